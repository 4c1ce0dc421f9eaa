"""How far the decoding operators' results are off as a whole: the 2-norm of the errors beside that
of the results.

The worst-case bounds of single elements (cache_helpers.attend_tol) take every rounding of a score's D
products at its worst and of one sign, and grow with D until fp32 results held in bf16 would pass.
Roundings of independent operands do not conspire: D of them, each of at most u = 2^-24 of a partial
sum that is no larger than |q * k|_2 in the root mean square, add up to sqrt(D) u |q * k|_2.
"""
import numpy as np

import cache_helpers as C

U = C.U32


def score_rms(Q, K, Kd, lens, scale=None):
    """[B][H][T]: root mean square error of a token's scores in fp32 arithmetic, of the largest
    |q * k|_2 of its keys; and of the exponentials' arguments, a few steps of the largest score."""
    B, H, T, D = Q.shape
    rep = H // K.shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else abs(scale)
    out = np.zeros((B, H, T))
    for b in range(B):
        for h in range(H):
            k = K[b, h // rep, :lens[b]]
            if Kd is not None:
                k = np.concatenate([k, Kd[b, h // rep]])
            k, q = k.astype(np.float64), Q[b, h].astype(np.float64)
            norm = np.sqrt(((q * q) @ (k * k).T).max(-1)) * scale
            top = np.abs(q @ k.T).max(-1) * scale
            out[b, h] = (np.sqrt(D) * norm + 8 * top) * U
    return out


def rms(x):
    return float(np.sqrt(np.mean(np.square(x, dtype=np.float64))))


def out_tol(dtype, rows, keys):
    """Relative, of the output's 2-norm: the scores' errors and their mean's (the sum of the
    weights), the sums over the keys and the last steps -- with values of random sign an error of
    the weights counts as much as the weights do; twice, for what a few rows deviate from the mean.
    bf16: the weights and the output rounded once each, half a step (2^-8) at most, evenly
    spread: 2^-8 / sqrt(3) each."""
    tol = 2 * (np.sqrt(2) * rms(rows) + (np.sqrt(keys) + 16) * U)
    return tol + (np.sqrt(2.0 / 3.0) * 2.0 ** -8 if dtype == "bf16" else 0.0)


def lse_tol(rows, keys, want):
    """Absolute, in the root mean square: a weighted mean of the scores' errors, the sum's, and the
    result's own steps.  The same for bf16: scores and sums are fp32."""
    return 2 * (rms(rows) + (np.sqrt(keys) + 16) * U) + 4 * U * rms(want)


def out_error(got, want):
    return float(np.linalg.norm((got - want).ravel()) / np.linalg.norm(want.ravel()))


def attend_accurate(dtype, got, got_lse, want, want_lse, rows, keys):
    """What attention gave for tokens that all count and attend something.  Returns the errors in
    tolerances."""
    out = out_error(got, want) / out_tol(dtype, rows, keys)
    lse = rms(got_lse - want_lse) / lse_tol(rows, keys, want_lse)
    assert out <= 1, f"output off by {out} tolerances"
    assert lse <= 1, f"lse off by {lse} tolerances"
    return out, lse


def weights_tol(rows, terms):
    """Relative, of the 2-norm of what was added: the scores' errors, the exponentials' steps and
    the sum's."""
    return 2 * (rms(rows) + (16 + np.sqrt(terms)) * U)
