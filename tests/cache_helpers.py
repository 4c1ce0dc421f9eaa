"""Inputs, float64 definitions and tolerances of the decoding operators' tests."""
import numpy as np

U32 = 2.0 ** -24              # half a step of fp32, relative
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
LOG2E = 1.4426950408889634


def rounded(x, dtype):
    """x as the device holds it."""
    import hip_rt
    x = np.asarray(x, dtype=np.float32)
    return x if dtype == "f32" else hip_rt.bf16_bits_to_f32(hip_rt.f32_to_bf16_bits(x))


class Tensor:
    """A [B][heads][rows][D] tensor on the device in one of two memory orders ("heads":
    [B][heads][rows][D]; "rows": [B][rows][heads][D]), starting `offset` elements into its buffer,
    rows `pad` elements longer than D; `host` is its content.  What lies between rows is NaN."""

    def __init__(self, x, dtype, order="heads", offset=0, pad=0):
        import hip_rt
        self.dtype, self.order, self.offset = dtype, order, offset
        self.host = rounded(x, dtype)
        B, Hh, R, D = x.shape
        ld = D + pad
        self.phys = (B, Hh, R, ld) if order == "heads" else (B, R, Hh, ld)
        self.base = hip_rt.DeviceArray.from_numpy(self._flat(self.host), dtype)
        s = (Hh * R * ld, R * ld, ld, 1) if order == "heads" else (Hh * R * ld, ld, Hh * ld, 1)
        self.dev = hip_rt.DeviceArray.wrap(self.base.ptr + offset * self.base.itemsize, x.shape,
                                           dtype, strides=s, keep=self.base)

    def _flat(self, x):
        full = np.full(self.phys, np.nan, np.float32)
        full[..., :x.shape[3]] = x if self.order == "heads" else x.transpose(0, 2, 1, 3)
        return np.concatenate([np.full(self.offset, np.nan, np.float32), full.ravel()])

    def numpy(self):
        """The content now; what lies around it must still be what it was."""
        flat = self.base.numpy()
        D = self.dev.shape[3]
        full = flat[self.offset:].reshape(self.phys)
        assert np.isnan(flat[:self.offset]).all() and np.isnan(full[..., D:]).all()
        x = full[..., :D]
        return np.ascontiguousarray(x if self.order == "heads" else x.transpose(0, 2, 1, 3))


def ints(x):
    import hip_rt
    return hip_rt.DeviceArray.from_numpy(np.asarray(x), "i32")


def floats(x):
    import hip_rt
    return hip_rt.DeviceArray.from_numpy(np.asarray(x, dtype=np.float32), "f32")


def visible(T, count, mask_words, b):
    """[T][T] bool: draft t attends draft j."""
    t = np.arange(T)
    see = t[:, None] >= t[None] if mask_words is None else \
        ((mask_words[b][:, t // 32] >> (t % 32)) & 1).astype(bool)
    return see & (t < count)[None]


def attend64(Q, K, V, Kd, Vd, lens, counts, mask_words=None, scale=None):
    """The definition in float64.  Returns out, lse and, for tolerances, per element: the sum
    of p |v|, and per row: the largest sum of |q k| scale, the largest |score| and the keys."""
    B, H, T, D = Q.shape
    G = K.shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out = np.zeros((B, H, T, D))
    pv = np.zeros((B, H, T, D))
    lse = np.full((B, H, T), -np.inf)
    sabs, smax, keys = np.zeros((B, H, T)), np.zeros((B, H, T)), np.zeros((B, H, T))
    for b in range(B):
        L, n = lens[b], counts[b]
        see = visible(T, n, mask_words, b)
        for h in range(H):
            g = h // (H // G)
            kc, vc = K[b, g, :L].astype(np.float64), V[b, g, :L].astype(np.float64)
            for t in range(n):
                on = see[t] if Kd is not None else np.zeros(T, bool)
                k = np.concatenate([kc, Kd[b, g][on].astype(np.float64)]) if on.any() else kc
                v = np.concatenate([vc, Vd[b, g][on].astype(np.float64)]) if on.any() else vc
                if len(k) == 0:
                    continue
                q = Q[b, h, t].astype(np.float64)
                s = k @ q * scale
                m = s.max()
                if m == -np.inf:
                    continue
                e = np.exp(s - m)
                l = e.sum()
                out[b, h, t] = e @ v / l
                pv[b, h, t] = e @ np.abs(v) / l
                lse[b, h, t] = m + np.log(l)
                sabs[b, h, t] = (np.abs(k) @ np.abs(q)).max() * abs(scale)
                smax[b, h, t] = np.abs(s).max()
                keys[b, h, t] = len(k)
    return out, lse, dict(pv=pv, sabs=sabs, smax=smax, keys=keys)


def score_error(D, info):
    """Bound of a score's absolute error: D products summed in fp32 in some order (fp32 inputs:
    each product rounded once; a term passes at most D additions), the multiplication by the scale
    (itself rounded) and by log2(e), and the rounding of differences of scores."""
    return (D + 4) * U32 * info["sabs"] + 8 * U32 * info["smax"]


def attend_tol(dtype, D, out, info):
    """Absolute tolerances of out and lse: each weight is off by a factor of exp(2 score errors)
    (its own and the maximum's) and the exponential's own few steps, sums of `keys` terms by keys
    steps, twice (numerator, denominator); bf16 rounds the weights in the product with V once
    and the output once."""
    d = score_error(D, info)
    w = np.expm1(2 * d) + (16 + 2 * info["keys"]) * U32 + (HALF["bf16"] if dtype == "bf16" else 0.0)
    tol = w[..., None] * info["pv"] * 1.01 + HALF[dtype] * np.abs(out) + 1e-30
    with np.errstate(invalid="ignore"):
        lse = 2 * d + (16 + info["keys"]) * U32
    return tol, lse


def attend_close(dtype, D, got, got_lse, want, want_lse, info, counts):
    tol, tol_lse = attend_tol(dtype, D, want, info)
    for b, n in enumerate(counts):
        err = np.abs(got[b, :, :n] - want[b, :, :n])
        bad = ~(err <= tol[b, :, :n])
        assert not bad.any(), (f"sequence {b}: {bad.sum()} of {bad.size} off, worst "
                               f"{np.nanmax(err / tol[b, :, :n])} tolerances at "
                               f"{np.argwhere(bad)[:4].tolist()}")
        if got_lse is not None:
            w, x = want_lse[b, :, :n], got_lse[b, :, :n]
            assert np.array_equal(np.isneginf(w), np.isneginf(x))
            f = np.isfinite(w)
            assert (np.abs(x[f] - w[f]) <= tol_lse[b, :, :n][f] + U32 * 4 * np.abs(w[f])).all()


def accepted_rows(path, accepted, counts, lens, cap, path_len):
    """Rows that commit writes, of each sequence."""
    out = []
    for b, n in enumerate(counts):
        a = path_len if accepted is None else min(max(accepted[b], 0), path_len)
        if path is None:
            a = min(a, n)
        else:
            bad = [i for i in range(a) if not 0 <= path[b][i] < n]
            a = bad[0] if bad else a
        out.append(min(a, cap - lens[b]))
    return out


def evict_moves(weight, pos, L, seen, budget, recent):
    """(to, from) of one head by the definition: recent rows first, the lower ones where there are
    more than the budget, then by weight, NaN last, the lower row of equal ones."""
    if L <= budget:
        return []

    def rank_of(r):
        old = int(pos[r]) < int(seen) - recent
        nan = old and np.isnan(weight[r])
        return old, nan, -float(weight[r]) if old and not nan else 0.0, r

    rank = sorted(range(L), key=rank_of)
    keep = set(rank[:budget])
    to = [r for r in range(budget) if r not in keep]
    frm = sorted(r for r in keep if r >= budget)
    return list(zip(to, frm))
