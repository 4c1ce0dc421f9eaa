"""A serving program's run on the GPU: prompts that share a beginning enter a paged cache in parts,
then tokens follow one by one, every step an append with rotation, attention and an advance; the
same run over the contiguous cache and in float64."""
import numpy as np
import pytest

import cache_helpers as C
import paged_helpers as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [("f32", 64), ("bf16", 128), ("f32", 512), ("bf16", 640)])
@pytest.mark.parametrize("page", [16, 12])
def test_run(am, dev, dtype, D, page):
    import hip_rt
    rng = np.random.default_rng(4)
    B, H, G, rot, shared = 3, 4, 2, D // 2, 48
    prompts, steps = [70, 48, 91], [48, 30, 13, 1, 1, 1]  # tokens of a step; the first is the shared part
    pages, slots = 40, 12
    freq, amplitude = am.rope_frequencies(rot, scaling="parts", factor=8.0, original=64)
    rotary = am.Rotary(C.floats(freq), "half", rot, amplitude)
    K, V = (C.Tensor(np.full((pages, G, page, D), np.nan), dtype) for _ in range(2))
    order = rng.permutation(pages)
    whole = shared // page
    table = np.full((B, slots), -1, np.int32)
    table[:, :whole] = order[:whole]
    table[:, whole:] = order[whole:whole + B * (slots - whole)].reshape(B, -1)
    lens, tab = C.ints([0] * B), C.ints(table)
    cache = am.PagedCache(K.dev, V.dev, tab, lens)
    prefix = am.SharedPrefix(C.ints([0, B]), C.ints([shared]))
    s = hip_rt.Stream()
    first = rng.standard_normal((3, 1, H, shared, D))
    old_k, old_v = [[np.zeros((G, 0, D))] * B for _ in range(2)]
    at = [0] * B
    for step, T in enumerate(steps):
        # what is left of each prompt, then a token each
        counts = [min(T, prompts[b] - at[b]) if at[b] < prompts[b] else (1 if T == 1 else 0)
                  for b in range(B)]
        q, k, v = (rng.standard_normal((B, n, T, D)) for n in (H, G, G))
        if step == 0:  # the same tokens in all
            q, k, v = (np.tile(x[:, :n], (B, 1, 1, 1)) for x, n in zip(first, (H, G, G)))
        Q, Kd, Vd = (C.Tensor(x, dtype, order="rows") for x in (q, k, v))
        out = C.Tensor(np.full((B, H, T, D), 7.0), dtype, order="rows")
        lse = C.floats(np.full((B, H, T), 7.0))
        drafts = am.Drafts(Q.dev, Kd.dev, Vd.dev, count=C.ints(counts))
        append = am.paged_append_call(cache, drafts, rotary, q_out=Q.dev)
        attend = am.paged_attention_call(cache, drafts, out.dev, lse, max_len=128,
                                         prefix=prefix if step else None)
        if step == 0:  # (the shared pages are one sequence's to write)
            one = am.Drafts(Q.dev, Kd.dev, Vd.dev, count=C.ints([T, 0, 0]))
            am.paged_append_ex(cache, one, rotary, stream=s)
            rest = T - whole * page  # ... and each one's copy of the last page's rows
            s.synchronize()
            if rest:
                for x in (K, V):
                    y = x.numpy()
                    for b in range(1, B):
                        y[table[b, whole], :, :rest] = y[table[0, whole], :, :rest]
                    x.base.upload(x._flat(y))
            am.rotary_ex(rotary, [(Q.dev, Q.dev)], stream=s)
        else:
            append(s)
        attend(s)
        am.paged_advance_ex(cache, drafts, stream=s)
        s.synchronize()
        # the same in float64, from the turned and rounded queries and keys as the library holds them
        pos = np.array(at)[:, None] + np.arange(T)
        got_q, pools = Q.numpy(), [K.numpy(), V.numpy()]
        for x, host, where in ((got_q, Q.host, None), (pools[0], Kd.host, 1)):
            want, size = P.turned(host, pos, freq, True, rot, amplitude)
            tol = P.turned_tol(dtype, want, size, pos, freq, amplitude)
            for b in range(B):
                n = counts[b]
                g = x[b, :, :n] if where is None else \
                    P.rows_at(x, table, b, at[b] + n, page)[:, at[b]:]
                assert (np.abs(g - want[b, :, :n]) <= tol[b, :, :n]).all()
        for b in range(B):
            r = P.rows_at(pools[1], table, b, at[b] + counts[b], page)[:, at[b]:]
            assert np.array_equal(r, Vd.host[b, :, :counts[b]])
        Kc, Vc, Kn, Vn = (np.zeros((B, G, n, D)) for n in (max(at) + 1, max(at) + 1, T, T))
        for b in range(B):
            for pool, c, n in ((pools[0], Kc, Kn), (pools[1], Vc, Vn)):
                rows = P.rows_at(pool, table, b, at[b] + counts[b], page)
                c[b, :, :at[b]], n[b, :, :counts[b]] = rows[:, :at[b]], rows[:, at[b]:]
        want, wl, info = C.attend64(got_q, Kc, Vc, Kn, Vn, at, counts)
        got, got_lse = out.numpy(), lse.numpy()
        C.attend_close(dtype, D, got, got_lse, want, wl, info, counts)
        # ... and by the library over a contiguous cache
        lay = [C.Tensor(x, dtype) for x in (Kc, Vc, Kn, Vn)]
        tree_out, tree_lse = C.Tensor(np.full((B, H, T, D), 7.0), dtype), C.floats(np.zeros((B, H, T)))
        td = am.Drafts(Q.dev, lay[2].dev, lay[3].dev, count=drafts.count)
        am.tree_attention_ex(am.KvCache(lay[0].dev, lay[1].dev, C.ints(at)), td, tree_out.dev, tree_lse)
        C.attend_close(dtype, D, tree_out.numpy(), tree_lse.numpy(), want, wl, info, counts)
        at = [a + n for a, n in zip(at, counts)]
        assert lens.numpy().tolist() == at
    assert at == [73, 51, 94]
    s.destroy()


@pytest.mark.parametrize("dtype,D,T", [("bf16", 128, 1), ("bf16", 64, 40), ("f32", 80, 3), ("f32", 512, 2)])
def test_captured_steps(am, dev, dtype, D, T):
    """Append, attention and advance in one graph, replayed with other tokens, counts and tables between
    the replays, beside the same program run eagerly on another stream: the same bits."""
    import hip_rt
    B, H, G, page, slots, pages = 3, 4, 2, 16, 64, 150
    freq, _ = am.rope_frequencies(D)
    rng = np.random.default_rng(8)
    order = rng.permutation(pages)
    start, shared = [540, 530, 560], 512
    rows = rng.standard_normal((2, pages, G, page, D))

    class Program:
        def __init__(self):
            self.K, self.V = (C.Tensor(x, dtype) for x in rows)
            self.table = np.full((B, slots), -1, np.int32)
            self.table[:, :32] = order[:32]
            self.table[:, 32:62] = order[32:122].reshape(B, 30)
            self.tab, self.lens = C.ints(self.table), C.ints(start)
            cache = am.PagedCache(self.K.dev, self.V.dev, self.tab, self.lens)
            self.Q, self.Kd, self.Vd = (C.Tensor(np.zeros((B, n, T, D)), dtype, order="rows")
                                        for n in (H, G, G))
            self.count = C.ints([T] * B)
            self.out = C.Tensor(np.full((B, H, T, D), 7.0), dtype, order="rows")
            self.lse = C.floats(np.full((B, H, T), 7.0))
            drafts = am.Drafts(self.Q.dev, self.Kd.dev, self.Vd.dev, count=self.count)
            rotary = am.Rotary(C.floats(freq), "half", D)
            prefix = am.SharedPrefix(C.ints([0, B]), C.ints([shared]))
            self.calls = [am.paged_append_call(cache, drafts, rotary, q_out=self.Q.dev),
                          am.paged_attention_call(cache, drafts, self.out.dev, self.lse, prefix=prefix),
                          am.paged_advance_call(cache, drafts)]
            self.stream = hip_rt.Stream()

        def step(self):
            for call in self.calls:
                call(self.stream)

        def put(self, q, k, v, counts):
            for x, y in ((self.Q, q), (self.Kd, k), (self.Vd, v)):
                x.base.upload(x._flat(y.astype(np.float32)))
            self.count.upload(np.array(counts))

    a, b = Program(), Program()
    b.step()  # (the stream's workspace has to be there before the capture)
    b.stream.synchronize()
    for x, y in zip((b.K, b.V), rows):
        x.base.upload(x._flat(y.astype(np.float32)))
    b.lens.upload(np.array(start))
    graph = hip_rt.Graph(b.stream, b.step)
    at = list(start)
    for i in range(5):
        q, k, v = (rng.standard_normal((B, n, T, D)) for n in (H, G, G))
        counts = [T, (T + i) % (T + 1), max(0, T - i)]
        if i == 3:  # a page of each moves elsewhere
            for p in (a, b):
                for x in (p.K, p.V):
                    y = x.numpy()
                    y[order[122:125]] = y[p.table[:, 33]]
                    x.base.upload(x._flat(y))
                p.table[:, 33] = order[122:125]
                p.tab.upload(p.table)
        for p in (a, b):
            p.put(q, k, v, counts)
        a.step()
        graph.launch()
        for p in (a, b):
            p.stream.synchronize()
        at = [x + n for x, n in zip(at, counts)]
        assert a.lens.numpy().tolist() == b.lens.numpy().tolist() == at
        for x, y in ((a.K, b.K), (a.V, b.V), (a.out, b.out), (a.Q, b.Q)):
            assert np.array_equal(x.base.bits(), y.base.bits())
        assert np.array_equal(a.lse.bits(), b.lse.bits())
        # ... and they are what they should be
        old = [n - m for n, m in zip(at, counts)]
        Kc, Vc, Kn, Vn = (np.zeros((B, G, n, D)) for n in (max(old), max(old), T, T))
        for pool, c, n in ((b.K.numpy(), Kc, Kn), (b.V.numpy(), Vc, Vn)):
            for s in range(B):
                r = P.rows_at(pool, b.table, s, at[s], page)
                c[s, :, :old[s]], n[s, :, :counts[s]] = r[:, :old[s]], r[:, old[s]:]
        want, wl, info = C.attend64(b.Q.numpy(), Kc, Vc, Kn, Vn, old, counts)
        got, got_lse = b.out.numpy(), b.lse.numpy()
        C.attend_close(dtype, D, got, got_lse, want, wl, info, counts)
    graph.destroy()
    for p in (a, b):
        p.stream.destroy()
