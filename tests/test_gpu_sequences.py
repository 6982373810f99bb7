"""Attention over a batch of sequences (paged caches, packed prompts) and the paged append, against
the formula in 64 bits.

Tolerances, per output value with A = sum p |v| / sum p (64 bits) and N = |q| |k| (largest over the
row's keys), from the roundings that the kernels make:
  scores    products are exact, 16 of them are added at a time, hd / 16 additions into f32 (twice
            with the split queries): each off by at most 2^-23 N, the exponent's fma by another
            2^-23 of a value below N; p then moves by at most that much relative, and the sum of p
            likewise: 2 (hd / 8 + 2) 2^-23 N A
  p         one rounding to f16 (2^-11) or bf16 (2^-8), or the split's 2^-22 for f32: times A; its
            exponential 2^-22 A, twice; f32 sums over len keys in at most len / 16 + 64 additions
            of 2^-24 each, twice
  out       one rounding to the output type
A tanh score adds 2^-20 softcap, once for each of p and its sum.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
P_EPS = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def env():
    import torch
    import rust_interference_engine_b200 as rie
    return torch, rie, rie.Context(0, torch.cuda.current_stream())


def dtype(torch, t):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def ref_row(q, k, v, softcap):
    """One query over its attended keys in 64 bits: (out, A, N)."""
    s = k @ q
    if softcap:
        s = softcap * np.tanh(s / softcap)
    p = np.exp(s - s.max())
    return p @ v / p.sum(), p @ np.abs(v) / p.sum(), np.linalg.norm(q) * np.linalg.norm(k, axis=1).max()


def check_rows(got, q, ks, vs, spans, n_head, n_kv, hd, window, softcap, ty):
    """got, q: rows [n_tok][n_head * hd]; ks / vs: per sequence [len][n_kv][hd]; spans: (first row,
    new tokens, len)."""
    G = n_head // n_kv
    for i, (first, n, length) in enumerate(spans):
        for t in range(n):
            pos = length - n + t
            lo = max(0, pos + 1 - window) if window else 0
            for h in range(n_head):
                kk, vv = ks[i][lo:pos + 1, h // G], vs[i][lo:pos + 1, h // G]
                want, A, N = ref_row(q[first + t, h * hd:(h + 1) * hd], kk, vv, softcap)
                x = got[first + t, h * hd:(h + 1) * hd]
                rel = (2 * (hd / 8 + 2) * 2.0 ** -23 * N + P_EPS[ty] + 2 * 2.0 ** -22
                       + 2 * ((pos + 1 - lo) / 16 + 64) * 2.0 ** -24 + (2 * 2.0 ** -20 * softcap if softcap else 0))
                tol = rel * A * (1 + 2.0 ** -7) + EPS[ty] * np.abs(want) + 2.0 ** -24
                bad = ~(np.abs(x - want) <= tol)
                assert not bad.any(), (i, t, h, np.abs(x - want).max(), tol[bad][:3], x[bad][:3], want[bad][:3])


class Case:
    """Sequences in a pool of pages whose other places hold NaN."""

    def __init__(self, torch, rie, ctx, seqs, n_head, n_kv, hd, ps, ty, seed=0, tail=3, scale=2.0):
        rng = np.random.default_rng(seed)
        self.seqs, self.n_head, self.n_kv, self.hd, self.ps, self.ty = seqs, n_head, n_kv, hd, ps, ty
        self.ks = [rng.standard_normal((n, n_kv, hd)).astype(np.float16).astype(np.float64) for _, n in seqs]
        self.vs = [rng.standard_normal((n, n_kv, hd)).astype(np.float16).astype(np.float64) for _, n in seqs]
        need = [-(-n // ps) for _, n in seqs]
        n_pages, width = sum(need) + 3, max(max(need), 1) + 1
        order = rng.permutation(n_pages)
        self.pages = np.full((len(seqs), width), -7, dtype=np.int32)  # unused entries are never followed
        kp = np.full((n_pages, n_kv, ps, hd), np.nan, dtype=np.float16)
        vp = np.full((n_pages, n_kv, ps, hd), np.nan, dtype=np.float16)
        at = 0
        for i, (_, n) in enumerate(seqs):
            mine = order[at:at + need[i]]
            at += need[i]
            self.pages[i, :need[i]] = mine
            for p in range(n):
                kp[mine[p // ps], :, p % ps] = self.ks[i][p]
                vp[mine[p // ps], :, p % ps] = self.vs[i][p]
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.n_tok = int(self.cu[-1]) + tail
        self.q = torch.from_numpy(rng.standard_normal((self.n_tok, n_head * hd)) * (scale / np.sqrt(hd))).to(dtype(torch, ty)).cuda()
        self.k_pool, self.v_pool = torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda()
        self.cache = rie.PagedCache(ctx, n_kv, hd, ps, n_pages, k=self.k_pool, v=self.v_pool)
        self.dev = [torch.from_numpy(x).cuda() for x in (self.cu, np.array([n for _, n in seqs], dtype=np.int32), self.pages)]
        self.torch, self.rie, self.ctx = torch, rie, ctx

    def batch(self, max_len=0):
        return self.rie.SeqBatch(*self.dev, self.n_tok, max_len=max_len)

    def spans(self):
        return [(int(self.cu[i]), n, length) for i, (n, length) in enumerate(self.seqs)]

    def run(self, window=0, softcap=0.0, max_len=0):
        out = self.torch.full_like(self.q, 7.5)
        self.rie.paged_attention(self.ctx, self.cache, self.batch(max_len), self.q, self.n_head, out, window=window, softcap=softcap)
        self.ctx.sync()
        return out

    def check(self, out, window=0, softcap=0.0):
        got = out.double().cpu().numpy()
        check_rows(got, self.q.double().cpu().numpy(), self.ks, self.vs, self.spans(), self.n_head, self.n_kv, self.hd, window, softcap, self.ty)
        assert (got[int(self.cu[-1]):] == 7.5).all()  # rows behind the last sequence


MIXED = [(1, 1), (1, 16), (1, 17), (0, 9), (3, 3), (5, 64), (37, 100), (1, 333), (0, 0), (2, 130)]


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("n_head,n_kv,hd,ps", [(4, 4, 64, 16), (6, 2, 128, 64), (4, 1, 96, 32), (7, 1, 128, 16), (16, 2, 32, 128),
                                               (2, 1, 256, 64), (24, 1, 64, 256), (40, 1, 128, 1024)])
def test_paged_mixed(env, ty, n_head, n_kv, hd, ps):
    c = Case(*env, MIXED, n_head, n_kv, hd, ps, ty)
    c.check(c.run())


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (7, 0.0), (16, 20.0), (64, 0.0), (1000, 5.0), (0, 30.0)])
def test_paged_window_and_softcap(env, ty, window, softcap):
    c = Case(*env, MIXED, 8, 2, 128, 16, ty, seed=1)
    c.check(c.run(window, softcap), window, softcap)


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("seqs", [[(1, 2500)], [(1, 4097), (1, 31)], [(2, 3000)], [(130, 700)], [(200, 1500), (1, 900), (65, 65)]])
def test_paged_long_axis_is_split(env, ty, seqs):
    """Few rows over a long context share a tile between CTAs; chunks cross tile borders."""
    c = Case(*env, seqs, 4, 2, 128, 64, ty, seed=2)
    for max_len in (0, max(n for _, n in seqs), 1):
        c.check(c.run(max_len=max_len))


@pytest.mark.parametrize("n_head,n_kv,hd,n", [(8, 2, 128, 257), (4, 4, 64, 300), (14, 2, 128, 150), (6, 1, 96, 129), (3, 1, 256, 140)])
@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_paged_chunks(env, ty, n_head, n_kv, hd, n):
    c = Case(*env, [(n, n + 500), (n // 2, n // 2), (1, 77)], n_head, n_kv, hd, 32, ty, seed=3)
    c.check(c.run())
    c.check(c.run(window=100), window=100)


@pytest.mark.parametrize("scale", [1e-4, 3000.0])
def test_f32_queries_of_any_size(env, scale):
    """f32 queries far below and above f16's range."""
    c = Case(*env, [(1, 400), (40, 90)], 4, 2, 64, 16, "f32", seed=4, scale=scale)
    c.q[:, :64] *= 1e-3
    c.q[1, 0] = 7e4
    c.check(c.run())


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("n", [20, 200])
def test_masked_infinities_do_not_count(env, ty, n):
    """A later token's values are infinite or NaN: the tokens before it must not see them, the
    tokens from it on follow the formula."""
    torch, rie, ctx = env
    c = Case(torch, rie, ctx, [(n, n + 50)], 4, 2, 128, 16, ty, seed=5)
    bad = n + 50 - n // 2
    pg, slot = int(c.pages[0, bad // 16]), bad % 16
    c.v_pool[pg, :, slot] = float("inf")
    c.v_pool[pg, 1, slot, 3] = float("nan")
    out = c.run().double().cpu().numpy()
    t0 = bad - 50
    G = 2
    for t in range(n):
        for h in range(4):
            x = out[t, h * 128:(h + 1) * 128]
            if t < t0:
                want, A, N = ref_row(c.q[t, h * 128:(h + 1) * 128].double().cpu().numpy(), c.ks[0][:51 + t, h // G], c.vs[0][:51 + t, h // G], 0)
                assert np.isfinite(x).all() and np.abs(x - want).max() <= 2.0 ** -8
            else:
                nan = np.zeros(128, bool)
                nan[3] = h // G == 1
                assert (np.isnan(x) == nan).all() and (x[~nan] == np.inf).all()
    # a NaN key makes the rows that attend it NaN, and no others
    c = Case(torch, rie, ctx, [(n, n + 50)], 4, 2, 128, 16, ty, seed=6)
    c.k_pool[int(c.pages[0, bad // 16]), :, slot] = float("nan")
    out = c.run().double().cpu().numpy()[:n]
    assert np.isfinite(out[:t0]).all() and np.isnan(out[t0:]).all()


def test_strided_rows(env):
    """q, out and the appended k / v are slices of wider rows."""
    torch, rie, ctx = env
    c = Case(torch, rie, ctx, MIXED, 4, 2, 64, 16, "f32", seed=7)
    wide_q = torch.randn(c.n_tok, 4 * 64 + 2 * 2 * 64, device="cuda")
    wide_q[:, :256] = c.q
    wide_o = torch.full((c.n_tok, 512), 7.5, device="cuda")
    rie.paged_attention(ctx, c.cache, c.batch(), wide_q[:, :256], 4, wide_o[:, 128:384])
    ctx.sync()
    c.check(wide_o[:, 128:384])
    assert (wide_o[:, :128] == 7.5).all() and (wide_o[:, 384:] == 7.5).all()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,hd,ps", [(2, 64, 16), (1, 32, 64), (8, 128, 32), (3, 96, 16), (5, 256, 16)])
def test_store(env, ty, n_kv, hd, ps):
    torch, rie, ctx = env
    c = Case(torch, rie, ctx, MIXED + [(1, 1)] * 40 + [(33, 80)], n_kv, n_kv, hd, ps, "f16", seed=8)
    wide = (torch.randn(c.n_tok, 2 * n_kv * hd + 64, device="cuda") * 3).to(dtype(torch, ty))
    k, v = wide[:, :n_kv * hd], wide[:, n_kv * hd:2 * n_kv * hd]
    want_k, want_v = c.k_pool.clone(), c.v_pool.clone()
    c.cache.store(c.batch(), k, v)
    ctx.sync()
    for i, (first, n, length) in enumerate(c.spans()):
        for t in range(n):
            p = length - n + t
            pg = int(c.pages[i, p // ps])
            want_k[pg, :, p % ps] = k[first + t].view(n_kv, hd).half()
            want_v[pg, :, p % ps] = v[first + t].view(n_kv, hd).half()
    for got, want in ((c.k_pool, want_k), (c.v_pool, want_v)):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))  # NaN elsewhere, untouched


@pytest.mark.parametrize("ty,kv", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("n_head,n_kv,hd,lens", [(4, 2, 64, [37]), (4, 4, 128, [1, 16, 0, 17, 128, 129, 3]), (14, 2, 128, [70, 260]),
                                                 (6, 2, 96, [33, 200]), (2, 1, 256, [5, 150]), (8, 1, 32, [64, 1, 1, 90]),
                                                 (8, 2, 128, [600, 31])])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (20, 0.0), (0, 15.0)])
def test_packed(env, ty, kv, n_head, n_kv, hd, lens, window, softcap):
    torch, rie, ctx = env
    rng = np.random.default_rng(9)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n_tok = int(cu[-1]) + 5
    wide = torch.from_numpy(rng.standard_normal((n_tok, 2 * n_kv * hd))).to(dtype(torch, kv)).cuda()
    k, v = wide[:, :n_kv * hd], wide[:, n_kv * hd:]  # slices of one projection
    wide[int(cu[-1]):] = float("nan")
    q = torch.from_numpy(rng.standard_normal((n_tok, n_head * hd)) * 2 / np.sqrt(hd)).to(dtype(torch, ty)).cuda()
    out = torch.full_like(q, 7.5)
    rie.packed_attention(ctx, q, k, v, torch.from_numpy(cu).cuda(), n_head, n_kv, hd, out, window=window, softcap=softcap)
    ctx.sync()
    got = out.double().cpu().numpy()
    ks = [k[a:b].double().cpu().numpy().reshape(-1, n_kv, hd) for a, b in zip(cu, cu[1:])]
    vs = [v[a:b].double().cpu().numpy().reshape(-1, n_kv, hd) for a, b in zip(cu, cu[1:])]
    check_rows(got, q.double().cpu().numpy(), ks, vs, [(int(a), n, n) for a, n in zip(cu, lens)], n_head, n_kv, hd, window, softcap, ty)
    assert (got[int(cu[-1]):] == 7.5).all()


def test_packed_prompt_next_to_infinities(env):
    """The rows behind a prompt belong to the next one, whose values may be anything."""
    torch, rie, ctx = env
    lens, hd = [21, 40], 64
    cu = torch.tensor([0, 21, 61], dtype=torch.int32, device="cuda")
    q = torch.randn(61, 2 * hd, device="cuda").half() / 8
    k, v = torch.randn(61, hd, device="cuda").half(), torch.randn(61, hd, device="cuda").half()
    out = torch.zeros_like(q)
    rie.packed_attention(ctx, q, k, v, cu, 2, 1, hd, out)
    v2, out2 = v.clone(), torch.zeros_like(q)
    v2[21:] = float("inf")
    rie.packed_attention(ctx, q, k, v2, cu, 2, 1, hd, out2)
    ctx.sync()
    assert torch.isfinite(out2[:21]).all()
    assert (out2[:21].float() - out[:21].float()).abs().max() <= 2.0 ** -9 * 4
    assert torch.isinf(out2[21:]).all()


@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_bad_device_data_is_reported(env, ty):
    """Page numbers outside the pool, lengths beyond the table or below the new tokens, offsets
    that fall: nothing is followed, the next sync says so, and the context works on."""
    torch, rie, ctx = env

    def broken(change, store=False):
        c = Case(torch, rie, ctx, [(1, 40), (3, 70), (100, 140)], 4, 2, 64, 16, ty, seed=10)
        change(c.dev)
        out = torch.zeros_like(c.q)
        if store:
            kv = torch.zeros(c.n_tok, 128, device="cuda")
            c.cache.store(c.batch(), kv, kv)
        else:
            rie.paged_attention(ctx, c.cache, c.batch(), c.q, 4, out)
        with pytest.raises(rie.RcuError, match="0x8"):
            ctx.sync()

    def page(v):
        def f(dev):
            dev[2][1, 4] = v
        return f

    def length(v):
        def f(dev):
            dev[1][1] = v
        return f

    def offset(i, v):
        def f(dev):
            dev[0][i] = v
        return f

    for store in (False, True):
        for change in (page(-1), page(1 << 20), length(1 << 30), length(1), length(-5), offset(1, 1 << 29), offset(2, 0)):
            broken(change, store)
    ctx.sync()
    c = Case(torch, rie, ctx, MIXED, 4, 2, 64, 16, ty, seed=11)
    c.check(c.run())


def test_captured_graph_follows_the_batch(env):
    """Append and attention captured once; replayed with other lengths, pages and rows."""
    torch, rie, _ = env
    s = torch.cuda.Stream()
    ctx = rie.Context(0, s)
    a = Case(torch, rie, ctx, [(1, 30), (1, 500), (1, 77)], 8, 2, 128, 16, "f32", seed=12, tail=0)
    b = Case(torch, rie, ctx, [(1, 31), (1, 501), (1, 78)], 8, 2, 128, 16, "f32", seed=13, tail=0)
    k = torch.zeros(3, 256, device="cuda")
    v = torch.zeros(3, 256, device="cuda")
    out = torch.zeros_like(a.q)
    torch.cuda.synchronize()

    def step():
        a.cache.store(a.batch(512), k, v)
        rie.paged_attention(ctx, a.cache, a.batch(512), a.q, 8, out)

    with torch.cuda.stream(s):
        step()
        ctx.sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    for c in (a, b):  # b's pool, lengths, pages and queries take a's place
        with torch.cuda.stream(s):
            if c is b:
                assert b.k_pool.numel() == a.k_pool.numel() and b.dev[2].shape == a.dev[2].shape
                a.k_pool.copy_(b.k_pool)
                a.v_pool.copy_(b.v_pool)
                a.q.copy_(b.q)
                for x, y in zip(a.dev, b.dev):
                    x.copy_(y)
            k.copy_(torch.from_numpy(np.stack([ks[-1].reshape(-1) for ks in c.ks])))
            v.copy_(torch.from_numpy(np.stack([vs[-1].reshape(-1) for vs in c.vs])))
            g.replay()
        ctx.sync()
        check_rows(out.double().cpu().numpy(), c.q.double().cpu().numpy(), c.ks, c.vs, c.spans(), 8, 2, 128, 0, 0.0, "f32")
    del g


def test_calls_on_two_streams_do_not_share_anything(env):
    torch, rie, _ = env
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [rie.Context(0, s) for s in streams]
    cases = [Case(torch, rie, c, [(1, 3000 + i), (30, 200)], 8, 2, 128, 64, "f16", seed=14 + i) for i, c in enumerate(ctxs)]
    torch.cuda.synchronize()
    outs = [[torch.full_like(c.q, 7.5) for _ in range(20)] for c in cases]
    torch.cuda.synchronize()
    for j in range(20):
        for c, o in zip(cases, outs):
            rie.paged_attention(c.ctx, c.cache, c.batch(), c.q, 8, o[j])
    for c, o in zip(cases, outs):
        c.ctx.sync()
        c.check(o[0])
        for x in o[1:]:
            assert torch.equal(x, o[0])  # the same bits every time


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("hd", [160, 224])
def test_head_dims_between(env, ty, hd):
    c = Case(*env, [(1, 70), (9, 33), (40, 80)], 4, 2, hd, 16, ty, seed=20)
    c.check(c.run())


@pytest.mark.parametrize("new", [1, 2])
def test_hundreds_of_sequences(env, new):
    """The lookup of a tile's sequence goes over many groups of 32, empty sequences among them."""
    seqs = [(new if i % 7 else 0, 3 + (i * 37) % 90) for i in range(333)]
    c = Case(*env, seqs, 4, 2, 64, 16, "f16", seed=21)
    c.check(c.run())
    c.check(c.run(max_len=100))


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("window", [0, 300, 1500])
def test_chunk_split_over_a_cluster(env, ty, window):
    """A chunk late in a long context: its keys are split, windows leave some parts without any."""
    c = Case(*env, [(70, 6000)], 4, 1, 128, 64, ty, seed=22)
    c.check(c.run(window), window)
    c.check(c.run(window, 25.0), window, 25.0)


@pytest.mark.parametrize("max_new", [0, 1, 12, 500])
def test_max_new_shapes_the_launch_only(env, max_new):
    """A wrong max_new chooses another kernel, with the same result."""
    torch, rie, ctx = env
    c = Case(torch, rie, ctx, [(12, 90), (1, 400), (500, 500), (3, 17)], 8, 2, 128, 32, "f16", seed=23)
    out = torch.full_like(c.q, 7.5)
    rie.paged_attention(ctx, c.cache, rie.SeqBatch(*c.dev, c.n_tok, max_new=max_new), c.q, 8, out)
    ctx.sync()
    c.check(out)


@pytest.mark.parametrize("n", [17, 300])
def test_nan_and_infinite_queries(env, n):
    """A query that is not finite makes its own row NaN, and no other."""
    torch, rie, ctx = env
    for ty in ("f32", "f16"):
        c = Case(torch, rie, ctx, [(n, n + 20)], 4, 2, 128, 16, ty, seed=24)
        want = c.run()
        c.q[3, 128 + 5] = float("nan")
        c.q[7, 5] = float("inf")
        out = c.run()
        bad = torch.zeros(c.n_tok, 4, dtype=torch.bool)
        bad[3, 1] = bad[7, 0] = True
        rows = out.view(c.n_tok, 4, 128).cpu()
        assert torch.isnan(rows[bad]).all()
        assert torch.equal(rows[~bad], want.view(c.n_tok, 4, 128).cpu()[~bad])


def test_pages_shared_by_two_sequences(env):
    """A common prefix in the same pages, and the same page twice in a table."""
    torch, rie, ctx = env
    c = Case(torch, rie, ctx, [(1, 64), (1, 64)], 4, 2, 64, 16, "f16", seed=25)
    c.dev[2][1, :3] = c.dev[2][0, :3]
    c.dev[2][1, 1] = c.dev[2][0, 0]
    for x in (c.ks, c.vs):
        x[1][:48] = x[0][:48]
        x[1][16:32] = x[0][:16]
    c.check(c.run())


def test_owned_pool_starts_zeroed_and_serves(env):
    """Pages of the library's own; append, then attention, step by step next to one LayerCache a
    sequence: two f32 attentions over the same f16 rows."""
    torch, rie, ctx = env
    n_head, n_kv, hd, ps, n_pages = 8, 2, 128, 16, 40
    cache = rie.PagedCache(ctx, n_kv, hd, ps, n_pages)
    k_ptr, v_ptr = cache.data_ptrs()
    assert k_ptr and v_ptr and k_ptr != v_ptr
    lens = [0, 0, 0]
    flat = [rie.LayerCache(ctx, rie.KvType.F16, n_kv, hd, 256) for _ in lens]
    pages = torch.arange(30, dtype=torch.int32, device="cuda").reshape(10, 3).t().contiguous()
    g = torch.Generator(device="cuda").manual_seed(26)
    for new in ([50, 3, 17], [1, 1, 1], [1, 0, 1], [20, 1, 2], [1, 1, 1]):
        n = sum(new)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        lens = [a + b for a, b in zip(lens, new)]
        batch = rie.SeqBatch(cu, torch.tensor(lens, dtype=torch.int32, device="cuda"), pages, n, max_len=max(lens))
        q, k, v = (torch.randn(n, h * hd, generator=g, device="cuda") * s for h, s in ((n_head, hd ** -0.5), (n_kv, 1), (n_kv, 1)))
        out, want = torch.zeros_like(q), torch.zeros_like(q)
        cache.store(batch, k, v)
        rie.paged_attention(ctx, cache, batch, q, n_head, out)
        at = 0
        for c, length, m in zip(flat, lens, new):
            if m:
                c.store(k[at:at + m], v[at:at + m], m, length - m)
                rie.attention(ctx, c, q[at:at + m], m, n_head, length - m, want[at:at + m])
            at += m
        ctx.sync()
        # both are the same sums in f32, in another order: 2^-20 of values below 4 (the split parts carry 2^-22)
        assert (out - want).abs().max().item() <= 4 * 2.0 ** -18


@pytest.mark.parametrize("hd", [160, 256])
@pytest.mark.parametrize("window", [0, 700])
def test_wide_heads_in_chunks(env, hd, window):
    """16-bit queries of head_dim above 128: one tile a CTA, keys split over a cluster or not."""
    c = Case(*env, [(60, 3000)], 4, 1, hd, 64, "f16", seed=27)
    c.check(c.run(window), window)
    c = Case(*env, [(100, 300), (1, 50), (33, 33)], 6, 2, hd, 16, "f16", seed=28)
    c.check(c.run(window, 20.0), window, 20.0)


@pytest.mark.parametrize("hd", [160, 224, 256])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (700, 0.0), (0, 20.0)])
def test_wide_heads_of_f32_queries(env, hd, window, softcap):
    """f32 queries of head_dim above 128 in chunks: keys split over a cluster or not, rows that are part of a tile."""
    for seqs, n_head, n_kv, ps, seed in (([(60, 3000)], 4, 1, 64, 31), ([(100, 300), (1, 50), (33, 33)], 6, 2, 16, 32),
                                         ([(11, 5000)], 16, 4, 16, 33), ([(150, 150)] * 4, 8, 8, 128, 34)):
        c = Case(*env, seqs, n_head, n_kv, hd, ps, "f32", seed=seed)
        c.check(c.run(window, softcap), window, softcap)


def test_a_nan_query_of_a_wide_head_stays_in_its_row(env):
    torch = env[0]
    c = Case(*env, [(80, 200)], 4, 1, 256, 16, "f32", seed=35)
    out = c.run()
    c.q[40, :256] = float("nan")
    got = c.run()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[40, :256] = False
    assert got[40, :256].isnan().all()
    assert torch.equal(got[keep], out[keep])


@pytest.mark.parametrize("hd,ty", [(64, "f16"), (128, "f32"), (256, "f32")])
def test_single_tokens_of_large_groups(env, hd, ty):
    """17 to 39 query rows a KV head: enough sequences to fill the device, and few."""
    for n, seed in ((64, 36), (3, 37)):
        c = Case(*env, [(1, 1 + 17 * i % 300) for i in range(n)] + [(0, 5)], 20, 1, hd, 32, ty, seed=seed)
        c.check(c.run())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs,n_kv", [([(300, 2300)], 4), ([(40, 6000)], 2), ([(200, 900), (130, 1400)] * 8, 8)])
def test_f32_chunks_have_the_same_bits_every_time(env, hd, seqs, n_kv):
    """A tile's O is read back block by block while the tensor core goes on: whichever warp is late,
    the sums are the same. One tile a CTA and two, keys split over a cluster and whole."""
    torch, rie, ctx = env
    g = torch.Generator(device="cuda").manual_seed(38)
    n_head, ps = 2 * n_kv, 32
    need = [-(-n // ps) for _, n in seqs]
    pages = torch.zeros(len(seqs), max(need), dtype=torch.int32, device="cuda")
    for i, n in enumerate(need):
        pages[i, :n] = torch.arange(sum(need[:i]), sum(need[:i]) + n, dtype=torch.int32)
    cache_k, cache_v = (torch.randn(sum(need), n_kv, ps, hd, generator=g, device="cuda").half() for _ in "kv")
    cache = rie.PagedCache(ctx, n_kv, hd, ps, sum(need), k=cache_k, v=cache_v)
    n_tok = sum(n for n, _ in seqs)
    cu = torch.tensor(np.concatenate([[0], np.cumsum([n for n, _ in seqs])]), dtype=torch.int32, device="cuda")
    batch = rie.SeqBatch(cu, torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda"), pages, n_tok)
    q = torch.randn(n_tok, n_head * hd, generator=g, device="cuda") * (2 / np.sqrt(hd))
    first, again = torch.zeros_like(q), torch.zeros_like(q)
    rie.paged_attention(ctx, cache, batch, q, n_head, first)
    for _ in range(40):
        again.zero_()
        rie.paged_attention(ctx, cache, batch, q, n_head, again)
        ctx.sync()
        assert torch.equal(first, again)
    i, (new, length) = len(seqs) - 1, seqs[-1]
    ks, vs = (x[pages[i, :need[i]].long()].transpose(1, 2).reshape(-1, n_kv, hd)[:length].double().cpu().numpy() for x in (cache_k, cache_v))
    a = n_tok - new
    check_rows(first[a:a + 3].double().cpu().numpy(), q[a:a + 3].double().cpu().numpy(), [ks[:length - new + 3]], [vs[:length - new + 3]],
               [(0, 3, length - new + 3)], n_head, n_kv, hd, 0, 0.0, "f32")


@pytest.mark.parametrize("ty,times", [("f16", 3), ("f32", 12)])
@pytest.mark.parametrize("shape", ["decode", "chunk", "packed"])
def test_a_nan_key_does_not_slow_the_call(env, ty, times, shape):
    """Rows that attend a NaN key are NaN, and known to be: the formula is not gone through again key by
    key (some thousand times the call's own time). f32 rows go through it as far as the NaN, which is early here."""
    torch, rie, ctx = env
    T, g = dtype(torch, ty), torch.Generator(device="cuda").manual_seed(39)
    n_head, n_kv, hd, ps = 8, 2, 128, 64
    new, length = {"decode": (1, 60000), "chunk": (200, 9000), "packed": (3000, 3000)}[shape]
    n_pages = -(-length // ps)
    kp, vp = (torch.randn(n_pages, n_kv, ps, hd, generator=g, device="cuda").half() for _ in "kv")
    cache = rie.PagedCache(ctx, n_kv, hd, ps, n_pages, k=kp, v=vp)
    cu, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [length]))
    batch = rie.SeqBatch(cu, ln, torch.arange(n_pages, dtype=torch.int32, device="cuda")[None], new, max_len=length, max_new=new)
    q = (torch.randn(new, n_head * hd, generator=g, device="cuda") / 8).to(T)
    k, v = (x.transpose(1, 2).reshape(-1, n_kv * hd)[:length].contiguous() for x in (kp, vp))
    out = torch.zeros_like(q)

    def call():
        if shape == "packed":
            rie.packed_attention(ctx, q, k, v, cu, n_head, n_kv, hd, out, max_len=length)
        else:
            rie.paged_attention(ctx, cache, batch, q, n_head, out)

    def time():
        call()
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(6)]
        for e in ends:
            e.record()
            call()
        ctx.sync()
        return min(a.elapsed_time(b) for a, b in zip(ends, ends[1:]))

    clean = time()
    assert torch.isfinite(out).all()
    kp[0, :, 5] = float("nan")
    k[5] = float("nan")
    assert time() <= times * clean
    first = 5 if shape == "packed" else 0
    assert torch.isfinite(out[:first]).all() and torch.isnan(out[first:]).all()


def test_a_pool_of_another_device_is_refused(env):
    """By the C entry points too, before they launch anything; and a pool outlives the context that made it."""
    import ctypes
    torch, rie, ctx = env
    lib = ctx._lib
    own = rie.Context(0, torch.cuda.current_stream())
    pool = ctypes.c_void_p()
    assert lib.rcu_paged_create(own.ptr, 0, 2, 64, 16, 8, None, None, ctypes.byref(pool)) == 0
    own.sync()
    own.close()
    cu, ln, pages = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [3], [[0]]))
    batch = rie.SeqBatch(cu, ln, pages, 1)
    q, out = torch.randn(1, 256, device="cuda"), torch.ones(1, 256, device="cuda")
    assert lib.rcu_paged_attention(ctx.ptr, pool, batch._ref, q.data_ptr(), 0, 256, 4, 0, 0.0, out.data_ptr(), 256) == 0
    ctx.sync()
    assert (out == 0).all()  # zeroed pages
    if torch.cuda.device_count() > 1:
        other = rie.Context(1)
        for st in (lib.rcu_paged_attention(other.ptr, pool, batch._ref, q.data_ptr(), 0, 256, 4, 0, 0.0, out.data_ptr(), 256),
                   lib.rcu_paged_store(other.ptr, pool, batch._ref, q.data_ptr(), q.data_ptr(), 0, 128)):
            assert st == 1 and b"another device" in lib.rcu_last_error(other.ptr)
    lib.rcu_paged_free(pool)


@pytest.mark.parametrize("length", [50, 65, 1000, 2 ** 31 - 1, 2, -5, -2 ** 31])
def test_a_wrong_length_overwrites_no_other_position(env, length):
    """A table of three pages of 16, three new tokens and a length that does not fit: positions within the
    table are written, the others dropped, and what lies in the pages stays."""
    torch, rie, ctx = env
    n_kv, hd, ps = 2, 64, 16
    kp, vp = (torch.full((4, n_kv, ps, hd), x, dtype=torch.float16, device="cuda") for x in (1.0, 2.0))
    cache = rie.PagedCache(ctx, n_kv, hd, ps, 4, k=kp, v=vp)
    cu, ln, pages = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [length], [[2, 0, 3]]))
    k = torch.arange(3, device="cuda").view(3, 1).expand(3, n_kv * hd).float() + 10
    want_k, want_v = kp.clone(), vp.clone()
    for t in range(3):
        pos = length - 3 + t
        if 0 <= pos < 48:
            want_k[[2, 0, 3][pos // ps], :, pos % ps] = 10.0 + t
            want_v[[2, 0, 3][pos // ps], :, pos % ps] = 20.0 + t
    cache.store(rie.SeqBatch(cu, ln, pages, 3), k.contiguous(), (k + 10).contiguous())
    with pytest.raises(rie.RcuError, match="0x8"):
        ctx.sync()
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_the_largest_batch(env):
    """16384 sequences, empty ones and a few chunks among them: append and attention."""
    torch, rie, ctx = env
    n_kv, n_head, hd, ps, n_seq = 1, 2, 64, 16, 1 << 14
    rng = np.random.default_rng(40)
    new = np.where(np.arange(n_seq) % 5 == 3, 0, 1)
    new[[7, 9000, n_seq - 1]] = [20, 3, 5]
    lens = new + rng.integers(0, 12, n_seq)
    need = -(-lens // ps)
    pages = np.zeros((n_seq, need.max()), dtype=np.int32)
    order = rng.permutation(need.sum())
    for i, at in enumerate(np.cumsum(need) - need):
        pages[i, :need[i]] = order[at:at + need[i]]
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n_tok = int(cu[-1])
    pools = [torch.from_numpy(rng.standard_normal((int(need.sum()), n_kv, ps, hd)).astype(np.float16)).cuda() for _ in "kv"]
    cache = rie.PagedCache(ctx, n_kv, hd, ps, int(need.sum()), k=pools[0], v=pools[1])
    dev = [torch.from_numpy(x).cuda() for x in (cu, lens.astype(np.int32), pages)]
    q, k, v = (torch.from_numpy(rng.standard_normal((n_tok, w)).astype(np.float32)).cuda() for w in (n_head * hd, hd, hd))
    q /= 8
    cache.store(rie.SeqBatch(*dev, n_tok), k, v)
    out = torch.full_like(q, 7.5)
    for max_new in (0, 1):
        rie.paged_attention(ctx, cache, rie.SeqBatch(*dev, n_tok, max_new=max_new), q, n_head, out)
        ctx.sync()
        kn, vn = (x.double().cpu().numpy() for x in pools)
        qn, got = q.double().cpu().numpy(), out.double().cpu().numpy()
        for i in [*range(0, n_seq, 37), 7, 9000, n_seq - 1]:
            rows = [(pages[i, p // ps], p % ps) for p in range(lens[i])]
            ks, vs = (np.array([x[pg, :, sl] for pg, sl in rows]).reshape(-1, n_kv, hd) for x in (kn, vn))
            assert (ks[lens[i] - new[i]:, 0] == k[cu[i]:cu[i + 1]].half().double().cpu().numpy()).all()
            check_rows(got, qn, [ks], [vs], [(int(cu[i]), int(new[i]), int(lens[i]))], n_head, n_kv, hd, 0, 0.0, "f32")


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("n_head,n_kv,hd", [(300, 1, 32), (514, 2, 64), (129, 1, 256)])
def test_groups_larger_than_a_tile(env, ty, n_head, n_kv, hd):
    """One token's heads alone fill a tile of query rows, or more than one."""
    c = Case(*env, [(1, 40), (3, 200), (1, 1)], n_head, n_kv, hd, 16, ty, seed=41)
    c.check(c.run())
    c.check(c.run(window=30), window=30)


@pytest.mark.parametrize("new,ty", [(1, "f32"), (3, "f16"), (70, "f32"), (70, "f16")])
def test_pools_past_32_bits(env, new, ty):
    """Pages whose values lie more than 2^32 elements into the pool."""
    torch, rie, ctx = env
    n_kv, hd, ps, length = 1, 256, 1024, 1500
    n_pages = (1 << 32) // (hd * ps) + 3
    kp, vp = (torch.zeros(n_pages, n_kv, ps, hd, dtype=torch.float16, device="cuda") for _ in "kv")
    g = torch.Generator(device="cuda").manual_seed(42)
    k, v = (torch.randn(length, hd, generator=g, device="cuda").half() for _ in "kv")
    cache = rie.PagedCache(ctx, n_kv, hd, ps, n_pages, k=kp, v=vp)
    pages = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32, device="cuda")
    for cu, ln in (([0, 1000], 1000), ([0, 500], 1500)):
        cu, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, [ln]))
        n, first = int(cu[1]), int(ln[0]) - int(cu[1])
        cache.store(rie.SeqBatch(cu, ln, pages, n), k[first:first + n], v[first:first + n])
    ctx.sync()
    assert torch.equal(kp[n_pages - 1, 0], k[:ps]) and torch.equal(vp[n_pages - 2, 0, :length - ps], v[ps:])
    assert not kp[:n_pages - 2].any()
    q = (torch.randn(new, 2 * hd, generator=g, device="cuda") / 8).to(dtype(torch, ty))
    out = torch.zeros_like(q)
    cu, ln = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, new], [length]))
    rie.paged_attention(ctx, cache, rie.SeqBatch(cu, ln, pages, new), q, 2, out)
    ctx.sync()
    check_rows(out.double().cpu().numpy(), q.double().cpu().numpy(), [k.view(-1, 1, hd).double().cpu().numpy()],
               [v.view(-1, 1, hd).double().cpu().numpy()], [(0, new, length)], 2, 1, hd, 0, 0.0, ty)
