"""Log probabilities, entropy and alternatives of rows of logits against 64 bits, alone and through
the backend.

Tolerances: with m the row's maximum, log p = (x - m) - ln z. x - m is rounded once (2^-24 of it),
exp(x - m) comes with 2^-22 and, from the rounded x - m and its product with log2 e, another
2 * 2^-24 |x - m| whose weight exp(x - m) keeps below 2^-24; z is a sum of positive values in
chains of at most vocab / 4096 + 64 additions of 2^-24 (times z): ln z is off by at most
(8 + vocab / 4096 + 64) 2^-24, its logarithm rounds once more, and the result once. The entropy
ln z - w / z adds the same relative error on w / z, whose size is the entropy's at most plus ln z.
"""
import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import rust_interference_engine_b200 as rie
    return torch, rie, rie.Context(0, torch.cuda.current_stream())


def exact(x):
    """(log softmax, entropy) in 64 bits."""
    x = x.astype(np.float64)
    d = x - x.max(axis=1, keepdims=True)
    e = np.exp(d)
    z = e.sum(axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        w = np.where(e > 0, e * d, 0.0).sum(axis=1, keepdims=True)
    return d - np.log(z), (np.log(z) - w / z)[:, 0], np.log(z)[:, 0]


def order(x, k):
    """Indices of the k largest, NaN first, ties to the lowest index."""
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    nan = np.isnan(x)
    return np.stack([np.lexsort((np.arange(x.shape[1]), -key[r], ~nan[r]))[:k] for r in range(x.shape[0])])


def run(env, x, targets, k):
    torch, rie, ctx = env
    n = x.shape[0]
    o = dict(logprob=torch.full((n,), 9.0, device="cuda"), entropy=torch.full((n,), 9.0, device="cuda"),
             top_ids=torch.full((n, k), -9, dtype=torch.int32, device="cuda"), top_logprobs=torch.full((n, k), 9.0, device="cuda"))
    rie.logprobs(ctx, x, torch.from_numpy(targets.astype(np.int32)).cuda(), o["logprob"], o["entropy"], o["top_ids"], o["top_logprobs"])
    ctx.sync()
    return {a: b.cpu().numpy() for a, b in o.items()}


def check(x, targets, k, got, vocab):
    lp, ent, lnz = exact(x)
    step = (8 + vocab / 4096 + 64) * 2.0 ** -24
    rows = np.arange(x.shape[0])
    want = np.where(targets >= 0, lp[rows, np.maximum(targets, 0)], 0.0)
    fin = np.isfinite(want)
    assert (np.isneginf(got["logprob"]) == np.isneginf(want)).all()
    assert (np.abs(got["logprob"][fin] - want[fin]) <= step + 2.0 ** -23 * (1 + np.abs(want[fin]) + lnz[fin])).all()
    assert (np.abs(got["entropy"] - ent) <= 2 * step * (1 + np.abs(ent) + lnz) + 2.0 ** -23).all()
    ids = order(x, k)
    assert (got["top_ids"] == ids).all()
    want = np.take_along_axis(lp, ids, axis=1)
    fin = np.isfinite(want)
    assert (np.isneginf(got["top_logprobs"]) == ~fin).all()
    tol = step + 2.0 ** -23 * (1 + np.abs(np.where(fin, want, 0.0)) + lnz[:, None])
    assert (np.abs(got["top_logprobs"][fin] - want[fin]) <= tol[fin]).all()


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 7), (2, 255, 128), (5, 384, 0), (1, 4096, 20), (4, 4097, 64), (3, 32000, 5),
                                          (2, 50257, 50), (1, 151936, 20), (33, 20001, 128), (700, 513, 3)])
def test_logprobs(env, ty, rows, vocab, k):
    torch = env[0]
    rng = np.random.default_rng(vocab)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[ty]
    wide = torch.from_numpy(rng.standard_normal((rows, vocab + 3)) * 4).to(t).cuda()
    x = wide[:, 1:vocab + 1]  # rows that start and end anywhere
    xn = x.float().cpu().numpy()
    targets = rng.integers(-1, vocab, rows)
    check(xn, targets, k, run(env, x, targets, k), vocab)


@pytest.mark.parametrize("k", [1, 20, 128])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "one_thread", "few_values", "mostly_masked", "blocks"])
def test_orders_that_defeat_the_bound(env, k, kind):
    """Rows whose largest values lie where the running bound helps least, ties everywhere."""
    torch = env[0]
    n = 60001
    rng = np.random.default_rng(1)
    i = np.arange(n)
    x = {"equal": np.zeros(n), "rising": i / 3000.0, "falling": -i / 3000.0,
         "one_thread": np.where(i // 4 % 256 == 7, 5.0 + i / n, rng.standard_normal(n)),
         "few_values": rng.integers(0, 3, n).astype(float), "mostly_masked": np.where(i % 1009 == 5, rng.standard_normal(n), -np.inf),
         "blocks": np.where(i > 55000, 3.0, 0.0) + np.where(i % 2, 0.0, -0.0)}[kind].astype(np.float32)
    x = np.stack([x, x[::-1], np.roll(x, 12345)])
    targets = np.array([0, n - 1, 77])
    check(x, targets, k, run(env, torch.from_numpy(x.copy()).cuda(), targets, k), n)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("value", ["lowest", -1e38, -3e37, -1e34, -2e3])
@pytest.mark.parametrize("k", [0, 3])
def test_masks_of_very_low_values(env, ty, value, k):
    """Tokens masked by a finite value, in runs that fill a thread's, a warp's and a CTA's values, and
    rows that are all of it: the entropy is that of the other tokens."""
    torch = env[0]
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[ty]
    n, low = 60001, torch.finfo(t).min if value == "lowest" else value
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((7, n)) * 4)
    keep = torch.zeros(7, n, dtype=torch.bool)
    keep[0, n // 2:] = True
    keep[1, :n // 2] = True
    keep[2, [5, 777, 30000, 59999]] = True
    keep[3] = True
    keep[3, 20000:26000] = False
    keep[4, n - 1] = True
    keep[5, ::16] = True  # row 6: nothing but the mask
    x = torch.where(keep, x, torch.tensor(float(low), dtype=torch.float64)).to(t).cuda()
    xn = x.double().cpu().numpy()
    targets = np.array([n - 1, 0, 777, 21000, n - 1, 16, 9])
    for rows in (slice(0, 7), slice(0, 4), slice(4, 7)):
        check(xn[rows], targets[rows], k, run(env, x[rows], targets[rows], k), n)


@pytest.mark.parametrize("rows", [2, 9])
def test_rows_that_span_more_than_the_largest_number(env, rows):
    """Finite logits whose distance from the maximum has no f32 value: they add nothing."""
    torch = env[0]
    x = np.full((rows, 20000), -3e38, dtype=np.float32)
    x[:, 3::5] = np.random.default_rng(4).standard_normal((rows, 4000))
    x[:, 100:200] = 3e38
    got = run(env, torch.from_numpy(x).cuda(), np.full(rows, 150), 100)
    want = np.log(100.0)  # of 100 equal values; ln z rounds once, a sum of 100 ones is exact
    assert (np.abs(got["entropy"] - want) <= 2.0 ** -22 * want).all()
    assert (np.abs(got["logprob"] + want) <= 2.0 ** -22 * want).all()
    assert (got["top_ids"] == np.arange(100, 200)).all()


def test_rows_without_a_distribution(env):
    torch, rie, ctx = env
    n = 5000
    x = np.random.default_rng(2).standard_normal((6, n)).astype(np.float32)
    x[0, 4000] = np.nan
    x[1, 17] = np.inf
    x[2] = -np.inf
    x[3] = -np.inf
    x[3, 9] = np.nan
    x[4, 10:] = -np.inf
    got = run(env, torch.from_numpy(x).cuda(), np.array([1, 17, 3, 9, 20, -1]), 4)
    for r in range(4):
        assert np.isnan(got["logprob"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["top_logprobs"][r]).all()
    assert (got["top_ids"] == order(x, 4)).all()
    assert np.isneginf(got["logprob"][4]) and got["logprob"][5] == 0.0
    lp, ent, _ = exact(x[4:])
    assert np.abs(got["entropy"][4:] - ent).max() <= 1e-4


def test_target_outside_the_vocabulary_is_reported(env):
    torch, rie, ctx = env
    x = torch.randn(3, 100, device="cuda")
    for bad in (100, -2, 2 ** 31 - 1):
        t = torch.tensor([5, bad, 7], dtype=torch.int32, device="cuda")
        lp = torch.zeros(3, device="cuda")
        rie.logprobs(ctx, x, t, lp)
        with pytest.raises(rie.RcuError, match="0x8"):
            ctx.sync()
        v = lp.cpu().numpy()
        assert np.isnan(v[1]) and np.isfinite(v[[0, 2]]).all()
    rie.logprobs(ctx, x, entropy=torch.zeros(3, device="cuda"))  # nothing but the entropy
    ctx.sync()


def test_logits_past_32_bits(env):
    """Rows whose values lie more than 2^32 elements into the logits."""
    torch = env[0]
    rows, vocab = 29000, 151936
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    pick = [0, 14000, 28400, rows - 1]
    x[pick] = (torch.randn(len(pick), vocab, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") * 4).half()
    targets = np.random.default_rng(6).integers(0, vocab, rows)
    got = run(env, x, targets, 3)
    check(x[pick].float().cpu().numpy(), targets[pick], 3, {n: a[pick] for n, a in got.items()}, vocab)
    rest = np.setdiff1d(np.arange(rows), pick)
    step = (8 + vocab / 4096 + 64) * 2.0 ** -24  # equal values: -ln of the vocabulary, ties in order
    assert (np.abs(got["logprob"][rest] + np.log(vocab)) <= step + 2.0 ** -23 * (1 + 2 * np.log(vocab))).all()
    assert (got["top_ids"][rest] == np.arange(3)).all()


@pytest.fixture(scope="module")
def backend(env):
    torch, rie, ctx = env
    from rust_interference_engine_b200 import model as M
    spec = M.SyntheticSpec.tiny("qwen3", rie.GgmlType.Q4_0)
    rng = O.Rng(4711)
    m = M.Model(ctx, spec.config())
    for name, t, r, c, data in M.synthetic_tensors(spec, lambda t, r, c: rng.weight(int(t), r, c), lambda n, s: rng.vec(n, s),
                                                   lambda n: np.ones(n, dtype=np.float32)):
        m.set_tensor(name, t, r, c, data)
    return M.CudaBackend(m, 64, 16), spec


@pytest.mark.parametrize("n,pos,k", [(1, 0, 5), (7, 0, 20), (16, 0, 0), (4, 12, 3)])
def test_backend_score_matches_its_logits(backend, n, pos, k):
    """score() is the forward's own logits, scored: the same rows through numpy."""
    b, spec = backend
    toks = np.random.default_rng(n).integers(0, spec.n_vocab, pos + n)
    if pos:
        b.forward(toks[:pos], 0)
    logits = b.forward(toks[pos:], pos, all_logits=True)
    targets = np.concatenate([toks[pos + 1:], [-1]])
    if pos:
        b.forward(toks[:pos], 0)
    for _ in range(3):  # eager, captured and replayed for single tokens
        got = b.score(toks[pos:], pos, targets, k)
        check(logits, targets, k, got, spec.n_vocab)
    plain = b.score(toks[pos:], pos)
    assert "logprob" not in plain and plain["top_ids"].shape == (n, 0)


def test_backend_score_refuses(backend, env):
    rie = env[1]
    b, spec = backend
    with pytest.raises(rie.RcuError, match="target id"):
        b.score([1, 2], 0, [3, spec.n_vocab])
    with pytest.raises(rie.RcuError, match="token id"):
        b.score([spec.n_vocab], 0, [3])
    with pytest.raises(rie.RcuError, match="context window full"):
        b.score([1] * 16, 60)
    with pytest.raises(rie.RcuError, match="exceeds max batch"):
        b.score([1] * 17, 0)
    with pytest.raises(rie.RcuError, match="alternatives"):
        b.score([1], 0, top_k=129)
    with pytest.raises(ValueError, match="targets"):
        b.score([1, 2], 0, [3])
