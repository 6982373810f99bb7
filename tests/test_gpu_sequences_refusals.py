"""Refusals of the operators over batches of sequences and of the scores, each by its message: the
calls differ from one that is accepted in the named argument alone, and are refused on the host
before anything is launched."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

INVALID, UNSUPPORTED, RUNTIME = 1, 3, 6
F32, F16, BF16, Q8_0 = 0, 1, 30, 8


@pytest.fixture(scope="module")
def env():
    import torch
    import rust_interference_engine_b200 as rie
    ctx = rie.Context(0, torch.cuda.current_stream())
    room = torch.zeros(1 << 22, device="cuda")  # whatever a call is given lies in here
    cache = rie.PagedCache(ctx, 2, 64, 16, 8)
    cu, ln, pages = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 3], [5, 20], [[0, 1], [2, 3]]))
    ctx.sync()
    return ctx, room, cache, (cu, ln, pages)


def outcome(ctx, status):
    """(status, message); what was accepted has run."""
    message = ctx._lib.rcu_last_error(ctx.ptr).decode() if status else ""
    if not status:
        ctx.sync()
    return status, message


def batch(env, **kw):
    cu, ln, pages = (x.data_ptr() for x in env[3])
    from rust_interference_engine_b200._lib import RcuSeqs
    a = dict(cu=cu, len=ln, pages=pages, n_seq=2, n_tok=3, ld_pages=2, max_len=0, max_new=0)
    a.update(kw)
    return RcuSeqs(*(a[n] for n, _ in RcuSeqs._fields_))


def refused(got, status, message):
    assert got[0] == status and message in got[1], got


PAGE_TABLES = [(dict(ld_pages=0), INVALID, "page table"), (dict(ld_pages=1 << 27), INVALID, "page table"),
               (dict(ld_pages=1 << 60), INVALID, "page table"), (dict(ld_pages=(1 << 60) + 1), INVALID, "page table")]


@pytest.mark.parametrize("kw,status,message", PAGE_TABLES)
def test_page_tables_are_refused(env, kw, status, message):
    """Widths whose positions leave 31 bits, or whose product with the page size leaves 64."""
    ctx, room, cache, _ = env
    b, p = batch(env, **kw), room.data_ptr()
    refused(outcome(ctx, ctx._lib.rcu_paged_attention(ctx.ptr, cache.ptr, C.byref(b), p, F32, 256, 4, 0, 0.0, p + (1 << 20), 256)), status, message)
    refused(outcome(ctx, ctx._lib.rcu_paged_store(ctx.ptr, cache.ptr, C.byref(b), p, p, F32, 128)), status, message)


NULL = (INVALID, "null argument")
BATCHES = [(dict(cu=None), *NULL), (dict(len=None), *NULL), (dict(pages=None), *NULL), (dict(n_tok=0), RUNTIME, "empty batch"),
           (dict(n_seq=0), RUNTIME, "empty batch"), (dict(n_tok=(1 << 30) + 1), INVALID, "batch too large"),
           (dict(n_seq=(1 << 14) + 1), INVALID, "batch too large")]
HEADS = [(dict(n_head=5), INVALID, "not divisible"), (dict(n_head=0), INVALID, "not divisible"),
         (dict(n_head=8192, ld_q=1 << 19, ld_out=1 << 19), INVALID, "4096 query heads"),
         (dict(window=1 << 31), INVALID, "window must be below"), (dict(softcap=float("nan")), INVALID, "softcap must be finite"),
         (dict(softcap=float("inf")), INVALID, "softcap must be finite")]


def paged(env, **kw):
    ctx, room, cache, _ = env
    a = dict(pool=cache.ptr, batch={}, q=0, type=F32, ld_q=256, n_head=4, window=0, softcap=0.0, out=1 << 20, ld_out=256)
    assert set(kw) <= set(a)
    a.update(kw)
    q, out = (None if x is None else room.data_ptr() + x for x in (a["q"], a["out"]))
    b = None if a["batch"] is None else C.byref(batch(env, **a["batch"]))
    return outcome(ctx, ctx._lib.rcu_paged_attention(ctx.ptr, a["pool"], b, q, a["type"], a["ld_q"], a["n_head"], a["window"], a["softcap"], out, a["ld_out"]))


@pytest.mark.parametrize("kw,status,message", [
    (dict(pool=None), *NULL), (dict(batch=None), *NULL), (dict(q=None), *NULL), (dict(out=None), *NULL),
    *[(dict(batch=b), st, m) for b, st, m in BATCHES], *HEADS,
    (dict(batch=dict(n_tok=1 << 30), n_head=4096), INVALID, "batch too large"),
    (dict(type=BF16), UNSUPPORTED, "queries are f32 or f16"), (dict(type=Q8_0), UNSUPPORTED, "queries are f32 or f16"),
    (dict(out=0), INVALID, "out must not be q"),
    (dict(q=4), INVALID, "q: rows must start on 16-byte"), (dict(q=8, type=F16), INVALID, "q: rows must start on 16-byte"),
    (dict(ld_q=257), INVALID, "q: rows must start on 16-byte"), (dict(ld_q=260, type=F16), INVALID, "q: rows must start on 16-byte"),
    (dict(out=(1 << 20) + 4), INVALID, "out: rows must start on 16-byte"), (dict(ld_out=258), INVALID, "out: rows must start on 16-byte"),
    (dict(ld_q=252), INVALID, "q: row stride smaller"), (dict(ld_out=252), INVALID, "out: row stride smaller"),
    (dict(ld_q=(1 << 32) + 4), INVALID, "q: row stride too large"), (dict(ld_out=1 << 62), INVALID, "out: row stride too large"),
    (dict(), 0, "")])
def test_paged_attention_refuses(env, kw, status, message):
    refused(paged(env, **kw), status, message)


def store(env, **kw):
    ctx, room, cache, _ = env
    a = dict(pool=cache.ptr, batch={}, k=0, v=1 << 20, type=F32, ld=128)
    assert set(kw) <= set(a)
    a.update(kw)
    k, v = (None if x is None else room.data_ptr() + x for x in (a["k"], a["v"]))
    b = None if a["batch"] is None else C.byref(batch(env, **a["batch"]))
    return outcome(ctx, ctx._lib.rcu_paged_store(ctx.ptr, a["pool"], b, k, v, a["type"], a["ld"]))


@pytest.mark.parametrize("kw,status,message", [
    (dict(pool=None), *NULL), (dict(batch=None), *NULL), (dict(k=None), *NULL), (dict(v=None), *NULL),
    *[(dict(batch=b), st, m) for b, st, m in BATCHES],
    (dict(type=Q8_0), UNSUPPORTED, "rows are f32, f16 or bf16"), (dict(k=4), INVALID, "k: rows must start on 16-byte"),
    (dict(v=(1 << 20) + 8), INVALID, "v: rows must start on 16-byte"), (dict(ld=130), INVALID, "k: rows must start on 16-byte"),
    (dict(ld=132, type=BF16), INVALID, "k: rows must start on 16-byte"), (dict(ld=124), INVALID, "k: row stride smaller"),
    (dict(ld=(1 << 32) + 4), INVALID, "k: row stride too large"), (dict(), 0, "")])
def test_paged_store_refuses(env, kw, status, message):
    refused(store(env, **kw), status, message)


def packed(env, **kw):
    ctx, room, _, dev = env
    a = dict(q=0, q_type=F16, ld_q=256, k=1 << 20, v=2 << 20, kv=F16, ld_kv=128, cu=dev[0].data_ptr(), n_seq=2, n_tok=3, max_len=0,
             n_head=4, n_head_kv=2, hd=64, window=0, softcap=0.0, out=3 << 20, ld_out=256)
    assert set(kw) <= set(a)
    a.update(kw)
    q, k, v, out = (None if a[n] is None else room.data_ptr() + a[n] for n in ("q", "k", "v", "out"))
    return outcome(ctx, ctx._lib.rcu_packed_attention(ctx.ptr, q, a["q_type"], a["ld_q"], k, v, a["kv"], a["ld_kv"], a["cu"], a["n_seq"],
                                                      a["n_tok"], a["max_len"], a["n_head"], a["n_head_kv"], a["hd"], a["window"],
                                                      a["softcap"], out, a["ld_out"]))


@pytest.mark.parametrize("kw,status,message", [
    (dict(q=None), *NULL), (dict(k=None), *NULL), (dict(v=None), *NULL), (dict(cu=None), *NULL), (dict(out=None), *NULL),
    (dict(n_tok=0), RUNTIME, "empty batch"), (dict(n_seq=0), RUNTIME, "empty batch"), (dict(n_tok=1 << 31), INVALID, "batch too large"),
    (dict(n_seq=16385), INVALID, "batch too large"), *HEADS, (dict(n_head_kv=0), INVALID, "not divisible"),
    (dict(n_tok=1 << 30, n_head=4096, n_head_kv=1, ld_q=1 << 19, ld_out=1 << 19), INVALID, "batch too large"),
    (dict(hd=0), INVALID, "head_dim must be"), (dict(hd=48), INVALID, "head_dim must be"), (dict(hd=288), INVALID, "head_dim must be"),
    (dict(q_type=BF16), UNSUPPORTED, "queries are f32 or f16 over"), (dict(q_type=F32, kv=F32), UNSUPPORTED, "queries are f32 or f16 over"),
    (dict(q_type=F32, kv=BF16), UNSUPPORTED, "queries are f32 or f16 over"), (dict(kv=BF16), UNSUPPORTED, "queries are f32 or f16 over"),
    (dict(out=0), INVALID, "out must not be an input"), (dict(out=1 << 20), INVALID, "out must not be an input"),
    (dict(out=2 << 20), INVALID, "out must not be an input"),
    (dict(q=2), INVALID, "q: rows must start on 16-byte"), (dict(k=(1 << 20) + 8), INVALID, "k: rows must start on 16-byte"),
    (dict(v=(2 << 20) + 8), INVALID, "v: rows must start on 16-byte"), (dict(out=(3 << 20) + 8), INVALID, "out: rows must start on 16-byte"),
    (dict(ld_q=260), INVALID, "q: rows must start on 16-byte"), (dict(ld_kv=132), INVALID, "k: rows must start on 16-byte"),
    (dict(ld_out=257), INVALID, "out: rows must start on 16-byte"), (dict(ld_q=248), INVALID, "q: row stride smaller"),
    (dict(ld_kv=120), INVALID, "k: row stride smaller"), (dict(ld_out=248), INVALID, "out: row stride smaller"),
    (dict(ld_kv=(1 << 32) + 8), INVALID, "k: row stride too large"), (dict(), 0, "")])
def test_packed_attention_refuses(env, kw, status, message):
    refused(packed(env, **kw), status, message)


def logprobs(env, **kw):
    ctx, room, _, _ = env
    a = dict(x=0, type=F32, rows=3, vocab=200, ld=200, targets=1 << 20, logprob=2 << 20, entropy=3 << 20, top_k=5, ids=4 << 20, tlp=5 << 20)
    assert set(kw) <= set(a)
    a.update(kw)
    at = {n: None if a[n] is None else room.data_ptr() + a[n] for n in ("x", "targets", "logprob", "entropy", "ids", "tlp")}
    return outcome(ctx, ctx._lib.rcu_logprobs(ctx.ptr, at["x"], a["type"], a["rows"], a["vocab"], a["ld"], at["targets"], at["logprob"],
                                              at["entropy"], a["top_k"], at["ids"], at["tlp"]))


@pytest.mark.parametrize("kw,status,message", [
    (dict(x=None), *NULL), (dict(rows=0), RUNTIME, "empty batch"), (dict(type=2), UNSUPPORTED, "logits are"), (dict(type=Q8_0), UNSUPPORTED, "logits are"),
    (dict(targets=None), INVALID, "targets and logprob"), (dict(logprob=None), INVALID, "targets and logprob"),
    (dict(ids=None), INVALID, "top_k without"), (dict(tlp=None), INVALID, "top_k without"), (dict(vocab=0), INVALID, "out of range"),
    (dict(vocab=1 << 31, ld=1 << 31), INVALID, "out of range"), (dict(rows=(1 << 26) + 1), INVALID, "out of range"),
    (dict(ld=199), INVALID, "ld smaller"), (dict(top_k=129), INVALID, "at most 128"), (dict(vocab=4, top_k=5), INVALID, "no more than the vocabulary"),
    (dict(x=2), INVALID, "misaligned"), (dict(x=1, type=F16), INVALID, "misaligned"), (dict(x=3, type=BF16), INVALID, "misaligned"),
    (dict(), 0, "")])
def test_logprobs_refuses(env, kw, status, message):
    refused(logprobs(env, **kw), status, message)


def create(env, **kw):
    ctx, room, _, _ = env
    a = dict(kv_type=0, n_kv=2, hd=64, page=16, pages=8, k=0, v=1 << 20)
    assert set(kw) <= set(a)
    a.update(kw)
    k, v = (None if x is None else room.data_ptr() + x for x in (a["k"], a["v"]))
    pool = C.c_void_p(77)
    got = outcome(ctx, ctx._lib.rcu_paged_create(ctx.ptr, a["kv_type"], a["n_kv"], a["hd"], a["page"], a["pages"], k, v, C.byref(pool)))
    assert bool(pool.value) == (got[0] == 0)
    ctx._lib.rcu_paged_free(pool)
    return got


@pytest.mark.parametrize("kw,status,message", [
    (dict(kv_type=3), INVALID, "unknown kv type"), (dict(kv_type=-1), INVALID, "unknown kv type"), (dict(kv_type=1), UNSUPPORTED, "f16 pages only"),
    (dict(kv_type=2), UNSUPPORTED, "f16 pages only"), (dict(n_kv=0), INVALID, "n_head_kv 1..4096"), (dict(n_kv=4097), INVALID, "n_head_kv 1..4096"),
    (dict(hd=0), INVALID, "head_dim must be"), (dict(hd=40), INVALID, "head_dim must be"), (dict(hd=288), INVALID, "head_dim must be"),
    (dict(page=8), INVALID, "power of two"), (dict(page=48), INVALID, "power of two"), (dict(page=2048), INVALID, "power of two"),
    (dict(pages=0), INVALID, "n_pages out of range"), (dict(pages=1 << 31), INVALID, "n_pages out of range"),
    (dict(k=None), INVALID, "both pools"), (dict(v=None), INVALID, "both pools"), (dict(k=8), INVALID, "pools must be 16-byte"),
    (dict(v=(1 << 20) + 8), INVALID, "pools must be 16-byte"), (dict(), 0, "")])
def test_paged_create_refuses(env, kw, status, message):
    refused(create(env, **kw), status, message)


def test_the_mirror_checks_its_tensors(env):
    """Shapes, types, strides and devices of the Python calls."""
    import torch
    import rust_interference_engine_b200 as rie
    ctx, _, cache, dev = env
    b = rie.SeqBatch(*dev, 3)
    q, kv = torch.zeros(3, 256, device="cuda"), torch.zeros(3, 128, device="cuda")
    bad = [(lambda: rie.paged_attention(ctx, cache, b, q[:2], 4, q.clone()), "q: expected 3 x 256"),
           (lambda: rie.paged_attention(ctx, cache, b, q, 4, q.clone().half()), "same type"),
           (lambda: rie.paged_attention(ctx, cache, b, q.cpu(), 4, q.clone()), "q: expected a CUDA"),
           (lambda: rie.paged_attention(ctx, cache, b, torch.zeros(3, 512, device="cuda")[:, ::2], 4, q), "contiguous"),
           (lambda: rie.paged_attention(ctx, cache, b, q.int(), 4, q.clone()), "f32, f16 or bf16"),
           (lambda: cache.store(b, kv, kv.half()), "same type and row stride"), (lambda: cache.store(b, kv, q[:, :128]), "same type and row stride"),
           (lambda: cache.store(b, kv, kv.cpu()), "v: expected a CUDA"), (lambda: cache.store(b, kv.view(-1), kv), "k: expected 3 x 128"),
           (lambda: rie.packed_attention(ctx, q, kv, kv, dev[0].long(), 4, 2, 64, q.clone()), "cu: expected"),
           (lambda: rie.packed_attention(ctx, q, kv.half(), kv, dev[0], 4, 2, 64, q.clone()), "same type"),
           (lambda: rie.SeqBatch(dev[0], dev[1], dev[2][:1], 3), "2 sequences need"), (lambda: rie.SeqBatch(dev[0][1:], dev[1], dev[2], 3), "2 sequences need"),
           (lambda: rie.SeqBatch(*dev, -1), "must not be negative"), (lambda: rie.SeqBatch(dev[0], dev[1], dev[2][:, :1], 3), "contiguous"),
           (lambda: rie.logprobs(ctx, q.view(-1)), "expected rows"), (lambda: rie.logprobs(ctx, q, dev[1]), "pass targets with logprob"),
           (lambda: rie.logprobs(ctx, q, entropy=torch.zeros(2, device="cuda")), "entropy: expected"),
           (lambda: rie.logprobs(ctx, q, top_ids=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), "pass targets with logprob"),
           (lambda: rie.PagedCache(ctx, 2, 64, 16, 8, k=kv), "both pools"),
           (lambda: rie.PagedCache(ctx, 2, 64, 16, 8, k=kv.half(), v=kv.half()), "contiguous f16 values"),
           (lambda: rie.PagedCache(ctx, 2, 64, 16, 8, ty=rie.KvType.Q8_0), "f16 pages only")]
    for i, (call, message) in enumerate(bad):
        with pytest.raises((ValueError, rie.RcuError), match=message):
            call()
            raise AssertionError(f"call {i} was accepted")
    ctx.sync()
