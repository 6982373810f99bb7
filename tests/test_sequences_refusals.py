"""Refusals of the operators over batches of sequences and of the scores. What the C entry points
can tell from their arguments alone they tell before they touch the context, so the packed and the
score entry points are tested here without a GPU (a null context, addresses that are never read)."""
import ctypes as C

import pytest

from rust_interference_engine_b200 import _lib

INVALID, UNSUPPORTED, RUNTIME = _lib.RCU_ERR_INVALID, _lib.RCU_ERR_UNSUPPORTED, _lib.RCU_ERR_RUNTIME
F32, F16, BF16 = 0, 1, 30
A = 0x10000  # an aligned address


def packed(**kw):
    a = dict(q=A, q_type=F16, ld_q=256, k=A, v=A, kv=F16, ld_kv=128, cu=A, n_seq=2, n_tok=10, max_len=0, n_head=4, n_head_kv=2,
             hd=64, window=0, softcap=0.0, out=2 * A, ld_out=256)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().rcu_packed_attention(None, a["q"], a["q_type"], a["ld_q"], a["k"], a["v"], a["kv"], a["ld_kv"], a["cu"],
                                            a["n_seq"], a["n_tok"], a["max_len"], a["n_head"], a["n_head_kv"], a["hd"],
                                            a["window"], a["softcap"], a["out"], a["ld_out"])


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(cu=None), INVALID), (dict(out=None), INVALID),
    (dict(n_tok=0), RUNTIME), (dict(n_seq=0), RUNTIME), (dict(n_tok=1 << 31), INVALID), (dict(n_seq=1 << 25), INVALID),
    (dict(n_head=5), INVALID), (dict(n_head=0), INVALID), (dict(n_head_kv=0), INVALID), (dict(n_head=8192, ld_q=1 << 20, ld_out=1 << 20), INVALID),
    (dict(hd=0), INVALID), (dict(hd=48), INVALID), (dict(hd=288), INVALID),
    (dict(window=1 << 31), INVALID), (dict(softcap=float("nan")), INVALID), (dict(softcap=float("inf")), INVALID),
    (dict(q_type=BF16), UNSUPPORTED), (dict(kv=F32, q_type=F32), UNSUPPORTED), (dict(kv=BF16), UNSUPPORTED), (dict(q_type=2), UNSUPPORTED),
    (dict(q=A + 2), INVALID), (dict(k=A + 8), INVALID), (dict(v=A + 8), INVALID), (dict(out=A + 8), INVALID),
    (dict(ld_q=255), INVALID), (dict(ld_q=260), INVALID), (dict(ld_kv=120), INVALID), (dict(ld_kv=132), INVALID), (dict(ld_out=248), INVALID),
    (dict(out=A), INVALID), (dict(n_seq=16385, n_tok=20000), INVALID),
    (dict(n_tok=1 << 30, n_head=4096, n_head_kv=1, ld_q=1 << 19, ld_out=1 << 19), INVALID),
    (dict(), INVALID),  # nothing but the context is missing
])
def test_packed_attention_refuses(kw, status):
    assert packed(**kw) == status


def logprobs(**kw):
    a = dict(x=A, type=F32, rows=3, vocab=100, ld=100, targets=A, logprob=A, entropy=A, top_k=5, ids=A, tlp=A)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().rcu_logprobs(None, a["x"], a["type"], a["rows"], a["vocab"], a["ld"], a["targets"], a["logprob"],
                                    a["entropy"], a["top_k"], a["ids"], a["tlp"])


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), INVALID), (dict(rows=0), RUNTIME), (dict(type=2), UNSUPPORTED), (dict(type=12), UNSUPPORTED),
    (dict(targets=None), INVALID), (dict(logprob=None), INVALID), (dict(ids=None), INVALID), (dict(tlp=None), INVALID),
    (dict(vocab=0), INVALID), (dict(vocab=1 << 31, ld=1 << 31), INVALID), (dict(rows=1 << 27), INVALID), (dict(ld=99), INVALID),
    (dict(top_k=129, vocab=200, ld=200), INVALID), (dict(top_k=101), INVALID), (dict(x=A + 2), INVALID), (dict(type=F16, x=A + 1), INVALID),
    (dict(), INVALID),
])
def test_logprobs_refuses(kw, status):
    assert logprobs(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(kv_type=3), INVALID), (dict(kv_type=1), UNSUPPORTED), (dict(kv_type=2), UNSUPPORTED), (dict(n_kv=0), INVALID), (dict(hd=40), INVALID),
    (dict(hd=512), INVALID), (dict(page=8), INVALID), (dict(page=48), INVALID), (dict(page=2048), INVALID), (dict(pages=0), INVALID),
    (dict(pages=1 << 31), INVALID), (dict(k=A), INVALID), (dict(v=A), INVALID), (dict(k=A + 8, v=A), INVALID), (dict(), INVALID)])
def test_paged_create_refuses(kw, status):
    a = dict(kv_type=0, n_kv=2, hd=64, page=16, pages=8, k=None, v=None)
    a.update(kw)
    out = C.c_void_p(77)
    assert _lib.load().rcu_paged_create(None, a["kv_type"], a["n_kv"], a["hd"], a["page"], a["pages"], a["k"], a["v"], C.byref(out)) == status
    assert not out.value


def test_null_handles():
    lib = _lib.load()
    lib.rcu_paged_free(None)
    assert lib.rcu_paged_device_ptrs(None, None, None) == INVALID
    assert lib.rcu_paged_store(None, None, None, None, None, F32, 64) == INVALID
    assert lib.rcu_paged_attention(None, None, None, None, F32, 64, 1, 0, 0.0, None, 64) == INVALID
    assert lib.rcu_backend_score(None, None, 0, 0, None, None, None, 0, None, None) == INVALID


def test_seq_batch_checks_its_tensors():
    torch = pytest.importorskip("torch")
    import rust_interference_engine_b200 as rie
    cu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        rie.SeqBatch(cu, cu[:2].clone(), torch.zeros(2, 4, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="int32"):
        rie.SeqBatch(cu.long(), cu[:2].clone(), torch.zeros(2, 4, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="2-dimensional"):
        rie.SeqBatch(cu, cu[:2].clone(), cu, 1)


def test_a_cache_of_another_device_is_refused():
    """Before anything of it is used."""
    import rust_interference_engine_b200 as rie

    class At:
        def __init__(self, **kw):
            self.__dict__.update(kw)

    cache = At(ctx=At(device=0), head_dim=64, ptr=None)
    with pytest.raises(ValueError, match="cache: on device 0, the context is on 1"):
        rie.paged_attention(At(device=1), cache, At(n_tok=1), None, 1, None)
