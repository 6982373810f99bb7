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
