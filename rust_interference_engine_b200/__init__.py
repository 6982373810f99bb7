"""B200 (sm_100a) implementation of the Rust Inference Engine's quantized-matmul and
turbo4 KV-cache hot path.

The compute lives in librie_cuda.so behind a C ABI (include/rie_cuda.h). This module is
the host-side mirror of the reference's kernel-level interface, with the same names and
argument meaning:

  reference (crates/rie-core/src/...)           here
  quant::GgmlType / ActFormat                    GgmlType / ActFormat
  tensor::Weight (+ slice_rows)                  Weight
  kernels::matmul::QuantActs::prepare            QuantActs.prepare
  kernels::matmul::{MatmulJob, matmul, matmul_multi, formats_for}
  turbo::{row_bytes_4, quantize_4, Rotation}     turbo.row_bytes_4 / quantize_4 / rotate
  model::cpu::{KvType, LayerCache, attention}    KvType / LayerCache / attention

Several sequences at once, which the reference's caches and samplers do not hold: PagedCache and
SeqBatch with paged_attention, packed_attention over whole prompts, and logprobs.

Device memory is passed as torch CUDA tensors (or raw device pointers); torch is only the
allocator and stream plumbing. There is no CPU fallback: without the CUDA library or a
GPU every call raises.
"""
from __future__ import annotations

import ctypes as C
import enum
from dataclasses import dataclass
from typing import Iterable, Sequence

from . import _lib
from ._lib import RcuError, RcuJob, RcuSeqs

__all__ = ["GgmlType", "ActFormat", "KvType", "Rounding", "PrefillGemm", "Context", "Weight", "QuantActs", "MatmulJob",
           "matmul", "matmul_multi", "matmul_f32_static", "formats_for", "block_sums", "quantize_weight", "LayerCache",
           "attention", "PagedCache", "SeqBatch", "paged_attention", "packed_attention", "logprobs", "turbo", "RcuError"]


class GgmlType(enum.IntEnum):  # quant/mod.rs:15-68 (GGUF ids)
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q4_1 = 3
    Q5_0 = 6
    Q5_1 = 7
    Q8_0 = 8
    Q2_K = 10
    Q3_K = 11
    Q4_K = 12
    Q5_K = 13
    Q6_K = 14
    BF16 = 30

    @property
    def block_size(self) -> int:
        if self in (GgmlType.F32, GgmlType.F16, GgmlType.BF16):
            return 1
        return 32 if self in (GgmlType.Q4_0, GgmlType.Q4_1, GgmlType.Q5_0, GgmlType.Q5_1, GgmlType.Q8_0) else 256

    def row_bytes(self, n: int) -> int:
        return int(_lib.load().rcu_row_bytes(int(self), n))

    def act_format(self) -> "ActFormat":  # quant/mod.rs:118-124
        if self in (GgmlType.Q4_0, GgmlType.Q4_1, GgmlType.Q5_0, GgmlType.Q5_1, GgmlType.Q8_0):
            return ActFormat.Q8_0
        if self in (GgmlType.Q4_K, GgmlType.Q5_K, GgmlType.Q6_K, GgmlType.Q2_K, GgmlType.Q3_K):
            return ActFormat.Q8K
        return ActFormat.F32


class ActFormat(enum.IntFlag):  # quant/mod.rs:127-132 (as flags of the C ABI)
    F32 = 1
    Q8_0 = 2
    Q8K = 4


class KvType(enum.IntEnum):  # model/cpu.rs:12-36
    F16 = 0
    Q8_0 = 1
    Turbo4 = 2

    @staticmethod
    def parse(s: str) -> "KvType | None":
        return {"f16": KvType.F16, "q8": KvType.Q8_0, "q8_0": KvType.Q8_0, "turbo4": KvType.Turbo4,
                "tq4": KvType.Turbo4, "turbo": KvType.Turbo4}.get(s.lower())


class Rounding(enum.IntEnum):
    NEAREST_EVEN = 0  # AVX2 / NEON tiers of the reference
    HALF_AWAY = 1     # scalar tier (RIE_DISABLE=simd)


class PrefillGemm(enum.IntEnum):
    F16 = 0  # every weight type: f16-dequantized operands on the tensor cores (default)
    I8 = 1   # Q4_0: int8 MMA with the exact per-block int32 sums


def _check(ctx_ptr, status: int):
    if status != 0:
        msg = _lib.load().rcu_last_error(ctx_ptr) if ctx_ptr else b""
        raise RcuError(status, (msg or b"").decode(errors="replace"))


def _dptr(x) -> int:
    """Device address of a torch CUDA tensor (or a raw integer pointer)."""
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        if not x.is_cuda:
            raise ValueError("expected a CUDA tensor")
        if not x.is_contiguous():
            raise ValueError("expected a contiguous tensor")
        return int(x.data_ptr())
    raise TypeError(f"not a device buffer: {type(x)}")


class Context:
    """A device + stream the library issues work on (replaces the CPU ThreadPool)."""

    def __init__(self, device: int = 0, stream=None, rounding: Rounding = Rounding.NEAREST_EVEN):
        lib = _lib.load()
        self._lib = lib
        ptr = C.c_void_p()
        err = C.create_string_buffer(512)
        handle = _stream_handle(stream)
        st = lib.rcu_ctx_create(device, handle, C.byref(ptr), err, 512)
        if st != 0:
            raise RcuError(st, err.value.decode(errors="replace"))
        self.ptr = ptr
        self.device = device
        self.set_rounding(rounding)

    def set_stream(self, stream) -> None:
        _check(self.ptr, self._lib.rcu_set_stream(self.ptr, _stream_handle(stream)))

    def set_rounding(self, mode: Rounding) -> None:
        _check(self.ptr, self._lib.rcu_set_rounding(self.ptr, int(mode)))

    def set_static_weights(self, on: bool) -> None:
        """Promise that weights are never written by a kernel after upload (lets matmuls
        stream them before the previous kernel finishes)."""
        _check(self.ptr, self._lib.rcu_set_static_weights(self.ptr, int(bool(on))))

    def set_wait_limit_ms(self, ms: int) -> None:
        """Limit of the device-side waits on other ranks (the fused all-reduce)."""
        _check(self.ptr, self._lib.rcu_set_wait_limit_ms(self.ptr, int(ms)))

    def set_prefill_gemm(self, kind: "PrefillGemm") -> None:
        _check(self.ptr, self._lib.rcu_set_prefill_gemm(self.ptr, int(kind)))

    def sync(self) -> None:
        _check(self.ptr, self._lib.rcu_sync(self.ptr))

    def device_error_bits(self) -> int:
        bits = C.c_uint32(0)
        st = self._lib.rcu_check_device(self.ptr, C.byref(bits))
        if st != 0 and not bits.value:
            _check(self.ptr, st)
        return int(bits.value)

    def close(self) -> None:
        if getattr(self, "ptr", None):
            self._lib.rcu_ctx_destroy(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _stream_handle(stream) -> C.c_void_p:
    if stream is None:
        return C.c_void_p(0)
    if isinstance(stream, int):
        return C.c_void_p(stream)
    return C.c_void_p(int(stream.cuda_stream))


class Weight:
    """A rows x cols weight in GGUF block layout on the device (tensor.rs:6-98)."""

    def __init__(self, ctx: Context, ptr: C.c_void_p, ty: GgmlType, rows: int, cols: int, keep=None):
        self.ctx, self.ptr, self.ty, self.rows, self.cols = ctx, ptr, GgmlType(ty), rows, cols
        self._keep = keep

    @classmethod
    def upload(cls, ctx: Context, ty: GgmlType, rows: int, cols: int, data) -> "Weight":
        """Copy raw GGUF block bytes (bytes / numpy uint8 array) to the device."""
        import numpy as np
        buf = np.ascontiguousarray(np.frombuffer(data, dtype=np.uint8) if isinstance(data, (bytes, bytearray))
                                   else np.asarray(data, dtype=np.uint8))
        if buf.size != rows * GgmlType(ty).row_bytes(cols):
            raise ValueError("weight size mismatch")
        ptr = C.c_void_p()
        _check(ctx.ptr, ctx._lib.rcu_weight_upload(ctx.ptr, int(ty), rows, cols, buf.ctypes.data_as(C.c_void_p),
                                                   C.byref(ptr)))
        return cls(ctx, ptr, ty, rows, cols)

    @classmethod
    def view(cls, ctx: Context, ty: GgmlType, rows: int, cols: int, dev) -> "Weight":
        """Zero-copy view of GGUF bytes already on the device (16-byte aligned)."""
        ptr = C.c_void_p()
        _check(ctx.ptr, ctx._lib.rcu_weight_view(ctx.ptr, int(ty), rows, cols, C.c_void_p(_dptr(dev)), C.byref(ptr)))
        return cls(ctx, ptr, ty, rows, cols, keep=dev)

    def slice_rows(self, start: int, n: int) -> "Weight":
        ptr = C.c_void_p()
        _check(self.ctx.ptr, self.ctx._lib.rcu_weight_slice_rows(self.ptr, start, n, C.byref(ptr)))
        return Weight(self.ctx, ptr, self.ty, n, self.cols, keep=self)

    @property
    def row_bytes(self) -> int:
        return self.ty.row_bytes(self.cols)

    def data_ptr(self) -> int:
        return int(self.ctx._lib.rcu_weight_device_ptr(self.ptr) or 0)

    def free(self) -> None:
        if getattr(self, "ptr", None):
            self.ctx._lib.rcu_weight_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def formats_for(ws: Iterable[Weight]) -> ActFormat:  # matmul.rs:119-128
    f = ActFormat(0)
    for w in ws:
        f |= w.ty.act_format()
    return f


class QuantActs:
    """One batch of quantized activations on the device (matmul.rs:19-97)."""

    def __init__(self, ctx: Context, max_tok: int, max_k: int):
        self.ctx = ctx
        self.ptr = C.c_void_p()
        _check(ctx.ptr, ctx._lib.rcu_acts_create(ctx.ptr, max_tok, max_k, C.byref(self.ptr)))
        self.n_tok = 0
        self.k = 0

    def prepare(self, x, n_tok: int, k: int, formats: ActFormat) -> None:
        """Quantize x (n_tok x k f32, device) once into every format in `formats`."""
        fl = int(formats) & ~int(ActFormat.F32)
        _check(self.ctx.ptr, self.ctx._lib.rcu_acts_prepare(self.ctx.ptr, self.ptr, C.c_void_p(_dptr(x)), n_tok, k, fl))
        self.n_tok, self.k = n_tok, k

    def export(self, fmt: ActFormat):
        """Blocks in the reference's layout (BlockQ8_0: 48 B, BlockQ8K: 304 B) as numpy bytes."""
        import numpy as np
        bs, sz = (32, 48) if fmt == ActFormat.Q8_0 else (256, 304)
        out = np.zeros(self.n_tok * (self.k // bs) * sz, dtype=np.uint8)
        _check(self.ctx.ptr, self.ctx._lib.rcu_acts_export(self.ctx.ptr, self.ptr, int(fmt),
                                                           out.ctypes.data_as(C.c_void_p)))
        return out

    def free(self) -> None:
        if getattr(self, "ptr", None):
            self.ctx._lib.rcu_acts_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


@dataclass
class MatmulJob:  # matmul.rs:110-116
    w: Weight
    out: object  # device tensor / pointer: out[t * ld + r]
    ld: int | None = None


def matmul_multi(ctx: Context, acts: QuantActs, jobs: Sequence[MatmulJob]) -> None:
    """Several matmuls sharing one activation batch, in one launch (matmul.rs:136-176)."""
    arr = (RcuJob * len(jobs))()
    for i, j in enumerate(jobs):
        arr[i].w = j.w.ptr.value
        arr[i].out = _dptr(j.out)
        arr[i].ld = j.ld if j.ld is not None else j.w.rows
    _check(ctx.ptr, ctx._lib.rcu_matmul_multi(ctx.ptr, acts.ptr, arr, len(jobs)))


def matmul(ctx: Context, acts: QuantActs, w: Weight, out) -> None:  # matmul.rs:130-133
    matmul_multi(ctx, acts, [MatmulJob(w, out, w.rows)])


def matmul_f32_static(ctx: Context, w: Weight, x, n_tok: int, out, ld: int | None = None) -> None:
    """W . X for f32 activations without allocating device memory.

    For callers that cannot cudaMalloc when they run a matmul (their device memory belongs
    to a pool such as PyTorch's caching allocator, or allocation would stall a decode step):
    the activations are quantized into a fixed scratch area inside the library. At most 8
    tokens and rows of at most 16384 values; calls that overlap on the GPU share that
    scratch and must not run concurrently."""
    _check(ctx.ptr, ctx._lib.rcu_matmul_f32_static(ctx.ptr, w.ptr, C.c_void_p(_dptr(x)), n_tok,
                                                   C.c_void_p(_dptr(out)), w.rows if ld is None else ld))


def quantize_weight(ctx: Context, ty: GgmlType, rows: int, cols: int, x, out, ld: int | None = None) -> None:
    """f32 weights (rows x cols, row stride ld, device) -> GGUF blocks of `ty` in `out` (device,
    rows x row_bytes(cols) bytes). Q8_0 / Q4_0 follow the reference's quantizers
    (quant/mod.rs:262-307); the other block types use this library's own rules."""
    _check(ctx.ptr, ctx._lib.rcu_quantize_weight(ctx.ptr, int(ty), rows, cols, C.c_void_p(_dptr(x)),
                                                 cols if ld is None else ld, C.c_void_p(_dptr(out))))


def block_sums(ctx: Context, acts: QuantActs, w: Weight, row: int, tok: int, out) -> None:
    """Exact per-block int32 sums of W[row] . X[tok] into a device int32 buffer."""
    _check(ctx.ptr, ctx._lib.rcu_block_sums(ctx.ptr, acts.ptr, w.ptr, row, tok, C.c_void_p(_dptr(out))))


def matmul_block_sums(ctx: Context, acts: QuantActs, w: Weight, out, sums, kernel: int) -> None:
    """Row 0 of acts times every row of w on the named GEMV (0: lane kernel, 1: tensor-core
    kernel), f32 results in `out` and the exact per-block int32 sums that kernel formed in
    `sums` (rows x blocks per row, the block_sums layout; device buffers)."""
    _check(ctx.ptr, ctx._lib.rcu_matmul_block_sums(ctx.ptr, acts.ptr, w.ptr, C.c_void_p(_dptr(out)),
                                                   C.c_void_p(_dptr(sums)), int(kernel)))


class LayerCache:
    """One layer's KV cache, layout [kv_head][slot][row] (model/cpu.rs:38-50)."""

    def __init__(self, ctx: Context, ty: KvType, n_head_kv: int, head_dim: int, slots: int):
        self.ctx, self.ty, self.n_head_kv, self.head_dim, self.slots = ctx, KvType(ty), n_head_kv, head_dim, slots
        self.ptr = C.c_void_p()
        _check(ctx.ptr, ctx._lib.rcu_kv_create(ctx.ptr, int(ty), n_head_kv, head_dim, slots, C.byref(self.ptr)))

    @property
    def row_bytes(self) -> int:
        if self.ty == KvType.F16:
            return 2 * self.head_dim
        if self.ty == KvType.Q8_0:
            return self.head_dim // 32 * 34
        return turbo.row_bytes_4(self.head_dim)

    def store(self, k, v, n_tok: int, pos0: int) -> None:
        """Append n_tok tokens' keys/values (n_tok x n_head_kv*head_dim f32, device)."""
        _check(self.ctx.ptr, self.ctx._lib.rcu_kv_store(self.ctx.ptr, self.ptr, C.c_void_p(_dptr(k)),
                                                        C.c_void_p(_dptr(v)), n_tok, pos0))

    def export(self):
        import numpy as np
        n = self.n_head_kv * self.slots * self.row_bytes
        k = np.zeros(n, dtype=np.uint8)
        v = np.zeros(n, dtype=np.uint8)
        _check(self.ctx.ptr, self.ctx._lib.rcu_kv_export(self.ctx.ptr, self.ptr, k.ctypes.data_as(C.c_void_p),
                                                         v.ctypes.data_as(C.c_void_p)))
        return k.reshape(self.n_head_kv * self.slots, -1), v.reshape(self.n_head_kv * self.slots, -1)

    def import_(self, k, v) -> None:
        import numpy as np
        k = np.ascontiguousarray(k, dtype=np.uint8)
        v = np.ascontiguousarray(v, dtype=np.uint8)
        _check(self.ctx.ptr, self.ctx._lib.rcu_kv_import(self.ctx.ptr, self.ptr, k.ctypes.data_as(C.c_void_p),
                                                         v.ctypes.data_as(C.c_void_p)))

    def free(self) -> None:
        if getattr(self, "ptr", None):
            self.ctx._lib.rcu_kv_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def attention(ctx: Context, cache: LayerCache, q, n_tok: int, n_head: int, pos0: int, out, window: int = 0,
              softcap: float | None = None) -> None:
    """Causal GQA attention over the cache (model/cpu.rs:552-634); q already x attn_scale."""
    _check(ctx.ptr, ctx._lib.rcu_attention(ctx.ptr, cache.ptr, C.c_void_p(_dptr(q)), n_tok, n_head, pos0, window,
                                           float(softcap or 0.0), C.c_void_p(_dptr(out))))


_ELEM: dict = {}   # torch dtype -> GGUF type id
_DTYPE: dict = {}  # name -> torch dtype


def _torch_types() -> None:
    import torch
    _ELEM.update({torch.float32: int(GgmlType.F32), torch.float16: int(GgmlType.F16), torch.bfloat16: int(GgmlType.BF16)})
    _DTYPE.update(f32=torch.float32, i32=torch.int32)


def _elem(x) -> int:
    """GGUF type id of a tensor's elements."""
    ty = _ELEM.get(x.dtype)
    if ty is None:
        if not _ELEM:
            _torch_types()
            return _elem(x)
        raise ValueError(f"f32, f16 or bf16 values expected, not {x.dtype}")
    return ty


def _elsewhere(ctx: Context, x, what: str):
    return ValueError(f"{what}: expected a CUDA tensor" if x.get_device() < 0 else
                      f"{what}: on device {x.get_device()}, the context is on {ctx.device}")


def _on(ctx: Context, x, what: str) -> int:
    """Device address of a tensor that must live on the context's device."""
    if x.get_device() != ctx.device:  # -1: not a CUDA tensor
        raise _elsewhere(ctx, x, what)
    return x.data_ptr()


def _rows(ctx: Context, x, n: int, width: int, what: str):
    """(address, type, row stride) of n rows of `width` values; the rows may be slices of wider
    ones, their values must be contiguous. (One call for each tensor of a small launch: nothing in
    here is done twice.)"""
    if x.shape != (n, width):
        raise ValueError(f"{what}: expected {n} x {width} values, not {tuple(x.shape)}")
    ld, step = x.stride()
    if step != 1 and width > 1:
        raise ValueError(f"{what}: the values of a row must be contiguous")
    if x.get_device() != ctx.device:
        raise _elsewhere(ctx, x, what)
    ty = _ELEM.get(x.dtype)
    return x.data_ptr(), _elem(x) if ty is None else ty, ld if n > 1 else max(ld, width)


def _vector(ctx: Context, x, dtype: str, shape, what: str) -> int:
    if not _DTYPE:
        _torch_types()
    if x.dtype is not _DTYPE[dtype] or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous {dtype} tensor of shape {tuple(shape)}, not {x.dtype} {tuple(x.shape)}")
    if x.get_device() != ctx.device:
        raise _elsewhere(ctx, x, what)
    return x.data_ptr()


class SeqBatch:
    """The new tokens of several sequences (rcu_seqs): rows cu[i] .. cu[i + 1] - 1 of a batch of
    n_tok rows are sequence i's, len[i] counts its positions with them, pages[i] lists its pages.

    cu (n_seq + 1), len (n_seq) and pages (n_seq x width) are int32 CUDA tensors; the kernels read
    them when they run, so a captured graph replays with what they hold then. max_len (the longest
    len) and max_new (the most new tokens of one sequence), when the program knows them, shape the
    launches; results differ by roundings alone. Give max_new where sequences have a few new tokens
    each: without it one of them is taken to have them all."""

    def __init__(self, cu, len, pages, n_tok: int, max_len: int = 0, max_new: int = 0):  # noqa: A002
        for x, what, dims in ((cu, "cu", 1), (len, "len", 1), (pages, "pages", 2)):
            if str(x.dtype) != "torch.int32" or x.dim() != dims or not x.is_contiguous():
                raise ValueError(f"{what}: expected a contiguous {dims}-dimensional int32 tensor")
        for x, what in ((cu, "cu"), (len, "len"), (pages, "pages")):
            if not x.is_cuda or x.get_device() != cu.get_device():
                raise ValueError(f"{what}: expected a CUDA tensor on the batch's device")
        n_seq = len.shape[0]
        if cu.shape[0] != n_seq + 1 or pages.shape[0] != n_seq:
            raise ValueError(f"{n_seq} sequences need {n_seq + 1} offsets and {n_seq} rows of pages")
        if n_tok < 0 or max_len < 0 or max_new < 0:
            raise ValueError("n_tok, max_len and max_new must not be negative")
        self.n_seq, self.n_tok, self.device = n_seq, n_tok, cu.get_device()
        self._keep = (cu, len, pages)
        self._c = RcuSeqs(cu.data_ptr(), len.data_ptr(), pages.data_ptr(), n_seq, n_tok, pages.shape[1], max_len, max_new)
        self._ref = C.byref(self._c)

    def _on(self, ctx: Context):
        if self.device != ctx.device:
            raise ValueError(f"batch: on device {self.device}, the context is on {ctx.device}")
        return self._ref


class PagedCache:
    """A pool of key / value pages for any number of sequences, [page][kv_head][slot][head_dim] f16
    (rcu_paged_create). k and v: the program's own pools (f16 CUDA tensors of that many values),
    or the library's when left out."""

    def __init__(self, ctx: Context, n_head_kv: int, head_dim: int, page_size: int, n_pages: int,
                 ty: KvType = KvType.F16, k=None, v=None):
        self.ctx, self.ty, self.n_head_kv, self.head_dim = ctx, KvType(ty), n_head_kv, head_dim
        self.page_size, self.n_pages = page_size, n_pages
        self.ptr = C.c_void_p()
        if (k is None) != (v is None):
            raise ValueError("pass both pools or neither")
        for x, what in ((k, "k"), (v, "v")):
            if x is None:
                continue
            if _elem(x) != GgmlType.F16 or not x.is_contiguous() or x.numel() != n_pages * n_head_kv * page_size * head_dim:
                raise ValueError(f"{what}: expected {n_pages * n_head_kv * page_size * head_dim} contiguous f16 values")
            _on(ctx, x, what)
        self._keep = (k, v)
        _check(ctx.ptr, ctx._lib.rcu_paged_create(ctx.ptr, int(ty), n_head_kv, head_dim, page_size, n_pages,
                                                  k.data_ptr() if k is not None else None,
                                                  v.data_ptr() if v is not None else None, C.byref(self.ptr)))

    def store(self, batch: SeqBatch, k, v) -> None:
        """Append the batch's keys and values (n_tok x n_head_kv*head_dim f32, f16 or bf16)."""
        ctx, width = self.ctx, self.n_head_kv * self.head_dim
        kp, ty, ld = _rows(ctx, k, batch.n_tok, width, "k")
        vp, ty_v, ld_v = _rows(ctx, v, batch.n_tok, width, "v")
        if ty != ty_v or ld != ld_v:
            raise ValueError("k and v must have the same type and row stride")
        _check(ctx.ptr, ctx._lib.rcu_paged_store(ctx.ptr, self.ptr, batch._on(ctx), kp, vp, ty, ld))

    def data_ptrs(self):
        k, v = C.c_void_p(), C.c_void_p()
        _check(self.ctx.ptr, self.ctx._lib.rcu_paged_device_ptrs(self.ptr, C.byref(k), C.byref(v)))
        return int(k.value), int(v.value)

    def free(self) -> None:
        if getattr(self, "ptr", None):
            self.ctx._lib.rcu_paged_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def paged_attention(ctx: Context, cache: PagedCache, batch: SeqBatch, q, n_head: int, out, window: int = 0,
                    softcap: float | None = None) -> None:
    """Causal GQA attention of the batch's new tokens over their pages (rcu_paged_attention); q
    (n_tok x n_head*head_dim, f32 or f16) already x attn_scale, out the same type."""
    if cache.ctx.device != ctx.device:
        raise ValueError(f"cache: on device {cache.ctx.device}, the context is on {ctx.device}")
    width = n_head * cache.head_dim
    qp, ty, ld = _rows(ctx, q, batch.n_tok, width, "q")
    op, ty_o, ld_o = _rows(ctx, out, batch.n_tok, width, "out")
    if ty_o != ty:
        raise ValueError("q and out must have the same type")
    _check(ctx.ptr, ctx._lib.rcu_paged_attention(ctx.ptr, cache.ptr, batch._on(ctx), qp, ty, ld, n_head, window,
                                                 softcap or 0.0, op, ld_o))


def packed_attention(ctx: Context, q, k, v, cu, n_head: int, n_head_kv: int, head_dim: int, out, window: int = 0,
                     softcap: float | None = None, max_len: int = 0) -> None:
    """Causal GQA attention within each of the packed prompts, rows cu[i] .. cu[i + 1] - 1
    (rcu_packed_attention): q (already x attn_scale) and out f32 or f16 over f16 k and v, or all bf16."""
    n_tok = q.shape[0]
    qp, ty, ld = _rows(ctx, q, n_tok, n_head * head_dim, "q")
    kp, ty_k, ld_k = _rows(ctx, k, n_tok, n_head_kv * head_dim, "k")
    vp, ty_v, ld_v = _rows(ctx, v, n_tok, n_head_kv * head_dim, "v")
    op, ty_o, ld_o = _rows(ctx, out, n_tok, n_head * head_dim, "out")
    if ty_k != ty_v or ld_k != ld_v or ty_o != ty:
        raise ValueError("k and v must have the same type and row stride, q and out the same type")
    n_seq = cu.shape[0] - 1
    _check(ctx.ptr, ctx._lib.rcu_packed_attention(ctx.ptr, qp, ty, ld, kp, vp, ty_k, ld_k,
                                                  _vector(ctx, cu, "i32", (n_seq + 1,), "cu"), n_seq, n_tok,
                                                  max_len, n_head, n_head_kv, head_dim, window, softcap or 0.0, op, ld_o))


def logprobs(ctx: Context, logits, targets=None, logprob=None, entropy=None, top_ids=None, top_logprobs=None) -> None:
    """Scores of rows of logits (n_rows x n_vocab, f32, f16 or bf16) into the tensors that are given
    (rcu_logprobs): logprob of targets (int32, -1: none), entropy (both n_rows f32), and the
    largest top_k as top_ids (n_rows x top_k int32) and top_logprobs (n_rows x top_k f32)."""
    if logits.dim() != 2:
        raise ValueError(f"logits: expected rows, not {tuple(logits.shape)}")
    n, width = logits.shape
    lp, ty, ld = _rows(ctx, logits, n, width, "logits")
    if (targets is None) != (logprob is None) or (top_ids is None) != (top_logprobs is None):
        raise ValueError("pass targets with logprob, and top_ids with top_logprobs")
    top_k = 0 if top_ids is None else top_ids.shape[-1]

    def arg(x, dtype, shape, what):
        return None if x is None else _vector(ctx, x, dtype, shape, what)

    ids = arg(top_ids, "i32", (n, top_k), "top_ids")
    tlp = arg(top_logprobs, "f32", (n, top_k), "top_logprobs")
    _check(ctx.ptr, ctx._lib.rcu_logprobs(ctx.ptr, lp, ty, n, width, ld, arg(targets, "i32", (n,), "targets"),
                                          arg(logprob, "f32", (n,), "logprob"),
                                          arg(entropy, "f32", (n,), "entropy"), top_k, ids if top_k else None,
                                          tlp if top_k else None))


class turbo:  # noqa: N801  (namespace mirroring turbo.rs)
    KV_SEED = 0x7542_6F51_7561_6E74

    @staticmethod
    def row_bytes_4(d: int) -> int:
        return int(_lib.load().rcu_turbo4_row_bytes(d))

    @staticmethod
    def quantize_4(ctx: Context, x, n_rows: int, d: int, out) -> None:
        """Rotate + 4-bit encode n_rows rows of d f32 (device) into reference-format rows."""
        _check(ctx.ptr, ctx._lib.rcu_turbo4_quantize(ctx.ptr, C.c_void_p(_dptr(x)), n_rows, d, C.c_void_p(_dptr(out))))

    @staticmethod
    def rotate(ctx: Context, x, n_rows: int, d: int, inverse: bool = False) -> None:
        _check(ctx.ptr, ctx._lib.rcu_turbo4_rotate(ctx.ptr, C.c_void_p(_dptr(x)), n_rows, d, int(inverse)))
