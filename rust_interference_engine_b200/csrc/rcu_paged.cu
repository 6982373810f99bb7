// rcu_paged.cu -- a pool of key / value pages shared by many sequences, the append of new tokens to
// it, and the C entry points of attention over a batch of sequences.
//
// A page holds page_size positions of one sequence, [page][kv head][slot][head_dim] f16, so that a
// head's rows of a page are one stretch of memory. Sequence i's position P lives in page
// pages[i][P / page_size], slot P % page_size. The page numbers, lengths and row offsets are device
// memory: a captured graph replays with whatever they hold by then.
#include <cstring>
#include <new>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"

struct rcu_paged {
    int device = 0;  // not the context: a pool may outlive the one that made it
    uint64_t n_kv = 0, hd = 0, page_size = 0, n_pages = 0;
    uint32_t page_shift = 0;
    void *k = nullptr, *v = nullptr;
    bool owned = false;
    rcu::SeqKvMaps few, tile;  // boxes of 16 rows, and of a page's rows (128 at most)
};

namespace rcu {

// Eight values rounded to f16.
template <typename T>
struct Eight {
    uint4 a, b;  // as loaded (f32: two pieces)
    __device__ __forceinline__ void load(const T *p) {
        a = __ldcs(reinterpret_cast<const uint4 *>(p));
        if constexpr (sizeof(T) == 4) b = __ldcs(reinterpret_cast<const uint4 *>(p) + 1);
    }
    __device__ __forceinline__ uint4 half8() const {
        if constexpr (sizeof(T) == 4) {
            const float4 x = *reinterpret_cast<const float4 *>(&a), y = *reinterpret_cast<const float4 *>(&b);
            return make_uint4(pack2<__half>(x.x, x.y), pack2<__half>(x.z, x.w), pack2<__half>(y.x, y.y), pack2<__half>(y.z, y.w));
        } else if constexpr (std::is_same<T, __half>::value) {
            return a;
        } else {
            const float2 x = unpack2<T>(a.x), y = unpack2<T>(a.y), z = unpack2<T>(a.z), w = unpack2<T>(a.w);
            return make_uint4(pack2<__half>(x.x, x.y), pack2<__half>(y.x, y.y), pack2<__half>(z.x, z.y), pack2<__half>(w.x, w.y));
        }
    }
};

// One warp per (new token, k or v), 8 values a lane and step. The row's first values are on their way
// before the warp looks up where they go (its sequence: rows cu[i + 1] <= t are counted, 32 sequences
// a step; then length and page, one after the other): bound by bytes, if enough of them are in flight.
template <typename T>
__global__ void __launch_bounds__(256) k_paged_store(const SeqView b, const T *__restrict__ k, const T *__restrict__ v,
                                                     uint64_t ld, uint32_t n_kv, uint32_t hd, __half *kp, __half *vp) {
    pdl_wait();
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), t = w >> 1;
    if (t >= b.n_tok) return;
    constexpr int kAhead = 4;
    const T *src = (w & 1 ? v : k) + (uint64_t)t * ld;
    const uint32_t vecs = n_kv * hd / 8, per = hd / 8;
    Eight<T> x[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++)
        if (lane + 32 * j < vecs) x[j].load(src + 8 * (lane + 32 * j));
    uint32_t seq = 0;
    for (uint32_t s0 = 0; s0 < b.n_seq; s0 += 32)
        seq += __popc(__ballot_sync(0xffffffffu, s0 + lane < b.n_seq && b.cu[s0 + lane + 1] <= (int32_t)t));
    if (seq >= b.n_seq) return;  // a row behind the last sequence
    uint32_t first;
    const uint32_t n = seq_rows(b, seq, &first);
    if (t < first || t - first >= n) return;  // offsets out of order (reported)
    // a length that does not fit (reported): rows whose own position is outside the table are dropped
    const int32_t len = b.len[seq];
    seq_len(b, len, n);
    const int64_t pos = (int64_t)len - n + (t - first);
    if (pos < 0 || pos >= (int64_t)b.ld_pages << b.page_shift) return;
    const uint32_t pg = seq_page(b, seq, (uint32_t)(pos >> b.page_shift));
    if (pg == kNoRow) return;
    const uint32_t ps = 1u << b.page_shift, slot = (uint32_t)pos & (ps - 1);
    __half *dst = w & 1 ? vp : kp;
    for (uint32_t i0 = 0; i0 < vecs; i0 += 32 * kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const uint32_t i = i0 + 32 * j + lane;
            if (i >= vecs) continue;
            const uint32_t h = i / per, c = i - h * per;
            const uint64_t row = ((uint64_t)pg * n_kv + h) * ps + slot;
            *reinterpret_cast<uint4 *>(dst + row * hd + 8 * c) = x[j].half8();
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const uint32_t i = i0 + 32 * (kAhead + j) + lane;
            if (i < vecs) x[j].load(src + 8 * i);
        }
    }
}

static uint64_t elem_size(int t) { return t == T_F32 ? 4 : t == T_F16 || t == T_BF16 ? 2 : 0; }
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
// Row strides: whole rows, and every row on a 16-byte boundary.
static int check_rows(rcu_ctx *ctx, const char *what, const void *p, uint64_t ld, uint64_t need, int type) {
    const std::string w(what);
    if (!aligned16(p) || ld * elem_size(type) % 16) return set_err(ctx, RCU_ERR_INVALID, w + ": rows must start on 16-byte boundaries");
    if (ld < need) return set_err(ctx, RCU_ERR_INVALID, w + ": row stride smaller than a row");
    if (ld > (1ull << 32)) return set_err(ctx, RCU_ERR_INVALID, w + ": row stride too large");
    return RCU_OK;
}
static int check_batch(rcu_ctx *ctx, uint64_t n_tok, uint64_t n_seq) {
    if (n_tok == 0 || n_seq == 0) return set_err(ctx, RCU_ERR_RUNTIME, "empty batch");
    // every CTA looks for its sequence among all of them
    if (n_tok > (1u << 30) || n_seq > (1u << 14)) return set_err(ctx, RCU_ERR_INVALID, "batch too large");
    return RCU_OK;
}
static int check_seqs(rcu_ctx *ctx, const rcu_paged *pg, const rcu_seqs *s, SeqView *v) {
    if (!pg || !s || !s->cu || !s->len || !s->pages) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    if (ctx && pg->device != ctx->device) return set_err(ctx, RCU_ERR_INVALID, "paged cache: on another device than the context");
    if (int st = check_batch(ctx, s->n_tok, s->n_seq)) return st;
    if (s->ld_pages == 0 || s->ld_pages > 0x7fffffffull / pg->page_size)
        return set_err(ctx, RCU_ERR_INVALID, "page table: 1 .. 2^31 / page_size pages a sequence");
    *v = SeqView{s->cu, s->len, s->pages, (uint32_t)s->n_seq, (uint32_t)s->n_tok, (uint32_t)s->ld_pages,
                 (uint32_t)pg->n_pages, pg->page_shift, ctx ? ctx->dev_err : nullptr};
    return RCU_OK;
}
static int check_heads(rcu_ctx *ctx, uint64_t n_tok, uint64_t n_head, uint64_t n_kv, uint64_t hd, uint64_t window, float softcap) {
    if (n_head == 0 || n_kv == 0 || n_head % n_kv) return set_err(ctx, RCU_ERR_INVALID, "n_head not divisible by n_head_kv");
    if (hd == 0 || hd % 32 || hd > 256) return set_err(ctx, RCU_ERR_INVALID, "head_dim must be a multiple of 32 and <= 256");
    if (n_tok * (n_head / n_kv) > 0x7fffff00ull) return set_err(ctx, RCU_ERR_INVALID, "batch too large");
    if (n_head > 4096) return set_err(ctx, RCU_ERR_INVALID, "more than 4096 query heads");
    if (window > 0x7fffffffull) return set_err(ctx, RCU_ERR_INVALID, "window must be below 2^31 (0: none)");
    if (!(softcap < 3e38f)) return set_err(ctx, RCU_ERR_INVALID, "softcap must be finite (<= 0: none)");
    return RCU_OK;
}

}  // namespace rcu

using namespace rcu;

extern "C" {

int32_t rcu_paged_create(rcu_ctx *ctx, int32_t kv_type, uint64_t n_head_kv, uint64_t head_dim, uint64_t page_size,
                         uint64_t n_pages, void *k_dev, void *v_dev, rcu_paged **out) {
    RCU_GUARD_BEGIN
    if (!out) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    *out = nullptr;
    if (kv_type < RCU_KV_F16 || kv_type > RCU_KV_TURBO4) return set_err(ctx, RCU_ERR_INVALID, "unknown kv type");
    if (kv_type != RCU_KV_F16) return set_err(ctx, RCU_ERR_UNSUPPORTED, "paged cache: f16 pages only");
    if (n_head_kv == 0 || n_head_kv > 4096 || head_dim == 0 || head_dim % 32 || head_dim > 256)
        return set_err(ctx, RCU_ERR_INVALID, "paged cache: head_dim must be a multiple of 32 and <= 256, n_head_kv 1..4096");
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
        return set_err(ctx, RCU_ERR_INVALID, "paged cache: page_size must be a power of two, 16..1024");
    if (n_pages == 0 || n_pages > 0x7ffffff0ull / (n_head_kv * page_size))
        return set_err(ctx, RCU_ERR_INVALID, "paged cache: n_pages out of range");
    if (!k_dev != !v_dev) return set_err(ctx, RCU_ERR_INVALID, "paged cache: pass both pools or neither");
    if (k_dev && (!aligned16(k_dev) || !aligned16(v_dev)))
        return set_err(ctx, RCU_ERR_INVALID, "paged cache: pools must be 16-byte aligned");
    if (!ctx) return RCU_ERR_INVALID;
    DeviceGuard guard(ctx);
    rcu_paged *pg = new (std::nothrow) rcu_paged();
    if (!pg) return set_err(ctx, RCU_ERR_OOM, "host allocation failed");
    pg->device = ctx->device;
    pg->n_kv = n_head_kv;
    pg->hd = head_dim;
    pg->page_size = page_size;
    pg->n_pages = n_pages;
    while ((1ull << pg->page_shift) < page_size) pg->page_shift++;
    pg->k = k_dev;
    pg->v = v_dev;
    if (!k_dev) {
        const uint64_t bytes = n_pages * n_head_kv * page_size * head_dim * 2;
        pg->owned = true;
        cudaError_t e = cudaMalloc(&pg->k, bytes);
        if (e == cudaSuccess) e = cudaMalloc(&pg->v, bytes);
        if (e == cudaSuccess) e = cudaMemsetAsync(pg->k, 0, bytes, ctx->stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(pg->v, 0, bytes, ctx->stream);
        if (e != cudaSuccess) {
            rcu_paged_free(pg);
            return cuda_err(ctx, e, "paged cache alloc");
        }
    }
    const SeqKvDesc kv{pg->k, pg->v, true, n_pages * n_head_kv * page_size, head_dim, head_dim, nullptr, nullptr};
    int st = seq_kv_maps(ctx, kv, head_dim, n_head_kv, kSeqFewBox, &pg->few);
    if (!st) st = seq_kv_maps(ctx, kv, head_dim, n_head_kv, (uint32_t)std::min<uint64_t>(page_size, kSeqTileBox), &pg->tile);
    if (st) {
        rcu_paged_free(pg);
        return st;
    }
    *out = pg;
    return RCU_OK;
    RCU_GUARD_END(ctx)
}

void rcu_paged_free(rcu_paged *pg) {
    if (!pg) return;
    if (pg->owned) {
        DeviceGuard guard(pg->device);
        cudaFree(pg->k);
        cudaFree(pg->v);
    }
    delete pg;
}

int32_t rcu_paged_device_ptrs(const rcu_paged *pg, void **k_dev, void **v_dev) {
    if (!pg) return RCU_ERR_INVALID;
    if (k_dev) *k_dev = pg->k;
    if (v_dev) *v_dev = pg->v;
    return RCU_OK;
}

int32_t rcu_paged_store(rcu_ctx *ctx, rcu_paged *pg, const rcu_seqs *seqs, const void *k_dev, const void *v_dev,
                        uint32_t type, uint64_t ld) {
    RCU_GUARD_BEGIN
    SeqView b{};
    if (!ctx || !k_dev || !v_dev) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    if (int st = check_seqs(ctx, pg, seqs, &b)) return st;
    if (!elem_size((int)type)) return set_err(ctx, RCU_ERR_UNSUPPORTED, "paged store: rows are f32, f16 or bf16");
    const uint64_t row = pg->n_kv * pg->hd;
    if (int st = check_rows(ctx, "paged store: k", k_dev, ld, row, (int)type)) return st;
    if (int st = check_rows(ctx, "paged store: v", v_dev, ld, row, (int)type)) return st;
    DeviceGuard guard(ctx);
    const dim3 grid((uint32_t)((2ull * b.n_tok + 7) / 8)), block(256);
    const uint32_t n_kv = (uint32_t)pg->n_kv, hd = (uint32_t)pg->hd;
    __half *kp = (__half *)pg->k, *vp = (__half *)pg->v;
    if (type == T_F32)
        RCU_CUDA_TRY(ctx, launch_k(ctx, k_paged_store<float>, grid, block, 0, b, (const float *)k_dev, (const float *)v_dev, ld, n_kv, hd, kp, vp));
    else if (type == T_F16)
        RCU_CUDA_TRY(ctx, launch_k(ctx, k_paged_store<__half>, grid, block, 0, b, (const __half *)k_dev, (const __half *)v_dev, ld, n_kv, hd, kp, vp));
    else
        RCU_CUDA_TRY(ctx, launch_k(ctx, k_paged_store<__nv_bfloat16>, grid, block, 0, b, (const __nv_bfloat16 *)k_dev, (const __nv_bfloat16 *)v_dev, ld, n_kv, hd, kp, vp));
    return RCU_OK;
    RCU_GUARD_END(ctx)
}

int32_t rcu_paged_attention(rcu_ctx *ctx, const rcu_paged *pg, const rcu_seqs *seqs, const void *q_dev, uint32_t type,
                            uint64_t ld_q, uint64_t n_head, uint64_t window, float softcap, void *out_dev, uint64_t ld_out) {
    RCU_GUARD_BEGIN
    SeqAttnParams p{};
    if (!ctx || !q_dev || !out_dev) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    if (int st = check_seqs(ctx, pg, seqs, &p.b)) return st;
    if (int st = check_heads(ctx, seqs->n_tok, n_head, pg->n_kv, pg->hd, window, softcap)) return st;
    if (type != T_F32 && type != T_F16) return set_err(ctx, RCU_ERR_UNSUPPORTED, "paged attention: queries are f32 or f16");
    if (q_dev == out_dev) return set_err(ctx, RCU_ERR_INVALID, "paged attention: out must not be q");
    if (int st = check_rows(ctx, "paged attention: q", q_dev, ld_q, n_head * pg->hd, (int)type)) return st;
    if (int st = check_rows(ctx, "paged attention: out", out_dev, ld_out, n_head * pg->hd, (int)type)) return st;
    p.q = q_dev;
    p.out = out_dev;
    p.k = pg->k;
    p.v = pg->v;
    p.ld_q = ld_q;
    p.ld_out = ld_out;
    p.ld_kv = pg->hd;
    p.kv_rows = (uint32_t)(pg->n_pages * pg->n_kv * pg->page_size);
    p.n_head = (uint32_t)n_head;
    p.n_kv = (uint32_t)pg->n_kv;
    set_group(p, (uint32_t)(n_head / pg->n_kv));
    p.hd = (uint32_t)pg->hd;
    p.window = (uint32_t)window;
    p.softcap = softcap;
    const uint64_t cap = seqs->ld_pages * pg->page_size;
    DeviceGuard guard(ctx);
    const SeqKvDesc kv{pg->k, pg->v, true, p.kv_rows, pg->hd, pg->hd, &pg->few, &pg->tile};
    return launch_seq_attention(ctx, p, (int)type, kv, seqs->max_len ? std::min(seqs->max_len, cap) : cap, seqs->max_new);
    RCU_GUARD_END(ctx)
}

int32_t rcu_packed_attention(rcu_ctx *ctx, const void *q_dev, uint32_t q_type, uint64_t ld_q, const void *k_dev,
                             const void *v_dev, uint32_t kv_elem, uint64_t ld_kv, const int32_t *cu, uint64_t n_seq,
                             uint64_t n_tok, uint64_t max_len, uint64_t n_head, uint64_t n_head_kv, uint64_t head_dim,
                             uint64_t window, float softcap, void *out_dev, uint64_t ld_out) {
    RCU_GUARD_BEGIN
    if (!q_dev || !k_dev || !v_dev || !cu || !out_dev) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    if (int st = check_batch(ctx, n_tok, n_seq)) return st;
    if (int st = check_heads(ctx, n_tok, n_head, n_head_kv, head_dim, window, softcap)) return st;
    if (!((q_type == T_F32 && kv_elem == T_F16) || (q_type == kv_elem && (q_type == T_F16 || q_type == T_BF16))))
        return set_err(ctx, RCU_ERR_UNSUPPORTED, "packed attention: queries are f32 or f16 over f16 keys and values, or bf16 over bf16");
    if (q_dev == out_dev || k_dev == out_dev || v_dev == out_dev)
        return set_err(ctx, RCU_ERR_INVALID, "packed attention: out must not be an input");
    if (int st = check_rows(ctx, "packed attention: q", q_dev, ld_q, n_head * head_dim, (int)q_type)) return st;
    if (int st = check_rows(ctx, "packed attention: k", k_dev, ld_kv, n_head_kv * head_dim, (int)kv_elem)) return st;
    if (int st = check_rows(ctx, "packed attention: v", v_dev, ld_kv, n_head_kv * head_dim, (int)kv_elem)) return st;
    if (int st = check_rows(ctx, "packed attention: out", out_dev, ld_out, n_head * head_dim, (int)q_type)) return st;
    if (!ctx) return RCU_ERR_INVALID;
    SeqAttnParams p{};
    p.b = SeqView{cu, nullptr, nullptr, (uint32_t)n_seq, (uint32_t)n_tok, 0, 0, 0, ctx->dev_err};
    p.q = q_dev;
    p.out = out_dev;
    p.k = k_dev;
    p.v = v_dev;
    p.ld_q = ld_q;
    p.ld_out = ld_out;
    p.ld_kv = ld_kv;
    p.head_kv = head_dim;
    p.kv_rows = (uint32_t)n_tok;
    p.n_head = (uint32_t)n_head;
    p.n_kv = (uint32_t)n_head_kv;
    set_group(p, (uint32_t)(n_head / n_head_kv));
    p.hd = (uint32_t)head_dim;
    p.window = (uint32_t)window;
    p.softcap = softcap;
    DeviceGuard guard(ctx);
    const SeqKvDesc kv{k_dev, v_dev, false, n_tok, ld_kv, head_dim, nullptr, nullptr};
    return launch_seq_attention(ctx, p, (int)q_type, kv, max_len ? std::min(max_len, n_tok) : n_tok, max_len);
    RCU_GUARD_END(ctx)
}

}  // extern "C"
