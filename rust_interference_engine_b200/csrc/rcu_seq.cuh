// rcu_seq.cuh -- what the kernels over a batch of sequences share: the batch's description, the
// lookup of a work tile's sequence, element conversion, and the row-by-row attention that the
// tiled kernels fall back to for rows with values that are not finite.
//
// A batch is `n_tok` rows of new tokens; rows cu[i] .. cu[i + 1] - 1 belong to sequence i, whose
// last new token has position len[i] - 1. All of it is device memory that the host never reads, so
// every kernel clamps what it takes from there before it forms an address: a wrong value costs an
// error bit (ERR_BAD_ARG) and rows without a meaning, never an access out of range.
#pragma once
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_tc.cuh"

namespace rcu {

constexpr float kLog2e = 1.4426950408889634f;

struct SeqView {
    const int32_t *cu;     // [n_seq + 1]
    const int32_t *len;    // [n_seq]; nullptr: a sequence is its new tokens (packed prompts)
    const int32_t *pages;  // [n_seq][ld_pages]; nullptr: keys and values are packed rows
    uint32_t n_seq, n_tok, ld_pages, n_pages, page_shift;
    uint32_t *err;
};

// What one sequence of the batch is, clamped to the batch and to its page table.
struct SeqSpan {
    uint32_t seq, first, n_new;  // rows first .. first + n_new - 1
    int32_t len;                 // positions 0 .. len - 1 are in the cache (the host keeps tables below 2^31)
    // position of new token t: negative where a wrong len is shorter than n_new (no keys then)
    __device__ __forceinline__ int32_t pos(uint32_t t) const { return len - (int32_t)n_new + (int32_t)t; }
};

__device__ __forceinline__ uint32_t seq_rows(const SeqView &b, uint32_t s, uint32_t *first) {
    const int32_t c0 = b.cu[s], c1 = b.cu[s + 1];
    const int32_t a0 = min(max(c0, 0), (int32_t)b.n_tok), a1 = min(max(c1, a0), (int32_t)b.n_tok);
    if (a0 != c0 || a1 != c1) atomicOr(b.err, (uint32_t)ERR_BAD_ARG);
    *first = (uint32_t)a0;
    return (uint32_t)(a1 - a0);
}
// The length l that the batch gives for a sequence of n_new new tokens, clamped to its table.
__device__ __forceinline__ int32_t seq_len(const SeqView &b, int32_t l, uint32_t n_new) {
    if (!b.len) return (int32_t)n_new;
    const int32_t cap = (int32_t)(b.ld_pages << b.page_shift);  // the host keeps it below 2^31
    if (l < (int32_t)n_new || l > cap) atomicOr(b.err, (uint32_t)ERR_BAD_ARG);
    return min(max(l, 0), cap);
}

// The sequence that holds work tile `ti` when each sequence takes ceil(n_new * group / rows) tiles,
// and the tile's number within it; false behind the last tile. One whole warp; the scan reads
// 2 * n_seq words that stay in L1 / L2.
__device__ __forceinline__ bool seq_find_tile(const SeqView &b, uint32_t group, uint32_t rows, uint32_t ti, SeqSpan *sp,
                                              uint32_t *tile) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t base = 0;
    for (uint32_t s0 = 0; s0 < b.n_seq; s0 += 32) {
        uint32_t first = 0, n = 0;
        int32_t len = 0;
        if (s0 + lane < b.n_seq) {
            const int32_t l = b.len ? b.len[s0 + lane] : 0;  // on its way together with the offsets
            n = seq_rows(b, s0 + lane, &first);
            len = seq_len(b, l, n);
        }
        const uint32_t t = (n * group + rows - 1) / rows;  // below 2^31: the host checks n_tok * group
        uint32_t inc = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= (uint32_t)d) inc += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, ti - base < inc);  // ti >= base here
        if (hit) {
            const int l = __ffs((int)hit) - 1;
            sp->seq = s0 + l;
            sp->first = __shfl_sync(0xffffffffu, first, l);
            sp->n_new = __shfl_sync(0xffffffffu, n, l);
            *tile = ti - base - (__shfl_sync(0xffffffffu, inc, l) - __shfl_sync(0xffffffffu, t, l));
            sp->len = __shfl_sync(0xffffffffu, len, l);
            return true;
        }
        base += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
}
// An upper bound of the tiles of a batch, from what the host knows.
inline uint64_t seq_tiles_bound(uint64_t n_tok, uint64_t n_seq, uint64_t group, uint64_t rows) {
    return std::min<uint64_t>((n_tok * group + n_seq * (rows - 1)) / rows, n_tok * ((group + rows - 1) / rows));
}

// Row of position `pos` of a sequence in the key / value tensors: a row of the page pool (kv head
// included) or of the packed prompts. Page numbers out of range give `none` and an error bit.
constexpr uint32_t kNoRow = 0xffffffffu;
__device__ __forceinline__ uint32_t seq_page(const SeqView &b, uint32_t seq, uint32_t idx) {
    if (idx >= b.ld_pages) return kNoRow;
    const int32_t pg = b.pages[(uint64_t)seq * b.ld_pages + idx];
    if (pg < 0 || (uint32_t)pg >= b.n_pages) {
        atomicOr(b.err, (uint32_t)ERR_BAD_ARG);
        return kNoRow;
    }
    return (uint32_t)pg;
}
__device__ __forceinline__ uint32_t seq_kv_row(const SeqView &b, const SeqSpan &sp, uint32_t n_kv, uint32_t kvh,
                                               uint32_t pos) {
    if (!b.pages) return sp.first + pos;
    const uint32_t pg = seq_page(b, sp.seq, pos >> b.page_shift);
    if (pg == kNoRow) return kNoRow;
    return ((pg * n_kv + kvh) << b.page_shift) + (pos & ((1u << b.page_shift) - 1));
}

// ---- elements ---------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// Two values rounded to E in one register (lo in the low half).
template <typename E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename E>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 lanes in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t x, y, z, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t x, y, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t x, y, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}
// Largest of three, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A bounded wait whose polls suspend the thread until the phase changes (at most 0.1 ms each), and
// that reads the clock, which takes longer than a wake-up, only between them.
__device__ __forceinline__ bool mbar_wait_spin(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code) {
    constexpr uint32_t kHintNs = 100000;
    if (mbar_try_wait_hint(bar, parity, kHintNs)) return true;
    if (mbar_try_wait_hint(bar, parity, kHintNs)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 16; i++)
            if (mbar_try_wait_hint(bar, parity, kHintNs)) return true;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            atomicOr(err, code);
            return false;
        }
    }
}

// Whether the phase is complete, without suspending the thread.
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// ---- thread-block clusters ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t smem, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// ---- attention over a batch of sequences --------------------------------------------------------
struct SeqAttnParams {
    SeqView b;
    const void *q;
    void *out;
    const void *k, *v;          // for the row-by-row path
    uint64_t ld_q, ld_out;      // elements between rows of q / out
    uint64_t ld_kv, head_kv;    // elements between rows of k / v, and between a row's kv heads
    uint32_t kv_rows;           // rows of k / v
    uint32_t n_head, n_kv, group, hd, window, n_tiles, splits;
    uint64_t group_mul;         // n / group = n * group_mul >> group_shift for n < 2^31
    uint32_t group_shift;
    float softcap;
};

// n < 2^31 divided by the group: with 2^s >= group, group_mul = floor(2^(31 + s) / group) + 1 is off by
// at most one part in 2^(31 + s) / group, which n < 2^31 cannot carry to the next whole number.
__device__ __forceinline__ uint32_t div_group(const SeqAttnParams &p, uint32_t n) {
    return (uint32_t)((uint64_t)n * p.group_mul >> p.group_shift);
}
inline void set_group(SeqAttnParams &p, uint32_t group) {
    uint32_t s = 0;
    while ((1u << s) < group) s++;
    p.group = group;
    p.group_shift = 31 + s;
    p.group_mul = (1ull << (31 + s)) / group + 1;
}

// One output row by one warp, from the formula, over the attended keys alone. The tiled kernels
// multiply the probability 0 of a masked key with its value, which is NaN where that value is an
// infinity or NaN; a row that comes out not finite is made again here, where masked keys are not
// touched. An attended NaN or infinity stays what the formula makes of it. 32 keys a step, four at a
// time: eight lanes take a key, each the 16-byte pieces sub, sub + 8, .. of its row. A row of its own on
// an SM is bound by the latency of its loads (0.16 us a key; taken one a step it was 2.4 us), the
// rows of a tile by the instructions (512 tokens over 12,800 keys, 32 heads, a tile in which every row
// is made again: 14 ms against 175). Unrolled further or with the next rows fetched ahead it was slower.
template <typename T, typename E, int HDP>
__device__ __noinline__ void seq_attn_row(const SeqAttnParams &p, const SeqSpan &sp, uint32_t t, uint32_t kvh, uint32_t g) {
    constexpr int NC = HDP / 64;
    const uint32_t lane = threadIdx.x & 31, sub = lane & 7, grp = lane >> 3, pieces = p.hd / 8, head = kvh * p.group + g;
    const int32_t pos = sp.pos(t), lo = p.window > 0 ? max(pos - (int32_t)p.window + 1, 0) : 0;
    const T *q = reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + t) * p.ld_q + (uint64_t)head * p.hd;
    T *out = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + t) * p.ld_out + (uint64_t)head * p.hd;
    const uint32_t kvo = p.b.pages ? 0u : kvh * (uint32_t)p.head_kv;
    float qv[NC][8], o[NC][8];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            qv[c][i] = sub + 8 * c < pieces ? to_f32(q[8 * (sub + 8 * c) + i]) : 0.0f;
            o[c][i] = 0.0f;
        }
    // this lane's pieces of row r of x; loads without a branch, so that several are in flight
    auto fetch = [&](const void *x, uint32_t r, uint4 (&u)[NC]) {
        const E *src = reinterpret_cast<const E *>(x) + (uint64_t)(r == kNoRow ? 0 : r) * p.ld_kv + kvo;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            u[c] = *reinterpret_cast<const uint4 *>(src + 8 * min(sub + 8 * c, pieces - 1));
            if (r == kNoRow || sub + 8 * c >= pieces) u[c] = make_uint4(0, 0, 0, 0);
        }
    };
    // the group's keys are 4 i + grp, i = 0 .. 7; lane `sub` of it holds key i = sub's row and score
    auto place = [&](int64_t j0) { return j0 + 4 * sub + grp <= pos ? seq_kv_row(p.b, sp, p.n_kv, kvh, (uint32_t)j0 + 4 * sub + grp) : kNoRow; };
    float m = -INFINITY, l = 0.0f;
    uint32_t next = place(lo);
    for (int64_t j0 = lo; j0 <= pos; j0 += 32) {  // pos may be 2^31 - 1
        const bool in = j0 + 4 * sub + grp <= pos;
        const uint32_t row = next;
        next = place(j0 + 32);
        float s = -INFINITY;
#pragma unroll 4
        for (uint32_t i = 0; i < 8; i++) {
            uint4 u[NC];
            fetch(p.k, __shfl_sync(0xffffffffu, row, (lane & 24) | i), u);
            float x = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 f = unpack2<E>(w[k]);
                    x = fmaf(qv[c][2 * k + 1], f.y, fmaf(qv[c][2 * k], f.x, x));
                }
            }
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            if (sub == i && in) s = x;
        }
        if (p.softcap > 0.0f && in) s = p.softcap * tanhf(s / p.softcap);
        float mn = fmaxf(m, s);  // leaves a NaN out
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
        const float a = m == mn ? 1.0f : expf(m - mn), e = s == -INFINITY ? 0.0f : expf(s - mn);
        float sum = e;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        m = mn;
        l = l * a + sum;
        if (l != l) break;  // a score is NaN or +inf: so is the row, whatever follows
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) o[c][i] *= a;
#pragma unroll 4
        for (uint32_t i = 0; i < 8; i++) {
            const float ei = __shfl_sync(0xffffffffu, e, (lane & 24) | i);
            uint4 u[NC];
            fetch(p.v, __shfl_sync(0xffffffffu, row, (lane & 24) | i), u);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 f = unpack2<E>(w[k]);
                    o[c][2 * k] = fmaf(ei, f.x, o[c][2 * k]);
                    o[c][2 * k + 1] = fmaf(ei, f.y, o[c][2 * k + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            o[c][i] += __shfl_xor_sync(0xffffffffu, o[c][i], 8);
            o[c][i] += __shfl_xor_sync(0xffffffffu, o[c][i], 16);
            if (grp == 0 && sub + 8 * c < pieces) out[8 * (sub + 8 * c) + i] = from_f32<T>(lo > pos ? 0.0f : o[c][i] / l);
        }
}
// Whether a row that came out not finite, with the largest score m (in units of log2) and the sum l, is
// its answer already. A masked score adds 0 to the sum whatever it is, so that a NaN there is from an
// attended score that is NaN or +inf. Not so where m overflowed; nor for f32 queries, whose two parts
// make NaN of a score of -inf: those rows are made again.
template <typename T>
__device__ __forceinline__ bool seq_row_settled(float m, float l) {
    return !std::is_same<T, float>::value && l != l && m < INFINITY;
}

// ---- host ---------------------------------------------------------------------------------------
// Tensor maps of k and v with boxes of `box` rows of 64 elements (128-byte swizzle).
struct SeqKvMaps {
    CUtensorMap k, v;
};
inline int seq_kv_maps(rcu_ctx *ctx, const SeqKvDesc &kv, uint64_t hd, uint64_t n_kv, uint32_t box, SeqKvMaps *m) {
    for (int i = 0; i < 2; i++)
        if (int st = make_map_3d(ctx, i ? &m->v : &m->k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, i ? kv.v : kv.k, hd, kv.pages ? 1 : n_kv,
                                 kv.rows, kv.head_stride * 2, kv.row_stride * 2, 64, 1, box, CU_TENSOR_MAP_SWIZZLE_128B))
            return st;
    return RCU_OK;
}
// The maps that a launch with boxes of `box` rows uses: the pool's own, made with it, or new ones.
inline int seq_pick_maps(rcu_ctx *ctx, const SeqAttnParams &p, const SeqKvDesc &kv, uint32_t box, const SeqKvMaps *made,
                         SeqKvMaps *room, const SeqKvMaps **use) {
    *use = made;
    if (made) return RCU_OK;
    *use = room;
    return seq_kv_maps(ctx, kv, p.hd, p.n_kv, box, room);
}
// Shared memory and cluster attributes of a kernel, set by its first use on a device.
template <auto Kern>
inline int prepare_cluster_k(rcu_ctx *ctx, size_t smem) {
    static std::atomic<uint64_t> ready{0};  // devices, of the first 64
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (ctx->device >= 64 || !(ready.load(std::memory_order_acquire) & bit)) {
        const void *fn = reinterpret_cast<const void *>(Kern);
        RCU_CUDA_TRY(ctx, prefer_max_shared(fn));
        RCU_CUDA_TRY(ctx, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        RCU_CUDA_TRY(ctx, cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ready.fetch_or(bit, std::memory_order_release);
    }
    return RCU_OK;
}
// Clusters of 2^e CTAs (e below 4) of a kernel that the device runs at the same time.
template <auto Kern>
inline int cluster_slots(rcu_ctx *ctx, uint32_t threads, size_t smem, int e, int *slots) {
    static std::atomic<int> known[64][4];
    const bool keep = ctx->device < 64;
    if (keep && (*slots = known[ctx->device][e].load(std::memory_order_relaxed)) > 0) return RCU_OK;
    if (int st = prepare_cluster_k<Kern>(ctx, smem)) return st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << e;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << e);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    RCU_CUDA_TRY(ctx, cudaOccupancyMaxActiveClusters(slots, Kern, &cfg));
    *slots = std::max(*slots, 1);
    if (keep) known[ctx->device][e].store(*slots, std::memory_order_relaxed);
    return RCU_OK;
}
// Clusters of cs CTAs, programmatic dependent launch as launch_k.
template <auto Kern, typename... Args>
inline int launch_cluster_k(rcu_ctx *ctx, uint32_t grid, uint32_t threads, size_t smem, uint32_t cs, const Args &...args) {
    if (int st = prepare_cluster_k<Kern>(ctx, smem)) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (cs > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = cs;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        na++;
    }
    if (ctx->pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    RCU_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, Kern, args...));
    return RCU_OK;
}

}  // namespace rcu
