// rcu_attn_tile.cu -- attention of a batch of sequences with many query rows per KV head (chunks,
// whole prompts) on the 5th-generation tensor cores. Formula and batch as in rcu_attn_seq.cu.
//
// A CTA takes 256 query rows (token, head of the group) of one sequence and KV head as two tiles of
// 128 rows, and walks the attended keys in blocks of 128:
//   * warp 8     producer: K and V blocks by tiled TMA (128-byte swizzle) into a ring of stages; a
//                page may be smaller than a block (one box per page) or larger;
//   * warp 9     owns tensor memory; one thread issues S_t = Q_t K^T (M 128, N 128) and O_t += P_t V
//                (P read from tensor memory, V in its own layout as an MN-major operand);
//   * warps 0-3, 4-7  softmax of tile 0 / 1, one thread per query row: S out of tensor memory, mask,
//                running maximum and sum in f32, P = 2^(s - m) back as packed 16-bit values over S.
// While one tile's warps are at their softmax, the tensor core works on the other tile.
// 16-bit queries: O stays in tensor memory; it is rescaled only when a row's maximum has grown by
// more than 2^kTlLazy since its last rescale (p then is at most 2^(kTlLazy + kTlShift)).
// f32 queries: q (scaled by a power of two per row) and p are each split into two f16 parts, so each
// product is two MMAs; O is added up in registers block by block, because a long chain of additions
// inside the tensor core, which does not round to nearest, would drift (8e-6 at 12k keys).
// Few tiles over a long context: a cluster of CTAs splits the keys and joins through distributed
// shared memory. All waits are bounded; TMEM is freed on every path.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"
#include "rcu_tc.cuh"

namespace rcu {

constexpr int kTlRows = 256;       // query rows per CTA (two tiles)
constexpr int kTlBlk = 128;        // keys per block
constexpr int kTlThreads = 384;  // two softmax warpgroups; a third for the producer and the MMA issuer
// registers a thread: the third warpgroup gives its own up (2 x 224 + 56 = 3 x 168, the launch's)
constexpr int kTlRegsSoftmax = 224, kTlRegsOther = 56;
constexpr int kTlMaxCluster = 8;
constexpr int kTlJoinWarps = 8;    // the softmax warps write the result
constexpr int kTlPoly = 2;         // of 8 exponential pairs: on the FMA pipe, beside the special-function unit
constexpr float kTlLazy = 8.0f, kTlShift = 7.0f;

template <int HDP, bool SPLIT>
struct TlCfg {
    static constexpr int kPart = 128 * HDP * 2;              // one tile's Q (one part of it)
    static constexpr int kParts = SPLIT ? 2 : 1;
    static constexpr int kQ = 2 * kParts * kPart;
    static constexpr int kStage = kTlBlk * HDP * 2;          // one K or V block
    static constexpr int kStages = HDP == 64 ? 8 : SPLIT ? 3 : 5;
    static constexpr int kData = kQ + kStages * kStage;
    static_assert(kData >= kTlRows * HDP * 4, "the joined O overlays Q and the ring");
};
template <int HDP, bool SPLIT>
struct TlSmem {
    using C = TlCfg<HDP, SPLIT>;
    uint8_t data[C::kData];  // Q, then the ring; at the end O (f32, 16-byte chunks swizzled by row)
    float m[kTlRows], l[kTlRows];
    uint64_t full[C::kStages], empty[C::kStages], q_full[2], s_full[2], p_half[2], p_full[2], done;
    uint32_t tmem;
};

// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tl_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void tl_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// Shared-memory descriptor of an MN-major operand with the 128-byte swizzle: rows of 64 elements
// along N, 8 rows (k) 128 bytes apart to a group, groups 1024 bytes apart, the next 64 elements of
// N `n_stride` bytes on.
__device__ __forceinline__ uint64_t sw128_desc_mn(const void *p, uint32_t n_stride) {
    uint64_t d = (smem_u32(p) >> 4) & 0x3fffull;
    d |= (uint64_t)(n_stride >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void tl_tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tl_tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
        "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
        "r"(v[31])
        : "memory");
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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// max over 32 values and mx (a tree, so that few steps wait for one another), NaN if one of them is
__device__ __forceinline__ float tl_max32(const uint32_t (&s)[32], float mx) {
    float c[11];
#pragma unroll
    for (int i = 0; i < 10; i++)
        c[i] = max3_nan(__uint_as_float(s[3 * i]), __uint_as_float(s[3 * i + 1]), __uint_as_float(s[3 * i + 2]));
    c[10] = max3_nan(__uint_as_float(s[30]), __uint_as_float(s[31]), mx);
    const float d0 = max3_nan(c[0], c[1], c[2]), d1 = max3_nan(c[3], c[4], c[5]), d2 = max3_nan(c[6], c[7], c[8]);
    return max3_nan(max3_nan(d0, d1, d2), c[9], c[10]);
}
// 2^x of two values on the FMA pipe, x <= 127 (below -126: 2^-126): x = n + f with n the nearest
// whole number (from the addition of 1.5 * 2^23), 2^f by the polynomial of least relative error on
// [-1/2, 1/2] (degree 4: 2.6e-6, degree 3: 7.5e-5; exchange algorithm in 64 bits), n into the exponent.
template <int DEG>
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    x.x = fmaxf(x.x, -126.0f), x.y = fmaxf(x.y, -126.0f);
    const float2 t = add2(x, make_float2(12582912.0f, 12582912.0f));
    const float2 n = add2(t, make_float2(-12582912.0f, -12582912.0f));
    const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
    constexpr float c[2][5] = {{0.9999280571937561f, 0.6932609677314758f, 0.2426111251115799f, 0.0551716685295105f, 0.0f},
                               {0.9999992847442627f, 0.6931217908859253f, 0.240247443318367f, 0.05591785907745361f, 0.009570102207362652f}};
    float2 y = make_float2(c[DEG - 3][DEG], c[DEG - 3][DEG]);
#pragma unroll
    for (int i = DEG - 1; i >= 0; i--) y = fma2(y, f, make_float2(c[DEG - 3][i], c[DEG - 3][i]));
    y.x = __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23));
    y.y = __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23));
    return y;
}

// Blocks [lo, hi) of keys that rows [r0, r1) of a sequence attend (r1 > r0).
struct TlSpan {
    int32_t lo, hi;
};
__device__ __forceinline__ TlSpan tl_span(const SeqAttnParams &p, const SeqSpan &sp, uint32_t r0, uint32_t r1) {
    const int64_t a = sp.pos(r0 / p.group), b = sp.pos((r1 - 1) / p.group);
    if (b < 0) return {0, 0};
    const int64_t lo = p.window > 0 && a + 1 > (int64_t)p.window ? a + 1 - p.window : 0;
    return {(int32_t)(lo / kTlBlk), (int32_t)(b / kTlBlk) + 1};
}

template <typename T, typename E, int HDP>
__global__ void __launch_bounds__(kTlThreads, 1) k_attn_tile(const __grid_constant__ CUtensorMap mk,
                                                             const __grid_constant__ CUtensorMap mv,
                                                             const __grid_constant__ SeqAttnParams p) {
    constexpr bool kSplit = std::is_same<T, float>::value;
    using C = TlCfg<HDP, kSplit>;
    using S = TlSmem<HDP, kSplit>;
    constexpr int kChunks = HDP / 64;
    extern __shared__ __align__(1024) uint8_t tl_raw[];  // swizzled tiles start on 1024-byte boundaries
    S &sm = *reinterpret_cast<S *>(tl_raw);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const uint32_t item = blockIdx.x / p.splits, kvh = item % p.n_kv, ti = p.n_tiles - 1 - item / p.n_kv;
    pdl_wait();
    pdl_trigger();
    SeqSpan sp;
    uint32_t tile;
    if (!seq_find_tile(p.b, p.group, kTlRows, p.rows_lo, p.rows_hi, ti, &sp, &tile)) return;  // the same for the whole cluster
    const uint32_t row0 = tile * kTlRows, n_rows = min(sp.n_new * p.group - row0, (uint32_t)kTlRows);
    const uint32_t n_tiles = n_rows > 128 ? 2 : 1;
    // this CTA's part of the blocks, and each tile's part of those
    const TlSpan all = tl_span(p, sp, row0, row0 + n_rows);
    const int32_t per = (all.hi - all.lo + (int32_t)p.splits - 1) / (int32_t)p.splits;
    const int32_t j0 = min(all.lo + (int32_t)rank * per, all.hi), j1 = min(j0 + per, all.hi);
    int32_t jb[2], je[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        jb[t] = je[t] = j0;
        if (t < (int)n_tiles) {
            const TlSpan s = tl_span(p, sp, row0 + 128 * t, min(row0 + n_rows, row0 + 128 * t + 128));
            jb[t] = min(max(s.lo, j0), j1), je[t] = max(min(s.hi, j1), jb[t]);
        }
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; s++) mbar_init(&sm.full[s], 1), mbar_init(&sm.empty[s], 1);
        for (int t = 0; t < 2; t++) mbar_init(&sm.q_full[t], 128), mbar_init(&sm.s_full[t], 1), mbar_init(&sm.p_half[t], 4), mbar_init(&sm.p_full[t], 4);
        mbar_init(&sm.done, 1);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc<512>(&sm.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    uint8_t *ring = sm.data + C::kQ;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTlRegsOther));
    }
    if (warp == 8) {  // ---- producer ----
        const uint32_t box = p.b.pages ? min(1u << p.b.page_shift, (uint32_t)kTlBlk) : (uint32_t)kTlBlk;
        const uint32_t n_box = kTlBlk / box;  // boxes of rows per block (8 at most, pages of 16)
        const int64_t end = sp.pos((row0 + n_rows - 1) / p.group) + 1;
        uint32_t it = 0;
        bool ok = true;
        for (int32_t j = j0; j < j1 && ok; j++) {
            // lane l < n_box * kChunks brings box l % n_box of 64-element chunk l / n_box
            const uint32_t bx = lane % n_box, ch = lane / n_box;
            const int64_t pos = (int64_t)j * kTlBlk + bx * box;
            uint32_t row = p.kv_rows;  // behind the tensor: zeros
            if (ch < kChunks && pos < end) row = min(seq_kv_row(p.b, sp, p.n_kv, kvh, (uint32_t)pos), p.kv_rows);
#pragma unroll
            for (int kv = 0; kv < 2; kv++, it++) {
                const uint32_t s = it % C::kStages, n = it / C::kStages;
                if (n > 0) ok = ok && mbar_wait_sleep(&sm.empty[s], (n - 1) & 1, p.b.err, ERR_TIMEOUT_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&sm.full[s], C::kStage);
                __syncwarp();
                if (ch < kChunks)
                    tma_load_3d(ring + s * C::kStage + ch * (kTlBlk * 128) + bx * box * 128, kv ? &mv : &mk, 64 * ch,
                                p.b.pages ? 0 : (int)kvh, (int)row, &sm.full[s]);
            }
        }
        // every copy has landed before this CTA goes on to its end
        for (uint32_t i = it > C::kStages ? it - C::kStages : 0; i < it; i++)
            mbar_wait_sleep(&sm.full[i % C::kStages], (i / C::kStages) & 1, p.b.err, ERR_TIMEOUT_FULL);
    } else if (warp == 9) {  // ---- MMA ----
        // The whole warp walks the blocks and one elected lane issues: the loop's state is the same in
        // every lane (taken from lane 0), so the descriptors stay in uniform registers. Issued from a
        // branch of lane 0 alone, an MMA cost 107 cycles of moves into them, against 64 of work.
        constexpr uint32_t kFmt = std::is_same<E, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t kIdS = (1u << 4) | kFmt | ((uint32_t)(kTlBlk >> 3) << 17) | (8u << 24);
        constexpr uint32_t kIdO = (1u << 4) | kFmt | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | (8u << 24);
        auto uni = [](int32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
        const int32_t n_blk = uni(j1 - j0), b0 = uni(jb[0] - j0), e0 = uni(je[0] - j0), b1 = uni(jb[1] - j0), e1 = uni(je[1] - j0);
        const uint32_t tm = uni((int32_t)tmem);
        const uint64_t dq = sw128_desc(sm.data), dk = sw128_desc(ring), dv = sw128_desc_mn(ring, kTlBlk * 128);
        const bool elected = elect_one();
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(bar, parity, p.b.err, ERR_TIMEOUT_FULL));
            tc_fence_after();
            return ok;
        };
        wait(&sm.q_full[0], 0);
        if (uni((int32_t)n_tiles) > 1) wait(&sm.q_full[1], 0);
        uint32_t np[2] = {0, 0};
        uint32_t sk = 0, pk = 0, sv = 1, pv = 0;  // ring stage and parity of K(j), V(j - 1)
        for (int32_t j = 0; j <= n_blk && ok; j++) {
            const bool last = j == n_blk;
            if (j > 0) wait(&sm.full[sv], pv);
            if (!last) wait(&sm.full[sk], pk);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t ts = tm + 128 * t, to = tm + 256 + HDP * t;
                const int32_t b = t ? b1 : b0, e = t ? e1 : e0;
                if (j - 1 >= b && j - 1 < e && ok) {  // O_t += P_t V(j - 1)
                    const uint64_t v = dv + sv * (C::kStage >> 4);
#pragma unroll
                    for (int half = 0; half < 2; half++) {  // keys 64 half .. 64 half + 63
                        if (!wait(half ? &sm.p_full[t] : &sm.p_half[t], np[t] & 1)) break;
                        if (elected) {
#pragma unroll
                            for (int kk = 4 * half; kk < 4 * half + 4; kk++) {
                                const uint32_t a = ts + 32 * (kk >> 1) + 8 * (kk & 1);
                                tl_mma_ts(to, a, v + (2048 >> 4) * kk, kIdO, kk > 0 || (!kSplit && j - 1 > b));
                                if constexpr (kSplit) tl_mma_ts(to, a + 16, v + (2048 >> 4) * kk, kIdO, true);
                            }
                        }
                    }
                    np[t]++;
                }
                if (t == 1 && j > 0 && elected) mma_commit(&sm.empty[sv]);
                if (j >= b && j < e && ok) {  // S_t = Q_t K(j)^T
                    if (elected) {
                        const uint64_t k = dk + sk * (C::kStage >> 4), q = dq + t * ((C::kParts * C::kPart) >> 4);
                        if constexpr (kSplit) {
#pragma unroll
                            for (int kk = 0; kk < HDP / 16; kk++) {
                                const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
                                tl_mma_ss(ts, q + (C::kPart >> 4) + off, k + off, kIdS, kk > 0);
                            }
                        }
#pragma unroll
                        for (int kk = 0; kk < HDP / 16; kk++) {
                            const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
                            tl_mma_ss(ts, q + off, k + off, kIdS, kSplit || kk > 0);
                        }
                        mma_commit(&sm.s_full[t]);
                    }
                    __syncwarp();
                }
            }
            if (!last && elected) mma_commit(&sm.empty[sk]);
            // K and V blocks take turns in the ring
            auto next = [](uint32_t &s, uint32_t &par) {
                s += 2;
                if (s >= (uint32_t)C::kStages) s -= C::kStages, par ^= 1;
            };
            if (j > 0) next(sv, pv);
            next(sk, pk);
        }
        if (elected) mma_commit(&sm.done);  // every MMA issued, on an early end too
        __syncwarp();
        mbar_wait_sleep(&sm.done, 0, p.b.err, ERR_TIMEOUT_DRAIN);
    } else if (warp < 8) {  // ---- softmax: thread r of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTlRegsSoftmax));
        const uint32_t t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (32 * (warp & 3)) << 16;  // this warp's TMEM lanes
        const uint32_t ts = tmem + 128 * t + lanes, to = tmem + 256 + HDP * t + lanes;
        const bool live = 128 * t + r < n_rows;
        const uint32_t row = row0 + min(128 * t + r, n_rows - 1), tok = row / p.group;
        const int64_t hi = live ? sp.pos(tok) : -1;
        const int64_t lo = p.window > 0 && hi + 1 > (int64_t)p.window ? hi + 1 - p.window : 0;
        float unscale = 1.0f;
        if (t < n_tiles) {  // Q row into shared memory (K-major, 128-byte swizzle)
            const T *src = reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + tok) * p.ld_q +
                           (uint64_t)(kvh * p.group + row % p.group) * p.hd;
            uint8_t *q = sm.data + t * C::kParts * C::kPart + r * 128;
            float scale = 1.0f;
            if constexpr (kSplit) {
                float mx = 0.0f;
                if (live)
                    for (uint32_t c = 0; c < p.hd; c += 4) {
                        const float4 x = *reinterpret_cast<const float4 *>(src + c);
                        mx = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), mx);
                    }
                const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255), 2), 252) - 127;
                scale = __uint_as_float((uint32_t)(127 - e) << 23);
                unscale = __uint_as_float((uint32_t)(127 + e) << 23);
            }
#pragma unroll 4
            for (int c = 0; c < HDP / 8; c++) {
                uint8_t *d = q + (c >> 3) * (128 * 128) + (((c & 7) ^ (r & 7)) << 4);
                const bool in = live && 8 * c < (int)p.hd;
                if constexpr (kSplit) {
                    float x[8] = {};
                    if (in) {
                        *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(src + 8 * c);
                        *reinterpret_cast<float4 *>(x + 4) = *reinterpret_cast<const float4 *>(src + 8 * c + 4);
                    }
                    uint32_t h[4], w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float a = x[2 * i] * scale, b = x[2 * i + 1] * scale;
                        h[i] = pack2<E>(a, b);
                        const float2 f = unpack2<E>(h[i]);
                        w[i] = pack2<E>(a - f.x, b - f.y);
                    }
                    *reinterpret_cast<uint4 *>(d) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(d + C::kPart) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    *reinterpret_cast<uint4 *>(d) = in ? *reinterpret_cast<const uint4 *>(src + 8 * c) : make_uint4(0, 0, 0, 0);
                }
            }
            fence_async_smem();
            mbar_arrive(&sm.q_full[t]);
        }
        // keys that every live row of the tile attends: blocks inside need no mask
        int64_t all_hi = -1, all_lo = 0;
        if (t < n_tiles) {
            const int64_t last = sp.pos((min(row0 + n_rows, row0 + 128 * t + 128) - 1) / p.group);
            all_hi = sp.pos((row0 + 128 * t) / p.group);
            all_lo = p.window > 0 && last + 1 > (int64_t)p.window ? last + 1 - p.window : 0;
        }
        const float cs = p.softcap > 0.0f ? 1.0f : unscale * kLog2e;
        float m = -INFINITY, l = 0.0f;  // m in units of log2, as last rescaled to
        float o[kSplit ? HDP : 1];
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < HDP; i++) o[i] = 0.0f;
        }
        bool ok = true;
        for (int32_t j = jb[t]; j < je[t]; j++) {
            ok = mbar_wait_bounded(&sm.s_full[t], (j - jb[t]) & 1, p.b.err, ERR_TIMEOUT_FULL);
            if (!ok) break;
            tc_fence_after();
            const int64_t key0 = (int64_t)j * kTlBlk;
            const bool part = key0 < all_lo || key0 + kTlBlk - 1 > all_hi;
            const int32_t rlo = (int32_t)max(lo - key0, (int64_t)0), rhi = (int32_t)max(min(hi - key0, (int64_t)kTlBlk), (int64_t)-1);
            // one block's columns 32 c .. 32 c + 31 of this row: softcapped, masked
            auto fetch = [&](int c, uint32_t (&s)[32]) { tmem_ld32(ts + 32 * c, s); };
            auto shape = [&](int c, uint32_t (&s)[32]) {
                if (p.softcap > 0.0f) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        s[i] = __float_as_uint(p.softcap * kLog2e * tanhf(__uint_as_float(s[i]) * unscale / p.softcap));
                }
                if (part) {
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (32 * c + i > rhi || 32 * c + i < rlo) s[i] = 0xff800000u;
                }
            };
            float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
            auto pack = [&](int c, const uint32_t (&s)[32], float off) {  // p, and its sum; the first 64 keys' P may go
                uint32_t h[16], w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float2 x = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), make_float2(cs, cs),
                                          make_float2(-off, -off));
                    float2 e;
                    if (!kSplit && i % 8 < kTlPoly) e = ex2_poly<std::is_same<E, __half>::value ? 4 : 3>(x);
                    else e = make_float2(ex2(x.x), ex2(x.y));
                    if (i & 1) sum1 = add2(sum1, e);
                    else sum0 = add2(sum0, e);
                    h[i] = pack2<E>(e.x, e.y);
                    if constexpr (kSplit) {
                        const float2 f = unpack2<E>(h[i]);
                        w[i] = pack2<E>(e.x - f.x, e.y - f.y);
                    }
                }
                tl_tmem_st16(ts + 32 * c, h);
                if constexpr (kSplit) tl_tmem_st16(ts + 32 * c + 16, w);
                if (c & 1) {
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(c == 1 ? &sm.p_half[t] : &sm.p_full[t]);
                }
            };
            float mx = -INFINITY;
            if constexpr (!kSplit) {
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++) fetch(c, s[c]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    shape(c, s[c]);
                    mx = tl_max32(s[c], mx);
                }
                mx *= cs;
                const bool grow = mx > m + kTlLazy || (m == -INFINITY && mx > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mn = grow ? mx : m;
                    const float a = mn == m ? 1.0f : ex2(m - mn);
                    m = mn;
                    l *= a;
                    if (j > jb[t]) {  // the S that was waited for comes after the last P V
#pragma unroll
                        for (int c = 0; c < HDP / 32; c++) {
                            uint32_t v[32];
                            tmem_ld32(to + 32 * c, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
                            tl_tmem_st32(to + 32 * c, v);
                        }
                    }
                }
                const float off = (m == -INFINITY ? 0.0f : m) - kTlShift;
#pragma unroll
                for (int c = 0; c < 4; c++) pack(c, s[c], off);
            } else {
                uint32_t s[32];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    fetch(c, s);
                    tmem_wait_ld();
                    shape(c, s);
                    mx = tl_max32(s, mx);
                }
                mx *= cs;
                if (j > jb[t]) {  // add the last block's P V
#pragma unroll
                    for (int c = 0; c < HDP / 32; c++) {
                        tmem_ld32(to + 32 * c, s);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) o[32 * c + i] += __uint_as_float(s[i]);
                    }
                }
                if (__any_sync(0xffffffffu, mx > m)) {
                    const float mn = mx > m ? mx : m;
                    const float a = mn == m ? 1.0f : ex2(m - mn);
                    m = mn;
                    l *= a;
#pragma unroll
                    for (int i = 0; i < HDP; i++) o[i] *= a;
                }
                const float off = (m == -INFINITY ? 0.0f : m) - kTlShift;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    fetch(c, s);
                    tmem_wait_ld();
                    shape(c, s);
                    pack(c, s, off);
                }
            }
            l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
            if (mx != mx) l = mx;  // a NaN among the scores (the polynomial does not carry it)
        }
        // every MMA has ended: Q and the ring are free for O
        ok = mbar_wait_sleep(&sm.done, 0, p.b.err, ERR_TIMEOUT_DRAIN) && ok;
        tc_fence_after();
        if (t < n_tiles) {
            float *orow = reinterpret_cast<float *>(sm.data) + (128 * t + r) * HDP;
            constexpr uint32_t kMask = HDP / 4 - 1;
            const bool any = je[t] > jb[t] && ok;
#pragma unroll
            for (int c = 0; c < HDP / 32; c++) {
                uint32_t v[32];
                if (any) {
                    tmem_ld32(to + 32 * c, v);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float x[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        x[k] = any ? __uint_as_float(v[4 * i + k]) : 0.0f;
                        if constexpr (kSplit) x[k] += o[32 * c + 4 * i + k];
                    }
                    *reinterpret_cast<float4 *>(orow + (((8 * c + i) ^ (r & kMask)) << 2)) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
            sm.m[128 * t + r] = m;
            sm.l[128 * t + r] = l;
        }
        tc_fence_before();
        if (p.splits > 1) cluster_sync_all();
        else __syncthreads();
        // ---- rows of the result over the warps of the cluster ----
        constexpr int VE = HDP / 32;  // values a lane
        for (uint32_t r = rank * kTlJoinWarps + warp; r < n_rows; r += p.splits * kTlJoinWarps) {
            float acc[VE] = {};
            float L;
            // lane's values: 16-byte chunk lane * VE / 4, swizzled by the row
            const uint32_t ch = (lane * VE / 4) ^ (r & (HDP / 4 - 1)), at = r * HDP * 4 + ch * 16 + (lane * VE % 4) * 4;
            if (p.splits == 1) {
                L = sm.l[r];
    #pragma unroll
                for (int i = 0; i < VE; i++) acc[i] = *reinterpret_cast<const float *>(sm.data + at + 4 * i);
            } else {
                const uint32_t am = smem_u32(&sm.m[r]), al = smem_u32(&sm.l[r]), ao = smem_u32(sm.data) + at;
                const float mc = lane < p.splits ? ld_cluster_f32(cluster_addr(am, lane)) : -INFINITY;
                const float lc = lane < p.splits ? ld_cluster_f32(cluster_addr(al, lane)) : 0.0f;
                float M = mc;
    #pragma unroll
                for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
                const float ac = mc == -INFINITY ? 0.0f : ex2(mc - M);
                L = ac * lc;
    #pragma unroll
                for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
                for (uint32_t c = 0; c < p.splits; c++) {
                    const float w = __shfl_sync(0xffffffffu, ac, c);
                    if (w == 0.0f) continue;
                    const uint32_t a = cluster_addr(ao, c);
    #pragma unroll
                    for (int i = 0; i < VE; i++) acc[i] = fmaf(w, ld_cluster_f32(a + 4 * i), acc[i]);
                }
            }
            const uint32_t rr = row0 + r, tk = rr / p.group, gq = rr % p.group, d0 = lane * VE;
            T *orow = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + tk) * p.ld_out + (uint64_t)(kvh * p.group + gq) * p.hd;
            bool fine = true;
            if (d0 < p.hd) {
                alignas(16) T v[VE];
    #pragma unroll
                for (int i = 0; i < VE; i++) {
                    const float x = acc[i] / L;
                    fine = fine && isfinite(x);
                    v[i] = from_f32<T>(x);
                }
                if constexpr (VE * sizeof(T) == 16) *reinterpret_cast<uint4 *>(orow + d0) = *reinterpret_cast<const uint4 *>(v);
                else if constexpr (VE * sizeof(T) == 8) *reinterpret_cast<uint2 *>(orow + d0) = *reinterpret_cast<const uint2 *>(v);
                else *reinterpret_cast<uint32_t *>(orow + d0) = *reinterpret_cast<const uint32_t *>(v);
            }
            if (!__all_sync(0xffffffffu, fine)) {
                __syncwarp();
                seq_attn_row<T, E>(p, sp, tk, kvh, gq);
            }
        }
        if (p.splits > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
        return;
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_free<512>(tmem);
    }
    if (p.splits > 1) cluster_sync_all();
}

// ---- host ---------------------------------------------------------------------------------------
bool attention_tile_ok(uint64_t hd) { return hd <= 128; }

template <typename T, typename E, int HDP>
static int launch_tile(rcu_ctx *ctx, const CUtensorMap &mk, const CUtensorMap &mv, SeqAttnParams p, uint64_t max_len) {
    constexpr size_t smem = sizeof(TlSmem<HDP, std::is_same<T, float>::value>);
    static_assert(smem <= 232448, "shared memory of one CTA");
    const uint64_t items = (uint64_t)p.n_tiles * p.n_kv, span = p.window > 0 ? std::min<uint64_t>(max_len, p.window + kTlRows) : max_len;
    uint32_t cs = 1;  // one CTA for each SM, four blocks of keys for each
    while (cs < kTlMaxCluster && items * cs * 2 <= (uint64_t)ctx->num_sms && span >= (uint64_t)cs * 2 * 4 * kTlBlk) cs *= 2;
    p.splits = cs;
    if (items * cs > 0x7fffffffull) return set_err(ctx, RCU_ERR_INVALID, "attention: too many work tiles");
    return launch_cluster_k(ctx, k_attn_tile<T, E, HDP>, (uint32_t)(items * cs), kTlThreads, smem, cs, mk, mv, p);
}

template <typename T, typename E>
static int launch_tile_hd(rcu_ctx *ctx, SeqAttnParams &p, const SeqKvDesc &kv, uint64_t max_len) {
    CUtensorMap mk, mv;
    const uint32_t box = kv.pages ? std::min<uint32_t>(1u << p.b.page_shift, kTlBlk) : kTlBlk;
    if (int st = seq_kv_maps(ctx, p, kv, box, &mk, &mv)) return st;
    // sequences of this class have at least rows_lo rows (or there is one class only)
    const uint64_t rows = (uint64_t)p.b.n_tok * p.group;
    p.n_tiles = (uint32_t)std::min<uint64_t>(seq_tiles_bound(p.b.n_tok, p.b.n_seq, p.group, kTlRows),
                                             rows / kTlRows + rows / std::max(1u, p.rows_lo) + 1);
    return p.hd <= 64 ? launch_tile<T, E, 64>(ctx, mk, mv, p, max_len) : launch_tile<T, E, 128>(ctx, mk, mv, p, max_len);
}

int launch_attention_tile(rcu_ctx *ctx, const SeqAttnParams &params, int q_type, const SeqKvDesc &kv, uint64_t max_len) {
    SeqAttnParams p = params;
    if (q_type == T_F32) return launch_tile_hd<float, __half>(ctx, p, kv, max_len);
    if (q_type == T_F16) return launch_tile_hd<__half, __half>(ctx, p, kv, max_len);
    return launch_tile_hd<__nv_bfloat16, __nv_bfloat16>(ctx, p, kv, max_len);
}

}  // namespace rcu
