// rcu_attn_tile.cu -- attention of a batch of sequences with many query rows per KV head (chunks,
// whole prompts) on the 5th-generation tensor cores. Formula and batch as in rcu_attn_seq.cu.
//
// A CTA takes 256 query rows (token, head of the group) of one sequence and KV head as two tiles of
// 128 rows, or 128 as one, and walks the attended keys in blocks of 128 (one tile: 16-bit queries
// whose CTAs are short, two CTAs to an SM, so that one's start and end run beside the other's blocks;
// head_dim above 128, since O fills tensor memory):
//   * warp 0     owns tensor memory; one lane issues S_t = Q_t K^T (M 128, N 128) and O_t += P_t V
//                (P read from tensor memory, V in its own layout as an MN-major operand);
//   * warp 1     producer: K and V blocks by tiled TMA (128-byte swizzle) into a ring of stages; a
//                page may be smaller than a block (one box per page) or larger. Warps 2 and 3 only
//                give their registers up;
//   * the others softmax, 8 warps for each tile: two threads share a query row, one for the first 64
//                keys of the block and one for the others: S out of tensor memory, mask, running
//                maximum (the two exchange theirs) and sum in f32, P = 2^(s - m) back as packed
//                16-bit values over S, each half handed on by itself.
// While one tile's warps are at their softmax, the tensor core works on the other tile (CTA).
// 16-bit queries: O stays in tensor memory; it is rescaled only when a row's maximum has grown by
// more than 2^kTlLazy since its last rescale (p then is at most 2^(kTlLazy + kTlShift)). p is rounded
// to the type of V, its sum is not: kind::f16 takes both operands in one type, and a second part of p
// would double the products (as f32 queries do); 2^-11 or 2^-8 of p, as much as the output's rounding.
// f32 queries: q (scaled by a power of two per row) and p are each split into two f16 parts, so each
// product is two MMAs (head_dim above 128: Q's low part in the tensor memory that S and O leave); O is added up in registers block by block, because a long chain of additions
// inside the tensor core, which does not round to nearest, would drift (8e-6 at 12k keys).
// Few tiles over a long context: a cluster of CTAs splits the keys and joins through distributed
// shared memory. All waits are bounded; TMEM is freed on every path.
// Bound: a block's 4 x 128 x 128 x 128 products take 2048 cycles of the tensor pipe, and about 3000
// pass, since a tile's S, softmax and P V follow one another and only the other tile's fill the gap;
// one bf16 prompt of 8192 tokens, 32 heads of 128: 547 to 557 us run for seconds, at the 1000 W limit
// (power cap active, 1.70 GHz), and 460 to 487 us (1.15 P/s) in the first milliseconds; with constants in
// place of the exponentials, or with fewer instructions in the issuing warp, the time was the same.
// A softcap costs more than all of it (1800 us): tanhf for each score, for f32 queries twice.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"
#include "rcu_tc.cuh"

namespace rcu {

constexpr int kTlBlk = kSeqTileBox;  // keys per block
constexpr int kTlMaxCluster = 8;
constexpr float kTlLazy = 8.0f, kTlShift = 7.0f;

template <int HDP, bool SPLIT, int TILES>
struct TlCfg {
    static_assert(TILES == 1 || HDP < 256, "O of two tiles does not fit tensor memory");
    static constexpr int kTiles = TILES;
    static constexpr int kPerSm = TILES == 1 && HDP < 256 ? 2 : 1;  // CTAs on an SM
    static constexpr int kTmem = 512 / kPerSm;               // tensor memory columns: 128 for S and HDP for O, each tile
    static constexpr int kRows = 128 * kTiles;               // query rows per CTA
    static constexpr int kSoftWarps = 8 * kTiles;
    static constexpr int kThreads = 32 * (kSoftWarps + 4);   // a warpgroup for the MMA issuer and the producer
    // registers a thread: the first warpgroup gives its own up (4 x 112 + 32 = 5 x 96, 2 x 104 + 32 = 3 x 80
    // or 2 x 224 + 56 = 3 x 168, the launch's)
    static constexpr int kRegsSoftmax = kTiles == 2 ? 112 : kPerSm == 2 ? 104 : 224, kRegsOther = kTiles == 2 || kPerSm == 2 ? 32 : 56;
    static constexpr int kPart = 128 * HDP * 2;              // one tile's Q (one part of it)
    static constexpr bool kLowTmem = SPLIT && HDP == 256;    // Q's low part in tensor memory, behind S and O
    static constexpr int kParts = SPLIT && !kLowTmem ? 2 : 1;  // of Q in shared memory
    static constexpr int kQ = kTiles * kParts * kPart;
    static constexpr int kStage = kTlBlk * HDP * 2;          // one K or V block
    static constexpr int kStages = kPerSm == 2 ? (HDP == 64 ? 5 : 2) : HDP == 64 ? 8 : HDP == 256 ? 2 : SPLIT ? 3 : 5;
    static constexpr int kData = kQ + kStages * kStage;
    static_assert(kData >= kRows * HDP * 4 + kTlMaxCluster * kRows * 4, "the joined O and its weights overlay Q and the ring");
    static_assert(!SPLIT || TILES == 2 || HDP == 256, "Q's two parts leave too little room for a ring");
};
template <int HDP, bool SPLIT, int TILES>
struct TlSmem {
    using C = TlCfg<HDP, SPLIT, TILES>;
    uint8_t data[C::kData];  // Q, then the ring; at the end O and its weights when a cluster joins
    float mx[2][C::kRows];   // [half of the block's keys]: row maxima; at the end the row's m and l
    uint64_t full[C::kStages], empty[C::kStages], s_full[2], p_half[2], p_full[2], o_done[2], done;
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
__device__ __forceinline__ void tl_tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tl_tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// max of 16 values (a tree, so that few steps wait for one another), NaN if one of them is
__device__ __forceinline__ float tl_max16(const uint32_t (&s)[16]) {
    float c[5];
#pragma unroll
    for (int i = 0; i < 5; i++)
        c[i] = max3_nan(__uint_as_float(s[3 * i]), __uint_as_float(s[3 * i + 1]), __uint_as_float(s[3 * i + 2]));
    return max3_nan(max3_nan(c[0], c[1], c[2]), max3_nan(c[3], c[4], __uint_as_float(s[15])), -INFINITY);
}
// Blocks [lo, hi) of keys that rows [r0, r1) of a sequence attend (r1 > r0).
struct TlSpan {
    int32_t lo, hi;
};
__device__ __forceinline__ TlSpan tl_span(const SeqAttnParams &p, const SeqSpan &sp, uint32_t r0, uint32_t r1) {
    const int32_t a = sp.pos(div_group(p, r0)), b = sp.pos(div_group(p, r1 - 1));
    if (b < 0) return {0, 0};
    return {p.window > 0 ? max(a - (int32_t)p.window + 1, 0) / kTlBlk : 0, b / kTlBlk + 1};
}

template <typename T, typename E, int HDP, int TILES>
__global__ void __launch_bounds__(TlCfg<HDP, std::is_same<T, float>::value, TILES>::kThreads, TlCfg<HDP, std::is_same<T, float>::value, TILES>::kPerSm) k_attn_tile(const __grid_constant__ CUtensorMap mk,
                                                             const __grid_constant__ CUtensorMap mv,
                                                             const __grid_constant__ SeqAttnParams p) {
    constexpr bool kSplit = std::is_same<T, float>::value;
    using C = TlCfg<HDP, kSplit, TILES>;
    using S = TlSmem<HDP, kSplit, TILES>;
    constexpr int kChunks = HDP / 64, kTiles = C::kTiles, kTlRows = C::kRows, kTlSoftWarps = C::kSoftWarps;
    extern __shared__ __align__(1024) uint8_t tl_raw[];  // swizzled tiles start on 1024-byte boundaries
    S &sm = *reinterpret_cast<S *>(tl_raw);
    constexpr uint32_t kMmaWarp = 0, kLoadWarp = 1, kSoft0 = 4;  // warps by role
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), sw = warp - kSoft0, lane = threadIdx.x & 31;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const uint32_t item = blockIdx.x / p.splits, kvh = item % p.n_kv, ti = p.n_tiles - 1 - item / p.n_kv;
    // what needs no input first: tensor memory, and the barriers by the warp that uses them at once
    if (warp == kMmaWarp) tmem_alloc<C::kTmem>(&sm.tmem);
    if (warp == kLoadWarp) {
        if (lane == 0) {
            for (int s = 0; s < C::kStages; s++) mbar_init(&sm.full[s], 1), mbar_init(&sm.empty[s], 1);
            for (int t = 0; t < kTiles; t++)
                mbar_init(&sm.s_full[t], 1), mbar_init(&sm.p_half[t], 4), mbar_init(&sm.p_full[t], 4), mbar_init(&sm.o_done[t], 1);
            mbar_init(&sm.done, 1);
            fence_mbar_init();
        }
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();
    SeqSpan sp;
    uint32_t tile;
    if (!seq_find_tile(p.b, p.group, kTlRows, ti, &sp, &tile)) {  // the same for the whole cluster
        if (warp == kMmaWarp) tmem_free<C::kTmem>(sm.tmem);
        return;
    }
    const uint32_t row0 = tile * kTlRows, n_rows = min(sp.n_new * p.group - row0, (uint32_t)kTlRows);
    const uint32_t n_tiles = n_rows > 128 ? 2 : 1;  // 1 where there is one
    // this CTA's part of the blocks, and each tile's part of those
    const TlSpan all = tl_span(p, sp, row0, row0 + n_rows);
    const int32_t per = (all.hi - all.lo + (int32_t)p.splits - 1) / (int32_t)p.splits;
    const int32_t j0 = min(all.lo + (int32_t)rank * per, all.hi), j1 = min(j0 + per, all.hi);
    int32_t jb[2] = {j0, j0}, je[2] = {j0, j0};
#pragma unroll
    for (int t = 0; t < kTiles; t++) {
        jb[t] = je[t] = j0;
        if (t < (int)n_tiles) {
            const TlSpan s = tl_span(p, sp, row0 + 128 * t, min(row0 + n_rows, row0 + 128 * t + 128));
            jb[t] = min(max(s.lo, j0), j1), je[t] = max(min(s.hi, j1), jb[t]);
        }
    }
    uint8_t *ring = sm.data + C::kQ;
    if (warp >= kSoft0) {
        const uint32_t t = sw >> 3;
        if (t < n_tiles) {  // Q into shared memory (K-major, 128-byte swizzle), whole rows by neighbouring lanes
            uint8_t *q = sm.data + t * C::kParts * C::kPart;
            const uint32_t w8 = sw & 7;
            auto source = [&](uint32_t i) {  // row i of the tile
                const uint32_t rr = row0 + min(128 * t + i, n_rows - 1);
                const uint32_t tk = div_group(p, rr);
                return reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + tk) * p.ld_q +
                       (uint64_t)(kvh * p.group + rr - tk * p.group) * p.hd;
            };
            if constexpr (kSplit && HDP == 256) {  // a row a step; the low parts go to tensor memory below
#pragma unroll 4
                for (uint32_t k = 0; k < 16; k++) {
                    const uint32_t i = w8 * 16 + k;
                    const bool in = 128 * t + i < n_rows;
                    const T *src = source(i);
                    float4 x[2];
                    float mx = 0.0f;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t c4 = lane + 32 * u;
                        x[u] = in && 4 * c4 < p.hd ? *reinterpret_cast<const float4 *>(src + 4 * c4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[u].x), fabsf(x[u].y)), fmaxf(fabsf(x[u].z), fabsf(x[u].w))));
                    }
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255), 2), 252) - 127;
                    const float scale = __uint_as_float((uint32_t)(127 - e) << 23);
                    if (lane == 0) sm.mx[0][128 * t + i] = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t c4 = lane + 32 * u, c = c4 >> 1;
                        *reinterpret_cast<uint2 *>(q + (c >> 3) * (128 * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4) + 8 * (c4 & 1)) =
                            make_uint2(pack2<E>(x[u].x * scale, x[u].y * scale), pack2<E>(x[u].z * scale, x[u].w * scale));
                    }
                }
            } else if constexpr (kSplit) {
                constexpr int kLanes = HDP / 4, kPer = 32 / kLanes;  // lanes of a row (4 values each), rows a warp and step
                const uint32_t c4 = lane % kLanes, sub = lane / kLanes;
#pragma unroll
                for (int g = 0; g < 16 / kPer; g += 4) {
                    float4 x[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t i = (w8 * (16 / kPer) + g + k) * kPer + sub;
                        const bool in = 128 * t + i < n_rows && 4 * c4 < p.hd;
                        x[k] = in ? *reinterpret_cast<const float4 *>(source(i) + 4 * c4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t i = (w8 * (16 / kPer) + g + k) * kPer + sub;
                        float mx = fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
#pragma unroll
                        for (int d = kLanes / 2; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        // exponents at which both 2^e and 2^-e are normal numbers
                        const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255), 2), 252) - 127;
                        const float scale = __uint_as_float((uint32_t)(127 - e) << 23);
                        if (c4 == 0) sm.mx[0][128 * t + i] = __uint_as_float((uint32_t)(127 + e) << 23);
                        uint32_t u[2], w[2];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const float a = (j ? x[k].z : x[k].x) * scale, b = (j ? x[k].w : x[k].y) * scale;
                            u[j] = pack2<E>(a, b);
                            const float2 f = unpack2<E>(u[j]);
                            w[j] = pack2<E>(a - f.x, b - f.y);
                        }
                        const uint32_t c = c4 >> 1;
                        uint8_t *d = q + (c >> 3) * (128 * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4) + 8 * (c4 & 1);
                        *reinterpret_cast<uint2 *>(d) = make_uint2(u[0], u[1]);
                        *reinterpret_cast<uint2 *>(d + C::kPart) = make_uint2(w[0], w[1]);
                    }
                }
            } else {
                constexpr int kLanes = HDP / 8, kPer = 32 / kLanes, kIt = 16 / kPer;
                const uint32_t c = lane % kLanes, sub = lane / kLanes;
                uint4 x[kIt];
#pragma unroll
                for (int k = 0; k < kIt; k++) {
                    const uint32_t i = (w8 * kIt + k) * kPer + sub;
                    x[k] = 128 * t + i < n_rows && 8 * c < p.hd ? *reinterpret_cast<const uint4 *>(source(i) + 8 * c) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int k = 0; k < kIt; k++) {
                    const uint32_t i = (w8 * kIt + k) * kPer + sub;
                    *reinterpret_cast<uint4 *>(q + (c >> 3) * (128 * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4)) = x[k];
                }
            }
            fence_async_smem();
        }
    }
    uint32_t tmem = 0;
    auto meet = [&]() {  // Q, the barriers and tensor memory are there
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = sm.tmem;
    };
    if (warp != kLoadWarp) meet();  // the producer has its copies on their way first
    if (warp < kSoft0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsOther));
    }
    if (warp == kLoadWarp) {  // ---- producer ----
        bool met = false;
        const uint32_t box = p.b.pages ? min(1u << p.b.page_shift, (uint32_t)kTlBlk) : (uint32_t)kTlBlk;
        const uint32_t n_box = kTlBlk / box;  // boxes of rows per block (8 at most, pages of 16)
        const int32_t end = sp.pos(div_group(p, row0 + n_rows - 1)) + 1;
        uint32_t it = 0;
        bool ok = true;
        for (int32_t j = j0; j < j1 && ok; j++) {
            if (it + 2 > C::kStages && !met) met = true, meet();
            // lane l < n_box * kChunks brings box l % n_box of 64-element chunk l / n_box
            const uint32_t bx = lane % n_box, ch = lane / n_box;
            const int32_t pos = j * kTlBlk + (int32_t)(bx * box);
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
        if (!met) meet();
        // every copy has landed before this CTA goes on to its end
        for (uint32_t i = it > C::kStages ? it - C::kStages : 0; i < it; i++)
            mbar_wait_sleep(&sm.full[i % C::kStages], (i / C::kStages) & 1, p.b.err, ERR_TIMEOUT_FULL);
    } else if (warp == kMmaWarp) {  // ---- MMA ----
        // The whole warp walks the blocks and one elected lane issues: the loop's state is the same in
        // every lane (taken from lane 0), so the descriptors stay in uniform registers. Issued from a
        // branch of lane 0 alone, an MMA cost 107 cycles of moves into them, against 64 of work.
        constexpr uint32_t kFmt = std::is_same<E, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t kIdS = (1u << 4) | kFmt | ((uint32_t)(kTlBlk >> 3) << 17) | (8u << 24);
        constexpr uint32_t kIdO = (1u << 4) | kFmt | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | (8u << 24);
        auto uni = [](int32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
        const int32_t n_blk = uni(j1 - j0), b0 = uni(jb[0] - j0), e0 = uni(je[0] - j0), b1 = uni(jb[1] - j0), e1 = uni(je[1] - j0);
        // keys from this CTA's first block to the last one that a row attends
        const int32_t n_keys = uni(sp.pos(div_group(p, row0 + n_rows - 1)) + 1 - j0 * kTlBlk);
        const uint32_t tm = uni((int32_t)tmem);
        const uint64_t dq = sw128_desc(sm.data), dk = sw128_desc(ring), dv = sw128_desc_mn(ring, kTlBlk * 128);
        const bool elected = elect_one();
        // After a wait that ran out (the result is void) the walk goes on without waiting.
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            bool there = false;
#pragma unroll 1
            for (int i = 0; i < 64 && !there; i++) there = __all_sync(0xffffffffu, mbar_test(bar, parity));
            if (!there && ok) ok = __all_sync(0xffffffffu, mbar_wait_spin(bar, parity, p.b.err, ERR_TIMEOUT_FULL));
            tc_fence_after();
        };
        uint32_t np = 0;                          // bit t: parity of tile t's P
        uint32_t sk = 0, pk = 0, sv = 1, pv = 0;  // ring stage and parity of K(j), V(j - 1)
        // K and V blocks take turns in the ring
        auto next = [](uint32_t &s, uint32_t &par) {
            s += 2;
            if (s >= (uint32_t)C::kStages) s -= C::kStages, par ^= 1;
        };
        auto wait_v = [&](int32_t j, uint32_t s, uint32_t par) {  // V(j)
            wait(&sm.full[s], par);
            if ((j + 1) * kTlBlk > n_keys) {  // rows behind the last key hold anything: 0 * v must stay 0
                uint8_t *v = ring + s * C::kStage;
#pragma unroll 1
                for (uint32_t i = (uint32_t)(n_keys - j * kTlBlk) * 8 + lane; i < kTlBlk * 8; i += 32)
#pragma unroll
                    for (int c = 0; c < kChunks; c++) *reinterpret_cast<uint4 *>(v + c * (kTlBlk * 128) + i * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
                __syncwarp();
            }
        };
        // Where the ring has room for them, the next blocks are waited for while the tensor core is at
        // work, not between a tile's P and its products (the time is the same while the copies are
        // ahead; a late copy then delays one tile and not both).
        constexpr bool kEarlyV = C::kStages >= 3, kEarlyK = C::kStages >= 4;
        if constexpr (C::kLowTmem) {
            named_bar_sync(11, 288);
            tc_fence_after();
        }
        if (n_blk > 0) wait(&sm.full[sk], pk);
        for (int32_t j = 0; j <= n_blk; j++) {
            const bool last = j == n_blk;
            if (!kEarlyV && j > 0) wait_v(j - 1, sv, pv);
            if (!kEarlyK && j > 0 && !last) wait(&sm.full[sk], pk);
#pragma unroll 1
            for (int t = 0; t < kTiles; t++) {
                const uint32_t ts = tm + 128 * t, to = tm + 128 * kTiles + HDP * t;
                const int32_t b = t ? b1 : b0, e = t ? e1 : e0;
                if (j > b && j <= e) {  // O_t += P_t V(j - 1)
                    const uint64_t v = dv + sv * (C::kStage >> 4);
#pragma unroll 1
                    for (int half = 0; half < 2; half++) {  // keys 64 half .. 64 half + 63
                        wait(half ? &sm.p_full[t] : &sm.p_half[t], np >> t & 1);
                        if (elected) {
#pragma unroll
                            for (int kk = 0; kk < 4; kk++) {
                                const uint32_t a = ts + 64 * half + 16 * kk;
                                const uint64_t vk = v + (2048 >> 4) * (4 * half + kk);
                                tl_mma_ts(to, a, vk, kIdO, kk > 0 || half > 0 || (!kSplit && j - 1 > b));
                                if constexpr (kSplit) tl_mma_ts(to, a + 8, vk, kIdO, true);
                            }
                        }
                    }
                    np ^= 1u << t;
                    if (j == e && elected) mma_commit(&sm.o_done[t]);
                }
                if (t == kTiles - 1 && j > 0 && elected) mma_commit(&sm.empty[sv]);
                if (j >= b && j < e) {  // S_t = Q_t K(j)^T
                    if (elected) {
                        const uint64_t k = dk + sk * (C::kStage >> 4), q = dq + t * ((C::kParts * C::kPart) >> 4);
                        if constexpr (kSplit) {
#pragma unroll
                            for (int kk = 0; kk < HDP / 16; kk++) {
                                const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
                                if constexpr (C::kLowTmem) tl_mma_ts(ts, tm + 384 + 8 * kk, k + off, kIdS, kk > 0);
                                else tl_mma_ss(ts, q + (C::kPart >> 4) + off, k + off, kIdS, kk > 0);
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
                if (t == 0 && !last) {
                    uint32_t s = sv, par = pv;
                    if (j > 0) next(s, par);
                    if (kEarlyV) wait_v(j, s, par);
                    s = sk, par = pk;
                    next(s, par);
                    if (kEarlyK && j + 1 < n_blk) wait(&sm.full[s], par);
                }
            }
            if (!last && elected) mma_commit(&sm.empty[sk]);
            if (j > 0) next(sv, pv);
            next(sk, pk);
        }
        if (elected) {
            mma_commit(&sm.done);  // every MMA issued
        }
        __syncwarp();
        mbar_wait_sleep(&sm.done, 0, p.b.err, ERR_TIMEOUT_DRAIN);
    } else if (warp >= kSoft0) {  // ---- softmax: row r of tile t, keys 64 h .. 64 h + 63 of each block ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
        const uint32_t t = sw >> 3, h = (sw >> 2) & 1, r = threadIdx.x & 127, tr = 128 * t + r;
        const uint32_t pair = 1 + 4 * t + (warp & 3);    // barrier of the two warps that share these rows
        const uint32_t lanes = (32 * (warp & 3)) << 16;  // their TMEM lanes
        const uint32_t ts = tmem + 128 * t + 64 * h + lanes, to = tmem + 128 * kTiles + HDP * t + HDP / 2 * h + lanes;
        const bool live = tr < n_rows;
        const uint32_t tok = div_group(p, row0 + min(tr, n_rows - 1));
        // positions stay below 2^31
        const int32_t hi = live ? sp.pos(tok) : -1;
        const int32_t lo = p.window > 0 ? max(hi - (int32_t)p.window + 1, 0) : 0;
        // keys that every live row of the tile attends: blocks inside need no mask
        int32_t all_hi = -1, all_lo = 0;
        if (t < n_tiles) {
            const int32_t last = sp.pos(div_group(p, min(row0 + n_rows, row0 + 128 * t + 128) - 1));
            all_hi = sp.pos(div_group(p, row0 + 128 * t));
            all_lo = p.window > 0 ? max(last - (int32_t)p.window + 1, 0) : 0;
        }
        float unscale = 1.0f;
        if constexpr (kSplit) {
            unscale = t < n_tiles ? sm.mx[0][tr] : 1.0f;
            named_bar_sync(pair, 64);  // both have read it before either writes a maximum there
        }
        if constexpr (C::kLowTmem) {  // this thread's half of its row of q once more: what the high part leaves
            const float scale = 1.0f / unscale;  // a power of two
            const uint32_t rr = row0 + min(tr, n_rows - 1);
            const T *src = reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + tok) * p.ld_q +
                           (uint64_t)(kvh * p.group + rr - tok * p.group) * p.hd;
#pragma unroll 2
            for (uint32_t c = 0; c < 8; c++) {
                uint32_t w[8];
#pragma unroll
                for (uint32_t u = 0; u < 4; u++) {
                    const uint32_t d = 128 * h + 16 * c + 4 * u;
                    const float4 x = live && d < p.hd ? *reinterpret_cast<const float4 *>(src + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const float2 a = make_float2(x.x * scale, x.y * scale), b = make_float2(x.z * scale, x.w * scale);
                    const float2 ah = unpack2<E>(pack2<E>(a.x, a.y)), bh = unpack2<E>(pack2<E>(b.x, b.y));
                    w[2 * u] = pack2<E>(a.x - ah.x, a.y - ah.y);
                    w[2 * u + 1] = pack2<E>(b.x - bh.x, b.y - bh.y);
                }
                tl_tmem_st8(tmem + 384 + 64 * h + 8 * c + lanes, w);
            }
            tmem_wait_st();
            tc_fence_before();
            named_bar_sync(11, 288);
        }
        const float cs = p.softcap > 0.0f ? 1.0f : unscale * kLog2e;
        float m = -INFINITY, l = 0.0f;  // m in units of log2, as last rescaled to
        float o[kSplit ? HDP / 2 : 1];  // f32: this thread's half of O's columns, without the last block
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < HDP / 2; i++) o[i] = 0.0f;
        }
        // After a wait that ran out (the result is void) the warps go on without waiting, so that no
        // barrier among them lacks one.
        bool ok = true;
        for (int32_t j = jb[t]; j < je[t]; j++) {
            ok = ok && mbar_wait_spin(&sm.s_full[t], (j - jb[t]) & 1, p.b.err, ERR_TIMEOUT_FULL);
            tc_fence_after();
            const int32_t key0 = j * kTlBlk + 64 * (int32_t)h;
            const bool part = key0 < all_lo || key0 + 63 > all_hi;
            const int32_t rlo = lo - key0, rhi = hi - key0;
            // 16 scores of chunk c: softcapped (then in units of log2), masked
            auto shape = [&](int c, uint32_t (&s)[16]) {
                if (p.softcap > 0.0f) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[i] = __float_as_uint(p.softcap * kLog2e * tanhf(__uint_as_float(s[i]) * unscale / p.softcap));
                }
                if (part) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (16 * c + i > rhi || 16 * c + i < rlo) s[i] = 0xff800000u;
                }
            };
            const bool shaped = part || p.softcap > 0.0f;
            // 16-bit: the scores stay in registers. f32: they are read again after the maximum, since
            // the registers hold O.
            uint32_t s[kSplit ? 2 : 4][16];
            float mx = -INFINITY;
            if constexpr (!kSplit) {
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld16(ts + 16 * c, s[c]);
                tmem_wait_ld();
                if (shaped) {
#pragma unroll
                    for (int c = 0; c < 4; c++) shape(c, s[c]);
                }
                mx = max3_nan(max3_nan(tl_max16(s[0]), tl_max16(s[1]), tl_max16(s[2])), tl_max16(s[3]), -INFINITY);
            } else {
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    tmem_ld16(ts + 16 * c, s[0]);
                    tmem_ld16(ts + 16 * c + 16, s[1]);
                    tmem_wait_ld();
                    if (shaped) shape(c, s[0]), shape(c + 1, s[1]);
                    mx = max3_nan(mx, tl_max16(s[0]), tl_max16(s[1]));
                }
            }
            sm.mx[h][tr] = mx;
            if constexpr (kSplit) {
                // Add the last block's P V, before the pair's barrier: the next P V starts when the first
                // half's P is there and writes all of O's columns, the other half's among them.
                if (j > jb[t]) {
#pragma unroll
                    for (int c = 0; c < HDP / 16; c++) {
                        uint32_t v[8];
                        tl_tmem_ld8(to + 8 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++) o[8 * c + i] += __uint_as_float(v[i]);
                    }
                    tc_fence_before();
                }
            }
            named_bar_sync(pair, 64);
            if constexpr (kSplit) tc_fence_after();
            mx = max3_nan(mx, sm.mx[h ^ 1][tr], -INFINITY) * cs;
            const bool grow = kSplit ? mx > m : mx > m + kTlLazy || (m == -INFINITY && mx > m);
            if (__any_sync(0xffffffffu, grow)) {  // the same for the other warp of these rows
                const float mn = grow ? mx : m;
                const float a = mn == m ? 1.0f : ex2(m - mn);
                m = mn;
                l *= a;
                if constexpr (kSplit) {
#pragma unroll
                    for (int i = 0; i < HDP / 2; i++) o[i] *= a;
                } else if (j > jb[t]) {  // the S that was waited for comes after the last P V
#pragma unroll
                    for (int c = 0; c < HDP / 16; c++) {  // few registers at a time: the scores hold most
                        uint32_t v[8];
                        tl_tmem_ld8(to + 8 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * a);
                        tl_tmem_st8(to + 8 * c, v);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    named_bar_sync(pair, 64);  // neither half's P goes on before all of O is rescaled
                    tc_fence_after();
                }
            }
            const float off = (m == -INFINITY ? 0.0f : m) - kTlShift;
            float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t (&x)[16] = s[kSplit ? 0 : c];
                if constexpr (kSplit) {
                    tmem_ld16(ts + 16 * c, x);
                    tmem_wait_ld();
                    if (shaped) shape(c, x);
                }
                uint32_t u[8], w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float2 y = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])),
                                          make_float2(cs, cs), make_float2(-off, -off));
                    const float2 e = make_float2(ex2(y.x), ex2(y.y));
                    if (i & 1) sum1 = add2(sum1, e);
                    else sum0 = add2(sum0, e);
                    u[i] = pack2<E>(e.x, e.y);
                    if constexpr (kSplit) {
                        const float2 f = unpack2<E>(u[i]);
                        w[i] = pack2<E>(e.x - f.x, e.y - f.y);
                    }
                }
                tl_tmem_st8(ts + 16 * c, u);
                if constexpr (kSplit) tl_tmem_st8(ts + 16 * c + 8, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(h ? &sm.p_full[t] : &sm.p_half[t]);
            l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
        }
        // this tile's MMAs have ended (when a cluster joins, every MMA: O goes over Q and the ring)
        const bool own = je[t] > jb[t];
        if (p.splits > 1 || own) ok = ok && mbar_wait_spin(p.splits > 1 ? &sm.done : &sm.o_done[t], 0, p.b.err, ERR_TIMEOUT_DRAIN);
        tc_fence_after();
        const bool any = own && ok;
        if (t < n_tiles) {
            if (h == 1) sm.mx[1][tr] = l;
            named_bar_sync(pair, 64);
            if (h == 0) l += sm.mx[1][tr], sm.mx[0][tr] = m, sm.mx[1][tr] = l;
            named_bar_sync(pair, 64);
            l = sm.mx[1][tr];
        }
        // this thread's half of O's columns, 8 at a time
        auto columns = [&](int c, float (&x)[8]) {
            uint32_t v[8];
            if (any) {
                tl_tmem_ld8(to + 8 * c, v);
                tmem_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = any ? __uint_as_float(v[i]) : 0.0f;
                if constexpr (kSplit) x[i] += o[8 * c + i];
            }
        };
        if (p.splits == 1) {
            // rounded rows through shared memory (over the tile's own Q, 16-byte chunks swizzled by row),
            // so that neighbouring lanes store neighbouring bytes: a row of each lane's own cost 9000
            // cycles a CTA against 3000
            if (t < n_tiles) {
                constexpr int kRowB = HDP * sizeof(T), kVec = kRowB / 16, kPer = 16 / sizeof(T);  // bytes, chunks, values a chunk
                uint8_t *st = sm.data + t * 128 * kRowB;
                const float inv = 1.0f / l;
                float chk = 0.0f;
#pragma unroll
                for (int c = 0; c < HDP / 16; c++) {
                    float x[8];
                    columns(c, x);
                    alignas(16) T y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float f = x[i] * inv;
                        chk = fmaf(f, 0.0f, chk);  // NaN from a value that is not finite
                        y[i] = from_f32<T>(f);
                    }
#pragma unroll
                    for (int i = 0; i < (int)sizeof(T) / 2; i++)
                        *reinterpret_cast<uint4 *>(st + r * kRowB + ((((kVec / 2 * h) + (int)sizeof(T) / 2 * c + i) ^ (r & 7)) << 4)) =
                            reinterpret_cast<const uint4 *>(y)[i];
                }
                tc_fence_before();
                named_bar_sync(9 + t, 256);
                constexpr int kLanes = kVec < 32 ? kVec : 32, kRows = 32 / kLanes;
#pragma unroll 4
                for (uint32_t k = 0; k < 16 / kRows; k++) {
                    const uint32_t i = ((sw & 7) * (16 / kRows) + k) * kRows + lane / kLanes;
                    if (128 * t + i >= n_rows) continue;
                    const uint32_t rr = row0 + 128 * t + i;
                    const uint32_t tk = div_group(p, rr);
                    T *orow = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + tk) * p.ld_out +
                              (uint64_t)(kvh * p.group + rr - tk * p.group) * p.hd;
#pragma unroll
                    for (uint32_t ch = lane % kLanes; ch < (uint32_t)kVec; ch += kLanes)
                        if (ch * kPer < p.hd)
                            *reinterpret_cast<uint4 *>(orow + ch * kPer) = *reinterpret_cast<const uint4 *>(st + i * kRowB + ((ch ^ (i & 7)) << 4));
                }
                uint32_t bad = __ballot_sync(0xffffffffu, live && chk != 0.0f && !seq_row_settled<T>(m, l));
                if (lane == 0) sm.mx[h][128 * t + 32 * (warp & 3)] = __uint_as_float(bad);
                named_bar_sync(9 + t, 256);  // every row is written: now the ones that are not finite again
                bad |= __float_as_uint(sm.mx[h ^ 1][128 * t + 32 * (warp & 3)]);
                bad &= h ? 0xaaaaaaaau : 0x55555555u;  // shared by the two warps of these rows
                while (bad) {
                    const int b = __ffs((int)bad) - 1;
                    bad &= bad - 1;
                    const uint32_t rr = row0 + 128 * t + 32 * (warp & 3) + b;
                    seq_attn_row<T, E, HDP>(p, sp, div_group(p, rr), kvh, rr - div_group(p, rr) * p.group);
                }
            }
            tc_fence_before();
            __syncthreads();  // tensor memory may go
            return;
        }
        // ---- joined over the cluster: every CTA's O in its shared memory (16-byte chunks swizzled by
        // row, over Q and the ring), then the rows are shared out over the cluster's warps ----
        if (t < n_tiles) {
            float *orow = reinterpret_cast<float *>(sm.data) + tr * HDP;
#pragma unroll
            for (int c = 0; c < HDP / 16; c++) {
                float x[8];
                columns(c, x);
#pragma unroll
                for (int i = 0; i < 2; i++)
                    *reinterpret_cast<float4 *>(orow + (((HDP / 8 * h + 2 * c + i) ^ (r & (HDP / 4 - 1))) << 2)) =
                        make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
        }
        tc_fence_before();
        cluster_sync_all();
        // weight of each CTA's part of row i: 2^(m_c - max m) / sum_c l_c 2^(m_c - max m)
        constexpr uint32_t kSettled = 0x7ffffffeu;  // a NaN
        float *wt = reinterpret_cast<float *>(sm.data + kTlRows * HDP * 4);
        if (threadIdx.x - 32 * kSoft0 < n_rows) {
            const uint32_t i = threadIdx.x - 32 * kSoft0, am = smem_u32(&sm.mx[0][i]), al = smem_u32(&sm.mx[1][i]);
            float mc[kTlMaxCluster], lc[kTlMaxCluster], M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int c = 0; c < kTlMaxCluster; c++) {
                mc[c] = c < (int)p.splits ? ld_cluster_f32(cluster_addr(am, c)) : -INFINITY;
                lc[c] = c < (int)p.splits ? ld_cluster_f32(cluster_addr(al, c)) : 0.0f;
                M = fmaxf(M, mc[c]);
            }
#pragma unroll
            for (int c = 0; c < kTlMaxCluster; c++) {
                mc[c] = mc[c] == -INFINITY ? 0.0f : ex2(mc[c] - M);
                if (c < (int)p.splits) L = fmaf(mc[c], lc[c], L);
            }
            const float inv = 1.0f / L;
#pragma unroll
            for (int c = 0; c < kTlMaxCluster; c++)
                if (c < (int)p.splits) wt[c * kTlRows + i] = mc[c] * inv;
            // no keys, or a NaN: the row is made again, unless NaN is its answer
            if (!isfinite(inv)) wt[i] = __uint_as_float(seq_row_settled<T>(M, L) ? kSettled : 0x7fffffffu);
        }
        named_bar_sync(15, kTlSoftWarps * 32);
        constexpr int kVec = HDP / 4, kLn = kVec < 32 ? kVec : 32, kPerRow = kVec / kLn;  // 16-byte chunks of a row, lanes, chunks a lane
        const uint32_t step = p.splits * kTlSoftWarps * 32 / kLn;
#pragma unroll 2
        for (uint32_t i = (rank * kTlSoftWarps + sw) * (32 / kLn) + lane / kLn; i - lane / kLn < n_rows; i += step) {
            const bool in = i < n_rows;
            const uint32_t rr = row0 + (in ? i : 0), tk = div_group(p, rr), gq = rr - tk * p.group;
            T *orow = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + tk) * p.ld_out + (uint64_t)(kvh * p.group + gq) * p.hd;
            bool fine = true;
#pragma unroll
            for (int u = 0; u < kPerRow; u++) {
                const uint32_t ch = lane % kLn + 32 * u;
                const uint32_t a = smem_u32(sm.data) + (in ? i * HDP * 4 + ((ch ^ (i & (kVec - 1))) << 4) : 0);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < kTlMaxCluster; c++) {
                    if (c >= (int)p.splits || !in) continue;
                    const float w = wt[c * kTlRows + i];
                    const float4 x = ld_cluster_f32x4(cluster_addr(a, c));
                    if (w != 0.0f) v = make_float4(fmaf(w, x.x, v.x), fmaf(w, x.y, v.y), fmaf(w, x.z, v.z), fmaf(w, x.w, v.w));
                }
                if (!in || 4 * ch >= p.hd) continue;
                fine = fine && isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(orow + 4 * ch) = v;
                else *reinterpret_cast<uint2 *>(orow + 4 * ch) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
            }
            if (in && __float_as_uint(wt[i]) == kSettled) fine = true;
            uint32_t bad = __ballot_sync(0xffffffffu, !fine);
            if (bad) {
                __syncwarp();
#pragma unroll 1
                for (int r = 0; r < 32 / kLn; r++)
                    if (bad >> (r * kLn) & (kLn == 32 ? 0xffffffffu : (1u << kLn) - 1)) {
                        const uint32_t rb = __shfl_sync(0xffffffffu, rr, r * kLn);
                        seq_attn_row<T, E, HDP>(p, sp, div_group(p, rb), kvh, rb - div_group(p, rb) * p.group);
                    }
            }
        }
        cluster_sync_all();  // no CTA leaves while another reads its shared memory
        return;
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_free<C::kTmem>(tmem);
    }
    if (p.splits > 1) cluster_sync_all();
}

// ---- host ---------------------------------------------------------------------------------------
// How many CTAs share a tile's keys, by the time that the launch takes in blocks of keys (about 1.8 us
// each): a CTA's share of the blocks and, for its start and end, 5 more (7 with the join). Two CTAs on
// an SM hide a part of those (3.5 and 6), but bring each block in twice and take 9 % longer. A launch
// that does not fill the device takes as long as its longest tile. Beyond that tiles of unequal
// lengths share the SMs evenly and end a fifth of a tile late, equal ones run in whole waves. The
// average tile of a prompt over itself has half the keys, one of several sequences 0.6 of the longest.
// (128 rows over 8128 keys, 8 KV heads, f16: two tiles a CTA 123, 71, 43, 57 us by 1, 2, 4, 8 CTAs,
// where the device does not hold all clusters of 8; one tile 116, 65, 39, 30. 16 sequences of 250 ..
// 5333 keys, two chunks of 333 rows among them: 75, 64, 87, 156 and 107, 59, 67, 109. 16 prompts of 65
// .. 2047 tokens: 295 and 278 by one CTA. One prompt of 8192: 480 and 510. 512 rows over 12,800 keys:
// 190, 106, 118, 187 and 181, 111, 120, 151.)
struct TlPlan {
    uint32_t splits;
    double cost;
};
template <typename T, typename E, int HDP, int TILES>
static int plan_tile(rcu_ctx *ctx, const SeqAttnParams &p, uint64_t max_len, TlPlan *plan) {
    using C = TlCfg<HDP, std::is_same<T, float>::value, TILES>;
    constexpr size_t smem = sizeof(TlSmem<HDP, std::is_same<T, float>::value, TILES>);
    const double items = (double)seq_tiles_bound(p.b.n_tok, p.b.n_seq, p.group, C::kRows) * p.n_kv;
    const uint64_t span = p.window > 0 ? std::min<uint64_t>(max_len, p.window + C::kRows) : max_len;
    const double blocks = (double)((span + kTlBlk - 1) / kTlBlk);
    const double part = p.window > 0 ? 0.0 : std::min(1.0, (double)p.b.n_tok / ((double)p.b.n_seq * max_len));
    const double mean = (p.b.n_seq > 1 ? 0.6 : 1.0) * (1.0 - 0.5 * part);  // of `blocks`
    *plan = {1, 0.0};
    for (int e = 0; 1 << e <= kTlMaxCluster && (e == 0 || blocks >= 2.0 * (1 << e)); e++) {
        int slots = ctx->num_sms * C::kPerSm;
        if (e > 0 && C::kPerSm == 1) {
            if (int st = cluster_slots<k_attn_tile<T, E, HDP, TILES>>(ctx, C::kThreads, smem, e, &slots)) return st;
        } else if (e > 0) {  // n SMs hold as many clusters of 2^e with two CTAs each as of half the size with one
            using W = TlCfg<HDP, false, HDP == 256 ? 1 : 2>;
            constexpr size_t wide = sizeof(TlSmem<HDP, false, W::kTiles>);
            if (e == 1) slots = ctx->num_sms;
            else if (int st = cluster_slots<k_attn_tile<T, E, HDP, W::kTiles>>(ctx, W::kThreads, wide, e - 1, &slots)) return st;
        }
        const double f = items / slots, ends = C::kPerSm == 2 ? (e ? 6.0 : 3.5) : (e ? 7.0 : 5.0);
        const double longest = blocks / (1 << e) + ends, usual = blocks * mean / (1 << e) + ends;
        double cost = f <= 1.0 ? longest : std::max(longest, (mean < 0.8 ? f + 0.2 : std::ceil(f)) * usual);
        if (C::kPerSm == 2) cost *= 1.09;
        if (e == 0 || cost < plan->cost) *plan = {1u << e, cost};
    }
    return RCU_OK;
}

template <typename T, typename E, int HDP, int TILES>
static int launch_tile(rcu_ctx *ctx, const SeqKvMaps &m, SeqAttnParams p, uint32_t splits) {
    using C = TlCfg<HDP, std::is_same<T, float>::value, TILES>;
    constexpr size_t smem = sizeof(TlSmem<HDP, std::is_same<T, float>::value, TILES>);
    static_assert(smem <= 232448 && (smem + 1024) * C::kPerSm <= 233472, "shared memory of one CTA, of an SM");
    p.n_tiles = (uint32_t)seq_tiles_bound(p.b.n_tok, p.b.n_seq, p.group, C::kRows);
    p.splits = splits;
    const uint64_t grid = (uint64_t)p.n_tiles * p.n_kv * splits;
    if (grid > 0x7fffffffull) return set_err(ctx, RCU_ERR_INVALID, "attention: too many work tiles");
    return launch_cluster_k<k_attn_tile<T, E, HDP, TILES>>(ctx, (uint32_t)grid, C::kThreads, smem, splits, m.k, m.v, p);
}

// The form with the smaller cost. head_dim above 128 has one tile a CTA, f32 queries below have two:
// O, or Q's two parts, leave no room for the other form.
template <typename T, typename E, int HDP>
static int launch_tile_form(rcu_ctx *ctx, const SeqKvMaps &m, const SeqAttnParams &p, uint64_t max_len) {
    TlPlan one, two;
    if constexpr (HDP == 256) {
        if (int st = plan_tile<T, E, HDP, 1>(ctx, p, max_len, &one)) return st;
        return launch_tile<T, E, HDP, 1>(ctx, m, p, one.splits);
    } else {
        if (int st = plan_tile<T, E, HDP, 2>(ctx, p, max_len, &two)) return st;
        if constexpr (!std::is_same<T, float>::value) {
            if (int st = plan_tile<T, E, HDP, 1>(ctx, p, max_len, &one)) return st;
            if (one.cost < two.cost) return launch_tile<T, E, HDP, 1>(ctx, m, p, one.splits);
        }
        return launch_tile<T, E, HDP, 2>(ctx, m, p, two.splits);
    }
}

template <typename T, typename E>
static int launch_tile_hd(rcu_ctx *ctx, SeqAttnParams &p, const SeqKvDesc &kv, uint64_t max_len) {
    SeqKvMaps room;
    const SeqKvMaps *m;
    if (int st = seq_pick_maps(ctx, p, kv, kSeqTileBox, kv.tile, &room, &m)) return st;
    if (p.hd <= 64) return launch_tile_form<T, E, 64>(ctx, *m, p, max_len);
    if (p.hd > 128) return launch_tile_form<T, E, 256>(ctx, *m, p, max_len);
    return launch_tile_form<T, E, 128>(ctx, *m, p, max_len);
}

int launch_attention_tile(rcu_ctx *ctx, const SeqAttnParams &params, int q_type, const SeqKvDesc &kv, uint64_t max_len) {
    SeqAttnParams p = params;
    if (q_type == T_F32) return launch_tile_hd<float, __half>(ctx, p, kv, max_len);
    if (q_type == T_F16) return launch_tile_hd<__half, __half>(ctx, p, kv, max_len);
    return launch_tile_hd<__nv_bfloat16, __nv_bfloat16>(ctx, p, kv, max_len);
}

}  // namespace rcu
