// rcu_attn_seq.cu -- attention of a batch of sequences: each sequence's new tokens over its pages
// (chunks of prompts and single-token steps mixed), or whole packed prompts over themselves.
//
// For the new token at position P of a sequence, head h of KV head h / G:
//   s_j = q . k_j  (c * tanh(s_j / c) with a softcap c),  j = max(0, P + 1 - window) .. P
//   o = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
//
// k_attn_seq is the kernel for few query rows per KV head (decode steps, short chunks): it reads
// every key and value once per work tile (4, 8 or 16 rows: token, head of the group) and is bound by
// that reading. A cluster of CTAs shares a tile, and every warp of the cluster takes chunks of 16
// keys in turn, on its own:
//   * its lane 0 brings a chunk's K and V rows in by tiled TMA (128-byte swizzle) two chunks
//     ahead, one mbarrier per stage; a chunk lies in one page, so a page may end anywhere;
//   * S^T = K Q^T and O^T += V^T P^T with mma.sync m16n8k16: keys, then values' columns, fill the 16
//     rows of a fragment and the queries its 8 columns. (With the queries on the 16 rows, four heads
//     of a group waste three quarters of the products, and mma.sync, at a sixteenth of tcgen05's
//     rate, becomes the bound: 278 us against 160 us for two f32 sequences of 131,071 keys.)
//   * running maximum and sum per row in f32; the maximum is raised, and O rescaled, only when a
//     score passes it by more than 2^kSqLazy, which a vote finds without a reduction over the keys.
// No warp waits for another before its last chunk. Then the warps of a CTA join their states in
// shared memory and the CTAs of the cluster through distributed shared memory: one launch, and no
// workspace that two calls or graphs could share.
// 16-bit queries: p is rounded to the values' type, which the MMA takes on both sides (2^-11 or 2^-8 of
// it, no more than the output's own rounding; a second part would double the products). Its sum is not.
// f32 queries: q (scaled by a power of two per row) and p are each split into two f16 parts that take
// columns c and c + 4 of one fragment, so both products carry 22 bits; keys and values are f16 as the
// cache holds them. O is added up outside the MMA, whose own additions do not round to nearest
// (5.6e-6 off after 131,071 keys).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"
#include "rcu_tc.cuh"

namespace rcu {

constexpr int kSqKeys = kSeqFewBox;  // keys of a chunk
constexpr int kSqWarps = 4;
constexpr int kSqStages = 2;  // three CTAs to an SM; with three stages two, of which clusters of 16 leave SMs idle (199 against 159 us)
constexpr int kSqMaxCluster = 16;
constexpr int kSqMaxRows = 16;
// p is held as 2^kSqShift * exp(s - m), the row's largest at most 2^(kSqShift + kSqLazy): in f16 its
// relative precision then reaches down to 2^-21 of exp(0); the sum carries the same factor.
constexpr float kSqLazy = 8.0f, kSqShift = 7.0f;

template <typename E>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void sq_ldsm_x4(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p));
}
__device__ __forceinline__ void sq_ldsm_x4_t(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p));
}
// Byte offset of 16-byte chunk `ch` (of a row's HDP / 8) of row `r` in a tile of `rows` rows that
// TMA wrote as HDP / 64 boxes of 64 elements with the 128-byte swizzle.
__device__ __forceinline__ uint32_t sq_off(uint32_t r, uint32_t ch, uint32_t rows) {
    return (ch >> 3) * (rows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}
// Transposes an 8 x 8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t sq_transpose(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int HDP>
struct SqSmem {
    static constexpr int kTile = kSqKeys * HDP * 2;  // bytes of one chunk's K (or V) rows
    static constexpr int kWarp = kSqStages * 2 * kTile;
    static constexpr int kLd = HDP + 4;              // floats between rows of O
    uint8_t ring[kSqWarps][kWarp];  // at the end: each warp's O, then the CTA's (f32 [rows][kLd])
    float m[kSqWarps][kSqMaxRows], l[kSqWarps][kSqMaxRows];
    float cm[kSqMaxRows], cl[kSqMaxRows];  // of the CTA
    uint64_t full[kSqWarps][kSqStages];
    static_assert(kSqMaxRows * kLd * 4 <= kWarp, "O overlays the ring");
};

template <typename T, typename E, int HDP, int NT>
__global__ void __launch_bounds__(kSqWarps * 32) k_attn_seq(const __grid_constant__ CUtensorMap mk,
                                                            const __grid_constant__ CUtensorMap mv,
                                                            const __grid_constant__ SeqAttnParams p) {
    using S = SqSmem<HDP>;
    constexpr bool kSplit = std::is_same<T, float>::value;
    constexpr int KS = HDP / 16;
    constexpr int kPer = kSplit ? 4 : 8, kRows = kPer * NT;  // rows of a fragment, of the tile
    extern __shared__ uint8_t sq_raw[];
    S &sm = *reinterpret_cast<S *>((reinterpret_cast<uintptr_t>(sq_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const uint32_t item = blockIdx.x / p.splits, kvh = item % p.n_kv, ti = p.n_tiles - 1 - item / p.n_kv;
    pdl_wait();  // the batch, q, k and v may come from the kernel before
    pdl_trigger();
    SeqSpan sp;
    uint32_t tile;
    if (!seq_find_tile(p.b, p.group, kRows, ti, &sp, &tile)) return;  // the same for the whole cluster
    if (lane == 0) {
        for (int s = 0; s < kSqStages; s++) mbar_init(&sm.full[warp][s], 1);
        fence_mbar_init();
    }
    __syncwarp();
    const uint32_t row0 = tile * kRows, n_rows = min(sp.n_new * p.group - row0, (uint32_t)kRows);
    // the tile's attended positions k_lo .. k_hi; positions stay below 2^31
    const int32_t p_first = sp.pos(div_group(p, row0)), k_hi = sp.pos(div_group(p, row0 + n_rows - 1));
    const int32_t k_lo = p.window > 0 ? max(p_first - (int32_t)p.window + 1, 0) : 0;
    const uint32_t c_lo = (uint32_t)(k_lo / kSqKeys), c_all = k_hi >= 0 ? (uint32_t)(k_hi / kSqKeys) + 1 : 0;
    const uint32_t n_chunks = c_all > c_lo ? c_all - c_lo : 0;
    // keys that every live row attends: chunks inside need no mask
    const int32_t all_lo = p.window > 0 ? max(k_hi - (int32_t)p.window + 1, 0) : 0, all_hi = p_first;

    // this warp's chunks: w0, w0 + stride, ... of the tile's n_chunks
    const uint32_t stride = p.splits * kSqWarps, w0 = rank * kSqWarps + warp;
    const uint32_t mine = n_chunks > w0 ? (n_chunks - w0 + stride - 1) / stride : 0;
    uint8_t *ring = sm.ring[warp];
    uint32_t rows_ahead = 0;  // lane l: first key row of chunk (32-chunk group) + l
    auto fetch_rows = [&](uint32_t i0) {
        const uint32_t i = i0 + lane;
        rows_ahead = i < mine ? seq_kv_row(p.b, sp, p.n_kv, kvh, (c_lo + w0 + i * stride) * kSqKeys) : 0;
    };
    auto issue = [&](uint32_t i, uint32_t st) {  // whole warp; brings chunk i into stage st = i % kSqStages
        if ((i & 31) == 0) fetch_rows(i);
        const uint32_t r = __shfl_sync(0xffffffffu, rows_ahead, i & 31);
        if (lane == 0) {
            uint8_t *kd = ring + st * 2 * S::kTile, *vd = kd + S::kTile;
            // a page number out of range reads as zeros: rows behind the tensor's end
            const int y = (int)min(r, p.kv_rows), h = p.b.pages ? 0 : (int)kvh;
            mbar_arrive_expect_tx(&sm.full[warp][st], 2 * S::kTile);
#pragma unroll
            for (int c = 0; c < HDP / 64; c++) {
                tma_load_3d(kd + c * (kSqKeys * 128), &mk, 64 * c, h, y, &sm.full[warp][st]);
                tma_load_3d(vd + c * (kSqKeys * 128), &mv, 64 * c, h, y, &sm.full[warp][st]);
            }
        }
    };
    for (uint32_t i = 0; i < min(mine, (uint32_t)kSqStages); i++) issue(i, i);

    // q as B fragments: column g of fragment n (f32: row 4 n + g % 4, its high part in columns 0-3, the
    // rest in 4-7, the row scaled by 2^-e, e from its largest value)
    uint32_t q[NT][KS][2];
    float unscale[NT][2];  // 2^e of this thread's score rows
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t r = kPer * n + g % kPer, rr = row0 + min(r, n_rows - 1);
        const bool live = r < n_rows;
        const uint32_t tok = div_group(p, rr);
        const T *src = reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + tok) * p.ld_q +
                       (uint64_t)(kvh * p.group + rr - tok * p.group) * p.hd;
        if constexpr (kSplit) {
            float2 x[KS][2];
            float mx = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t col = 16 * ks + 8 * j + 2 * t4;
                    x[ks][j] = live && col < p.hd ? *reinterpret_cast<const float2 *>(src + col) : make_float2(0.0f, 0.0f);
                    mx = fmaxf(mx, fmaxf(fabsf(x[ks][j].x), fabsf(x[ks][j].y)));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // exponents at which both 2^e and 2^-e are normal numbers
            const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255), 2), 252) - 127;
            const float scale = __uint_as_float((uint32_t)(127 - e) << 23), un = __uint_as_float((uint32_t)(127 + e) << 23);
            unscale[n][0] = __shfl_sync(0xffffffffu, un, 4 * (2 * (t4 & 1)));
            unscale[n][1] = __shfl_sync(0xffffffffu, un, 4 * (2 * (t4 & 1) + 1));
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float a = x[ks][j].x * scale, b = x[ks][j].y * scale;
                    const uint32_t h = pack2<E>(a, b);
                    const float2 f = unpack2<E>(h);
                    q[n][ks][j] = g < 4 ? h : pack2<E>(a - f.x, b - f.y);
                }
        } else {
            unscale[n][0] = unscale[n][1] = 1.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t col = 16 * ks + 8 * j + 2 * t4;
                    q[n][ks][j] = live && col < p.hd ? *reinterpret_cast<const uint32_t *>(src + col) : 0u;
                }
        }
    }
    float sc[NT][2];  // scores times sc are in units of log2
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) sc[n][i] = p.softcap > 0.0f ? 1.0f : unscale[n][i] * kLog2e;
    // this thread's scores: keys g and g + 8 of a chunk, rows srow[n][0..1] of the tile, which attend
    // positions slo .. shi
    int32_t slo[NT][2], shi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t r = kPer * n + (2 * t4 + i) % kPer;
            shi[n][i] = r < n_rows ? sp.pos(div_group(p, row0 + r)) : -1;
            slo[n][i] = p.window > 0 ? max(shi[n][i] - (int32_t)p.window + 1, 0) : 0;
        }
    float o[NT][KS][4];  // O^T: columns 16 ks + g (+ 8) of rows as the scores' (f32: high parts, the rest)
    float m[NT][2], l[NT][2];  // m in units of log2
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) o[n][ks][0] = o[n][ks][1] = o[n][ks][2] = o[n][ks][3] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }

    bool ok = true;
    uint32_t st = 0, parity = 0;
    const uint32_t mi = lane >> 3, l7 = lane & 7;
    for (uint32_t i = 0; i < mine; i++) {
        ok = mbar_wait_spin(&sm.full[warp][st], parity, p.b.err, ERR_TIMEOUT_FULL);
        if (!ok) {  // the result is void; the copies still in flight must land before the CTA ends
            for (uint32_t j = i + 1; j < min(mine, i + kSqStages); j++)
                mbar_wait_spin(&sm.full[warp][j % kSqStages], (j / kSqStages) & 1, p.b.err, ERR_TIMEOUT_FULL);
            break;
        }
        uint8_t *vrows = ring + st * 2 * S::kTile + S::kTile;
        const uint32_t kb = smem_u32(ring + st * 2 * S::kTile), vb = kb + S::kTile;
        const int32_t c0 = (int32_t)(c_lo + w0 + i * stride) * kSqKeys;
        const bool part = c0 < all_lo || c0 + kSqKeys - 1 > all_hi;
        if (c0 + kSqKeys - 1 > k_hi) {  // rows behind the last key hold anything: 0 * v must stay 0
            for (uint32_t r = (uint32_t)(k_hi - c0 + 1); r < kSqKeys; r++)
                for (uint32_t c = lane; c < HDP / 8; c += 32)
                    *reinterpret_cast<uint4 *>(vrows + sq_off(r, c, kSqKeys)) = make_uint4(0, 0, 0, 0);
            fence_async_smem();
            __syncwarp();
        }
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t r[4];
            sq_ldsm_x4(r, kb + sq_off(8 * (mi & 1) + l7, 2 * ks + (mi >> 1), kSqKeys));
#pragma unroll
            for (int n = 0; n < NT; n++) mma_16816<E>(s[n], r, q[n][ks][0], q[n][ks][1]);
        }
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) {  // key g + 8 (j >> 1), row j & 1
                float v = s[n][j];
                if constexpr (kSplit) v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (p.softcap > 0.0f) v = p.softcap * kLog2e * tanhf(v * unscale[n][j & 1] / p.softcap);
                if (part) {
                    const int32_t key = c0 + (int32_t)g + 8 * (j >> 1);
                    if (key > shi[n][j & 1] || key < slo[n][j & 1]) v = -INFINITY;
                }
                s[n][j] = v;
                v *= sc[n][j & 1];
                grow |= v > m[n][j & 1] + kSqLazy || (m[n][j & 1] == -INFINITY && v > -INFINITY);
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float mx = fmaxf(fmaxf(s[n][k], s[n][2 + k]) * sc[n][k], m[n][k]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float a = mx == m[n][k] ? 1.0f : ex2(m[n][k] - mx);
                    m[n][k] = mx;
                    l[n][k] *= a;
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) o[n][ks][k] *= a, o[n][ks][2 + k] *= a;
                }
        }
        uint32_t b[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                e[j] = ex2(fmaf(s[n][j], sc[n][j & 1], kSqShift - (m[n][j & 1] == -INFINITY ? 0.0f : m[n][j & 1])));
                l[n][j & 1] += e[j];
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                uint32_t u = pack2<E>(e[2 * k], e[2 * k + 1]);
                if constexpr (kSplit) {
                    const float2 f = unpack2<E>(u);
                    if (t4 >= 2) u = pack2<E>(e[2 * k] - f.x, e[2 * k + 1] - f.y);
                }
                b[n][k] = sq_transpose(u);
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t r[4];
            sq_ldsm_x4_t(r, vb + sq_off(8 * (mi >> 1) + l7, 2 * ks + (mi & 1), kSqKeys));
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if constexpr (kSplit) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_16816<E>(d, r, b[n][0], b[n][1]);
#pragma unroll
                    for (int j = 0; j < 4; j++) o[n][ks][j] += d[j];
                } else {
                    mma_16816<E>(o[n][ks], r, b[n][0], b[n][1]);
                }
            }
        }
        __syncwarp();  // every lane has read the stage
        if (i + kSqStages < mine) issue(i + kSqStages, st);
        if (++st == kSqStages) st = 0, parity ^= 1;
    }
    // ---- join: warps of the CTA, then CTAs of the cluster -----------------------------------------
    // this warp's ring is free (all its copies were waited for, or its wait ran out and the result is void)
    float *ow = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 4);
            l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 8);
            l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 16);
            if (g == 0 && 2 * t4 < kPer) sm.m[warp][kPer * n + 2 * t4 + k] = m[n][k], sm.l[warp][kPer * n + 2 * t4 + k] = l[n][k];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float v = o[n][ks][j];
                if constexpr (kSplit) v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (2 * t4 < kPer && ok) ow[(kPer * n + 2 * t4 + (j & 1)) * S::kLd + 16 * ks + g + 8 * (j >> 1)] = v;
            }
    }
    __syncthreads();
    float *oc = reinterpret_cast<float *>(sm.ring[0]);
    constexpr int kOw = S::kWarp / 4;  // floats between two warps' O
    for (uint32_t r = warp; r < n_rows; r += kSqWarps) {
        float M = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kSqWarps; w++) M = fmaxf(M, sm.m[w][r]);
        float a[kSqWarps], L = 0.0f;
#pragma unroll
        for (int w = 0; w < kSqWarps; w++) {
            a[w] = sm.m[w][r] == -INFINITY ? 0.0f : ex2(sm.m[w][r] - M);
            L += a[w] * sm.l[w][r];
        }
        for (uint32_t d = lane; d < HDP; d += 32) {
            float acc = 0.0f;
#pragma unroll
            for (int w = 0; w < kSqWarps; w++)
                if (a[w] != 0.0f) acc += a[w] * oc[w * kOw + r * S::kLd + d];
            oc[r * S::kLd + d] = acc;
        }
        if (lane == 0) sm.cm[r] = M, sm.cl[r] = L;
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    // rows of the result are shared out over the warps of the cluster
    for (uint32_t r = w0; r < n_rows; r += stride) {
        float L, M;
        float acc[HDP / 32] = {};
        if (p.splits == 1) {
            L = sm.cl[r], M = sm.cm[r];
            for (int i = 0; i < HDP / 32; i++) acc[i] = oc[r * S::kLd + lane + 32 * i];
        } else {
            const uint32_t am = smem_u32(&sm.cm[r]), al2 = smem_u32(&sm.cl[r]), ao = smem_u32(oc + r * S::kLd + lane);
            const float mc = lane < p.splits ? ld_cluster_f32(cluster_addr(am, lane)) : -INFINITY;
            const float lc = lane < p.splits ? ld_cluster_f32(cluster_addr(al2, lane)) : 0.0f;
            M = mc;
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
                for (int i = 0; i < HDP / 32; i++) acc[i] = fmaf(w, ld_cluster_f32(a + 128 * i), acc[i]);
            }
        }
        const uint32_t rr = row0 + r, t = div_group(p, rr), gq = rr - t * p.group;
        T *orow = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + t) * p.ld_out + (uint64_t)(kvh * p.group + gq) * p.hd;
        bool fine = true;
#pragma unroll
        for (int i = 0; i < HDP / 32; i++) {
            const uint32_t d = lane + 32 * i;
            const float v = acc[i] / L;
            fine = fine && (isfinite(v) || d >= p.hd);
            if (d < p.hd) orow[d] = from_f32<T>(v);
        }
        if (!__all_sync(0xffffffffu, fine) && !seq_row_settled<T>(M, L)) {
            __syncwarp();
            seq_attn_row<T, E, HDP>(p, sp, t, kvh, gq);
        }
    }
    if (p.splits > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// ---- host ---------------------------------------------------------------------------------------
template <typename T, typename E, int HDP, int NT>
static int launch_few(rcu_ctx *ctx, const SeqKvMaps &m, SeqAttnParams p, uint64_t max_len) {
    const size_t smem = sizeof(SqSmem<HDP>) + 1024;
    p.n_tiles = (uint32_t)seq_tiles_bound(p.b.n_tok, p.b.n_seq, p.group, (std::is_same<T, float>::value ? 4 : 8) * NT);
    // CTAs per tile: up to three for each SM in all, and at least 64 keys each (a chunk for each warp;
    // eight warps a CTA instead were slower: clusters of 16 such CTAs do not all find SMs at once)
    const uint64_t items = (uint64_t)p.n_tiles * p.n_kv, span = p.window > 0 ? std::min<uint64_t>(max_len, p.window + 16) : max_len;
    const uint32_t most = HDP == 256 ? 8 : kSqMaxCluster;  // one CTA to an SM: eight SMs of a GPC are sure to be there
    uint32_t cs = 1;
    while (cs < most && items * cs * 2 <= 3ull * ctx->num_sms && span >= (uint64_t)cs * 2 * 64) cs *= 2;
    p.splits = cs;
    if (items * cs > 0x7fffffffull) return set_err(ctx, RCU_ERR_INVALID, "attention: too many work tiles");
    return launch_cluster_k<k_attn_seq<T, E, HDP, NT>>(ctx, (uint32_t)(items * cs), kSqWarps * 32, smem, cs, m.k, m.v, p);
}

// One fragment of rows where they fill no more (a group's heads for single tokens), else two.
template <typename T, typename E>
static int launch_few_hd(rcu_ctx *ctx, const SeqAttnParams &p, const SeqKvDesc &kv, uint64_t max_len, uint64_t most) {
    SeqKvMaps room;
    const SeqKvMaps *m;
    if (int st = seq_pick_maps(ctx, p, kv, kSeqFewBox, kv.few, &room, &m)) return st;
    if (most <= (std::is_same<T, float>::value ? 4u : 8u)) {
        if (p.hd <= 64) return launch_few<T, E, 64, 1>(ctx, *m, p, max_len);
        if (p.hd <= 128) return launch_few<T, E, 128, 1>(ctx, *m, p, max_len);
        return launch_few<T, E, 256, 1>(ctx, *m, p, max_len);
    }
    if (p.hd <= 64) return launch_few<T, E, 64, 2>(ctx, *m, p, max_len);
    if (p.hd <= 128) return launch_few<T, E, 128, 2>(ctx, *m, p, max_len);
    return launch_few<T, E, 256, 2>(ctx, *m, p, max_len);
}

static int launch_attention_few(rcu_ctx *ctx, const SeqAttnParams &p, int q_type, const SeqKvDesc &kv, uint64_t max_len,
                                uint64_t most) {
    if (q_type == T_F32) return launch_few_hd<float, __half>(ctx, p, kv, max_len, most);
    if (q_type == T_F16) return launch_few_hd<__half, __half>(ctx, p, kv, max_len, most);
    return launch_few_hd<__nv_bfloat16, __nv_bfloat16>(ctx, p, kv, max_len, most);
}

int launch_seq_attention(rcu_ctx *ctx, const SeqAttnParams &p, int q_type, const SeqKvDesc &kv, uint64_t max_len,
                         uint64_t max_new) {
    // The most query rows that a sequence may have in one KV head. Without max_new, as many new rows as
    // sequences are taken for single tokens, and more for one sequence's; what is there in fact decides
    // only how fast the launch is (32 sequences of 2 tokens over 2000 keys, 8 KV heads of 4: f32 103 us
    // so and 58 with max_new, f16 56 and 54). One kernel takes the whole batch: in a mixed one the single
    // tokens ride along with the chunks (two chunks of 333 tokens beside 14 single ones: 59 us; 37 us
    // for the chunks and 23 us for the single tokens in launches of their own).
    const uint64_t new_max = max_new ? max_new : p.b.n_tok <= p.b.n_seq ? 1 : p.b.n_tok;
    const uint64_t most = std::min<uint64_t>(new_max, p.b.n_tok) * p.group;
    // Above kSqMaxRows rows k_attn_seq reads keys and values more than once, which costs most where the
    // sequences fill the device.
    const bool full = most > kSqMaxRows && p.b.n_seq * p.n_kv >= kTileMinPairs;
    if (most < kTileMinRows && !full) return launch_attention_few(ctx, p, q_type, kv, max_len, most);
    return launch_attention_tile(ctx, p, q_type, kv, max_len);
}

}  // namespace rcu
