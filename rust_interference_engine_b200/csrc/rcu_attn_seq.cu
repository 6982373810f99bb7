// rcu_attn_seq.cu -- attention of a batch of sequences: each sequence's new tokens over its pages
// (chunks of prompts and single-token steps mixed), or whole packed prompts over themselves.
//
// For the new token at position P of a sequence, head h of KV head h / G:
//   s_j = q . k_j  (c * tanh(s_j / c) with a softcap c),  j = max(0, P + 1 - window) .. P
//   o = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
//
// k_attn_seq is the kernel for few query rows per KV head (decode steps, short chunks): it reads
// every key and value once per 16 query rows and is bound by that reading. A work tile is 16 rows
// (token, head of the group) of one sequence and KV head; a cluster of CTAs shares it, and every
// warp of the cluster takes chunks of 16 keys in turn, on its own:
//   * its lane 0 brings a chunk's K and V rows in by tiled TMA (128-byte swizzle) three chunks
//     ahead, one mbarrier per stage; a chunk lies in one page, so a page may end anywhere;
//   * S = Q K^T and O += P V with mma.sync m16n8k16 (f32 accumulation): 16 rows fill one fragment;
//   * running maximum and sum per row in f32. No warp waits for another before its last chunk.
// Then the warps of a CTA join their states in shared memory and the CTAs of the cluster through
// distributed shared memory: one launch, and no workspace that two calls or graphs could share.
// f32 queries: q (scaled by a power of two per row) and p are each split into two f16 parts, so
// both products carry 22 bits; keys and values are f16 as the cache holds them.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"
#include "rcu_tc.cuh"

namespace rcu {

constexpr int kSqRows = 16;     // query rows of a work tile
constexpr int kSqKeys = 16;     // keys of a chunk
constexpr int kSqWarps = 4;
constexpr int kSqStages = 3;
constexpr int kSqMaxCluster = 16;
// p is held as 2^kPShift * exp(s - max): in f16 its relative precision then reaches down to
// 2^-26 of the largest probability; the sum carries the same factor.
constexpr float kPShift = 12.0f;

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
template <int HDP>
struct SqSmem {
    static constexpr int kTile = kSqKeys * HDP * 2;  // bytes of one chunk's K (or V) rows
    static constexpr int kWarp = kSqStages * 2 * kTile;
    uint8_t ring[kSqWarps][kWarp];  // at the end: each warp's O, then the CTA's (f32 [16][HDP])
    float m[kSqWarps][kSqRows], l[kSqWarps][kSqRows];
    float cm[kSqRows], cl[kSqRows];  // of the CTA
    uint64_t full[kSqWarps][kSqStages];
};

// q as fragments: rows g and g + 8 of the tile, 16 columns a step; f32 rows are scaled by 2^-e
// (e from the row's largest value) and split in two, and `unscale` is then 2^e.
template <typename T, typename E, int HDP>
struct SqFrag {
    static constexpr bool kSplit = std::is_same<T, float>::value;
    static constexpr int KS = HDP / 16;
    uint32_t hi[KS][4], lo[kSplit ? KS : 1][4];
    float unscale[2];

    __device__ __forceinline__ void load(const SeqAttnParams &p, const SeqSpan &sp, uint32_t kvh, const uint32_t (&row)[2],
                                         const bool (&live)[2]) {
        const uint32_t t4 = threadIdx.x & 3;
        const T *src[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            src[i] = reinterpret_cast<const T *>(p.q) + (uint64_t)(sp.first + row[i] / p.group) * p.ld_q +
                     (uint64_t)(kvh * p.group + row[i] % p.group) * p.hd;
        float scale[2] = {1.0f, 1.0f};
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float mx = 0.0f;
                for (uint32_t c = 2 * t4; c < p.hd; c += 8)
                    if (live[i]) mx = fmaxf(mx, fmaxf(fabsf(to_f32(src[i][c])), fabsf(to_f32(src[i][c + 1]))));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                // exponents at which both 2^e and 2^-e are normal numbers
                const int e = min(max((int)((__float_as_uint(mx) >> 23) & 255), 2), 252) - 127;
                scale[i] = __uint_as_float((uint32_t)(127 - e) << 23);
                unscale[i] = __uint_as_float((uint32_t)(127 + e) << 23);
            }
        } else {
            unscale[0] = unscale[1] = 1.0f;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = j & 1;
                const uint32_t col = 16 * ks + 2 * t4 + (j >= 2 ? 8 : 0);
                float2 x = make_float2(0.0f, 0.0f);
                if constexpr (kSplit) {
                    if (live[i] && col < p.hd) x = *reinterpret_cast<const float2 *>(src[i] + col);
                    x.x *= scale[i], x.y *= scale[i];
                    hi[ks][j] = pack2<E>(x.x, x.y);
                    const float2 h = unpack2<E>(hi[ks][j]);
                    lo[ks][j] = pack2<E>(x.x - h.x, x.y - h.y);
                } else {
                    hi[ks][j] = live[i] && col < p.hd ? *reinterpret_cast<const uint32_t *>(src[i] + col) : 0u;
                }
            }
        }
    }
};

template <typename T, typename E, int HDP>
__global__ void __launch_bounds__(kSqWarps * 32) k_attn_seq(const __grid_constant__ CUtensorMap mk,
                                                            const __grid_constant__ CUtensorMap mv,
                                                            const __grid_constant__ SeqAttnParams p) {
    using S = SqSmem<HDP>;
    constexpr bool kSplit = std::is_same<T, float>::value;
    constexpr int KS = HDP / 16, NO = HDP / 8;
    extern __shared__ uint8_t sq_raw[];
    S &sm = *reinterpret_cast<S *>((reinterpret_cast<uintptr_t>(sq_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const uint32_t item = blockIdx.x / p.splits, kvh = item % p.n_kv, ti = p.n_tiles - 1 - item / p.n_kv;
    pdl_wait();  // the batch, q, k and v may come from the kernel before
    pdl_trigger();
    SeqSpan sp;
    uint32_t tile;
    if (!seq_find_tile(p.b, p.group, kSqRows, ti, &sp, &tile)) return;  // the same for the whole cluster
    if (lane == 0) {
        for (int s = 0; s < kSqStages; s++) mbar_init(&sm.full[warp][s], 1);
        fence_mbar_init();
    }
    __syncwarp();
    const uint32_t row0 = tile * kSqRows, n_rows = min(sp.n_new * p.group - row0, (uint32_t)kSqRows);
    // attended positions [lo, hi] of this thread's two rows (none: hi = -1) and of the whole tile
    uint32_t row[2];
    bool live[2];
    int64_t lo[2], hi[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        live[i] = g + 8 * i < n_rows;
        row[i] = row0 + min(g + 8 * i, n_rows - 1);
        hi[i] = live[i] ? sp.pos(row[i] / p.group) : -1;
        lo[i] = p.window > 0 && hi[i] + 1 > (int64_t)p.window ? hi[i] + 1 - p.window : 0;
    }
    const int64_t p_first = sp.pos(row0 / p.group), k_hi = sp.pos((row0 + n_rows - 1) / p.group);
    const int64_t k_lo = p.window > 0 && p_first + 1 > (int64_t)p.window ? p_first + 1 - p.window : 0;
    const uint32_t c_lo = (uint32_t)(k_lo / kSqKeys), c_all = k_hi >= 0 ? (uint32_t)(k_hi / kSqKeys) + 1 : 0;
    const uint32_t n_chunks = c_all > c_lo ? c_all - c_lo : 0;
    // keys that every live row attends: chunks inside need no mask
    const int64_t all_lo = p.window > 0 && k_hi + 1 > (int64_t)p.window ? k_hi + 1 - p.window : 0, all_hi = p_first;

    // this warp's chunks: w0, w0 + stride, ... of the tile's n_chunks
    const uint32_t stride = p.splits * kSqWarps, w0 = rank * kSqWarps + warp;
    const uint32_t mine = n_chunks > w0 ? (n_chunks - w0 + stride - 1) / stride : 0;
    uint8_t *ring = sm.ring[warp];
    uint32_t rows_ahead = 0;  // lane l: first key row of chunk (32-chunk group) + l
    auto fetch_rows = [&](uint32_t i0) {
        const uint32_t i = i0 + lane;
        rows_ahead = i < mine ? seq_kv_row(p.b, sp, p.n_kv, kvh, (c_lo + w0 + i * stride) * kSqKeys) : 0;
    };
    auto issue = [&](uint32_t i) {  // whole warp; brings chunk i into stage i % kSqStages
        if ((i & 31) == 0) fetch_rows(i);
        const uint32_t r = __shfl_sync(0xffffffffu, rows_ahead, i & 31);
        if (lane == 0) {
            const uint32_t st = i % kSqStages;
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
    const uint32_t pre = min(mine, (uint32_t)kSqStages);
    for (uint32_t i = 0; i < pre; i++) issue(i);

    SqFrag<T, E, HDP> q;
    q.load(p, sp, kvh, row, live);
    const float sc[2] = {q.unscale[0] * kLog2e, q.unscale[1] * kLog2e};
    float o[NO][4];
#pragma unroll
    for (int n = 0; n < NO; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // m in units of log2

    bool ok = true;
    for (uint32_t i = 0; i < mine; i++) {
        const uint32_t st = i % kSqStages;
        ok = mbar_wait_bounded(&sm.full[warp][st], (i / kSqStages) & 1, p.b.err, ERR_TIMEOUT_FULL);
        if (!ok) {  // the result is void; the copies still in flight must land before the CTA ends
            for (uint32_t j = i + 1; j < min(mine, i + kSqStages); j++)
                mbar_wait_bounded(&sm.full[warp][j % kSqStages], (j / kSqStages) & 1, p.b.err, ERR_TIMEOUT_FULL);
            break;
        }
        const uint32_t kb = smem_u32(ring + st * 2 * S::kTile), vb = kb + S::kTile;
        const int64_t c0 = (int64_t)(c_lo + w0 + i * stride) * kSqKeys;
        float s[2][4] = {};
        const int mi = lane >> 3;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t r[4];
            sq_ldsm_x4(r, kb + sq_off(8 * (mi >> 1) + (lane & 7), 2 * ks + (mi & 1), kSqKeys));
            mma_16816<E>(s[0], q.hi[ks], r[0], r[1]);
            mma_16816<E>(s[1], q.hi[ks], r[2], r[3]);
            if constexpr (kSplit) {
                mma_16816<E>(s[0], q.lo[ks], r[0], r[1]);
                mma_16816<E>(s[1], q.lo[ks], r[2], r[3]);
            }
        }
        // s in units of log2, masked where the chunk is not attended by every row
        if (p.softcap > 0.0f) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[n][j] = p.softcap * kLog2e * tanhf(s[n][j] * q.unscale[j >> 1] / p.softcap);
        }
        const bool part = c0 < all_lo || c0 + kSqKeys - 1 > all_hi;
        float mx[2] = {-INFINITY, -INFINITY};
        if (part) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t kp = c0 + 8 * n + 2 * t4 + (j & 1);
                    if (kp > hi[j >> 1] || kp < lo[j >> 1]) s[n][j] = -INFINITY;
                }
        }
        const float cs[2] = {p.softcap > 0.0f ? 1.0f : sc[0], p.softcap > 0.0f ? 1.0f : sc[1]};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) mx[j >> 1] = fmaxf(mx[j >> 1], s[n][j]);
        bool grew = false;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 1));
            mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 2));
            mx[k] *= cs[k];  // cs > 0
            grew |= mx[k] > m[k];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float mn = fmaxf(m[k], mx[k]);
                const float a = mn == -INFINITY ? 1.0f : ex2(m[k] - mn);
                m[k] = mn;
                l[k] *= a;
#pragma unroll
                for (int n = 0; n < NO; n++) o[n][2 * k] *= a, o[n][2 * k + 1] *= a;
            }
        }
        float pr[2][4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float off = (m[k] == -INFINITY ? 0.0f : m[k]) - kPShift;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float e = ex2(fmaf(s[n][2 * k + j], cs[k], -off));
                    pr[n][2 * k + j] = e;
                    l[k] += e;
                }
        }
        uint32_t ah[4], al[4];
        const float pv[4][2] = {{pr[0][0], pr[0][1]}, {pr[0][2], pr[0][3]}, {pr[1][0], pr[1][1]}, {pr[1][2], pr[1][3]}};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            ah[j] = pack2<E>(pv[j][0], pv[j][1]);
            if constexpr (kSplit) {
                const float2 h = unpack2<E>(ah[j]);
                al[j] = pack2<E>(pv[j][0] - h.x, pv[j][1] - h.y);
            }
        }
#pragma unroll
        for (int nd = 0; nd < HDP / 16; nd++) {
            uint32_t r[4];
            sq_ldsm_x4_t(r, vb + sq_off(8 * (mi & 1) + (lane & 7), 2 * nd + (mi >> 1), kSqKeys));
            mma_16816<E>(o[2 * nd], ah, r[0], r[1]);
            mma_16816<E>(o[2 * nd + 1], ah, r[2], r[3]);
            if constexpr (kSplit) {
                mma_16816<E>(o[2 * nd], al, r[0], r[1]);
                mma_16816<E>(o[2 * nd + 1], al, r[2], r[3]);
            }
        }
        __syncwarp();  // every lane has read the stage
        if (i + kSqStages < mine) issue(i + kSqStages);
    }
    // ---- join: warps of the CTA, then CTAs of the cluster -----------------------------------------
#pragma unroll
    for (int k = 0; k < 2; k++) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 1);
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], 2);
        if (t4 == 0) sm.m[warp][g + 8 * k] = m[k], sm.l[warp][g + 8 * k] = l[k];
    }
    // this warp's ring is free (all its copies were waited for, or its wait ran out and the result is void)
    float *ow = reinterpret_cast<float *>(ring);
    if (ok) {
#pragma unroll
        for (int n = 0; n < NO; n++)
#pragma unroll
            for (int k = 0; k < 2; k++)
                *reinterpret_cast<float2 *>(ow + (g + 8 * k) * HDP + 8 * n + 2 * t4) = make_float2(o[n][2 * k], o[n][2 * k + 1]);
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
                if (a[w] != 0.0f) acc += a[w] * oc[w * kOw + r * HDP + d];
            oc[r * HDP + d] = acc;
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
            L = sm.cl[r];
            for (int i = 0; i < HDP / 32; i++) acc[i] = oc[r * HDP + lane + 32 * i];
        } else {
            const uint32_t am = smem_u32(&sm.cm[r]), al2 = smem_u32(&sm.cl[r]), ao = smem_u32(oc + r * HDP + lane);
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
        const uint32_t rr = row0 + r, t = rr / p.group, gq = rr % p.group;
        T *orow = reinterpret_cast<T *>(p.out) + (uint64_t)(sp.first + t) * p.ld_out + (uint64_t)(kvh * p.group + gq) * p.hd;
        bool fine = true;
#pragma unroll
        for (int i = 0; i < HDP / 32; i++) {
            const uint32_t d = lane + 32 * i;
            const float v = acc[i] / L;
            fine = fine && (isfinite(v) || d >= p.hd);
            if (d < p.hd) orow[d] = from_f32<T>(v);
        }
        if (!__all_sync(0xffffffffu, fine)) {
            __syncwarp();
            seq_attn_row<T, E>(p, sp, t, kvh, gq);
        }
    }
    if (p.splits > 1) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// ---- host ---------------------------------------------------------------------------------------
template <typename T, typename E, int HDP>
static int launch_few(rcu_ctx *ctx, const CUtensorMap &mk, const CUtensorMap &mv, SeqAttnParams p, uint64_t max_len) {
    const size_t smem = sizeof(SqSmem<HDP>) + 1024;
    // CTAs per tile: up to two for each SM in all, and at least 128 keys each
    const uint64_t items = (uint64_t)p.n_tiles * p.n_kv, span = p.window > 0 ? std::min<uint64_t>(max_len, p.window + 16) : max_len;
    const uint32_t most = HDP == 256 ? 8 : kSqMaxCluster;  // 197 KB of shared memory each: eight SMs of a GPC are sure to be there
    uint32_t cs = 1;
    while (cs < most && items * cs * 2 <= 2ull * ctx->num_sms && span >= (uint64_t)cs * 2 * 128) cs *= 2;
    p.splits = cs;
    if (items * cs > 0x7fffffffull) return set_err(ctx, RCU_ERR_INVALID, "attention: too many work tiles");
    return launch_cluster_k(ctx, k_attn_seq<T, E, HDP>, (uint32_t)(items * cs), kSqWarps * 32, smem, cs, mk, mv, p);
}

template <typename T, typename E>
static int launch_few_hd(rcu_ctx *ctx, SeqAttnParams p, const SeqKvDesc &kv, uint64_t max_len) {
    CUtensorMap mk, mv;
    if (int st = seq_kv_maps(ctx, p, kv, kSqKeys, &mk, &mv)) return st;
    p.n_tiles = (uint32_t)seq_tiles_bound(p.b.n_tok, p.b.n_seq, p.group, kSqRows);
    if (p.hd <= 64) return launch_few<T, E, 64>(ctx, mk, mv, p, max_len);
    if (p.hd <= 128) return launch_few<T, E, 128>(ctx, mk, mv, p, max_len);
    return launch_few<T, E, 256>(ctx, mk, mv, p, max_len);
}

static int launch_attention_few(rcu_ctx *ctx, const SeqAttnParams &p, int q_type, const SeqKvDesc &kv, uint64_t max_len) {
    if (q_type == T_F32) return launch_few_hd<float, __half>(ctx, p, kv, max_len);
    if (q_type == T_F16) return launch_few_hd<__half, __half>(ctx, p, kv, max_len);
    return launch_few_hd<__nv_bfloat16, __nv_bfloat16>(ctx, p, kv, max_len);
}

int launch_seq_attention(rcu_ctx *ctx, const SeqAttnParams &p, int q_type, const SeqKvDesc &kv, uint64_t max_len,
                         uint64_t max_new) {
    // The most query rows that a sequence may have in one KV head. As many new rows as sequences are
    // taken for single tokens; what is there in fact decides only how fast the launch is. One kernel
    // takes the whole batch: in a mixed one the single tokens ride along with the chunks (two chunks
    // of 333 tokens beside 14 single ones: 64 us for the chunks alone and 62 us for the single
    // tokens in a launch of their own).
    const uint64_t most = std::min<uint64_t>(max_new ? max_new : p.b.n_tok, p.b.n_tok) * p.group;
    if (!attention_tile_ok(p.hd) || most < kTileMinRows || (!max_new && p.b.n_tok <= p.b.n_seq))
        return launch_attention_few(ctx, p, q_type, kv, max_len);
    return launch_attention_tile(ctx, p, q_type, kv, max_len);
}

}  // namespace rcu
