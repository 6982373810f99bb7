// rcu_logprobs.cu -- log probabilities of given tokens, entropy and the most likely alternatives of
// rows of logits, in one pass over the logits.
//
// For a row x of `vocab` logits, m = max x, z = sum exp(x - m):
//   log p(i) = (x_i - m) - ln z          entropy = ln z - (sum exp(x - m) (x - m)) / z
// and the top_k largest, ties to the lowest index (a NaN counts as the largest value, -0 as 0).
//
// Reading the logits is the bound. A cluster of `splits` CTAs shares a row; each thread keeps a
// running (m, z, sum) over the values it reads, 16 a step. For many rows the steps' values come
// through a ring of bulk copies (from registers one step ahead, half as many bytes were in flight and
// 512 rows of 151,936 took 83 us without alternatives); a few rows take one step of larger
// CTAs. The alternatives need no second pass: a value is a 64-bit key (ordered value, ~index),
// and the k-th largest of the maxima of 128 or 256 groups of values is a bound below which nothing
// can be among the k largest of the row. A value reaches the candidate list in shared memory only
// from the bound on, which is taken from the first step's groups and again from the list now and then
// (less often as the row goes on); no other step has a barrier. Should the list run over all the same (logits that rise
// along the row, or many equal ones at the bound), the CTA reads its part again with a check after
// every step. The candidates' ranks, by counting larger keys, are the order of a CTA's answer; in a
// cluster every CTA ranks its own keys among the others' ordered lists and writes them where they go.
#include <cstdint>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"

namespace rcu {

constexpr int kLpPer = 16;                       // values a thread reads per step
constexpr int kLpMaxTop = 128;
constexpr int kLpMaxSplits = 16;
constexpr int kLpCap = 2048;                     // candidates
constexpr int kLpGroups = 256;                   // groups whose maxima give a bound, at most
// A checked step adds at most kLpCap / 2 candidates to at most as many that are kept.
constexpr int kLpKeep = kLpCap / 2;

constexpr int kLpStages = 2;
// exp(d) is 0 in f32 from here on down. Farther distances (-inf; masks of the type's lowest value,
// whose products with d leave f32's range) are taken for this one, so that 0 * d stays 0.
constexpr float kLpFar = -1000.0f;

struct LpSmem {
    uint64_t full[kLpStages], empty[kLpStages];
    uint64_t cand[kLpCap];
    uint64_t top[kLpMaxTop];      // this CTA's largest keys in order
    uint32_t gmax[kLpGroups];
    float sum[3][32];             // (m, z, w) of the warps; then [0..2][0] of the CTA
    float row[3];                 // of the row
    uint32_t n, bound;
};

// Orders as the value does; NaN above everything.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    if (x != x) return 0xffffffffu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    if (o == 0xffffffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t idx) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~idx; }

// State of a softmax sum: maximum, sum of exp(x - m) and of exp(x - m) (x - m).
struct LpSum {
    float m = -INFINITY, z = 0.0f, w = 0.0f;
    __device__ __forceinline__ void raise(float mn) {  // mn >= m
        if (mn == m || z == 0.0f) {
            m = mn;
            return;
        }
        const float d = m - mn, a = ex2(d * kLog2e);
        w = a * fmaf(fmaxf(d, kLpFar), z, w);  // where a is 0, d z may be past the largest number; a NaN stays in z
        z *= a;
        m = mn;
    }
    // 16 values, none above m; far: one of them is kLpFar or more below m and adds nothing
    __device__ __forceinline__ void add16(const float (&f)[16], bool far) {
        const float2 nm = make_float2(-m, -m), c = make_float2(kLog2e, kLog2e);
        float2 z2[2] = {}, w2[2] = {};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float2 d = add2(make_float2(f[2 * i], f[2 * i + 1]), nm);
            const float2 y = mul2(d, c), e = make_float2(ex2(y.x), ex2(y.y));
            if (far) d.x = fmaxf(d.x, kLpFar), d.y = fmaxf(d.y, kLpFar);  // a NaN stays in e
            z2[i & 1] = add2(z2[i & 1], e);
            w2[i & 1] = fma2(e, d, w2[i & 1]);
        }
        z += (z2[0].x + z2[0].y) + (z2[1].x + z2[1].y);
        w += (w2[0].x + w2[0].y) + (w2[1].x + w2[1].y);
    }
    __device__ __forceinline__ void join(float m2, float z2, float w2) {
        const float mn = fmaxf(m, m2);
        LpSum o{m2, z2, w2};
        raise(mn);
        o.raise(mn);
        z += o.z;
        w += o.w;
    }
};

// The order (lp_order) of the k-th largest of n group maxima: all values from it on are candidates.
// The thread that holds group id < n's maximum passes it (0: the group has no value). 0 when fewer
// than k groups have one. The whole CTA; threads 0 .. n - 1 count.
__device__ __forceinline__ uint32_t lp_bound(LpSmem &sm, uint32_t id, uint32_t mine, uint32_t n, uint32_t k) {
    if (id < n) sm.gmax[id] = mine;
    if (threadIdx.x == 0) sm.bound = 0;
    __syncthreads();
    if (threadIdx.x < n) {
        const uint32_t own = sm.gmax[threadIdx.x];
        uint32_t above = 0, same = 0;
        const uint4 *t = reinterpret_cast<const uint4 *>(sm.gmax);
#pragma unroll 8
        for (uint32_t i = 0; i < n / 4; i++) {
            const uint4 x = t[i];
            above += (x.x > own) + (x.y > own) + (x.z > own) + (x.w > own);
            same += (x.x == own) + (x.y == own) + (x.z == own) + (x.w == own);
        }
        if (own != 0 && above < k && above + same >= k) sm.bound = own;  // equal ones write the same
    }
    __syncthreads();
    return sm.bound;
}
// Cuts a short candidate list (n <= the CTA's threads) down to its k largest; returns the last one's
// order. The whole CTA, of which a thread for each candidate counts.
__device__ __forceinline__ uint32_t lp_tighten(LpSmem &sm, uint32_t n, uint32_t k) {
    uint64_t key = 0;
    uint32_t above = 0;
    if (threadIdx.x < n) {
        key = sm.cand[threadIdx.x];
#pragma unroll 4
        for (uint32_t j = 0; j < n; j++) above += sm.cand[j] > key;
        if (above == k - 1) sm.bound = (uint32_t)(key >> 32);
    }
    __syncthreads();
    if (threadIdx.x < n && above < k) sm.cand[above] = key;
    if (threadIdx.x == 0) sm.n = k;
    __syncthreads();
    return sm.bound;
}
// Cuts the candidate list down to the k largest keys or a few more: the bound of 256 stretches of the
// list by whole keys, so that equal values do not keep it long (at most k * ceil(n / 256) <= n / 2 +
// 128 stay). Returns the order below which nothing is a candidate any more. The whole CTA.
__device__ __noinline__ uint32_t lp_compact(LpSmem &sm, uint32_t n, uint32_t k) {
    constexpr int kMost = kLpCap / kLpGroups;
    __shared__ uint64_t kmax[kLpGroups], kbound;
    uint64_t own[kMost], mx = 0;
#pragma unroll
    for (int i = 0; i < kMost; i++) {
        const uint32_t j = threadIdx.x + i * kLpGroups;
        own[i] = threadIdx.x < kLpGroups && j < n ? sm.cand[j] : 0;
        mx = own[i] > mx ? own[i] : mx;
    }
    if (threadIdx.x < kLpGroups) kmax[threadIdx.x] = mx;
    if (threadIdx.x == 0) sm.n = 0, kbound = 0;
    __syncthreads();
    if (threadIdx.x < kLpGroups && mx != 0) {
        uint32_t above = 0;
#pragma unroll 8
        for (int i = 0; i < kLpGroups; i++) above += kmax[i] > mx;
        if (above == k - 1) kbound = mx;  // keys differ: one thread at most
    }
    __syncthreads();
    const uint64_t bound = kbound;
#pragma unroll
    for (int i = 0; i < kMost; i++)
        if (own[i] != 0 && own[i] >= bound) sm.cand[atomicAdd(&sm.n, 1u)] = own[i];
    __syncthreads();
    return (uint32_t)(bound >> 32);
}

// A row's part as a CTA reads it: 16-byte pieces v0 .. v1 - 1, counted from the boundary at or below
// the row's start; a row may start and end inside one.
template <typename T>
struct LpPart {
    static constexpr int VE = 16 / sizeof(T);
    const T *x;
    uint32_t off, vocab, v0, v1;
    __device__ __forceinline__ uint32_t index(uint32_t v, int i) const { return v * VE + i - off; }  // of value i of piece v
    __device__ __forceinline__ bool inside(uint32_t v) const { return v < v1 && v * VE >= off && v * VE + VE - off <= vocab; }
    __device__ __forceinline__ bool valid(uint32_t v, int i) const { return v < v1 && v * VE + i >= off && v * VE + i - off < vocab; }
    // piece v (outside values: -inf)
    __device__ __forceinline__ uint4 load(uint32_t v) const {
        if (inside(v)) return __ldcs(reinterpret_cast<const uint4 *>(x - off) + v);
        alignas(16) T t[VE];
#pragma unroll
        for (int i = 0; i < VE; i++) t[i] = valid(v, i) ? x[index(v, i)] : from_f32<T>(-INFINITY);
        return *reinterpret_cast<const uint4 *>(t);
    }
    static __device__ __forceinline__ void values(const uint4 &u, float *f) {
        if constexpr (sizeof(T) == 4) {
            f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
        } else {
            const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
            f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
        }
    }
};

// The candidates once more, for a list that ran over: one piece a thread and step (at most kLpKeep
// values), the list cut down after each.
template <typename T, int THREADS>
__device__ __noinline__ void lp_checked(LpSmem &sm, const LpPart<T> &part, uint32_t k) {
    constexpr int VE = LpPart<T>::VE, kTake = kLpKeep / VE < THREADS ? kLpKeep / VE : THREADS;
    uint32_t bound = 0;
    __syncthreads();
    if (threadIdx.x == 0) sm.n = 0;
    __syncthreads();
    for (uint32_t s = part.v0; s < part.v1; s += kTake) {
        const uint32_t v = s + threadIdx.x;
        if (threadIdx.x < kTake && v < part.v1) {
            float f[VE];
            LpPart<T>::values(part.load(v), f);
#pragma unroll
            for (int i = 0; i < VE; i++)
                if (part.valid(v, i)) {
                    const uint64_t key = lp_key(f[i], part.index(v, i));
                    if ((uint32_t)(key >> 32) >= bound) sm.cand[atomicAdd(&sm.n, 1u)] = key;
                }
        }
        __syncthreads();
        uint32_t n = sm.n;
        __syncthreads();
        while (n > (uint32_t)kLpKeep) {
            bound = lp_compact(sm, n, k);
            n = sm.n;
            __syncthreads();
        }
    }
}

constexpr uint32_t kRingAt = (sizeof(LpSmem) + 127) / 128 * 128;
template <int THREADS>
constexpr size_t lp_smem() {
    return THREADS == 256 ? kRingAt + kLpStages * THREADS * kLpPer * 4 : sizeof(LpSmem);
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : 1) k_logprobs(const LogprobParams p, uint32_t splits) {
    using Part = LpPart<T>;
    constexpr int VE = Part::VE, NV = kLpPer / VE;  // values of a 16-byte load, loads a step
    constexpr uint32_t kStep = THREADS * NV;
    extern __shared__ __align__(128) uint8_t lp_raw[];
    LpSmem &sm = *reinterpret_cast<LpSmem *>(lp_raw);
    const uint32_t rank = splits > 1 ? cluster_ctarank() : 0, r = blockIdx.x / splits, k = p.top_k;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        sm.n = 0;
        for (int i = 0; i < kLpStages; i++) mbar_init(&sm.full[i], 1), mbar_init(&sm.empty[i], THREADS / 32);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    Part part;
    part.x = reinterpret_cast<const T *>(p.logits) + (uint64_t)r * p.ld;
    part.off = (uint32_t)(((uintptr_t)part.x & 15) / sizeof(T));
    part.vocab = p.vocab;
    const uint32_t n_vec = (part.off + p.vocab + VE - 1) / VE, per = (n_vec + splits - 1) / splits;
    part.v0 = min(rank * per, n_vec), part.v1 = min(part.v0 + per, n_vec);
    const T *x = part.x;

    LpSum a;
    uint32_t bound = 0;  // order from which a value is a candidate
    float boundf = -INFINITY;
    // steps so far; the list is looked at after 1, 2, 3, 4, 6, 8, 12, 16, 24 and then every 16 steps
    uint32_t done = 0;
    constexpr uint32_t looks = 1u << 1 | 1u << 2 | 1u << 3 | 1u << 4 | 1u << 6 | 1u << 8 | 1u << 12 | 1u << 24;
    // pieces [full0, full1) lie inside the row and this CTA's part
    const uint32_t full0 = part.v0 + (part.v0 == 0 && part.off > 0);
    const uint32_t full1 = part.v1 - (part.v1 == n_vec && (n_vec * VE - part.off) > p.vocab && part.v1 > full0);
    // the step's pieces that lie inside, by one bulk copy into its stage of the ring
    constexpr bool kRing = THREADS == 256;
    constexpr uint32_t kStageB = kStep * 16;
    uint8_t *ring = lp_raw + kRingAt;
    auto inner = [&](uint32_t s, uint32_t *lo) {  // and how many there are
        *lo = max(s, full0);
        const uint32_t hi = min(s + kStep, full1);
        return hi > *lo ? hi - *lo : 0u;
    };
    auto issue = [&](uint32_t s, uint32_t st) {
        uint32_t lo;
        const uint32_t c = inner(s, &lo);
        if (s >= part.v1 || c == 0) return;
        mbar_arrive_expect_tx(&sm.full[st], c * 16);
        bulk_g2s(ring + st * kStageB + (lo - s) * 16, reinterpret_cast<const uint4 *>(x - part.off) + lo, c * 16, &sm.full[st],
                 policy_evict_first());
    };
    if (kRing && threadIdx.x == 0)
        for (int st = 0; st < kLpStages; st++) issue(part.v0 + st * kStep, st);
    uint32_t st = 0, parity = 0;
    for (uint32_t s = part.v0; s < part.v1; s += kStep) {
        float f[kLpPer];
        if constexpr (kRing) {
            uint32_t lo;
            const uint32_t c = inner(s, &lo);
            if (c > 0) mbar_wait_spin(&sm.full[st], parity, p.err, ERR_TIMEOUT_FULL);
            const uint4 *there = reinterpret_cast<const uint4 *>(ring + st * kStageB) + threadIdx.x;
            if (c == kStep) {
#pragma unroll
                for (int j = 0; j < NV; j++) Part::values(there[j * THREADS], f + j * VE);
            } else {
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    const uint32_t v = s + j * THREADS + threadIdx.x;
                    Part::values(v - lo < c ? there[j * THREADS] : part.load(v), f + j * VE);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
            if (threadIdx.x == 0 && s + kLpStages * kStep < part.v1) {
                mbar_wait_spin(&sm.empty[st], parity, p.err, ERR_TIMEOUT_EMPTY);
                issue(s + kLpStages * kStep, st);
            }
            if (++st == kLpStages) st = 0, parity ^= 1;
        } else {
#pragma unroll
            for (int j = 0; j < NV; j++) Part::values(part.load(s + j * THREADS + threadIdx.x), f + j * VE);
        }
        const bool full = s >= full0 && s + kStep <= full1;
        float pm[NV];  // the pieces' maxima, NaN if a value is
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const float *g = f + j * VE;
            pm[j] = max3_nan(max3_nan(g[0], g[1], g[2]), g[3], -INFINITY);
            if constexpr (VE == 8) pm[j] = max3_nan(max3_nan(g[4], g[5], g[6]), g[7], pm[j]);
        }
        float top = max3_nan(pm[0], pm[1], -INFINITY);
        if constexpr (NV == 4) top = max3_nan(pm[2], pm[3], top);
        float l[5];
#pragma unroll
        for (int i = 0; i < 5; i++) l[i] = fminf(fminf(f[3 * i], f[3 * i + 1]), f[3 * i + 2]);
        const float low = fminf(fminf(fminf(l[0], l[1]), fminf(l[2], l[3])), fminf(l[4], f[15]));
        if (top > a.m) a.raise(top);
        if (top != top) a.z = top;
        if (a.m != -INFINITY) {
            if (low - a.m < kLpFar) a.add16(f, true);
            else a.add16(f, false);
        }
        if (k == 0) continue;
        if (done == 0) {
            // groups of neighbouring threads: all values of the step stand for one of them
            const uint32_t groups = k <= 32 ? kLpGroups / 2 : kLpGroups, each = THREADS / groups;
            uint32_t mx = lp_order(top);
            if (!full && top == -INFINITY) {  // nothing of the row among a thread's values, or -inf
                bool any = false;
#pragma unroll
                for (int i = 0; i < kLpPer; i++) any |= part.valid(s + (i / VE) * THREADS + threadIdx.x, i % VE);
                if (!any) mx = 0;
            }
            for (uint32_t d = 1; d < each; d <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            bound = lp_bound(sm, threadIdx.x % each == 0 ? threadIdx.x / each : groups, mx, groups, k);
        } else if (looks >> min(done, 31u) & 1 || (done & 15) == 0) {
            __syncthreads();
            const uint32_t n = sm.n;
            __syncthreads();
            if (n >= k + k / 2 + 8 && n <= (uint32_t)kLpCap)
                bound = max(bound, n <= (uint32_t)THREADS ? lp_tighten(sm, n, k) : lp_compact(sm, n, k));
        }
        done++;
        boundf = bound ? lp_value(bound) : -INFINITY;
        if (!(top < boundf)) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (pm[j] < boundf) continue;
                const uint32_t v = s + j * THREADS + threadIdx.x;
#pragma unroll
                for (int i = 0; i < VE; i++)
                    if (!(f[j * VE + i] < boundf) && (full || part.valid(v, i))) {
                        const uint64_t key = lp_key(f[j * VE + i], part.index(v, i));
                        if ((uint32_t)(key >> 32) >= bound) {
                            const uint32_t at = atomicAdd(&sm.n, 1u);
                            if (at < (uint32_t)kLpCap) sm.cand[at] = key;
                        }
                    }
            }
        }
    }
    // ---- join the threads' sums ----
    auto join_lanes = [&](LpSum &t, int lanes) {
#pragma unroll
        for (int d = lanes / 2; d > 0; d >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, t.m, d), z2 = __shfl_xor_sync(0xffffffffu, t.z, d),
                        w2 = __shfl_xor_sync(0xffffffffu, t.w, d);
            t.join(m2, z2, w2);
        }
    };
    join_lanes(a, 32);
    if (lane == 0) sm.sum[0][warp] = a.m, sm.sum[1][warp] = a.z, sm.sum[2][warp] = a.w;
    for (uint32_t i = threadIdx.x; i < k; i += THREADS) sm.top[i] = 0;
    __syncthreads();
    if (k > 0 && sm.n > (uint32_t)kLpCap) lp_checked<T, THREADS>(sm, part, k);
    if (warp == 0) {
        LpSum t;
        if (lane < THREADS / 32) t.m = sm.sum[0][lane], t.z = sm.sum[1][lane], t.w = sm.sum[2][lane];
        join_lanes(t, THREADS / 32);
        __syncwarp();
        if (lane == 0) {
            sm.sum[0][0] = t.m, sm.sum[1][0] = t.z, sm.sum[2][0] = t.w;
            if (splits == 1) sm.row[0] = t.m, sm.row[1] = t.z, sm.row[2] = t.w;
        }
    }
    // ---- this CTA's largest keys, in order ----
    const uint32_t n = sm.n;
    for (uint32_t i = threadIdx.x; i < n && k > 0; i += THREADS) {
        const uint64_t key = sm.cand[i];
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; j++) above += sm.cand[j] > key;
        if (above < k) sm.top[above] = key;
    }
    if (splits > 1) {
        cluster_sync_all();
        if (warp == 0) {  // the row's sums, in every CTA
            LpSum t;
            if (lane < splits) {
                t.m = ld_cluster_f32(cluster_addr(smem_u32(&sm.sum[0][0]), lane));
                t.z = ld_cluster_f32(cluster_addr(smem_u32(&sm.sum[1][0]), lane));
                t.w = ld_cluster_f32(cluster_addr(smem_u32(&sm.sum[2][0]), lane));
            }
            join_lanes(t, kLpMaxSplits);
            if (lane == 0) sm.row[0] = t.m, sm.row[1] = t.z, sm.row[2] = t.w;
        }
        for (uint32_t i = threadIdx.x; i < splits * k; i += THREADS) {  // the others' lists
            const uint32_t src = cluster_addr(smem_u32(&sm.top[i % k]), i / k);
            uint64_t key;
            asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(src) : "memory");
            sm.cand[i] = key;
        }
        cluster_sync_all();  // everything has been read; and this CTA's copies are written
    } else {
        __syncthreads();
    }
    const float m = sm.row[0], z = sm.row[1], lz = logf(z);
    if (threadIdx.x == 0 && rank == 0) {
        if (p.entropy) p.entropy[r] = lz - sm.row[2] / z;
        if (p.targets) {
            const int32_t t = p.targets[r];
            float lp = 0.0f;
            if (t >= 0 && (uint32_t)t < p.vocab) {
                lp = to_f32(x[t]) - m - lz;
            } else if (t != -1) {
                atomicOr(p.err, (uint32_t)ERR_BAD_ARG);
                lp = __uint_as_float(0x7fffffffu);
            }
            p.logprob[r] = lp;
        }
    }
    auto put = [&](uint32_t at, uint64_t key) {
        p.top_ids[(uint64_t)r * k + at] = (int32_t)~(uint32_t)key;
        p.top_logprobs[(uint64_t)r * k + at] = lp_value((uint32_t)(key >> 32)) - m - lz;
    };
    if (splits == 1) {
        for (uint32_t i = threadIdx.x; i < k; i += THREADS) put(i, sm.top[i]);
    } else {
        // `splits` lanes a key, each with one list: keys above it in the list, by halving
        const uint32_t keys = THREADS / splits, c = threadIdx.x % splits;
        for (uint32_t i0 = 0; i0 < k; i0 += keys) {
            const uint32_t i = i0 + threadIdx.x / splits;
            const uint64_t key = i < k ? sm.top[i] : 0;
            const uint64_t *list = sm.cand + c * k;
            uint32_t a0 = 0, a1 = k;  // list[.. a0) are above, list[a1 ..] are not
            while (a0 < a1) {
                const uint32_t mid = (a0 + a1) / 2;
                if (list[mid] > key) a0 = mid + 1;
                else a1 = mid;
            }
            uint32_t above = a0;
            for (uint32_t d = splits / 2; d > 0; d >>= 1) above += __shfl_xor_sync(0xffffffffu, above, d);
            if (c == 0 && key != 0 && above < k) put(above, key);
        }
    }
}

// CTAs a row: as many as make the waves of `slots` CTAs end soonest, a CTA costing its share of the
// row and as much as 8192 values beside it.
template <typename T, int THREADS>
static int launch_lp_threads(rcu_ctx *ctx, const LogprobParams &p, uint32_t per_sm) {
    const uint64_t slots = (uint64_t)per_sm * ctx->num_sms;
    uint32_t cs = 1;
    uint64_t best = ~0ull;
    for (uint32_t c = 1; c <= kLpMaxSplits && (c == 1 || p.vocab >= (uint64_t)c * 2048); c *= 2) {
        const uint64_t cost = ((uint64_t)p.rows * c + slots - 1) / slots * (p.vocab / c + 8192);
        if (cost < best) best = cost, cs = c;
    }
    return launch_cluster_k<k_logprobs<T, THREADS>>(ctx, p.rows * cs, THREADS, lp_smem<THREADS>(), cs, p, cs);
}
template <typename T>
static int launch_lp(rcu_ctx *ctx, const LogprobParams &p) {
    return p.rows <= 4 ? launch_lp_threads<T, 1024>(ctx, p, 1) : launch_lp_threads<T, 256>(ctx, p, 4);
}

int launch_logprobs(rcu_ctx *ctx, const LogprobParams &p, int type) {
    if (type == T_F32) return launch_lp<float>(ctx, p);
    if (type == T_F16) return launch_lp<__half>(ctx, p);
    return launch_lp<__nv_bfloat16>(ctx, p);
}

}  // namespace rcu

using namespace rcu;

extern "C" {

int32_t rcu_logprobs(rcu_ctx *ctx, const void *logits_dev, uint32_t type, uint64_t n_rows, uint64_t n_vocab, uint64_t ld,
                     const int32_t *targets_dev, float *logprob_dev, float *entropy_dev, uint64_t top_k,
                     int32_t *top_ids_dev, float *top_logprobs_dev) {
    RCU_GUARD_BEGIN
    if (!logits_dev) return set_err(ctx, RCU_ERR_INVALID, "null argument");
    if (n_rows == 0) return set_err(ctx, RCU_ERR_RUNTIME, "empty batch");
    if (type != T_F32 && type != T_F16 && type != T_BF16)
        return set_err(ctx, RCU_ERR_UNSUPPORTED, "logprobs: logits are f32, f16 or bf16");
    if (!targets_dev != !logprob_dev) return set_err(ctx, RCU_ERR_INVALID, "logprobs: pass targets and logprob, or neither");
    if (top_k && (!top_ids_dev || !top_logprobs_dev)) return set_err(ctx, RCU_ERR_INVALID, "logprobs: top_k without its outputs");
    if (n_vocab == 0 || n_vocab > 0x7ffffff0ull || n_rows > (1ull << 26))
        return set_err(ctx, RCU_ERR_INVALID, "logprobs: vocabulary or batch out of range");
    if (ld < n_vocab) return set_err(ctx, RCU_ERR_INVALID, "ld smaller than n_vocab");
    if (top_k > kLpMaxTop || top_k > n_vocab)
        return set_err(ctx, RCU_ERR_INVALID, "logprobs: at most " + std::to_string(kLpMaxTop) + " alternatives, and no more than the vocabulary");
    if ((uintptr_t)logits_dev % (type == T_F32 ? 4 : 2)) return set_err(ctx, RCU_ERR_INVALID, "logprobs: misaligned logits");
    if (!ctx) return RCU_ERR_INVALID;
    DeviceGuard guard(ctx);
    const LogprobParams p{logits_dev, targets_dev, logprob_dev, entropy_dev, top_logprobs_dev, top_ids_dev, ld,
                          (uint32_t)n_rows, (uint32_t)n_vocab, (uint32_t)top_k, ctx->dev_err};
    return launch_logprobs(ctx, p, (int)type);
    RCU_GUARD_END(ctx)
}

}  // extern "C"
