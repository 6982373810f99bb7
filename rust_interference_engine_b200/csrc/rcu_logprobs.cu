// rcu_logprobs.cu -- log probabilities of given tokens, entropy and the most likely alternatives of
// rows of logits, in one pass over the logits.
//
// For a row x of `vocab` logits, m = max x, z = sum exp(x - m):
//   log p(i) = (x_i - m) - ln z          entropy = ln z - (sum exp(x - m) (x - m)) / z
// and the top_k largest, ties to the lowest index (a NaN counts as the largest value, -0 as 0).
//
// Reading the logits is the bound. A cluster of `splits` CTAs shares a row; each thread keeps a
// running (m, z, sum) over the values it reads, 16 a step, the next step's loads on their way
// meanwhile. The alternatives need no second pass: a value is a 64-bit key (ordered value, ~index),
// and the k-th largest of some threads' own maxima is a bound below which nothing can be among the k
// largest of the row. A value reaches the candidate list in shared memory only above the bound, which
// is taken from the first step's maxima and again from the list after 2, 4, 8, ... steps; no other
// step has a barrier. Should the list run over all the same (logits that rise along the row), the
// CTA reads its part again with a check after every step. The candidates' ranks, by counting larger
// keys, are the order of the answer.
#include <cstdint>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"

namespace rcu {

constexpr int kLpPer = 16;                       // values a thread reads per step
constexpr int kLpMaxTop = 128;
constexpr int kLpMaxSplits = 16;
constexpr int kLpCap = 2048;                     // candidates
constexpr int kLpBound = 256;                    // threads whose maxima give a bound
// A checked step adds at most kLpCap / 2 candidates to at most as many that are kept.
constexpr int kLpKeep = kLpCap / 2;

struct LpSmem {
    uint64_t cand[kLpCap];
    uint64_t tmax[kLpBound];
    uint64_t top[kLpMaxTop];      // this CTA's largest keys in order
    float rm[32], rz[32], rw[32];
    float cm, cz, cw;             // of the CTA
    uint32_t n;
    uint64_t bound;
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
        w = a * fmaf(d, z, w);
        z *= a;
        m = mn;
    }
    __device__ __forceinline__ void add(float x) {  // after raise(>= x)
        const float d = x - m;
        const float e = ex2(d * kLog2e);
        z += e;
        w = fmaf(e, fmaxf(d, -1000.0f), w);  // -inf adds nothing; NaN stays in e
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

// k-th largest of the keys `mine` of threads 0 .. kLpBound - 1 (0: no key): a lower bound of the
// k-th largest of all keys that these threads' own maxima stand for; 0 when fewer than k have one.
__device__ __forceinline__ uint64_t lp_bound(LpSmem &sm, uint64_t mine, uint32_t k) {
    if (threadIdx.x < kLpBound) sm.tmax[threadIdx.x] = mine;
    if (threadIdx.x == 0) sm.bound = 0;
    __syncthreads();
    if (threadIdx.x < kLpBound && mine != 0) {
        uint32_t above = 0;
        const ulonglong2 *t = reinterpret_cast<const ulonglong2 *>(sm.tmax);
#pragma unroll 8
        for (int i = 0; i < kLpBound / 2; i++) {
            const ulonglong2 x = t[i];
            above += (x.x > mine) + (x.y > mine);
        }
        if (above == k - 1) sm.bound = mine;  // keys differ: one thread at most
    }
    __syncthreads();
    return sm.bound;
}
// Raises the bound from the candidate list itself and drops what lies below it: at most
// k * ceil(n / kLpBound) <= n / 2 + 128 candidates stay. The whole CTA.
__device__ __noinline__ uint64_t lp_compact(LpSmem &sm, uint32_t n, uint32_t k) {
    constexpr int kMost = kLpCap / kLpBound;
    uint64_t own[kMost], mx = 0;
#pragma unroll
    for (int i = 0; i < kMost; i++) {
        const uint32_t j = threadIdx.x + i * kLpBound;
        own[i] = threadIdx.x < kLpBound && j < n ? sm.cand[j] : 0;
        mx = own[i] > mx ? own[i] : mx;
    }
    const uint64_t bound = lp_bound(sm, mx, k);
    if (threadIdx.x == 0) sm.n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMost; i++)
        if (own[i] != 0 && own[i] >= bound) sm.cand[atomicAdd(&sm.n, 1u)] = own[i];
    __syncthreads();
    return bound;
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
    uint64_t bound = 0;
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
                    if (key >= bound) sm.cand[atomicAdd(&sm.n, 1u)] = key;
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

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_logprobs(const LogprobParams p, uint32_t splits) {
    using Part = LpPart<T>;
    constexpr int VE = Part::VE, NV = kLpPer / VE;  // values of a 16-byte load, loads a step
    constexpr uint32_t kStep = THREADS * NV;
    extern __shared__ __align__(16) uint8_t lp_raw[];
    LpSmem &sm = *reinterpret_cast<LpSmem *>(lp_raw);
    const uint32_t rank = splits > 1 ? cluster_ctarank() : 0, r = blockIdx.x / splits, k = p.top_k;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) sm.n = 0;
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
    uint64_t bound = 0;
    float boundf = -INFINITY;
    uint32_t done = 0;  // steps
    uint4 next[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) next[j] = part.load(part.v0 + j * THREADS + threadIdx.x);
    for (uint32_t s = part.v0; s < part.v1; s += kStep) {
        float f[kLpPer];
#pragma unroll
        for (int j = 0; j < NV; j++) Part::values(next[j], f + j * VE);
        if (s + kStep < part.v1) {
#pragma unroll
            for (int j = 0; j < NV; j++) next[j] = part.load(s + kStep + j * THREADS + threadIdx.x);
        }
        float c[4] = {f[0], f[1], f[2], f[3]};
#pragma unroll
        for (int i = 4; i < kLpPer; i++) c[i & 3] = fmaxf(c[i & 3], f[i]);
        const float top = fmaxf(fmaxf(c[0], c[1]), fmaxf(c[2], c[3]));
        if (top > a.m) a.raise(top);
        if (a.m != -INFINITY) {
            LpSum b{a.m};  // two chains
#pragma unroll
            for (int i = 0; i < kLpPer; i += 2) a.add(f[i]), b.add(f[i + 1]);
            a.z += b.z, a.w += b.w;
        } else {  // nothing above -inf so far: only a NaN counts
#pragma unroll
            for (int i = 0; i < kLpPer; i++)
                if (f[i] != f[i]) a.z = f[i];
        }
        if (k == 0) continue;
        auto piece = [&](int i) { return s + (i / VE) * THREADS + threadIdx.x; };
        if (done == 0) {
            uint64_t mx = 0;
#pragma unroll
            for (int i = 0; i < kLpPer; i++) {
                const uint64_t key = part.valid(piece(i), i % VE) ? lp_key(f[i], part.index(piece(i), i % VE)) : 0;
                mx = key > mx ? key : mx;
            }
            bound = lp_bound(sm, mx, k);
        } else if ((done & (done - 1)) == 0 && done > 1) {  // 2, 4, 8, ... steps are in the list
            __syncthreads();
            const uint32_t n = sm.n;
            __syncthreads();
            if (n > 2 * k && n <= (uint32_t)kLpCap) bound = lp_compact(sm, n, k);
        }
        done++;
        boundf = bound ? lp_value((uint32_t)(bound >> 32)) : -INFINITY;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kLpPer; i++) any |= !(f[i] < boundf);
        if (any) {
#pragma unroll
            for (int i = 0; i < kLpPer; i++)
                if (!(f[i] < boundf) && part.valid(piece(i), i % VE)) {
                    const uint64_t key = lp_key(f[i], part.index(piece(i), i % VE));
                    if (key >= bound) {
                        const uint32_t at = atomicAdd(&sm.n, 1u);
                        if (at < (uint32_t)kLpCap) sm.cand[at] = key;
                    }
                }
        }
    }
    if (k > 0) {
        __syncthreads();
        if (sm.n > (uint32_t)kLpCap) lp_checked<T, THREADS>(sm, part, k);
    }
    // ---- join the threads' sums ----
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, a.m, d), z2 = __shfl_xor_sync(0xffffffffu, a.z, d),
                    w2 = __shfl_xor_sync(0xffffffffu, a.w, d);
        a.join(m2, z2, w2);
    }
    if (lane == 0) sm.rm[warp] = a.m, sm.rz[warp] = a.z, sm.rw[warp] = a.w;
    __syncthreads();
    if (threadIdx.x == 0) {
        LpSum t{sm.rm[0], sm.rz[0], sm.rw[0]};
        for (int i = 1; i < THREADS / 32; i++) t.join(sm.rm[i], sm.rz[i], sm.rw[i]);
        sm.cm = t.m, sm.cz = t.z, sm.cw = t.w;
    }
    // ---- this CTA's largest keys, in order ----
    if (k > 0) {
        for (uint32_t i = threadIdx.x; i < k; i += THREADS) sm.top[i] = 0;
        __syncthreads();
        const uint32_t n = sm.n;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const uint64_t key = sm.cand[i];
            uint32_t above = 0;
            for (uint32_t j = 0; j < n; j++) above += sm.cand[j] > key;
            if (above < k) sm.top[above] = key;
        }
    }
    if (splits > 1) {
        cluster_sync_all();
        if (rank == 0) {  // join the cluster's states and candidates
            if (threadIdx.x == 0) {
                LpSum t{sm.cm, sm.cz, sm.cw};
                for (uint32_t c = 1; c < splits; c++)
                    t.join(ld_cluster_f32(cluster_addr(smem_u32(&sm.cm), c)), ld_cluster_f32(cluster_addr(smem_u32(&sm.cz), c)),
                           ld_cluster_f32(cluster_addr(smem_u32(&sm.cw), c)));
                sm.rm[0] = t.m, sm.rz[0] = t.z, sm.rw[0] = t.w;
            }
            const uint32_t n = splits * k;  // <= 2048
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint32_t src = cluster_addr(smem_u32(&sm.top[i % k]), i / k);
                uint64_t key;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(src) : "memory");
                sm.cand[i] = key;
            }
            __syncthreads();
            uint64_t keys[kLpMaxTop * kLpMaxSplits / THREADS];
            uint32_t ranks[kLpMaxTop * kLpMaxSplits / THREADS];
#pragma unroll
            for (int q = 0; q < kLpMaxTop * kLpMaxSplits / THREADS; q++) {
                const uint32_t i = threadIdx.x + q * THREADS;
                keys[q] = i < n ? sm.cand[i] : 0;
                uint32_t above = 0;
                if (keys[q])
                    for (uint32_t j = 0; j < n; j++) above += sm.cand[j] > keys[q];
                ranks[q] = above;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kLpMaxTop * kLpMaxSplits / THREADS; q++)
                if (keys[q] && ranks[q] < k) sm.cand[ranks[q]] = keys[q];
            __syncthreads();
        }
        cluster_sync_all();
        if (rank != 0) return;
    } else {
        if (threadIdx.x == 0) sm.rm[0] = sm.cm, sm.rz[0] = sm.cz, sm.rw[0] = sm.cw;
        __syncthreads();
    }
    const float m = sm.rm[0], z = sm.rz[0], lz = logf(z);
    if (threadIdx.x == 0) {
        if (p.entropy) p.entropy[r] = lz - sm.rw[0] / z;
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
    const uint64_t *top = splits > 1 ? sm.cand : sm.top;
    for (uint32_t i = threadIdx.x; i < k; i += THREADS) {
        const uint64_t key = top[i];
        p.top_ids[(uint64_t)r * k + i] = (int32_t)~(uint32_t)key;
        p.top_logprobs[(uint64_t)r * k + i] = lp_value((uint32_t)(key >> 32)) - m - lz;
    }
}

template <typename T, int THREADS>
static int launch_lp_threads(rcu_ctx *ctx, const LogprobParams &p, uint32_t per_sm) {
    uint32_t cs = 1;  // up to per_sm CTAs for each SM, and no CTA without a step's values
    while (cs < kLpMaxSplits && (uint64_t)p.rows * cs * 2 <= (uint64_t)per_sm * ctx->num_sms && p.vocab >= (uint64_t)cs * THREADS * kLpPer) cs *= 2;
    return launch_cluster_k(ctx, k_logprobs<T, THREADS>, p.rows * cs, THREADS, sizeof(LpSmem), cs, p, cs);
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
