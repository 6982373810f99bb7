// rcu_logprobs.cu -- log probabilities of given tokens, entropy and the most likely alternatives of
// rows of logits, in one pass over the logits.
//
// For a row x of `vocab` logits, m = max x, z = sum exp(x - m):
//   log p(i) = (x_i - m) - ln z          entropy = ln z - (sum exp(x - m) (x - m)) / z
// and the top_k largest, ties to the lowest index (a NaN counts as the largest value, -0 as 0).
//
// Reading the logits is the bound. A cluster of `splits` CTAs shares a row, each thread keeps a
// running (m, z, sum) over the values it reads, 16 a step. The alternatives need no second pass: a
// value is a 64-bit key (ordered value, ~index), and after the first step the k-th largest of the
// threads' own maxima is a bound below which nothing can be among the k largest of the row; a later
// value reaches the candidate list in shared memory only above it. When that list could run over,
// the same bound is taken again from the list itself. The list's ranks, by counting larger keys,
// are the order of the answer.
#include <cstdint>
#include <type_traits>

#include "rcu_kernels.h"
#include "rcu_seq.cuh"

namespace rcu {

constexpr int kLpThreads = 256;
constexpr int kLpPer = 16;                       // values a thread reads per step
constexpr int kLpStep = kLpThreads * kLpPer;
constexpr int kLpMaxTop = 128;
constexpr int kLpMaxSplits = 16;
constexpr int kLpKeep = 1024;                    // candidates kept over a step at most
constexpr int kLpCap = kLpKeep + kLpStep;

struct LpSmem {
    uint64_t cand[kLpCap];
    uint64_t tmax[kLpThreads];
    uint64_t top[kLpMaxTop];      // this CTA's largest keys in order
    float rm[8], rz[8], rw[8];
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

// k-th largest of the threads' keys `mine` (0: no key): a lower bound of the k-th largest of all
// keys that the threads' own maxima stand for; 0 when fewer than k threads have a key.
__device__ __forceinline__ uint64_t lp_bound(LpSmem &sm, uint64_t mine, uint32_t k) {
    sm.tmax[threadIdx.x] = mine;
    if (threadIdx.x == 0) sm.bound = 0;
    __syncthreads();
    uint32_t above = 0;
#pragma unroll 8
    for (int i = 0; i < kLpThreads; i++) above += sm.tmax[i] > mine;
    if (mine != 0 && above == k - 1) sm.bound = mine;  // keys differ: one thread at most
    __syncthreads();
    return sm.bound;
}
// Raises the bound from the candidate list itself and drops what lies below it.
__device__ __noinline__ uint64_t lp_compact(LpSmem &sm, uint32_t n, uint32_t k) {
    constexpr int kMost = (kLpCap + kLpThreads - 1) / kLpThreads;
    uint64_t own[kMost], mx = 0;
#pragma unroll
    for (int i = 0; i < kMost; i++) {
        const uint32_t j = threadIdx.x + i * kLpThreads;
        own[i] = j < n ? sm.cand[j] : 0;
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

template <typename T>
__global__ void __launch_bounds__(kLpThreads) k_logprobs(const LogprobParams p, uint32_t splits) {
    constexpr int VE = 16 / sizeof(T);      // values of a 16-byte load
    constexpr int NV = kLpPer / VE;         // loads a step
    extern __shared__ __align__(16) uint8_t lp_raw[];
    LpSmem &sm = *reinterpret_cast<LpSmem *>(lp_raw);
    const uint32_t rank = splits > 1 ? cluster_ctarank() : 0, r = blockIdx.x / splits, k = p.top_k;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) sm.n = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const T *x = reinterpret_cast<const T *>(p.logits) + (uint64_t)r * p.ld;
    // 16-byte pieces of the row, counted from the boundary at or below its start
    const uint32_t off = (uint32_t)(((uintptr_t)x & 15) / sizeof(T));
    const T *base = x - off;
    const uint32_t n_vec = (off + p.vocab + VE - 1) / VE, per = (n_vec + splits - 1) / splits;
    const uint32_t v0 = min(rank * per, n_vec), v1 = min(v0 + per, n_vec);

    LpSum a;
    uint64_t bound = 0;
    float boundf = -INFINITY;
    for (uint32_t s = v0; s < v1; s += kLpThreads * NV) {
        float f[kLpPer];
        bool in = true;  // every value of this thread's pieces is one of the row
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t v = s + j * kLpThreads + threadIdx.x;
            const int64_t e0 = (int64_t)v * VE - off;
            if (v < v1 && e0 >= 0 && e0 + VE <= (int64_t)p.vocab) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(base) + v);
                const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
                for (int i = 0; i < VE; i++) f[j * VE + i] = to_f32(t[i]);
            } else {
                in = false;
#pragma unroll
                for (int i = 0; i < VE; i++)
                    f[j * VE + i] = v < v1 && e0 + i >= 0 && e0 + i < (int64_t)p.vocab ? to_f32(x[e0 + i]) : -INFINITY;
            }
        }
        float c = f[0];
#pragma unroll
        for (int i = 1; i < kLpPer; i++) c = fmaxf(c, f[i]);
        if (c > a.m) a.raise(c);
        if (a.m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < kLpPer; i++) a.add(f[i]);
        } else {  // nothing above -inf so far: only a NaN counts
#pragma unroll
            for (int i = 0; i < kLpPer; i++)
                if (f[i] != f[i]) a.z = f[i];
        }
        if (k == 0) continue;
        auto index = [&](int i) {  // of value i, below vocab
            return (uint32_t)((int64_t)(s + (i / VE) * kLpThreads + threadIdx.x) * VE - off + i % VE);
        };
        auto valid = [&](int i) { return in || (s + (i / VE) * kLpThreads + threadIdx.x < v1 && index(i) < p.vocab); };
        if (s == v0) {
            uint64_t mx = 0;
#pragma unroll
            for (int i = 0; i < kLpPer; i++) {
                const uint64_t key = valid(i) ? lp_key(f[i], index(i)) : 0;
                mx = key > mx ? key : mx;
            }
            bound = lp_bound(sm, mx, k);
            if (bound) boundf = lp_value((uint32_t)(bound >> 32));
        }
        bool any = false;
#pragma unroll
        for (int i = 0; i < kLpPer; i++) any |= !(f[i] < boundf);
        if (any) {
#pragma unroll
            for (int i = 0; i < kLpPer; i++)
                if (!(f[i] < boundf) && valid(i)) {
                    const uint64_t key = lp_key(f[i], index(i));
                    if (key >= bound) sm.cand[atomicAdd(&sm.n, 1u)] = key;
                }
        }
        __syncthreads();
        uint32_t n = sm.n;
        __syncthreads();
        while (n > (uint32_t)kLpKeep) {  // at most k * ceil(n / 256) <= n / 2 + 128 keys stay
            bound = lp_compact(sm, n, k);
            boundf = bound ? lp_value((uint32_t)(bound >> 32)) : -INFINITY;
            n = sm.n;
            __syncthreads();
        }
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
        for (int i = 1; i < kLpThreads / 32; i++) t.join(sm.rm[i], sm.rz[i], sm.rw[i]);
        sm.cm = t.m, sm.cz = t.z, sm.cw = t.w;
    }
    // ---- this CTA's largest keys, in order ----
    if (k > 0) {
        for (uint32_t i = threadIdx.x; i < k; i += kLpThreads) sm.top[i] = 0;
        __syncthreads();
        const uint32_t n = sm.n;
        for (uint32_t i = threadIdx.x; i < n; i += kLpThreads) {
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
            for (uint32_t i = threadIdx.x; i < n; i += kLpThreads) {
                const uint32_t src = cluster_addr(smem_u32(&sm.top[i % k]), i / k);
                uint64_t key;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(src) : "memory");
                sm.cand[i] = key;
            }
            __syncthreads();
            uint64_t keys[kLpMaxTop * kLpMaxSplits / kLpThreads];
            uint32_t ranks[kLpMaxTop * kLpMaxSplits / kLpThreads];
#pragma unroll
            for (int q = 0; q < kLpMaxTop * kLpMaxSplits / kLpThreads; q++) {
                const uint32_t i = threadIdx.x + q * kLpThreads;
                keys[q] = i < n ? sm.cand[i] : 0;
                uint32_t above = 0;
                if (keys[q])
                    for (uint32_t j = 0; j < n; j++) above += sm.cand[j] > keys[q];
                ranks[q] = above;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kLpMaxTop * kLpMaxSplits / kLpThreads; q++)
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
    for (uint32_t i = threadIdx.x; i < k; i += kLpThreads) {
        const uint64_t key = top[i];
        p.top_ids[(uint64_t)r * k + i] = (int32_t)~(uint32_t)key;
        p.top_logprobs[(uint64_t)r * k + i] = lp_value((uint32_t)(key >> 32)) - m - lz;
    }
}

template <typename T>
static int launch_lp(rcu_ctx *ctx, const LogprobParams &p) {
    uint32_t cs = 1;  // up to four CTAs for each SM, two steps of values for each
    while (cs < kLpMaxSplits && (uint64_t)p.rows * cs * 2 <= 4ull * ctx->num_sms && p.vocab >= (uint64_t)cs * 2 * kLpStep) cs *= 2;
    return launch_cluster_k(ctx, k_logprobs<T>, p.rows * cs, kLpThreads, sizeof(LpSmem), cs, p, cs);
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
