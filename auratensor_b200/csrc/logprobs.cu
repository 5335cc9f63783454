// Log probabilities of given tokens, with entropy and top alternatives, from
// rows of logits x[V]:
//   m = max x, s = sum e^(x - m), lse = m + log s, log p_t = (x_t - m) - log s
//   (not x_t - lse: lse loses log s's digits when |m| is large),
//   H = log s - (sum (x - m) e^(x - m)) / s   (terms with e = 0 count 0),
// and the k largest logits in descending order, equal ones by the lower id.
// Rows without a distribution: all -inf gives lse -inf, log p -inf, H 0;
// a NaN or +inf gives NaN for lse, log p and H. The alternatives are ordered
// all the same, NaN above +inf.
//
// One pass over the logits, which is what bounds it: each thread keeps its own
// running maximum and sums (FP32, joined at the end), 64 bytes of a row per
// thread and step in flight. The alternatives ride along: what exceeds a bound
// tau, which leaves at least k logits of the row at or above it, goes to a
// shared-memory list (a few times k values) that is ranked at the end. tau is
// the k-th largest of the running maxima of 64 groups of lanes, found after
// 1, 2, 4, 8 .. steps with the whole CTA (each halves what passes per step),
// and between those by any warp that sees many of its lanes above tau, from
// its own lanes' maxima, so that a row whose large logits come late does not
// flood the list. Ties: tau is set just below its value, so that the logits
// equal to it are listed, unless there are many (constant or masked rows);
// then they are left out and the first ids equal to tau fill up at the end. A
// row is one CTA, or a cluster of up to 8 whose parts meet in distributed
// shared memory when there are too few rows to fill the GPU.
// 2048 rows of 128256 logits, k = 20: 139 us in BF16 (3.8 TB/s: 70 % of the
// issue slots and 45 % of ex2's rate; the rest is waiting, at the CTA's
// barriers and for a step's loads, which are not in flight while the step
// before is summed or a row's list is ranked), 183 to 199 us in FP32 (5.5
// TB/s). 8 rows of FP32, k = 5: 8.8 us, its launch, the list's ranking and the
// cluster's join. 256 threads are as fast for many rows and slower for few
// (10.5 us); the next step's loads ahead of time need 64 registers and lose a
// CTA (167 us).
#include <cooperative_groups.h>

#include <cstdint>
#include <string>

#include "kvblock.cuh"

namespace at {

namespace {

namespace cg = cooperative_groups;

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOP_MAX = 32;
constexpr int LP_VECS = 4;                       // 16-byte vectors per thread and step
constexpr int LP_GROUP = 8;                      // lanes whose maximum counts as one for tau
constexpr int LP_GROUPS = LP_THREADS / LP_GROUP; // >= LP_TOP_MAX
constexpr int LP_LIST = 2048;                    // values above tau
constexpr int LP_RAISE = 12;                     // lanes of a warp above tau that make the warp raise it
constexpr int LP_TIES = 16;                      // maxima beyond k at or above a new tau: more are ties, and it is set on, not below, its value
constexpr int LP_MAX_CLUSTER = 8;
constexpr uint32_t LP_NINF = 0x007FFFFFu;        // lp_key(-inf)

// Order-preserving bits: NaN on top, -0 equal to +0.
__device__ __forceinline__ uint32_t lp_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// Larger value first, then the lower id.
__device__ __forceinline__ unsigned long long lp_pack(float v, int i) {
    return ((unsigned long long)lp_key(v) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}
// The value of a key, and the key just below (-0 is skipped: it is +0's equal).
__device__ __forceinline__ float lp_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint32_t lp_below(uint32_t k) { return k == 0x80000000u ? k - 2u : k - 1u; }
__device__ __forceinline__ int lp_id(unsigned long long p) { return (int)(0xFFFFFFFFu - (uint32_t)p); }

__device__ __forceinline__ float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Word w of a 16-byte vector: two 16-bit logits, or one FP32 logit.
template <class T>
struct Words;
template <>
struct Words<float> {
    static constexpr uint32_t NINF = 0xFF800000u;  // -inf in every lane of a word
    static __device__ __forceinline__ float max_of(const uint4& v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ float2 pair(const uint4& v, int j) {  // j 0..1
        return j ? make_float2(__uint_as_float(v.z), __uint_as_float(v.w)) : make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    }
};
template <class H2>
__device__ __forceinline__ float max16(const uint4& v) {
    const H2* h = reinterpret_cast<const H2*>(&v);
    const H2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf((float)m.x, (float)m.y);
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }
template <>
struct Words<__half> {
    static constexpr uint32_t NINF = 0xFC00FC00u;
    static __device__ __forceinline__ float max_of(const uint4& v) { return max16<__half2>(v); }
    static __device__ __forceinline__ float2 pair(const uint4& v, int j) {
        const uint32_t w = word_of(v, j);
        return __half22float2(reinterpret_cast<const __half2&>(w));
    }
};
template <>
struct Words<__nv_bfloat16> {
    static constexpr uint32_t NINF = 0xFF80FF80u;
    static __device__ __forceinline__ float max_of(const uint4& v) { return max16<__nv_bfloat162>(v); }
    static __device__ __forceinline__ float2 pair(const uint4& v, int j) {
        const uint32_t w = word_of(v, j);
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
};

// Running maximum and sums of one thread (or of a joined set): s = sum e^(x - m),
// t = sum (x - m) e^(x - m).
struct Sums {
    float m, s, t;
    __device__ __forceinline__ void move(float to) {  // to >= m
        const float d = m - to, a = __expf(d);
        t = a == 0.f ? 0.f : a * fmaf(d, s, t);  // d may be -inf
        s *= a;                                  // a NaN stays
        m = to;
    }
    // The sums of all lanes (of groups of W lanes), in every lane.
    template <int W>
    __device__ __forceinline__ void join_lanes() {
        float to = m;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
        if (m != to) move(to);  // to is not -inf then
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
    }
    __device__ __forceinline__ void add(float x) {
        if (x > m) move(x);
        const float d = x - (m == -INFINITY ? 0.f : m), e = __expf(d);
        s += e;
        t += e == 0.f ? 0.f : e * d;
    }
};

struct LpShared {
    unsigned long long list[LP_LIST];
    unsigned long long top[LP_TOP_MAX];          // the CTA's k best, in order (0: fewer)
    unsigned long long best_of_row[LP_TOP_MAX];  // the cluster's
    unsigned long long best[LP_WARPS];
    float group[LP_GROUPS];
    Sums part[LP_WARPS], sums;
    unsigned count;
    int eq[LP_WARPS];
    float bound;
    uint32_t tau;  // a key
};

struct LpParams {
    const void* logits;
    int64_t stride;
    int V, k, splits, log_splits;
    const int32_t* tokens;
    float *lp, *lse, *ent;
    int32_t* ids;
    float* alt;
};

// The CTA's k best by rounds of "the largest below the last": for rows with
// NaN or +inf, and for lists that overflowed.
template <class T>
__device__ void lp_top_slow(const T* x, int lo, int hi, int k, LpShared* sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long last = ~0ull;
    for (int j = 0; j < k; ++j) {
        unsigned long long b = 0;
        for (int i = lo + tid; i < hi; i += LP_THREADS) {
            const unsigned long long p = lp_pack(to_f32<T>(x[i]), i);
            if (p < last && p > b) b = p;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
            b = c > b ? c : b;
        }
        __syncthreads();
        if (lane == 0) sh->best[warp] = b;
        __syncthreads();
        for (int w = 0; w < LP_WARPS; ++w) b = sh->best[w] > b ? sh->best[w] : b;
        last = b;
        if (tid == 0) sh->top[j] = b;
        if (b == 0) break;  // fewer than k logits here (the rest of top is 0)
    }
}

template <class T>
__global__ void __launch_bounds__(LP_THREADS, 3) logprobs_kernel(const LpParams p) {
    using W = Words<T>;
    constexpr int VE = 16 / (int)sizeof(T);                 // logits per vector
    constexpr float L2E = 1.44269504088896341f;
    __shared__ LpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x >> p.log_splits, part = blockIdx.x & (p.splits - 1);
    const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.stride;
    const int k = p.k;
    // this CTA's ids [lo, hi); vectors of the row start at its first 16-byte boundary
    const int head = min(p.V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int nv = (p.V - head) / VE;
    const int v0 = (int)(((int64_t)nv * part) >> p.log_splits), v1 = (int)(((int64_t)nv * (part + 1)) >> p.log_splits);
    const int lo = part == 0 ? 0 : head + v0 * VE, hi = part == p.splits - 1 ? p.V : head + v1 * VE;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);

    if (tid == 0) {
        sh.count = 0;
        sh.tau = LP_NINF;
    }
    if (tid < LP_TOP_MAX) sh.top[tid] = 0;
    __syncthreads();
    Sums mine{-INFINITY, 0.f, 0.f};
    // what lies outside the vectors, one logit per thread, listed as it is
    {
        const int before = part == 0 ? head : 0, after = part == p.splits - 1 ? p.V - head - nv * VE : 0;
        const int i = tid < before ? tid : tid - before < after ? head + nv * VE + tid - before : -1;
        if (i >= 0) {
            const float v = to_f32<T>(x[i]);
            mine.add(v);
            if (k > 0) sh.list[atomicAdd(&sh.count, 1u)] = lp_pack(v, i);
        }
    }
    float bound = -INFINITY;
    for (int b = v0, step = 0; b < v1; b += LP_THREADS * LP_VECS, ++step) {
        uint4 v[LP_VECS];
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i) {
            const int at = b + i * LP_THREADS + tid;
            v[i] = make_uint4(W::NINF, W::NINF, W::NINF, W::NINF);
            if (at < v1) v[i] = ld_stream_u4(xv + at);
        }
        float vtop[LP_VECS], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i) {
            vtop[i] = W::max_of(v[i]);
            top = fmaxf(top, vtop[i]);
        }
        bool some = b + tid < v1;
        if (some && top == -INFINITY) {  // all -inf adds nothing (NaN would: it is not in the maximum)
            uint32_t differs = 0;
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) differs |= (v[i].x ^ W::NINF) | (v[i].y ^ W::NINF) | (v[i].z ^ W::NINF) | (v[i].w ^ W::NINF);
            some = differs != 0;
        }
        if (some) {
            if (top > mine.m) mine.move(top);
            const float ref = mine.m == -INFINITY ? 0.f : mine.m;
            const float2 neg = make_float2(-ref, -ref), l2 = make_float2(L2E, L2E);
            float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < LP_VECS; ++i) {
                if (b + i * LP_THREADS + tid >= v1) break;
#pragma unroll
                for (int j = 0; j < VE / 2; ++j) {
                    const float2 d = add2(W::pair(v[i], j), neg);
                    const float2 a = mul2(d, l2), e = make_float2(lp_ex2(a.x), lp_ex2(a.y));
                    s = add2(s, e);
                    t = fma2(e, d, t);
                }
            }
            float tt = t.x + t.y;
            if (tt != tt) {  // -inf logits (0 (-inf)), or NaN, which s shows
                tt = 0.f;
#pragma unroll
                for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
                    for (int j = 0; j < VE / 2; ++j) {
                        const float2 d = add2(W::pair(v[i], j), neg);
                        const float ex = lp_ex2(d.x * L2E), ey = lp_ex2(d.y * L2E);
                        tt += (ex == 0.f ? 0.f : ex * d.x) + (ey == 0.f ? 0.f : ey * d.y);
                    }
            }
            mine.s += s.x + s.y;
            mine.t += tt;
        }
        if (k > 0) {
            if (((step & (step + 1)) == 0 && (step == 0 || b + LP_THREADS * LP_VECS < v1)) || bound == -INFINITY) {  // uniform
                float g = mine.m;
#pragma unroll
                for (int o = LP_GROUP / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
                if ((tid & (LP_GROUP - 1)) == 0) sh.group[tid / LP_GROUP] = g;
                __syncthreads();
                // LP_GROUP threads rank a group together
                const int grp = tid / LP_GROUP, sub = tid % LP_GROUP;
                const float own = sh.group[grp];
                int rank = 0, at_least = 0;
#pragma unroll
                for (int j = sub; j < LP_GROUPS; j += LP_GROUP) {
                    const float o = sh.group[j];
                    at_least += o >= own;
                    rank += o > own || (o == own && j < grp);
                }
#pragma unroll
                for (int o = LP_GROUP / 2; o > 0; o >>= 1) {
                    rank += __shfl_xor_sync(0xffffffffu, rank, o);
                    at_least += __shfl_xor_sync(0xffffffffu, at_least, o);
                }
                if (sub == 0 && rank == k - 1) {
                    sh.bound = own;
                    if (own > -INFINITY) atomicMax(&sh.tau, at_least > k + LP_TIES ? lp_key(own) : lp_below(lp_key(own)));
                }
                __syncthreads();
                bound = sh.bound;
            } else if (__popc(__ballot_sync(0xffffffffu, top > lp_value(*reinterpret_cast<volatile uint32_t*>(&sh.tau)))) > LP_RAISE) {
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < 32; ++j) {
                    const float o = __shfl_sync(0xffffffffu, top, j);
                    rank += o > top || (o == top && j < lane);
                }
                const uint32_t who = __ballot_sync(0xffffffffu, rank == k - 1);
                const float c = __shfl_sync(0xffffffffu, top, __ffs(who) - 1);
                const int at_least = __popc(__ballot_sync(0xffffffffu, top >= c));
                if (lane == 0 && c > -INFINITY) atomicMax(&sh.tau, at_least > k + LP_TIES ? lp_key(c) : lp_below(lp_key(c)));
                __syncwarp();
            }
            const float tau = lp_value(*reinterpret_cast<volatile uint32_t*>(&sh.tau));
            if (top > tau) {
#pragma unroll
                for (int i = 0; i < LP_VECS; ++i) {
                    if (vtop[i] <= tau) continue;
#pragma unroll
                    for (int j = 0; j < VE / 2; ++j) {
                        const float2 y = W::pair(v[i], j);
                        const int id = head + (b + i * LP_THREADS + tid) * VE + 2 * j;
                        if (y.x > tau) {
                            const unsigned at = atomicAdd(&sh.count, 1u);
                            if (at < LP_LIST) sh.list[at] = lp_pack(y.x, id);
                        }
                        if (y.y > tau) {
                            const unsigned at = atomicAdd(&sh.count, 1u);
                            if (at < LP_LIST) sh.list[at] = lp_pack(y.y, id + 1);
                        }
                    }
                }
            }
        }
    }
    // the CTA's sums
    mine.join_lanes<32>();
    if (lane == 0) sh.part[warp] = mine;
    __syncthreads();
    Sums all = sh.part[lane % LP_WARPS];
    all.join_lanes<LP_WARPS>();
    // its k best
    if (k > 0) {
        const unsigned n = sh.count;
        const uint32_t tau = sh.tau;
        if (all.s != all.s || n > LP_LIST) {
            lp_top_slow(x, lo, hi, k, &sh);
        } else {
            // above tau: ranked; then the first ids equal to tau
            unsigned long long kept[LP_LIST / LP_THREADS];
#pragma unroll
            for (int i = 0; i < LP_LIST / LP_THREADS; ++i) {
                const unsigned at = i * LP_THREADS + tid;
                kept[i] = at < n ? sh.list[at] : 0;
                if ((uint32_t)(kept[i] >> 32) <= tau) kept[i] = 0;  // listed before tau rose
            }
            __syncthreads();
            if (tid == 0) sh.count = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LP_LIST / LP_THREADS; ++i)
                if (kept[i] != 0) sh.list[atomicAdd(&sh.count, 1u)] = kept[i];
            __syncthreads();
            const unsigned above = sh.count;
            for (unsigned base = 0; base < above; base += LP_GROUPS) {  // LP_GROUP threads rank a logit together
                const unsigned i = base + tid / LP_GROUP;
                const unsigned long long mk = i < above ? sh.list[i] : 0;
                unsigned rank = 0;
                for (unsigned j = tid % LP_GROUP; j < above; j += LP_GROUP) rank += sh.list[j] > mk;
#pragma unroll
                for (int o = LP_GROUP / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
                if (mk != 0 && rank < (unsigned)k) sh.top[rank] = mk;
            }
            for (int base = lo, have = (int)above; base < hi && have < k; base += LP_THREADS) {  // uniform
                const int i = base + tid;
                const bool eq = i < hi && lp_key(to_f32<T>(x[i])) == tau;
                const uint32_t ballot = __ballot_sync(0xffffffffu, eq);
                if (lane == 0) sh.eq[warp] = __popc(ballot);
                __syncthreads();
                int before = have, total = 0;
                for (int w = 0; w < LP_WARPS; ++w) {
                    before += w < warp ? sh.eq[w] : 0;
                    total += sh.eq[w];
                }
                const int at = before + __popc(ballot & ((1u << lane) - 1u));
                if (eq && at < k) sh.top[at] = lp_pack(lp_value(tau), i);
                have += total;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    cg::cluster_group cluster = cg::this_cluster();
    if (p.splits > 1) {
        if (tid == 0) sh.sums = all;
        cluster.sync();
        if (part == 0) {
            all = lane < p.splits ? cluster.map_shared_rank(&sh, lane)->sums : Sums{-INFINITY, 0.f, 0.f};
            all.join_lanes<32>();
            const int n = p.splits * k;
            for (int i = tid; i < n; i += LP_THREADS) sh.list[i] = cluster.map_shared_rank(&sh, i / k)->top[i % k];
            __syncthreads();
            for (int base = 0; base < n; base += LP_GROUPS) {
                const int i = base + tid / LP_GROUP;
                const unsigned long long mk = i < n ? sh.list[i] : 0;
                int rank = 0;
                for (int j = tid % LP_GROUP; j < n; j += LP_GROUP) rank += sh.list[j] > mk;
#pragma unroll
                for (int o = LP_GROUP / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
                if (mk != 0 && rank < k) sh.best_of_row[rank] = mk;
            }
            __syncthreads();
        }
        cluster.sync();  // the other CTAs' shared memory has been read
        if (part != 0) return;
    }
    const float nan = __uint_as_float(0x7FC00000u);
    const float ls = logf(all.s);
    float lse = all.m + ls, h = ls - all.t / all.s;
    if (all.s == 0.f) {  // -inf only
        lse = -INFINITY;
        h = 0.f;
    } else if (all.s != all.s) {
        lse = h = nan;
    }
    auto logp = [&](float v) { return lse != lse ? nan : v == -INFINITY ? v : (v - all.m) - ls; };
    if (tid == 0) {
        p.lse[row] = lse;
        p.ent[row] = h;
        if (p.lp) {
            const int tok = p.tokens[row];
            p.lp[row] = (unsigned)tok < (unsigned)p.V ? logp(to_f32<T>(x[tok])) : nan;
        }
    }
    if (tid < k) {
        const int id = lp_id(p.splits > 1 ? sh.best_of_row[tid] : sh.top[tid]);
        p.ids[(int64_t)row * k + tid] = id;
        p.alt[(int64_t)row * k + tid] = logp(to_f32<T>(x[id]));
    }
}

template <class T>
void launch_logprobs(LpParams p, int rows, int num_sms, cudaStream_t s) {
    // As many CTAs per row as fill the GPU once (three are resident per SM),
    // each with a step of logits at least.
    const int step = LP_THREADS * LP_VECS * (16 / (int)sizeof(T));
    int splits = 1;
    while (splits < LP_MAX_CLUSTER && (int64_t)rows * splits * 2 <= 3 * num_sms && (p.V + 2 * splits - 1) / (2 * splits) >= step / 2) splits *= 2;
    p.splits = splits;
    p.log_splits = splits == 1 ? 0 : splits == 2 ? 1 : splits == 4 ? 2 : 3;
    AT_REQUIRE((int64_t)rows * splits <= INT32_MAX, AT_ERR_INVALID_ARG, "logprobs: too many rows for one call");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * splits);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)splits, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    AT_CUDA(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p));
}

}  // namespace

}  // namespace at

using namespace at;

extern "C" {

int at_logprobs(at_ctx* ctx, const void* logits, int dtype, int rows, int vocab, int64_t row_stride, const int32_t* tokens,
                int n_top, float* logprob, float* logsumexp, float* entropy, int32_t* top_ids, float* top_logprobs) {
    return guard([&] {
        AT_REQUIRE(ctx, AT_ERR_INVALID_ARG, "null context");
        AT_REQUIRE(dtype == AT_GGML_F32 || dtype == AT_GGML_F16 || dtype == AT_GGML_BF16, AT_ERR_UNSUPPORTED,
                   "logits must be F32, F16 or BF16");
        AT_REQUIRE(rows >= 0 && vocab > 0, AT_ERR_INVALID_ARG, "logprobs: rows must not be negative, vocab must be positive");
        AT_REQUIRE(row_stride >= vocab || rows <= 1, AT_ERR_INVALID_ARG, "logprobs: rows overlap");
        AT_REQUIRE(n_top >= 0 && n_top <= vocab, AT_ERR_INVALID_ARG, "logprobs: n_top must be in [0, vocab]");
        AT_REQUIRE(n_top <= LP_TOP_MAX, AT_ERR_UNSUPPORTED, "logprobs: at most " + std::to_string(LP_TOP_MAX) + " alternatives");
        if (rows == 0) return;
        AT_REQUIRE(logits && logsumexp && entropy, AT_ERR_INVALID_ARG, "logprobs: null argument");
        AT_REQUIRE((tokens != nullptr) == (logprob != nullptr), AT_ERR_INVALID_ARG, "logprobs: tokens and logprob go together");
        AT_REQUIRE(n_top == 0 || (top_ids && top_logprobs), AT_ERR_INVALID_ARG, "logprobs: null alternatives");
        AT_REQUIRE(((uintptr_t)logits & (kvb_elem_bytes(dtype) - 1)) == 0, AT_ERR_INVALID_ARG, "logits must be aligned to their elements");
        AT_CUDA(cudaSetDevice(ctx->device));
        kvb_dispatch(dtype, [&](auto t) {
            using T = decltype(t);
            launch_logprobs<T>(LpParams{logits, row_stride, vocab, n_top, 1, 0, tokens, logprob, logsumexp, entropy, top_ids, top_logprobs}, rows,
                               ctx->num_sms, ctx->stream);
        });
    });
}

}  // extern "C"
