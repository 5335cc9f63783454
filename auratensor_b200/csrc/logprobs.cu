// Log probabilities of given tokens, with entropy and top alternatives, from
// rows of logits x[V]:
//   m = max x, s = sum e^(x - m), lse = m + log s, log p_t = (x_t - m) - log s
//   (not x_t - lse: lse loses log s's digits when |m| is large),
//   H = log s - (sum (x - m) e^(x - m)) / s   (terms with e = 0 count 0),
// and the k largest logits in descending order, equal ones by the lower id.
// Rows without a distribution: all -inf gives lse -inf, log p -inf, H 0;
// a NaN or +inf gives NaN for lse, log p and H. The alternatives are ordered
// all the same, NaN above +inf.
#include <cstdint>
#include <string>

#include "kvblock.cuh"

namespace at {

namespace {

constexpr int LP_THREADS = 512;
constexpr int LP_TOP_MAX = 32;

// Order-preserving bits: NaN on top, -0 equal to +0.
__device__ __forceinline__ uint32_t lp_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long lp_pack(float v, int i) {
    return ((unsigned long long)lp_key(v) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}

template <class R, class F>
__device__ __forceinline__ R lp_block_reduce(R v, R* s, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) s[warp] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < LP_THREADS / 32; ++w) v = f(v, s[w]);
    return v;
}

template <class T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const T* __restrict__ logits, int V, int64_t stride,
                                                              const int32_t* __restrict__ tokens, int k, float* __restrict__ lp,
                                                              float* __restrict__ lse_out, float* __restrict__ ent,
                                                              int32_t* __restrict__ ids, float* __restrict__ alt) {
    __shared__ float s_f[LP_THREADS / 32];
    __shared__ unsigned long long s_k[LP_THREADS / 32];
    const T* x = logits + (int64_t)blockIdx.x * stride;
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < V; i += LP_THREADS) best = max(best, lp_pack(to_f32<T>(x[i]), i));
    best = lp_block_reduce(best, s_k, [](unsigned long long a, unsigned long long c) { return a > c ? a : c; });
    const int top = (int)(0xFFFFFFFFu - (uint32_t)best);
    const float m = to_f32<T>(x[top]);
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < V; i += LP_THREADS) {
        const float d = to_f32<T>(x[i]) - m, e = expf(d);
        s += e;
        t += e > 0.f ? d * e : 0.f;
    }
    auto add = [](float a, float c) { return a + c; };
    s = lp_block_reduce(s, s_f, add);
    t = lp_block_reduce(t, s_f, add);
    const float nan = __uint_as_float(0x7FC00000u);
    const float ls = logf(s);
    float lse = m + ls, h = ls - t / s;
    if (m == -INFINITY) {
        lse = -INFINITY;
        h = 0.f;
    } else if (!(m < INFINITY)) {
        lse = h = nan;
    }
    auto logp = [&](float v) { return lse != lse ? nan : v == -INFINITY ? v : (v - m) - ls; };
    if (threadIdx.x == 0) {
        const int r = blockIdx.x;
        lse_out[r] = lse;
        ent[r] = h;
        if (lp) {
            const int tok = tokens[r];
            lp[r] = (unsigned)tok < (unsigned)V ? logp(to_f32<T>(x[tok])) : nan;
        }
    }
    for (int j = 0; j < k; ++j) {
        if (j > 0) {
            unsigned long long nb = 0;
            for (int i = threadIdx.x; i < V; i += LP_THREADS) {
                const unsigned long long p = lp_pack(to_f32<T>(x[i]), i);
                if (p < best) nb = max(nb, p);
            }
            best = lp_block_reduce(nb, s_k, [](unsigned long long a, unsigned long long c) { return a > c ? a : c; });
        }
        if (threadIdx.x == 0) {
            const int id = (int)(0xFFFFFFFFu - (uint32_t)best);
            ids[(int64_t)blockIdx.x * k + j] = id;
            alt[(int64_t)blockIdx.x * k + j] = logp(to_f32<T>(x[id]));
        }
    }
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
            logprobs_kernel<T><<<rows, LP_THREADS, 0, ctx->stream>>>(static_cast<const T*>(logits), vocab, row_stride, tokens, n_top,
                                                                     logprob, logsumexp, entropy, top_ids, top_logprobs);
        });
        AT_CUDA(cudaGetLastError());
    });
}

}  // extern "C"
