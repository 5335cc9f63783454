// Attention over the block-quantized KV cache (kvblock.cu).
//
// The query at position p of a sequence sees the keys j <= p (and
// j > p - window when a window is set):
//   s_j = scale * d_k(j) * sum_c q_c k8_jc,   out = sum_j e^(s_j - m) d_v(j) v8_j / sum_j e^(s_j - m)
// with m the running maximum; statistics and sums in FP32. A hidden key is
// left out by its index, so what its bytes or scale hold never matters; a
// visible key of a poisoned block (scale NaN) makes the row NaN.
#include <cstdint>
#include <string>

#include "kvblock.cuh"

namespace at {

namespace {

constexpr int SIMPLE_THREADS = 128;

// One CTA per query token and query head: each warp walks every fourth key
// with the lanes across the head dimension, then the warps are joined.
template <class T, int HD>
__global__ void __launch_bounds__(SIMPLE_THREADS) kvb_attn_simple_kernel(KvbDev c, KvbBatch b, const T* __restrict__ q,
                                                                         int64_t q_ts, int64_t q_hs, T* __restrict__ out, int H,
                                                                         float scale, int window) {
    constexpr int E = HD / 32, W = SIMPLE_THREADS / 32;
    __shared__ float s_m[W], s_l[W], s_o[W][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.x % H, i = (blockIdx.x / H) % b.max_tokens, s = blockIdx.x / H / b.max_tokens;
    const KvbSeq sq = kvb_seq(c, b, s);
    if (i >= sq.n) return;
    const int kvh = h / (H / c.hkv), pos = (int)sq.start + i;
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = to_f32<T>(q[(int64_t)(sq.off + i) * q_ts + (int64_t)h * q_hs + lane * E + e]) * scale;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = lo + warp; j <= pos; j += W) {
        const int page = kvb_page(c, sq.slot, j >> c.lb);
        const size_t ph = (size_t)max(page, 0) * c.hkv + kvh;
        const float dk = page < 0 ? __uint_as_float(0x7FC00000u) : c.ks[ph], dv = page < 0 ? dk : c.vs[ph];
        const size_t at = ((ph << c.lb) + (j & ((1 << c.lb) - 1))) * HD + lane * E;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) dot = fmaf(qv[e], (float)c.k[at + e], dot);
        const float sc = warp_sum(dot) * dk;
        const float mn = fmaxf(m, sc);
        const float a = mn == -INFINITY ? 1.f : expf(m - mn), p = expf(sc - mn);
        l = fmaf(l, a, p);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], a, p * dv * (float)c.v[at + e]);
        m = mn;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    __syncthreads();
    float mx = -INFINITY;
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w]);
    float lt = 0.f;
    for (int w = 0; w < W; ++w) lt += s_l[w] == 0.f ? 0.f : s_l[w] * expf(s_m[w] - mx);
    for (int d = threadIdx.x; d < HD; d += SIMPLE_THREADS) {
        float acc = 0.f;
        for (int w = 0; w < W; ++w) acc += s_l[w] == 0.f ? 0.f : s_o[w][d] * expf(s_m[w] - mx);
        out[((size_t)(sq.off + i) * H + h) * HD + d] = from_f32<T>(acc / lt);
    }
}

}  // namespace

}  // namespace at

using namespace at;

extern "C" {

int at_kvb_attention_workspace(at_ctx* ctx, const at_kvb* cache, const at_token_batch* batch, int n_heads, int window,
                               size_t* bytes) {
    return guard([&] {
        kvb_dev(ctx, cache, false);
        kvb_batch(cache, batch);
        AT_REQUIRE(bytes, AT_ERR_INVALID_ARG, "null output");
        AT_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0, AT_ERR_INVALID_ARG,
                   "query heads must be a multiple of the KV heads");
        (void)window;
        *bytes = 0;
    });
}

int at_kvb_attention(at_ctx* ctx, const at_kvb* cache, const at_token_batch* batch, int dtype, int n_heads, const void* q,
                     int64_t q_token_stride, int64_t q_head_stride, void* out, float scale, int window, void* workspace,
                     size_t workspace_bytes) {
    return guard([&] {
        const KvbDev c = kvb_dev(ctx, cache, false);
        const KvbBatch b = kvb_batch(cache, batch);
        AT_REQUIRE(dtype == AT_GGML_F32 || dtype == AT_GGML_F16 || dtype == AT_GGML_BF16, AT_ERR_UNSUPPORTED,
                   "query type must be F32, F16 or BF16");
        AT_REQUIRE(n_heads > 0 && n_heads % c.hkv == 0, AT_ERR_INVALID_ARG, "query heads must be a multiple of the KV heads");
        AT_REQUIRE(window >= 0, AT_ERR_INVALID_ARG, "window must not be negative");
        AT_REQUIRE(scale > 0.f && scale < INFINITY, AT_ERR_INVALID_ARG, "scale must be positive and finite");
        if (b.n_seqs == 0 || b.max_tokens == 0) return;
        AT_REQUIRE(q && out, AT_ERR_INVALID_ARG, "null q or out");
        AT_REQUIRE(((uintptr_t)out & 15) == 0 && ((uintptr_t)q & (kvb_elem_bytes(dtype) - 1)) == 0, AT_ERR_INVALID_ARG,
                   "out must be 16-byte aligned, q aligned to its elements");
        (void)workspace;
        (void)workspace_bytes;
        const int64_t grid = (int64_t)b.n_seqs * b.max_tokens * n_heads;
        AT_REQUIRE(grid <= INT32_MAX, AT_ERR_INVALID_ARG, "the batch is too large for one call");
        AT_CUDA(cudaSetDevice(ctx->device));
        kvb_dispatch(dtype, [&](auto t) {
            using T = decltype(t);
            auto kern = c.hd == 128 ? kvb_attn_simple_kernel<T, 128> : kvb_attn_simple_kernel<T, 64>;
            kern<<<(int)grid, SIMPLE_THREADS, 0, ctx->stream>>>(c, b, static_cast<const T*>(q), q_token_stride, q_head_stride,
                                                                static_cast<T*>(out), n_heads, scale, window);
        });
        AT_CUDA(cudaGetLastError());
    });
}

}  // extern "C"
