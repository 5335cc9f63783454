// Shared by the two attention kernels over the block-quantized KV cache: the
// step kernel (kvblock_attn.cu) and the prompt kernel (kvblock_prompt.cu).
#pragma once

#include "kvblock.cuh"

namespace at {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {  // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
// Bytes 0 and 2 (odd: 1 and 3) of w as f16 pairs: q exactly, or, BIASED,
// (q + 128) 2^-24.
template <bool BIASED>
__device__ __forceinline__ uint32_t bytes_h2(uint32_t w, bool odd) {
    if (odd) w >>= 8;
    if constexpr (BIASED) {
        return (w & 0x00FF00FFu) ^ 0x00800080u;
    } else {
        const uint32_t m = (w & 0x00FF00FFu) ^ 0x64806480u, c = 0x64806480u;  // 1024 + 128 + q; 1152
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&c));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
// Power of two that brings a row whose largest |x| is `top` to [512, 1024).
__device__ __forceinline__ float row_scale(float top) {
    const int e = (int)(__float_as_uint(top) >> 23) - 127;  // -127: zero or subnormal
    return __uint_as_float((uint32_t)(127 + min(9 - e, 126)) << 23);
}

// log2 d_v of a block as the attention kernels use it: weights are kept as
// 2^(s + lv), their sum as 2^(s + lv) iv. A zero scale holds zeros only, so any
// weight will do for its values: it counts as 2^-80, far below the scales that
// stand next to it, and 2^31 keys of the largest weight, 2^14, still sum to
// less than FP32's end. The bounds of this form: a sum of n such weights over
// blocks of scale d overflows at n 2^14 / d = 2^128 (2^17 keys: all visible
// scales below 2^-97), and what lies 2^-134 below the largest t is lost, so
// that scales up to 2^110 apart leave the sum its 24 bits.
// EXACT splits d_v into a power of two (lv, iv) and a mantissa mv that
// multiplies the weights; else lv is the whole logarithm (its error, 2^-20 at
// most, is far below 16-bit outputs) and mv 1.
template <bool EXACT>
__device__ __forceinline__ void value_scale(float dv, float* lv, float* iv, float* mv) {
    const float d = dv == 0.f ? 0x1p-80f : dv;
    if constexpr (EXACT) {
        const uint32_t u = __float_as_uint(d);
        const int e = (int)(u >> 23) - 127;  // d is normal, or NaN
        *lv = d != d ? d : (float)e;
        *iv = d != d ? d : __uint_as_float((uint32_t)(127 - e) << 23);
        *mv = d != d ? d : __uint_as_float((u & 0x007FFFFFu) | 0x3F800000u);
    } else {
        *lv = __log2f(d);
        *iv = __fdividef(1.f, d);
        *mv = 1.f;
    }
}

// The prompt kernel, for sequences of more than min_rows query rows per KV head.
void launch_kvb_attn_prompt(const KvbDev& c, const KvbBatch& b, int dtype, int n_heads, const void* q, int64_t q_ts, int64_t q_hs, void* out,
                            float scale, int window, int min_rows, cudaStream_t s);

}  // namespace at
