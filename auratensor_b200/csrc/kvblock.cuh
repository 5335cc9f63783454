// Shared by the kernels of the block-quantized KV cache (kvblock.cu,
// kvblock_attn.cu): the cache and batch descriptors on the device, and the
// checks that keep a bad descriptor from turning into a bad address.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "at_internal.h"
#include "dev_common.cuh"

namespace at {

// Bits of the cache's status word (at_kvb.status).
constexpr int KVB_BAD_SEQ = 1;    // a slot, start or offset outside its range: the sequence was skipped
constexpr int KVB_STALLED = 4;    // a bounded wait inside a kernel ran out: its output is not valid
constexpr int KVB_BAD_BLOCK = 2;  // a block-table entry outside the pool: reads give NaN, writes are dropped
constexpr int KVB_STALE_TAIL = 8;  // an append inside a block whose older rows the tail no longer has: that block was not written

struct KvbDev {
    int hkv, hd, lb;  // lb: log2(block_tokens)
    int n_blocks, max_seqs, max_blocks;
    int8_t *k, *v;
    float *ks, *vs;
    void *kt, *vt;
    float *ktm, *vtm;
    const int32_t* table;
    int32_t* status;
};

struct KvbBatch {
    int n_seqs, n_tokens, max_tokens;
    const int32_t* slots;
    const int64_t* starts;
    const int32_t* offsets;
};

// Host checks (kvblock.cu); fail() with the framework's status classes.
KvbDev kvb_dev(const at_ctx* ctx, const at_kvb* c, bool with_tail);
KvbBatch kvb_batch(const at_kvb* c, const at_token_batch* b);

struct KvbSeq {
    int slot, n, off;
    int64_t start;
};

__device__ __forceinline__ void kvb_flag(int32_t* status, int bit) {
    if (status) atomicOr(status, bit);
}

// Sequence s of the batch; n = 0 (and the status bit) when it is out of range.
__device__ __forceinline__ KvbSeq kvb_seq(const KvbDev& c, const KvbBatch& b, int s) {
    KvbSeq q;
    q.slot = b.slots[s];
    q.start = b.starts[s];
    q.off = b.offsets[s];
    q.n = b.offsets[s + 1] - q.off;
    const int64_t room = (int64_t)c.max_blocks << c.lb;
    if (q.n < 0 || q.n > b.max_tokens || q.off < 0 || q.off > b.n_tokens - q.n || (unsigned)q.slot >= (unsigned)c.max_seqs ||
        q.start < 0 || q.start > room - q.n) {
        kvb_flag(c.status, KVB_BAD_SEQ);
        q.n = 0;
    }
    return q;
}

// Page of a sequence's block, or -1 (and the status bit).
__device__ __forceinline__ int kvb_page(const KvbDev& c, int slot, int blk) {
    const int p = c.table[(size_t)slot * c.max_blocks + blk];
    if ((unsigned)p < (unsigned)c.n_blocks) return p;
    kvb_flag(c.status, KVB_BAD_BLOCK);
    return -1;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Calls f with a value of the C++ type of a dtype code.
template <class F>
inline void kvb_dispatch(int dtype, F&& f) {
    switch (dtype) {
        case AT_GGML_F32: f(float{}); return;
        case AT_GGML_F16: f(__half{}); return;
        case AT_GGML_BF16: f(__nv_bfloat16{}); return;
        default: fail(AT_ERR_UNSUPPORTED, "element type must be F32, F16 or BF16, got " + std::to_string(dtype));
    }
}
// Two FP32 lanes in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r)) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r)) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(r))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return r;
}

// Eight consecutive elements as they are; vec: p is 16-byte aligned.
template <class T>
struct alignas(16) Raw8 {
    T t[8];
};
template <class T>
__device__ __forceinline__ void load_raw8(const T* __restrict__ p, bool vec, Raw8<T>& x) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(x.t)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.t[i] = p[i];
    }
}
template <class T>
__device__ __forceinline__ void to_f32x8(const Raw8<T>& r, float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(r.t[i]);
}
// Eight consecutive elements as FP32.
template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool vec, float* x) {
    Raw8<T> r;
    load_raw8<T>(p, vec, r);
    to_f32x8<T>(r, x);
}

inline int kvb_elem_bytes(int dtype) { return dtype == AT_GGML_F32 ? 4 : 2; }

// Whether every row of head_dim elements starts on a 16-byte boundary.
inline bool aligned_rows(const void* x, int elem_bytes, int64_t token_stride, int64_t head_stride) {
    return (((uintptr_t)x | (uintptr_t)(token_stride * elem_bytes) | (uintptr_t)(head_stride * elem_bytes)) & 15) == 0;
}

}  // namespace at
