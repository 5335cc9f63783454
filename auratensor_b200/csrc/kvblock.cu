// The block-quantized KV cache: K and V in 8 bits, one scale for each block of
// tokens and KV head, blocks ("pages") found through a per-sequence table.
//
//   d = max|x| / 127 over the block's values so far (FP32 division; a d below
//       2^-126 is held as 0, a NaN or infinity in the block makes d NaN, so
//       that every read of the block gives NaN)
//   q = round-half-even(x * (1 / d)), read back as q * d.
//
// A block fills token by token, and its scale grows with its maximum. The
// original values of a sequence's last two blocks stay in a ring of 2 B rows
// (the tail, with each row's max|x|), so when a new token raises the maximum
// the block's older rows are quantized again from the originals: what a block
// holds depends on its tokens alone, not on how appends cut them, and no
// error builds up. Two blocks, so that the next append may also start
// anywhere in the last block written or the one before it (a rejected draft
// is overwritten). The ring holds, of the even and of the odd blocks, the one
// written last: an append that starts inside another block would take that
// one's rows for its own, so the row before its first is compared with what
// the page holds of it, and where they differ the append is reported instead.
#include <algorithm>
#include <cstdint>
#include <string>

#include "kvblock.cuh"

namespace at {

KvbDev kvb_dev(const at_ctx* ctx, const at_kvb* c, bool with_tail) {
    AT_REQUIRE(ctx && c, AT_ERR_INVALID_ARG, "null argument");
    AT_REQUIRE(c->dtype == AT_GGML_F32 || c->dtype == AT_GGML_F16 || c->dtype == AT_GGML_BF16, AT_ERR_UNSUPPORTED,
               "cache type must be F32, F16 or BF16, got " + std::to_string(c->dtype));
    AT_REQUIRE(c->head_dim == 64 || c->head_dim == 128, AT_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    AT_REQUIRE(c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128,
               AT_ERR_INVALID_ARG, "block_tokens must be 16, 32, 64 or 128");
    AT_REQUIRE(c->n_kv_heads > 0 && c->n_blocks > 0 && c->max_seqs > 0 && c->max_blocks > 0, AT_ERR_INVALID_ARG,
               "cache dimensions must be positive");
    AT_REQUIRE((int64_t)c->max_blocks * c->block_tokens <= INT32_MAX, AT_ERR_INVALID_ARG, "positions must fit 31 bits");
    AT_REQUIRE(c->k && c->v && c->k_scale && c->v_scale && c->block_table, AT_ERR_INVALID_ARG, "null cache buffer");
    AT_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, AT_ERR_INVALID_ARG, "cache blocks must be 16-byte aligned");
    if (with_tail) {
        AT_REQUIRE(c->k_tail && c->v_tail && c->k_tail_max && c->v_tail_max, AT_ERR_STATE,
                   "the cache has no tail buffers: it can only be read");
        AT_REQUIRE((((uintptr_t)c->k_tail | (uintptr_t)c->v_tail) & 15) == 0, AT_ERR_INVALID_ARG,
                   "tail buffers must be 16-byte aligned");
    }
    KvbDev d;
    d.hkv = c->n_kv_heads;
    d.hd = c->head_dim;
    d.lb = c->block_tokens == 16 ? 4 : c->block_tokens == 32 ? 5 : c->block_tokens == 64 ? 6 : 7;
    d.n_blocks = c->n_blocks;
    d.max_seqs = c->max_seqs;
    d.max_blocks = c->max_blocks;
    d.k = c->k; d.v = c->v;
    d.ks = c->k_scale; d.vs = c->v_scale;
    d.kt = c->k_tail; d.vt = c->v_tail;
    d.ktm = c->k_tail_max; d.vtm = c->v_tail_max;
    d.table = c->block_table;
    d.status = c->status;
    return d;
}

KvbBatch kvb_batch(const at_kvb* c, const at_token_batch* b) {
    AT_REQUIRE(b, AT_ERR_INVALID_ARG, "null batch");
    AT_REQUIRE(b->n_seqs >= 0 && b->n_tokens >= 0 && b->max_tokens >= 0 && b->max_tokens <= b->n_tokens && b->max_end >= 0,
               AT_ERR_INVALID_ARG, "bad batch sizes");
    AT_REQUIRE(b->n_seqs == 0 || (b->slots && b->starts && b->offsets), AT_ERR_INVALID_ARG, "null batch buffer");
    AT_REQUIRE(b->max_end <= (int64_t)c->max_blocks * c->block_tokens, AT_ERR_STATE,
               "position " + std::to_string(b->max_end) + " is past the cache's " +
                   std::to_string((int64_t)c->max_blocks * c->block_tokens) + " positions per sequence");
    // a run is no longer than a sequence's positions, whatever the host's bound
    const int most = (int)std::min<int64_t>(b->max_tokens, (int64_t)c->max_blocks * c->block_tokens);
    return KvbBatch{b->n_seqs, b->n_tokens, most, b->slots, b->starts, b->offsets};
}

namespace {

constexpr uint32_t F32_INF = 0x7F800000u;

template <class T>
__device__ __forceinline__ void store_raw8(T* __restrict__ p, const Raw8<T>& x) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(x.t)[i];
}
template <class T>
__device__ __forceinline__ void store8(T* __restrict__ p, const float* x) {
    Raw8<T> t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t.t[i] = from_f32<T>(x[i]);
    store_raw8<T>(p, t);
}

// The largest |x| as ordered bits (finite < infinity < NaN), two 16-bit lanes
// at a time for 16-bit types: their magnitudes order like their bits.
template <class T>
__device__ __forceinline__ uint32_t max_bits(const Raw8<T>& x, uint32_t m) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x.t);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    }
    return m;
}
// ... as the bits of an FP32 value.
template <class T>
__device__ __forceinline__ uint32_t max_bits_f32(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
        return m;
    } else {
        const unsigned short h = (unsigned short)max(m & 0xFFFFu, m >> 16);
        return __float_as_uint(to_f32<T>(reinterpret_cast<const T&>(h))) & 0x7FFFFFFFu;
    }
}

// A quant in the low byte, and eight. 1.5 2^23 + x rounds x to the nearest integer (ties to even) in
// the low bits of the sum: its low byte is q in two's complement (one addition
// instead of a conversion, which runs at an eighth of its rate).
__device__ __forceinline__ uint32_t quant1(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
__device__ __forceinline__ uint2 quant8(const float* x, float inv) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = quant1(x[i], inv);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    return make_uint2(w[0], w[1]);
}

// Whether a row of the ring is what its row of the page was quantized from
// (warp-uniform). A poisoned block, whose scale is NaN, cannot be told.
template <class T, int HD>
__device__ __forceinline__ bool tail_intact(const int8_t* page_row, const T* tail_row, float row_max, float held) {
    constexpr int E = HD / 32;  // elements per lane
    const int col = E * (threadIdx.x & 31);
    const float inv = held > 0.f ? __fdiv_rn(1.f, held) : 0.f, d = __fdiv_rn(row_max, 127.f);
    bool differs = !((d < 0x1p-126f ? 0.f : d) <= held);
#pragma unroll
    for (int i = 0; i < E; ++i) differs |= (int8_t)quant1(to_f32<T>(tail_row[col + i]), inv) != page_row[col + i];
    return held != held || !__any_sync(0xffffffffu, differs);
}

template <class T>
struct AppendSrc {
    const T* x;
    int64_t ts, hs;  // token and head strides, elements
    bool vec;
};

// One CTA: one touched block of one sequence and KV head, of K or of V. The
// block's new rows stay in registers (NCH chunks of 8 values per thread)
// between the maximum and the quantization, so every value is read once. NT
// threads: 256 for whole blocks, one warp (its barriers wait for no other) for
// a few tokens. 8 BF16 prompts up to 8191 tokens, 8 heads of 128, written and
// read back: 120 us, 5.2 TB/s over both kernels; the write is bound by its
// instructions (packed maxima, products and roundings fill 86 % of the issue
// slots), not by memory. K and V of a block in one CTA spill: 125 us. One token
// of one sequence, written and read back: 5.1 us, 0.4 of it the look at the
// tail (held in eight values per lane that look took 57 registers for 48, a
// CTA per SM, and 5 us of the prompts; a row spread over the warp takes none).
template <class T, int HD, int NT, int NCH>
__global__ void __launch_bounds__(NT) kvb_append_kernel(KvbDev c, KvbBatch b, AppendSrc<T> sk, AppendSrc<T> sv, int max_touched) {
    constexpr int CPR = HD / 8;  // chunks per row: a row's chunks are neighbouring lanes
    __shared__ uint32_t s_max[NT / 32];
    const int tid = threadIdx.x;
    const bool is_v = blockIdx.y & 1;
    const int h = blockIdx.y >> 1, s = blockIdx.x / max_touched, j = blockIdx.x - s * max_touched;
    const KvbSeq q = kvb_seq(c, b, s);
    const int B = 1 << c.lb;
    const int start = (int)q.start, end = start + q.n;
    const int first = start >> c.lb, blk = first + j, base = blk << c.lb;
    if (q.n == 0 || base >= end) return;
    const AppendSrc<T> src = is_v ? sv : sk;
    const T* x0 = src.x + (int64_t)q.off * src.ts + (int64_t)h * src.hs;
    const int lo = max(start, base), hi = min(end, base + B);
    // the source's rows first: they do not wait for the page
    Raw8<T> x[NCH];
    const int r0 = tid / CPR, col = 8 * (tid % CPR);  // chunk i of this thread: row r0 + i NT / CPR
    const int rows = hi - lo - r0;                    // chunk i exists when i NT / CPR < rows
    {
        const T* xp = x0 + (int64_t)(lo - start + r0) * src.ts + col;
        const int64_t step = src.ts * (NT / CPR);
#pragma unroll
        for (int i = 0; i < NCH; ++i, xp += step)
            if (i * (NT / CPR) < rows) load_raw8<T>(xp, src.vec, x[i]);
    }
    const int page = kvb_page(c, q.slot, blk);
    if (page < 0) return;
    const size_t row0 = ((size_t)page * c.hkv + h) << c.lb;
    int8_t* dst = (is_v ? c.v : c.k) + row0 * HD;
    float* scale = (is_v ? c.vs : c.ks) + (size_t)page * c.hkv + h;
    const float held = *scale;  // the scale of the block's older rows
    const size_t ring0 = ((size_t)q.slot * c.hkv + h) << (c.lb + 1);
    T* tail = static_cast<T*>(is_v ? c.vt : c.kt) + ring0 * HD;
    float* tail_max = (is_v ? c.vtm : c.ktm) + ring0;
    const int last = (end - 1) >> c.lb;
    const int ring_mask = 2 * B - 1;
    // An append inside a block needs the block's older rows in the ring. Every
    // warp looks for itself, before the CTA writes anything: all leave together.
    if (lo > base) {
        const int p = (lo - 1) & ring_mask;
        if (!tail_intact<T, HD>(dst + (size_t)(lo - 1 - base) * HD, tail + (size_t)p * HD, tail_max[p], held)) {
            if (tid == 0) kvb_flag(c.status, KVB_STALE_TAIL);
            return;
        }
    }
    // The rows of blocks last - 1 and last go to the ring. If this append
    // begins inside a block and another block of the same parity is kept, the
    // ring rows that the first block still reads are the ones that block
    // overwrites: then the first block's CTA copies them, after its reads.
    const bool open = start > (first << c.lb);
    const int clash = (open && last >= first + 2) ? last - ((last - first) & 1) : -1;
    const bool keep = blk >= last - 1 && blk != clash;

    uint32_t m16 = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * (NT / CPR) < rows) m16 = max_bits<T>(x[i], m16);
    uint32_t m = max_bits_f32<T>(m16);
    for (int r = base + tid; r < lo; r += NT) m = max(m, __float_as_uint(tail_max[r & ring_mask]) & 0x7FFFFFFFu);
    if (keep) {  // CTA-uniform
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const bool live = i * (NT / CPR) < rows;
            const int p = (lo + r0 + i * (NT / CPR)) & ring_mask;
            uint32_t rm = live ? max_bits_f32<T>(max_bits<T>(x[i], 0u)) : 0u;
#pragma unroll
            for (int o = CPR >> 1; o > 0; o >>= 1) rm = max(rm, __shfl_xor_sync(0xffffffffu, rm, o));
            if (live) {
                store_raw8<T>(tail + (size_t)p * HD + col, x[i]);
                if (col == 0) tail_max[p] = __uint_as_float(rm);
            }
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (NT > 32) {
        if ((tid & 31) == 0) s_max[tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) m = max(m, s_max[i]);
    }
    float d = __fdiv_rn(__uint_as_float(m), 127.f), inv = 0.f;
    const bool poison = m >= F32_INF;
    if (poison) d = __uint_as_float(0x7FC00000u);
    else if (d < 0x1p-126f) d = 0.f;
    else inv = __fdiv_rn(1.f, d);
    int8_t* dp = dst + (lo - base + r0) * HD + col;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * (NT / CPR) < rows) {
            float f[8];
            to_f32x8<T>(x[i], f);
            *reinterpret_cast<uint2*>(dp + i * (NT / CPR) * HD) = poison ? make_uint2(0u, 0u) : quant8(f, inv);
        }
    if (__float_as_uint(held) != __float_as_uint(d)) {
        for (int p = base + r0; p < lo; p += NT / CPR) {
            float y[8];
            load8<T>(tail + (size_t)(p & ring_mask) * HD + col, true, y);
            *reinterpret_cast<uint2*>(dst + (size_t)(p - base) * HD + col) = poison ? make_uint2(0u, 0u) : quant8(y, inv);
        }
        if (tid == 0) *scale = d;
    }
    if (j == 0 && clash >= 0) {
        __syncthreads();  // every read of the ring rows is done
        const int cb = clash << c.lb, n = min(end, cb + B) - cb;
        for (int r = r0; r < B; r += NT / CPR) {  // whole warps: B is a multiple of the rows per pass, or all lanes leave together
            uint32_t rm = 0;
            if (r < n) {
                Raw8<T> y;
                load_raw8<T>(x0 + (int64_t)(cb + r - start) * src.ts + col, src.vec, y);
                rm = max_bits_f32<T>(max_bits<T>(y, 0u));
                store_raw8<T>(tail + (size_t)((cb + r) & ring_mask) * HD + col, y);
            }
#pragma unroll
            for (int o = CPR >> 1; o > 0; o >>= 1) rm = max(rm, __shfl_xor_sync(0xffffffffu, rm, o));
            if (r < n && col == 0) tail_max[(cb + r) & ring_mask] = __uint_as_float(rm);
        }
    }
}

constexpr int READ_THREADS = 256;
constexpr int READ_TOKENS = 64;  // positions per CTA

// A CTA reads READ_TOKENS positions of one KV head, K or V, and writes them
// token-major: 8 values per thread and row, all of its loads in flight at once.
// Bound by memory traffic: 131071 tokens of 8 heads of 128 as F16: 135 us, 5.9
// TB/s; 2048 tokens of 8 heads of 64 as FP32: 5.4 us.
template <class T, int HD>
__global__ void __launch_bounds__(READ_THREADS) kvb_read_kernel(KvbDev c, KvbBatch b, T* __restrict__ ok, T* __restrict__ ov,
                                                                int chunks) {
    constexpr int CPR = HD / 8, ROWS = READ_THREADS / CPR, U = READ_TOKENS / ROWS;
    const bool is_v = ok ? (ov ? blockIdx.y & 1 : false) : true;
    const int h = ok && ov ? blockIdx.y >> 1 : blockIdx.y;
    const int s = blockIdx.x / chunks, i0 = (blockIdx.x - s * chunks) * READ_TOKENS;
    const KvbSeq q = kvb_seq(c, b, s);
    const int n = min(READ_TOKENS, q.n - i0);
    if (n <= 0) return;
    const int8_t* src = is_v ? c.v : c.k;
    const float* sc = is_v ? c.vs : c.ks;
    T* out = (is_v ? ov : ok) + ((size_t)(q.off + i0) * c.hkv + h) * HD;
    const int r0 = threadIdx.x / CPR, col = 8 * (threadIdx.x % CPR), mask = (1 << c.lb) - 1;
    uint2 x[U];
    float d[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int r = r0 + i * ROWS;
        x[i] = make_uint2(0u, 0u);
        d[i] = 0.f;
        if (r < n) {
            const int p = (int)q.start + i0 + r;
            const int page = kvb_page(c, q.slot, p >> c.lb);
            const size_t ph = (size_t)max(page, 0) * c.hkv + h;
            d[i] = page < 0 ? __uint_as_float(0x7FC00000u) : sc[ph];
            x[i] = *reinterpret_cast<const uint2*>(src + ((ph << c.lb) + (p & mask)) * HD + col);
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int r = r0 + i * ROWS;
        if (r >= n) break;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t w = e < 4 ? x[i].x : x[i].y;
            y[e] = __fmul_rn(magic_byte(w ^ 0x80808080u, e & 3) - 8388736.f, d[i]);  // 2^23 + 128 + q, exact
        }
        store8<T>(out + (size_t)r * c.hkv * HD + col, y);
    }
}

template <class T, int HD>
void launch_append(const KvbDev& c, const KvbBatch& b, const AppendSrc<T>& k, const AppendSrc<T>& v, cudaStream_t s) {
    const int B = 1 << c.lb;
    const int touched = (int)(((int64_t)b.max_tokens + B - 2) / B) + 1;
    AT_REQUIRE((int64_t)b.n_seqs * touched <= INT32_MAX && c.hkv <= 32767, AT_ERR_INVALID_ARG, "the batch is too large for one append");
    const dim3 grid(b.n_seqs * touched, 2 * c.hkv);
    const int few = std::min(b.max_tokens, B) * (HD / 8);  // chunks of a sequence's new rows in one block at most
    if (few <= 32) kvb_append_kernel<T, HD, 32, 1><<<grid, 32, 0, s>>>(c, b, k, v, touched);
    else if (few <= 128) kvb_append_kernel<T, HD, 32, 4><<<grid, 32, 0, s>>>(c, b, k, v, touched);
    else {
        switch (B * HD / 8 / 256) {
            case 8: kvb_append_kernel<T, HD, 256, 8><<<grid, 256, 0, s>>>(c, b, k, v, touched); break;
            case 4: kvb_append_kernel<T, HD, 256, 4><<<grid, 256, 0, s>>>(c, b, k, v, touched); break;
            case 2: kvb_append_kernel<T, HD, 256, 2><<<grid, 256, 0, s>>>(c, b, k, v, touched); break;
            default: kvb_append_kernel<T, HD, 256, 1><<<grid, 256, 0, s>>>(c, b, k, v, touched); break;
        }
    }
    AT_CUDA(cudaGetLastError());
}

template <class T>
AppendSrc<T> append_src(const void* x, int64_t ts, int64_t hs) {
    return AppendSrc<T>{static_cast<const T*>(x), ts, hs, aligned_rows(x, (int)sizeof(T), ts, hs)};
}

}  // namespace

}  // namespace at

using namespace at;

extern "C" {

int at_kvb_append(at_ctx* ctx, const at_kvb* cache, const at_token_batch* batch, const void* k, int64_t k_token_stride,
                  int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride) {
    return guard([&] {
        const KvbDev c = kvb_dev(ctx, cache, true);
        const KvbBatch b = kvb_batch(cache, batch);
        if (b.n_seqs == 0 || b.max_tokens == 0) return;
        AT_REQUIRE(k && v, AT_ERR_INVALID_ARG, "null K or V");
        const uintptr_t e = kvb_elem_bytes(cache->dtype);
        AT_REQUIRE((((uintptr_t)k | (uintptr_t)v) & (e - 1)) == 0, AT_ERR_INVALID_ARG, "K and V must be aligned to their elements");
        AT_CUDA(cudaSetDevice(ctx->device));
        kvb_dispatch(cache->dtype, [&](auto t) {
            using T = decltype(t);
            const AppendSrc<T> sk = append_src<T>(k, k_token_stride, k_head_stride), sv = append_src<T>(v, v_token_stride, v_head_stride);
            if (c.hd == 128) launch_append<T, 128>(c, b, sk, sv, ctx->stream);
            else launch_append<T, 64>(c, b, sk, sv, ctx->stream);
        });
    });
}

int at_kvb_read(at_ctx* ctx, const at_kvb* cache, const at_token_batch* batch, int out_type, void* k_out, void* v_out) {
    return guard([&] {
        const KvbDev c = kvb_dev(ctx, cache, false);
        const KvbBatch b = kvb_batch(cache, batch);
        AT_REQUIRE(out_type == AT_GGML_F32 || out_type == AT_GGML_F16 || out_type == AT_GGML_BF16, AT_ERR_UNSUPPORTED,
                   "output type must be F32, F16 or BF16");
        if (b.n_seqs == 0 || b.max_tokens == 0) return;
        AT_REQUIRE(k_out || v_out, AT_ERR_INVALID_ARG, "null outputs");
        AT_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, AT_ERR_INVALID_ARG, "outputs must be 16-byte aligned");
        const int chunks = (int)(((int64_t)b.max_tokens + READ_TOKENS - 1) / READ_TOKENS);
        AT_REQUIRE((int64_t)b.n_seqs * chunks <= INT32_MAX && c.hkv <= 32767, AT_ERR_INVALID_ARG, "the batch is too large for one read");
        const dim3 grid(b.n_seqs * chunks, c.hkv * (k_out && v_out ? 2 : 1));
        AT_CUDA(cudaSetDevice(ctx->device));
        kvb_dispatch(out_type, [&](auto t) {
            using T = decltype(t);
            auto kern = c.hd == 128 ? kvb_read_kernel<T, 128> : kvb_read_kernel<T, 64>;
            kern<<<grid, READ_THREADS, 0, ctx->stream>>>(c, b, static_cast<T*>(k_out), static_cast<T*>(v_out), chunks);
        });
        AT_CUDA(cudaGetLastError());
    });
}

}  // extern "C"
