// Attention over the block-quantized KV cache (kvblock.cu).
//
// The query at position p of a sequence sees the keys j <= p (and
// j > p - window when a window is set):
//   s_j = scale * d_k(j) * sum_c q_c k8_jc,   out = sum_j e^(s_j - m) d_v(j) v8_j / sum_j e^(s_j - m)
// with m the running maximum; statistics and sums in FP32. A hidden key is
// left out by its index, so what its bytes or scale hold never matters; a
// visible key of a poisoned block (scale NaN) makes the row NaN.
#include <algorithm>
#include <cstdint>
#include <string>

#include <cooperative_groups.h>

#include "kvblock.cuh"
#include "kvblock_attn.cuh"

namespace at {

namespace {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------
// Few query rows per KV head (decode steps, drafted tokens)
// ---------------------------------------------------------------------------
// Rows r = token * G + query head of one (sequence, KV head) form the N side
// (8 per tile, NT tiles) of mma.sync m16n8k16 (f16 operands, FP32 sums); keys
// are the M side of S^T = K Q^T, head dimensions the M side of O^T = V^T P^T.
// Both A operands are built in registers from the int8 bytes as they come
// from memory, exact in f16 (|q| <= 127), so K and V cross shared memory
// nowhere: a warp's unit is 32 or 64 keys, 16-byte loads straight into the
// lanes that multiply them. A byte q becomes 1024 + 128 + q by one masked xor and
// loses the offset in one packed subtraction; for F16/BF16 queries K skips the
// subtraction: its f16 bits are q + 128 alone, a subnormal worth
// (q + 128) 2^-24, and 128 sum(q_c) leaves the finished dot product (the
// offset is 3 to 4 times the dot's own size, which costs FP32 sums two bits). Which key or dimension a lane's bytes are is free, as
// long as both operands agree, and is chosen so that
//   K: lane (g, t) holds 16-byte chunks of key rows 4 J (g / 2) + 4 j + (g & 1), + 2;
//   V: lane (g, t) holds HD / 8 bytes of keys 4 J t + 4 j .. + 3 (J 16-key tiles per unit);
//   the S^T accumulators, packed to f16 pairs and transposed by movmatrix,
//   are the P^T operand.
// tcgen05 would want the converted tiles in shared memory and 128 rows; here
// there are 8 or 16 and the time goes to the K and V bytes.
// FP32 queries are split into two f16 parts (22 bits), and so are the weights;
// F16/BF16 queries are exact in one (each row is scaled by a power of two
// into f16's range) and their weights are rounded once to 11 bits. The values'
// scale is part of the weights' exponent: with t_j = s_j + log2 d_v(j) and m
// their running maximum, P_j = 2^(t_j - m + 12) fills f16's range whatever the
// blocks' scales are (value_scale says how far apart they may lie), and weights down to 2^-26 of the largest keep its full
// precision; out = sum P_j v8_j / sum P_j / d_v(j).
//
// 64 sequences of 4096 to 8191 tokens, 64 BF16 heads over 8 of 128: 149 us, 5.3
// TB/s of K and V, four fifths of a copy's rate: half of the issue slots and
// 58 % of the integer pipe go to turning bytes into f16, with 12 warps per SM
// to cover the loads. (K Q^T on the int8 form of mma.sync, with no work per key
// byte: 142 us with queries as two int8 parts, which lose what is small beside
// a row's largest value; 148 us with three, which do not.) In FP32, with twice
// the products and registers spilled (below): 229 us. One sequence of 131072
// tokens over 8 heads of 64: 39 us, 3.4 TB/s; of 513 tokens: 7.6 us, the time
// of its launch and of three loads one after another.
constexpr int ST_WARPS = 4;
constexpr int ST_THREADS = 32 * ST_WARPS;
constexpr float ST_ROOM = 12.f;
// Keys of a warp's unit: 8 KB of K and V each at a time. At head_dim 128 a
// unit of 64 keys needs 252 registers and leaves two warps per scheduler to
// cover each other's latencies (64 sequences up to 8191 tokens: 163 us); with
// 16-bit queries 32 keys fit 168 registers and three (149 us). FP32 queries do
// not fit either: 180 bytes are spilled and 108 loaded again per thread with 8
// rows, 256 and 212 of 255 registers with 16 (229 us).
constexpr int st_unit(int hd) { return hd == 128 ? 32 : 64; }

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int N>
struct Bytes;
template <>
struct Bytes<16> { uint32_t w[4]; };
template <>
struct Bytes<8> { uint32_t w[2]; };
__device__ __forceinline__ void ld_bytes(Bytes<16>& b, const int8_t* p) {
    const uint4 v = ld_stream_u4(p);
    b.w[0] = v.x; b.w[1] = v.y; b.w[2] = v.z; b.w[3] = v.w;
}
__device__ __forceinline__ void ld_bytes(Bytes<8>& b, const int8_t* p) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(b.w[0]), "=r"(b.w[1]) : "l"(p));
}

struct StepParams {
    KvbDev c;
    KvbBatch b;
    const void* q;
    int64_t q_ts, q_hs;
    void* out;
    int H, G, groups, splits, window, max_rows;  // groups: row groups of 8 NT; sequences above max_rows rows are skipped
    int q_vec;                                   // q rows are 16-byte aligned
    int single;                                  // one token per sequence: row r is query head r
    int cluster;                                 // the splits of an item are one cluster
    float scale;
    float* part_o;   // [item][split][8 NT][HD]
    float2* part_ml; // [item][split][8 NT]
};

// Four outputs of a row: o / l (0 for a row that saw no key).
template <class T>
__device__ __forceinline__ void store_row4(T* out, float4 o, float l) {
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
    alignas(16) T y[4] = {from_f32<T>(o.x * inv), from_f32<T>(o.y * inv), from_f32<T>(o.z * inv), from_f32<T>(o.w * inv)};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(y);
    else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(y);
}

template <class T, int HD, int NT>
__global__ void __launch_bounds__(ST_THREADS, NT == 1 ? 3 : 2) kvb_attn_step_kernel(const StepParams p) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    constexpr bool BIASED = TERMS == 1;
    constexpr int KS = HD / 16;    // k-steps of K Q^T
    constexpr int KC = HD / 64;    // 16-byte chunks of a key row per lane
    constexpr int MT = HD / 16;    // M tiles of V^T P^T
    constexpr int VB = HD / 8;     // bytes of a value row per lane
    constexpr int ROWS = 8 * NT;
    constexpr int UNIT = st_unit(HD), J = UNIT / 16, SUB = 4 * J;  // SUB consecutive keys share a lane's page
    const KvbDev& c = p.c;
    __shared__ float s_ml[ST_WARPS][ROWS][2], s_w[ST_WARPS][ROWS], s_lt[ROWS], s_mx[ROWS];
    __shared__ float s_o[ST_WARPS][ROWS][HD];
    if (!p.cluster) pdl_trigger();  // the join may be launched; it waits for this kernel
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, s = blockIdx.z, kvh = p.groups == 1 ? blockIdx.y : blockIdx.y / p.groups, rg = blockIdx.y - kvh * p.groups;
    const int item = s * gridDim.y + blockIdx.y;
    auto token_of = [&](int r) { return p.single ? 0 : r / p.G; };
    const KvbSeq sq = kvb_seq(c, p.b, s);
    const int R = sq.n * p.G, r0 = rg * ROWS;
    if (r0 >= R || R > p.max_rows) return;
    const int start = (int)sq.start;
    const int first_pos = start + token_of(r0), last_pos = start + token_of(min(R, r0 + ROWS) - 1);
    const int lo = p.window > 0 ? max(0, first_pos - p.window + 1) : 0, hi = last_pos + 1;
    const int u_lo = lo / UNIT, nu = (hi - 1) / UNIT + 1 - u_lo;
    const int share = nu / p.splits, more = nu - share * p.splits;  // the first `more` splits have one unit more
    const int u0 = u_lo + share * split + min(split, more), u1 = u0 + share + (split < more);

    // queries: row g of each tile, 4 dims per k-step
    uint32_t qf[NT][TERMS][KS][2];
    float qs[NT][2];  // score factors of rows 2 t, 2 t + 1 (log2 units)
    float qb[NT][2];  // 128 sum(q_c) of the same rows (the K offset)
    int qp[NT][2];    // their positions (padding rows: -1, they see nothing)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + 8 * nt + g;
        float x[KC][16];
        float top = 0.f;
        if (r < R) {
            const int tok = token_of(r);
            const T* row = static_cast<const T*>(p.q) + (int64_t)(sq.off + tok) * p.q_ts + (int64_t)(kvh * p.G + r - tok * p.G) * p.q_hs + 16 * t;
#pragma unroll
            for (int cc = 0; cc < KC; ++cc) {
                load8<T>(row + 64 * cc, p.q_vec, x[cc]);
                load8<T>(row + 64 * cc + 8, p.q_vec, x[cc] + 8);
            }
        } else {
#pragma unroll
            for (int cc = 0; cc < KC; ++cc)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[cc][i] = 0.f;
        }
#pragma unroll
        for (int cc = 0; cc < KC; ++cc)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[cc][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float rs = row_scale(top);
        float sum = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float a0 = x[kk >> 2][4 * (kk & 3) + b] * rs, a1 = x[kk >> 2][4 * (kk & 3) + b + 2] * rs;
                const uint32_t hi2 = pack_h2(a0, a1);
                const float2 h = unpack_h2(hi2);
                qf[nt][0][kk][b] = hi2;
                sum += h.x + h.y;
                if constexpr (TERMS == 2) qf[nt][1][kk][b] = pack_h2(a0 - h.x, a1 - h.y);
            }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float f = p.scale * 1.44269504088896341f / rs;  // exact division: rs is a power of two
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            qs[nt][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
            qb[nt][e] = 128.f * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
            const int rr = r0 + 8 * nt + 2 * t + e;
            qp[nt][e] = rr < R ? start + token_of(rr) : -1;
        }
    }

    float o[NT][MT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }

    // page of this lane's sub-block t of a unit (-2: past the last key, -1: outside the pool)
    auto lookup = [&](int u) { return (u < u1 && u * UNIT + SUB * t < hi) ? kvb_page(c, sq.slot, (u * UNIT + SUB * t) >> c.lb) : -2; };
    const int bmask = (1 << c.lb) - 1;
    auto load_k = [&](Bytes<16> (&kr)[J][2][KC], int u, int pk) {  // pk: page of sub-block g / 2
        const int8_t* base = c.k + ((((size_t)max(pk, 0) * c.hkv + kvh) << c.lb) + ((u * UNIT + SUB * (g >> 1)) & bmask)) * HD + 16 * t;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int cc = 0; cc < KC; ++cc) ld_bytes(kr[j][e][cc], base + (4 * j + (g & 1) + 2 * e) * HD + 64 * cc);
    };
    auto load_d = [&](int pk, float* dk, float* dv) {
        const size_t i = (size_t)max(pk, 0) * c.hkv + kvh;
        *dk = pk == -1 ? __uint_as_float(0x7FC00000u) : pk < 0 ? 0.f : c.ks[i];
        *dv = pk == -1 ? __uint_as_float(0x7FC00000u) : pk < 0 ? 0.f : c.vs[i];
    };

    int u = u0 + warp;
    int pv = lookup(u), pv_next = lookup(u + ST_WARPS);
    Bytes<16> kr[J][2][KC];
    float dk, dv;
    {
        const int pk = __shfl_sync(0xffffffffu, pv, g >> 1);
        load_k(kr, u, pk);
        load_d(pk, &dk, &dv);
    }
    for (; u < u1; u += ST_WARPS) {
        // the values' bytes are asked for before the keys are multiplied
        Bytes<VB> vr[J][4];
        {
            const int8_t* base = c.v + ((((size_t)max(pv, 0) * c.hkv + kvh) << c.lb) + ((u * UNIT + SUB * t) & bmask)) * HD + VB * g;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) ld_bytes(vr[j][e], base + (4 * j + e) * HD);
        }
        float sc[J][NT][4];
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[j][nt][0] = sc[j][nt][1] = sc[j][nt][2] = sc[j][nt][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const uint32_t w0 = kr[j][0][kk >> 2].w[kk & 3], w1 = kr[j][1][kk >> 2].w[kk & 3];
                const uint32_t a0 = bytes_h2<BIASED>(w0, false), a1 = bytes_h2<BIASED>(w1, false);
                const uint32_t a2 = bytes_h2<BIASED>(w0, true), a3 = bytes_h2<BIASED>(w1, true);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) mma16816(sc[j][nt], a0, a1, a2, a3, qf[nt][e][kk][0], qf[nt][e][kk][1]);
            }
        }
        // the next unit's keys and scales, and the pages of the one after it
        const float dk_u = dk, dv_u = dv;
        pv = pv_next;
        if (u + ST_WARPS < u1) {
            const int pk = __shfl_sync(0xffffffffu, pv_next, g >> 1);
            load_k(kr, u + ST_WARPS, pk);
            load_d(pk, &dk, &dv);
            pv_next = lookup(u + 2 * ST_WARPS);
        }
        // softmax: lane (g, t) has keys base + 4 j + 2 e of rows 2 t, 2 t + 1
        const int kbase = u * UNIT + SUB * (g >> 1) + (g & 1);
        const bool whole = u * UNIT + UNIT - 1 <= first_pos && (p.window <= 0 || u * UNIT > last_pos - p.window);
        float lv, iv, mv;
        value_scale<!BIASED>(dv_u, &lv, &iv, &mv);
        [[maybe_unused]] bool moved = false;
        float alpha[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float f0 = dk_u * qs[nt][q], f = BIASED ? f0 * 0x1p24f : f0, off = BIASED ? -qb[nt][q] * f0 : 0.f;
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sc[j][nt][2 * e + q] = fmaf(sc[j][nt][2 * e + q], f, off);
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = kbase + 4 * j + 2 * e;
                            if (key > qp[nt][q] || (p.window > 0 && key <= qp[nt][q] - p.window)) sc[j][nt][2 * e + q] = -INFINITY;
                        }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < J; ++j) mx = fmaxf(mx, fmaxf(sc[j][nt][q], sc[j][nt][2 + q]));
                mx += lv;
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[nt][q], mx);
                const float a = mn == m[nt][q] ? 1.f : ex2(m[nt][q] - mn);
                m[nt][q] = mn;
                l[nt][q] *= a;
                alpha[nt][q] = a;
                moved |= a != 1.f;
                const float sub = mn == -INFINITY ? 0.f : mn - ST_ROOM - lv;
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sc[j][nt][2 * e + q] = ex2(sc[j][nt][2 * e + q] - sub);
                auto hide = [&] {  // a hidden key has no weight whatever its block's scales hold (0 NaN is NaN)
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = kbase + 4 * j + 2 * e;
                            if (key > qp[nt][q] || (p.window > 0 && key <= qp[nt][q] - p.window)) sc[j][nt][2 * e + q] = 0.f;
                        }
                };
                if (!whole) hide();
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < J; ++j) sum += sc[j][nt][q] + sc[j][nt][2 + q];
                if (sum != 0.f) l[nt][q] = fmaf(sum, iv, l[nt][q]);
                if constexpr (!BIASED) {
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) sc[j][nt][2 * e + q] *= mv;
                    if (!whole) hide();
                }
            }
        // O^T = O^T alpha + V^T P^T. The tensor cores truncate what they
        // accumulate: each product in a chain loses some 10^-8 of the sum. FP32
        // queries therefore start each unit's product from zero and add it in
        // FP32 (150 sequences of 8000 tokens: 0.7e-6 off instead of 3.5e-6). The
        // 2000 products of a 16-bit warp over 131072 keys lose 2e-5, a tenth of
        // what rounding to F16 does, and the additions would cost an eighth of
        // the time (169 us instead of 149).
        if constexpr (TERMS == 2) {
            uint32_t pf[J][NT][TERMS][2];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float a = sc[j][nt][2 * e], b = sc[j][nt][2 * e + 1];
                        const uint32_t h = pack_h2(a, b);
                        const float2 f = unpack_h2(h);
                        pf[j][nt][0][e] = transpose8(h);
                        pf[j][nt][1][e] = transpose8(pack_h2(a - f.x, b - f.y));
                    }
#pragma unroll
            for (int w = 0; w < VB / 4; ++w)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {  // dims 4 w + 2 hf, + 1 of the lane's VB
                    float part[NT][4] = {};
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const uint32_t k01 = __byte_perm(vr[j][0].w[w], vr[j][1].w[w], hf ? 0x7632 : 0x5410);
                        const uint32_t k23 = __byte_perm(vr[j][2].w[w], vr[j][3].w[w], hf ? 0x7632 : 0x5410);
                        const uint32_t a0 = bytes_h2<false>(k01, false), a1 = bytes_h2<false>(k01, true);
                        const uint32_t a2 = bytes_h2<false>(k23, false), a3 = bytes_h2<false>(k23, true);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = TERMS - 1; e >= 0; --e) mma16816(part[nt], a0, a1, a2, a3, pf[j][nt][e][0], pf[j][nt][e][1]);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float* y = o[nt][2 * w + hf];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], alpha[nt][e & 1], part[nt][e]);
                    }
                }
        } else {
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[nt][i][0] *= alpha[nt][0];
                        o[nt][i][1] *= alpha[nt][1];
                        o[nt][i][2] *= alpha[nt][0];
                        o[nt][i][3] *= alpha[nt][1];
                    }
            }
            // O^T += V^T P^T
#pragma unroll
            for (int j = 0; j < J; ++j) {
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        pf[nt][e] = transpose8(pack_h2(sc[j][nt][2 * e], sc[j][nt][2 * e + 1]));
#pragma unroll
                for (int w = 0; w < VB / 4; ++w) {
                    uint32_t x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = vr[j][e].w[w];
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {  // dims 4 w + 2 hf, + 1 of the lane's VB
                        const uint32_t k01 = __byte_perm(x[0], x[1], hf ? 0x7632 : 0x5410), k23 = __byte_perm(x[2], x[3], hf ? 0x7632 : 0x5410);
                        const uint32_t a0 = bytes_h2<false>(k01, false), a1 = bytes_h2<false>(k01, true);
                        const uint32_t a2 = bytes_h2<false>(k23, false), a3 = bytes_h2<false>(k23, true);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * w + hf], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                    }
                }
            }
        }
    }

    // join the warps (in order), then write the row or the split's part
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float x = l[nt][q];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int row = 8 * nt + 2 * t + q;
            if (g == 0) {
                s_ml[warp][row][0] = m[nt][q];
                s_ml[warp][row][1] = x;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                s_o[warp][row][VB * g + 2 * i] = o[nt][i][q];
                s_o[warp][row][VB * g + 2 * i + 1] = o[nt][i][2 + q];
            }
        }
    __syncthreads();
    if (threadIdx.x < ROWS) {
        const int row = threadIdx.x;
        float mx = -INFINITY, lt = 0.f;
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) mx = fmaxf(mx, s_ml[w][row][0]);
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) {
            const float lw = s_ml[w][row][1], a = s_ml[w][row][0] == mx ? 1.f : ex2(s_ml[w][row][0] - mx);
            s_w[w][row] = lw == 0.f ? 0.f : a;  // 0: this warp saw no key of the row
            if (lw != 0.f) lt = fmaf(lw, a, lt);
        }
        s_lt[row] = lt;
        s_mx[row] = mx;
    }
    __syncthreads();
    const int rows = min(ROWS, R - r0);
    auto out_row = [&](int row) {
        const int r = r0 + row, tok = token_of(r);
        return static_cast<T*>(p.out) + ((size_t)(sq.off + tok) * p.H + kvh * p.G + r - tok * p.G) * HD;
    };
    for (int i = threadIdx.x; i < rows * (HD / 4); i += ST_THREADS) {
        const int row = i / (HD / 4), d = 4 * (i % (HD / 4));
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < ST_WARPS; ++w) {
            const float a = s_w[w][row];
            if (a == 0.f) continue;
            const float4 x = *reinterpret_cast<const float4*>(&s_o[w][row][d]);
            acc.x = fmaf(x.x, a, acc.x);
            acc.y = fmaf(x.y, a, acc.y);
            acc.z = fmaf(x.z, a, acc.z);
            acc.w = fmaf(x.w, a, acc.w);
        }
        if (p.splits == 1) {
            store_row4<T>(out_row(row) + d, acc, s_lt[row]);
        } else if (p.cluster) {
            *reinterpret_cast<float4*>(&s_o[0][row][d]) = acc;  // this thread alone reads and writes it here
        } else {
            const size_t at = ((size_t)item * p.splits + split) * ROWS + row;
            *reinterpret_cast<float4*>(p.part_o + at * HD + d) = acc;
            if (d == 0) p.part_ml[at] = make_float2(s_mx[row], s_lt[row]);
        }
    }
    if (p.cluster) {
        // the splits meet in distributed shared memory: each CTA joins a share of the outputs, in split order
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int n = rows * (HD / 4), per = (n + p.splits - 1) / p.splits;
        for (int i = split * per + threadIdx.x; i < min(n, (split + 1) * per); i += ST_THREADS) {
            const int row = i / (HD / 4), d = 4 * (i % (HD / 4));
            float m8[8], l8[8];
            float4 x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                m8[k] = -INFINITY;
                l8[k] = 0.f;
                if (k < p.splits) {
                    m8[k] = *cluster.map_shared_rank(&s_mx[row], k);
                    l8[k] = *cluster.map_shared_rank(&s_lt[row], k);
                    x[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(&s_o[0][row][d], k));
                }
            }
            float mx = m8[0], lt = 0.f;
#pragma unroll
            for (int k = 1; k < 8; ++k) mx = fmaxf(mx, m8[k]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k >= p.splits || l8[k] == 0.f) continue;
                const float a = m8[k] == mx ? 1.f : ex2(m8[k] - mx);
                lt = fmaf(l8[k], a, lt);
                acc.x = fmaf(x[k].x, a, acc.x);
                acc.y = fmaf(x[k].y, a, acc.y);
                acc.z = fmaf(x[k].z, a, acc.z);
                acc.w = fmaf(x[k].w, a, acc.w);
            }
            store_row4<T>(out_row(row) + d, acc, lt);
        }
        cluster.sync();  // the others have read this CTA's shared memory
    }
}

// Joins the splits of a row, in split order: HD / 4 threads per row. The
// weights of up to 32 splits are found by the lanes of a warp together.
template <class T, int HD>
__global__ void __launch_bounds__(128) kvb_attn_join_kernel(const StepParams p, int rows, int total) {
    constexpr int TPR = HD / 4;  // threads per row: 16 or 32
    const int lane = threadIdx.x % TPR;
    const uint32_t mask = TPR == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    pdl_wait();
    const int gr = blockIdx.x * (128 / TPR) + threadIdx.x / TPR;
    if (gr >= total) return;
    const int row = gr % rows, item = gr / rows;
    const int rg = item % p.groups, kvh = (item / p.groups) % p.c.hkv, s = item / p.groups / p.c.hkv;
    const KvbSeq sq = kvb_seq(p.c, p.b, s);
    const int R = sq.n * p.G, r = rg * rows + row;
    if (r >= R || R > p.max_rows) return;
    const size_t at = (size_t)item * p.splits * rows + row;
    float mx = -INFINITY;
    for (int i = lane; i < p.splits; i += TPR) mx = fmaxf(mx, p.part_ml[at + (size_t)i * rows].x);
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o, TPR));
    float lt = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < p.splits; i0 += TPR) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (i0 + lane < p.splits) ml = p.part_ml[at + (size_t)(i0 + lane) * rows];
        const float a = ml.y == 0.f ? 0.f : ml.x == mx ? 1.f : ex2(ml.x - mx);
        lt += ml.y == 0.f ? 0.f : ml.y * a;
        const int n = min(TPR, p.splits - i0);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(p.part_o + (at + (size_t)(i0 + i) * rows) * HD + 4 * lane);
            const float w = __shfl_sync(mask, a, i, TPR);
            if (w == 0.f) continue;
            acc.x = fmaf(x.x, w, acc.x);
            acc.y = fmaf(x.y, w, acc.y);
            acc.z = fmaf(x.z, w, acc.z);
            acc.w = fmaf(x.w, w, acc.w);
        }
    }
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) lt += __shfl_xor_sync(mask, lt, o, TPR);
    store_row4<T>(static_cast<T*>(p.out) + ((size_t)(sq.off + r / p.G) * p.H + kvh * p.G + r % p.G) * HD + 4 * lane, acc, lt);
}

struct StepPlan {
    int rows, groups, splits, cluster;
    size_t ml_bytes, bytes;
};

// Splits along the keys. Three CTAs are resident per SM (two for 16 rows).
// Fewer items than that: as many splits as fill the GPU once (more only
// lengthen the join: one sequence of 131072 tokens, 8 KV heads of 64: 39 us
// at 1 wave, 51 at 3). More items: several waves, because sequences differ in
// length (64 sequences of 4096 to 8191 tokens: 187 us at 2 waves, 148 to 156
// from 2.5 to 9, 157 at 16). A split keeps at least one unit per warp.
StepPlan step_plan(const at_ctx* ctx, const KvbDev& c, const KvbBatch& b, int64_t max_end, int n_heads, int window, int max_rows) {
    const int G = n_heads / c.hkv;
    const int most = (int)std::min<int64_t>((int64_t)b.max_tokens * G, max_rows);
    StepPlan s;
    s.rows = most <= 8 ? 8 : 16;
    s.groups = (most + s.rows - 1) / s.rows;
    const int64_t items = (int64_t)b.n_seqs * c.hkv * s.groups;
    int64_t keys = max_end;
    if (window > 0) keys = std::min<int64_t>(keys, (int64_t)window + b.max_tokens + 64);
    const int64_t units = (keys + st_unit(c.hd) - 1) / st_unit(c.hd);
    const int64_t slots = (s.rows == 8 ? 3 : 2) * (int64_t)ctx->num_sms;
    const int64_t want = items >= slots ? (7 * slots / 2 + items - 1) / items : slots / items;
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, (units + ST_WARPS - 1) / ST_WARPS));
    // Up to 8 splits that fit the GPU at once are one thread-block cluster (of
    // 2, 4 or 8 CTAs) and need neither workspace nor a second launch (one
    // sequence of 513 tokens: 3.1 us less). In several waves a cluster's
    // CTAs hold their places until the last is done (64 sequences: 163 us
    // against 149 with the join as a kernel).
    const int pow2 = s.splits <= 2 ? s.splits : s.splits <= 4 ? 4 : 8;
    s.cluster = s.splits > 1 && s.splits <= 8 && items * pow2 <= slots;
    if (s.cluster) s.splits = pow2;
    AT_REQUIRE(b.n_seqs <= 65535 && (int64_t)c.hkv * s.groups <= 65535 && items * s.rows <= INT32_MAX, AT_ERR_INVALID_ARG,
               "the batch is too large for one call");
    const bool parts = s.splits > 1 && !s.cluster;
    s.ml_bytes = parts ? (size_t)items * s.splits * s.rows * sizeof(float2) : 0;
    s.bytes = parts ? s.ml_bytes + (size_t)items * s.splits * s.rows * c.hd * sizeof(float) : 0;
    return s;
}

template <class T, int HD>
void launch_step(const StepParams& p, const StepPlan& s, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    cfg.gridDim = dim3(s.splits, p.c.hkv * s.groups, p.b.n_seqs);
    cfg.blockDim = dim3(ST_THREADS);
    cfg.stream = st;
    cfg.attrs = &attr;
    if (s.cluster) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {(unsigned)s.splits, 1, 1};
        cfg.numAttrs = 1;
    }
    AT_CUDA(s.rows == 8 ? cudaLaunchKernelEx(&cfg, kvb_attn_step_kernel<T, HD, 1>, p) : cudaLaunchKernelEx(&cfg, kvb_attn_step_kernel<T, HD, 2>, p));
    if (s.bytes) {
        const int total = p.b.n_seqs * p.c.hkv * s.groups * s.rows, per = 128 / (HD / 4);
        cfg.gridDim = dim3((total + per - 1) / per);
        cfg.blockDim = dim3(128);
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
        AT_CUDA(cudaLaunchKernelEx(&cfg, kvb_attn_join_kernel<T, HD>, p, s.rows, total));
    }
}

// Rows per KV head up to which the step kernel serves a sequence. It reads and
// converts K and V once per 16 rows, the prompt kernel once per 256 (128 in
// FP32), but only the step kernel splits the keys. 64 BF16 heads over 8 of 128,
// us, step / prompt kernel (FP32 in brackets):
//                              16 rows       32 rows       64 rows
//    1 sequence, 512 tokens    9 / 19        10 / 19       11 / 19
//    1 sequence, 32768        32 / 585       45 / 585      73 / 585   (108 / 639)
//   16 sequences to 4096      41 / 83        71 / 83      129 / 84    (193 / 93)
//   64 sequences to 4096     135 / 261      227 / 250     415 / 268   (648 / 298)
// Up to 64 rows it is at most 2.2 times slower where many sequences fill the
// GPU, and 8 times faster where one has to.
constexpr int STEP_MAX_ROWS = 64;

// The step kernel serves every sequence of at most STEP_MAX_ROWS query rows
// per KV head. The host's sizes are upper bounds, so a run may always be
// shorter than they say; where they leave no room for it (equal prompts) the
// step kernel is left out, and the prompt kernel takes every sequence.
bool uses_step(const KvbBatch& b, int G) {
    return (int64_t)b.max_tokens * G <= STEP_MAX_ROWS || (int64_t)b.n_seqs * b.max_tokens > b.n_tokens;
}

}  // namespace

}  // namespace at

using namespace at;

extern "C" {

int at_kvb_attention_workspace(at_ctx* ctx, const at_kvb* cache, const at_token_batch* batch, int n_heads, int window,
                               size_t* bytes) {
    return guard([&] {
        AT_REQUIRE(ctx && cache && batch, AT_ERR_INVALID_ARG, "null argument");
        AT_REQUIRE(bytes, AT_ERR_INVALID_ARG, "null output");
        const KvbDev c = kvb_dev(ctx, cache, false);
        const KvbBatch b = kvb_batch(cache, batch);
        AT_REQUIRE(n_heads > 0 && n_heads % c.hkv == 0, AT_ERR_INVALID_ARG, "query heads must be a multiple of the KV heads");
        *bytes = 0;
        if (b.n_seqs == 0 || b.max_tokens == 0) return;
        if (uses_step(b, n_heads / c.hkv)) *bytes = step_plan(ctx, c, b, batch->max_end, n_heads, window, STEP_MAX_ROWS).bytes;
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
        AT_REQUIRE(n_heads / c.hkv <= 128, AT_ERR_UNSUPPORTED, "at most 128 query heads per KV head");
        AT_REQUIRE(window >= 0, AT_ERR_INVALID_ARG, "window must not be negative");
        AT_REQUIRE(scale > 0.f && scale < INFINITY, AT_ERR_INVALID_ARG, "scale must be positive and finite");
        if (b.n_seqs == 0 || b.max_tokens == 0) return;
        AT_REQUIRE(q && out, AT_ERR_INVALID_ARG, "null q or out");
        AT_REQUIRE(((uintptr_t)out & 15) == 0 && ((uintptr_t)q & (kvb_elem_bytes(dtype) - 1)) == 0, AT_ERR_INVALID_ARG,
                   "out must be 16-byte aligned, q aligned to its elements");
        AT_CUDA(cudaSetDevice(ctx->device));
        const bool step = uses_step(b, n_heads / c.hkv);
        if (step) {
            const StepPlan s = step_plan(ctx, c, b, batch->max_end, n_heads, window, STEP_MAX_ROWS);
            AT_REQUIRE(workspace_bytes >= s.bytes && (s.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0)), AT_ERR_INVALID_ARG,
                       "attention: the workspace must be 16-byte aligned and hold at_kvb_attention_workspace bytes");
            StepParams p{c, b, q, q_token_stride, q_head_stride, out, n_heads, n_heads / c.hkv, s.groups, s.splits, window, STEP_MAX_ROWS, 0, b.max_tokens == 1, s.cluster, scale,
                         reinterpret_cast<float*>(static_cast<char*>(workspace) + s.ml_bytes), static_cast<float2*>(workspace)};
            p.q_vec = aligned_rows(q, kvb_elem_bytes(dtype), q_token_stride, q_head_stride);
            kvb_dispatch(dtype, [&](auto t) {
                using T = decltype(t);
                if (c.hd == 128) launch_step<T, 128>(p, s, ctx->stream);
                else launch_step<T, 64>(p, s, ctx->stream);
            });
        }
        if ((int64_t)b.max_tokens * (n_heads / c.hkv) > STEP_MAX_ROWS)
            launch_kvb_attn_prompt(c, b, dtype, n_heads, q, q_token_stride, q_head_stride, out, scale, window, step ? STEP_MAX_ROWS : 0,
                                   ctx->stream);
    });
}

}  // extern "C"
