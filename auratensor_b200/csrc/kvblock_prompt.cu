// Attention over the block-quantized KV cache for many query rows (prompts)
// on the 5th-generation tensor cores.
//
// A CTA holds NQ tiles of 128 query rows of one (sequence, KV head): the
// tokens of consecutive query blocks times the G heads of the KV head, so
// every K and V byte is read and converted once for all of them. The keys
// are walked in tiles of 128:
//   warps 8..11 (producers) bring a tile's int8 K and V rows from their pages
//     into registers, turn them into f16 (exact, |q| <= 127) and store them
//     into a two-stage ring: K K-major, V MN-major, 128-byte swizzle;
//   warp 12 (one thread) issues S = Q K^T into TMEM, and O += P V with P read
//     from TMEM; with two query tiles one's products run under the other's
//     softmax;
//   warps 0..3 and 4..7 (one thread per query row) run the online softmax of
//     their tile: S from TMEM, P back over S's own columns as packed f16.
// Arithmetic, per row, in log2 units: t_j = s_j + log2 d_v(j), P_j = 2^(t_j - r)
// with a reference r that follows the row's largest t; out = sum P_j v8_j /
// sum P_j / d_v(j). The values' scale is part of the exponent, so P fills
// f16's range whatever the blocks' scales are, and costs no product; FP32
// queries keep log2 d_v to its integer part and multiply by the mantissa, as
// its logarithm is not exact. r is moved (and O, in TMEM, rescaled) only when
// the maximum outgrows it by 2^8, which f16 holds.
// FP32 queries take two f16 parts of Q and of P (22 bits) and one query tile.
// Within a group of 4 head dimensions the f16 order is 0, 2, 1, 3 (how bytes
// unpack); Q is stored alike and the output is put back in order.
// Every wait is bounded: one that runs out sets the status bit, and all roles
// leave.
#include <cstdint>
#include <string>

#include "kvblock.cuh"
#include "kvblock_attn.cuh"

namespace at {

namespace {

constexpr int PR_KT = 128;             // keys per tile
constexpr int PR_ROWS = 128;           // query rows per tile
constexpr int PR_PRODUCERS = 128;
constexpr uint32_t PR_TMEM_COLS = 512;
constexpr int kPrSpinLimit = 1 << 20;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

struct PrShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_full, s_full[2], p_full[2], o_done;
    uint32_t tmem;
    int bad;
    float dk[2][8], lv[2][8], iv[2][8], mv[2][8];  // per stage and 16 keys: d_k, log2 part and reciprocal of d_v, mantissa
};

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// False when the wait ran out, here or in another role.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, PrShared* sh) {
    const uint32_t b = smem_u32(bar);
    for (int it = 0; it < kPrSpinLimit; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(b), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*reinterpret_cast<volatile int*>(&sh->bad)) return false;
    }
    *reinterpret_cast<volatile int*>(&sh->bad) = 1;
    return false;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Instruction descriptor of kind::f16: D f32 (bits 4-5 = 1), A and B f16
// (bits 7-9, 10-12 = 0), B K-major (bit 16 = 0) or MN-major (1), N >> 3 at
// bits 17-22, M >> 4 at bits 24-28.
constexpr uint32_t pr_idesc(int m, int n, bool b_mn) {
    return (1u << 4) | (b_mn ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Shared-memory descriptors, 128-byte swizzle (layout type 2 at bits 61-63),
// version 1 (bit 46); addresses and offsets in 16-byte units.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) |
           (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// 32 consecutive 32-bit columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte chunk c (0..7) of row r in a K-major tile of
// 64-element (128-byte) rows.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4)); }

template <class T>
constexpr int pr_terms() { return sizeof(T) == 4 ? 2 : 1; }
template <class T>
constexpr int pr_tiles() { return sizeof(T) == 4 ? 1 : 2; }  // query tiles per CTA
template <class T>
constexpr int pr_threads() { return 128 * pr_tiles<T>() + PR_PRODUCERS + 32; }
template <class T, int HD>
constexpr size_t pr_smem() {
    return (size_t)pr_terms<T>() * pr_tiles<T>() * PR_ROWS * HD * 2 + 2 * (2 * PR_KT * HD * 2) + 1024;
}

struct PromptParams {
    KvbDev c;
    KvbBatch b;
    const void* q;
    int64_t q_ts, q_hs;
    void* out;
    int H, G, window, q_vec, blocks, min_rows;  // blocks: query blocks per sequence; sequences up to min_rows rows are skipped
    float scale;
};

template <class T, int HD>
__global__ void __launch_bounds__(pr_threads<T>(), 1) kvb_attn_prompt_kernel(const PromptParams p) {
    constexpr int NQ = pr_tiles<T>(), TERMS = pr_terms<T>();
    constexpr int NA = HD / 64;                        // 128-byte atom columns of a row
    constexpr uint32_t ATOM_COL = 128 * 128;           // bytes of one atom column of a 128-row K-major tile
    constexpr uint32_t TILE = 128 * HD * 2;            // bytes of a Q, K or V tile
    constexpr uint32_t IDESC_S = pr_idesc(PR_ROWS, PR_KT, false), IDESC_O = pr_idesc(PR_ROWS, HD, true);
    constexpr int SM_WARPS = 4 * NQ;
    extern __shared__ uint8_t pr_raw[];
    __shared__ PrShared sh;
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ks = qs + NQ * TERMS * TILE;
    uint8_t* vs = ks + 2 * TILE;
    const KvbDev& c = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // late query blocks see the most keys: they go first
    const int blk = p.blocks - 1 - (int)(blockIdx.x / (c.hkv * p.b.n_seqs));
    const int kvh = blockIdx.x % c.hkv, s = (blockIdx.x / c.hkv) % p.b.n_seqs;
    const KvbSeq sq = kvb_seq(c, p.b, s);
    const int QB = PR_ROWS / p.G;                      // tokens per query tile
    const int t0 = blk * NQ * QB;                      // first token of the CTA
    if (t0 >= sq.n || sq.n * p.G <= p.min_rows) return;
    const int start = (int)sq.start;
    // key tiles of query tile i: [lo_tile(i), hi_tile(i))
    int k_lo[NQ], k_hi[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int a = t0 + i * QB, b = min(sq.n, a + QB) - 1;
        const bool live = a < sq.n;
        k_lo[i] = live && p.window > 0 ? max(0, start + a - p.window + 1) / PR_KT : 0;
        k_hi[i] = live ? (start + b) / PR_KT + 1 : 0;
    }
    const int lo = k_lo[0], hi = NQ == 2 ? max(k_hi[0], k_hi[NQ - 1]) : k_hi[0];
    const int end = start + min(sq.n, t0 + NQ * QB);   // keys at or past it are not read

    if (warp == SM_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(PR_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&sh.k_full[i], PR_PRODUCERS);
            bar_init(&sh.v_full[i], PR_PRODUCERS);
            bar_init(&sh.k_empty[i], 1);
            // V's scales are read by the softmax threads until their P is done
            bar_init(&sh.v_empty[i], 1);
            bar_init(&sh.s_full[i], 1);
            bar_init(&sh.p_full[i], 128);
        }
        bar_init(&sh.q_full, 128 * NQ);
        bar_init(&sh.o_done, 1);
        sh.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp < SM_WARPS) {
        // ------------------------------------------------------------ softmax
        const int i = warp >> 2, row = tid & 127;
        const uint32_t trow = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t t_s = trow + 128 * i, t_o = trow + 128 * NQ + 128 * i;
        const int tok = t0 + i * QB + row / p.G;
        const bool live = row / p.G < QB && tok < sq.n;
        const int qpos = live ? start + tok : -1;
        float qf;  // score factor of the row, log2 units
        {
            const T* src = static_cast<const T*>(p.q) + (int64_t)(sq.off + tok) * p.q_ts + (int64_t)(kvh * p.G + row % p.G) * p.q_hs;
            float top = 0.f;
            if (live) {
#pragma unroll 4
                for (int d = 0; d < HD; d += 8) {
                    float x[8];
                    load8<T>(src + d, p.q_vec, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
                }
            }
            const float rs = row_scale(top);
            qf = p.scale * 1.44269504088896341f / rs;
            uint8_t* dst = qs + i * TERMS * TILE;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
                if (live) load8<T>(src + d, p.q_vec, x);
                uint32_t h[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // pairs (0, 2), (1, 3), (4, 6), (5, 7)
                    const float a = x[4 * (e >> 1) + (e & 1)] * rs, b = x[4 * (e >> 1) + (e & 1) + 2] * rs;
                    h[e] = pack_h2(a, b);
                    const float2 f = unpack_h2(h[e]);
                    l[e] = pack_h2(a - f.x, b - f.y);
                }
                const uint32_t at = (d >> 6) * ATOM_COL + sw128(row, (d >> 3) & 7);
                *reinterpret_cast<uint4*>(dst + at) = make_uint4(h[0], h[1], h[2], h[3]);
                if constexpr (TERMS == 2) *reinterpret_cast<uint4*>(dst + TILE + at) = make_uint4(l[0], l[1], l[2], l[3]);
            }
            fence_async();
            bar_arrive(&sh.q_full);
        }
        float r = -INFINITY, l = 0.f;
        bool ok = true;
        int n = 0;
        for (int k = lo; k < hi && ok; ++k) {
            if (k < k_lo[i] || k >= k_hi[i]) continue;
            const int st = (k - lo) & 1, k0 = k * PR_KT;
            // the scales come with K
            ok = bar_wait(&sh.k_full[st], ((k - lo) >> 1) & 1, &sh) && bar_wait(&sh.s_full[i], n & 1, &sh);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            fence_after();
            const bool edge = __any_sync(0xffffffffu, k0 + PR_KT - 1 > qpos || (p.window > 0 && k0 <= qpos - p.window));
            float mx = -INFINITY;
            uint32_t sv[32];
#pragma unroll 1
            for (int cc = 0; cc < 4; ++cc) {
                tmem_ld32(t_s + 32 * cc, sv);
                tmem_ld_wait();
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int key = k0 + 32 * cc + e;
                        if (key > qpos || (p.window > 0 && key <= qpos - p.window)) sv[e] = 0xFF800000u;
                    }
                }
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float m = __uint_as_float(sv[16 * hf]);
#pragma unroll
                    for (int e = 1; e < 16; ++e) m = fmaxf(m, __uint_as_float(sv[16 * hf + e]));
                    if (m != -INFINITY) mx = fmaxf(mx, fmaf(m, sh.dk[st][2 * cc + hf] * qf, sh.lv[st][2 * cc + hf]));
                }
            }
            float alpha = 1.f;
            if (mx > r + 8.f) {
                alpha = ex2(r - mx);  // 0 for the first
                r = mx;
            }
            const float sub = r == -INFINITY ? 0.f : r;
            float sum = 0.f;
#pragma unroll 1
            for (int cc = 0; cc < 4; ++cc) {
                uint32_t pk[16], pl[16];
                tmem_ld32(t_s + 32 * cc, sv);
                tmem_ld_wait();
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float f = sh.dk[st][2 * cc + hf] * qf, off = sh.lv[st][2 * cc + hf] - sub, mv = sh.mv[st][2 * cc + hf];
                    float a0 = 0.f, a1 = 0.f;
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float x = ex2(fmaf(__uint_as_float(sv[16 * hf + e]), f, off)), y = ex2(fmaf(__uint_as_float(sv[16 * hf + e + 1]), f, off));
                        const int key = k0 + 32 * cc + 16 * hf + e;
                        bool hx = false, hy = false;
                        if (edge) {
                            hx = key > qpos || (p.window > 0 && key <= qpos - p.window);
                            hy = key + 1 > qpos || (p.window > 0 && key + 1 <= qpos - p.window);
                            x = hx ? 0.f : x;
                            y = hy ? 0.f : y;
                        }
                        a0 += x;
                        a1 += y;
                        if constexpr (TERMS == 2) {
                            x = hx ? 0.f : x * mv;
                            y = hy ? 0.f : y * mv;
                        }
                        const uint32_t h = pack_h2(x, y);
                        pk[8 * hf + e / 2] = h;
                        if constexpr (TERMS == 2) {
                            const float2 u = unpack_h2(h);
                            pl[8 * hf + e / 2] = pack_h2(x - u.x, y - u.y);
                        }
                    }
                    const float a = a0 + a1;
                    if (a != 0.f) sum = fmaf(a, sh.iv[st][2 * cc + hf], sum);
                }
                tmem_st16(t_s + 16 * cc, pk);
                if constexpr (TERMS == 2) tmem_st16(t_o + 128 + 16 * cc, pl);
            }
            l = fmaf(l, alpha, sum);
            // O of the earlier tiles is complete: its products were issued before this S
            if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                for (int cc = 0; cc < HD / 32; ++cc) {
                    tmem_ld32(t_o + 32 * cc, sv);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) sv[e] = __float_as_uint(__uint_as_float(sv[e]) * alpha);
                    tmem_st32(t_o + 32 * cc, sv);
                }
            }
            tmem_st_wait();
            fence_before();
            bar_arrive(&sh.p_full[i]);
            ++n;
        }
        if (ok && n > 0) ok = bar_wait(&sh.o_done, 0, &sh);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && n > 0) {
            fence_after();
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
            T* dst = static_cast<T*>(p.out) + ((size_t)(sq.off + tok) * p.H + kvh * p.G + row % p.G) * HD;
#pragma unroll 1
            for (int cc = 0; cc < HD / 32; ++cc) {
                uint32_t ov[32];
                tmem_ld32(t_o + 32 * cc, ov);
                tmem_ld_wait();
                if (live) {
                    constexpr int PER = 16 / sizeof(T);
#pragma unroll
                    for (int d = 0; d < 32; d += PER) {
                        alignas(16) T y[PER];
#pragma unroll
                        for (int e = 0; e < PER; ++e) {  // dimension 4 g + (0, 1, 2, 3) sits at 4 g + (0, 2, 1, 3)
                            const int at = d + e, w = at & 3;
                            y[e] = from_f32<T>(__uint_as_float(ov[(at & ~3) + ((w & 1) << 1 | (w >> 1))]) * inv);
                        }
                        *reinterpret_cast<uint4*>(dst + 32 * cc + d) = *reinterpret_cast<const uint4*>(y);
                    }
                }
            }
        }
    } else if (warp < SM_WARPS + 4) {
        // ---------------------------------------------------------- producers
        constexpr int CPR = HD / 16;                   // 16-byte chunks per row
        constexpr int CH = PR_KT * CPR / PR_PRODUCERS; // chunks per thread of K, and of V
        const int pt = tid - 32 * SM_WARPS;
        const int bmask = (1 << c.lb) - 1;
        for (int k = lo; k < hi; ++k) {
            const int st = (k - lo) & 1, use = (k - lo) >> 1, k0 = k * PR_KT;
            // lanes 0..7: the page and scales of each 16 keys
            int page = -2;
            float dk = 0.f, dv = 0.f;
            if (lane < 8 && k0 + 16 * lane < end) {
                page = kvb_page(c, sq.slot, (k0 + 16 * lane) >> c.lb);
                const size_t i = (size_t)max(page, 0) * c.hkv + kvh;
                dk = page < 0 ? __uint_as_float(0x7FC00000u) : c.ks[i];
                dv = page < 0 ? __uint_as_float(0x7FC00000u) : c.vs[i];
            }
            uint4 x[2][CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int ch = i * PR_PRODUCERS + pt, r = ch / CPR, col = 16 * (ch % CPR);
                const int pg = __shfl_sync(0xffffffffu, page, r >> 4);
                x[0][i] = x[1][i] = make_uint4(0u, 0u, 0u, 0u);
                if (k0 + r < end && pg >= 0) {
                    const size_t at = ((((size_t)pg * c.hkv + kvh) << c.lb) + ((k0 + r) & bmask)) * HD + col;
                    x[0][i] = ld_stream_u4(c.k + at);
                    x[1][i] = ld_stream_u4(c.v + at);
                }
            }
            if (use > 0 && !(bar_wait(&sh.k_empty[st], (use - 1) & 1, &sh) && bar_wait(&sh.v_empty[st], (use - 1) & 1, &sh))) break;
            if (pt < 8) {
                sh.dk[st][pt] = dk;
                value_scale<TERMS == 2>(dv, &sh.lv[st][pt], &sh.iv[st][pt], &sh.mv[st][pt]);
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                uint8_t* dst = (kv ? vs : ks) + st * TILE;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int ch = i * PR_PRODUCERS + pt, r = ch / CPR, c8 = 2 * (ch % CPR);
                    const uint32_t w[4] = {x[kv][i].x, x[kv][i].y, x[kv][i].z, x[kv][i].w};
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const uint4 y = make_uint4(bytes_h2<false>(w[2 * hf], false), bytes_h2<false>(w[2 * hf], true),
                                                   bytes_h2<false>(w[2 * hf + 1], false), bytes_h2<false>(w[2 * hf + 1], true));
                        const int cc = c8 + hf;
                        const uint32_t at = kv == 0 ? (cc >> 3) * ATOM_COL + sw128(r, cc & 7)
                                                    : (r >> 3) * (NA * 1024) + (cc >> 3) * 1024 + (r & 7) * 128 + (((cc & 7) ^ (r & 7)) << 4);
                        *reinterpret_cast<uint4*>(dst + at) = y;
                    }
                }
                fence_async();
                bar_arrive(kv ? &sh.v_full[st] : &sh.k_full[st]);
            }
        }
    } else if (lane == 0) {
        // ---------------------------------------------------------------- MMA
        bool ok = bar_wait(&sh.q_full, 0, &sh);
        fence_after();
        auto scores = [&](int i, int st) {
            const uint32_t ka = smem_u32(ks + st * TILE);
#pragma unroll
            for (int e = 0; e < TERMS; ++e) {
                const uint32_t qa = smem_u32(qs + (i * TERMS + e) * TILE);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    mma_ss(tmem + 128 * i, desc_k_major(qa + (kk >> 2) * ATOM_COL + 32 * (kk & 3)),
                           desc_k_major(ka + (kk >> 2) * ATOM_COL + 32 * (kk & 3)), IDESC_S, (e > 0 || kk > 0) ? 1u : 0u);
            }
            mma_commit(&sh.s_full[i]);
        };
        auto values = [&](int i, int st, bool first) {
            const uint32_t va = smem_u32(vs + st * TILE);
            const uint32_t o = tmem + 128 * NQ + 128 * i;
#pragma unroll
            for (int e = 0; e < TERMS; ++e)
#pragma unroll
                for (int kk = 0; kk < PR_KT / 16; ++kk)
                    mma_ts(o, (e == 0 ? tmem + 128 * i : o + 128) + 8 * kk, desc_mn_major(va + kk * 2 * (NA * 1024), 1024, NA * 1024), IDESC_O,
                           (!first || e > 0 || kk > 0) ? 1u : 0u);
        };
        int n[NQ] = {};
        for (int k = lo; k <= hi && ok; ++k) {
            const int st = (k - lo) & 1, pst = st ^ 1;
            if (k < hi) ok = bar_wait(&sh.k_full[st], ((k - lo) >> 1) & 1, &sh);
            if (ok && k > lo) ok = bar_wait(&sh.v_full[pst], ((k - 1 - lo) >> 1) & 1, &sh);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int q = k - 1;
                if (q >= max(lo, k_lo[i]) && q < k_hi[i]) {
                    if (!(ok = bar_wait(&sh.p_full[i], n[i] & 1, &sh))) break;
                    fence_after();
                    values(i, pst, n[i] == 0);
                    ++n[i];
                }
                if (k < hi && k >= k_lo[i] && k < k_hi[i]) scores(i, st);
            }
            if (!ok) break;
            if (k > lo) mma_commit(&sh.v_empty[pst]);
            if (k < hi) mma_commit(&sh.k_empty[st]);
        }
        mma_commit(&sh.o_done);
        bar_wait(&sh.o_done, 0, &sh);  // nothing in flight when TMEM is freed
    }
    fence_before();
    __syncthreads();
    if (sh.bad && tid == 0) kvb_flag(c.status, KVB_STALLED);
    if (warp == SM_WARPS)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PR_TMEM_COLS) : "memory");
}

template <class T, int HD>
void prompt_launch(PromptParams p, cudaStream_t s) {
    auto kern = kvb_attn_prompt_kernel<T, HD>;
    AT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pr_smem<T, HD>()));
    const int per = pr_tiles<T>() * (PR_ROWS / p.G);
    p.blocks = (p.b.max_tokens + per - 1) / per;
    const int64_t grid = (int64_t)p.blocks * p.c.hkv * p.b.n_seqs;
    AT_REQUIRE(grid <= INT32_MAX, AT_ERR_INVALID_ARG, "the batch is too large for one call");
    kern<<<(int)grid, pr_threads<T>(), pr_smem<T, HD>(), s>>>(p);
    AT_CUDA(cudaGetLastError());
}

}  // namespace

void launch_kvb_attn_prompt(const KvbDev& c, const KvbBatch& b, int dtype, int n_heads, const void* q, int64_t q_ts, int64_t q_hs, void* out,
                            float scale, int window, int min_rows, cudaStream_t s) {
    const PromptParams p{c, b, q, q_ts, q_hs, out, n_heads, n_heads / c.hkv, window, aligned_rows(q, kvb_elem_bytes(dtype), q_ts, q_hs) ? 1 : 0,
                         0, min_rows, scale};
    kvb_dispatch(dtype, [&](auto t) {
        using T = decltype(t);
        if (c.hd == 128) prompt_launch<T, 128>(p, s);
        else prompt_launch<T, 64>(p, s);
    });
}

}  // namespace at
