// Attention over the block-quantized KV cache for many query rows (prompts)
// on the 5th-generation tensor cores.
//
// A CTA holds NQ tiles of 128 query rows of one (sequence, KV head): the
// tokens of consecutive query blocks times the G heads of the KV head, so
// every K and V byte is read and converted once for all of them. The keys
// are walked in tiles of 128:
//   two warpgroups of producers, one for K and one for V, copy a tile's int8
//     rows from their pages into shared memory (cp.async, each thread its own
//     chunks: the next tile's are in flight while this one's are converted),
//     turn them into f16, or K into bf16 for BF16 queries (both exact,
//     |q| <= 127), and store them into a two-stage ring: K K-major, V MN-major,
//     128-byte swizzle;
//   one thread issues S = Q K^T into TMEM, and O += P V with P read from TMEM;
//     with two query tiles one's products run under the other's softmax, with
//     one (FP32) S has two buffers and the next S runs under this softmax;
//   softmax threads, one per query row with two query tiles, two per row (64
//     columns of S each, exchanging their maxima) with one: S from TMEM, twice
//     (its maximum, then the weights: 128 values would not stay in registers),
//     P back over their own S columns as packed f16. With two tiles two
//     threads per row were slower (375 us where one takes 344).
// Arithmetic, per row, in log2 units: t_j = s_j + log2 d_v(j), P_j = 2^(t_j - r)
// with a reference r that follows the row's largest t; out = sum P_j v8_j /
// sum P_j / d_v(j). The values' scale is part of the exponent, so P fills
// f16's range whatever the blocks' scales are (value_scale says how far apart
// they may lie), and costs no product; FP32
// queries keep log2 d_v to its integer part and multiply by the mantissa, as
// its logarithm is not exact. r is set 2^8 below the row's maximum, and moved
// (with O, in TMEM, rescaled) only when the maximum outgrows it by 2^14, which
// f16 holds: weights down to 2^-22 of the largest keep its full precision.
// FP32 queries take two f16 parts of Q and of P (22 bits) and one query tile.
// The tensor cores truncate what they accumulate, so each product in a chain
// loses some 10^-8 of the sum: for FP32 queries O leaves TMEM after every key
// tile and is added in FP32 registers (128 tokens behind 30000: 7e-5 off
// before). 16-bit queries keep it in TMEM, where 131072 keys lose 3e-4, as
// much as half the last place of F16.
// Within a group of 4 head dimensions the f16 order is 0, 2, 1, 3 (how bytes
// unpack); Q is stored alike and the output is put back in order.
//
// Two prompts up to 4096 tokens, 32 BF16 heads over 8 of 128: 321 us, 725
// TFLOP/s of causal products, 45 % of a plain matrix product's rate; in FP32,
// with two products for one, one query tile and a few spilled registers (28
// bytes stored, 36 loaded at head_dim 128): 614 us, 512 tokens 21 us. What
// bounds it: a tile of 128 x 128 weights costs 1024 cycles of ex2 and 1024 of
// tensor work, and a query tile's softmax, P V and next S follow one another
// (4500 cycles for two tiles); 15 % of a block's time is its first loads and
// its last stores.
// S in two buffers of 64 keys breaks that chain but pays for each product as
// for one of 128 (415 us); releasing P in halves holds up the other tile's
// products (332 us).
// The loops are kept short on purpose (unrolled over 32 columns or one chunk):
// five roles run apart in the code and share the instruction caches. The
// conversion unrolled by four: 337 us; the weights of 128 columns straight on,
// though they save a TMEM load: 347 us.
// Every wait is bounded: one that runs out sets the status bit, and all roles
// leave.
#include <atomic>
#include <cstdint>
#include <string>
#include <type_traits>

#include "kvblock.cuh"
#include "kvblock_attn.cuh"

namespace at {

namespace {

constexpr int PR_KT = 128;             // keys per tile
constexpr int PR_ROWS = 128;           // query rows per tile
constexpr int PR_PRODUCERS = 128;      // for K, and as many for V
constexpr uint32_t PR_TMEM_COLS = 512;
constexpr float PR_ROOM = 8.f, PR_GROW = 14.f;  // the reference lies so far below the maximum; it moves when that outgrows it by so much
constexpr int kPrSpinLimit = 1 << 20;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// s_full and p_full are per query tile, or per S buffer when there is one tile.
// The scales' ring is four deep: tile k + 4 is written once S of tile k + 2 is
// done, which was issued after the softmax of tile k.
struct PrShared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], sc_full[4];
    uint64_t q_full, s_full[2], p_full[2], pv_done, o_done, pair;  // pair: the two threads of each row
    uint32_t tmem;
    int bad;
    float top[2][2][PR_ROWS];  // maxima that a row's two threads exchange: [parity of the tile][half][row]
    float dk[4][8], lv[4][8], iv[4][8], mv[4][8];  // per 16 keys: d_k, log2 part and reciprocal of d_v, mantissa
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
// The same, not cut short by another role's failure: for what must be over
// before the block may leave.
__device__ __forceinline__ void bar_drain(uint64_t* bar, uint32_t parity, PrShared* sh) {
    for (int it = 0; it < kPrSpinLimit; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return;
    }
    *reinterpret_cast<volatile int*>(&sh->bad) = 1;
}

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// The MMA warp runs as a whole, with operands that the compiler knows to be
// the same in every lane (tile addresses are constants of the block, TMEM
// addresses literals): they then live in uniform registers, where the
// instruction wants them. Issued by one elected thread with operands of its
// own, an MMA took 110 to 150 cycles, twice its 64 on the tensor cores. Only
// the leader's executes.
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(leader)
        : "memory");
}
// Instruction descriptor of kind::f16: D f32 (bits 4-5 = 1), A and B f16
// (bits 7-9, 10-12 = 0) or both bf16 (1), B K-major (bit 16 = 0) or MN-major (1), N >> 3 at
// bits 17-22, M >> 4 at bits 24-28.
constexpr uint32_t pr_idesc(int m, int n, bool b_mn, bool bf16) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Shared-memory descriptors, 128-byte swizzle (layout type 2 at bits 61-63),
// version 1 (bit 46); addresses and offsets in 16-byte units: the low word
// holds the address and the leading offset, the high word the stride. A
// further byte offset is added to the low word.
constexpr uint32_t desc_high(uint32_t stride_bytes) { return (stride_bytes >> 4) | (1u << 14) | (2u << 29); }
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead_units) { return (addr >> 4) | (lead_units << 16); }
template <uint32_t AHI, uint32_t BHI>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %7};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(leader), "n"(AHI), "n"(BHI)
        : "memory");
}
template <uint32_t BHI>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 y, {%2, %6};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(leader), "n"(BHI)
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

// Bytes 0 and 2 of w, signed, as bf16 pairs, exactly: 128 + the low seven bits
// less 128, or 256 when the sign bit is set.
__device__ __forceinline__ uint32_t bytes_bf2(uint32_t w) {
    const uint32_t m = (w & 0x007F007Fu) | 0x43004300u, c = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), *reinterpret_cast<const __nv_bfloat162*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Byte offset of 16-byte chunk c (0..7) of row r in a K-major tile of
// 64-element (128-byte) rows.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4)); }

template <class T>
constexpr int pr_terms() { return sizeof(T) == 4 ? 2 : 1; }
template <class T>
constexpr int pr_tiles() { return sizeof(T) == 4 ? 1 : 2; }  // query tiles per CTA
template <class T>
constexpr int pr_halves() { return pr_tiles<T>() == 1 ? 2 : 1; }  // softmax threads per row
template <class T>
constexpr int pr_softmax() { return 128 * pr_tiles<T>() * pr_halves<T>(); }
template <class T>
constexpr int pr_threads() { return pr_softmax<T>() + 2 * PR_PRODUCERS + 128; }
// Registers per thread of the softmax, producer and MMA warpgroups. Their sums
// must stay within what the block is launched with (threads x the compiler's
// bound for that many): a setmaxnreg.inc beyond it would wait for ever.
template <class T>
constexpr int pr_softmax_regs() { return pr_tiles<T>() == 2 ? 112 : 144; }
template <class T>
constexpr int pr_producer_regs() { return pr_tiles<T>() == 2 ? 80 : 72; }
template <class T>
constexpr int pr_mma_regs() { return pr_tiles<T>() == 2 ? 56 : 40; }
template <class T>
constexpr int pr_launch_regs() { return 65536 / pr_threads<T>() / 8 * 8; }
template <class T>
constexpr bool pr_regs_fit() {
    return pr_softmax<T>() * pr_softmax_regs<T>() + 2 * PR_PRODUCERS * pr_producer_regs<T>() + 128 * pr_mma_regs<T>() <=
           pr_threads<T>() * pr_launch_regs<T>();
}
static_assert(pr_regs_fit<float>() && pr_regs_fit<__half>(), "register shares");
template <class T, int HD>
constexpr size_t pr_smem() {
    return (size_t)pr_terms<T>() * pr_tiles<T>() * PR_ROWS * HD * 2 + 2 * (2 * PR_KT * HD * 2) + 2 * PR_KT * HD;
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

static_assert(sizeof(PrShared) <= 3072, "what the tiles leave of an SM's 227 KB");

template <class T, int HD>
__global__ void __launch_bounds__(pr_threads<T>(), 1) kvb_attn_prompt_kernel(const PromptParams p) {
    constexpr int NQ = pr_tiles<T>(), TERMS = pr_terms<T>();
    constexpr int NA = HD / 64;                        // 128-byte atom columns of a row
    constexpr uint32_t ATOM_COL = 128 * 128;           // bytes of one atom column of a 128-row K-major tile
    constexpr uint32_t TILE = 128 * HD * 2;            // bytes of a Q, K or V tile
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t IDESC_S = pr_idesc(PR_ROWS, PR_KT, false, BF16), IDESC_O = pr_idesc(PR_ROWS, HD, true, false);
    constexpr int HV = pr_halves<T>(), SM_WARPS = pr_softmax<T>() / 32;
    constexpr uint32_t T_O = 256, T_LO = 384;          // TMEM columns: S at 0 and 128, O (per tile), low parts of P (one tile, per buffer)
    extern __shared__ __align__(1024) uint8_t pr_raw[];
    __shared__ PrShared sh;
    uint8_t* qs = pr_raw;
    uint8_t* ks = qs + NQ * TERMS * TILE;
    uint8_t* vs = ks + 2 * TILE;
    uint8_t* raw = vs + 2 * TILE;                      // int8 of K's and V's next tile
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
            bar_init(&sh.v_empty[i], 1);
            bar_init(&sh.sc_full[i], 2);
            bar_init(&sh.sc_full[2 + i], 2);
            bar_init(&sh.s_full[i], 1);
            bar_init(&sh.p_full[i], 128 * HV);
        }
        bar_init(&sh.q_full, pr_softmax<T>());
        bar_init(&sh.pv_done, 1);
        bar_init(&sh.pair, 256);
        bar_init(&sh.o_done, 1);
        sh.bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    // all 512 columns are this block's, so the allocation begins at 0; the
    // swizzled tiles need their 1024-byte alignment
    const bool placed = sh.tmem == 0 && (smem_u32(pr_raw) & 1023) == 0;
    constexpr uint32_t tmem = 0;
    if (placed) {

    if (warp < SM_WARPS) {
        // ------------------------------------------------------------ softmax
        regs_inc<pr_softmax_regs<T>()>();
        const int i = NQ == 2 ? warp >> 2 : 0, half = HV == 2 ? warp >> 2 : 0, row = tid & 127;
        const uint32_t trow = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t t_o = trow + T_O + 128 * i;
        const int tq = row / p.G, hq = kvh * p.G + row - tq * p.G;  // the row's token of the tile, and its query head
        const int tok = t0 + i * QB + tq;
        const bool live = tq < QB && tok < sq.n;
        const int qpos = start + min(tok, min(sq.n, t0 + (i + 1) * QB) - 1);  // padding rows: the last row's, so that they need no edge of their own
        [[maybe_unused]] float* row_qf = sh.top[1][0];  // FP32 queries: the rows' scaling (free until the second tile)
        float qf = 1.f;  // power of two of the row (FP32 queries), then its score factor, log2 units
        {
            // HD / 8 lanes take a row together (a thread's own row would touch
            // 32 lines per load).
            constexpr int LPR = HD / 8, RPP = 32 / LPR, PASSES = 32 / RPP, IN_FLIGHT = TERMS == 2 ? 4 : PASSES;
            const int sub = lane / LPR, d = 8 * (lane % LPR), r_w = 32 * (warp & 3);
            const int64_t own = live ? (int64_t)(sq.off + tok) * p.q_ts + (int64_t)hq * p.q_hs : -1;
            uint8_t* dst = qs + i * TERMS * TILE + (d >> 6) * ATOM_COL;
#pragma unroll 1
            for (int b = half * (PASSES / HV); b < (half + 1) * (PASSES / HV); b += IN_FLIGHT) {
                Raw8<T> raw8[IN_FLIGHT];
#pragma unroll
                for (int j = 0; j < IN_FLIGHT; ++j) {
                    const int64_t at = __shfl_sync(0xffffffffu, own, (b + j) * RPP + sub);
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) reinterpret_cast<uint4*>(raw8[j].t)[e] = make_uint4(0u, 0u, 0u, 0u);
                    if (at >= 0) load_raw8<T>(static_cast<const T*>(p.q) + at + d, p.q_vec, raw8[j]);
                }
#pragma unroll
                for (int j = 0; j < IN_FLIGHT; ++j) {
                    uint8_t* to = dst + sw128(r_w + (b + j) * RPP + sub, (d >> 3) & 7);
                    if constexpr (TERMS == 1) {
                        // 16-bit queries go in as they are (BF16 against BF16 K), pairs (0, 2), (1, 3), ..
                        const uint4 v = *reinterpret_cast<const uint4*>(raw8[j].t);
                        *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632),
                                                                   __byte_perm(v.z, v.w, 0x5410), __byte_perm(v.z, v.w, 0x7632));
                    } else {
                        float x[8], top = 0.f;
                        to_f32x8<T>(raw8[j], x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
                        for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const float rs = row_scale(top);
                        if (lane % LPR == 0) row_qf[r_w + (b + j) * RPP + sub] = rs;
                        uint32_t h[4], l[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float a = x[4 * (e >> 1) + (e & 1)] * rs, c2 = x[4 * (e >> 1) + (e & 1) + 2] * rs;
                            h[e] = pack_h2(a, c2);
                            const float2 g = unpack_h2(h[e]);
                            l[e] = pack_h2(a - g.x, c2 - g.y);
                        }
                        *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4*>(to + TILE) = make_uint4(l[0], l[1], l[2], l[3]);
                    }
                }
            }
            fence_async();
            bar_arrive(&sh.q_full);
        }
        bool ok = true;
        uint32_t pairs = 0;
        [[maybe_unused]] auto pair_sync = [&] {  // between the two threads of each row; bounded like every wait
            bar_arrive(&sh.pair);
            ok = __all_sync(0xffffffffu, bar_wait(&sh.pair, pairs++ & 1, &sh));
        };
        if constexpr (TERMS == 2) {
            pair_sync();
            qf = row_qf[row];
        }
        qf = p.scale * 1.44269504088896341f / qf;
        float r = -INFINITY, l = 0.f, alpha = 1.f;
        [[maybe_unused]] float acc[NQ == 1 ? HD / HV : 1] = {};  // one query tile: this thread's part of O
        int n = 0;
        // acc = (acc + the last tile's product) f
        [[maybe_unused]] auto collect = [&](float f) {
#pragma unroll
            for (int cc = 0; cc < (int)(sizeof(acc) / sizeof(float)) / 32; ++cc) {
                uint32_t y[32];
                tmem_ld32(t_o + half * (HD / HV) + 32 * cc, y);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[32 * cc + e] = (acc[32 * cc + e] + __uint_as_float(y[e])) * f;
            }
        };
        const int k_first = NQ == 2 && i ? max(lo, k_lo[NQ - 1]) : lo, k_end = NQ == 2 && i ? k_hi[NQ - 1] : k_hi[0];
        for (int k = k_first; k < k_end && ok; ++k, ++n) {
            const int k0 = k * PR_KT, sc = (k - lo) & 3;
            const int buf = NQ == 2 ? i : n & 1;       // S buffer and its barriers
            const uint32_t t_s = trow + 128 * buf;
            ok = bar_wait(&sh.sc_full[sc], ((k - lo) >> 2) & 1, &sh) && bar_wait(&sh.s_full[buf], (NQ == 2 ? n : n >> 1) & 1, &sh);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            fence_after();
            const float *dk = sh.dk[sc], *lv = sh.lv[sc], *iv = sh.iv[sc], *mv = sh.mv[sc];
            const int hide_from = min(qpos + 1 - k0, PR_KT);                                // columns at or past it are hidden
            const int hide_to = p.window > 0 ? max(qpos + 1 - p.window - k0, 0) : 0;       // and those before it
            const bool edge = __any_sync(0xffffffffu, hide_from < PR_KT || hide_to > 0);
            auto tile = [&](auto is_edge) {
                constexpr bool EDGE = decltype(is_edge)::value;
                uint32_t x[32];
                [[maybe_unused]] uint32_t sees = ~0u;  // the chunk's visible columns, a bit each
                auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
                auto load = [&](int cc) {
                    tmem_ld32(t_s + 32 * cc, x);
                    if (EDGE) sees = below(hide_from - 32 * cc) & ~below(hide_to - 32 * cc);
                    tmem_ld_wait();
                };
                auto chunk_max = [&](int cc) {  // largest t of the chunk's visible keys
                    float mx = -INFINITY;
                    if (EDGE) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(sees & (1u << e))) x[e] = 0xFF800000u;
                    }
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float m[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            m[e] = fmaxf(fmaxf(__uint_as_float(x[16 * hf + e]), __uint_as_float(x[16 * hf + e + 4])),
                                         fmaxf(__uint_as_float(x[16 * hf + e + 8]), __uint_as_float(x[16 * hf + e + 12])));
                        const float mm = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                        const float t = fmaf(mm, dk[2 * cc + hf] * qf, lv[2 * cc + hf]);
                        mx = fmaxf(mx, EDGE && mm == -INFINITY ? -INFINITY : t);
                    }
                    return mx;
                };
                float mx = -INFINITY;
#pragma unroll 1
                for (int cc = 4 / HV * half; cc < 4 / HV * (half + 1); ++cc) {
                    load(cc);
                    mx = fmaxf(mx, chunk_max(cc));
                }
                if constexpr (HV == 2) {
                    float* share = &sh.top[n & 1][0][row];
                    share[half * PR_ROWS] = mx;
                    pair_sync();
                    if (!ok) return;
                    mx = fmaxf(mx, share[(half ^ 1) * PR_ROWS]);
                }
                float sum = 0.f;
                alpha = 1.f;
                if (mx > r + PR_GROW) {
                    alpha = ex2(r - (mx - PR_ROOM));  // 0 for the first
                    r = mx - PR_ROOM;
                }
                const float sub = r == -INFINITY ? 0.f : r;
#pragma unroll 1
                for (int cc = 4 / HV * half; cc < 4 / HV * (half + 1); ++cc) {
                    uint32_t pk[16];
                    [[maybe_unused]] uint32_t pl[16];
                    load(cc);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        const float f = dk[2 * cc + hf] * qf, off = lv[2 * cc + hf] - sub;
                        const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
                        float2 a = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const bool h0 = EDGE && !(sees & (1u << (16 * hf + e))), h1 = EDGE && !(sees & (2u << (16 * hf + e)));
                            const float2 t = fma2(make_float2(__uint_as_float(x[16 * hf + e]), __uint_as_float(x[16 * hf + e + 1])), f2, off2);
                            float2 w = make_float2(ex2(h0 ? -INFINITY : t.x), ex2(h1 ? -INFINITY : t.y));
                            a = add2(a, w);
                            if constexpr (TERMS == 2) {
                                const float m = mv[2 * cc + hf];
                                w = make_float2(h0 ? 0.f : w.x * m, h1 ? 0.f : w.y * m);
                            }
                            const uint32_t h = pack_h2(w.x, w.y);
                            pk[8 * hf + e / 2] = h;
                            if constexpr (TERMS == 2) {
                                const float2 u = unpack_h2(h);
                                pl[8 * hf + e / 2] = pack_h2(w.x - u.x, w.y - u.y);
                            }
                        }
                        const float as = a.x + a.y;
                        sum = EDGE && as == 0.f ? sum : fmaf(as, iv[2 * cc + hf], sum);
                    }
                    // over this thread's own S columns, which have been read: 64 columns, or 32 from 0 and from 64
                    tmem_st16(t_s + (HV == 2 ? 64 * half + 16 * (cc & 1) : 16 * cc), pk);
                    if constexpr (TERMS == 2) tmem_st16(trow + T_LO + 64 * buf + 16 * cc, pl);
                }
                l = fmaf(l, alpha, sum);
                // with two query tiles O stays in TMEM; its last product was issued before this S
                if (NQ == 2 && n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                    for (int cc = 0; cc < HD / 32; ++cc) {
                        tmem_ld32(t_o + 32 * cc, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
                        tmem_st32(t_o + 32 * cc, x);
                    }
                }
            };
            if (edge) tile(std::true_type{});
            else tile(std::false_type{});
            if (!ok) break;
            if constexpr (NQ == 1) {
                if (n > 0) {
                    if (!(ok = __all_sync(0xffffffffu, bar_wait(&sh.pv_done, (n - 1) & 1, &sh)))) break;
                    fence_after();
                    collect(alpha);
                }
            }
            tmem_st_wait();
            fence_before();
            bar_arrive(&sh.p_full[buf]);
        }
        if (ok && n > 0) ok = bar_wait(&sh.o_done, 0, &sh);
        ok = __all_sync(0xffffffffu, ok);
        if (HV == 2 && ok && n > 0) {
            float* share = reinterpret_cast<float*>(raw) + row;  // the last tile has left it
            share[half * PR_ROWS] = l;
            pair_sync();
            l = share[0] + share[PR_ROWS];  // in the same order in both
        }
        if (ok && n > 0) {
            fence_after();
            const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
            // rows go through the query tiles' shared memory (their last product
            // is done) to leave as whole lines; chunks are XOR-swizzled by row
            constexpr int PER = 16 / sizeof(T), CPR = HD / PER, LINE = HD * (int)sizeof(T), CPH = CPR / HV;
            uint8_t* own_row = qs + i * TERMS * TILE + row * LINE;
            auto put = [&](int cc, const uint32_t* ov) {
#pragma unroll
                for (int d = 0; d < 32; d += PER) {
                    alignas(16) T y[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) {  // dimension 4 g + (0, 1, 2, 3) sits at 4 g + (0, 2, 1, 3)
                        const int at = d + e, w = at & 3;
                        y[e] = from_f32<T>(__uint_as_float(ov[(at & ~3) + ((w & 1) << 1 | (w >> 1))]) * inv);
                    }
                    const int ch = (32 * cc + d) / PER;
                    *reinterpret_cast<uint4*>(own_row + 16 * (ch ^ (row & (CPR - 1)))) = *reinterpret_cast<const uint4*>(y);
                }
            };
            if constexpr (NQ == 1) {
                collect(1.f);
#pragma unroll
                for (int cc = 0; cc < HD / 32 / HV; ++cc) put(half * (HD / 32 / HV) + cc, reinterpret_cast<const uint32_t*>(acc) + 32 * cc);
            } else {
#pragma unroll 1
                for (int cc = 0; cc < HD / 32; ++cc) {
                    uint32_t ov[32];
                    tmem_ld32(t_o + 32 * cc, ov);
                    tmem_ld_wait();
                    put(cc, ov);
                }
            }
            __syncwarp();
            constexpr int RPP = 32 / CPH;
            const int64_t own = live ? ((int64_t)(sq.off + tok) * p.H + hq) * HD : -1;
            const int sub = lane / CPH, ch = half * CPH + lane % CPH;
#pragma unroll 4
            for (int b = 0; b < 32 / RPP; ++b) {
                const int rw = b * RPP + sub, rr = 32 * (warp & 3) + rw;
                const int64_t at = __shfl_sync(0xffffffffu, own, rw);
                const uint4 y = *reinterpret_cast<const uint4*>(qs + i * TERMS * TILE + rr * LINE + 16 * (ch ^ (rr & (CPR - 1))));
                if (at >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at + PER * ch) = y;
            }
        }
    } else if (warp < SM_WARPS + 8) {
        // ---------------------------------------------------------- producers
        if constexpr (pr_producer_regs<T>() < pr_launch_regs<T>()) regs_dec<pr_producer_regs<T>()>();
        // Four lanes take 64 bytes of a row, the next four the next row's: in
        // the swizzled tile their 16-byte stores then fall into distinct banks.
        // A thread has rows pt / 4 + 32 j, NA 16-byte chunks of each.
        const bool is_v = warp >= SM_WARPS + 4;
        const int pt = tid - 32 * SM_WARPS - (is_v ? PR_PRODUCERS : 0);
        const int bmask = (1 << c.lb) - 1, r0 = pt >> 2, col = 16 * (pt & 3);
        const int8_t* src = (is_v ? c.v : c.k) + col;
        const float* scales = is_v ? c.vs : c.ks;
        // lanes 0..7: the page of each 16 keys of a tile (-1: outside the pool, -2: past the last key)
        auto lookup = [&](int k) {
            const int pos = k * PR_KT + 16 * lane;
            return lane < 8 && k < hi && pos < end ? kvb_page(c, sq.slot, pos >> c.lb) : -2;
        };
        const uint32_t slot = smem_u32(raw) + (is_v ? PR_KT * HD : 0) + 16 * pt;  // chunk i at slot + i * 16 * PR_PRODUCERS
        // rows r0 + 32 j of tile k, into their slots
        auto fetch = [&](int k, int page, int j) {
            const int at = k * PR_KT + r0 + 32 * j;
            const int pg = __shfl_sync(0xffffffffu, page, (r0 >> 4) + 2 * j);
            const int8_t* from = src + ((((size_t)max(pg, 0) * c.hkv + kvh) << c.lb) + (at & bmask)) * HD;
            const int n = at < end && pg >= 0 ? 16 : 0;
#pragma unroll
            for (int a = 0; a < NA; ++a)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + (j * NA + a) * 16 * PR_PRODUCERS), "l"(from + 64 * a), "r"(n)
                             : "memory");
        };
        // the swizzled place of chunk (j, a): swz[half] + j step_j + a step_a (32 rows keep r & 7)
        const uint32_t step_j = 4096 * (is_v ? NA : 1), step_a = is_v ? 1024 : ATOM_COL;
        const uint32_t row_at = (r0 >> 3) * (is_v ? NA * 1024 : 1024) + (r0 & 7) * 128;
        const uint32_t swz[2] = {row_at + (((col >> 3) ^ (r0 & 7)) << 4), row_at + ((((col >> 3) + 1) ^ (r0 & 7)) << 4)};
        const uint8_t* mine = raw + (is_v ? PR_KT * HD : 0) + 16 * pt;
        auto scale_of = [&](int page) {
            return page == -1 ? __uint_as_float(0x7FC00000u) : page < 0 ? 0.f : scales[(size_t)page * c.hkv + kvh];
        };
        auto store = [&](int k, float d, int next_page) {
            const int st = (k - lo) & 1, use = (k - lo) >> 1, sc = (k - lo) & 3;
            if (use > 0 && !__all_sync(0xffffffffu, bar_wait(is_v ? &sh.v_empty[st] : &sh.k_empty[st], (use - 1) & 1, &sh))) return false;
            if (pt < 32) {
                if (lane < 8) {
                    if (is_v) value_scale<TERMS == 2>(d, &sh.lv[sc][lane], &sh.iv[sc][lane], &sh.mv[sc][lane]);
                    else sh.dk[sc][lane] = d;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.sc_full[sc]);
            }
            uint8_t* dst = (is_v ? vs : ks) + st * TILE;
            auto convert = [&](auto v_) {
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int a = 0; a < NA; ++a) {
                        const uint4 x = *reinterpret_cast<const uint4*>(mine + (j * NA + a) * 16 * PR_PRODUCERS);
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            uint4 y;
                            if constexpr (BF16 && !decltype(v_)::value)
                                y = make_uint4(bytes_bf2(w[2 * hf]), bytes_bf2(w[2 * hf] >> 8), bytes_bf2(w[2 * hf + 1]), bytes_bf2(w[2 * hf + 1] >> 8));
                            else
                                y = make_uint4(bytes_h2<false>(w[2 * hf], false), bytes_h2<false>(w[2 * hf], true),
                                               bytes_h2<false>(w[2 * hf + 1], false), bytes_h2<false>(w[2 * hf + 1], true));
                            *reinterpret_cast<uint4*>(dst + swz[hf] + j * step_j + a * step_a) = y;
                        }
                    }
                    if (k + 1 < hi) fetch(k + 1, next_page, j);  // into the slots just read
                }
            };
            if (BF16 && !is_v) convert(std::false_type{});
            else convert(std::true_type{});
            fence_async();
            bar_arrive(is_v ? &sh.v_full[st] : &sh.k_full[st]);
            return true;
        };
        int page = lookup(lo), next = lookup(lo + 1);
#pragma unroll 1
        for (int j = 0; j < 4; ++j) fetch(lo, page, j);
        float d = scale_of(page);
        for (int k = lo; k < hi; ++k) {
            const float d_next = scale_of(next);
            const int after = lookup(k + 2);
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (!store(k, d, next)) break;
            d = d_next;
            next = after;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        regs_dec<pr_mma_regs<T>()>();
        if (warp == SM_WARPS + 8) {
        // ---------------------------------------------------------------- MMA
        const uint32_t leader = lane == 0;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait(bar, parity, &sh)) != 0; };
        bool ok = wait(&sh.q_full, 0);
        fence_after();
        auto scores = [&](auto i_, auto buf_, auto st_) {
            constexpr int i = i_(), buf = buf_(), st = st_();
            const uint32_t kd = desc_low(smem_u32(pr_raw) + (NQ * TERMS + st) * TILE, 1);
#pragma unroll
            for (int e = TERMS - 1; e >= 0; --e) {  // the small parts first
                const uint32_t qd = desc_low(smem_u32(pr_raw) + (i * TERMS + e) * TILE, 1);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t off = ((kk >> 2) * ATOM_COL + 32 * (kk & 3)) >> 4;
                    mma_ss<desc_high(1024), desc_high(1024)>(128 * buf, qd + off, kd + off, IDESC_S, (e < TERMS - 1 || kk > 0) ? 1u : 0u, leader);
                }
            }
            mma_commit(&sh.s_full[buf], leader);
        };
        auto values = [&](auto i_, auto buf_, auto st_, uint32_t acc) {
            constexpr int i = i_(), buf = buf_(), st = st_();
            const uint32_t vd = desc_low(smem_u32(pr_raw) + (NQ * TERMS + 2 + st) * TILE, 64);
#pragma unroll
            for (int e = TERMS - 1; e >= 0; --e) {  // the small parts first
#pragma unroll
                for (int kk = 0; kk < PR_KT / 16; ++kk)
                    mma_ts<desc_high(NA * 1024)>(T_O + 128 * i, (e == 0 ? 128 * buf + (HV == 2 ? (kk >> 2) * 32 : 0) : T_LO + 64 * buf) + 8 * kk, vd + ((kk * 2 * (NA * 1024)) >> 4),
                                                 IDESC_O, (e < TERMS - 1 || kk > 0) ? 1u : acc, leader);
            }
        };
        const std::integral_constant<int, 0> c0;
        const std::integral_constant<int, 1> c1;
        if constexpr (NQ == 1) {
            // S of tile k + 1 is issued before P V of tile k
            for (int k = lo - 1; k < hi && ok; ++k) {
                const int n = k - lo;
                if (k + 1 < hi) {
                    if (!(ok = wait(&sh.k_full[(n + 1) & 1], ((n + 1) >> 1) & 1))) break;
                    fence_after();
                    if ((n + 1) & 1) scores(c0, c1, c1);
                    else scores(c0, c0, c0);
                    mma_commit(&sh.k_empty[(n + 1) & 1], leader);
                }
                if (k < lo) continue;
                ok = wait(&sh.v_full[n & 1], (n >> 1) & 1) && wait(&sh.p_full[n & 1], (n >> 1) & 1);
                if (!ok) break;
                fence_after();
                if (n & 1) values(c0, c1, c1, 0u);
                else values(c0, c0, c0, 0u);
                mma_commit(&sh.pv_done, leader);
                mma_commit(&sh.v_empty[n & 1], leader);
            }
        } else {
            int n0 = 0, n1 = 0;
            // tile k - 1's products with V, then tile k's scores, one query tile after the other
            auto step = [&](int k, auto st, auto pst) {
                if (k < hi && !wait(&sh.k_full[st], ((k - lo) >> 1) & 1)) return false;
                if (k > lo && !wait(&sh.v_full[pst], ((k - 1 - lo) >> 1) & 1)) return false;
                fence_after();
                auto query_tile = [&](auto i, int& n) {
                    if (k > lo && k - 1 >= k_lo[i] && k - 1 < k_hi[i]) {
                        if (!wait(&sh.p_full[i], n & 1)) return false;
                        fence_after();
                        values(i, i, pst, n > 0);
                        ++n;
                    }
                    if (k < hi && k >= k_lo[i] && k < k_hi[i]) scores(i, i, st);
                    return true;
                };
                if (!query_tile(c0, n0) || !query_tile(c1, n1)) return false;
                if (k > lo) mma_commit(&sh.v_empty[pst], leader);
                if (k < hi) mma_commit(&sh.k_empty[st], leader);
                return true;
            };
            for (int k = lo; k <= hi && ok; ++k) ok = (k - lo) & 1 ? step(k, c1, c0) : step(k, c0, c1);
        }
        mma_commit(&sh.o_done, leader);
        bar_drain(&sh.o_done, 0, &sh);  // nothing in flight when TMEM is freed, also after a wait that ran out
        }
    }
    }  // placed
    fence_before();
    __syncthreads();
    if ((sh.bad || !placed) && tid == 0) kvb_flag(c.status, KVB_STALLED);
    if (warp == SM_WARPS)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(PR_TMEM_COLS) : "memory");
}

template <class T, int HD>
void prompt_launch(PromptParams p, cudaStream_t s) {
    auto kern = kvb_attn_prompt_kernel<T, HD>;
    static std::atomic<uint64_t> ready{0};  // per instance: the devices it was set up on (the attribute is a device's)
    int dev = 0;
    AT_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (!(ready.load() & bit)) {
        AT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pr_smem<T, HD>()));
        cudaFuncAttributes a;
        AT_CUDA(cudaFuncGetAttributes(&a, kern));
        AT_REQUIRE(a.numRegs == pr_launch_regs<T>(), AT_ERR_CUDA, "prompt attention was built with another register count than its warpgroups share");
        ready.fetch_or(bit);
    }
    const int per = pr_tiles<T>() * (PR_ROWS / p.G);
    p.blocks = (int)(((int64_t)p.b.max_tokens + per - 1) / per);
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
