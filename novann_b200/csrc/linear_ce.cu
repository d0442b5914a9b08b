// Softmax cross entropy of a linear layer's output, the logits never kept.
//
//   l = X W^T + b;   lse_m = log sum_v exp(l_mv);   loss_m = lse_m - l_m,y(m)   (rows that count)
//   g = s (exp(l - lse) - onehot(y)),  s = grad_scale / (rows that count, or 1 for a sum)
//   dX = g W,  dW = g^T X,  db = sum over m of g
//
// One kernel does all four contractions: a pair of CTAs per 256 x 256 output tile, operands by TMA into
// a six-stage ring, tcgen05.mma (cta_group::2) into two TMEM accumulators, so that the epilogue of one
// tile runs under the MMAs of the next.  What differs is which of an operand's two dimensions is
// contiguous (the contraction for X W^T and for g in dX; the other one for W in dX and for both
// operands of dW - the tensor core reads either, so nothing is ever transposed) and the epilogue:
//   kLse   per row the maximum and the sum of exp over 128 columns, and the label's logit
//   kProb  softmax(l) - onehot as 16-bit values, a piece of the vocabulary at a time (kProbDb: and the
//          column sums of the fp32 values, for db)
//   kSum   fp32 sums: added to a buffer, or scaled and rounded to the gradient's type
// The backward pass computes the logits of a piece a second time instead of keeping M x V of them:
// 8 M V K operations where 6 M V K are needed, against reading and writing the logits twice.
#include <type_traits>

#include "gemm_common.cuh"
#include "packet.cuh"

namespace {

constexpr int BM = 256, BN = 256, BK = 64, UMMA_K = 16;
constexpr int A_BYTES = 128 * BK * 2, B_BYTES = 128 * BK * 2;   // per CTA
constexpr int STAGES = 6;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 8192;
constexpr int TMEM_COLS = 512;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// fp16 values of g below 2^-14 would lose bits: they are kept times 2^14 (|g| <= 1 stays in range)
constexpr float F16_GAIN = 16384.f;

enum { kLse = 0, kProb = 1, kSum = 2, kProbDb = 3 };
constexpr bool is_prob(int epi) { return epi == kProb || epi == kProbDb; }
// Epilogue warps: eight with 128 columns of 32 rows each, in registers (168 a thread).  kProb, which has the most to do
// per column, is faster with sixteen of 64 columns (2048 x 32000 x 1024: 114 us against 124), the others are not (kLse
// 107 against 102).
template <int EPI> struct Cfg {
    static constexpr int WARPS = is_prob(EPI) ? 16 : 8;
    static constexpr int THREADS = 64 + 32 * WARPS;
    static constexpr int COLGRPS = WARPS / 4, COLS = BN / COLGRPS;
};
constexpr int MAX_WARPS = 16, LSE_SLOTS = Cfg<kLse>::COLGRPS;      // partial maxima and sums per 256 columns
enum { ERR_PRODUCER = 81, ERR_MMA_FULL = 82, ERR_MMA_TMEM = 83, ERR_EPILOGUE = 84, ERR_LABEL = 85 };

// One contraction: (M x K) times (K x N) in 256 x 256 tiles
struct Problem : LinearParams {
    int splits, kb_per;          // the contraction cut into `splits` parts of kb_per k-blocks
    int a_mn;                    // kSum: A is stored with M contiguous instead of the contraction
    const float* add;            // fp32 sums of earlier pieces (M x N), or nullptr
    float* sum;                  // where fp32 sums go (M x N each; split s at s * M * N), or nullptr
    void* out;                   // final result, or nullptr
    int vec32;                   // out's rows start on 32-byte boundaries
};

struct CeParams {
    Problem q[2];                // kSum: up to two contractions in one launch, the longer items first
    int lead;                    // see nth_item
    int* status;
    // kLse, kProb
    const float* bias;
    const int32_t* labels;
    float2* partial;             // kLse: (LSE_SLOTS * n_blocks) x M maxima and sums
    float* label_logit;          // kLse: M
    const float* stats;          // kProb: M row maxima, then M logarithms of the sums of exp(l - maximum)
    int v0, vocab, ignore;       // kProb: first vocabulary entry of this piece, vocabulary, label that does not count
    uint16_t* prob;              // kProb: M x ldp, ldp a multiple of 16, 0 past the piece
    int ldp;
    float* col_partial;          // ceil(M / 32) x ldp column sums of 32 rows each (kProbDb writes, kSum adds up)
    // kSum
    int out_type;
    float scale;                 // factor of the final results, over the count of rows where `count` is set
    const float* count;
    float* db;                   // the column sums' sums, db_n of them over `groups` groups of rows, times db_scale
    int db_n, groups;
    float db_scale;
};

struct Shared {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t tmem_full[4];
    uint64_t tmem_empty[4];
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float bias[2][BN];
    float db_part[MAX_WARPS][32];
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Waits for the kernel before this one; the kernel after it may then be set up beside this one (it waits alike).
__device__ __forceinline__ void chain() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// a + b, and in `lost` exactly what its rounding left out (Knuth's two-sum)
__device__ __forceinline__ float two_sum(float a, float b, float& lost) {
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    lost = __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t));
    return s;
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Keeps what follows a wait for TMEM loads behind it: the loaded registers are touched here.
template <int N>
__device__ __forceinline__ void pin(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+f"(v[i]));
}

// Shared-memory descriptor of a tile whose rows run along the contraction and hold 64 elements of the
// other dimension (128 bytes, 128-byte swizzle): groups of 8 rows are 1024 bytes apart, the next 64
// elements of the other dimension 64 rows (8192 bytes) further on.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(8192 >> 4) << 16;                      // leading byte offset
    d |= (uint64_t)(1024 >> 4) << 32;                      // stride byte offset
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

struct Item { const Problem* q; TileRef tile; int kb0, kb1, split; bool second; };
__device__ __forceinline__ Item item_of(const CeParams& p, int t) {
    Item it;
    it.second = t >= p.q[0].num_items;
    it.q = &p.q[it.second];
    if (it.second) t -= p.q[0].num_items;
    it.split = 0;
    it.kb0 = 0;
    it.kb1 = (it.q->K + BK - 1) / BK;
    if (it.q->splits > 1) {          // num_items = tiles * splits, a tile's parts next to one another
        it.split = t % it.q->splits;
        t /= it.q->splits;
        it.kb0 = it.split * it.q->kb_per;
        it.kb1 = min(it.kb1, it.kb0 + it.q->kb_per);
    }
    it.tile = tile_ref(*it.q, t);
    return it;
}

// The n-th item of a pair, or -1.  The first contraction's items are dealt out in turn; the pairs that got one less then take
// `lead` of the second's each (as many as last as long as the item that they did not get), and what is left is
// dealt out to all.
__device__ __forceinline__ int nth_item(const CeParams& p, int pair, int num_pairs, int n) {
    const int n0 = p.q[0].num_items, n1 = p.q[1].num_items, r0 = n0 % num_pairs;
    const int mine = n0 / num_pairs + (pair < r0);
    if (n < mine) return pair + n * num_pairs;
    n -= mine;
    const int idle = num_pairs - r0;
    int i;
    if (pair >= r0 && n < p.lead) i = pair - r0 + n * idle;
    else i = idle * p.lead + pair + (pair >= r0 ? n - p.lead : n) * num_pairs;
    return i < n1 ? n0 + i : -1;
}

// kLse and kProbDb keep at most this many k-blocks (512 of K) in one TMEM accumulator: the tensor core cuts off where it
// adds, by up to a step of the running sum each time.  Over 4096 of K the logits were off by 1e-6 of themselves, all
// towards zero; in parts of 1024 the row losses are 6e-7 off, in parts of 512 3e-7 (and scoring 4095 x 50001 x 2048
// takes 517 us instead of 506).  The parts are joined in registers; MMAs and epilogue alternate between the two
// accumulators as they do between tiles.  db needs the probabilities from logits summed alike: from one
// accumulator they missed a sum of 1 by 3e-5 at K = 4096.
constexpr int PART_KB = 8;
constexpr bool in_parts(int epi) { return epi == kLse || epi == kProbDb; }

template <bool F16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}

// `columns` of one row's sums, times s; wide: dst lies on a 32-byte boundary, else on a 16-byte one
template <int COLS>
__device__ __forceinline__ void store_f32(float* dst, const float (&v)[COLS], int columns, float s, bool wide) {
#pragma unroll
    for (int g = 0; g < COLS; g += 8) {
        if (g >= columns) break;
        u32x8 o;
#pragma unroll
        for (int j = 0; j < 8; j++) o.v[j] = __float_as_uint(v[g + j] * s);
        if (wide) {
            stg_stream_256(dst + g, o);
        } else {
            stg_stream_128(dst + g, make_uint4(o.v[0], o.v[1], o.v[2], o.v[3]));
            stg_stream_128(dst + g + 4, make_uint4(o.v[4], o.v[5], o.v[6], o.v[7]));
        }
    }
}
template <bool F16, int COLS>
__device__ __forceinline__ void store_16(uint16_t* dst, const float (&v)[COLS], int columns, float s, bool wide) {
#pragma unroll
    for (int g = 0; g < COLS; g += 16) {
        if (g >= columns) break;
        u32x8 o;
#pragma unroll
        for (int j = 0; j < 8; j++) o.v[j] = pack16<F16>(v[g + 2 * j] * s, v[g + 2 * j + 1] * s);
        if (wide && g + 16 <= columns) {
            stg_stream_256(dst + g, o);
        } else {
            stg_stream_128(dst + g, make_uint4(o.v[0], o.v[1], o.v[2], o.v[3]));
            if (g + 16 <= columns) stg_stream_128(dst + g + 8, make_uint4(o.v[4], o.v[5], o.v[6], o.v[7]));
        }
    }
}

// 32 lanes x 8 consecutive fp32 columns
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, float* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// kLse, kProb: both operands with the contraction contiguous.  kSum: B with N contiguous, A as Problem::a_mn says.
// F16: operands (and 16-bit results) are fp16, else bf16.
template <int EPI, bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<EPI>::THREADS, 1)
ce_gemm_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
               const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
               const __grid_constant__ CeParams p) {
    constexpr bool B_MN = EPI == kSum;
    constexpr int EPI_WARPS = Cfg<EPI>::WARPS, COLGRPS = Cfg<EPI>::COLGRPS, COLS = Cfg<EPI>::COLS;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = tc::smem_u32(smem_raw);
    const uint32_t tiles = (raw + 1023u) & ~1023u;
    Shared* sh = (Shared*)(smem_raw + (tiles - raw) + STAGES * STAGE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_ctarank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    volatile int* abort_flag = &sh->abort_flag;
    // accumulators: two of 256 columns
    auto acc_of = [&](int n, uint32_t& acc, uint32_t& acc_phase) { acc = n & 1; acc_phase = (n >> 1) & 1; };
    constexpr int part_kb = in_parts(EPI) ? PART_KB : 1 << 30;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            tc::mbar_init(tc::smem_u32(&sh->full[s]), 1);
            tc::mbar_init(tc::smem_u32(&sh->empty[s]), 1);
        }
        for (int a = 0; a < 2; a++) {
            tc::mbar_init(tc::smem_u32(&sh->tmem_full[a]), 1);
            tc::mbar_init(tc::smem_u32(&sh->tmem_empty[a]), 2 * EPI_WARPS);
        }
        sh->abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&map_a0);
        tc::tma_prefetch_desc(&map_b0);
        if (EPI == kSum) {
            tc::tma_prefetch_desc(&map_a1);
            tc::tma_prefetch_desc(&map_b1);
        }
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tc::smem_u32(&sh->tmem_base), TMEM_COLS);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync_all();
    tc::tc_fence_after();
    const uint32_t tmem_base = sh->tmem_base;
    chain();

    if (warp == 0) {
        // ------------------------------------------------------------ producer (both CTAs)
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int i = 0, t; ok && (t = nth_item(p, pair, num_pairs, i)) >= 0; i++) {
                const Item it = item_of(p, t);
                const CUtensorMap* map_a = it.second ? &map_a1 : &map_a0;
                const CUtensorMap* map_b = it.second ? &map_b1 : &map_b0;
                const int rows_b = it.tile.is_half ? BN / 4 : BN / 2;       // per CTA
                const int m0 = it.tile.m_blk * BM + (int)rank * 128;
                const int n0 = it.tile.n_blk * BN + it.tile.half * (BN / 2) + (int)rank * rows_b;
                for (int kb = it.kb0; kb < it.kb1; kb++) {
                    ok = tc::mbar_wait(tc::smem_u32(&sh->empty[stage]), phase ^ 1, abort_flag, ERR_PRODUCER);
                    if (!ok) break;
                    const uint32_t dst = tiles + stage * STAGE_BYTES;
                    const uint32_t lead_full = tc::mapa(tc::smem_u32(&sh->full[stage]), 0);
                    if (rank == 0)       // the leader expects the bytes of both CTAs
                        tc::mbar_arrive_expect_tx(tc::smem_u32(&sh->full[stage]), 2 * (A_BYTES + rows_b * BK * 2));
                    if (EPI == kSum && it.q->a_mn) {
                        tc::tma_load_2d_pair(dst, map_a, lead_full, m0, kb * BK);
                        tc::tma_load_2d_pair(dst + A_BYTES / 2, map_a, lead_full, m0 + 64, kb * BK);
                    } else {
                        tc::tma_load_2d_pair(dst, map_a, lead_full, kb * BK, m0);
                    }
                    if constexpr (B_MN) {
                        tc::tma_load_2d_pair(dst + A_BYTES, map_b, lead_full, n0, kb * BK);
                        if (rows_b == 128)
                            tc::tma_load_2d_pair(dst + A_BYTES + B_BYTES / 2, map_b, lead_full, n0 + 64, kb * BK);
                    } else {
                        tc::tma_load_2d_pair(dst + A_BYTES, map_b, lead_full, kb * BK, n0);
                        if (rows_b == 128)
                            tc::tma_load_2d_pair(dst + A_BYTES + B_BYTES / 2, map_b, lead_full, kb * BK, n0 + 64);
                    }
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader only)
        if (lane == 0 && rank == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true, ready = false;
            int n = 0;
            constexpr uint32_t fmt = F16 ? 0u : 1u;
            for (int i = 0, t; ok && (t = nth_item(p, pair, num_pairs, i)) >= 0; i++) {
                const Item it = item_of(p, t);
                const bool a_mn = EPI == kSum && it.q->a_mn;
                const uint32_t idesc = tc::idesc_f16(BM, it.tile.is_half ? BN / 2 : BN, fmt, fmt) |
                                       (a_mn ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);
                // 16 contraction steps: 32 bytes along a row, or 16 rows of 128 bytes
                const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4;
                constexpr uint32_t b_step = B_MN ? 2048 >> 4 : 32 >> 4;
                for (int k0 = it.kb0; k0 < it.kb1 && ok; k0 += part_kb, n++) {
                    const int k1 = it.kb1 - k0 < part_kb ? it.kb1 : k0 + part_kb;
                    uint32_t acc, acc_phase;
                    acc_of(n, acc, acc_phase);
                    ok = tc::mbar_wait(tc::smem_u32(&sh->tmem_empty[acc]), acc_phase ^ 1, abort_flag, ERR_MMA_TMEM);
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t d_tmem = tmem_base + acc * BN;
                    for (int kb = k0; kb < k1; kb++) {
                        if (!ready) {
                            ok = tc::mbar_wait(tc::smem_u32(&sh->full[stage]), phase, abort_flag, ERR_MMA_FULL);
                            if (!ok) break;
                        }
                        tc::tc_fence_after();
                        const uint32_t nstage = stage + 1 == (uint32_t)STAGES ? 0u : stage + 1;
                        const uint32_t nphase = nstage == 0 ? phase ^ 1u : phase;
                        const uint32_t a_addr = tiles + stage * STAGE_BYTES, b_addr = a_addr + A_BYTES;
                        const uint64_t a_desc = a_mn ? smem_desc_mn_sw128(a_addr) : tc::smem_desc_k_sw128(a_addr);
                        const uint64_t b_desc = B_MN ? smem_desc_mn_sw128(b_addr) : tc::smem_desc_k_sw128(b_addr);
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; k++) {
                            tc::tc_mma_f16_pair(d_tmem, a_desc + a_step * k, b_desc + b_step * k, idesc,
                                                kb > k0 || k > 0);
                            if (k == 0) ready = tc::mbar_test_wait(tc::smem_u32(&sh->full[nstage]), nphase);
                        }
                        tc::tc_commit_pair(tc::smem_u32(&sh->empty[stage]), 3);
                        stage = nstage;
                        phase = nphase;
                    }
                    if (ok) tc::tc_commit_pair(tc::smem_u32(&sh->tmem_full[acc]), 3);
                }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const int quarter = warp & 3;                 // the TMEM lanes this warp may read
        const int colgrp = (warp - 2) >> 2;           // which COLS (COLS / 2) columns of the tile
        const int et = threadIdx.x - 64;
        bool ok = true;
        int n_acc = 0;
        // the accumulator that comes next, complete; every epilogue thread takes part, whatever its lane found
        auto take = [&](uint32_t& taddr) -> uint32_t {
            uint32_t acc, acc_phase;
            acc_of(n_acc++, acc, acc_phase);
            __syncwarp();            // rows past the end have skipped the stores of the tile before
            ok = tc::mbar_wait(tc::smem_u32(&sh->tmem_full[acc]), acc_phase, abort_flag, ERR_EPILOGUE);
            ok = epilogue_all<32 * EPI_WARPS>(ok);
            tc::tc_fence_after();
            taddr = tmem_base + acc * BN + ((uint32_t)(quarter * 32) << 16);
            return acc;
        };
        auto give_back = [&](uint32_t acc) {
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive_remote(tc::mapa(tc::smem_u32(&sh->tmem_empty[acc]), 0));
        };

        if constexpr (EPI == kSum) {
            // db, while the first tile's MMAs run: 32 columns a warp where there are few groups of rows to add up,
            // else 32 columns a CTA
            if (p.db) {
                const float s_db = p.count ? p.db_scale / fmaxf(*p.count, 1.f) : p.db_scale;
                const bool alone = p.groups <= EPI_WARPS;
                const int wide = alone ? 32 * EPI_WARPS : 32;
                for (int c0 = (int)blockIdx.x * wide; c0 < p.db_n; c0 += (int)gridDim.x * wide) {
                    float s = 0.f;
                    const int c = c0 + (alone ? (warp - 2) * 32 : 0) + lane;
                    if (c < p.db_n)
#pragma unroll 4
                        for (int g = alone ? 0 : warp - 2; g < p.groups; g += alone ? 1 : EPI_WARPS)
                            s += p.col_partial[(size_t)g * p.ldp + c];
                    if (!alone) {
                        sh->db_part[warp - 2][lane] = s;
                        epilogue_all<32 * EPI_WARPS>(true);
                        s = 0.f;
                        if (warp == 2)
                            for (int w = 0; w < EPI_WARPS; w++) s += sh->db_part[w][lane];
                        epilogue_all<32 * EPI_WARPS>(true);
                    }
                    if (c < p.db_n && (alone || warp == 2)) p.db[c] = s * s_db;
                }
            }
        }

        for (int n_tile = 0, t; ok && (t = nth_item(p, pair, num_pairs, n_tile)) >= 0; n_tile++) {
            const Item it = item_of(p, t);
            const Problem& q = *it.q;
            const int bn = it.tile.is_half ? BN / 2 : BN;
            const int m0 = it.tile.m_blk * BM + (int)rank * 128;
            const int n0 = it.tile.n_blk * BN + it.tile.half * (BN / 2);
            const int row = m0 + quarter * 32 + lane;
            const bool valid = row < q.M;
            uint32_t taddr;

            // All columns of this warp (COLS, or half as many of a half-width tile) go to registers before anything is
            // done with them: the loads overlap, and the accumulator goes back at once.
            const int width = bn / COLGRPS, n_first = n0 + colgrp * width;
            float v[COLS];
            auto load_columns = [&]() {
                const uint32_t acc = take(taddr);
                if (!ok) return;
#pragma unroll
                for (int i = 0; i < COLS / 32; i++)
                    if (i * 32 < width) tc::tmem_ld_32x32(taddr + colgrp * width + i * 32, (uint32_t*)v + i * 32);
                tc::tmem_ld_wait();
                pin(v);
                give_back(acc);
            };

            if constexpr (EPI == kSum) {
                load_columns();
                if (!ok) break;
                const int columns = min(width, q.N - n_first);       // N % 8 == 0: eight at a time are in or out
                const size_t at = (size_t)row * q.N + n_first;
                if (valid && q.add) {
#pragma unroll
                    for (int g = 0; g < COLS; g += 8) {
                        if (g < columns) {
                            float a[8];
                            load8_f32(a, q.add + at + g);
#pragma unroll
                            for (int j = 0; j < 8; j++) v[g + j] += a[j];
                        }
                    }
                }
                if (valid && q.out == nullptr)
                    store_f32(q.sum + (size_t)it.split * q.M * q.N + at, v, columns, 1.f, true);
                else if (valid) {
                    const float scale = p.count ? p.scale / fmaxf(*p.count, 1.f) : p.scale;
                    if (p.out_type == NVQ_F32) store_f32((float*)q.out + at, v, columns, scale, q.vec32);
                    else store_16<F16>((uint16_t*)q.out + at, v, columns, scale, q.vec32);
                }
            } else {
                // Two bias buffers, by the tile's parity: the barrier in take() lies between the last reads of one
                // and its next writes.
                float* bi = sh->bias[n_tile & 1];
                for (int c = et; c < bn; c += 32 * EPI_WARPS)
                    bi[c] = p.bias && n0 + c < q.N ? p.bias[n0 + c] : 0.f;
                int label = -1;              // column of this launch, or out of its range
                [[maybe_unused]] float row_max = 0.f, log_sum = 0.f;
                [[maybe_unused]] bool counts = false;
                if (valid) {
                    label = p.labels[row];
                    if constexpr (is_prob(EPI)) {
                        row_max = p.stats[row];
                        log_sum = p.stats[(size_t)q.M + row];
                        // a row whose every entry is taken out (-inf) has no gradient
                        counts = label != p.ignore && label >= 0 && label < p.vocab && row_max != -INFINITY;
                        label -= p.v0;
                    }
                }
                load_columns();
                if (!ok) break;
                if constexpr (in_parts(EPI)) {
                    constexpr int W = EPI == kLse ? 16 : 8;      // columns at a time: what the registers leave room for
                    for (int k0 = PART_KB; k0 < it.kb1; k0 += PART_KB) {
                        const uint32_t acc = take(taddr);
                        if (!ok) break;
#pragma unroll
                        for (int i = 0; i < COLS / W; i++) {
                            if (i * W >= width) continue;
                            float r[W];
                            if constexpr (W == 16) tc::tmem_ld_32x16(taddr + colgrp * width + i * W, (uint32_t*)r);
                            else tmem_ld_32x8(taddr + colgrp * width + i * W, r);
                            tc::tmem_ld_wait();
                            pin(r);
#pragma unroll
                            for (int j = 0; j < W; j += 2)
                                unpair2(add2(pair2(v[i * W + j], v[i * W + j + 1]), pair2(r[j], r[j + 1])), v[i * W + j],
                                        v[i * W + j + 1]);
                        }
                        give_back(acc);
                    }
                    if (!ok) break;
                }
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < COLS; j += 8) {
                        float b8[8];
                        load8_f32(b8, bi + colgrp * width + j);
#pragma unroll
                        for (int k = 0; k < 8; k += 2)
                            unpair2(add2(pair2(v[j + k], v[j + k + 1]), pair2(b8[k], b8[k + 1])), v[j + k], v[j + k + 1]);
                    }
                }
                const int columns = min(width, q.N - n_first);     // the rest lies past the vocabulary
                if (columns < COLS) {
#pragma unroll
                    for (int j = 0; j < COLS; j++)
                        if (j >= columns) v[j] = -INFINITY;
                }
                const int hit = label - n_first;          // the label's place among this warp's columns

                if constexpr (EPI == kLse) {
                    if (hit >= 0 && hit < columns) {
#pragma unroll
                        for (int j = 0; j < COLS; j++)
                            if (j == hit) p.label_logit[row] = v[j];
                    }
                    float m[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) m[j] = v[j];
#pragma unroll
                    for (int j = 4; j < COLS - 4; j += 8) {
#pragma unroll
                        for (int k = 0; k < 4; k++) m[k] = max3(m[k], v[j + 2 * k], v[j + 2 * k + 1]);
                    }
                    const float top = max3(max3(m[0], m[1], m[2]), m[3],
                                           max3(fmaxf(v[COLS - 4], v[COLS - 3]), v[COLS - 2], v[COLS - 1]));
                    // exp(l - top) by one multiply-add
                    float s1 = -top * LOG2E;
                    if (!__all_sync(0xFFFFFFFFu, fabsf(top) < 1e30f)) {
                        // Logits near the lowest fp32 value, whose product with log2 e overflows, or nothing but -inf: a
                        // row whose entries are all taken out has sum 0 relative to 0.
                        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                        for (int j = 0; j < COLS; j++) v[j] -= ref;
                        s1 = 0.f;
                    }
                    const uint64_t scale = pair2(LOG2E, LOG2E), shift = pair2(s1, s1);
                    uint64_t s2[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < COLS; j += 2) {
                        float a, b;
                        unpair2(fma2(pair2(v[j], v[j + 1]), scale, shift), a, b);
                        s2[j / 2 % 4] = add2(s2[j / 2 % 4], pair2(ex2(a), ex2(b)));
                    }
                    float s_even, s_odd;
                    unpair2(add2(add2(s2[0], s2[1]), add2(s2[2], s2[3])), s_even, s_odd);
                    float sum = s_even + s_odd;
                    // what the shift lost in rounding, as a factor 2^e = 1 + e ln 2 of all of them
                    if (s1 != 0.f) sum = fmaf(sum * fmaf(-top, LOG2E, -s1), LN2, sum);
                    // the maximum and sum of this warp's columns, for each of its rows (kLse tiles are never cut in
                    // two, so a 256-column block has these two entries)
                    if (valid)
                        p.partial[(size_t)(it.tile.n_blk * COLGRPS + colgrp) * q.M + row] = make_float2(top, sum);
                } else {
                    // softmax(l) - onehot, times F16_GAIN (2^14, part of the exponent) for fp16
                    constexpr float gain = F16 ? F16_GAIN : 1.f, log2_gain = F16 ? 14.f : 0.f;
                    // by one multiply-add, whose shift is off by 2^-15 of a probability at most; kProbDb adds what it lost
                    const float a_hi = row_max * LOG2E, b_hi = log_sum * LOG2E;
                    const float b_lo = fmaf(log_sum, LOG2E, -b_hi);
                    float lost, left;
                    float s1 = two_sum(log2_gain, -two_sum(a_hi, b_hi, lost), left);
                    [[maybe_unused]] float s0 = left - (lost + fmaf(row_max, LOG2E, -a_hi) + b_lo);
                    if (!__all_sync(0xFFFFFFFFu, fabsf(row_max) < 256.f)) {
#pragma unroll
                        for (int j = 0; j < COLS; j++) v[j] -= row_max;
                        s1 = log2_gain - b_hi;
                        s0 = -b_lo;
                    }
                    const uint64_t scale = pair2(LOG2E, LOG2E), shift = pair2(s1, s1);
#pragma unroll
                    for (int j = 0; j < COLS; j += 2) {
                        uint64_t t = fma2(pair2(v[j], v[j + 1]), scale, shift);
                        if constexpr (EPI == kProbDb) t = add2(t, pair2(s0, s0));
                        float a, b;
                        unpair2(t, a, b);
                        v[j] = ex2(a);
                        v[j + 1] = ex2(b);
                    }
                    if (hit >= 0 && hit < columns) {
#pragma unroll
                        for (int j = 0; j < COLS; j++)
                            if (j == hit) v[j] -= gain;
                    }
                    // a row that does not count gives zeros whatever its logits are
                    const uint32_t keep = counts ? 0xFFFFFFFFu : 0u;
                    if (valid) {
                        uint16_t* dst = p.prob + (size_t)row * p.ldp + n_first;
#pragma unroll
                        for (int g = 0; g < COLS; g += 16) {
                            if (g < width && n_first + g < p.ldp) {
                                u32x8 o;
#pragma unroll
                                for (int j = 0; j < 8; j++)
                                    o.v[j] = pack16<F16>(v[g + 2 * j], v[g + 2 * j + 1]) & keep;
                                stg_stream_256(dst + g, o);
                            }
                        }
                    }
                    if constexpr (EPI == kProbDb) {
                        // Sums of 32 columns over the warp's 32 rows: at each step a lane keeps the half of its
                        // columns that its lane bit names and adds its partner's; after five steps lane l holds
                        // column l.
#pragma unroll
                        for (int c = 0; c < COLS; c += 32) {
                            if (c >= width) continue;
                            float f[32];
#pragma unroll
                            for (int j = 0; j < 32; j++) f[j] = __uint_as_float(__float_as_uint(v[c + j]) & keep);
#pragma unroll
                            for (int h = 16; h; h >>= 1) {
                                const bool upper = (lane & h) != 0;
#pragma unroll
                                for (int j = 0; j < h; j++) {
                                    const float stay = upper ? f[j + h] : f[j], give = upper ? f[j] : f[j + h];
                                    f[j] = stay + __shfl_xor_sync(0xFFFFFFFFu, give, h);
                                }
                            }
                            if (n_first + c + lane < p.ldp && m0 + quarter * 32 < q.M)
                                p.col_partial[(size_t)((m0 >> 5) + quarter) * p.ldp + n_first + c + lane] = f[0];
                        }
                    }
                }
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    if (*abort_flag) {
        for (int i = 0; i < 64; i++) __nanosleep(20000);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync_all();
    tc::tc_fence_after();
    if (warp == 1) tc::tmem_dealloc_pair(tmem_base, TMEM_COLS);
    if (threadIdx.x == 0 && *abort_flag && p.status) atomicCAS(p.status, 0, *abort_flag);
}

// ---------------------------------------------------------------- joining what the tiles left
// Row statistics, row loss and the label checks, one row per lane.
constexpr int JOIN_WARPS = 32;

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    const float ref = top == -INFINITY ? 0.f : top;
    s = s * ex2((m - ref) * LOG2E) + s2 * ex2((m2 - ref) * LOG2E);
    m = top;
}

// loss[0] = sum of the row losses (over their count for the mean; 0 when no row counts), loss[1] = count
__device__ __forceinline__ void put_loss(float* loss, double sum, double count, int mean) {
    loss[0] = (float)(mean ? sum / (count > 1.0 ? count : 1.0) : sum);
    loss[1] = (float)count;
}

// WAYS warps share 32 rows; a block takes 32 / WAYS groups of rows.  With one block the loss is complete.
template <int WAYS>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
join_rows_kernel(float* __restrict__ loss_out, float* __restrict__ stats, float* __restrict__ row_loss,
                 double2* __restrict__ block_sum, const float2* __restrict__ partial,
                 const float* __restrict__ label_logit, const int32_t* __restrict__ labels, int M, int slots, int vocab,
                 int ignore, int mean, int* __restrict__ status) {
    __shared__ float2 part[WAYS > 1 ? JOIN_WARPS : 1][32];
    __shared__ double sums[JOIN_WARPS], counts[JOIN_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = (blockIdx.x * (JOIN_WARPS / WAYS) + warp / WAYS) * 32 + lane;
    chain();
    float m = -INFINITY, s = 0.f;
    if (row < M) {
        int i = warp % WAYS;
        for (; i + 3 * WAYS < slots; i += 4 * WAYS) {
            float2 q[4];
#pragma unroll
            for (int k = 0; k < 4; k++) q[k] = partial[(size_t)(i + k * WAYS) * M + row];
#pragma unroll
            for (int k = 0; k < 4; k++) join(m, s, q[k].x, q[k].y);
        }
        for (; i < slots; i += WAYS) {
            const float2 q = partial[(size_t)i * M + row];
            join(m, s, q.x, q.y);
        }
    }
    if constexpr (WAYS > 1) {
        part[warp][lane] = make_float2(m, s);
        __syncthreads();
        if (warp % WAYS == 0)
            for (int w = 1; w < WAYS; w++) join(m, s, part[warp + w][lane].x, part[warp + w][lane].y);
    }
    double loss = 0.0, n = 0.0;
    if (warp % WAYS == 0 && row < M) {
        // maximum and logarithm are kept apart: their sum would lose the logarithm where the logits are large
        const float log_sum = m == -INFINITY ? 0.f : logf(s);
        const int y = labels[row];
        float mine = 0.f;
        if (y != ignore) {
            if (y >= 0 && y < vocab) {
                mine = m == -INFINITY ? INFINITY : (m - label_logit[row]) + log_sum;
                n = 1.0;
            } else if (status) {
                atomicCAS(status, 0, (int)ERR_LABEL);
            }
        }
        loss = mine;
        stats[row] = m;
        stats[(size_t)M + row] = log_sum;
        if (row_loss) row_loss[row] = mine;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        loss += __shfl_xor_sync(0xFFFFFFFFu, loss, o);
        n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    }
    if (lane == 0) { sums[warp] = loss; counts[warp] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < JOIN_WARPS; w++) { loss += sums[w]; n += counts[w]; }
        if (gridDim.x == 1) put_loss(loss_out, loss, n, mean);
        else block_sum[blockIdx.x] = make_double2(loss, n);
    }
}

__global__ void __launch_bounds__(256)
loss_kernel(float* __restrict__ loss_out, const double2* __restrict__ block_sum, int blocks, int mean) {
    __shared__ double sums[8], counts[8];
    chain();
    double s = 0.0, n = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 256) {
        s += block_sum[i].x;
        n += block_sum[i].y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    }
    if ((threadIdx.x & 31) == 0) { sums[threadIdx.x >> 5] = s; counts[threadIdx.x >> 5] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) { s += sums[w]; n += counts[w]; }
        put_loss(loss_out, s, n, mean);
    }
}

// (sum of the parts of a split contraction + add) -> fp32 buffer, or scaled to the final type; n % 8 == 0
template <int DT>
__global__ void __launch_bounds__(256)
join_splits_kernel(void* out, const float* __restrict__ parts, int splits, const float* add, size_t n,
                   float scale, const float* __restrict__ count) {
    chain();
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; s++) {
        const float4 v = *(const float4*)(parts + (size_t)s * n + i);
        f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    }
    if (add) {
        const float4 v = *(const float4*)(add + i);
        f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    }
    const float s = count ? scale / fmaxf(*count, 1.f) : scale;
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] *= s;
    if constexpr (DT == NVQ_F32) {
        *(float4*)((float*)out + i) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        *(uint2*)((uint16_t*)out + i) = make_uint2(Elem<DT>::narrow(f), Elem<DT>::narrow(f + 2));
    }
}

// db = scale * the column sums' sum over the groups of 32 rows
__global__ void __launch_bounds__(256)
bias_grad_kernel(float* __restrict__ db, const float* __restrict__ col_partial, int groups, int ld, int N, float scale,
                 const float* __restrict__ count) {
    __shared__ float part[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = blockIdx.x * 32 + lane;
    chain();
    float s = 0.f;
    if (c < N)
#pragma unroll 4
        for (int g = warp; g < groups; g += 8) s += col_partial[(size_t)g * ld + c];
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < N) {
        for (int w = 1; w < 8; w++) s += part[w][lane];
        db[c] = s * (count ? scale / fmaxf(*count, 1.f) : scale);
    }
}

// ---------------------------------------------------------------- host
template <typename... KArgs, typename... Args>
nvq_status launch_after(void (*kernel)(KArgs...), size_t grid, int threads, int smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // may start under the tail
    attr[0].val.programmaticStreamSerializationAllowed = 1;            // of the previous kernel
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NVQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...));
    NVQ_LAUNCHED();
    return NVQ_OK;
}

int item_cost(int kb);
template <int EPI, bool F16>
nvq_status launch_gemm_typed(CeParams& p, const CUtensorMap& a0, const CUtensorMap& b0, const CUtensorMap& a1,
                       const CUtensorMap& b1, int device, cudaStream_t st) {
    static std::atomic<bool> attr_set[64];   // per device; setting the attribute twice is harmless
    if (!attr_set[device]) {
        NVQ_CUDA(cudaFuncSetAttribute(ce_gemm_kernel<EPI, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      SMEM_BYTES));
        attr_set[device] = true;
    }
    nvq_status s = nvq_status_word(device, &p.status);
    if (s != NVQ_OK) return s;
    const int pairs = nvq_sm_count(device) / 2;
    for (Problem& q : p.q) {
        q.m_blocks = (q.M + BM - 1) / BM;
        q.n_blocks = (q.N + BN - 1) / BN;
        // row blocks walked together: a panel of about 32 MB of A stays in L2 while B streams past it
        const int kb = q.splits > 1 ? q.kb_per : (q.K + BK - 1) / BK;
        const int most = (int)((32u << 20) / (BM * BK * 2) / (kb ? kb : 1));
        q.group_m = most < 4 ? 4 : (most > 16 ? 16 : most);
        q.num_big = q.num_items = q.m_blocks * q.n_blocks * q.splits;
    }
    // a partial last wave that would occupy at most half of the pairs is cut into half-width tiles
    Problem& tail = p.q[p.q[1].num_items ? 1 : 0];
    const int total = p.q[0].num_items + p.q[1].num_items, rem = total % pairs;
    if (EPI != kLse && tail.splits == 1 && tail.N > BN / 2 && total > pairs && 2 * rem <= pairs && rem <= tail.num_items) {
        tail.num_big -= rem;
        tail.num_items += rem;
    }
    const int items = p.q[0].num_items + p.q[1].num_items;
    const int used = items < pairs ? items : pairs;
    p.lead = 0;
    if (p.q[1].num_items && p.q[0].num_items % used) {
        const int kb0 = p.q[0].splits > 1 ? p.q[0].kb_per : (p.q[0].K + BK - 1) / BK;
        const int kb1 = p.q[1].splits > 1 ? p.q[1].kb_per : (p.q[1].K + BK - 1) / BK;
        p.lead = (item_cost(kb0) + item_cost(kb1) / 2) / item_cost(kb1);
    }
    return launch_after(ce_gemm_kernel<EPI, F16>, 2 * (size_t)used, Cfg<EPI>::THREADS, SMEM_BYTES, st, a0, b0, a1, b1, p);
}
template <int EPI>
nvq_status launch_gemm(CeParams& p, bool f16, const CUtensorMap& a0, const CUtensorMap& b0, const CUtensorMap& a1,
                       const CUtensorMap& b1, int device, cudaStream_t st) {
    return f16 ? launch_gemm_typed<EPI, true>(p, a0, b0, a1, b1, device, st)
               : launch_gemm_typed<EPI, false>(p, a0, b0, a1, b1, device, st);
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

constexpr int kPairs = 74;      // what the splits are made for: workspace sizes are asked for without a device

// The contractions of one launch as tiles and their length in k-blocks.  A tile takes as long as its MMAs or, with fewer than
// EPILOGUE_KB k-blocks, as the writing of its result.  splits[i] > 1: one item of a tile would take longer than an
// even share of all work, and the tile is cut into parts of about that share, eight k-blocks at least.
constexpr int EPILOGUE_KB = 6;
int item_cost(int kb) { return kb > EPILOGUE_KB ? kb : EPILOGUE_KB; }
struct Shape { size_t M, N, K; };
struct Cut { int splits, kb_per; };
void cut_long(const Shape* q, Cut* cut, int n) {
    size_t total = 0;
    for (int i = 0; i < n; i++)
        total += (q[i].M + BM - 1) / BM * ((q[i].N + BN - 1) / BN) * item_cost((int)((q[i].K + BK - 1) / BK));
    size_t share = (total + kPairs - 1) / kPairs;
    if (share < 8) share = 8;
    for (int i = 0; i < n; i++) {
        const size_t kb = (q[i].K + BK - 1) / BK;
        size_t parts = (kb + share - 1) / share;
        if (parts < 1) parts = 1;
        cut[i].kb_per = (int)((kb + parts - 1) / parts);
        cut[i].splits = (int)((kb + cut[i].kb_per - 1) / cut[i].kb_per);
    }
}
size_t part_bytes(const Shape& q, const Cut& c) { return c.splits > 1 ? align256(c.splits * q.M * q.N * 4) : 0; }

// Vocabulary entries per piece of the backward pass: 64 Mi values of g, 8192 entries at least, so that adding a
// piece to the fp32 dX costs little beside its contractions.
size_t piece_of(size_t M, size_t V) {
    size_t most = ((size_t)64 << 20) / M;
    if (most < 8192) most = 8192;
    const size_t pieces = (V + most - 1) / most;
    const size_t each = (V + pieces - 1) / pieces;
    return (each + 255) / 256 * 256;
}

struct FwdSpace { size_t partial, logit, block, total; };
FwdSpace fwd_space(size_t M, size_t V) {
    FwdSpace s;
    s.partial = align256((V + BN - 1) / BN * LSE_SLOTS * M * sizeof(float2));
    s.logit = align256(M * 4);
    s.block = align256((M + 31) / 32 * sizeof(double2));
    s.total = s.partial + s.logit + s.block;
    return s;
}

// Parts of the split contractions of one piece, whichever of dX and dW are wanted
size_t parts_space(size_t M, size_t nv, size_t K) {
    const Shape q[2] = {{M, K, nv}, {nv, K, M}};
    Cut c[2];
    cut_long(q, c, 2);
    size_t most = part_bytes(q[0], c[0]) + part_bytes(q[1], c[1]);
    for (int i = 0; i < 2; i++) {
        cut_long(q + i, c + i, 1);
        const size_t one = part_bytes(q[i], c[i]);
        if (one > most) most = one;
    }
    return most;
}
struct BwdSpace { size_t prob, cols, sum, total; };
BwdSpace bwd_space(size_t M, size_t V, size_t K) {
    BwdSpace s;
    const size_t piece = piece_of(M, V), nv = piece < V ? piece : V, ld = (nv + 15) / 16 * 16;
    s.prob = align256(M * ld * 2);
    s.cols = align256((M + 31) / 32 * ld * 4);
    s.sum = piece < V ? align256(M * K * 4) : 0;
    size_t parts = parts_space(M, nv, K);
    if (V % piece && piece < V) {       // the last, shorter piece
        const size_t last = parts_space(M, V % piece, K);
        if (last > parts) parts = last;
    }
    s.total = s.prob + s.cols + s.sum + parts;
    return s;
}

nvq_status join_parts(const Problem& q, const CeParams& p, const float* parts, cudaStream_t st) {
    const size_t n = (size_t)q.M * q.N, grid = (n / 4 + 255) / 256;
    if (q.out == nullptr)
        return launch_after(join_splits_kernel<NVQ_F32>, grid, 256, 0, st, (void*)q.sum, parts, q.splits, q.add, n, 1.f,
                            nullptr);
    if (p.out_type == NVQ_F32)
        return launch_after(join_splits_kernel<NVQ_F32>, grid, 256, 0, st, q.out, parts, q.splits, q.add, n, p.scale,
                            p.count);
    if (p.out_type == NVQ_F16)
        return launch_after(join_splits_kernel<NVQ_F16>, grid, 256, 0, st, q.out, parts, q.splits, q.add, n, p.scale,
                            p.count);
    return launch_after(join_splits_kernel<NVQ_BF16>, grid, 256, 0, st, q.out, parts, q.splits, q.add, n, p.scale,
                        p.count);
}

nvq_status check_shape(const char* who, const void* x, const void* w, int dtype, const float* bias,
                       const int32_t* labels, size_t M, size_t V, size_t K, int reduction) {
    NVQ_REQUIRE(dtype == NVQ_BF16 || dtype == NVQ_F16, "%s: operand type %d; f16 and bf16 are taken", who, dtype);
    NVQ_REQUIRE(V > 0 && K > 0 && M <= (1u << 30) && V <= (1u << 30) && K <= (1u << 20),
                "%s: M up to 2^30, V in [1, 2^30], K in [1, 2^20]", who);
    NVQ_REQUIRE(K % 8 == 0, "%s: K (%zu) must be a multiple of 8", who, K);
    NVQ_REQUIRE((M + BM - 1) / BM * ((V + BN - 1) / BN) < ((size_t)1 << 30), "%s: M * V is too large", who);
    NVQ_REQUIRE(reduction == NVQ_REDUCE_SUM || reduction == NVQ_REDUCE_MEAN, "%s: unknown reduction %d", who, reduction);
    NVQ_REQUIRE(w && nvq_aligned(w, 16) && (M == 0 || (x && nvq_aligned(x, 16))), "%s: x and w must be 16-byte aligned",
                who);
    NVQ_REQUIRE(M == 0 || (labels && nvq_aligned(labels, 4)), "%s: null or misaligned labels", who);
    NVQ_REQUIRE(nvq_aligned(bias, 4), "%s: misaligned bias", who);
    return NVQ_OK;
}

}  // namespace

extern "C" nvq_status nvq_linear_ce_workspace_bytes(size_t M, size_t V, size_t K, int backward, size_t* bytes) {
    NVQ_REQUIRE(bytes, "null out pointer");
    NVQ_REQUIRE(V > 0 && K > 0 && M <= (1u << 30) && V <= (1u << 30) && K <= (1u << 20),
                "nvq_linear_ce_workspace_bytes: M up to 2^30, V in [1, 2^30], K in [1, 2^20]");
    *bytes = 0;
    if (M == 0) return NVQ_OK;
    *bytes = fwd_space(M, V).total;
    if (backward) {
        const size_t b = bwd_space(M, V, K).total;
        if (b > *bytes) *bytes = b;
    }
    return NVQ_OK;
}

extern "C" nvq_status nvq_linear_ce_fwd(float* d_loss_count, float* d_row_loss, float* d_row_stats, const void* d_x,
                                        const void* d_w, nvq_dtype dtype, const float* d_bias, const int32_t* d_labels,
                                        size_t M, size_t V, size_t K, int32_t ignore_index, int reduction,
                                        void* d_workspace, size_t workspace_bytes, int device, void* stream) {
    nvq_status s = check_shape("nvq_linear_ce_fwd", d_x, d_w, dtype, d_bias, d_labels, M, V, K, reduction);
    if (s != NVQ_OK) return s;
    NVQ_REQUIRE(d_loss_count && nvq_aligned(d_loss_count, 4) && nvq_aligned(d_row_loss, 4) &&
                    (M == 0 || (d_row_stats && nvq_aligned(d_row_stats, 4))),
                "nvq_linear_ce_fwd: null or misaligned output");
    const FwdSpace sp = fwd_space(M, V);
    NVQ_REQUIRE(M == 0 || (d_workspace && workspace_bytes >= sp.total && nvq_aligned(d_workspace, 256)),
                "nvq_linear_ce_fwd: workspace of %zu bytes (256-byte aligned) required", sp.total);
    s = nvq_use_device(device);
    if (s != NVQ_OK) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (M == 0) {
        NVQ_CUDA(cudaMemsetAsync(d_loss_count, 0, 2 * sizeof(float), st));
        return NVQ_OK;
    }
    CUtensorMap a, b;
    s = nvq_make_tmap_2d(&a, d_x, M, K, 128, BK, 2, 1);
    if (s != NVQ_OK) return s;
    s = nvq_make_tmap_2d(&b, d_w, V, K, 64, BK, 2, 1);
    if (s != NVQ_OK) return s;
    char* ws = (char*)d_workspace;
    float2* partial = (float2*)ws;
    float* logit = (float*)(ws + sp.partial);
    double2* block_sum = (double2*)(ws + sp.partial + sp.logit);
    CeParams p = {};
    p.q[0].M = (int)M;
    p.q[0].N = (int)V;
    p.q[0].K = (int)K;
    p.q[0].splits = 1;
    p.bias = d_bias;
    p.labels = d_labels;
    p.partial = partial;
    p.label_logit = logit;
    s = launch_gemm<kLse>(p, dtype == NVQ_F16, a, b, a, b, device, st);
    if (s != NVQ_OK) return s;
    // up to eight partial sums a row: a warp adds up 32 rows by itself; more: the whole block does
    const int slots = LSE_SLOTS * p.q[0].n_blocks, mean = reduction == NVQ_REDUCE_MEAN;
    const int rows = slots <= 8 ? 32 * JOIN_WARPS : 32, blocks = (int)((M + rows - 1) / rows);
    s = slots <= 8 ? launch_after(join_rows_kernel<1>, blocks, JOIN_WARPS * 32, 0, st, d_loss_count, d_row_stats,
                                  d_row_loss, block_sum, partial, logit, d_labels, (int)M, slots, (int)V, ignore_index,
                                  mean, p.status)
                   : launch_after(join_rows_kernel<JOIN_WARPS>, blocks, JOIN_WARPS * 32, 0, st, d_loss_count,
                                  d_row_stats, d_row_loss, block_sum, partial, logit, d_labels, (int)M, slots, (int)V,
                                  ignore_index, mean, p.status);
    if (s != NVQ_OK || blocks == 1) return s;
    return launch_after(loss_kernel, 1, 256, 0, st, d_loss_count, block_sum, blocks, mean);
}

extern "C" nvq_status nvq_linear_ce_bwd(void* d_dx, void* d_dw, nvq_dtype grad_dtype, float* d_db, const void* d_x,
                                        const void* d_w, nvq_dtype dtype, const float* d_bias, const int32_t* d_labels,
                                        const float* d_row_stats, const float* d_loss_count, float grad_scale, size_t M,
                                        size_t V, size_t K, int32_t ignore_index, int reduction, void* d_workspace,
                                        size_t workspace_bytes, int device, void* stream) {
    nvq_status s = check_shape("nvq_linear_ce_bwd", d_x, d_w, dtype, d_bias, d_labels, M, V, K, reduction);
    if (s != NVQ_OK) return s;
    NVQ_REQUIRE(grad_dtype == NVQ_F32 || grad_dtype == dtype,
                "nvq_linear_ce_bwd: gradients are f32 or of the operands' type, not %d", (int)grad_dtype);
    NVQ_REQUIRE(nvq_aligned(d_dx, 16) && nvq_aligned(d_dw, 16) && nvq_aligned(d_db, 4),
                "nvq_linear_ce_bwd: dx and dw must be 16-byte aligned");
    NVQ_REQUIRE(M == 0 || (d_row_stats && d_loss_count && nvq_aligned(d_row_stats, 4) && nvq_aligned(d_loss_count, 4)),
                "nvq_linear_ce_bwd: needs the row statistics, loss and count that nvq_linear_ce_fwd left");
    const size_t size = grad_dtype == NVQ_F32 ? 4 : 2;
    BwdSpace sp = {};
    if (M) sp = bwd_space(M, V, K);
    NVQ_REQUIRE(M == 0 || (d_workspace && workspace_bytes >= sp.total && nvq_aligned(d_workspace, 256)),
                "nvq_linear_ce_bwd: workspace of %zu bytes (256-byte aligned) required", sp.total);
    s = nvq_use_device(device);
    if (s != NVQ_OK) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (M == 0) {
        if (d_dw) NVQ_CUDA(cudaMemsetAsync(d_dw, 0, V * K * size, st));
        if (d_db) NVQ_CUDA(cudaMemsetAsync(d_db, 0, V * sizeof(float), st));
        return NVQ_OK;
    }
    if (!d_dx && !d_dw && !d_db) return NVQ_OK;
    char* ws = (char*)d_workspace;
    uint16_t* prob = (uint16_t*)ws;
    float* cols = (float*)(ws + sp.prob);
    float* sum = (float*)(ws + sp.prob + sp.cols);
    char* parts = ws + sp.prob + sp.cols + sp.sum;
    const float* count = reduction == NVQ_REDUCE_MEAN ? d_loss_count + 1 : nullptr;
    const bool f16 = dtype == NVQ_F16;
    const size_t piece = piece_of(M, V);
    CUtensorMap x_k, x_mn;      // X with the contraction along its rows, and across them
    s = nvq_make_tmap_2d(&x_k, d_x, M, K, 128, BK, 2, 1);
    if (s != NVQ_OK) return s;
    s = nvq_make_tmap_2d(&x_mn, d_x, M, K, BK, 64, 2, 1);
    if (s != NVQ_OK) return s;
    for (size_t v0 = 0; v0 < V; v0 += piece) {
        const size_t nv = V - v0 < piece ? V - v0 : piece, ld = (nv + 15) / 16 * 16;
        const bool last = v0 + nv == V;
        const uint16_t* w = (const uint16_t*)d_w + v0 * K;
        CUtensorMap w_k, w_mn, g_k, g_mn;
        if ((s = nvq_make_tmap_2d(&w_k, w, nv, K, 64, BK, 2, 1)) != NVQ_OK) return s;
        if ((s = nvq_make_tmap_2d(&w_mn, w, nv, K, BK, 64, 2, 1)) != NVQ_OK) return s;
        if ((s = nvq_make_tmap_2d(&g_k, prob, M, ld, 128, BK, 2, 1)) != NVQ_OK) return s;
        if ((s = nvq_make_tmap_2d(&g_mn, prob, M, ld, BK, 64, 2, 1)) != NVQ_OK) return s;
        CeParams p = {};
        p.q[0].M = (int)M;
        p.q[0].N = (int)nv;
        p.q[0].K = (int)K;
        p.q[0].splits = 1;
        p.bias = d_bias ? d_bias + v0 : nullptr;
        p.labels = d_labels;
        p.stats = d_row_stats;
        p.v0 = (int)v0;
        p.vocab = (int)V;
        p.ignore = ignore_index;
        p.prob = prob;
        p.ldp = (int)ld;
        p.col_partial = d_db ? cols : nullptr;
        s = d_db ? launch_gemm<kProbDb>(p, f16, x_k, w_k, x_k, w_k, device, st)
                 : launch_gemm<kProb>(p, f16, x_k, w_k, x_k, w_k, device, st);
        if (s != NVQ_OK) return s;

        // dX and dW of the piece in one launch, and db beside them
        CeParams u = {};
        u.out_type = grad_dtype;
        u.scale = grad_scale / (f16 ? F16_GAIN : 1.f);
        u.count = count;
        u.col_partial = cols;
        u.ldp = (int)ld;
        u.db = d_db ? d_db + v0 : nullptr;
        u.db_n = (int)nv;
        u.groups = (int)((M + 31) / 32);
        u.db_scale = u.scale;
        Problem dx = {}, dw = {};
        dx.M = (int)M;
        dx.N = dw.N = (int)K;
        dx.K = dw.M = (int)nv;
        dw.K = (int)M;
        dw.a_mn = 1;
        dx.add = v0 ? sum : nullptr;
        dx.sum = last ? nullptr : sum;
        dx.out = last ? d_dx : nullptr;
        dx.vec32 = K * size % 32 == 0 && nvq_aligned(d_dx, 32);
        dw.out = d_dw ? (char*)d_dw + v0 * K * size : nullptr;
        dw.vec32 = K * size % 32 == 0 && nvq_aligned(d_dw, 32);
        Shape shape[2];
        Cut cut[2];
        Problem* wanted[2];
        int n = 0;
        if (d_dx) { shape[n] = {M, K, nv}; wanted[n++] = &dx; }
        if (d_dw) { shape[n] = {nv, K, M}; wanted[n++] = &dw; }
        cut_long(shape, cut, n);
        char* at = parts;
        Problem whole[2];              // as wanted, for joining the parts
        for (int i = 0; i < n; i++) {
            Problem& q = *wanted[i];
            q.splits = cut[i].splits;
            q.kb_per = cut[i].kb_per;
            whole[i] = q;
            if (q.splits > 1) {
                q.add = nullptr;
                q.out = nullptr;
                q.sum = (float*)at;
                at += part_bytes(shape[i], cut[i]);
            }
        }
        // the longer items first
        const bool swap = n == 2 && cut[1].kb_per > cut[0].kb_per;
        if (n > 0) u.q[swap ? 1 : 0] = *wanted[0];
        if (n > 1) u.q[swap ? 0 : 1] = *wanted[1];
        const bool first_dw = n > 0 && wanted[swap ? 1 : 0] == &dw;
        if (n == 0) {
            s = launch_after(bias_grad_kernel, (nv + 31) / 32, 256, 0, st, u.db, cols, u.groups, u.ldp, u.db_n, u.db_scale,
                             count);
        } else {
            s = first_dw ? launch_gemm<kSum>(u, f16, g_mn, x_mn, g_k, w_mn, device, st)
                         : launch_gemm<kSum>(u, f16, g_k, w_mn, g_mn, x_mn, device, st);
        }
        if (s != NVQ_OK) return s;
        for (int i = 0; i < n; i++) {
            if (cut[i].splits == 1) continue;
            s = join_parts(whole[i], u, wanted[i]->sum, st);
            if (s != NVQ_OK) return s;
        }
    }
    return NVQ_OK;
}
