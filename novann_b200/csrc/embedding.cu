// Embedding lookup, out[t] = scale * table[id_t], and the gradient of its table,
//   dtable[v] = scale * sum over t with id_t == v of dout[t]        (+ dtable[v] when accumulating)
// added for every v in a fixed order, in fp32, without atomics: equal inputs give equal bits.
#include "packet.cuh"

nvq_status nvq_status_word(int device, int** dev_ptr);

namespace {

enum { ERR_ID_RANGE = 71 };   // an id outside [0, V): recorded for nvq_device_error_flag

// ---------------------------------------------------------------- lookup
// A group of `lanes` threads (a power of two, at most the block) copies ROWS rows at a time, so that
// ROWS x (packets per thread) loads are in flight for every id that had to be fetched first.
constexpr int FWD_THREADS = 256;

template <int DT, int V, int ROWS>
__global__ void __launch_bounds__(FWD_THREADS)
embedding_kernel(void* __restrict__ out, const void* __restrict__ table, const int32_t* __restrict__ ids, size_t T,
                 int vocab, int packets, int lanes_log2, float scale, int* __restrict__ status) {
    constexpr int BYTES = Packet<DT, V>::BYTES;
    const int lane = threadIdx.x & ((1 << lanes_log2) - 1);
    const size_t group = ((size_t)blockIdx.x * FWD_THREADS + threadIdx.x) >> lanes_log2;
    const size_t t0 = group * ROWS;
    if (t0 >= T) return;
    const size_t pitch = (size_t)packets * BYTES;
    const char* src[ROWS];
    bool live[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int id = t0 + r < T ? ids[t0 + r] : 0;
        live[r] = id >= 0 && id < vocab;
        if (!live[r] && lane == 0 && status) atomicCAS(status, 0, ERR_ID_RANGE);
        src[r] = (const char*)table + (live[r] ? (size_t)id : 0) * pitch;
    }
    char* dst = (char*)out + t0 * pitch;
    for (int p = lane; p < packets; p += 1 << lanes_log2) {
        Packet<DT, V> q[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) q[r].load(src[r] + (size_t)p * BYTES);
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            float f[V];
            q[r].widen(f);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = live[r] ? f[j] * scale : 0.f;
            q[r].narrow(f);
            if (t0 + r < T) q[r].store(dst + r * pitch + (size_t)p * BYTES);
        }
    }
}

template <int DT, int V>
nvq_status launch_lookup(void* out, const void* table, const int32_t* ids, size_t T, size_t vocab, size_t D,
                         float scale, int* status, int device, cudaStream_t st) {
    const int packets = (int)(D / V);
    int lg = 0;
    while ((1 << lg) < packets && (1 << lg) < FWD_THREADS) lg++;
    const size_t groups_per_block = FWD_THREADS >> lg;
    // four rows per group once that still fills every SM with eight blocks
    const bool wide = T >= (size_t)4 * 8 * nvq_sm_count(device) * groups_per_block;
    const size_t per_block = groups_per_block * (wide ? 4 : 1);
    const size_t grid = (T + per_block - 1) / per_block;
    if (wide)
        embedding_kernel<DT, V, 4><<<(unsigned)grid, FWD_THREADS, 0, st>>>(out, table, ids, T, (int)vocab, packets, lg,
                                                                           scale, status);
    else
        embedding_kernel<DT, V, 1><<<(unsigned)grid, FWD_THREADS, 0, st>>>(out, table, ids, T, (int)vocab, packets, lg,
                                                                           scale, status);
    NVQ_LAUNCHED();
    return NVQ_OK;
}

// the widest packet that divides a row and that both pointers are aligned to
template <int DT>
nvq_status lookup(void* out, const void* table, const int32_t* ids, size_t T, size_t vocab, size_t D, float scale,
                  int* status, int device, cudaStream_t st) {
    constexpr int V16 = 16 / Elem<DT>::SIZE, V4 = 4 / Elem<DT>::SIZE;
    if (D % V16 == 0 && nvq_aligned(out, 16) && nvq_aligned(table, 16))
        return launch_lookup<DT, V16>(out, table, ids, T, vocab, D, scale, status, device, st);
    if (V4 > 1 && D % V4 == 0 && nvq_aligned(out, 4) && nvq_aligned(table, 4))
        return launch_lookup<DT, V4>(out, table, ids, T, vocab, D, scale, status, device, st);
    return launch_lookup<DT, 1>(out, table, ids, T, vocab, D, scale, status, device, st);
}

// ---------------------------------------------------------------- sorting the tokens
// The ids of up to SORT_MAX tokens are sorted, stably, with their positions, by one thread-block
// cluster: each CTA holds a run of at most CTA_ITEMS (id, position) pairs in its shared memory and a
// pass of least-significant-digit radix sort moves them between the CTAs through distributed shared
// memory, so that the whole sort is one launch without a global round trip.  The other clusters of the
// same launch meanwhile clear the gradient table, which takes longer than the sort for any large one.
constexpr int SORT_THREADS = 1024;
constexpr int WARPS = SORT_THREADS / 32;
constexpr int ITEMS = 16;                              // pairs per thread
constexpr int CTA_ITEMS = SORT_THREADS * ITEMS;
constexpr int MAX_CLUSTER = 8;
constexpr int SORT_MAX = CTA_ITEMS * MAX_CLUSTER;      // 131072
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;

struct SortShared {
    uint2 item[CTA_ITEMS];
    uint16_t hist[WARPS][MAX_BINS];         // per warp: count, then count of the warps before
    uint32_t cta_count[MAX_CLUSTER][MAX_BINS];
    uint32_t local_base[MAX_BINS];          // first place of a digit among this CTA's pairs
    uint32_t base[MAX_BINS];                // ... among all pairs, less local_base
    uint32_t scan[WARPS];
};

// sum of v over the threads before this one; barriers before and after the use of sh.scan
__device__ __forceinline__ uint32_t scan_exclusive(SortShared& sh, uint32_t v) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    uint32_t before = lane < warp ? sh.scan[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    __syncthreads();
    return incl - v + before;
}

__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t r, a = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

struct SortParams {
    const int32_t* ids;
    int32_t* sorted_id;      // ids that take no part (padding, out of range) come last, as `vocab`
    int32_t* sorted_pos;
    int n, vocab;
    int padding_id;          // < 0: none
    int bits, passes;        // digit width and count: passes * bits covers `vocab` itself
    int chunk_log2;          // pairs per CTA
    float* clear;            // table to clear, or nullptr
    int D;
    int skip_used;           // leave the rows out that have a token: they are written later
    int* status;
};

// a warp writes n zeros, 32 bytes a lane between the boundaries
__device__ __forceinline__ void clear_row(float* row, int n, int lane) {
    const int head = min(n, (int)((32 - ((uintptr_t)row & 31)) & 31) / 4), octs = (n - head) / 8;
    const u32x8 zero = {};
    if (lane < head) row[lane] = 0.f;
#pragma unroll 4
    for (int i = lane; i < octs; i += 32) stg_stream_256(row + head + i * 8, zero);
    const int tail = head + octs * 8 + lane;
    if (tail < n) row[tail] = 0.f;
}

// this block's share of the whole table
__device__ __forceinline__ void clear_flat(const SortParams& p, size_t block, size_t blocks, int threads) {
    const size_t floats = (size_t)p.vocab * p.D;
    const size_t first = block * threads + threadIdx.x, step = blocks * threads;
    const size_t octs = ((uintptr_t)p.clear & 31) == 0 ? floats / 8 : 0;
    const u32x8 zero = {};
#pragma unroll 4
    for (size_t i = first; i < octs; i += step) stg_stream_256(p.clear + 8 * i, zero);
    for (size_t i = octs * 8 + first; i < floats; i += step) p.clear[i] = 0.f;
}
// this warp's share of the rows whose bit is not set
__device__ __forceinline__ void clear_unused(const SortParams& p, const uint32_t* used, size_t warp, size_t warps,
                                             int lane) {
    for (size_t r = warp; r < (size_t)p.vocab; r += warps)
        if (!(used[r >> 5] >> (r & 31) & 1u)) clear_row(p.clear + r * p.D, p.D, lane);
}
// the sets of the bits of this thread's ids, every `step`-th from `first`
__device__ __forceinline__ void mark_used(const SortParams& p, uint32_t* used, int first, int step) {
    for (int i0 = first; i0 < p.n; i0 += 8 * step) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * step;
            id[k] = i < p.n ? p.ids[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (id[k] >= 0 && id[k] < p.vocab && id[k] != p.padding_id) {
                const uint32_t bit = 1u << (id[k] & 31);
                if (!(*(volatile uint32_t*)&used[id[k] >> 5] & bit)) atomicOr(&used[id[k] >> 5], bit);
            }
    }
}

__global__ void __launch_bounds__(SORT_THREADS, 1) sort_tokens_kernel(const SortParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    SortShared& sh = *(SortShared*)smem;
    uint32_t ctas, rank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (blockIdx.x >= ctas) {               // not the sorting cluster: clear the table
        const size_t block = blockIdx.x - ctas, blocks = gridDim.x - ctas;
        if (!p.skip_used) {
            clear_flat(p, block, blocks, SORT_THREADS);
            return;
        }
        // One bit per row: each CTA of the cluster looks at its share of the ids, then the shares are joined.
        const int words = (p.vocab + 31) / 32;
        uint32_t *share = (uint32_t*)smem, *used = share + (ctas > 1 ? words : 0);
        for (int i = tid; i < words; i += SORT_THREADS) share[i] = 0;
        __syncthreads();
        mark_used(p, share, (int)rank * SORT_THREADS + tid, (int)ctas * SORT_THREADS);
        __syncthreads();
        if (ctas > 1) {
            cluster_barrier();
            for (int i = tid; i < words; i += SORT_THREADS) {
                uint32_t w = 0;
                for (uint32_t c = 0; c < ctas; c++) {
                    uint32_t v;
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(&share[i], c)) : "memory");
                    w |= v;
                }
                used[i] = w;
            }
            cluster_barrier();      // nobody reads this CTA's share any more
        }
        __syncthreads();
        clear_unused(p, used, block * WARPS + warp, blocks * WARPS, lane);
        return;
    }

    const int chunk = 1 << p.chunk_log2;
    const int lo = (int)rank << p.chunk_log2;
    const int count = max(0, min(chunk, p.n - lo));
    const int bins = 1 << p.bits;
    // warp w owns items [w * 32 * rounds, ...) of the CTA's run, in rounds of 32
    const int rounds = max(1, chunk / SORT_THREADS);
    const int w0 = warp * 32 * rounds;
    uint32_t key[ITEMS], pos[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; r++) {       // all loads under way before the first is looked at
        const int i = r * SORT_THREADS + tid;
        if (i < count) key[r] = (uint32_t)p.ids[lo + i];
    }
    bool outside = false;
#pragma unroll
    for (int r = 0; r < ITEMS; r++) {
        const int i = r * SORT_THREADS + tid;
        if (i < count) {
            const bool in = key[r] < (uint32_t)p.vocab;          // a negative id is a large number here
            outside |= !in;
            sh.item[i] = make_uint2(in && (int)key[r] != p.padding_id ? key[r] : (uint32_t)p.vocab, (uint32_t)(lo + i));
        }
    }
    if (outside && p.status) atomicCAS(p.status, 0, ERR_ID_RANGE);
    for (int pass = 0; pass < p.passes; pass++) {
        const int shift = pass * p.bits;
        for (int i = tid; i < WARPS * MAX_BINS / 2; i += SORT_THREADS) ((uint32_t*)sh.hist)[i] = 0;
        __syncthreads();
        uint32_t before[ITEMS / 2];         // 16-bit ranks within the warp's run, packed in pairs
#pragma unroll
        for (int r = 0; r < ITEMS; r++) {
            if (r >= rounds) break;
            const int i = w0 + r * 32 + lane;
            const bool live = i < count;
            key[r] = 0;
            pos[r] = 0;
            if (live) {
                const uint2 q = sh.item[i];
                key[r] = q.x;
                pos[r] = q.y;
            }
            const uint32_t d = (key[r] >> shift) & (bins - 1);
            // the lanes with this lane's digit, by one vote per bit (with match.any 131072 tokens took 51 us instead of 43)
            uint32_t same = __ballot_sync(0xFFFFFFFFu, live);
#pragma unroll
            for (int b = 0; b < MAX_BITS; b++) {
                if (b >= p.bits) break;
                const uint32_t ones = __ballot_sync(0xFFFFFFFFu, d >> b & 1u);
                same &= d >> b & 1u ? ones : ~ones;
            }
            const uint32_t lower = __popc(same & ((1u << lane) - 1u));
            uint32_t rank_in_warp = 0;
            if (live) rank_in_warp = sh.hist[warp][d] + lower;
            __syncwarp();
            if (live && lower == 0) sh.hist[warp][d] = (uint16_t)(rank_in_warp + __popc(same));
            __syncwarp();
            if (r & 1) before[r >> 1] |= rank_in_warp << 16;
            else before[r >> 1] = rank_in_warp;
        }
        __syncthreads();
        // counts -> counts of the warps before; the CTA's total goes to every CTA of the cluster
        uint32_t total = 0;
        if (tid < bins) {
#pragma unroll
            for (int w0 = 0; w0 < WARPS; w0 += 16) {
                uint32_t c[16];
#pragma unroll
                for (int w = 0; w < 16; w++) c[w] = sh.hist[w0 + w][tid];
#pragma unroll
                for (int w = 0; w < 16; w++) {
                    sh.hist[w0 + w][tid] = (uint16_t)total;
                    total += c[w];
                }
            }
            for (uint32_t c = 0; c < ctas; c++)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&sh.cta_count[rank][tid], c)),
                             "r"(total)
                             : "memory");
        }
        const uint32_t local = scan_exclusive(sh, total);
        if (tid < bins) sh.local_base[tid] = local;
        __syncthreads();
        // Sorted within the CTA first: pairs of one digit then lie side by side, and what is written to the other CTAs (or
        // to memory) goes there in runs instead of one by one.
#pragma unroll
        for (int r = 0; r < ITEMS; r++) {
            const int i = w0 + r * 32 + lane;
            if (r >= rounds || i >= count) break;
            const uint32_t d = (key[r] >> shift) & (bins - 1);
            const uint32_t rk = (r & 1) ? before[r >> 1] >> 16 : before[r >> 1] & 0xFFFFu;
            sh.item[sh.local_base[d] + sh.hist[warp][d] + rk] = make_uint2(key[r], pos[r]);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; r++) {
            const int i = r * SORT_THREADS + tid;
            if (i >= count) break;
            const uint2 q = sh.item[i];
            key[r] = q.x;
            pos[r] = q.y;
        }
        cluster_barrier();       // all counts are here, and every CTA holds its pairs in registers
        // first place of each digit among all pairs, plus what the CTAs before this one hold of it
        uint32_t all = 0, mine = 0;
        if (tid < bins)
            for (uint32_t c = 0; c < ctas; c++) {
                const uint32_t v = sh.cta_count[c][tid];
                if (c < rank) mine += v;
                all += v;
            }
        const uint32_t first = scan_exclusive(sh, all);
        if (tid < bins) sh.base[tid] = first + mine - sh.local_base[tid];
        __syncthreads();
        const bool last = pass == p.passes - 1;
#pragma unroll
        for (int r = 0; r < ITEMS; r++) {
            const int i = r * SORT_THREADS + tid;
            if (i >= count) break;
            const uint32_t to = sh.base[(key[r] >> shift) & (bins - 1)] + (uint32_t)i;
            if (last) {
                p.sorted_id[to] = (int32_t)key[r];
                p.sorted_pos[to] = (int32_t)pos[r];
            } else {
                const uint32_t a = cluster_addr(&sh.item[to & (chunk - 1)], to >> p.chunk_log2);
                asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(key[r]), "r"(pos[r]) : "memory");
            }
        }
        cluster_barrier();       // every pair has landed, and nobody writes here any more at the end
    }
}

// ---------------------------------------------------------------- sums over runs of one id
// A warp adds the rows of PIECE consecutive sorted tokens over a tile of columns.  A run of one id
// that lies inside the piece goes straight to the table; the two that may cross its ends are joined in shared
// memory over the pieces of the block, in their order.  The two that may cross the block's ends leave partial
// sums in `carry` (slot 0: a run that began in an earlier block, slot 1: one that begins here and goes
// on), which join_runs_kernel adds up in the order of the blocks.
constexpr int PIECE = 32;
constexpr int SUM_WARPS = 4;
constexpr int BLOCK_TOKENS = PIECE * SUM_WARPS;

template <int DT, int V> struct Tile {
    // Packets per lane: one of 16 bytes, or narrow ones of 8 bytes in all and twice as many rows under way (65536 rows of
    // 1001 bf16: 60 us against 70 with 16 bytes; two rows of one wide packet more: 79 us against 70)
    static constexpr bool NARROW = V * Elem<DT>::SIZE < 16;
    static constexpr int NV = NARROW ? (8 / Elem<DT>::SIZE) / V : 1;
    static constexpr int AHEAD = NARROW ? 16 : 8;
    static constexpr int E = V * NV;
    static constexpr int COLS = 32 * E;
};

// this lane's E sums of columns [c0, c0 + COLS) to (or onto) a row of fp32
template <typename TL, int V>
__device__ __forceinline__ void put_row(float* row, const float* acc, int c0, int lane, int D, float scale, bool add) {
#pragma unroll
    for (int k = 0; k < TL::NV; k++) {
        const int c = c0 + (k * 32 + lane) * V;
        if (c >= D) continue;
        if constexpr (V >= 4) {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                float4 v = make_float4(acc[k * V + j] * scale, acc[k * V + j + 1] * scale, acc[k * V + j + 2] * scale,
                                       acc[k * V + j + 3] * scale);
                float4* at = (float4*)(row + c + j);
                if (add) {
                    const float4 o = *at;
                    v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                }
                *at = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float v = acc[k * V + j] * scale;
                row[c + j] = add ? row[c + j] + v : v;
            }
        }
    }
}

template <int DT, int V>
__global__ void __launch_bounds__(SUM_WARPS * 32, 5)       // 96 registers: narrow packets would take 128
sum_runs_kernel(float* __restrict__ dtable, float* __restrict__ carry, const void* __restrict__ dout,
                const int32_t* __restrict__ sorted_id, const int32_t* __restrict__ sorted_pos, int n, int vocab, int D,
                float scale, int accumulate) {
    using TL = Tile<DT, V>;
    using E = Elem<DT>;
    // the sums of a piece's first run, if it began earlier, and of its last, if it goes on; HEAD_TAIL: they are one
    enum { HEAD = 1, TAIL = 2, HEAD_TAIL = 4 };
    __shared__ float head_sum[SUM_WARPS][TL::COLS], tail_sum[SUM_WARPS][TL::COLS];
    __shared__ int kinds[SUM_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int piece = blockIdx.x * SUM_WARPS + warp;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the next one waits alike
    const int c0 = blockIdx.y * TL::COLS;
    const int i0 = piece * PIECE;          // past the last token: a piece without any
    const int my = i0 + lane;
    const int id = my < n ? sorted_id[my] : vocab;
    const int pos = my < n ? sorted_pos[my] : 0;
    const int prev = i0 > 0 && i0 < n ? sorted_id[i0 - 1] : -1;
    const int next = i0 + PIECE < n ? sorted_id[i0 + PIECE] : vocab;
    const int live = __popc(__ballot_sync(0xFFFFFFFFu, id < vocab));     // the tokens that count come first
    // bit j: the run that item j belongs to ends with it, inside this piece
    const int right = __shfl_down_sync(0xFFFFFFFFu, id, 1);
    const uint32_t ends = __ballot_sync(0xFFFFFFFFu, lane == PIECE - 1 || right != id);
    const char* base = (const char*)dout;
    const size_t pitch = (size_t)D * E::SIZE;
    float acc[TL::E];
#pragma unroll
    for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
    bool head = __shfl_sync(0xFFFFFFFFu, id, 0) == prev;      // the first run began in an earlier piece
    int kind = 0, tail_id = 0;
    constexpr int AHEAD = TL::AHEAD;
    for (int j0 = 0; j0 < live; j0 += AHEAD) {
        Packet<DT, V> q[AHEAD][TL::NV];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int at = __shfl_sync(0xFFFFFFFFu, pos, j0 + a);
            const char* row = base + (size_t)at * pitch;
#pragma unroll
            for (int k = 0; k < TL::NV; k++) {
                const int c = c0 + (k * 32 + lane) * V;
                if (j0 + a < live && c < D) q[a][k].load_stream(row + (size_t)c * E::SIZE);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int j = j0 + a;
            if (j >= live) break;
#pragma unroll
            for (int k = 0; k < TL::NV; k++) {
                float f[V];
                q[a][k].widen(f);
#pragma unroll
                for (int v = 0; v < V; v++) acc[k * V + v] += f[v];
            }
            if ((ends >> j) & 1u) {
                const int run = __shfl_sync(0xFFFFFFFFu, id, j);
                const bool tail = j == PIECE - 1 && run == next;
                if (head || tail) {
                    float* keep = head ? head_sum[warp] : tail_sum[warp];
#pragma unroll
                    for (int e = 0; e < TL::E; e++) keep[e * 32 + lane] = acc[e];
                    kind |= head ? (tail ? HEAD | HEAD_TAIL : HEAD) : TAIL;
                    tail_id = run;
                } else {
                    put_row<TL, V>(dtable + (size_t)run * D, acc, c0, lane, D, scale, accumulate);
                }
                head = false;
#pragma unroll
                for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
            }
        }
    }
    if (lane == 0) kinds[warp] = kind;
    __syncthreads();
    auto add = [&](const float* from) {
#pragma unroll
        for (int e = 0; e < TL::E; e++) acc[e] += from[e * 32 + lane];
    };
    float* out = carry + (size_t)blockIdx.x * 2 * D;
    if (kind & TAIL) {
#pragma unroll
        for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
        add(tail_sum[warp]);
        bool on = true;             // the run goes on behind this block
        for (int w = warp + 1; w < SUM_WARPS && on; w++) {
            add(head_sum[w]);
            on = kinds[w] & HEAD_TAIL;
        }
        if (on) put_row<TL, V>(out + D, acc, c0, lane, D, 1.f, false);
        else put_row<TL, V>(dtable + (size_t)tail_id * D, acc, c0, lane, D, scale, accumulate);
    }
    if (warp == 0 && (kind & HEAD)) {
#pragma unroll
        for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
        bool on = true;
        for (int w = 0; w < SUM_WARPS && on; w++) {
            add(head_sum[w]);
            on = kinds[w] & HEAD_TAIL;
        }
        put_row<TL, V>(out, acc, c0, lane, D, 1.f, false);
    }
}

// The runs that cross those blocks: slot 1 of the block where one begins, then slot 0 of every block that it
// reaches.  A warp looks at one of them and adds up a run of at most LONG_RUN by itself; a longer one
// (a frequent token: one in sixteen tokens of a 65536-token batch makes 32 blocks) is cut into equal
// shares for the warps, whose sums are then added in order.
constexpr int JOIN_WARPS = 8, LONG_RUN = 16;

// 256 columns a warp and four blocks an SM: most blocks see within three loads that no run begins in their parts, and
// the few that have something to add up should all be there at once.
template <int V> struct JoinTile {
    static constexpr int NV = 8 / V, E = 8, COLS = 256;
};

template <int V>
__global__ void __launch_bounds__(JOIN_WARPS * 32, 4)
join_runs_kernel(float* __restrict__ dtable, const float* __restrict__ carry, const int32_t* __restrict__ sorted_id,
                 int n, int vocab, int D, int parts, float scale, int accumulate) {
    using TL = JoinTile<V>;
    __shared__ int run_parts[JOIN_WARPS];      // parts after the first, for the block to add up; 0: none
    __shared__ float share[JOIN_WARPS][TL::COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = blockIdx.y * TL::COLS;
    auto fetch = [&](const float* row, float* f) {
#pragma unroll
        for (int k = 0; k < TL::NV; k++) {
            const int c = c0 + (k * 32 + lane) * V;
            Packet<NVQ_F32, V> q;
#pragma unroll
            for (int w = 0; w < Packet<NVQ_F32, V>::WORDS; w++) q.w[w] = 0;
            if (c < D) q.load(row + c);
            q.widen(f + k * V);
        }
    };
    auto add_slots = [&](float* acc, int first, int many) {       // slot 0 of `many` parts from `first`
        constexpr int AHEAD = 4;
        for (int a0 = 0; a0 < many; a0 += AHEAD) {
            float f[AHEAD][TL::E];
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (a0 + a < many) fetch(carry + (size_t)(first + a0 + a) * 2 * D, f[a]);
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (a0 + a < many)
#pragma unroll
                    for (int e = 0; e < TL::E; e++) acc[e] += f[a][e];
        }
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int part0 = blockIdx.x * JOIN_WARPS;
    const int part = part0 + warp;
    int many = 0, id = vocab;
    if (part + 1 < parts) {
        const int i0 = part * BLOCK_TOKENS, i1 = i0 + BLOCK_TOKENS;      // i1 < n: another part follows
        id = sorted_id[i1 - 1];
        const bool begins = id < vocab && sorted_id[i1] == id &&
                            !(sorted_id[i0] == id && i0 > 0 && sorted_id[i0 - 1] == id);
        // a part belongs to the run while its first token has the run's id
        for (int q0 = part + 1; begins && q0 < parts; q0 += 32) {
            const int mine = q0 + lane;
            const bool in = mine < parts && sorted_id[(size_t)mine * BLOCK_TOKENS] == id;
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, in);
            many += hit == 0xFFFFFFFFu ? 32 : __ffs(~hit) - 1;
            if (hit != 0xFFFFFFFFu) break;
        }
    }
    if (many > 0 && many <= LONG_RUN) {
        float acc[TL::E];
        fetch(carry + ((size_t)part * 2 + 1) * D, acc);
        add_slots(acc, part + 1, many);
        put_row<TL, V>(dtable + (size_t)id * D, acc, c0, lane, D, scale, accumulate);
    }
    if (lane == 0) run_parts[warp] = many > LONG_RUN ? many : 0;
    __syncthreads();
    for (int w = 0; w < JOIN_WARPS; w++) {
        const int total = run_parts[w];
        if (total == 0) continue;
        const int each = (total + JOIN_WARPS - 1) / JOIN_WARPS;
        const int first = warp * each, mine = max(0, min(each, total - first));
        float acc[TL::E];
#pragma unroll
        for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
        if (warp == 0) fetch(carry + ((size_t)(part0 + w) * 2 + 1) * D, acc);
        add_slots(acc, part0 + w + 1 + first, mine);
#pragma unroll
        for (int e = 0; e < TL::E; e++) share[warp][e * 32 + lane] = acc[e];
        __syncthreads();
        if (warp == w) {
#pragma unroll
            for (int e = 0; e < TL::E; e++) {
                acc[e] = share[0][e * 32 + lane];
                for (int x = 1; x < JOIN_WARPS; x++) acc[e] += share[x][e * 32 + lane];
            }
            put_row<TL, V>(dtable + (size_t)id * D, acc, c0, lane, D, scale, accumulate);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- few tokens: one launch, no sort
// Up to FEW_TOKENS tokens, comparing every id with every other costs less than sorting: a warp per token looks for its
// id among all T.  If an earlier token has it there is nothing to do; else the warp adds up the rows of all its
// tokens, in order, and writes the table row.  An id with more than FEW_LIST tokens is left to the block, whose warps
// then take a stretch of the tokens each.  The first blocks of the grid clear the rows that no token has.
// Gradient of an 8191 x 1001 table: 64 tokens 8 us (sort, sums and join 19), 512 tokens 12 (19), 2048 tokens 30 (20):
// the comparisons grow with T * T, and with them the time of an id that many tokens share.
constexpr int FEW_WARPS = 8, FEW_LIST = 64, FEW_TOKENS = 512;
constexpr size_t FEW_VOCAB = 262144;          // 32 KB of one bit per row

template <int DT, int V>
__global__ void __launch_bounds__(FEW_WARPS * 32, 4)
few_tokens_kernel(float* __restrict__ dtable, const void* __restrict__ dout, const int32_t* __restrict__ ids, int T,
                  int vocab, int D, float scale, int padding_id, int accumulate, int clear_blocks, int groups,
                  int tiles_per_group, int* __restrict__ status) {
    using TL = Tile<DT, V>;
    using E = Elem<DT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int list[FEW_WARPS][FEW_LIST];
    __shared__ int hot[FEW_WARPS];
    __shared__ float part[FEW_WARPS][TL::COLS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((int)blockIdx.x < clear_blocks) {
        uint32_t* used = (uint32_t*)smem;
        for (int i = threadIdx.x; i < (vocab + 31) / 32; i += FEW_WARPS * 32) used[i] = 0;
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < T; i += FEW_WARPS * 32) {
            const int id = ids[i];
            if (id >= 0 && id < vocab && id != padding_id) atomicOr(&used[id >> 5], 1u << (id & 31));
        }
        __syncthreads();
        for (int r = (int)blockIdx.x * FEW_WARPS + warp; r < vocab; r += clear_blocks * FEW_WARPS) {
            if (used[r >> 5] >> (r & 31) & 1u) continue;
            clear_row(dtable + (size_t)r * D, D, lane);
        }
        return;
    }

    const int block = (int)blockIdx.x - clear_blocks;
    const int t = block / groups * FEW_WARPS + warp;
    const int tile0 = block % groups * tiles_per_group;
    const int tile1 = min(tile0 + tiles_per_group, (D + TL::COLS - 1) / TL::COLS);
    const int id = t < T ? ids[t] : -1;
    const bool inside = id >= 0 && id < vocab;
    if (t < T && !inside && lane == 0 && status) atomicCAS(status, 0, ERR_ID_RANGE);
    const char* base = (const char*)dout;
    const size_t pitch = (size_t)D * E::SIZE;
    // acc += the rows at[0 .. n) of one column tile
    auto add_rows = [&](float* acc, const int* at, int n, int c0) {
        constexpr int AHEAD = 4;
        for (int j0 = 0; j0 < n; j0 += AHEAD) {
            Packet<DT, V> q[AHEAD][TL::NV];
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
#pragma unroll
                for (int k = 0; k < TL::NV; k++) {
                    const int c = c0 + (k * 32 + lane) * V;
                    if (j0 + a < n && c < D) q[a][k].load(base + (size_t)at[j0 + a] * pitch + (size_t)c * E::SIZE);
                }
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (j0 + a < n)
#pragma unroll
                    for (int k = 0; k < TL::NV; k++) {
                        float f[V];
                        q[a][k].widen(f);
#pragma unroll
                        for (int v = 0; v < V; v++) acc[k * V + v] += f[v];
                    }
        }
    };

    int n = 0;                  // tokens with this id, or FEW_LIST + 1 for more than the list holds
    bool first = inside && id != padding_id;
    for (int i0 = 0; i0 < T && first && n <= FEW_LIST; i0 += 8 * 32) {
        int other[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * 32 + lane;
            other[k] = i < T ? ids[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int i = i0 + k * 32 + lane;
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, other[k] == id);
            if (hit == 0 || n > FEW_LIST) continue;
            const int at = i0 + k * 32 + __ffs(hit) - 1;
            if (at < t) {
                first = false;
                n = FEW_LIST + 1;       // ends the search
                continue;
            }
            const int place = n + __popc(hit & ((1u << lane) - 1u));
            if ((hit >> lane & 1u) && place < FEW_LIST) list[warp][place] = i;
            n += __popc(hit);
        }
    }
    __syncwarp();
    if (first && n <= FEW_LIST)
        for (int tile = tile0; tile < tile1; tile++) {
            float acc[TL::E];
#pragma unroll
            for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
            add_rows(acc, list[warp], n, tile * TL::COLS);
            put_row<TL, V>(dtable + (size_t)id * D, acc, tile * TL::COLS, lane, D, scale, accumulate);
        }
    if (lane == 0) hot[warp] = first && n > FEW_LIST ? id : -1;
    __syncthreads();
    const int stretch = (T + FEW_WARPS * 32 - 1) / (FEW_WARPS * 32) * 32;      // tokens per warp, whole votes
    for (int w = 0; w < FEW_WARPS; w++) {
        const int id_w = hot[w];
        if (id_w < 0) continue;
        for (int tile = tile0; tile < tile1; tile++) {
            float acc[TL::E];
#pragma unroll
            for (int e = 0; e < TL::E; e++) acc[e] = 0.f;
            int held = 0;
            for (int i0 = warp * stretch; i0 < min(T, (warp + 1) * stretch); i0 += 32) {
                const int i = i0 + lane;
                const bool same = i < T && ids[i] == id_w;
                const uint32_t hit = __ballot_sync(0xFFFFFFFFu, same);
                if (same) list[warp][held + __popc(hit & ((1u << lane) - 1u))] = i;     // at most 31 + 32
                held += __popc(hit);
                __syncwarp();
                if (held >= 32) {
                    add_rows(acc, list[warp], held, tile * TL::COLS);
                    held = 0;
                    __syncwarp();
                }
            }
            add_rows(acc, list[warp], held, tile * TL::COLS);
#pragma unroll
            for (int e = 0; e < TL::E; e++) part[warp][e * 32 + lane] = acc[e];
            __syncthreads();
            if (warp == w) {
#pragma unroll
                for (int e = 0; e < TL::E; e++) {
                    acc[e] = part[0][e * 32 + lane];
                    for (int x = 1; x < FEW_WARPS; x++) acc[e] += part[x][e * 32 + lane];
                }
                put_row<TL, V>(dtable + (size_t)id_w * D, acc, tile * TL::COLS, lane, D, scale, accumulate);
            }
            __syncthreads();
        }
    }
}

template <int DT, int V>
nvq_status few_tokens(float* dtable, const void* dout, const int32_t* ids, int T, int vocab, int D, float scale,
                      int padding_id, int accumulate, int* status, int device, cudaStream_t st) {
    const int sms = nvq_sm_count(device), blocks = (T + FEW_WARPS - 1) / FEW_WARPS;
    const int tiles = (D + Tile<DT, V>::COLS - 1) / Tile<DT, V>::COLS;
    // column tiles go to more blocks until there are about 24 a SM
    int groups = (24 * sms + blocks - 1) / blocks;
    if (groups > tiles) groups = tiles;
    const int per_group = (tiles + groups - 1) / groups;
    groups = (tiles + per_group - 1) / per_group;
    const size_t bytes = accumulate ? 0 : ((size_t)vocab + 31) / 32 * 4;
    size_t clear = accumulate ? 0 : ((size_t)vocab * D + 8191) / 8192;
    if (clear > (size_t)2 * sms) clear = 2 * sms;
    few_tokens_kernel<DT, V><<<(unsigned)(clear + (size_t)blocks * groups), FEW_WARPS * 32, bytes, st>>>(
        dtable, dout, ids, T, vocab, D, scale, padding_id, accumulate, (int)clear, groups, per_group, status);
    NVQ_LAUNCHED();
    return NVQ_OK;
}

template <int DT>
nvq_status few_tokens_of(float* dtable, const void* dout, const int32_t* ids, int T, int vocab, int D, float scale,
                         int padding_id, int accumulate, int* status, int device, cudaStream_t st) {
    constexpr int V16 = 16 / Elem<DT>::SIZE, V4 = 4 / Elem<DT>::SIZE;
    if (D % V16 == 0 && nvq_aligned(dout, 16) && nvq_aligned(dtable, 16))
        return few_tokens<DT, V16>(dtable, dout, ids, T, vocab, D, scale, padding_id, accumulate, status, device, st);
    if (V4 > 1 && D % V4 == 0 && nvq_aligned(dout, 4))
        return few_tokens<DT, V4>(dtable, dout, ids, T, vocab, D, scale, padding_id, accumulate, status, device, st);
    return few_tokens<DT, 1>(dtable, dout, ids, T, vocab, D, scale, padding_id, accumulate, status, device, st);
}

cudaLaunchConfig_t sort_launch(size_t grid, int cluster, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(SORT_THREADS);
    cfg.dynamicSmemBytes = sizeof(SortShared);
    cfg.stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = cluster;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

struct BwdSpace { size_t ids, pos, carry, total; };
BwdSpace bwd_space(size_t T, size_t D) {
    const size_t n = T < (size_t)SORT_MAX ? T : SORT_MAX;
    BwdSpace s;
    s.ids = align256(n * 4);
    s.pos = align256(n * 4);
    s.carry = align256((n + BLOCK_TOKENS - 1) / BLOCK_TOKENS * 2 * D * 4);
    s.total = s.ids + s.pos + s.carry;
    return s;
}

// a kernel that waits (griddepcontrol.wait) for the one before it and may be set up under its tail
template <typename... KArgs, typename... Args>
void launch_after(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

template <int DT>
nvq_status sum_runs(float* dtable, float* carry, const char* dout, const int32_t* sid, const int32_t* spos, int n,
                    int vocab, int D, float scale, int accumulate, cudaStream_t st) {
    constexpr int V16 = 16 / Elem<DT>::SIZE, V4 = 4 / Elem<DT>::SIZE;
    const int parts = (n + BLOCK_TOKENS - 1) / BLOCK_TOKENS;
    const bool wide = D % V16 == 0 && nvq_aligned(dout, 16) && nvq_aligned(dtable, 16);
    const dim3 block(SUM_WARPS * 32);
    auto grid = [&](int cols, int each = 1) { return dim3((parts + each - 1) / each, (D + cols - 1) / cols); };
    const int join = JOIN_WARPS * 32;
    if (wide)
        launch_after(sum_runs_kernel<DT, V16>, grid(Tile<DT, V16>::COLS), block, st, dtable, carry, dout, sid, spos, n,
                     vocab, D, scale, accumulate);
    else if (V4 > 1 && D % V4 == 0 && nvq_aligned(dout, 4))
        launch_after(sum_runs_kernel<DT, V4>, grid(Tile<DT, V4>::COLS), block, st, dtable, carry, dout, sid, spos, n,
                     vocab, D, scale, accumulate);
    else
        launch_after(sum_runs_kernel<DT, 1>, grid(Tile<DT, 1>::COLS), block, st, dtable, carry, dout, sid, spos, n, vocab,
                     D, scale, accumulate);
    NVQ_LAUNCHED();
    if (parts > 1) {
        if (D % 4 == 0 && nvq_aligned(dtable, 16))
            launch_after(join_runs_kernel<4>, grid(JoinTile<4>::COLS, JOIN_WARPS), join, st, dtable, carry, sid, n, vocab,
                         D, parts, scale, accumulate);
        else
            launch_after(join_runs_kernel<1>, grid(JoinTile<1>::COLS, JOIN_WARPS), join, st, dtable, carry, sid, n, vocab,
                         D, parts, scale, accumulate);
        NVQ_LAUNCHED();
    }
    return NVQ_OK;
}

}  // namespace

extern "C" nvq_status nvq_embedding_fwd(void* d_out, const void* d_table, nvq_dtype dtype, const int32_t* d_ids,
                                        size_t T, size_t V, size_t D, float scale, int device, void* stream) {
    NVQ_REQUIRE(dtype == NVQ_F32 || dtype == NVQ_F16 || dtype == NVQ_BF16,
                "nvq_embedding_fwd: table type %d; f32, f16 and bf16 are taken", (int)dtype);
    NVQ_REQUIRE(V > 0 && V < (1u << 31) && D > 0 && D < (1u << 31) && T < ((size_t)1 << 31),
                "nvq_embedding_fwd: V and D in [1, 2^31), T below 2^31");
    if (T == 0) return NVQ_OK;
    const size_t size = dtype == NVQ_F32 ? 4 : 2;
    NVQ_REQUIRE(d_out && d_table && d_ids, "nvq_embedding_fwd: null buffer");
    NVQ_REQUIRE(nvq_aligned(d_out, size) && nvq_aligned(d_table, size) && nvq_aligned(d_ids, 4),
                "nvq_embedding_fwd: misaligned buffer");
    nvq_status s = nvq_use_device(device);
    if (s != NVQ_OK) return s;
    int* status = nullptr;
    s = nvq_status_word(device, &status);
    if (s != NVQ_OK) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == NVQ_F32) return lookup<NVQ_F32>(d_out, d_table, d_ids, T, V, D, scale, status, device, st);
    if (dtype == NVQ_F16) return lookup<NVQ_F16>(d_out, d_table, d_ids, T, V, D, scale, status, device, st);
    return lookup<NVQ_BF16>(d_out, d_table, d_ids, T, V, D, scale, status, device, st);
}

extern "C" nvq_status nvq_embedding_bwd_workspace_bytes(size_t T, size_t V, size_t D, size_t* bytes) {
    NVQ_REQUIRE(bytes, "null out pointer");
    (void)V;
    *bytes = bwd_space(T, D).total;
    return NVQ_OK;
}

extern "C" nvq_status nvq_embedding_bwd(float* d_dtable, const void* d_dout, nvq_dtype dout_dtype,
                                        const int32_t* d_ids, size_t T, size_t V, size_t D, float scale,
                                        int32_t padding_id, int accumulate, void* d_workspace, size_t workspace_bytes,
                                        int device, void* stream) {
    NVQ_REQUIRE(dout_dtype == NVQ_F32 || dout_dtype == NVQ_F16 || dout_dtype == NVQ_BF16,
                "nvq_embedding_bwd: gradient type %d; f32, f16 and bf16 are taken", (int)dout_dtype);
    NVQ_REQUIRE(V > 0 && V < (1u << 31) - 1 && D > 0 && D <= (1u << 21) && T < ((size_t)1 << 31),
                "nvq_embedding_bwd: V in [1, 2^31 - 1), D in [1, 2^21], T below 2^31");
    const size_t size = dout_dtype == NVQ_F32 ? 4 : 2;
    NVQ_REQUIRE(d_dtable && nvq_aligned(d_dtable, 4), "nvq_embedding_bwd: null or misaligned table gradient");
    NVQ_REQUIRE(T == 0 || (d_dout && d_ids && nvq_aligned(d_dout, size) && nvq_aligned(d_ids, 4)),
                "nvq_embedding_bwd: null or misaligned buffer");
    const BwdSpace sp = bwd_space(T, D);
    NVQ_REQUIRE(T == 0 || (d_workspace && workspace_bytes >= sp.total && nvq_aligned(d_workspace, 256)),
                "nvq_embedding_bwd: workspace of %zu bytes (256-byte aligned) required", sp.total);
    nvq_status s = nvq_use_device(device);
    if (s != NVQ_OK) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        if (!accumulate) NVQ_CUDA(cudaMemsetAsync(d_dtable, 0, V * D * sizeof(float), st));
        return NVQ_OK;
    }
    int* status = nullptr;
    s = nvq_status_word(device, &status);
    if (s != NVQ_OK) return s;
    if (T <= (size_t)FEW_TOKENS && (accumulate || V <= FEW_VOCAB)) {
        const int t = (int)T, v = (int)V, d = (int)D;
        if (dout_dtype == NVQ_F32)
            return few_tokens_of<NVQ_F32>(d_dtable, d_dout, d_ids, t, v, d, scale, padding_id, accumulate, status, device, st);
        if (dout_dtype == NVQ_F16)
            return few_tokens_of<NVQ_F16>(d_dtable, d_dout, d_ids, t, v, d, scale, padding_id, accumulate, status, device, st);
        return few_tokens_of<NVQ_BF16>(d_dtable, d_dout, d_ids, t, v, d, scale, padding_id, accumulate, status, device, st);
    }
    static std::atomic<int> clusters[64];    // per device: sorting clusters that run at once (found twice: harmless)
    if (!clusters[device]) {
        NVQ_CUDA(cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)sizeof(SortShared)));
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = sort_launch(MAX_CLUSTER, MAX_CLUSTER, st, attr);
        int n = 0;
        NVQ_CUDA(cudaOccupancyMaxActiveClusters(&n, sort_tokens_kernel, &cfg));
        clusters[device] = n < 2 ? 2 : n;
    }
    int32_t* sid = (int32_t*)d_workspace;
    int32_t* spos = (int32_t*)((char*)d_workspace + sp.ids);
    float* carry = (float*)((char*)d_workspace + sp.ids + sp.pos);
    int value_bits = 1;
    while (((size_t)1 << value_bits) <= V) value_bits++;      // V itself marks a token that takes no part
    // more tokens than one cluster sorts: one part after the other, each adding to the table
    for (size_t t0 = 0; t0 < T; t0 += SORT_MAX) {
        const int n = (int)(T - t0 < (size_t)SORT_MAX ? T - t0 : SORT_MAX);
        const int add = accumulate || t0 > 0;
        SortParams q;
        q.ids = d_ids + t0;
        q.sorted_id = sid;
        q.sorted_pos = spos;
        q.n = n;
        q.vocab = (int)V;
        q.padding_id = padding_id;
        q.passes = (value_bits + MAX_BITS - 1) / MAX_BITS;
        q.bits = (value_bits + q.passes - 1) / q.passes;
        q.clear = add ? nullptr : d_dtable;
        q.D = (int)D;
        // Finding the used rows costs the clearing clusters a pass over the ids, leaving them out saves their bytes: worth
        // it for rows of 1024 floats and more, with two bits per row in shared memory (and only where this part's
        // tokens are all there are: later parts add to rows that have to be 0).
        q.skip_used = D >= 1024 && V <= sizeof(SortShared) * 4 - 64 && T <= (size_t)SORT_MAX;
        q.status = status;
        const int ctas = n <= SORT_THREADS ? 1 : MAX_CLUSTER;      // the last part of many may be short
        q.chunk_log2 = 5;
        while (((size_t)ctas << q.chunk_log2) < (size_t)n) q.chunk_log2++;
        // Further clusters clear the table: as many as run beside the sorting one (128 of 148 SMs take clusters of eight;
        // with a second wave of them a 410 MB table took 90 us instead of 67), fewer for a small one.
        size_t clearing = add ? 0 : (V * D + 32767) / 32768;
        const size_t most = (size_t)(ctas == 1 ? nvq_sm_count(device) : clusters[device].load() * ctas) - ctas;
        if (clearing > most) clearing = most;
        clearing = (clearing + ctas - 1) / ctas * ctas;
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = sort_launch(ctas + clearing, ctas, st, attr);
        NVQ_CUDA(cudaLaunchKernelEx(&cfg, sort_tokens_kernel, q));
        NVQ_LAUNCHED();
        const char* part = (const char*)d_dout + t0 * D * size;
        if (dout_dtype == NVQ_F32)
            s = sum_runs<NVQ_F32>(d_dtable, carry, part, sid, spos, n, (int)V, (int)D, scale, add, st);
        else if (dout_dtype == NVQ_F16)
            s = sum_runs<NVQ_F16>(d_dtable, carry, part, sid, spos, n, (int)V, (int)D, scale, add, st);
        else
            s = sum_runs<NVQ_BF16>(d_dtable, carry, part, sid, spos, n, (int)V, (int)D, scale, add, st);
        if (s != NVQ_OK) return s;
    }
    return NVQ_OK;
}
