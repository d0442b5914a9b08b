// The norm of many gradient tensors taken as one vector, and the clipping by it.
//
//   norm = sqrt(sum over tensors, sum over elements of g^2)
//   coef = 1 if norm <= max_norm, else max_norm / norm;   out = g * coef
//
// Both kernels walk one list of chunks of 32 KB; a chunk lies in one tensor and belongs to a fixed block (the
// blocks take neighbouring chunks at the same time, which is what DRAM likes best), so that the sum is always added in the same order (equal inputs give equal bits)
// and nothing is counted by atomics.  The tensor list travels in the kernel's parameters: no copy
// to the device, and a captured graph keeps its own.  Squares are added in fp64 (one conversion and
// one fused multiply-add per element, which the memory rate leaves room for): no gradient that fits
// its type overflows the sum or falls out of it, as fp32 squares above 1.8e19 and below 1e-23 would.
#include "packet.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int CHUNK_BYTES = 32768;     // 128 per thread: four 32-byte loads (16 KB: 3 % slower at 577 M fp32, 7 % at 234 M bf16)
constexpr int BLOCKS_PER_SM = 8;       // of the first kernel; four made fp32 4 % faster and bf16 11 % slower
constexpr int MAX_BLOCKS = 148 * BLOCKS_PER_SM;
constexpr int CLIP_BLOCKS_PER_SM = 4, MAX_CLIP_BLOCKS = 148 * CLIP_BLOCKS_PER_SM;

template <int NT>
struct TensorList {
    const void* src[NT];
    void* dst[NT];
    unsigned long long count[NT];
    uint32_t first[NT + 1];     // chunk number at which the tensor starts
    uint8_t dtype[NT];
    uint8_t vec[NT];            // src and dst lie alike within 32 bytes
    int n;
};

template <int NT>
__device__ __forceinline__ int find_tensor(const TensorList<NT>& L, uint32_t chunk) {
    int lo = 0, hi = L.n - 1;   // the last tensor whose first chunk is <= chunk (empty tensors own none)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (L.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) s += sh[i];
    return s;
}

__host__ __device__ constexpr int elem_size(int dt) { return dt == NVQ_F64 ? 8 : (dt == NVQ_F32 ? 4 : 2); }
__host__ __device__ constexpr int chunk_elems(int dt) { return CHUNK_BYTES / elem_size(dt); }

__device__ __forceinline__ u32x8 ld256(const void* p) {
    u32x8 r;
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]),
                   "=r"(r.v[7])
                 : "l"(p)
                 : "memory");
    return r;
}

// Calls wide(i) for every 32-byte packet of a chunk of n elements at p (pairs(i, i + THREADS) where both exist) and
// one(k) for the elements before the first and after the last of them.
template <int SIZE, typename Pairs, typename Wide, typename One>
__device__ __forceinline__ void walk(const void* p, int n, bool vec, Pairs pairs, Wide wide, One one) {
    constexpr int V = 32 / SIZE;
    const int head = vec ? min(n, (int)((32 - ((uintptr_t)p & 31)) & 31) / SIZE) : n;
    const int packets = (n - head) / V, tail = head + packets * V;
    int i = threadIdx.x;
    for (; i + THREADS < packets; i += 2 * THREADS) pairs(head, i, i + THREADS);
    if (i < packets) wide(head, i);
    for (int k = threadIdx.x; k < head; k += THREADS) one(k);
    for (int k = tail + threadIdx.x; k < n; k += THREADS) one(k);
}

// sum of squares of a chunk of n elements at p, this thread's share
template <int DT>
__device__ __forceinline__ double chunk_squares(const char* p, int n, bool vec) {
    using E = Elem<DT>;
    double s = 0.0;
    auto add = [&](const u32x8& q) {
#pragma unroll
        for (int w = 0; w < 8; w++) {
            float f[2];
            E::widen(q.v[w], f);
#pragma unroll
            for (int j = 0; j < E::PER_WORD; j++) s = fma((double)f[j], (double)f[j], s);
        }
    };
    walk<E::SIZE>(
        p, n, vec,
        [&](int h, int i, int k) {
            const u32x8 a = ld256(p + h * E::SIZE + i * 32), b = ld256(p + h * E::SIZE + k * 32);
            add(a);
            add(b);
        },
        [&](int h, int i) { add(ld256(p + h * E::SIZE + i * 32)); },
        [&](int k) {
            const double f = (double)E::load(p + k * E::SIZE);
            s = fma(f, f, s);
        });
    return s;
}
__device__ __forceinline__ double chunk_squares_f64(const double* p, int n) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) s = fma(p[i], p[i], s);
    return s;
}

// partial[block] = (add ? partial[block] : 0) + the block's share of the sum of squares
template <int NT>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
square_sum_kernel(const __grid_constant__ TensorList<NT> L, double* __restrict__ partial, uint32_t chunks, int add) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the next kernel is set up, and waits
    __shared__ double sh[THREADS / 32];
    double s = 0.0;
    int t = 0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        if (c >= L.first[t + 1]) t = find_tensor(L, c);
        const int dt = L.dtype[t];
        const size_t at = (size_t)(c - L.first[t]) * chunk_elems(dt);
        const int n = (int)min((unsigned long long)chunk_elems(dt), L.count[t] - at);
        const char* p = (const char*)L.src[t] + at * elem_size(dt);
        if (dt == NVQ_F32) s += chunk_squares<NVQ_F32>(p, n, L.vec[t]);
        else if (dt == NVQ_BF16) s += chunk_squares<NVQ_BF16>(p, n, L.vec[t]);
        else if (dt == NVQ_F16) s += chunk_squares<NVQ_F16>(p, n, L.vec[t]);
        else s += chunk_squares_f64((const double*)p, n);
    }
    s = block_sum(s, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = (add ? partial[blockIdx.x] : 0.0) + s;
}

// norm and coefficient from the partial sums, the same additions in the same order in every block
__device__ __forceinline__ double total_norm(const double* __restrict__ partial, int blocks, double* sh) {
    double s = 0.0;
    for (int i = threadIdx.x; i < blocks; i += THREADS) s += partial[i];
    return sqrt(block_sum(s, sh));
}
// A NaN norm is not <= max_norm, so it makes the coefficient, and every clipped gradient, NaN; an
// infinite one makes the coefficient 0 (and the infinite gradients themselves NaN).
__device__ __forceinline__ double clip_coef(double norm, double max_norm) {
    return norm <= max_norm ? 1.0 : max_norm / norm;
}

__global__ void __launch_bounds__(THREADS)
norm_kernel(float* __restrict__ out, const double* __restrict__ partial, int blocks, double max_norm) {
    __shared__ double sh[THREADS / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const double norm = total_norm(partial, blocks, sh);
    if (threadIdx.x == 0) {
        out[0] = (float)norm;
        out[1] = (float)clip_coef(norm, max_norm);
    }
}

template <int DT>
__device__ __forceinline__ void chunk_scale(char* d, const char* p, int n, bool vec, float coef) {
    using E = Elem<DT>;
    auto cut = [&](u32x8 q, char* to) {
#pragma unroll
        for (int w = 0; w < 8; w++) {
            float f[2];
            E::widen(q.v[w], f);
#pragma unroll
            for (int j = 0; j < E::PER_WORD; j++) f[j] *= coef;
            q.v[w] = E::narrow(f);
        }
        stg_stream_256(to, q);
    };
    walk<E::SIZE>(
        p, n, vec,
        [&](int h, int i, int k) {
            const u32x8 a = ld256(p + h * E::SIZE + i * 32), b = ld256(p + h * E::SIZE + k * 32);
            cut(a, d + h * E::SIZE + i * 32);
            cut(b, d + h * E::SIZE + k * 32);
        },
        [&](int h, int i) { cut(ld256(p + h * E::SIZE + i * 32), d + h * E::SIZE + i * 32); },
        [&](int k) { E::store(d + k * E::SIZE, E::load(p + k * E::SIZE) * coef); });
}

// Every block adds the (at most 1184) partial sums up again, which costs less than a launch between
// the two kernels.  The chunks are walked backwards: the ones that the first kernel read last are those that
// still lie in L2 (160 MB of fp32: 47 us against 51 forwards).
template <int NT>
__global__ void __launch_bounds__(THREADS, CLIP_BLOCKS_PER_SM)
clip_kernel(const __grid_constant__ TensorList<NT> L, float* __restrict__ out, const double* __restrict__ partial,
            int blocks, double max_norm, uint32_t chunks) {
    __shared__ double sh[THREADS / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const double norm = total_norm(partial, blocks, sh);
    const double coef64 = clip_coef(norm, max_norm);
    const float coef = (float)coef64;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        out[0] = (float)norm;
        out[1] = coef;
    }
    int t = L.n - 1;
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t c = chunks - 1 - k;
        if (c < L.first[t]) t = find_tensor(L, c);
        const int dt = L.dtype[t];
        const size_t at = (size_t)(c - L.first[t]) * chunk_elems(dt);
        const int n = (int)min((unsigned long long)chunk_elems(dt), L.count[t] - at);
        const char* p = (const char*)L.src[t] + at * elem_size(dt);
        char* d = (char*)L.dst[t] + at * elem_size(dt);
        if (coef64 == 1.0 && p == d) continue;      // in place and nothing to cut
        if (dt == NVQ_F32) chunk_scale<NVQ_F32>(d, p, n, L.vec[t], coef);
        else if (dt == NVQ_BF16) chunk_scale<NVQ_BF16>(d, p, n, L.vec[t], coef);
        else if (dt == NVQ_F16) chunk_scale<NVQ_F16>(d, p, n, L.vec[t], coef);
        else
            for (int i = threadIdx.x; i < n; i += THREADS) ((double*)d)[i] = ((const double*)p)[i] * coef64;
    }
}

template <typename... KArgs, typename... Args>
void launch_after(void (*kernel)(KArgs...), int grid, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// The tensors [begin, n) from which the list takes as many as it holds; returns the first one left.
template <int NT>
size_t fill(TensorList<NT>& L, const void* const* src, void* const* dst, const size_t* counts, const int32_t* dtypes,
            size_t begin, size_t n, uint32_t* chunks) {
    uint64_t total = 0;
    L.n = 0;
    size_t t = begin;
    for (; t < n && L.n < NT; t++) {
        if (counts[t] == 0) continue;
        const uint64_t each = chunk_elems(dtypes[t]), c = (counts[t] + each - 1) / each;
        if (total + c > 0x7FFFFFFFull) break;
        L.src[L.n] = src[t];
        L.dst[L.n] = dst ? dst[t] : const_cast<void*>(src[t]);
        L.count[L.n] = counts[t];
        L.first[L.n] = (uint32_t)total;
        L.dtype[L.n] = (uint8_t)dtypes[t];
        L.vec[L.n] = !dst || ((uintptr_t)src[t] & 31) == ((uintptr_t)dst[t] & 31);
        total += c;
        L.n++;
    }
    L.first[L.n] = (uint32_t)total;
    *chunks = (uint32_t)total;
    return t;
}

int blocks_for(uint32_t chunks, int most) { return chunks < (uint32_t)most ? (int)chunks : most; }

// Few tensors take the short list (2 KB of parameters); more take lists of up to 1024.
constexpr int SHORT_LIST = 64, LONG_LIST = 1000;

template <int NT>
nvq_status run_lists(float* d_out, void* const* dst, const void* const* src, const size_t* counts,
                     const int32_t* dtypes, size_t n, double max_norm, double* partial, bool clip, cudaStream_t st) {
    TensorList<NT> L;
    uint32_t chunks = 0;
    int blocks = 0;
    for (size_t t = 0; t < n;) {
        t = fill(L, src, dst, counts, dtypes, t, n, &chunks);
        if (chunks == 0) break;
        const int grid = blocks_for(chunks, MAX_BLOCKS);
        // a later list adds to the partial sums of the first ones, block by block
        if (blocks && blocks < grid)
            NVQ_CUDA(cudaMemsetAsync(partial + blocks, 0, (grid - blocks) * sizeof(double), st));
        square_sum_kernel<NT><<<grid, THREADS, 0, st>>>(L, partial, chunks, blocks != 0);
        NVQ_LAUNCHED();
        if (grid > blocks) blocks = grid;
    }
    if (!clip || blocks == 0) {
        launch_after(norm_kernel, 1, st, d_out, (const double*)partial, blocks, max_norm);
        NVQ_LAUNCHED();
        return NVQ_OK;
    }
    for (size_t t = 0; t < n;) {
        t = fill(L, src, dst, counts, dtypes, t, n, &chunks);
        if (chunks == 0) break;
        launch_after(clip_kernel<NT>, blocks_for(chunks, MAX_CLIP_BLOCKS), st, L, d_out, (const double*)partial, blocks,
                     max_norm, chunks);
        NVQ_LAUNCHED();
    }
    return NVQ_OK;
}

nvq_status run(const char* who, float* d_out, void* const* dst, const void* const* src, const size_t* counts,
               const int32_t* dtypes, size_t n, double max_norm, void* ws, size_t ws_bytes, bool clip, int device,
               void* stream) {
    NVQ_REQUIRE(d_out && nvq_aligned(d_out, 4), "%s: null or misaligned output", who);
    NVQ_REQUIRE(n == 0 || (src && counts && dtypes), "%s: null tensor list", who);
    NVQ_REQUIRE(max_norm > 0.0, "%s: max_norm must be above 0", who);
    NVQ_REQUIRE(ws && nvq_aligned(ws, 8) && ws_bytes >= MAX_BLOCKS * sizeof(double),
                "%s: workspace of %zu bytes (8-byte aligned) required", who, MAX_BLOCKS * sizeof(double));
    size_t used = 0;
    for (size_t t = 0; t < n; t++) {
        const int32_t dt = dtypes[t];
        NVQ_REQUIRE(dt == NVQ_F32 || dt == NVQ_F16 || dt == NVQ_BF16 || dt == NVQ_F64,
                    "%s: tensor %zu has type %d; f32, f16, bf16 and f64 are taken", who, t, (int)dt);
        if (counts[t] == 0) continue;
        NVQ_REQUIRE(counts[t] < ((size_t)1 << 42), "%s: tensor %zu is too large", who, t);
        NVQ_REQUIRE(src[t] && nvq_aligned(src[t], elem_size(dt)), "%s: tensor %zu is null or misaligned", who, t);
        NVQ_REQUIRE(!dst || (dst[t] && nvq_aligned(dst[t], elem_size(dt))), "%s: output %zu is null or misaligned",
                    who, t);
        used++;
    }
    nvq_status s = nvq_use_device(device);
    if (s != NVQ_OK) return s;
    cudaStream_t st = (cudaStream_t)stream;
    if (used <= SHORT_LIST)
        return run_lists<SHORT_LIST>(d_out, dst, src, counts, dtypes, n, max_norm, (double*)ws, clip, st);
    return run_lists<LONG_LIST>(d_out, dst, src, counts, dtypes, n, max_norm, (double*)ws, clip, st);
}

}  // namespace

extern "C" nvq_status nvq_grad_norm_workspace_bytes(size_t* bytes) {
    NVQ_REQUIRE(bytes, "null out pointer");
    *bytes = MAX_BLOCKS * sizeof(double);
    return NVQ_OK;
}

extern "C" nvq_status nvq_grad_norm(float* d_norm_coef, const void* const* h_grads, const size_t* h_counts,
                                    const int32_t* h_dtypes, size_t n_tensors, double max_norm, void* d_workspace,
                                    size_t workspace_bytes, int device, void* stream) {
    return run("nvq_grad_norm", d_norm_coef, nullptr, h_grads, h_counts, h_dtypes, n_tensors, max_norm, d_workspace,
               workspace_bytes, false, device, stream);
}

extern "C" nvq_status nvq_clip_grads(float* d_norm_coef, void* const* h_out, void* const* h_grads,
                                     const size_t* h_counts, const int32_t* h_dtypes, size_t n_tensors,
                                     double max_norm, void* d_workspace, size_t workspace_bytes, int device,
                                     void* stream) {
    return run("nvq_clip_grads", d_norm_coef, h_out, (const void* const*)h_grads, h_counts, h_dtypes, n_tensors,
               max_norm, d_workspace, workspace_bytes, true, device, stream);
}
