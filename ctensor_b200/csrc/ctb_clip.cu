// The norm of all gradients of a model, and scaling them down to a given norm.
//
//   N = (sum over all tensors and elements of |g|^p)^(1/p), p = 1, 2 or infinity;
//   g <- g * (max_norm / N)   if max_norm < N < infinity, else g as it is.
//
// Two launches for every 1024 tensors: the first leaves one fp64 partial per block, every block of the second
// folds all partials in the same order (so all of them agree on the factor bit for bit, with no atomics and
// no block that waits for another) and scales.
// The list of tensors travels in the kernel's arguments: nothing is copied ahead of the launch and a
// captured graph keeps its own list.
//
// Bound by HBM: 4 bytes per Float32 element for the norm and 8 more where the gradients have to be
// scaled (what the first launch read last is still in L2 and is scaled first).  Measured: 1.07 billion
// gradients in 193 tensors, scaled out of place, 1965 us = 6.55 TB/s over 12 bytes per element; the norm of
// 202 million alone 122 us = 6.6 TB/s; four small tensors 6.2 us, two launches; 196
// tensors of 1 to 140000 values, side by side at every alignment, 10.7 us; 50 million values, the two sides at
// different alignments, 131 us.  Squares and sums are fp64: a
// square of an fp32 value neither overflows nor vanishes there.
#include "ctb_clip.cuh"
#include "ctb_team.cuh"

namespace ctb {

namespace {

constexpr int kClipThreads = 256;
constexpr int kClipLoads = 8;                            // 32-byte loads in flight per thread
constexpr int kClipVecBytes = 32;
constexpr int kClipRagged = 4;                           // and in a tensor's ragged first or last chunk
constexpr int kClipApart = 16;                           // elements in flight per thread where two sides differ in alignment
constexpr int kClipChunkBytes = kClipThreads * kClipLoads * kClipVecBytes;      // 64 KiB
// Resident blocks: eight loads a thread and three blocks read 202 million gradients in 122 us, four loads and five or
// six blocks in 130 and 140 (spilled sums), eight and four in 127.  The scaling pass, which stores as well, is
// launched with four blocks an SM and its registers left free: bounding them to four spills (2034 us for 1.07 billion).
constexpr int kNormBlocksPerSm = 3, kScaleBlocksPerSm = 4;
constexpr int kClipMaxBlocks = 1024;                     // partials of one launch
// Tables: every launch carries a whole one, 28 bytes an entry (300 tiny tensors with 1024 entries 11.5 us).
constexpr int kClipSmallTable = 128, kClipMidTable = 384, kClipLargeTable = 1024;

// Tensors of one launch.  Tensor t is cut into chunks of 64 KiB counted from its first element's
// address rounded down to 32 bytes, so that all vector accesses are aligned wherever it starts;
// `first[t]` is its first chunk's number, first[count] the number of chunks.
template <int N>
struct ClipTable {
    const void* src[N];
    void* dst[N];
    int64_t n[N];
    uint32_t first[N + 1];
    int32_t count;
};

template <typename T> struct ClipVec { static constexpr int kElems = kClipVecBytes / (int)sizeof(T); };

// ---- folding ------------------------------------------------------------------------------------------
// The running value is a double; for the maximum it holds the bits of |g|, compared as integers,
// which orders non-negative numbers like their values and puts NaN above infinity: a NaN survives.
template <int KIND> __device__ __forceinline__ double clip_fold(double acc, double v) {
    if (KIND == kNormInf) {
        const unsigned long long a = (unsigned long long)__double_as_longlong(acc), b = (unsigned long long)__double_as_longlong(v);
        return a > b ? acc : v;
    }
    return __dadd_rn(acc, v);
}
template <int KIND> __device__ __forceinline__ double clip_term(double acc, double g) {
    if (KIND == kNormP2) return fma(g, g, acc);
    return clip_fold<KIND>(acc, fabs(g));
}

// Fold over the block; the result is valid in every thread.
template <int KIND> __device__ __forceinline__ double clip_block_fold(double v, double* smem) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = clip_fold<KIND>(v, __shfl_xor_sync(0xffffffffu, v, off));
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    double r = smem[0];
#pragma unroll
    for (int i = 1; i < kClipThreads / 32; ++i) r = clip_fold<KIND>(r, smem[i]);
    return r;
}

// The vector at `p`, zeros where that lies outside [lo, hi); and its way back.
template <typename T> __device__ __forceinline__ Vec<T, ClipVec<T>::kElems> clip_load_some(const T* src, int64_t p, int64_t lo, int64_t hi) {
    constexpr int VEC = ClipVec<T>::kElems;
    Vec<T, VEC> v;
    if (p >= lo && p + VEC <= hi) {
        v = ldg_stream(reinterpret_cast<const Vec<T, VEC>*>(src + p));
    } else {
        const bool some = p + VEC > lo && p < hi;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v.v[k] = some && p + k >= lo && p + k < hi ? src[p + k] : (T)0;
    }
    return v;
}
template <typename T> __device__ __forceinline__ void clip_store_some(T* dst, int64_t p, int64_t lo, int64_t hi, const Vec<T, ClipVec<T>::kElems>& v) {
    constexpr int VEC = ClipVec<T>::kElems;
    if (p >= lo && p + VEC <= hi) {
        stg_stream(reinterpret_cast<Vec<T, VEC>*>(dst + p), v);
    } else if (p + VEC > lo && p < hi) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (p + k >= lo && p + k < hi) dst[p + k] = v.v[k];
    }
}

// The chunks of one block: [lo, hi).
__device__ __forceinline__ void clip_range(uint32_t chunks, uint32_t* lo, uint32_t* hi) {
    *lo = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x);
    *hi = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
}
// The tensor that chunk `c` belongs to.
template <int N> __device__ __forceinline__ int clip_tensor_of(const ClipTable<N>& t, uint32_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int KIND, typename T, int N>
__global__ void __launch_bounds__(kClipThreads, kNormBlocksPerSm)
clip_norm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ partials) {
    constexpr int VEC = ClipVec<T>::kElems;
    using V = Vec<T, VEC>;
    __shared__ double smem[kClipThreads / 32];
    uint32_t c, hi;
    clip_range(t.first[t.count], &c, &hi);
    double acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.0;
    int which = c < hi ? clip_tensor_of(t, c) : 0;
    for (; c < hi; ++c) {
        while (c >= t.first[which + 1]) ++which;
        const T* src = (const T*)t.src[which];
        const int phase = (int)(((uintptr_t)src % kClipVecBytes) / sizeof(T));
        const int64_t end = t.n[which] + phase;                        // in elements from the rounded address
        src -= phase;
        const int64_t at = (int64_t)(c - t.first[which]) * (kClipChunkBytes / (int)sizeof(T)) + (int64_t)threadIdx.x * VEC;
        const int64_t chunk_end = (int64_t)(c - t.first[which] + 1) * (kClipChunkBytes / (int)sizeof(T));
        if (chunk_end <= end && (phase == 0 || c != t.first[which])) {
            V v[kClipLoads];
#pragma unroll
            for (int i = 0; i < kClipLoads; ++i) v[i] = ldg_stream(reinterpret_cast<const V*>(src + at + i * (kClipThreads * VEC)));
#pragma unroll
            for (int i = 0; i < kClipLoads; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[k] = clip_term<KIND>(acc[k], (double)v[i].v[k]);
        } else {                                                       // a tensor's ragged first or last chunk
#pragma unroll 1
            for (int64_t p = at; p < end; p += kClipRagged * kClipThreads * VEC) {
                if (p >= chunk_end) break;
                V v[kClipRagged];
#pragma unroll
                for (int i = 0; i < kClipRagged; ++i) v[i] = clip_load_some<T>(src, p + i * (kClipThreads * VEC), phase, end);
#pragma unroll
                for (int i = 0; i < kClipRagged; ++i)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] = clip_term<KIND>(acc[k], (double)v[i].v[k]);
            }
        }
    }
    let_next_start();
    double sum = acc[0];
#pragma unroll
    for (int k = 1; k < VEC; ++k) sum = clip_fold<KIND>(sum, acc[k]);
    sum = clip_block_fold<KIND>(sum, smem);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// Fold of all partials, in the same order in every block of every launch.
template <int KIND> __device__ __forceinline__ double clip_total(const double* partials, int count, double* smem) {
    double v = 0.0;
    for (int i = threadIdx.x; i < count; i += kClipThreads) v = clip_fold<KIND>(v, partials[i]);
    v = clip_block_fold<KIND>(v, smem);
    return KIND == kNormP2 ? sqrt(v) : v;
}
__device__ __forceinline__ void clip_store_norm(double total, void* norm, int norm_dtype) {
    if (norm_dtype == CTB_F64) *(double*)norm = total;
    else *(float*)norm = (float)total;
}

template <int KIND>
__global__ void __launch_bounds__(kClipThreads)
clip_finish_kernel(const double* __restrict__ partials, int count, void* norm, int norm_dtype) {
    __shared__ double smem[kClipThreads / 32];
    wait_for_previous();
    const double total = clip_total<KIND>(partials, count, smem);
    if (threadIdx.x == 0) clip_store_norm(total, norm, norm_dtype);
}

// The factor is rounded to T once (the product once more): two roundings of 2^-24 for Float32.  A factor so small that T
// would hold it with fewer bits, or as 0, is applied in fp64 in two steps, of which the first is exact.
template <typename T> __device__ __forceinline__ double clip_smallest() { return sizeof(T) == 4 ? 0x1p-100 : 0x1p-960; }
template <int KIND, typename T, int N>
__global__ void __launch_bounds__(kClipThreads)
clip_scale_kernel(const __grid_constant__ ClipTable<N> t, const double* __restrict__ partials, int count, double max_norm,
                  void* norm, int norm_dtype) {
    constexpr int VEC = ClipVec<T>::kElems;
    constexpr int CHUNK = kClipChunkBytes / (int)sizeof(T);
    using V = Vec<T, VEC>;
    __shared__ double smem[kClipThreads / 32];
    wait_for_previous();
    const double total = clip_total<KIND>(partials, count, smem);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) clip_store_norm(total, norm, norm_dtype);
    const bool clipped = total > max_norm && total < INFINITY;
    const T factor = clipped ? (T)(max_norm / total) : (T)1;
    const bool tiny = clipped && max_norm / total < clip_smallest<T>();
    const double rest = max_norm * 0x1p512 / total;
    uint32_t lo, c;
    clip_range(t.first[t.count], &lo, &c);
    int which = lo < c ? clip_tensor_of(t, c - 1) : 0;
    // last chunk first: what the first launch read last is what L2 still holds
    while (c > lo) {
        --c;
        while (c < t.first[which]) --which;
        const T* src = (const T*)t.src[which];
        T* dst = (T*)t.dst[which];
        if (!clipped && dst == src) continue;
        const int phase = (int)(((uintptr_t)src % kClipVecBytes) / sizeof(T));
        const int64_t end = t.n[which] + phase;
        const bool together = ((uintptr_t)dst % kClipVecBytes) / sizeof(T) == (uintptr_t)phase;
        src -= phase;
        dst -= phase;
        const int64_t begin = (int64_t)(c - t.first[which]) * CHUNK;
        if (!together || tiny) {                            // other alignment on the two sides: element by element
            const int64_t stop = begin + CHUNK < end ? begin + CHUNK : end;
            for (int64_t p = begin + threadIdx.x; p < stop; p += kClipThreads * kClipApart) {
                T v[kClipApart];
#pragma unroll
                for (int i = 0; i < kClipApart; ++i) v[i] = p + i * kClipThreads >= phase && p + i * kClipThreads < stop ? src[p + i * kClipThreads] : (T)0;
#pragma unroll
                for (int i = 0; i < kClipApart; ++i)
                    if (p + i * kClipThreads >= phase && p + i * kClipThreads < stop)
                        dst[p + i * kClipThreads] = tiny ? (T)((double)v[i] * 0x1p-512 * rest) : clipped ? v[i] * factor : v[i];
            }
            continue;
        }
        const int64_t at = begin + (int64_t)threadIdx.x * VEC;
        if (begin + CHUNK <= end && (phase == 0 || begin > 0)) {
            V v[kClipLoads];
#pragma unroll
            for (int i = 0; i < kClipLoads; ++i) v[i] = ldg_stream(reinterpret_cast<const V*>(src + at + i * (kClipThreads * VEC)));
#pragma unroll
            for (int i = 0; i < kClipLoads; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[i].v[k] = v[i].v[k] * factor;
                stg_stream(reinterpret_cast<V*>(dst + at + i * (kClipThreads * VEC)), v[i]);
            }
        } else {
#pragma unroll 1
            for (int64_t p = at; p < end; p += kClipRagged * kClipThreads * VEC) {
                if (p >= begin + CHUNK) break;
                V v[kClipRagged];                           // loads ahead of stores: these may be to the same tensor
#pragma unroll
                for (int i = 0; i < kClipRagged; ++i) v[i] = clip_load_some<T>(src, p + i * (kClipThreads * VEC), phase, end);
#pragma unroll
                for (int i = 0; i < kClipRagged; ++i) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[i].v[k] = v[i].v[k] * factor;
                    clip_store_some<T>(dst, p + i * (kClipThreads * VEC), phase, end, v[i]);
                }
            }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------
template <typename T> int64_t clip_chunks(const ClipTensor& t) {
    const int64_t phase = (int64_t)(((uintptr_t)t.src % kClipVecBytes) / sizeof(T));
    return t.n == 0 ? 0 : ceil_div(phase + t.n, (int64_t)(kClipChunkBytes / (int)sizeof(T)));
}

template <typename T, int N>
int clip_fill(ClipTable<N>* table, const ClipTensor* list, int64_t count) {
    int64_t chunks = 0;
    table->count = (int32_t)count;
    for (int64_t i = 0; i < count; ++i) {
        table->src[i] = list[i].src;
        table->dst[i] = list[i].dst;
        table->n[i] = list[i].n;
        table->first[i] = (uint32_t)chunks;
        chunks += clip_chunks<T>(list[i]);
        if (chunks > 0x7FFFFFFFll) return set_error(CTB_ERR_LIMIT, "clip_grad_norm: too many elements for one launch");
    }
    table->first[count] = (uint32_t)chunks;
    return CTB_OK;
}

// One block per SM slot, never more blocks than chunks (and at least one, which writes its partial).
unsigned clip_grid(uint32_t chunks, int sm_count, int per_sm) {
    int64_t g = (int64_t)sm_count * per_sm;
    if (g > kClipMaxBlocks) g = kClipMaxBlocks;
    if (g > chunks) g = chunks;
    return (unsigned)(g < 1 ? 1 : g);
}

struct ClipCall {
    double* partials;
    int total_partials;       // of all launches of the first phase
    double max_norm;
    void* norm;
    int norm_dtype;
    int sm_count;
    cudaStream_t st;
};

template <int KIND, typename T, int N>
int clip_launch_table(int phase, const ClipTensor* list, int64_t count, ClipCall& call) {
    ClipTable<N> table;
    if (int rc = clip_fill<T, N>(&table, list, count)) return rc;
    const unsigned grid = clip_grid(table.first[count], call.sm_count, phase == 0 ? kNormBlocksPerSm : kScaleBlocksPerSm);
    if (phase == 0) {
        clip_norm_kernel<KIND, T, N><<<grid, kClipThreads, 0, call.st>>>(table, call.partials + call.total_partials);
        call.total_partials += (int)grid;
    } else {
        // (a second scaling launch may start early too: it waits for the first, which waited for the norm)
        const int rc = launch_early(clip_scale_kernel<KIND, T, N>, grid, kClipThreads, call.st, table, call.partials, call.total_partials, call.max_norm, call.norm, call.norm_dtype);
        call.norm = nullptr;                                // written once
        return rc;
    }
    return cuda_error(cudaGetLastError(), "clip_grad_norm launch");
}

template <int KIND, typename T>
int clip_phase(int phase, const ClipTensor* list, int64_t count, ClipCall& call) {
    for (int64_t at = 0; at < count; at += kClipLargeTable) {
        const int64_t n = count - at < kClipLargeTable ? count - at : kClipLargeTable;
        const int rc = n <= kClipSmallTable ? clip_launch_table<KIND, T, kClipSmallTable>(phase, list + at, n, call)
                       : n <= kClipMidTable ? clip_launch_table<KIND, T, kClipMidTable>(phase, list + at, n, call)
                                            : clip_launch_table<KIND, T, kClipLargeTable>(phase, list + at, n, call);
        if (rc) return rc;
    }
    return CTB_OK;
}

template <int KIND>
int clip_run(const ClipTensor* t32, int64_t n32, const ClipTensor* t64, int64_t n64, int scale, ClipCall& call) {
    int rc;
    if ((rc = clip_phase<KIND, float>(0, t32, n32, call))) return rc;
    if ((rc = clip_phase<KIND, double>(0, t64, n64, call))) return rc;
    if (scale) {
        if ((rc = clip_phase<KIND, float>(1, t32, n32, call))) return rc;
        if ((rc = clip_phase<KIND, double>(1, t64, n64, call))) return rc;
    }
    if (call.norm) {                                        // no scaling launch wrote it
        return launch_early(clip_finish_kernel<KIND>, 1, kClipThreads, call.st, call.partials, call.total_partials, call.norm, call.norm_dtype);
    }
    return CTB_OK;
}

}  // namespace

size_t clip_workspace_bytes(int64_t n32, int64_t n64) {
    const int64_t launches = ceil_div(n32, (int64_t)kClipLargeTable) + ceil_div(n64, (int64_t)kClipLargeTable);
    return (size_t)launches * kClipMaxBlocks * sizeof(double);
}

int launch_clip(int kind, const ClipTensor* t32, int64_t n32, const ClipTensor* t64, int64_t n64, int scale,
                double max_norm, void* norm, int norm_dtype, void* workspace, cudaStream_t stream) {
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    ClipCall call{(double*)workspace, 0, max_norm, norm, norm_dtype, di.sm_count, stream};
    switch (kind) {
    case kNormP1: return clip_run<kNormP1>(t32, n32, t64, n64, scale, call);
    case kNormInf: return clip_run<kNormInf>(t32, n32, t64, n64, scale, call);
    default: return clip_run<kNormP2>(t32, n32, t64, n64, scale, call);
    }
}

}  // namespace ctb
