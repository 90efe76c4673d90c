// Teams of threads that own one row: a warp, several warps of a CTA, a CTA, or the CTAs of a thread-block
// cluster.  Folds over a team give every thread the same bits.
#pragma once
#include "ctb_common.cuh"

namespace ctb {

constexpr int kMaxCluster = 8;                           // portable cluster size

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
    cluster_arrive();
    cluster_wait();
}
// The address of this CTA's shared object `p` in the CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_shared(const void* p, uint32_t rank) {
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(p);
    uint32_t theirs;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(mine), "r"(rank));
    return theirs;
}
__device__ __forceinline__ void store_peer(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void store_peer(uint32_t at, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory"); }

struct FoldSum {
    template <typename S> static __device__ __forceinline__ S of(S a, S b) { return a + b; }
    static __device__ __forceinline__ float none() { return 0.0f; }
};
struct FoldMax {      // like fmaxf, ignores a NaN
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float none() { return -INFINITY; }
};

// A CTA's shared memory may be written by another of its cluster only once it is known to run.  A kernel therefore
// makes a TeamEntry first of all, which arrives at the cluster's barrier, and gets the FoldTurn that every fold asks
// for from met(), which waits there: the row's loads lie between the two.  Every thread of a cluster calls
// both; with one CTA to a team (cs == 1) neither does anything.
class FoldTurn {
public:
    const int cs;                                        // CTAs of a team
    int slot = 0;

private:
    __device__ __forceinline__ explicit FoldTurn(int ctas) : cs(ctas) {}
    friend class TeamEntry;
};
class TeamEntry {
public:
    __device__ __forceinline__ explicit TeamEntry(int ctas) : cs_(ctas) {
        if (cs_ > 1) cluster_arrive();
    }
    __device__ __forceinline__ FoldTurn met() const {
        if (cs_ > 1) {
            __syncwarp();
            cluster_wait();
        }
        return FoldTurn(cs_);
    }

private:
    const int cs_;
};

// Two sets of slots used in turn: a slot is written again only after every reader has passed the barrier
// of the fold in between.
template <int THREADS, int N, typename S>
struct TeamSlots {
    S warps[2][kMaxCluster * (THREADS / 32)][N];         // entries of this CTA's warps, or of all warps of the cluster
};

// v[n] = fold over i < count of p[i * N + n], in every lane: lane l reads the entries l, l + 32, ... (all of
// the same n = l % N), the lanes of equal n join theirs, and lane n passes the result on.
template <typename OP, int N, typename S>
__device__ __forceinline__ void lane_fold(S (&v)[N], const S* p, int count) {
    const int lane = threadIdx.x & 31;
    S x = (S)OP::none();
    for (int i = lane; i < count * N; i += 32) x = OP::of(x, p[i]);
#pragma unroll
    for (int off = N; off < 32; off <<= 1) x = OP::of(x, __shfl_xor_sync(0xffffffffu, x, off));
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, x, n);
}

// Folds N (a power of two) values over a team of T threads of a CTA of THREADS, and over the CTAs of a
// cluster when turn.cs > 1 (a team is then a whole CTA).  Every thread of the team calls it and gets the same
// bits.  Within a warp the values are folded in halves — a lane passes on half of its values, then half of
// the rest — so that eight sums cost 9 shuffles instead of 40; lane l then holds value l / (32 / N).
template <typename OP, int THREADS, int T, int N, typename S>
__device__ __forceinline__ void team_fold(S (&v)[N], TeamSlots<THREADS, N, S>& sh, FoldTurn& turn) {
    if constexpr (T < 32) {                              // several teams in a warp, all of whose lanes take part
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int off = T / 2; off > 0; off >>= 1) v[n] = OP::of(v[n], __shfl_xor_sync(0xffffffffu, v[n], off));
        return;
    }
    const int lane = threadIdx.x & 31;
    int off = 16;
#pragma unroll
    for (int have = N; have > 1; have >>= 1, off >>= 1) {
        const bool upper = lane & off;
#pragma unroll
        for (int n = 0; n < have / 2; ++n) {
            const S give = upper ? v[n] : v[n + have / 2], keep = upper ? v[n + have / 2] : v[n];
            v[n] = OP::of(keep, __shfl_xor_sync(0xffffffffu, give, off));
        }
    }
#pragma unroll
    for (int rest = 16 / N; rest > 0; rest >>= 1) v[0] = OP::of(v[0], __shfl_xor_sync(0xffffffffu, v[0], rest));
    if (T == 32) {
        const S mine = v[0];
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, mine, n * (32 / N));
        return;
    }
    const int warp = threadIdx.x >> 5, team = threadIdx.x / T;
    if (T == THREADS && turn.cs > 1) {
        // every warp leaves its values with every CTA: one barrier for warps and CTAs together
        const uint32_t rank = cluster_rank();
        const S mine = __shfl_sync(0xffffffffu, v[0], (lane % N) * (32 / N));
        for (int peer = lane / N; peer < turn.cs; peer += 32 / N) store_peer(peer_shared(&sh.warps[turn.slot][rank * (THREADS / 32) + warp][lane % N], peer), mine);
        __syncwarp();
        cluster_barrier();
        lane_fold<OP, N>(v, &sh.warps[turn.slot][0][0], turn.cs * (THREADS / 32));
    } else {
        if (lane % (32 / N) == 0) sh.warps[turn.slot][warp][lane / (32 / N)] = v[0];
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(T) : "memory");
        lane_fold<OP, N>(v, &sh.warps[turn.slot][team * (T / 32)][0], T / 32);
    }
    turn.slot ^= 1;
}

// How many clusters of `cs` CTAs of this kernel the current device runs at once.
int resident_clusters(const void* kernel, int threads, size_t smem, int cs, int* count);

// A kernel that was launched with `early` may start before the one ahead of it in the stream has ended; it
// calls wait_for_previous() before it touches what that one writes.  The one ahead calls let_next_start() when
// it has little left to do.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
int launch_early(void (*kernel)(Params...), unsigned blocks, int threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
    return CTB_OK;
}

// One-dimensional launch, in clusters of `cs` CTAs when cs > 1.
template <typename... Params, typename... Args>
int launch_clusters(const char* who, void (*kernel)(Params...), int64_t blocks, int threads, size_t smem, int cs, cudaStream_t st, Args... args) {
    if (blocks > 0x7FFFFFFFll) return set_error(CTB_ERR_LIMIT, "%s: too many rows for one launch", who);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    if (smem > 48 * 1024) CTB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...));
    return CTB_OK;
}

}  // namespace ctb
