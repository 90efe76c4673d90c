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
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
};
struct FoldMax {      // like fmaxf, ignores a NaN
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// Two sets of slots used in turn: a slot is written again only after every reader has passed the barrier
// of the fold in between.  (One object serves folds of different kinds as long as all of them use `turn`.)
template <int THREADS, int N, typename S>
struct TeamSlots {
    S warps[2][THREADS / 32][N];
    S peers[2][kMaxCluster][N];
};

// Folds N values over a team of T threads of a CTA of THREADS, and over the `cs` CTAs of a cluster when
// cs > 1 (a team is then a whole CTA).  Every thread of the team calls it.
template <typename OP, int THREADS, int T, int N, typename S>
__device__ __forceinline__ void team_fold(S (&v)[N], TeamSlots<THREADS, N, S>& sh, int& turn, int cs) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v[n] = OP::of(v[n], __shfl_xor_sync(0xffffffffu, v[n], off));
    if (T == 32) return;
    const int warp = threadIdx.x >> 5, team = threadIdx.x / T;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) sh.warps[turn][warp][n] = v[n];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(T) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n) {
        S r = sh.warps[turn][team * (T / 32)][n];
#pragma unroll
        for (int i = 1; i < T / 32; ++i) r = OP::of(r, sh.warps[turn][team * (T / 32) + i][n]);
        v[n] = r;
    }
    if (cs > 1) {
        if ((int)threadIdx.x < cs) {
            const uint32_t at = peer_shared(&sh.peers[turn][cluster_rank()][0], threadIdx.x);
#pragma unroll
            for (int n = 0; n < N; ++n) store_peer(at + n * (uint32_t)sizeof(S), v[n]);
        }
        __syncwarp();
        cluster_barrier();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            S r = sh.peers[turn][0][n];
            for (int i = 1; i < cs; ++i) r = OP::of(r, sh.peers[turn][i][n]);
            v[n] = r;
        }
    }
    turn ^= 1;
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
