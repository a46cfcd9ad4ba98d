// Shared by the 16-bit operators: conversions, and the walk over segments of rows (experts, adapters).
#pragma once
#include <atomic>

#include "common.cuh"

namespace gsb {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
// h of the FFN: a finite value beyond fp16 saturates instead of turning into infinity and then NaN in the next product;
// infinities and NaN are the activations' own and go on (the minimum and maximum of a NaN would be the border)
template <typename T> __device__ __forceinline__ T h_from_f(float v) { return from_f<T>(v); }
template <> __device__ __forceinline__ __half h_from_f(float v) {
    return isfinite(v) ? sat_half(v) : __float2half_rn(v);
}

// Segment bounds as read from device memory, forced into [0, P], so that no list leads outside the buffers; the
// kernels write nothing for one that descends.
__device__ __forceinline__ int seg_bound(const int* offsets, int e, int P) { return min(max(offsets[e], 0), P); }

constexpr int kMaxE = 1024;     // segments at most
constexpr int kMaxDim = 1 << 30;    // of a row; sums of a dimension and a tile stay ints

// The walk over the segments: the first 256 threads hold four segments each (n[j] = rows of segment 4 tid + j), all call.
// Returns non-zero in a thread that saw the list descend.
__device__ __forceinline__ int seg_count(const int* offsets, int E, int P, int (&n)[4]) {
    int descending = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = (int)threadIdx.x * 4 + j;
        n[j] = 0;
        if (e < E) {
            n[j] = seg_bound(offsets, e + 1, P) - seg_bound(offsets, e, P);
            descending |= n[j] < 0;
        }
    }
    return descending;
}
// pre[e] = tiles of at most 2^lg rows before segment e, e = 0..E (E <= kMaxE).  `wsum`: shared scratch of 8 ints.
__device__ __forceinline__ void seg_scan(const int (&n)[4], int E, int lg, int* pre, int* wsum) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int c[4], sum = 0, incl = 0;
    if (tid < 256) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c[j] = sum;
            sum += n[j] > 0 ? (n[j] + (1 << lg) - 1) >> lg : 0;
        }
        incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        if (lane == 31) wsum[warp] = incl;
    }
    __syncthreads();
    if (tid < 256) {
        int base = incl - sum;
        for (int w = 0; w < warp; ++w) base += wsum[w];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (tid * 4 + j <= E) pre[tid * 4 + j] = base + c[j];
        if (tid == 255 && E == kMaxE) pre[kMaxE] = base + sum;
    }
}
__device__ __forceinline__ int seg_scan(const int* offsets, int E, int P, int lg, int* pre, int* wsum) {
    int n[4];
    const int descending = seg_count(offsets, E, P, n);
    seg_scan(n, E, lg, pre, wsum);
    return descending;
}

inline int sm_count_of(int dev) {
    static std::atomic<int> cached[64];
    int v = dev < 64 ? cached[dev].load() : 0;
    if (!v) {
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        if (dev < 64) cached[dev].store(v);
    }
    return v;
}

// Programmatic dependent launch: a kernel started with launch_after() may begin before the one ahead of it in the stream
// has ended, once all of that one's blocks have called pdl_trigger(); it touches nothing that another kernel writes, or
// still reads, before pdl_wait(), which returns when the kernel ahead is complete.  Every kernel here waits, so what a
// kernel two places ahead wrote is there as well.  What it reads may still be written while it is already there (unless an
// ordinary launch stands between), so none of that goes through the read-only path (__ldg, const __restrict__): it asks for
// data that no one writes meanwhile, and its loads may be moved ahead of the wait.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename K, typename... A>
inline int launch_after(K kernel, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return GSB_OK;
    cudaGetLastError();     // the status says it; a later call must not find it again
    return GSB_ERR_LAUNCH;
}

inline bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }
// whether two pieces of memory share a byte; sizes are products of up to three dimensions (below 2^73), null has none
inline bool overlap(const void* p, __int128 p_bytes, const void* q, __int128 q_bytes) {
    const __int128 a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return p && q && a < b + q_bytes && b < a + p_bytes;
}

}  // namespace gsb
