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
// h of the FFN: fp16 saturates instead of turning into infinity and then NaN in the next product
template <typename T> __device__ __forceinline__ T h_from_f(float v) { return from_f<T>(v); }
template <> __device__ __forceinline__ __half h_from_f(float v) { return sat_half(v); }

// Segment bounds as read from device memory, forced into [0, P]: a list that is not ascending gives wrong rows,
// never an access outside the buffers.
__device__ __forceinline__ int seg_bound(const int* offsets, int e, int P) { return min(max(__ldg(offsets + e), 0), P); }

constexpr int kMaxE = 1024;     // segments at most

// pre[e] = tiles of at most NT rows before segment e, e = 0..E (E <= kMaxE); the first 256 threads work, all call.
// Returns non-zero in a thread that saw the list descend.  `wsum`: shared scratch of 8 ints.
template <int NT>
__device__ __forceinline__ int seg_scan(const int* offsets, int E, int P, int* pre, int* wsum) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int c[4], sum = 0, incl = 0, descending = 0;
    if (tid < 256) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = tid * 4 + j;
            c[j] = sum;
            if (e < E) {
                const int lo = seg_bound(offsets, e, P), hi = seg_bound(offsets, e + 1, P);
                sum += hi > lo ? (hi - lo + NT - 1) / NT : 0;
                descending |= hi < lo;
            }
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

inline bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

}  // namespace gsb
