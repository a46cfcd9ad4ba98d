// Shared by the two tensor-core kernels of the 16-bit expert products (expert16.cu, expert16_pair.cu).
#pragma once
#include <atomic>
#include <type_traits>

#include "launchers.cuh"
#include "tc5.cuh"

namespace gsb {

struct GroupedArgs {
    const void* x;          // [n, K]
    const void* w;          // [E, N, K]; the gate matrices when w2 is given
    const void* w2;         // [E, N, K] up matrices or null
    const int* offsets;     // [E + 1]
    const int* rows;        // [P] row of x for every p, or null (row p)
    int n, P, K, N, E;
    void* y;                // [P, N]
};

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

constexpr int kMaxE = 1024;
constexpr long long kGrWaitLimit = 2000000000LL;    // about a second of SM clocks

struct GrItem { int e, p0, cnt, f0; };

// pre[e] = token tiles of at most NT rows before expert e, e = 0..E; at least 256 threads, all call.
// Returns non-zero when the list descends somewhere.  `wsum`: shared scratch of 8 ints.
template <int NT>
__device__ __forceinline__ int gr_scan(const GroupedArgs& a, int* pre, int* wsum) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int c[4], sum = 0, incl = 0, descending = 0;
    if (tid < 256) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = tid * 4 + j;
            c[j] = sum;
            if (e < a.E) {
                const int lo = seg_bound(a.offsets, e, a.P), hi = seg_bound(a.offsets, e + 1, a.P);
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
            if (tid * 4 + j <= a.E) pre[tid * 4 + j] = base + c[j];
        if (tid == 255 && a.E == kMaxE) pre[kMaxE] = base + sum;
    }
    return descending;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
    }();
    return fn;
}

// [d2, d1, d0] row-major 16-bit tensor (d2 = 0: two dims), boxes of 64 columns x box_rows rows, 128-byte swizzle.
inline bool encode(CUtensorMap* m, const void* base, bool bf16, uint64_t d0, uint64_t d1, uint64_t d2, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {d0, d1, d2}, strides[2] = {d0 * 2, d0 * d1 * 2};
    const cuuint32_t box[3] = {64, box_rows, 1}, estr[3] = {1, 1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, d2 ? 3 : 2, const_cast<void*>(base),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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

// The two kernels; types as in gsb_grouped_gemm (a.w2 given: SwiGLU of two products, y of x's type).
int launch_grouped_split(const GroupedArgs& a, int type, int y_type, cudaStream_t s);
int take_pair_status();      // status word of the pair kernel, cleared
int launch_grouped_pair(const GroupedArgs& a, int type, int y_type, cudaStream_t s);

}  // namespace gsb
