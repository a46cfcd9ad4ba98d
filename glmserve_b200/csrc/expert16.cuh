// Shared by the two tensor-core kernels of the 16-bit expert products (expert16.cu, expert16_pair.cu).
#pragma once
#include <atomic>
#include <type_traits>

#include "launchers.cuh"
#include "segments.cuh"
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

constexpr long long kGrWaitLimit = 2000000000LL;    // about a second of SM clocks

struct GrItem { int e, p0, cnt, f0; };

// Weight rows of an item (128, 64 or 32, not under `least`) for `tiles` token tiles x `rows` weight rows each on
// `workers` CTAs that take items in turn: the one with the shortest way through, an item costing its rows and the time of
// about 8 more.
__device__ __forceinline__ int best_width(int tiles, int rows, int workers, int least) {
    int best = 128;
    int64_t cost = 0;
    for (int w = 128; w >= least; w >>= 1) {
        const int64_t items = (int64_t)tiles * ((rows + w - 1) / w), c = (items + workers - 1) / workers * (w + 8);
        if (w == 128 || c < cost) { best = w; cost = c; }
    }
    return best;
}

// AND over the four epilogue warps
__device__ __forceinline__ int epilogue_agree(int ok) {
    int all;
    asm volatile("{\n\t.reg .pred p, r;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred r, 1, 128, p;\n\tselp.u32 %0, 1, 0, r;\n\t}"
                 : "=r"(all) : "r"(ok) : "memory");
    return all;
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

// The two kernels; types as in gsb_grouped_gemm (a.w2 given: SwiGLU of two products, y of x's type).
int launch_grouped_split(const GroupedArgs& a, int type, int y_type, cudaStream_t s);
int take_pair_status();      // status word of the pair kernel, cleared
// scratch (16-byte aligned, grouped_pair_scratch_bytes): a copy of the rows in expert order, used when a.rows is given
size_t grouped_pair_scratch_bytes(int P, int K);
int launch_grouped_pair(const GroupedArgs& a, int type, int y_type, void* scratch, cudaStream_t s);

}  // namespace gsb
