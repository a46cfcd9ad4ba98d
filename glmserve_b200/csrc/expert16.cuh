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
    // SwiGLU of few slots: the ids to make offsets and rows from (P = n * topk <= kFewSlots of them; offsets and rows are
    // null), and where to leave the offsets and every slot's place
    const int* ids;
    int topk;
    int* offsets_out;
    int* slot_pos_out;
    long long sum_limit;    // clocks to wait for a whole sum over K
};

constexpr long long kGrWaitLimit = 2000000000LL;    // about a second of SM clocks
// The wait for a whole sum over K lasts as long as the sum: a second more for every 250,000 k-blocks of 64 columns.  (A
// block alone on the GPU takes 270 clocks for one; 38 experts of one row, 2^29 to 1, are 2.2 G clocks.)
inline long long gr_sum_limit(int K) { return kGrWaitLimit + ((long long)K + 63) / 64 * 8192; }

constexpr int kFewSlots = 256;

struct GrItem { int e, p0, cnt, f0; };

// AND over the four warps that meet at named barrier `bar`
__device__ __forceinline__ int epilogue_agree(int ok, int bar) {
    int all;
    asm volatile("{\n\t.reg .pred p, r;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred r, %2, 128, p;\n\tselp.u32 %0, 1, 0, r;\n\t}"
                 : "=r"(all) : "r"(ok), "r"(bar) : "memory");
    return all;
}
__device__ __forceinline__ void epilogue_sync(int bar) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(bar) : "memory"); }

// silu(gate) * up.  expf and the divide are good to 2^-21 together; the result is rounded to 16 bits next.  (An IEEE divide
// here is a third of an epilogue's instructions; where 1 + exp passes 2^126 this one gives 0 for a silu below 2^-119.)
__device__ __forceinline__ float swiglu(float g, float u) { return __fmul_rn(__fdividef(g, 1.0f + expf(-g)), u); }

// status words of the kernels in the other files, cleared
int take_pair_status();
int take_lora_status();
// The kernel for many rows; types as in gsb_grouped_gemm (a.w2 given: SwiGLU of two products, y of x's type).  scratch
// (16-byte aligned, grouped_pair_scratch_bytes): a copy of the rows in expert order, used when a.rows is given
size_t grouped_pair_scratch_bytes(int P, int K);
int launch_grouped_pair(const GroupedArgs& a, int type, int y_type, void* scratch, cudaStream_t s);

}  // namespace gsb
