// Low-rank adapters of many requests beside a shared projection:
//   v[p, :] = scale[a] * A[a] x[t, :],   y[t, :] += B[a] v[p, :]        t = rows[p], a = the adapter of p's segment
// Two launches: the first takes the long sum over the input dim, the second spreads the few values v over the output.
#include "common.cuh"
#include "launchers.cuh"

namespace gsb {

namespace {

struct LoraArgs {
    const void *x, *A, *B;
    const int *offsets, *rows, *ranks;
    const float* scales;
    int n, P, K, N, nA, R;
    float* v;       // [P, R]
    void* y;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// adapter whose segment holds p, or -1
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int p) {
    for (int i = 0; i < a.nA; ++i)
        if (__ldg(a.offsets + i) <= p && p < __ldg(a.offsets + i + 1)) return i;
    return -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs& a, int ad) {
    return a.ranks ? min(max(__ldg(a.ranks + ad), 0), a.R) : a.R;
}

template <typename T>
__global__ void __launch_bounds__(256) lora_shrink_simple_kernel(const LoraArgs a) {
    const int p = blockIdx.x, ad = adapter_of(a, p);
    const int t = __ldg(a.rows + p);
    if (ad < 0 || t < 0 || t >= a.n) return;
    const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)t * a.K;
    const float sc = a.scales ? __ldg(a.scales + ad) : 1.f;
    for (int r = threadIdx.x >> 5; r < rank_of(a, ad); r += 8) {
        const T* w = reinterpret_cast<const T*>(a.A) + ((int64_t)ad * a.R + r) * a.K;
        float s = 0.f;
        for (int k = threadIdx.x & 31; k < a.K; k += 32) s = fmaf(to_f(x[k]), to_f(w[k]), s);
        s = warp_sum(s);
        if ((threadIdx.x & 31) == 0) a.v[(int64_t)p * a.R + r] = sc * s;
    }
}

template <typename T, typename Y>
__global__ void __launch_bounds__(256) lora_expand_simple_kernel(const LoraArgs a) {
    const int p = blockIdx.x, ad = adapter_of(a, p);
    const int t = __ldg(a.rows + p);
    if (ad < 0 || t < 0 || t >= a.n) return;
    Y* y = reinterpret_cast<Y*>(a.y) + (int64_t)t * a.N;
    const int rank = rank_of(a, ad);
    for (int o = threadIdx.x; o < a.N; o += 256) {
        const T* b = reinterpret_cast<const T*>(a.B) + ((int64_t)ad * a.N + o) * a.R;
        float s = 0.f;
        for (int r = 0; r < rank; ++r) s = fmaf(to_f(b[r]), a.v[(int64_t)p * a.R + r], s);
        y[o] = from_f<Y>(to_f(y[o]) + s);
    }
}

template <typename T, typename Y>
int run_lora(const LoraArgs& a, cudaStream_t s) {
    lora_shrink_simple_kernel<T><<<a.P, 256, 0, s>>>(a);
    lora_expand_simple_kernel<T, Y><<<a.P, 256, 0, s>>>(a);
    return launch_status();
}

inline bool misaligned(const void* p, size_t al) { return reinterpret_cast<uintptr_t>(p) % al != 0; }

}  // namespace

}  // namespace gsb

using namespace gsb;

extern "C" size_t gsb_lora_scratch_bytes(int P, int max_rank, int n_adapters) {
    if (P <= 0 || max_rank <= 0 || n_adapters <= 0) return 0;
    return (size_t)P * max_rank * 4;
}

extern "C" int gsb_lora_add(const void* x, const void* A, const void* B, int type, const int* adapter_offsets,
                            const int* rows, const int* ranks, const float* scales, int n, int P, int in, int out,
                            int n_adapters, int max_rank, void* y, int y_type, void* scratch, size_t scratch_bytes,
                            void* stream) {
    if ((type != GSB_TYPE_BF16 && type != GSB_TYPE_F16) || (y_type != type && y_type != GSB_TYPE_F32)) return GSB_ERR_INVALID_ARG;
    if (n < 0 || P < 0 || P > n || in <= 0 || out <= 0 || n_adapters <= 0 || max_rank <= 0) return GSB_ERR_INVALID_ARG;
    if (P == 0) return GSB_OK;
    if (!x || !A || !B || !adapter_offsets || !rows || !y) return GSB_ERR_INVALID_ARG;
    if (misaligned(x, 16) || misaligned(A, 16) || misaligned(B, 2) || misaligned(y, y_type == GSB_TYPE_F32 ? 4 : 2) ||
        misaligned(adapter_offsets, 4) || misaligned(rows, 4) || misaligned(ranks, 4) || misaligned(scales, 4))
        return GSB_ERR_INVALID_ARG;
    if (in % 8 || max_rank > 256 || n_adapters > 1024) return GSB_ERR_UNSUPPORTED;
    if (!scratch || misaligned(scratch, 256)) return GSB_ERR_INVALID_ARG;
    if (scratch_bytes < gsb_lora_scratch_bytes(P, max_rank, n_adapters)) return GSB_ERR_WORKSPACE;
    LoraArgs a{};
    a.x = x; a.A = A; a.B = B; a.offsets = adapter_offsets; a.rows = rows; a.ranks = ranks; a.scales = scales;
    a.n = n; a.P = P; a.K = in; a.N = out; a.nA = n_adapters; a.R = max_rank;
    a.v = reinterpret_cast<float*>(scratch); a.y = y;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (type == GSB_TYPE_BF16)
        return y_type == GSB_TYPE_F32 ? run_lora<__nv_bfloat16, float>(a, s) : run_lora<__nv_bfloat16, __nv_bfloat16>(a, s);
    return y_type == GSB_TYPE_F32 ? run_lora<__half, float>(a, s) : run_lora<__half, __half>(a, s);
}
