// Expert products with 16-bit (bf16 / fp16) weights: the ragged grouped product
//   y[p, :] = W[e] x[rows[p], :]                        for offsets[e] <= p < offsets[e + 1]
// and the expert FFN built from it
//   h[p, :] = silu(gate[e] x) * (up[e] x),  y[p, :] = down[e] h[p, :],  out[t, :] = sum_k w[t, k] y[slot(t, k), :].
// Products are summed in fp32; h is rounded once to the weights' type (the tensor cores read it in that type,
// fp16 saturating at +-65504), the per-slot rows y stay fp32 and the sum over slots is taken in slot order.
#include "common.cuh"
#include "launchers.cuh"

namespace gsb {

namespace {

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

// Plain form: 64 rows x 64 features per block, 4 x 4 per thread.
template <typename T, typename Y, bool GU>
__global__ void __launch_bounds__(256)
grouped_simple_kernel(const GroupedArgs a) {
    __shared__ float sx[64][17], sw[64][17], su[GU ? 64 : 1][17];
    __shared__ int seg[3], srow[64];
    const int tid = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(a.x);
    if (tid == 0) {
        int t = blockIdx.y;
        seg[0] = -1;
        for (int e = 0; e < a.E; ++e) {
            const int lo = seg_bound(a.offsets, e, a.P), hi = seg_bound(a.offsets, e + 1, a.P);
            const int nt = hi > lo ? (hi - lo + 63) / 64 : 0;
            if (t < nt) { seg[0] = e; seg[1] = lo + t * 64; seg[2] = min(64, hi - lo - t * 64); break; }
            t -= nt;
        }
    }
    __syncthreads();
    const int e = seg[0], p0 = seg[1], cnt = seg[2], f0 = blockIdx.x * 64;
    if (e < 0) return;
    if (tid < 64) {
        const int r = tid < cnt ? (a.rows ? __ldg(a.rows + p0 + tid) : p0 + tid) : -1;
        srow[tid] = r >= 0 && r < a.n ? r : -1;
    }
    const T* w = reinterpret_cast<const T*>(a.w) + (int64_t)e * a.N * a.K;
    const T* u = reinterpret_cast<const T*>(a.w2) + (int64_t)e * a.N * a.K;
    float acc[4][4] = {}, acu[4][4] = {};
    const int tr = tid >> 4, tf = tid & 15;
    for (int k0 = 0; k0 < a.K; k0 += 16) {
        __syncthreads();
        for (int i = tid; i < 64 * 16; i += 256) {
            const int r = i >> 4, k = k0 + (i & 15), f = f0 + r;
            sx[r][i & 15] = srow[r] >= 0 && k < a.K ? to_f(x[(int64_t)srow[r] * a.K + k]) : 0.f;
            sw[r][i & 15] = f < a.N && k < a.K ? to_f(w[(int64_t)f * a.K + k]) : 0.f;
            if (GU) su[r][i & 15] = f < a.N && k < a.K ? to_f(u[(int64_t)f * a.K + k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = fmaf(sx[tr * 4 + i][k], sw[j * 16 + tf][k], acc[i][j]);
                    if (GU) acu[i][j] = fmaf(sx[tr * 4 + i][k], su[j * 16 + tf][k], acu[i][j]);
                }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = tr * 4 + i, f = f0 + j * 16 + tf;
            if (srow[r] < 0 || f >= a.N) continue;
            reinterpret_cast<Y*>(a.y)[(int64_t)(p0 + r) * a.N + f] =
                GU ? h_from_f<Y>(__fmul_rn(silu_ref(acc[i][j]), acu[i][j])) : from_f<Y>(acc[i][j]);
        }
}

template <typename T, typename Y, bool GU>
int run_grouped(const GroupedArgs& a, cudaStream_t s) {
    const int tiles = a.P / 64 + (a.E < a.P ? a.E : a.P);
    grouped_simple_kernel<T, Y, GU><<<dim3((a.N + 63) / 64, tiles), 256, 0, s>>>(a);
    return launch_status();
}

template <typename T>
int run_grouped_any(const GroupedArgs& a, int y_type, cudaStream_t s) {
    if (a.w2) return run_grouped<T, T, true>(a, s);
    return y_type == GSB_TYPE_F32 ? run_grouped<T, float, false>(a, s) : run_grouped<T, T, false>(a, s);
}

int launch_grouped(const GroupedArgs& a, int type, int y_type, cudaStream_t s) {
    return type == GSB_TYPE_BF16 ? run_grouped_any<__nv_bfloat16>(a, y_type, s) : run_grouped_any<__half>(a, y_type, s);
}

// out[t] = sum over k, in order, of w[t, k] * y[slot_pos[t, k]]; slots whose id is outside [0, E) add nothing.
template <typename O>
__global__ void __launch_bounds__(256)
combine16_kernel(const float* __restrict__ y, const int* __restrict__ ids, const int* __restrict__ slot_pos,
                 const float* __restrict__ w, int topk, int H, int E, O* __restrict__ out) {
    const int64_t t = blockIdx.x;
    for (int c = (blockIdx.y * 256 + threadIdx.x) * 4; c < H; c += gridDim.y * 1024) {   // H is a multiple of 8
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < topk; ++k) {
            const int id = __ldg(ids + t * topk + k);
            if (id < 0 || id >= E) continue;
            const float4 v = __ldg(reinterpret_cast<const float4*>(y + (int64_t)__ldg(slot_pos + t * topk + k) * H + c));
            const float wk = __ldg(w + t * topk + k);
            acc.x = fmaf(wk, v.x, acc.x); acc.y = fmaf(wk, v.y, acc.y);
            acc.z = fmaf(wk, v.z, acc.z); acc.w = fmaf(wk, v.w, acc.w);
        }
        O* o = out + t * H + c;
        o[0] = from_f<O>(acc.x); o[1] = from_f<O>(acc.y); o[2] = from_f<O>(acc.z); o[3] = from_f<O>(acc.w);
    }
}

template <typename O>
int run_combine16(const float* y, const int* ids, const int* slot_pos, const float* w, int n, int topk, int H, int E,
                  void* out, cudaStream_t s) {
    combine16_kernel<O><<<dim3(n, (H + 1023) / 1024), 256, 0, s>>>(y, ids, slot_pos, w, topk, H, E, reinterpret_cast<O*>(out));
    return launch_status();
}

// Scratch of the FFN; every buffer starts on a 256-byte boundary.
struct Ffn16Ws { int *offsets, *tok, *row, *slot_pos, *disp; uint8_t* h; float* y; size_t total; };
Ffn16Ws carve16(int n, int topk, int H, int I, int E, void* base) {
    const size_t P = (size_t)n * topk;
    Ffn16Ws ws{};
    uint8_t* p = reinterpret_cast<uint8_t*>(base);
    size_t at = 0;
    auto take = [&](size_t bytes) { uint8_t* q = p + at; at += (bytes + 255) / 256 * 256; return q; };
    ws.offsets = reinterpret_cast<int*>(take((size_t)(E + 1) * 4));
    ws.tok = reinterpret_cast<int*>(take(P * 4));
    ws.row = reinterpret_cast<int*>(take(P * 4));
    ws.slot_pos = reinterpret_cast<int*>(take(P * 4));
    ws.disp = reinterpret_cast<int*>(take(dispatch_scratch_bytes(n, topk, E)));
    ws.h = take(P * I * 2);
    ws.y = reinterpret_cast<float*>(take(P * H * 4));
    ws.total = at;
    return ws;
}

inline bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }
inline bool is16(int type) { return type == GSB_TYPE_BF16 || type == GSB_TYPE_F16; }
inline size_t type_bytes(int type) { return type == GSB_TYPE_F32 ? 4 : 2; }
constexpr int64_t kMaxSlots = (int64_t)1 << 30;

}  // namespace

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_grouped_gemm(const void* x, const void* w, int type, const int* expert_offsets, const int* rows,
                                int n, int P, int in, int out, int E, void* y, int y_type, void* stream) {
    if (!is16(type) || (y_type != type && y_type != GSB_TYPE_F32)) return GSB_ERR_INVALID_ARG;
    if (n < 0 || P < 0 || in <= 0 || out <= 0 || E <= 0 || (!rows && P > n)) return GSB_ERR_INVALID_ARG;
    if (P == 0 || n == 0) return GSB_OK;
    if (!x || !w || !expert_offsets || !y) return GSB_ERR_INVALID_ARG;
    if (misaligned(x, 16) || misaligned(w, 16) || misaligned(expert_offsets, 4) || misaligned(rows, 4) ||
        misaligned(y, type_bytes(y_type)))
        return GSB_ERR_INVALID_ARG;
    if (in % 8 || E > 1024 || P > kMaxSlots) return GSB_ERR_UNSUPPORTED;
    GroupedArgs a{};
    a.x = x; a.w = w; a.offsets = expert_offsets; a.rows = rows;
    a.n = n; a.P = P; a.K = in; a.N = out; a.E = E; a.y = y;
    return launch_grouped(a, type, y_type, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t gsb_moe_expert_ffn_w16_workspace_bytes(int n, int topk, int hidden, int moe_inter, int E) {
    if (n <= 0 || topk <= 0 || hidden <= 0 || moe_inter <= 0 || E <= 0) return 0;
    return carve16(n, topk, hidden, moe_inter, E, nullptr).total;
}

extern "C" int gsb_moe_expert_ffn_w16(const void* x, const int* topk_ids, const float* topk_weights, const void* gate_w,
                                      const void* up_w, const void* down_w, int type, int n, int topk, int hidden,
                                      int moe_inter, int E, void* out, int out_type, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (!is16(type) || (out_type != type && out_type != GSB_TYPE_F32)) return GSB_ERR_INVALID_ARG;
    if (n < 0 || topk <= 0 || hidden <= 0 || moe_inter <= 0 || E <= 0) return GSB_ERR_INVALID_ARG;
    if (n == 0) return GSB_OK;
    if (!x || !topk_ids || !topk_weights || !gate_w || !up_w || !down_w || !out) return GSB_ERR_INVALID_ARG;
    if (misaligned(x, 16) || misaligned(gate_w, 16) || misaligned(up_w, 16) || misaligned(down_w, 16) ||
        misaligned(out, 16) || misaligned(topk_ids, 4) || misaligned(topk_weights, 4))
        return GSB_ERR_INVALID_ARG;
    if (hidden % 8 || moe_inter % 8 || E > 1024 || (int64_t)n * topk > kMaxSlots) return GSB_ERR_UNSUPPORTED;
    if (!workspace || misaligned(workspace, 256)) return GSB_ERR_INVALID_ARG;
    const Ffn16Ws ws = carve16(n, topk, hidden, moe_inter, E, workspace);
    if (workspace_bytes < ws.total) return GSB_ERR_WORKSPACE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int st = launch_dispatch(topk_ids, n, topk, E, ws.offsets, ws.tok, ws.row, ws.slot_pos, s, ws.disp);
    if (st) return st;
    GroupedArgs g{};
    g.x = x; g.w = gate_w; g.w2 = up_w; g.offsets = ws.offsets; g.rows = ws.tok;
    g.n = n; g.P = n * topk; g.K = hidden; g.N = moe_inter; g.E = E; g.y = ws.h;
    st = launch_grouped(g, type, type, s);
    if (st) return st;
    GroupedArgs d{};
    d.x = ws.h; d.w = down_w; d.offsets = ws.offsets;
    d.n = d.P = n * topk; d.K = moe_inter; d.N = hidden; d.E = E; d.y = ws.y;
    st = launch_grouped(d, type, GSB_TYPE_F32, s);
    if (st) return st;
    if (out_type == GSB_TYPE_F32) return run_combine16<float>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
    if (type == GSB_TYPE_BF16) return run_combine16<__nv_bfloat16>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
    return run_combine16<__half>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
}

extern "C" int gsb_operators16_status(void) {
    return cudaDeviceSynchronize() == cudaSuccess ? GSB_OK : GSB_ERR_CUDA;
}
