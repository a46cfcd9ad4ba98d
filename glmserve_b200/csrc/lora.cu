// Low-rank adapters of many requests beside a shared projection:
//   v[p, :] = scale[a] * A[a] x[t, :],   y[t, :] += B[a] v[p, :]        t = rows[p], a = the adapter of p's segment
// Two launches, both over tiles of one adapter's rows: the first takes the long sum over the input dim (x and A are
// read once), the second spreads the few values v over the output (y is read and written once, B read once per tile).
// Both are bound by those bytes; the tensor cores only keep the arithmetic out of the way, so mma.sync fed straight from
// global memory does: every lane loads 16 (B: 8) contiguous bytes of a row and takes them as its k positions in the
// fragments of BOTH operands - a sum does not care in which order k runs.
#include "launchers.cuh"
#include "segments.cuh"

namespace gsb {

namespace {

struct LoraArgs {
    const void *x, *A, *B;
    const int *offsets, *rows, *ranks;
    const float* scales;
    int n, P, K, N, nA, R;
    int S;          // parts of the sum over K
    float* part;    // [S, P, R]
    void* y;
};

constexpr int kShWarps = 8;

__device__ __forceinline__ int rank_of(const LoraArgs& a, int ad) {
    return a.ranks ? min(max(__ldg(a.ranks + ad), 0), a.R) : a.R;
}

struct LoraTile { int ad, p0, cnt; };

// tile i of all adapters' rows (NT rows each); ad < 0 past the last
template <int NT>
__device__ __forceinline__ LoraTile lora_tile(const LoraArgs& a, const int* pre, int i, int descending) {
    LoraTile t{-1, 0, 0};
    if (descending || i >= pre[a.nA]) return t;
    int lo = 0, hi = a.nA - 1;                     // the last adapter with pre[ad] <= i (empty ones have pre[ad + 1] == pre[ad])
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= i) lo = mid; else hi = mid - 1;
    }
    t.ad = lo;
    const int beg = seg_bound(a.offsets, lo, a.P), end = seg_bound(a.offsets, lo + 1, a.P);
    t.p0 = beg + (i - pre[lo]) * NT;
    t.cnt = min(NT, end - t.p0);
    return t;
}

template <typename T> __device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_k16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_k16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)),
                   "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// ---- first launch: v ---------------------------------------------------------------------------
// Block: up to 8 * NTK rows of one adapter x 16 * MT ranks, D[rank, row]; its eight warps and a.S blocks share the sum
// over K (adjacent 32-column chunks go to adjacent warps).  The warps' tiles are added in shared memory in warp order,
// the blocks' parts by the second launch in block order.
template <typename T, int MT, int NTK>
__global__ void __launch_bounds__(kShWarps * 32)
lora_shrink_kernel(const LoraArgs a) {
    extern __shared__ float s_red[];                  // [warps][16 * MT ranks][8 * NTK rows]
    __shared__ int pre[kMaxE + 4], wsum[8];
    constexpr int RT = 16 * MT, TT = 8 * NTK;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int descending = seg_scan<TT>(a.offsets, a.nA, a.P, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<TT>(a, pre, blockIdx.x, descending);
    if (tile.ad < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.z * RT, rank = rank_of(a, tile.ad);
    if (r0 >= rank) return;
    const T* A = reinterpret_cast<const T*>(a.A) + ((int64_t)tile.ad * a.R + r0) * a.K + t * 8;
    const T* xr[NTK];
    bool xin[NTK];
#pragma unroll
    for (int j = 0; j < NTK; ++j) {
        const int c = j * 8 + g;
        const int row = c < tile.cnt ? __ldg(a.rows + tile.p0 + c) : -1;
        xin[j] = row >= 0 && row < a.n;
        xr[j] = reinterpret_cast<const T*>(a.x) + (int64_t)(xin[j] ? row : 0) * a.K + t * 8;
    }
    float acc[MT][NTK][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int chunks = (a.K + 31) / 32, stride = kShWarps * a.S;
    constexpr int U = MT * NTK >= 8 ? 1 : MT * NTK >= 4 ? 2 : 4;      // chunks in flight
    for (int c0 = blockIdx.y * kShWarps + warp; c0 < chunks; c0 += stride * U) {
        uint4 fa[U][MT][2], fx[U][NTK];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c0 + u * stride) * 32;
            const bool in = k + t * 8 < a.K;
#pragma unroll
            for (int j = 0; j < NTK; ++j) fx[u][j] = in && xin[j] ? __ldg(reinterpret_cast<const uint4*>(xr[j] + k)) : zero;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = m * 16 + h * 8 + g;          // what lies behind the adapter's rank counts as zero
                    fa[u][m][h] = in && r0 + r < rank ? __ldg(reinterpret_cast<const uint4*>(A + (int64_t)r * a.K + k)) : zero;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NTK; ++j) {
                    mma_k16<T>(acc[m][j], fa[u][m][0].x, fa[u][m][1].x, fa[u][m][0].y, fa[u][m][1].y, fx[u][j].x, fx[u][j].y);
                    mma_k16<T>(acc[m][j], fa[u][m][0].z, fa[u][m][1].z, fa[u][m][0].w, fa[u][m][1].w, fx[u][j].z, fx[u][j].w);
                }
    }
    float* mine = s_red + warp * RT * TT;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NTK; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h)
                mine[(m * 16 + (h >> 1) * 8 + g) * TT + j * 8 + t * 2 + (h & 1)] = acc[m][j][h];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * TT; i += kShWarps * 32) {
        const int c = i / RT, r = i - c * RT;
        if (c >= tile.cnt || r0 + r >= rank) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kShWarps; ++w) s += s_red[(w * RT + r) * TT + c];
        a.part[((int64_t)blockIdx.y * a.P + tile.p0 + c) * a.R + r0 + r] = s;
    }
}

// ---- second launch: y += B v ---------------------------------------------------------------------
// Block: up to 16 * MT rows of one adapter x a range of features, 32 features a warp at a time, D[row, feature].  v is
// applied as the sum of two tf32 numbers (together 22 bits of it; B's 16-bit values are exact in tf32), so y's fp32 sums
// keep fp32 accuracy.  n-tile j of a warp's chunk holds features 8 (c / 2) + 2 j + c % 2 in its columns c: lane t of a quad
// then owns eight contiguous features of a row.
template <typename T> __device__ __forceinline__ float2 pair_f(uint32_t v);
template <> __device__ __forceinline__ float2 pair_f<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <> __device__ __forceinline__ float2 pair_f<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

__device__ __forceinline__ float tf32_of(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return __uint_as_float(r);
}

template <typename Y>
__device__ __forceinline__ void load8(const Y* p, int have, bool vec, float (&v)[8]) {
    if (vec && have == 8) {
        if constexpr (sizeof(Y) == 4) {
            const float4 q0 = *reinterpret_cast<const float4*>(p), q1 = *(reinterpret_cast<const float4*>(p) + 1);
            v[0] = q0.x; v[1] = q0.y; v[2] = q0.z; v[3] = q0.w; v[4] = q1.x; v[5] = q1.y; v[6] = q1.z; v[7] = q1.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float2 f = pair_f<Y>(w[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < have ? to_f(p[i]) : 0.f;
}
template <typename Y>
__device__ __forceinline__ void store8(Y* p, int have, bool vec, const float (&v)[8]) {
    if (vec && have == 8) {
        if constexpr (sizeof(Y) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            Y o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = from_f<Y>(v[i]);
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(o);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = from_f<Y>(v[i]);
}

template <typename T, typename Y, int MT>
__global__ void __launch_bounds__(256)
lora_expand_kernel(const LoraArgs a, int feats, int vec_b, int vec_y) {
    extern __shared__ float4 s_v[];                   // [row tile of 16][16 ranks][hi g, hi g + 8, lo g, lo g + 8][lane]
    __shared__ int pre[kMaxE + 4], wsum[8], srow[16 * MT];
    int descending = seg_scan<16 * MT>(a.offsets, a.nA, a.P, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<16 * MT>(a, pre, blockIdx.x, descending);
    if (tile.ad < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = rank_of(a, tile.ad), kgs = (rank + 15) / 16;
    if (rank == 0) return;
    if (threadIdx.x < 16 * MT) {
        const int r = (int)threadIdx.x < tile.cnt ? __ldg(a.rows + tile.p0 + threadIdx.x) : -1;
        srow[threadIdx.x] = r >= 0 && r < a.n ? r : -1;
    }
    const float sc = a.scales ? __ldg(a.scales + tile.ad) : 1.f;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // v comes from the first launch
    for (int i = threadIdx.x; i < MT * kgs * 64; i += 256) {
        // (row tile, group of 16 ranks, half of the 16 rows, lane): four ranks of one row
        const int l = i & 31, h = (i >> 5) & 1, kg = (i >> 6) % kgs, m = (i >> 6) / kgs;
        const int c = m * 16 + h * 8 + (l >> 2), r = kg * 16 + (l & 3) * 4;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float s = 0.f;
            if (c < tile.cnt && r + j < rank)
                for (int q = 0; q < a.S; ++q) s += a.part[((int64_t)q * a.P + tile.p0 + c) * a.R + r + j];
            v[j] = sc * s;
        }
        float4* d = s_v + (int64_t)((m * kgs + kg) * 4) * 32 + l;
        float4 hi = make_float4(tf32_of(v[0]), tf32_of(v[1]), tf32_of(v[2]), tf32_of(v[3]));
        // what tf32 cannot hold of v; an infinite or NaN v has no rest
        float4 lo = make_float4(v[0] - hi.x, v[1] - hi.y, v[2] - hi.z, v[3] - hi.w);
        d[h * 32] = hi;
        d[(2 + h) * 32] = make_float4(isfinite(v[0]) ? tf32_of(lo.x) : 0.f, isfinite(v[1]) ? tf32_of(lo.y) : 0.f,
                                      isfinite(v[2]) ? tf32_of(lo.z) : 0.f, isfinite(v[3]) ? tf32_of(lo.w) : 0.f);
    }
    __syncthreads();
    const T* B = reinterpret_cast<const T*>(a.B) + (int64_t)tile.ad * a.N * a.R;
    Y* y = reinterpret_cast<Y*>(a.y);
    const int f_end = min(a.N, (int)(blockIdx.y + 1) * feats), mts = (tile.cnt + 15) / 16;
    for (int f0 = blockIdx.y * feats + warp * 32; f0 < f_end; f0 += 256) {
        float acc[MT][4][4] = {};
        for (int kg = 0; kg < kgs; ++kg) {
            const int r = kg * 16 + t * 4;
            float2 b[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int f = f0 + 8 * (g >> 1) + 2 * j + (g & 1);
                uint32_t w0 = 0, w1 = 0;
                if (f < a.N) {
                    const T* br = B + (int64_t)f * a.R + r;
                    if (vec_b && r + 4 <= rank) {
                        const uint2 q = __ldg(reinterpret_cast<const uint2*>(br));
                        w0 = q.x; w1 = q.y;
                    } else {
                        const unsigned short* bs = reinterpret_cast<const unsigned short*>(br);
                        if (r < rank) w0 = bs[0];
                        if (r + 1 < rank) w0 |= (uint32_t)bs[1] << 16;
                        if (r + 2 < rank) w1 = bs[2];
                        if (r + 3 < rank) w1 |= (uint32_t)bs[3] << 16;
                    }
                }
                b[j][0] = pair_f<T>(w0);
                b[j][1] = pair_f<T>(w1);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (m >= mts) break;
                const float4* d = s_v + (m * kgs + kg) * 128 + lane;
                const float4 h0 = d[0], h1 = d[32], l0 = d[64], l1 = d[96];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma_tf32(acc[m][j], l0.x, l1.x, l0.y, l1.y, b[j][0].x, b[j][0].y);
                    mma_tf32(acc[m][j], l0.z, l1.z, l0.w, l1.w, b[j][1].x, b[j][1].y);
                    mma_tf32(acc[m][j], h0.x, h1.x, h0.y, h1.y, b[j][0].x, b[j][0].y);
                    mma_tf32(acc[m][j], h0.z, h1.z, h0.w, h1.w, b[j][1].x, b[j][1].y);
                }
            }
        }
        const int f = f0 + 8 * t, have = min(8, a.N - f);
        if (have <= 0) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = srow[m * 16 + h * 8 + g];
                if (row < 0) continue;
                Y* p = y + (int64_t)row * a.N + f;
                float v[8];
                load8(p, have, vec_y, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[2 * j] += acc[m][j][2 * h];
                    v[2 * j + 1] += acc[m][j][2 * h + 1];
                }
                store8(p, have, vec_y, v);
            }
    }
}

// How the first launch is cut: a rule on P and the number of adapters alone, because the scratch is sized by it.
// Eight-row tiles (the least mma.sync multiplies) while an adapter has few rows, 32-row tiles above (each A is then
// read once per 32 rows); the sum over K is spread until two blocks per SM have work.
inline bool lora_wide(int P, int nA) { return P > 8 * (int64_t)nA; }
inline int lora_split(int P, int nA) {
    const int64_t tiles = (nA < P ? nA : P) + P / (lora_wide(P, nA) ? 32 : 8);
    const int64_t s = 296 / tiles;
    return s < 1 ? 1 : s > 8 ? 8 : (int)s;
}

template <typename T, int MT, int NTK>
int run_shrink(const LoraArgs& a, cudaStream_t s) {
    constexpr size_t smem = (size_t)kShWarps * 16 * MT * 8 * NTK * 4;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(lora_shrink_kernel<T, MT, NTK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return GSB_ERR_CUDA;
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / (8 * NTK);
    lora_shrink_kernel<T, MT, NTK><<<dim3(tiles, a.S, (a.R + 16 * MT - 1) / (16 * MT)), kShWarps * 32, smem, s>>>(a);
    return launch_status();
}

template <typename T, typename Y, int MT>
int run_expand(const LoraArgs& a, cudaStream_t s) {
    const size_t smem = (size_t)MT * ((a.R + 15) / 16) * 128 * sizeof(float4);
    auto kernel = lora_expand_kernel<T, Y, MT>;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return GSB_ERR_CUDA;
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / (16 * MT);
    // features in ranges of whole passes of the block (256), until about four blocks per SM have work
    const int passes = (a.N + 255) / 256;
    int per = (int)(((int64_t)passes * tiles + 591) / 592);
    per = per < 1 ? 1 : per > passes ? passes : per;
    const int vec_b = a.R % 4 == 0 && !misaligned(a.B, 8);
    const int vec_y = a.N % (16 / (int)sizeof(Y)) == 0 && !misaligned(a.y, 16);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles, (passes + per - 1) / per); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, per * 256, vec_b, vec_y) == cudaSuccess ? GSB_OK : GSB_ERR_LAUNCH;
}

template <typename T, typename Y>
int run_lora(const LoraArgs& a, cudaStream_t s) {
    const bool wide = lora_wide(a.P, a.nA);
    int st;
    if (wide) st = a.R <= 16 ? run_shrink<T, 1, 4>(a, s) : a.R <= 32 ? run_shrink<T, 2, 4>(a, s) : run_shrink<T, 4, 4>(a, s);
    else st = a.R <= 16 ? run_shrink<T, 1, 1>(a, s) : a.R <= 32 ? run_shrink<T, 2, 1>(a, s) : run_shrink<T, 4, 1>(a, s);
    if (st) return st;
    return wide && a.R <= 64 ? run_expand<T, Y, 4>(a, s) : run_expand<T, Y, 1>(a, s);
}

}  // namespace

}  // namespace gsb

using namespace gsb;

extern "C" size_t gsb_lora_scratch_bytes(int P, int max_rank, int n_adapters) {
    if (P <= 0 || max_rank <= 0 || n_adapters <= 0) return 0;
    return (size_t)lora_split(P, n_adapters) * P * max_rank * 4;
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
    a.S = lora_split(P, n_adapters); a.part = reinterpret_cast<float*>(scratch); a.y = y;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (type == GSB_TYPE_BF16)
        return y_type == GSB_TYPE_F32 ? run_lora<__nv_bfloat16, float>(a, s) : run_lora<__nv_bfloat16, __nv_bfloat16>(a, s);
    return y_type == GSB_TYPE_F32 ? run_lora<__half, float>(a, s) : run_lora<__half, __half>(a, s);
}
