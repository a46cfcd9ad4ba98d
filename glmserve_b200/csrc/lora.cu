// Low-rank adapters of many requests beside a shared projection:
//   v[p, :] = scale[a] * A[a] x[t, :],   y[t, :] += B[a] v[p, :]        t = rows[p], a = the adapter of p's segment
// Two launches, both over tiles of one adapter's rows: the first takes the long sum over the input dim (x and A are
// read once), the second spreads the few values v over the output (y is read and written once, B read once per tile).
// Both are bound by those bytes; the tensor cores only keep the arithmetic out of the way, so mma.sync fed straight from
// global memory does: every lane loads 16 (B: 8) contiguous bytes of a row and takes them as its k positions in the
// fragments of BOTH operands - a sum does not care in which order k runs.
#include <type_traits>

#include "launchers.cuh"
#include "segments.cuh"
#include "tc5.cuh"

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
    return a.ranks ? min(max(a.ranks[ad], 0), a.R) : a.R;
}

constexpr int kMaxRank = 256, kMaxSplit = 8;

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
// ---- first launch: v ---------------------------------------------------------------------------
// Early: the kernel may be there while its inputs are written (before the second launch of two stands an ordinary one).
template <bool Early, typename V> __device__ __forceinline__ V load_in(const V* p) {
    if constexpr (Early) return *p;
    else return __ldg(p);
}
// This warp's share of D[rank, row] for eight rows of one adapter and 16 * MT ranks from r0 on: the 32-column chunks
// c0, c0 + stride, ... of the sum over K.
template <typename T, int MT, bool Early>
__device__ __forceinline__ void shrink_sum(const LoraArgs& a, const LoraTile& tile, int rank, int r0, int c0, int stride, float (&acc)[MT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const T* A = reinterpret_cast<const T*>(a.A) + ((int64_t)tile.ad * a.R + r0) * a.K + t * 8;
    const int row = g < tile.cnt ? a.rows[tile.p0 + g] : -1;
    const bool xin = row >= 0 && row < a.n;
    const T* xr = reinterpret_cast<const T*>(a.x) + (int64_t)(xin ? row : 0) * a.K + t * 8;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int chunks = (a.K + 31) / 32;
    constexpr int U = MT >= 4 ? 2 : 4;                 // chunks in flight
    for (; c0 < chunks; c0 += stride * U) {
        uint4 fa[U][MT][2], fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c0 + u * stride) * 32;
            const bool in = k + t * 8 < a.K;
            fx[u] = in && xin ? load_in<Early>(reinterpret_cast<const uint4*>(xr + k)) : zero;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = m * 16 + h * 8 + g;  // what lies behind the adapter's rank counts as zero
                    fa[u][m][h] = in && r0 + r < rank ? load_in<Early>(reinterpret_cast<const uint4*>(A + (int64_t)r * a.K + k)) : zero;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mma_k16<T>(acc[m], fa[u][m][0].x, fa[u][m][1].x, fa[u][m][0].y, fa[u][m][1].y, fx[u].x, fx[u].y);
                mma_k16<T>(acc[m], fa[u][m][0].z, fa[u][m][1].z, fa[u][m][0].w, fa[u][m][1].w, fx[u].z, fx[u].w);
            }
    }
}

// The warps' shares through shared memory ([warp][rank][row]), then put(row, rank, sum over the warps in order).
template <int MT, typename F>
__device__ __forceinline__ void shrink_add(const float (&acc)[MT][4], float* s_red, F put) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int RT = 16 * MT;
    float* mine = s_red + (threadIdx.x >> 5) * RT * 8;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 4; ++h) mine[(m * 16 + (h >> 1) * 8 + g) * 8 + t * 2 + (h & 1)] = acc[m][h];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 8; i += kShWarps * 32) {
        const int c = i / RT, r = i - c * RT;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kShWarps; ++w) s += s_red[(w * RT + r) * 8 + c];
        put(c, r, s);
    }
}

// Block: up to eight rows of one adapter x 16 * MT ranks; its eight warps and a.S blocks share the sum over K (adjacent
// chunks go to adjacent warps).  The warps' tiles are added in shared memory in warp order, the blocks' parts by the
// second launch in block order.
template <typename T, int MT>
__global__ void __launch_bounds__(kShWarps * 32)
lora_shrink_kernel(const LoraArgs a) {
    extern __shared__ float s_red[];
    __shared__ int pre[kMaxE + 4], wsum[8];
    pdl_trigger();    // (an ordinary launch: what the kernels ahead wrote is there, for the second launch too)
    int descending = seg_scan(a.offsets, a.nA, a.P, 3, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<8>(a, pre, blockIdx.x, descending);
    if (tile.ad < 0) return;
    const int r0 = blockIdx.z * 16 * MT, rank = rank_of(a, tile.ad);
    if (r0 >= rank) return;
    float acc[MT][4] = {};
    shrink_sum<T, MT, false>(a, tile, rank, r0, blockIdx.y * kShWarps + (threadIdx.x >> 5), kShWarps * a.S, acc);
    shrink_add<MT>(acc, s_red, [&](int c, int r, float s) {
        if (c < tile.cnt && r0 + r < rank) a.part[((int64_t)blockIdx.y * a.P + tile.p0 + c) * a.R + r0 + r] = s;
    });
}

// The same for adapters with many rows: 64 rows x 16 * MT ranks, D[row, rank], over K steps of 64 columns that 16-byte
// asynchronous copies bring into a ring in shared memory (rows of 128 bytes, 16-byte piece c of row q at c ^ q % 8), so
// that 48 KB a block stay in flight without a register: the direct kernel above, at 32 rows x 64 ranks a block, has room
// for one step and measured 91 us for 8192 rows of 6144 at rank 64, this one 33 us.  Warps: four groups of 16 rows x two
// halves of each K step.
constexpr int kWdRows = 64, kWdStages = 4;
template <int MT> constexpr int wd_stage_bytes() { return (kWdRows + 16 * MT) * 128; }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T, int MT>
__global__ void __launch_bounds__(256, 2)
lora_shrink_wide_kernel(const LoraArgs a) {
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ int pre[kMaxE + 4], wsum[8];
    constexpr int RT = 16 * MT, SB = wd_stage_bytes<MT>();
    pdl_trigger();    // (an ordinary launch: what the kernels ahead wrote is there, for the second launch too)
    int descending = seg_scan(a.offsets, a.nA, a.P, 6, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<kWdRows>(a, pre, blockIdx.x, descending);
    if (tile.ad < 0) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = blockIdx.z * RT, rank = rank_of(a, tile.ad);
    if (r0 >= rank) return;
    const int steps = (a.K + 63) / 64, k_lo = steps * (int)blockIdx.y / a.S, k_hi = steps * ((int)blockIdx.y + 1) / a.S;
    // copies: thread = 16-byte piece tid % 8 of rows tid / 8 + 32 i
    const int piece = tid & 7, q0 = tid >> 3;
    const T* xs[2];
    bool xin[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = q0 + 32 * i, row = c < tile.cnt ? a.rows[tile.p0 + c] : -1;
        xin[i] = row >= 0 && row < a.n;
        xs[i] = reinterpret_cast<const T*>(a.x) + (int64_t)(xin[i] ? row : 0) * a.K + piece * 8;
    }
    const T* A = reinterpret_cast<const T*>(a.A) + ((int64_t)tile.ad * a.R + r0) * a.K + piece * 8;
    const uint32_t ring = smem_u32(s_ring), sw = (uint32_t)((piece ^ (q0 & 7)) << 4);
    auto copy = [&](int step) {
        if (step < k_hi) {
            const uint32_t base = ring + (uint32_t)((step - k_lo) % kWdStages) * SB;
            const bool in = step * 64 + piece * 8 < a.K;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                tc5::cp_async16(base + (uint32_t)((q0 + 32 * i) * 128) + sw, in && xin[i] ? xs[i] + step * 64 : xs[i], in && xin[i]);
#pragma unroll
            for (int i = 0; i < (RT + 31) / 32; ++i) {
                const int r = q0 + 32 * i;
                const bool have = in && r < RT && r0 + r < rank;    // what lies behind the adapter's rank counts as zero
                if (r < RT) tc5::cp_async16(base + (uint32_t)((kWdRows + r) * 128) + sw, have ? A + (int64_t)r * a.K + step * 64 : A, have);
            }
        }
        tc5::cp_async_commit();
    };
    for (int i = 0; i < kWdStages - 1; ++i) copy(k_lo + i);
    const int wr = (warp & 3) * 16, wk = warp >> 2;        // this warp's rows, and its half of the step
    float acc[2 * MT][4] = {};
    for (int step = k_lo; step < k_hi; ++step) {
        tc5::cp_async_wait<kWdStages - 2>();
        __syncthreads();                                   // the step is there, and the stage copied into next is free
        copy(step + kWdStages - 1);
        const uint32_t base = ring + (uint32_t)((step - k_lo) % kWdStages) * SB;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c0 = wk * 4 + kk * 2;                // first 16-byte piece of these 16 columns
            uint32_t fx[4], fa[4];
            const int xr = wr + (lane & 15);
            ldsm4(base + (uint32_t)(xr * 128 + (((c0 + (lane >> 4)) ^ (xr & 7)) << 4)), fx);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                // ranks m * 16 + 0..7 in fa[0], fa[1], ranks m * 16 + 8..15 in fa[2], fa[3]
                const int ar = m * 16 + (lane & 7) + ((lane >> 4) << 3);
                ldsm4(base + (uint32_t)((kWdRows + ar) * 128 + (((c0 + ((lane >> 3) & 1)) ^ (ar & 7)) << 4)), fa);
                mma_k16<T>(acc[2 * m], fx[0], fx[1], fx[2], fx[3], fa[0], fa[1]);
                mma_k16<T>(acc[2 * m + 1], fx[0], fx[1], fx[2], fx[3], fa[2], fa[3]);
            }
        }
    }
    tc5::cp_async_wait<0>();
    __syncthreads();
    // the second half's sums are added to the first's
    float* red = reinterpret_cast<float*>(s_ring);
    const int g = lane >> 2, t = lane & 3;
    if (wk == 1)
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h) red[((warp & 3) * 8 * MT + j * 4 + h) * 32 + lane] = acc[j][h];
    __syncthreads();
    if (wk == 0)
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int c = wr + (h >> 1) * 8 + g, r = r0 + j * 8 + t * 2 + (h & 1);
                if (c < tile.cnt && r < rank)
                    a.part[((int64_t)blockIdx.y * a.P + tile.p0 + c) * a.R + r] = acc[j][h] + red[(warp * 8 * MT + j * 4 + h) * 32 + lane];
            }
}

// ---- second launch: y += B v ---------------------------------------------------------------------
// Block: up to 16 * MT rows of one adapter x a range of features, 32 features a warp at a time, D[row, feature].
// v enters the 16-bit tensor cores as a sum of three 16-bit numbers, so that y's fp32 sums keep fp32 accuracy: three bf16
// numbers hold all 24 bits.  For fp16 each row of v is scaled by a power of two to a largest finite value in
// [2^14, 2^15), and every part holds 2^11 times the rest that the part before left, or its bits would fall below fp16's
// range: v = p0 + 2^-11 p1 + 2^-22 p2 holds all 24 bits of what is above 2^-37 of the row's largest, and is off by at most
// 2^-61 of the largest below that.  The sums over the parts are scaled alike, the last part's first.  (tf32 would do it in
// two for both types, but mma.sync runs tf32 at the rate of plain fp32 multiply-adds here: 192 us instead of 121 for 8192
// rows of 6144 at rank 64.)  n-tile j of a warp's chunk holds features 8 (c / 2) + 2 j + c % 2 in its columns c: lane t
// of a quad then owns eight contiguous features of a row.
template <typename T> __device__ __forceinline__ float2 pair_f(uint32_t v);
template <> __device__ __forceinline__ float2 pair_f<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <> __device__ __forceinline__ float2 pair_f<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

template <typename T> struct Split;      // v as the sum of N numbers of type T, each after the first times 2^lg
template <> struct Split<__nv_bfloat16> { static constexpr int N = 3, lg = 0; static constexpr bool scaled = false; };
template <> struct Split<__half> { static constexpr int N = 3, lg = 11; static constexpr bool scaled = true; };

// One part of v, and in v what the next is taken from.  Infinity and NaN have no rest; a finite value that rounds to
// infinity is cut instead.
template <typename T>
__device__ __forceinline__ T next_part(float& v) {
    T p = from_f<T>(v);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        if (isinf(to_f(p)) && isfinite(v)) p = __float2bfloat16_rz(v);
    }
    v = isfinite(v) ? (v - to_f(p)) * (float)(1 << Split<T>::lg) : 0.f;
    return p;
}

// The power of two that lifts `top` into [2^14, 2^15), kept where it and its inverse are normal; 0 for zero.
__device__ __forceinline__ int row_exponent(float top) {
    const int ex = 14 - ((int)((__float_as_uint(top) >> 23) & 0xff) - 127);
    return top > 0.f ? min(max(ex, -126), 126) : 0;
}
// what a value counts for the row's largest: infinity and NaN nothing, or the finite ones beside them would leave the range
__device__ __forceinline__ float magnitude(float v) { return isfinite(v) ? fabsf(v) : 0.f; }

template <typename T> __device__ __forceinline__ uint32_t pack2(T a, T b) {
    const unsigned short x = *reinterpret_cast<const unsigned short*>(&a), y = *reinterpret_cast<const unsigned short*>(&b);
    return (uint32_t)x | ((uint32_t)y << 16);
}

// eight values of y as they lie in memory
template <typename Y> struct Raw8 { uint4 q[sizeof(Y) / 2]; };
template <typename Y>
__device__ __forceinline__ Raw8<Y> load8(const Y* p, int have, bool vec) {
    Raw8<Y> v;
    if (vec && have == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(Y) / 2; ++i) v.q[i] = *(reinterpret_cast<const uint4*>(p) + i);
    } else {
        uint32_t w[sizeof(Y) * 2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(Y) == 4) w[i] = i < have ? __float_as_uint(p[i]) : 0u;
            else {
                const uint32_t h = i < have ? (uint32_t)reinterpret_cast<const unsigned short*>(p)[i] : 0u;
                if (i & 1) w[i >> 1] |= h << 16; else w[i >> 1] = h;
            }
        }
#pragma unroll
        for (int i = 0; i < (int)sizeof(Y) / 2; ++i) v.q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    return v;
}
template <typename Y>
__device__ __forceinline__ void add_store8(Y* p, int have, bool vec, const Raw8<Y>& raw, const float (&d)[8]) {
    float v[8];
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(Y) == 4) v[i] = __uint_as_float(w[i]) + d[i];
        else { const float2 f = pair_f<Y>(w[i >> 1]); v[i] = (i & 1 ? f.y : f.x) + d[i]; }
    }
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

// The parts of v[p, r] added in order, all loads in flight at once.
__device__ __forceinline__ float sum_parts(const LoraArgs& a, int p, int r) {
    const float* q0 = a.part + (int64_t)p * a.R + r;
    const int64_t step = (int64_t)a.P * a.R;
    float v[kMaxSplit], s = 0.f;
#pragma unroll
    for (int q = 0; q < kMaxSplit; ++q) v[q] = q < a.S ? __ldcg(q0 + q * step) : 0.f;
#pragma unroll
    for (int q = 0; q < kMaxSplit; ++q) s += v[q];
    return s;
}

// v of a tile into shared memory as A fragments ([row tile of 16][16 ranks][part][lane]), eight lanes a row, each every
// eighth run of two ranks; up to 16 * KG ranks (0: any number, read twice where a row is scaled).  of(row, rank) is v.
template <typename T, int MT, int KG, typename F>
__device__ __forceinline__ void stage_v(int cnt, int rank, F of, uint4* s_v, float* s_scale) {
    constexpr int NS = Split<T>::N;
    const int kgs = (rank + 15) / 16, l8 = threadIdx.x & 7, cr = threadIdx.x >> 3;
    if (cr >= 16 * MT) return;                           // (whole warps: 16 rows are four)
    auto value = [&](int r) { return cr < cnt && r < rank ? of(cr, r) : 0.f; };
    float v[KG ? 2 * KG : 2], up = 1.f;
    if (KG) {
#pragma unroll
        for (int i = 0; i < KG; ++i) { v[2 * i] = value(i * 16 + l8 * 2); v[2 * i + 1] = value(i * 16 + l8 * 2 + 1); }
    }
    if (Split<T>::scaled) {
        float top = 0.f;
        if (KG) {
#pragma unroll
            for (int i = 0; i < 2 * KG; ++i) top = fmaxf(top, magnitude(v[i]));
        } else {
            for (int r = l8 * 2; r < kgs * 16; r += 16) top = fmaxf(top, fmaxf(magnitude(value(r)), magnitude(value(r + 1))));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = row_exponent(top);
        up = __int_as_float((ex + 127) << 23);
        if (l8 == 0) s_scale[cr] = __int_as_float((127 - ex) << 23);
    }
#pragma unroll
    for (int kg = 0; kg < (KG ? KG : kMaxRank / 16); ++kg) {
        if (kg >= kgs) break;
        const int r = kg * 16 + l8 * 2;
        float v0 = up * (KG ? v[KG ? 2 * kg : 0] : value(r)), v1 = up * (KG ? v[KG ? 2 * kg + 1 : 0] : value(r + 1));
        // ranks 4 t' .. 4 t' + 3 of a group are lane t' of the quad: two in the first, two in the last register pair
        const int tq = l8 >> 1, hi_pair = l8 & 1;
        uint32_t* d = reinterpret_cast<uint32_t*>(s_v + (((cr >> 4) * kgs + kg) * NS) * 32 + (cr & 7) * 4 + tq) +
                      hi_pair * 2 + ((cr >> 3) & 1);
#pragma unroll
        for (int u = 0; u < NS; ++u) {
            const T p0 = next_part<T>(v0), p1 = next_part<T>(v1);
            d[u * 128] = pack2(p0, p1);
        }
    }
}

// One warp's way through features of a tile of 16 * MT rows, 32 at a time.  KG: groups of 16 ranks whose B values are
// loaded ahead together with y (0: any number of ranks, B loaded in turn).
template <typename T, typename Y, int MT, int KG, bool Early>
struct Expand {
    static constexpr int NS = Split<T>::N;
    struct Ahead { Raw8<Y> y[2 * MT]; uint2 b[KG ? KG : 1][4]; };
    const LoraArgs& a;
    const T* B;
    const uint4* s_v;
    const float* s_scale;
    int rank, kgs, f_end, row[2 * MT];
    bool vec_b, vec_y;

    __device__ __forceinline__ Expand(const LoraArgs& args, const LoraTile& tile, int rk, const uint4* v, const float* scale, int end, int flags)
        : a(args), B(reinterpret_cast<const T*>(args.B) + (int64_t)tile.ad * args.N * args.R), s_v(v), s_scale(scale), rank(rk),
          kgs((rk + 15) / 16), f_end(end), vec_b(flags & 1), vec_y(flags & 2) {
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) {
            const int c = m * 8 + ((threadIdx.x & 31) >> 2), r = c < tile.cnt ? a.rows[tile.p0 + c] : -1;
            row[m] = r < a.n ? r : -1;
        }
    }
    // four ranks of feature n of n-tile j, as two packed pairs
    __device__ __forceinline__ uint2 load_b(int f0, int kg, int j) const {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
        const int f = f0 + 8 * (g >> 1) + 2 * j + (g & 1), r = kg * 16 + t * 4;
        uint2 w = make_uint2(0, 0);
        if (f < a.N) {
            const T* br = B + (int64_t)f * a.R + r;
            if (vec_b && r + 4 <= rank) w = load_in<Early>(reinterpret_cast<const uint2*>(br));
            else {
                const unsigned short* bs = reinterpret_cast<const unsigned short*>(br);
                if (r < rank) w.x = bs[0];
                if (r + 1 < rank) w.x |= (uint32_t)bs[1] << 16;
                if (r + 2 < rank) w.y = bs[2];
                if (r + 3 < rank) w.y |= (uint32_t)bs[3] << 16;
            }
        }
        return w;
    }
    __device__ __forceinline__ void load(Ahead& q, int f0) const {
        if (f0 >= f_end) return;
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int j = 0; j < 4; ++j) q.b[kg][j] = kg < kgs ? load_b(f0, kg, j) : make_uint2(0, 0);
        const int f = f0 + 8 * (threadIdx.x & 3);
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m)
            if (row[m] >= 0 && f < a.N) q.y[m] = load8(reinterpret_cast<const Y*>(a.y) + (int64_t)row[m] * a.N + f, min(8, a.N - f), vec_y);
    }
    __device__ __forceinline__ static void lower(float (&d)[4]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) d[h] *= 1.f / (1 << Split<T>::lg);
    }
    __device__ __forceinline__ void finish(const Ahead& q, int f0) const {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        float acc[MT][4][4] = {};
        // small parts first; where the parts are scaled, so are the sums between two parts: all of them where B is in
        // registers, else those of 16 ranks
        if constexpr (Split<T>::scaled && KG > 0) {
#pragma unroll
            for (int u = NS - 1; u >= 0; --u) {
                if (u < NS - 1) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) lower(acc[m][j]);
                }
#pragma unroll
                for (int kg = 0; kg < KG; ++kg) {
                    if (kg >= kgs) break;
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint4 v = s_v[((m * kgs + kg) * NS + u) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma_k16<T>(acc[m][j], v.x, v.y, v.z, v.w, q.b[kg][j].x, q.b[kg][j].y);
                    }
                }
            }
        } else {
            for (int kg = 0; kg < (KG ? KG : kgs); ++kg) {
                if (kg >= kgs) break;
                uint2 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = KG ? q.b[kg][j] : load_b(f0, kg, j);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float rest[4][4] = {};
#pragma unroll
                    for (int u = NS - 1; u >= 0; --u) {
                        const uint4 v = s_v[((m * kgs + kg) * NS + u) * 32 + lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (Split<T>::scaled && u) {
                                mma_k16<T>(rest[j], v.x, v.y, v.z, v.w, b[j].x, b[j].y);
                                lower(rest[j]);
                            } else {
                                if (Split<T>::scaled) {
#pragma unroll
                                    for (int h = 0; h < 4; ++h) acc[m][j][h] += rest[j][h];
                                }
                                mma_k16<T>(acc[m][j], v.x, v.y, v.z, v.w, b[j].x, b[j].y);
                            }
                        }
                    }
                }
            }
        }
        const int f = f0 + 8 * (lane & 3), have = min(8, a.N - f);
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) {
            if (row[m] < 0 || have <= 0) continue;
            float d[8];
            const float back = Split<T>::scaled ? s_scale[m * 8 + g] : 1.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[2 * j] = back * acc[m >> 1][j][2 * (m & 1)];
                d[2 * j + 1] = back * acc[m >> 1][j][2 * (m & 1) + 1];
            }
            add_store8(reinterpret_cast<Y*>(a.y) + (int64_t)row[m] * a.N + f, have, vec_y, q.y[m], d);
        }
    }
};

template <typename T, typename Y, int MT, int KG>
__global__ void __launch_bounds__(256, MT == 1 && KG == 1 ? 3 : 2)
lora_expand_kernel(const LoraArgs a, int feats, int flags) {
    extern __shared__ uint4 s_v[];                    // [row tile of 16][16 ranks][part][lane]: A fragments
    __shared__ int pre[kMaxE + 4], wsum[8];
    __shared__ float s_scale[16 * MT];                // what a row's sums are multiplied by at the end
    int descending = seg_scan(a.offsets, a.nA, a.P, MT == 1 ? 4 : 5, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<16 * MT>(a, pre, blockIdx.x, descending);
    const int rank = tile.ad < 0 ? 0 : rank_of(a, tile.ad);
    if (rank == 0) {
        pdl_wait();                                      // this launch does not end before the first
        return;
    }
    const float sc = a.scales ? a.scales[tile.ad] : 1.f;
    const Expand<T, Y, MT, KG, false> ex(a, tile, rank, s_v, s_scale, min(a.N, (int)(blockIdx.y + 1) * feats), flags);
    int f0 = blockIdx.y * feats + (threadIdx.x >> 5) * 32;
    typename Expand<T, Y, MT, KG, false>::Ahead q;
    ex.load(q, f0);                                      // B and y do not wait for the first launch
    pdl_wait();                                          // v comes from it
    // 32-row tiles take ranks up to 64, which registers hold where v would be read twice (8192 rows of 6144 to 6144 at rank
    // 64, fp16 and a 16-bit y: 135 us against 163)
    stage_v<T, MT, MT == 2 && !KG && Split<T>::scaled ? 4 : KG>(tile.cnt, rank, [&](int c, int r) { return sc * sum_parts(a, tile.p0 + c, r); }, s_v, s_scale);
    __syncthreads();
    for (; f0 < ex.f_end; f0 += 256) {
        ex.finish(q, f0);
        ex.load(q, f0 + 256);
    }
}

// ---- both sums in one launch, for few rows -------------------------------------------------------
// A cluster of eight blocks takes eight rows of one adapter: each block an eighth of the sum over K, then, with the
// others' parts read from their shared memory and added in rank order, an eighth of the output features.  One launch and
// no scratch: with few rows the two-launch form waits for launches and its partial sums more than for memory.
constexpr int kClusterBlocks = 8;
template <typename T, typename Y, int KG>
__global__ void __launch_bounds__(256, 2)
lora_cluster_kernel(const LoraArgs a, int feats, int flags) {
    constexpr int RT = 16 * KG;
    __shared__ uint4 s_v[KG * Split<T>::N * 32];
    __shared__ float s_red[kShWarps * RT * 8], s_part[RT * 8], s_scale[16];
    __shared__ int pre[kMaxE + 4], wsum[8];
    pdl_trigger();
    pdl_wait();
    int descending = seg_scan(a.offsets, a.nA, a.P, 3, pre, wsum);
    descending = __syncthreads_or(descending);
    const LoraTile tile = lora_tile<8>(a, pre, blockIdx.x / kClusterBlocks, descending);
    const int rank = tile.ad < 0 ? 0 : rank_of(a, tile.ad), block = (int)tc5::cluster_rank(), warp = threadIdx.x >> 5;
    if (rank == 0) return;                               // (the same for all blocks of the cluster)
    const float sc = a.scales ? a.scales[tile.ad] : 1.f;
    const Expand<T, Y, 1, KG, true> ex(a, tile, rank, s_v, s_scale, min(a.N, (block + 1) * feats), flags);
    int f0 = block * feats + warp * 32;
    float acc[KG][4] = {};
    shrink_sum<T, KG, true>(a, tile, rank, 0, block * kShWarps + warp, kShWarps * kClusterBlocks, acc);
    typename Expand<T, Y, 1, KG, true>::Ahead q;
    ex.load(q, f0);                                      // on its way while the parts of v are put together
    shrink_add<KG>(acc, s_red, [&](int c, int r, float s) { s_part[r * 8 + c] = s; });
    tc5::cluster_sync_all();
    const uint32_t part = smem_u32(s_part);
    stage_v<T, 1, KG>(tile.cnt, rank, [&](int c, int r) {
        float v[kClusterBlocks], s = 0.f;
#pragma unroll
        for (int b = 0; b < kClusterBlocks; ++b) v[b] = tc5::ld_cluster(tc5::map_rank(part + (uint32_t)((r * 8 + c) * 4), (uint32_t)b));
#pragma unroll
        for (int b = 0; b < kClusterBlocks; ++b) s += v[b];
        return sc * s;
    }, s_v, s_scale);
    __syncthreads();
    tc5::cluster_arrive();                               // this block has read the others' parts
    for (; f0 < ex.f_end; f0 += 256) {
        ex.finish(q, f0);
        ex.load(q, f0 + 256);
    }
    __syncwarp();
    tc5::cluster_wait();                                 // and they have read its own
}

// The same on tcgen05, for ranks up to 64: D[feature, row] = sum over v's parts of B[feature, :] v_part[row, :], 128
// features (TMEM lanes) x up to 64 rows of one adapter a unit, the CTAs taking equal runs of the sequence (tile, its
// feature blocks).  The product is nothing; what this buys is the way y is met: a lane holds one feature of every row, so
// a warp reads and writes whole 128-byte lines straight from registers, one load, one add and one store a value, with the
// loads of 32 rows on their way before the product is waited for.  (mma.sync's fragments are 8-byte pieces of eight rows:
// the kernel above took 121 us for 8192 rows of 6144 at rank 64, bound by its instructions, this one 85 us.)
// B comes by TMA as 128-byte rows of 64 ranks, zeros behind R, where R % 8 == 0; columns between an adapter's rank and the
// next multiple of 16 are zeroed in shared memory, since v's zeros would not hide a NaN there.  With any other R the tile's
// 128 rows are one piece of memory without 16-byte rows: it is copied as it lies and two warps lay it out.  Needs B
// 16-byte aligned.
constexpr int kTcNT = 64;                  // rows per tile at most
constexpr int kTcStages = 4;               // ring of B tiles
constexpr int kTcABytes = 128 * 128;
constexpr int kTcVBytes = kTcNT * 128;     // one part of v: 64 rows x 64 ranks
constexpr int kTcGroups = 4;               // of four epilogue warps, units in turn; accumulator slots
constexpr int kTcThreads = 128 + kTcGroups * 128;   // warps: 0 B, 1 MMA, 2 zeroes, 3 TMEM (2 and 3 lay B out), 4-19 epilogue
constexpr int kTcLinBytes = 128 * 64 * 2 + 256, kTcLin = 2;     // B tiles as they lie in memory: ring of two
constexpr long long kTcWaitLimit = 2000000000LL;
template <typename T> constexpr size_t tc_smem(bool tma) {
    return (size_t)kTcStages * kTcABytes + (size_t)Split<T>::N * kTcVBytes + (kMaxE + 4) * 4 + 1280 + (tma ? 0 : kTcLin * kTcLinBytes);
}

__device__ int g_lora_status;

__device__ __forceinline__ void lora_timeout(volatile int* abort_flag) {
    *abort_flag = 1;
    atomicCAS(&g_lora_status, 0, GSB_ERR_TIMEOUT);
}

// v of a tile as 128-byte swizzled rows of 64 ranks, a copy per part, for 512 threads: eight a row, eight ranks each.
template <typename T>
__device__ __forceinline__ void stage_v_rows(const LoraArgs& a, const LoraTile& tile, int rank, int e, uint8_t* s_vp, int64_t* s_off, float* s_back) {
    constexpr int NS = Split<T>::N;
    const int c = e >> 3, p8 = e & 7;
    const bool in = c < tile.cnt;
    if (p8 == 0) {
        const int r = in ? a.rows[tile.p0 + c] : -1;
        s_off[c] = r >= 0 && r < a.n ? (int64_t)r * a.N : -1;
    }
    const float sc = a.scales ? a.scales[tile.ad] : 1.f;
    float v[8], top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int r = p8 * 8 + j;
        v[j] = in && r < rank ? sc * sum_parts(a, tile.p0 + c, r) : 0.f;
        top = fmaxf(top, magnitude(v[j]));
    }
    if (Split<T>::scaled) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int ex = row_exponent(top);
        const float up = __int_as_float((ex + 127) << 23);
        if (p8 == 0) s_back[c] = __int_as_float((127 - ex) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= up;
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T h0 = next_part<T>(v[2 * j]), h1 = next_part<T>(v[2 * j + 1]);
            w[j] = pack2(h0, h1);
        }
        *reinterpret_cast<uint4*>(s_vp + u * kTcNT * 128 + c * 128 + ((p8 ^ (c & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// B's 128 rows from feature f0 on as one piece of memory: 16-byte aligned start and size, `head` elements before the first
// row.  The piece stays inside B; the last elements of B that a whole 16 bytes would overshoot are left out of it.
struct TcLin { const uint8_t* src; int bytes, head; };
__device__ __forceinline__ TcLin tc_lin(const LoraArgs& a, int ad, int f0) {
    const int64_t first = ((int64_t)ad * a.N + f0) * a.R * 2, last = first + (int64_t)min(128, a.N - f0) * a.R * 2;
    const int64_t all = (int64_t)a.nA * a.N * a.R * 2, beg = first & ~(int64_t)15, end = min((last + 15) & ~(int64_t)15, all & ~(int64_t)15);
    TcLin l;
    l.src = reinterpret_cast<const uint8_t*>(a.B) + beg;
    l.bytes = end > beg ? (int)(end - beg) : 0;
    l.head = (int)(first - beg) / 2;
    return l;
}

template <typename T, typename Y>
__global__ void __launch_bounds__(kTcThreads, 1)
lora_expand_tc_kernel(const LoraArgs a, const __grid_constant__ CUtensorMap tm_b, int tma) {
    constexpr int NS = Split<T>::N;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* s_vp = smem + kTcStages * kTcABytes;                       // parts of v, 128-byte swizzled rows
    int* pre = reinterpret_cast<int*>(s_vp + NS * kTcVBytes);
    uint64_t* b_full = reinterpret_cast<uint64_t*>(pre + kMaxE + 4);    // TMA -> zeroing warp
    uint64_t* b_ready = b_full + kTcStages;                            // zeroing warp -> MMA
    uint64_t* b_empty = b_ready + kTcStages;                           // MMA -> TMA
    uint64_t* acc_full = b_empty + kTcStages;                          // MMA -> epilogue group
    uint64_t* acc_empty = acc_full + kTcGroups;
    uint64_t* v_full = acc_empty + kTcGroups;                          // epilogue warps -> MMA: v of the next tile is there
    int64_t* s_off = reinterpret_cast<int64_t*>(v_full + 1);           // [64] where a row of y begins (elements), -1: no such row
    float* s_back = reinterpret_cast<float*>(s_off + kTcNT);           // [64] what a row's sums are multiplied by
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_back + kTcNT);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* wsum = reinterpret_cast<int*>(tmem_slot + 2);                 // [8]
    uint64_t* lin_full = reinterpret_cast<uint64_t*>(wsum + 8);        // [2] tile as it lies in memory -> warps 2 and 3
    uint64_t* lin_empty = lin_full + kTcLin;
    uint8_t* s_lin = smem + kTcStages * kTcABytes + NS * kTcVBytes + (kMaxE + 4) * 4 + 1280;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kTcStages; ++i) { mbar_init(&b_full[i], 1); mbar_init(&b_ready[i], tma ? 1 : 2); mbar_init(&b_empty[i], 1); }
        for (int i = 0; i < kTcLin; ++i) { mbar_init(&lin_full[i], 1); mbar_init(&lin_empty[i], 2); }
        for (int i = 0; i < kTcGroups; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4); }
        mbar_init(v_full, 4 * kTcGroups);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 3) { tc5::tmem_alloc(tmem_slot, kTcGroups * kTcNT); tc5::tmem_relinquish(); }
    int descending = (smem_u32(smem) & 1023u) != 0;
    descending |= seg_scan(a.offsets, a.nA, a.P, 6, pre, wsum);
    tc5::fence_before();
    descending = __syncthreads_or(descending);
    tc5::fence_after();
    const uint32_t tmem = *tmem_slot;
    const int FB = (a.N + 127) / 128;
    const int units = descending ? 0 : pre[a.nA] * FB;                  // (checked to fit by the host)
    const int u_beg = (int)((int64_t)units * blockIdx.x / gridDim.x), u_end = (int)((int64_t)units * (blockIdx.x + 1) / gridDim.x);

    if (u_beg == u_end) pdl_wait();        // this launch does not end before the first

    if (warp == 0) {                       // ---- B tiles
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0;
        const uint32_t ring = tma ? kTcStages : kTcLin;
        const int ahead = tma ? kTcStages : kTcStages + kTcLin;      // tiles that need no MMA before them
        uint64_t *fullb = tma ? b_full : lin_full, *emptyb = tma ? b_empty : lin_empty;
        LoraTile tile{-1, 0, 0};
        for (int u = u_beg; u < u_end && !tc5::warp_set(abort_flag); ++u) {
            if (u == u_beg || u % FB == 0) tile = lora_tile<kTcNT>(a, pre, u / FB, 0);
            if (u - u_beg == ahead) pdl_wait();    // bounded waits count from where the first launch has ended, which may take its time
            if (!tc5::warp_wait(&emptyb[st], ph ^ 1u, kTcWaitLimit)) { lora_timeout(abort_flag); break; }
            if (leader) {
                const int f0 = u % FB * 128;
                if (tma) {
                    mbar_arrive_expect_tx(&fullb[st], kTcABytes);
                    tc5::tma_load_3d(smem + st * kTcABytes, &tm_b, 0, f0, tile.ad, &fullb[st]);
                } else {
                    const TcLin l = tc_lin(a, tile.ad, f0);
                    mbar_arrive_expect_tx(&fullb[st], (uint32_t)l.bytes);
                    if (l.bytes) bulk_g2s(s_lin + st * kTcLinBytes, l.src, (uint32_t)l.bytes, &fullb[st]);
                }
            }
            if (++st == ring) { st = 0; ph ^= 1u; }
        }
        pdl_wait();
        for (uint32_t j = 0; j < ring && !tc5::warp_set(abort_flag); ++j) {           // the last tiles are done with, their signals in
            tc5::warp_wait(&emptyb[st], ph ^ 1u, kTcWaitLimit);
            if (++st == ring) { st = 0; ph ^= 1u; }
        }
        if (tc5::warp_set(abort_flag))                   // after a time-out: nothing may still be copying when the block ends
            for (uint32_t j = 0; j < ring; ++j) {
                if (st == 0) { st = ring; ph ^= 1u; }
                --st;
                tc5::warp_wait(&fullb[st], ph, kTcWaitLimit / 16);
            }
    } else if (warp == 2 || (warp == 3 && !tma)) {
        // ---- tma: zeroes between an adapter's rank and the next multiple of 16; else: the tile laid out, a warp 64 rows
        uint32_t st = 0, ph = 0, ls = 0, lph = 0;
        LoraTile tile{-1, 0, 0};
        int rank = 0;
        for (int u = u_beg; u < u_end && !tc5::warp_set(abort_flag); ++u) {
            if (u == u_beg || u % FB == 0) { tile = lora_tile<kTcNT>(a, pre, u / FB, 0); rank = rank_of(a, tile.ad); }
            uint8_t* at = smem + st * kTcABytes;
            if (u - u_beg == kTcStages) pdl_wait();
            if (tma) {
                if (!tc5::warp_wait(&b_full[st], ph, kTcWaitLimit)) { lora_timeout(abort_flag); break; }
                if (rank & 15) {
                    for (int f = lane; f < 128; f += 32)
                        for (int r = rank; r < ((rank + 15) & ~15); ++r)    // piece c of row f lies at c ^ f % 8
                            *reinterpret_cast<unsigned short*>(at + f * 128 + (((r >> 3) ^ (f & 7)) << 4) + (r & 7) * 2) = 0;
                    fence_proxy_async();
                }
            } else {
                if (!tc5::warp_wait(&lin_full[ls], lph, kTcWaitLimit) || !tc5::warp_wait(&b_empty[st], ph ^ 1u, kTcWaitLimit)) { lora_timeout(abort_flag); break; }
                const int f0 = u % FB * 128;
                const TcLin l = tc_lin(a, tile.ad, f0);
                const uint32_t* s32 = reinterpret_cast<const uint32_t*>(s_lin + ls * kTcLinBytes);
                const bool whole = (l.head + min(128, a.N - f0) * a.R) * 2 <= l.bytes;      // all but the last tile of B
                for (int f = (warp - 2) * 64 + lane, k = 0; k < 2; ++k, f += 32) {
                    const bool have = f0 + f < a.N;
                    const int i0 = have ? l.head + f * a.R : 0;                 // the row's first element in the piece
                    const uint32_t shift = (uint32_t)(i0 & 1) * 16;
                    const uint32_t* src = s32 + (i0 >> 1);
                    uint32_t low = src[0];
                    for (int c = 0; c < (rank + 15) / 16 * 2; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {       // two elements at once, half a word on where the row starts odd
                            const int r = c * 8 + j * 2;
                            if (whole || !have) {
                                const uint32_t high = src[(r >> 1) + 1];
                                w[j] = __funnelshift_r(low, high, shift);
                                low = high;
                            } else {
                                const unsigned short *in = reinterpret_cast<const unsigned short*>(s32), *out = reinterpret_cast<const unsigned short*>(l.src);
                                w[j] = 0;
                                for (int h = 0; h < 2; ++h)
                                    if (r + h < rank) w[j] |= (uint32_t)((i0 + r + h + 1) * 2 <= l.bytes ? in[i0 + r + h] : out[i0 + r + h]) << (16 * h);
                            }
                            if (!have || r >= rank) w[j] = 0;
                            else if (r + 1 == rank) w[j] &= 0xffffu;
                        }
                        *reinterpret_cast<uint4*>(at + f * 128 + ((c ^ (f & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&lin_empty[ls]);
                if (++ls == kTcLin) { ls = 0; lph ^= 1u; }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_ready[st]);
            if (++st == kTcStages) { st = 0; ph ^= 1u; }
        }
        pdl_wait();
        if (!tma)
            for (int j = 0; j < kTcStages && !tc5::warp_set(abort_flag); ++j) {       // the last MMAs' signals have arrived
                tc5::warp_wait(&b_empty[st], ph ^ 1u, kTcWaitLimit);
                if (++st == kTcStages) { st = 0; ph ^= 1u; }
            }
    } else if (warp == 1) {                // ---- MMA issue
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0, n = 0, vph = 0;
        constexpr uint32_t ab = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint64_t b0 = tc5::desc_sw128(smem_u32(smem)), v0 = tc5::desc_sw128(smem_u32(s_vp));
        LoraTile tile{-1, 0, 0};
        int kgs = 0;
        for (int u = u_beg; u < u_end && !tc5::warp_set(abort_flag); ++u, ++n) {
            if (u == u_beg || u % FB == 0) {
                tile = lora_tile<kTcNT>(a, pre, u / FB, 0);
                kgs = (rank_of(a, tile.ad) + 15) / 16;
                if (u == u_beg) pdl_wait();
                if (!tc5::warp_wait(v_full, vph, kTcWaitLimit)) { lora_timeout(abort_flag); break; }
                vph ^= 1u;
            }
            const uint32_t slot = n % kTcGroups;
            if (!tc5::warp_wait(&b_ready[st], ph, kTcWaitLimit) || !tc5::warp_wait(&acc_empty[slot], ((n / kTcGroups) & 1u) ^ 1u, kTcWaitLimit)) {
                lora_timeout(abort_flag);
                break;
            }
            tc5::fence_after();
            if (leader) {
                const uint32_t idesc = tc5::idesc_f16(ab, 128, (uint32_t)((tile.cnt + 15) & ~15));
                const uint64_t bd = b0 + (uint64_t)(st * (uint32_t)(kTcABytes >> 4));
                uint32_t acc = 0;
                for (int p = NS - 1; p >= 0; --p)          // small parts first; their sum is scaled by the next part's first product
                    for (int k = 0; k < kgs; ++k) {
                        const uint64_t vd = v0 + (uint64_t)(p * (kTcVBytes >> 4) + k * 2);
                        if (Split<T>::lg && !k && acc) tc5::mma_f16_ss_lower<Split<T>::lg>(tmem + slot * kTcNT, bd, vd, idesc);
                        else tc5::mma_f16_ss(tmem + slot * kTcNT, bd + (uint64_t)(k * 2), vd, idesc, acc);
                        acc = 1u;
                    }
                tc5::commit(&b_empty[st]);
                tc5::commit(&acc_full[slot]);
            }
            if (++st == kTcStages) { st = 0; ph ^= 1u; }
        }
        // after a time-out: no MMA is at work, and no signal on its way, when the block ends (otherwise the others have
        // waited for all of them)
        if (tc5::warp_set(abort_flag) && n) {
            if (st == 0) { st = kTcStages; ph ^= 1u; }
            tc5::warp_wait(&b_empty[st - 1], ph, kTcWaitLimit);
            tc5::warp_wait(&acc_full[(n - 1) % kTcGroups], ((n - 1) / kTcGroups) & 1u, kTcWaitLimit);
        }
    } else if (warp >= 4) {                // ---- v of a tile, then y of this group's units
        const int e = tid - 128, group = (warp - 4) >> 2, q = warp & 3;
        for (int us = u_beg; us < u_end;) {                // units of one tile
            const int ti = us / FB, ue = min(u_end, (ti + 1) * FB);
            const LoraTile tile = lora_tile<kTcNT>(a, pre, ti, 0);
            const int rank = rank_of(a, tile.ad);
            if (us == u_beg) pdl_wait();
            // every group is done with the units of the tile before, hence the MMAs with its v
            asm volatile("barrier.cta.sync 1, %0;" ::"n"(kTcGroups * 128) : "memory");
            stage_v_rows<T>(a, tile, rank, e, s_vp, s_off, s_back);
            fence_proxy_async();
            asm volatile("barrier.cta.sync 1, %0;" ::"n"(kTcGroups * 128) : "memory");
            if (lane == 0) mbar_arrive(v_full);

            // this group's units of the tile, 16 rows at a time, the next 16 rows' loads ahead of the sums of the last
            const int chunks = (tile.cnt + 15) / 16, u0 = us + ((group - (us - u_beg)) & (kTcGroups - 1));
            const int total = u0 < ue ? ((ue - 1 - u0) / kTcGroups + 1) * chunks : 0;
            // rows without a gap from the first on: the common case needs no test per row
            const uint32_t l0 = __ballot_sync(0xffffffffu, s_off[lane] >= 0), l1 = __ballot_sync(0xffffffffu, s_off[32 + lane] >= 0);
            const int s_live = ~l0 ? __ffs(~l0) - 1 : 32 + (~l1 ? __ffs(~l1) - 1 : 32);
            struct At { int u, c0; };
            At next{u0, 0};
            auto load = [&](float (&v)[16]) {
                const int f = (next.u - ti * FB) * 128 + q * 32 + lane;
                const Y* yf = reinterpret_cast<const Y*>(a.y) + f;
                const bool have = f < a.N && rank > 0;
                if (__all_sync(0xffffffffu, have) && next.c0 + 16 <= s_live) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = to_f(__ldcs(yf + s_off[next.c0 + j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int64_t o = s_off[next.c0 + j];
                        v[j] = have && o >= 0 ? to_f(__ldcs(yf + o)) : 0.f;
                    }
                }
                next.c0 += 16;
                if (next.c0 >= tile.cnt) { next.c0 = 0; next.u += kTcGroups; }
            };
            At now{u0, 0};
            auto finish = [&](const float (&v)[16]) {
                const int n = now.u - u_beg;
                if (now.c0 == 0) {
                    if (tc5::warp_set(abort_flag) || !tc5::warp_wait(&acc_full[group], (n / kTcGroups) & 1u, kTcWaitLimit)) {
                        if (!*abort_flag) lora_timeout(abort_flag);
                    }
                    tc5::fence_after();
                }
                uint32_t d[16];
                tc5::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(group * kTcNT + now.c0), d);
                tc5::tmem_ld_wait();
                const int f = (now.u - ti * FB) * 128 + q * 32 + lane;
                Y* yf = reinterpret_cast<Y*>(a.y) + f;
                const bool have = f < a.N && rank > 0 && !*abort_flag;
                float s[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    s[j] = v[j] + (Split<T>::scaled ? s_back[now.c0 + j] * __uint_as_float(d[j]) : __uint_as_float(d[j]));
                if (__all_sync(0xffffffffu, have) && now.c0 + 16 <= s_live) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) __stcs(yf + s_off[now.c0 + j], from_f<Y>(s[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int64_t o = s_off[now.c0 + j];
                        if (have && o >= 0) __stcs(yf + o, from_f<Y>(s[j]));
                    }
                }
                now.c0 += 16;
                if (now.c0 >= tile.cnt) {
                    now.c0 = 0;
                    now.u += kTcGroups;
                    tc5::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[group]);
                }
            };
            float v0[16], v1[16];
            if (total) load(v0);
            for (int k = 0; k < total; k += 2) {
                if (k + 1 < total) load(v1);
                finish(v0);
                if (k + 1 >= total) break;
                if (k + 2 < total) load(v0);
                finish(v1);
            }
            us = ue;
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    if (warp == 3) { tc5::fence_after(); tc5::tmem_dealloc(tmem, kTcGroups * kTcNT); }
}

// One launch for few tiles of eight rows and ranks up to 32.  (Measured, one launch against two: rank 16, 1024 to 1024, one
// row 4.2 us and 4.9, 64 rows of 2 adapters 5.1 and 6.1, 256 rows of 8 9.3 and 6.3; rank 64, 6144 to 6144, one row 13.2 and
// 9.1.  On the host it is one launch and no scratch.)
inline bool lora_one_launch(int P, int R, int nA) { return R <= 32 && (nA < P ? nA : P) + P / 8 <= 24; }

// How the first launch is cut: a rule on P and the number of adapters alone, because the scratch is sized by it.
// Eight-row tiles (the least mma.sync multiplies) while an adapter has few rows, 64-row tiles above; the sum over K is
// spread until two blocks per SM have work.
inline bool lora_wide(int P, int nA) { return P > 8 * (int64_t)nA; }
inline int lora_split(int P, int nA) {
    // (each adapter's last tile is on average half filled; counted as full, 8192 rows of 32 adapters, 6144 to 256 at rank
    // 64, took 54 us in one part per tile, 41 in two)
    const int64_t tiles = lora_wide(P, nA) ? nA / 2 + (P + kWdRows - 1) / kWdRows : (nA < P ? nA : P) + P / 8;
    const int64_t s = 296 / tiles;
    return s < 1 ? 1 : s > kMaxSplit ? kMaxSplit : (int)s;
}
// ... and no more than leave a warp (a block of the pipelined form) four 64-column steps.
inline int lora_split_used(int P, int nA, int K) {
    const int most = lora_wide(P, nA) ? K / 256 : K / 1024, s = lora_split(P, nA);
    return most < 1 ? 1 : s < most ? s : most;
}

template <typename T, int MT>
int run_shrink_wide(const LoraArgs& a, cudaStream_t s) {
    constexpr size_t smem = (size_t)kWdStages * wd_stage_bytes<MT>();
    if (smem > 40 * 1024 && cudaFuncSetAttribute(lora_shrink_wide_kernel<T, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return GSB_ERR_CUDA;
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / kWdRows;
    lora_shrink_wide_kernel<T, MT><<<dim3(tiles, a.S, (a.R + 16 * MT - 1) / (16 * MT)), 256, smem, s>>>(a);
    return launch_status();
}

template <typename T, int MT>
int run_shrink(const LoraArgs& a, cudaStream_t s) {
    constexpr size_t smem = (size_t)kShWarps * 16 * MT * 8 * 4;
    if (smem > 40 * 1024 && cudaFuncSetAttribute(lora_shrink_kernel<T, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return GSB_ERR_CUDA;
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / 8;
    lora_shrink_kernel<T, MT><<<dim3(tiles, a.S, (a.R + 16 * MT - 1) / (16 * MT)), kShWarps * 32, smem, s>>>(a);
    return launch_status();
}

// whether B (1) and y (2) can be read in pieces of eight and sixteen bytes
template <typename Y>
int expand_flags(const LoraArgs& a) {
    return (a.R % 4 == 0 && !misaligned(a.B, 8) ? 1 : 0) + (a.N % (16 / (int)sizeof(Y)) == 0 && !misaligned(a.y, 16) ? 2 : 0);
}

template <typename T, typename Y, int KG>
int run_cluster(const LoraArgs& a, cudaStream_t s) {
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / 8, feats = ((a.N + 31) / 32 + kClusterBlocks - 1) / kClusterBlocks * 32;
    return launch_after(lora_cluster_kernel<T, Y, KG>, dim3((unsigned)tiles * kClusterBlocks), 256, 0, kClusterBlocks, s, a, feats, expand_flags<Y>(a));
}

template <typename T, typename Y, int MT, int KG>
int run_expand(const LoraArgs& a, cudaStream_t s) {
    const size_t smem = (size_t)MT * ((a.R + 15) / 16) * Split<T>::N * 32 * sizeof(uint4);
    auto kernel = lora_expand_kernel<T, Y, MT, KG>;
    if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return GSB_ERR_CUDA;
    const int tiles = (a.nA < a.P ? a.nA : a.P) + a.P / (16 * MT);
    // features in ranges of whole passes of the block (256), until about four blocks per SM have work
    const int passes = (a.N + 255) / 256;
    int per = (int)(((int64_t)passes * tiles + 591) / 592);
    per = per < 1 ? 1 : per > passes ? passes : per;
    return launch_after(kernel, dim3(tiles, (passes + per - 1) / per), 256, smem, 1, s, a, per * 256, expand_flags<Y>(a));
}

template <typename T, typename Y>
int run_expand_tc(const LoraArgs& a, cudaStream_t s) {
    auto kernel = lora_expand_tc_kernel<T, Y>;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return GSB_ERR_CUDA;
    const int sms = sm_count_of(dev);
    const bool tma = a.R % 8 == 0;
    if (!sms || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tc_smem<T>(false)) != cudaSuccess) return GSB_ERR_CUDA;
    const int64_t units = ((int64_t)(a.nA < a.P ? a.nA : a.P) + a.P / kTcNT) * ((a.N + 127) / 128);
    if (units >= (int64_t)1 << 31) return GSB_ERR_TOO_LARGE;
    CUtensorMap tb{};
    if (tma && !encode(&tb, a.B, std::is_same<T, __nv_bfloat16>::value, a.R, a.N, a.nA, 128)) return GSB_ERR_CUDA;
    return launch_after(kernel, dim3((unsigned)(units < sms ? units : sms)), kTcThreads, tc_smem<T>(tma), 1, s, a, tb, (int)tma);
}

template <typename T, typename Y>
int run_lora(const LoraArgs& a, cudaStream_t s) {
    if (lora_one_launch(a.P, a.R, a.nA))
        return a.R <= 16 ? run_cluster<T, Y, 1>(a, s) : run_cluster<T, Y, 2>(a, s);
    const bool wide = lora_wide(a.P, a.nA);
    int st;
    if (wide) st = a.R <= 16 ? run_shrink_wide<T, 1>(a, s) : a.R <= 32 ? run_shrink_wide<T, 2>(a, s) : run_shrink_wide<T, 4>(a, s);
    else st = a.R <= 16 ? run_shrink<T, 1>(a, s) : a.R <= 32 ? run_shrink<T, 2>(a, s) : run_shrink<T, 4>(a, s);
    if (st) return st;
    // Times of a whole call on the device, 8 adapters, bf16.  16-row tiles with B loaded ahead while there are few rows (rank
    // 64, 256 rows of 1024 to 1024: 11 us against 13 for 32-row tiles and 16 for tcgen05); 32-row tiles halve the reads of B
    // above (rank 16, 8192 rows of 6144 to 6144: 111 us against 135).  tcgen05 where fp32 outputs and the rank are large,
    // against 32-row tiles, 8192 rows of 256 to 6144: rank 64 103 us and 169, rank 32 100 and 144, rank 16 98 and 102; 2048
    // rows of 256 to 4096: 31 and 41, 30 and 32, 29 and 24; rank 49, whose B it lays out itself, 159 and 191, 39 and 44.
    // With a 16-bit y its lanes move 2 bytes at a time: rank 64 110 and 109, rank 32 105 and 84, rank 49 160 and 139 (fp16
    // 110 and 120, 104 and 90, 162 and 145).  And tcgen05 for outputs whose rows are not 16-byte pieces, which the others
    // take value by value (8192 rows of 256 to 3941: rank 16 74 us against 235, rank 49 108 and 197).
    const int64_t outputs = (int64_t)a.P * a.N;
    const bool pieces = expand_flags<Y>(a) & 2, rows8 = a.R % 8 == 0;
    const int64_t enough = !pieces ? 5 << 19 : sizeof(Y) == 2 ? INT64_MAX : a.R > 32 ? (rows8 ? 6 << 20 : 20 << 20) : a.R > 16 && rows8 ? 12 << 20 : INT64_MAX;
    if (a.R <= 64 && !misaligned(a.B, 16) && outputs >= enough) return run_expand_tc<T, Y>(a, s);
    if (a.R > 64) return run_expand<T, Y, 1, 0>(a, s);
    if (wide && a.P >= 1024) return a.R <= 16 ? run_expand<T, Y, 2, 1>(a, s) : run_expand<T, Y, 2, 0>(a, s);
    return a.R <= 16 ? run_expand<T, Y, 1, 1>(a, s) : a.R <= 32 ? run_expand<T, Y, 1, 2>(a, s) : run_expand<T, Y, 1, 4>(a, s);
}

}  // namespace

int take_lora_status() {
    int st = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&st, g_lora_status, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    if (st && cudaMemcpyToSymbol(g_lora_status, &zero, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    return st;
}

}  // namespace gsb

using namespace gsb;

extern "C" size_t gsb_lora_scratch_bytes(int P, int max_rank, int n_adapters) {
    if (P <= 0 || max_rank <= 0 || n_adapters <= 0) return 0;
    return lora_one_launch(P, max_rank, n_adapters) ? 0 : (size_t)lora_split(P, n_adapters) * P * max_rank * 4;
}

extern "C" int gsb_lora_add(const void* x, const void* A, const void* B, int type, const int* adapter_offsets,
                            const int* rows, const int* ranks, const float* scales, int n, int P, int in, int out,
                            int n_adapters, int max_rank, void* y, int y_type, void* scratch, size_t scratch_bytes,
                            void* stream) {
    if ((type != GSB_TYPE_BF16 && type != GSB_TYPE_F16) || (y_type != type && y_type != GSB_TYPE_F32)) return GSB_ERR_INVALID_ARG;
    if (n < 0 || P < 0 || P > n || in <= 0 || out <= 0 || n_adapters <= 0 || max_rank <= 0) return GSB_ERR_INVALID_ARG;
    if (P == 0) return GSB_OK;
    if (!x || !A || !B || !adapter_offsets || !rows || !y || y == x) return GSB_ERR_INVALID_ARG;
    if (misaligned(x, 16) || misaligned(A, 16) || misaligned(B, 2) || misaligned(y, y_type == GSB_TYPE_F32 ? 4 : 2) ||
        misaligned(adapter_offsets, 4) || misaligned(rows, 4) || misaligned(ranks, 4) || misaligned(scales, 4))
        return GSB_ERR_INVALID_ARG;
    if (in % 8 || max_rank > kMaxRank || n_adapters > 1024 || in > kMaxDim || out > kMaxDim || P > kMaxDim) return GSB_ERR_UNSUPPORTED;
    const size_t need = gsb_lora_scratch_bytes(P, max_rank, n_adapters);
    if (need && (!scratch || misaligned(scratch, 256))) return GSB_ERR_INVALID_ARG;
    if (scratch_bytes < need) return GSB_ERR_WORKSPACE;
    const __int128 y_bytes = (__int128)n * out * (y_type == GSB_TYPE_F32 ? 4 : 2), per = (__int128)n_adapters * max_rank * 2;
    if (overlap(y, y_bytes, x, (__int128)n * in * 2) || overlap(y, y_bytes, A, per * in) || overlap(y, y_bytes, B, per * out) ||
        overlap(y, y_bytes, adapter_offsets, (n_adapters + 1) * 4) || overlap(y, y_bytes, rows, (__int128)P * 4) ||
        overlap(y, y_bytes, ranks, n_adapters * 4) || overlap(y, y_bytes, scales, n_adapters * 4))
        return GSB_ERR_INVALID_ARG;
    LoraArgs a{};
    a.x = x; a.A = A; a.B = B; a.offsets = adapter_offsets; a.rows = rows; a.ranks = ranks; a.scales = scales;
    a.n = n; a.P = P; a.K = in; a.N = out; a.nA = n_adapters; a.R = max_rank;
    a.S = lora_split_used(P, n_adapters, in); a.part = reinterpret_cast<float*>(scratch); a.y = y;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (type == GSB_TYPE_BF16)
        return y_type == GSB_TYPE_F32 ? run_lora<__nv_bfloat16, float>(a, s) : run_lora<__nv_bfloat16, __nv_bfloat16>(a, s);
    return y_type == GSB_TYPE_F32 ? run_lora<__half, float>(a, s) : run_lora<__half, __half>(a, s);
}
