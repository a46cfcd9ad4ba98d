// Expert products with 16-bit (bf16 / fp16) weights: the ragged grouped product
//   y[p, :] = W[e] x[rows[p], :]                        for offsets[e] <= p < offsets[e + 1]
// and the expert FFN built from it
//   h[p, :] = silu(gate[e] x) * (up[e] x),  y[p, :] = down[e] h[p, :],  out[t, :] = sum_k w[t, k] y[slot(t, k), :].
// Products are summed in fp32; h is rounded once to the weights' type (the tensor cores read it in that type,
// fp16 saturating at +-65504), the per-slot rows y stay fp32 and the sum over slots is taken in slot order.
#include "expert16.cuh"

namespace gsb {

namespace {

// ---- the tensor-core kernel -------------------------------------------------------------------
// One item = 128 weight rows x up to NT token rows of one expert, as D[weight row, token] = sum_k W[row, k] X[token, k]
// (M = 128 weight rows in the 128 TMEM lanes, N = tokens rounded up to 16): a decode batch pads tokens to 16, not to 128.
// The 128 rows are two boxes of 64: consecutive rows of one matrix, or 64 gate rows and their 64 up rows, so that SwiGLU
// pairs meet in the epilogue.  X rows are gathered by TMA (four rows an instruction), so no sorted copy is made.
// A cluster of S CTAs works on one item, each on 1/S of K: the partial tiles are exchanged through distributed shared
// memory, CTA r finishing the r-th part of the columns, and added in rank order - no atomics, the same bits every time.
constexpr int kGrThreads = 256;            // warps: 0 weights, 1 MMA, 2 TMEM, 3 token rows, 4-7 epilogue
constexpr int kCh = 16;                    // accumulator columns a pass of the epilogue exchanges
constexpr int kABytes = 128 * 128;         // 128 weight rows x 64 columns

template <int NT> struct GrCfg {
    static constexpr int kps = NT <= 16 ? 2 : 1;                   // k-blocks of 64 columns per stage
    static constexpr int stages = NT <= 16 ? 5 : NT <= 64 ? 8 : 4;
    static constexpr int bbytes = NT * 128;
    static constexpr int stage_bytes = kps * (kABytes + bbytes);
    static constexpr int red_bytes = 2 * kCh * 128 * 4;
    static constexpr int tmem_cols = 2 * NT < 32 ? 32 : 2 * NT;
    static constexpr size_t smem = (size_t)stages * stage_bytes + red_bytes + (kMaxE + 4) * 4 + 256;
    static_assert(smem <= 227 * 1024, "stages exceed the shared memory of an SM");
};

__device__ int g_op16_status;

// item i: experts in order; inside one, all token tiles of a feature block run next to each other (they read the
// same weights, which the second one finds in L2).  `e` only moves forward.
template <int NT, int FW>
__device__ __forceinline__ GrItem gr_item(const GroupedArgs& a, const int* pre, int i, int fb_count, int& e) {
    while (i >= pre[e + 1] * fb_count) ++e;
    const int nt = pre[e + 1] - pre[e], local = i - pre[e] * fb_count;
    const int fb = local / nt, tt = local - fb * nt;
    GrItem it;
    it.e = e;
    it.f0 = fb * FW;
    const int lo = seg_bound(a.offsets, e, a.P), hi = seg_bound(a.offsets, e + 1, a.P);
    it.p0 = lo + tt * NT;
    it.cnt = min(NT, hi - it.p0);
    return it;
}

__device__ __forceinline__ void gr_timeout(volatile int* abort_flag) {
    *abort_flag = 1;
    atomicCAS(&g_op16_status, 0, GSB_ERR_TIMEOUT);
}

template <int NT, typename T, typename Y, bool GU>
__global__ void __launch_bounds__(kGrThreads, 1)
grouped_kernel(const GroupedArgs a, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w2,
               const __grid_constant__ CUtensorMap tm_x) {
    using Cfg = GrCfg<NT>;
    constexpr int FW = GU ? 64 : 128;      // output features of an item
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* s_stage = smem;
    float* s_red = reinterpret_cast<float*>(smem + Cfg::stages * Cfg::stage_bytes);
    int* pre = reinterpret_cast<int*>(s_red + 2 * kCh * 128);               // [E + 1] token tiles before expert e
    uint64_t* full = reinterpret_cast<uint64_t*>(pre + kMaxE + 4);
    uint64_t* empty = full + Cfg::stages;
    uint64_t* acc_full = empty + Cfg::stages;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* red_full = acc_empty + 2;
    uint64_t* red_free = red_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(red_free + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = (int)tc5::cluster_size(), rank = (int)tc5::cluster_rank();
    if (tid == 0) {
        for (int i = 0; i < Cfg::stages; ++i) { mbar_init(&full[i], 2); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4);
            mbar_init(&red_full[i], 4 * S); mbar_init(&red_free[i], 4 * S);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 2) { tc5::tmem_alloc(tmem_slot, Cfg::tmem_cols); tc5::tmem_relinquish(); }
    int descending = (smem_u32(smem) & 1023u) != 0;    // (the swizzled tiles need a 1 KiB boundary: as good as no list)
    descending |= seg_scan<NT>(a.offsets, a.E, a.P, pre, reinterpret_cast<int*>(s_red));
    tc5::fence_before();
    descending = __syncthreads_or(descending);
    tc5::fence_after();
    if (S > 1) tc5::cluster_sync_all();    // the peers' barriers exist before anyone arrives on them
    const uint32_t tmem = *tmem_slot;
    const int nkb = (a.K + 63) >> 6, kb0 = nkb * rank / S, kb1 = nkb * (rank + 1) / S;
    const int FB = (a.N + FW - 1) / FW;
    // at most (E + P / NT) * FB, which the host has checked to fit; a list that is not ascending is no list
    const int items = descending ? 0 : pre[a.E] * FB;
    const int first = blockIdx.x / S, step = gridDim.x / S;

    if (warp == 0) {
        if (lane == 0) {                   // ---- weights
            uint32_t st = 0, ph = 0;
            int e = 0;
            bool dead = false;
            for (int i = first; i < items && !dead && !*abort_flag; i += step) {
                const GrItem it = gr_item<NT, FW>(a, pre, i, FB, e);
                for (int kb = kb0; kb < kb1; kb += Cfg::kps) {
                    if (!mbar_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                    const int nk = min(Cfg::kps, kb1 - kb);
                    mbar_arrive_expect_tx(&full[st], (uint32_t)nk * kABytes);
                    uint8_t* dst = s_stage + st * Cfg::stage_bytes;
                    for (int j = 0; j < nk; ++j) {
                        tc5::tma_load_3d(dst + j * kABytes, &tm_w, (kb + j) * 64, it.f0, it.e, &full[st]);
                        tc5::tma_load_3d(dst + j * kABytes + kABytes / 2, GU ? &tm_w2 : &tm_w, (kb + j) * 64,
                                         GU ? it.f0 : it.f0 + 64, it.e, &full[st]);
                    }
                    if (++st == Cfg::stages) { st = 0; ph ^= 1u; }
                }
            }
            // after a time-out elsewhere: nothing may still be copying into this block's memory when it ends
            if (*abort_flag)
                for (int j = 0; j < Cfg::stages; ++j) {
                    if (st == 0) { st = Cfg::stages; ph ^= 1u; }
                    --st;
                    mbar_wait(&full[st], ph, kGrWaitLimit / 16);
                }
        }
    } else if (warp == 3) {                // ---- token rows
        uint32_t st = 0, ph = 0;
        int e = 0;
        bool dead = false;
        constexpr int G = NT > 128 ? NT / 128 : 1;    // groups of four rows per lane
        for (int i = first; i < items && !dead && !*abort_flag; i += step) {
            const GrItem it = gr_item<NT, FW>(a, pre, i, FB, e);
            const int nr = (it.cnt + 15) & ~15;
            int r[G][4];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int q = (g * 32 + lane) * 4 + j;
                    // columns behind the tile's last row, and rows that do not exist, read row 0; neither is stored
                    int v = 0;
                    if (q < it.cnt) v = a.rows ? __ldg(a.rows + it.p0 + q) : it.p0 + q;
                    r[g][j] = v >= 0 && v < a.n ? v : 0;
                }
            for (int kb = kb0; kb < kb1; kb += Cfg::kps) {
                if (!mbar_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                const int nk = min(Cfg::kps, kb1 - kb);
                if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(nk * nr * 128));
                __syncwarp();
                uint8_t* dst = s_stage + st * Cfg::stage_bytes + Cfg::kps * kABytes;
                for (int j = 0; j < nk; ++j)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const int q = (g * 32 + lane) * 4;
                        if (q < nr) tc5::tma_gather4(dst + j * Cfg::bbytes + q * 128, &tm_x, (kb + j) * 64, r[g][0], r[g][1], r[g][2], r[g][3], &full[st]);
                    }
                if (++st == Cfg::stages) { st = 0; ph ^= 1u; }
            }
            dead = __any_sync(0xffffffffu, dead);
        }
    } else if (warp == 1) {
        if (lane == 0) {                   // ---- MMA issue
            uint32_t st = 0, ph = 0, tl = 0;
            int e = 0;
            bool dead = false;
            constexpr uint32_t ab = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            const uint64_t d0 = tc5::desc_sw128(smem_u32(s_stage));
            for (int i = first; i < items && !dead && !*abort_flag; i += step, ++tl) {
                const GrItem it = gr_item<NT, FW>(a, pre, i, FB, e);
                const uint32_t buf = tl & 1u;
                if (!mbar_wait(&acc_empty[buf], ((tl >> 1) & 1u) ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); break; }
                tc5::fence_after();
                const uint32_t idesc = tc5::idesc_f16(ab, 128, (uint32_t)((it.cnt + 15) & ~15));
                uint32_t acc = 0;
                for (int kb = kb0; kb < kb1; kb += Cfg::kps) {
                    if (!mbar_wait(&full[st], ph, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                    tc5::fence_after();
                    const int nk = min(Cfg::kps, kb1 - kb);
                    const uint64_t ad = d0 + (uint64_t)(st * (uint32_t)(Cfg::stage_bytes >> 4));
                    const uint64_t bd = ad + (uint64_t)(Cfg::kps * kABytes >> 4);
                    for (int j = 0; j < nk; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            tc5::mma_f16_ss(tmem + buf * NT, ad + (uint64_t)(j * (kABytes >> 4) + k * 2),
                                            bd + (uint64_t)(j * (Cfg::bbytes >> 4) + k * 2), idesc, acc);
                            acc = 1u;
                        }
                    tc5::commit(&empty[st]);
                    if (++st == Cfg::stages) { st = 0; ph ^= 1u; }
                }
                if (!dead) tc5::commit(&acc_full[buf]);
            }
        }
    } else if (warp >= 4) {                // ---- epilogue: this thread's TMEM lane = weight row
        const int q = warp & 3, row = q * 32 + lane;
        const int lsh = S == 4 ? 2 : S == 2 ? 1 : 0, per = kCh >> lsh;     // columns of a pass that one CTA finishes
        const uint32_t red0 = smem_u32(s_red);
        uint32_t tl = 0, cc = 0;
        int e = 0;
        bool dead = false;
        Y* y = reinterpret_cast<Y*>(a.y);
        for (int i = first; i < items && !dead; i += step, ++tl) {
            const GrItem it = gr_item<NT, FW>(a, pre, i, FB, e);
            const uint32_t buf = tl & 1u;
            if (*abort_flag || !mbar_wait(&acc_full[buf], (tl >> 1) & 1u, kGrWaitLimit)) {
                if (!*abort_flag) gr_timeout(abort_flag);
                break;
            }
            tc5::fence_after();
            for (int c0 = 0; c0 < it.cnt; c0 += kCh, ++cc) {
                const uint32_t rb = cc & 1u, rph = (cc >> 1) & 1u;
                uint32_t v[kCh];
                tc5::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + buf * NT + (uint32_t)c0, v);
                tc5::tmem_ld_wait();
                if (!tc5::wait_cluster(&red_free[rb], rph ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
#pragma unroll
                for (int j = 0; j < kCh; ++j) {
                    const int owner = j >> (4 - lsh), jl = j & (per - 1);
                    tc5::st_cluster(tc5::map_rank(red0 + (uint32_t)(((rb * kCh + rank * per + jl) * 128 + row) * 4), (uint32_t)owner),
                                    __uint_as_float(v[j]));
                }
                __syncwarp();
                if (lane < S) tc5::arrive_cluster(tc5::map_rank(smem_u32(&red_full[rb]), (uint32_t)lane));
                if (!tc5::wait_cluster(&red_full[rb], rph, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                const float* red = s_red + rb * kCh * 128;
                const int f = it.f0 + (GU ? (row & 63) : row);
                for (int jl = GU ? row >> 6 : 0; jl < per; jl += GU ? 2 : 1) {
                    const int c = c0 + rank * per + jl;
                    if (c >= it.cnt || f >= a.N) continue;
                    const int p = it.p0 + c;
                    if (a.rows) { const int r = __ldg(a.rows + p); if (r < 0 || r >= a.n) continue; }
                    float s0 = 0.f, s1 = 0.f;
                    for (int src = 0; src < S; ++src) {
                        s0 += red[(src * per + jl) * 128 + (GU ? (row & 63) : row)];
                        if (GU) s1 += red[(src * per + jl) * 128 + (row & 63) + 64];
                    }
                    y[(int64_t)p * a.N + f] = GU ? h_from_f<Y>(__fmul_rn(silu_ref(s0), s1)) : from_f<Y>(s0);
                }
                __syncwarp();
                if (lane < S) tc5::arrive_cluster(tc5::map_rank(smem_u32(&red_free[rb]), (uint32_t)lane));
            }
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    if (S > 1) tc5::cluster_sync_all();    // peers may still read or signal this block's memory
    if (warp == 2) { tc5::fence_after(); tc5::tmem_dealloc(tmem, Cfg::tmem_cols); }
}

template <int NT, typename T, typename Y, bool GU>
int run_grouped_nt(const GroupedArgs& a, int S, cudaStream_t s) {
    using Cfg = GrCfg<NT>;
    constexpr int FW = GU ? 64 : 128;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return GSB_ERR_CUDA;
    const int sms = sm_count_of(dev);
    if (!sms) return GSB_ERR_CUDA;
    auto kernel = grouped_kernel<NT, T, Y, GU>;
    static std::atomic<uint64_t> ready{0};     // devices on which the shared-memory size was raised
    if (dev >= 64 || !((ready.load() >> dev) & 1u)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::smem) != cudaSuccess) return GSB_ERR_CUDA;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    const int64_t fbs = (a.N + FW - 1) / FW, tiles = (a.E < a.P ? a.E : a.P) + a.P / NT;
    const int64_t items = tiles * fbs;
    if (items + sms >= (int64_t)1 << 31) return GSB_ERR_TOO_LARGE;
    CUtensorMap tw, tw2, tx;
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    if (!encode(&tw, a.w, bf, a.K, a.N, a.E, 64) || (GU && !encode(&tw2, a.w2, bf, a.K, a.N, a.E, 64)) ||
        !encode(&tx, a.x, bf, a.K, a.n, 0, 1))
        return GSB_ERR_CUDA;
    const int64_t groups = items < sms / S ? items : sms / S;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(groups * S)); cfg.blockDim = dim3(kGrThreads); cfg.dynamicSmemBytes = Cfg::smem; cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)S; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, tw, GU ? tw2 : tw, tx) == cudaSuccess ? GSB_OK : GSB_ERR_LAUNCH;
}

template <typename T, typename Y, bool GU>
int run_grouped(const GroupedArgs& a, cudaStream_t s) {
    const int64_t per_expert = a.P / a.E, nkb = (a.K + 63) / 64;
    const int nt = per_expert <= 16 ? 16 : per_expert <= 64 ? 64 : 256;
    const int64_t fbs = (a.N + (GU ? 63 : 127)) / (GU ? 64 : 128), items = ((a.E < a.P ? a.E : a.P) + a.P / nt) * fbs;
    int S = items >= 1184 ? 1 : items >= 592 ? 2 : 4;
    while (S > nkb) S >>= 1;
    if (nt == 16) return run_grouped_nt<16, T, Y, GU>(a, S, s);
    if (nt == 64) return run_grouped_nt<64, T, Y, GU>(a, S, s);
    return run_grouped_nt<256, T, Y, GU>(a, S, s);
}

template <typename T>
int run_grouped_any(const GroupedArgs& a, int y_type, cudaStream_t s) {
    if (a.w2) return run_grouped<T, T, true>(a, s);
    return y_type == GSB_TYPE_F32 ? run_grouped<T, float, false>(a, s) : run_grouped<T, T, false>(a, s);
}

bool use_pair(int P, int E) { return P / E > 64; }

int launch_grouped(const GroupedArgs& a, int type, int y_type, void* scratch, cudaStream_t s) {
    if (use_pair(a.P, a.E)) return launch_grouped_pair(a, type, y_type, scratch, s);
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
struct Ffn16Ws { int *offsets, *tok, *row, *slot_pos, *disp; uint8_t *h, *xs; float* y; size_t total; };
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
    // the rows in expert order are done with when the per-slot rows are written
    ws.y = reinterpret_cast<float*>(take(P * H * 4));
    ws.xs = reinterpret_cast<uint8_t*>(ws.y);
    ws.total = at;
    return ws;
}

inline bool is16(int type) { return type == GSB_TYPE_BF16 || type == GSB_TYPE_F16; }
inline size_t type_bytes(int type) { return type == GSB_TYPE_F32 ? 4 : 2; }
constexpr int64_t kMaxSlots = (int64_t)1 << 30;

}  // namespace

}  // namespace gsb

using namespace gsb;

extern "C" size_t gsb_grouped_gemm_workspace_bytes(int P, int in, int E) {
    return P > 0 && in > 0 && E > 0 && use_pair(P, E) ? grouped_pair_scratch_bytes(P, in) : 0;
}

extern "C" int gsb_grouped_gemm(const void* x, const void* w, int type, const int* expert_offsets, const int* rows,
                                int n, int P, int in, int out, int E, void* y, int y_type, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (!is16(type) || (y_type != type && y_type != GSB_TYPE_F32)) return GSB_ERR_INVALID_ARG;
    if (n < 0 || P < 0 || in <= 0 || out <= 0 || E <= 0 || (!rows && P > n)) return GSB_ERR_INVALID_ARG;
    if (P == 0 || n == 0) return GSB_OK;
    if (!x || !w || !expert_offsets || !y) return GSB_ERR_INVALID_ARG;
    if (misaligned(x, 16) || misaligned(w, 16) || misaligned(expert_offsets, 4) || misaligned(rows, 4) ||
        misaligned(y, type_bytes(y_type)))
        return GSB_ERR_INVALID_ARG;
    if (in % 8 || E > 1024 || P > kMaxSlots) return GSB_ERR_UNSUPPORTED;
    const size_t need = rows ? gsb_grouped_gemm_workspace_bytes(P, in, E) : 0;
    if (need && (!workspace || misaligned(workspace, 256))) return GSB_ERR_INVALID_ARG;
    if (need > workspace_bytes) return GSB_ERR_WORKSPACE;
    GroupedArgs a{};
    a.x = x; a.w = w; a.offsets = expert_offsets; a.rows = rows;
    a.n = n; a.P = P; a.K = in; a.N = out; a.E = E; a.y = y;
    return launch_grouped(a, type, y_type, workspace, reinterpret_cast<cudaStream_t>(stream));
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
    st = launch_grouped(g, type, type, ws.xs, s);
    if (st) return st;
    GroupedArgs d{};
    d.x = ws.h; d.w = down_w; d.offsets = ws.offsets;
    d.n = d.P = n * topk; d.K = moe_inter; d.N = hidden; d.E = E; d.y = ws.y;
    st = launch_grouped(d, type, GSB_TYPE_F32, nullptr, s);
    if (st) return st;
    if (out_type == GSB_TYPE_F32) return run_combine16<float>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
    if (type == GSB_TYPE_BF16) return run_combine16<__nv_bfloat16>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
    return run_combine16<__half>(ws.y, topk_ids, ws.slot_pos, topk_weights, n, topk, hidden, E, out, s);
}

extern "C" int gsb_operators16_status(void) {
    int st = 0;
    const int zero = 0;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&st, g_op16_status, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    if (st && cudaMemcpyToSymbol(g_op16_status, &zero, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    const int pair = take_pair_status();
    return st ? st : pair;
}
