// The grouped product for many rows per expert: two CTAs of a cluster share one tile (tcgen05 cta_group::2).
//
// D[weight row, token] = sum_k W[row, k] X[token, k]: 256 weight rows (128 in each CTA's TMEM lanes) x up to 256 token
// rows of one expert.  Each CTA stages its own 128 weight rows and half of the tokens; the tensor cores of both read
// both halves, so a byte of shared memory feeds twice the products of a one-CTA tile - with a 128 x 256 tile per CTA the
// operand reads plus the writes of the copies need 1.5 times the shared-memory bandwidth of an SM.
// Both operands come by TMA, so the token rows lie in expert order: rows named by a list are copied into that order
// first (16384 rows of 2048: 16 us, the rate of a copy).  Gathering inside this kernel was slower: 16384 rows of 8 experts,
// 2048 to 4096, take 190 us in order, 211 with the copy, 307 with TMA's gather (~26 cycles per four rows, where a k-block
// of 64 columns multiplies for 512) and 309 with half the rows by TMA's gather and half by cp.async.
// SwiGLU: a CTA's 128 weight rows are 64 gate rows and their 64 up rows; the epilogue warps swap halves through shared
// memory.  Two accumulators (2 x 256 TMEM columns), so the epilogue of a tile runs under the next one's main loop.  A
// TMEM lane holds one feature of 32 tokens where memory wants a token's features side by side: 16-bit results are turned
// round in shared memory and stored 16 bytes a lane (2-byte stores took as long as the main loop of K = 2048).
#include "expert16.cuh"

namespace gsb {

namespace {

constexpr int kPrNT = 256;                 // token rows per tile at most
constexpr int kPrStages = 6;
constexpr int kPrHalf = 128 * 128;         // 128 rows x 64 columns: weights, or this CTA's tokens
constexpr int kPrStageBytes = 2 * kPrHalf;
constexpr int kPrXch = 2 * 2 * 2 * 8 * 64 * 4;   // per epilogue group: two buffers of 2 x 8 columns x 64 rows fp32
constexpr int kPrTurn = 8 * 16 * 32 * 2;   // per epilogue warp: 16 tokens x 32 features, 16-bit
constexpr int kPrThreads = 384;            // warps: 0 weights, 1 MMA, 2 TMEM, 3 tokens, 4-11 epilogue (two groups)
constexpr size_t kPrSmem = (size_t)kPrStages * kPrStageBytes + kPrXch + kPrTurn + (kMaxE + 4) * 4 + 256;
static_assert(kPrSmem <= 227 * 1024, "stages exceed the shared memory of an SM");

__device__ int g_pair_status;

__device__ __forceinline__ void pr_timeout(volatile int* abort_flag) {
    *abort_flag = 1;
    atomicCAS(&g_pair_status, 0, GSB_ERR_TIMEOUT);
}

// Item i: experts in order, inside one the token tiles of a feature block next to each other (same weights).  An
// expert's rows are cut into equal tiles (multiples of 32 rows) instead of full ones and a rest.
__device__ __forceinline__ GrItem pr_item(const GroupedArgs& a, const int* pre, int i, int fb_count, int fw, int& e) {
    while (i >= pre[e + 1] * fb_count) ++e;
    const int nt = pre[e + 1] - pre[e], local = i - pre[e] * fb_count;
    const int fb = local / nt, tt = local - fb * nt;
    const int lo = seg_bound(a.offsets, e, a.P), hi = seg_bound(a.offsets, e + 1, a.P);
    const int rows = ((hi - lo + nt - 1) / nt + 31) & ~31;
    GrItem it;
    it.e = e;
    it.f0 = fb * fw;
    it.p0 = lo + tt * rows;
    it.cnt = min(rows, hi - it.p0);
    return it;
}

template <typename T, typename Y, bool GU>
__global__ void __launch_bounds__(kPrThreads, 1)
grouped_pair_kernel(const GroupedArgs a, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w2,
                    const __grid_constant__ CUtensorMap tm_x, int vec) {
    extern __shared__ __align__(1024) uint8_t smem[];
    float* s_xch = reinterpret_cast<float*>(smem + kPrStages * kPrStageBytes);
    uint8_t* s_turn = smem + kPrStages * kPrStageBytes + kPrXch;
    int* pre = reinterpret_cast<int*>(s_turn + kPrTurn);
    uint64_t* full = reinterpret_cast<uint64_t*>(pre + kMaxE + 4);     // the leader's are used, for both CTAs' data
    uint64_t* empty = full + kPrStages;
    uint64_t* acc_full = empty + kPrStages;
    uint64_t* acc_empty = acc_full + 2;                                // the leader's are used
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_tot = reinterpret_cast<int*>(tmem_slot + 2);                // [3] token tiles if cut into 32, 64, 128 rows

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)tc5::cluster_rank();
    if (tid == 0) {
        for (int i = 0; i < kPrStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * 8); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) { tc5::prefetch_map(&tm_w); tc5::prefetch_map(&tm_x); if (GU) tc5::prefetch_map(&tm_w2); }
    if (tid < 3) s_tot[tid] = 0;
    tc5::cluster_sync_all();
    if (warp == 2) { tc5::tmem_alloc2(tmem_slot, 512); tc5::tmem_relinquish2(); }
    tc5::fence_before();
    tc5::cluster_sync_all();               // the peer has its barriers and its TMEM
    tc5::fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();
    constexpr int fc = GU ? 64 : 128, fw = 2 * fc;     // output features of this CTA, and of an item (both CTAs)
    const int FB = (a.N + fw - 1) / fw;
    int n[4], descending = (smem_u32(smem) & 1023u) != 0;
    descending |= seg_count(a.offsets, a.E, a.P, n);
    // Tiles of 256 rows, or of fewer (down to 32) where all of them still run at once: a small problem is then spread over
    // more SMs and its epilogues are shorter (256 rows for each of 4 experts, 1024 x 1024: 12 us with 256 rows a tile, 8 with
    // 64, 11 with 32, which take two rounds).  Only the device knows how many rows the list names.
    if (tid < 256)
        for (int k = 0; k < 3; ++k) {
            int t = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) t += n[j] > 0 ? (n[j] + (32 << k) - 1) >> (5 + k) : 0;
            t = __reduce_add_sync(0xffffffffu, t);
            if (lane == 0 && t) atomicAdd(&s_tot[k], t);
        }
    descending = __syncthreads_or(descending);
    int lg = 8;
    while (lg > 5 && (int64_t)s_tot[lg - 6] * FB <= (int)gridDim.x >> 1) --lg;
    seg_scan(n, a.E, lg, pre, reinterpret_cast<int*>(s_xch));
    __syncthreads();
    const int nkb = (a.K + 63) >> 6;
    const int items = descending ? 0 : pre[a.E] * FB;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int fr = rank * fc;              // this CTA's features start here inside an item

    if (warp == 0) {                       // ---- weights of this CTA; bytes are counted on the leader's barrier
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0;
        int e = 0;
        bool dead = false;
        for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step) {
            const GrItem it = pr_item(a, pre, i, FB, fw, e);
            const int nb = ((it.cnt + 31) / 32 * 16 + 31) / 32;         // token boxes of 32 rows per CTA
            for (int kb = 0; kb < nkb; ++kb) {
                if (!tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { pr_timeout(abort_flag); dead = true; break; }
                if (leader) {
                    if (rank == 0) mbar_arrive_expect_tx(&full[st], 2u * (kPrHalf + (uint32_t)nb * 4096u));
                    const uint32_t bar = tc5::map_rank(smem_u32(&full[st]), 0);
                    uint8_t* dst = smem + st * kPrStageBytes;
                    tc5::tma2_load_3d(dst, &tm_w, kb * 64, it.f0 + fr, it.e, bar);
                    if (GU) tc5::tma2_load_3d(dst + kPrHalf / 2, &tm_w2, kb * 64, it.f0 + fr, it.e, bar);
                }
                if (++st == kPrStages) { st = 0; ph ^= 1u; }
            }
        }
        // the signals of the last MMAs have arrived before the block ends
        for (int j = 0; j < kPrStages && !tc5::warp_set(abort_flag); ++j) {
            tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit);
            if (++st == kPrStages) { st = 0; ph ^= 1u; }
        }
        // after a time-out: nothing may still be copying into this block's memory when it ends
        if (tc5::warp_set(abort_flag) && rank == 0)
            for (int j = 0; j < kPrStages; ++j) {
                if (st == 0) { st = kPrStages; ph ^= 1u; }
                --st;
                tc5::warp_wait(&full[st], ph, kGrWaitLimit / 16);
            }
    } else if (warp == 3) {                // ---- this CTA's half of the token rows
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0;
        int e = 0;
        bool dead = false;
        for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step) {
            const GrItem it = pr_item(a, pre, i, FB, fw, e);
            const int half = (it.cnt + 31) / 32 * 16, nb = (half + 31) / 32;
            for (int kb = 0; kb < nkb; ++kb) {
                if (!tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { pr_timeout(abort_flag); dead = true; break; }
                if (leader) {
                    const uint32_t bar = tc5::map_rank(smem_u32(&full[st]), 0);
                    for (int b = 0; b < nb; ++b)
                        tc5::tma2_load_2d(smem + st * kPrStageBytes + kPrHalf + b * 4096, &tm_x, kb * 64, it.p0 + rank * half + b * 32, bar);
                }
                if (++st == kPrStages) { st = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {                // ---- MMA issue for the pair
        if (rank == 0) {
            const bool leader = tc5::elect_one();
            uint32_t st = 0, ph = 0, tl = 0;
            int e = 0;
            bool dead = false;
            constexpr uint32_t ab = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            const uint64_t d0 = tc5::desc_sw128(smem_u32(smem));
            for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step, ++tl) {
                const GrItem it = pr_item(a, pre, i, FB, fw, e);
                const uint32_t buf = tl & 1u;
                if (!tc5::warp_wait_cluster(&acc_empty[buf], ((tl >> 1) & 1u) ^ 1u, kGrWaitLimit)) { pr_timeout(abort_flag); break; }
                tc5::fence_after();
                const uint32_t idesc = tc5::idesc_f16(ab, 256, (uint32_t)((it.cnt + 31) & ~31));
                uint32_t acc = 0;
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!tc5::warp_wait_cluster(&full[st], ph, kGrWaitLimit)) { pr_timeout(abort_flag); dead = true; break; }
                    tc5::fence_after();
                    if (leader) {
                        const uint64_t ad = d0 + (uint64_t)(st * (uint32_t)(kPrStageBytes >> 4));
                        const uint64_t bd = ad + (uint64_t)(kPrHalf >> 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc5::mma2_f16_ss(tmem + buf * kPrNT, ad + (uint64_t)(k * 2), bd + (uint64_t)(k * 2), idesc, k ? 1u : acc);
                        tc5::commit2(&empty[st]);
                    }
                    acc = 1u;
                    if (++st == kPrStages) { st = 0; ph ^= 1u; }
                }
                if (!dead && leader) tc5::commit2(&acc_full[buf]);
            }
            // after a time-out: no MMA is at work, and no signal on its way, when the blocks end (otherwise the others have
            // waited for all of them)
            if (tc5::warp_set(abort_flag)) {
                if (st == 0) { st = kPrStages; ph ^= 1u; }
                tc5::warp_wait(&empty[st - 1], ph, kGrWaitLimit);      // (at once where there was none)
                if (dead) --tl;                                        // (counted, but not announced)
                if (tl) tc5::warp_wait(&acc_full[(tl - 1) & 1u], ((tl - 1) >> 1) & 1u, kGrWaitLimit);
            }
        }
    } else if (warp >= 4) {                // ---- epilogue: this thread's TMEM lane = weight row of this CTA
        // two groups of four warps take 16 token columns in turn
        const int group = (warp - 4) >> 2, bar = 1 + group, q = warp & 3, row = q * 32 + lane;
        uint32_t tl = 0, xb = 0;
        int e = 0;
        Y* y = reinterpret_cast<Y*>(a.y);
        Y* turn = reinterpret_cast<Y*>(s_turn + (warp - 4) * 1024);
        for (int i = first; i < items; i += step, ++tl) {
            const GrItem it = pr_item(a, pre, i, FB, fw, e);
            const uint32_t buf = tl & 1u;
            int ok = tc5::warp_set(abort_flag) ? 0 : (int)tc5::warp_wait(&acc_full[buf], (tl >> 1) & 1u, a.sum_limit);
            if (!ok) pr_timeout(abort_flag);
            // the group's four warps must agree to go on: they meet at a barrier in the loop below
            if (GU) ok = epilogue_agree(ok, bar);
            if (!ok) break;
            tc5::fence_after();
            const int f = it.f0 + fr + (GU ? row & 63 : row);
            for (int c0 = group * 16; c0 < it.cnt; c0 += 32) {
                uint32_t v[16];
                tc5::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + buf * kPrNT + (uint32_t)c0, v);
                // which of the 16 tokens exist
                int r = lane < 16 && c0 + lane < it.cnt ? 0 : -1;
                if (a.rows && r == 0) r = a.rows[it.p0 + c0 + lane];
                const uint32_t live = __ballot_sync(0xffffffffu, r >= 0 && r < a.n);
                tc5::tmem_ld_wait();
                constexpr int NC = GU ? 8 : 16;        // columns this thread finishes, from column cb on
                const int cb = GU && q >= 2 ? 8 : 0;
                float d[NC];
                if (GU) {
                    // warps 0, 1 of the group hold gate rows, 2, 3 the up rows of the same features: each side keeps 8 of
                    // the 16 columns and passes the other 8 on
                    float* xs = s_xch + group * 2048 + xb * 1024 + (q >> 1) * 512 + (row & 63);
#pragma unroll
                    for (int j = 0; j < 8; ++j) xs[j * 64] = __uint_as_float(q < 2 ? v[8 + j] : v[j]);
                    epilogue_sync(bar);
                    const float* xo = s_xch + group * 2048 + xb * 1024 + ((q >> 1) ^ 1) * 512 + (row & 63);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float mine = __uint_as_float(q < 2 ? v[j] : v[8 + j]), other = xo[j * 64];
                        d[j] = swiglu(q < 2 ? mine : other, q < 2 ? other : mine);
                    }
                    xb ^= 1u;
                } else {
#pragma unroll
                    for (int j = 0; j < NC; ++j) d[j] = __uint_as_float(v[j]);
                }
                Y* o = y + (int64_t)(it.p0 + c0 + cb) * a.N + f;
                if (GU || (sizeof(Y) == 2 && vec)) {      // (h has rows of whole 16-byte pieces, from the workspace's border on)
#pragma unroll
                    for (int j = 0; j < NC; ++j) turn[j * 32 + lane] = GU ? h_from_f<Y>(d[j]) : from_f<Y>(d[j]);
                    __syncwarp();
                    const int f8 = f - lane + (lane & 3) * 8;
#pragma unroll
                    for (int k = 0; k < NC / 8; ++k) {
                        const int c = k * 8 + (lane >> 2);
                        const uint4 o8 = *reinterpret_cast<const uint4*>(turn + c * 32 + (lane & 3) * 8);
                        if (f8 < a.N && ((live >> (cb + c)) & 1u))
                            *reinterpret_cast<uint4*>(y + (int64_t)(it.p0 + c0 + cb + c) * a.N + f8) = o8;
                    }
                    __syncwarp();
                } else if (live == 0xffffu && f - lane + 32 <= a.N) {
#pragma unroll
                    for (int j = 0; j < NC; ++j, o += a.N) *o = from_f<Y>(d[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < NC; ++j)
                        if (f < a.N && ((live >> (cb + j)) & 1u)) o[(int64_t)j * a.N] = from_f<Y>(d[j]);
                }
            }
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) tc5::arrive_cluster(tc5::map_rank(smem_u32(&acc_empty[buf]), 0));
        }
    }
    __syncwarp();
    tc5::fence_before();
    __syncthreads();
    tc5::cluster_sync_all();               // the peer's MMAs and signals reach into this block's memory
    if (warp == 2) { tc5::fence_after(); tc5::tmem_dealloc2(tmem, 512); }
}

// Rows named by the list, in order: a warp takes a row, eight 16-byte loads a lane on their way.  Rows that do not exist
// are left out (their results are not stored).
__global__ void __launch_bounds__(256)
gather_rows_kernel(const uint4* x, const int* rows, const int* offsets, int n, int P, int K8, int E, uint4* out) {
    pdl_trigger();
    pdl_wait();
    const int end = seg_bound(offsets, E, P);
    const int64_t p = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (p >= end) return;
    const int r = rows[p];
    if (r < 0 || r >= n) return;
    const uint4* src = x + (int64_t)r * K8;
    uint4* dst = out + p * K8;
    for (int c = threadIdx.x & 31; c < K8; c += 256) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c + u * 32 < K8) v[u] = src[c + u * 32];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c + u * 32 < K8) dst[c + u * 32] = v[u];
    }
}

template <typename T, typename Y, bool GU>
int run_pair(const GroupedArgs& a, void* scratch, cudaStream_t s) {
    constexpr int FW = GU ? 128 : 256;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return GSB_ERR_CUDA;
    const int sms = sm_count_of(dev);
    if (sms < 2) return GSB_ERR_CUDA;
    auto kernel = grouped_pair_kernel<T, Y, GU>;
    static std::atomic<uint64_t> ready{0};
    if (dev >= 64 || !((ready.load() >> dev) & 1u)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPrSmem) != cudaSuccess) return GSB_ERR_CUDA;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    const int64_t fbs = (a.N + FW - 1) / FW, hit = a.E < a.P ? a.E : a.P;
    const int64_t items = (hit + (a.P >> 8)) * fbs, most = (hit + (a.P >> 5)) * fbs;    // with tiles of 256 and of 32 rows
    if (items + sms >= (int64_t)1 << 31) return GSB_ERR_TOO_LARGE;
    const void* sorted = a.x;
    if (a.rows) {
        const int st = launch_after(gather_rows_kernel, dim3((unsigned)((a.P + 7) / 8)), 256, 0, 1, s, reinterpret_cast<const uint4*>(a.x),
                                    a.rows, a.offsets, a.n, a.P, a.K / 8, a.E, reinterpret_cast<uint4*>(scratch));
        if (st) return st;
        sorted = scratch;
    }
    CUtensorMap tw, tw2, tx;
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    if (!encode(&tw, a.w, bf, a.K, a.N, a.E, GU ? 64 : 128) || (GU && !encode(&tw2, a.w2, bf, a.K, a.N, a.E, 64)) ||
        !encode(&tx, sorted, bf, a.K, a.rows ? a.P : a.n, 0, 32))
        return GSB_ERR_CUDA;
    const int64_t pairs = most < sms / 2 ? most : sms / 2;
    return launch_after(kernel, dim3((unsigned)(pairs * 2)), kPrThreads, kPrSmem, 2, s, a, tw, GU ? tw2 : tw, tx, (int)(a.N % 8 == 0 && !misaligned(a.y, 16)));
}

template <typename T>
int run_pair_any(const GroupedArgs& a, int y_type, void* scratch, cudaStream_t s) {
    if (a.w2) return run_pair<T, T, true>(a, scratch, s);
    return y_type == GSB_TYPE_F32 ? run_pair<T, float, false>(a, scratch, s) : run_pair<T, T, false>(a, scratch, s);
}

}  // namespace

size_t grouped_pair_scratch_bytes(int P, int K) { return (size_t)P * K * 2; }

int launch_grouped_pair(const GroupedArgs& a, int type, int y_type, void* scratch, cudaStream_t s) {
    return type == GSB_TYPE_BF16 ? run_pair_any<__nv_bfloat16>(a, y_type, scratch, s) : run_pair_any<__half>(a, y_type, scratch, s);
}

int take_pair_status() {
    int st = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&st, g_pair_status, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    if (st && cudaMemcpyToSymbol(g_pair_status, &zero, sizeof(int)) != cudaSuccess) return GSB_ERR_CUDA;
    return st;
}

}  // namespace gsb
