// Expert products with 16-bit (bf16 / fp16) weights: the ragged grouped product
//   y[p, :] = W[e] x[rows[p], :]                        for offsets[e] <= p < offsets[e + 1]
// and the expert FFN built from it
//   h[p, :] = silu(gate[e] x) * (up[e] x),  y[p, :] = down[e] h[p, :],  out[t, :] = sum_k w[t, k] y[slot(t, k), :].
// Products are summed in fp32; h is rounded once to the weights' type (the tensor cores read it in that type,
// fp16 saturating at +-65504), the per-slot rows y stay fp32 and the sum over slots is taken in slot order.
#include "expert16.cuh"

namespace gsb {

namespace {

// ---- few rows per expert ----------------------------------------------------------------------
// Bound by the weights, which are read once; everything is arranged around keeping that stream going.
// One item = w weight rows (128 or 64) x up to 16 token rows of one expert, as D[weight row, token] = sum_k W[row, k]
// X[token, k]: the weights are tcgen05's M operand (128 TMEM lanes), so the tokens are padded to 16, not to 128.  For
// SwiGLU w is made of gate rows followed by as many up rows.  The copies of the next items run while this one is
// multiplied and stored (one ring over all items of a CTA).  Token rows are gathered by warps with 16-byte cp.async, only
// as many as there are; TMA is left to the weights.
// w is chosen on the device, where the number of experts with rows is known: 64 where items of 128 would leave half the
// SMs without one (2 experts of 4096 x 2048, one row each: 14.0 us against 14.5), else 128 - a last round that fills few
// SMs does not matter, they get the whole bandwidth (32 experts of 6144 x 2048, two rows each: 121 us with 4 rounds of 128
// rows, 119 with 7 of 64, 199 with 14 of 32, where the MMAs no longer keep up).
// With so few items that a cluster of blocks can share each, every block sums its part of K; the partial tiles meet in
// distributed shared memory, each block finishing some columns and adding the parts in rank order - no atomics, the same
// bits every time.
constexpr int kGrThreads = 384;            // warps: 0 weights, 1 MMA, 2 TMEM, 4-7 epilogue, 8-11 token rows
constexpr int kABytes = 128 * 128;         // at most 128 weight rows x 64 columns
constexpr int kNT = 16;                    // token rows per item at most (seg_scan is given its logarithm, 4)
constexpr int kBBytes = kNT * 128;
constexpr int kKps = 2;                    // k-blocks of 64 columns per stage
constexpr int kTokWarps = 4;
constexpr int kRing = 5 * kKps * (kABytes + kBBytes);   // five stages of 128 weight rows, 9 of 64
constexpr int kMaxStages = 9;
constexpr int kXch = 2 * kNT * 128 * 4;    // SwiGLU: two buffers of 16 columns x 128 rows
constexpr int kBars = (2 * kMaxStages + 4) * 8 + 16;     // barriers, TMEM address, abort flag
constexpr int kLists = kRing + kXch + (kMaxE + 4) * 4 + kBars;   // lists of a few slots: offsets, tokens, ids
constexpr size_t kGrSmem = (size_t)kLists + (kMaxE + 4) * 4 + 2 * kFewSlots * 4;
static_assert(kLists % 16 == 0, "the lists are read 16 bytes at a time");
// A token warp comes back to the ring kTokWarps stages later.  With fewer stages than that it could be two uses of a stage
// ahead, where the parity it waits for is the one that an unfinished phase shows as well.
static_assert(kRing / (kKps * (kABytes + kBBytes)) >= kTokWarps, "ring too short for the token warps");
static_assert(kGrSmem <= 227 * 1024, "stages exceed the shared memory of an SM");

__device__ int g_op16_status;

// item i: experts in order; inside one, all token tiles of a feature block run next to each other (they read the
// same weights, which the second one finds in L2).  `e` only moves forward.
__device__ __forceinline__ GrItem gr_item(const int* offsets, int P, const int* pre, int i, int fb_count, int fw, int& e) {
    while (i >= pre[e + 1] * fb_count) ++e;
    const int nt = pre[e + 1] - pre[e], local = i - pre[e] * fb_count;
    const int fb = local / nt, tt = local - fb * nt;
    GrItem it;
    it.e = e;
    it.f0 = fb * fw;
    const int lo = seg_bound(offsets, e, P), hi = seg_bound(offsets, e + 1, P);
    it.p0 = lo + tt * kNT;
    it.cnt = min(kNT, hi - it.p0);
    return it;
}

__device__ __forceinline__ void gr_timeout(volatile int* abort_flag) {
    *abort_flag = 1;
    atomicCAS(&g_op16_status, 0, GSB_ERR_TIMEOUT);
}

// The lists of moe_dispatch for a few slots, by counting instead of sorting: slot i's place is the number of slots with a
// smaller id plus the earlier ones of its own, expert e's start the number of slots below it.  off [E + 1], tok and id
// [kFewSlots] in shared memory; block 0 leaves the offsets and the slots' places in memory.  All threads call, and meet.
__device__ __forceinline__ void few_lists(const GroupedArgs& a, int* off, int* tok, int* id) {
    for (int i = threadIdx.x; i < kFewSlots; i += blockDim.x) {
        const int v = i < a.P ? a.ids[i] : -1;
        id[i] = v >= 0 && v < a.E ? v : a.E;               // what is nobody's sorts behind the last expert
        tok[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= a.E || i < a.P; i += blockDim.x) {
        const int mine = i < a.P ? id[i] : 0;
        int below = 0, before = 0, start = 0;
        for (int j = 0; j < a.P; j += 4) {
            const int4 v = *reinterpret_cast<const int4*>(id + j);
            const int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                below += w[u] < mine;
                before += w[u] == mine && j + u < i;
                start += w[u] < i;
            }
        }
        if (i <= a.E) {
            off[i] = start;
            if (blockIdx.x == 0) a.offsets_out[i] = start;
        }
        if (i < a.P && mine < a.E) {
            tok[below + before] = i / a.topk;
            if (blockIdx.x == 0) a.slot_pos_out[i] = below + before;
        }
    }
    __syncthreads();
}

template <typename T, typename Y, bool GU>
__global__ void __launch_bounds__(kGrThreads, 1)
grouped_kernel(const GroupedArgs a, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_w2) {
    extern __shared__ __align__(1024) uint8_t smem[];
    float* s_xch = reinterpret_cast<float*>(smem + kRing);
    int* pre = reinterpret_cast<int*>(smem + kRing + kXch);   // [E + 1] token tiles before expert e
    uint64_t* full = reinterpret_cast<uint64_t*>(pre + kMaxE + 4);
    uint64_t* empty = full + kMaxStages;
    uint64_t* acc_full = empty + kMaxStages;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) { mbar_init(&full[i], 2); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 4); }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) { tc5::prefetch_map(&tm_w); if (GU) tc5::prefetch_map(&tm_w2); }
    if (warp == 2) { tc5::tmem_alloc(tmem_slot, 2 * kNT); tc5::tmem_relinquish(); }
    const int S = (int)tc5::cluster_size(), rank = (int)tc5::cluster_rank();
    pdl_trigger();
    pdl_wait();
    int descending = (smem_u32(smem) & 1023u) != 0;    // (the swizzled tiles need a 1 KiB boundary: as good as no list)
    const int *offsets = a.offsets, *rows = a.rows;
    if (GU && a.ids) {                     // every block makes the lists of a few slots for itself
        int* s_off = reinterpret_cast<int*>(smem + kLists);
        few_lists(a, s_off, s_off + kMaxE + 4, s_off + kMaxE + 4 + kFewSlots);
        offsets = s_off;
        rows = s_off + kMaxE + 4;
    }
    descending |= seg_scan(offsets, a.E, a.P, 4, pre, reinterpret_cast<int*>(s_xch));
    tc5::fence_before();
    descending = __syncthreads_or(descending);
    tc5::fence_after();
    if (S > 1) tc5::cluster_arrive();      // this block runs, and s_xch is no longer the scan's
    const uint32_t tmem = *tmem_slot;
    const int nkb = (a.K + 63) >> 6;
    // at most (E + P / 16) token tiles, and so many items as the host has checked to fit; a list that descends is no list
    const int tiles = descending ? 0 : pre[a.E];
    const int64_t wide = (int64_t)tiles * ((a.N + (GU ? 63 : 127)) / (GU ? 64 : 128));
    const int w = S == 1 && wide * 2 <= (int)gridDim.x ? 64 : 128;      // weight rows of an item
    const int fw = GU ? w / 2 : w;         // output features of an item
    const int FB = (a.N + fw - 1) / fw;
    const int items = tiles * FB;
    // the ring's stages are as long as w rows need, so a narrow item has as many bytes on their way as a wide one (the
    // MMA's unused rows read on into what follows; their lanes are not stored)
    const int abytes = w * 128, stage_bytes = kKps * (abytes + kBBytes), stages = min(kMaxStages, kRing / stage_bytes);
    const int first = (int)blockIdx.x / S, step = (int)gridDim.x / S;
    const int kb0 = nkb * rank / S, kb1 = nkb * (rank + 1) / S;     // this block's part of the sum

    // which of an item's tokens exist, as a mask (whole warps ask)
    auto live_tokens = [&](const GrItem& it) {
        int r = lane < it.cnt ? 0 : -1;
        if (rows && r == 0) r = rows[it.p0 + lane];
        return __ballot_sync(0xffffffffu, r >= 0 && r < a.n);
    };

    bool met = false;                      // S > 1: whether this warp has waited for the cluster's first meeting

    if (warp == 0) {                       // ---- weights
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0;
        int e = 0;
        bool dead = false;
        for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step) {
            const GrItem it = gr_item(offsets, a.P, pre, i, FB, fw, e);
            for (int kb = kb0; kb < kb1; kb += kKps) {
                if (!tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                if (leader) {
                    const int nk = min(kKps, kb1 - kb);
                    mbar_arrive_expect_tx(&full[st], (uint32_t)(nk * w * 128));
                    uint8_t* dst = smem + st * stage_bytes;
                    for (int j = 0; j < nk; ++j)
                        for (int r = 0; r < fw; r += 32) {
                            tc5::tma_load_3d(dst + j * abytes + r * 128, &tm_w, (kb + j) * 64, it.f0 + r, it.e, &full[st]);
                            if (GU) tc5::tma_load_3d(dst + j * abytes + (fw + r) * 128, &tm_w2, (kb + j) * 64, it.f0 + r, it.e, &full[st]);
                        }
                }
                if (++st == (uint32_t)stages) { st = 0; ph ^= 1u; }
            }
        }
        // the signals of the last MMAs have arrived before the block ends
        for (int j = 0; j < stages && !tc5::warp_set(abort_flag); ++j) {
            tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit);
            if (++st == (uint32_t)stages) { st = 0; ph ^= 1u; }
        }
        // after a time-out: nothing may still be copying into this block's memory when it ends
        if (tc5::warp_set(abort_flag))
            for (int j = 0; j < stages; ++j) {
                if (st == 0) { st = (uint32_t)stages; ph ^= 1u; }
                --st;
                tc5::warp_wait(&full[st], ph, kGrWaitLimit / 16);
            }
    } else if (warp >= 8) {                // ---- token rows: the four warps take stages in turn
        // eight lanes copy the 128 bytes of a row's k-block; a warp fences its copies before it hands the stage over, and
        // the other three's are on their way meanwhile
        const int group = warp - 8, piece = lane & 7;
        const T* x = reinterpret_cast<const T*>(a.x) + piece * 8;
        uint32_t st = 0, ph = 0, cnt = 0;
        int e = 0;
        bool dead = false;
        for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step) {
            const GrItem it = gr_item(offsets, a.P, pre, i, FB, fw, e);
            int r[kNT / 4];
#pragma unroll
            for (int j = 0; j < kNT / 4; ++j) {
                // rows that do not exist read row 0 and are not stored; what lies in the place of the columns behind the
                // tile's last reaches only those columns
                const int q = j * 4 + (lane >> 3);
                r[j] = -1;
                if (q < it.cnt) {
                    const int v = rows ? rows[it.p0 + q] : it.p0 + q;
                    r[j] = v >= 0 && v < a.n ? v : 0;
                }
            }
            for (int kb = kb0; kb < kb1; kb += kKps, ++cnt) {
                if ((int)(cnt % kTokWarps) == group) {
                    if (!tc5::warp_wait(&empty[st], ph ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                    const uint32_t base = smem_u32(smem) + st * stage_bytes + kKps * abytes + (uint32_t)((lane >> 3) * 128);
#pragma unroll
                    for (int u = 0; u < kKps; ++u) {
                        const bool in = (kb + u) * 64 + piece * 8 < a.K;
                        const T* xk = in ? x + (kb + u) * 64 : x;
#pragma unroll
                        for (int j = 0; j < kNT / 4; ++j)     // 128-byte swizzle: piece c of row q lies at c ^ q % 8
                            if (r[j] >= 0 && kb + u < kb1)
                                tc5::cp_async16(base + (uint32_t)(u * kBBytes + j * 512 + ((piece ^ ((j * 4 + (lane >> 3)) & 7)) << 4)),
                                                xk + (int64_t)r[j] * a.K, in);
                    }
                    tc5::cp_async_commit();
                    tc5::cp_async_wait<0>();
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[st]);
                }
                if (++st == (uint32_t)stages) { st = 0; ph ^= 1u; }
            }
        }
        tc5::cp_async_wait<0>();
    } else if (warp == 1) {                // ---- MMA issue
        const bool leader = tc5::elect_one();
        uint32_t st = 0, ph = 0, tl = 0;
        bool dead = false;
        constexpr uint32_t idesc_ab = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t idesc = tc5::idesc_f16(idesc_ab, 128, kNT);
        const uint64_t d0 = tc5::desc_sw128(smem_u32(smem));
        for (int i = first; i < items && !dead && !tc5::warp_set(abort_flag); i += step, ++tl) {
            const uint32_t buf = tl & 1u;
            if (!tc5::warp_wait(&acc_empty[buf], ((tl >> 1) & 1u) ^ 1u, kGrWaitLimit)) { gr_timeout(abort_flag); break; }
            tc5::fence_after();
            uint32_t acc = 0;
            for (int kb = kb0; kb < kb1; kb += kKps) {
                if (!tc5::warp_wait(&full[st], ph, kGrWaitLimit)) { gr_timeout(abort_flag); dead = true; break; }
                tc5::fence_after();
                if (leader) {
                    const uint64_t ad = d0 + (uint64_t)(st * (uint32_t)(stage_bytes >> 4));
                    const uint64_t bd = ad + (uint64_t)(kKps * abytes >> 4);
#pragma unroll
                    for (int j = 0; j < kKps; ++j)
                        if (kb + j < kb1)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                tc5::mma_f16_ss(tmem + buf * kNT, ad + (uint64_t)(j * (abytes >> 4) + k * 2),
                                                bd + (uint64_t)(j * (kBBytes >> 4) + k * 2), idesc, j + k ? 1u : acc);
                    tc5::commit(&empty[st]);
                }
                acc = 1u;
                if (++st == (uint32_t)stages) { st = 0; ph ^= 1u; }
            }
            if (!dead && leader) tc5::commit(&acc_full[buf]);
        }
        // after a time-out: no MMA is at work, and no signal on its way, when the block ends (otherwise the others have
        // waited for all of them)
        if (tc5::warp_set(abort_flag)) {
            if (st == 0) { st = (uint32_t)stages; ph ^= 1u; }
            tc5::warp_wait(&empty[st - 1], ph, kGrWaitLimit);      // (at once where there was none)
            if (dead) --tl;                                        // (counted, but not announced)
            if (tl) tc5::warp_wait(&acc_full[(tl - 1) & 1u], ((tl - 1) >> 1) & 1u, kGrWaitLimit);
        }
    } else if (warp >= 4) {                // ---- epilogue: this thread's TMEM lane = weight row
        const int q = warp & 3, row = q * 32 + lane;
        uint32_t tl = 0;
        int e = 0;
        Y* y = reinterpret_cast<Y*>(a.y);
        for (int i = first; i < items; i += step, ++tl) {
            const GrItem it = gr_item(offsets, a.P, pre, i, FB, fw, e);
            const uint32_t buf = tl & 1u;
            int ok = tc5::warp_set(abort_flag) ? 0 : (int)tc5::warp_wait(&acc_full[buf], (tl >> 1) & 1u, a.sum_limit);
            if (!ok) gr_timeout(abort_flag);
            // all four warps must agree to go on: they meet at a barrier below
            if (GU) ok = epilogue_agree(ok, 1);
            if (!ok) break;
            tc5::fence_after();
            uint32_t u[kNT];
            tc5::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + buf * kNT, u);
            const uint32_t live = live_tokens(it);
            tc5::tmem_ld_wait();
            tc5::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
            if (S > 1) {                   // to the block that finishes the column: [source][column][row]
                const int per = kNT / S;
                __syncwarp();
                if (!met) tc5::cluster_wait();
                met = true;                // (one item per cluster)
#pragma unroll
                for (int j = 0; j < kNT; ++j)
                    tc5::st_cluster(tc5::map_rank(smem_u32(s_xch + (rank * per + j % per) * 128 + row), (uint32_t)(j / per)), __uint_as_float(u[j]));
            } else if (GU) {
                // rows [0, fw) are gate, [fw, 2 fw) the up rows of the same features
                float* xs = s_xch + buf * kNT * 128;
#pragma unroll
                for (int j = 0; j < kNT; ++j) xs[j * 128 + row] = __uint_as_float(u[j]);
                epilogue_sync(1);
                const int fl = row & (fw - 1), f = it.f0 + fl, groups = 128 / fw;     // fw is 64 or 32
                for (int c = row / fw; c < it.cnt; c += groups)
                    if (f < a.N && ((live >> c) & 1u))
                        y[(int64_t)(it.p0 + c) * a.N + f] = h_from_f<Y>(swiglu(xs[c * 128 + fl], xs[c * 128 + fw + fl]));
            } else {
                const int f = it.f0 + row;
                if (row < w && f < a.N)
#pragma unroll
                    for (int j = 0; j < kNT; ++j)
                        if ((live >> j) & 1u) y[(int64_t)(it.p0 + j) * a.N + f] = from_f<Y>(__uint_as_float(u[j]));
            }
        }
    }
    __syncwarp();
    tc5::fence_before();
    if (S > 1) {
        if (!met) tc5::cluster_wait();
        tc5::cluster_sync_all();
        if (first < items && warp >= 4 && warp < 8 && !tc5::warp_set(abort_flag)) {
            int e = 0;
            const GrItem it = gr_item(offsets, a.P, pre, first, FB, fw, e);
            const uint32_t live = live_tokens(it);
            const int per = kNT / S, row = (warp & 3) * 32 + lane, fl = GU ? row & 63 : row, f = it.f0 + fl;
            for (int cl = GU ? row >> 6 : 0; cl < per; cl += GU ? 2 : 1) {
                const int c = rank * per + cl;
                if (f >= a.N || !((live >> c) & 1u)) continue;
                float s0 = 0.f, s1 = 0.f;
                for (int src = 0; src < S; ++src) {
                    s0 += s_xch[(src * per + cl) * 128 + fl];
                    if (GU) s1 += s_xch[(src * per + cl) * 128 + 64 + fl];
                }
                reinterpret_cast<Y*>(a.y)[(int64_t)(it.p0 + c) * a.N + f] = GU ? h_from_f<Y>(swiglu(s0, s1)) : from_f<Y>(s0);
            }
        }
    }
    __syncthreads();
    if (warp == 2) { tc5::fence_after(); tc5::tmem_dealloc(tmem, 2 * kNT); }
}

template <typename T, typename Y, bool GU>
int run_grouped(const GroupedArgs& a, cudaStream_t s) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return GSB_ERR_CUDA;
    const int sms = sm_count_of(dev);
    if (!sms) return GSB_ERR_CUDA;
    auto kernel = grouped_kernel<T, Y, GU>;
    static std::atomic<uint64_t> ready{0};     // devices on which the shared-memory size was raised
    if (dev >= 64 || !((ready.load() >> dev) & 1u)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGrSmem) != cudaSuccess) return GSB_ERR_CUDA;
        if (dev < 64) ready.fetch_or(1ull << dev);
    }
    const int64_t fbs = (a.N + (GU ? 31 : 63)) / (GU ? 32 : 64), tiles = (a.E < a.P ? a.E : a.P) + a.P / kNT, items = tiles * fbs;
    if (items + sms >= (int64_t)1 << 31) return GSB_ERR_TOO_LARGE;
    CUtensorMap tw, tw2;
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    if (!encode(&tw, a.w, bf, a.K, a.N, a.E, 32) || (GU && !encode(&tw2, a.w2, bf, a.K, a.N, a.E, 32))) return GSB_ERR_CUDA;
    // A cluster of four blocks per item where that many still run at once and the sum is long (1 expert, one row of 6144 to
    // 2048: 10.9 us against 17.4, 4 experts, 4096 to 1000: 9.6 against 13.3; at 1024 the cluster costs 1 us more than it
    // saves, at 2048 the two are equal; two or eight blocks were no better).
    const int64_t wide = tiles * ((a.N + (GU ? 63 : 127)) / (GU ? 64 : 128));
    const int S = a.K > 2048 && wide * 4 <= sms ? 4 : 1;
    const int grid = S > 1 ? (int)wide * S : (int)(items < sms ? items : sms);
    return launch_after(kernel, dim3(grid), kGrThreads, kGrSmem, S, s, a, tw, GU ? tw2 : tw);
}

template <typename T>
int run_grouped_any(const GroupedArgs& a, int y_type, cudaStream_t s) {
    if (a.w2) return run_grouped<T, T, true>(a, s);
    return y_type == GSB_TYPE_F32 ? run_grouped<T, float, false>(a, s) : run_grouped<T, T, false>(a, s);
}

// The kernel for many rows above 16 rows per expert on average: the host knows the length of the list, not what is in it.
// Few rows against many, us, 32 experts of 6144 to 2048: 8 rows an expert 124 and 136, 16 rows 126 and 137, 20 rows 149 and
// 138, 32 rows 181 and 141; the same with Zipf-like loads (exponent 1.1): 131 and 136, 141 and 138, 159 and 137, 190 and
// 140.  8 experts of 4096 to 4096: 8 rows 45 and 51, 16 rows 54 and 52, 32 rows 70 and 53.  Small products change places
// later (16 experts of 1024 to 512: 24 rows 8.0 and 10.1, 32 rows 11.6 and 10.6).  Where the average says little it can be
// wrong: all rows on one of 32 experts, 256 rows 44 and 28, 512 rows 83 and 29; and a shard whose list is mostly slots of
// other GPUs (FFN, 32 of 256 experts, 6144 x 2048): 128 tokens 359 and 379, 512 tokens 394 and 400, 1024 tokens 514 and 422.
bool use_pair(int P, int E) { return P / E > 16; }

int launch_grouped(GroupedArgs a, int type, int y_type, void* scratch, cudaStream_t s) {
    a.sum_limit = gr_sum_limit(a.K);
    if (use_pair(a.P, a.E)) return launch_grouped_pair(a, type, y_type, scratch, s);
    return type == GSB_TYPE_BF16 ? run_grouped_any<__nv_bfloat16>(a, y_type, s) : run_grouped_any<__half>(a, y_type, s);
}

// The lists alone, for the pair kernel.
__global__ void __launch_bounds__(1024)
dispatch_few_kernel(const GroupedArgs a, int* tok) {
    __shared__ __align__(16) int s_list[kMaxE + 4 + 2 * kFewSlots];
    pdl_trigger();
    few_lists(a, s_list, s_list + kMaxE + 4, s_list + kMaxE + 4 + kFewSlots);
    if (threadIdx.x < a.P) tok[threadIdx.x] = s_list[kMaxE + 4 + threadIdx.x];
}

// out[t] = sum over k, in order, of w[t, k] * y[slot_pos[t, k]]; slots whose id is outside [0, E) add nothing.  A block
// takes 1024 * U features of a token: where the slots' rows lie is read once, then every thread has the loads of J
// slots on their way, U each of 16 bytes: four of one slot (16384 rows of 4096 in 50 us, the rate of a copy), or one of
// eight slots, which spreads a few tokens over more blocks.
template <typename O, int U>
__global__ void __launch_bounds__(256)
combine16_kernel(const float* y, const int* ids, const int* slot_pos, const float* w, int topk, int H, int E, O* out) {
    const int64_t t = U == 1 ? blockIdx.y : blockIdx.x;
    __shared__ int s_pos[256];
    __shared__ float s_w[256];
    pdl_trigger();
    pdl_wait();
    constexpr int J = U == 1 ? 8 : 1;
    float4 acc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int c0 = (int)(U == 1 ? blockIdx.x : blockIdx.y) * 1024 * U + threadIdx.x * 4;     // H is a multiple of 8
    for (int k0 = 0; k0 < topk; k0 += 256) {
        __syncthreads();
        if (k0 + (int)threadIdx.x < topk) {
            const int64_t i = t * topk + k0 + threadIdx.x;
            const int id = ids[i];
            const bool have = id >= 0 && id < E;
            s_pos[threadIdx.x] = have ? slot_pos[i] : -1;
            s_w[threadIdx.x] = have ? w[i] : 0.f;
        }
        __syncthreads();
        const int kn = min(256, topk - k0);
        for (int k = 0; k < kn; k += J) {
            float4 v[J][U];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int pos = k + j < kn ? s_pos[k + j] : -1;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    v[j][u] = pos >= 0 && c0 + u * 1024 < H ? __ldcs(reinterpret_cast<const float4*>(y + (int64_t)pos * H + c0 + u * 1024))
                                                            : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float wk = k + j < kn ? s_w[k + j] : 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    acc[u].x = fmaf(wk, v[j][u].x, acc[u].x); acc[u].y = fmaf(wk, v[j][u].y, acc[u].y);
                    acc[u].z = fmaf(wk, v[j][u].z, acc[u].z); acc[u].w = fmaf(wk, v[j][u].w, acc[u].w);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (c0 + u * 1024 >= H) continue;
        __align__(16) O o[4] = {from_f<O>(acc[u].x), from_f<O>(acc[u].y), from_f<O>(acc[u].z), from_f<O>(acc[u].w)};
        O* dst = out + t * H + c0 + u * 1024;
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(o);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
    }
}

constexpr int kManyTokens = 256;

template <typename O>
int run_combine16(const float* y, const int* ids, const int* slot_pos, const float* w, int n, int topk, int H, int E,
                  void* out, cudaStream_t s) {
    O* o = reinterpret_cast<O*>(out);
    // a grid's second dimension ends at 65535: few tokens may have more feature blocks than that (256 tokens and more would
    // need per-slot rows of 275 GB for it, and are refused)
    if (n < kManyTokens) return launch_after(combine16_kernel<O, 1>, dim3((H + 1023) / 1024, n), 256, 0, 1, s, y, ids, slot_pos, w, topk, H, E, o);
    return launch_after(combine16_kernel<O, 4>, dim3(n, (H + 4095) / 4096), 256, 0, 1, s, y, ids, slot_pos, w, topk, H, E, o);
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
    if (in % 8 || E > 1024 || P > kMaxSlots || in > kMaxDim || out > kMaxDim) return GSB_ERR_UNSUPPORTED;
    const size_t need = rows ? gsb_grouped_gemm_workspace_bytes(P, in, E) : 0;
    if (need && (!workspace || misaligned(workspace, 256))) return GSB_ERR_INVALID_ARG;
    if (need > workspace_bytes) return GSB_ERR_WORKSPACE;
    const __int128 y_bytes = (__int128)P * out * type_bytes(y_type);
    if (overlap(y, y_bytes, x, (__int128)n * in * 2) || overlap(y, y_bytes, w, (__int128)E * out * in * 2) ||
        overlap(y, y_bytes, expert_offsets, (E + 1) * 4) || overlap(y, y_bytes, rows, (__int128)P * 4))
        return GSB_ERR_INVALID_ARG;
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
    if (hidden % 8 || moe_inter % 8 || E > 1024 || (int64_t)n * topk > kMaxSlots || hidden > kMaxDim || moe_inter > kMaxDim)
        return GSB_ERR_UNSUPPORTED;
    if (n >= kManyTokens && (hidden + 4095) / 4096 > 65535) return GSB_ERR_TOO_LARGE;
    if (!workspace || misaligned(workspace, 256)) return GSB_ERR_INVALID_ARG;
    const Ffn16Ws ws = carve16(n, topk, hidden, moe_inter, E, workspace);
    if (workspace_bytes < ws.total) return GSB_ERR_WORKSPACE;
    // (x has been read when the last launch writes out; the ids and weights are read by it)
    const __int128 out_bytes = (__int128)n * hidden * type_bytes(out_type), slot_bytes = (__int128)n * topk * 4;
    if (overlap(out, out_bytes, topk_ids, slot_bytes) || overlap(out, out_bytes, topk_weights, slot_bytes)) return GSB_ERR_INVALID_ARG;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    GroupedArgs g{};
    g.x = x; g.w = gate_w; g.w2 = up_w; g.offsets = ws.offsets; g.rows = ws.tok;
    g.n = n; g.P = n * topk; g.K = hidden; g.N = moe_inter; g.E = E; g.y = ws.h;
    int st = GSB_OK;
    if (g.P <= kFewSlots) {
        g.ids = topk_ids; g.topk = topk; g.offsets_out = ws.offsets; g.slot_pos_out = ws.slot_pos;
        if (use_pair(g.P, E)) {
            dispatch_few_kernel<<<1, 1024, 0, s>>>(g, ws.tok);
            st = launch_status();
            g.ids = nullptr;
        } else {
            g.offsets = nullptr; g.rows = nullptr;
        }
    } else {
        st = launch_dispatch(topk_ids, n, topk, E, ws.offsets, ws.tok, ws.row, ws.slot_pos, s, ws.disp);
    }
    if (st) return st;
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
    const int pair = take_pair_status(), lora = take_lora_status();
    return st ? st : pair ? pair : lora;
}
