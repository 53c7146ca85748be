// ============================================================================
// mxk_matmul.cuh — 8-bit products with UE8M0 block scales, apart from the layer.
//
//   out[m, n] = sum_k x[m, k] 2^(sx[m, k/128] - 127) * w[n, k] 2^(sw[.., k/128] - 127)
//
// dense (one weight matrix) or grouped (rows offsets[e] .. offsets[e+1] of x meet w[e]).
// The scales are powers of two, one per 128 columns, so the block-scaled tensor-core MMA
// applies them exactly on its way into one FP32 accumulator over all of K.
//
// Orientation: the WEIGHT rows are the M side of the MMA (128 per CTA) and the rows of x its N
// side, whose extent is a run-time multiple of 16.  An expert with 3 rows then costs an N = 16
// MMA instead of a 128-row tile, a group of 1100 rows is cut into five equal tiles of 224 instead
// of nine of 128, and one kernel body serves a single token and a prefill.  The accumulators come out
// transposed (lane = output column), which the epilogue's stores turn round: the 32 lanes of a
// warp write 32 neighbouring columns of one output row.
//
// A unit of work is a tile of 128 (CTA pair: 256) weight rows x up to bt_max rows of x.  Units
// are dealt out round-robin; every role walks the same list from the sanitised group table in
// shared memory, so there is no task queue, no counter in global memory and no workspace: launches
// on several streams or in several graphs share nothing.
//
// Warp roles (384 threads) as in the layer's GEMM phase: warp 0 TMA producer, warp 1 MMA issuer,
// warps 2-3 scale tiles (global bytes -> shared tile -> tensor memory), warps 4-11 epilogue.  Tensor
// memory holds two accumulators of up to 224 columns that alternate between tiles, so that the drain
// of one hides under the MMAs of the next.  (Both as the halves of one tile of 448 rows were slower, although a
// quarter fewer bytes cross L2: MMAs that alternate between two accumulators ran at 75 % of the pipe.)
//
// What bounds it: many rows, the tensor pipe at the clock that the 1 kW cap leaves (4096 x 4096 x 7168: 93 us = 2.57
// PFLOP/s in a burst, 112 us in a loop of seconds, at 1.55 - 1.6 GHz); few rows, the weights' stream (32 groups of 4
// rows x 4096 x 6144: 121 us = 6.7 TB/s); the smallest calls, a chain of round trips of some 5 us that starts under
// the predecessor's end (programmatic launch).  Rows of an operand that are no multiple of 32 bytes apart cost a
// third: half of the tile loads' rows then straddle a sector (2043 x 1111 x 4016: 17.6 us, at depth 4000 14.5, 4096 13.4).
//
// Few tiles (small batches): the K extent is split over the CTAs of a cluster, the partial tiles
// are exchanged through distributed shared memory and added in the order of the splits, so results
// do not depend on timing.
//
// Every wait is bounded; on expiry the CTA records a status word, unwinds and frees its TMEM.
// ============================================================================
#pragma once

constexpr int kMmThreads = 384;
constexpr int kMmEpiWarps = 8;
constexpr int kMmFirstEpi = 4;
constexpr int kMmMaxStages = 8;
constexpr int kMmMaxSfSlots = 8;
constexpr int kMmSfTile = 512;                 // 128 rows x 4 scale bytes
constexpr int kMmStageKb = 2;                  // K blocks of a ring stage
constexpr int kMmRowsMax = 224;                // columns of an accumulator: 2 x 224 leave 64 TMEM columns to the scales
constexpr int kMmWBytes = 128 * 128;           // weight tile of one K block
constexpr int kMmMaxExperts = 1024;
constexpr int kMmTmemCols = 512;
constexpr int kMmSmemLimit = 227 * 1024;

struct MmArgs {
    const uint8_t* x_sf;       // [rows][x_sf_stride] or null (all 127)
    const uint8_t* w_sf;       // [experts][w_sf_rows][nkb] or null
    uint16_t* out;             // bf16 [rows][out_stride]
    const int* offsets;        // [experts + 1] or null (dense)
    long long x_sf_stride, out_stride;
    int rows, cols, nkb, experts;
    int n_tiles;               // weight tiles of a group
    int bt_max, box;           // rows of x per tile at most; rows per TMA box (pairs: half of them)
    int n_stages, sf_slots, sf_col;
    int splits;                // CTAs of a cluster that share a tile's K extent: 1, 2, 4 or 8; pairs take it whole
    int w_sf_rows, w_per_row;  // rows of a group's weight scale plane; 1: one scale row per weight row
    int zero_tail;             // clear out rows behind the last group
    FastDiv fbt, fnt;          // division by bt_max and n_tiles
    uint32_t formats;          // operand format bits of the instruction descriptor
    unsigned long long wait_ns;
};

struct MmSmem {
    uint64_t full[kMmMaxStages], empty[kMmMaxStages];
    uint64_t sf_full[kMmMaxSfSlots], sf_empty[kMmMaxSfSlots], sf_peer[kMmMaxSfSlots];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t red_full, red_free;     // split-K exchange: all partials have come in / every split has added its rows up
    uint32_t tmem_base;
    int abort_flag;
};

// the barriers of MmSmem lie behind one another; what each expects
constexpr int kMmBarriers = 2 * kMmMaxStages + 3 * kMmMaxSfSlots + 6;
__device__ __forceinline__ uint32_t mm_barrier_count(int i, uint32_t ctas, uint32_t splits) {
    const int k = i - (2 * kMmMaxStages + 3 * kMmMaxSfSlots);
    return k == 2 || k == 3 ? kMmEpiWarps * ctas : k == 5 ? kMmEpiWarps * splits : 1u;   // acc_empty; red_free; copies, commits and stores
}
static_assert(offsetof(MmSmem, tmem_base) == kMmBarriers * sizeof(uint64_t), "barriers first, without gaps");

struct MmTile {
    int group, w_row, x_row, bt, valid;    // w_row: first weight row inside the group; x_row, bt: rows of x
};

// status word of the products on this device: 0, or the first wait that expired
__device__ int g_mm_status = 0;

// Tile t of the list: groups in order; inside a group the operand with fewer rows turns fastest,
// so that the other one is read from memory once while the first stays in L2.
template <bool kPair>
__device__ __forceinline__ bool mm_tile(const MmArgs& a, const int* start, const int* before, int t, MmTile& o) {
    if (t >= before[a.experts]) return false;
    int lo = 0, hi = a.experts;   // last group with before[g] <= t; empty groups share a value with their successor
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= t) lo = mid; else hi = mid;
    }
    const int n = start[lo + 1] - start[lo], i = t - before[lo];
    int xt = 0, wt = i, per = n;
    if (n > a.bt_max) {
        const int tt = a.fbt.div(n + a.bt_max - 1);
        if (n <= a.cols) { wt = i / tt; xt = i - wt * tt; }
        else { xt = a.fnt.div(i); wt = i - xt * a.n_tiles; }
        per = (n + tt - 1) / tt;
    }
    o.group = lo;
    o.bt = (per + 15) & ~15;   // the group's rows spread evenly over its tiles
    o.w_row = wt * (kPair ? 256 : 128);
    o.x_row = start[lo] + xt * o.bt;
    o.valid = min(o.bt, n - xt * o.bt);
    return true;
}

__device__ __forceinline__ void mm_raise(MmSmem* S, int code) {
    atomicCAS(&g_mm_status, 0, code);
    *(volatile int*)&S->abort_flag = 1;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
// A store into another CTA of the cluster that reports its four bytes to a barrier there: no fence, no
// separate arrival (with ordinary stores, a release and an arrival the exchange of a 1 x 4096 x 6144 product took 0.6 us longer).
__device__ __forceinline__ void st_async_b32(uint32_t addr, uint32_t v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(v), "r"(bar) : "memory");
}
// v = the word at p if `has`, else v as it was
__device__ __forceinline__ void ld_if(uint32_t& v, const void* p, bool has) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\n@q ld.global.b32 %0, [%1];\n}\n" : "+r"(v) : "l"(p), "r"((int)has));
}
// An arrival, here or in another CTA of the cluster, that orders no memory: what it reports are reads of tensor memory,
// which tcgen05.wait and tcgen05.fence have ordered before it.  As a release it would wait for the warp's stores of the
// result, some 1700 clocks a tile (32 groups of 300 rows x 2048 x 512: 33 us with it, 26 without).
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
    return p != 0;
}
// commit of a pair's MMAs onto the barrier at this offset in both of its CTAs (a signal inside one
// cluster; no load, no other GPU's memory)
__device__ __forceinline__ void umma_commit_pair_both(uint32_t bar_smem_addr) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar_smem_addr), "h"((uint16_t)3)
                 : "memory");
}

template <bool kPair>
__device__ __forceinline__ void mm_body(const MmArgs& a, const CUtensorMap* tm_x, const CUtensorMap* tm_w) {
    extern __shared__ uint8_t mm_smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(mm_smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kXTiles = kPair ? 2 : 1, kSfTiles = 1 + kXTiles;   // scale tiles: weight rows, then 128 rows of x each
    constexpr uint32_t kSfSlotBytes = kSfTiles * kMmSfTile, kSfSlotCols = kSfTiles * 4;
    const uint32_t x_bytes = (uint32_t)a.box * 128u;
    const uint32_t stage_bytes = (uint32_t)kMmStageKb * ((uint32_t)kMmWBytes + x_bytes);   // [w]..[x].., tiles of 128-byte rows
    uint8_t* sf_tiles = tiles + (size_t)a.n_stages * stage_bytes;
    float* red = reinterpret_cast<float*>(sf_tiles + a.sf_slots * kSfSlotBytes);   // [bt_max][128] partial sums, splits > 1 only
    const int splits = kPair ? 1 : a.splits;
    MmSmem* S = reinterpret_cast<MmSmem*>(reinterpret_cast<uint8_t*>(red) + (splits > 1 ? (size_t)a.bt_max * 512 : 0));
    int* start = reinterpret_cast<int*>(S + 1);
    int* before = start + a.experts + 1;  // both [experts + 1]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a cluster is a pair, or the splits of a tile
    constexpr uint32_t kCtas = kPair ? 2u : 1u;               // CTAs of a unit that share a tile of accumulators
    const bool clustered = kPair || splits > 1;
    const uint32_t crank = clustered ? cluster_ctarank() : 0u;
    const uint32_t half = kPair ? crank : 0u;                 // which CTA of the pair; the first one leads
    const bool leader = half == 0;
    const int split = kPair ? 0 : (int)crank;
    volatile int* abort_flag = &S->abort_flag;
    const uint64_t wait_ns = a.wait_ns;

    // Start-up, kept short because it is a fifth of a small product: warp 0 initialises the barriers, builds the
    // group table and goes on to its first loads without waiting for the others; warp 1 meanwhile allocates TMEM.
    // Every role waits for the kernels before this one (grid_wait) where it first touches memory or first waits for one that
    // does, and not earlier, so that its way there, instruction fetches included, lies under their end.  Not later either: a
    // bounded wait that began under a long kernel (a collective behind a late rank) would run out in a healthy product.
    grid_let_next_begin();
    if (clustered && warp != 0) cluster_arrive();
    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(tm_w);
            tma_prefetch_desc(tm_x);
        }
        for (int i = lane; i < kMmBarriers; i += 32) mbar_init(&S->full[0] + i, mm_barrier_count(i, kCtas, (uint32_t)splits));
        if (lane == 0) S->abort_flag = 0;
        mbar_fence_init();
        fence_proxy_async_smem();
        if (clustered) {
            __syncwarp();
            cluster_arrive();
        }
        // Group table.  Offsets come from the device and are not trusted: clamped into [0, rows] and made
        // ascending (a running maximum), groups are disjoint whatever they held and no tile reaches outside.
        if (!a.offsets) {
            if (lane == 0) {
                start[0] = before[0] = 0;
                start[1] = a.rows;
                before[1] = a.fbt.div(a.rows + a.bt_max - 1) * a.n_tiles;
            }
        } else {
            grid_wait();   // the first read of memory
#pragma unroll 4
            for (int e = lane; e <= a.experts; e += 32) start[e] = min(max(a.offsets[e], 0), a.rows);
            __syncwarp();
            // every lane walks a contiguous share of the groups; the shares are joined by warp scans
            const int share = a.experts / 32 + 1, e0 = lane * share, e1 = min(e0 + share, a.experts + 1);
            int top = 0;
            for (int e = e0; e < e1; ++e) start[e] = top = max(top, start[e]);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = max(top, __shfl_up_sync(0xFFFFFFFFu, top, d));   // lanes below d get their own value
            int below = __shfl_up_sync(0xFFFFFFFFu, top, 1);
            if (lane == 0) below = 0;
            for (int e = e0; e < e1; ++e) start[e] = max(below, start[e]);
            __syncwarp();
            int sum = 0;
            for (int e = e0; e < e1; ++e) {
                before[e] = sum;
                if (e < a.experts) sum += a.fbt.div(start[e + 1] - start[e] + a.bt_max - 1) * a.n_tiles;
            }
            const int own = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xFFFFFFFFu, sum, d);
                if (lane >= d) sum += o;
            }
            for (int e = e0; e < e1; ++e) before[e] += sum - own;
        }
        __syncwarp();
        asm volatile("barrier.cta.arrive 1, %0;" ::"n"(kMmThreads) : "memory");
    } else {
        if (warp == 1) {
            if constexpr (kPair) { tmem_alloc_pair(&S->tmem_base, kMmTmemCols); tmem_relinquish_pair(); }
            else { tmem_alloc(&S->tmem_base, kMmTmemCols); tmem_relinquish(); }
        }
        tc_fence_before();
        asm volatile("barrier.cta.sync 1, %0;" ::"n"(kMmThreads) : "memory");
        tc_fence_after();
    }
    // the partner's barriers must exist before anything arrives on them; a split's producer has no partner
    if (kPair || (clustered && warp != 0)) cluster_wait();
    const uint32_t tmem_base = warp == 0 ? 0u : *(volatile uint32_t*)&S->tmem_base;

    const int cluster = (int)kCtas * splits, unit = (int)blockIdx.x / cluster, n_units = (int)gridDim.x / cluster;
    // K blocks of this split, cut at multiples of four blocks (one scale word holds four)
    const int groups_all = (a.nkb + 3) >> 2;
    const int g_first = groups_all * split / splits, g_last = groups_all * (split + 1) / splits;
    const int kb_first = g_first * 4, kb_last = min(a.nkb, g_last * 4);

    auto wait_bar = [&](uint64_t* bar, uint32_t parity) -> bool {
        if constexpr (kPair) return mbar_wait_cluster(bar, parity, wait_ns, abort_flag);
        else return mbar_wait(bar, parity, wait_ns, abort_flag);
    };
    auto arrive_leader = [&](uint64_t* bar) {
        if constexpr (kPair) mbar_arrive_cluster(mapa_u32(smem_u32(bar), 0));
        else mbar_arrive(bar);
    };
    auto drained = [&](uint64_t* bar) {
        if constexpr (kPair) mbar_arrive_relaxed(mapa_u32(smem_u32(bar), 0));
        else mbar_arrive(bar);
    };
    MmTile tl;
    bool left = false;   // this thread has arrived at the closing cluster barrier

    if (warp == 0) {
        // --------------------------------------------------------------- TMA producer
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            unsigned long long issued = 0;
            bool dead = false, waited = false;
            for (int t = unit; !dead && mm_tile<kPair>(a, start, before, t, tl); t += n_units) {
                // rows of all experts lie behind one another in the weight map; a tile that runs past its
                // expert's last row reads the next expert's, and those output columns are not stored
                const int w_row = (int)((long long)tl.group * a.cols) + tl.w_row + 128 * (int)half;
                const int x_row = tl.x_row + (kPair ? (int)half * (tl.bt >> 1) : 0);
                for (int kb = kb_first; kb < kb_last; kb += kMmStageKb) {
                    if (!mbar_wait(&S->empty[stage], phase ^ 1, wait_ns, abort_flag)) { dead = true; break; }
                    uint8_t* sw = tiles + (size_t)stage * stage_bytes;
                    uint8_t* sx = sw + kMmStageKb * kMmWBytes;
                    const bool two = kb + 1 < kb_last;
                    const uint32_t tx = kCtas * ((uint32_t)kMmWBytes + x_bytes) * (two ? 2u : 1u);
                    uint32_t bar = 0;
                    if constexpr (kPair) {
                        if (leader) mbar_expect_tx(&S->full[stage], tx);
                        bar = mapa_u32(smem_u32(&S->full[stage]), 0);
                    } else {
                        mbar_expect_tx(&S->full[stage], tx);
                    }
                    auto load = [&](uint8_t* dst, const CUtensorMap* map, int k, int row) {
                        if constexpr (kPair) tma_load_2d_pair(dst, map, k * 128, row, bar);
                        else tma_load_2d(dst, map, k * 128, row, &S->full[stage]);
                    };
                    if (!waited) {
                        grid_wait();
                        waited = true;
                    }
                    load(sw, tm_w, kb, w_row);
                    load(sx, tm_x, kb, x_row);
                    if (two) {
                        load(sw + kMmWBytes, tm_w, kb + 1, w_row);
                        load(sx + x_bytes, tm_x, kb + 1, x_row);
                    }
                    ++issued;
                    if (++stage == (uint32_t)a.n_stages) { stage = 0; phase ^= 1; }
                }
            }
            if (dead || *abort_flag) {
                if (dead) mm_raise(S, MXK_DEV_TIMEOUT_PIPE);
                // nothing may still be on its way into this shared memory when the CTA ends
                const unsigned long long n = issued < (unsigned long long)a.n_stages ? issued : (unsigned long long)a.n_stages;
                for (unsigned long long i = issued - n; leader && i < issued; ++i)
                    (void)mbar_wait(&S->full[i % a.n_stages], (uint32_t)((i / a.n_stages) & 1), 100000000ull, nullptr);
            }
        }
    } else if (warp == 1) {
        // ----------------------------------------------------------------- MMA issuer
        // The whole warp walks the loop, one elected lane issues: descriptors and barrier addresses
        // stay warp-uniform, which keeps the issue path short.  It has to be: a K block of a 256 x 208 tile is 416
        // tensor-pipe cycles, the pipe queues only a few MMAs, and every wait and commit costs this warp on the
        // order of 100 cycles.  Hence two K blocks per stage (one wait, one commit for eight MMAs) and waits at
        // CTA scope wherever a commit is what arrives (one wait at cluster scope took 290 cycles).
        if (leader) {
            uint32_t stage = 0, phase = 0, slot = 0, slot_phase = 0, it = 0;
            bool dead = false;
            const bool elected = elect_one();
            const uint64_t desc0 = umma_smem_desc_sw128(smem_u32(tiles));
            const uint32_t w_step = (uint32_t)kMmWBytes >> 4, x_step = x_bytes >> 4, desc_step = stage_bytes >> 4;
            const uint32_t n_stages = (uint32_t)a.n_stages, sf_slots = (uint32_t)a.sf_slots;
            auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity) ? 1 : 0)) return true;
                return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, wait_ns, abort_flag) ? 1 : 0) != 0;
            };
            auto mma = [&](uint32_t d, uint64_t wdesc, uint64_t xdesc, uint32_t idesc, uint32_t tsf, uint32_t acc) {
                if constexpr (kPair) umma_mxf8_pair(d, wdesc, xdesc, idesc, tsf, tsf + 4, acc);
                else umma_mxf8(d, wdesc, xdesc, idesc, tsf, tsf + 4, acc);
            };
            auto commit = [&](uint64_t* bar) {
                if constexpr (kPair) umma_commit_pair_both(smem_u32(bar));
                else umma_commit(bar);
            };
            grid_wait();   // nothing arrives before the loads do: the bounded waits shall not count the kernels before this one
            for (int t = unit; !dead && mm_tile<kPair>(a, start, before, t, tl); t += n_units, ++it) {
                const uint32_t idesc0 = umma_idesc_mx_e4m3(kPair ? 256 : 128, tl.bt, 0, 0) | a.formats;
                const uint32_t buf = it & 1u, use = it >> 1;
                const uint32_t tacc = tmem_base + buf * (uint32_t)a.bt_max;
                // the epilogue must have drained this accumulator's previous tile
                if (!__all_sync(0xFFFFFFFFu, wait_bar(&S->acc_empty[buf], (use & 1u) ^ 1u) ? 1 : 0)) { dead = true; break; }
                tc_fence_after();
                uint32_t acc = 0;
                for (int kb0 = kb_first; kb0 < kb_last; kb0 += 4) {
                    if (!warp_wait(&S->sf_full[slot], slot_phase)) { dead = true; break; }
                    const uint32_t tsf = tmem_base + (uint32_t)a.sf_col + slot * kSfSlotCols;
#pragma unroll
                    for (int i = 0; i < 4; i += kMmStageKb) {
                        if (kb0 + i >= kb_last) break;
                        if (!warp_wait(&S->full[stage], phase)) { dead = true; break; }
                        tc_fence_after();
                        const uint64_t wdesc = desc0 + (uint64_t)(stage * desc_step);
                        const uint64_t xdesc = wdesc + (uint64_t)((kMmStageKb * kMmWBytes) >> 4);
                        const uint32_t id0 = idesc0 | ((uint32_t)i << 4) | ((uint32_t)i << 29);        // scale byte i of the group
                        const uint32_t id1 = idesc0 | ((uint32_t)(i + 1) << 4) | ((uint32_t)(i + 1) << 29);
                        if (elected) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) mma(tacc, wdesc + 2 * k, xdesc + 2 * k, id0, tsf, k ? 1u : acc);
                            if (kb0 + i + 1 < kb_last) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) mma(tacc, wdesc + w_step + 2 * k, xdesc + x_step + 2 * k, id1, tsf, 1u);
                            }
                            commit(&S->empty[stage]);
                        }
                        __syncwarp();
                        acc = 1u;
                        if (++stage == n_stages) { stage = 0; phase ^= 1; }
                    }
                    if (dead) break;
                    if (elected) commit(&S->sf_empty[slot]);
                    __syncwarp();
                    if (++slot == sf_slots) { slot = 0; slot_phase ^= 1; }
                }
                if (dead) break;
                if (elected) commit(&S->acc_full[buf]);
                __syncwarp();
            }
            if (dead && elected) mm_raise(S, MXK_DEV_TIMEOUT_PIPE);
        }
    } else if (warp == 2 || warp == 3) {
        // -------------------------------------------------------- scale-tile builders
        // The two warps take the groups of four K blocks in turn.  Tile byte 16*l + 4*j + i is the
        // scale of row l + 32*j for K block i of the group (what tcgen05.cp 32x128b.warpx4 wants).
        const uint32_t mine = (uint32_t)(warp - 2);
        const bool x_words = a.x_sf && ((a.x_sf_stride | (long long)(reinterpret_cast<uintptr_t>(a.x_sf))) & 3) == 0;
        const bool w_words = a.w_sf && ((a.nkb | (int)(reinterpret_cast<uintptr_t>(a.w_sf) & 3)) & 3) == 0;
        // Four scale bytes of a row from K block kb on; 127 where there is no row (`has`) or no further block.  The word
        // form leaves the load under way: a value chosen after the load would wait for it here.
        auto load_word = [&](uint32_t& v, const uint8_t* p, bool has, int kb, bool words) {
            v = 0x7F7F7F7Fu;
            if (words && kb + 4 <= a.nkb) {
                ld_if(v, p + kb, has);
            } else if (has) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kb + i < a.nkb) v = (v & ~(0xFFu << (8 * i))) | ((uint32_t)p[kb + i] << (8 * i));
            }
        };
        constexpr int kXj = 4 * kXTiles;   // rows of an accumulator per lane
        // The loads run one group ahead of the copies, over the end of a tile too: group n of this CTA's list is group
        // n % n_groups of its tile n / n_groups.
        const int n_groups = g_last - g_first;
        const uint8_t *wsf = nullptr, *xsf = nullptr;
        int t = unit - n_units, w_here = 0, valid = 0, g = n_groups + (int)mine;   // w_here: weight rows of this CTA's half that exist
        uint32_t wx[kXj], ww[4];
        bool waited = false;
        auto load_next = [&]() -> bool {   // this warp's next group, if there is one
            bool entered = false;
            while (g >= n_groups) {
                g -= n_groups;
                t += n_units;
                entered = true;
            }
            if (entered) {
                if (!mm_tile<kPair>(a, start, before, t, tl)) return false;
                const int r0 = tl.w_row + 128 * (int)half;
                const long long plane = (long long)tl.group * a.w_sf_rows;
                if (a.w_sf) wsf = a.w_sf + (plane + (a.w_per_row ? r0 : r0 >> 7)) * a.nkb;
                if (a.x_sf) xsf = a.x_sf + (long long)tl.x_row * a.x_sf_stride;
                w_here = a.cols - r0;
                valid = tl.valid;
            }
            const int kb = (g_first + g) * 4;
            if (!waited) {
                grid_wait();
                waited = true;
            }
#pragma unroll
            for (int j = 0; j < kXj; ++j) {
                const int r = lane + 32 * j;
                load_word(wx[j], xsf + (long long)r * a.x_sf_stride, xsf && r < valid, kb, x_words);
            }
            if (!a.w_per_row) {   // a 128 x 128 block: one word for all rows
                load_word(ww[0], wsf, wsf && w_here > 0, kb, w_words);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = lane + 32 * j;
                    load_word(ww[j], wsf + (long long)r * a.nkb, wsf && r < w_here, kb, w_words);
                }
            }
            g += 2;
            return true;
        };
        bool dead = false, loaded = load_next();
        uint32_t slot = mine, par = 0;   // sf_slots is at least two
        while (loaded) {
            bool ok = true;
            if (lane == 0) ok = mbar_wait(&S->sf_empty[slot], par ^ 1u, wait_ns, abort_flag);
            ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
            if (!ok) { dead = true; break; }
            uint4* dst = reinterpret_cast<uint4*>(sf_tiles + slot * kSfSlotBytes);
            dst[lane] = a.w_per_row ? make_uint4(ww[0], ww[1], ww[2], ww[3]) : make_uint4(ww[0], ww[0], ww[0], ww[0]);
#pragma unroll
            for (int j = 0; j < kXTiles; ++j) dst[32 * (j + 1) + lane] = make_uint4(wx[4 * j], wx[4 * j + 1], wx[4 * j + 2], wx[4 * j + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            // the arrival is a release and would wait for loads under way, so it comes before them
            if (kPair && !leader && lane == 0) arrive_leader(&S->sf_peer[slot]);
            loaded = load_next();   // in flight while the copy is issued and the slot awaited
            if (leader && lane == 0) {
                const uint32_t tsf = tmem_base + (uint32_t)a.sf_col + slot * kSfSlotCols;
                const uint64_t sfdesc = umma_smem_desc_sf(smem_u32(dst));
                if constexpr (kPair) {   // one copy serves both CTAs: the partner's tile must be in place
                    ok = wait_bar(&S->sf_peer[slot], par);
                    if (ok) {
                        tc_fence_after();
#pragma unroll
                        for (int j = 0; j < kSfTiles; ++j) utccp_32x128b_warpx4_pair(tsf + 4 * j, sfdesc + (j * kMmSfTile >> 4));
                        umma_commit_pair(mapa_u32(smem_u32(&S->sf_full[slot]), 0));
                    }
                } else {
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < kSfTiles; ++j) utccp_32x128b_warpx4(tsf + 4 * j, sfdesc + (j * kMmSfTile >> 4));
                    umma_commit(&S->sf_full[slot]);
                }
            }
            ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
            if (!ok) { dead = true; break; }
            slot += 2;
            if (slot >= (uint32_t)a.sf_slots) { slot -= (uint32_t)a.sf_slots; par ^= 1u; }
        }
        if (dead && lane == 0) mm_raise(S, MXK_DEV_TIMEOUT_PIPE);
    } else {
        // ------------------------------------------------------------------- epilogue
        // Warp (q, part) reads TMEM lanes 32q .. 32q+31 (its output columns) and every second chunk of
        // 16 accumulator columns (rows of x), and stores each row's 32 columns as one 64-byte piece straight from
        // registers.  Beside the running MMAs that was faster than fewer, wider stores: 4096 x 4096 x 1024
        // 25.4 us like this, 27.6 with chunks turned round in shared memory and 16 bytes a lane, 32.0 with shuffles
        // and 4 bytes (rows off every alignment, 4095 columns: 28.0, 40.6, 29.0; all before the arrival behind them
        // stopped waiting for the stores, 23.9 like this since).
        const int q = warp & 3, part = (warp - kMmFirstEpi) >> 2;
        grid_wait();   // kernels before this one may still read what is written here
        uint32_t it = 0;
        bool dead = false;
        for (int t = unit; mm_tile<kPair>(a, start, before, t, tl); t += n_units, ++it) {
            const uint32_t buf = it & 1u, use = it >> 1;
            bool ok = true;
            if (lane == 0) ok = wait_bar(&S->acc_full[buf], use & 1u);
            ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;
            // every split has added up the previous tile's partials before they are overwritten
            if (ok && splits > 1 && it > 0) ok = mbar_wait_cluster(&S->red_free, (it - 1) & 1u, wait_ns, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok ? 1 : 0) != 0;
            if (!ok) { dead = true; break; }
            tc_fence_after();
            const int n_chunks = tl.bt >> 4;
            const uint32_t tacc = tmem_base + buf * (uint32_t)a.bt_max + ((uint32_t)(q * 32) << 16);
            // split K: row r of the tile is added up by split r % splits, into whose shared memory every split writes
            // its partial row, [split][r / splits][128]
            const int log_splits = __ffs(splits) - 1, own_rows = a.bt_max >> log_splits;
            auto push = [&](int c) {
                uint32_t v[16];
                tmem_ld16(tacc + c * 16, v);
                tmem_wait_ld();
                const uint32_t at = smem_u32(red + split * own_rows * 128 + q * 32 + lane), bar = smem_u32(&S->red_full);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int r = c * 16 + j;
                    if (r >= tl.valid) break;
                    const uint32_t owner = (uint32_t)(r & (splits - 1));
                    st_async_b32(mapa_u32(at + (uint32_t)(r >> log_splits) * 512u, owner), v[j], mapa_u32(bar, owner));
                }
            };
            if (splits > 1) {
                // what this CTA will be sent: its rows of the tile, from every split
                if (warp == kMmFirstEpi && lane == 0)
                    mbar_expect_tx(&S->red_full, (uint32_t)((tl.valid + splits - 1 - split) >> log_splits) * (uint32_t)splits * 512u);
#pragma unroll 1
                for (int c = part; c < n_chunks; c += 2) push(c);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) drained(&S->acc_empty[buf]);
            } else {
                const int col = tl.w_row + 128 * (int)half + q * 32 + lane;
                uint32_t v[16];
                if (part < n_chunks) tmem_ld16(tacc + part * 16, v);
                tmem_wait_ld();
#pragma unroll 1
                for (int c = part; c < n_chunks; c += 2) {
                    uint32_t pk[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) pk[j] = pack_bf16x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                    const bool more = c + 2 < n_chunks;
                    if (more) tmem_ld16(tacc + (c + 2) * 16, v);   // in flight while this chunk is stored
                    uint16_t* dst = a.out + (long long)(tl.x_row + c * 16) * a.out_stride + col;
                    const int n_rows = col < a.cols ? tl.valid - c * 16 : 0;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (j < n_rows) *dst = (uint16_t)(pk[j >> 1] >> (16 * (j & 1)));
                        dst += a.out_stride;
                    }
                    if (more) tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) drained(&S->acc_empty[buf]);
            }
            if (splits > 1) {
                ok = mbar_wait_cluster(&S->red_full, it & 1u, wait_ns, abort_flag);
                ok = __all_sync(0xFFFFFFFFu, ok ? 1 : 0) != 0;
                if (!ok) { dead = true; break; }
                const bool more = t + n_units < before[a.experts];
                if (!more) { cluster_arrive(); left = true; }   // nothing of this CTA touches another one's memory from here on
                const int c0 = tl.w_row + lane * 4;
                for (int r = split + splits * (warp - kMmFirstEpi); r < tl.valid; r += splits * kMmEpiWarps) {
                    const float4* part_row = reinterpret_cast<const float4*>(red + (r >> log_splits) * 128) + lane;
                    float4 sum = part_row[0];
                    for (int s = 1; s < splits; ++s) {
                        const float4 o = part_row[s * own_rows * 32];
                        sum.x += o.x; sum.y += o.y; sum.z += o.z; sum.w += o.w;
                    }
                    uint16_t* dst = a.out + (long long)(tl.x_row + r) * a.out_stride + c0;
                    const uint32_t lo = pack_bf16x2(sum.x, sum.y), hi = pack_bf16x2(sum.z, sum.w);
                    if (c0 + 4 <= a.cols && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
                        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
                    } else {
                        if (c0 < a.cols) dst[0] = (uint16_t)lo;
                        if (c0 + 1 < a.cols) dst[1] = (uint16_t)(lo >> 16);
                        if (c0 + 2 < a.cols) dst[2] = (uint16_t)hi;
                        if (c0 + 3 < a.cols) dst[3] = (uint16_t)(hi >> 16);
                    }
                }
                if (more) {
                    __syncwarp();
                    if (lane < splits) mbar_arrive_cluster(mapa_u32(smem_u32(&S->red_free), (uint32_t)lane));
                }
            }
        }
        if (dead && lane == 0) mm_raise(S, MXK_DEV_TIMEOUT_PIPE);
        if (a.zero_tail) {   // rows of no group: out was allocated for them, nothing computes them
            const int head = start[0], end = start[a.experts], n = head + a.rows - end;
            const int tid = (int)threadIdx.x - kMmFirstEpi * 32;
            for (int i = (int)blockIdx.x; i < n; i += (int)gridDim.x) {
                const long long r = i < head ? i : (long long)end + (i - head);
                for (int c = tid; c < a.cols; c += kMmEpiWarps * 32) a.out[r * a.out_stride + c] = 0;
            }
        }
    }
    // nobody leaves while a partner may still signal or write this CTA's shared memory
    tc_fence_before();
    if (clustered) {
        __syncwarp();
        if (!kPair && warp == 0) cluster_wait();   // the arrival at the start is still open
        if (!left) cluster_arrive();
        cluster_wait();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        if constexpr (kPair) tmem_dealloc_pair(tmem_base, kMmTmemCols); else tmem_dealloc(tmem_base, kMmTmemCols);
    }
}

// one CTA per tile of 128 weight rows: few rows of x, the weights' stream is all that counts
__global__ void __launch_bounds__(kMmThreads, 1)
k_matmul(const MmArgs a, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w) {
    mm_body<false>(a, &tm_x, &tm_w);
}
// a CTA pair per tile of 256 weight rows (2-CTA MMA)
__global__ void __launch_bounds__(kMmThreads, 1)
k_matmul_pair(const MmArgs a, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w) {
    mm_body<true>(a, &tm_x, &tm_w);
}
