// ============================================================================
// mxk_rows.cuh — tokens sorted by expert and back, apart from the layer.
//
// P = tokens * topk pairs, pair p = token * topk + j.  The plan gives every pair whose id lies in
// [first, first + experts) a row: rows of one expert are neighbours, in ascending pair order (the
// order of the layer's own dispatch), so the plan is the same on every run.  Everything that
// follows is a gather by the plan's tables: no atomics on data, no order that could vary.
// ============================================================================
#pragma once

constexpr int kPlanThreads = 1024;   // at most
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanClusterMax = 16;
constexpr int kPlanKeep = 4;         // ids a lane keeps in registers between the two passes
constexpr int kRowsMaxExperts = 1024;

// ---- plan -------------------------------------------------------------------------
// One cluster.  Every warp owns a contiguous slice of the pairs.  Pass 1 counts the slice per expert
// (lanes with equal ids find one another with one ballot per id bit, their lowest lane adds the count, so no two
// threads touch one counter); the counts of the warps below, of the CTAs below (read through
// distributed shared memory) and of the experts below turn into the warp's first row per expert; pass
// 2 hands the rows out.  Bound by the latency of its steps, not by bytes, so each step is one round trip: ids and
// places of a slice of up to 128 pairs stay in registers, counters are read in batches, the peers' counts are requested
// together.  Up to 1024 pairs one CTA of few warps, up to 16384 a cluster of 8 CTAs, beyond that of 16 (1024 pairs, 256
// experts: 1 CTA 6.3 us, 8 CTAs 8.3; 32768 pairs, 32 experts: 8 CTAs 10.3 us, 16 CTAs 8.3; of which a launch that
// starts under its predecessor's end hides some 2 us).  Long slices: pass 1 only needs numbers, so beyond the kept ids it adds them
// with shared-memory atomics (524288 pairs, 128 experts: 45 us, with ballots there too 60, with match.any 80).
struct PlanArgs {
    const void* idx;
    long long idx_stride;      // elements between two tokens' ids
    int idx64;
    int pairs, topk, first, experts;
    int bits;                  // 2^bits > experts: ids and the -1 of a dropped pair differ in these bits
    int per_cta, per_warp;     // pairs of a CTA and of a warp, multiples of 32
    FastDiv ftopk;
    int* row_of_pair;
    int* pair_of_row;
    int* offsets;
};

__device__ __forceinline__ int plan_id(const PlanArgs& a, int p, int end) {
    if (p >= end) return -1;
    const int t = a.ftopk.div(p), j = p - t * a.topk;
    const long long at = (long long)t * a.idx_stride + j;
    const long long e = (a.idx64 ? reinterpret_cast<const long long*>(a.idx)[at] : (long long)reinterpret_cast<const int*>(a.idx)[at]) - a.first;
    return e >= 0 && e < a.experts ? (int)e : -1;
}
__device__ __forceinline__ unsigned plan_peers(int e, int bits) {   // lanes whose id equals this lane's
    unsigned m = 0xFFFFFFFFu;
#pragma unroll
    for (int b = 0; b < 11; ++b) {
        if (b >= bits) break;
        const bool on = (e >> b) & 1;
        const unsigned v = __ballot_sync(0xFFFFFFFFu, on);
        m &= on ? v : ~v;
    }
    return m;
}
// counters of a warp, an odd distance apart
__host__ __device__ constexpr int plan_stride(int experts) { return experts | 1; }

__global__ void __launch_bounds__(kPlanThreads, 1) k_plan(const PlanArgs a) {
    grid_let_next_begin();
    extern __shared__ int plan_smem[];
    const int stride = plan_stride(a.experts);
    int* mine = plan_smem;                        // [experts] pairs of this CTA
    int* first_row = mine + stride;               // [experts] this CTA's first row
    int* wcnt = first_row + stride;               // [warps][stride]: counts, then rows handed out inside the CTA
    __shared__ int s_part[kPlanWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_ctas = (int)gridDim.x, cta = (int)blockIdx.x, n_warps = (int)blockDim.x >> 5;
    const int c_end = min(a.pairs, (cta + 1) * a.per_cta);
    const int p0 = cta * a.per_cta + warp * a.per_warp;
    const int p1 = min(c_end, p0 + a.per_warp);
    int* my = wcnt + warp * stride;

    for (int e = lane; e < a.experts; e += 32) my[e] = 0;
    grid_wait();

    int keep[kPlanKeep], rank[kPlanKeep];   // ids of the slice's first pairs, and their place among the warp's pairs of that id
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i) keep[i] = plan_id(a, p0 + i * 32 + lane, p1);
    __syncwarp();
    auto count = [&](int e) -> int {
        const unsigned m = plan_peers(e, a.bits);
        const int seen = e >= 0 ? my[e] : 0;
        __syncwarp();
        if (e >= 0 && lane == __ffs(m) - 1) my[e] = seen + __popc(m);
        __syncwarp();
        return seen + __popc(m & ((1u << lane) - 1u));
    };
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i) rank[i] = p0 + i * 32 < p1 ? count(keep[i]) : 0;
#pragma unroll 1
    for (int p = p0 + kPlanKeep * 32; p < p1; p += kPlanKeep * 32) {
        int e[kPlanKeep];
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i) e[i] = plan_id(a, p + i * 32 + lane, p1);
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i)
            if (e[i] >= 0) atomicAdd(my + e[i], 1);   // a number, whatever the order
    }
    __syncthreads();
    const int e = threadIdx.x;   // one expert per thread from here on
    int total = 0, below = 0;
    if (e < a.experts) {
        for (int w0 = 0; w0 < n_warps; w0 += 8) {   // counts of the warps below (warps are a multiple of 8)
            int v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = wcnt[(w0 + i) * stride + e];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                wcnt[(w0 + i) * stride + e] = total;
                total += v[i];
            }
        }
        mine[e] = total;
    }
    if (n_ctas > 1) {
        cluster_sync_all();
        if (e < a.experts) {
            const uint32_t at = smem_u32(mine + e);
            int v[kPlanClusterMax];
#pragma unroll
            for (int c = 0; c < kPlanClusterMax; ++c) {
                v[c] = 0;
                if (c < n_ctas) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[c]) : "r"(mapa_u32(at, (uint32_t)c)) : "memory");
            }
            total = 0;
#pragma unroll
            for (int c = 0; c < kPlanClusterMax; ++c) {
                if (c < cta) below += v[c];
                total += v[c];
            }
        }
        __syncwarp();
        cluster_arrive();   // this CTA has read its peers' counts
    }
    // exclusive sum over the experts
    int s = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= d) s += o;
    }
    if (lane == 31) s_part[warp] = s;
    __syncthreads();
    int part = lane < n_warps ? s_part[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, part, d);
        if (lane >= d) part += o;
    }
    const int all = __shfl_sync(0xFFFFFFFFu, part, 31);
    const int warps_below = __shfl_sync(0xFFFFFFFFu, part, max(warp - 1, 0));
    const int base = s - total + (warp ? warps_below : 0);
    if (e < a.experts) {
        if (cta == 0) {
            a.offsets[e] = base;
            if (e == a.experts - 1) a.offsets[a.experts] = all;
        }
        first_row[e] = base + below;
    }
    __syncthreads();
    auto put = [&](int row, int p) {
        if (p < p1) a.row_of_pair[p] = row;
        if (row >= 0) a.pair_of_row[row] = p;
    };
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i)
        if (p0 + i * 32 < p1) put(keep[i] >= 0 ? first_row[keep[i]] + my[keep[i]] + rank[i] : -1, p0 + i * 32 + lane);
    if (p0 + kPlanKeep * 32 < p1) {   // the rest is ranked again: first past the kept ones, then on
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i)
            if (keep[i] >= 0) atomicAdd(my + keep[i], 1);
        __syncwarp();
#pragma unroll 1
        for (int p = p0 + kPlanKeep * 32; p < p1; p += kPlanKeep * 32) {
            int id[kPlanKeep];
#pragma unroll
            for (int i = 0; i < kPlanKeep; ++i) id[i] = plan_id(a, p + i * 32 + lane, p1);
#pragma unroll
            for (int i = 0; i < kPlanKeep; ++i)
                if (p + i * 32 < p1) {
                    const int row = count(id[i]);
                    put(id[i] >= 0 ? first_row[id[i]] + row : -1, p + i * 32 + lane);
                }
        }
    }
    for (int r = all + cta * (int)blockDim.x + (int)threadIdx.x; r < a.pairs; r += n_ctas * (int)blockDim.x) a.pair_of_row[r] = -1;
    if (n_ctas > 1) cluster_wait();       // and they this one's
}

// ---- vectors ------------------------------------------------------------------------
template <int kBytes> struct VecOf;
template <> struct VecOf<16> { typedef uint4 T; };
template <> struct VecOf<8> { typedef uint2 T; };
template <> struct VecOf<4> { typedef uint32_t T; };
template <> struct VecOf<2> { typedef uint16_t T; };
template <> struct VecOf<1> { typedef uint8_t T; };

constexpr int kTypeBf16 = 0, kTypeFp16 = 1, kTypeFp32 = 2;
template <int kType> __device__ __forceinline__ float elem_load(const void* p) {
    if constexpr (kType == kTypeBf16) return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
    else if constexpr (kType == kTypeFp16) return __half2float(*reinterpret_cast<const __half*>(p));
    else return *reinterpret_cast<const float*>(p);
}
template <int kType> __device__ __forceinline__ void elem_store(void* p, float v) {
    if constexpr (kType == kTypeBf16) *reinterpret_cast<uint16_t*>(p) = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else if constexpr (kType == kTypeFp16) *reinterpret_cast<__half*>(p) = __float2half_rn(v);
    else *reinterpret_cast<float*>(p) = v;
}
template <int kType> __host__ __device__ constexpr int elem_bytes() { return kType == kTypeFp32 ? 4 : 2; }

// ---- the row kernels' frame -------------------------------------------------------------------
// A CTA is a tile of `tall` tokens x `wide` threads over one column part of the rows; a thread owns U vectors
// of V bytes of its token, `wide` apart.  CTAs walk the tokens with the grid's stride; the rows' numbers
// (and weights) of the next tokens are fetched into shared memory in batches, so that the only latency in the
// walk is the rows' own.  U * V is 16 bytes and more: rows whose width no wide vector divides have as many
// bytes in flight as the others.
constexpr int kRowThreads = 256;
constexpr int kRowBatch = 1024;      // table entries per batch

struct RowFrame {
    const int* row_of_pair;
    int tokens, topk, pairs;
    int row_bytes;             // of the contiguous side
    int wide, tall, part_vecs, vecs, batch;   // batch: steps of a token walk per fetch
    FastDiv fwide, ftopk;
};

template <int V, int U> struct RowCols {   // this thread's place in the tile
    int row, first;
    bool on[U];
    __device__ __forceinline__ RowCols(const RowFrame& f) {
        row = f.fwide.div((int)threadIdx.x);
        const int c = (int)threadIdx.x - row * f.wide, v0 = (int)blockIdx.y * f.part_vecs;
        first = v0 + c;
#pragma unroll
        for (int u = 0; u < U; ++u) on[u] = row < f.tall && c + u * f.wide < f.part_vecs && first + u * f.wide < f.vecs;
    }
};

// Rows (and weights) of the CTA's next `batch` steps: entry (step * tall + row) * topk + j.  A dropped pair, or a row
// out of range, is -1.
template <bool kWeights>
__device__ __forceinline__ void row_fetch(const RowFrame& f, const float* w, long long w_stride, long long step0, int* s_row, float* s_w) {
    __syncthreads();
    const int n = f.batch * f.tall * f.topk;
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
        const int q = f.ftopk.div(i), j = i - q * f.topk, step = q / f.tall;
        const long long t = ((step0 + step) * gridDim.x + blockIdx.x) * f.tall + (q - step * f.tall);
        int r = -1;
        float wt = 0.0f;
        if (t < f.tokens) {
            r = f.row_of_pair[t * f.topk + j];
            if (r < 0 || r >= f.pairs) r = -1;
            if (kWeights && r >= 0) wt = w ? w[t * w_stride + j] : 1.0f;
        }
        s_row[i] = r;
        if (kWeights) s_w[i] = wt;
    }
    __syncthreads();
}

template <int V>
__device__ __forceinline__ void clear_row(uint8_t* row, int bytes) {   // by one warp
    typedef typename VecOf<V>::T T;
    T z;
    memset(&z, 0, sizeof(z));
    for (int i = threadIdx.x & 31; i < bytes / V; i += 32) reinterpret_cast<T*>(row)[i] = z;
}

// Rows that no pair names are cleared: those behind the last expert's, and those of pairs that the caller's tables drop
// although a row was planned for them.  pair_of_row tells which: it names no pair, or one that is dropped now.  Without it
// (null) only rows behind the end are cleared.  A row behind the end counts as named where the two tables agree on it.
struct RowTables {
    const int* row_of_pair;
    const int* pair_of_row;    // or null
    const int* end;            // offsets[experts]: rows in use
    int pairs;
};
__device__ __forceinline__ long long row_looked_up(long long first, long long ctas) {   // by this thread, one of 256 from `first` on
    return first + (long long)((threadIdx.x & 31) * (kRowThreads / 32) + (threadIdx.x >> 5)) * ctas;
}
__device__ __forceinline__ int pair_of(const RowTables& a, long long r) { return a.pair_of_row && r < a.pairs ? a.pair_of_row[r] : -1; }
__device__ __forceinline__ int row_of(const RowTables& a, int p) { return p >= 0 && p < a.pairs ? a.row_of_pair[p] : -1; }
// CTA `cta` of `ctas` sees to the rows cta, cta + ctas, ...: a lane looks one of its warp's up, the warp clears what its lanes
// found.  `back` is row_of(pair_of()) of the thread's first row, asked for ahead of the CTA's work: two round trips at the end of
// every CTA cost 1 us of a sort of 128 tokens x 8 and 6 us of 110 in the gradient of 2048 tokens x 8 x 6144.
template <class Clear>
__device__ __forceinline__ void clear_unnamed(const RowTables& a, long long cta, long long ctas, int back, Clear&& clear) {
    const int end = min(max(*a.end, 0), a.pairs);
    for (long long first = cta; first < a.pairs; first += ctas * kRowThreads) {
        const long long r = row_looked_up(first, ctas);
        if (first != cta) back = row_of(a, pair_of(a, r));
        const bool named = !a.pair_of_row ? r < end : r < end ? back >= 0 && back < a.pairs : back == (int)r;
        for (unsigned m = __ballot_sync(0xFFFFFFFFu, r < a.pairs && !named); m; m &= m - 1)
            clear(first + (long long)((__ffs(m) - 1) * (kRowThreads / 32) + (int)(threadIdx.x >> 5)) * ctas);
    }
}

// ---- sort: rows[row_of_pair[p]] = x[p / topk] -----------------------------------------------
// A byte copy, so it serves every element type.  A vector of x is loaded once and stored to the token's topk rows:
// memory sees tokens * row bytes in and pairs * row bytes out.
// 4096 tokens x 8, 7168 bytes: 48 us = 5.5 TB/s; bulk copies from shared memory, wider CTAs or streaming stores ran
// within 3 % of it, a plain fill of the same bytes (no scatter, no reads) at 6.6 TB/s.
struct SortArgs {
    RowFrame f;
    const uint8_t* x;
    const uint8_t* x_sf;       // scale bytes that travel with the rows, or null
    uint8_t* rows;
    uint8_t* rows_sf;
    RowTables tables;
    long long x_stride, sf_stride;   // bytes between tokens
    int sf_bytes, sf_vec;
};

// Scales wider than this are copied in parts, so that the count over a batch of tiles stays below 2^31.
constexpr int kScalePart = 1 << 20;
static_assert((long long)kRowBatch * kScalePart + kRowThreads < (1ll << 31), "32-bit index");
template <int V>
__device__ __forceinline__ void copy_scales(const SortArgs& a, const int* s_row, long long step0) {
    typedef typename VecOf<V>::T T;
    const int all = a.sf_bytes / V, tiles = a.f.batch * a.f.tall;   // tiles <= kRowBatch
    for (int first = 0; first < all; first += kScalePart) {
        const int n = min(all - first, kScalePart);
        for (int i = threadIdx.x; i < tiles * n; i += kRowThreads) {
            const int q = i / n, at = first + i - q * n, step = q / a.f.tall;
            const long long t = ((step0 + step) * gridDim.x + blockIdx.x) * a.f.tall + (q - step * a.f.tall);
            if (t >= a.f.tokens) continue;
            const T v = *reinterpret_cast<const T*>(a.x_sf + t * a.sf_stride + (long long)at * V);
            for (int j = 0; j < a.f.topk; ++j) {
                const int r = s_row[q * a.f.topk + j];
                if (r >= 0) *reinterpret_cast<T*>(a.rows_sf + (long long)r * a.sf_bytes + (long long)at * V) = v;
            }
        }
    }
}

template <int V, int U>
__global__ void __launch_bounds__(kRowThreads) k_sort_rows(const SortArgs a) {
    grid_let_next_begin();
    typedef typename VecOf<V>::T T;
    __shared__ int s_row[kRowBatch];
    const RowFrame& f = a.f;
    const RowCols<V, U> c(f);
    const long long steps = (f.tokens + (long long)gridDim.x * f.tall - 1) / ((long long)gridDim.x * f.tall);
    const long long cta = (long long)blockIdx.y * gridDim.x + blockIdx.x, ctas = (long long)gridDim.x * gridDim.y;
    grid_wait();
    const int pair = pair_of(a.tables, row_looked_up(cta, ctas));
    int back = -1;
    for (long long step0 = 0; step0 < steps; step0 += f.batch) {
        row_fetch<false>(f, nullptr, 0, step0, s_row, nullptr);
        if (step0 == 0) back = row_of(a.tables, pair);
        const int here = (int)min((long long)f.batch, steps - step0);
        for (int s = 0; s < here; ++s) {
            const long long t = ((step0 + s) * gridDim.x + blockIdx.x) * f.tall + c.row;
            if (t >= f.tokens || !c.on[0]) break;
            T v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c.on[u]) v[u] = reinterpret_cast<const T*>(a.x + t * a.x_stride)[c.first + u * f.wide];
            const int* rp = s_row + (s * f.tall + c.row) * f.topk;
            for (int j = 0; j < f.topk; ++j) {
                const int r = rp[j];
                if (r < 0) continue;
                T* dst = reinterpret_cast<T*>(a.rows + (long long)r * f.row_bytes) + c.first;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (c.on[u]) dst[u * f.wide] = v[u];
            }
        }
        if (a.x_sf && blockIdx.y == 0) {
            switch (a.sf_vec) {
                case 16: copy_scales<16>(a, s_row, step0); break;
                case 8: copy_scales<8>(a, s_row, step0); break;
                case 4: copy_scales<4>(a, s_row, step0); break;
                default: copy_scales<1>(a, s_row, step0); break;
            }
        }
    }
    clear_unnamed(a.tables, cta, ctas, back, [&](long long r) {
        clear_row<V>(a.rows + r * f.row_bytes, f.row_bytes);
        if (a.x_sf) clear_row<1>(a.rows_sf + r * a.sf_bytes, a.sf_bytes);
    });
}

// ---- unsort: y[t] = sum_j w[t, j] rows[row_of_pair[t, j]] ------------------------------------
// j ascending, FP32, one rounding at the end.  A thread has its vectors of up to eight of the token's rows in
// flight; memory sees pairs * row bytes in, tokens * row bytes out.
// 4096 tokens x 8, 7168 bf16: 85 us = 6.2 TB/s (249 us with the rows' numbers loaded in front of every vector).
struct UnsortArgs {
    RowFrame f;
    const uint8_t* rows;
    const float* w;            // [tokens][topk] or null (all one)
    uint8_t* y;
    long long rows_stride, w_stride;   // bytes between rows; floats between tokens
};

template <int kType, int V, int U>
__global__ void __launch_bounds__(kRowThreads, 4) k_unsort_rows(const UnsortArgs a) {
    grid_let_next_begin();
    constexpr int kEl = elem_bytes<kType>(), kN = V / kEl;
    typedef typename VecOf<V>::T T;
    __shared__ int s_row[kRowBatch];
    __shared__ float s_w[kRowBatch];
    const RowFrame& f = a.f;
    const RowCols<V, U> c(f);
    const long long steps = (f.tokens + (long long)gridDim.x * f.tall - 1) / ((long long)gridDim.x * f.tall);
    grid_wait();
    for (long long step0 = 0; step0 < steps; step0 += f.batch) {
        row_fetch<true>(f, a.w, a.w_stride, step0, s_row, s_w);
        const int here = (int)min((long long)f.batch, steps - step0);
        for (int s = 0; s < here; ++s) {
            const long long t = ((step0 + s) * gridDim.x + blockIdx.x) * f.tall + c.row;
            if (t >= f.tokens || !c.on[0]) break;
            const int at = (s * f.tall + c.row) * f.topk;
            float acc[U][kN];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < kN; ++i) acc[u][i] = 0.0f;
            for (int j0 = 0; j0 < f.topk; j0 += 8) {
                T v[8][U];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int r = j0 + j < f.topk ? s_row[at + j0 + j] : -1;
                    memset(&v[j], 0, sizeof(v[j]));     // a dropped pair adds nothing, whatever its row holds
                    if (r >= 0) {
                        const T* src = reinterpret_cast<const T*>(a.rows + (long long)r * a.rows_stride) + c.first;
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (c.on[u]) v[j][u] = src[u * f.wide];
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float w = j0 + j < f.topk ? s_w[at + j0 + j] : 0.0f;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int i = 0; i < kN; ++i)
                            acc[u][i] = fmaf(w, elem_load<kType>(reinterpret_cast<const uint8_t*>(&v[j][u]) + i * kEl), acc[u][i]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                T o;
#pragma unroll
                for (int i = 0; i < kN; ++i) elem_store<kType>(reinterpret_cast<uint8_t*>(&o) + i * kEl, acc[u][i]);
                if (c.on[u]) reinterpret_cast<T*>(a.y + t * f.row_bytes)[c.first + u * f.wide] = o;
            }
        }
    }
}

// ---- gradient of the weighted unsort -----------------------------------------------------------
// drows[row(t, j)] = w[t, j] dy[t], 0 in rows that no pair names;  dw[t, j] = <dy[t], rows[row(t, j)]>.  A team of 1, 2, 4 or 8 warps (by the row's
// width) takes one token.  dy is read once per eight pairs, the eight rows' vectors are requested together; a dot is
// summed per lane, over the warp, over the team, always in that order.
// 2048 tokens x 8, 6144 bf16: 69 us = 6.2 TB/s; with the loads one after the other 92 us, and with the 64 registers that
// four CTAs per SM leave (spills) 120 us: two CTAs with everything in registers keep enough bytes in flight.
struct UnsortGradArgs {
    const uint8_t* dy;
    const uint8_t* rows;       // needed for dw only
    const float* w;
    uint8_t* drows;            // or null
    float* dw;                 // [tokens][topk] or null
    RowTables tables;
    long long dy_stride, rows_stride, w_stride;
    int row_bytes;             // of drows (contiguous)
    int tokens, topk, vecs, team;
};

template <int kType, int V, bool kRows, bool kDots>
__global__ void __launch_bounds__(kRowThreads, 2) k_unsort_grad(const UnsortGradArgs a) {
    grid_let_next_begin();
    grid_wait();
    constexpr int kEl = elem_bytes<kType>(), kN = V / kEl;
    typedef typename VecOf<V>::T T;
    __shared__ float s_dot[2][8][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int teams = 8 / a.team, team = warp / a.team, member = warp - team * a.team;
    const int step = a.team * 32;
    const long long t = (long long)blockIdx.x * teams + team;
    int pair = -1, back = -1;
    if constexpr (kRows) {
        pair = pair_of(a.tables, row_looked_up(blockIdx.x, gridDim.x));
        if (t >= a.tokens) back = row_of(a.tables, pair);
    }
    if (t < a.tokens) {
        const int* rp = a.tables.row_of_pair + t * a.topk;
        const uint8_t* dy = a.dy + t * a.dy_stride;
        for (int j0 = 0, turn = 0; j0 < a.topk; j0 += 8, turn ^= 1) {
            int r[8];
            float w[8], dot[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                r[j] = j0 + j < a.topk ? rp[j0 + j] : -1;
                dot[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (r[j] >= a.tables.pairs) r[j] = -1;
                w[j] = r[j] >= 0 ? a.w[t * a.w_stride + j0 + j] : 0.0f;
            }
            if (kRows && j0 == 0) back = row_of(a.tables, pair);
            for (int i = member * 32 + lane; i < a.vecs; i += step) {
                const long long at = (long long)i * V;
                const T g = *reinterpret_cast<const T*>(dy + at);
                T v[8];
                if constexpr (kDots) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        memset(&v[j], 0, sizeof(T));
                        if (r[j] >= 0) v[j] = *reinterpret_cast<const T*>(a.rows + (long long)r[j] * a.rows_stride + at);
                    }
                }
                float gf[kN];
#pragma unroll
                for (int k = 0; k < kN; ++k) gf[k] = elem_load<kType>(reinterpret_cast<const uint8_t*>(&g) + k * kEl);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (kRows && r[j] >= 0) {
                        T o;
#pragma unroll
                        for (int k = 0; k < kN; ++k) elem_store<kType>(reinterpret_cast<uint8_t*>(&o) + k * kEl, w[j] * gf[k]);
                        *reinterpret_cast<T*>(a.drows + (long long)r[j] * a.row_bytes + at) = o;
                    }
                    if constexpr (kDots) {
#pragma unroll
                        for (int k = 0; k < kN; ++k)
                            dot[j] = fmaf(gf[k], elem_load<kType>(reinterpret_cast<const uint8_t*>(&v[j]) + k * kEl), dot[j]);
                    }
                }
            }
            if constexpr (kDots) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], d);
                    if (lane == 0) s_dot[turn][warp][j] = dot[j];
                }
                // one barrier per eight pairs: the next eight use the other copy of the partial sums
                if (a.team > 1) asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + team), "r"(step) : "memory");
                else __syncwarp();
                if (member == 0 && lane < 8 && j0 + lane < a.topk) {
                    float sum = s_dot[turn][warp][lane];
                    for (int k = 1; k < a.team; ++k) sum += s_dot[turn][warp + k][lane];
                    const int own = rp[j0 + lane];
                    a.dw[t * a.topk + j0 + lane] = own >= 0 && own < a.tables.pairs ? sum : 0.0f;   // a dropped pair has no gradient, whatever dy holds
                }
            }
        }
    }
    if constexpr (kRows) {
        clear_unnamed(a.tables, blockIdx.x, gridDim.x, back, [&](long long r) { clear_row<V>(a.drows + r * a.row_bytes, a.row_bytes); });
    }
}
