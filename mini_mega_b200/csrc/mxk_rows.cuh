// ============================================================================
// mxk_rows.cuh — tokens sorted by expert and back, apart from the layer.
//
// P = tokens * topk pairs, pair p = token * topk + j.  The plan gives every pair whose id lies in
// [first, first + experts) a row: rows of one expert are neighbours, in ascending pair order (the
// order of the layer's own dispatch), so the plan is the same on every run.  Everything that
// follows is a gather by the plan's tables: no atomics on data, no order that could vary.
// ============================================================================
#pragma once

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanClusterMax = 8;
constexpr int kPlanKeep = 4;         // ids a lane keeps in registers between the two passes
constexpr int kRowsMaxExperts = 1024;

// ---- plan -------------------------------------------------------------------------
// One cluster.  Every warp owns a contiguous slice of the pairs.  Pass 1 counts the slice per expert
// (lanes with equal ids find one another with match.any, their lowest lane adds the count, so no two
// threads touch one counter); the counts of the warps below, of the CTAs below (read through
// distributed shared memory) and of the experts below turn into the warp's first row per expert; pass
// 2 walks the slice again and hands the rows out.
struct PlanArgs {
    const void* idx;
    long long idx_stride;      // elements between two tokens' ids
    int idx64;
    int pairs, topk, first, experts;
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

__global__ void __launch_bounds__(kPlanThreads, 1) k_plan(const PlanArgs a) {
    extern __shared__ int plan_smem[];
    int* mine = plan_smem;                        // [experts] pairs of this CTA
    int* wcnt = mine + a.experts;                 // [warps][experts]: counts, then next rows
    __shared__ int s_part[kPlanWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_ctas = (int)gridDim.x, cta = (int)blockIdx.x;
    const int c_end = min(a.pairs, (cta + 1) * a.per_cta);
    const int p0 = cta * a.per_cta + warp * a.per_warp;
    const int p1 = min(c_end, p0 + a.per_warp);
    int* my = wcnt + warp * a.experts;
    for (int e = lane; e < a.experts; e += 32) my[e] = 0;
    __syncwarp();

    int keep[kPlanKeep];
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i) keep[i] = plan_id(a, p0 + i * 32 + lane, p1);
    auto count = [&](int e) {
        const unsigned m = __match_any_sync(0xFFFFFFFFu, e);
        if (e >= 0 && lane == __ffs(m) - 1) my[e] += __popc(m);
        __syncwarp();
    };
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i)
        if (p0 + i * 32 < p1) count(keep[i]);
    for (int p = p0 + kPlanKeep * 32; p < p1; p += kPlanKeep * 32) {
        int e[kPlanKeep];
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i) e[i] = plan_id(a, p + i * 32 + lane, p1);
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i)
            if (p + i * 32 < p1) count(e[i]);
    }
    __syncthreads();
    const int e = threadIdx.x;
    int total = 0;
    if (e < a.experts) {
        for (int w = 0; w < kPlanWarps; ++w) {   // counts of the warps below
            const int v = wcnt[w * a.experts + e];
            wcnt[w * a.experts + e] = total;
            total += v;
        }
        mine[e] = total;
    }
    int below = 0;
    if (n_ctas > 1) {
        cluster_sync_all();
        if (e < a.experts) {
            const uint32_t at = smem_u32(mine + e);
            total = 0;
            for (int c = 0; c < n_ctas; ++c) {
                int v;
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(at, (uint32_t)c)) : "memory");
                if (c < cta) below += v;
                total += v;
            }
        }
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
    int base = s - total, all = 0;
    for (int w = 0; w < kPlanWarps; ++w) {
        const int v = s_part[w];
        if (w < warp) base += v;
        all += v;
    }
    if (e < a.experts) {
        if (cta == 0) {
            a.offsets[e] = base;
            if (e == a.experts - 1) a.offsets[a.experts] = all;
        }
        base += below;
        for (int w = 0; w < kPlanWarps; ++w) wcnt[w * a.experts + e] += base;
    }
    __syncthreads();
    auto place = [&](int e_, int p) {
        const unsigned m = __match_any_sync(0xFFFFFFFFu, e_);
        const int row = e_ >= 0 ? my[e_] + __popc(m & ((1u << lane) - 1u)) : -1;
        __syncwarp();
        if (e_ >= 0 && lane == __ffs(m) - 1) my[e_] += __popc(m);
        __syncwarp();
        if (p < p1) a.row_of_pair[p] = row;
        if (row >= 0) a.pair_of_row[row] = p;
    };
#pragma unroll
    for (int i = 0; i < kPlanKeep; ++i)
        if (p0 + i * 32 < p1) place(keep[i], p0 + i * 32 + lane);
    for (int p = p0 + kPlanKeep * 32; p < p1; p += kPlanKeep * 32) {
        int id[kPlanKeep];
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i) id[i] = plan_id(a, p + i * 32 + lane, p1);
#pragma unroll
        for (int i = 0; i < kPlanKeep; ++i)
            if (p + i * 32 < p1) place(id[i], p + i * 32 + lane);
    }
    for (int r = all + cta * kPlanThreads + (int)threadIdx.x; r < a.pairs; r += n_ctas * kPlanThreads) a.pair_of_row[r] = -1;
    if (n_ctas > 1) cluster_sync_all();   // the peers have read this CTA's counts
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

// ---- sort: rows[row_of_pair[p]] = x[p / topk] -----------------------------------------------
// A byte copy, so it serves every element type.  A CTA takes `span` tokens (or a column part of one
// token when tokens are few): a thread loads its vector of x ONCE and stores it to the token's topk
// rows, so memory sees tokens * row bytes in and pairs * row bytes out.
struct SortArgs {
    const uint8_t* x;
    const uint8_t* x_sf;       // scale bytes that travel with the rows, or null
    uint8_t* rows;
    uint8_t* rows_sf;
    const int* row_of_pair;
    const int* end;            // offsets[experts]: rows in use
    long long x_stride, sf_stride;   // bytes between tokens
    int row_bytes, sf_bytes, sf_vec;
    int tokens, topk, pairs, span, vecs, part_vecs;
    FastDiv fvecs;
};

template <int V>
__device__ __forceinline__ void copy_part(const uint8_t* src, uint8_t* dst, const int* row_of_pair, int topk, int pairs, int row_bytes, int at) {
    typedef typename VecOf<V>::T T;
    const T v = *reinterpret_cast<const T*>(src + (long long)at * V);
    for (int j = 0; j < topk; ++j) {
        const int r = row_of_pair[j];
        if (r >= 0 && r < pairs) *reinterpret_cast<T*>(dst + (long long)r * row_bytes + (long long)at * V) = v;
    }
}
template <int V>
__device__ __forceinline__ void clear_row(uint8_t* row, int bytes) {
    typedef typename VecOf<V>::T T;
    T z;
    memset(&z, 0, sizeof(z));
    for (int i = threadIdx.x; i < bytes / V; i += blockDim.x) reinterpret_cast<T*>(row)[i] = z;
}

template <int V>
__global__ void __launch_bounds__(256) k_sort_rows(const SortArgs a) {
    const int t0 = (int)blockIdx.x * a.span;
    const int n_tok = min(a.span, a.tokens - t0);
    const int v0 = (int)blockIdx.y * a.part_vecs, vn = min(a.part_vecs, a.vecs - v0);
    for (int i = threadIdx.x; i < n_tok * vn; i += blockDim.x) {
        const int dt = a.span == 1 ? 0 : a.fvecs.div(i);   // several tokens per CTA only with whole rows
        const int t = t0 + dt, at = v0 + i - dt * vn;
        copy_part<V>(a.x + (long long)t * a.x_stride, a.rows, a.row_of_pair + (long long)t * a.topk, a.topk, a.pairs, a.row_bytes, at);
    }
    if (a.x_sf && blockIdx.y == 0) {
        const int n = a.sf_bytes / a.sf_vec;
        for (int i = threadIdx.x; i < n_tok * n; i += blockDim.x) {
            const int dt = i / n, t = t0 + dt, at = i - dt * n;
            const uint8_t* src = a.x_sf + (long long)t * a.sf_stride;
            const int* rp = a.row_of_pair + (long long)t * a.topk;
            switch (a.sf_vec) {
                case 16: copy_part<16>(src, a.rows_sf, rp, a.topk, a.pairs, a.sf_bytes, at); break;
                case 8: copy_part<8>(src, a.rows_sf, rp, a.topk, a.pairs, a.sf_bytes, at); break;
                case 4: copy_part<4>(src, a.rows_sf, rp, a.topk, a.pairs, a.sf_bytes, at); break;
                default: copy_part<1>(src, a.rows_sf, rp, a.topk, a.pairs, a.sf_bytes, at); break;
            }
        }
    }
    // rows behind the last expert's
    const int end = min(max(*a.end, 0), a.pairs);
    for (long long r = end + (long long)blockIdx.y * gridDim.x + blockIdx.x; r < a.pairs; r += (long long)gridDim.x * gridDim.y) {
        clear_row<V>(a.rows + r * a.row_bytes, a.row_bytes);
        if (a.x_sf) clear_row<1>(a.rows_sf + r * a.sf_bytes, a.sf_bytes);
    }
}

// ---- unsort: y[t] = sum_j w[t, j] rows[row_of_pair[t, j]] ------------------------------------
// j ascending, FP32, one rounding at the end.  A thread owns one vector of columns of one token and
// has up to eight of the token's rows in flight; memory sees pairs * row bytes in, tokens * row bytes out.
struct UnsortArgs {
    const uint8_t* rows;
    const float* w;            // [tokens][topk] or null (all one)
    uint8_t* y;
    const int* row_of_pair;
    long long rows_stride, w_stride;   // bytes between rows; floats between tokens
    int row_bytes;             // of y (contiguous)
    int tokens, topk, pairs, span, vecs, part_vecs;
    FastDiv fvecs;
};

template <int kType, int V>
__global__ void __launch_bounds__(256, 4) k_unsort_rows(const UnsortArgs a) {
    constexpr int kEl = elem_bytes<kType>(), kN = V / kEl;
    typedef typename VecOf<V>::T T;
    const int t0 = (int)blockIdx.x * a.span;
    const int n_tok = min(a.span, a.tokens - t0);
    const int v0 = (int)blockIdx.y * a.part_vecs, vn = min(a.part_vecs, a.vecs - v0);
    for (int i = threadIdx.x; i < n_tok * vn; i += blockDim.x) {
        const int dt = a.span == 1 ? 0 : a.fvecs.div(i);
        const long long t = t0 + dt;
        const long long at = (long long)(v0 + i - dt * vn) * V;
        const int* rp = a.row_of_pair + t * a.topk;
        float acc[kN];
#pragma unroll
        for (int c = 0; c < kN; ++c) acc[c] = 0.0f;
        for (int j0 = 0; j0 < a.topk; j0 += 8) {
            T v[8];
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = j0 + j < a.topk ? __ldg(rp + j0 + j) : -1;
                const bool ok = r >= 0 && r < a.pairs;
                w[j] = ok ? (a.w ? __ldg(a.w + t * a.w_stride + j0 + j) : 1.0f) : 0.0f;
                memset(&v[j], 0, sizeof(T));     // a dropped pair adds nothing, whatever its row holds
                if (ok) v[j] = __ldg(reinterpret_cast<const T*>(a.rows + (long long)r * a.rows_stride + at));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < kN; ++c)
                    acc[c] = fmaf(w[j], elem_load<kType>(reinterpret_cast<const uint8_t*>(&v[j]) + c * kEl), acc[c]);
        }
        T o;
#pragma unroll
        for (int c = 0; c < kN; ++c) elem_store<kType>(reinterpret_cast<uint8_t*>(&o) + c * kEl, acc[c]);
        *reinterpret_cast<T*>(a.y + t * a.row_bytes + at) = o;
    }
}

// ---- gradient of the weighted unsort -----------------------------------------------------------
// drows[row(t, j)] = w[t, j] dy[t];  dw[t, j] = <dy[t], rows[row(t, j)]>.  One CTA per token: dy is read
// once per eight pairs, the dots are summed per thread, then over the CTA in a fixed order.
struct UnsortGradArgs {
    const uint8_t* dy;
    const uint8_t* rows;       // needed for dw only
    const float* w;
    uint8_t* drows;            // or null
    float* dw;                 // [tokens][topk] or null
    const int* row_of_pair;
    const int* end;
    long long dy_stride, rows_stride, w_stride;
    int row_bytes;             // of drows (contiguous)
    int tokens, topk, pairs, vecs;
};

template <int kType, int V>
__global__ void __launch_bounds__(256) k_unsort_grad(const UnsortGradArgs a) {
    constexpr int kEl = elem_bytes<kType>(), kN = V / kEl;
    typedef typename VecOf<V>::T T;
    __shared__ float s_dot[8][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
    for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const int* rp = a.row_of_pair + t * a.topk;
        const uint8_t* dy = a.dy + t * a.dy_stride;
        for (int j0 = 0; j0 < a.topk; j0 += 8) {
            int r[8];
            float w[8], dot[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                r[j] = j0 + j < a.topk ? rp[j0 + j] : -1;
                if (r[j] >= a.pairs) r[j] = -1;
                w[j] = r[j] >= 0 ? a.w[t * a.w_stride + j0 + j] : 0.0f;
                dot[j] = 0.0f;
            }
            for (int i = threadIdx.x; i < a.vecs; i += blockDim.x) {
                const long long at = (long long)i * V;
                const T g = *reinterpret_cast<const T*>(dy + at);
                float gf[kN];
#pragma unroll
                for (int c = 0; c < kN; ++c) gf[c] = elem_load<kType>(reinterpret_cast<const uint8_t*>(&g) + c * kEl);
                if (a.dw) {
                    T v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        memset(&v[j], 0, sizeof(T));
                        if (r[j] >= 0) v[j] = *reinterpret_cast<const T*>(a.rows + (long long)r[j] * a.rows_stride + at);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int c = 0; c < kN; ++c)
                            dot[j] = fmaf(gf[c], elem_load<kType>(reinterpret_cast<const uint8_t*>(&v[j]) + c * kEl), dot[j]);
                }
                if (a.drows) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (r[j] >= 0) {
                            T o;
#pragma unroll
                            for (int c = 0; c < kN; ++c) elem_store<kType>(reinterpret_cast<uint8_t*>(&o) + c * kEl, w[j] * gf[c]);
                            *reinterpret_cast<T*>(a.drows + (long long)r[j] * a.row_bytes + at) = o;
                        }
                }
            }
            if (a.dw) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], d);
                    if (lane == 0) s_dot[j][warp] = dot[j];
                }
                __syncthreads();
                if (threadIdx.x < 8 && j0 + (int)threadIdx.x < a.topk) {
                    const int rr = rp[j0 + threadIdx.x];
                    float sum = 0.0f;
                    for (int k = 0; k < n_warps; ++k) sum += s_dot[threadIdx.x][k];
                    // a dropped pair has no gradient, whatever dy holds
                    a.dw[t * a.topk + j0 + threadIdx.x] = rr >= 0 && rr < a.pairs ? sum : 0.0f;
                }
                __syncthreads();
            }
        }
    }
    if (a.drows) {
        const int end = min(max(*a.end, 0), a.pairs);
        for (long long r = end + (long long)blockIdx.x; r < a.pairs; r += gridDim.x) clear_row<V>(a.drows + r * a.row_bytes, a.row_bytes);
    }
}
