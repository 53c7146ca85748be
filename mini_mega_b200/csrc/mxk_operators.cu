// ============================================================================
// mxk_operators.cu — operators beside the layer, behind the C ABI of include/mxk_b200.h: tokens
// sorted by expert and back with their gradients (mxk_rows.cuh), 8-bit products with block scales,
// dense and grouped by expert (mxk_matmul.cuh).
// ============================================================================
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/mxk_b200.h"
#include "mxk_device.cuh"

// mxk_last_error()'s message of this thread (mxk_kernels.cu)
__attribute__((visibility("hidden"))) int mxk_set_error(int code, const std::string& msg);

namespace {

using namespace mxk;

#include "mxk_rows.cuh"
#include "mxk_matmul.cuh"

constexpr int kSms = 148;

int fail(int code, const std::string& msg) { return mxk_set_error(code, msg); }
int cuda_fail(cudaError_t e, const char* what) { return mxk_set_error((int)e, std::string(what) + ": " + cudaGetErrorString(e)); }

// Every launch allows its kernel to begin while the one before it in the stream ends (grid_wait in the kernels).
template <class... K, class... A>
cudaError_t launch(void (*kernel)(K...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads, 1, 1); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[2];
    std::memset(at, 0, sizeof(at));
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
int launched(cudaError_t e, const char* what) { return e == cudaSuccess ? 0 : cuda_fail(e, what); }

// Largest power of two up to 16 that divides every given address, stride and length (in bytes).
int common_vec(uint64_t bits) {
    bits |= 16;
    return (int)(bits & (~bits + 1));
}
uint64_t addr(const void* p) { return (uint64_t)reinterpret_cast<uintptr_t>(p); }
template <class... P> bool words(const P*... p) { return ((0 | ... | addr(p)) & 3) == 0; }   // tables and FP32 factors on 4-byte addresses

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device.
int allow_smem(const void* fn, int slot, int bytes) {
    static thread_local uint64_t done[3] = {0, 0, 0};   // bit = device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
    if (dev < 64 && (done[slot] >> dev) & 1) return 0;
    int major = 0;
    if ((e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev)) != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    if (major != 10) return fail(MXK_ERR_DEVICE, "the operators run on sm_100 devices only");
    if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    if (dev < 64) done[slot] |= 1ull << dev;
    return 0;
}

// Whether a cluster of 16 plan CTAs can run on the current device (more than the portable 8: asked once).
bool sixteen_fit(int smem) {
    static thread_local uint64_t asked = 0, fits = 0;   // bit = device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
    if (!((asked >> dev) & 1)) {
        cudaLaunchConfig_t cfg;
        std::memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(16, 1, 1); cfg.blockDim = dim3(kPlanThreads, 1, 1); cfg.dynamicSmemBytes = (size_t)smem;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = 16; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
        cfg.attrs = &at; cfg.numAttrs = 1;
        int n = 0;
        const bool ok = cudaFuncSetAttribute((const void*)k_plan, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&n, k_plan, &cfg) == cudaSuccess && n >= 1;
        if (!ok) (void)cudaGetLastError();
        if (ok) fits |= 1ull << dev;
        asked |= 1ull << dev;
    }
    return (fits >> dev) & 1;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}
// bytes [rows][k] with `stride` bytes between rows, tiles of box_rows x 128 bytes, 128-byte swizzle, zero outside
int byte_map(CUtensorMap* m, const void* base, int64_t rows, int64_t k, int64_t stride, int box_rows) {
    const EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(MXK_ERR_NO_DRIVER, "cuTensorMapEncodeTiled not available from the CUDA driver");
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : fail(MXK_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled failed, CUresult " + std::to_string((int)r));
}

// Tile of the row kernels: column parts of at most 256 threads x u vectors, as many tokens beside one another
// as fit the CTA; with few tokens, more and narrower parts, so that every SM has some.
dim3 row_frame(RowFrame& f, int tokens, int topk, int row_bytes, int vec, int u, const int32_t* row_of_pair) {
    f.row_of_pair = row_of_pair;
    f.tokens = tokens; f.topk = topk; f.pairs = tokens * topk; f.row_bytes = row_bytes;
    f.vecs = row_bytes / vec;
    const int most = kRowThreads * u;
    int parts = (f.vecs + most - 1) / most;
    if ((int64_t)tokens * parts < 2 * kSms) parts = std::min<int64_t>((f.vecs + 32 * u - 1) / (32 * u), (2 * kSms + tokens - 1) / tokens);
    parts = std::min(std::max(parts, (f.vecs + most - 1) / most), 65535);
    // a part is `wide` threads x u vectors; rows so wide that 65535 parts do not cover them are refused by the callers
    f.wide = (f.vecs + parts * u - 1) / (parts * u);
    f.part_vecs = f.wide * u;
    parts = (f.vecs + f.part_vecs - 1) / f.part_vecs;
    f.tall = std::max(1, std::min(kRowThreads / f.wide, kRowBatch / topk));
    f.tall = (int)std::min<int64_t>(f.tall, std::max<int64_t>(1, (tokens * (int64_t)parts + 2 * kSms - 1) / (2 * kSms)));
    f.batch = std::max(1, kRowBatch / (f.tall * topk));
    f.fwide = FastDiv::make((uint32_t)f.wide); f.ftopk = FastDiv::make((uint32_t)topk);
    const int64_t columns = (tokens + f.tall - 1) / f.tall, resident = std::max<int64_t>(1, kSms * 8 / parts);
    const int grid = (int)std::min(columns, resident);
    f.batch = (int)std::min<int64_t>(f.batch, (columns + grid - 1) / grid);
    return dim3((unsigned)grid, (unsigned)parts, 1);
}
constexpr int kMaxRowBytes = 1 << 24;

int bad_tables(int64_t tokens, int topk) { return tokens < 0 || topk < 1 || topk > 256 || tokens * topk > (1 << 30); }

template <int kType>
int unsort_launch(const UnsortArgs& a, int vec, dim3 grid, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    switch (vec) {
        case 16: e = launch(k_unsort_rows<kType, 16, 1>, grid, kRowThreads, 0, 1, st, a); break;
        case 8: e = launch(k_unsort_rows<kType, 8, 2>, grid, kRowThreads, 0, 1, st, a); break;
        case 4: e = launch(k_unsort_rows<kType, 4, 4>, grid, kRowThreads, 0, 1, st, a); break;
        default:
            if constexpr (kType != kTypeFp32) e = launch(k_unsort_rows<kType, 2, 4>, grid, kRowThreads, 0, 1, st, a);
    }
    return launched(e, "launch k_unsort_rows");
}
template <int kType, int V>
int unsort_grad_vec(const UnsortGradArgs& a, int grid, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    if (a.drows && a.dw) e = launch(k_unsort_grad<kType, V, true, true>, grid, kRowThreads, 0, 1, st, a);
    else if (a.drows) e = launch(k_unsort_grad<kType, V, true, false>, grid, kRowThreads, 0, 1, st, a);
    else e = launch(k_unsort_grad<kType, V, false, true>, grid, kRowThreads, 0, 1, st, a);
    return launched(e, "launch k_unsort_grad");
}
template <int kType>
int unsort_grad_launch(const UnsortGradArgs& a, int vec, int grid, cudaStream_t st) {
    switch (vec) {
        case 16: return unsort_grad_vec<kType, 16>(a, grid, st);
        case 8: return unsort_grad_vec<kType, 8>(a, grid, st);
        case 4: return unsort_grad_vec<kType, 4>(a, grid, st);
        default: return unsort_grad_vec<kType, kType == kTypeFp32 ? 4 : 2>(a, grid, st);
    }
}
int unroll_of(int vec) { return vec >= 16 ? 1 : vec == 8 ? 2 : 4; }

// How a product is cut: CTA pairs or single CTAs, rows of x per tile, CTAs that share a tile's K extent.  The cut
// with the least estimated time, from the parts that were measured on a B200 (us, launches back to back; K blocks of 128;
// `full`: the part of the GPU that has a tile):
//   start and end                     single 3.5 + full (0.6 + 0.014 x rows of x in a tile), pair 5.0 + 0.022 x rows x full
//   one K block of a tile             single 153 ns + 0.64 ns x rows (32 rows: 173, 64: 195, 128: 234), pair 145 ns +
//                                     0.6 ns x rows (128 rows: 230, 192: 267, 224: 279)
//   a further round of tiles          0.25
//   partial sums between splits       0.8 + full (1.1 + 0.018 x rows)
// and, for grouped products only, the operands' way from memory (6.3 TB/s) and, for every tile of rows after a group's first,
// its weights' way from L2 once more (12 TB/s).  Both sides, measured: 1 x 4096 x 6144 in 1 / 2 / 4 splits 11.3 / 8.7 / 8.0 us; 16 x 1024 x 2048 6.3 / 6.5 / 5.5;
// 128 x 4096 x 7168 tiles of 64 rows in 2 splits 12.2, of 32 rows unsplit 13.6; 512 x 4096 x 7168 single 17.5, pairs 20.1;
// 2048 x 4096 x 7168 single 57, pairs 52; 32 groups of 200 rows x 4096 x 7168 pairs with one tile a group 192, with two 282,
// single CTAs with two 252.  Splits only while every tile is expected to run at once (unevenly loaded groups can have more
// tiles than their mean tells: some clusters then take a second one): a second round costs 7 us (20 groups of 40 rows x
// 1000 x 2992: 21 us without splits, 24 in two, 45 in four), and 8 of them only for a few tiles, because few clusters of
// eight fit the GPU at once (1 x 2048 x 6144: 14.3 us, in four 8.8).
struct MmShape { bool pair; int bt, splits; };
MmShape mm_shape(int64_t rows, int64_t cols, int64_t depth, int64_t experts, bool grouped) {
    const int nkb = (int)((depth + 127) / 128), k_groups = (nkb + 3) / 4;
    double mean = (double)rows / (double)experts;
    if (grouped) mean = std::max(48.0, mean + 1.5 * std::sqrt(mean));   // groups differ in size: most shall fit one tile
    const int64_t n = std::max<int64_t>(1, (int64_t)std::ceil(mean)), groups = std::min(experts, rows);
    const double weights = (double)groups * (double)cols * (double)depth;
    const double memory = (weights + (double)rows * (double)depth + 2.0 * (double)rows * (double)cols) / 6.3e6;
    MmShape best{false, 16, 1};
    double least = 1e30;
    auto offer = [&](bool pair, int bt, int splits, int64_t units) {
        const int64_t tt = (n + bt - 1) / bt, real = ((n + tt - 1) / tt + 15) / 16 * 16;
        const int64_t tiles = groups * tt * ((cols + (pair ? 255 : 127)) / (pair ? 256 : 128)), waves = (tiles + units - 1) / units;
        if (splits > 1 && (grouped ? tiles + tiles / 2 : tiles) > units) return;
        const double block = pair ? 0.145 + 0.0006 * real : 0.153 + 0.00064 * bt;
        const double compute = (double)waves * (double)((nkb + splits - 1) / splits) * block;
        const double full = std::min(1.0, (double)tiles * splits / (double)(pair ? kSms / 2 : kSms));   // of the GPU that works at once
        const double time = (pair ? 5.0 + 0.022 * real * full : 3.5 + (0.6 + 0.014 * real) * full) +
                            std::max(compute, grouped ? memory : 0.0) + (grouped ? (double)(tt - 1) * weights / 12e6 : 0.0) +
                            0.25 * (double)(waves - 1) + (splits > 1 ? 0.8 + (1.1 + 0.018 * real) * full : 0.0);
        if (time < least) { least = time; best = MmShape{pair, bt, splits}; }
    };
    for (int bt : {16, 32, 48, 64, 96, 128}) {
        if (bt > 16 && bt >= n + 32) break;
        offer(false, bt, 1, kSms);
        if (k_groups >= 2) offer(false, bt, 2, 72);
        if (k_groups >= 4) offer(false, bt, 4, 34);
        if (k_groups >= 8) offer(false, bt, 8, 8);
    }
    if (cols > 128)
        for (int bt = 64; bt <= kMmRowsMax && bt < n + 32; bt += 16) offer(true, bt, 1, kSms / 2);
    return best;
}

// A wait that expires ends its CTA, which must not happen while copies or MMAs of a healthy product are still on their
// way into that CTA's memory: bounds below this are refused, no wait begins before the kernels in front have ended
// (grid_wait in every role), and the longest wait (a tile's whole K loop) gets 4 us per
// K block on top, more than ten times what one takes.
constexpr int kMmLeastSpins = 8000000;

bool bad_product(int64_t rows, int64_t cols, int64_t depth, int64_t experts) {
    return rows < 0 || cols < 1 || depth < 16 || depth % 16 || rows > (1 << 30) || depth > (1 << 30) || experts < 1 || experts > kMmMaxExperts || experts * cols > (1 << 30);
}

int dtype_bytes(int dtype) { return dtype == MXK_DTYPE_FP32 ? 4 : 2; }

}  // namespace

extern "C" {

int mxk_plan_tokens(const void* topk_idx, int32_t idx_bytes, int64_t idx_stride, int32_t tokens, int32_t topk,
                    int32_t first_expert, int32_t num_experts, int32_t* row_of_pair, int32_t* pair_of_row,
                    int32_t* offsets, void* stream) {
    if (bad_tables(tokens, topk) || num_experts < 1 || num_experts > kRowsMaxExperts || first_expert < 0 || (idx_bytes != 4 && idx_bytes != 8))
        return fail(MXK_ERR_BAD_ARG, "plan_tokens: need tokens * topk <= 2^30, 1 <= topk <= 256, 1 <= num_experts <= 1024, ids of 4 or 8 bytes");
    if (idx_stride < 0) return fail(MXK_ERR_BAD_ARG, "plan_tokens: strides must not be negative");
    if (!offsets || (tokens > 0 && (!topk_idx || !row_of_pair || !pair_of_row)))
        return fail(MXK_ERR_BAD_ARG, "plan_tokens: pointers must be non-null");
    if (!words(row_of_pair, pair_of_row, offsets) || addr(topk_idx) % (uint64_t)idx_bytes)
        return fail(MXK_ERR_BAD_ARG, "plan_tokens: ids and tables must be aligned to their element type");
    PlanArgs a;
    std::memset(&a, 0, sizeof(a));
    a.idx = topk_idx; a.idx_stride = idx_stride; a.idx64 = idx_bytes == 8;
    a.pairs = tokens * topk; a.topk = topk; a.first = first_expert; a.experts = num_experts;
    a.ftopk = FastDiv::make((uint32_t)topk);
    a.row_of_pair = row_of_pair; a.pair_of_row = pair_of_row; a.offsets = offsets;
    while ((1 << a.bits) <= num_experts) ++a.bits;
    const int smem_most = (kPlanWarps + 2) * plan_stride(kRowsMaxExperts) * 4;
    if (int rc = allow_smem((const void*)k_plan, 0, smem_most)) return rc;
    int ctas = 1, threads = std::max(256, (num_experts + 255) / 256 * 256);
    if (a.pairs > 8 * 32 * kPlanKeep) {
        threads = kPlanThreads;
        ctas = a.pairs > 16384 && sixteen_fit(smem_most) ? 16 : 8;
    }
    const int warps = threads / 32;
    a.per_warp = std::max(32, ((a.pairs + ctas * warps - 1) / (ctas * warps) + 31) / 32 * 32);
    a.per_cta = a.per_warp * warps;
    return launched(launch(k_plan, dim3(ctas, 1, 1), threads, (size_t)(warps + 2) * plan_stride(num_experts) * 4, ctas, static_cast<cudaStream_t>(stream), a), "launch k_plan");
}

int mxk_sort_tokens(const void* x, int64_t x_stride, int64_t row_bytes, const void* x_sf, int64_t sf_stride, int64_t sf_bytes,
                    int32_t tokens, int32_t topk, int32_t num_experts, const int32_t* row_of_pair, const int32_t* offsets,
                    void* rows, void* rows_sf, void* stream) {
    return mxk_sort_tokens_by_plan(x, x_stride, row_bytes, x_sf, sf_stride, sf_bytes, tokens, topk, num_experts, row_of_pair, nullptr,
                                   offsets, rows, rows_sf, stream);
}

int mxk_sort_tokens_by_plan(const void* x, int64_t x_stride, int64_t row_bytes, const void* x_sf, int64_t sf_stride, int64_t sf_bytes,
                            int32_t tokens, int32_t topk, int32_t num_experts, const int32_t* row_of_pair, const int32_t* pair_of_row,
                            const int32_t* offsets, void* rows, void* rows_sf, void* stream) {
    if (bad_tables(tokens, topk) || num_experts < 1 || num_experts > kRowsMaxExperts || row_bytes < 1 || row_bytes > kMaxRowBytes || (x_sf && (sf_bytes < 1 || sf_bytes > (1 << 24))))
        return fail(MXK_ERR_BAD_ARG, "sort_tokens: sizes out of range");
    if (x_stride < 0 || sf_stride < 0) return fail(MXK_ERR_BAD_ARG, "sort_tokens: strides must not be negative");
    if (tokens == 0) return 0;
    if (!x || !rows || !row_of_pair || !offsets || (x_sf && !rows_sf)) return fail(MXK_ERR_BAD_ARG, "sort_tokens: pointers must be non-null");
    if (!words(row_of_pair, pair_of_row, offsets)) return fail(MXK_ERR_BAD_ARG, "sort_tokens: tables must be aligned to their element type");
    const int vec = common_vec(addr(x) | addr(rows) | (uint64_t)x_stride | (uint64_t)row_bytes);
    SortArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x = static_cast<const uint8_t*>(x); a.x_sf = static_cast<const uint8_t*>(x_sf);
    a.rows = static_cast<uint8_t*>(rows); a.rows_sf = static_cast<uint8_t*>(rows_sf);
    a.tables = RowTables{row_of_pair, pair_of_row, offsets + num_experts, tokens * topk};
    a.x_stride = x_stride; a.sf_stride = sf_stride; a.sf_bytes = (int)sf_bytes;
    if (x_sf) {
        const int v = common_vec(addr(x_sf) | addr(rows_sf) | (uint64_t)sf_stride | (uint64_t)sf_bytes);
        a.sf_vec = v == 2 ? 1 : v;
    }
    const dim3 grid = row_frame(a.f, tokens, topk, (int)row_bytes, vec, unroll_of(vec), row_of_pair);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    switch (vec) {
        case 16: e = launch(k_sort_rows<16, 1>, grid, kRowThreads, 0, 1, st, a); break;
        case 8: e = launch(k_sort_rows<8, 2>, grid, kRowThreads, 0, 1, st, a); break;
        case 4: e = launch(k_sort_rows<4, 4>, grid, kRowThreads, 0, 1, st, a); break;
        case 2: e = launch(k_sort_rows<2, 4>, grid, kRowThreads, 0, 1, st, a); break;
        default: e = launch(k_sort_rows<1, 4>, grid, kRowThreads, 0, 1, st, a); break;
    }
    return launched(e, "launch k_sort_rows");
}

int mxk_unsort_tokens(const void* rows, int32_t dtype, int64_t rows_stride, const float* weights, int64_t weights_stride,
                      int32_t tokens, int32_t topk, int32_t hidden, const int32_t* row_of_pair, void* y, void* stream) {
    if (bad_tables(tokens, topk) || hidden < 1 || hidden > kMaxRowBytes / 4 || dtype < MXK_DTYPE_BF16 || dtype > MXK_DTYPE_FP32)
        return fail(MXK_ERR_BAD_ARG, "unsort_tokens: sizes or type out of range");
    if (rows_stride < 0 || weights_stride < 0) return fail(MXK_ERR_BAD_ARG, "unsort_tokens: strides must not be negative");
    if (tokens == 0) return 0;
    if (!rows || !row_of_pair || !y) return fail(MXK_ERR_BAD_ARG, "unsort_tokens: pointers must be non-null");
    UnsortArgs a;
    std::memset(&a, 0, sizeof(a));
    a.rows = static_cast<const uint8_t*>(rows); a.w = weights; a.y = static_cast<uint8_t*>(y);
    a.rows_stride = rows_stride; a.w_stride = weights_stride;
    const int row_bytes = hidden * dtype_bytes(dtype);
    const int vec = common_vec(addr(rows) | addr(y) | (uint64_t)rows_stride | (uint64_t)row_bytes);
    if (vec < dtype_bytes(dtype) || !words(weights, row_of_pair)) return fail(MXK_ERR_BAD_ARG, "unsort_tokens: tensors must be aligned to their element type");
    const dim3 grid = row_frame(a.f, tokens, topk, row_bytes, vec, unroll_of(vec), row_of_pair);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MXK_DTYPE_BF16) return unsort_launch<kTypeBf16>(a, vec, grid, st);
    if (dtype == MXK_DTYPE_FP16) return unsort_launch<kTypeFp16>(a, vec, grid, st);
    return unsort_launch<kTypeFp32>(a, vec, grid, st);
}

int mxk_unsort_tokens_grad(const void* dy, int64_t dy_stride, const void* rows, int64_t rows_stride, int32_t dtype,
                           const float* weights, int64_t weights_stride, int32_t tokens, int32_t topk, int32_t num_experts,
                           int32_t hidden, const int32_t* row_of_pair, const int32_t* offsets, void* drows, float* dweights,
                           void* stream) {
    return mxk_unsort_tokens_grad_by_plan(dy, dy_stride, rows, rows_stride, dtype, weights, weights_stride, tokens, topk, num_experts,
                                          hidden, row_of_pair, nullptr, offsets, drows, dweights, stream);
}

int mxk_unsort_tokens_grad_by_plan(const void* dy, int64_t dy_stride, const void* rows, int64_t rows_stride, int32_t dtype,
                                   const float* weights, int64_t weights_stride, int32_t tokens, int32_t topk, int32_t num_experts,
                                   int32_t hidden, const int32_t* row_of_pair, const int32_t* pair_of_row, const int32_t* offsets,
                                   void* drows, float* dweights, void* stream) {
    if (bad_tables(tokens, topk) || num_experts < 1 || num_experts > kRowsMaxExperts || hidden < 1 || hidden > kMaxRowBytes / 4 || dtype < MXK_DTYPE_BF16 || dtype > MXK_DTYPE_FP32)
        return fail(MXK_ERR_BAD_ARG, "unsort_tokens_grad: sizes or type out of range");
    if (dy_stride < 0 || rows_stride < 0 || weights_stride < 0) return fail(MXK_ERR_BAD_ARG, "unsort_tokens_grad: strides must not be negative");
    if (tokens == 0 || (!drows && !dweights)) return 0;
    if (!dy || !weights || !row_of_pair || !offsets || (dweights && !rows)) return fail(MXK_ERR_BAD_ARG, "unsort_tokens_grad: pointers must be non-null");
    UnsortGradArgs a;
    std::memset(&a, 0, sizeof(a));
    a.dy = static_cast<const uint8_t*>(dy); a.rows = static_cast<const uint8_t*>(rows); a.w = weights;
    a.drows = static_cast<uint8_t*>(drows); a.dw = dweights;
    a.tables = RowTables{row_of_pair, pair_of_row, offsets + num_experts, tokens * topk};
    a.dy_stride = dy_stride; a.rows_stride = rows_stride; a.w_stride = weights_stride;
    a.row_bytes = hidden * dtype_bytes(dtype); a.tokens = tokens; a.topk = topk;
    uint64_t bits = addr(dy) | (uint64_t)dy_stride | (uint64_t)a.row_bytes;
    if (drows) bits |= addr(drows);
    if (dweights) bits |= addr(rows) | (uint64_t)rows_stride;
    const int vec = common_vec(bits);
    if (vec < dtype_bytes(dtype) || !words(weights, row_of_pair, pair_of_row, offsets, dweights)) return fail(MXK_ERR_BAD_ARG, "unsort_tokens_grad: tensors must be aligned to their element type");
    a.vecs = a.row_bytes / vec;
    a.team = 1;   // warps per token: as many as the row has columns for
    while (a.team < 8 && a.vecs > 32 * a.team) a.team *= 2;
    const int grid = (int)(((int64_t)tokens * a.team + 7) / 8);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MXK_DTYPE_BF16) return unsort_grad_launch<kTypeBf16>(a, vec, grid, st);
    if (dtype == MXK_DTYPE_FP16) return unsort_grad_launch<kTypeFp16>(a, vec, grid, st);
    return unsort_grad_launch<kTypeFp32>(a, vec, grid, st);
}

int mxk_fp8_matmul(const MxkMatmulArgs* p, void* stream) {
    if (!p) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: null arguments");
    const int64_t rows = p->rows, cols = p->cols, depth = p->depth, experts = p->offsets ? p->experts : 1;
    if (bad_product(rows, cols, depth, experts))
        return fail(MXK_ERR_BAD_ARG, "fp8_matmul: need depth a multiple of 16, 1 <= experts <= 1024, rows and experts * cols <= 2^30");
    if (p->x_format < MXK_FP8_E4M3 || p->x_format > MXK_FP8_E5M2 || p->w_format < MXK_FP8_E4M3 || p->w_format > MXK_FP8_E5M2)
        return fail(MXK_ERR_BAD_ARG, "fp8_matmul: operand formats are MXK_FP8_E4M3 and MXK_FP8_E5M2");
    if (p->max_spins != 0 && p->max_spins < kMmLeastSpins)
        return fail(MXK_ERR_BAD_ARG, "fp8_matmul: max_spins is 0 or at least 8000000 (2 s)");
    if (rows == 0) return 0;
    if (!p->x || !p->w || !p->out) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: pointers must be non-null");
    if ((addr(p->x) | addr(p->w) | (uint64_t)p->x_stride | (uint64_t)p->w_stride) & 15 || p->x_stride < depth || p->w_stride < depth)
        return fail(MXK_ERR_BAD_ARG, "fp8_matmul: x and w need 16-byte aligned rows");
    if (!words(p->offsets)) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: offsets must be aligned to their element type");
    if (p->x_sf && rows > 1 && p->x_sf_stride < (depth + 127) / 128) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: rows of x_sf overlap");
    if ((addr(p->out) & 1) || (rows > 1 && p->out_stride < cols)) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: out must be bf16 rows that do not overlap");
    MmArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x_sf = p->x_sf; a.w_sf = p->w_sf; a.out = p->out; a.offsets = p->offsets;
    a.x_sf_stride = p->x_sf_stride; a.out_stride = p->out_stride;
    a.rows = (int)rows; a.cols = (int)cols; a.nkb = (int)((depth + 127) / 128); a.experts = (int)experts;
    a.w_per_row = p->w_sf_per_row ? 1 : 0;
    a.w_sf_rows = a.w_per_row ? a.cols : (a.cols + 127) / 128;
    a.zero_tail = p->offsets && p->zero_tail;
    a.formats = ((uint32_t)p->w_format << 7) | ((uint32_t)p->x_format << 10);   // w is the MMA's A operand, x its B
    a.wait_ns = (p->max_spins ? (unsigned long long)p->max_spins * 250ull : 2000000000ull) + (unsigned long long)a.nkb * 4000ull;

    const MmShape sh = mm_shape(rows, cols, depth, experts, p->offsets != nullptr);
    const bool pair = sh.pair;
    a.bt_max = sh.bt;
    a.splits = sh.splits;
    a.n_tiles = (a.cols + (pair ? 255 : 127)) / (pair ? 256 : 128);
    a.box = pair ? a.bt_max / 2 : a.bt_max;
    a.fbt = FastDiv::make((uint32_t)a.bt_max);
    a.fnt = FastDiv::make((uint32_t)a.n_tiles);
    const int sf_tiles = pair ? 3 : 2;
    a.sf_col = 2 * a.bt_max;
    a.sf_slots = std::min(kMmMaxSfSlots, (kMmTmemCols - a.sf_col) / (4 * sf_tiles));
    const int stage = kMmStageKb * (kMmWBytes + a.box * 128);
    const int fixed = 1024 + a.sf_slots * sf_tiles * kMmSfTile + (a.splits > 1 ? a.bt_max * 512 : 0) + (int)sizeof(MmSmem) + 2 * (a.experts + 1) * 4;
    a.n_stages = std::min(kMmMaxStages, (kMmSmemLimit - fixed) / stage);
    const int smem = fixed + a.n_stages * stage;
    CUtensorMap tm_x, tm_w;
    if (int rc = byte_map(&tm_x, p->x, rows, depth, p->x_stride, a.box)) return rc;
    if (int rc = byte_map(&tm_w, p->w, experts * cols, depth, p->w_stride, 128)) return rc;
    const auto fn = pair ? k_matmul_pair : k_matmul;
    if (int rc = allow_smem((const void*)fn, pair ? 1 : 2, kMmSmemLimit)) return rc;
    const int cluster = pair ? 2 : a.splits;   // mm_shape gives pairs no splits
    const int64_t tiles_most = ((p->offsets ? std::min<int64_t>(experts, rows) : 0) + (rows + a.bt_max - 1) / a.bt_max) * a.n_tiles;
    if (tiles_most > (1 << 30)) return fail(MXK_ERR_BAD_ARG, "fp8_matmul: more than 2^30 tiles");
    const dim3 grid((unsigned)(std::min<int64_t>(tiles_most, kSms / cluster) * cluster), 1, 1);
    return launched(launch(fn, grid, kMmThreads, (size_t)smem, cluster, static_cast<cudaStream_t>(stream), a, tm_x, tm_w), "launch k_matmul");
}

int mxk_matmul_cut(int32_t rows, int32_t cols, int32_t depth, int32_t experts, int32_t grouped, int32_t cut[3]) {
    if (!cut || rows < 1 || bad_product(rows, cols, depth, grouped ? experts : 1)) return fail(MXK_ERR_BAD_ARG, "matmul_cut: null argument or sizes out of range");
    const MmShape sh = mm_shape(rows, cols, depth, grouped ? experts : 1, grouped != 0);
    cut[0] = sh.pair; cut[1] = sh.bt; cut[2] = sh.splits;
    return 0;
}

int mxk_matmul_status(int32_t* out) {
    if (!out) return fail(MXK_ERR_BAD_ARG, "matmul_status: null argument");
    int v = 0;
    cudaError_t e = cudaDeviceSynchronize();   // products on every stream
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceSynchronize(matmul status)");
    e = cudaMemcpyFromSymbol(&v, g_mm_status, sizeof(v));
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemcpyFromSymbol(matmul status)");
    *out = v;
    return 0;
}

}  // extern "C"
