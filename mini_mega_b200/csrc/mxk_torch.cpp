// ============================================================================
// mxk_torch.cpp — torch binding of the operators beside the layer (experts.py, matmul.py).
//
// The layer's own calls go through ctypes: one of them is 150 us and more of GPU work.  An operator
// can be a few microseconds of it, and the same binding in Python (argument checks, allocation,
// stream look-up, ctypes) took 17 to 19 us of host time per call and 130 us for a forward and backward
// pass; here it is 4 to 5 us and 49 to 58 (torch's own product: 47 to 51).  Checks raise before anything touches a device, so they hold on a host
// without one.  All compute is in libmxk_b200.so, reached through its C ABI.
// ============================================================================
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cstring>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "../../include/mxk_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

constexpr int64_t kMaxExperts = 1024, kMaxTopk = 256, kMaxRows = int64_t(1) << 30, kMaxHidden = int64_t(1) << 22;

template <class E, class... A>
[[noreturn]] void raise(const A&... parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw E(s.str());
}
#define MXK_VALUE(cond, ...) do { if (!(cond)) raise<py::value_error>(__VA_ARGS__); } while (0)
#define MXK_TYPE(cond, ...) do { if (!(cond)) raise<py::type_error>(__VA_ARGS__); } while (0)

void done(int rc, const char* what) {
    if (rc != 0) throw std::runtime_error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + mxk_last_error());
}

void same_device(const char* fn, const Tensor& first, std::initializer_list<const Tensor*> rest) {
    const at::Device d = first.device();
    for (const Tensor* t : rest)
        if (t && t->defined()) MXK_VALUE(t->device() == d, fn, ": all tensors must be on one device, got ", d.str(), " and ", t->device().str());
    MXK_VALUE(d.is_cuda(), fn, " runs on CUDA tensors only, got ", d.str());
}

// The calls pass the dispatcher by, so whoever follows a computation through it sees a fresh result without a past: a
// tangent would be lost and a tracer would store the result as a constant, both without a word.  They are refused.
void not_followed(const char* fn, std::initializer_list<const Tensor*> inputs) {
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
        throw std::runtime_error(std::string(fn) + ": cannot be traced");
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : inputs)
        if (t && t->defined() && t->_fw_grad(0).defined())
            throw std::runtime_error(std::string(fn) + ": has no forward-mode derivative, got an input with a tangent");
}

Tensor rows_contiguous(const Tensor& t) {
    if (t.is_neg()) return t.resolve_neg().contiguous();   // a view that carries its sign in a flag
    return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
}
int64_t row_bytes_apart(const Tensor& t) { return t.stride(0) * (int64_t)t.element_size(); }
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int32_t* table(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// Allocation without the dispatcher (0.3 us of 1.1), on the device of `like`.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// Part of an int32 tensor's memory as a tensor of its own: 0.1 us where an allocation takes 0.8.
Tensor part_of(const Tensor& whole, int64_t first, at::IntArrayRef sizes) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(first);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

// ---- tokens sorted by expert and back ---------------------------------------------------
int type_code(at::ScalarType t) {
    return t == at::kBFloat16 ? MXK_DTYPE_BF16 : t == at::kHalf ? MXK_DTYPE_FP16 : t == at::kFloat ? MXK_DTYPE_FP32 : -1;
}

std::tuple<Tensor, Tensor, Tensor> plan_tokens(const Tensor& topk_idx, int64_t num_experts, int64_t first_expert) {
    const char* fn = "plan_tokens_by_expert";
    not_followed(fn, {});
    MXK_TYPE(topk_idx.scalar_type() == at::kLong || topk_idx.scalar_type() == at::kInt, fn, ": topk_idx must be an int64 or int32 tensor");
    MXK_VALUE(topk_idx.dim() == 2 && topk_idx.size(1) >= 1 && topk_idx.size(1) <= kMaxTopk, fn, ": topk_idx must be [tokens, topk] with 1 <= topk <= ", kMaxTopk, ", got ", topk_idx.sizes());
    MXK_VALUE(num_experts >= 1 && num_experts <= kMaxExperts, fn, ": num_experts must be in [1, ", kMaxExperts, "], got ", num_experts);
    MXK_VALUE(first_expert >= 0 && first_expert < (int64_t(1) << 31), fn, ": first_expert must be in [0, 2^31), got ", first_expert);
    const int64_t tokens = topk_idx.size(0), topk = topk_idx.size(1);
    MXK_VALUE(tokens * topk <= kMaxRows, fn, ": tokens * topk must be at most 2^30, got ", tokens * topk);
    same_device(fn, topk_idx, {});
    const c10::cuda::CUDAGuard guard(topk_idx.device());
    const Tensor idx = rows_contiguous(topk_idx);
    const int64_t pairs = tokens * topk;
    const Tensor tables = fresh({2 * pairs + num_experts + 1}, at::kInt, idx);
    Tensor row_of_pair = part_of(tables, 0, {tokens, topk}), pair_of_row = part_of(tables, pairs, {pairs}), offsets = part_of(tables, 2 * pairs, {num_experts + 1});
    done(mxk_plan_tokens(idx.data_ptr(), (int32_t)idx.element_size(), idx.stride(0), (int32_t)tokens, (int32_t)topk, (int32_t)first_expert,
                         (int32_t)num_experts, table(row_of_pair), table(pair_of_row), table(offsets), stream_of(idx)),
         "mxk_plan_tokens");
    return {row_of_pair, pair_of_row, offsets};
}

void check_plan(const char* fn, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
    for (const Tensor* t : {&row_of_pair, &pair_of_row, &offsets}) {
        MXK_TYPE(t->scalar_type() == at::kInt, fn, ": the plan's tables must be int32 tensors");
        MXK_VALUE(t->is_contiguous(), fn, ": the plan's tables must be contiguous");
    }
    MXK_VALUE(row_of_pair.dim() == 2 && row_of_pair.size(1) >= 1 && row_of_pair.size(1) <= kMaxTopk && row_of_pair.numel() <= kMaxRows, fn, ": row_of_pair must be [tokens, topk], got ", row_of_pair.sizes());
    MXK_VALUE(pair_of_row.dim() == 1 && pair_of_row.size(0) == row_of_pair.numel(), fn, ": pair_of_row must be [tokens * topk], got ", pair_of_row.sizes());
    MXK_VALUE(offsets.dim() == 1 && offsets.size(0) >= 2 && offsets.size(0) <= kMaxExperts + 1, fn, ": offsets must be [num_experts + 1], got ", offsets.sizes());
}

// A leaf's gradient is accumulated on the stream of the leaf's first use for as long as a graph of that
// use lives.  When that was another stream than the one under capture, the captured backward pass would have to
// wait on it, which invalidates the capture and ends the process; such a call is refused instead.
void check_leaf_under_capture(const char* fn, const Tensor& t) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return;
    const auto made_on = node->stream();
    if (made_on && *made_on != at::cuda::getCurrentCUDAStream(t.device().index()).unwrap())
        throw std::runtime_error(std::string(fn) + ": a graph of an earlier call with the same leaf tensor is still alive and belongs to "
                                 "another stream; drop its outputs before the capture begins");
}

Tensor sort_rows(const Tensor& x_in, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets, const Tensor& sf_in, Tensor* rows_sf) {
    const c10::cuda::CUDAGuard guard(x_in.device());
    const int64_t tokens = row_of_pair.size(0), topk = row_of_pair.size(1);
    const Tensor x = rows_contiguous(x_in);
    Tensor rows = fresh({tokens * topk, x.size(1)}, x.scalar_type(), x), sf;
    if (sf_in.defined()) {
        sf = rows_contiguous(sf_in);
        *rows_sf = fresh({tokens * topk, sf.size(1)}, at::kByte, sf);
    }
    done(mxk_sort_tokens_by_plan(x.data_ptr(), row_bytes_apart(x), x.size(1) * (int64_t)x.element_size(), sf.defined() ? sf.data_ptr() : nullptr,
                                 sf.defined() ? sf.stride(0) : 0, sf.defined() ? sf.size(1) : 0, (int32_t)tokens, (int32_t)topk,
                                 (int32_t)(offsets.size(0) - 1), table(row_of_pair), table(pair_of_row), table(offsets), rows.data_ptr(),
                                 sf.defined() ? rows_sf->data_ptr() : nullptr, stream_of(x)),
         "mxk_sort_tokens_by_plan");
    return rows;
}

Tensor unsort_rows(const Tensor& rows_in, const Tensor& weights_in, const Tensor& row_of_pair) {
    const c10::cuda::CUDAGuard guard(rows_in.device());
    const int64_t tokens = row_of_pair.size(0), topk = row_of_pair.size(1);
    const Tensor rows = rows_contiguous(rows_in);
    const Tensor weights = weights_in.defined() ? rows_contiguous(weights_in) : weights_in;
    Tensor y = fresh({tokens, rows.size(1)}, rows.scalar_type(), rows);
    done(mxk_unsort_tokens(rows.data_ptr(), type_code(rows.scalar_type()), row_bytes_apart(rows),
                           weights.defined() ? static_cast<const float*>(weights.data_ptr()) : nullptr, weights.defined() ? weights.stride(0) : 0,
                           (int32_t)tokens, (int32_t)topk, (int32_t)rows.size(1), table(row_of_pair), y.data_ptr(), stream_of(rows)),
         "mxk_unsort_tokens");
    return y;
}

// Sort and plain unsort are linear and each other's gradient, so they can be differentiated again;
// the weighted unsort cannot, and says so.
Tensor sort_differentiable(const Tensor& x, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets);
Tensor unsort_differentiable(const Tensor& rows, const Tensor& weights, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets);

struct SortFunction : torch::autograd::Function<SortFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
        ctx->save_for_backward({row_of_pair, pair_of_row, offsets});
        return sort_rows(x, row_of_pair, pair_of_row, offsets, Tensor(), nullptr);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        not_followed("sort_tokens_by_expert (backward)", {&grads[0]});
        return {unsort_differentiable(grads[0], Tensor(), saved[0], saved[1], saved[2]), Tensor(), Tensor(), Tensor()};
    }
};

struct SumFunction : torch::autograd::Function<SumFunction> {   // unsort without weights
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
        ctx->save_for_backward({row_of_pair, pair_of_row, offsets});
        return unsort_rows(rows, Tensor(), row_of_pair);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        not_followed("unsort_tokens_by_expert (backward)", {&grads[0]});
        return {sort_differentiable(grads[0], saved[0], saved[1], saved[2]), Tensor(), Tensor(), Tensor()};
    }
};

struct UnsortFunction : torch::autograd::Function<UnsortFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
        // rows are kept for the gradient of the weights only
        ctx->save_for_backward({weights.requires_grad() ? rows : Tensor(), weights, row_of_pair, pair_of_row, offsets});
        ctx->saved_data["rows_grad"] = rows.requires_grad();
        return unsort_rows(rows, weights, row_of_pair);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &weights_in = saved[1], &row_of_pair = saved[2], &pair_of_row = saved[3], &offsets = saved[4];
        not_followed("unsort_tokens_by_expert (backward)", {&grads[0]});
        if (at::GradMode::is_enabled()) throw std::runtime_error("unsort_tokens_by_expert: the weighted sum has no second derivative (create_graph)");
        const c10::cuda::CUDAGuard guard(grads[0].device());
        const int64_t tokens = row_of_pair.size(0), topk = row_of_pair.size(1);
        const Tensor dy = rows_contiguous(grads[0]), weights = rows_contiguous(weights_in);
        const Tensor rows = saved[0].defined() ? rows_contiguous(saved[0]) : Tensor();
        Tensor drows, dweights;
        if (ctx->saved_data["rows_grad"].toBool()) drows = fresh({tokens * topk, dy.size(1)}, dy.scalar_type(), dy);
        if (rows.defined()) dweights = fresh({tokens, topk}, at::kFloat, weights);
        done(mxk_unsort_tokens_grad_by_plan(dy.data_ptr(), row_bytes_apart(dy), rows.defined() ? rows.data_ptr() : nullptr,
                                    rows.defined() ? row_bytes_apart(rows) : 0, type_code(dy.scalar_type()),
                                    static_cast<const float*>(weights.data_ptr()), weights.stride(0), (int32_t)tokens, (int32_t)topk,
                                    (int32_t)(offsets.size(0) - 1), (int32_t)dy.size(1), table(row_of_pair), table(pair_of_row), table(offsets),
                                    drows.defined() ? drows.data_ptr() : nullptr,
                                    dweights.defined() ? static_cast<float*>(dweights.data_ptr()) : nullptr, stream_of(dy)),
             "mxk_unsort_tokens_grad_by_plan");
        return {drows, dweights, Tensor(), Tensor(), Tensor()};
    }
};

Tensor sort_differentiable(const Tensor& x, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
    if (!at::GradMode::is_enabled() || !x.requires_grad()) return sort_rows(x, row_of_pair, pair_of_row, offsets, Tensor(), nullptr);
    return SortFunction::apply(x, row_of_pair, pair_of_row, offsets);
}
Tensor unsort_differentiable(const Tensor& rows, const Tensor& weights, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets) {
    if (!at::GradMode::is_enabled() || !(rows.requires_grad() || (weights.defined() && weights.requires_grad())))
        return unsort_rows(rows, weights, row_of_pair);
    return weights.defined() ? UnsortFunction::apply(rows, weights, row_of_pair, pair_of_row, offsets) : SumFunction::apply(rows, row_of_pair, pair_of_row, offsets);
}

bool byte_type(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kFloat8_e5m2 || t == at::kByte || t == at::kChar; }
bool under_capture() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

py::object sort_tokens(const Tensor& x, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets, const MaybeTensor& x_sf) {
    const char* fn = "sort_tokens_by_expert";
    not_followed(fn, {&x});
    check_plan(fn, row_of_pair, pair_of_row, offsets);
    MXK_TYPE(type_code(x.scalar_type()) >= 0 || byte_type(x.scalar_type()), fn, ": x must be a bf16, fp16, fp32 or 8-bit tensor");
    MXK_VALUE(x.dim() == 2 && x.size(0) == row_of_pair.size(0) && x.size(1) >= 1 && x.size(1) <= kMaxHidden, fn, ": x must be [", row_of_pair.size(0), ", hidden], got ", x.sizes());
    if (x_sf) {
        MXK_TYPE(x_sf->scalar_type() == at::kByte && x.element_size() == 1, fn, ": x_sf are uint8 exponents of 8-bit rows");
        MXK_VALUE(x_sf->dim() == 2 && x_sf->size(0) == x.size(0) && x_sf->size(1) >= 1 && x_sf->size(1) <= kMaxHidden, fn, ": x_sf must be [", x.size(0), ", hidden / 128], got ", x_sf->sizes());
    }
    same_device(fn, x, {&row_of_pair, &pair_of_row, &offsets, x_sf ? &*x_sf : nullptr});
    const bool grad = x.requires_grad() && at::GradMode::is_enabled();
    MXK_TYPE(!grad || type_code(x.scalar_type()) >= 0, fn, ": only bf16, fp16 and fp32 rows have a gradient");
    if (x_sf) {
        Tensor rows_sf;
        const Tensor rows = sort_rows(x, row_of_pair, pair_of_row, offsets, *x_sf, &rows_sf);
        return py::cast(std::make_pair(rows, rows_sf));
    }
    const c10::cuda::CUDAGuard guard(x.device());
    if (grad && under_capture()) check_leaf_under_capture(fn, x);
    return py::cast(sort_differentiable(x, row_of_pair, pair_of_row, offsets));
}

Tensor unsort_tokens(const Tensor& rows, const Tensor& row_of_pair, const Tensor& pair_of_row, const Tensor& offsets, const MaybeTensor& topk_weights) {
    const char* fn = "unsort_tokens_by_expert";
    not_followed(fn, {&rows, topk_weights ? &*topk_weights : nullptr});
    check_plan(fn, row_of_pair, pair_of_row, offsets);
    MXK_TYPE(type_code(rows.scalar_type()) >= 0, fn, ": rows must be a bf16, fp16 or fp32 tensor");
    MXK_VALUE(rows.dim() == 2 && rows.size(0) == row_of_pair.numel() && rows.size(1) >= 1 && rows.size(1) <= kMaxHidden, fn, ": rows must be [", row_of_pair.numel(), ", hidden], got ", rows.sizes());
    const Tensor weights = topk_weights ? *topk_weights : Tensor();
    if (weights.defined()) {
        MXK_TYPE(weights.scalar_type() == at::kFloat, fn, ": topk_weights must be a float32 tensor");
        MXK_VALUE(weights.sizes() == row_of_pair.sizes(), fn, ": topk_weights must be ", row_of_pair.sizes(), ", got ", weights.sizes());
    }
    same_device(fn, rows, {&row_of_pair, &pair_of_row, &offsets, &weights});
    const c10::cuda::CUDAGuard guard(rows.device());
    if (at::GradMode::is_enabled() && (rows.requires_grad() || (weights.defined() && weights.requires_grad())) && under_capture()) {
        check_leaf_under_capture(fn, rows);
        check_leaf_under_capture(fn, weights);
    }
    return unsort_differentiable(rows, weights, row_of_pair, pair_of_row, offsets);
}

// ---- 8-bit products -----------------------------------------------------------------------
int format_code(at::ScalarType t) {
    return t == at::kFloat8_e4m3fn || t == at::kByte ? MXK_FP8_E4M3 : t == at::kFloat8_e5m2 ? MXK_FP8_E5M2 : -1;
}

Tensor matmul(const char* fn, const Tensor& x, const MaybeTensor& x_sf, const Tensor& w, const MaybeTensor& w_sf, const MaybeTensor& offsets, const MaybeTensor& out_in) {
    const int64_t w_dim = offsets ? 3 : 2;
    not_followed(fn, {&x, &w, out_in ? &*out_in : nullptr});
    MXK_TYPE(format_code(x.scalar_type()) >= 0, fn, ": x must be a float8_e4m3fn, float8_e5m2 (or raw uint8 E4M3) tensor");
    MXK_TYPE(format_code(w.scalar_type()) >= 0, fn, ": w must be a float8_e4m3fn, float8_e5m2 (or raw uint8 E4M3) tensor");
    MXK_TYPE(!at::GradMode::is_enabled() || !(x.requires_grad() || w.requires_grad()), fn, ": has no gradient: detach the operands, or call it under no_grad");
    MXK_VALUE(x.dim() == 2, fn, ": x must have 2 dimensions, got ", x.sizes());
    MXK_VALUE(w.dim() == w_dim, fn, ": w must have ", w_dim, " dimensions, got ", w.sizes());
    MXK_TYPE(!x_sf || x_sf->scalar_type() == at::kByte, fn, ": x scales must be uint8 exponents");
    MXK_TYPE(!w_sf || w_sf->scalar_type() == at::kByte, fn, ": w scales must be uint8 exponents");
    const int64_t rows = x.size(0), depth = x.size(1), cols = w.size(-2), experts = offsets ? w.size(0) : 1, blocks = (depth + 127) / 128;
    MXK_VALUE(w.size(-1) == depth, fn, ": x has ", depth, " columns, w ", w.size(-1));
    MXK_VALUE(depth >= 16 && depth % 16 == 0 && cols >= 1 && experts >= 1 && experts <= kMaxExperts, fn, ": needs a depth that is a multiple of 16, at least one weight row and 1 to ", kMaxExperts, " experts, got x ", x.sizes(), " and w ", w.sizes());
    MXK_VALUE(rows <= kMaxRows && depth <= kMaxRows && experts * cols <= kMaxRows, fn, ": more than 2^30 rows");
    if (x_sf)
        MXK_VALUE(x_sf->dim() == 2 && x_sf->size(0) == rows && x_sf->size(1) == blocks && (blocks == 1 || x_sf->stride(1) == 1), fn, ": x scales must be [", rows, ", ", blocks, "] with contiguous rows, got ", x_sf->sizes());
    int per_row = 0;
    if (w_sf) {
        const int64_t d = w_sf->dim(), tall = d == w_dim ? w_sf->size(-2) : -1;
        MXK_VALUE(d == w_dim && w_sf->size(-1) == blocks && (d == 2 || w_sf->size(0) == experts) && (tall == (cols + 127) / 128 || tall == cols), fn, ": w scales must be one byte per 128 x 128 block or per row and 128 columns of w ", w.sizes(), ", got ", w_sf->sizes());
        MXK_VALUE(w_sf->is_contiguous(), fn, ": w scales must be contiguous");
        per_row = tall != (cols + 127) / 128;
    }
    const auto misaligned = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15; };
    MXK_VALUE(x.stride(1) == 1 && (rows <= 1 || (x.stride(0) >= depth && x.stride(0) % 16 == 0)) && !misaligned(x), fn, ": x needs contiguous rows, 16-byte aligned and not overlapping");
    const int64_t w_stride = cols > 1 ? w.stride(-2) : experts > 1 ? w.stride(0) : depth;
    MXK_VALUE(w.stride(-1) == 1 && w_stride >= depth && w_stride % 16 == 0 && !misaligned(w) && (experts == 1 || w.stride(0) == cols * w_stride), fn, ": w needs contiguous rows, 16-byte aligned, and the experts' matrices one behind the other");
    if (offsets) {
        MXK_VALUE(offsets->scalar_type() == at::kInt && offsets->dim() == 1 && offsets->size(0) == experts + 1 && offsets->is_contiguous(), fn, ": offsets must be a contiguous int32 tensor of ", experts + 1, " entries");
    }
    if (out_in)
        MXK_VALUE(out_in->scalar_type() == at::kBFloat16 && out_in->dim() == 2 && out_in->size(0) == rows && out_in->size(1) == cols && (cols <= 1 || out_in->stride(1) == 1) && (rows <= 1 || out_in->stride(0) >= cols), fn, ": out must be a bf16 [", rows, ", ", cols, "] tensor with contiguous rows");
    if (out_in) MXK_VALUE(!out_in->requires_grad() && (!out_in->is_inference() || c10::InferenceMode::is_enabled()), fn, ": out must not require a gradient, nor be an inference tensor outside inference mode");
    const auto at_of = [](const MaybeTensor& t) { return t ? &*t : nullptr; };
    same_device(fn, x, {&w, at_of(x_sf), at_of(w_sf), at_of(offsets), at_of(out_in)});
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor out = out_in ? *out_in : fresh({rows, cols}, at::kBFloat16, x);
    if (rows == 0) return out;
    MxkMatmulArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x = static_cast<const uint8_t*>(x.data_ptr()); a.w = static_cast<const uint8_t*>(w.data_ptr());
    a.x_sf = x_sf ? static_cast<const uint8_t*>(x_sf->data_ptr()) : nullptr;
    a.w_sf = w_sf ? static_cast<const uint8_t*>(w_sf->data_ptr()) : nullptr;
    a.out = static_cast<uint16_t*>(out.data_ptr());
    a.offsets = offsets ? table(*offsets) : nullptr;
    a.x_stride = rows > 1 ? x.stride(0) : depth; a.x_sf_stride = x_sf ? x_sf->stride(0) : 0; a.w_stride = w_stride; a.out_stride = out.stride(0);
    a.rows = (int32_t)rows; a.cols = (int32_t)cols; a.depth = (int32_t)depth; a.experts = (int32_t)experts;
    a.x_format = format_code(x.scalar_type()); a.w_format = format_code(w.scalar_type());
    a.w_sf_per_row = per_row; a.zero_tail = out_in ? 0 : 1;
    done(mxk_fp8_matmul(&a, stream_of(x)), "mxk_fp8_matmul");
    if (out_in) torch::autograd::impl::bump_version(out);   // a graph that has saved the given tensor shall notice
    return out;
}

Tensor fp8_matmul(const Tensor& x, const MaybeTensor& x_sf, const Tensor& w, const MaybeTensor& w_sf, const MaybeTensor& out) {
    return matmul("fp8_matmul", x, x_sf, w, w_sf, std::nullopt, out);
}
Tensor fp8_grouped_matmul(const Tensor& x, const MaybeTensor& x_sf, const Tensor& w, const MaybeTensor& w_sf, const Tensor& offsets, const MaybeTensor& out) {
    return matmul("fp8_grouped_matmul", x, x_sf, w, w_sf, offsets, out);
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
    m.def("plan_tokens", &plan_tokens);
    m.def("sort_tokens", &sort_tokens);
    m.def("unsort_tokens", &unsort_tokens);
    m.def("fp8_matmul", &fp8_matmul);
    m.def("fp8_grouped_matmul", &fp8_grouped_matmul);
}
