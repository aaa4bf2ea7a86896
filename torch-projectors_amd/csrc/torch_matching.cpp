// PyTorch dispatcher registration of the matching operators
// (torch_projectors/matching.py): scores in 8-bit blocks, log probabilities,
// rows sorted by class.  No counterpart in the reference.  The ops join the
// namespace that torch_projectors.cpp defines; each checks its arguments,
// allocates its outputs and workspace from PyTorch's allocator, and calls the
// C ABI on PyTorch's current stream.
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>
#include <torch/torch.h>

#include <tuple>

#include "../../include/torch_projectors_hip.h"

namespace {

using at::Tensor;
using c10::optional;

constexpr int64_t kBlock = 128;

void* current_stream(const c10::Device& dev) {
    return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream());
}

void check_rc(int rc) { TORCH_CHECK(rc == TP_OK, "torch_projectors HIP backend: ", tp_last_error()); }

int dtype_code(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return TP_F32;
        case at::kHalf: return TP_F16;
        case at::kBFloat16: return TP_BF16;
        default: TORCH_CHECK(false, what, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

void same_device(const Tensor& t, const c10::Device& dev) {
    TORCH_CHECK(t.device() == dev, "all tensors must be on the same GPU (", dev, "), got one on ", t.device());
}

// An output or a workspace, straight from the GPU's allocator (at::empty's way there through the dispatcher
// costs as much again, and a small call is as long as its host side).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const c10::Device& dev) {
    return Tensor(at::detail::empty_cuda(sizes, dtype, dev, c10::nullopt));
}
Tensor workspace(int64_t bytes, const c10::Device& dev) { return bytes ? fresh({bytes}, at::kByte, dev) : Tensor(); }

// Values as they lie in memory (a view of a conjugate's imaginary part holds their negatives).
Tensor as_held(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// Adjacent, from a 16-byte boundary on.
Tensor adjacent16(const Tensor& t) {
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// The op's device, and no autograd inside it.
struct Scope {
    c10::hip::HIPGuardMasqueradingAsCUDA guard;
    at::AutoDispatchBelowADInplaceOrView no_autograd;
    explicit Scope(const c10::Device& dev) : guard(dev) {}
};
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------ 8-bit blocks
// Rows any distance apart, the values of each adjacent.
Tensor rows_of(const Tensor& x, const char* what) {
    TORCH_CHECK(x.dim() == 2, what, " must be (rows, values)");
    TORCH_CHECK(x.size(1) >= 1, what, ": rows must hold at least one value");
    const Tensor v = as_held(x);
    return v.size(1) == 1 || v.stride(1) == 1 ? v : v.contiguous();
}

std::tuple<Tensor, Tensor> quantize_blocks(const Tensor& x) {
    const int dt = dtype_code(x, "quantize_blocks: x");
    const auto dev = x.device();
    const Scope scope(dev);
    const Tensor v = rows_of(x, "quantize_blocks: x");
    const int64_t R = v.size(0), nb = (v.size(1) + kBlock - 1) / kBlock;
    Tensor codes = fresh({R, nb * kBlock}, at::kFloat8_e4m3fn, dev);
    Tensor scales = fresh({nb, tp_scale_rows(R)}, at::kByte, dev);
    check_rc(tp_quantize_blocks(dt, v.data_ptr(), R, v.size(1), v.stride(0), codes.data_ptr(), scales.data_ptr(),
                                current_stream(dev)));
    return {codes, scales};
}

void check_blocks(const Tensor& codes, const Tensor& scales, const char* what) {
    TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn && codes.dim() == 2 && codes.size(1) >= kBlock &&
                    codes.size(1) % kBlock == 0,
                what, ": codes must be float8_e4m3fn (rows, 128 * blocks)");
    TORCH_CHECK(scales.scalar_type() == at::kByte && scales.dim() == 2 && scales.size(0) == codes.size(1) / kBlock &&
                    scales.size(1) == tp_scale_rows(codes.size(0)),
                what, ": scales must be uint8 (blocks, rows padded to 16)");
}

// images: float rows, quantised on the way, or codes with their scales
Tensor block_scores(const Tensor& images, const optional<Tensor>& image_scales, const Tensor& codes,
                    const Tensor& scales, const optional<Tensor>& bias, at::ScalarType out_dtype) {
    check_blocks(codes, scales, "references");
    TORCH_CHECK(out_dtype == at::kFloat || out_dtype == at::kBFloat16,
                "block_scores: out_dtype must be float32 or bfloat16");
    const auto dev = codes.device();
    same_device(scales, dev);
    same_device(images, dev);
    const Scope scope(dev);
    const int64_t N = codes.size(0), nb = codes.size(1) / kBlock;
    Tensor f;
    if (bias.has_value()) {
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N && bias->scalar_type() == at::kFloat,
                    "block_scores: bias must be float32 (references)");
        same_device(*bias, dev);
        f = as_held(*bias).contiguous();
    }
    const Tensor b = adjacent16(codes), sb = adjacent16(scales);
    const int out_dt = out_dtype == at::kFloat ? TP_F32 : TP_BF16;
    auto same_blocks = [&](int64_t blocks) {
        TORCH_CHECK(blocks == nb, "block_scores: images have ", blocks, " blocks a row, references ", nb);
    };
    if (image_scales.has_value()) {
        check_blocks(images, *image_scales, "images");
        same_blocks(images.size(1) / kBlock);
        same_device(*image_scales, dev);
        const Tensor a = adjacent16(images), sa = adjacent16(*image_scales);
        const int64_t M = a.size(0), bytes = tp_block_scores_work(M, N, nb);
        Tensor out = fresh({M, N}, out_dtype, dev);
        const Tensor work = workspace(bytes, dev);
        check_rc(tp_block_scores(a.data_ptr(), sa.data_ptr(), M, b.data_ptr(), sb.data_ptr(), N, nb, ptr(f), out_dt,
                                 out.data_ptr(), ptr(work), bytes, current_stream(dev)));
        return out;
    }
    const int dt = dtype_code(images, "block_scores: images");
    const Tensor a = rows_of(images, "block_scores: images");
    same_blocks((a.size(1) + kBlock - 1) / kBlock);
    const int64_t M = a.size(0), bytes = tp_score_images_work(M, N, a.size(1));
    Tensor out = fresh({M, N}, out_dtype, dev);
    const Tensor work = workspace(bytes, dev);
    check_rc(tp_score_images(dt, a.data_ptr(), M, a.size(1), a.stride(0), b.data_ptr(), sb.data_ptr(), N, ptr(f),
                             out_dt, out.data_ptr(), ptr(work), bytes, current_stream(dev)));
    return out;
}

// ------------------------------------------------------------------ log probabilities
struct Probs {
    int dt;
    Tensor scores, given, mask;
    int64_t T, V, stride, G = 0, mask_stride = 0;
};
Probs probs(const Tensor& scores, const optional<Tensor>& given, const optional<Tensor>& mask) {
    Probs p;
    TORCH_CHECK(scores.dim() == 2, "log_probs: scores must be (rows, candidates)");
    TORCH_CHECK(scores.size(1) >= 1, "log_probs: there must be at least one candidate");
    p.dt = dtype_code(scores, "log_probs: scores");
    const auto dev = scores.device();
    p.T = scores.size(0);
    p.V = scores.size(1);
    p.scores = as_held(scores);
    if (p.V > 1 && p.scores.stride(1) != 1) p.scores = p.scores.contiguous();
    p.stride = p.scores.stride(0);
    if (given.has_value()) {
        TORCH_CHECK(given->scalar_type() == at::kLong && (given->dim() == 1 || given->dim() == 2) &&
                        given->size(0) == p.T,
                    "log_probs: given must be int64 with the scores' leading dimensions");
        same_device(*given, dev);
        p.given = given->contiguous();
        p.G = given->dim() == 1 ? 1 : given->size(1);
    }
    if (mask.has_value()) {
        const int64_t d = mask->dim();
        TORCH_CHECK(mask->scalar_type() == at::kBool && (d == 1 || d == 2) && mask->size(d - 1) == p.V &&
                        (d == 1 || mask->size(0) == p.T),
                    "log_probs: mask must be bool (candidates) or of the scores' shape");
        same_device(*mask, dev);
        p.mask = p.V == 1 || mask->stride(d - 1) == 1 ? *mask : mask->contiguous();
        p.mask_stride = d == 1 ? 0 : p.mask.stride(0);
    }
    return p;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> log_probs_of(const Tensor& scores,
                                                                        const optional<Tensor>& given,
                                                                        const optional<Tensor>& mask, int64_t top,
                                                                        double temperature, bool with_stats) {
    const Probs p = probs(scores, given, mask);
    TORCH_CHECK(top >= 0 && top <= 64, "log_probs: top must be in [0, 64]");
    const auto dev = scores.device();
    const Scope scope(dev);
    Tensor given_out = given.has_value() ? fresh(given->sizes(), at::kFloat, dev) : Tensor();
    Tensor entropy = fresh({p.T}, at::kFloat, dev), log_sum = fresh({p.T}, at::kFloat, dev);
    Tensor top_out = fresh({p.T, top}, at::kFloat, dev), top_index = fresh({p.T, top}, at::kLong, dev);
    Tensor stats = with_stats ? fresh({p.T, 4}, at::kFloat, dev) : Tensor();
    const int64_t bytes = tp_log_probs_work(p.T, p.V, top);
    const Tensor work = workspace(bytes, dev);
    check_rc(tp_log_probs(p.dt, p.scores.data_ptr(), p.T, p.V, p.stride, ptr(p.given), p.G, ptr(p.mask),
                          p.mask_stride, top, temperature, ptr(given_out), entropy.data_ptr(),
                          log_sum.data_ptr(), top_out.data_ptr(), top_index.data_ptr(), ptr(stats), ptr(work),
                          bytes, current_stream(dev)));
    return {given_out, entropy, log_sum, top_out, top_index, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> log_probs(const Tensor& scores, const optional<Tensor>& given,
                                                                     const optional<Tensor>& mask, int64_t top,
                                                                     double temperature) {
    return log_probs_of(scores, given, mask, top, temperature, true);
}

Tensor log_probs_back(const Tensor& scores, const optional<Tensor>& given, const optional<Tensor>& mask,
                      const Tensor& top_index, const Tensor& stats, double temperature,
                      const optional<Tensor>& d_given, const optional<Tensor>& d_entropy,
                      const optional<Tensor>& d_log_sum, const optional<Tensor>& d_top) {
    const Probs p = probs(scores, given, mask);
    const auto dev = scores.device();
    const int64_t top = top_index.dim() == 2 ? top_index.size(1) : -1;
    TORCH_CHECK(top >= 0 && top <= 64 && top_index.size(0) == p.T && top_index.scalar_type() == at::kLong,
                "log_probs_back: top_index must be int64 (rows, top)");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == p.T && stats.size(1) == 4,
                "log_probs_back: stats must be float32 (rows, 4)");
    auto upstream = [&](const optional<Tensor>& g, int64_t n, const char* what) {
        if (!g.has_value()) return Tensor();
        TORCH_CHECK(g->scalar_type() == at::kFloat && g->numel() == n, "log_probs_back: ", what,
                    " must be float32 of its output's shape");
        same_device(*g, dev);
        return as_held(*g).contiguous();
    };
    const Tensor dg = upstream(d_given, p.T * p.G, "d_given"), dh = upstream(d_entropy, p.T, "d_entropy");
    const Tensor dl = upstream(d_log_sum, p.T, "d_log_sum"), dt = upstream(d_top, p.T * top, "d_top");
    same_device(top_index, dev);
    same_device(stats, dev);
    const Scope scope(dev);
    const Tensor index = top_index.contiguous(), st = adjacent16(stats);
    Tensor out = fresh({p.T, p.V}, scores.scalar_type(), dev);
    check_rc(tp_log_probs_back(p.dt, p.scores.data_ptr(), p.T, p.V, p.stride, ptr(p.given), p.G, ptr(p.mask),
                               p.mask_stride, top, temperature, index.data_ptr(), st.data_ptr(),
                               p.G ? ptr(dg) : nullptr, ptr(dh), ptr(dl), top ? ptr(dt) : nullptr, out.data_ptr(),
                               current_stream(dev)));
    return out;
}

// ------------------------------------------------------------------ rows by class
std::tuple<Tensor, Tensor, Tensor> sort_by_class(const Tensor& classes, int64_t num_classes) {
    TORCH_CHECK(classes.dim() == 1 || classes.dim() == 2, "sort_by_class: classes must be (rows) or (rows, choices)");
    TORCH_CHECK(classes.scalar_type() == at::kLong || classes.scalar_type() == at::kInt,
                "sort_by_class: classes must be int64 or int32, got ", classes.scalar_type());
    TORCH_CHECK(num_classes >= 1 && num_classes <= 4096, "sort_by_class: num_classes must be in [1, 4096]");
    const auto dev = classes.device();
    const Scope scope(dev);
    const Tensor ids = classes.contiguous();
    const int64_t n = ids.numel();
    Tensor order = fresh({n}, at::kInt, dev), slot = fresh({ids.size(0), ids.dim() == 1 ? 1 : ids.size(1)}, at::kInt, dev);
    Tensor offsets = fresh({num_classes + 1}, at::kInt, dev);
    const int64_t bytes = tp_sort_by_class_work(n, num_classes);
    const Tensor work = workspace(bytes, dev);
    check_rc(tp_sort_by_class(int(ids.element_size()), ids.data_ptr(), n, num_classes, order.data_ptr(),
                              slot.data_ptr(), offsets.data_ptr(), ptr(work), bytes, current_stream(dev)));
    return {order, slot, offsets};
}

struct Route {
    Tensor slot, offsets, weights;
    int64_t T, k;
    const void* kept() const { return static_cast<const int*>(offsets.data_ptr()) + offsets.numel() - 1; }
};
Route route(const Tensor& slot, const Tensor& offsets, const optional<Tensor>& weights, const c10::Device& dev) {
    TORCH_CHECK(slot.scalar_type() == at::kInt && slot.dim() == 2, "slot must be int32 (rows, choices)");
    TORCH_CHECK(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.numel() >= 2,
                "offsets must be int32 (classes + 1)");
    same_device(slot, dev);
    same_device(offsets, dev);
    Route r{slot.contiguous(), offsets.contiguous(), Tensor(), slot.size(0), slot.size(1)};
    if (weights.has_value()) {
        TORCH_CHECK(weights->scalar_type() == at::kFloat && weights->sizes() == slot.sizes(),
                    "weights must be float32 (rows, choices)");
        same_device(*weights, dev);
        r.weights = as_held(*weights).contiguous();
    }
    return r;
}
// rows of a tensor: n along dimension 0, the rest of it one row
int64_t row_size(const Tensor& t, int64_t n, const char* what) {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == n, what, " must be (", n, ", values)");
    return t.size(1);
}

// x [T, D] -> sorted [T k, D]; with other [T k, D] also the weights' gradient <x[t], other[slot]> (else None)
std::tuple<Tensor, Tensor> spread_rows(const Tensor& x, const Tensor& slot, const Tensor& offsets,
                                       const optional<Tensor>& weights, const optional<Tensor>& other) {
    const auto dev = x.device();
    const Route r = route(slot, offsets, weights, dev);
    const int64_t D = row_size(x, r.T, "rows");
    const int dt = dtype_code(x, "rows");
    const Scope scope(dev);
    const Tensor v = as_held(x).contiguous();
    Tensor sorted = fresh({r.T * r.k, D}, x.scalar_type(), dev), o, dw;
    if (other.has_value()) {
        TORCH_CHECK(other->scalar_type() == x.scalar_type(), "both sides' rows must have the same dtype");
        TORCH_CHECK(row_size(*other, r.T * r.k, "sorted rows") == D, "both sides' rows must have the same size");
        same_device(*other, dev);
        o = as_held(*other).contiguous();
        dw = fresh(slot.sizes(), at::kFloat, dev);
    }
    check_rc(tp_spread_rows(dt, v.data_ptr(), r.T, D, r.k, r.slot.data_ptr(), r.kept(), ptr(r.weights),
                            sorted.data_ptr(), ptr(o), ptr(dw), current_stream(dev)));
    return {sorted, dw};
}

// sorted [T k, D] -> out [T, D]; with other [T, D] also the weights' gradient <other[t], sorted[slot]> (else None)
std::tuple<Tensor, Tensor> gather_rows(const Tensor& sorted, const Tensor& slot, const Tensor& offsets,
                                       const optional<Tensor>& weights, const optional<Tensor>& other) {
    const auto dev = sorted.device();
    const Route r = route(slot, offsets, weights, dev);
    const int64_t D = row_size(sorted, r.T * r.k, "sorted rows");
    const int dt = dtype_code(sorted, "sorted rows");
    const Scope scope(dev);
    const Tensor v = as_held(sorted).contiguous();
    Tensor out = fresh({r.T, D}, sorted.scalar_type(), dev), o, dw;
    if (other.has_value()) {
        TORCH_CHECK(other->scalar_type() == sorted.scalar_type(), "both sides' rows must have the same dtype");
        TORCH_CHECK(row_size(*other, r.T, "rows") == D, "both sides' rows must have the same size");
        same_device(*other, dev);
        o = as_held(*other).contiguous();
        dw = fresh(slot.sizes(), at::kFloat, dev);
    }
    check_rc(tp_gather_rows(dt, v.data_ptr(), r.T, D, r.k, r.slot.data_ptr(), r.kept(), ptr(r.weights),
                            out.data_ptr(), ptr(o), ptr(dw), current_stream(dev)));
    return {out, dw};
}

// ------------------------------------------------------------------ gradients
// Autograd in C++, as the ops above: a step takes as long as by a Python function (log_probs of 500 rows of 4099,
// forward and backward: 70 us against 71), but its backward does not hold the interpreter.

// The gradients are computed without a graph of their own: asking for one fails where it is used.
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto refuse = std::make_shared<torch::autograd::DelayedError>(
        "torch_projectors: the matching operators are differentiable once", int64_t(grads.size()));
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    return (*refuse)(std::move(grads));
}
optional<Tensor> given_or_none(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }
// There are no forward-mode derivatives: a tangent would be lost without a word.
void refuse_forward_mode(const optional<Tensor>& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t),
                                "torch_projectors: the matching operators have no forward-mode derivatives");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct LogProbsGrad : torch::autograd::Function<LogProbsGrad> {
    static variable_list forward(AutogradContext* ctx, const Tensor& scores, const optional<Tensor>& given,
                                 const optional<Tensor>& mask, int64_t top, double temperature) {
        auto [g, entropy, log_sum, best, index, stats] = log_probs(scores, given, mask, top, temperature);
        ctx->save_for_backward({scores, given.value_or(Tensor()), mask.value_or(Tensor()), index, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->mark_non_differentiable({index, stats});
        ctx->set_materialize_grads(false);
        if (!g.defined()) return {entropy, log_sum, best, index, stats};
        return {entropy, log_sum, best, index, stats, g};
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto v = ctx->get_saved_variables();
        Tensor out;
        {
            at::AutoGradMode off(false);
            auto up = [&](size_t i) { return i < d.size() ? given_or_none(d[i]) : c10::nullopt; };
            out = log_probs_back(v[0], given_or_none(v[1]), given_or_none(v[2]), v[3], v[4],
                                 ctx->saved_data["temperature"].toDouble(), up(5), up(0), up(1), up(2));
        }
        return once({out, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> log_probs_grad(const Tensor& scores,
                                                                          const optional<Tensor>& given,
                                                                          const optional<Tensor>& mask, int64_t top,
                                                                          double temperature) {
    refuse_forward_mode(scores);
    if (!at::GradMode::is_enabled() || !wants(scores))  // (no statistics: None)
        return log_probs_of(scores, given, mask, top, temperature, false);
    auto r = LogProbsGrad::apply(scores, given, mask, top, temperature);
    return {r.size() > 5 ? r[5] : Tensor(), r[0], r[1], r[2], r[3], r[4]};
}

// SPREAD: rows to their places; else back.  Each one's backward is the other.
template <bool SPREAD> struct RowsGrad : torch::autograd::Function<RowsGrad<SPREAD>> {
    static std::tuple<Tensor, Tensor> move(bool spread, const Tensor& x, const Tensor& slot, const Tensor& offsets,
                                           const optional<Tensor>& weights, const optional<Tensor>& other) {
        return spread ? spread_rows(x, slot, offsets, weights, other) : gather_rows(x, slot, offsets, weights, other);
    }
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& slot, const Tensor& offsets,
                          const optional<Tensor>& weights) {
        ctx->save_for_backward({wants(weights) ? x : Tensor(), slot, offsets, weights.value_or(Tensor())});
        return std::get<0>(move(SPREAD, x, slot, offsets, weights, c10::nullopt));
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto v = ctx->get_saved_variables();
        Tensor dx, dw;
        if (d[0].defined()) {
            at::AutoGradMode off(false);
            std::tie(dx, dw) = move(!SPREAD, d[0], v[1], v[2], given_or_none(v[3]), given_or_none(v[0]));
        }
        return once({dx, Tensor(), Tensor(), dw});
    }
};
template <bool SPREAD>
std::tuple<Tensor, Tensor> rows_grad(const Tensor& x, const Tensor& slot, const Tensor& offsets,
                                     const optional<Tensor>& weights, const optional<Tensor>& other) {
    using F = RowsGrad<SPREAD>;
    refuse_forward_mode(x);
    refuse_forward_mode(weights);
    if (!at::GradMode::is_enabled() || other.has_value() || !(wants(x) || wants(weights)))
        return F::move(SPREAD, x, slot, offsets, weights, other);
    return {F::apply(x, slot, offsets, weights), Tensor()};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torch_projectors, m) {
    m.def("quantize_blocks(Tensor x) -> (Tensor, Tensor)");
    m.def("block_scores(Tensor images, Tensor? image_scales, Tensor codes, Tensor scales, Tensor? bias, ScalarType out_dtype) -> Tensor");
    m.def("log_probs(Tensor scores, Tensor? given, Tensor? mask, int top, float temperature) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("log_probs_back(Tensor scores, Tensor? given, Tensor? mask, Tensor top_index, Tensor stats, float temperature, Tensor? d_given, Tensor? d_entropy, Tensor? d_log_sum, Tensor? d_top) -> Tensor");
    m.def("sort_by_class(Tensor classes, int num_classes) -> (Tensor, Tensor, Tensor)");
    m.def("spread_rows(Tensor x, Tensor slot, Tensor offsets, Tensor? weights, Tensor? other) -> (Tensor, Tensor)");
    m.def("gather_rows(Tensor sorted, Tensor slot, Tensor offsets, Tensor? weights, Tensor? other) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(torch_projectors, CUDA, m) {
    m.impl("quantize_blocks", &quantize_blocks);
    m.impl("block_scores", &block_scores);
    m.impl("log_probs", &log_probs);
    m.impl("log_probs_back", &log_probs_back);
    m.impl("sort_by_class", &sort_by_class);
    m.impl("spread_rows", &spread_rows);
    m.impl("gather_rows", &gather_rows);
}

// What is differentiable takes its gradient from above; the others are called as they are.
TORCH_LIBRARY_IMPL(torch_projectors, AutogradCUDA, m) {
    m.impl("log_probs", &log_probs_grad);
    m.impl("spread_rows", &rows_grad<true>);
    m.impl("gather_rows", &rows_grad<false>);
    for (const char* name : {"quantize_blocks", "block_scores", "log_probs_back", "sort_by_class"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}
