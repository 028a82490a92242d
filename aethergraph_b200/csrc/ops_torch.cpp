// The row operators as PyTorch functions: argument checks, outputs from PyTorch's allocator,
// PyTorch's current stream and autograd around the C ABI (include/aethergpu.h).  In C++ because the
// kernels of a small batch take less time than Python needs to make one call: a norm with its gradients
// spends 120 us of host time written in Python, most of it in the autograd engine's thread.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "../../include/aethergpu.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;
using MaybeType = std::optional<at::ScalarType>;

constexpr int64_t kF8Block = 128;  // columns per scale

template <typename... Args> [[noreturn]] void refuse(const Args &...args) { throw py::value_error(c10::str(args...)); }

void check(int32_t status) {
    if (status == AG_OK) return;
    if (status == AG_ERR_VALUE) throw py::value_error(ag_last_error());
    throw std::runtime_error(ag_last_error());
}

int tag_of(at::ScalarType t) {
    return t == at::kFloat ? AG_F32 : t == at::kHalf ? AG_F16 : t == at::kBFloat16 ? AG_BF16 : -1;
}

std::string say(const Tensor &t) { return t.defined() ? c10::str(t.sizes(), " ", t.scalar_type(), " on ", t.device()) : "nothing"; }

// A traced program would keep this call's results as constants: nothing here goes through PyTorch's dispatcher.
void no_trace(const char *what) {
    if (torch::jit::tracer::isTracing()) throw std::runtime_error(c10::str(what, " cannot be traced by torch.jit.trace"));
}

int check_rows(const Tensor &x, const char *what) {
    no_trace("a row operator");
    if (!x.is_cuda()) refuse(what, " must be a CUDA tensor");
    const int tag = tag_of(x.scalar_type());
    if (tag < 0) refuse(what, " must be float32, float16 or bfloat16, got ", x.scalar_type());
    if (x.dim() == 0 || x.size(-1) == 0) refuse(what, " must have at least one column, got shape ", x.sizes());
    return tag;
}

// The imaginary part of a conjugate keeps its values with the other sign.
Tensor plain(const Tensor &x) { return x.is_neg() ? x.resolve_neg() : x; }

// A tensor as rows of consecutive columns; copied only where it is laid out otherwise.
struct Rows {
    Tensor t;
    int64_t rows, dim, pitch;
    explicit Rows(const Tensor &x) : t(plain(x)), dim(x.size(-1)) {
        if (!t.is_contiguous()) {
            if (t.dim() == 2 && (t.stride(1) == 1 || dim == 1) && t.stride(0) >= 0) {
                rows = t.size(0);
                pitch = t.stride(0);
                return;
            }
            t = t.contiguous();
        }
        rows = t.numel() / dim;
        pitch = dim;
    }
};

// PyTorch's allocator without its dispatcher, which takes as long as the allocation.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
Tensor fresh_like(const Tensor &x) { return fresh(x.sizes(), x.scalar_type(), x); }
void *stream_of(const Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }
bool has(const MaybeTensor &t) { return t.has_value() && t->defined(); }
// Derivatives are reverse mode only.  A forward-mode tangent is not in the memory that a kernel is given, and
// would be gone without a word.
void no_tangent(const char *what, std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
        if (t && t->defined() && t->_fw_grad(0).defined()) refuse(what, " has no forward-mode derivative");
}
const Tensor *ptr(const MaybeTensor &t) { return has(t) ? &*t : nullptr; }
void once(const char *what) {
    if (at::GradMode::is_enabled()) throw std::runtime_error(c10::str(what, " is differentiable once; call the backward pass without create_graph"));
}
void no_gradient(const char *what, std::initializer_list<const Tensor *> tensors) {
    no_tangent(what, tensors);
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor *t : tensors)
        if (t && t->defined() && t->requires_grad()) refuse(what, " has no gradient; call it under torch.no_grad()");
}

// ----------------------------------------------------------------- dropout --
Tensor run_dropout(const Tensor &x, double p, uint64_t seed, uint64_t offset) {
    const Rows r(x);
    Tensor y = fresh_like(x);
    check(ag_rows_dropout(r.t.data_ptr(), y.data_ptr(), r.rows, r.dim, r.pitch, r.dim, tag_of(x.scalar_type()), p, seed, offset,
                          x.get_device(), stream_of(x)));
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, int64_t seed, int64_t offset) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        return run_dropout(x, p, (uint64_t)seed, (uint64_t)offset);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("dropout");
        return {run_dropout(grads[0], ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                            (uint64_t)ctx->saved_data["offset"].toInt()),
                Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor &x, double p, uint64_t seed, uint64_t offset) {
    no_tangent("dropout", {&x});
    check_rows(x, "x");
    if (x.requires_grad() && at::GradMode::is_enabled()) return Dropout::apply(x, p, (int64_t)seed, (int64_t)offset);
    return run_dropout(x, p, seed, offset);
}

void dropout_(const Tensor &x, double p, uint64_t seed, uint64_t offset) {
    no_tangent("dropout_", {&x});
    const int tag = check_rows(x, "x");
    if (x.requires_grad() && at::GradMode::is_enabled()) refuse("dropout_ is for rows that need no gradient; use dropout");
    const Rows r(x);
    if (!r.t.is_same(x) || (r.rows > 1 && r.pitch < r.dim)) refuse("dropout_ needs rows of consecutive columns that do not overlap");
    const int64_t pitch = std::max(r.pitch, r.dim);  // the pitch of a single row is free
    check(ag_rows_dropout(x.data_ptr(), x.data_ptr(), r.rows, r.dim, pitch, pitch, tag, p, seed, offset, x.get_device(), stream_of(x)));
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();  // whoever saved x for a backward pass is told
}

// -------------------------------------------------------------------- norm --
void check_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual) {
    check_rows(x, "x");
    if (has(weight)) {
        const Tensor &w = *weight;
        if (w.dim() != 1 || w.size(0) != x.size(-1) || w.device() != x.device() || (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat))
            refuse("weight must be [", x.size(-1), "] of ", x.scalar_type(), " or float32 on ", x.device(), ", got ", say(w));
    }
    if (has(residual)) {
        const Tensor &r = *residual;
        if (r.sizes() != x.sizes() || r.scalar_type() != x.scalar_type() || r.device() != x.device())
            refuse("residual must have the shape, type and device of x: got ", say(r), ", x is ", say(x));
    }
}

// The call's arguments without its outputs, and the tensors that they name.
struct NormCall {
    ag_norm n{};
    Rows x;
    std::optional<Rows> res;
    Tensor w;
    NormCall(const Tensor &x_, const MaybeTensor &weight, const MaybeTensor &residual, double eps) : x(x_) {
        n.x = x.t.data_ptr(); n.rows = x.rows; n.dim = x.dim; n.x_stride = x.pitch; n.eps = (float)eps; n.dtype = tag_of(x_.scalar_type());
        if (has(residual)) {
            res.emplace(*residual);
            n.residual = res->t.data_ptr(); n.residual_stride = res->pitch;
        }
        if (has(weight)) {
            w = plain(*weight).contiguous();
            n.weight = w.data_ptr(); n.weight_dtype = tag_of(w.scalar_type());
        }
    }
};

struct NormOut { Tensor y, h, rstd; };
NormOut run_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps, double p, uint64_t seed, uint64_t offset, bool want_rstd) {
    NormCall c(x, weight, residual, eps);
    c.n.p = p; c.n.seed = seed; c.n.offset = offset;
    NormOut out{fresh_like(x), x, Tensor()};
    c.n.y = out.y.data_ptr(); c.n.y_stride = c.x.dim;
    if (has(residual) || p > 0) {
        out.h = fresh_like(x);
        c.n.h = out.h.data_ptr(); c.n.h_stride = c.x.dim;
    }
    if (want_rstd) {
        out.rstd = fresh({c.x.rows}, at::kFloat, x);
        c.n.rstd = out.rstd.data_ptr<float>();
    }
    check(ag_rows_norm(&c.n, x.get_device(), stream_of(x)));
    return out;
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps, double p,
                                 int64_t seed, int64_t offset) {
        NormOut out = run_norm(x, weight, residual, eps, p, (uint64_t)seed, (uint64_t)offset, true);
        // 16-bit rows: not the rounded h but what it is made of, if that is not x alone
        const bool again = x.scalar_type() != at::kFloat && !out.h.is_same(x);
        auto kept = [](const Tensor &t) { return t.is_inference() ? t.clone() : t; };  // autograd keeps no tensor of inference mode
        ctx->save_for_backward({again ? kept(x) : out.h, has(weight) ? *weight : Tensor(), out.rstd, again && has(residual) ? kept(*residual) : Tensor()});
        ctx->saved_data["again"] = again;
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = has(residual);
        ctx->set_materialize_grads(false);
        return {out.y, out.h};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        once("add_rms_norm");
        variable_list got(7);
        if (!grads[0].defined() && !grads[1].defined()) return got;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &weight = saved[1], &rstd = saved[2], &res = saved[3];  // h, or x where it is made again
        const bool again = ctx->saved_data["again"].toBool();
        const double p = ctx->saved_data["p"].toDouble();
        const bool residual = ctx->saved_data["residual"].toBool();
        // what autograd counts is the tensors that there were
        const bool need_x = ctx->needs_input_grad(0), need_w = weight.defined() && ctx->needs_input_grad(1),
                   need_res = residual && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        const Rows r(h);
        ag_norm_grad n{};
        std::optional<Rows> rr;
        (again ? n.x : n.h) = r.t.data_ptr();
        (again ? n.x_stride : n.h_stride) = r.pitch;
        if (res.defined()) { rr.emplace(res); n.residual = rr->t.data_ptr(); n.residual_stride = rr->pitch; }
        n.rstd = rstd.data_ptr<float>(); n.rows = r.rows; n.dim = r.dim; n.p = p;
        n.seed = (uint64_t)ctx->saved_data["seed"].toInt(); n.offset = (uint64_t)ctx->saved_data["offset"].toInt();
        n.dtype = tag_of(h.scalar_type());
        std::optional<Rows> dy, dh;
        if (grads[0].defined()) { dy.emplace(grads[0]); n.dy = dy->t.data_ptr(); n.dy_stride = dy->pitch; }
        if (grads[1].defined()) { dh.emplace(grads[1]); n.dh = dh->t.data_ptr(); n.dh_stride = dh->pitch; }
        if (need_x) {
            got[0] = fresh_like(h);
            n.dx = got[0].data_ptr();
        }
        if (need_res) {
            if (p > 0 || !need_x) {
                got[2] = fresh_like(h);
                n.dresidual = got[2].data_ptr();
            } else {
                got[2] = got[0];  // without dropout the two are one
            }
        }
        Tensor w, scratch;
        if (weight.defined()) {
            w = plain(weight).contiguous();
            n.weight = w.data_ptr(); n.weight_dtype = tag_of(w.scalar_type());
            if (need_w && !dy) {  // h alone was used: the weights have no part in it
                got[1] = at::zeros_like(w);
            } else if (need_w) {
                check(ag_rows_norm_backward_scratch(r.rows, r.dim, n.dtype, h.get_device(), &n.scratch_bytes));
                got[1] = fresh_like(w);
                scratch = fresh({(int64_t)n.scratch_bytes}, at::kByte, h);
                n.dw = got[1].data_ptr(); n.scratch = scratch.data_ptr();
            }
        }
        check(ag_rows_norm_backward(&n, h.get_device(), stream_of(h)));
        return got;
    }
};

std::pair<Tensor, Tensor> add_rms_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps, double p, uint64_t seed,
                                       uint64_t offset) {
    no_tangent("add_rms_norm", {&x, ptr(weight), ptr(residual)});
    check_norm(x, weight, residual);
    if (at::GradMode::is_enabled() && (x.requires_grad() || (has(weight) && weight->requires_grad()) || (has(residual) && residual->requires_grad()))) {
        const variable_list out = AddRmsNorm::apply(x, weight, residual, eps, p, (int64_t)seed, (int64_t)offset);
        return {out[0], out[1]};
    }
    NormOut out = run_norm(x, weight, residual, eps, p, seed, offset, false);
    return {out.y, out.h};
}

// ------------------------------------------------------------- 8-bit rows --
int64_t blocks_of(int64_t n) { return (n + kF8Block - 1) / kF8Block; }
int64_t f8_pitch(int64_t dim) { return (dim + 15) / 16 * 16; }
Tensor empty_codes(int64_t rows, int64_t dim, const Tensor &like) {
    const int64_t pitch = f8_pitch(dim);
    Tensor t = fresh({rows, pitch}, at::kFloat8_e4m3fn, like);
    return pitch == dim ? t : t.narrow(1, 0, dim);
}
Tensor empty_scales(int64_t rows, int64_t dim, const Tensor &like) { return fresh({rows, blocks_of(dim)}, at::kFloat, like); }

std::pair<Tensor, Tensor> to_f8(NormCall &c, const Tensor &x) {
    Tensor codes = empty_codes(c.x.rows, c.x.dim, x), scales = empty_scales(c.x.rows, c.x.dim, x);
    c.n.codes = codes.data_ptr(); c.n.scales = scales.data_ptr<float>(); c.n.code_stride = f8_pitch(c.x.dim);
    if (c.x.rows) check(ag_rows_norm(&c.n, x.get_device(), stream_of(x)));
    return {codes, scales};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_f8(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps) {
    no_gradient("add_rms_norm_f8", {&x, ptr(weight), ptr(residual)});
    check_norm(x, weight, residual);
    NormCall c(x, weight, residual, eps);
    Tensor h = x;
    if (has(residual)) {
        h = fresh_like(x);
        c.n.h = h.data_ptr(); c.n.h_stride = c.x.dim;
    }
    auto [codes, scales] = to_f8(c, x);
    return {codes, scales, h};
}

std::pair<Tensor, Tensor> encode_f8(const Tensor &x) {
    no_gradient("encode_f8", {&x});
    check_rows(x, "x");
    NormCall c(x, std::nullopt, std::nullopt, 0.0);
    c.n.encode_only = 1;
    return to_f8(c, x);
}

std::pair<Tensor, Tensor> encode_weight_f8(const Tensor &w) {
    no_gradient("encode_weight_f8", {&w});
    const int tag = check_rows(w, "w");
    if (w.dim() != 2) refuse("weights must be [out, dim], got shape ", w.sizes());
    const Rows r(w);
    Tensor codes = empty_codes(r.rows, r.dim, w), scales = empty_scales(blocks_of(r.rows), r.dim, w);
    check(ag_rows_encode_weight(r.t.data_ptr(), r.rows, r.dim, r.pitch, tag, codes.data_ptr(), f8_pitch(r.dim), scales.data_ptr<float>(), w.get_device(),
                                stream_of(w)));
    return {codes, scales};
}

void check_f8(const Tensor &codes, const Tensor &scales, const char *what, int64_t rows_per_scale) {
    if (!codes.is_cuda() || codes.dim() != 2 || codes.scalar_type() != at::kFloat8_e4m3fn)
        refuse(what, " must be a CUDA tensor [rows, dim] of torch.float8_e4m3fn");
    const int64_t rows = codes.size(0), dim = codes.size(1), pitch = codes.stride(0);
    if (dim == 0 || (dim > 1 && codes.stride(1) != 1) || pitch % 16 || pitch < dim || (uintptr_t)codes.data_ptr() % 16)
        refuse(what, " must start on 16 bytes, with consecutive columns and a row pitch that is a multiple of 16 bytes");
    const int64_t want = (rows + rows_per_scale - 1) / rows_per_scale;
    if (!scales.is_cuda() || scales.get_device() != codes.get_device() || scales.scalar_type() != at::kFloat || scales.dim() != 2 || scales.size(0) != want ||
        scales.size(1) != blocks_of(dim) || !scales.is_contiguous() || scales.is_neg())
        refuse(what, "' scales must be contiguous float32 [", want, ", ", blocks_of(dim), "] on ", codes.device());
}

Tensor decode_f8(const Tensor &codes, const Tensor &scales) {
    no_trace("decode_f8");
    no_tangent("decode_f8", {&scales});
    check_f8(codes, scales, "codes", 1);
    Tensor out = fresh({codes.size(0), codes.size(1)}, at::kFloat, codes);
    check(ag_rows_decode(codes.data_ptr(), scales.data_ptr<float>(), codes.size(0), codes.size(1), codes.stride(0), out.data_ptr<float>(), codes.get_device(),
                         stream_of(codes)));
    return out;
}

// Where 8-bit rows lie: a pair of tensors, or a feature store.
struct Held { const void *codes; const float *scales; int64_t rows, dim, pitch; int device; const ag_features *store; };

Tensor product(const Held &held, const Tensor &weight, const Tensor &weight_scales, const MaybeTensor &ids, const MaybeTensor &bias, MaybeType type) {
    const at::ScalarType dtype = type.value_or(at::kBFloat16);
    no_trace("a product of 8-bit rows");
    no_tangent("a product of 8-bit rows", {&weight_scales});
    no_gradient("a product of 8-bit rows", {ptr(bias)});
    check_f8(weight, weight_scales, "weight", kF8Block);
    const int64_t out_dim = weight.size(0);
    if (weight.get_device() != held.device || weight.size(1) != held.dim || out_dim == 0)
        refuse("weight must be [out, ", held.dim, "] on cuda:", held.device, ", got ", say(weight));
    ag_product p{};
    Tensor plain_bias;
    p.out_dtype = tag_of(dtype);
    if (p.out_dtype < 0) refuse("dtype must be float32, float16 or bfloat16, got ", dtype);
    p.codes = held.codes; p.scales = held.scales; p.weight = weight.data_ptr(); p.weight_scales = weight_scales.data_ptr<float>();
    p.rows = p.held = held.rows; p.dim = held.dim; p.out_dim = out_dim; p.code_stride = held.pitch; p.store = held.store; p.weight_stride = weight.stride(0); p.out_stride = out_dim;
    if (has(ids)) {
        if (!ids->is_cuda() || ids->get_device() != held.device || ids->dim() != 1 || !ids->is_contiguous() ||
            (ids->scalar_type() != at::kLong && ids->scalar_type() != at::kInt))
            refuse("ids must be a contiguous 1-d tensor of dtype int64 or int32 on cuda:", held.device);
        p.ids = ids->data_ptr(); p.ids_are_i64 = ids->scalar_type() == at::kLong; p.rows = ids->size(0);
    }
    if (has(bias)) {
        if (!bias->is_cuda() || bias->get_device() != held.device || bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != out_dim ||
            !bias->is_contiguous())
            refuse("bias must be contiguous float32 [", out_dim, "] on cuda:", held.device);
        plain_bias = plain(*bias);
        p.bias = plain_bias.data_ptr<float>();
    }
    Tensor out = fresh({(int64_t)p.rows, out_dim}, dtype, weight);
    p.out = out.data_ptr();
    if (p.rows) check(ag_rows_product(&p, held.device, stream_of(weight)));
    return out;
}

Tensor product_f8(const Tensor &codes, const Tensor &scales, const Tensor &weight, const Tensor &weight_scales, const MaybeTensor &ids, const MaybeTensor &bias,
                  MaybeType dtype) {
    no_trace("a product of 8-bit rows");
    no_tangent("a product of 8-bit rows", {&scales});
    check_f8(codes, scales, "codes", 1);
    return product({codes.data_ptr(), scales.data_ptr<float>(), codes.size(0), codes.size(1), codes.stride(0), (int)codes.get_device(), nullptr}, weight, weight_scales,
                   ids, bias, dtype);
}

// `store`: an ag_features handle of 8-bit float rows.
Tensor project(uintptr_t store, const Tensor &ids, const Tensor &weight, const Tensor &weight_scales, const MaybeTensor &bias, MaybeType dtype) {
    const ag_features *f = (const ag_features *)store;
    uint64_t rows = 0, dim = 0;
    int32_t device = 0, kind = 0;
    check(ag_features_info(f, &rows, &dim, &kind, &device, nullptr));
    if (kind != AG_F8) refuse("the store does not hold 8-bit float rows");
    return product({nullptr, nullptr, (int64_t)rows, (int64_t)dim, 0, device, f}, weight, weight_scales, ids, bias, dtype);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto release = py::call_guard<py::gil_scoped_release>();
    m.def("dropout", &dropout, release);
    m.def("dropout_", &dropout_, release);
    m.def("add_rms_norm", &add_rms_norm, release);
    m.def("add_rms_norm_f8", &add_rms_norm_f8, release);
    m.def("encode_f8", &encode_f8, release);
    m.def("encode_weight_f8", &encode_weight_f8, release);
    m.def("decode_f8", &decode_f8, release);
    m.def("check_f8", &check_f8, release);
    m.def("product_f8", &product_f8, release);
    m.def("project", &project, release);
}
