// torch binding of the row-wise operators: argument checks, output buffers,
// the current stream, and their autograd nodes, over the C entry points of
// peer_b200.h.  The kernels are in libpeer_b200.so, which stays free of torch.
//
// The nodes are C++ because the operators are short: as torch.autograd.Function
// classes with ctypes calls a training pass through layer_norm cost 124 us of
// host time (two changes of the interpreter's lock between the caller's thread
// and the engine's, 20 arguments converted one by one), more than its kernels
// take at 16384 x 2048 (67 us); as here the whole pass costs 71 us.
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../../include/peer_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

template <typename... A> std::string text(A&&... a) { return c10::str(std::forward<A>(a)...); }

// dtypes as Python writes them
std::string dtype_name(at::ScalarType t) {
    switch (t) {
        case at::kDouble: return "torch.float64";
        case at::kFloat: return "torch.float32";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kByte: return "torch.uint8";
        case at::kShort: return "torch.int16";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return c10::toString(t);
    }
}

// return codes as in _lib.check
void check(int rc) {
    if (rc == PEER_OK) return;
    const char* msg = peer_last_error(nullptr);
    if (rc == PEER_ERR_INVALID_ARG || rc == PEER_ERR_UNSUPPORTED) throw py::value_error(text("peer_b200: ", msg));
    throw std::runtime_error(text("peer_b200 (code ", rc, "): ", msg));
}

void need_cuda(const Tensor& t, const char* name) {
    if (!t.is_cuda())
        throw std::runtime_error(text(name, " is on ", t.device(), ": peer_b200 runs on CUDA devices only (sm_100a); there is no CPU path"));
}

// A tangent would be dropped: the kernels see the values only, and the result would look like a constant.
bool has_tangent(const Tensor& t) {
    return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined();
}
void refuse_tangent(const Tensor& t, const char* name) {
    if (has_tangent(t))
        throw std::runtime_error(text(name, " carries a tangent: peer_b200 differentiates backward only, not in forward-mode"));
}

int code_of(at::ScalarType t, const char* name) {
    switch (t) {
        case at::kFloat: return PEER_DTYPE_F32;
        case at::kBFloat16: return PEER_DTYPE_BF16;
        case at::kHalf: return PEER_DTYPE_F16;
        default: throw py::type_error(text(name, " is ", dtype_name(t), "; float32, bfloat16 and float16 are implemented"));
    }
}

void need_rows(const Tensor& t, const char* name) {
    if (t.dim() < 1 || t.size(-1) < 1)
        throw py::value_error(text(name, " must have rows of at least one value, got shape ", t.sizes()));
}

// t [..., D] as [rows, D] with consecutive values in a row: a view wherever one exists (row strides of any size, zero
// included, are the kernels' business), else a contiguous copy.  A negated view (the imaginary part of a conjugate) has
// the wrong signs in memory and is resolved first; where a table or parameters are one, the call is refused.
Tensor as_rows(const Tensor& t) {
    const int64_t D = t.size(-1);
    Tensor rows = t.dim() == 2 ? t : t.reshape({t.numel() / D, D});
    rows = rows.resolve_neg();
    return D == 1 || rows.stride(1) == 1 ? rows : rows.contiguous();
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor workspace(int64_t bytes, const Tensor& like) {
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// What a second derivative through one of the nodes meets: an error, not a gradient that ignores the node.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto& g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(in.size()));
    return (*error)(std::move(in));
}

// ---- layer norm -----------------------------------------------------------------------------------------------------

struct NormCodes { int x, param; };

NormCodes check_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
    refuse_tangent(x, "x");
    refuse_tangent(w, "weight");
    refuse_tangent(b, "bias");
    need_cuda(x, "x");
    NormCodes c{code_of(x.scalar_type(), "x"), PEER_DTYPE_F32};
    need_rows(x, "x");
    if (!(eps >= 0.0)) throw py::value_error(text("eps=", eps, " must not be negative"));
    const auto one = [&](const Tensor& p, const char* name) {
        if (!p.defined()) return;
        if (p.dim() != 1 || p.size(0) != x.size(-1))
            throw py::value_error(text(name, " is ", p.sizes(), ", expected (", x.size(-1), ",)"));
        if (p.device() != x.device()) throw std::runtime_error(text(name, " is on ", p.device(), ", x on ", x.device()));
        if (p.scalar_type() != at::kFloat && p.scalar_type() != x.scalar_type())
            throw py::type_error(text(name, " is ", dtype_name(p.scalar_type()), ": parameters are float32 or of x's dtype, ", dtype_name(x.scalar_type())));
        if (!p.is_contiguous() || p.is_neg()) throw py::value_error(text(name, " must be contiguous"));
        c.param = code_of(p.scalar_type(), name);
    };
    one(w, "weight");
    one(b, "bias");
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
        throw py::type_error(text("weight is ", dtype_name(w.scalar_type()), " and bias ", dtype_name(b.scalar_type()), ": both parameters have one dtype"));
    return c;
}

struct NormOut { Tensor y, stats, payload, scale; };       // stats [2, rows]: means, 1/deviations

NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, NormCodes c, bool keep, bool pack) {
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor rows = as_rows(x);
    const int64_t R = rows.size(0), D = rows.size(1);
    NormOut o;
    o.y = at::empty(x.sizes(), x.options());
    float *mean = nullptr, *rstd = nullptr;
    if (keep) {
        o.stats = at::empty({2, R}, x.options().dtype(at::kFloat));
        mean = o.stats.data_ptr<float>();
        rstd = mean + R;
    }
    if (pack) {
        o.payload = at::empty({R, D}, x.options().dtype(at::kFloat8_e4m3fn));
        o.scale = at::empty({R}, x.options().dtype(at::kFloat));
    }
    check(peer_layer_norm(rows.data_ptr(), rows.stride(0), c.x, ptr(w), ptr(b), c.param, static_cast<float>(eps), R, D,
                          o.y.data_ptr(), mean, rstd, ptr(o.payload), static_cast<float*>(ptr(o.scale)), stream_of(x)));
    return o;
}

// x, or its packed form; add: contiguous, of grad's shape, added to dx before its rounding
variable_list norm_backward(const Tensor& grad, const Tensor& x, const Tensor& payload, const Tensor& scale, const Tensor& stats,
                            const Tensor& w, NormCodes c, at::ScalarType w_type, at::ScalarType b_type, bool want_x, bool want_w,
                            bool want_b, const Tensor& add) {
    const c10::cuda::CUDAGuard guard(grad.device());
    const Tensor dy = as_rows(grad), rows = x.defined() ? as_rows(x) : Tensor();
    const int64_t R = dy.size(0), D = dy.size(1);
    Tensor dx, dw, db;
    if (want_x) dx = at::empty(grad.sizes(), grad.options());
    if (want_w) dw = at::empty({D}, grad.options().dtype(w_type));
    if (want_b) db = at::empty({D}, grad.options().dtype(b_type));
    const int64_t bytes = want_w || want_b ? peer_layer_norm_workspace(R, D) : 0;
    const Tensor ws = workspace(bytes, grad);
    const float* mean = stats.data_ptr<float>();
    check(peer_layer_norm_backward(dy.data_ptr(), dy.stride(0), ptr(rows), rows.defined() ? rows.stride(0) : 0, ptr(payload),
                                   static_cast<float*>(ptr(scale)), mean, mean + R, ptr(w), c.x, c.param, ptr(add), R, D, ptr(dx),
                                   ptr(dw), ptr(db), ptr(ws), bytes, stream_of(grad)));
    return {dx, dw, db};
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                          bool packed, int64_t x_code, int64_t param_code) {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        const NormCodes c{static_cast<int>(x_code), static_cast<int>(param_code)};
        NormOut o = norm_forward(x, w, b, eps, c, true, packed);
        ctx->save_for_backward({packed ? Tensor() : x, w, o.payload, o.scale, o.stats});
        ctx->saved_data["codes"] = x_code * 16 + param_code;
        ctx->saved_data["bias"] = b.defined() ? static_cast<int64_t>(b.scalar_type()) : int64_t(-1);
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t codes = ctx->saved_data["codes"].toInt(), bias = ctx->saved_data["bias"].toInt();
        const bool has_w = saved[1].defined();
        size_t edge = 0;                                     // parameters that are missing have no edge
        const bool want_x = ctx->needs_input_grad(edge++);
        const bool want_w = has_w && ctx->needs_input_grad(edge++);
        const bool want_b = bias >= 0 && ctx->needs_input_grad(edge++);
        variable_list g;
        {
            const at::AutoGradMode off(false);
            g = norm_backward(grads[0], saved[0], saved[2], saved[3], saved[4], saved[1],
                              NormCodes{static_cast<int>(codes / 16), static_cast<int>(codes % 16)},
                              has_w ? saved[1].scalar_type() : at::kFloat,
                              bias >= 0 ? static_cast<at::ScalarType>(bias) : at::kFloat, want_x, want_w, want_b, Tensor());
        }
        g = once(std::move(g));
        return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, const std::optional<std::string>& checkpoint) {
    if (checkpoint && *checkpoint != "e4m3") throw py::value_error(text("checkpoint='", *checkpoint, "': None or 'e4m3'"));
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    const NormCodes c = check_norm(x, w, b, eps);
    if (at::GradMode::is_enabled() && (needs_grad(x) || needs_grad(w) || needs_grad(b)))
        return LayerNormNode::apply(x, weight, bias, eps, checkpoint.has_value(), int64_t(c.x), int64_t(c.param));
    return norm_forward(x, w, b, eps, c, false, false).y;
}

// ---- 8-bit rows -------------------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> pack_rows(const Tensor& x_in) {
    refuse_tangent(x_in, "x");
    need_cuda(x_in, "x");
    const int code = code_of(x_in.scalar_type(), "x");
    need_rows(x_in, "x");
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor rows = as_rows(x_in);
    Tensor payload = at::empty(x_in.sizes(), x_in.options().dtype(at::kFloat8_e4m3fn));
    Tensor scale = at::empty(x_in.sizes().slice(0, x_in.dim() - 1), x_in.options().dtype(at::kFloat));
    check(peer_pack_rows(rows.data_ptr(), rows.stride(0), code, rows.size(0), rows.size(1), payload.data_ptr(),
                         scale.data_ptr<float>(), stream_of(x_in)));
    return {payload, scale};
}

Tensor unpack_rows(const Tensor& payload_in, const Tensor& scale_in, at::ScalarType dtype) {
    refuse_tangent(scale_in, "scale");
    need_cuda(payload_in, "payload");
    if (payload_in.scalar_type() != at::kFloat8_e4m3fn || scale_in.scalar_type() != at::kFloat)
        throw py::type_error(text("payload is ", dtype_name(payload_in.scalar_type()), " and scale ", dtype_name(scale_in.scalar_type()),
                                  ", expected float8_e4m3fn and float32"));
    const int code = code_of(dtype, "dtype");
    if (payload_in.dim() < 1 || payload_in.size(-1) < 1 || scale_in.sizes() != payload_in.sizes().slice(0, payload_in.dim() - 1))
        throw py::value_error(text("payload ", payload_in.sizes(), " and scale ", scale_in.sizes(), " do not belong together"));
    if (scale_in.device() != payload_in.device())
        throw std::runtime_error(text("scale is on ", scale_in.device(), ", payload on ", payload_in.device()));
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard guard(payload_in.device());
    const Tensor payload = payload_in.contiguous(), scale = scale_in.contiguous().resolve_neg();
    Tensor out = at::empty(payload.sizes(), payload.options().dtype(dtype));
    const int64_t D = payload.size(-1);
    check(peer_unpack_rows(payload.data_ptr(), scale.data_ptr<float>(), code, payload.numel() / D, D, out.data_ptr(), stream_of(payload)));
    return out;
}

// ---- embedding --------------------------------------------------------------------------------------------------------

Tensor lookup(const Tensor& weight, const Tensor& ids, double scale, const Tensor& dropped) {
    const c10::cuda::CUDAGuard guard(weight.device());
    std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
    shape.push_back(weight.size(1));
    Tensor out = at::empty(shape, weight.options());
    check(peer_embedding(ids.data_ptr(), static_cast<int>(ids.element_size()), ids.numel(), weight.data_ptr(),
                         code_of(weight.scalar_type(), "weight"), weight.size(0), weight.size(1), static_cast<float>(scale),
                         out.data_ptr(), static_cast<int64_t*>(ptr(dropped)), stream_of(weight)));
    return out;
}

struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, double scale, int64_t padding_idx,
                          const OptTensor& dropped) {
        ctx->save_for_backward({ids});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding_idx;
        ctx->saved_data["rows"] = weight.size(0);
        return lookup(weight, ids, scale, dropped.value_or(Tensor()));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor ids = ctx->get_saved_variables()[0], grad = grads[0];
        const int64_t V = ctx->saved_data["rows"].toInt(), D = grad.size(-1);
        variable_list g(1);
        {
            const at::AutoGradMode off(false);
            const c10::cuda::CUDAGuard guard(grad.device());
            const Tensor rows = as_rows(grad);
            g[0] = at::empty({V, D}, grad.options());
            const int64_t bytes = peer_embedding_workspace(ids.numel(), D);
            const Tensor ws = workspace(bytes, grad);
            check(peer_embedding_backward(ids.data_ptr(), static_cast<int>(ids.element_size()), ids.numel(), rows.data_ptr(),
                                          rows.stride(0), code_of(grad.scalar_type(), "grad"), V, D,
                                          static_cast<float>(ctx->saved_data["scale"].toDouble()), ctx->saved_data["padding"].toInt(),
                                          g[0].data_ptr(), ptr(ws), bytes, stream_of(grad)));
        }
        g = once(std::move(g));
        return {g[0], Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor embedding(const Tensor& ids_in, const Tensor& weight, double scale, std::optional<int64_t> padding_idx, const OptTensor& dropped) {
    refuse_tangent(weight, "weight");
    need_cuda(weight, "weight");
    code_of(weight.scalar_type(), "weight");
    if (weight.dim() != 2 || weight.size(0) < 1 || weight.size(1) < 1)
        throw py::value_error(text("weight must be a [rows, width] table, got ", weight.sizes()));
    if (!weight.is_contiguous() || weight.is_neg()) throw py::value_error("weight must be contiguous");
    if (ids_in.scalar_type() != at::kInt && ids_in.scalar_type() != at::kLong)
        throw py::type_error(text("ids is ", dtype_name(ids_in.scalar_type()), ", expected int32 or int64"));
    if (ids_in.device() != weight.device())
        throw std::runtime_error(text("ids is on ", ids_in.device(), ", weight on ", weight.device()));
    if (padding_idx && (*padding_idx < 0 || *padding_idx >= weight.size(0)))
        throw py::value_error(text("padding_idx=", *padding_idx, " of a table of ", weight.size(0), " rows"));
    if (dropped && (dropped->scalar_type() != at::kLong || dropped->numel() != 1 || dropped->device() != weight.device()))
        throw py::type_error("dropped must be one int64 on the table's device");
    if (ids_in.numel() > PEER_SORT_IDS_MAX || weight.size(0) > PEER_SORT_IDS_MAX)
        throw py::value_error("more than 2^31 - 2 ids or table rows");
    const Tensor ids = ids_in.contiguous();
    if (at::GradMode::is_enabled() && weight.requires_grad())
        return EmbeddingNode::apply(weight, ids, scale, padding_idx.value_or(-1), dropped);
    return lookup(weight, ids, scale, dropped.value_or(Tensor()));
}

// ---- for autograd.py: the norm inside the block's node ------------------------------------------------------------------

// The forward pass's values again (peer_block_norm), and the statistics [2, rows].
std::pair<Tensor, Tensor> block_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    const NormCodes c = check_norm(x, w, b, eps);
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor rows = as_rows(x).contiguous(), w32 = w.defined() ? w.to(at::kFloat) : w, b32 = b.defined() ? b.to(at::kFloat) : b;
    const int64_t R = rows.size(0), D = rows.size(1);
    Tensor y = at::empty(x.sizes(), x.options()), stats = at::empty({2, R}, x.options().dtype(at::kFloat));
    float* mean = stats.data_ptr<float>();
    check(peer_block_norm(rows.data_ptr(), c.x, static_cast<const float*>(ptr(w32)), static_cast<const float*>(ptr(b32)),
                          static_cast<float>(eps), R, D, y.data_ptr(), mean, mean + R, stream_of(x)));
    return {y, stats};
}

std::tuple<OptTensor, OptTensor, OptTensor> block_norm_grad(const Tensor& grad, const Tensor& x, const Tensor& stats, const OptTensor& weight,
                                                            const OptTensor& bias, const Tensor& add, bool want_x, bool want_w, bool want_b) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    const variable_list g = norm_backward(grad, x, Tensor(), Tensor(), stats, w, check_norm(x, w, b, 0.0),
                                          w.defined() ? w.scalar_type() : at::kFloat, b.defined() ? b.scalar_type() : at::kFloat,
                                          want_x, want_w, want_b, add);
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    return {opt(g[0]), opt(g[1]), opt(g[2])};
}

void check_norm_arguments(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    check_norm(x, weight.value_or(Tensor()), bias.value_or(Tensor()), eps);
}

// for peer.py: whether any of the layer's tensors carries one
bool any_tangent(const std::vector<OptTensor>& tensors) {
    for (const auto& t : tensors)
        if (t && has_tangent(*t)) return true;
    return false;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.attr("abi_version") = PEER_B200_ABI_VERSION;
    m.def("layer_norm", &layer_norm);
    m.def("pack_rows", &pack_rows);
    m.def("unpack_rows", &unpack_rows);
    m.def("embedding", &embedding);
    m.def("block_norm", &block_norm);
    m.def("block_norm_grad", &block_norm_grad);
    m.def("check_norm_arguments", &check_norm_arguments);
    m.def("any_tangent", &any_tangent);
}
