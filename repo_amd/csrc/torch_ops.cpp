// `_cs_torch`, a CPython extension on torch's C++ tensors, for what costs the host
// most in Python: the autograd nodes of group norm, tokens' log-probabilities and the
// policy loss (their backward then runs in the engine's thread without the
// interpreter), and the checks that an AdamW step makes of every parameter and
// gradient.  The kernels are reached through the C ABI of libcubicsplat_hip.so, as
// everywhere.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <Python.h>
#include <optional>

#include "../../include/cubicsplat_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc, const char* what) {
    TORCH_CHECK(rc == CS_OK, what, ": ",
                rc == CS_ERR_ARGS ? "invalid arguments" : "HIP launch failure", " (status ", rc,
                ")");
}

int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Sizes {
    int64_t n, s;
    int32_t c;
    explicit Sizes(const Tensor& x)
        : n(x.size(0)), s(x.numel() / (x.size(0) * x.size(1))), c((int32_t)x.size(1)) {}
};

Tensor workspace(const Tensor& x, const Sizes& z, int64_t groups, int backward) {
    const size_t elems = cs_group_norm_workspace_elems(z.n, z.s, z.c, (int32_t)groups,
                                                       type_code(x), backward);
    return at::empty({(int64_t)elems}, x.options().dtype(at::kFloat));
}

hipStream_t stream(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()); }

// The capture that x's current stream belongs to, 0 for none, -1 where it cannot be told.
int64_t capture_of(const Tensor& x) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(stream(x), &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return -1;
    }
    return status == hipStreamCaptureStatusNone ? 0 : (int64_t)id;
}

// t if its channels lie together without gaps, else a copy that does.
Tensor channels_last(const Tensor& t) {
    const Tensor last = t.movedim(1, -1);
    return last.is_contiguous() ? t : last.contiguous().movedim(-1, 1);
}

int affine_code(const Tensor& weight, const Tensor& bias) {
    return weight.defined() ? type_code(weight) : bias.defined() ? type_code(bias) : 0;
}

Tensor forward(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups,
               double eps, int64_t act, Tensor* stats) {
    const Sizes z(x);
    Tensor y = at::empty_like(x);
    const Tensor work = workspace(x, z, groups, 0);
    float *mean = nullptr, *rstd = nullptr;
    if (stats) {
        *stats = at::empty({2, z.n, groups}, x.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
        rstd = mean + z.n * groups;
    }
    check(cs_group_norm_forward(x.data_ptr(), z.n, z.s, z.c, (int32_t)groups, type_code(x),
                                pointer(weight), pointer(bias), affine_code(weight, bias), eps,
                                (int32_t)act, work.data_ptr<float>(), mean, rstd, y.data_ptr(),
                                stream(x)),
          "cs_group_norm_forward");
    return y;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x,
                          const std::optional<Tensor>& given_weight,
                          const std::optional<Tensor>& given_bias, int64_t groups, double eps,
                          int64_t act) {
        const Tensor weight = given_weight.value_or(Tensor()), bias = given_bias.value_or(Tensor());
        Tensor stats;
        Tensor y = ::forward(x, weight, bias, groups, eps, act, &stats);
        ctx->save_for_backward({x, weight, bias, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        const Sizes z(x);
        variable_list out(6);
        {
            at::AutoGradMode off(false);
            const Tensor dy = channels_last(grads[0]);
            // The node's edges are those of the tensors that there are.
            if (ctx->needs_input_grad(0)) out[0] = at::empty_like(x);
            if (weight.defined() && ctx->needs_input_grad(1)) out[1] = at::empty_like(weight);
            if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1))
                out[2] = at::empty_like(bias);
            const Tensor work = workspace(x, z, groups, 1);
            const float* mean = stats.data_ptr<float>();
            check(cs_group_norm_backward(
                      x.data_ptr(), dy.data_ptr(), z.n, z.s, z.c, (int32_t)groups, type_code(x),
                      pointer(weight), pointer(bias), affine_code(weight, bias),
                      (int32_t)ctx->saved_data["act"].toInt(), mean, mean + z.n * groups,
                      work.data_ptr<float>(), pointer(out[0]), pointer(out[1]), pointer(out[2]),
                      stream(x)),
                  "cs_group_norm_backward");
        }
        if (at::GradMode::is_enabled()) {
            // Under create_graph the gradients get a node that refuses to be
            // differentiated, rather than none.
            variable_list given;
            for (int k = 0; k < 3; ++k)
                if (out[k].defined()) given.push_back(out[k].detach().set_requires_grad(true));
            auto refuse = std::make_shared<torch::autograd::DelayedError>(
                "group_norm is differentiable once", (int)given.size());
            variable_list refused = (*refuse)(std::move(given));
            for (int k = 0, j = 0; k < 3; ++k)
                if (out[k].defined()) out[k] = refused[j++];
        }
        return out;
    }
};

std::optional<Tensor> optional_tensor(PyObject* o) {
    if (o == Py_None) return std::nullopt;
    return THPVariable_Unpack(o);
}

bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

// group_norm(x, weight | None, bias | None, groups, eps, act): x channels last
// without gaps, all arguments checked by the caller.
PyObject* py_group_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 6, "group_norm: expected 6 arguments");
    TORCH_CHECK_TYPE(THPVariable_Check(args[0]), "group_norm: x must be a tensor");
    for (int k = 1; k < 3; ++k)
        TORCH_CHECK_TYPE(args[k] == Py_None || THPVariable_Check(args[k]),
                         "group_norm: weight and bias must be tensors or None");
    const Tensor& x = THPVariable_Unpack(args[0]);
    const std::optional<Tensor> weight = optional_tensor(args[1]), bias = optional_tensor(args[2]);
    const int64_t groups = PyLong_AsLongLong(args[3]), act = PyLong_AsLongLong(args[5]);
    const double eps = PyFloat_AsDouble(args[4]);
    if (PyErr_Occurred()) return nullptr;
    TORCH_CHECK_VALUE(x.is_cuda() && type_code(x) >= 0 && x.dim() >= 2 && x.numel() > 0 &&
                          x.movedim(1, -1).is_contiguous(),
                      "group_norm: x must be on the GPU, channels last without gaps");
    for (const auto& p : {weight, bias})
        TORCH_CHECK_VALUE(!p || (p->device() == x.device() && p->numel() == x.size(1) &&
                                 type_code(*p) >= 0 && p->is_contiguous()),
                          "group_norm: weight and bias must lie beside x");
    // A tangent of forward mode goes to the node too, which refuses it.
    const bool node = (at::GradMode::is_enabled() &&
                       (x.requires_grad() || (weight && weight->requires_grad()) ||
                        (bias && bias->requires_grad()))) ||
                      has_tangent(x) || (weight && has_tangent(*weight)) ||
                      (bias && has_tangent(*bias));
    Tensor y = node ? GroupNorm::apply(x, weight, bias, groups, eps, act)
                    : forward(x, weight.value_or(Tensor()), bias.value_or(Tensor()), groups, eps,
                              act, nullptr);
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// A gradient under create_graph gets a node that refuses to be differentiated, rather
// than none.
Tensor once(Tensor grad, const char* what) {
    if (!at::GradMode::is_enabled()) return grad;
    auto refuse = std::make_shared<torch::autograd::DelayedError>(what, 1);
    return (*refuse)(variable_list{grad.detach().set_requires_grad(true)})[0];
}

// Logits as [batch, length, vocab] rows that the entry points can read, and what belongs
// to them: whole-number tokens and a mask, contiguous.
struct Rows {
    Tensor z, tokens, mask;
    double temperature;

    Rows(Tensor z_, Tensor tokens_, Tensor mask_, double t)
        : z(std::move(z_)), tokens(std::move(tokens_)), mask(std::move(mask_)), temperature(t) {}

    static Rows of(const Tensor& logits, const Tensor& tokens, const std::optional<Tensor>& mask,
                   double temperature) {
        Tensor z = logits.detach();
        if (z.dim() < 3) z = z.reshape({1, z.dim() < 2 ? 1 : z.size(0), z.size(-1)});
        else if (z.dim() > 3) z = z.reshape({-1, z.size(-2), z.size(-1)});
        if (z.size(2) != 1 && z.stride(2) != 1) z = z.contiguous();
        return Rows(z, tokens.detach().to(at::kLong).contiguous(),
                    mask ? mask->detach().contiguous() : Tensor(), temperature);
    }
    int64_t batch() const { return z.size(0); }
    int64_t length() const { return z.size(1); }
    at::TensorOptions fp32() const { return z.options().dtype(at::kFloat); }
    const uint8_t* mask_pointer() const { return (const uint8_t*)pointer(mask); }

    // The gradient for slopes of the log-probabilities, times *factor; into `into`, which
    // holds it for a factor of one, or a new tensor.
    Tensor gradient(const Tensor& stats, const Tensor& slopes, const Tensor& factor, Tensor into,
                    at::IntArrayRef shape) const {
        const bool fresh = !into.defined();
        if (fresh) into = at::empty(shape, z.options());
        check(cs_token_logprobs_backward(z.data_ptr(), batch(), length(), z.size(2), z.stride(0),
                                         z.stride(1), type_code(z), tokens.data_ptr<int64_t>(),
                                         mask_pointer(), temperature, stats.data_ptr<float>(),
                                         slopes.data_ptr<float>(), (const float*)pointer(factor),
                                         fresh ? 0 : 1, into.data_ptr(), stream(z)),
              "cs_token_logprobs_backward");
        return into;
    }
};

Tensor logprobs_forward(const Rows& a, Tensor* stats) {
    *stats = at::empty({a.batch(), a.length(), 2}, a.fp32());
    Tensor lp = at::empty(a.tokens.sizes(), a.fp32());
    check(cs_token_logprobs_forward(a.z.data_ptr(), a.batch(), a.length(), a.z.size(2),
                                    a.z.stride(0), a.z.stride(1), type_code(a.z),
                                    a.tokens.data_ptr<int64_t>(), a.mask_pointer(), a.temperature,
                                    stats->data_ptr<float>(), lp.data_ptr<float>(), stream(a.z)),
          "cs_token_logprobs_forward");
    return lp;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                          const std::optional<Tensor>& mask, double temperature) {
        const Rows a = Rows::of(logits, tokens, mask, temperature);
        Tensor stats, lp = logprobs_forward(a, &stats);
        ctx->save_for_backward({a.z, a.tokens, a.mask, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["shape"] = logits.sizes().vec();
        return lp;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Rows a(saved[0], saved[1], saved[2], ctx->saved_data["temperature"].toDouble());
        Tensor grad;
        {
            at::AutoGradMode off(false);
            grad = a.gradient(saved[3], grads[0].contiguous(), Tensor(), Tensor(),
                              ctx->saved_data["shape"].toIntVector());
        }
        return {once(grad, "token_logprobs is differentiable once"), Tensor(), Tensor(), Tensor()};
    }
};

// What the loss takes besides the rows: constants, and numbers.
struct LossArgs {
    Tensor advantages, old_logprobs, ref_logprobs;
    double clip_low, clip_high, kl_weight, scale;
    int64_t reduction;
};

// [loss, KL, clipped], the log-probabilities; with `grad` the gradient for an incoming one.
struct LossOut { Tensor out, logprobs, stats, slopes, grad; };

LossOut loss_forward(const Rows& a, const LossArgs& f, at::IntArrayRef shape, bool with_grad) {
    LossOut y;
    y.out = at::empty({3}, a.fp32());
    y.logprobs = at::empty(a.tokens.sizes(), a.fp32());
    y.slopes = at::empty({a.batch(), a.length()}, a.fp32());
    y.stats = at::empty({a.batch(), a.length(), 2}, a.fp32());
    if (with_grad) y.grad = at::empty(shape, a.z.options());
    const Tensor work = at::empty(
        {(int64_t)cs_policy_loss_workspace_elems(a.batch(), a.length())}, a.fp32());
    const Tensor adv = f.advantages.detach().to(at::kFloat).expand(a.tokens.sizes()).reshape(
        {a.batch(), a.length()});
    const Tensor old = f.old_logprobs.detach().to(at::kFloat).contiguous();
    const Tensor ref = f.ref_logprobs.defined()
                           ? f.ref_logprobs.detach().to(at::kFloat).contiguous() : Tensor();
    check(cs_policy_loss(a.z.data_ptr(), a.batch(), a.length(), a.z.size(2), a.z.stride(0),
                         a.z.stride(1), type_code(a.z), a.tokens.data_ptr<int64_t>(),
                         a.mask_pointer(), a.temperature, adv.data_ptr<float>(), adv.stride(0),
                         adv.stride(1), old.data_ptr<float>(), (const float*)pointer(ref),
                         f.clip_low, f.clip_high, f.kl_weight, (int32_t)f.reduction, f.scale,
                         work.data_ptr<float>(), y.stats.data_ptr<float>(),
                         y.slopes.data_ptr<float>(), y.logprobs.data_ptr<float>(),
                         y.out.data_ptr<float>(), pointer(y.grad), stream(a.z)),
          "cs_policy_loss");
    return y;
}

// Loss, log-probabilities, KL estimate and clipped share: tensors of their own, which callers may write
// in place, and not views of one.
variable_list results(const LossOut& y) {
    return {y.out[0].variable_data(), y.logprobs, y.out[1].variable_data(),
            y.out[2].variable_data()};
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                                 const std::optional<Tensor>& mask, double temperature,
                                 const LossArgs* f) {
        const Rows a = Rows::of(logits, tokens, mask, temperature);
        LossOut y = loss_forward(a, *f, logits.sizes(), true);
        variable_list out = results(y);
        ctx->mark_non_differentiable({out[1], out[2], out[3]});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({a.z, a.tokens, a.mask, y.stats, y.slopes});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["shape"] = logits.sizes().vec();
        ctx->saved_data["grad"] = y.grad;
        ctx->saved_data["capture"] = capture_of(a.z);
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        // The gradient for an incoming one is there; another one's is computed from the
        // logits, not from that one's rounded values.  A second backward pass finds it given
        // away.  Of a loss that is in another graph than this pass, or of which one is in none, it
        // is left: replays of one without the other would find what the last has made of it.
        const variable_list saved = ctx->get_saved_variables();
        const Rows a(saved[0], saved[1], saved[2], ctx->saved_data["temperature"].toDouble());
        Tensor grad;
        auto held = ctx->saved_data.find("grad");
        if (held != ctx->saved_data.end()) {
            const int64_t capture = capture_of(a.z);
            if (capture >= 0 && capture == ctx->saved_data["capture"].toInt())
                grad = held->second.toTensor();
            ctx->saved_data.erase("grad");
        }
        if (!grads[0].defined()) return variable_list(5);
        {
            at::AutoGradMode off(false);
            grad = a.gradient(saved[3], saved[4], grads[0].to(at::kFloat).contiguous(), grad,
                              ctx->saved_data["shape"].toIntVector());
        }
        return {once(grad, "policy_loss is differentiable once"), Tensor(), Tensor(), Tensor(),
                Tensor()};
    }
};

bool wants_node(const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || has_tangent(t);
}

void check_rows(const char* what, PyObject* const* args) {
    for (int k : {0, 1})
        TORCH_CHECK_TYPE(THPVariable_Check(args[k]), what, ": expected tensors");
    TORCH_CHECK_TYPE(args[2] == Py_None || THPVariable_Check(args[2]), what,
                     ": mask must be a tensor or None");
    const Tensor &z = THPVariable_Unpack(args[0]), &t = THPVariable_Unpack(args[1]);
    TORCH_CHECK_VALUE(z.is_cuda() && type_code(z) >= 0 && z.dim() >= 1 && t.numel() > 0 &&
                          z.numel() > 0 && z.numel() / z.size(-1) == t.numel() &&
                          t.device() == z.device(),
                      what, ": logits and tokens do not fit");
    if (args[2] != Py_None) {
        const Tensor& m = THPVariable_Unpack(args[2]);
        TORCH_CHECK_VALUE(m.scalar_type() == at::kBool && m.sizes() == t.sizes() &&
                              m.device() == z.device(), what, ": the mask does not fit");
    }
}

// token_logprobs(logits, tokens, mask | None, temperature): all arguments checked by the caller.
PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 4, "token_logprobs: expected 4 arguments");
    check_rows("token_logprobs", args);
    const Tensor &logits = THPVariable_Unpack(args[0]), &tokens = THPVariable_Unpack(args[1]);
    const std::optional<Tensor> mask = optional_tensor(args[2]);
    const double temperature = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    Tensor stats;
    Tensor lp = wants_node(logits)
                    ? TokenLogprobs::apply(logits, tokens, mask, temperature)
                    : logprobs_forward(Rows::of(logits, tokens, mask, temperature), &stats);
    return THPVariable_Wrap(std::move(lp));
    END_HANDLE_TH_ERRORS
}

// policy_loss(logits, tokens, mask | None, temperature, advantages, old, ref | None, clip_low,
// clip_high, kl_weight, reduction, scale) -> (loss, logprobs, kl, clipped): all arguments
// checked by the caller.
PyObject* py_policy_loss(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 12, "policy_loss: expected 12 arguments");
    check_rows("policy_loss", args);
    for (int k : {4, 5}) TORCH_CHECK_TYPE(THPVariable_Check(args[k]), "policy_loss: expected tensors");
    TORCH_CHECK_TYPE(args[6] == Py_None || THPVariable_Check(args[6]),
                     "policy_loss: ref must be a tensor or None");
    const Tensor &logits = THPVariable_Unpack(args[0]), &tokens = THPVariable_Unpack(args[1]);
    const std::optional<Tensor> mask = optional_tensor(args[2]);
    LossArgs f{THPVariable_Unpack(args[4]), THPVariable_Unpack(args[5]),
               optional_tensor(args[6]).value_or(Tensor()), PyFloat_AsDouble(args[7]),
               PyFloat_AsDouble(args[8]), PyFloat_AsDouble(args[9]), PyFloat_AsDouble(args[11]),
               PyLong_AsLongLong(args[10])};
    const double temperature = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    for (const Tensor& t : {f.old_logprobs, f.ref_logprobs})
        TORCH_CHECK_VALUE(!t.defined() || (t.sizes() == tokens.sizes() &&
                                           t.device() == logits.device()),
                          "policy_loss: the constants do not fit");
    TORCH_CHECK_VALUE(f.advantages.device() == logits.device(),
                      "policy_loss: the constants do not fit");
    variable_list out;
    if (wants_node(logits)) {
        out = PolicyLoss::apply(logits, tokens, mask, temperature, &f);
    } else {
        out = results(loss_forward(Rows::of(logits, tokens, mask, temperature), f, {}, false));
    }
    PyObject* tuple = PyTuple_New(4);
    if (!tuple) return nullptr;
    for (int k = 0; k < 4; ++k) PyTuple_SET_ITEM(tuple, k, THPVariable_Wrap(std::move(out[k])));
    return tuple;
    END_HANDLE_TH_ERRORS
}

// Where and how a tensor's elements lie: what a launch's table says of it as long as
// all of this is unchanged.  order: 0 for the logical one, which the sizes do not
// change; sizes of one have no stride.
struct Place {
    int64_t address, type, numel, order;
    explicit Place(const Tensor& t)
        : address((int64_t)t.const_data_ptr()),
          type((int64_t)t.scalar_type()),
          numel(t.numel()),
          order(0) {
        if (t.is_contiguous()) return;
        uint64_t mix = (uint64_t)t.dim();
        for (int64_t d = 0; d < t.dim(); ++d) {
            const int64_t size = t.size(d);
            mix = (mix ^ (uint64_t)size) * 0x9E3779B97F4A7C15u;
            mix = (mix ^ (uint64_t)(size == 1 ? 0 : t.stride(d))) * 0xC2B2AE3D27D4EB4Fu;
            mix ^= mix >> 29;
        }
        order = (int64_t)mix;
    }
};

// adamw_unchanged(groups, params, sizes, state, keys, values): whether the groups' lists
// of parameters are `params`, one list after the other and sizes[k] of them each, and
// the dict `state` has these keys and values, the same objects in the same order.
PyObject* py_adamw_unchanged(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 6 && PyDict_Check(args[3]), "adamw_unchanged: expected 6 arguments");
    for (int k : {0, 1, 2, 4, 5})
        TORCH_CHECK_TYPE(PyList_Check(args[k]), "adamw_unchanged: expected lists");
    PyObject *params = args[1], *sizes = args[2], *keys = args[4], *values = args[5];
    const Py_ssize_t ngroups = PyList_GET_SIZE(args[0]), n = PyDict_Size(args[3]);
    if (ngroups != PyList_GET_SIZE(sizes) || n != PyList_GET_SIZE(keys) ||
        n != PyList_GET_SIZE(values))
        Py_RETURN_FALSE;
    Py_ssize_t at = 0;
    for (Py_ssize_t k = 0; k < ngroups; ++k) {
        PyObject* group = PyList_GET_ITEM(args[0], k);
        PyObject* list = PyDict_Check(group) ? PyDict_GetItemString(group, "params") : nullptr;
        if (!list || !PyList_Check(list)) Py_RETURN_FALSE;
        const Py_ssize_t size = PyList_GET_SIZE(list);
        if (PyLong_AsSsize_t(PyList_GET_ITEM(sizes, k)) != size ||
            at + size > PyList_GET_SIZE(params))
            Py_RETURN_FALSE;
        for (Py_ssize_t i = 0; i < size; ++i, ++at)
            if (PyList_GET_ITEM(list, i) != PyList_GET_ITEM(params, at)) Py_RETURN_FALSE;
    }
    if (at != PyList_GET_SIZE(params)) Py_RETURN_FALSE;
    PyObject *key, *value;
    Py_ssize_t pos = 0;
    for (Py_ssize_t i = 0; PyDict_Next(args[3], &pos, &key, &value); ++i)
        if (key != PyList_GET_ITEM(keys, i) || value != PyList_GET_ITEM(values, i))
            Py_RETURN_FALSE;
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// adamw_place(tensors, places): writes each tensor's Place into the array by that
// address; adamw_held(tensors, places): whether all still are what it holds.
PyObject* with_places(PyObject* const* args, Py_ssize_t nargs, bool write) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 2 && PyTuple_Check(args[0]), "expected a tuple and an address");
    Place* places = (Place*)PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyTuple_GET_SIZE(args[0]);
    bool same = true;
    for (Py_ssize_t i = 0; i < n && same; ++i) {
        PyObject* o = PyTuple_GET_ITEM(args[0], i);
        TORCH_CHECK_TYPE(THPVariable_Check(o), "expected tensors");
        const Place now(THPVariable_Unpack(o));
        if (write)
            places[i] = now;
        else
            same = now.address == places[i].address && now.type == places[i].type &&
                   now.numel == places[i].numel && now.order == places[i].order;
    }
    return PyBool_FromLong(same);
    END_HANDLE_TH_ERRORS
}

PyObject* py_adamw_place(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return with_places(args, nargs, true);
}

PyObject* py_adamw_held(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return with_places(args, nargs, false);
}

// adamw_current(params, states, keys, tensors, table, steps, gradients): whether
// each parameter still is what its row of the table (int64 [n][8], by address)
// says, and each states[i][keys[i][j]] the object tensors[i][j] (whose place adamw_held
// has found unchanged: the step counts are read by address); with `gradients`,
// whether each parameter has a gradient that can be read as it is, whose address
// goes into the row, and whether all step counts (float pointers, by the address of
// their array) agree.  The count with `gradients`, else 0; -1 where anything is not
// so.
PyObject* py_adamw_current(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 7, "adamw_current: expected 7 arguments");
    for (int k = 0; k < 4; ++k)
        TORCH_CHECK_TYPE(PyList_Check(args[k]) &&
                             PyList_GET_SIZE(args[k]) == PyList_GET_SIZE(args[0]),
                         "adamw_current: expected lists of one length");
    int64_t* table = (int64_t*)PyLong_AsVoidPtr(args[4]);
    float* const* steps = (float* const*)PyLong_AsVoidPtr(args[5]);
    const int gradients = PyObject_IsTrue(args[6]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    double step = 0.0;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* po = PyList_GET_ITEM(args[0], i);
        PyObject* state = PyList_GET_ITEM(args[1], i);
        PyObject* keys = PyList_GET_ITEM(args[2], i);
        PyObject* tensors = PyList_GET_ITEM(args[3], i);
        TORCH_CHECK_TYPE(THPVariable_Check(po) && PyDict_Check(state) && PyTuple_Check(keys) &&
                             PyTuple_Check(tensors) &&
                             PyTuple_GET_SIZE(keys) == PyTuple_GET_SIZE(tensors),
                         "adamw_current: expected tensors, dicts and tuples");
        for (Py_ssize_t j = 0; j < PyTuple_GET_SIZE(keys); ++j) {
            PyObject* held = PyDict_GetItemWithError(state, PyTuple_GET_ITEM(keys, j));
            if (!held && PyErr_Occurred()) return nullptr;
            if (held != PyTuple_GET_ITEM(tensors, j)) return PyFloat_FromDouble(-1.0);
        }
        const Tensor& p = THPVariable_Unpack(po);
        int64_t* row = table + 8 * i;
        if ((int64_t)p.data_ptr() != row[0] || p.numel() != row[5] ||
            type_code(p) != (int)(row[6] & 0xF) || !p.is_contiguous())
            return PyFloat_FromDouble(-1.0);
        if (!gradients) continue;
        const Tensor& g = p.grad();
        if (!g.defined() || g.layout() != at::kStrided || g.scalar_type() != p.scalar_type() ||
            g.device() != p.device() || g.sizes() != p.sizes() || !g.is_contiguous())
            return PyFloat_FromDouble(-1.0);
        row[1] = (int64_t)g.data_ptr();
        if (i == 0) step = *steps[0];
        if (*steps[i] != step) return PyFloat_FromDouble(-1.0);
    }
    return PyFloat_FromDouble(step);
    END_HANDLE_TH_ERRORS
}

// adamw_count(steps, n, value): sets the n step counts.
PyObject* py_adamw_count(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 3, "adamw_count: expected 3 arguments");
    float* const* steps = (float* const*)PyLong_AsVoidPtr(args[0]);
    const Py_ssize_t n = PyLong_AsSsize_t(args[1]);
    const double value = PyFloat_AsDouble(args[2]);
    if (PyErr_Occurred()) return nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) *steps[i] = (float)value;
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// What autograd counts of a tensor's writes in place, for those that it counts.
int64_t version_of(const Tensor& t) {
    return t.is_inference() ? 0
                            : (int64_t)t.unsafeGetTensorImpl()->version_counter().current_version();
}

// adamw_unwritten(params, versions): whether each 16-bit parameter's version counter
// is the one in the array (int64, by address); adamw_written(params, versions): raises
// all counters and then puts those of the 16-bit parameters there (views of one buffer
// share theirs).
PyObject* with_versions(PyObject* const* args, Py_ssize_t nargs, bool write) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(nargs == 2 && PyList_Check(args[0]), "expected a list and an address");
    int64_t* versions = (int64_t*)PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    for (Py_ssize_t i = 0; i < n; ++i)
        TORCH_CHECK_TYPE(THPVariable_Check(PyList_GET_ITEM(args[0], i)), "expected tensors");
    for (Py_ssize_t i = 0; i < n && write; ++i) {
        const Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
        if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
    }
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(args[0], i));
        if (p.scalar_type() == at::kFloat) continue;
        if (write)
            versions[i] = version_of(p);
        else if (version_of(p) != versions[i])
            Py_RETURN_FALSE;
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

PyObject* py_adamw_unwritten(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return with_versions(args, nargs, false);
}

PyObject* py_adamw_written(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    return with_versions(args, nargs, true);
}

PyObject* py_signature_hash(PyObject*, PyObject*) {
    return PyUnicode_FromString(CS_SIGNATURE_HASH);
}

PyMethodDef methods[] = {
    {"group_norm", (PyCFunction)(void (*)(void))py_group_norm, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void (*)(void))py_token_logprobs, METH_FASTCALL, nullptr},
    {"policy_loss", (PyCFunction)(void (*)(void))py_policy_loss, METH_FASTCALL, nullptr},
    {"adamw_unchanged", (PyCFunction)(void (*)(void))py_adamw_unchanged, METH_FASTCALL, nullptr},
    {"adamw_place", (PyCFunction)(void (*)(void))py_adamw_place, METH_FASTCALL, nullptr},
    {"adamw_held", (PyCFunction)(void (*)(void))py_adamw_held, METH_FASTCALL, nullptr},
    {"adamw_current", (PyCFunction)(void (*)(void))py_adamw_current, METH_FASTCALL, nullptr},
    {"adamw_count", (PyCFunction)(void (*)(void))py_adamw_count, METH_FASTCALL, nullptr},
    {"adamw_unwritten", (PyCFunction)(void (*)(void))py_adamw_unwritten, METH_FASTCALL, nullptr},
    {"adamw_written", (PyCFunction)(void (*)(void))py_adamw_written, METH_FASTCALL, nullptr},
    {"signature_hash", py_signature_hash, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cs_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__cs_torch(void) { return PyModule_Create(&module); }
