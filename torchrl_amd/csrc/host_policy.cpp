// Host-side fast path of the token-policy and 8-bit-activation entry points (part of the CPython module _trl_host, host_fast.cpp):
// checks, allocations, autograd nodes and the C-ABI calls in C++, so that a call costs about its launches.  Plumbing only.
//
// process_logits(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask, temperature)
// token_log_prob(logits, action, entropy, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask, temperature)
// checkpointed_linear(x, weight, bias)   quantize(x) -> (codes, exponents)   dequantize(codes, exponents, features, dtype code)
//   -> the result
//   -> None    not a fast-path call (python's general path takes it, and raises what is to be raised)
//   -> int     non-zero status of the C-ABI call
// Eligible: logits [B, V] or [B, T, V] on the current HIP device with dense rows, tokens [B, L], dense lengths / prompt lengths / action, numbers
// as penalties and temperature, bias and mask of the logits' rank or [V].
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/hip/HIPStream.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "../../include/trl_value.h"
#include "host_policy.h"

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

decltype(&trl_process_logits_fwd) g_process_fwd = nullptr;
decltype(&trl_process_logits_bwd) g_process_bwd = nullptr;
decltype(&trl_token_workspace_bytes) g_token_ws = nullptr;
decltype(&trl_token_log_prob_fwd) g_log_prob_fwd = nullptr;
decltype(&trl_token_log_prob_bwd) g_log_prob_bwd = nullptr;
decltype(&trl_act_quantize) g_quantize = nullptr;
decltype(&trl_act_dequantize) g_dequantize = nullptr;
decltype(&trl_act_weight_grad_workspace_bytes) g_weight_grad_ws = nullptr;
decltype(&trl_act_weight_grad) g_weight_grad = nullptr;
decltype(&trl_act_head_fwd) g_head_fwd = nullptr;
decltype(&trl_act_head_bwd) g_head_bwd = nullptr;
decltype(&trl_last_error) g_last_error = nullptr;

int dtype_code(at::ScalarType t) { return t == at::kFloat ? TRL_F32 : t == at::kBFloat16 ? TRL_BF16 : t == at::kHalf ? TRL_F16 : -1; }
at::ScalarType int_type(int wide) { return wide ? at::kLong : at::kInt; }
bool is_int(const at::Tensor &t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }
bool on_current_device(const at::Tensor &t) {
    return t.is_cuda() && c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice().index() == t.device().index();
}
void *stream_of(const at::Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check_status(int rc, const char *what) {
    TORCH_CHECK(rc == 0, "torchrl_amd native call failed (status ", rc, "): ", g_last_error ? g_last_error() : what);
}
bool wants_grad(const at::Tensor &t) { return t.defined() && t.requires_grad() && c10::GradMode::is_enabled(); }
// a tensor with memory of its own kind: no function transform's or subclass's wrapper, no forward-mode tangent, and nothing that records the call
bool plain_tensor(PyObject *o, at::Tensor &t) {
    if (!THPVariable_Check(o) || maybe_recorded()) return false;
    t = THPVariable_Unpack(o);
    using c10::DispatchKey;
    constexpr c10::DispatchKeySet wrapped({DispatchKey::FuncTorchGradWrapper, DispatchKey::FuncTorchBatched, DispatchKey::Functionalize, DispatchKey::Python,
                                           DispatchKey::Negative, DispatchKey::ZeroTensor});
    return !t.key_set().has_any(wrapped) && !t._fw_grad(0).defined();
}
bool optional_tensor(PyObject *o, at::Tensor &t) { return o == Py_None || plain_tensor(o, t); }
bool number(PyObject *o, bool positive, float &out) {
    double x;
    if (PyFloat_CheckExact(o)) x = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) x = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) { PyErr_Clear(); return false; }
    out = (float)x;
    return std::isfinite(x) && std::isfinite(out) && (!positive || out >= FLT_MIN);
}

// The tensors of a call's processing, in the order in which autograd keeps them.
struct Processing {
    at::Tensor logits, tokens, lengths, prompt, bias, mask;
    trl_token_args a{};
    bool steps = false;  // [B, T, V]

    // strides of [V], [B, V] or [B, T, V]; false: not that
    bool row_strides(const at::Tensor &t, int64_t last, int64_t &sb, int64_t &st) const {
        const int64_t nd = steps ? 3 : 2, es = t.element_size();
        if (t.dim() < 1 || t.size(-1) != last || (t.stride(-1) != 1 && last != 1)) return false;
        sb = st = 0;
        if (t.dim() == 1) return true;
        if (t.dim() != nd) return false;
        for (int64_t k = 0; k + 1 < nd; ++k) {
            const int64_t rows = k == 0 ? a.B : a.T;
            if (t.size(k) != 1 && t.size(k) != rows) return false;
            (k == 0 ? sb : st) = t.size(k) == 1 ? 0 : t.stride(k) * es;
        }
        return true;
    }
    bool bias_strides() { return row_strides(bias, a.V, a.bias_sb, a.bias_st); }
    bool mask_strides() { return row_strides(mask, mask.scalar_type() == at::kInt ? (a.V + 31) / 32 : a.V, a.mask_sb, a.mask_st); }
    // pointers and strides of the tensors as they are now
    bool bind() {
        if (logits.defined()) {
            a.logits = logits.data_ptr();
            a.logits_sb = logits.stride(0);
            a.logits_st = steps ? logits.stride(1) : 0;
        }
        a.tokens = tokens.defined() ? tokens.data_ptr() : nullptr;
        a.tokens_sb = tokens.defined() ? tokens.stride(0) : 0;
        a.lengths = lengths.defined() ? lengths.data_ptr() : nullptr;
        a.prompt = prompt.defined() ? prompt.data_ptr() : nullptr;
        a.bias = bias.defined() ? bias.data_ptr() : nullptr;
        a.mask = mask.defined() ? mask.data_ptr() : nullptr;
        return true;
    }

    // o: tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask, temperature; false: not a fast-path call
    bool parse(PyObject *z, PyObject *const *o) {
        if (!plain_tensor(z, logits)) return false;
        const int64_t nd = logits.dim();
        a.dtype = dtype_code(logits.scalar_type());
        if (nd < 2 || nd > 3 || a.dtype < 0 || !on_current_device(logits) || logits.numel() == 0 || logits.stride(-1) != 1) return false;
        steps = nd == 3;
        a.B = logits.size(0);
        a.T = steps ? logits.size(1) : 1;
        a.V = logits.size(-1);
        if (!optional_tensor(o[0], tokens) || !optional_tensor(o[1], lengths) || !optional_tensor(o[2], prompt) || !optional_tensor(o[6], bias) ||
            !optional_tensor(o[7], mask))
            return false;
        if (!number(o[3], true, a.rep) || !number(o[4], false, a.pres) || !number(o[5], false, a.freq) || !number(o[8], true, a.temp)) return false;
        const auto dev = logits.device();
        const bool penalised = a.rep != 1.0f || a.pres != 0.0f || a.freq != 0.0f;
        if (tokens.defined()) {
            if (!is_int(tokens) || tokens.device() != dev || tokens.dim() != 2 || tokens.size(0) != a.B || (tokens.stride(1) != 1 && tokens.size(1) > 1)) return false;
            if (lengths.defined() ? !is_int(lengths) || lengths.device() != dev || lengths.sizes() != logits.sizes().slice(0, nd - 1) || !lengths.is_contiguous() : steps)
                return false;
            if (prompt.defined() && (!is_int(prompt) || prompt.device() != dev || prompt.dim() != 1 || prompt.size(0) != a.B || !prompt.is_contiguous()))
                return false;
            a.L = tokens.size(1);
            if (!penalised || a.L == 0) {
                tokens = lengths = prompt = at::Tensor();
                a.L = 0;
            }
        } else if (penalised || lengths.defined() || prompt.defined()) {
            return false;
        }
        a.tokens_wide = tokens.defined() && tokens.scalar_type() == at::kLong;
        a.lengths_wide = lengths.defined() && lengths.scalar_type() == at::kLong;
        a.prompt_wide = prompt.defined() && prompt.scalar_type() == at::kLong;
        if (bias.defined()) {
            const int code = dtype_code(bias.scalar_type());
            if (code < 0 || bias.device() != dev || wants_grad(bias) || !bias_strides()) return false;
            a.bias_kind = 1 + code;
        }
        if (mask.defined()) {
            const bool bits = mask.scalar_type() == at::kInt;
            if ((!bits && mask.scalar_type() != at::kBool) || mask.device() != dev || !mask_strides()) return false;
            a.mask_kind = bits ? TRL_MASK_BITS : TRL_MASK_BOOL;
        }
        return bind();
    }
    int64_t rows() const { return a.B * a.T; }
    bool reads_sign() const { return a.tokens && a.rep != 1.0f; }
};

// A hook hands back what it likes in place of a kept tensor; the kernels read what the kept sizes say, so anything but another layout is refused.
void check_kept(const at::Tensor &t, const at::Device &device, bool fits, const char *what) {
    TORCH_CHECK(t.layout() == at::kStrided && t.device() == device && fits, "torchrl_amd: the kept ", what,
                " came back from its saved-tensor hook with another type, shape or device");
}
void check_kept(const at::Tensor &t, const at::Device &device, at::ScalarType type, int64_t numel, const char *what) {
    check_kept(t, device, t.scalar_type() == type && t.numel() == numel, what);
}

// What a node keeps of a Processing: the tensors through SavedVariable (writes in place are noticed, hooks are honoured).
struct KeptProcessing {
    SavedVariable t[6];
    trl_token_args a{};
    bool steps = false;
    std::vector<int64_t> sizes;
    at::TensorOptions options;
    void keep(const Processing &p, bool with_logits) {
        const at::Tensor *all[6] = {&p.logits, &p.tokens, &p.lengths, &p.prompt, &p.bias, &p.mask};
        for (int k = with_logits ? 0 : 1; k < 6; ++k)
            if (all[k]->defined()) t[k] = SavedVariable(*all[k], false);
        a = p.a;
        steps = p.steps;
        sizes = p.logits.sizes().vec();
        options = p.logits.options();
    }
    Processing get() {
        Processing p;
        at::Tensor *all[6] = {&p.logits, &p.tokens, &p.lengths, &p.prompt, &p.bias, &p.mask};
        for (int k = 0; k < 6; ++k) *all[k] = t[k].unpack();
        p.a = a;
        p.a.logits = nullptr;
        p.steps = steps;
        const at::Device dev = options.device();
        if (p.logits.defined()) check_kept(p.logits, dev, dtype_code(p.logits.scalar_type()) == a.dtype && p.logits.sizes() == sizes, "logits");
        if (p.tokens.defined())
            check_kept(p.tokens, dev, p.tokens.scalar_type() == int_type(a.tokens_wide) && p.tokens.dim() == 2 && p.tokens.size(0) == a.B && p.tokens.size(1) == a.L,
                       "tokens");
        if (p.lengths.defined()) check_kept(p.lengths, dev, int_type(a.lengths_wide), a.B * a.T, "lengths");
        if (p.prompt.defined()) check_kept(p.prompt, dev, int_type(a.prompt_wide), a.B, "prompt lengths");
        if (p.bias.defined()) check_kept(p.bias, dev, 1 + dtype_code(p.bias.scalar_type()) == a.bias_kind, "bias");
        if (p.mask.defined()) check_kept(p.mask, dev, p.mask.scalar_type() == (a.mask_kind == TRL_MASK_BITS ? at::kInt : at::kBool), "mask");
        // a hook may hand back the values in another layout: the strides are those of the tensors as they are now
        for (at::Tensor *t : {&p.lengths, &p.prompt})
            if (t->defined()) *t = t->contiguous();
        for (at::Tensor *t : {&p.logits, &p.tokens, &p.bias, &p.mask})
            if (t->defined() && t->stride(-1) != 1) *t = t->contiguous();
        TORCH_CHECK((!p.bias.defined() || p.bias_strides()) && (!p.mask.defined() || p.mask_strides()), "torchrl_amd: a kept bias or mask changed its shape");
        p.bind();
        return p;
    }
    void release() { for (auto &v : t) v.reset_data(); }
};

// A gradient of a result that was computed before a recording began has no operator to write down: the recording would lack the kernel.
void check_not_recorded() {
    TORCH_CHECK(!c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() && !torch::jit::tracer::isTracing(),
                "torchrl_amd: this gradient cannot be recorded: record its forward pass too");
}

// The gradients of these operators are not differentiable again: where the incoming ones are, the results say so when that is tried.
bool differentiable(const variable_list &grads) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const auto &g : grads)
        if (g.defined() && g.requires_grad()) return true;
    return false;
}
variable_list once(variable_list &&grads, bool asked_again) {
    if (!asked_again) return std::move(grads);
    for (auto &g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
    return (*error)(std::move(grads));
}

struct ProcessLogitsBackward : torch::autograd::Node {
    KeptProcessing kept;
    variable_list apply(variable_list &&grads) override {
        if (!grads[0].defined()) return {at::Tensor()};
        check_not_recorded();
        const bool again = differentiable(grads);
        at::Tensor d;
        {
            c10::DeviceGuard guard(grads[0].device());
            c10::AutoGradMode off(false);
            Processing p = kept.get();
            const at::Tensor g = grads[0].contiguous();
            d = at::empty(kept.sizes, kept.options);
            p.a.grad_out = g.data_ptr();
            p.a.out = d.data_ptr();
            p.a.out_st = p.a.V;
            p.a.out_sb = p.a.T * p.a.V;
            check_status(g_process_bwd(stream_of(d), &p.a), "trl_process_logits_bwd");
        }
        return once({d}, again);
    }
    void release_variables() override { kept.release(); }
    std::string name() const override { return "ProcessLogitsBackward"; }
};

struct TokenLogProbBackward : torch::autograd::Node {
    KeptProcessing kept;
    SavedVariable action, entropy, stats;
    at::Tensor row_grad(const at::Tensor &g) { return g.defined() ? g.to(at::kFloat).contiguous() : g; }
    variable_list apply(variable_list &&grads) override {
        at::Tensor g_lp = grads[0], g_h = grads.size() > 1 ? grads[1] : at::Tensor(), d;
        if (!g_lp.defined() && !g_h.defined()) return {at::Tensor()};
        check_not_recorded();
        const bool again = differentiable(grads);
        {
            c10::DeviceGuard guard((g_lp.defined() ? g_lp : g_h).device());
            c10::AutoGradMode off(false);
            Processing p = kept.get();
            const at::Tensor act = action.unpack().contiguous(), st = stats.unpack().contiguous(),
                             h = g_h.defined() ? entropy.unpack(shared_from_this()).contiguous() : at::Tensor();
            const at::Device dev = kept.options.device();
            check_kept(act, dev, int_type(p.a.action_wide), p.rows(), "action");
            check_kept(st, dev, at::kFloat, 2 * p.rows(), "statistics");
            if (h.defined()) check_kept(h, dev, at::kFloat, p.rows(), "entropy");
            g_lp = row_grad(g_lp);
            g_h = row_grad(g_h);
            d = at::empty(kept.sizes, kept.options);
            p.a.action = act.data_ptr();
            p.a.stats = st.data_ptr<float>();
            p.a.entropy = h.defined() ? h.data_ptr<float>() : nullptr;
            p.a.g_log_prob = g_lp.defined() ? g_lp.data_ptr<float>() : nullptr;
            p.a.g_entropy = g_h.defined() ? g_h.data_ptr<float>() : nullptr;
            p.a.out = d.data_ptr();
            p.a.out_st = p.a.V;
            p.a.out_sb = p.a.T * p.a.V;
            check_status(g_log_prob_bwd(stream_of(d), &p.a), "trl_token_log_prob_bwd");
        }
        return once({d}, again);
    }
    void release_variables() override {
        kept.release();
        action.reset_data();
        entropy.reset_data();
        stats.reset_data();
    }
    std::string name() const override { return "TokenLogProbBackward"; }
};

// (N, D) view of [*B, D] with dense rows
at::Tensor as_rows(const at::Tensor &x) {
    const at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
void empty_kept(const at::Tensor &x, at::Tensor &codes, at::Tensor &exponents) {
    auto shape = x.sizes().vec();
    const int64_t blocks = (shape.back() + 31) / 32;
    shape.back() = blocks * 32;
    codes = at::empty(shape, x.options().dtype(at::kChar));
    shape.back() = blocks;
    exponents = at::empty(shape, x.options().dtype(at::kByte));
}
int quantize(const at::Tensor &x, at::Tensor &codes, at::Tensor &exponents) {
    empty_kept(x, codes, exponents);
    const at::Tensor r = as_rows(x);
    return g_quantize(stream_of(x), dtype_code(x.scalar_type()), r.data_ptr(), r.stride(0), r.size(0), r.size(1), (int8_t *)codes.data_ptr(),
                      (uint8_t *)exponents.data_ptr());
}
// the layer of one output (w, b) of x, which is quantized on the way if it is to be kept
int head(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, bool keep, at::Tensor &y, at::Tensor &codes, at::Tensor &exponents) {
    auto shape = x.sizes().vec();
    shape.back() = 1;
    y = at::empty(shape, x.options());
    if (keep) empty_kept(x, codes, exponents);
    const at::Tensor r = as_rows(x), row = w.contiguous();
    return g_head_fwd(stream_of(x), dtype_code(x.scalar_type()), r.data_ptr(), r.stride(0), r.size(0), r.size(1), row.data_ptr(),
                      b.defined() ? b.data_ptr() : nullptr, keep ? (int8_t *)codes.data_ptr() : nullptr, keep ? (uint8_t *)exponents.data_ptr() : nullptr,
                      y.data_ptr());
}

// Up to here a layer of one output runs in one pass over x, whether x is kept or not: the same bits in training and evaluation.  Against the library's
// product and a quantization, us, bf16: 8192 x 4096 19 and 36, 256 x 16384 17 and 20, 300 x 65536 75 and 88; a wave walks a row, so with few rows the
// width decides: 1 x 16384 14 and 19, 1 x 65536 51 and 49, 64 x 65536 58 and 52, 1000 x 100000 158 and 166 -- wider ones are the library's.  Without
// keeping: 4096 x 4096 5 and 15, 1 x 65536 26 and 47.  fp32 4 to 10 times ahead of the library's product.
constexpr int64_t kHeadFeatures = 65536;

struct CheckpointedLinearBackward : torch::autograd::Node {
    SavedVariable codes, exponents, weight;
    int64_t features = 0;
    bool need_x = false, need_w = false, need_b = false;
    variable_list apply(variable_list &&grads) override {
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
        check_not_recorded();
        const bool again = differentiable(grads);
        at::Tensor dx, dw, db;
        {
            c10::DeviceGuard guard(grads[0].device());
            c10::AutoGradMode off(false);
            const at::Tensor &g = grads[0];
            at::Tensor dy = as_rows(g);
            const int64_t N = dy.size(0), O = dy.size(1);
            const bool w = need_w && task_should_compute_output(1), b = need_b && task_should_compute_output(2), head = w && O == 1;
            at::Tensor row;  // one output: the input's gradient beside the weight's
            if (need_x && task_should_compute_output(0)) {
                auto shape = g.sizes().vec();
                shape.back() = features;
                if (head) {
                    row = weight.unpack().contiguous();
                    check_kept(row, dy.device(), dy.scalar_type(), features, "weight");
                    dx = at::empty(shape, dy.options());
                } else {
                    dx = at::_unsafe_view(at::mm(dy, weight.unpack()), shape);
                }
            }
            if (w || b) {
                const at::Tensor c = w ? codes.unpack().contiguous() : at::Tensor(), e = w ? exponents.unpack().contiguous() : at::Tensor();
                const int64_t blocks = (features + 31) / 32;
                if (w) check_kept(c, dy.device(), at::kChar, N * blocks * 32, "codes");
                if (w) check_kept(e, dy.device(), at::kByte, N * blocks, "exponents");
                const int code = dtype_code(dy.scalar_type());
                if (w) dw = at::empty({O, features}, dy.options());
                if (b) db = at::empty({O}, dy.options());
                const size_t need = g_weight_grad_ws(code, N, O, w ? features : 0);
                const at::Tensor ws = need ? at::empty({(int64_t)need}, dy.options().dtype(at::kByte)) : at::Tensor();
                if (head)
                    check_status(g_head_bwd(stream_of(dy), code, dy.data_ptr(), dy.stride(0), (const int8_t *)c.data_ptr(), (const uint8_t *)e.data_ptr(), N,
                                            features, row.defined() ? row.data_ptr() : nullptr, dw.data_ptr(), b ? db.data_ptr() : nullptr,
                                            dx.defined() ? dx.data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, need),
                                 "trl_act_head_bwd");
                else
                    check_status(g_weight_grad(stream_of(dy), code, dy.data_ptr(), dy.stride(0), w ? (const int8_t *)c.data_ptr() : nullptr,
                                           w ? (const uint8_t *)e.data_ptr() : nullptr, N, O, w ? features : 0, w ? dw.data_ptr() : nullptr,
                                           b ? db.data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, need),
                             "trl_act_weight_grad");
            }
        }
        return once({dx, dw, db}, again);
    }
    void release_variables() override {
        codes.reset_data();
        exponents.reset_data();
        weight.reset_data();
    }
    std::string name() const override { return "CheckpointedLinearBackward"; }
};

template <typename N>
std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

bool count_ok(Py_ssize_t nargs, Py_ssize_t want, const char *name) {
    if (nargs != want) PyErr_Format(PyExc_TypeError, "_trl_host.%s takes %zd positional arguments", name, want);
    else if (!g_process_fwd) PyErr_SetString(PyExc_RuntimeError, "_trl_host called before init_policy");
    else return true;
    return false;
}

PyObject *py_process_logits(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (!count_ok(nargs, 10, "process_logits")) return nullptr;
    Processing p;
    if (!p.parse(o[0], o + 1)) Py_RETURN_NONE;
    const bool grad = wants_grad(p.logits);
    at::Tensor out;
    {
        c10::AutoGradMode off(false);
        out = at::empty(p.logits.sizes(), p.logits.options());
        p.a.out = out.data_ptr();
        p.a.out_st = p.a.V;
        p.a.out_sb = p.a.T * p.a.V;
        const int rc = g_process_fwd(stream_of(out), &p.a);
        if (rc) return PyLong_FromLong(rc);
    }
    if (grad) {
        auto node = make_node<ProcessLogitsBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(p.logits));
        node->kept.keep(p, p.reads_sign());
        torch::autograd::set_history(out, node);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyObject *py_token_log_prob(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (!count_ok(nargs, 12, "token_log_prob")) return nullptr;
    Processing p;
    at::Tensor action;
    if (!plain_tensor(o[1], action) || !p.parse(o[0], o + 3)) Py_RETURN_NONE;
    const bool want_entropy = o[2] == Py_True, grad = wants_grad(p.logits);
    if (!is_int(action) || action.device() != p.logits.device() || action.sizes() != p.logits.sizes().slice(0, p.logits.dim() - 1) || !action.is_contiguous())
        Py_RETURN_NONE;
    at::Tensor log_prob, entropy, stats;
    {
        c10::AutoGradMode off(false);
        const auto f32 = p.logits.options().dtype(at::kFloat);
        log_prob = at::empty(action.sizes(), f32);
        if (want_entropy) entropy = at::empty(action.sizes(), f32);
        if (grad) stats = at::empty({p.rows(), 2}, f32);
        const size_t need = g_token_ws(p.a.B, p.a.T, p.a.V);
        const at::Tensor ws = at::empty({(int64_t)need}, p.logits.options().dtype(at::kByte));
        trl_token_args a = p.a;
        a.action = action.data_ptr();
        a.action_wide = p.a.action_wide = action.scalar_type() == at::kLong;
        a.log_prob = log_prob.data_ptr<float>();
        a.entropy = want_entropy ? entropy.data_ptr<float>() : nullptr;
        a.stats = grad ? stats.data_ptr<float>() : nullptr;
        const int rc = g_log_prob_fwd(stream_of(log_prob), &a, ws.data_ptr(), need);
        if (rc) return PyLong_FromLong(rc);
    }
    if (grad) {
        auto node = make_node<TokenLogProbBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(p.logits));
        node->kept.keep(p, true);
        node->action = SavedVariable(action, false);
        node->stats = SavedVariable(stats, false);
        torch::autograd::set_history(log_prob, node);
        if (want_entropy) {
            torch::autograd::set_history(entropy, node);
            node->entropy = SavedVariable(entropy, true);
        }
    }
    if (!want_entropy) return THPVariable_Wrap(std::move(log_prob));
    PyObject *out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(log_prob)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(entropy)));
    return out;
    END_HANDLE_TH_ERRORS
}

PyObject *py_checkpointed_linear(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (!count_ok(nargs, 3, "checkpointed_linear")) return nullptr;
    at::Tensor x, w, b;
    if (!plain_tensor(o[0], x) || !plain_tensor(o[1], w) || !optional_tensor(o[2], b)) Py_RETURN_NONE;
    const auto dt = x.scalar_type();
    if (dtype_code(dt) < 0 || !on_current_device(x) || x.numel() == 0 || x.dim() < 1 || w.dim() != 2 || w.numel() == 0 || w.size(1) != x.size(-1) ||
        w.scalar_type() != dt || w.device() != x.device())
        Py_RETURN_NONE;
    if (b.defined() && (b.dim() != 1 || b.size(0) != w.size(0) || b.scalar_type() != dt || b.device() != x.device())) Py_RETURN_NONE;
    const bool gx = wants_grad(x), gw = wants_grad(w), gb = wants_grad(b);
    at::Tensor y, codes, exponents;
    {
        c10::AutoGradMode off(false);
        int rc = 0;
        if (w.size(0) == 1 && w.size(1) <= kHeadFeatures) {
            rc = head(x, w, b, gw, y, codes, exponents);
        } else {
            // below the view tracking: the product folds batch dims and comes back as a view, which may not be written in place once it has a history
            at::AutoDispatchBelowADInplaceOrView untracked;
            y = at::linear(x, w, b.defined() ? std::optional<at::Tensor>(b) : std::nullopt);
            if (gw) rc = quantize(x, codes, exponents);
        }
        if (rc) return PyLong_FromLong(rc);
    }
    if (gx || gw || gb) {
        auto node = make_node<CheckpointedLinearBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
        node->features = x.size(-1);
        node->need_x = gx;
        node->need_w = gw;
        node->need_b = gb;
        if (gw) {
            node->codes = SavedVariable(codes, false);
            node->exponents = SavedVariable(exponents, false);
        }
        if (gx) node->weight = SavedVariable(w, false);
        torch::autograd::set_history(y, node);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

PyObject *py_quantize(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (!count_ok(nargs, 1, "quantize")) return nullptr;
    at::Tensor x;
    if (!plain_tensor(o[0], x)) Py_RETURN_NONE;
    if (dtype_code(x.scalar_type()) < 0 || !on_current_device(x) || x.numel() == 0 || x.dim() < 1) Py_RETURN_NONE;
    c10::AutoGradMode off(false);
    at::Tensor codes, exponents;
    const int rc = quantize(x, codes, exponents);
    if (rc) return PyLong_FromLong(rc);
    PyObject *out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(codes)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(exponents)));
    return out;
    END_HANDLE_TH_ERRORS
}

PyObject *py_dequantize(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (!count_ok(nargs, 4, "dequantize")) return nullptr;
    at::Tensor codes, exponents;
    if (!plain_tensor(o[0], codes) || !plain_tensor(o[1], exponents)) Py_RETURN_NONE;
    const int64_t D = PyLong_AsLongLong(o[2]);
    const int code = (int)PyLong_AsLong(o[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!on_current_device(codes) || codes.numel() == 0 || !codes.is_contiguous() || !exponents.is_contiguous() || codes.scalar_type() != at::kChar ||
        exponents.scalar_type() != at::kByte || D <= 0 || codes.size(-1) != (D + 31) / 32 * 32 || exponents.numel() * 32 != codes.numel() ||
        exponents.device() != codes.device())
        Py_RETURN_NONE;
    c10::AutoGradMode off(false);
    auto shape = codes.sizes().vec();
    shape.back() = D;
    at::Tensor out = at::empty(shape, codes.options().dtype(code == TRL_F32 ? at::kFloat : code == TRL_BF16 ? at::kBFloat16 : at::kHalf));
    const int rc = g_dequantize(stream_of(out), code, (const int8_t *)codes.data_ptr(), (const uint8_t *)exponents.data_ptr(),
                                codes.numel() / codes.size(-1), D, out.data_ptr());
    if (rc) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyObject *py_init_policy(PyObject *, PyObject *args) {
    unsigned long long p[12];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8, p + 9, p + 10, p + 11)) return nullptr;
    g_process_fwd = (decltype(g_process_fwd))(uintptr_t)p[0];
    g_process_bwd = (decltype(g_process_bwd))(uintptr_t)p[1];
    g_token_ws = (decltype(g_token_ws))(uintptr_t)p[2];
    g_log_prob_fwd = (decltype(g_log_prob_fwd))(uintptr_t)p[3];
    g_log_prob_bwd = (decltype(g_log_prob_bwd))(uintptr_t)p[4];
    g_quantize = (decltype(g_quantize))(uintptr_t)p[5];
    g_dequantize = (decltype(g_dequantize))(uintptr_t)p[6];
    g_weight_grad_ws = (decltype(g_weight_grad_ws))(uintptr_t)p[7];
    g_weight_grad = (decltype(g_weight_grad))(uintptr_t)p[8];
    g_head_fwd = (decltype(g_head_fwd))(uintptr_t)p[9];
    g_head_bwd = (decltype(g_head_bwd))(uintptr_t)p[10];
    g_last_error = (decltype(g_last_error))(uintptr_t)p[11];
    Py_RETURN_NONE;
}

}  // namespace

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL
PyMethodDef trl_policy_methods[] = {
    {"init_policy", py_init_policy, METH_VARARGS,
     "init_policy(trl_process_logits_fwd, trl_process_logits_bwd, trl_token_workspace_bytes, trl_token_log_prob_fwd, trl_token_log_prob_bwd, "
     "trl_act_quantize, trl_act_dequantize, trl_act_weight_grad_workspace_bytes, trl_act_weight_grad, trl_act_head_fwd, trl_act_head_bwd, trl_last_error)"},
    {"process_logits", FAST(py_process_logits), "see host_policy.cpp"},
    {"token_log_prob", FAST(py_token_log_prob), "see host_policy.cpp"},
    {"checkpointed_linear", FAST(py_checkpointed_linear), "see host_policy.cpp"},
    {"quantize", FAST(py_quantize), "see host_policy.cpp"},
    {"dequantize", FAST(py_dequantize), "see host_policy.cpp"},
    {nullptr, nullptr, 0, nullptr}};
