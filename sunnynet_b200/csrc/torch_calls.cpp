// The parts of kernels.py that cost more in Python than their kernels take.
//
// read: the lists of torch tensors of an AdamW step, as the addresses and sizes
// that the C entry point takes, and the checks of types, layout and device. In
// Python each question to each tensor costs about 0.07 us: for 12 layers of a
// model (146 tensors, six lists with 8-bit states) 200 us of calls, as long as
// the update itself takes on the GPU; here 25 us.
//
// layer_norm: the call and its node in the autograd graph. A call and its
// gradients take 75 us of the host's time (torch's own layer norm 70), as a
// Function in Python 110; a call without a graph 8 us instead of 11.
//
// embedding, linear_attention (calls and nodes alike), linear_attention_step and
// grad_norm: with their checks in Python they took 20 to 30 us of the host's time
// a call, longer than most of their kernels.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "sn_abi.h"

namespace {

// The library's entry points (it is loaded by ctypes).
struct {
    decltype(&sn_abi_layer_norm) norm = nullptr;
    decltype(&sn_abi_layer_norm_bwd) norm_bwd = nullptr;
    decltype(&sn_abi_layer_norm_bwd_ws) norm_bwd_ws = nullptr;
    decltype(&sn_abi_last_error) last_error = nullptr;
    decltype(&sn_abi_embedding) embedding = nullptr;
    decltype(&sn_abi_embedding_bwd) embedding_bwd = nullptr;
    decltype(&sn_abi_embedding_bwd_ws) embedding_bwd_ws = nullptr;
    decltype(&sn_abi_linear_attention) attention = nullptr;
    decltype(&sn_abi_linear_attention_bwd) attention_bwd = nullptr;
    decltype(&sn_abi_linear_attention_ws) attention_ws = nullptr;
    decltype(&sn_abi_linear_attention_step) attention_step = nullptr;
    decltype(&sn_abi_arrays_on) arrays_on = nullptr;
    decltype(&sn_abi_grad_norm_ws) grad_norm_ws = nullptr;
    decltype(&sn_abi_grad_norm) grad_norm = nullptr;
    decltype(&sn_abi_clip_grads) clip_grads = nullptr;
} lib;

std::string last_error() {
    char text[512] = "";
    lib.last_error(text, sizeof text);
    return text;
}

int32_t code(at::ScalarType t) {
    return t == at::kFloat ? SN_F32 : t == at::kBFloat16 ? SN_BF16 : SN_F16;
}

// t as rows of D values at one stride; ld: that stride in elements.
at::Tensor rows_of(const at::Tensor& t, int64_t D, int64_t* ld) {
    *ld = D;
    if (t.is_contiguous()) return t;
    at::Tensor r = t.reshape({-1, D});  // a view wherever the rows lie at one stride
    if (r.stride(1) != 1 || (r.size(0) > 1 && r.stride(0) < D))
        return r.contiguous();  // among these what a sum's gradient broadcasts
    *ld = std::max(r.stride(0), D);
    return r;
}

void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const at::Tensor& t) {
    return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// The library's next call takes all arrays to be on t's GPU, and does not ask for
// each. Constructed right before that call.
struct Known {
    explicit Known(const at::Tensor& t) { lib.arrays_on(t.get_device()); }
    ~Known() { lib.arrays_on(-1); }
    Known(const Known&) = delete;
};

int32_t weight_code(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b) {
    return code(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
}

// y; x, w, b: what was given, made rows and contiguous. stats: (2, rows), or none.
at::Tensor norm_forward(at::Tensor& x, at::Tensor& w, at::Tensor& b, double eps,
                        at::Tensor* stats) {
    const int64_t D = x.size(-1), rows = x.numel() / D;
    at::Tensor y = x.is_contiguous() ? at::empty_like(x) : at::empty(x.sizes(), x.options());
    int64_t ld;
    x = rows_of(x, D, &ld);
    if (w.defined()) w = w.contiguous();
    if (b.defined()) b = b.contiguous();
    float* mean = nullptr;
    if (stats) {
        *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
    }
    const int rc = lib.norm(address(x), ld, address(w), address(b), address(y), mean,
                            stats ? mean + rows : nullptr, code(x.scalar_type()),
                            weight_code(x, w, b), rows, (int32_t)D, (float)eps, stream_of(x));
    TORCH_CHECK(rc == SN_OK, "layer_norm: ", last_error());
    return y;
}

struct Norm : torch::autograd::Function<Norm> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x_,
                              const std::optional<at::Tensor>& w_,
                              const std::optional<at::Tensor>& b_, double eps) {
        at::Tensor x = x_, w = w_.value_or(at::Tensor()), b = b_.value_or(at::Tensor()), stats;
        const int32_t wcode = weight_code(x, w, b);
        const bool has_w = w.defined(), has_b = b.defined();
        at::Tensor y = norm_forward(x, w, b, eps, &stats);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["call"] = (int64_t)(wcode | has_w << 4 | has_b << 5);
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        // with create_graph: its own gradient is not there
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm can be differentiated once");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &stats = saved[2], &dy = grads[0];
        const int64_t call = ctx->saved_data["call"].toInt();
        const int32_t wcode = (int32_t)(call & 15);
        const bool has_w = call >> 4 & 1, has_b = call >> 5 & 1;
        const bool want_x = ctx->needs_input_grad(0), want_w = has_w && ctx->needs_input_grad(1),
                   want_b = has_b && ctx->needs_input_grad(1 + has_w);
        const int64_t D = dy.size(-1), rows = dy.numel() / D;
        int64_t ldx, ldg;
        const at::Tensor xr = rows_of(x, D, &ldx), g = rows_of(dy, D, &ldg);
        const int32_t c = code(x.scalar_type());
        at::Tensor dx, dw, db, ws;
        if (want_x) dx = at::empty(dy.sizes(), dy.options());
        const auto wide = dy.options().dtype(wcode == SN_F32 ? at::kFloat : dy.scalar_type());
        if (want_w) dw = at::empty({D}, wide);
        if (want_b) db = at::empty({D}, wide);
        int64_t need = 0;
        if (want_w || want_b) {
            need = lib.norm_bwd_ws(rows, (int32_t)D, c);
            ws = at::empty({need}, dy.options().dtype(at::kByte));
        }
        const float* mean = stats.data_ptr<float>();
        const int rc = lib.norm_bwd(address(g), ldg, address(xr), ldx, address(w), mean,
                                    mean + rows, address(dx), address(dw), address(db),
                                    address(ws), need, c, wcode, rows, (int32_t)D, stream_of(x));
        TORCH_CHECK(rc == SN_OK, "layer_norm_bwd: ", last_error());
        return {dx, dw, db, at::Tensor()};
    }
};

// A tensor or None (an undefined one); false with an error set for others.
bool tensor_of(const char* what, PyObject* o, at::Tensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: tensors are wanted", what);
        return false;
    }
    *t = THPVariable_Unpack(o);
    return true;
}

// layer_norm(x, weight, bias, eps), the arguments as kernels.layer_norm checked them.
PyObject* layer_norm(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *xo, *wo, *bo;
    double eps;
    if (!PyArg_ParseTuple(args, "OOOd", &xo, &wo, &bo, &eps)) return nullptr;
    at::Tensor x, w, b;
    const char* const what = "layer_norm";
    if (!tensor_of(what, xo, &x) || !tensor_of(what, wo, &w) || !tensor_of(what, bo, &b)) return nullptr;
    // (neither path carries a tangent on)
    const auto moves = [](const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); };
    TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
                  (moves(x) || moves(w) || moves(b))),
                "layer_norm has no forward-mode derivative");
    const auto grows = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
    if (at::GradMode::is_enabled() && (grows(x) || grows(w) || grows(b)))
        return THPVariable_Wrap(
            Norm::apply(x, w.defined() ? std::optional<at::Tensor>(w) : std::nullopt,
                        b.defined() ? std::optional<at::Tensor>(b) : std::nullopt, eps));
    return THPVariable_Wrap(norm_forward(x, w, b, eps, nullptr));
    END_HANDLE_TH_ERRORS
}

bool float_type(const at::Tensor& t) {
    const at::ScalarType k = t.scalar_type();
    return k == at::kFloat || k == at::kBFloat16 || k == at::kHalf;
}

bool wants_grad(std::initializer_list<at::Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// (no call here carries a tangent on)
void no_tangent(const char* what, std::initializer_list<at::Tensor> ts) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const at::Tensor& t : ts)
        TORCH_CHECK(!(t.defined() && t._fw_grad(0).defined()), what, " has no forward-mode derivative");
}

// Views whose sign is not in memory (the imaginary part of a conjugate) become tensors as they read.
void signed_values(std::initializer_list<at::Tensor*> ts) {
    for (at::Tensor* t : ts)
        if (t->defined() && t->is_neg()) *t = t->resolve_neg();
}

at::Tensor space(int64_t bytes, const at::Tensor& like) {
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// ------------------------------------------------------------------ embedding
at::Tensor embedding_forward(const at::Tensor& tokens, const at::Tensor& w, double scale) {
    std::vector<int64_t> sizes(tokens.sizes().begin(), tokens.sizes().end());
    sizes.push_back(w.size(1));
    at::Tensor out = at::empty(sizes, w.options());
    const Known known(w);
    const int rc = lib.embedding(address(tokens), 8 * (int32_t)tokens.element_size(), tokens.numel(), address(w),
                                 w.stride(0), w.size(0), (int32_t)w.size(1), code(w.scalar_type()), (float)scale,
                                 address(out), stream_of(w));
    TORCH_CHECK(rc == SN_OK, "embedding: ", last_error());
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& tokens,
                              const at::Tensor& w, double scale) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["rows"] = w.size(0);
        ctx->saved_data["scale"] = scale;
        return embedding_forward(tokens, w, scale);
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "embedding can be differentiated once");
        const at::Tensor tokens = ctx->get_saved_variables()[0];
        at::Tensor& dout = grads[0];
        signed_values({&dout});
        const int64_t V = ctx->saved_data["rows"].toInt(), D = dout.size(-1), n = tokens.numel();
        at::Tensor rows = dout.reshape({n, D});  // a view wherever the rows lie at one stride
        if (D > 1 && rows.stride(1) != 1) rows = rows.contiguous();
        at::Tensor dw = at::empty({V, D}, dout.options());
        const int64_t need = lib.embedding_bwd_ws(n, V, (int32_t)D);
        const at::Tensor ws = space(need, dout);
        const Known known(dout);
        const int rc = lib.embedding_bwd(address(tokens), 8 * (int32_t)tokens.element_size(), n, address(rows),
                                         rows.stride(0), V, (int32_t)D, code(dout.scalar_type()),
                                         (float)ctx->saved_data["scale"].toDouble(), address(dw), address(ws),
                                         need, stream_of(dout));
        TORCH_CHECK(rc == SN_OK, "embedding_bwd: ", last_error());
        return {at::Tensor(), dw, at::Tensor()};
    }
};

// embedding(tokens, weight, scale)
PyObject* embedding(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *to, *wo;
    double scale;
    if (!PyArg_ParseTuple(args, "OOd", &to, &wo, &scale)) return nullptr;
    at::Tensor tokens, w;
    if (!tensor_of("embedding", to, &tokens) || !tensor_of("embedding", wo, &w)) return nullptr;
    TORCH_CHECK_VALUE(w.defined() && w.dim() == 2 && w.is_cuda() && w.size(1) <= 1 << 22 && w.size(0) < 0x7fffffff,
                      "embedding: weight (V, D) on a GPU is wanted, D at most 2^22");
    TORCH_CHECK_TYPE(float_type(w), "embedding: weight is float32, bfloat16 or float16");
    TORCH_CHECK_VALUE(tokens.defined() && (tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong) &&
                          tokens.device() == w.device() && tokens.numel() <= 0x7ffff000,
                      "embedding: tokens are int32 or int64 on the weight's GPU, fewer than 2^31");
    TORCH_CHECK_VALUE(std::isfinite(scale), "embedding: the scale is not finite");
    no_tangent("embedding", {w});
    signed_values({&w});
    tokens = tokens.contiguous();
    if (w.size(1) > 1 && w.stride(1) != 1) w = w.contiguous();
    if (wants_grad({w})) return THPVariable_Wrap(Embedding::apply(tokens, w, scale));
    return THPVariable_Wrap(embedding_forward(tokens, w, scale));
    END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------- linear attention
constexpr int64_t kMaxHead = 128;

// The checked arguments of a call. Tensors are made fit for it in place. A single
// token's have no axis of tokens.
SnAbiLinearAttention attention_call(const char* what, at::Tensor& q, at::Tensor& k, at::Tensor& v,
                                    at::Tensor& decay, at::Tensor* state, at::Tensor* lengths, double scale,
                                    bool one = false) {
    const int64_t n = 4 - one;
    TORCH_CHECK_VALUE(q.dim() == n && v.dim() == n && k.sizes() == q.sizes() && v.size(0) == q.size(0) &&
                          (one || v.size(1) == q.size(1)),
                      what, one ? ": q and k are (B, Hk, dk), v (B, H, dv)"
                                : ": q and k are (B, T, Hk, dk), v (B, T, H, dv)");
    const int64_t B = q.size(0), T = one ? 1 : q.size(1), Hk = q.size(n - 2), dk = q.size(n - 1), H = v.size(n - 2),
                  dv = v.size(n - 1);
    TORCH_CHECK_VALUE(Hk > 0 && H > 0 && H % Hk == 0 && dk > 0 && dk <= kMaxHead && dv > 0 && dv <= kMaxHead, what,
                      ": heads of 1 to 128 values, H a multiple of Hk");
    TORCH_CHECK_VALUE(T < 0x7fffffff - 128 && B * H <= 0x7fffffff, what, ": sizes beyond 31 bits");
    TORCH_CHECK_TYPE(float_type(v), what, ": q, k and v are float32, bfloat16 or float16");
    TORCH_CHECK_VALUE(v.is_cuda() && q.scalar_type() == v.scalar_type() && k.scalar_type() == v.scalar_type() &&
                          q.device() == v.device() && k.device() == v.device(),
                      what, ": q, k and v are of one type, on one GPU");
    TORCH_CHECK_VALUE(decay.scalar_type() == at::kFloat && decay.device() == v.device() &&
                          (decay.sizes() == at::IntArrayRef({H}) ||
                           (one ? decay.sizes() == at::IntArrayRef({B, H}) : decay.sizes() == at::IntArrayRef({B, T, H}))),
                      what, one ? ": log_decay is float32 of (H) or (B, H) on the GPU of the others"
                                : ": log_decay is float32 of (H) or (B, T, H) on the GPU of the others");
    TORCH_CHECK_VALUE(std::isfinite(scale), what, ": the scale is not finite");
    SnAbiLinearAttention a = {};
    if (state && state->defined()) {
        TORCH_CHECK_VALUE(state->scalar_type() == at::kFloat && state->device() == v.device() &&
                              state->sizes() == at::IntArrayRef({B, H, dk, dv}),
                          what, ": state is float32 of (B, H, dk, dv) on the GPU of the others");
        *state = state->contiguous();
        a.state = state->data_ptr<float>();
    }
    if (lengths && lengths->defined()) {
        TORCH_CHECK_VALUE(lengths->scalar_type() == at::kInt && lengths->device() == v.device() &&
                              lengths->sizes() == at::IntArrayRef({B}),
                          what, ": lengths are (B) int32 values on the GPU of the others");
        *lengths = lengths->contiguous();
        a.lengths = lengths->data_ptr<int32_t>();
    }
    const auto rows = [&](at::Tensor& t, const void** p, int64_t* stride) {
        if (t.size(n - 1) > 1 && t.stride(n - 1) != 1) t = t.contiguous();
        *p = t.data_ptr();
        stride[0] = t.stride(0);
        stride[1] = one ? 0 : t.stride(1);
        stride[2] = t.stride(n - 2);
    };
    rows(q, &a.q, a.q_stride);
    rows(k, &a.k, a.k_stride);
    rows(v, &a.v, a.v_stride);
    a.log_decay = decay.data_ptr<float>();
    const bool each = decay.dim() > 1;  // token's
    a.log_decay_stride[0] = each ? decay.stride(0) : 0;
    a.log_decay_stride[1] = each && !one ? decay.stride(1) : 0;
    a.log_decay_stride[2] = decay.stride(decay.dim() - 1);
    a.dtype = code(v.scalar_type());
    a.B = (int32_t)B, a.T = (int32_t)T, a.H = (int32_t)H, a.Hk = (int32_t)Hk, a.dk = (int32_t)dk, a.dv = (int32_t)dv;
    a.scale = (float)scale;
    return a;
}

std::pair<at::Tensor, at::Tensor> attention_forward(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor decay,
                                                    at::Tensor state, at::Tensor lengths, double scale) {
    const SnAbiLinearAttention a = attention_call("linear_attention", q, k, v, decay, &state, &lengths, scale);
    at::Tensor out = at::empty(v.sizes(), v.options());
    at::Tensor end = at::empty({a.B, a.H, a.dk, a.dv}, v.options().dtype(at::kFloat));
    const int64_t need = lib.attention_ws(&a, 0, 0);
    const at::Tensor ws = space(need, v);
    const Known known(v);
    const int rc = lib.attention(&a, address(out), end.data_ptr<float>(), address(ws), need, stream_of(v));
    TORCH_CHECK(rc == SN_OK, "linear_attention: ", last_error());
    return {out, end};
}

struct Attention : torch::autograd::Function<Attention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                  const at::Tensor& k, const at::Tensor& v,
                                                  const at::Tensor& decay,
                                                  const std::optional<at::Tensor>& state_,
                                                  const std::optional<at::Tensor>& lengths_, double scale) {
        const at::Tensor state = state_.value_or(at::Tensor()), lengths = lengths_.value_or(at::Tensor());
        ctx->save_for_backward({q, k, v, decay, state, lengths});
        ctx->set_materialize_grads(false);
        ctx->saved_data["scale"] = scale;
        auto [out, end] = attention_forward(q, k, v, decay, state, lengths, scale);
        return {out, end};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_attention can be differentiated once");
        auto saved = ctx->get_saved_variables();
        at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &decay = saved[3], &state = saved[4];
        const bool has_state = state.defined();
        const auto qs = q.sizes().vec(), ks = k.sizes().vec();
        const SnAbiLinearAttention a = attention_call("linear_attention_bwd", q, k, v, decay, &state, &saved[5],
                                                      ctx->saved_data["scale"].toDouble());
        at::Tensor dout = grads[0], dend = grads[1];
        signed_values({&dout, &dend});
        if (!dout.defined()) dout = at::zeros(v.sizes(), v.options());
        if (a.dv > 1 && dout.stride(3) != 1) dout = dout.contiguous();
        if (dend.defined()) dend = dend.contiguous();
        at::Tensor dq = at::empty(qs, q.options()), dk = at::empty(ks, k.options()),
                   dv = at::empty(v.sizes(), v.options()), dg, ds;
        if (ctx->needs_input_grad(3)) dg = at::empty(decay.sizes(), decay.options());
        if (has_state && ctx->needs_input_grad(4)) ds = at::empty(state.sizes(), state.options());
        const int32_t heads = dg.defined() && decay.dim() == 1;
        if (a.B) {
            const int64_t need = lib.attention_ws(&a, 1, heads);
            const at::Tensor ws = space(need, v);
            const int64_t stride[3] = {dout.stride(0), dout.stride(1), dout.stride(2)};
            const Known known(v);
            const int rc = lib.attention_bwd(&a, address(dout), stride, static_cast<float*>(address(dend)),
                                             address(dq), address(dk), address(dv),
                                             static_cast<float*>(address(dg)), heads,
                                             static_cast<float*>(address(ds)), address(ws), need, stream_of(v));
            TORCH_CHECK(rc == SN_OK, "linear_attention_bwd: ", last_error());
        } else if (dg.defined()) {
            dg.zero_();
        }
        return {dq, dk, dv, dg, ds, at::Tensor(), at::Tensor()};
    }
};

// The tensors of a call's arguments and its scale (None: 1 / sqrt of q's last axis).
bool attention_args(const char* what, PyObject* const* o, int n, at::Tensor* t, PyObject* scale, double* to) {
    for (int i = 0; i < n; ++i) {
        if (!tensor_of(what, o[i], t + i)) return false;
        if (i < 4 && !t[i].defined()) {
            PyErr_Format(PyExc_TypeError, "%s: tensors are wanted", what);
            return false;
        }
    }
    if (scale != Py_None) {
        *to = PyFloat_AsDouble(scale);
        return !(*to == -1.0 && PyErr_Occurred());
    }
    *to = t[0].dim() && t[0].size(-1) > 0 ? 1.0 / std::sqrt((double)t[0].size(-1)) : 1.0;
    return true;
}

// linear_attention(q, k, v, log_decay, state, lengths, scale) -> (out, state)
PyObject* linear_attention(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *o[6], *so;
    if (!PyArg_ParseTuple(args, "OOOOOOO", o, o + 1, o + 2, o + 3, o + 4, o + 5, &so)) return nullptr;
    at::Tensor t[6];
    double scale;
    const char* const what = "linear_attention";
    if (!attention_args(what, o, 6, t, so, &scale)) return nullptr;
    no_tangent(what, {t[0], t[1], t[2], t[3], t[4]});
    signed_values({t, t + 1, t + 2, t + 3, t + 4});
    std::pair<at::Tensor, at::Tensor> r;
    if (wants_grad({t[0], t[1], t[2], t[3], t[4]})) {
        const auto some = [](const at::Tensor& x) { return x.defined() ? std::optional<at::Tensor>(x) : std::nullopt; };
        auto both = Attention::apply(t[0], t[1], t[2], t[3], some(t[4]), some(t[5]), scale);
        r = {both[0], both[1]};
    } else {
        r = attention_forward(t[0], t[1], t[2], t[3], t[4], t[5], scale);
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(r.first), THPVariable_Wrap(r.second));
    END_HANDLE_TH_ERRORS
}

// Whether each sequence's state is contiguous.
bool rows_of_state(const at::Tensor& s) {
    int64_t want = 1;
    for (int i = 3; i > 0; --i) {
        if (s.size(i) > 1 && s.stride(i) != want) return false;
        want *= s.size(i);
    }
    return true;
}

// linear_attention_step(q, k, v, log_decay, state, scale) -> out; state is updated
PyObject* linear_attention_step(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *o[5], *so;
    if (!PyArg_ParseTuple(args, "OOOOOO", o, o + 1, o + 2, o + 3, o + 4, &so)) return nullptr;
    at::Tensor t[5];
    double scale;
    const char* const what = "linear_attention_step";
    if (!attention_args(what, o, 5, t, so, &scale)) return nullptr;
    at::Tensor &q = t[0], &k = t[1], &v = t[2], &decay = t[3], &state = t[4];
    no_tangent(what, {q, k, v, decay, state});
    TORCH_CHECK_VALUE(!wants_grad({q, k, v, decay, state}), what, " has no gradient: call linear_attention");
    signed_values({&q, &k, &v, &decay});
    at::Tensor out = at::empty(v.sizes(), v.options());
    const SnAbiLinearAttention a = attention_call(what, q, k, v, decay, nullptr, nullptr, scale, true);
    TORCH_CHECK_VALUE(state.defined() && state.scalar_type() == at::kFloat && state.device() == v.device() &&
                          state.sizes() == at::IntArrayRef({a.B, a.H, a.dk, a.dv}) &&
                          rows_of_state(state) && !state.is_neg(),
                      what, ": state is float32 of (B, H, dk, dv) on the GPU of the others, each sequence's contiguous");
    TORCH_CHECK_VALUE(a.B < 2 || state.stride(0) >= (int64_t)a.H * a.dk * a.dv, what, ": the states overlap");
    state.unsafeGetTensorImpl()->bump_version();  // a graph that saved it must not use it
    const Known known(v);
    const int rc = lib.attention_step(&a, static_cast<float*>(address(state)), a.B ? state.stride(0) : 0,
                                      address(out), stream_of(v));
    TORCH_CHECK(rc == SN_OK, last_error());
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// use(addresses of the library's entry points, in the order below)
PyObject* use(PyObject*, PyObject* args) {
    unsigned long long p[15];
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8, p + 9,
                          p + 10, p + 11, p + 12, p + 13, p + 14))
        return nullptr;
    lib.norm = reinterpret_cast<decltype(lib.norm)>(p[0]);
    lib.norm_bwd = reinterpret_cast<decltype(lib.norm_bwd)>(p[1]);
    lib.norm_bwd_ws = reinterpret_cast<decltype(lib.norm_bwd_ws)>(p[2]);
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(p[3]);
    lib.embedding = reinterpret_cast<decltype(lib.embedding)>(p[4]);
    lib.embedding_bwd = reinterpret_cast<decltype(lib.embedding_bwd)>(p[5]);
    lib.embedding_bwd_ws = reinterpret_cast<decltype(lib.embedding_bwd_ws)>(p[6]);
    lib.attention = reinterpret_cast<decltype(lib.attention)>(p[7]);
    lib.attention_bwd = reinterpret_cast<decltype(lib.attention_bwd)>(p[8]);
    lib.attention_ws = reinterpret_cast<decltype(lib.attention_ws)>(p[9]);
    lib.attention_step = reinterpret_cast<decltype(lib.attention_step)>(p[10]);
    lib.grad_norm_ws = reinterpret_cast<decltype(lib.grad_norm_ws)>(p[11]);
    lib.grad_norm = reinterpret_cast<decltype(lib.grad_norm)>(p[12]);
    lib.clip_grads = reinterpret_cast<decltype(lib.clip_grads)>(p[13]);
    lib.arrays_on = reinterpret_cast<decltype(lib.arrays_on)>(p[14]);
    Py_RETURN_NONE;
}

// The tensors of a list or tuple, or null with an error set.
PyObject** items(PyObject* list, Py_ssize_t* n) {
    if (!PyList_Check(list) && !PyTuple_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "lists or tuples of tensors are wanted");
        return nullptr;
    }
    *n = PySequence_Fast_GET_SIZE(list);
    return PySequence_Fast_ITEMS(list);
}

// read(lists, dtypes, block) -> (addresses, sizes): of k lists of n tensors, as
// k * n unsigned and n signed 64-bit numbers. List i has tensors of dtypes[i],
// all contiguous and on one GPU. Lists 0 to 3 agree in their sizes, the others
// have one value for each `block` of those. No memory of lists 0, 2, 3 ...
// (what is written) belongs to two of their tensors.
PyObject* read(PyObject*, PyObject* args) {
    PyObject *lists, *dtypes;
    long long block;
    if (!PyArg_ParseTuple(args, "O!O!L", &PyTuple_Type, &lists, &PyTuple_Type, &dtypes, &block))
        return nullptr;
    const Py_ssize_t k = PyTuple_GET_SIZE(lists);
    if (k < 1 || PyTuple_GET_SIZE(dtypes) != k || block < 1) {
        PyErr_SetString(PyExc_ValueError, "one dtype for each list is wanted");
        return nullptr;
    }
    try {
        Py_ssize_t n = 0;
        if (!items(PyTuple_GET_ITEM(lists, 0), &n)) return nullptr;
        std::vector<uint64_t> at(k * n);
        std::vector<std::pair<uint64_t, uint64_t>> written;  // begin and end
        std::vector<int64_t> sizes(n);
        c10::Device device(c10::kCPU);
        for (Py_ssize_t i = 0; i < k; ++i) {
            Py_ssize_t m = 0;
            PyObject** const of = items(PyTuple_GET_ITEM(lists, i), &m);
            if (!of) return nullptr;
            if (m != n) {
                PyErr_SetString(PyExc_ValueError, "the lists differ in length");
                return nullptr;
            }
            PyObject* const kind = PyTuple_GET_ITEM(dtypes, i);
            if (!THPDtype_Check(kind)) {
                PyErr_SetString(PyExc_TypeError, "a dtype is wanted for each list");
                return nullptr;
            }
            const at::ScalarType type = reinterpret_cast<THPDtype*>(kind)->scalar_type;
            for (Py_ssize_t j = 0; j < n; ++j) {
                if (!THPVariable_Check(of[j])) {
                    PyErr_SetString(PyExc_TypeError, "tensors are wanted");
                    return nullptr;
                }
                const at::Tensor& t = THPVariable_Unpack(of[j]);
                if (t.scalar_type() != type) {
                    PyErr_Format(PyExc_TypeError, "list %zd has tensors of %R", i, kind);
                    return nullptr;
                }
                if (i == 0 && j == 0) device = t.device();
                if (!t.device().is_cuda() || t.device() != device) {
                    PyErr_SetString(PyExc_ValueError, "every tensor must be on one GPU");
                    return nullptr;
                }
                if (!t.is_contiguous()) {
                    PyErr_SetString(PyExc_ValueError, "every tensor must be contiguous");
                    return nullptr;
                }
                const int64_t size = t.numel();
                if (i == 0) {
                    sizes[j] = size;
                } else if (size != (i < 4 ? sizes[j] : (sizes[j] + block - 1) / block)) {
                    PyErr_SetString(PyExc_ValueError,
                                    i < 4 ? "a gradient or state differs in size from its parameter"
                                          : "there is one scale for each block of values");
                    return nullptr;
                }
                at[i * n + j] = reinterpret_cast<uint64_t>(size ? t.data_ptr() : nullptr);
                if (size && i != 1)
                    written.emplace_back(at[i * n + j], at[i * n + j] + size * t.element_size());
            }
        }
        std::sort(written.begin(), written.end());
        if (std::adjacent_find(written.begin(), written.end(), [](const auto& a, const auto& b) {
                return b.first < a.second;
            }) != written.end()) {
            PyErr_SetString(PyExc_ValueError, "a parameter or state appears twice, or overlaps another");
            return nullptr;
        }
        return Py_BuildValue("(y#y#)", reinterpret_cast<const char*>(at.data()),
                             static_cast<Py_ssize_t>(at.size() * 8),
                             reinterpret_cast<const char*>(sizes.data()),
                             static_cast<Py_ssize_t>(sizes.size() * 8));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// grad_norm(list, max_norm, clip) -> (norm, factor), with `clip` the norm alone, of the gradients in a list or
// tuple: tensors of float types on one GPU, each filling one run of memory in any
// order. With `clip` they are scaled in place; no memory then belongs to two of them.
PyObject* grad_norm(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject* list;
    double max_norm;
    int clip;
    if (!PyArg_ParseTuple(args, "Odp", &list, &max_norm, &clip)) return nullptr;
    Py_ssize_t n = 0;
    PyObject** const of = items(list, &n);
    if (!of && PyErr_Occurred()) return nullptr;  // (an empty list may have no items at all)
    const char* const what = clip ? "clip_grads" : "grad_norm";
    TORCH_CHECK_VALUE(n > 0 && n < 0x7fffffff, what, ": no gradients");
    TORCH_CHECK_VALUE(max_norm >= 0, what, ": max_norm must not be negative");
    std::vector<void*> at(n);
    std::vector<int64_t> sizes(n);
    std::vector<int32_t> types(n);
    std::vector<std::pair<uint64_t, uint64_t>> written;
    for (Py_ssize_t j = 0; j < n; ++j) {
        TORCH_CHECK_TYPE(THPVariable_Check(of[j]), what, ": tensors are wanted");
        const at::Tensor& t = THPVariable_Unpack(of[j]);
        TORCH_CHECK_VALUE(t.layout() == at::kStrided, what, ": sparse gradients are not supported");
        TORCH_CHECK_TYPE(float_type(t), what, ": gradients are of float32, bfloat16 or float16");
        TORCH_CHECK_VALUE(t.is_cuda() && t.device() == THPVariable_Unpack(of[0]).device(), what,
                          ": every gradient must be on one GPU");
        TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense(), what,
                          ": a gradient's values must fill one run of memory");
        sizes[j] = t.numel();
        types[j] = code(t.scalar_type());
        at[j] = sizes[j] ? t.data_ptr() : nullptr;
        if (clip && sizes[j]) {
            const uint64_t begin = reinterpret_cast<uint64_t>(at[j]);
            written.emplace_back(begin, begin + sizes[j] * t.element_size());
        }
    }
    std::sort(written.begin(), written.end());
    TORCH_CHECK_VALUE(std::adjacent_find(written.begin(), written.end(),
                                         [](const auto& a, const auto& b) { return b.first < a.second; }) ==
                          written.end(),
                      what, ": a gradient appears twice, or overlaps another");
    const at::Tensor& first = THPVariable_Unpack(of[0]);
    const int64_t need = lib.grad_norm_ws((int32_t)n, sizes.data());
    TORCH_CHECK_VALUE(need >= 0, what, ": too many values");
    const at::Tensor ws = at::empty({2 + need / 4}, first.options().dtype(at::kFloat));
    float* const to = ws.data_ptr<float>();
    if (clip)  // a graph that saved one must not use it
        for (Py_ssize_t j = 0; j < n; ++j) THPVariable_Unpack(of[j]).unsafeGetTensorImpl()->bump_version();
    const Known known(first);
    const int rc = clip ? lib.clip_grads((int32_t)n, at.data(), sizes.data(), types.data(), max_norm, to, to + 1,
                                         to + 2, need, stream_of(first))
                        : lib.grad_norm((int32_t)n, at.data(), sizes.data(), types.data(), max_norm, to, to + 1,
                                        to + 2, need, stream_of(first));
    TORCH_CHECK(rc == SN_OK, last_error());
    if (clip) return THPVariable_Wrap(ws.select(0, 0));
    return Py_BuildValue("(NN)", THPVariable_Wrap(ws.select(0, 0)), THPVariable_Wrap(ws.select(0, 1)));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"read", read, METH_VARARGS, "read(lists, dtypes, block) -> (addresses, sizes)"},
    {"grad_norm", grad_norm, METH_VARARGS, "grad_norm(list, max_norm, clip) -> (norm, factor)"},
    {"layer_norm", layer_norm, METH_VARARGS, "layer_norm(x, weight, bias, eps) -> y"},
    {"embedding", embedding, METH_VARARGS, "embedding(tokens, weight, scale) -> rows"},
    {"linear_attention", linear_attention, METH_VARARGS,
     "linear_attention(q, k, v, log_decay, state, lengths, scale) -> (out, state)"},
    {"linear_attention_step", linear_attention_step, METH_VARARGS,
     "linear_attention_step(q, k, v, log_decay, state, scale) -> out"},
    {"use", use, METH_VARARGS, "use(addresses of the library's entry points)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls() { return PyModule_Create(&module); }
