// Host path of the eager layer calls: a CPython extension over libadder_b200.so that does in C++ what the Python layer
// (adder.py, adder_cuda.py, inference.py) does around a launch - checks, output allocation, the autograd node, the side stream
// of the weight gradient.  A small layer's kernels take 10-20 us; the Python around its forward and backward took 150.
//
// Every entry point takes the common case only (contiguous CUDA tensors, fp32 and of a geometry the fused kernels are built for where it
// is a layer) and returns None for anything else, errors included: the caller then goes through the Python layer, which handles or rejects it.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>

#include <array>
#include <atomic>
#include <cmath>
#include <mutex>

#include "../../include/adder_b200.h"

namespace {

struct Api {      // entry points of the loaded libadder_b200.so
    decltype(&adder_b200_status_string) status_string = nullptr;
    decltype(&adder_b200_forward) forward = nullptr;
    decltype(&adder_b200_forward_stat_slices) forward_stat_slices = nullptr;
    decltype(&adder_b200_forward_with_stats) forward_with_stats = nullptr;
    decltype(&adder_b200_forward_affine) forward_affine = nullptr;
    decltype(&adder_b200_affine_forward) affine_forward = nullptr;
    decltype(&adder_b200_backward_input_workspace_bytes) backward_input_workspace_bytes = nullptr;
    decltype(&adder_b200_backward_input_with_workspace) backward_input_with_workspace = nullptr;
    decltype(&adder_b200_backward_weight_workspace_bytes) backward_weight_workspace_bytes = nullptr;
    decltype(&adder_b200_backward_weight) backward_weight = nullptr;
    decltype(&adder_b200_conv_forward) conv_forward = nullptr;
    decltype(&adder_b200_conv_backward_input_workspace_bytes) conv_backward_input_workspace_bytes = nullptr;
    decltype(&adder_b200_conv_backward_input_with_workspace) conv_backward_input_with_workspace = nullptr;
    decltype(&adder_b200_conv_backward_weight_workspace_bytes) conv_backward_weight_workspace_bytes = nullptr;
    decltype(&adder_b200_conv_backward_weight) conv_backward_weight = nullptr;
    decltype(&adder_b200_layernorm_forward) layernorm_forward = nullptr;
    decltype(&adder_b200_layernorm_backward_workspace_bytes) layernorm_backward_workspace_bytes = nullptr;
    decltype(&adder_b200_layernorm_backward) layernorm_backward = nullptr;
    decltype(&adder_b200_log_probs_forward) log_probs_forward = nullptr;
    decltype(&adder_b200_log_probs_backward) log_probs_backward = nullptr;
    decltype(&adder_b200_rmsnorm_forward) rmsnorm_forward = nullptr;
    decltype(&adder_b200_rmsnorm_forward_8bit) rmsnorm_forward_8bit = nullptr;
    decltype(&adder_b200_rmsnorm_backward_workspace_bytes) rmsnorm_backward_workspace_bytes = nullptr;
    decltype(&adder_b200_rmsnorm_backward) rmsnorm_backward = nullptr;
    decltype(&adder_b200_quantize_rows) quantize_rows = nullptr;
    decltype(&adder_b200_linear_8bit) linear_8bit = nullptr;
    decltype(&adder_b200_distillation_forward) distillation_forward = nullptr;
    decltype(&adder_b200_distillation_backward) distillation_backward = nullptr;
    decltype(&adder_b200_verify_drafts) verify_drafts = nullptr;
    decltype(&adder_b200_adamw_step) adamw_step = nullptr;
};
// Written once, by the first bind to the product library, which is never unloaded: autograd nodes made by this path call through it
// for as long as they live, from any thread.  `enabled` is what bind() switches, and only the Python entry points look at it.
Api api;
std::atomic<bool> enabled{false};
PyObject* g_adder_dict = nullptr;          // module dictionaries that hold FAST_CLAMP, OVERLAP_BACKWARD and ETA
PyObject* g_cuda_dict = nullptr;

// A torch.jit trace records the Python layer's autograd functions as operators; what runs here would leave a constant in it.
bool available() { return enabled.load(std::memory_order_acquire) && !torch::jit::tracer::isTracing(); }

// ValueError for what the caller can mend, RuntimeError otherwise, as _lib.check raises.
void check(int status, const char* what) {
    const bool runtime = status == ADDER_ERR_CUDA || status == ADDER_ERR_INTERNAL || status == ADDER_ERR_TIMEOUT;
    TORCH_CHECK(status == ADDER_OK || !runtime, what, ": ", api.status_string(status), " (status ", status, ")");
    TORCH_CHECK_VALUE(status == ADDER_OK, what, ": ", api.status_string(status), " (status ", status, ")");
}

cudaStream_t current_stream(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type = at::kFloat) {
    return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

struct Layer {      // geometry arguments of the C interface
    int n, ci, h, w, co, k, stride, pad, ho, wo;
};
#define ADDER_GEOM(L) (L).n, (L).ci, (L).h, (L).w, (L).co, (L).k, (L).stride, (L).pad

// What the kernels take.  A dual tensor of forward-mode differentiation is left to the Python layer, which refuses it: without a node,
// its tangent would be dropped without a word.
bool unwrapped(const at::Tensor& t) {
    static const c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                              c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                              c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
    return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) && !t._fw_grad(0).defined();
}
bool plain(const at::Tensor& t) { return unwrapped(t) && t.scalar_type() == at::kFloat && t.is_contiguous(); }

bool layer_of(const at::Tensor& x, const at::Tensor& w, int64_t stride, int64_t pad, Layer* L) {
    if (!plain(x) || !plain(w) || x.device() != w.device() || x.dim() != 4 || w.dim() != 4) return false;
    const int64_t k = w.size(2);
    if (w.size(3) != k || (k != 1 && k != 3) || (stride != 1 && stride != 2) || pad < 0 || pad >= k) return false;
    if (w.size(1) != x.size(1) || x.numel() == 0 || w.numel() == 0) return false;
    const int64_t h = x.size(2), wd = x.size(3), ho = (h + 2 * pad - k) / stride + 1, wo = (wd + 2 * pad - k) / stride + 1;
    if (h + 2 * pad < k || wd + 2 * pad < k) return false;
    constexpr int64_t lim = 2147483647;
    if (x.numel() > lim || w.numel() > lim || x.size(0) * w.size(0) * ho * wo > lim) return false;
    *L = Layer{(int)x.size(0), (int)x.size(1), (int)h, (int)wd, (int)w.size(0), (int)k, (int)stride, (int)pad, (int)ho, (int)wo};
    return true;
}

// ------------------------------------------------------------------------------------------ the operations

at::Tensor forward(const at::Tensor& x, const at::Tensor& w, const Layer& L) {
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = empty_on(x, {L.n, L.co, L.ho, L.wo});
    check(api.forward(x.const_data_ptr<float>(), w.const_data_ptr<float>(), out.mutable_data_ptr<float>(), ADDER_GEOM(L), current_stream(x)),
          "adder_b200_forward");
    return out;
}

std::pair<at::Tensor, at::Tensor> forward_with_stats(const at::Tensor& x, const at::Tensor& w, const Layer& L) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int slices = api.forward_stat_slices(ADDER_GEOM(L));
    at::Tensor st = empty_on(x, {L.co, slices > 0 ? slices : 0, 2}, at::kDouble);
    if (slices <= 0) return {forward(x, w, L), st};
    at::Tensor out = empty_on(x, {L.n, L.co, L.ho, L.wo});
    check(api.forward_with_stats(x.const_data_ptr<float>(), w.const_data_ptr<float>(), out.mutable_data_ptr<float>(),
                                 st.mutable_data_ptr<double>(), slices, ADDER_GEOM(L), current_stream(x)), "adder_b200_forward_with_stats");
    return {out, st};
}

// The scratch comes from torch's caching allocator on the current stream: a cached block most of the time, safe with any number
// of threads and streams, and part of the graph's own pool under capture.
void backward_input(const at::Tensor& g, const at::Tensor& x, const at::Tensor& w, const at::Tensor& gx, const Layer& L, bool fast) {
    const size_t bytes = api.backward_input_workspace_bytes(ADDER_GEOM(L));
    at::Tensor ws;
    if (bytes > 0) ws = empty_on(x, {(int64_t)bytes}, at::kByte);
    check(api.backward_input_with_workspace(g.const_data_ptr<float>(), x.const_data_ptr<float>(), w.const_data_ptr<float>(), gx.mutable_data_ptr<float>(),
                                            bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, ADDER_GEOM(L), fast ? ADDER_FLAG_FAST_CLAMP : 0,
                                            current_stream(x)), "adder_b200_backward_input");
}

void backward_weight(const at::Tensor& g, const at::Tensor& x, const at::Tensor& w, const at::Tensor& gw, const Layer& L, float eta) {
    const int64_t bytes = (int64_t)api.backward_weight_workspace_bytes(ADDER_GEOM(L));
    at::Tensor ws = empty_on(x, {bytes}, at::kByte);
    check(api.backward_weight(g.const_data_ptr<float>(), x.const_data_ptr<float>(), w.const_data_ptr<float>(), gw.mutable_data_ptr<float>(), eta,
                              nullptr, ws.mutable_data_ptr(), (size_t)bytes, ADDER_GEOM(L), 0, current_stream(x)), "adder_b200_backward_weight");
}

c10::cuda::CUDAStream side_stream(c10::DeviceIndex dev) {
    static std::mutex mu;
    static std::array<std::unique_ptr<c10::cuda::CUDAStream>, 64> streams;
    std::lock_guard<std::mutex> lock(mu);
    auto& s = streams.at(dev);
    if (!s) s = std::make_unique<c10::cuda::CUDAStream>(c10::cuda::getStreamFromPool(false, dev));
    return *s;
}

// Both gradients; with `overlap` the weight gradient runs on a side stream beside the input gradient.
// What that gives depends on what else runs.  Among other passes (250 drawn layers) it saves 4 % from 1.5e8 to 2.5e8 terms, 2 % up to
// 1e9, less above.  A pass that is waited for gains or loses: where the input gradient is one long chain on few CTAs, the weight
// gradient's CTAs, each of which fills an SM, may take the SMs first and leave it crowded on the rest (256->256 14x14 at batch 2:
// 356 us, 200 one after the other; the other order loses as much on 256->512 14x14 stride 2 at batch 4, 596 against 250).  Below 1.5e8
// terms one after the other is the faster on average there, and the events cost 6 us of host time; inside a graph capture they
// cost nothing.
constexpr double OVERLAP_TERMS = 1.5e8;

template <class Input, class Weight>
void run_both(const at::Tensor& x, bool overlap, double terms, Input input, Weight weight) {
    if (!overlap || (terms < OVERLAP_TERMS && at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None)) {
        input();
        weight();
        return;
    }
    const auto cur = c10::cuda::getCurrentCUDAStream(x.device().index());
    const auto side = side_stream(x.device().index());
    at::cuda::CUDAEvent ready, done;
    ready.record(cur);
    ready.block(side);
    {
        const c10::cuda::CUDAStreamGuard on_side(side);
        weight();
        done.record(side);
    }
    input();
    done.block(cur);
}

void backward_both(const at::Tensor& g, const at::Tensor& x, const at::Tensor& w, const at::Tensor& gx, const at::Tensor& gw,
                   const Layer& L, float eta, bool fast, bool overlap) {
    run_both(x, overlap, (double)L.n * L.ho * L.wo * L.co * L.ci * L.k * L.k, [&] { backward_input(g, x, w, gx, L, fast); }, [&] { backward_weight(g, x, w, gw, L, eta); });
}

// ------------------------------------------------------------------------------------------ any other geometry

// n, ci, h, w, co, kh, kw, sh, sw, ph, pw, dh, dw; then ho, wo
using Conv = std::array<int, 15>;
#define ADDER_CONV_GEOM(c) c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7], c[8], c[9], c[10], c[11], c[12]

bool conv_of(const at::Tensor& x, const at::Tensor& w, const std::array<int64_t, 6>& p, Conv* c) {
    if (!plain(x) || !plain(w) || x.device() != w.device() || x.dim() != 4 || w.dim() != 4) return false;
    if (w.size(1) != x.size(1) || x.numel() == 0 || w.numel() == 0) return false;
    constexpr int64_t lim = 2147483647;
    for (int i = 0; i < 6; ++i)
        if (p[i] < (i == 2 || i == 3 ? 0 : 1) || p[i] > (1 << 20)) return false;      // stride, padding, dilation
    // Beyond 24x24 the input gradient is mostly zeros between the pixels that a window reaches, which columns fold faster (16->16 on
    // 256x256 at batch 8, forward and backward: 1x1 stride 64 1220 us here, 395 as columns; 2x2 stride 24 452 and 399, 1x1 stride 17
    // 177 and 401).
    if (p[0] * p[1] > 600) return false;
    const int64_t h = x.size(2), wd = x.size(3), kh = w.size(2), kw = w.size(3);
    const int64_t eh = h + 2 * p[2] - p[4] * (kh - 1) - 1, ew = wd + 2 * p[3] - p[5] * (kw - 1) - 1;
    if (eh < 0 || ew < 0) return false;
    const int64_t ho = eh / p[0] + 1, wo = ew / p[1] + 1;
    if (x.numel() > lim || w.numel() > lim || x.size(0) * w.size(0) * ho * wo > lim) return false;
    *c = Conv{(int)x.size(0), (int)x.size(1), (int)h, (int)wd, (int)w.size(0), (int)kh, (int)kw, (int)p[0], (int)p[1], (int)p[2], (int)p[3],
              (int)p[4], (int)p[5], (int)ho, (int)wo};
    return api.conv_backward_weight_workspace_bytes(ADDER_CONV_GEOM((*c))) > 0;
}

at::Tensor conv_forward(const at::Tensor& x, const at::Tensor& w, const Conv& c) {
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = empty_on(x, {c[0], c[4], c[13], c[14]});
    check(api.conv_forward(x.const_data_ptr<float>(), w.const_data_ptr<float>(), out.mutable_data_ptr<float>(), ADDER_CONV_GEOM(c),
                           current_stream(x)), "adder_b200_conv_forward");
    return out;
}

void conv_backward_input(const at::Tensor& g, const at::Tensor& x, const at::Tensor& w, const at::Tensor& gx, const Conv& c, bool fast) {
    const size_t bytes = api.conv_backward_input_workspace_bytes(ADDER_CONV_GEOM(c));
    at::Tensor ws;
    if (bytes > 0) ws = empty_on(x, {(int64_t)bytes}, at::kByte);
    check(api.conv_backward_input_with_workspace(g.const_data_ptr<float>(), x.const_data_ptr<float>(), w.const_data_ptr<float>(),
                                                 gx.mutable_data_ptr<float>(), bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, ADDER_CONV_GEOM(c),
                                                 fast ? ADDER_FLAG_FAST_CLAMP : 0, current_stream(x)), "adder_b200_conv_backward_input");
}

void conv_backward_weight(const at::Tensor& g, const at::Tensor& x, const at::Tensor& w, const at::Tensor& gw, const Conv& c, float eta) {
    const int64_t bytes = (int64_t)api.conv_backward_weight_workspace_bytes(ADDER_CONV_GEOM(c));
    at::Tensor ws = empty_on(x, {bytes}, at::kByte);
    check(api.conv_backward_weight(g.const_data_ptr<float>(), x.const_data_ptr<float>(), w.const_data_ptr<float>(),
                                   gw.mutable_data_ptr<float>(), eta, ws.mutable_data_ptr(), (size_t)bytes, ADDER_CONV_GEOM(c),
                                   current_stream(x)), "adder_b200_conv_backward_weight");
}

// ------------------------------------------------------------------------------------------ autograd nodes

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// What a saved-tensor hook hands back need not be what it was given: every backward looks at its tensors again.
constexpr const char* SAVED = "the saved tensors came back in another form: contiguous float32 CUDA tensors of the forward's shapes are needed";

at::Tensor gradient(const Variable& grad, const at::Tensor& x, at::IntArrayRef shape) {
    const at::Tensor g = grad.contiguous();
    TORCH_CHECK(g.scalar_type() == at::kFloat && g.device() == x.device(), "grad_out must be a float32 tensor on the layer's device");
    TORCH_CHECK(g.sizes() == shape, "grad_out has shape ", g.sizes(), ", expected ", shape);
    return g;
}

struct Settings { bool fast, overlap; float eta; };

// The module-level switches are read when the backward runs, as the Python layer reads them.
Settings settings() {
    pybind11::gil_scoped_acquire gil;
    auto flag = [](PyObject* dict, const char* name) {
        PyObject* v = PyDict_GetItemString(dict, name);
        return v != nullptr && PyObject_IsTrue(v) == 1;
    };
    PyObject* eta = PyDict_GetItemString(g_cuda_dict, "ETA");
    return {flag(g_adder_dict, "FAST_CLAMP"), flag(g_adder_dict, "OVERLAP_BACKWARD"), eta != nullptr ? (float)PyFloat_AsDouble(eta) : 0.2f};
}


// adder2d on NCHW tensors (adder.py:22-80 of the reference).
struct AdderLayer : public torch::autograd::Function<AdderLayer> {
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Variable& w, int64_t stride, int64_t pad, bool stats) {
        Layer L;
        TORCH_CHECK(layer_of(x, w, stride, pad, &L));
        ctx->save_for_backward({x, w});
        ctx->saved_data["stride"] = stride;
        ctx->saved_data["pad"] = pad;
        if (!stats) return {::forward(x, w, L)};
        auto r = ::forward_with_stats(x, w, L);
        ctx->mark_non_differentiable({r.second});
        ctx->set_materialize_grads(false);
        return {r.first, r.second};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return {Variable(), Variable(), Variable(), Variable(), Variable()};
        const auto saved = ctx->get_saved_variables();
        const Variable &x = saved[0], &w = saved[1];
        Layer L;
        TORCH_CHECK(layer_of(x, w, ctx->saved_data["stride"].toInt(), ctx->saved_data["pad"].toInt(), &L), SAVED);
        const at::Tensor g = gradient(grads[0], x, {L.n, L.co, L.ho, L.wo});
        const c10::cuda::CUDAGuard guard(x.device());
        const Settings set = settings();
        at::Tensor gx, gw;
        if (ctx->needs_input_grad(0)) gx = empty_on(x, x.sizes());
        if (ctx->needs_input_grad(1)) gw = empty_on(w, w.sizes());
        if (gx.defined() && gw.defined()) backward_both(g, x, w, gx, gw, L, set.eta, set.fast, set.overlap);
        else if (gx.defined()) backward_input(g, x, w, gx, L, set.fast);
        else if (gw.defined()) backward_weight(g, x, w, gw, L, set.eta);
        return {gx, gw, Variable(), Variable(), Variable()};
    }
};

struct ConvLayer : public torch::autograd::Function<ConvLayer> {
    static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& w, const std::vector<int64_t>& p) {
        Conv c;
        TORCH_CHECK(conv_of(x, w, {p[0], p[1], p[2], p[3], p[4], p[5]}, &c));
        ctx->save_for_backward({x, w});
        ctx->saved_data["p"] = p;
        return conv_forward(x, w, c);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Variable &x = saved[0], &w = saved[1];
        const auto p = ctx->saved_data["p"].toIntVector();
        Conv c;
        TORCH_CHECK(conv_of(x, w, {p[0], p[1], p[2], p[3], p[4], p[5]}, &c), SAVED);
        const at::Tensor g = gradient(grads[0], x, {c[0], c[4], c[13], c[14]});
        const c10::cuda::CUDAGuard guard(x.device());
        const Settings set = settings();
        at::Tensor gx, gw;
        if (ctx->needs_input_grad(0)) gx = empty_on(x, x.sizes());
        if (ctx->needs_input_grad(1)) gw = empty_on(w, w.sizes());
        auto input = [&] { conv_backward_input(g, x, w, gx, c, set.fast); };
        auto weight = [&] { conv_backward_weight(g, x, w, gw, c, set.eta); };
        if (gx.defined() && gw.defined()) run_both(x, set.overlap, (double)w.numel() * g.size(0) * c[13] * c[14], input, weight);
        else if (gx.defined()) input();
        else if (gw.defined()) weight();
        return {gx, gw, Variable()};
    }
};

// The column-matrix op (adder.py:43-80 of the reference): X[K,P] is the 1x1 layer [1,K,1,P], W[Co,K] its kernel.
bool column_of(const at::Tensor& w, const at::Tensor& x, Layer* L) {
    if (!plain(w) || !plain(x) || w.dim() != 2 || x.dim() != 2 || w.size(1) != x.size(0) || w.numel() == 0 || x.numel() == 0 ||
        w.device() != x.device())
        return false;
    constexpr int64_t lim = 2147483647;
    if (w.numel() > lim || x.numel() > lim || w.size(0) * x.size(1) > lim) return false;
    *L = Layer{1, (int)x.size(0), 1, (int)x.size(1), (int)w.size(0), 1, 1, 0, 1, (int)x.size(1)};
    return true;
}

struct AdderColumn : public torch::autograd::Function<AdderColumn> {
    static Variable forward(AutogradContext* ctx, const Variable& w, const Variable& x) {
        Layer L;
        TORCH_CHECK(column_of(w, x, &L));
        ctx->save_for_backward({w, x});
        return ::forward(x, w, L).view({L.co, L.w});
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Variable &w = saved[0], &x = saved[1];
        Layer L;
        TORCH_CHECK(column_of(w, x, &L), SAVED);
        const at::Tensor g = gradient(grads[0], x, {L.co, L.w});
        const c10::cuda::CUDAGuard guard(x.device());
        at::Tensor gx = empty_on(x, x.sizes()), gw = empty_on(w, w.sizes());
        backward_both(g, x, w, gx, gw, L, 0.2f, false, true);
        return {gw, gx};
    }
};

// ------------------------------------------------------------------------------------------ layer norm, log probabilities, AdamW

// ADDER_TYPE_* of a tensor, or -1
int type_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return ADDER_TYPE_F32;
        case at::kBFloat16: return ADDER_TYPE_BF16;
        case at::kHalf: return ADDER_TYPE_F16;
        default: return -1;
    }
}

// The last `inner` extents of t lie one after the other, and so do the rows that they make, *stride elements apart.
bool rows_of(const at::Tensor& t, int64_t inner, int64_t d, int64_t* stride) {
    if (t.is_contiguous()) {
        *stride = d;
        return true;
    }
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t want = 1, i = t.dim() - 1;
    for (; i >= t.dim() - inner; --i) {
        if (sizes[i] != 1 && strides[i] != want) return false;
        want *= sizes[i];
    }
    bool first = true;
    for (; i >= 0; --i) {
        if (sizes[i] == 1) continue;
        if (first) *stride = want = strides[i];
        else if (strides[i] != want) return false;
        first = false;
        want *= sizes[i];
    }
    if (first) *stride = d;
    return true;
}

struct Norm {      // a checked call
    int64_t rows, d, x_stride, r_stride;
    int type, weight_type;
    double eps;
};

bool norm_of(const at::Tensor& x, const at::Tensor* r, const at::Tensor* w, const at::Tensor* b, at::IntArrayRef shape, double eps, Norm* n) {
    n->type = type_code(x);
    if (n->type < 0 || !unwrapped(x) || shape.empty() || x.dim() < (int64_t)shape.size() || !(eps >= 0.0)) return false;
    if (x.sizes().slice(x.dim() - shape.size()) != shape) return false;
    n->d = c10::multiply_integers(shape);
    if (n->d == 0 || x.numel() == 0) return false;
    n->rows = x.numel() / n->d;
    n->r_stride = 0;
    if (!rows_of(x, shape.size(), n->d, &n->x_stride)) return false;
    if (r != nullptr && (!unwrapped(*r) || r->device() != x.device() || r->scalar_type() != x.scalar_type() || r->sizes() != x.sizes() ||
                         !rows_of(*r, shape.size(), n->d, &n->r_stride)))
        return false;
    n->weight_type = n->type;
    for (const at::Tensor* t : {w, b}) {
        if (t == nullptr) continue;
        if (!unwrapped(*t) || !t->is_contiguous() || t->device() != x.device() || t->sizes() != shape) return false;
        n->weight_type = type_code(*t);
        if (n->weight_type != n->type && n->weight_type != ADDER_TYPE_F32) return false;
    }
    if (w != nullptr && b != nullptr && w->scalar_type() != b->scalar_type()) return false;
    n->eps = eps;
    return true;
}

// A gradient as its memory stands: contiguous, and no lazy negation (which a view of a conjugate's imaginary part is).
at::Tensor whole_gradient(const at::Tensor& g) { return (g.is_neg() ? g.resolve_neg() : g).contiguous(); }

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct NormResult { at::Tensor y, h, mean, rstd; };

NormResult norm_forward(const at::Tensor& x, const at::Tensor& r, const at::Tensor& w, const at::Tensor& b, const Norm& n, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    NormResult out;
    out.y = empty_on(x, x.sizes(), x.scalar_type());
    if (r.defined()) out.h = empty_on(x, x.sizes(), x.scalar_type());
    if (keep) {
        out.mean = empty_on(x, {n.rows});
        out.rstd = empty_on(x, {n.rows});
    }
    check(api.layernorm_forward(ptr(x), ptr(r), ptr(w), ptr(b), ptr(out.y), ptr(out.h), static_cast<float*>(ptr(out.mean)),
                                static_cast<float*>(ptr(out.rstd)), n.rows, n.d, n.x_stride, n.r_stride, n.type, n.weight_type, (float)n.eps,
                                current_stream(x)), "adder_b200_layernorm_forward");
    return out;
}

using Optional = std::optional<at::Tensor>;

// `grad` of an operator that is differentiable once, computed from the tensors in `from`.  Where the backward pass is itself recorded
// (create_graph) it must not count as a constant: it gets a node that raises when it is differentiated.  The node's edges lead to what the
// gradient depends on, so that a call for the gradients of some inputs alone comes by it, too.
void once(const char* name, const at::Tensor& grad, std::initializer_list<const at::Tensor*> from) {
    if (!grad.defined() || !at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges;
    for (const at::Tensor* t : from)
        if (t->defined() && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
    if (edges.empty()) return;
    torch::autograd::set_history(grad, std::make_shared<torch::autograd::Error>(std::string(name) + " is differentiable once", std::move(edges)));
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Optional& r, const Optional& w, const Optional& b, const Norm& n) {
        const at::Tensor none;
        auto out = norm_forward(x, r.value_or(none), w.value_or(none), b.value_or(none), n, true);
        ctx->save_for_backward({r ? out.h : x, w.value_or(none), out.mean, out.rstd});
        ctx->saved_data["sizes"] = std::vector<int64_t>{n.rows, n.d, n.type, n.weight_type, r.has_value(), b.has_value()};
        if (b) ctx->saved_data["shape"] = b->sizes().vec();
        ctx->set_materialize_grads(false);
        return r ? variable_list{out.y, out.h} : variable_list{out.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Variable none;
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int64_t rows = sizes[0], d = sizes[1];
        const int type = (int)sizes[2], weight_type = (int)sizes[3];
        const bool has_r = sizes[4], has_b = sizes[5];
        at::Tensor dy = grads[0], dh = has_r ? grads[1] : none;
        if (!dy.defined() && !dh.defined()) return {none, none, none, none, none};
        const auto saved = ctx->get_saved_variables();
        const Variable &h = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
        int64_t stride;
        TORCH_CHECK(unwrapped(h) && type_code(h) == type && h.numel() == rows * d && plain(mean) && plain(rstd) && mean.numel() == rows &&
                    rstd.numel() == rows && mean.device() == h.device() && rstd.device() == h.device(), SAVED);
        TORCH_CHECK(!w.defined() || (unwrapped(w) && w.is_contiguous() && type_code(w) == weight_type && w.numel() == d && w.device() == h.device()), SAVED);
        const c10::cuda::CUDAGuard guard(h.device());
        at::Tensor h2 = h;      // rows of consecutive elements
        if (!rows_of(h, 1, d, &stride) || h.dim() == 0 || h.size(-1) != d) {
            h2 = h.contiguous();
            stride = d;
        }
        if (!dy.defined()) dy = at::zeros_like(h, at::MemoryFormat::Contiguous);
        dy = whole_gradient(dy);
        if (dh.defined()) dh = whole_gradient(dh);
        for (const at::Tensor* g : {&dy, &dh})
            TORCH_CHECK(!g->defined() || (g->scalar_type() == h.scalar_type() && g->device() == h.device() && g->sizes() == h.sizes()),
                        "the gradient must have the type, device and shape of the output");
        int edge = 0;
        const bool need_x = ctx->needs_input_grad(edge++), need_r = has_r && ctx->needs_input_grad(edge++);
        const bool need_w = w.defined() && ctx->needs_input_grad(edge++), need_b = has_b && ctx->needs_input_grad(edge++);
        at::Tensor dx, dw, db, ws;
        if (need_x || need_r) dx = empty_on(h, h.sizes(), h.scalar_type());
        const at::ScalarType weight_scalar = weight_type == ADDER_TYPE_F32 ? at::kFloat : h.scalar_type();
        if (need_w) dw = empty_on(h, w.sizes(), weight_scalar);
        if (need_b) db = empty_on(h, ctx->saved_data["shape"].toIntVector(), weight_scalar);
        const size_t bytes = need_w || need_b ? api.layernorm_backward_workspace_bytes(rows, d) : 0;
        if (bytes > 0) ws = empty_on(h, {(int64_t)bytes}, at::kByte);
        check(api.layernorm_backward(ptr(dy), ptr(dh), ptr(h2), ptr(w), mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(), ptr(dx), ptr(dw),
                                     ptr(db), ptr(ws), bytes, rows, d, stride, type, weight_type, current_stream(h)), "adder_b200_layernorm_backward");
        const Variable& input = need_x || need_r ? h : none;      // h is an output as well, and asks for gradients whatever the inputs do
        once("layer_norm", dx, {&dy, &dh, &input, &w});
        once("layer_norm", dw, {&dy, &input});
        once("layer_norm", db, {&dy});
        return {need_x ? dx : none, need_r ? dx : none, dw, db, none};
    }
};

struct LogProbs {      // a checked call
    int64_t rows, classes, stride, ignore;
    int type, top_k;
    bool entropy;
};

bool log_probs_of(const at::Tensor& x, const at::Tensor* targets, int64_t top_k, LogProbs* n) {
    n->type = type_code(x);
    if (n->type < 0 || !unwrapped(x) || x.dim() < 1 || x.numel() == 0) return false;
    n->classes = x.size(-1);
    n->rows = x.numel() / n->classes;
    if (top_k < 0 || top_k > 32 || top_k > n->classes || !rows_of(x, 1, n->classes, &n->stride)) return false;
    n->top_k = (int)top_k;
    return targets == nullptr || (unwrapped(*targets) && targets->scalar_type() == at::kLong && targets->is_contiguous() &&
                                  targets->device() == x.device() && targets->sizes() == x.sizes().slice(0, x.dim() - 1));
}

struct LogProbsResult { at::Tensor log_prob, entropy, top, indices, stats; };

LogProbsResult log_probs_forward(const at::Tensor& x, const at::Tensor& targets, const LogProbs& n, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    LogProbsResult out;
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    if (targets.defined()) out.log_prob = empty_on(x, lead);
    if (n.entropy) out.entropy = empty_on(x, lead);
    if (n.top_k > 0) {
        c10::SmallVector<int64_t, 5> sizes(lead.begin(), lead.end());
        sizes.push_back(n.top_k);
        out.top = empty_on(x, sizes);
        out.indices = empty_on(x, sizes, at::kLong);
    }
    if (keep) out.stats = empty_on(x, {n.rows, 2});
    check(api.log_probs_forward(ptr(x), n.type, n.rows, n.classes, n.stride, static_cast<const long long*>(ptr(targets)), n.ignore, n.top_k,
                                static_cast<float*>(ptr(out.log_prob)), static_cast<float*>(ptr(out.entropy)), static_cast<float*>(ptr(out.stats)),
                                static_cast<float*>(ptr(out.top)), static_cast<long long*>(ptr(out.indices)), current_stream(x)),
          "adder_b200_log_probs_forward");
    return out;
}

struct LogProbsNode : public torch::autograd::Function<LogProbsNode> {
    // the outputs that there are, in the order of LogProbsResult
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Optional& targets, const LogProbs& n) {
        const at::Tensor none;
        auto out = log_probs_forward(x, targets.value_or(none), n, true);
        ctx->save_for_backward({x, targets.value_or(none), out.stats, out.entropy, out.indices});
        ctx->saved_data["args"] = std::vector<int64_t>{n.rows, n.classes, n.ignore, n.type, n.top_k, targets.has_value(), n.entropy};
        ctx->set_materialize_grads(false);
        if (out.indices.defined()) ctx->mark_non_differentiable({out.indices});
        variable_list list;
        for (const at::Tensor* t : {&out.log_prob, &out.entropy, &out.top, &out.indices})
            if (t->defined()) list.push_back(*t);
        return list;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Variable none;
        const auto a = ctx->saved_data["args"].toIntVector();
        const int64_t rows = a[0], classes = a[1], ignore = a[2];
        const int type = (int)a[3], top_k = (int)a[4];
        size_t at = 0;
        at::Tensor g_lp, g_ent, g_top;
        if (a[5]) g_lp = grads[at++];
        if (a[6]) g_ent = grads[at++];
        if (top_k > 0) g_top = grads[at++];
        if (!g_lp.defined() && !g_ent.defined() && !g_top.defined()) return {none, none, none};
        const auto saved = ctx->get_saved_variables();
        const Variable &x = saved[0], &targets = saved[1], &stats = saved[2], &entropy = saved[3], &indices = saved[4];
        TORCH_CHECK(unwrapped(x) && type_code(x) == type && x.dim() >= 1 && x.size(-1) == classes && x.numel() == rows * classes && plain(stats) &&
                    stats.numel() == 2 * rows && stats.device() == x.device() &&
                    (!a[6] || (plain(entropy) && entropy.numel() == rows && entropy.device() == x.device())), SAVED);
        const auto whole = [&](const Variable& t, int64_t count) {
            return unwrapped(t) && t.scalar_type() == at::kLong && t.is_contiguous() && t.numel() == count && t.device() == x.device();
        };
        TORCH_CHECK((!a[5] || whole(targets, rows)) && (top_k == 0 || whole(indices, rows * top_k)), SAVED);
        const c10::cuda::CUDAGuard guard(x.device());
        for (at::Tensor* g : {&g_lp, &g_ent, &g_top})
            if (g->defined()) {
                *g = whole_gradient(*g);
                TORCH_CHECK(g->scalar_type() == at::kFloat && g->device() == x.device() && g->numel() == (g == &g_top ? rows * top_k : rows),
                            "the gradient must be a float32 tensor of the output's shape and device");
            }
        at::Tensor x2 = x;
        int64_t stride;
        if (!rows_of(x, 1, classes, &stride)) {
            x2 = x.contiguous();
            stride = classes;
        }
        at::Tensor dx = empty_on(x, x.sizes(), x.scalar_type());
        check(api.log_probs_backward(ptr(x2), type, rows, classes, stride, static_cast<const long long*>(ptr(targets)), ignore, top_k,
                                     static_cast<const long long*>(ptr(indices)), stats.const_data_ptr<float>(), static_cast<const float*>(ptr(entropy)),
                                     static_cast<const float*>(ptr(g_lp)), static_cast<const float*>(ptr(g_ent)), static_cast<const float*>(ptr(g_top)),
                                     ptr(dx), current_stream(x)), "adder_b200_log_probs_backward");
        once("token_log_probs", dx, {&x, &g_lp, &g_ent, &g_top});
        return {dx, none, none};
    }
};

struct RmsResult { at::Tensor y, h, rstd; };

RmsResult rms_forward(const at::Tensor& x, const at::Tensor& r, const at::Tensor& w, const Norm& n, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    RmsResult out;
    out.y = empty_on(x, x.sizes(), x.scalar_type());
    if (r.defined()) out.h = empty_on(x, x.sizes(), x.scalar_type());
    if (keep) out.rstd = empty_on(x, {n.rows});
    check(api.rmsnorm_forward(ptr(x), ptr(r), ptr(w), ptr(out.y), ptr(out.h), static_cast<float*>(ptr(out.rstd)), n.rows, n.d, n.x_stride,
                              n.r_stride, n.type, n.weight_type, (float)n.eps, current_stream(x)), "adder_b200_rmsnorm_forward");
    return out;
}

struct RmsNorm : public torch::autograd::Function<RmsNorm> {
    static variable_list forward(AutogradContext* ctx, const Variable& x, const Optional& r, const Optional& w, const Norm& n) {
        const at::Tensor none;
        auto out = rms_forward(x, r.value_or(none), w.value_or(none), n, true);
        ctx->save_for_backward({r ? out.h : x, w.value_or(none), out.rstd});
        ctx->saved_data["sizes"] = std::vector<int64_t>{n.rows, n.d, n.type, n.weight_type, r.has_value()};
        ctx->set_materialize_grads(false);
        return r ? variable_list{out.y, out.h} : variable_list{out.y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Variable none;
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const int64_t rows = sizes[0], d = sizes[1];
        const int type = (int)sizes[2], weight_type = (int)sizes[3];
        const bool has_r = sizes[4];
        at::Tensor dy = grads[0], dh = has_r ? grads[1] : none;
        if (!dy.defined() && !dh.defined()) return {none, none, none, none};
        const auto saved = ctx->get_saved_variables();
        const Variable &h = saved[0], &w = saved[1], &rstd = saved[2];
        int64_t stride;
        TORCH_CHECK(unwrapped(h) && type_code(h) == type && h.numel() == rows * d && plain(rstd) && rstd.numel() == rows && rstd.device() == h.device(), SAVED);
        TORCH_CHECK(!w.defined() || (unwrapped(w) && w.is_contiguous() && type_code(w) == weight_type && w.numel() == d && w.device() == h.device()), SAVED);
        const c10::cuda::CUDAGuard guard(h.device());
        at::Tensor h2 = h;      // rows of consecutive elements
        if (!rows_of(h, 1, d, &stride) || h.dim() == 0 || h.size(-1) != d) {
            h2 = h.contiguous();
            stride = d;
        }
        if (!dy.defined()) dy = at::zeros_like(h, at::MemoryFormat::Contiguous);
        dy = whole_gradient(dy);
        if (dh.defined()) dh = whole_gradient(dh);
        for (const at::Tensor* g : {&dy, &dh})
            TORCH_CHECK(!g->defined() || (g->scalar_type() == h.scalar_type() && g->device() == h.device() && g->sizes() == h.sizes()),
                        "the gradient must have the type, device and shape of the output");
        int edge = 0;
        const bool need_x = ctx->needs_input_grad(edge++), need_r = has_r && ctx->needs_input_grad(edge++);
        const bool need_w = w.defined() && ctx->needs_input_grad(edge++);
        at::Tensor dx, dw, ws;
        if (need_x || need_r) dx = empty_on(h, h.sizes(), h.scalar_type());
        if (need_w) dw = empty_on(h, w.sizes(), w.scalar_type());
        const size_t bytes = need_w ? api.rmsnorm_backward_workspace_bytes(rows, d) : 0;
        if (bytes > 0) ws = empty_on(h, {(int64_t)bytes}, at::kByte);
        check(api.rmsnorm_backward(ptr(dy), ptr(dh), ptr(h2), ptr(w), rstd.const_data_ptr<float>(), ptr(dx), ptr(dw), ptr(ws), bytes, rows, d, stride,
                                   type, weight_type, current_stream(h)), "adder_b200_rmsnorm_backward");
        const Variable& input = need_x || need_r ? h : none;      // h is an output as well, and asks for gradients whatever the inputs do
        once("rms_norm", dx, {&dy, &dh, &input, &w});
        once("rms_norm", dw, {&dy, &input});
        return {need_x ? dx : none, need_r ? dx : none, dw, none};
    }
};

struct Distill {      // a checked call
    int64_t rows, classes, stride, ignore;
    int type, teacher_type, k;
    double temperature;
};

bool whole_long(const at::Tensor& t, const at::Device& dev) {
    return unwrapped(t) && t.scalar_type() == at::kLong && t.is_contiguous() && t.device() == dev;
}

bool distill_of(const at::Tensor& x, const at::Tensor& teacher, const at::Tensor& indices, const at::Tensor* targets, Distill* n) {
    n->type = type_code(x);
    n->teacher_type = type_code(teacher);
    if (n->type < 0 || n->teacher_type < 0 || !unwrapped(x) || x.dim() < 1 || x.numel() == 0) return false;
    n->classes = x.size(-1);
    n->rows = x.numel() / n->classes;
    if (!rows_of(x, 1, n->classes, &n->stride) || !(n->temperature > 0.0) || !std::isfinite(n->temperature)) return false;
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    if (!unwrapped(teacher) || !teacher.is_contiguous() || teacher.device() != x.device() || teacher.dim() != x.dim() ||
        teacher.sizes().slice(0, lead.size()) != lead || teacher.size(-1) < 1 || teacher.size(-1) > 256 || (at::GradMode::is_enabled() && teacher.requires_grad()))
        return false;
    n->k = (int)teacher.size(-1);
    return whole_long(indices, x.device()) && indices.sizes() == teacher.sizes() && (targets == nullptr || (whole_long(*targets, x.device()) && targets->sizes() == lead));
}

struct DistillResult { at::Tensor divergence, log_prob, stats, mass; };

DistillResult distill_forward(const at::Tensor& x, const at::Tensor& teacher, const at::Tensor& indices, const at::Tensor& targets, const Distill& n, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    DistillResult out;
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    out.divergence = empty_on(x, lead);
    if (targets.defined()) out.log_prob = empty_on(x, lead);
    if (keep) {
        out.stats = empty_on(x, {n.rows, 3});
        out.mass = empty_on(x, {n.rows, n.k});
    }
    check(api.distillation_forward(ptr(x), n.type, n.rows, n.classes, n.stride, ptr(teacher), n.teacher_type,
                                   static_cast<const long long*>(ptr(indices)), n.k, (float)n.temperature, static_cast<const long long*>(ptr(targets)), n.ignore, static_cast<float*>(ptr(out.divergence)),
                                   static_cast<float*>(ptr(out.log_prob)), static_cast<float*>(ptr(out.stats)), static_cast<float*>(ptr(out.mass)),
                                   current_stream(x)), "adder_b200_distillation_forward");
    return out;
}

struct DistillNode : public torch::autograd::Function<DistillNode> {
    static variable_list forward(AutogradContext* ctx, const Variable& x, const at::Tensor& teacher, const at::Tensor& indices, const Optional& targets,
                                 const Distill& n) {
        const at::Tensor none;
        auto out = distill_forward(x, teacher, indices, targets.value_or(none), n, true);
        ctx->save_for_backward({x, indices, targets.value_or(none), out.stats, out.mass});
        ctx->saved_data["args"] = std::vector<int64_t>{n.rows, n.classes, n.ignore, n.type, n.k, targets.has_value()};
        ctx->saved_data["temperature"] = n.temperature;
        ctx->set_materialize_grads(false);
        variable_list list{out.divergence};
        if (targets) list.push_back(out.log_prob);
        return list;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Variable none;
        const auto a = ctx->saved_data["args"].toIntVector();
        const int64_t rows = a[0], classes = a[1], ignore = a[2];
        const int type = (int)a[3], k = (int)a[4];
        at::Tensor g_div = grads[0], g_lp = a[5] ? grads[1] : none;
        if (!g_div.defined() && !g_lp.defined()) return {none, none, none, none, none};
        const auto saved = ctx->get_saved_variables();
        const Variable &x = saved[0], &indices = saved[1], &targets = saved[2], &stats = saved[3], &mass = saved[4];
        TORCH_CHECK(unwrapped(x) && type_code(x) == type && x.dim() >= 1 && x.size(-1) == classes && x.numel() == rows * classes && plain(stats) &&
                    stats.numel() == 3 * rows && stats.device() == x.device() && plain(mass) && mass.numel() == rows * k && mass.device() == x.device(), SAVED);
        TORCH_CHECK(whole_long(indices, x.device()) && indices.numel() == rows * k && (!a[5] || (whole_long(targets, x.device()) && targets.numel() == rows)), SAVED);
        const c10::cuda::CUDAGuard guard(x.device());
        for (at::Tensor* g : {&g_div, &g_lp})
            if (g->defined()) {
                *g = whole_gradient(*g);
                TORCH_CHECK(g->scalar_type() == at::kFloat && g->device() == x.device() && g->numel() == rows,
                            "the gradient must be a float32 tensor of the output's shape and device");
            }
        at::Tensor x2 = x;
        int64_t stride;
        if (!rows_of(x, 1, classes, &stride)) {
            x2 = x.contiguous();
            stride = classes;
        }
        at::Tensor dx = empty_on(x, x.sizes(), x.scalar_type());
        check(api.distillation_backward(ptr(x2), type, rows, classes, stride, static_cast<const long long*>(ptr(indices)), k,
                                        (float)ctx->saved_data["temperature"].toDouble(), static_cast<const long long*>(ptr(targets)), ignore,
                                        stats.const_data_ptr<float>(), mass.const_data_ptr<float>(), static_cast<const float*>(ptr(g_div)),
                                        static_cast<const float*>(ptr(g_lp)), ptr(dx), current_stream(x)), "adder_b200_distillation_backward");
        once("distillation", dx, {&x, &g_div, &g_lp});
        return {dx, none, none, none, none};
    }
};

// Codes whose rows begin at multiples of 16 bytes.
struct Codes {
    at::Tensor values;
    int64_t stride;
};
Codes empty_codes(const at::Tensor& like, at::IntArrayRef sizes) {
    c10::SmallVector<int64_t, 5> whole(sizes.begin(), sizes.end());
    const int64_t d = whole.back(), stride = (d + 15) / 16 * 16;
    whole.back() = stride;
    at::Tensor t = empty_on(like, whole, at::kFloat8_e4m3fn);
    return {stride == d ? t : t.slice(-1, 0, d), stride};
}
at::Tensor empty_scales(const at::Tensor& like, at::IntArrayRef sizes) {
    c10::SmallVector<int64_t, 5> whole(sizes.begin(), sizes.end());
    whole.back() = (whole.back() + 127) / 128;
    return empty_on(like, whole);
}
// Codes as the product takes them; false: they have to be copied, or are none.
bool codes_of(const at::Tensor& values, const at::Tensor& scales, int64_t* rows, int64_t* stride) {
    if (!unwrapped(values) || values.scalar_type() != at::kFloat8_e4m3fn || values.dim() < 1 || values.numel() == 0 || !plain(scales) ||
        scales.device() != values.device() || scales.dim() != values.dim())
        return false;
    const int64_t d = values.size(-1);
    *rows = values.numel() / d;
    if (!rows_of(values, 1, d, stride)) return false;
    if (*rows == 1) *stride = (d + 15) / 16 * 16;
    return *stride % 16 == 0 && *stride >= d && ((uintptr_t)values.data_ptr() & 15) == 0 && scales.size(-1) == (d + 127) / 128;
}

// ------------------------------------------------------------------------------------------ Python entry points

const at::Tensor* tensor_arg(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool int_arg(PyObject* o, int64_t* v) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

bool needs_node(const at::Tensor& a, const at::Tensor& b) { return at::GradMode::is_enabled() && (a.requires_grad() || b.requires_grad()); }

// layer(x, w, stride, padding) -> out, or None
PyObject* py_layer(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *w = tensor_arg(args[1]);
    int64_t stride, pad;
    Layer L;
    if (x == nullptr || w == nullptr || !int_arg(args[2], &stride) || !int_arg(args[3], &pad) || !layer_of(*x, *w, stride, pad, &L)) Py_RETURN_NONE;
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = needs_node(*x, *w) ? AdderLayer::apply(*x, *w, stride, pad, false)[0] : forward(*x, *w, L);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// conv(x, w, sh, sw, ph, pw, dh, dw) -> out, or None
PyObject* py_conv(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *w = tensor_arg(args[1]);
    std::array<int64_t, 6> p;
    for (int i = 0; i < 6; ++i)
        if (!int_arg(args[2 + i], &p[i])) Py_RETURN_NONE;
    Conv c;
    if (x == nullptr || w == nullptr || !conv_of(*x, *w, p, &c)) Py_RETURN_NONE;
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        out = needs_node(*x, *w) ? ConvLayer::apply(*x, *w, std::vector<int64_t>(p.begin(), p.end())) : conv_forward(*x, *w, c);
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// layer_with_stats(x, w, stride, padding) -> (out, statistics), or None
PyObject* py_layer_with_stats(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *w = tensor_arg(args[1]);
    int64_t stride, pad;
    Layer L;
    if (x == nullptr || w == nullptr || !int_arg(args[2], &stride) || !int_arg(args[3], &pad) || !layer_of(*x, *w, stride, pad, &L)) Py_RETURN_NONE;
    at::Tensor out, st;
    {
        pybind11::gil_scoped_release no_gil;
        if (needs_node(*x, *w)) {
            auto r = AdderLayer::apply(*x, *w, stride, pad, true);
            out = r[0]; st = r[1];
        } else {
            std::tie(out, st) = forward_with_stats(*x, *w, L);
        }
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(st)));
    END_HANDLE_TH_ERRORS
}

bool affine_args(PyObject* scale, PyObject* shift, PyObject* residual, const at::Tensor& like, int64_t channels, at::IntArrayRef shape,
                 const at::Tensor** sc, const at::Tensor** sh, const at::Tensor** res) {
    *sc = tensor_arg(scale); *sh = tensor_arg(shift);
    *res = residual == Py_None ? nullptr : tensor_arg(residual);
    if (*sc == nullptr || *sh == nullptr || (residual != Py_None && *res == nullptr)) return false;
    for (const at::Tensor* t : {*sc, *sh})
        if (!plain(*t) || t->numel() != channels || t->device() != like.device()) return false;
    return *res == nullptr || (plain(**res) && (*res)->sizes() == shape && (*res)->device() == like.device() && !(*res)->requires_grad());
}

// layer_affine(x, w, stride, padding, scale, shift, residual, relu) -> relu?(layer * scale + shift + residual) without autograd, or None
PyObject* py_layer_affine(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *w = tensor_arg(args[1]), *sc, *sh, *res;
    int64_t stride, pad;
    Layer L;
    if (x == nullptr || w == nullptr || !int_arg(args[2], &stride) || !int_arg(args[3], &pad) || !layer_of(*x, *w, stride, pad, &L) || needs_node(*x, *w))
        Py_RETURN_NONE;
    const std::array<int64_t, 4> shape{L.n, L.co, L.ho, L.wo};
    if (!affine_args(args[4], args[5], args[6], *x, L.co, shape, &sc, &sh, &res)) Py_RETURN_NONE;
    const int relu = PyObject_IsTrue(args[7]);
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::cuda::CUDAGuard guard(x->device());
        out = empty_on(*x, shape);
        check(api.forward_affine(x->const_data_ptr<float>(), w->const_data_ptr<float>(), sc->const_data_ptr<float>(), sh->const_data_ptr<float>(),
                                 res != nullptr ? res->const_data_ptr<float>() : nullptr, relu, out.mutable_data_ptr<float>(), ADDER_GEOM(L),
                                 current_stream(*x)), "adder_b200_forward_affine");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// affine(y, scale, shift, residual, relu) -> the same behind a tensor, or None
PyObject* py_affine(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !available()) Py_RETURN_NONE;
    const at::Tensor *y = tensor_arg(args[0]), *sc, *sh, *res;
    if (y == nullptr || !plain(*y) || y->dim() != 4 || y->numel() == 0 || y->numel() > 2147483647) Py_RETURN_NONE;
    if (!affine_args(args[1], args[2], args[3], *y, y->size(1), y->sizes(), &sc, &sh, &res)) Py_RETURN_NONE;
    const int relu = PyObject_IsTrue(args[4]);
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::cuda::CUDAGuard guard(y->device());
        out = empty_on(*y, y->sizes());
        check(api.affine_forward(y->const_data_ptr<float>(), sc->const_data_ptr<float>(), sh->const_data_ptr<float>(),
                                 res != nullptr ? res->const_data_ptr<float>() : nullptr, out.mutable_data_ptr<float>(), relu, (int)y->size(0),
                                 (int)y->size(1), (int)(y->size(2) * y->size(3)), current_stream(*y)), "adder_b200_affine_forward");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// column(W[Co,K], X[K,P]) -> [Co,P], or None
PyObject* py_column(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 2 || !available()) Py_RETURN_NONE;
    const at::Tensor *w = tensor_arg(args[0]), *x = tensor_arg(args[1]);
    Layer L;
    if (w == nullptr || x == nullptr || !column_of(*w, *x, &L)) Py_RETURN_NONE;
    at::Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        if (needs_node(*w, *x)) out = AdderColumn::apply(*w, *x);
        else out = forward(*x, *w, L).view({L.co, L.w});
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// A tensor that may be left out (None); false: something else.
bool optional_tensor(PyObject* o, const at::Tensor** t) {
    *t = o == Py_None ? nullptr : tensor_arg(o);
    return o == Py_None || *t != nullptr;
}
bool double_arg(PyObject* o, double* v) {
    if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
    else if (PyLong_CheckExact(o)) *v = PyLong_AsDouble(o);
    else return false;
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
Optional optional(const at::Tensor* t) { return t != nullptr ? Optional(*t) : Optional(); }
PyObject* wrap_or_none(at::Tensor t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(t));
}

// layer_norm(x, residual or None, weight or None, bias or None, shape, eps) -> y, or (y, h) with a residual, or None
PyObject* py_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *r, *w, *b;
    double eps;
    if (x == nullptr || !optional_tensor(args[1], &r) || !optional_tensor(args[2], &w) || !optional_tensor(args[3], &b) ||
        !PyTuple_CheckExact(args[4]) || !double_arg(args[5], &eps))
        Py_RETURN_NONE;
    c10::SmallVector<int64_t, 5> shape(PyTuple_GET_SIZE(args[4]));
    for (size_t i = 0; i < shape.size(); ++i)
        if (!int_arg(PyTuple_GET_ITEM(args[4], i), &shape[i])) Py_RETURN_NONE;
    Norm c;
    if (!norm_of(*x, r, w, b, shape, eps, &c)) Py_RETURN_NONE;
    at::Tensor y, h;
    {
        pybind11::gil_scoped_release no_gil;
        bool node = false;
        if (at::GradMode::is_enabled())
            for (const at::Tensor* t : {x, r, w, b}) node = node || (t != nullptr && t->requires_grad());
        if (node) {
            auto out = LayerNorm::apply(*x, optional(r), optional(w), optional(b), c);
            y = out[0];
            if (r != nullptr) h = out[1];
        } else {
            const at::Tensor none;
            auto out = norm_forward(*x, r != nullptr ? *r : none, w != nullptr ? *w : none, b != nullptr ? *b : none, c, false);
            y = out.y; h = out.h;
        }
    }
    if (r == nullptr) return THPVariable_Wrap(std::move(y));
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(h)));
    END_HANDLE_TH_ERRORS
}

// log_probs(logits, targets or None, top_k, entropy, ignore_index) -> (log_prob, entropy, top_log_probs, top_indices), or None
PyObject* py_log_probs(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *targets;
    int64_t top_k;
    LogProbs c;
    if (x == nullptr || !optional_tensor(args[1], &targets) || !int_arg(args[2], &top_k) || !PyBool_Check(args[3]) || !int_arg(args[4], &c.ignore) ||
        !log_probs_of(*x, targets, top_k, &c))
        Py_RETURN_NONE;
    c.entropy = args[3] == Py_True;
    if (targets == nullptr && top_k == 0 && !c.entropy) Py_RETURN_NONE;
    at::Tensor out[4];
    {
        pybind11::gil_scoped_release no_gil;
        if (at::GradMode::is_enabled() && x->requires_grad()) {
            auto list = LogProbsNode::apply(*x, optional(targets), c);
            size_t at = 0;
            const bool there[4] = {targets != nullptr, c.entropy, top_k > 0, top_k > 0};
            for (int i = 0; i < 4; ++i)
                if (there[i]) out[i] = list[at++];
        } else {
            const at::Tensor none;
            auto r = log_probs_forward(*x, targets != nullptr ? *targets : none, c, false);
            out[0] = r.log_prob; out[1] = r.entropy; out[2] = r.top; out[3] = r.indices;
        }
    }
    return Py_BuildValue("(NNNN)", wrap_or_none(std::move(out[0])), wrap_or_none(std::move(out[1])), wrap_or_none(std::move(out[2])),
                         wrap_or_none(std::move(out[3])));
    END_HANDLE_TH_ERRORS
}

// rms_norm(x, residual or None, weight or None, shape, eps) -> y, or (y, h) with a residual, or None
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *r, *w;
    double eps;
    if (x == nullptr || !optional_tensor(args[1], &r) || !optional_tensor(args[2], &w) || !PyTuple_CheckExact(args[3]) || !double_arg(args[4], &eps))
        Py_RETURN_NONE;
    c10::SmallVector<int64_t, 5> shape(PyTuple_GET_SIZE(args[3]));
    for (size_t i = 0; i < shape.size(); ++i)
        if (!int_arg(PyTuple_GET_ITEM(args[3], i), &shape[i])) Py_RETURN_NONE;
    Norm c;
    if (!norm_of(*x, r, w, nullptr, shape, eps, &c)) Py_RETURN_NONE;
    at::Tensor y, h;
    {
        pybind11::gil_scoped_release no_gil;
        bool node = false;
        if (at::GradMode::is_enabled())
            for (const at::Tensor* t : {x, r, w}) node = node || (t != nullptr && t->requires_grad());
        if (node) {
            auto out = RmsNorm::apply(*x, optional(r), optional(w), c);
            y = out[0];
            if (r != nullptr) h = out[1];
        } else {
            const at::Tensor none;
            auto out = rms_forward(*x, r != nullptr ? *r : none, w != nullptr ? *w : none, c, false);
            y = out.y; h = out.h;
        }
    }
    if (r == nullptr) return THPVariable_Wrap(std::move(y));
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(h)));
    END_HANDLE_TH_ERRORS
}

// rms_norm_8bit(x, weight or None, eps, residual or None) -> (values, scales, h or None), or None
PyObject* py_rms_norm_8bit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *r, *w;
    double eps;
    if (x == nullptr || !optional_tensor(args[1], &w) || !double_arg(args[2], &eps) || !optional_tensor(args[3], &r) || x->dim() < 1) Py_RETURN_NONE;
    Norm c;
    if (!norm_of(*x, r, w, nullptr, x->sizes().slice(x->dim() - 1), eps, &c)) Py_RETURN_NONE;
    if (at::GradMode::is_enabled())
        for (const at::Tensor* t : {x, r, w})
            if (t != nullptr && t->requires_grad()) Py_RETURN_NONE;
    Codes y;
    at::Tensor scales, h;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::cuda::CUDAGuard guard(x->device());
        const at::Tensor none;
        y = empty_codes(*x, x->sizes());
        scales = empty_scales(*x, x->sizes());
        if (r != nullptr) h = empty_on(*x, x->sizes(), x->scalar_type());
        check(api.rmsnorm_forward_8bit(ptr(*x), ptr(r != nullptr ? *r : none), ptr(w != nullptr ? *w : none), ptr(y.values), scales.mutable_data_ptr<float>(), ptr(h),
                                       c.rows, c.d, c.x_stride, c.r_stride, y.stride, c.type, c.weight_type, (float)eps, current_stream(*x)),
              "adder_b200_rmsnorm_forward_8bit");
    }
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(y.values)), THPVariable_Wrap(std::move(scales)), wrap_or_none(std::move(h)));
    END_HANDLE_TH_ERRORS
}

// Both tensors of a pair such as Rows8
bool pair_arg(PyObject* o, const at::Tensor** a, const at::Tensor** b) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
    *a = tensor_arg(PyTuple_GET_ITEM(o, 0));
    *b = tensor_arg(PyTuple_GET_ITEM(o, 1));
    return *a != nullptr && *b != nullptr;
}

// linear_8bit(x or (values, scales), (values, scales), bias or None, dtype or None) -> y, or None
PyObject* py_linear_8bit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *xv = nullptr, *xs = nullptr, *wv, *ws, *bias;
    if ((x == nullptr && !pair_arg(args[0], &xv, &xs)) || !pair_arg(args[1], &wv, &ws) || !optional_tensor(args[2], &bias)) Py_RETURN_NONE;
    at::ScalarType out_type = x != nullptr ? x->scalar_type() : at::kBFloat16;
    if (args[3] != Py_None) {
        if (!THPDtype_Check(args[3])) Py_RETURN_NONE;
        out_type = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
    }
    const int out_code = out_type == at::kFloat ? ADDER_TYPE_F32 : out_type == at::kBFloat16 ? ADDER_TYPE_BF16 : out_type == at::kHalf ? ADDER_TYPE_F16 : -1;
    int64_t outer, w_stride, rows, x_stride;
    if (out_code < 0 || !codes_of(*wv, *ws, &outer, &w_stride) || wv->dim() != 2 || ws->size(0) != (outer + 127) / 128 || needs_node(*wv, *ws)) Py_RETURN_NONE;
    const int64_t inner = wv->size(1);
    const at::Tensor& first = x != nullptr ? *x : *xv;
    if (first.dim() < 1 || first.size(-1) != inner || first.device() != wv->device()) Py_RETURN_NONE;
    const auto lead = first.sizes().slice(0, first.dim() - 1);
    int type = 0;
    if (x != nullptr) {
        type = type_code(*x);
        if (type < 0 || !unwrapped(*x) || x->numel() == 0 || !rows_of(*x, 1, inner, &x_stride) || needs_node(*x, *x)) Py_RETURN_NONE;
        rows = x->numel() / inner;
    } else if (!codes_of(*xv, *xs, &rows, &x_stride) || xs->sizes().slice(0, lead.size()) != lead || needs_node(*xv, *xs)) {
        Py_RETURN_NONE;
    }
    if (bias != nullptr && (!unwrapped(*bias) || !bias->is_contiguous() || bias->device() != wv->device() || bias->scalar_type() != out_type || bias->dim() != 1 ||
                            bias->size(0) != outer || needs_node(*bias, *bias)))
        Py_RETURN_NONE;
    at::Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::cuda::CUDAGuard guard(wv->device());
        const cudaStream_t stream = current_stream(*wv);
        at::Tensor values, scales;
        if (x != nullptr) {
            Codes codes = empty_codes(*x, {rows, inner});
            values = codes.values;
            scales = empty_scales(*x, {rows, inner});
            check(api.quantize_rows(ptr(*x), static_cast<unsigned char*>(ptr(values)), scales.mutable_data_ptr<float>(), rows, inner, x_stride, codes.stride, type, stream),
                  "adder_b200_quantize_rows");
            x_stride = codes.stride;
        } else {
            values = *xv;
            scales = *xs;
        }
        c10::SmallVector<int64_t, 5> sizes(lead.begin(), lead.end());
        sizes.push_back(outer);
        y = empty_on(*wv, sizes, out_type);
        const at::Tensor none;
        check(api.linear_8bit(static_cast<const unsigned char*>(ptr(values)), scales.const_data_ptr<float>(), static_cast<const unsigned char*>(ptr(*wv)),
                              ws->const_data_ptr<float>(), ptr(bias != nullptr ? *bias : none), ptr(y), rows, inner, outer, x_stride, w_stride, out_code, stream),
              "adder_b200_linear_8bit");
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// distillation(logits, teacher, indices, temperature, targets or None, ignore_index) -> (divergence, log_prob or None), or None
PyObject* py_distillation(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6 || !available()) Py_RETURN_NONE;
    const at::Tensor *x = tensor_arg(args[0]), *teacher = tensor_arg(args[1]), *indices = tensor_arg(args[2]), *targets;
    Distill c;
    if (x == nullptr || teacher == nullptr || indices == nullptr || !double_arg(args[3], &c.temperature) || !optional_tensor(args[4], &targets) ||
        !int_arg(args[5], &c.ignore) || !distill_of(*x, *teacher, *indices, targets, &c))
        Py_RETURN_NONE;
    at::Tensor divergence, log_prob;
    {
        pybind11::gil_scoped_release no_gil;
        if (at::GradMode::is_enabled() && x->requires_grad()) {
            auto list = DistillNode::apply(*x, *teacher, *indices, optional(targets), c);
            divergence = list[0];
            if (targets != nullptr) log_prob = list[1];
        } else {
            const at::Tensor none;
            auto r = distill_forward(*x, *teacher, *indices, targets != nullptr ? *targets : none, c, false);
            divergence = r.divergence; log_prob = r.log_prob;
        }
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(divergence)), wrap_or_none(std::move(log_prob)));
    END_HANDLE_TH_ERRORS
}

// verify_drafts(target_probs, draft_probs or None, draft_tokens, uniforms, lengths or None) -> (tokens, accepted), or None
PyObject* py_verify_drafts(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5 || !available()) Py_RETURN_NONE;
    const at::Tensor *p = tensor_arg(args[0]), *q, *tokens = tensor_arg(args[2]), *u = tensor_arg(args[3]), *lengths;
    if (p == nullptr || !optional_tensor(args[1], &q) || tokens == nullptr || u == nullptr || !optional_tensor(args[4], &lengths)) Py_RETURN_NONE;
    const int type = type_code(*p);
    if (type < 0 || !unwrapped(*p) || p->dim() != 3 || p->numel() == 0) Py_RETURN_NONE;
    const int64_t b = p->size(0), places = p->size(1), classes = p->size(2);
    const std::array<int64_t, 3> of_draft{b, places - 1, classes};
    if (q != nullptr && (!unwrapped(*q) || q->device() != p->device() || q->scalar_type() != p->scalar_type() || q->sizes() != at::IntArrayRef(of_draft))) Py_RETURN_NONE;
    for (const at::Tensor* t : {p, q})
        if (t != nullptr && classes > 1 && t->stride(2) != 1) Py_RETURN_NONE;
    if (!whole_long(*tokens, p->device()) || tokens->dim() != 2 || tokens->size(0) != b || tokens->size(1) != places - 1 || !plain(*u) || u->device() != p->device() ||
        u->dim() != 2 || u->size(0) != b || u->size(1) != places)
        Py_RETURN_NONE;
    if (lengths != nullptr && (!whole_long(*lengths, p->device()) || lengths->dim() != 1 || lengths->size(0) != b)) Py_RETURN_NONE;
    at::Tensor out, accepted;
    {
        pybind11::gil_scoped_release no_gil;
        const c10::cuda::CUDAGuard guard(p->device());
        const at::Tensor none;
        out = empty_on(*p, {b, places}, at::kLong);
        accepted = empty_on(*p, {b}, at::kLong);
        check(api.verify_drafts(ptr(*p), ptr(q != nullptr ? *q : none), type, static_cast<const long long*>(ptr(*tokens)), u->const_data_ptr<float>(),
                                lengths != nullptr ? static_cast<const long long*>(ptr(*lengths)) : nullptr, static_cast<long long*>(ptr(out)),
                                static_cast<long long*>(ptr(accepted)), b, places - 1, classes, p->stride(0), p->stride(1), q != nullptr ? q->stride(0) : 0,
                                q != nullptr ? q->stride(1) : 0, current_stream(*p)), "adder_b200_verify_drafts");
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(accepted)));
    END_HANDLE_TH_ERRORS
}

// The addresses that one step writes to: no two may be equal.
class Addresses {
public:
    explicit Addresses(size_t n) {
        size_t size = 64;
        while (size < 2 * n) size *= 2;
        slots_.assign(size, 0);
    }
    bool add(const void* p) { return probe((uintptr_t)p, true); }
    bool has(const void* p) { return !probe((uintptr_t)p, false); }

private:
    bool probe(uintptr_t p, bool insert) {      // false: it was there
        for (size_t i = (p >> 3) * 0x9E3779B97F4A7C15ull >> 32;; ++i) {
            uintptr_t& slot = slots_[i & (slots_.size() - 1)];
            if (slot == p) return false;
            if (slot == 0) {
                if (insert) slot = p;
                return true;
            }
        }
    }
    std::vector<uintptr_t> slots_;
};

// The items of a list or tuple of exact tensors
bool tensor_list(PyObject* o, size_t n, std::vector<const at::Tensor*>* out) {
    if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
    if ((size_t)PySequence_Fast_GET_SIZE(o) != n) return false;
    PyObject** items = PySequence_Fast_ITEMS(o);
    out->resize(n);
    for (size_t i = 0; i < n; ++i) {
        PyObject* t = items[i];
        if (!THPVariable_CheckExact(t)) return false;
        (*out)[i] = &THPVariable_Unpack(t);
    }
    return true;
}

// A number, or a float32 tensor of one element on the device
bool scalar_arg(PyObject* o, const at::Device& dev, double* v, const float** device) {
    *device = nullptr;
    if (double_arg(o, v)) return true;
    const at::Tensor* t = tensor_arg(o);
    if (t == nullptr || !plain(*t) || t->numel() != 1 || t->device() != dev) return false;
    *v = 0.0;
    *device = t->const_data_ptr<float>();
    return true;
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, steps, lr, beta1, beta2, eps, weight_decay, scales or None, scales or None, grad_scale or None)
// -> True, or None where nothing was done
PyObject* py_adamw(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    if (nargs != 13 || !available() || (!PyList_CheckExact(args[0]) && !PyTuple_CheckExact(args[0]))) Py_RETURN_NONE;
    const size_t n = PySequence_Fast_GET_SIZE(args[0]);
    // kept from call to call for their memory alone
    static thread_local std::vector<const at::Tensor*> p, g, m, v, ms, vs, steps;
    static thread_local std::vector<adder_b200_adamw_tensor> tensors;
    const bool eight = args[10] != Py_None;
    if (n == 0 || !tensor_list(args[0], n, &p) || !tensor_list(args[1], n, &g) || !tensor_list(args[2], n, &m) || !tensor_list(args[3], n, &v)) Py_RETURN_NONE;
    if (eight != (args[11] != Py_None) || (eight && (!tensor_list(args[10], n, &ms) || !tensor_list(args[11], n, &vs)))) Py_RETURN_NONE;
    const at::Tensor* all_steps = tensor_arg(args[4]);
    if (all_steps == nullptr && !tensor_list(args[4], n, &steps)) Py_RETURN_NONE;
    const at::Device dev = p[0]->device();
    const int type = type_code(*p[0]);
    const at::ScalarType scalar = p[0]->scalar_type(), state = eight ? at::kByte : at::kFloat;
    double lr, b1, b2, eps, wd;
    const float *lr_device, *scale_device = nullptr;
    if (type < 0 || !dev.is_cuda() || !scalar_arg(args[5], dev, &lr, &lr_device) || !double_arg(args[6], &b1) || !double_arg(args[7], &b2) ||
        !double_arg(args[8], &eps) || !double_arg(args[9], &wd))
        Py_RETURN_NONE;
    if (args[12] != Py_None) {
        double ignored;
        if (tensor_arg(args[12]) == nullptr || !scalar_arg(args[12], dev, &ignored, &scale_device)) Py_RETURN_NONE;
    }
    // Tensors of one kind have one set of dispatch keys, so what the first parameter is is asked once; and without a level of forward-mode
    // differentiation no tensor has a tangent (asking each view for its own took as long as all the rest).
    if (!unwrapped(*p[0])) Py_RETURN_NONE;
    const c10::DispatchKeySet keys = p[0]->key_set();
    const bool no_tangents = torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr;
    const auto ordinary = [&](const at::Tensor& t, at::ScalarType type) {
        if (!t.defined()) return false;
        const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
        return impl->key_set() == keys && (no_tangents || !t._fw_grad(0).defined()) && impl->dtype() == c10::scalarTypeToTypeMeta(type) &&
               impl->device() == dev && impl->is_contiguous();
    };
    const auto fits = [&](const at::Tensor& t, at::ScalarType type, const at::Tensor& like) { return ordinary(t, type) && t.sizes() == like.sizes(); };
    const auto counts = [&](const at::Tensor& t, at::ScalarType type, int64_t count) { return ordinary(t, type) && t.numel() == count; };
    if (all_steps != nullptr && (!counts(*all_steps, at::kInt, 2 * (int64_t)n) || all_steps->dim() != 2 || all_steps->size(0) != (int64_t)n)) Py_RETURN_NONE;
    Addresses written(6 * n);
    tensors.resize(n);
    for (size_t i = 0; i < n; ++i) {
        const at::Tensor& q = *p[i];
        if (!fits(q, scalar, q) || !fits(*g[i], scalar, q) || !fits(*m[i], state, q) || !fits(*v[i], state, q)) Py_RETURN_NONE;
        if (all_steps == nullptr && !counts(*steps[i], at::kInt, 2)) Py_RETURN_NONE;
        const int64_t count = (q.numel() + 255) / 256;
        if (eight && (!counts(*ms[i], at::kFloat, count) || !counts(*vs[i], at::kFloat, count))) Py_RETURN_NONE;
        adder_b200_adamw_tensor& t = tensors[i];
        t.n = q.numel();
        if (t.n == 0) continue;
        t.param = q.data_ptr(); t.grad = g[i]->data_ptr(); t.exp_avg = m[i]->data_ptr(); t.exp_avg_sq = v[i]->data_ptr();
        t.exp_avg_scale = eight ? ms[i]->data_ptr<float>() : nullptr;
        t.exp_avg_sq_scale = eight ? vs[i]->data_ptr<float>() : nullptr;
        t.step = all_steps != nullptr ? all_steps->data_ptr<int>() + 2 * i : steps[i]->data_ptr<int>();
        if (!written.add(t.param) || !written.add(t.exp_avg) || !written.add(t.exp_avg_sq) || !written.add(t.step) ||
            (eight && (!written.add(t.exp_avg_scale) || !written.add(t.exp_avg_sq_scale))))
            Py_RETURN_NONE;
    }
    for (const auto& t : tensors)
        if (t.n > 0 && written.has(t.grad)) Py_RETURN_NONE;
    // The lock stays: the lists own the tensors, and another thread may change a list.
    const c10::cuda::CUDAGuard guard(dev);
    check(api.adamw_step(tensors.data(), (int)n, type, eight ? 8 : 32, lr, lr_device, b1, b2, eps, wd, scale_device,
                         c10::cuda::getCurrentCUDAStream(dev.index()).stream()), "adder_b200_adamw_step");
    for (const auto* list : {&p, &m, &v})
        for (const at::Tensor* t : *list)
            if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// bind({name: address}, adder module dict, adder_cuda module dict) switches the entry points on, bind(None, ...) off
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 3 && PyDict_Check(args[1]) && PyDict_Check(args[2]), "bind(addresses, dict, dict)");
    enabled.store(false, std::memory_order_release);
    const bool on = args[0] != Py_None;
    if (on && api.forward == nullptr) {
        Api a;
        auto get = [&](const char* name, auto* fn) {
            PyObject* v = PyDict_GetItemString(args[0], name);
            TORCH_CHECK(v != nullptr && PyLong_Check(v), "no address for ", name);
            *fn = reinterpret_cast<std::remove_pointer_t<decltype(fn)>>(PyLong_AsVoidPtr(v));
        };
        get("adder_b200_status_string", &a.status_string);
        get("adder_b200_forward", &a.forward);
        get("adder_b200_forward_stat_slices", &a.forward_stat_slices);
        get("adder_b200_forward_with_stats", &a.forward_with_stats);
        get("adder_b200_forward_affine", &a.forward_affine);
        get("adder_b200_affine_forward", &a.affine_forward);
        get("adder_b200_backward_input_workspace_bytes", &a.backward_input_workspace_bytes);
        get("adder_b200_backward_input_with_workspace", &a.backward_input_with_workspace);
        get("adder_b200_backward_weight_workspace_bytes", &a.backward_weight_workspace_bytes);
        get("adder_b200_backward_weight", &a.backward_weight);
        get("adder_b200_conv_forward", &a.conv_forward);
        get("adder_b200_conv_backward_input_workspace_bytes", &a.conv_backward_input_workspace_bytes);
        get("adder_b200_conv_backward_input_with_workspace", &a.conv_backward_input_with_workspace);
        get("adder_b200_conv_backward_weight_workspace_bytes", &a.conv_backward_weight_workspace_bytes);
        get("adder_b200_conv_backward_weight", &a.conv_backward_weight);
        get("adder_b200_layernorm_forward", &a.layernorm_forward);
        get("adder_b200_layernorm_backward_workspace_bytes", &a.layernorm_backward_workspace_bytes);
        get("adder_b200_layernorm_backward", &a.layernorm_backward);
        get("adder_b200_log_probs_forward", &a.log_probs_forward);
        get("adder_b200_log_probs_backward", &a.log_probs_backward);
        get("adder_b200_rmsnorm_forward", &a.rmsnorm_forward);
        get("adder_b200_rmsnorm_forward_8bit", &a.rmsnorm_forward_8bit);
        get("adder_b200_rmsnorm_backward_workspace_bytes", &a.rmsnorm_backward_workspace_bytes);
        get("adder_b200_rmsnorm_backward", &a.rmsnorm_backward);
        get("adder_b200_quantize_rows", &a.quantize_rows);
        get("adder_b200_linear_8bit", &a.linear_8bit);
        get("adder_b200_distillation_forward", &a.distillation_forward);
        get("adder_b200_distillation_backward", &a.distillation_backward);
        get("adder_b200_verify_drafts", &a.verify_drafts);
        get("adder_b200_adamw_step", &a.adamw_step);
        api = a;
    }
    Py_INCREF(args[1]); Py_INCREF(args[2]);
    Py_XDECREF(g_adder_dict); Py_XDECREF(g_cuda_dict);
    g_adder_dict = args[1]; g_cuda_dict = args[2];
    enabled.store(on, std::memory_order_release);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define ADDER_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ADDER_METHOD("bind", py_bind), ADDER_METHOD("layer", py_layer), ADDER_METHOD("conv", py_conv), ADDER_METHOD("layer_with_stats", py_layer_with_stats),
                         ADDER_METHOD("layer_affine", py_layer_affine), ADDER_METHOD("affine", py_affine), ADDER_METHOD("column", py_column),
                         ADDER_METHOD("layer_norm", py_layer_norm), ADDER_METHOD("log_probs", py_log_probs), ADDER_METHOD("adamw", py_adamw),
                         ADDER_METHOD("rms_norm", py_rms_norm), ADDER_METHOD("rms_norm_8bit", py_rms_norm_8bit), ADDER_METHOD("linear_8bit", py_linear_8bit),
                         ADDER_METHOD("distillation", py_distillation), ADDER_METHOD("verify_drafts", py_verify_drafts),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_adder_host", nullptr, -1, methods};

}  // namespace

#ifndef ADDER_HOST_MARK
#define ADDER_HOST_MARK ""
#endif

// The mark says which torch this file was linked with; build.py looks for it before it is loaded.
PyMODINIT_FUNC PyInit__adder_host() {
    PyObject* m = PyModule_Create(&module_def);
    if (m != nullptr) PyModule_AddStringConstant(m, "built_for", ADDER_HOST_MARK);
    return m;
}
