// ozk_torch.cpp -- the operators around linear layers as PyTorch calls: a Python
// module (_ozk_torch) that allocates results and workspaces, keeps what a backward
// pass needs and calls the C ABI (include/ozaki_amd.h).
//
// In C++ because these calls are short: an autograd node in Python costs its two
// passes 40 us of host time more than one here (a training step through 1999 x 520 x 1000
// 109 against 69), and a list of a hundred tensors is looked at in a few us.  Arguments
// are checked by the Python functions; what the calls here do not take as it is they
// refuse by returning None, before anything has happened, and the Python functions find
// out why.
//
// A tensor that stands for its memory's negative (the imaginary part of a conjugate) is
// written out first.
//
// A stream comes as its handle.  A backward pass runs on its gradient's device and the
// current stream there, which its memory comes from, too: autograd has made it that of
// the forward pass, a caller of the node itself may have another.
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <numeric>
#include <unordered_set>

#include "../../include/ozaki_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxStride = (int64_t)1 << 22;   // the kernels' limit on the distance of two rows

void check(const char *name, int status) {
    if (status != OZK_OK)
        throw std::runtime_error(std::string(name) + " failed: " + ozk_strerror(status) + " (status " +
                                 std::to_string(status) + ")");
}
int code(at::ScalarType t) {
    return t == at::kFloat      ? OZK_F32
           : t == at::kHalf     ? OZK_F16
           : t == at::kBFloat16 ? OZK_BF16
                                : -1;
}
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor written_out(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor workspace(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// The results of a backward pass that is itself recorded: a second derivative would
// be lost without a word, so taking one is an error.
void refuse_second(const char *name, variable_list &grads) {
    if (!at::GradMode::is_enabled()) return;
    variable_list some;
    for (const Tensor &g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_());
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate ") + name + " twice: its backward pass has no derivative",
        (int64_t)some.size());
    some = (*error)(std::move(some));
    size_t i = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = some[i++];
}

int64_t current_stream(const Tensor &t) {
    return (int64_t)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A backward pass that is captured on `stream` and reaches a node of the default stream
// further on (behind a reshape of x, say), as a leaf has while an earlier graph of it is
// alive: the engine would make the default stream wait for the capture, which ends the
// process.
void refuse_default_stream(const char *name, int64_t stream) {
    const auto node = torch::autograd::get_current_node();
    if (!stream || !node) return;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone)
        return;
    std::unordered_set<torch::autograd::Node *> seen;
    std::vector<torch::autograd::Node *> todo = {node.get()};
    while (!todo.empty()) {
        torch::autograd::Node *at = todo.back();
        todo.pop_back();
        for (size_t i = 0; i < at->next_edges().size(); ++i) {
            torch::autograd::Node *next = at->next_edge(i).function.get();
            if (!next || !at->task_should_compute_output(i) || !seen.insert(next).second) continue;
            const auto s = next->stream();
            if (s && s->id() == 0)
                throw std::runtime_error(std::string(name) + ": a captured backward pass reaches a tensor that has a "
                                         "graph on the default stream; delete that graph (its results) before the "
                                         "capture");
            todo.push_back(next);
        }
    }
}

// The engine hands a node gradients of its results' shape, type and device; who calls it
// by hand may not
void gradient_as(const Tensor &t, at::IntArrayRef sizes, at::ScalarType type, int64_t device) {
    if (!t.is_cuda() || t.device().index() != device || t.layout() != at::kStrided || t.sizes() != sizes ||
        t.scalar_type() != type)
        throw std::runtime_error("a gradient has another shape, type or device than its result");
}
// A hook may give back anything for a saved tensor: what the kernels take on trust
void saved_as(const Tensor &t, at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
    if (t.sizes() != sizes || t.scalar_type() != type || t.device() != like.device() || t.layout() != at::kStrided)
        throw std::runtime_error("a saved tensor came back with another shape, type or device");
}

variable_list saved_of(AutogradContext *ctx) {
    variable_list saved = ctx->get_saved_variables();
    for (Tensor &t : saved) t = written_out(t);
    return saved;
}

// t [rows, columns] with its columns contiguous, and its rows' distance within the
// kernels' limit (strides of dims of size 1 mean nothing)
Tensor rows(const Tensor &t, int64_t &stride) {
    const int64_t n = t.size(0), c = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
    stride = n <= 1 ? 0 : s0;
    if ((s1 == 1 || c <= 1) && stride < kMaxStride) return t;
    stride = n <= 1 ? 0 : c;
    return t.contiguous();
}
// W [N, K] with K or N contiguous, and its strides, the contiguous one 1
Tensor weight(const Tensor &W, int64_t (&s)[2]) {
    const int64_t N = W.size(0), K = W.size(1), s_n = N > 1 ? W.stride(0) : 0, s_k = W.stride(1);
    if ((s_k == 1 || K <= 1) && s_n < kMaxStride) {
        s[0] = s_n;
        s[1] = 1;
        return W;
    }
    if ((s_n == 1 || N <= 1) && s_k < kMaxStride) {
        s[0] = 1;
        s[1] = s_k;
        return W;
    }
    s[0] = N > 1 ? K : 0;
    s[1] = 1;
    return W.contiguous();
}

// ---- the dense product ----

Tensor linear_forward(const Tensor &x_, const Tensor &W_, const std::optional<Tensor> &bias_,
                      const std::optional<Tensor> &residual_, int64_t act, int64_t stream, Tensor *z) {
    const int64_t M = x_.size(0), K = x_.size(1), N = W_.size(0);
    int64_t sx, sr = 0, sw[2];
    const Tensor x = rows(x_, sx), W = weight(W_, sw);
    const Tensor bias = bias_ ? bias_->contiguous() : Tensor();
    const Tensor residual = residual_ ? rows(*residual_, sr) : Tensor();
    Tensor y = at::empty({M, N}, x.options());
    if (z) *z = at::empty({M, N}, x.options());
    size_t bytes = 0;
    check("ozk_linear_workspace_bytes",
          ozk_linear_workspace_bytes(ptr(x), sx, ptr(W), sw, M, N, K, &bytes));
    const Tensor ws = workspace(bytes, x);
    check("ozk_linear", ozk_linear(ptr(x), sx, ptr(W), sw, ptr(bias), ptr(residual), sr, (int)act, M, N, K,
                                   code(x.scalar_type()), ptr(y), N, z ? ptr(*z) : nullptr, ptr(ws), bytes,
                                   (void *)stream));
    return y;
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &W,
                          const std::optional<Tensor> &bias, const std::optional<Tensor> &residual,
                          int64_t act, int64_t stream) {
        const bool need_x = x.requires_grad(), need_W = W.requires_grad();
        const bool need_z = act != OZK_ACT_NONE && (need_x || need_W || (bias && bias->requires_grad()));
        Tensor z;
        const Tensor y = linear_forward(x, W, bias, residual, act, stream, need_z ? &z : nullptr);
        ctx->save_for_backward({need_W ? x : Tensor(), need_x ? W : Tensor(), z});
        ctx->saved_data["a"] =
            std::vector<int64_t>{act, bias.has_value(), residual.has_value(), x.size(0), W.size(0), x.size(1),
                                 (int64_t)x.scalar_type(), x.device().index()};
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto a = ctx->saved_data["a"].toIntVector();
        const int64_t act = a[0], M = a[3], N = a[4], K = a[5];
        const bool has_b = a[1], has_r = a[2];
        const variable_list saved = saved_of(ctx);
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const Tensor g = written_out(grads[0]);
        gradient_as(g, {M, N}, (at::ScalarType)a[6], a[7]);
        const c10::OptionalDeviceGuard device(g.device());
        const int64_t stream = current_stream(g);
        refuse_default_stream("fused_linear", stream);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const bool need_x = ctx->needs_input_grad(0), need_W = ctx->needs_input_grad(1);
            const bool need_b = has_b && ctx->needs_input_grad(2);
            if (need_W) saved_as(saved[0], {M, K}, g.scalar_type(), g);
            if (need_x) saved_as(saved[1], {N, K}, g.scalar_type(), g);
            if (saved[2].defined()) saved_as(saved[2], {M, N}, g.scalar_type(), g);
            int64_t sy, sx = 0, sw[2] = {0, 1};
            const Tensor dy = rows(g, sy), z = saved[2].defined() ? saved[2].contiguous() : Tensor();
            const Tensor x = need_W ? rows(saved[0], sx) : Tensor(), W = need_x ? weight(saved[1], sw) : Tensor();
            if (need_x) out[0] = at::empty({M, K}, dy.options());
            if (need_W) out[1] = at::empty({N, K}, dy.options());
            if (need_b) out[2] = at::empty({N}, dy.options());
            if (need_x || need_W || need_b) {
                const int want = (need_x ? 1 : 0) | (need_W ? 2 : 0) | (need_b ? 4 : 0);
                size_t bytes = 0;
                check("ozk_linear_backward_workspace_bytes",
                      ozk_linear_backward_workspace_bytes(ptr(dy), sy, ptr(x), sx, ptr(W), sw, (int)act, M,
                                                          N, K, want, &bytes));
                const Tensor ws = workspace(bytes, dy);
                check("ozk_linear_backward",
                      ozk_linear_backward(ptr(dy), sy, ptr(z), ptr(x), sx, ptr(W), sw, (int)act, M, N, K,
                                          code(dy.scalar_type()), ptr(out[0]), K, ptr(out[1]), K,
                                          ptr(out[2]), ptr(ws), bytes, (void *)stream));
            }
        }
        if (has_r && ctx->needs_input_grad(has_b ? 3 : 2)) out[3] = g;
        variable_list mine = {out[0], out[1], out[2]};
        refuse_second("fused_linear", mine);
        for (int i = 0; i < 3; ++i) out[i] = mine[i];
        return out;
    }
};

bool linear_ok(const Tensor &x, const Tensor &W, const std::optional<Tensor> &bias,
               const std::optional<Tensor> &residual) {
    if (x.dim() != 2 || W.dim() != 2 || !x.is_cuda() || x.size(1) != W.size(1)) return false;
    const auto t = x.scalar_type();
    if ((t != at::kHalf && t != at::kBFloat16) || W.scalar_type() != t || W.device() != x.device())
        return false;
    if (bias && (bias->dim() != 1 || bias->size(0) != W.size(0) || bias->scalar_type() != t ||
                 bias->device() != x.device()))
        return false;
    return !residual || (residual->dim() == 2 && residual->size(0) == x.size(0) &&
                         residual->size(1) == W.size(0) && residual->scalar_type() == t &&
                         residual->device() == x.device());
}
std::optional<Tensor> linear(const Tensor &x, const Tensor &W, const std::optional<Tensor> &bias,
                             const std::optional<Tensor> &residual, int64_t act, int64_t stream) {
    if (!linear_ok(x, W, bias, residual)) return std::nullopt;
    if (x.is_neg() || W.is_neg() || (bias && bias->is_neg()) || (residual && residual->is_neg())) {
        auto written = [](const std::optional<Tensor> &t) { return t ? t->resolve_neg() : t; };
        return linear(x.resolve_neg(), W.resolve_neg(), written(bias), written(residual), act, stream);
    }
    const bool grad = at::GradMode::is_enabled();
    const bool products = grad && (x.requires_grad() || W.requires_grad() || (bias && bias->requires_grad()));
    // what the backward pass would refuse: its dz has rows of N, with an activation padded
    const int64_t N = W.size(0);
    if (products && x.size(0) > 1 && (act == OZK_ACT_NONE ? N : (N + 7) / 8 * 8) >= kMaxStride)
        throw std::runtime_error("fused_linear: results of more than one row have gradients for fewer than 2^22 "
                                 "columns, got " + std::to_string(N));
    if (products || (grad && residual && residual->requires_grad()))
        return Linear::apply(x, W, bias, residual, act, stream);
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_forward(x, W, bias, residual, act, stream, nullptr);
}

// ---- the router ----

// experts, weights, order, place, offsets, counts, loss
variable_list route_forward(const Tensor &logits_, const std::optional<Tensor> &mask_, int64_t k,
                            bool normalize, int64_t stream) {
    const int64_t T = logits_.size(0), E = logits_.size(1), n = T * k;
    const Tensor signs = written_out(logits_);
    const Tensor logits = signs.stride(1) == 1 || E == 1 ? signs : signs.contiguous();
    const Tensor mask = mask_ ? mask_->contiguous() : Tensor();
    const auto ints = logits.options().dtype(at::kInt), floats = logits.options().dtype(at::kFloat);
    const Tensor all = at::empty({3 * n + 2 * E + 1}, ints);
    const Tensor experts = all.as_strided({T, k}, {k, 1}, 0), order = all.as_strided({n}, {1}, n);
    const Tensor place = all.as_strided({T, k}, {k, 1}, 2 * n);
    const Tensor offsets = all.as_strided({E + 1}, {1}, 3 * n);
    const Tensor counts = all.as_strided({E}, {1}, 3 * n + E + 1);
    const Tensor weights = at::empty({T, k}, floats), loss = at::empty({}, floats);
    size_t bytes = 0;
    check("ozk_route_workspace_bytes", ozk_route_workspace_bytes(T, E, k, &bytes));
    const Tensor ws = workspace(bytes, logits);
    check("ozk_route",
          ozk_route(ptr(logits), code(logits.scalar_type()), logits.stride(0), ptr(mask), T, E, k, normalize,
                    (int32_t *)ptr(experts), (float *)ptr(weights), (int32_t *)ptr(order),
                    (int32_t *)ptr(place), (int32_t *)ptr(offsets), (int32_t *)ptr(counts),
                    (float *)ptr(loss), ptr(ws), bytes, (void *)stream));
    return {experts, weights, order, place, offsets, counts, loss};
}

struct Route : torch::autograd::Function<Route> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const std::optional<Tensor> &mask,
                                 int64_t k, bool normalize, int64_t stream) {
        variable_list r;
        {
            // (views of one tensor that do not count each other's changes)
            at::AutoDispatchBelowADInplaceOrView below;
            r = route_forward(logits, mask, k, normalize, stream);
        }
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({r[0], r[2], r[3], r[4], r[5]});
        ctx->save_for_backward({logits, mask ? *mask : Tensor(), r[0], r[1], r[5]});
        ctx->saved_data["a"] = std::vector<int64_t>{
            normalize, mask.has_value(), logits.size(0), logits.size(1), k, (int64_t)logits.scalar_type(),
            logits.device().index()};
        return r;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(5);
        const Tensor gw = written_out(grads[1]), gl = written_out(grads[6]);
        if (!gw.defined() && !gl.defined()) return out;
        const auto a = ctx->saved_data["a"].toIntVector();
        const Tensor &like = gw.defined() ? gw : gl;
        const int64_t T = a[2], E = a[3], k = a[4];
        if (gw.defined()) gradient_as(gw, {T, k}, at::kFloat, a[6]);
        if (gl.defined()) gradient_as(gl, {}, at::kFloat, a[6]);
        const c10::OptionalDeviceGuard device(like.device());
        const int64_t stream = current_stream(like);
        refuse_default_stream("route_tokens", stream);
        const variable_list saved = saved_of(ctx);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            saved_as(saved[0], {T, E}, (at::ScalarType)a[5], like);
            if (a[1]) saved_as(saved[1], {T}, at::kBool, like);
            saved_as(saved[2], {T, k}, at::kInt, like);
            saved_as(saved[3], {T, k}, at::kFloat, like);
            saved_as(saved[4], {E}, at::kInt, like);
            const Tensor logits = saved[0].stride(1) == 1 || E == 1 ? saved[0] : saved[0].contiguous();
            const Tensor mask = a[1] ? saved[1].contiguous() : Tensor(), experts = saved[2].contiguous();
            const Tensor weights = saved[3].contiguous(), counts = saved[4].contiguous();
            const Tensor dw = gw.defined() ? gw.contiguous() : Tensor();
            out[0] = at::empty({T, E}, logits.options());
            check("ozk_route_backward",
                  ozk_route_backward(ptr(logits), code(logits.scalar_type()), logits.stride(0), ptr(mask), T, E,
                                     k, (int)a[0], (int32_t *)ptr(experts), (float *)ptr(weights),
                                     (int32_t *)ptr(counts), (float *)ptr(dw), (float *)ptr(gl), ptr(out[0]),
                                     (void *)stream));
        }
        variable_list mine = {out[0]};
        refuse_second("route_tokens", mine);
        out[0] = mine[0];
        return out;
    }
};

std::optional<variable_list> route(const Tensor &logits, const std::optional<Tensor> &mask, int64_t k,
                                   bool normalize, int64_t stream) {
    if (logits.dim() != 2 || !logits.is_cuda() || code(logits.scalar_type()) < 0) return std::nullopt;
    const int64_t E = logits.size(1);
    if (E < 1 || E > OZK_MAX_EXPERTS || k < 1 || k > E) return std::nullopt;
    if (mask && (mask->dim() != 1 || mask->size(0) != logits.size(0) ||
                 mask->scalar_type() != at::kBool || mask->device() != logits.device()))
        return std::nullopt;
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return Route::apply(logits, mask, k, normalize, stream);
    at::AutoDispatchBelowADInplaceOrView below;
    return route_forward(logits, mask, k, normalize, stream);
}

// ---- gradient norms ----

struct Table {
    std::vector<const void *> ins;
    std::vector<void *> outs;
    std::vector<int64_t> counts;
    std::vector<int> codes;
};
// false: not all on one GPU, contiguous, of a type with a kernel, without a gradient
bool table_of(const std::vector<Tensor> &in, const std::vector<Tensor> *out, Table &t) {
    const size_t n = in.size();
    if (!n || !in[0].is_cuda() || (out && out->size() != n)) return false;
    const bool grad = at::GradMode::is_enabled();
    t.ins.resize(n);
    t.outs.resize(out ? n : 0);
    t.counts.resize(n);
    t.codes.resize(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor &g = in[i];
        t.codes[i] = code(g.scalar_type());
        if (t.codes[i] < 0 || g.device() != in[0].device() || !g.is_contiguous() ||
            g.is_neg() || (grad && g.requires_grad()))
            return false;
        t.ins[i] = g.data_ptr();
        t.counts[i] = g.numel();
        if (!out) continue;
        const Tensor &o = (*out)[i];
        if (o.scalar_type() != g.scalar_type() || o.device() != g.device() || !o.is_contiguous() ||
            o.is_neg() || o.sizes() != g.sizes() || (grad && o.requires_grad()))
            return false;
        t.outs[i] = o.data_ptr();
    }
    return true;
}
Tensor norm_workspace(int64_t n, const Tensor &like, size_t &bytes) {
    check("ozk_gradient_norm_workspace_bytes", ozk_gradient_norm_workspace_bytes(n, &bytes));
    return workspace(bytes, like);
}
std::optional<Tensor> gradient_norm(const std::vector<Tensor> &grads, int64_t stream) {
    Table t;
    if (!table_of(grads, nullptr, t)) return std::nullopt;
    const int64_t n = (int64_t)grads.size();
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
    size_t bytes;
    const Tensor ws = norm_workspace(n, norm, bytes);
    check("ozk_gradient_norm", ozk_gradient_norm(t.ins.data(), t.counts.data(), t.codes.data(), n,
                                                 norm.data_ptr<float>(), ptr(ws), bytes, (void *)stream));
    return norm;
}
// nothing also where tensors share memory, which the Python function then says
std::optional<Tensor> clip_gradients(const std::vector<Tensor> &grads, const std::vector<Tensor> &outs,
                                     double max_norm, int64_t stream) {
    Table t;
    if (!(max_norm >= 0) || !table_of(grads, &outs, t)) return std::nullopt;
    const int64_t n = (int64_t)grads.size();
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
    size_t bytes;
    const Tensor ws = norm_workspace(n, norm, bytes);
    const int st = ozk_clip_gradients(t.ins.data(), t.outs.data(), t.counts.data(), t.codes.data(), n,
                                      max_norm, norm.data_ptr<float>(), ptr(ws), bytes, (void *)stream);
    if (st == OZK_ERR_SHAPE) return std::nullopt;
    check("ozk_clip_gradients", st);
    // written behind autograd's back
    for (const Tensor &o : outs)
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return norm;
}

// ---- tensors with gaps that lie in the same memory ----

// Whether sum of step k over the terms, each k within its lo .. hi, can be from `lo` to
// `hi` (with `moved`: any; else: with some k that is not 0).  Largest steps first, each k
// as far as the rest can make up for; what a common divisor leaves out is left out.
// Past `budget` steps the answer is yes.
struct Term {
    int64_t step, lo, hi;
};
bool reaches(const Term *t, size_t n, int64_t lo, int64_t hi, bool moved, int64_t &budget) {
    if (!n) return moved && lo <= 0 && hi >= 0;
    if (--budget < 0) return true;
    int64_t least = 0, most = 0, common = 0;   // of the rest; of all
    for (size_t i = 0; i < n; ++i) {
        common = std::gcd(common, t[i].step);
        if (!i) continue;
        least += t[i].step * t[i].lo;
        most += t[i].step * t[i].hi;
    }
    auto floor_of = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    if (floor_of(hi, common) * common < lo) return false;
    const int64_t step = t->step, first = std::max(t->lo, -floor_of(most - lo, step));
    const int64_t last = std::min(t->hi, floor_of(hi - least, step));
    for (int64_t k = first; k <= last; ++k)
        if (reaches(t + 1, n - 1, lo - step * k, hi - step * k, moved || k, budget)) return true;
    return false;
}
constexpr int64_t kReachBudget = 1 << 16;

struct Span {
    int64_t lo, hi, item;      // bytes
    std::vector<Term> dims;    // one element to the next, in bytes
    size_t of;                 // its place in the list
    bool out;
};
Span span_of(const Tensor &t, size_t of, bool out) {
    Span s = {(int64_t)(uintptr_t)t.data_ptr(), 0, (int64_t)t.element_size(), {}, of, out};
    s.hi = s.lo + s.item;
    for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1) {
            s.dims.push_back({t.stride(d) * s.item, 0, t.size(d) - 1});
            s.hi += s.dims.back().step * s.dims.back().hi;
        }
    return s;
}
// whether two indices are one element, or elements that overlap
bool meets_itself(const Span &s) {
    std::vector<Term> t;
    for (const Term &d : s.dims) {
        if (!d.step) return true;
        t.push_back({d.step, -d.hi, d.hi});
    }
    std::sort(t.begin(), t.end(), [](const Term &a, const Term &b) { return a.step > b.step; });
    int64_t budget = kReachBudget;
    return reaches(t.data(), t.size(), 1 - s.item, s.item - 1, false, budget);
}
bool meet(const Span &a, const Span &b) {
    std::vector<Term> t;
    for (const Term &d : a.dims)
        if (d.step) t.push_back(d);
    for (const Term &d : b.dims)
        if (d.step) t.push_back({d.step, -d.hi, 0});
    std::sort(t.begin(), t.end(), [](const Term &x, const Term &y) { return x.step > y.step; });
    size_t n = 0;   // those of one step as one
    for (size_t i = 0; i < t.size(); ++i)
        if (n && t[n - 1].step == t[i].step) {
            t[n - 1].lo += t[i].lo;
            t[n - 1].hi += t[i].hi;
        } else {
            t[n++] = t[i];
        }
    const int64_t d = a.lo - b.lo;
    int64_t budget = kReachBudget;
    return reaches(t.data(), n, 1 - a.item - d, b.item - 1 - d, true, budget);
}
// Whether an element of outs is in one of the other tensors, of ins or outs, or there
// twice (or cannot be shown not to be).
bool share_memory(const std::vector<Tensor> &ins, const std::vector<Tensor> &outs) {
    std::vector<Span> s;
    for (size_t i = 0; i < outs.size(); ++i) {
        if (!outs[i].numel()) continue;
        s.push_back(span_of(outs[i], i, true));
        if (meets_itself(s.back())) return true;
        if (!ins[i].is_same(outs[i])) s.push_back(span_of(ins[i], i, false));
    }
    std::sort(s.begin(), s.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    for (size_t i = 0; i < s.size(); ++i)
        for (size_t j = i + 1; j < s.size() && s[j].lo < s[i].hi; ++j)
            if ((s[i].out || s[j].out) && s[i].of != s[j].of && meet(s[i], s[j])) return true;
    return false;
}

}  // namespace

PYBIND11_MODULE(_ozk_torch, m) {
    m.def("linear", &linear);
    m.def("route", &route);
    m.def("gradient_norm", &gradient_norm);
    m.def("clip_gradients", &clip_gradients);
    m.def("share_memory", &share_memory);
}
