// Host side of the calls whose cost is the host's: the autograd node of the gated residual norm and the address lists of the optimizer.
//
// A training call on a few thousand rows is 30 us of GPU work; as a Python autograd.Function it is 160 us of host work, half of it in the
// backward, which autograd runs on another thread with the interpreter's lock in between.  Here the node is C++: checks, allocations and
// launches without the interpreter.  The kernels are those of the C ABI; their addresses are handed over by init(), from the library that
// the Python side has loaded, so there is one library whatever its path.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>

#include <string>
#include <vector>

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

typedef int (*fwd_fn)(int, int, const void*, int64_t, const void*, int64_t, const void*, int64_t, int, int, const float*, const float*, float, int, const float*,
                      const float*, int, const float*, const float*, double, void*, void*, float*, int64_t, int64_t, int, void*);
typedef int64_t (*ws_fn)(int64_t, int64_t, int, int, int, int, int);
typedef int (*bwd_fn)(int, int, const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, int64_t, const void*, int64_t, int, int,
                      const float*, const float*, float, int, const float*, const float*, int, const float*, const float*, void*, void*, void*, float*, int64_t,
                      int64_t, int, float*, int64_t, void*);
typedef int (*add_fn)(int, const float* const*, const int64_t*, const int64_t*, float* const*, const int64_t*, void*);
typedef const char* (*err_fn)();
fwd_fn resnorm_fwd = nullptr;
ws_fn resnorm_ws = nullptr;
bwd_fn resnorm_bwd = nullptr;
add_fn multi_add = nullptr;
err_fn last_error = nullptr;

void check(int rc) { TORCH_CHECK(rc == 0, "semseg_hip error ", rc, ": ", last_error()); }

template <typename E> [[noreturn]] void fail(const std::string& what) { throw E("gated_residual_norm: " + what); }
std::string str(c10::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + ")";
}

// sinks: the vectors' slots in a flat gradient buffer (engine.FlatParams), undefined where there is none
struct Cfg { int64_t rows, n, C; int mode, post, pre, act; double alpha, eps; std::vector<Tensor> sinks; };
int code(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
const float* f32(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
const void* raw(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

// [..., C] with unit inner stride and one stride between rows that the kernels' 32-bit lane offsets reach; a view or a copy only where the
// layout asks for one
Tensor rows_of(const Tensor& t, int64_t C, int64_t& ld) {
    ld = 0;
    if (!t.defined()) return t;
    ld = C;
    if (t.is_contiguous()) return t;
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, C});
    if (r.stride(1) != 1 || r.stride(0) >= (1 << 23)) return r.contiguous();
    ld = r.stride(0);
    return r;
}

struct Forward { Tensor h, y, stats; };
Forward launch_forward(const Tensor& x, const Tensor& b, const Tensor& gate, const Tensor& keep, const variable_list& v, const Cfg& c, bool want_stats) {
    c10::DeviceGuard guard(x.device());
    int64_t ldx, ldb, ldg;
    const Tensor xs = rows_of(x, c.C, ldx), bs = rows_of(b, c.C, ldb), gs = rows_of(gate, c.C, ldg);
    Forward r;
    r.h = at::empty(x.sizes(), x.options());
    if (c.pre) r.y = at::empty(x.sizes(), b.options());
    if (want_stats) r.stats = at::empty({c.rows, 4}, x.options().dtype(at::kFloat));
    check(resnorm_fwd(code(x), code(b), raw(xs), ldx, raw(bs), ldb, raw(gs), ldg, c.mode, c.act, f32(v[4]), f32(keep), (float)c.alpha, c.post, f32(v[2]), f32(v[3]),
                      c.pre, f32(v[0]), f32(v[1]), c.eps, r.h.mutable_data_ptr(), c.pre ? r.y.mutable_data_ptr() : nullptr,
                      want_stats ? r.stats.mutable_data_ptr<float>() : nullptr, c.rows, c.n, (int)c.C, stream_of(x)));
    return r;
}

typedef std::optional<Tensor> Maybe;
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

// What runtime.deliver_grads does: gradients whose parameter still has its slot as .grad are added there, all in one launch, and autograd is
// handed nothing for them.
void deliver(const std::vector<Tensor>& sinks, const variable_list& params, variable_list& out, void* stream) {
    const float* src[5];
    float* dst[5];
    int64_t n[5];
    int k = 0;
    for (int i = 0; i < 5; ++i) {
        Tensor& g = out[4 + i];
        if (!g.defined() || !sinks[i].defined() || !params[i].grad().defined() || params[i].grad().const_data_ptr() != sinks[i].const_data_ptr() ||
            sinks[i].numel() != g.numel() || !params[i].requires_grad()) continue;
        src[k] = g.const_data_ptr<float>(); dst[k] = sinks[i].mutable_data_ptr<float>(); n[k] = g.numel();
        ++k;
    }
    if (k) check(multi_add(k, src, n, n, dst, n, stream));
    for (int i = 0, j = 0; i < 5 && j < k; ++i)                              // the launch has read them: the allocator keeps stream order
        if (out[4 + i].defined() && out[4 + i].const_data_ptr<float>() == src[j]) { out[4 + i] = Tensor(); ++j; }
}

// A leaf's gradient is handed over on the stream on which the oldest living graph used the leaf.  In a capture that must not be the default
// stream: the capture cannot take its work in, and the process ends over it.  So such a backward is refused before it gets there.
void refuse_default_stream_leaves() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    for (const auto& edge : node->next_edges()) {
        auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get());
        if (!leaf) continue;
        if (info && !info->empty()) {                                        // autograd.grad: only what is asked for; it goes to the leaf's stream too
            const auto it = info->find(leaf);
            if (it == info->end() || !it->second.should_execute()) continue;
        }
        const auto s = leaf->stream();
        TORCH_CHECK(!s || s->id() != 0, "gated_residual_norm: backward captured while an eager graph of the same leaves, made on the default stream, is alive; "
                    "drop its outputs first, or run the eager passes on a side stream");
    }
}

// Inputs: x, branch, gate, keep, then the vectors: pre weight, pre bias, post weight, post bias, scale
struct ResnormNode : public torch::autograd::Function<ResnormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& b, const Maybe& gate_, const Maybe& keep_, const Maybe& pre_w_,
                                 const Maybe& pre_b_, const Maybe& post_w_, const Maybe& post_b_, const Maybe& scale_, const Cfg& c) {
        const Tensor gate = or_none(gate_), keep = or_none(keep_), pre_w = or_none(pre_w_), pre_b = or_none(pre_b_), post_w = or_none(post_w_),
                     post_b = or_none(post_b_), scale = or_none(scale_);
        Forward r = launch_forward(x, b, gate, keep, {pre_w, pre_b, post_w, post_b, scale}, c, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({r.h, b, gate, keep, r.stats, pre_w, pre_b, post_w, post_b, scale});
        auto& s = ctx->saved_data;
        s["i"] = std::vector<int64_t>{c.rows, c.n, c.C, c.mode, c.post, c.pre, c.act};
        s["alpha"] = c.alpha;
        if (!c.sinks.empty()) s["sinks"] = c.sinks;
        if (c.pre) return {r.h, r.y};
        return {r.h};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_residual_norm: no gradients of gradients (create_graph=True) are built");
        variable_list out(10);
        const Tensor dh = grads[0], dy = grads.size() > 1 ? grads[1] : Tensor();
        if (!dh.defined() && !dy.defined()) return out;
        refuse_default_stream_leaves();
        const auto saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &b = saved[1], &gate = saved[2], &keep = saved[3], &stats = saved[4], &pre_w = saved[5], &post_w = saved[7], &post_b = saved[8],
                     &scale = saved[9];
        const auto i = ctx->saved_data["i"].toIntVector();
        const int64_t rows = i[0], n = i[1], C = i[2];
        const int mode = (int)i[3], post = (int)i[4], pre = (int)i[5], act = (int)i[6], has_scale = scale.defined();
        c10::DeviceGuard guard(h.device());
        int64_t lddh, lddy, ldb, ldg;
        const Tensor dhs = rows_of(dh, C, lddh), dys = rows_of(dy, C, lddy), bs = rows_of(b, C, ldb), gs = rows_of(gate, C, ldg);
        out[0] = at::empty(h.sizes(), h.options());
        out[1] = at::empty(h.sizes(), b.options());
        if (mode) out[2] = at::empty(gate.sizes(), gate.options());
        const int slots = (pre != 0) + (pre == 1) + (post != 0) + (post == 1) + has_scale;
        const int64_t need = resnorm_ws(rows, n, (int)C, post, pre, mode, has_scale);
        // the vectors' gradients and the partial sums: from the allocator, two captured graphs may replay side by side
        const Tensor vec = at::empty({slots, C}, stats.options()), ws = at::empty({need / 4}, stats.options());
        check(resnorm_bwd(code(h), code(b), raw(dhs), lddh, raw(dys), lddy, raw(h), C, raw(bs), ldb, raw(gs), ldg, mode, act, f32(scale), f32(keep),
                          (float)ctx->saved_data["alpha"].toDouble(), post, f32(post_w), f32(post_b), pre, f32(pre_w), f32(stats), out[0].mutable_data_ptr(),
                          out[1].mutable_data_ptr(), mode ? out[2].mutable_data_ptr() : nullptr, slots ? vec.mutable_data_ptr<float>() : nullptr, rows, n, (int)C,
                          need ? ws.mutable_data_ptr<float>() : nullptr, need, stream_of(h)));
        int k = 0;                                                           // the slots' order; a LayerNorm without a bias has one all the same
        auto slot = [&](const Tensor& like) {
            const Tensor t = vec.select(0, k++);
            return !like.defined() || like.dim() == 1 ? t : t.view(like.sizes());
        };
        if (pre) out[4] = slot(pre_w);
        if (pre == 1) { const Tensor t = slot(saved[6]); if (saved[6].defined()) out[5] = t; }
        if (post) out[6] = slot(post_w);
        if (post == 1) { const Tensor t = slot(post_b); if (post_b.defined()) out[7] = t; }
        if (has_scale) out[8] = slot(scale);
        if (ctx->saved_data.count("sinks")) deliver(ctx->saved_data["sinks"].toTensorVector(), {pre_w, saved[6], post_w, post_b, scale}, out, stream_of(h));
        return out;
    }
};

py::object gated_residual_norm(const Tensor& x, const Tensor& branch, int post, const Maybe& post_w_, const Maybe& post_b_, const Maybe& gate_, int act,
                               const Maybe& scale_, const Maybe& keep_, double alpha, int pre, const Maybe& pre_w_, const Maybe& pre_b_, double eps,
                               int64_t samples, const std::vector<Maybe>& sinks) {
    const Tensor post_w = or_none(post_w_), post_b = or_none(post_b_), gate = or_none(gate_), scale = or_none(scale_), keep = or_none(keep_),
                 pre_w = or_none(pre_w_), pre_b = or_none(pre_b_);
    typedef py::value_error Value;
    typedef py::type_error Type;
    if (x.dim() < 2 || !x.sizes().equals(branch.sizes()))
        fail<Value>("x " + str(x.sizes()) + " and branch " + str(branch.sizes()) + " must be alike, [..., C]");
    Cfg c{0, 0, x.size(-1), 0, post, pre, act, alpha, eps, {}};
    for (const Maybe& t : sinks) c.sinks.push_back(or_none(t));
    if (x.numel() == 0) fail<Value>("nothing in x " + str(x.sizes()));
    c.rows = x.numel() / c.C;
    if (samples == 0) samples = x.dim() > 2 ? x.size(0) : 1;
    if (samples < 1 || c.rows % samples) fail<Value>(std::to_string(c.rows) + " rows do not divide into " + std::to_string(samples) + " samples");
    c.n = c.rows / samples;
    if (gate.defined()) {
        c.mode = gate.sizes().equals(x.sizes()) ? 2 : gate.dim() == 2 && gate.size(0) == samples && gate.size(1) == c.C ? 1 : 0;
        if (c.mode == 0 || gate.scalar_type() != branch.scalar_type())
            fail<Value>("gate must be branch's type, [" + std::to_string(samples) + ", " + std::to_string(c.C) + "] or like x, got " + str(gate.sizes()));
    }
    TORCH_CHECK(x.is_cuda(), "semseg_amd: tensors must live on a HIP device (no CPU fallback)");
    const auto dev = x.device();
    if (branch.device() != dev || (c.mode && gate.device() != dev)) fail<Value>("x, branch and gate must be on one device");
    const auto tx = x.scalar_type(), tb = branch.scalar_type();
    if (!((tx == at::kFloat && (tb == at::kFloat || tb == at::kBFloat16)) || (tx == at::kBFloat16 && tb == at::kBFloat16)))
        fail<Type>("stream / branch types must be f32 / f32, bf16 / bf16 or f32 / bf16");
    if ((post != 0) != post_w.defined() || (post_b.defined() && post != 1) || (pre != 0) != pre_w.defined() || (pre_b.defined() && pre != 1))
        fail<Value>("'layer' takes a weight and optionally a bias, 'rms' a weight, 'none' neither");
    const Tensor* vec[] = {&pre_w, &pre_b, &post_w, &post_b, &scale, &keep};
    const char* names[] = {"pre_weight", "pre_bias", "post_weight", "post_bias", "scale", "keep"};
    bool grad = x.requires_grad() || branch.requires_grad() || (c.mode && gate.requires_grad());
    for (int i = 0; i < 6; ++i) {
        const Tensor& t = *vec[i];
        if (!t.defined()) continue;
        const int64_t want = i == 5 ? samples : c.C;
        if (t.scalar_type() != at::kFloat || t.numel() != want || !t.is_contiguous() || t.device() != dev)
            fail<Value>(std::string(names[i]) + " must be contiguous float32 of " + std::to_string(want) + " elements on x's device, got " + str(t.sizes()));
        grad = grad || (i < 5 && t.requires_grad());
    }
    Tensor h, y;
    {
        py::gil_scoped_release nogil;
        if (grad && at::GradMode::is_enabled()) {
            const auto r = ResnormNode::apply(x, branch, gate_, keep_, pre_w_, pre_b_, post_w_, post_b_, scale_, c);
            h = r[0];
            if (c.pre) y = r[1];
        } else {
            const Forward r = launch_forward(x, branch, gate, keep, {pre_w, pre_b, post_w, post_b, scale}, c, false);
            h = r.h;
            y = r.y;
        }
    }
    return py::make_tuple(py::cast(h), c.pre ? py::cast(y) : py::none());
}

// Parameters and their .grad -> (gradient type code, parameters' addresses, gradients' addresses), host arrays of 64-bit words; everything
// that the step relies on is checked.
py::tuple addresses(const std::vector<Tensor>& params, const std::vector<int64_t>& numels, int dtype_code, int64_t device) {
    const at::ScalarType want = dtype_code ? at::kBFloat16 : at::kFloat;
    std::vector<uint64_t> pa(params.size()), ga(params.size(), 0);
    int gt = -1;
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor& p = params[i];
        TORCH_CHECK(p.scalar_type() == want && p.is_cuda() && p.device().index() == device && p.numel() == numels[i] && p.is_contiguous(),
                    "AdamW: a parameter changed its type, device, size or layout");
        pa[i] = (uint64_t)p.const_data_ptr();
        const Tensor& g = p.grad();
        if (!g.defined()) continue;
        const int t = g.scalar_type() == at::kFloat ? 0 : g.scalar_type() == at::kBFloat16 ? 1 : 2;
        if (gt < 0) gt = t;
        TORCH_CHECK(t == gt && t < 2 && g.layout() == at::kStrided && g.is_contiguous() && g.device() == p.device() && g.numel() == numels[i],
                    "AdamW: gradients must be contiguous, of one type (float32 or bfloat16) and like their parameters");
        ga[i] = (uint64_t)g.const_data_ptr();
    }
    return py::make_tuple(gt < 0 ? 0 : gt, py::bytes((const char*)pa.data(), pa.size() * 8), py::bytes((const char*)ga.data(), ga.size() * 8));
}

void init(uint64_t fwd, uint64_t ws, uint64_t bwd, uint64_t add, uint64_t err) {
    resnorm_fwd = (fwd_fn)fwd;
    resnorm_ws = (ws_fn)ws;
    resnorm_bwd = (bwd_fn)bwd;
    multi_add = (add_fn)add;
    last_error = (err_fn)err;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
    m.def("init", &init);
    m.def("gated_residual_norm", &gated_residual_norm);
    m.def("addresses", &addresses);
}
