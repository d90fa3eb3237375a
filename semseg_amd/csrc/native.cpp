// Host side of the calls whose cost is the host's: the autograd node of the gated residual norm and the address lists of the optimizer.
//
// A training call on a few thousand rows is 30 us of GPU work; as a Python autograd.Function it is 160 us of host work, half of it in the
// backward, which autograd runs on another thread with the interpreter's lock in between.  Here the node is C++: checks, allocations and
// launches without the interpreter, 78 us.  The kernels are those of the C ABI; their addresses are handed over by init(), from the library that
// the Python side has loaded, so there is one library whatever its path.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>
#include <unordered_set>
#include <vector>

using at::Tensor;
using torch::autograd::SavedVariable;
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

// autograd.grad and backward(inputs=...): gradients of some tensors only, or to be handed to the caller
bool some_gradients_only() {
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    return info && !info->empty();
}
// Whether a parameter's gradient is autograd's to place, not the node's: in such a pass it goes to the caller, or nowhere; and where the
// parameter's accumulator belongs to another stream than the one at work, only autograd's own hand-over makes the caller's stream wait
// (in a capture the node's launch is part of the graph, and a hand-over to a stream outside would break it).
bool left_to_autograd(const Tensor& p) {
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(p);
    if (some_gradients_only()) {
        const auto* info = torch::autograd::get_current_graph_task_exec_info();
        const auto it = info->find(accumulator.get());
        if (it == info->end() || !it->second.needed_ || it->second.captures_) return true;
    }
    if (!accumulator || !p.is_cuda() || c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) return false;
    const auto s = accumulator->stream();
    return s && *s != c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(p.device().index()).unwrap();
}

// What runtime.deliver_grads does: gradients whose parameter still has its slot as .grad are added there, all in one launch, and autograd is
// handed nothing for them.
void deliver(const std::vector<Tensor>& sinks, const variable_list& params, Tensor* grads, void* stream) {
    const float* src[5];
    float* dst[5];
    int64_t n[5];
    int at[5], k = 0;
    for (int i = 0; i < 5; ++i) {
        const Tensor &g = grads[i], &p = params[i];
        if (!g.defined() || !sinks[i].defined() || !p.requires_grad() || !p.grad().defined() || p.grad().const_data_ptr() != sinks[i].const_data_ptr() ||
            sinks[i].numel() != g.numel() || left_to_autograd(p)) continue;
        src[k] = g.const_data_ptr<float>(); dst[k] = sinks[i].mutable_data_ptr<float>(); n[k] = g.numel(); at[k++] = i;
    }
    if (k) check(multi_add(k, src, n, n, dst, n, stream));
    while (k) grads[at[--k]] = Tensor();                                     // the launch reads them in stream order, the allocator keeps it
}

// A leaf's gradient is handed over on the stream on which the oldest living graph used the leaf.  In a capture that must not be the default
// stream: the capture cannot take its work in, and the process ends over it.  The same holds for any other node that was made there.  So such
// a backward is refused before it gets there, for everything that this node's gradients reach, through views and other nodes too.  (Nodes
// that come before this one in the backward have had their turn by then.)
void refuse_default_stream_leaves(const torch::autograd::Node& node) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    std::vector<const torch::autograd::Node*> open{&node};
    std::unordered_set<const torch::autograd::Node*> seen;
    while (!open.empty()) {
        const torch::autograd::Node* at = open.back();
        open.pop_back();
        for (const auto& edge : at->next_edges()) {
            auto* next = edge.function.get();
            if (!next || !seen.insert(next).second) continue;
            if (info && !info->empty()) {                                    // autograd.grad: only what is asked for; it goes to the leaf's stream too
                const auto it = info->find(next);
                if (it == info->end() || !it->second.should_execute()) continue;
            }
            const auto s = next->stream();
            TORCH_CHECK(!s || s->id() != 0, "gated_residual_norm: backward captured while an eager graph of the same leaves, made on the default stream, is alive; "
                        "drop its outputs first, or run the eager passes on a side stream");
            open.push_back(next);
        }
    }
}
// for a node whose backward is Python, while it runs
void refuse_captured_leaves() {
    if (const auto node = torch::autograd::get_current_node()) refuse_default_stream_leaves(*node);
}

// The node itself, with members of its own: torch::autograd::Function keeps what it saves in a dictionary of boxed values and dispatches every
// allocation through autograd (forward and backward on 5223 x 97: 84 us of host time, 78 without; torch's own layer_norm takes 64, of which
// 34 are the hand-over to autograd's thread and back).
// Edges: x, branch, gate, then the vectors: pre weight, pre bias, post weight, post bias, scale
struct ResnormNode : public torch::autograd::Node {
    Cfg c;
    SavedVariable h, b, gate, keep, stats, vectors[5];

    std::string name() const override { return "GatedResidualNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        h.reset_data(); b.reset_data(); gate.reset_data(); keep.reset_data(); stats.reset_data();
        for (auto& v : vectors) v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_residual_norm: no gradients of gradients (create_graph=True) are built");
        variable_list out(8);
        const Tensor dh = grads[0], dy = grads.size() > 1 ? grads[1] : Tensor();
        if (!dh.defined() && !dy.defined()) return out;
        refuse_default_stream_leaves(*this);
        const Tensor h_ = h.unpack(getptr()), b_ = b.unpack(), gate_ = gate.unpack(), keep_ = keep.unpack(), stats_ = stats.unpack();
        variable_list v(5);
        for (int i = 0; i < 5; ++i) v[i] = vectors[i].unpack();
        const Tensor &pre_w = v[0], &post_w = v[2], &post_b = v[3], &scale = v[4];
        c10::DeviceGuard guard(h_.device());
        at::AutoDispatchBelowADInplaceOrView below;
        void* stream = stream_of(h_);
        int64_t lddh, lddy, ldb, ldg;
        const Tensor dhs = rows_of(dh, c.C, lddh), dys = rows_of(dy, c.C, lddy), bs = rows_of(b_, c.C, ldb), gs = rows_of(gate_, c.C, ldg);
        out[0] = at::empty(h_.sizes(), h_.options());
        out[1] = at::empty(h_.sizes(), b_.options());
        if (c.mode) out[2] = at::empty(gate_.sizes(), gate_.options());
        const int slots = (c.pre != 0) + (c.pre == 1) + (c.post != 0) + (c.post == 1) + scale.defined();
        const int64_t need = resnorm_ws(c.rows, c.n, (int)c.C, c.post, c.pre, c.mode, scale.defined());
        // the vectors' gradients and the partial sums: from the allocator, two captured graphs may replay side by side
        const Tensor vec = at::empty({slots, c.C}, stats_.options()), ws = at::empty({need / 4}, stats_.options());
        check(resnorm_bwd(code(h_), code(b_), raw(dhs), lddh, raw(dys), lddy, raw(h_), c.C, raw(bs), ldb, raw(gs), ldg, c.mode, c.act, f32(scale), f32(keep_),
                          (float)c.alpha, c.post, f32(post_w), f32(post_b), c.pre, f32(pre_w), f32(stats_), out[0].mutable_data_ptr(),
                          out[1].mutable_data_ptr(), c.mode ? out[2].mutable_data_ptr() : nullptr, slots ? vec.mutable_data_ptr<float>() : nullptr, c.rows, c.n,
                          (int)c.C, need ? ws.mutable_data_ptr<float>() : nullptr, need, stream));
        const bool has[5] = {c.pre != 0, c.pre == 1, c.post != 0, c.post == 1, scale.defined()};
        int k = 0;                                                           // the slots' order; a LayerNorm without a bias has one all the same
        for (int i = 0; i < 5; ++i) {
            if (!has[i]) continue;
            if (v[i].defined() && task_should_compute_output(3 + i)) {
                const Tensor t = vec.select(0, k);
                out[3 + i] = v[i].dim() == 1 ? t : t.view(v[i].sizes());
            }
            ++k;
        }
        if (!c.sinks.empty()) deliver(c.sinks, v, &out[3], stream);
        return out;
    }
};

Forward forward_with_graph(const Tensor& x, const Tensor& b, const Tensor& gate, const Tensor& keep, const variable_list& vectors, Cfg c) {
    Forward r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = launch_forward(x, b, gate, keep, vectors, c, true);
    }
    std::shared_ptr<ResnormNode> node(new ResnormNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, b, gate, vectors[0], vectors[1], vectors[2], vectors[3], vectors[4]));
    torch::autograd::set_history(r.h, node);
    if (r.y.defined()) torch::autograd::set_history(r.y, node);
    node->h = SavedVariable(r.h, true);
    node->b = SavedVariable(b, false);
    node->gate = SavedVariable(gate, false);
    node->keep = SavedVariable(keep, false);
    for (int i = 0; i < 5; ++i) node->vectors[i] = SavedVariable(vectors[i], false);
    node->stats = SavedVariable(r.stats, false);
    node->c = std::move(c);
    return r;
}

typedef std::optional<Tensor> Maybe;
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

typedef c10::impl::TorchDispatchModeTLS Modes;
// The kernels write new tensors behind the dispatcher's back: what follows a computation by watching it would see nothing of this one.
void refuse_watchers(const std::vector<Maybe>& inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY) &&
                                !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                                "gated_residual_norm: tracing would record outputs that nothing computes; it is not built");
    for (const Maybe& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), "gated_residual_norm: no forward-mode derivatives are built");
}

py::object gated_residual_norm(const Tensor& x, const Tensor& branch, int post, const Maybe& post_w_, const Maybe& post_b_, const Maybe& gate_, int act,
                               const Maybe& scale_, const Maybe& keep_, double alpha, int pre, const Maybe& pre_w_, const Maybe& pre_b_, double eps,
                               int64_t samples, const std::vector<Maybe>& sinks) {
    const Tensor post_w = or_none(post_w_), post_b = or_none(post_b_), gate = or_none(gate_), scale = or_none(scale_), keep = or_none(keep_),
                 pre_w = or_none(pre_w_), pre_b = or_none(pre_b_);
    typedef py::value_error Value;
    typedef py::type_error Type;
    refuse_watchers({x, branch, gate_, post_w_, post_b_, pre_w_, pre_b_, scale_, keep_});
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
        const variable_list vectors{pre_w, pre_b, post_w, post_b, scale};
        const Forward r = grad && at::GradMode::is_enabled() ? forward_with_graph(x, branch, gate, keep, vectors, std::move(c))
                                                             : launch_forward(x, branch, gate, keep, vectors, c, false);
        h = r.h;
        y = r.y;
    }
    return py::make_tuple(py::cast(h), y.defined() ? py::cast(y) : py::none());
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

// Parameters that are to lie, with their gradients, at `offsets` of two flat float buffers; the handles are kept, what they hold is looked at
// by each call (turning a list of 186 parameters into handles is 8 us)
struct FlatSlots {
    std::vector<Tensor> params;
    std::vector<int64_t> offsets;
    // -> the first that lies elsewhere, or -1
    int64_t first_stray(uint64_t data, uint64_t grad) const {
        for (size_t i = 0; i < params.size(); ++i) {
            const Tensor &p = params[i], &g = p.grad();
            if (p.numel() == 0) continue;
            if ((uint64_t)p.const_data_ptr() != data + 4 * offsets[i] || !g.defined() || (uint64_t)g.const_data_ptr() != grad + 4 * offsets[i]) return i;
        }
        return -1;
    }
};

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
    m.def("refuse_watchers", &refuse_watchers);
    m.def("refuse_captured_leaves", &refuse_captured_leaves);
    m.def("left_to_autograd", &left_to_autograd);
    m.def("addresses", &addresses);
    py::class_<FlatSlots>(m, "FlatSlots")
        .def(py::init([](std::vector<Tensor> params, std::vector<int64_t> offsets) {
            TORCH_CHECK(params.size() == offsets.size(), "FlatSlots: an offset for each parameter");
            return FlatSlots{std::move(params), std::move(offsets)};
        }))
        .def("first_stray", &FlatSlots::first_stray);
}
