// Host side of the operators whose calls are short beside their Python: group_norm_act (its checks, allocations and autograd node), the gradient
// lists of grad_norm / clip_grad_norm_ (one pass over the tensors) and the table of the fused SGD step.  A CPython extension over torch's C++ API;
// everything that runs on the GPU goes through the C ABI of include/lgd_hip.h, whose entry points lgd_amd/hip.py hands over (bind), so that both see
// the same library.
// What it is for: a training call on small maps costs the host two autograd.Function halves on two threads, 145 us on the MI355X host where the GPU needs
// 25; a list of 160 gradients 62 us for 16; the step over 10 (160) tensors 37 (60) us in Python, 13 (26) here.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <mutex>
#include <sstream>
#include <vector>

#include "../../include/lgd_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct {
    decltype(&lgd_gn_act_ws_bytes) gn_ws;
    decltype(&lgd_gn_act_fwd) gn_fwd;
    decltype(&lgd_gn_act_bwd) gn_bwd;
    decltype(&lgd_grad_norm_ws_bytes) norm_ws;
    decltype(&lgd_grad_norm) norm;
    decltype(&lgd_grad_clip) clip;
    decltype(&lgd_sgd_clip_step) sgd_clip;
    decltype(&lgd_sgd_norm_ws_bytes) sgd_norm_ws;
    decltype(&lgd_sgd_norm_step) sgd_norm;
    decltype(&lgd_sgd_norm_step_host) sgd_norm_host;
    decltype(&lgd_last_error) last_error;
    PyObject* error = nullptr;   // LgdHipError
} api;

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };   // becomes LgdHipError

template <typename... A> [[noreturn]] void refuse(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    throw Refused(s.str());
}
void check(int rc, const char* what) {
    if (rc != LGD_OK) refuse(what, " failed with code ", rc, " ", api.last_error());
}

int type_code(const Tensor& t) {   // LGD_F32 / LGD_BF16 / LGD_F16, -1: none of them
    switch (t.scalar_type()) {
        case at::kFloat: return LGD_F32;
        case at::kBFloat16: return LGD_BF16;
        case at::kHalf: return LGD_F16;
        default: return -1;
    }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// a tangent of forward-mode differentiation: these operators would drop it, which is a derivative of zero.  Tangents live while a dual level is open; asking
// that first costs a call 20 ns, asking 160 tensors 3 us of a norm's 17
bool duals_possible() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void refuse_dual(const Tensor& t, const char* what) {
    if (t.defined() && t._fw_grad(0).defined()) refuse(what, " has no forward-mode derivative: an input carries a tangent");
}
Tensor dense(const Tensor& t) { return t.is_contiguous(at::MemoryFormat::ChannelsLast) ? t : t.contiguous(at::MemoryFormat::ChannelsLast); }
void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------------------------------------- group_norm_act
struct GnCall {   // what forward and backward share: the non-empty maps and their shapes
    std::vector<int> live;
    std::vector<int32_t> hw;
    std::vector<const void*> x;
    int L = 0, B = 0, C = 0, type = 0, ptype = 0;
    GnCall(const variable_list& xs, const Tensor& w, const Tensor& b) {
        for (size_t i = 0; i < xs.size(); ++i) {
            if (xs[i].numel() == 0) continue;
            live.push_back((int)i);
            hw.push_back((int32_t)xs[i].size(2)); hw.push_back((int32_t)xs[i].size(3));
            x.push_back(xs[i].data_ptr());
        }
        L = (int)live.size(); B = (int)xs[0].size(0); C = (int)xs[0].size(1);
        type = type_code(xs[0]);
        ptype = w.defined() ? type_code(w) : b.defined() ? type_code(b) : LGD_F32;
    }
};

void gn_check(const variable_list& xs, int64_t groups, const Tensor& w, const Tensor& b, double eps) {
    const Tensor& x0 = xs[0];
    if (!(eps >= 0)) refuse("eps must not be negative, got ", eps);
    if (xs.size() > LGD_MAX_LEVELS) refuse("at most ", LGD_MAX_LEVELS, " maps per call (LGD_MAX_LEVELS), got ", xs.size());
    if (type_code(x0) < 0) refuse("group_norm_act takes fp32, bf16 or fp16 maps, got ", x0.scalar_type());
    for (const Tensor& x : xs) {
        if (x.dim() != 4 || x0.dim() != 4 || x.size(0) != x0.size(0) || x.size(1) != x0.size(1))
            refuse("maps of one call are (B,C,H_l,W_l) with the same B and C, got ", x0.sizes(), " and ", x.sizes());
        if (x.scalar_type() != x0.scalar_type() || x.device() != x0.device() || x.layout() != at::kStrided)
            refuse("maps of one call are strided, of one type and on one device, got ", x.layout(), " ", x.scalar_type(), " ", x.device(), " beside ",
                   x0.scalar_type(), " ", x0.device());
        for (int d = 0; d < 4; ++d) if (x.size(d) > INT32_MAX) refuse("a map's sizes are below 2^31, got ", x.sizes());
    }
    if (duals_possible()) {
        for (const Tensor& x : xs) refuse_dual(x, "group_norm_act");
        refuse_dual(w, "group_norm_act"); refuse_dual(b, "group_norm_act");
    }
    const int64_t C = x0.size(1);
    if (groups < 1 || C < 1 || groups > C || C % groups) refuse(C, " channels do not split into ", groups, " groups");
    for (const Tensor* p : {&w, &b})
        if (p->defined() && (type_code(*p) < 0 || p->dim() != 1 || p->size(0) != C || p->device() != x0.device() || p->layout() != at::kStrided))
            refuse(p == &w ? "weight" : "bias", " must be ", C, " fp32, bf16 or fp16 values on ", x0.device(), ", got ", p->sizes(), " ",
                   p->scalar_type(), " on ", p->device());
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type())
        refuse("weight and bias have one type, got ", w.scalar_type(), " and ", b.scalar_type());
}

// xs dense, w and b contiguous; stats: kept for a backward.  Below autograd
variable_list gn_forward(const variable_list& xs, int groups, int act, double eps, const Tensor& w, const Tensor& b, bool keep, Tensor& stats) {
    variable_list ys;
    ys.reserve(xs.size());
    for (const Tensor& x : xs) ys.push_back(at::empty_like(x));
    GnCall c(xs, w, b);
    if (c.L == 0) return ys;
    const c10::DeviceGuard guard(xs[0].device());
    const size_t n = api.gn_ws(c.hw.data(), c.L, c.B, c.C, groups, c.type, 0);
    if (n == (size_t)-1) refuse("group_norm_act: 2^31 elements per sample, or 2^30 groups of all maps and samples, or more are not supported");
    const int64_t words = 2LL * c.L * c.B * groups;
    const auto f64 = xs[0].options().dtype(at::kDouble).memory_format(at::MemoryFormat::Contiguous);
    // one allocation, unless the statistics outlive the workspace
    Tensor ws;
    const bool apart = keep && n > 0;
    stats = at::empty({words + (apart ? 0 : (int64_t)n / 8)}, f64);
    if (apart) ws = at::empty({(int64_t)n / 8}, f64);
    double* st = stats.data_ptr<double>();
    std::vector<void*> y;
    for (int i : c.live) y.push_back(ys[i].data_ptr());
    check(api.gn_fwd(c.x.data(), c.hw.data(), c.L, c.B, c.C, groups, c.type, ptr_or_null(w), ptr_or_null(b), c.ptype, eps, act,
                     n == 0 ? nullptr : apart ? ws.data_ptr() : st + words, st, y.data(), stream_of(xs[0])), "lgd_gn_act_fwd");
    return ys;
}

// stands behind a result that depends on its inputs in a way no graph holds: differentiating it must raise
struct NoDerivative : public Node {
    std::string who, what;
    NoDerivative(std::string w, std::string t) : who(std::move(w)), what(std::move(t)) {}
    variable_list apply(variable_list&&) override { throw std::runtime_error(who + " has no " + what); }
    std::string name() const override { return "NoDerivative"; }
};
std::shared_ptr<Node> no_derivative(const char* who, const char* what, torch::autograd::edge_list&& edges) {
    std::shared_ptr<Node> node(new NoDerivative(who, what), torch::autograd::deleteNode);
    node->set_next_edges(std::move(edges));
    return node;
}

// What is saved is read and released under the node's lock: two threads may differentiate one graph, one of them releasing it
struct GnBackward : public Node {
    std::vector<SavedVariable> x;
    SavedVariable w, b;
    Tensor stats;
    int groups = 0, act = 0;
    bool released = false;

    std::string name() const override { return "GroupNormActBackward"; }
    void release_variables() override {
        std::vector<SavedVariable> xs;   // let go of behind the lock: the last reference of a tensor may call into Python
        SavedVariable wv, bv;
        Tensor st;
        const std::lock_guard<std::mutex> lock(mutex_);
        std::swap(xs, x); std::swap(wv, w); std::swap(bv, b); std::swap(st, stats);
        released = true;
    }
    // A leaf whose gradient accumulator belongs to an older graph, made on another stream, would have the engine make that stream wait inside the capture:
    // an error that ends the process.  Refused before it gets there
    void refuse_capture() {
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
        const c10::StreamId here = c10::hip::getCurrentHIPStream().id();
        for (const auto& e : next_edges()) {
            if (!e.function || e.function->num_outputs() != 0) continue;   // (accumulators have no next functions)
            const auto s = e.function->stream();
            if (s && s->id() != here)
                throw std::runtime_error("group_norm_act: a leaf of this captured backward is held by a graph that was made on another stream; "
                                         "release that graph, or capture with leaves of its own");
        }
    }
    variable_list apply(variable_list&& dys) override {
        const bool again = at::GradMode::is_enabled();   // create_graph
        variable_list xs;
        Tensor wv, bv, st;
        {
            const std::lock_guard<std::mutex> lock(mutex_);
            TORCH_CHECK(!released, "group_norm_act: the graph has been freed; backward a second time needs retain_graph=True the first time");
            for (auto& v : x) xs.push_back(v.unpack());
            wv = w.unpack(); bv = b.unpack(); st = stats;
        }
        variable_list out(xs.size() + 2);
        bool any = false;
        for (const Tensor& d : dys) any = any || d.defined();
        if (!any) return out;
        if (duals_possible()) for (const Tensor& d : dys)
            if (d.defined() && d._fw_grad(0).defined()) throw std::runtime_error("group_norm_act has no forward-mode derivative: an output's gradient carries a tangent");
        refuse_capture();
        {
            at::AutoDispatchBelowADInplaceOrView below;
            run(xs, wv, bv, st, dys, out);
        }
        if (again) {
            torch::autograd::edge_list edges;
            for (const auto& e : next_edges()) if (e.is_valid()) edges.push_back(e);   // the call's own inputs: what is saved may be a copy of them
            for (const Tensor& t : dys)
                if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
            if (!edges.empty()) {
                const auto node = no_derivative("group_norm_act", "second derivative", std::move(edges));   // (of gradients computed under create_graph)
                for (Tensor& t : out) if (t.defined()) torch::autograd::set_history(t, node);
            }
        }
        return out;
    }
    void run(const variable_list& saved, const Tensor& w0, const Tensor& b0, const Tensor& st, const variable_list& dys, variable_list& out) {
        const size_t nx = saved.size();
        variable_list xs;   // (hooks on saved tensors may hand them back in another order)
        for (const Tensor& x : saved) xs.push_back(dense(x));
        const Tensor wv = w0.defined() ? w0.contiguous() : w0, bv = b0.defined() ? b0.contiguous() : b0;
        bool want_x = false;
        for (size_t i = 0; i < nx; ++i) want_x = want_x || task_should_compute_output(i);
        Tensor dw, db;
        if (wv.defined() && task_should_compute_output(nx)) dw = at::empty_like(wv);
        if (bv.defined() && task_should_compute_output(nx + 1)) db = at::empty_like(bv);
        variable_list dxs(nx);
        if (want_x) for (size_t i = 0; i < nx; ++i) dxs[i] = at::empty_like(xs[i]);
        GnCall c(xs, wv, bv);
        if (c.L == 0) {
            if (dw.defined()) dw.zero_();
            if (db.defined()) db.zero_();
        } else {
            const c10::DeviceGuard guard(xs[0].device());
            variable_list ds;
            std::vector<const void*> dy;
            std::vector<void*> dx;
            for (int i : c.live) {
                ds.push_back(dys[i].defined() ? dense(dys[i]) : at::zeros_like(xs[i]));
                dy.push_back(ds.back().data_ptr());
                if (want_x) dx.push_back(dxs[i].data_ptr());
            }
            const size_t n = api.gn_ws(c.hw.data(), c.L, c.B, c.C, groups, c.type, 1);
            Tensor ws;
            if (n) ws = at::empty({(int64_t)n}, xs[0].options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
            check(api.gn_bwd(c.x.data(), dy.data(), c.hw.data(), c.L, c.B, c.C, groups, c.type, ptr_or_null(wv), ptr_or_null(bv), c.ptype, act,
                             st.data_ptr<double>(), ptr_or_null(ws), want_x ? dx.data() : nullptr, ptr_or_null(dw), ptr_or_null(db), stream_of(xs[0])),
                  "lgd_gn_act_bwd");
        }
        for (size_t i = 0; i < nx; ++i) if (task_should_compute_output(i)) out[i] = dxs[i];
        out[nx] = dw; out[nx + 1] = db;
    }
};

variable_list gn_act(const variable_list& xs, int groups, int act, double eps, const Tensor& w, const Tensor& b) {
    bool grad = false;
    if (at::GradMode::is_enabled()) {
        for (const Tensor& x : xs) grad = grad || x.requires_grad();
        grad = grad || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad());
    }
    variable_list xd, ys;
    Tensor wd, bd, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        for (const Tensor& x : xs) xd.push_back(dense(x));
        if (w.defined()) wd = w.contiguous();
        if (b.defined()) bd = b.contiguous();
        ys = gn_forward(xd, groups, act, eps, wd, bd, grad, stats);
    }
    if (grad) {
        auto node = std::shared_ptr<GnBackward>(new GnBackward(), torch::autograd::deleteNode);
        torch::autograd::edge_list edges;
        auto edge = [&](const Tensor& t) {
            if (t.defined() && t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
            else edges.emplace_back();
        };
        for (const Tensor& x : xs) edge(x);
        edge(w); edge(b);
        node->set_next_edges(std::move(edges));
        for (const Tensor& x : xd) node->x.emplace_back(x, false);
        node->w = SavedVariable(wd, false);
        node->b = SavedVariable(bd, false);
        node->stats = stats;
        node->groups = groups; node->act = act;
        for (Tensor& y : ys) torch::autograd::set_history(y, node);
    }
    return ys;
}

// ------------------------------------------------------------------------------------------- lists of gradients
// the tensors of a Python sequence; grads: their gradients, where they have one
std::vector<Tensor> tensors_of(PyObject* seq, bool grads) {
    std::vector<Tensor> out;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    PyObject** items = PySequence_Fast_ITEMS(seq);
    out.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(items[i])) refuse("expected tensors, got ", Py_TYPE(items[i])->tp_name);
        const Tensor& t = THPVariable_Unpack(items[i]);
        if (!grads) out.push_back(t);
        else if (t.grad().defined()) out.push_back(t.grad());
    }
    return out;
}

using Runs = std::vector<std::pair<uintptr_t, uintptr_t>>;   // addresses: first, behind the last
void refuse_overlap(Runs& runs) {
    std::sort(runs.begin(), runs.end());
    for (size_t i = 1; i < runs.size(); ++i)
        if (runs[i - 1].second > runs[i].first) refuse("two of the gradients share memory: each element can be clipped once");
}

// in-place scaling needs every element once: a gradient listed twice, an expanded one, or views that overlap are refused.  copies: of the tensors that are
// not dense, undefined for the others
void refuse_shared(const std::vector<Tensor>& ts, const std::vector<Tensor>& copies) {
    Runs runs;
    std::vector<const void*> strided;
    for (size_t i = 0; i < ts.size(); ++i) {
        if (ts[i].numel() == 0) continue;
        const uintptr_t p = (uintptr_t)(copies[i].defined() ? copies[i] : ts[i]).data_ptr();
        runs.emplace_back(p, p + ts[i].numel() * ts[i].element_size());
        if (!copies[i].defined()) continue;
        strided.push_back(ts[i].data_ptr());
        for (int64_t d = 0; d < ts[i].dim(); ++d)
            if (ts[i].stride(d) == 0 && ts[i].size(d) > 1) refuse("a gradient that is expanded, or listed twice, cannot be clipped in place");
    }
    refuse_overlap(runs);
    std::sort(strided.begin(), strided.end());
    if (std::adjacent_find(strided.begin(), strided.end()) != strided.end()) refuse("a gradient that is expanded, or listed twice, cannot be clipped in place");
}

// the norm of the tensors (clip: and their scaling in place).  Undefined: they are not on a GPU
Tensor norm_of(const std::vector<Tensor>& ts, int norm_type, bool clip, double max_norm) {
    std::vector<Tensor> copies(ts.size());
    std::vector<lgd_grad_tensor> rec;
    rec.reserve(ts.size());
    const c10::Device dev = ts[0].device();
    const bool duals = duals_possible();
    at::AutoDispatchBelowADInplaceOrView below;
    for (size_t i = 0; i < ts.size(); ++i) {
        const Tensor& t = ts[i];
        const int type = type_code(t);
        if (t.layout() != at::kStrided || type < 0 || t.device() != dev)
            refuse("gradient norms take strided fp32, bf16 or fp16 tensors on one device, got ",
                   t.layout(), " ", t.scalar_type(), " ", t.device(), " (the first is on ", dev, ")");
        if (duals) refuse_dual(t, "the norm of gradients");
        if (!t.is_non_overlapping_and_dense()) copies[i] = t.contiguous();   // (any dense order is one run of memory)
        rec.push_back({(copies[i].defined() ? copies[i] : t).data_ptr(), t.numel(), type, 0});
    }
    if (clip) refuse_shared(ts, copies);
    if (!dev.is_cuda()) return Tensor();
    const c10::DeviceGuard guard(dev);
    const auto f32 = at::TensorOptions().device(dev).dtype(at::kFloat);
    Tensor out = at::empty({}, f32);
    const Tensor ws = at::empty({(int64_t)((api.norm_ws((int)rec.size()) + 7) / 8)}, f32.dtype(at::kDouble));
    if (clip) check(api.clip(rec.data(), (int)rec.size(), norm_type, (float)max_norm, ws.data_ptr(), out.data_ptr<float>(), stream_of(out)), "lgd_grad_clip");
    else check(api.norm(rec.data(), (int)rec.size(), norm_type, ws.data_ptr(), out.data_ptr<float>(), stream_of(out)), "lgd_grad_norm");
    if (clip)
        for (size_t i = 0; i < ts.size(); ++i) {
            if (copies[i].defined()) const_cast<Tensor&>(ts[i]).copy_(copies[i]);
            torch::autograd::impl::bump_version(ts[i]);   // written through a raw pointer
        }
    return out;
}

// ------------------------------------------------------------------------------------------- the fused step
bool dense_f32(const Tensor& t) { return t.layout() == at::kStrided && t.scalar_type() == at::kFloat && t.is_contiguous(); }

// what follows from the set of parameters that have a gradient, laid out by lgd_amd/optim.py
struct SgdPlan {
    const int32_t* rows;           // the parameters of the table's rows, ascending
    const lgd_sgd_tensor* table;   // n and reserved filled in
    const int32_t* blk;            // [k + 1]
    const int32_t* set;            // [k] which hyper-parameters
    const int32_t* border;         // [groups + 1] rows and blocks of the optimizers
    const int32_t* border_blk;
    int k, groups;
};
enum class Sgd { kDone, kOtherSet, kNotGpu };

Sgd sgd_step(PyObject* params, PyObject* momenta, const SgdPlan& plan, const std::vector<float>& hyper, bool by_norm, int norm_type, double clip,
             Tensor& norms) {
    const int n = (int)PyList_GET_SIZE(params), k = plan.k;
    std::vector<Tensor> ps, gs, ms;
    ps.reserve(k); gs.reserve(k); ms.reserve(k);
    for (int i = 0, j = 0; i < n; ++i) {
        const Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(params, i));
        const Tensor& g = p.grad();
        const bool row = j < k && plan.rows[j] == i;
        if (g.defined() != row) return Sgd::kOtherSet;
        if (!row) continue;
        ps.push_back(p); gs.push_back(g); ms.push_back(THPVariable_Unpack(PyList_GET_ITEM(momenta, i)));
        ++j;
    }
    const c10::Device dev = gs[0].device();
    if (!dev.is_cuda()) return Sgd::kNotGpu;
    const c10::DeviceGuard guard(dev);
    // (a replay would upload whatever the pinned block holds by then: addresses of nothing)
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        refuse("the fused step's table (addresses, learning rates) is the host's of this call: it cannot be captured into a graph");
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t bytes = (int64_t)k * sizeof(lgd_sgd_tensor) + 4 * (k + 1), room = (bytes + 15) / 16 * 16;
    const bool inl = by_norm && k <= LGD_SGD_INLINE;   // the table in the kernels' arguments: no upload
    // torch hands a pinned block out again only after the copies that read it
    const Tensor host = inl ? Tensor() : at::empty({bytes}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
    lgd_sgd_tensor own[LGD_SGD_INLINE];
    lgd_sgd_tensor* t = inl ? own : static_cast<lgd_sgd_tensor*>(host.data_ptr());
    memcpy(t, plan.table, (size_t)k * sizeof(lgd_sgd_tensor));
    Runs runs;
    for (int j = 0; j < k; ++j) {
        // (the sizes of parameters and momenta are checked against the plan's by the caller; `.data` can be anything by now)
        if (!dense_f32(gs[j]) || gs[j].device() != dev || gs[j].numel() != t[j].n)
            refuse("fused SGD needs dense contiguous fp32 gradients of their parameters' sizes on one device");
        if (!dense_f32(ps[j]) || ps[j].device() != dev) refuse("fused SGD needs dense contiguous fp32 parameters, beside their gradients");
        if (!dense_f32(ms[j]) || ms[j].device() != dev) refuse("fused SGD needs dense contiguous fp32 momentum buffers, beside their gradients");
        t[j].p = ps[j].data_ptr<float>(); t[j].g = gs[j].data_ptr<float>(); t[j].m = ms[j].data_ptr<float>();
        const float* h = &hyper[3 * (size_t)plan.set[j]];
        t[j].lr = h[0]; t[j].wd = h[1]; t[j].mu = h[2];
        if (by_norm && t[j].n > 0) runs.emplace_back((uintptr_t)t[j].g, (uintptr_t)(t[j].g + t[j].n));
    }
    refuse_overlap(runs);
    const int64_t ws = by_norm ? (int64_t)api.sgd_norm_ws(plan.groups) : 0;
    Tensor work = at::empty({(inl ? 0 : room) + ws}, at::TensorOptions().device(dev).dtype(at::kByte));
    char* base = static_cast<char*>(work.data_ptr());
    void* stream = stream_of(work);
    if (!inl) {
        memcpy(t + k, plan.blk, 4 * (size_t)(k + 1));
        work.narrow(0, 0, bytes).copy_(host, true);
    }
    const auto* table = reinterpret_cast<const lgd_sgd_tensor*>(base);
    const auto* blk = reinterpret_cast<const int32_t*>(table + k);
    if (by_norm) {
        norms = at::empty({plan.groups}, at::TensorOptions().device(dev).dtype(at::kFloat));
        float* out = norms.data_ptr<float>();
        check(inl ? api.sgd_norm_host(t, plan.blk, k, plan.blk[k], plan.border, plan.border_blk, plan.groups, norm_type, (float)clip, base, out, stream)
                  : api.sgd_norm(table, blk, k, plan.blk[k], plan.border, plan.border_blk, plan.groups, norm_type, (float)clip, base + room, out, stream),
              "lgd_sgd_norm_step");
    } else {
        check(api.sgd_clip(table, blk, k, plan.blk[k], (float)clip, stream), "lgd_sgd_clip_step");
    }
    // written through raw pointers: autograd's version counters, which the fold caches (ConvBN._frozen_fold, FrozenBatchNorm2d.scale_shift) key on and the
    // saved-tensor check reads
    for (int j = 0; j < k; ++j) {
        torch::autograd::impl::bump_version(ps[j]); torch::autograd::impl::bump_version(gs[j]); torch::autograd::impl::bump_version(ms[j]);
    }
    return Sgd::kDone;
}

// ------------------------------------------------------------------------------------------- Python
// bind(error class, address of every entry point in the order of `api`)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    constexpr int kEntries = 11;
    if (n != 1 + kEntries) { PyErr_SetString(PyExc_TypeError, "bind(error, addresses of the entry points)"); return nullptr; }
    void* p[kEntries];
    for (int i = 0; i < kEntries; ++i) {
        p[i] = PyLong_AsVoidPtr(a[i + 1]);
        if (!p[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point"); return nullptr; }
    }
    Py_INCREF(a[0]);
    Py_XDECREF(api.error);
    api.error = a[0];
    api.gn_ws = (decltype(api.gn_ws))p[0]; api.gn_fwd = (decltype(api.gn_fwd))p[1]; api.gn_bwd = (decltype(api.gn_bwd))p[2];
    api.norm_ws = (decltype(api.norm_ws))p[3]; api.norm = (decltype(api.norm))p[4]; api.clip = (decltype(api.clip))p[5];
    api.sgd_clip = (decltype(api.sgd_clip))p[6]; api.sgd_norm_ws = (decltype(api.sgd_norm_ws))p[7]; api.sgd_norm = (decltype(api.sgd_norm))p[8];
    api.sgd_norm_host = (decltype(api.sgd_norm_host))p[9]; api.last_error = (decltype(api.last_error))p[10];
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

bool opt_tensor(PyObject* o, Tensor& t, const char* what) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s must be a tensor or None, got %s", what, Py_TYPE(o)->tp_name); return false; }
    t = THPVariable_Unpack(o);
    return true;
}

struct Fast {   // a list or tuple of any Python iterable, released at the end
    PyObject* o;
    explicit Fast(PyObject* s) : o(PySequence_Fast(s, "expected an iterable of tensors")) {}
    ~Fast() { Py_XDECREF(o); }
};

// group_norm_act(maps, groups, act code, eps, weight, bias) -> list of outputs, or None where the maps are not on a GPU
PyObject* py_group_norm_act(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) { PyErr_SetString(PyExc_TypeError, "group_norm_act takes 6 arguments"); return nullptr; }
    Fast seq(a[0]);
    if (!seq.o) return nullptr;
    const long long groups = PyLong_AsLongLong(a[1]);
    const long act = PyLong_AsLong(a[2]);
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    Tensor w, b;
    if (!opt_tensor(a[4], w, "weight") || !opt_tensor(a[5], b, "bias")) return nullptr;
    try {
        const variable_list xs = tensors_of(seq.o, false);
        if (xs.empty()) return PyList_New(0);
        gn_check(xs, groups, w, b, eps);
        if (!xs[0].is_cuda()) Py_RETURN_NONE;
        const variable_list ys = gn_act(xs, (int)groups, (int)act, eps, w, b);
        PyObject* out = PyList_New((Py_ssize_t)ys.size());
        if (!out) return nullptr;
        for (size_t i = 0; i < ys.size(); ++i) {
            PyObject* y = THPVariable_Wrap(ys[i]);
            if (!y) { Py_DECREF(out); return nullptr; }
            PyList_SET_ITEM(out, (Py_ssize_t)i, y);
        }
        return out;
    } catch (const Refused& e) {
        PyErr_SetString(api.error, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// norm(tensors, take their gradients, norm code, max_norm or None) -> 0-dim tensor; None: no tensors; False: they are not on a GPU
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) { PyErr_SetString(PyExc_TypeError, "norm takes 4 arguments"); return nullptr; }
    Fast seq(a[0]);
    if (!seq.o) return nullptr;
    const int grads = PyObject_IsTrue(a[1]);
    const long code = PyLong_AsLong(a[2]);
    const bool clip = a[3] != Py_None;
    const double max_norm = clip ? PyFloat_AsDouble(a[3]) : 0.0;
    if (PyErr_Occurred()) return nullptr;
    try {
        const std::vector<Tensor> ts = tensors_of(seq.o, grads == 1);
        if (ts.empty()) Py_RETURN_NONE;
        Tensor out = norm_of(ts, (int)code, clip, max_norm);
        if (!out.defined()) Py_RETURN_FALSE;
        if (!clip && at::GradMode::is_enabled()) {
            torch::autograd::edge_list edges;
            for (const Tensor& t : ts)
                if (t.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(t));
            if (!edges.empty()) torch::autograd::set_history(out, no_derivative("grad_norm", "derivative", std::move(edges)));
        }
        return THPVariable_Wrap(out);
    } catch (const Refused& e) {
        PyErr_SetString(api.error, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// do the optimizers' states still hold what the plan was made with?  held: parameter, its state, its momentum buffer (or None), entry by entry; compared
// as objects.  1 yes, 0 no, -1 an error is set
int state_held(PyObject* states, PyObject* held) {
    static PyObject* const key = PyUnicode_InternFromString("momentum_buffer");
    const Py_ssize_t n = PyList_GET_SIZE(held);
    Py_ssize_t k = 0;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(states); ++i) {
        PyObject* state = PyList_GET_ITEM(states, i);
        if (!PyDict_Check(state)) { PyErr_SetString(PyExc_TypeError, "an optimizer's state must be a dict"); return -1; }
        PyObject *p, *entry;
        for (Py_ssize_t at = 0; PyDict_Next(state, &at, &p, &entry); k += 3) {
            if (k + 3 > n || PyList_GET_ITEM(held, k) != p || PyList_GET_ITEM(held, k + 1) != entry) return 0;
            if (!PyDict_Check(entry)) { PyErr_SetString(PyExc_TypeError, "a parameter's optimizer state must be a dict"); return -1; }
            PyObject* m = PyDict_GetItemWithError(entry, key);
            if (!m && PyErr_Occurred()) return -1;
            if (PyList_GET_ITEM(held, k + 2) != (m ? m : Py_None)) return 0;
        }
    }
    return k == n;
}

// sgd_step(parameters, momentum buffers, plan, [lr, weight decay, momentum] of every set, norm code or None, clip, the optimizers' states, what they held
// when the plan was made) -> the norms (by value: True); None: the parameters that have a gradient, or the states, are not the plan's; False: they are
// not on a GPU.  Lists of tensors (None where a parameter has no row); plan: six bytes objects in the order of SgdPlan
PyObject* py_sgd_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !PyList_Check(a[0]) || !PyList_Check(a[1]) || PyList_GET_SIZE(a[0]) != PyList_GET_SIZE(a[1]) || !PyTuple_Check(a[2]) ||
        PyTuple_GET_SIZE(a[2]) != 6 || !PyList_Check(a[3]) || !PyList_Check(a[6]) || !PyList_Check(a[7])) {
        PyErr_SetString(PyExc_TypeError, "sgd_step(list, list, plan, list, norm code, clip, list, list)");
        return nullptr;
    }
    const int same = state_held(a[6], a[7]);
    if (same < 0) return nullptr;
    if (!same) Py_RETURN_NONE;
    const void* part[6];
    Py_ssize_t size[6];
    for (int i = 0; i < 6; ++i) {
        PyObject* b = PyTuple_GET_ITEM(a[2], i);
        if (!PyBytes_Check(b)) { PyErr_SetString(PyExc_TypeError, "a plan holds bytes"); return nullptr; }
        part[i] = PyBytes_AS_STRING(b); size[i] = PyBytes_GET_SIZE(b);
    }
    const auto ints = [&](int i) { return static_cast<const int32_t*>(part[i]); };
    const SgdPlan plan = {ints(0), static_cast<const lgd_sgd_tensor*>(part[1]), ints(2), ints(3), ints(4), ints(5), (int)(size[0] / 4), (int)(size[4] / 4) - 1};
    std::vector<float> hyper;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[3]); ++i) hyper.push_back((float)PyFloat_AsDouble(PyList_GET_ITEM(a[3], i)));
    const bool by_norm = a[4] != Py_None;
    const long code = by_norm ? PyLong_AsLong(a[4]) : 0;
    const double clip = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) return nullptr;
    bool fits = plan.k > 0 && size[1] == (Py_ssize_t)(plan.k * sizeof(lgd_sgd_tensor)) && size[2] == 4 * (plan.k + 1) && size[3] == 4 * plan.k &&
                plan.groups > 0 && size[5] == size[4];
    for (Py_ssize_t i = 0; fits && i < PyList_GET_SIZE(a[0]); ++i) fits = THPVariable_Check(PyList_GET_ITEM(a[0], i));
    for (int j = 0; fits && j < plan.k; ++j) {
        const Py_ssize_t i = plan.rows[j];
        fits = i >= 0 && i < PyList_GET_SIZE(a[0]) && THPVariable_Check(PyList_GET_ITEM(a[1], i)) && plan.set[j] >= 0 &&
               3 * (size_t)plan.set[j] + 3 <= hyper.size() && plan.table[j].n == THPVariable_Unpack(PyList_GET_ITEM(a[0], i)).numel() &&
               plan.table[j].n == THPVariable_Unpack(PyList_GET_ITEM(a[1], i)).numel();
    }
    if (!fits) { PyErr_SetString(PyExc_ValueError, "the plan does not fit the lists"); return nullptr; }
    try {
        Tensor norms;
        switch (sgd_step(a[0], a[1], plan, hyper, by_norm, (int)code, clip, norms)) {
            case Sgd::kOtherSet: Py_RETURN_NONE;
            case Sgd::kNotGpu: Py_RETURN_FALSE;
            default: break;
        }
        if (!by_norm) Py_RETURN_TRUE;
        return THPVariable_Wrap(norms);
    } catch (const Refused& e) {
        PyErr_SetString(api.error, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)())py_bind, METH_FASTCALL, nullptr},
                         {"group_norm_act", (PyCFunction)(void (*)())py_group_norm_act, METH_FASTCALL, nullptr},
                         {"norm", (PyCFunction)(void (*)())py_norm, METH_FASTCALL, nullptr},
                         {"sgd_step", (PyCFunction)(void (*)())py_sgd_step, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lgd_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lgd_host(void) { return PyModule_Create(&module); }
