// The calls of marius_amd.hip on the encoder block's entry points (residual norm, neighbour attention, AdamW over many tensors): argument checks, outputs,
// workspaces and descriptors.  They are here and not in Python because that is where a small call's time goes: the checks and ctypes conversions of one norm took
// 15 us in Python, the kernel of 64 rows takes 4.
//
// Every function takes the address of the C entry point it calls (and of its workspace query) from marius_amd.hip, which is the one place that loads the kernel
// library; launches go to the current stream of the tensors' device, with that device current.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <sstream>

#include "marius_hip.h"

namespace py = pybind11;

namespace marius_amd {
namespace {

using Tensor = at::Tensor;
using MaybeTensor = std::optional<at::Tensor>;

[[noreturn]] void refuse(const std::string& message) {
    py::object error = py::module_::import("marius_amd.hip").attr("MariusHipError");
    PyErr_SetString(error.ptr(), message.c_str());
    throw py::error_already_set();
}
template <typename... A>
void require(bool ok, const A&... parts) {
    if (ok) return;
    std::ostringstream o;
    (o << ... << parts);
    refuse(o.str());
}
void check(int rc, const char* what) {
    if (rc != 0) py::module_::import("marius_amd.hip").attr("check")(rc, what);  // raises with the library's message
}
int type_of(const char* name, const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MARIUS_F32;
        case at::kBFloat16: return MARIUS_BF16;
        case at::kHalf: return MARIUS_F16;
        default: require(false, name, ": float32, bfloat16 or float16 required, got ", t.scalar_type()); return -1;
    }
}
void same_device(const at::Device& device, const char* name, const MaybeTensor& t) {
    if (t) require(t->device() == device, name, " is on ", t->device(), ", the call is on ", device);
}
void* data(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }
marius_stream_t stream_of(const at::Device& device) {
    return device.is_cuda() ? (marius_stream_t)c10::hip::getCurrentHIPStream(device.index()).stream() : nullptr;
}
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }

// rows [n, d] of contiguous elements that do not overlap (a copy where `t` is not laid out so) and their stride
struct Rows {
    Tensor t;
    int64_t ld = 0;
    Rows() = default;
    explicit Rows(const Tensor& given) : t(given) {
        const int64_t n = t.size(0), d = t.size(1);
        if ((d > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < d)) t = t.contiguous();
        ld = std::max(t.stride(0), d);
    }
    explicit Rows(const MaybeTensor& given) : Rows(given ? Rows(*given) : Rows()) {}
    void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

// ---------------------------------------------------------------------------------------------------------------- residual norm
struct NormCall {
    marius_residual_norm m{};
    Tensor keep[5];
    Rows gate;
};
void norm_call(NormCall& c, const Tensor& x, const MaybeTensor& block, const MaybeTensor& gate, const MaybeTensor (&weights)[4], bool post_norm, bool pre_norm,
               const std::string& kind, double eps, double residual_scale, const std::string& activation) {
    static const char* const names[] = {"post_weight", "post_bias", "pre_weight", "pre_bias"};
    require(x.dim() == 2, "residual_norm: rows [n, d] required, got ", x.sizes());
    const int64_t n = x.size(0), d = x.size(1);
    const at::Device device = x.device();
    marius_residual_norm& m = c.m;
    m.n = n;
    m.kind = kind == "RMS" ? MARIUS_NORM_RMS : kind == "LAYER" ? MARIUS_NORM_LAYER : -1;
    require(m.kind >= 0, "residual_norm: kind is one of RMS, LAYER");
    m.gate_activation = activation == "NONE" ? MARIUS_ACT_NONE : activation == "RELU" ? MARIUS_ACT_RELU : activation == "SIGMOID" ? MARIUS_ACT_SIGMOID : -1;
    require(m.gate_activation >= 0, "Unsupported activation function");
    require((d >= 1 || n == 0) && d <= 8192, "residual_norm: rows of 1 to 8192 elements, got ", d);
    require(eps >= 0, "residual_norm: eps must not be negative");
    m.d = (int32_t)d;
    m.stream_type = m.type = type_of("stream", x);
    m.has_block = block.has_value();
    if (block) {
        require(block->sizes() == x.sizes(), "residual_norm: block and stream differ in shape");
        m.type = type_of("block", *block);
        require(m.stream_type == m.type || m.stream_type == MARIUS_F32, "residual_norm: the stream is float32 or of the block's type (", block->scalar_type(), ")");
        same_device(device, "block", block);
    } else {
        require(pre_norm, "residual_norm: neither a block nor a norm: nothing to compute");
        require(!post_norm && !gate, "residual_norm: a post norm and a gate need a block");
        require(residual_scale == 1.0, "residual_norm: a residual scale needs a block");
    }
    m.post_norm = post_norm;
    m.pre_norm = pre_norm;
    m.eps = (float)eps;
    m.residual_scale = (float)residual_scale;
    int param = -1;
    const void** slots[] = {&m.post_weight, &m.post_bias, &m.pre_weight, &m.pre_bias};
    auto add_param = [&](const Tensor& t) {
        const int type = type_of("weights", t);
        require(param < 0 || param == type, "residual_norm: weights, biases and a channel gate are of one type");
        param = type;
    };
    for (int i = 0; i < 4; ++i) {
        if (!weights[i]) continue;
        require(i < 2 ? post_norm : pre_norm, "residual_norm: ", names[i], " of a norm that is not there");
        require(weights[i]->dim() == 1 && weights[i]->size(0) == d, "residual_norm: ", names[i], " has shape ", weights[i]->sizes(), ", rows have ", d, " elements");
        same_device(device, names[i], weights[i]);
        add_param(*weights[i]);
        c.keep[i] = weights[i]->contiguous();
        *slots[i] = c.keep[i].data_ptr();
    }
    if (gate) {
        same_device(device, "gate", gate);
        if (gate->dim() == 1 && gate->size(0) == d) {
            add_param(*gate);
            c.keep[4] = gate->contiguous();
            m.gate_mode = MARIUS_GATE_CHANNEL;
            m.gate = c.keep[4].data_ptr();
        } else {
            require(gate->sizes() == x.sizes(), "residual_norm: gate is [d] or [n, d], got ", gate->sizes());
            require(gate->scalar_type() == block->scalar_type(), "residual_norm: an element gate is of the block's type, got ", gate->scalar_type());
            c.gate = Rows(*gate);
            m.gate_mode = MARIUS_GATE_ELEMENT;
            m.gate = c.gate.ptr();
            m.gate_ld = c.gate.ld;
        }
    }
    m.param_type = param < 0 ? MARIUS_F32 : param;
}

std::pair<Tensor, MaybeTensor> residual_norm(uintptr_t entry, const Tensor& x, const MaybeTensor& block, const MaybeTensor& gate, const MaybeTensor& post_weight,
                                             const MaybeTensor& post_bias, const MaybeTensor& pre_weight, const MaybeTensor& pre_bias, bool post_norm, bool pre_norm,
                                             const std::string& kind, double eps, double residual_scale, const std::string& activation) {
    const MaybeTensor weights[4] = {post_weight, post_bias, pre_weight, pre_bias};
    NormCall c;
    norm_call(c, x, block, gate, weights, post_norm, pre_norm, kind, eps, residual_scale, activation);
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t d = x.size(1);
    Tensor y = block ? at::empty(x.sizes(), x.options()) : x;
    MaybeTensor h;
    if (pre_norm) h = at::empty(x.sizes(), (block ? *block : x).options());
    if (x.numel() == 0) return {y, h};
    const Rows xr(x), br(block);
    check(((decltype(&marius_residual_norm_forward))entry)(&c.m, xr.ptr(), xr.ld, br.ptr(), br.ld, block ? y.data_ptr() : nullptr, d, data(h), d, stream_of(x.device())),
          "residual_norm");
    return {y, h};
}

py::dict residual_norm_backward(uintptr_t entry, uintptr_t workspace_entry, const MaybeTensor& grad_y, const MaybeTensor& grad_h, const Tensor& y, const MaybeTensor& block,
                                const MaybeTensor& gate, const MaybeTensor& post_weight, const MaybeTensor& post_bias, const MaybeTensor& pre_weight, const MaybeTensor& pre_bias,
                                bool post_norm, bool pre_norm, const std::string& kind, double eps, double residual_scale, const std::string& activation, bool need_dx) {
    const MaybeTensor weights[4] = {post_weight, post_bias, pre_weight, pre_bias};
    NormCall c;
    norm_call(c, y, block, gate, weights, post_norm, pre_norm, kind, eps, residual_scale, activation);
    const Tensor& like = block ? *block : y;
    same_device(y.device(), "grad_y", grad_y);
    same_device(y.device(), "grad_h", grad_h);
    require(!grad_y || (grad_y->sizes() == y.sizes() && grad_y->scalar_type() == y.scalar_type()), "residual_norm_backward: grad_y is not like y");
    require(!grad_h || (pre_norm && grad_h->sizes() == y.sizes() && grad_h->scalar_type() == like.scalar_type()), "residual_norm_backward: grad_h is not like h");
    require(grad_y || grad_h, "residual_norm_backward: no gradient to go back from");
    const c10::OptionalDeviceGuard guard(y.device());
    const int64_t n = y.size(0), d = y.size(1);
    auto fresh = [](const MaybeTensor& t) -> MaybeTensor { return t ? MaybeTensor(at::empty(t->sizes(), t->options())) : MaybeTensor(); };
    MaybeTensor dx, dblock = fresh(block), dgate = fresh(gate), dw[4];
    if (need_dx) dx = at::empty(y.sizes(), y.options());
    for (int i = 0; i < 4; ++i) dw[i] = fresh(weights[i]);
    if (d > 0) {
        const Rows yr(y), br(block), gy(grad_y), gh(grad_h);
        marius_residual_norm_grads g{gy.ptr(), gh.ptr(), gy.ld, gh.ld, data(dx), data(dblock), data(dgate), d, d, d, data(dw[0]), data(dw[1]), data(dw[2]), data(dw[3])};
        const bool sums = c.m.gate_mode == MARIUS_GATE_CHANNEL || dw[0] || dw[1] || dw[2] || dw[3];
        const size_t need = sums ? ((decltype(&marius_residual_norm_workspace_bytes))workspace_entry)(n, (int32_t)d) : 0;
        const Tensor ws = need ? bytes(need, y) : Tensor();
        check(((decltype(&marius_residual_norm_backward))entry)(&c.m, &g, yr.ptr(), yr.ld, br.ptr(), br.ld, need ? ws.data_ptr() : nullptr, need, stream_of(y.device())),
              "residual_norm_backward");
    }
    py::dict got;
    got["dx"] = dx;
    got["dblock"] = dblock;
    got["dgate"] = dgate;
    got["dpost_weight"] = dw[0];
    got["dpost_bias"] = dw[1];
    got["dpre_weight"] = dw[2];
    got["dpre_bias"] = dw[3];
    return got;
}

// ---------------------------------------------------------------------------------------------------------------- neighbour attention
// [n, heads, dim] with contiguous heads (a copy where they are not) and its strides
struct Heads {
    Tensor t;
    int64_t row, head;
    explicit Heads(const Tensor& given) : t(given) {
        if (t.stride(2) != 1 && t.size(2) > 1) t = t.contiguous();
        row = t.size(0) > 1 ? t.stride(0) : 0;  // (of a single row or head: whatever a view left there)
        head = t.size(1) > 1 ? t.stride(1) : 0;
    }
};
struct AttentionCall {
    const marius_neighbor_plan* plan;
    marius_neighbor_attention m{};
    Tensor q, k, v, bias;
};
void attention_call(AttentionCall& c, uintptr_t plan, const Tensor& plan_index, const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scale, const MaybeTensor& bias) {
    c.plan = (const marius_neighbor_plan*)plan;
    const at::Device device = q.device();
    same_device(device, "k", k);
    same_device(device, "v", v);
    same_device(device, "the plan", plan_index);
    require(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes(), "neighbor_attention: q [n, heads, dim] and k, v [rows, kv_heads, dim] required");
    const int64_t n = q.size(0), heads = q.size(1), dim = q.size(2), rows = k.size(0), kv_heads = k.size(1);
    require(n == c.plan->n && rows == c.plan->rows, "neighbor_attention: the plan has ", c.plan->n, " targets over ", c.plan->rows, " rows, got ", n, " and ", rows);
    require(k.size(2) == dim && dim >= 1 && dim <= 256, "neighbor_attention: heads of 1 to 256 elements, the same in q, k and v");
    require(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 1024, "neighbor_attention: query heads (up to 1024) are a multiple of the key heads");
    require(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "neighbor_attention: q, k and v are of one type");
    marius_neighbor_attention& m = c.m;
    m.type = type_of("q", q);
    m.heads = (int32_t)heads;
    m.kv_heads = (int32_t)kv_heads;
    m.dim = (int32_t)dim;
    m.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)dim));
    const Heads hq(q), hk(k), hv(v);
    c.q = hq.t;
    c.k = hk.t;
    c.v = hv.t;
    m.q = c.q.data_ptr();
    m.k = c.k.data_ptr();
    m.v = c.v.data_ptr();
    m.q_row = hq.row;
    m.q_head = hq.head;
    m.k_row = hk.row;
    m.k_head = hk.head;
    m.v_row = hv.row;
    m.v_head = hv.head;
    if (bias) {
        require(bias->dim() == 2 && bias->size(0) == c.plan->T && bias->size(1) == heads && bias->scalar_type() == at::kFloat, "neighbor_attention: bias is float32 [", c.plan->T, ", ",
                heads, "]");
        same_device(device, "bias", bias);
        c.bias = bias->contiguous();
        m.bias = (const float*)c.bias.data_ptr();
    }
}
std::tuple<Tensor, Tensor, MaybeTensor> neighbor_attention(uintptr_t entry, uintptr_t workspace_entry, uintptr_t plan, const Tensor& plan_index, const Tensor& q, const Tensor& k,
                                                           const Tensor& v, std::optional<double> scale, const MaybeTensor& bias, bool return_lse) {
    AttentionCall c;
    attention_call(c, plan, plan_index, q, k, v, scale, bias);
    const c10::OptionalDeviceGuard guard(q.device());
    Tensor out = at::empty(q.sizes(), q.options()), stats = at::empty({q.size(0), q.size(1), 2}, q.options().dtype(at::kFloat));
    c.m.stats = (float*)stats.data_ptr();
    MaybeTensor lse;
    if (return_lse) lse = at::empty({q.size(0), q.size(1)}, stats.options());
    c.m.lse = (float*)data(lse);
    const size_t need = ((decltype(&marius_neighbor_attention_workspace_bytes))workspace_entry)(c.plan, c.m.heads, c.m.kv_heads, c.m.dim, 0);
    const Tensor ws = need ? bytes(need, q) : Tensor();
    check(((decltype(&marius_neighbor_attention_forward))entry)(c.plan, &c.m, out.data_ptr(), need ? ws.data_ptr() : nullptr, need, stream_of(q.device())), "neighbor_attention");
    return {out, stats, lse};
}
std::tuple<Tensor, Tensor, Tensor, MaybeTensor> neighbor_attention_backward(uintptr_t entry, uintptr_t workspace_entry, uintptr_t plan, const Tensor& plan_index, const Tensor& grad_out,
                                                                            const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& stats, std::optional<double> scale,
                                                                            const MaybeTensor& bias, bool need_dbias) {
    AttentionCall c;
    attention_call(c, plan, plan_index, q, k, v, scale, bias);
    same_device(q.device(), "grad_out", grad_out);
    same_device(q.device(), "stats", stats);
    require(grad_out.sizes() == q.sizes() && grad_out.scalar_type() == q.scalar_type(), "neighbor_attention_backward: grad_out is not like the output");
    require(stats.dim() == 3 && stats.size(0) == q.size(0) && stats.size(1) == q.size(1) && stats.size(2) == 2 && stats.scalar_type() == at::kFloat,
            "neighbor_attention_backward: stats is float32 [", q.size(0), ", ", q.size(1), ", 2]");
    const c10::OptionalDeviceGuard guard(q.device());
    const Heads g(grad_out);
    const Tensor st = stats.contiguous();
    c.m.stats = (float*)st.data_ptr();
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
    MaybeTensor dbias;
    if (bias && need_dbias) dbias = at::empty(bias->sizes(), bias->options());
    const size_t need = ((decltype(&marius_neighbor_attention_workspace_bytes))workspace_entry)(c.plan, c.m.heads, c.m.kv_heads, c.m.dim, 1);
    const Tensor ws = need ? bytes(need, q) : Tensor();
    check(((decltype(&marius_neighbor_attention_backward))entry)(c.plan, &c.m, g.t.data_ptr(), g.row, g.head, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), (float*)data(dbias),
                                                                 need ? ws.data_ptr() : nullptr, need, stream_of(q.device())),
          "neighbor_attention_backward");
    return {dq, dk, dv, dbias};
}

// ---------------------------------------------------------------------------------------------------------------- AdamW
// The tensors of an optimizer: parameters and states.  Both may be given new memory between steps: their addresses are read at every one, and looked over when one has changed.
struct AdamWTensors {
    std::vector<Tensor> params;
    std::vector<std::vector<Tensor>> states;  // exp_avg, exp_avg_sq (, their scales)
    std::vector<marius_adamw_tensor> table;
    std::vector<const void*> seen;            // the parameters' addresses when they were looked over
    int type = 0, bits = 32;
    at::Device device = at::kCPU;

    AdamWTensors(std::vector<Tensor> p, std::vector<Tensor> m, std::vector<Tensor> v, std::optional<std::vector<Tensor>> ms, std::optional<std::vector<Tensor>> vs)
        : params(std::move(p)) {
        require(!params.empty(), "AdamWTensors: no parameters");
        require(ms.has_value() == vs.has_value(), "AdamWTensors: lists of different lengths");
        bits = ms ? 8 : 32;
        states = {std::move(m), std::move(v)};
        if (ms) {
            states.push_back(std::move(*ms));
            states.push_back(std::move(*vs));
        }
        for (const auto& s : states) require(s.size() == params.size(), "AdamWTensors: lists of different lengths");
        type = type_of("parameters", params[0]);
        device = params[0].device();
        table.resize(params.size());
        for (size_t i = 0; i < params.size(); ++i) {
            const Tensor& w = params[i];
            require(w.scalar_type() == params[0].scalar_type() && w.is_contiguous(), "AdamWTensors: parameter ", i, " is not a contiguous ", params[0].scalar_type(), " tensor");
            require(w.device() == device, "AdamWTensors: tensors of parameter ", i, " are contiguous and on ", device);
            table[i].n = w.numel();
        }
        seen.resize(params.size());
        for (size_t i = 0; i < params.size(); ++i) look_at_states(i);
        look_for_overlaps();
    }
    // what a step writes besides the parameters, as it is now
    void look_at_states(size_t i) {
        marius_adamw_tensor& t = table[i];
        for (size_t k = 0; k < states.size(); ++k) {
            const Tensor& s = states[k][i];
            require(s.device() == device && s.is_contiguous(), "AdamWTensors: tensors of parameter ", i, " are contiguous and on ", device);
            if (k < 2)
                require(s.numel() == t.n && s.scalar_type() == (bits == 32 ? at::kFloat : at::kFloat8_e4m3fn), "AdamWTensors: states of parameter ", i, " are ",
                        bits == 32 ? "float32" : "float8_e4m3fn", " of its size");
            else
                require(s.scalar_type() == at::kFloat && s.numel() == (t.n + 255) / 256, "AdamWTensors: scales of parameter ", i, " are float32, one for 256");
        }
        t.exp_avg = states[0][i].data_ptr();
        t.exp_avg_sq = states[1][i].data_ptr();
        t.exp_avg_scale = bits == 8 ? (float*)states[2][i].data_ptr() : nullptr;
        t.exp_avg_sq_scale = bits == 8 ? (float*)states[3][i].data_ptr() : nullptr;
    }
    // no tensor twice, none inside another: every launch updates all of them at once
    void look_for_overlaps() {
        std::vector<std::pair<const char*, const char*>> spans;
        auto span = [&](const Tensor& t) {
            if (t.numel() > 0) spans.emplace_back((const char*)t.data_ptr(), (const char*)t.data_ptr() + t.nbytes());
        };
        for (const Tensor& w : params) span(w);
        for (const auto& s : states)
            for (const Tensor& t : s) span(t);
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i) require(spans[i - 1].second <= spans[i].first, "AdamWTensors: a tensor appears twice, or overlaps another");
        for (size_t i = 0; i < params.size(); ++i) seen[i] = params[i].data_ptr();
    }
    void refresh() {
        bool moved = false;
        for (size_t i = 0; i < params.size(); ++i) {
            const marius_adamw_tensor& t = table[i];
            bool same = states[0][i].data_ptr() == t.exp_avg && states[1][i].data_ptr() == t.exp_avg_sq && states[0][i].numel() == t.n && states[1][i].numel() == t.n;
            if (bits == 8) same = same && states[2][i].data_ptr() == t.exp_avg_scale && states[3][i].data_ptr() == t.exp_avg_sq_scale;
            if (!same) {
                seen[i] = nullptr;  // (looked over again next time, too, if this is refused)
                look_at_states(i);
            }
            moved = moved || !same || params[i].data_ptr() != seen[i];
        }
        if (moved) look_for_overlaps();
    }
};
// A step's arguments, checked; nothing is launched and nothing changes until they are used.  `step`: an int or an int64 device tensor (of one number, or one for each parameter)
struct AdamWCall {
    std::vector<marius_adamw_tensor> table;
    std::vector<size_t> strided;  // gradients that are not contiguous
    MaybeTensor counter;
    int64_t step = 0;
    int grad_type = -1;           // -1: no gradient at all
    int32_t steps() const { return counter ? (int32_t)counter->numel() : 1; }
};
AdamWCall adamw_call(uintptr_t check_entry, AdamWTensors& a, const std::vector<MaybeTensor>& grads, const py::object& step, double lr, double beta1, double beta2, double eps,
                     double weight_decay, const MaybeTensor& grad_scale, bool capturing) {
    const size_t count = a.params.size();
    require(grads.size() == count, "adamw_step: ", grads.size(), " gradients for ", count, " parameters");
    const at::Device device = a.device;
    AdamWCall c;
    a.refresh();
    c.table = a.table;  // (a copy: two threads may step at once)
    std::optional<at::ScalarType> kind;
    for (size_t i = 0; i < count; ++i) {
        marius_adamw_tensor& t = c.table[i];
        if (!grads[i]) {
            t.n = 0;
            continue;
        }
        const Tensor &g = *grads[i], &w = a.params[i];
        require(g.layout() == at::kStrided, "adamw_step: gradient ", i, " is not a dense tensor");
        if (!kind) kind = g.scalar_type();
        require(g.scalar_type() == *kind && g.device() == device && g.numel() == t.n, "adamw_step: gradient ", i, " is not a ", *kind, " tensor of ", t.n, " elements on ", device);
        require(w.device() == device && w.scalar_type() == a.params[0].scalar_type() && w.numel() == t.n && w.is_contiguous(), "adamw_step: parameter ", i,
                " is no longer what the states were made for");
        t.param = w.data_ptr();
        t.grad = g.data_ptr();
        if (!g.is_contiguous()) c.strided.push_back(i);
    }
    const bool on_device = THPVariable_Check(step.ptr());
    if (on_device) {
        c.counter = THPVariable_Unpack(step.ptr());
        require(c.counter->scalar_type() == at::kLong && (c.counter->numel() == 1 || c.counter->numel() == (int64_t)count) && c.counter->is_contiguous() && c.counter->device() == device,
                "adamw_step: a step on the device is one int64, or one for each parameter, on ", device);
    } else {
        c.step = step.cast<int64_t>();
    }
    require(!grad_scale || (grad_scale->scalar_type() == at::kFloat && grad_scale->numel() == 1 && grad_scale->device() == device), "adamw_step: grad_scale is one float32 on ", device);
    require(on_device || !capturing, "adamw_step: a captured step needs its number on the device (a replay would repeat this one's)");
    if (!kind) return c;
    require(*kind == at::kFloat || *kind == at::kBFloat16 || *kind == at::kHalf, "adamw_step: float32, bfloat16 or float16 gradients required, got ", *kind);
    c.grad_type = *kind == at::kFloat ? MARIUS_F32 : *kind == at::kBFloat16 ? MARIUS_BF16 : MARIUS_F16;
    if (check_entry)  // (marius_adamw_step makes these checks itself, before it launches)
        check(((decltype(&marius_adamw_check))check_entry)(c.table.data(), (int32_t)count, a.type, c.grad_type, a.bits, c.step, (const int64_t*)data(c.counter), c.steps(), lr,
                                                           beta1, beta2, eps, weight_decay),
              "adamw_step");
    return c;
}
void adamw_check(uintptr_t check_entry, AdamWTensors& a, const std::vector<MaybeTensor>& grads, const py::object& step, double lr, double beta1, double beta2, double eps,
                 double weight_decay, const MaybeTensor& grad_scale, bool capturing) {
    adamw_call(check_entry, a, grads, step, lr, beta1, beta2, eps, weight_decay, grad_scale, capturing);
}
void adamw_step(uintptr_t entry, uintptr_t workspace_entry, AdamWTensors& a, const std::vector<MaybeTensor>& grads, const py::object& step, double lr, double beta1,
                double beta2, double eps, double weight_decay, const MaybeTensor& grad_scale, bool capturing) {
    AdamWCall c = adamw_call(0, a, grads, step, lr, beta1, beta2, eps, weight_decay, grad_scale, capturing);
    if (c.grad_type < 0) return;
    const size_t count = a.params.size();
    const at::Device device = a.device;
    const c10::OptionalDeviceGuard guard(device);
    std::vector<Tensor> copies;
    for (size_t i : c.strided) {
        copies.push_back(grads[i]->contiguous());
        c.table[i].grad = copies.back().data_ptr();
    }
    const size_t need = ((decltype(&marius_adamw_workspace_bytes))workspace_entry)((int32_t)count);
    const Tensor ws = need ? bytes(need, a.states[0][0]) : Tensor();
    check(((decltype(&marius_adamw_step))entry)(c.table.data(), (int32_t)count, a.type, c.grad_type, a.bits, c.step, (const int64_t*)data(c.counter), c.steps(), lr, beta1, beta2, eps,
                                                weight_decay, (const float*)data(grad_scale), need ? ws.data_ptr() : nullptr, need, stream_of(device)),
          "adamw_step");
    for (size_t i = 0; i < count; ++i)  // a graph that saved the old values may not go back through the new ones
        if (grads[i] && !a.params[i].is_inference()) a.params[i].unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void bind_encoder_ops(py::module_& m) {
    m.def("residual_norm", &residual_norm);
    m.def("residual_norm_backward", &residual_norm_backward);
    m.def("neighbor_attention", &neighbor_attention);
    m.def("neighbor_attention_backward", &neighbor_attention_backward);
    py::class_<AdamWTensors>(m, "AdamWTensors")
        .def(py::init<std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, std::optional<std::vector<Tensor>>, std::optional<std::vector<Tensor>>>())
        .def_property_readonly("device", [](const AdamWTensors& a) { return a.device; })
        .def_readonly("params", &AdamWTensors::params);
    m.def("adamw_check", &adamw_check);
    m.def("adamw_step", &adamw_step);
}

}  // namespace marius_amd
