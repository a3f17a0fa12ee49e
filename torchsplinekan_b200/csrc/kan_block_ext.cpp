// PyTorch operators around a KAN layer: the norm in front of it, the gated residual connection behind it, and 8-bit
// checkpoints (kanb200_block_forward / _backward, kanb200_pack_activation / _unpack_activation).
//
// As in kan_torch_ext.cpp everything numerical of the native path happens behind the C ABI; this file validates,
// allocates outputs and scratch from the caching allocator (per call, so that calls on several streams and captured
// graphs share nothing), passes raw pointers and the current stream, and keeps the autograd bookkeeping.  The
// composite formulas serve CPU tensors and backward passes that are themselves recorded (create_graph=True).
#include <ATen/TensorUtils.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <array>
#include <cmath>
#include <functional>
#include <optional>
#include <tuple>
#include <vector>

#include "kan_ext_util.h"

namespace kan_ext {
namespace {

namespace py = pybind11;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

int stream_code(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return KANB200_F32;
        case at::kDouble: return KANB200_F64;
        case at::kHalf: return KANB200_F16;
        case at::kBFloat16: return KANB200_BF16;
        default:
            TORCH_CHECK(false, what, ": x must be float32, float64, float16 or bfloat16, got ", t.scalar_type());
    }
}
at::ScalarType branch_type(const Tensor& x) { return x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

// A tensor as rows with one stride: its own memory where the layout allows, a contiguous copy otherwise.
struct Rows {
    Tensor keep;
    int64_t stride = 0;
    const void* ptr() const { return keep.defined() ? keep.data_ptr() : nullptr; }
};
// A dense copy of a vector where it is not its own memory already.  (Memory says nothing of a view that negates lazily, such
// as the imaginary part of a conjugate.)
Tensor own_sign(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return t.defined() ? own_sign(t).contiguous() : t; }
Rows as_rows(const Tensor& given, int64_t rows, int64_t width) {
    if (!given.defined()) return {};
    const Tensor t = own_sign(given);
    const int64_t shape[2] = {rows, width};
    const auto strides = at::detail::computeStride(t.sizes(), t.strides(), at::IntArrayRef(shape, 2));
    if (strides && ((*strides)[1] == 1 || width == 1) && ((*strides)[0] >= 0)) return {t, (*strides)[0]};
    return {t.contiguous(), width};
}

void check_vector(const Tensor& t, const char* what, const char* name, int64_t width, at::ScalarType type,
                  const Tensor& x) {
    if (!t.defined()) return;
    TORCH_CHECK(t.dim() == 1 && t.size(0) == width, what, ": ", name, " must have shape [", width, "], got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == type, what, ": ", name, " must be ", type, " next to ", x.scalar_type(), " x, got ",
                t.scalar_type());
    TORCH_CHECK(t.device() == x.device(), what, ": ", name, " must be on x's device");
}

void check_settings(const char* what, const Tensor& x, double eps, int64_t checkpoint) {
    const double least = branch_type(x) == at::kDouble ? 2.2250738585072014e-308 : 1.17549435e-38;
    TORCH_CHECK(eps >= least && std::isfinite(eps), what, ": eps must be a positive normal number of the branch's type, got ",
                eps);
    TORCH_CHECK(checkpoint >= KANB200_PACK_NONE && checkpoint <= KANB200_PACK_E4M3, what, ": unknown checkpoint format");
}

// The native path reads memory: no tensors that stand for others (fake tensors, torch.func transforms, vmap, subclasses).
void check_memory(const char* what, std::initializer_list<std::reference_wrapper<const Tensor>> ts) {
    const c10::DispatchKeySet stands_in({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchGradWrapper});
    for (const Tensor& t : ts)
        TORCH_CHECK(!t.defined() || !t.key_set().has_any(stands_in), what,
                    ": fake tensors, tensor subclasses and torch.func transforms are not available on CUDA");
}

int64_t row_count(const Tensor& x) {
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < x.dim(); ++d) n *= x.size(d);
    return n;
}

// New memory from the caching allocator, past the dispatcher (a third of the time of at::empty; a training call of a few
// rows makes about ten).
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

int64_t group_count(int64_t width) { return (width + KANB200_PACK_GROUP - 1) / KANB200_PACK_GROUP; }

// What the forward leaves for the backward besides its inputs, in one piece of memory: the norms' statistics, and the codes and
// scales of y, of a gate per row and of the last norm's input.
struct Record {
    bool post = false, next = false, y = false, gate = false, x = false;

    // its size; with `base`, the places of its parts
    int64_t lay(kanb200_block_args& a, char* base) const {
        const int64_t value = a.dtype == KANB200_F64 ? 8 : 4;
        int64_t at = 0;
        const auto take = [&](bool there, int64_t bytes, void*& to) {
            if (!there) return;
            if (base) to = base + at;
            at += (bytes + 255) / 256 * 256;
        };
        take(post, 2 * a.rows * value, a.post_stats);
        take(next, 2 * a.rows * value, a.next_stats);
        const auto codes = [&](bool there, void*& c, void*& s) {
            take(there, a.rows * a.width, c);
            take(there, a.rows * group_count(a.width) * value, s);
        };
        codes(y, a.y_codes, a.y_scales);
        codes(gate, a.gate_codes, a.gate_scales);
        codes(x, a.x_codes, a.x_scales);
        return at;
    }
    Tensor make(kanb200_block_args& a, const Tensor& like) const {
        const int64_t bytes = lay(a, nullptr);
        if (bytes == 0) return Tensor();
        Tensor t = fresh({bytes}, at::kByte, like);
        lay(a, static_cast<char*>(t.data_ptr()));
        return t;
    }
    void find(kanb200_block_args& a, const Tensor& t) const {
        if (t.defined()) lay(a, static_cast<char*>(t.data_ptr()));
    }
};

void run_backward(kanb200_block_args& a, const Tensor& like, cudaStream_t st) {
    const size_t bytes = kanb200_block_backward_workspace_bytes(&a);
    Tensor ws;
    if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, like);
    check_rc(kanb200_block_backward(&a, mptr(ws), bytes, st));
}

// ------------------------------------------------------------------------------------------------
// composite formulas
// ------------------------------------------------------------------------------------------------
Tensor standardise(const Tensor& v, int64_t kind, double eps, Tensor* rstd = nullptr) {
    const Tensor c = kind == KANB200_NORM_LAYER ? v - v.mean(-1, true) : v;
    const Tensor r = (c.square().mean(-1, true) + eps).rsqrt();
    if (rstd) *rstd = r;
    return c * r;
}
Tensor affine(Tensor v, const Tensor& w, const Tensor& b) {
    if (w.defined()) v = v * w;
    if (b.defined()) v = v + b;
    return v;
}
Tensor over_rows(const Tensor& t) { return t.reshape({-1, t.size(-1)}).sum(0); }
Tensor activate(const Tensor& g, int64_t act) {
    return act == KANB200_ACT_NONE ? g : act == KANB200_ACT_SIGMOID ? at::sigmoid(g) : at::silu(g);
}
Tensor activate_grad(const Tensor& g, int64_t act) {
    if (act == KANB200_ACT_NONE) return at::ones_like(g);
    const Tensor s = at::sigmoid(g);
    return act == KANB200_ACT_SIGMOID ? s * (1.0 - s) : s * (1.0 + g * (1.0 - s));
}
// (d input, d weight, d bias) of affine(standardise(v)) for the gradient d of its value
std::tuple<Tensor, Tensor, Tensor> norm_gradient(const Tensor& v, const Tensor& w, const Tensor& d, int64_t kind,
                                                 double eps) {
    Tensor rstd;
    const Tensor vhat = standardise(v, kind, eps, &rstd), u = w.defined() ? d * w : d;
    Tensor inner = u - vhat * (u * vhat).mean(-1, true);
    if (kind == KANB200_NORM_LAYER) inner = inner - u.mean(-1, true);
    return std::make_tuple(rstd * inner, over_rows(d * vhat), over_rows(d));
}

Tensor norm_composite(const Tensor& x, const Tensor& w, const Tensor& b, int64_t kind, double eps) {
    return affine(standardise(x.to(branch_type(x)), kind, eps), w, b);
}

// ------------------------------------------------------------------------------------------------
// h = norm(x)
// ------------------------------------------------------------------------------------------------
void check_norm(const Tensor& x, const Tensor& w, const Tensor& b, int64_t kind, double eps, int64_t checkpoint) {
    const char* what = "block_norm";
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": x must have at least one column, got ", x.sizes());
    stream_code(x, what);
    TORCH_CHECK(kind == KANB200_NORM_RMS || kind == KANB200_NORM_LAYER, what, ": unknown norm");
    check_settings(what, x, eps, checkpoint);
    check_vector(w, what, "weight", x.size(-1), branch_type(x), x);
    check_vector(b, what, "bias", x.size(-1), branch_type(x), x);
}

Record norm_record(int64_t checkpoint) {
    Record r;
    r.next = true;
    r.x = checkpoint != KANB200_PACK_NONE;
    return r;
}
// `record`: where what the backward needs goes (NULL: no backward)
Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, int64_t kind, double eps, int64_t checkpoint,
                    Tensor* record) {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    Tensor h = fresh(x.sizes(), branch_type(x), x);
    kanb200_block_args a{};
    a.dtype = stream_code(x, "block_norm");
    a.rows = row_count(x);
    a.width = x.size(-1);
    a.next_norm = (int)kind;
    a.eps = eps;
    if (record) {
        a.checkpoint = (int)checkpoint;
        *record = norm_record(checkpoint).make(a, x);
    }
    const Rows xr = as_rows(x, a.rows, a.width);
    const Tensor wc = dense(w), bc = dense(b);
    a.x = xr.ptr();
    a.x_stride = xr.stride;
    a.next_weight = cptr(wc);
    a.next_bias = cptr(bc);
    a.h = h.data_ptr();
    check_rc(kanb200_block_forward(&a, st));
    return h;
}

bool wants_grad(std::initializer_list<Tensor> ts, const char* what) {
    bool wanted = false;
    for (const Tensor& t : ts) {
        if (!t.defined()) continue;
        TORCH_CHECK(!t._fw_grad(0).defined(), what, ": forward-mode derivatives are not available");
        wanted = wanted || t.requires_grad();
    }
    return wanted && at::GradMode::is_enabled();
}

// The autograd nodes are written out instead of through torch::autograd::Function: on small calls its context (a
// dictionary, generic wrapping of inputs and outputs) cost as much as the launch.
struct SavedNode : public torch::autograd::Node {
    std::vector<SavedVariable> saved;
    bool released = false;

    void keep(const Tensor& t, bool is_output = false) { saved.emplace_back(t, is_output); }
    Tensor kept(size_t i) {
        TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
        return saved[i].unpack(shared_from_this());
    }
    bool need(size_t i) const { return i < num_outputs() && task_should_compute_output(i); }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        released = true;
        for (SavedVariable& v : saved) v.reset_data();
    }
};
template <typename N> std::shared_ptr<N> new_node(std::initializer_list<Tensor> inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    edges.reserve(inputs.size());
    for (const Tensor& t : inputs)
        edges.push_back(t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
    node->set_next_edges(std::move(edges));
    return node;
}
int type_code(at::ScalarType t) {
    return t == at::kFloat ? KANB200_F32 : t == at::kDouble ? KANB200_F64 : t == at::kHalf ? KANB200_F16 : KANB200_BF16;
}

Tensor or_undefined(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

struct BlockNormNode : public SavedNode {
    int64_t kind = 0, checkpoint = 0;
    double eps = 0;
    at::ScalarType type = at::kFloat;                       // of the stream
    std::vector<int64_t> shape;
    std::string name() const override { return "BlockNormBackward"; }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(3);
        if (!grads[0].defined()) return result;
        const Tensor x = kept(0), w = kept(1), record = kept(2);
        if (at::GradMode::is_enabled()) {
            TORCH_CHECK(checkpoint == KANB200_PACK_NONE,
                        "block_norm: create_graph=True needs the input itself, not its 8-bit checkpoint");
            std::tie(result[0], result[1], result[2]) = norm_gradient(x.to(branch_type(x)), w, grads[0], kind, eps);
            result[0] = result[0].to(type);
            return result;
        }
        const Tensor& like = grads[0];
        c10::cuda::CUDAGuard guard(like.device());
        const cudaStream_t st = at::cuda::getCurrentCUDAStream();
        const at::ScalarType branch = type == at::kDouble ? at::kDouble : at::kFloat;
        kanb200_block_args a{};
        a.dtype = type_code(type);
        a.width = shape.back();
        a.rows = grads[0].numel() / a.width;
        const Rows xr = as_rows(x, a.rows, a.width), dr = as_rows(grads[0], a.rows, a.width);
        if (need(0)) result[0] = fresh(shape, type, like);
        if (need(1)) result[1] = fresh({a.width}, branch, like);
        if (need(2)) result[2] = fresh({a.width}, branch, like);
        a.next_norm = (int)kind;
        a.checkpoint = (int)checkpoint;
        a.eps = eps;
        a.x = xr.ptr();
        a.x_stride = xr.stride;
        const Tensor wc = dense(w);
        a.next_weight = cptr(wc);
        norm_record(checkpoint).find(a, record);
        a.dh = dr.ptr();
        a.dh_stride = dr.stride;
        a.dx = mptr(result[0]);
        a.dnext_weight = mptr(result[1]);
        a.dnext_bias = mptr(result[2]);
        run_backward(a, like, st);
        return result;
    }
};

Tensor block_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, int64_t kind,
                  double eps, int64_t checkpoint) {
    const Tensor w = or_undefined(weight), b = or_undefined(bias);
    check_norm(x, w, b, kind, eps, checkpoint);
    TORCH_CHECK(x.is_cuda() || checkpoint == KANB200_PACK_NONE, "block_norm: 8-bit checkpoints need CUDA tensors");
    if (!x.is_cuda() || x.numel() == 0) return norm_composite(x, w, b, kind, eps);
    check_memory("block_norm", {x, w, b});
    if (!wants_grad({x, w, b}, "block_norm")) return norm_forward(x, w, b, kind, eps, checkpoint, nullptr);
    Tensor record;
    Tensor h = norm_forward(x, w, b, kind, eps, checkpoint, &record);
    auto node = new_node<BlockNormNode>({x, w, b});
    node->kind = kind;
    node->eps = eps;
    node->checkpoint = checkpoint;
    node->type = x.scalar_type();
    node->shape = x.sizes().vec();
    node->saved.reserve(3);
    for (const Tensor& t : {checkpoint != KANB200_PACK_NONE ? Tensor() : x, w, record}) node->keep(t);
    torch::autograd::set_history(h, node);
    return h;
}

// ------------------------------------------------------------------------------------------------
// out = x + scale act(gate) post(y),  h = next(out)
// ------------------------------------------------------------------------------------------------
struct Gated {
    Tensor x, y, gate, scale, pw, pb, nw, nb;
    bool packed = false;               // y holds [value | gate] side by side
    int64_t act = 0, post = 0, next = 0, checkpoint = 0;
    double eps = 0;
    int64_t rows = 0, width = 0, gate_rows = 1;
    bool row_gate = false;             // a gate of its own for every row

    bool gated() const { return packed || gate.defined(); }
};

void check_gated(Gated& g) {
    const char* what = "gated_residual";
    const Tensor &x = g.x, &y = g.y;
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": x must have at least one column, got ", x.sizes());
    stream_code(x, what);
    check_settings(what, x, g.eps, g.checkpoint);
    TORCH_CHECK(g.act >= KANB200_ACT_NONE && g.act <= KANB200_ACT_SILU, what, ": unknown gate activation");
    for (int64_t n : {g.post, g.next})
        TORCH_CHECK(n >= KANB200_NORM_NONE && n <= KANB200_NORM_LAYER, what, ": unknown norm");
    const at::ScalarType type = branch_type(x);
    g.width = x.size(-1);
    g.rows = row_count(x);
    auto shape = x.sizes().vec();
    if (g.packed) shape.back() *= 2;
    TORCH_CHECK(y.sizes() == at::IntArrayRef(shape), what, ": y must have shape ", at::IntArrayRef(shape),
                g.packed ? " (value and gate side by side)" : "", ", got ", y.sizes());
    TORCH_CHECK(y.scalar_type() == type, what, ": y must be ", type, " next to ", x.scalar_type(), " x, got ",
                y.scalar_type());
    TORCH_CHECK(y.device() == x.device(), what, ": y must be on x's device");
    TORCH_CHECK(g.gated() || g.act == KANB200_ACT_NONE, what, ": a gate activation needs a gate");
    if (g.gate.defined()) {
        const Tensor& t = g.gate;
        TORCH_CHECK(t.scalar_type() == type, what, ": gate must be ", type, " next to ", x.scalar_type(), " x, got ",
                    t.scalar_type());
        TORCH_CHECK(t.device() == x.device(), what, ": gate must be on x's device");
        // a gate per row, or one for all rows of the trailing dimensions in which it has size 1
        bool ok = t.dim() >= 1 && t.size(-1) == g.width && (t.dim() == x.dim() || t.dim() == 1);
        int64_t own = 1;
        if (ok && t.dim() == x.dim()) {
            int64_t d = 0;
            while (d + 1 < x.dim() && t.size(d) == x.size(d)) own *= t.size(d++);
            for (; d + 1 < x.dim(); ++d) ok = ok && t.size(d) == 1;
        }
        TORCH_CHECK(ok, what, ": gate must have x's shape ", x.sizes(), " or size 1 in trailing row dimensions, got ",
                    t.sizes());
        g.gate_rows = own > 0 ? std::max<int64_t>(g.rows / own, 1) : 1;
    }
    g.row_gate = g.gated() && g.gate_rows == 1;
    check_vector(g.scale, what, "scale", g.width, type, x);
    check_vector(g.pw, what, "post_weight", g.width, type, x);
    check_vector(g.pb, what, "post_bias", g.width, type, x);
    check_vector(g.nw, what, "next_weight", g.width, type, x);
    check_vector(g.nb, what, "next_bias", g.width, type, x);
    TORCH_CHECK(g.post != KANB200_NORM_NONE || !(g.pw.defined() || g.pb.defined()), what,
                ": post_weight and post_bias need post_norm");
    TORCH_CHECK(g.next != KANB200_NORM_NONE || !(g.nw.defined() || g.nb.defined()), what,
                ": next_weight and next_bias need next_norm");
}

// value and gate of the branch as differentiable tensors
std::pair<Tensor, Tensor> halves(const Gated& g) {
    if (!g.packed) return {g.y, g.gate};
    return {g.y.narrow(-1, 0, g.width), g.y.narrow(-1, g.width, g.width)};
}

variable_list gated_composite(const Gated& g) {
    const auto [y, gate] = halves(g);
    Tensor t = affine(g.post != KANB200_NORM_NONE ? standardise(y, g.post, g.eps) : y, g.pw, g.pb);
    if (gate.defined()) t = t * activate(gate, g.act);
    if (g.scale.defined()) t = t * g.scale;
    const Tensor out = (g.x.to(branch_type(g.x)) + t).to(g.x.scalar_type());
    if (g.next == KANB200_NORM_NONE) return {out};
    return {out, norm_composite(out, g.nw, g.nb, g.next, g.eps)};
}

Record gated_record(const Gated& g) {
    Record r;
    r.post = g.post != KANB200_NORM_NONE;
    r.next = g.next != KANB200_NORM_NONE;
    r.y = g.checkpoint != KANB200_PACK_NONE;
    r.gate = r.y && g.row_gate;
    r.x = r.y && r.next;
    return r;
}

void fill(kanb200_block_args& a, const Gated& g) {
    a.gate_act = (int)g.act;
    a.post_norm = (int)g.post;
    a.next_norm = (int)g.next;
    a.eps = g.eps;
    a.rows = g.rows;
    a.width = g.width;
    a.gate_rows = g.gate_rows;
}

// y and gate as rows of the branch's memory: two tensors, or the two halves of one
void branch_rows(const Gated& g, Rows& y, const void*& gate, int64_t& gate_stride, Rows& gate_keep) {
    y = as_rows(g.y, g.rows, g.packed ? 2 * g.width : g.width);
    if (g.packed) {
        gate = static_cast<const char*>(y.ptr()) + g.width * g.y.element_size();
        gate_stride = y.stride;
    } else if (g.gate.defined()) {
        gate_keep = as_rows(g.gate, g.rows / g.gate_rows, g.width);
        gate = gate_keep.ptr();
        gate_stride = gate_keep.stride;
    }
}

variable_list gated_forward(const Gated& g, Tensor* record) {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(g.x.device());
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    Tensor out = fresh(g.x.sizes(), g.x.scalar_type(), g.x), h;
    if (g.next != KANB200_NORM_NONE) h = fresh(g.x.sizes(), branch_type(g.x), g.x);
    kanb200_block_args a{};
    a.dtype = stream_code(g.x, "gated_residual");
    fill(a, g);
    if (record) {
        a.checkpoint = (int)g.checkpoint;
        *record = gated_record(g).make(a, g.x);
    }
    const Rows xr = as_rows(g.x, g.rows, g.width);
    Rows yr, gr;
    branch_rows(g, yr, a.gate, a.gate_stride, gr);
    const Tensor scale = dense(g.scale), pw = dense(g.pw), pb = dense(g.pb), nw = dense(g.nw), nb = dense(g.nb);
    a.x = xr.ptr();
    a.x_stride = xr.stride;
    a.y = yr.ptr();
    a.y_stride = yr.stride;
    a.scale = cptr(scale);
    a.post_weight = cptr(pw);
    a.post_bias = cptr(pb);
    a.next_weight = cptr(nw);
    a.next_bias = cptr(nb);
    a.out = out.data_ptr();
    a.h = mptr(h);
    check_rc(kanb200_block_forward(&a, st));
    if (h.defined()) return {out, h};
    return {out};
}

// needs_input_grad / result slots
enum { kX, kY, kGate, kScale, kPostWeight, kPostBias, kNextWeight, kNextBias, kGatedInputs };

struct GatedResidualNode : public SavedNode {
    Gated settings;                                          // without tensors
    at::ScalarType type = at::kFloat;                        // of the stream
    std::vector<int64_t> shape, gate_shape;
    std::string name() const override { return "GatedResidualBackward"; }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        variable_list result(kGatedInputs);
        const Tensor dout = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        if (!dout.defined() && !dh.defined()) return result;
        std::array<Tensor, 8> v;
        for (size_t i = 0; i < v.size(); ++i) v[i] = kept(i);
        Gated g = settings;
        g.y = v[1];
        g.gate = v[2];
        g.scale = v[3];
        g.pw = v[4];
        g.pb = v[5];
        g.nw = v[6];
        if (at::GradMode::is_enabled()) {
            TORCH_CHECK(g.checkpoint == KANB200_PACK_NONE,
                        "gated_residual: create_graph=True needs the inputs themselves, not their 8-bit checkpoints");
            composite_backward(g, v[0], dout, dh, type, result);
            return result;
        }
        const Tensor& like = dout.defined() ? dout : dh;
        c10::cuda::CUDAGuard guard(like.device());
        const cudaStream_t st = at::cuda::getCurrentCUDAStream();
        const at::ScalarType branch = type == at::kDouble ? at::kDouble : at::kFloat;
        kanb200_block_args a{};
        fill(a, g);
        if (!dh.defined()) a.next_norm = KANB200_NORM_NONE;
        a.dtype = type_code(type);
        a.has_branch = 1;
        a.checkpoint = (int)g.checkpoint;
        Tensor dx, dy, dgate;
        if (need(kX)) {
            // without a norm behind, the stream's gradient passes through unchanged
            if (dh.defined()) dx = fresh(shape, type, like);
            else result[kX] = dout;
        }
        const bool want_gate = g.packed ? need(kY) : need(kGate);
        if (need(kY)) {
            auto s = shape;
            if (g.packed) s.back() *= 2;
            dy = fresh(s, branch, like);
            a.dy_stride = s.back();
        }
        if (want_gate && !g.packed) dgate = fresh(gate_shape, branch, like);
        const auto vec = [&](int i) {
            if (need(i)) result[i] = fresh({g.width}, branch, like);
            return mptr(result[i]);
        };
        a.dscale = vec(kScale);
        a.dpost_weight = vec(kPostWeight);
        a.dpost_bias = vec(kPostBias);
        if (dh.defined()) {
            a.dnext_weight = vec(kNextWeight);
            a.dnext_bias = vec(kNextBias);
        }
        const Rows xr = as_rows(dh.defined() ? v[0] : Tensor(), g.rows, g.width), dor = as_rows(dout, g.rows, g.width),
                   dhr = as_rows(dh, g.rows, g.width);
        Rows yr, gr;
        if (g.y.defined()) branch_rows(g, yr, a.gate, a.gate_stride, gr);
        else if (g.gate.defined()) {
            gr = as_rows(g.gate, g.rows / g.gate_rows, g.width);
            a.gate = gr.ptr();
            a.gate_stride = gr.stride;
        }
        const Tensor scale = dense(g.scale), pw = dense(g.pw), pb = dense(g.pb), nw = dense(g.nw);
        a.x = xr.ptr();
        a.x_stride = xr.stride;
        a.y = yr.ptr();
        a.y_stride = yr.stride;
        a.scale = cptr(scale);
        a.post_weight = cptr(pw);
        a.post_bias = cptr(pb);
        if (dh.defined()) a.next_weight = cptr(nw);
        gated_record(g).find(a, v[7]);
        if (!dh.defined()) a.x_codes = a.x_scales = nullptr;
        a.dout = dor.ptr();
        a.dout_stride = dor.stride;
        a.dh = dhr.ptr();
        a.dh_stride = dhr.stride;
        a.dx = mptr(dx);
        a.dy = mptr(dy);
        if (want_gate && g.packed) {
            a.dgate = has(dy) ? static_cast<char*>(dy.data_ptr()) + g.width * dy.element_size() : nullptr;
            a.dgate_stride = 2 * g.width;
        } else {
            a.dgate = mptr(dgate);
            a.dgate_stride = g.width;
        }
        if (a.dx || a.dy || a.dgate || a.dscale || a.dpost_weight || a.dpost_bias || a.dnext_weight || a.dnext_bias)
            run_backward(a, like, st);
        if (dx.defined()) result[kX] = dx;
        result[kY] = dy;
        result[kGate] = dgate;
        return result;
    }

    static void composite_backward(const Gated& g, const Tensor& out, const Tensor& dout, const Tensor& dh,
                                   at::ScalarType type, variable_list& result) {
        const auto btype = type == at::kDouble ? at::kDouble : at::kFloat;
        const auto [y, gate] = halves(g);
        Tensor grad = dout.defined() ? dout.to(btype) : Tensor();
        if (dh.defined()) {
            Tensor through;
            std::tie(through, result[kNextWeight], result[kNextBias]) = norm_gradient(out.to(btype), g.nw, dh, g.next, g.eps);
            grad = grad.defined() ? grad + through : through;
        }
        result[kX] = grad.to(type);
        const Tensor z = affine(g.post != KANB200_NORM_NONE ? standardise(y, g.post, g.eps) : y, g.pw, g.pb);
        const Tensor gs = g.scale.defined() ? grad * g.scale : grad;
        Tensor dz = gs, dgate;
        if (gate.defined()) {
            const Tensor act = activate(gate, g.act);
            dz = gs * act;
            dgate = (gs * activate_grad(gate, g.act) * z).sum_to_size(gate.sizes());
            result[kScale] = over_rows(grad * act * z);
        } else {
            result[kScale] = over_rows(grad * z);
        }
        if (g.post != KANB200_NORM_NONE)
            std::tie(result[kY], result[kPostWeight], result[kPostBias]) = norm_gradient(y, g.pw, dz, g.post, g.eps);
        else
            result[kY] = dz;
        if (g.packed) result[kY] = at::cat({result[kY], dgate}, -1);
        else result[kGate] = dgate;
        if (!g.scale.defined()) result[kScale] = Tensor();
    }
};

py::object gated_residual(const Tensor& x, const Tensor& y, const std::optional<Tensor>& gate, bool packed, int64_t act,
                          const std::optional<Tensor>& scale, int64_t post, const std::optional<Tensor>& pw,
                          const std::optional<Tensor>& pb, int64_t next, const std::optional<Tensor>& nw,
                          const std::optional<Tensor>& nb, double eps, int64_t checkpoint) {
    Gated g{x, y, or_undefined(gate), or_undefined(scale), or_undefined(pw), or_undefined(pb), or_undefined(nw),
            or_undefined(nb), packed, act, post, next, checkpoint, eps};
    check_gated(g);
    TORCH_CHECK(x.is_cuda() || checkpoint == KANB200_PACK_NONE, "gated_residual: 8-bit checkpoints need CUDA tensors");
    variable_list outs;
    if (x.is_cuda() && x.numel() > 0) check_memory("gated_residual", {g.x, g.y, g.gate, g.scale, g.pw, g.pb, g.nw, g.nb});
    if (!x.is_cuda() || x.numel() == 0) {
        outs = gated_composite(g);
    } else if (!wants_grad({g.x, g.y, g.gate, g.scale, g.pw, g.pb, g.nw, g.nb}, "gated_residual")) {
        outs = gated_forward(g, nullptr);
    } else {
        Tensor record;
        outs = gated_forward(g, &record);
        auto node = new_node<GatedResidualNode>({g.x, g.y, g.gate, g.scale, g.pw, g.pb, g.nw, g.nb});
        node->settings = g;
        for (Tensor Gated::*t : {&Gated::x, &Gated::y, &Gated::gate, &Gated::scale, &Gated::pw, &Gated::pb, &Gated::nw, &Gated::nb})
            node->settings.*t = Tensor();
        node->type = x.scalar_type();
        node->shape = x.sizes().vec();
        if (g.gate.defined()) node->gate_shape = g.gate.sizes().vec();
        for (Tensor& t : outs) torch::autograd::set_history(t, node);
        const bool codes = checkpoint != KANB200_PACK_NONE, keep_gate = !codes || g.gate_rows > 1;
        node->saved.reserve(8);
        node->keep(next != KANB200_NORM_NONE && !codes ? outs[0] : Tensor(), true);
        for (const Tensor& t : {codes ? Tensor() : g.y, keep_gate ? g.gate : Tensor(), g.scale, g.pw, g.pb, g.nw, record})
            node->keep(t);
    }
    if (outs.size() == 1) return py::cast(outs[0]);
    return py::make_tuple(outs[0], outs[1]);
}

}  // namespace

// ------------------------------------------------------------------------------------------------
// 8-bit checkpoints
// ------------------------------------------------------------------------------------------------
Packed pack_rows(const Tensor& x, int format) {
    const char* what = "pack_activation";
    const int code = stream_code(x, what);
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": x must have at least one column, got ", x.sizes());
    TORCH_CHECK(x.is_cuda(), what, ": x must be a CUDA tensor (this backend has no CPU kernels)");
    check_memory(what, {x});
    c10::cuda::CUDAGuard guard(x.device());
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    const int64_t rows = row_count(x), width = x.size(-1);
    auto shape = x.sizes().vec();
    Packed p{fresh({rows, width}, format == KANB200_PACK_INT8 ? at::kChar : at::kFloat8_e4m3fn, x),
             fresh({rows, group_count(width)}, branch_type(x), x)};
    const Rows xr = as_rows(x, rows, width);
    check_rc(kanb200_pack_activation(code, format, xr.ptr(), xr.stride, mptr(p.codes), mptr(p.scales), rows, width, st));
    if (x.dim() != 2) {
        p.codes = p.codes.view(shape);
        shape.back() = p.scales.size(1);
        p.scales = p.scales.view(shape);
    }
    return p;
}

Tensor unpack_rows(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
    const char* what = "unpack_activation";
    TORCH_CHECK(codes.scalar_type() == at::kChar || codes.scalar_type() == at::kFloat8_e4m3fn, what,
                ": codes must be int8 or float8_e4m3fn, got ", codes.scalar_type());
    TORCH_CHECK(codes.dim() >= 1 && codes.size(-1) >= 1, what, ": codes must have at least one column, got ", codes.sizes());
    auto shape = codes.sizes().vec();
    shape.back() = (shape.back() + KANB200_PACK_GROUP - 1) / KANB200_PACK_GROUP;
    TORCH_CHECK(scales.sizes() == at::IntArrayRef(shape), what, ": scales must have shape ", at::IntArrayRef(shape),
                ", got ", scales.sizes());
    TORCH_CHECK(dtype == at::kFloat || dtype == at::kDouble || dtype == at::kHalf || dtype == at::kBFloat16, what,
                ": dtype must be float32, float64, float16 or bfloat16, got ", dtype);
    const auto stype = dtype == at::kDouble ? at::kDouble : at::kFloat;
    TORCH_CHECK(scales.scalar_type() == stype, what, ": scales of ", dtype, " values must be ", stype, ", got ",
                scales.scalar_type());
    TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(), what,
                ": codes and scales must be CUDA tensors on one device");
    check_memory(what, {codes, scales});
    c10::cuda::CUDAGuard guard(codes.device());
    const cudaStream_t st = at::cuda::getCurrentCUDAStream();
    const Tensor cc = codes.contiguous(), sc = dense(scales);
    Tensor x = fresh(codes.sizes(), dtype, codes);
    check_rc(kanb200_unpack_activation(stream_code(x, what),
                                       codes.scalar_type() == at::kChar ? KANB200_PACK_INT8 : KANB200_PACK_E4M3, cptr(cc),
                                       cptr(sc), mptr(x), row_count(codes), codes.size(-1), st));
    return x;
}

void bind_block_operators(py::module_& m) {
    m.attr("PACK_GROUP") = KANB200_PACK_GROUP;
    m.def("block_norm", &block_norm, "norm(x) weight + bias, autograd-aware");
    m.def("gated_residual", &gated_residual, "x + scale act(gate) post(y) and, with a next norm, the norm of it");
    m.def("pack_activation",
          [](const Tensor& x, int64_t format) {
              Packed p = pack_rows(x, (int)format);
              return py::make_tuple(p.codes, p.scales);
          },
          "(codes, scales) of an 8-bit checkpoint");
    m.def("unpack_activation", [](const Tensor& codes, const Tensor& scales, py::object dtype) {
              return unpack_rows(codes, scales, torch::python::detail::py_object_to_dtype(dtype));
          },
          "the values of an 8-bit checkpoint");
}

}  // namespace kan_ext
