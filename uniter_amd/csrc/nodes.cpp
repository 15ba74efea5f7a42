// nodes.cpp — the autograd nodes of the operators whose calls are short: rotary positions and differential attention.
//
// A training call of these operators is two to four kernels of 5 to 25 us.  As Python autograd functions over ctypes their host work is
// 45 us in a loop that stays in the CPU's caches and twice that when autograd's own thread takes the backward half to another core; here
// it is C++ on both sides and the backward pass needs no interpreter (32 x 96, 12 heads, forward and gradients, call to call: 167 -> 93 us; one
// rotary training call 95 -> 49, one token 11.6 -> 7.5).  The kernels are reached through the C ABI all the same: the
// package hands over the addresses of the entry points of the library that it has loaded (init), nothing is linked.
//
// The arguments' checks are here too, for the same reason (ops.py holds the documentation); workspaces come from torch's caching allocator.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../include/uniter_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
    decltype(&uniter_rotary) rotary;
    decltype(&uniter_diff_attention_fwd_workspace_bytes) fwd_bytes;
    decltype(&uniter_diff_attention_fwd) fwd;
    decltype(&uniter_diff_attention_bwd_workspace_bytes) bwd_bytes;
    decltype(&uniter_diff_attention_bwd) bwd;
    decltype(&uniter_hip_last_error) last_error;
} lib{};
PyObject* error_type = nullptr;

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };

void ok(int rc, const char* name) {
    if (rc == 0) return;
    const char* why = lib.last_error();
    throw Error(std::string(name) + " failed with status " + std::to_string(rc) + ": " + (why ? why : ""));
}

template <class... T>
[[noreturn]] void refuse(const T&... words) { throw Error(c10::str(words...)); }

void check(const Tensor& t, at::ScalarType type, const char* what) {
    if (!t.defined() || !t.is_cuda())
        refuse(what, " must be a CUDA(HIP) tensor: the kernels exist for gfx950 only (no CPU / PyTorch fallback)");
    if (t.scalar_type() != type) refuse(what, " must be ", type, ", got ", t.scalar_type(), type == at::kBFloat16 ? " (cast the model with .bfloat16())" : "");
}
void check_beside(const Tensor& first, const char* name, const Tensor& t, at::ScalarType type, const char* what) {
    check(t, type, what);
    if (t.get_device() != first.get_device()) refuse(what, " is on ", t.device(), ", ", name, " on ", first.device());
}

// What neither a plain call nor a node here can carry on is refused, not dropped: a forward-mode tangent, and a trace (a launch through
// a raw pointer leaves nothing in it but the empty result).
void check_mode(const char* name, std::initializer_list<const Tensor*> inputs) {
    if (torch::jit::tracer::isTracing()) refuse(name, " cannot be traced: nothing of it would be recorded");
    for (const Tensor* t : inputs)
        if (t->defined() && t->_fw_grad(0).defined()) refuse(name, " has no forward-mode derivative");
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor get(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
Tensor rows_like(const Tensor& t) { return at::empty_like(t, t.options(), at::MemoryFormat::Contiguous); }
// strides of [.., rows, columns]; a dimension of one has one that no address uses and that may be anything
int64_t row_step(const Tensor& t) { return t.size(-2) == 1 ? t.size(-1) : t.stride(-2); }
int64_t batch_step(const Tensor& t) { return t.size(0) == 1 ? 0 : t.stride(0); }
// contiguous rows that start on 16 bytes (row strides of whole 8s); a copy where they do not
Tensor rows16(const Tensor& t) {
    if (t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0) return t;
    bool fits = t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0;
    for (int64_t i = 0; fits && i + 1 < t.dim(); ++i) fits = t.stride(i) % 8 == 0 || t.size(i) == 1;
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Gradients of a pass that has no derivative of its own: where the incoming gradient wants one, asking for it is an error.
variable_list once(variable_list grads, const Tensor& incoming) {
    if (!at::GradMode::is_enabled() || !incoming.requires_grad()) return grads;
    variable_list known;
    for (auto& g : grads)
        if (g.defined()) known.push_back(g);
    auto error = std::make_shared<torch::autograd::DelayedError>("the gradient of this operator has no derivative", (int64_t)known.size());
    known = (*error)(std::move(known));
    size_t i = 0;
    for (auto& g : grads)
        if (g.defined()) g = known[i++];
    return grads;
}

// ------------------------------------------------------------------------------------------------
// rotary positions
// ------------------------------------------------------------------------------------------------
struct Rotary {
    Tensor positions;                    // int64 [L] / [B, L] / [T], or undefined
    Tensor turns;                        // float64 [rot / 2]
    int64_t offset, rot;
    double multiplier;
    bool interleaved;
};

void rotary_run(const Tensor& x, const Tensor& y, const Rotary& r, bool inverse) {
    if (x.numel() == 0) return;
    const int64_t d = x.dim();
    UniterRotary a{};
    a.B = d == 4 ? x.size(0) : 1;
    a.L = x.size(-3); a.heads = x.size(-2); a.head_dim = x.size(-1);
    a.rot_dim = r.rot;
    a.freq = (const double*)r.turns.data_ptr();
    if (r.positions.defined()) {
        a.positions = (const int64_t*)r.positions.data_ptr();
        a.positions_batch_stride = r.positions.dim() == 2 ? r.positions.stride(0) : 0;
    }
    a.position_offset = r.offset;
    a.multiplier = (float)r.multiplier;
    a.interleaved = r.interleaved;
    a.inverse = inverse;
    auto step = [d](const Tensor& t, int64_t i) { return d < i || t.size(-i) == 1 ? (int64_t)0 : t.stride(-i); };      // (what nothing steps over may be anything)
    const int64_t sx[3] = {step(x, 4), step(x, 3), step(x, 2)}, sy[3] = {step(y, 4), step(y, 3), step(y, 2)};
    const c10::DeviceGuard on(x.device());
    ok(lib.rotary(&a, x.data_ptr(), sx, y.data_ptr(), sy, stream_of(x)), "uniter_rotary");
}

struct RotaryNode : torch::autograd::Function<RotaryNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Rotary& r) {
        Tensor y = rows_like(x);
        rotary_run(x, y, r, false);
        ctx->save_for_backward({r.positions, r.turns});
        ctx->saved_data["n"] = std::vector<int64_t>{r.offset, r.rot, r.interleaved};
        ctx->saved_data["m"] = r.multiplier;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list t = ctx->get_saved_variables();
        const auto n = ctx->saved_data["n"].toIntVector();
        const Rotary r{t[0], t[1], n[0], n[1], ctx->saved_data["m"].toDouble(), n[2] != 0};
        Tensor dy = grads[0];
        if (!dy.defined()) return {Tensor(), Tensor()};
        if (dy.stride(-1) != 1) dy = dy.contiguous();
        Tensor dx = rows_like(dy);
        rotary_run(dy, dx, r, true);
        return once({dx, Tensor()}, grads[0]);
    }
};

Tensor rotary(Tensor x, const optional<Tensor>& positions, int64_t offset, const optional<Tensor>& out, const Tensor& turns, int64_t head_dim,
              int64_t rot, double multiplier, bool interleaved) {
    check_mode("rotary", {&x, out.has_value() ? &*out : &x});
    check(x, at::kBFloat16, "rotary input");
    const int64_t d = x.dim();
    if ((d != 3 && d != 4) || x.size(-1) != head_dim)
        refuse("rotary input must be [B, L, heads, ", head_dim, "] or [T, heads, ", head_dim, "], got ", x.sizes());
    Tensor pos = get(positions);
    if (!pos.defined()) {
        if (d == 3) refuse("rotary: rows stored back to back need their positions");
    } else {
        if (pos.scalar_type() != at::kLong && pos.scalar_type() != at::kInt) refuse("rotary: positions must be an int64 or int32 tensor (or None)");
        if (!pos.is_cuda() || pos.get_device() != x.get_device()) refuse("positions is on ", pos.device(), ", x on ", x.device());
        if (d == 4 && pos.dim() == 2 && pos.size(0) == 1 && x.size(0) != 1) pos = pos[0];
        const auto rows = x.sizes().slice(0, d - 2), last = x.sizes().slice(d - 3, 1);
        if (pos.sizes() != rows && pos.sizes() != last) refuse("rotary: positions must be ", rows, " or ", last, ", got ", pos.sizes());
        if (pos.scalar_type() == at::kInt) pos = pos.to(at::kLong);
        if (pos.stride(-1) != 1) pos = pos.contiguous();
    }
    if (x.stride(-1) != 1) {
        if (out.has_value() && out->is_same(x)) refuse("rotary: in place needs contiguous heads");
        x = x.contiguous();
    }
    const Rotary r{pos, turns, offset, rot, multiplier, interleaved};
    if (!out.has_value()) {
        if (at::GradMode::is_enabled() && x.requires_grad()) return RotaryNode::apply(x, r);
        Tensor y = rows_like(x);
        rotary_run(x, y, r, false);
        return y;
    }
    const Tensor& y = *out;
    if (at::GradMode::is_enabled() && (x.requires_grad() || y.requires_grad()))
        refuse("rotary: out= writes outside autograd; call it without gradients or let it return a new tensor");
    check_beside(x, "x", y, at::kBFloat16, "rotary output");
    if (y.sizes() != x.sizes() || y.stride(-1) != 1) refuse("rotary: out must have x's shape and contiguous heads");
    // (the entry refuses an out that overlaps itself, or x without being x)
    rotary_run(x, y, r, false);
    if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();      // (a node that saved y, or what shares its memory, has to hear of it)
    return y;
}

// the kernel by itself, in place, on checked arguments
void rotary_turn(const Tensor& x, const optional<Tensor>& positions, const Tensor& turns, int64_t rot, double multiplier, bool interleaved, bool inverse) {
    rotary_run(x, x, Rotary{get(positions), turns, 0, rot, multiplier, interleaved}, inverse);
}

// ------------------------------------------------------------------------------------------------
// differential attention
// ------------------------------------------------------------------------------------------------
struct Fixed {                           // what a call has besides its differentiable tensors
    Tensor mask, cu_q, cu_k;
    int64_t heads, dim, max_q, max_k, seed, offset;
    double lambda_init, eps, p_drop;
    bool keep;                           // a backward pass will come
};
struct Operands {                        // k and v undefined: q is a fused [.., 3 H] projection
    Tensor q, k, v, weight, lams[4];
};

// q, k, v (or dq, dk, dv): three tensors, or the thirds of one projection's rows
template <class A>
void set_rows(A& a, const Tensor& q, const Tensor& k, const Tensor& v) {
    char* p = (char*)q.data_ptr();
    const bool fused = !k.defined();
    const int64_t third = fused ? q.size(-1) / 3 * 2 : 0;      // bytes
    a.q = p;
    a.k = fused ? (p ? p + third : nullptr) : k.data_ptr();
    a.v = fused ? (p ? p + 2 * third : nullptr) : v.data_ptr();
    a.q_row = row_step(q);
    a.k_row = fused ? a.q_row : row_step(k);
    a.v_row = fused ? a.q_row : row_step(v);
    a.q_batch = batch_step(q);
    a.k_batch = fused ? a.q_batch : batch_step(k);
    a.v_batch = fused ? a.q_batch : batch_step(v);
}

UniterDiffAttention args_of(const Operands& t, const Fixed& f) {
    UniterDiffAttention a{};
    set_rows(a, t.q, t.k, t.v);
    const bool fused = !t.k.defined();
    if (f.mask.defined()) {
        a.mask_bias = (const float*)f.mask.data_ptr();
        a.mask_row = f.mask.stride(0);
    }
    if (f.cu_q.defined()) {
        a.cu_seqlens_q = (const int32_t*)f.cu_q.data_ptr();
        a.cu_seqlens_k = (const int32_t*)f.cu_k.data_ptr();
        a.total_q = t.q.size(0);
        a.total_k = fused ? a.total_q : t.k.size(0);
        a.B = f.cu_q.size(0) - 1;
        a.Lq = f.max_q; a.Lk = f.max_k;
    } else {
        a.B = t.q.size(0);
        a.Lq = t.q.size(1);
        a.Lk = fused ? a.Lq : t.k.size(1);
    }
    a.lambda_q1 = t.lams[0].data_ptr(); a.lambda_k1 = t.lams[1].data_ptr();
    a.lambda_q2 = t.lams[2].data_ptr(); a.lambda_k2 = t.lams[3].data_ptr();
    a.lambda_per_head = t.lams[0].dim() == 2;
    a.norm_weight = ptr(t.weight);
    a.heads = f.heads; a.head_dim = f.dim;
    a.lambda_init = (float)f.lambda_init; a.norm_eps = (float)f.eps; a.p_drop = (float)f.p_drop;
    a.seed = (uint64_t)f.seed; a.offset = (uint64_t)f.offset;
    return a;
}

// (out, saved): saved (fp32: both maps' outputs, then the rows' statistics) only where a backward pass will want it
std::pair<Tensor, Tensor> diff_forward(const Operands& t, const Fixed& f) {
    UniterDiffAttention a = args_of(t, f);
    const int64_t H = f.heads * 2 * f.dim;
    // (rows of a packed batch that belong to no example are not written: they are zeros)
    Tensor out = f.cu_q.defined() ? at::zeros({t.q.size(0), H}, t.q.options()) : at::empty({a.B, a.Lq, H}, t.q.options());
    Tensor saved, ws;
    float *maps = nullptr, *stats = nullptr;
    if (f.keep) {
        const int64_t n = out.numel() * 2;
        saved = at::empty({n + a.B * a.heads * a.Lq * 4}, t.q.options().dtype(at::kFloat));
        maps = (float*)saved.data_ptr();
        stats = maps ? maps + n : nullptr;
    }
    const c10::DeviceGuard on(t.q.device());
    const size_t bytes = lib.fwd_bytes(&a);
    if (bytes) ws = at::empty({(int64_t)bytes}, t.q.options().dtype(at::kByte));
    ok(lib.fwd(&a, out.data_ptr(), H, out.stride(0), stats, maps, ptr(ws), bytes, stream_of(t.q)), "uniter_diff_attention_fwd");
    return {out, saved};
}

// dq / dk / dv: like q / k / v (one [.., 3 H] tensor for a fused projection); undefined parameter gradients are not formed
void diff_backward(const Operands& t, const Fixed& f, const Tensor& saved, const Tensor& incoming, const Operands& d, bool accumulate) {
    UniterDiffAttention a = args_of(t, f);
    UniterDiffAttentionGrads g{};
    set_rows(g, d.q, d.k, d.v);
    g.lambda_q1 = ptr(d.lams[0]); g.lambda_k1 = ptr(d.lams[1]); g.lambda_q2 = ptr(d.lams[2]); g.lambda_k2 = ptr(d.lams[3]);
    g.norm_weight = ptr(d.weight);
    g.accumulate_params = accumulate;
    const Tensor dout = rows16(incoming);
    const c10::DeviceGuard on(t.q.device());
    const size_t bytes = lib.bwd_bytes(&a);
    Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, t.q.options().dtype(at::kByte));
    const float* maps = (const float*)saved.data_ptr();
    ok(lib.bwd(&a, maps ? maps + 2 * dout.numel() : nullptr, maps, dout.data_ptr(), row_step(dout), batch_step(dout), &g, ws.data_ptr(), bytes,
               stream_of(t.q)), "uniter_diff_attention_bwd");
}

struct DiffNode : torch::autograd::Function<DiffNode> {
    static Tensor forward(AutogradContext* ctx, const Fixed& f, const Tensor& q, const optional<Tensor>& k, const optional<Tensor>& v,
                          const optional<Tensor>& weight, const Tensor& l0, const Tensor& l1, const Tensor& l2, const Tensor& l3) {
        const Operands t{q, get(k), get(v), get(weight), {l0, l1, l2, l3}};
        auto [out, saved] = diff_forward(t, f);
        ctx->save_for_backward({q, t.k, t.v, t.weight, l0, l1, l2, l3, f.mask, f.cu_q, f.cu_k, saved});
        ctx->saved_data["n"] = std::vector<int64_t>{f.heads, f.dim, f.max_q, f.max_k, f.seed, f.offset};
        ctx->saved_data["x"] = std::vector<double>{f.lambda_init, f.eps, f.p_drop};
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return variable_list(9);
        const variable_list s = ctx->get_saved_variables();
        const auto n = ctx->saved_data["n"].toIntVector();
        const auto x = ctx->saved_data["x"].toDoubleVector();
        const Operands t{s[0], s[1], s[2], s[3], {s[4], s[5], s[6], s[7]}};
        const Fixed f{s[8], s[9], s[10], n[0], n[1], n[2], n[3], n[4], n[5], x[0], x[1], x[2], true};
        const at::AutoDispatchBelowADInplaceOrView below;      // (buffers of kernels: nothing here is recorded)
        auto like = [&](const Tensor& a) { return !a.defined() ? Tensor() : f.cu_q.defined() ? at::zeros(a.sizes(), a.options()) : rows_like(a); };
        Operands d{like(t.q), like(t.k), like(t.v), t.weight.defined() ? rows_like(t.weight) : Tensor(), {}};
        for (int i = 0; i < 4; ++i) d.lams[i] = rows_like(t.lams[i]);
        diff_backward(t, f, s[11], grads[0], d, false);
        return once({Tensor(), d.q, d.k, d.v, d.weight, d.lams[0], d.lams[1], d.lams[2], d.lams[3]}, grads[0]);
    }
};

Fixed fixed_of(const optional<Tensor>& mask, const optional<Tensor>& cu_q, const optional<Tensor>& cu_k, int64_t heads, int64_t dim, double lambda_init,
               double eps, int64_t max_q, int64_t max_k, double p_drop, int64_t seed, int64_t offset, bool keep) {
    return Fixed{get(mask), get(cu_q), get(cu_k), heads, dim, max_q, max_k, seed, offset, lambda_init, eps, p_drop, keep};
}

// ops.differential_attention; k and v nullopt: q is a fused projection
Tensor diff_attention(Tensor q, const optional<Tensor>& k_, const optional<Tensor>& v_, int64_t heads, const std::vector<Tensor>& lams, double lambda_init,
                      const optional<Tensor>& weight_, const optional<Tensor>& mask_, const optional<Tensor>& cu_q_, const optional<Tensor>& cu_k_,
                      optional<int64_t> max_q, optional<int64_t> max_k, double eps, double p_drop, int64_t seed, int64_t offset) {
    const bool fused = !k_.has_value(), packed = cu_q_.has_value() || cu_k_.has_value();
    const char* name = fused ? "qkv" : "q";
    Tensor k = get(k_), v = get(v_), weight = get(weight_), mask = get(mask_), cu_q = get(cu_q_), cu_k = get(cu_k_), l[4];
    check_mode("differential attention", {&q, &k, &v, &weight, &mask});
    check(q, at::kBFloat16, name);
    if (!fused) {
        check_beside(q, name, k, at::kBFloat16, "k");
        check_beside(q, name, v, at::kBFloat16, "v");
    }
    const int64_t nd = packed ? 2 : 3;
    if (q.dim() != nd || (!fused && (k.dim() != nd || v.dim() != nd)))
        refuse(fused ? "qkv" : "q, k and v", " must be ", packed ? "[rows, columns] when cu_seqlens is given" : "[B, L, columns]", ", got ", q.sizes());
    const int64_t cols = q.size(-1), H = fused ? cols / 3 : cols, dim = heads > 0 ? H / (2 * heads) : 0;
    if ((fused && cols % 3 != 0) || (dim != 32 && dim != 64) || H != heads * 2 * dim)
        refuse("differential attention: a head is 64 or 128 columns (two maps of 32 or 64), got ", H, " columns for ", heads, " heads");
    if (!fused && (k.sizes() != v.sizes() || k.size(-1) != H || (!packed && k.size(0) != q.size(0))))
        refuse("differential attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not fit");
    if (lams.size() != 4) refuse("lambdas are four tensors: q1, k1, q2, k2");
    const bool per_head = lams[0].sizes() == at::IntArrayRef({heads, dim});
    if (!per_head && lams[0].sizes() != at::IntArrayRef({dim})) refuse("lambda vectors must be [", dim, "] or [", heads, ", ", dim, "], got ", lams[0].sizes());
    for (int i = 0; i < 4; ++i) {
        check_mode("differential attention", {&lams[i]});
        check_beside(q, name, lams[i], at::kBFloat16, "lambda vector");
        if (lams[i].sizes() != lams[0].sizes()) refuse("lambda vectors must have one shape, got ", lams[0].sizes(), " and ", lams[i].sizes());
        l[i] = lams[i].contiguous();
    }
    if (weight.defined()) {
        check_beside(q, name, weight, at::kBFloat16, "norm_weight");
        if (weight.sizes() != at::IntArrayRef({2 * dim})) refuse("norm_weight must be [", 2 * dim, "], got ", weight.sizes());
        weight = rows16(weight);
        if (!(eps > 0.0)) refuse("eps must be positive, got ", eps);
    }
    if (!(p_drop >= 0.0 && p_drop < 1.0)) refuse("dropout probability must be in [0, 1), got ", p_drop);
    if (packed) {
        if (mask.defined()) refuse("packed rows take no mask_bias: only real tokens are there");
        if (!cu_k.defined()) cu_k = cu_q;
        if (!max_k.has_value()) max_k = max_q;
        if (!cu_q.defined() || !max_q.has_value() || *max_q < 0 || *max_k < 0)
            refuse("packed rows need cu_seqlens and max_len (and those of the keys where they differ)");
        for (Tensor* c : {&cu_q, &cu_k}) {
            check_beside(q, name, *c, at::kInt, "cu_seqlens");
            if (c->dim() != 1 || c->numel() != cu_q.numel() || c->numel() < 1) refuse("cu_seqlens must be int32 [examples + 1]");
            *c = c->contiguous();
        }
    } else if (mask.defined()) {
        check_beside(q, name, mask, at::kFloat, "mask_bias");
        if (at::GradMode::is_enabled() && mask.requires_grad()) refuse("mask_bias has no gradient here: pass it detached");
        if (mask.dim() == 4 && mask.size(1) == 1 && mask.size(2) == 1) mask = mask.select(1, 0).select(1, 0);      // UniterModel's extended mask [B, 1, 1, L]
        const int64_t Lk = fused ? q.size(1) : k.size(1);
        if (mask.sizes() != at::IntArrayRef({q.size(0), Lk})) refuse("mask_bias must be [", q.size(0), ", ", Lk, "] (or [B, 1, 1, Lk]), got ", mask.sizes());
        if (mask.stride(1) != 1) mask = mask.contiguous();
    }
    q = rows16(q);
    if (!fused) {
        k = rows16(k);
        v = rows16(v);
    }
    auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    const bool keep = at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(weight) || wants(l[0]) || wants(l[1]) || wants(l[2]) || wants(l[3]));
    const Fixed f{mask, cu_q, cu_k, heads, dim, max_q.value_or(0), max_k.value_or(0), seed, offset, lambda_init, eps, p_drop, keep};
    if (!keep) return diff_forward(Operands{q, k, v, weight, {l[0], l[1], l[2], l[3]}}, f).first;
    auto given = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
    return DiffNode::apply(f, q, given(k), given(v), given(weight), l[0], l[1], l[2], l[3]);
}

void init(py::dict addresses, py::object error) {
    auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
    lib.rotary = (decltype(lib.rotary))at("uniter_rotary");
    lib.fwd_bytes = (decltype(lib.fwd_bytes))at("uniter_diff_attention_fwd_workspace_bytes");
    lib.fwd = (decltype(lib.fwd))at("uniter_diff_attention_fwd");
    lib.bwd_bytes = (decltype(lib.bwd_bytes))at("uniter_diff_attention_bwd_workspace_bytes");
    lib.bwd = (decltype(lib.bwd))at("uniter_diff_attention_bwd");
    lib.last_error = (decltype(lib.last_error))at("uniter_hip_last_error");
    error_type = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(uniter_nodes, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error& e) {
            PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, e.what());
        }
    });
    m.def("init", &init);
    // (without the interpreter lock, as torch's own operators: a launch may wait for room in its queue)
    using unlocked = py::call_guard<py::gil_scoped_release>;
    m.def("rotary", &rotary, unlocked());
    m.def("rotary_turn", &rotary_turn, unlocked());
    m.def("diff_attention", &diff_attention, unlocked());
    // the two passes by themselves, on a fused projection, for nodes that hold more than the attention
    m.def("diff_self_forward", [](const Tensor& qkv, const optional<Tensor>& weight, const std::vector<Tensor>& l, const optional<Tensor>& mask,
                                  const optional<Tensor>& cu, int64_t heads, int64_t dim, double lambda_init, double eps, int64_t max_len, double p_drop,
                                  int64_t seed, int64_t offset, bool keep) -> std::pair<Tensor, optional<Tensor>> {
        auto [out, saved] = diff_forward(Operands{qkv, Tensor(), Tensor(), get(weight), {l[0], l[1], l[2], l[3]}},
                                         fixed_of(mask, cu, cu, heads, dim, lambda_init, eps, max_len, max_len, p_drop, seed, offset, keep));
        return {out, saved.defined() ? optional<Tensor>(saved) : std::nullopt};
    }, unlocked());
    m.def("diff_self_backward", [](const Tensor& qkv, const optional<Tensor>& weight, const std::vector<Tensor>& l, const optional<Tensor>& mask,
                                   const optional<Tensor>& cu, int64_t heads, int64_t dim, double lambda_init, double eps, int64_t max_len, double p_drop,
                                   int64_t seed, int64_t offset, const Tensor& saved, const Tensor& dout, const Tensor& dqkv,
                                   const optional<Tensor>& dweight, const std::vector<optional<Tensor>>& dl, bool accumulate) {
        diff_backward(Operands{qkv, Tensor(), Tensor(), get(weight), {l[0], l[1], l[2], l[3]}},
                      fixed_of(mask, cu, cu, heads, dim, lambda_init, eps, max_len, max_len, p_drop, seed, offset, true), saved, dout,
                      Operands{dqkv, Tensor(), Tensor(), get(dweight), {get(dl[0]), get(dl[1]), get(dl[2]), get(dl[3])}}, accumulate);
    }, unlocked());
}
