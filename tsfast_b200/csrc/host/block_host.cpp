// Host path of the block operators (gated recurrence, block norms, quantised product): argument checks, allocations,
// autograd nodes and the call into the C ABI, for eager PyTorch. A single token's kernel runs for two or three
// microseconds, which is less than the same path costs in Python (17 to 20; the autograd of a small training step 150 more).
//
// The library is not linked: `bind` receives the entry points' addresses from the ctypes handle, so this module calls the
// library that _lib.py loaded, whichever that is. Every failure is a C++ exception, which reaches Python as RuntimeError.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <sstream>

#include "../../../include/b200scan.h"

// the torch and the Python that this is built for: looked for in the built file, which may not load with others
extern "C" __attribute__((used, visibility("default"))) const char b200_host_tag[] = B200_HOST_TAG;

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// ---- the library's entry points
#define B200_ENTRIES(F)                                                                                                      \
    F(b200_gated_chk_rows) F(b200_gated_fwd) F(b200_gated_bwd_workspace_bytes) F(b200_gated_bwd) F(b200_gated_step)          \
    F(b200_block_norm_fwd) F(b200_block_norm_bwd_workspace_bytes) F(b200_block_norm_bwd) F(b200_quant_weight)                \
    F(b200_quant_linear_workspace_bytes) F(b200_quant_linear)
#define DECLARE(name) decltype(&::name) name = nullptr;
struct {
    B200_ENTRIES(DECLARE)
} lib;

void bind(const std::map<std::string, uint64_t>& at) {
#define TAKE(name) lib.name = reinterpret_cast<decltype(&::name)>(at.at(#name));
    B200_ENTRIES(TAKE)
}
std::vector<std::string> entries() {
#define NAME(name) #name,
    return {B200_ENTRIES(NAME)};
}

// ---- refusals
template <typename... A>
[[noreturn]] void refuse(const char* op, const A&... why) {
    std::ostringstream s;
    s << "b200scan::" << op << ": ";
    (s << ... << why);
    throw std::runtime_error(s.str());
}
std::string name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "float32";
        case at::kDouble: return "float64";
        case at::kHalf: return "float16";
        case at::kBFloat16: return "bfloat16";
        case at::kFloat8_e4m3fn: return "float8_e4m3fn";
        case at::kInt: return "int32";
        case at::kLong: return "int64";
        default: return c10::toString(t);
    }
}
struct Say {  // a tensor as a refusal names it
    const Tensor& t;
};
std::ostream& operator<<(std::ostream& s, const Say& v) { return s << v.t.sizes() << " " << name_of(v.t.scalar_type()) << " on " << v.t.device(); }

void check(int status, const char* what) {
    if (status == B200_OK) return;
    static const char* names[] = {"",
                                  "B200_ERR_ARG (bad pointer, size or dtype)",
                                  "B200_ERR_WORKSPACE (workspace missing, misaligned or too small)",
                                  "B200_ERR_LAUNCH (the CUDA runtime refused a memset or launch)",
                                  "B200_ERR_UNSUPPORTED (size outside what the kernel handles)",
                                  "B200_ERR_TIMEOUT (a wait ran out of polls on the device)"};
    throw std::runtime_error(std::string(what) + " failed: " + (status > 0 && status <= 5 ? names[status] : "status " + std::to_string(status)));
}

int tag_of(at::ScalarType t) { return t == at::kFloat ? B200_F32 : t == at::kBFloat16 ? B200_BF16 : t == at::kHalf ? B200_F16 : -1; }

bool has(const Opt& t) { return t.has_value() && t->defined(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor get(const Opt& t) { return has(t) ? *t : Tensor(); }
bool wants(const Opt& t) { return has(t) && t->requires_grad(); }

// the tensors' device for a launch, and its current stream
struct Launch {
    int index, previous;
    explicit Launch(const Tensor& t) : index(t.device().index()), previous(c10::cuda::current_device()) {
        if (previous != index) c10::cuda::set_device(index);
    }
    ~Launch() {
        if (previous != index) (void)c10::cuda::SetDevice(previous);
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(index).stream(); }
};

// Whether somebody has to see the call: a tracer, a dispatch mode, a tensor with a dispatch of its own (a fake one). It is then
// left to the custom op, which goes through the dispatcher; here only the kernels' plain allocations would be seen.
bool recorded(std::initializer_list<const Tensor*> operands) {
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set()) return true;
    for (const Tensor* t : operands)
        if (t->defined() && t->unsafeGetTensorImpl()->is_python_dispatch()) return true;
    return false;
}

// Derivatives and transforms that the operators do not have: without a refusal a dual tensor's tangent would be dropped
void check_plain(const char* op, std::initializer_list<const Tensor*> operands) {
    for (const Tensor* t : operands) {
        if (!t->defined()) continue;
        if (t->key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched})))
            refuse(op, "it does not run inside the transforms of torch.func");
        if (t->_fw_grad(0).defined()) refuse(op, "there is no forward-mode derivative");
    }
}

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::empty(sizes, like.options().dtype(type).memory_format(std::nullopt).requires_grad(false)); }
Tensor workspace(size_t bytes, const Tensor& like) { return empty({(int64_t)std::max<size_t>(bytes, 256)}, at::kByte, like); }
// unit stride along the last axis (a copy only if it is strided)
Tensor unit(const Tensor& t) { return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
Tensor dense(const Tensor& t) { return !t.defined() ? t : t.contiguous(); }

void check_cuda_type(const char* op, const Tensor& x) {
    if (tag_of(x.scalar_type()) < 0) refuse(op, "x is ", name_of(x.scalar_type()), ", the kernel takes float32, bfloat16 or float16");
    if (!x.is_cuda()) refuse(op, "x lives on ", x.device(), ", the kernels only read CUDA memory");
}
void check_like(const char* op, const char* name, const Tensor& t, const Tensor& x) {
    if (t.sizes() != x.sizes() || t.scalar_type() != x.scalar_type() || t.device() != x.device())
        refuse(op, name, " is ", Say{t}, ", expected ", Say{x}, " like x");
}
void check_index(const char* op, const char* name, const Tensor& t, const Tensor& x) {
    if (t.dim() != 1 || (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.device() != x.device())
        refuse(op, name, " is ", Say{t}, ", expected a vector of int32 or int64 on ", x.device());
}
void check_sequences(const char* op, const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& lam, int64_t dims, double c) {
    check_cuda_type(op, x);
    if (x.dim() != dims || x.size(-1) < 1) refuse(op, "x is ", x.sizes(), ", expected ", dims, " axes with at least one channel");
    check_like(op, "r", r, x);
    check_like(op, "i", i, x);
    if (lam.scalar_type() != at::kFloat || lam.device() != x.device() || lam.dim() != 1 || lam.size(0) != x.size(-1))
        refuse(op, "lam is ", Say{lam}, ", expected float32 [", x.size(-1), "] on ", x.device());
    const float c32 = (float)c;  // as the kernels take it
    if (!(c32 > 0) || !std::isfinite(c32)) refuse(op, "c=", c, ", a positive number is needed, in the range of float32");
}

// Gradients that are not differentiable any further: their graph leads back through a node that raises to all that they depend on,
// which are the running node's own operands (those that are not kept for it included) and the upstream gradients.
variable_list once(const char* op, variable_list grads, const variable_list& upstream) {
    if (!at::GradMode::is_enabled()) return grads;
    torch::autograd::edge_list edges;
    if (const auto running = torch::autograd::get_current_node())
        for (const auto& edge : running->next_edges())
            if (edge.is_valid()) edges.push_back(edge);
    for (const auto& g : upstream)
        if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    auto node = std::make_shared<torch::autograd::Error>(std::string("b200scan::") + op + ": there is no second derivative", std::move(edges));
    for (auto& g : grads)
        if (g.defined()) torch::autograd::create_gradient_edge(g, node);
    return grads;
}

// ---------------------------------------------------------------------------------------------- gated recurrence
struct Extents {
    int64_t S, L, T, D;
};
Extents extents(const Tensor& x, const Tensor& cu) {
    if (!cu.defined()) return {x.size(0), x.size(1), 0, x.size(2)};
    return {cu.size(0) - 1, 0, x.size(0), x.size(1)};
}
int64_t batch_stride(const Tensor& t) { return t.dim() == 3 ? t.stride(0) : 0; }

// x, r, i [B, L, D], or [T, D] with cu; returns h, h_last and the kept states (undefined unless `keep`)
std::tuple<Tensor, Tensor, Tensor> gated_forward(const Tensor& x_, const Tensor& r_, const Tensor& i_, const Tensor& lam_, const Opt& h0_,
                                                 const Opt& cu_, double c, bool keep) {
    const char* op = "gated_recurrence";
    check_sequences(op, x_, r_, i_, lam_, has(cu_) ? 2 : 3, c);
    if (has(cu_)) {
        check_index(op, "cu_seqlens", *cu_, x_);
        if (cu_->size(0) < 1) refuse(op, "cu_seqlens needs at least one boundary");
    }
    const Tensor cu = dense(get(cu_)), h0 = dense(get(h0_));
    const Extents e = extents(x_, cu);
    if (h0.defined() && (h0.scalar_type() != at::kFloat || h0.device() != x_.device() || h0.dim() != 2 || h0.size(0) != e.S || h0.size(1) != e.D))
        refuse(op, "h0 is ", Say{h0}, ", expected float32 [", e.S, ", ", e.D, "] on ", x_.device());
    const Tensor x = unit(x_), r = unit(r_), i = unit(i_), lam = dense(lam_);
    const int tag = tag_of(x.scalar_type());
    Launch on(x);
    Tensor h = empty(x.sizes(), x.scalar_type(), x), last = empty({e.S, e.D}, at::kFloat, x), chk;
    if (keep) chk = empty({lib.b200_gated_chk_rows(tag, e.S, e.L, e.T, cu.defined()), e.D}, at::kFloat, x);
    check(lib.b200_gated_fwd(tag, e.S, e.L, e.T, e.D, (float)c, ptr(cu), cu.defined() && cu.scalar_type() == at::kLong, x.data_ptr(), batch_stride(x),
                             x.stride(-2), r.data_ptr(), batch_stride(r), r.stride(-2), i.data_ptr(), batch_stride(i), i.stride(-2), lam.data_ptr(),
                             ptr(h0), h.data_ptr(), last.data_ptr(), ptr(chk), on.stream()),
          "b200_gated_fwd");
    return {h, last, chk};
}

// gradients of x, r, i, lam and (want_h0) h0
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_backward(const Opt& gh_, const Opt& glast_, const Tensor& x_, const Tensor& r_, const Tensor& i_,
                                                                  const Tensor& lam_, const Opt& cu_, const Tensor& chk, double c, bool want_h0) {
    const Tensor x = unit(x_), r = unit(r_), i = unit(i_), lam = dense(lam_), cu = dense(get(cu_)), glast = dense(get(glast_));
    const Extents e = extents(x, cu);
    const int tag = tag_of(x.scalar_type());
    Launch on(x);
    const Tensor gh = has(gh_) ? unit(*gh_) : at::zeros(x.sizes(), x.options().memory_format(std::nullopt));
    Tensor gx = empty(x.sizes(), x.scalar_type(), x), gr = empty(x.sizes(), x.scalar_type(), x), gi = empty(x.sizes(), x.scalar_type(), x);
    Tensor glam = empty({e.D}, at::kFloat, x), gh0 = empty({want_h0 ? e.S : 0, e.D}, at::kFloat, x);
    Tensor ws = workspace(lib.b200_gated_bwd_workspace_bytes(tag, e.S, e.L, e.T, e.D, cu.defined()), x);
    check(lib.b200_gated_bwd(tag, e.S, e.L, e.T, e.D, (float)c, ptr(cu), cu.defined() && cu.scalar_type() == at::kLong, x.data_ptr(), batch_stride(x),
                             x.stride(-2), r.data_ptr(), batch_stride(r), r.stride(-2), i.data_ptr(), batch_stride(i), i.stride(-2), lam.data_ptr(),
                             chk.data_ptr(), gh.data_ptr(), batch_stride(gh), gh.stride(-2), ptr(glast), gx.data_ptr(), gr.data_ptr(), gi.data_ptr(),
                             glam.data_ptr(), want_h0 ? gh0.data_ptr() : nullptr, ws.data_ptr(), ws.numel(), on.stream()),
          "b200_gated_bwd");
    return {gx, gr, gi, glam, gh0};
}

struct GatedNode : Function<GatedNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& lam, const Opt& h0, const Opt& cu,
                                 double c) {
        auto [h, last, chk] = gated_forward(x, r, i, lam, h0, cu, c, true);
        ctx->save_for_backward({x, r, i, lam, get(cu), chk});
        ctx->saved_data["c"] = c;
        ctx->saved_data["h0"] = has(h0);
        ctx->set_materialize_grads(false);
        return {h, last};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const bool h0 = ctx->saved_data["h0"].toBool();
        auto [gx, gr, gi, glam, gh0] = [&] {
            at::NoGradGuard off;
            return gated_backward(g[0], g[1], s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["c"].toDouble(), h0);
        }();
        return once("gated_recurrence", {gx, gr, gi, glam, h0 ? gh0 : Tensor(), Tensor(), Tensor()}, g);
    }
};

// The calls of a user, as those below: nothing where the call is to be recorded
std::optional<std::tuple<Tensor, Tensor>> gated_recurrence(Tensor x, Tensor r, Tensor i, const Tensor& lam, Opt h0, const Opt& cu, double c) {
    const char* op = "gated_recurrence";
    const Tensor h0_ = get(h0), cu_ = get(cu);
    check_plain(op, {&x, &r, &i, &lam, &h0_});
    if (recorded({&x, &r, &i, &lam, &h0_, &cu_})) return {};
    const bool shaped = !has(cu) && x.dim() != 3;
    std::vector<int64_t> lead;
    if (shaped) {  // any number of leading axes, as one
        if (x.dim() < 2) refuse(op, "x is ", x.sizes(), ", expected at least [L, D]");
        const int64_t L = x.size(-2), D = x.size(-1);
        lead = x.sizes().slice(0, x.dim() - 2).vec();
        int64_t n = 1;
        for (int64_t k : lead) n *= k;
        std::vector<int64_t> state = lead;
        state.push_back(D);
        for (auto& [name, t] : {std::pair<const char*, Tensor*>{"r", &r}, {"i", &i}}) {
            if (t->sizes() != x.sizes()) refuse(op, name, " is ", t->sizes(), ", expected ", x.sizes(), " like x");
            *t = t->reshape({n, L, D});
        }
        x = x.reshape({n, L, D});
        if (has(h0)) {
            if (h0->sizes() != at::IntArrayRef(state)) refuse(op, "h0 is ", h0->sizes(), ", expected ", at::IntArrayRef(state));
            h0 = h0->reshape({n, D});
        }
    }
    Tensor h, last;
    if (at::GradMode::is_enabled() && (x.requires_grad() || r.requires_grad() || i.requires_grad() || lam.requires_grad() || wants(h0))) {
        auto out = GatedNode::apply(x, r, i, lam, h0, cu, c);
        h = out[0], last = out[1];
    } else {
        std::tie(h, last, std::ignore) = gated_forward(x, r, i, lam, h0, cu, c, false);
    }
    if (shaped) {
        std::vector<int64_t> rows = lead, state = lead;
        rows.push_back(h.size(1)), rows.push_back(h.size(2)), state.push_back(h.size(2));
        h = h.reshape(rows), last = last.reshape(state);
    }
    return std::tuple(h, last);
}

Tensor gated_step(const Tensor& x_, const Tensor& r_, const Tensor& i_, const Tensor& lam_, Tensor state, const Opt& slots_, double c) {
    const char* op = "gated_recurrence_step";
    check_sequences(op, x_, r_, i_, lam_, 2, c);
    const int64_t B = x_.size(0), D = x_.size(1);
    if (state.scalar_type() != at::kFloat || state.device() != x_.device() || state.dim() != 2 || state.size(1) != D)
        refuse(op, "state is ", Say{state}, ", expected float32 [slots, ", D, "] on ", x_.device());
    const int64_t n = state.size(0);
    if ((D > 1 && state.stride(1) != 1) || (n > 1 && state.stride(0) < D))
        refuse(op, "state is updated in place: rows of unit stride that do not overlap are needed, got strides ", state.strides());
    Tensor slots;
    if (has(slots_)) {
        check_index(op, "slots", *slots_, x_);
        if (slots_->size(0) != B) refuse(op, slots_->size(0), " slots for ", B, " rows");
        slots = slots_->contiguous();
    } else if (n < B) {
        refuse(op, B, " rows and ", n, " states: without slots row b has state b");
    }
    const Tensor x = unit(x_), r = unit(r_), i = unit(i_), lam = dense(lam_);
    state.unsafeGetTensorImpl()->bump_version();  // raises for a tensor of inference mode outside of it: before the update
    Launch on(x);
    Tensor h = empty({B, D}, x.scalar_type(), x);
    check(lib.b200_gated_step(tag_of(x.scalar_type()), B, D, n, (float)c, x.data_ptr(), x.stride(0), r.data_ptr(), r.stride(0), i.data_ptr(), i.stride(0),
                              lam.data_ptr(), state.data_ptr(), std::max(state.stride(0), D), ptr(slots), slots.defined() && slots.scalar_type() == at::kLong,
                              h.data_ptr(), on.stream()),
          "b200_gated_step");
    return h;
}
std::optional<Tensor> gated_recurrence_step(const Tensor& x, const Tensor& r, const Tensor& i, const Tensor& lam, const Tensor& state, const Opt& slots, double c) {
    if (at::GradMode::is_enabled() && (x.requires_grad() || r.requires_grad() || i.requires_grad() || lam.requires_grad() || state.requires_grad()))
        refuse("gated_recurrence_step", "it has no gradient (call it under torch.no_grad(), or train with gated_recurrence)");
    const Tensor at = get(slots);
    check_plain("gated_recurrence_step", {&x, &r, &i, &lam, &state});
    if (recorded({&x, &r, &i, &lam, &state, &at})) return {};
    return gated_step(x, r, i, lam, state, slots, c);
}

// ---------------------------------------------------------------------------------------------- block norms
constexpr int64_t kNormWidth = 8192;
constexpr int kParams = 5;
const char* const kParamNames[kParams] = {"post_weight", "post_bias", "scale", "weight", "bias"};
using Params = std::array<Tensor, kParams>;  // w1, b1, scale, w2, b2

int64_t pitch(const Tensor& t) { return t.defined() ? t.stride(0) : 0; }
int params_f32(const Params& w) { return (w[3].defined() ? w[3] : w[0]).scalar_type() == at::kFloat; }

// without a residual the parameters are those of the gated norm, which calls its own "weight" and "bias"
void check_norm(const char* op, const Tensor& x, const Tensor& residual, const Tensor& gate, const Params& w, int64_t kind, double eps) {
    if (!residual.defined() && (w[2].defined() || w[3].defined())) refuse(op, "residual is required");
    if (!(residual.defined() ? w[3] : w[0]).defined()) refuse(op, "weight is required");
    if (w[1].defined() && !w[0].defined()) refuse(op, "post_bias without post_weight: the norm of x is given by its weight");
    check_cuda_type(op, x);
    const int64_t D = x.dim() ? x.size(-1) : 0;
    if (D < 1 || D > kNormWidth) refuse(op, "rows of ", D, " features, the kernel takes 1 to ", kNormWidth);
    if (residual.defined()) check_like(op, "residual", residual, x);
    if (gate.defined()) check_like(op, "gate", gate, x);
    const bool seam = w[3].defined();
    const Tensor* first = nullptr;
    for (int k = 0; k < kParams; ++k) {
        const Tensor& t = w[k];
        if (!t.defined()) continue;
        const char* name = seam ? kParamNames[k] : kParamNames[k + 3];
        if (t.dim() != 1 || t.size(0) != D || t.device() != x.device() || (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat))
            refuse(op, name, " is ", Say{t}, ", expected [", D, "] of ", name_of(x.scalar_type()), " or float32 on ", x.device());
        if (first != nullptr && t.scalar_type() != first->scalar_type()) refuse(op, name, " is ", name_of(t.scalar_type()), " while other parameters are ", name_of(first->scalar_type()));
        first = &t;
    }
    if (kind == 0 && (w[1].defined() || w[4].defined())) refuse(op, "a bias goes with kind=\"layer\", an RMS norm has none");
    if (!(eps >= 0) || !std::isfinite((float)eps)) refuse(op, "eps=", eps, ", a number that is not negative is needed, in the range of float32");
}

// rows [M, D]; returns y, residual' (undefined without a residual) and the statistics (undefined unless `keep`)
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x_, const Tensor& residual_, const Tensor& gate_, const Params& w_, int64_t kind, int64_t act,
                                                double eps, bool keep) {
    const Tensor x = unit(x_), residual = unit(residual_), gate = unit(gate_);
    Params w;
    for (int k = 0; k < kParams; ++k) w[k] = dense(w_[k]);
    const int64_t M = x.size(0), D = x.size(1);
    Launch on(x);
    Tensor y = empty({M, D}, x.scalar_type(), x), r, stats;
    if (residual.defined()) r = empty({M, D}, x.scalar_type(), x);
    if (keep) stats = empty({M, 4}, at::kFloat, x);
    check(lib.b200_block_norm_fwd(tag_of(x.scalar_type()), M, D, (int)kind, (int)act, (float)eps, params_f32(w), x.data_ptr(), pitch(x), ptr(gate), pitch(gate),
                                  ptr(residual), pitch(residual), ptr(w[0]), ptr(w[1]), ptr(w[2]), ptr(w[3]), ptr(w[4]), y.data_ptr(), ptr(r), ptr(stats),
                                  on.stream()),
          "b200_block_norm_fwd");
    return {y, r, stats};
}

// gradients of x, residual, gate and the parameters, undefined where there is no such operand
std::vector<Tensor> norm_backward(const Tensor& gy_, const Tensor& gr_, const Tensor& x_, const Tensor& residual_, const Tensor& gate_, const Params& w_,
                                  const Tensor& stats, int64_t kind, int64_t act, double eps) {
    const Tensor x = unit(x_), residual = unit(residual_), gate = unit(gate_);
    Launch on(x);
    const Tensor gy = gy_.defined() ? unit(gy_) : at::zeros(x.sizes(), x.options().memory_format(std::nullopt));
    const Tensor gr = residual.defined() ? unit(gr_) : Tensor();
    Params w;
    for (int k = 0; k < kParams; ++k) w[k] = dense(w_[k]);
    const int64_t M = x.size(0), D = x.size(1);
    // where nothing stands between x and the sum, its gradient is the residual's
    const bool bare = residual.defined() && !gate.defined() && !w[0].defined() && !w[2].defined();
    std::vector<Tensor> g(3 + kParams);
    if (!bare) g[0] = empty({M, D}, x.scalar_type(), x);
    if (residual.defined()) g[1] = empty({M, D}, x.scalar_type(), x);
    if (gate.defined()) g[2] = empty({M, D}, x.scalar_type(), x);
    for (int k = 0; k < kParams; ++k)
        if (w[k].defined()) g[3 + k] = empty({D}, w[k].scalar_type(), x);
    Tensor ws = workspace(lib.b200_block_norm_bwd_workspace_bytes(M, D, (int)kind), x);
    check(lib.b200_block_norm_bwd(tag_of(x.scalar_type()), M, D, (int)kind, (int)act, (float)eps, params_f32(w), gy.data_ptr(), pitch(gy), ptr(gr), pitch(gr),
                                  x.data_ptr(), pitch(x), ptr(gate), pitch(gate), ptr(residual), pitch(residual), ptr(w[0]), ptr(w[1]), ptr(w[2]), ptr(w[3]),
                                  ptr(w[4]), stats.data_ptr(), ptr(g[0]), ptr(g[2]), ptr(g[1]), ptr(g[3]), ptr(g[4]), ptr(g[5]), ptr(g[6]), ptr(g[7]),
                                  ws.data_ptr(), ws.numel(), on.stream()),
          "b200_block_norm_bwd");
    if (bare) g[0] = g[1];
    return g;
}

struct NormNode : Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Opt& residual, const Opt& gate, const Opt& w1, const Opt& b1, const Opt& scale,
                                 const Opt& w2, const Opt& b2, int64_t kind, int64_t act, double eps) {
        const Params w = {get(w1), get(b1), get(scale), get(w2), get(b2)};
        auto [y, r, stats] = norm_forward(x, get(residual), get(gate), w, kind, act, eps, true);
        ctx->save_for_backward({x, get(residual), get(gate), w[0], w[1], w[2], w[3], w[4], stats});
        ctx->saved_data["kind"] = kind, ctx->saved_data["act"] = act, ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        if (r.defined()) return {y, r};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        variable_list grads;
        {
            at::NoGradGuard off;
            grads = norm_backward(g[0], g.size() > 1 ? g[1] : Tensor(), s[0], s[1], s[2], {s[3], s[4], s[5], s[6], s[7]}, s[8], ctx->saved_data["kind"].toInt(),
                                  ctx->saved_data["act"].toInt(), ctx->saved_data["eps"].toDouble());
        }
        for (int k = 0; k < 3; ++k) grads.emplace_back();
        return once("block_norm", grads, g);
    }
};

// the whole operator over [..., D]; without a residual the second result is undefined
std::optional<std::tuple<Tensor, Opt>> block_norm(const char* op, const Tensor& x, const Opt& residual, const Opt& gate, const Opt& w1, const Opt& b1, const Opt& scale,
                                   const Opt& w2, const Opt& b2, int64_t kind, int64_t act, double eps) {
    const Params w = {get(w1), get(b1), get(scale), get(w2), get(b2)};
    const Tensor residual_ = get(residual), gate_ = get(gate);
    check_plain(op, {&x, &residual_, &gate_, &w[0], &w[1], &w[2], &w[3], &w[4]});
    if (recorded({&x, &residual_, &gate_, &w[0], &w[1], &w[2], &w[3], &w[4]})) return {};
    check_norm(op, x, residual_, gate_, w, kind, eps);
    const bool flat = x.dim() == 2;
    const int64_t D = x.size(-1);
    auto rows = [&](const Opt& t) -> Opt { return !has(t) ? Opt() : flat ? t : Opt(t->reshape({x.numel() / D, D})); };
    const Tensor x2 = flat ? x : *rows(x);
    Tensor y, r;
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants(residual) || wants(gate) || wants(w1) || wants(b1) || wants(scale) || wants(w2) || wants(b2))) {
        auto out = NormNode::apply(x2, rows(residual), rows(gate), w1, b1, scale, w2, b2, kind, act, eps);
        y = out[0];
        if (out.size() > 1) r = out[1];
    } else {
        std::tie(y, r, std::ignore) = norm_forward(x2, get(rows(residual)), get(rows(gate)), w, kind, act, eps, false);
    }
    if (!flat) {
        y = y.reshape(x.sizes());
        if (r.defined()) r = r.reshape(x.sizes());
    }
    return std::tuple(y, r.defined() ? Opt(r) : Opt());
}

std::optional<Tensor> gated_norm(const Tensor& x, const Opt& gate, const Opt& weight, const Opt& bias, int64_t kind, int64_t act, double eps) {
    const auto out = block_norm("gated_norm", x, {}, gate, weight, bias, {}, {}, {}, kind, act, eps);
    return out ? std::optional(std::get<0>(*out)) : std::nullopt;
}
std::optional<std::tuple<Tensor, Opt>> residual_norm(const Tensor& x, const Opt& residual, const Opt& weight, const Opt& bias, const Opt& gate,
                                                     const Opt& scale, const Opt& post_weight, const Opt& post_bias, int64_t kind, int64_t act, double eps) {
    if (!has(residual)) refuse("residual_norm", "residual is required");  // (else it might pass for a gated norm)
    return block_norm("residual_norm", x, residual, gate, post_weight, post_bias, scale, weight, bias, kind, act, eps);
}

// ---------------------------------------------------------------------------------------------- quantised product
constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

std::tuple<Tensor, Tensor> quant_weight(const Tensor& w_) {
    const char* op = "quantize_weight";
    const int tag = tag_of(w_.scalar_type());
    if (tag < 0 || !w_.is_cuda() || w_.dim() != 2 || w_.numel() == 0)
        refuse(op, "w is ", Say{w_}, ", expected a float32, bfloat16 or float16 CUDA matrix [N, K]");
    const Tensor w = unit(w_.detach());
    const int64_t N = w.size(0), K = w.size(1);
    Launch on(w);
    Tensor q = at::zeros({N, blocks(K) * kBlock}, w.options().dtype(at::kByte).memory_format(std::nullopt)).view(at::kFloat8_e4m3fn).narrow(1, 0, K);
    Tensor scale = empty({blocks(N), blocks(K)}, at::kFloat, w);
    check(lib.b200_quant_weight(tag, N, K, w.data_ptr(), w.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), on.stream()), "b200_quant_weight");
    return {q, scale};
}

std::optional<std::tuple<Tensor, Tensor>> quantize_weight(const Tensor& w) {
    if (recorded({&w})) return {};
    return quant_weight(w);
}

// where TMA can read it: unit column stride, a row pitch that is a multiple of 16, a 16-byte aligned base; else a copy
Tensor readable(const Tensor& q) {
    const int64_t N = q.size(0), K = q.size(1);
    if ((q.stride(1) == 1 || K == 1) && q.stride(0) % 16 == 0 && q.stride(0) >= K && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0) return q;
    Tensor copy = empty({N, blocks(K) * kBlock}, at::kByte, q).view(at::kFloat8_e4m3fn).narrow(1, 0, K);
    copy.copy_(q);
    return copy;
}

Tensor quant_product(const Tensor& x_, const Tensor& q_, const Tensor& scale_, const Opt& bias_) {
    const char* op = "quant_linear";
    if ((x_.scalar_type() != at::kBFloat16 && x_.scalar_type() != at::kHalf) || !x_.is_cuda() || x_.dim() < 1)
        refuse(op, "x is ", Say{x_}, ", expected bfloat16 or float16 [..., K] in CUDA memory");
    if (q_.scalar_type() != at::kFloat8_e4m3fn || q_.device() != x_.device() || q_.dim() != 2 || q_.numel() == 0 || q_.size(1) != x_.size(-1))
        refuse(op, "q is ", Say{q_}, ", expected float8_e4m3fn [N, ", x_.size(-1), "] on ", x_.device());
    const int64_t N = q_.size(0), K = q_.size(1);
    if (scale_.scalar_type() != at::kFloat || scale_.device() != x_.device() || scale_.dim() != 2 || scale_.size(0) != blocks(N) || scale_.size(1) != blocks(K))
        refuse(op, "scale is ", Say{scale_}, ", expected float32 [", blocks(N), ", ", blocks(K), "] on ", x_.device());
    const Tensor bias = dense(get(bias_));
    if (bias.defined() && ((bias.scalar_type() != x_.scalar_type() && bias.scalar_type() != at::kFloat) || bias.device() != x_.device() || bias.dim() != 1 ||
                           bias.size(0) != N))
        refuse(op, "bias is ", Say{bias}, ", expected [", N, "] of ", name_of(x_.scalar_type()), " or float32 on ", x_.device());
    const int64_t M = x_.numel() / K;
    const bool flat = x_.dim() == 2;
    const Tensor x = unit(flat ? x_ : x_.reshape({M, K})), q = readable(q_), scale = dense(scale_);
    Launch on(x);
    Tensor y = empty({M, N}, x.scalar_type(), x);
    Tensor ws = workspace(lib.b200_quant_linear_workspace_bytes(M, N, K), x);
    check(lib.b200_quant_linear(tag_of(x.scalar_type()), M, N, K, x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), ptr(bias),
                                bias.defined() && bias.scalar_type() == at::kFloat, y.data_ptr(), N, ws.data_ptr(), ws.numel(), on.stream()),
          "b200_quant_linear");
    if (flat) return y;
    std::vector<int64_t> shape = x_.sizes().vec();
    shape.back() = N;
    return y.reshape(shape);
}
std::optional<Tensor> quant_linear(const Tensor& x, const Tensor& q, const Tensor& scale, const Opt& bias) {
    if (at::GradMode::is_enabled() && (x.requires_grad() || scale.requires_grad() || wants(bias)))
        refuse("quant_linear", "it has no gradient (call it under torch.no_grad())");
    const Tensor b = get(bias);
    check_plain("quant_linear", {&x, &q, &scale, &b});
    if (recorded({&x, &q, &scale, &b})) return {};
    return quant_product(x, q, scale, bias);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("bind", &bind);
    m.def("entries", &entries);
    m.def("gated_recurrence", &gated_recurrence);
    m.def("gated_forward", &gated_forward);
    m.def("gated_backward", &gated_backward);
    m.def("gated_recurrence_step", &gated_recurrence_step);
    m.def("gated_step", &gated_step);
    m.def("gated_norm", &gated_norm);
    m.def("residual_norm", &residual_norm);
    m.def("check_norm", [](const std::string& op, const Tensor& x, const Opt& residual, const Opt& gate, const std::vector<Opt>& w, int64_t kind, double eps) {
        check_norm(op.c_str(), x, get(residual), get(gate), {get(w[0]), get(w[1]), get(w[2]), get(w[3]), get(w[4])}, kind, eps);
    });
    m.def("norm_forward", [](const Tensor& x, const Opt& residual, const Opt& gate, const std::vector<Opt>& w, int64_t kind, int64_t act, double eps) {
        return norm_forward(x, get(residual), get(gate), {get(w[0]), get(w[1]), get(w[2]), get(w[3]), get(w[4])}, kind, act, eps, true);
    });
    m.def("norm_backward", [](const Opt& gy, const Opt& gr, const Tensor& x, const Opt& residual, const Opt& gate, const std::vector<Opt>& w, const Tensor& stats,
                              int64_t kind, int64_t act, double eps) {
        return norm_backward(get(gy), get(gr), x, get(residual), get(gate), {get(w[0]), get(w[1]), get(w[2]), get(w[3]), get(w[4])}, stats, kind, act, eps);
    });
    m.def("quantize_weight", &quantize_weight);
    m.def("quant_weight", &quant_weight);
    m.def("quant_linear", &quant_linear);
    m.def("quant_product", &quant_product);
}
