// The host side of the operators whose calls are short beside what Python costs around them: group normalisation, distillation, the
// relative position bias and the norms around a residual sum with their autograd
// nodes (a backward pass in Python waits for the interpreter on the engine's thread: 118 us for two launches of 10 us each), the
// global norm, and the walk over an optimizer's variables (28 variables: 34 us in Python).  Arguments are checked here, the kernels are
// called through the C ABI of libhgq_hip.so (bind()), outputs and workspaces are torch tensors on the current stream of their device.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>

#include "../../include/hgq_hip.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Library {  // the entry points that are called from here
    decltype(&hgq_last_error) last_error;
    decltype(&hgq_global_norm_parts) global_norm_parts;
    decltype(&hgq_global_norm) global_norm;
    decltype(&hgq_adamw_update_multi) adamw_update_multi;
    decltype(&hgq_group_norm_fwd_workspace) group_norm_fwd_workspace;
    decltype(&hgq_group_norm_fwd) group_norm_fwd;
    decltype(&hgq_group_norm_bwd_workspace) group_norm_bwd_workspace;
    decltype(&hgq_group_norm_bwd) group_norm_bwd;
    decltype(&hgq_distill_topk_workspace) distill_topk_workspace;
    decltype(&hgq_distill_topk_fwd) distill_topk_fwd;
    decltype(&hgq_distill_topk_bwd) distill_topk_bwd;
    decltype(&hgq_relative_bias_fwd) relative_bias_fwd;
    decltype(&hgq_relative_bias_bwd_workspace) relative_bias_bwd_workspace;
    decltype(&hgq_relative_bias_bwd) relative_bias_bwd;
    decltype(&hgq_residual_norm_fwd) residual_norm_fwd;
    decltype(&hgq_residual_norm_bwd_workspace) residual_norm_bwd_workspace;
    decltype(&hgq_residual_norm_bwd) residual_norm_bwd;
} lib;
PyObject *library_error = nullptr;  // hgq2_amd._lib.HGQLibraryError

std::atomic<bool> bound{false};

[[noreturn]] void rethrow(py::error_already_set &error) {  // as the Python exception that it is
    error.restore();
    python_error e;
    e.persist();
    throw e;
}

const Library &library() {
    if (!bound) {  // an operator called by its name alone, before anything else asked for the library
        const py::gil_scoped_acquire gil;
        try {
            py::module_::import("hgq2_amd._lib").attr("native")();
        } catch (py::error_already_set &e) {
            rethrow(e);
        }
    }
    return lib;
}

void check(int rc, const char *what) {
    if (rc == 0) return;
    const std::string message = std::string(what) + " failed with " + std::to_string(rc) + ": " + lib.last_error();
    const py::gil_scoped_acquire gil;  // (also called from the autograd engine's threads)
    PyErr_SetString(library_error, message.c_str());
    python_error e;
    e.persist();
    throw e;
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int type_code(at::ScalarType t) { return t == at::kFloat ? HGQ_TYPE_F32 : t == at::kBFloat16 ? HGQ_TYPE_BF16 : t == at::kHalf ? HGQ_TYPE_F16 : -1; }

float *floats(const Tensor &t) { return t.numel() ? t.data_ptr<float>() : nullptr; }

void *memory(const Tensor &t) { return t.numel() ? t.data_ptr() : nullptr; }

Tensor vector_like(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// A call's scratch memory on the current stream of the current device: the allocator hands it to later work of that stream only, and
// under capture it belongs to the graph.  (A tensor takes 1 us to make, this a quarter of that.)
template <typename T>
struct Workspace {
    c10::DataPtr memory;
    explicit Workspace(int64_t n) {
        if (n > 0) memory = c10::hip::HIPCachingAllocator::get()->allocate((size_t)n * sizeof(T));
    }
    T *get() const { return (T *)memory.get(); }
};

// ---- group normalisation ---------------------------------------------------------------------------------------------
struct GroupSizes {
    int64_t B, S, C;
    int G, type;
};

GroupSizes group_sizes(const Tensor &x, int64_t groups) {
    TORCH_CHECK_VALUE(x.is_cuda(), "x must be a GPU tensor (there is no CPU implementation), got device ", x.device());
    const int type = type_code(x.scalar_type());
    TORCH_CHECK_VALUE(type >= 0, "x must be float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 2 && x.size(-1) >= 1, "x must be [batch, ..., channels], got ", x.sizes());
    TORCH_CHECK_VALUE(x.is_contiguous(), "x must be contiguous");
    TORCH_CHECK_VALUE(groups >= 1 && x.size(-1) % groups == 0 && x.size(-1) <= INT32_MAX, x.size(-1), " channels do not fall into ", groups, " groups of one size");
    int64_t S = 1;
    for (int64_t d = 1; d + 1 < x.dim(); ++d) S *= x.size(d);
    return {x.size(0), S, x.size(-1), (int)groups, type};
}

void channel_vector(const char *name, const Tensor &t, const Tensor &x) {  // (empty: none)
    TORCH_CHECK_VALUE(t.numel() == 0 || (t.numel() == x.size(-1) && t.scalar_type() == at::kFloat && t.device() == x.device() && t.is_contiguous()), name,
                      " must be a contiguous float32 tensor of ", x.size(-1), " elements on ", x.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}

std::tuple<Tensor, Tensor> group_norm_fwd(const Tensor &x, const Tensor &gamma, const Tensor &beta, int64_t groups, double epsilon, int64_t act) {
    const GroupSizes s = group_sizes(x, groups);
    channel_vector("gamma", gamma, x), channel_vector("beta", beta, x);
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty_like(x), stats = at::empty({2, s.B, s.G}, x.options().dtype(at::kDouble));
    const Workspace<float> ws(library().group_norm_fwd_workspace(s.B, s.S, (int)s.C, s.G, s.type));
    double *mean = (double *)memory(stats);
    check(lib.group_norm_fwd(memory(x), floats(gamma), floats(beta), memory(y), mean, mean ? mean + s.B * s.G : nullptr, ws.get(),
                             s.B, s.S, (int)s.C, s.G, (float)epsilon, (int)act, s.type, stream_of(x)),
          "hgq_group_norm_fwd");
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> group_norm_bwd(const Tensor &dy, const Tensor &x, const Tensor &gamma, const Tensor &beta, const Tensor &stats,
                                                  int64_t groups, int64_t act, bool need_dx, bool need_dgamma, bool need_dbeta) {
    const GroupSizes s = group_sizes(x, groups);
    channel_vector("gamma", gamma, x), channel_vector("beta", beta, x);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device() && dy.is_contiguous(),
                      "dy must be contiguous and like x, got ", dy.scalar_type(), " ", dy.sizes(), " on ", dy.device());
    TORCH_CHECK_VALUE(stats.numel() == 2 * s.B * s.G && stats.scalar_type() == at::kDouble && stats.device() == x.device() && stats.is_contiguous(),
                      "stats must be what the forward call left");
    const c10::DeviceGuard guard(x.device());
    Tensor dx = need_dx ? at::empty_like(x) : at::empty({0}, x.options()), dgamma = vector_like(need_dgamma ? s.C : 0, x),
           dbeta = vector_like(need_dbeta ? s.C : 0, x);
    const Workspace<float> ws(library().group_norm_bwd_workspace(s.B, s.S, (int)s.C, s.G, s.type));
    const double *mean = (const double *)memory(stats);
    check(lib.group_norm_bwd(memory(dy), memory(x), floats(gamma), floats(beta), mean, mean ? mean + s.B * s.G : nullptr, memory(dx), floats(dgamma),
                             floats(dbeta), ws.get(), s.B, s.S, (int)s.C, s.G, (int)act, s.type, stream_of(x)),
          "hgq_group_norm_bwd");
    return {dx, dgamma, dbeta};
}

// Gradients that were asked for with create_graph: usable as they are, and refused where they are to be differentiated again (without
// this they would pass for constants).
struct OnceOnly : torch::autograd::Function<OnceOnly> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *, const Tensor &dx, const Tensor &dg, const Tensor &db, const Tensor &,
                                                  const Tensor &, const Tensor &, const Tensor &) {
        return {dx.view_as(dx), dg.view_as(dg), db.view_as(db)};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *, const torch::autograd::variable_list &) {
        TORCH_CHECK(false, "group_norm is differentiable once: its gradients have no gradient");
    }
};

// (through the dispatcher, so that fake tensors and tracing see the two operators)
const auto &forward_op() {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::group_norm_fwd", "").typed<decltype(group_norm_fwd)>();
    return op;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &gamma, const Tensor &beta, int64_t groups, double epsilon,
                          int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, stats] = forward_op().call(x, gamma, beta, groups, epsilon, act);
        ctx->save_for_backward({x, gamma, beta, stats});
        ctx->saved_data["groups"] = groups, ctx->saved_data["act"] = act;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::group_norm_bwd", "").typed<decltype(group_norm_bwd)>();
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gamma = saved[1], &beta = saved[2], &stats = saved[3];
        const bool wx = ctx->needs_input_grad(0), wg = ctx->needs_input_grad(1), wb = ctx->needs_input_grad(2);
        Tensor dx, dg, db;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            std::tie(dx, dg, db) = op.call(grads[0].contiguous(), x, gamma, beta, stats, ctx->saved_data["groups"].toInt(), ctx->saved_data["act"].toInt(), wx, wg, wb);
        }
        if (at::GradMode::is_enabled()) {
            const auto once = OnceOnly::apply(dx, dg, db, grads[0], x, gamma, beta);
            dx = once[0], dg = once[1], db = once[2];
        }
        return {wx ? dx : Tensor(), wg ? dg : Tensor(), wb ? db : Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// A recorded backward pass hands the gradient of a leaf to the leaf's one accumulating node, on the stream that the node was made on.  One that
// an earlier graph made on another stream, and keeps alive, would pull that stream into the recording, which ends the process.
bool accumulates_elsewhere(const Tensor &t) {
    if (!t.defined() || !t.requires_grad() || t.grad_fn()) return false;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    return stream && stream->id() != c10::hip::getCurrentHIPStream(t.device().index()).id();
}

void accumulates_here(const char *name, const Tensor &t) {
    if (!accumulates_elsewhere(t)) return;
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None, name,
                " belongs to a graph of another stream that is still alive: its backward pass cannot be recorded here (release what that graph gave, or "
                "make it on this stream)");
}

Tensor group_norm(const Tensor &x, int64_t groups, const std::optional<Tensor> &gamma, const std::optional<Tensor> &beta, double epsilon, int64_t act) {
    for (const auto &[name, t] : {std::make_pair("gamma", &gamma), std::make_pair("beta", &beta)})
        TORCH_CHECK_VALUE(!*t || ((*t)->dim() == 1 && x.dim() >= 1 && (*t)->numel() == x.size(-1)), name, " must be a vector with an element per channel");
    const auto differentiated = [](const Tensor &t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); };
    const bool graph = differentiated(x) || (gamma && differentiated(*gamma)) || (beta && differentiated(*beta));
    if (graph) {
        accumulates_here("x", x);
        if (gamma) accumulates_here("gamma", *gamma);
        if (beta) accumulates_here("beta", *beta);
    }
    const Tensor none = gamma && beta ? Tensor() : at::empty({0}, x.options().dtype(at::kFloat).requires_grad(false));
    const Tensor &ga = gamma ? *gamma : none, &be = beta ? *beta : none;
    if (graph) return GroupNorm::apply(x.contiguous(), ga, be, groups, epsilon, act);
    at::AutoDispatchBelowADInplaceOrView below;  // (no node to make)
    return std::get<0>(forward_op().call(x.contiguous(), ga, be, groups, epsilon, act));
}

// ---- what the three operators below share --------------------------------------------------------------------------------
void on_gpu(const char *name, const Tensor &t) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU tensor (there is no CPU implementation), got device ", t.device());
    TORCH_CHECK_VALUE(type_code(t.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

// float32 numbers, `n` of them (empty: none)
void numbers(const char *name, const Tensor &t, int64_t n, const Tensor &like) {
    TORCH_CHECK_VALUE(t.numel() == 0 || (t.numel() == n && t.scalar_type() == at::kFloat && t.device() == like.device() && t.is_contiguous()), name,
                      " must be a contiguous float32 tensor of ", n, " elements on ", like.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}

// (0.5 us less than empty_like takes)
Tensor whole_like(const Tensor &t) { return at::empty(t.sizes(), t.options()); }

bool differentiated(const Tensor &t) { return t.defined() && ((t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined()); }

Tensor plain(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// What is not given goes without a tensor (an empty one takes 1 us to make); the operators take an empty one for the same.
using Maybe = std::optional<Tensor>;

Tensor given(const Maybe &t) { return t ? *t : Tensor(); }

// Gradients asked for with create_graph, of any operator: see OnceOnly.
struct AllOnceOnly : torch::autograd::Function<AllOnceOnly> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, at::TensorList grads, at::TensorList inputs, std::string what) {
        ctx->saved_data["what"] = what;
        torch::autograd::variable_list out;
        for (const Tensor &g : grads) out.push_back(g.view_as(g));
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &) {
        TORCH_CHECK(false, ctx->saved_data["what"].toStringRef(), " is differentiable once: its gradients have no gradient");
    }
};

void once_only(torch::autograd::variable_list &grads, const std::vector<Tensor> &inputs, const char *what) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::variable_list there, from;
    for (const Tensor &g : grads)
        if (g.defined()) there.push_back(g);
    for (const Tensor &t : inputs)
        if (t.defined()) from.push_back(t);
    if (there.empty()) return;
    const auto out = AllOnceOnly::apply(at::TensorList(there), at::TensorList(from), std::string(what));
    size_t k = 0;
    for (Tensor &g : grads)
        if (g.defined()) g = out[k++];
}

// ---- distillation from a teacher's top logits --------------------------------------------------------------------------
struct DistillSizes {
    int64_t rows, V, K;
    int type, t_type, index_bytes;
};

DistillSizes distill_sizes(const Tensor &z, const Tensor &t, const Tensor &index, const Tensor &lse, const Tensor &weight, double T) {
    on_gpu("logits", z), on_gpu("teacher_logits", t);
    TORCH_CHECK_VALUE(z.dim() == 2 && t.dim() == 2 && t.size(0) == z.size(0), "logits [rows, vocabulary] and teacher_logits [rows, entries] expected, got ", z.sizes(), " and ", t.sizes());
    TORCH_CHECK_VALUE(z.size(1) >= 1 && t.size(1) >= 1, "logits and teacher_logits must have entries, got ", z.sizes(), " and ", t.sizes());
    TORCH_CHECK_VALUE((z.stride(1) == 1 || z.size(1) == 1) && z.stride(0) >= 0, "rows of logits must be contiguous");
    TORCH_CHECK_VALUE(index.sizes() == t.sizes() && (index.scalar_type() == at::kInt || index.scalar_type() == at::kLong), "teacher_indices must be int32 or int64 and like teacher_logits, got ",
                      index.scalar_type(), " ", index.sizes());
    TORCH_CHECK_VALUE(t.device() == z.device() && index.device() == z.device(), "logits and the teacher's list must be on one device");
    TORCH_CHECK_VALUE(t.is_contiguous() && index.is_contiguous(), "the teacher's list must be contiguous");
    numbers("teacher_lse", lse, z.size(0), z), numbers("sample_weight", weight, z.size(0), z);
    TORCH_CHECK_VALUE(T >= 1e-30 && T <= 1e30, "temperature must be positive, 1e-30 .. 1e30, got ", T);
    return {z.size(0), z.size(1), t.size(1), type_code(z.scalar_type()), type_code(t.scalar_type()), index.scalar_type() == at::kLong ? 8 : 4};
}

// stats and dz: where the gradient is wanted
Tensor distill_forward(const Tensor &z, const Tensor &t, const Tensor &index, const Tensor &lse, const Tensor &weight, double T, Tensor *stats, Tensor *dz) {
    const DistillSizes s = distill_sizes(z, t, index, lse, weight, T);
    const c10::DeviceGuard guard(z.device());
    const auto options = z.options().dtype(at::kFloat);
    Tensor loss = at::empty({}, options);
    if (stats) *stats = at::empty({s.rows, 4}, options), *dz = at::empty({s.rows, s.V}, z.options());
    const Workspace<float> ws(library().distill_topk_workspace(s.rows, s.V, s.K, lse.numel() > 0));
    check(lib.distill_topk_fwd(memory(z), z.stride(0), memory(t), s.t_type, memory(index), s.index_bytes, floats(lse), floats(weight), loss.data_ptr<float>(),
                               stats ? floats(*stats) : nullptr, dz ? memory(*dz) : nullptr, ws.get(), s.rows, s.V, s.K, T, s.type, stream_of(z)),
          "hgq_distill_topk_fwd");
    return loss;
}

std::tuple<Tensor, Tensor, Tensor> distill_topk_fwd(const Tensor &z, const Tensor &t, const Tensor &index, const Maybe &lse, const Maybe &weight, double T) {
    Tensor stats, dz, loss = distill_forward(z, t, index, given(lse), given(weight), T, &stats, &dz);
    return {loss, stats, dz};
}

Tensor distill_topk_loss(const Tensor &z, const Tensor &t, const Tensor &index, const Maybe &lse, const Maybe &weight, double T) {
    return distill_forward(z, t, index, given(lse), given(weight), T, nullptr, nullptr);
}

void distill_backward(const Tensor &up, const Tensor &z, const Tensor &t, const Tensor &index, const Tensor &lse, const Tensor &weight, const Tensor &stats, const Tensor &dz, bool holds_unit,
                      double T) {
    const DistillSizes s = distill_sizes(z, t, index, lse, weight, T);
    TORCH_CHECK_VALUE(up.numel() == 1 && up.scalar_type() == at::kFloat && up.device() == z.device(), "the loss' gradient must be one float32 on ", z.device());
    TORCH_CHECK_VALUE(stats.numel() == 4 * s.rows && stats.scalar_type() == at::kFloat && stats.device() == z.device() && stats.is_contiguous(), "stats must be what the forward call left");
    TORCH_CHECK_VALUE(dz.sizes() == z.sizes() && dz.scalar_type() == z.scalar_type() && dz.device() == z.device() && dz.is_contiguous(), "the logits' gradient must be contiguous and like them");
    const c10::DeviceGuard guard(z.device());
    check(library().distill_topk_bwd(memory(z), z.stride(0), memory(t), s.t_type, memory(index), s.index_bytes, floats(lse), floats(weight), up.data_ptr<float>(), floats(stats), memory(dz),
                                     holds_unit, s.rows, s.V, s.K, T, s.type, stream_of(z)),
          "hgq_distill_topk_bwd");
}

Tensor distill_topk_bwd(const Tensor &up, const Tensor &z, const Tensor &t, const Tensor &index, const Maybe &lse, const Maybe &weight, const Tensor &stats, double T) {
    on_gpu("logits", z);
    Tensor dz = at::empty(z.sizes(), z.options());
    distill_backward(up, z, t, index, given(lse), given(weight), stats, dz, false, T);
    return dz;
}

// `dz`: the gradient for an upstream of one, which is left as it is where the upstream is one
void distill_topk_bwd_(const Tensor &up, const Tensor &z, const Tensor &t, const Tensor &index, const Maybe &lse, const Maybe &weight, const Tensor &stats, double T, Tensor dz) {
    distill_backward(up, z, t, index, given(lse), given(weight), stats, dz, true, T);
}

// The forward pass writes the gradient for an upstream of one while the row is at hand.  The backward pass hands it on where the upstream is one - the
// kernel that looks at it ends at once - and forms it anew elsewhere, so there is one rounding whatever the upstream (a loss scaled
// for float16 gets the gradients it was scaled for).  A graph that is kept may be asked again: it gets a tensor of its own each time.
struct DistillTopk : torch::autograd::Function<DistillTopk> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &z, const Tensor &t, const Tensor &index, const Maybe &lse, const Maybe &weight, double T) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::distill_topk_fwd", "").typed<decltype(distill_topk_fwd)>();
        at::AutoDispatchBelowADInplaceOrView below;
        auto [loss, stats, dz] = op.call(z, t, index, lse, weight, T);
        ctx->save_for_backward({z, t, index, given(lse), given(weight), stats, dz});
        ctx->saved_data["T"] = T;
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        static const auto anew = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::distill_topk_bwd", "").typed<decltype(distill_topk_bwd)>();
        static const auto over = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::distill_topk_bwd_", "").typed<decltype(distill_topk_bwd_)>();
        const auto saved = ctx->get_saved_variables();
        torch::autograd::variable_list out(6);
        if (!ctx->needs_input_grad(0)) return out;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const Tensor up = plain(grads[0]).to(at::kFloat);
            const Maybe lse = saved[3].defined() ? Maybe(saved[3]) : Maybe(), weight = saved[4].defined() ? Maybe(saved[4]) : Maybe();
            if (torch::autograd::get_current_graph_task_keep_graph()) {
                out[0] = anew.call(up, saved[0], saved[1], saved[2], lse, weight, saved[5], ctx->saved_data["T"].toDouble());
            } else {
                out[0] = saved[6];
                over.call(up, saved[0], saved[1], saved[2], lse, weight, saved[5], ctx->saved_data["T"].toDouble(), out[0]);
            }
        }
        once_only(out, {grads[0], saved[0]}, "distill_topk");
        return out;
    }
};

Tensor distill_topk(const Tensor &logits, const Tensor &teacher, const Tensor &indices, double T, const std::optional<Tensor> &lse, const std::optional<Tensor> &weight) {
    const auto lead = [](const Tensor &t) { return t.sizes().slice(0, t.dim() - 1); };
    TORCH_CHECK_VALUE(logits.dim() >= 1 && teacher.dim() == logits.dim() && lead(teacher) == lead(logits), "teacher_logits must have the logits' leading axes, got ", teacher.sizes(), " for ", logits.sizes());
    TORCH_CHECK_VALUE(indices.sizes() == teacher.sizes(), "teacher_indices must be like teacher_logits, got ", indices.sizes(), " for ", teacher.sizes());
    for (const auto &[name, t] : {std::make_pair("teacher_lse", &lse), std::make_pair("sample_weight", &weight)})
        TORCH_CHECK_VALUE(!*t || (*t)->sizes() == lead(logits), name, " must have an element per row of logits, got ", (*t)->sizes(), " for ", logits.sizes());
    TORCH_CHECK_VALUE(!differentiated(teacher) && !(lse && differentiated(*lse)) && !(weight && differentiated(*weight)), "distill_topk is differentiable in the logits alone: detach the teacher's tensors and the weights");
    const bool graph = differentiated(logits);
    if (graph) accumulates_here("logits", logits);
    const int64_t V = logits.size(-1), K = teacher.size(-1);
    int64_t rows = 1;
    for (const int64_t n : lead(logits)) rows *= n;
    Tensor z = logits.dim() == 2 ? logits : logits.reshape({rows, V});
    if ((V > 1 && z.stride(1) != 1) || z.stride(0) < 0 || z.is_neg()) z = z.contiguous().resolve_neg();
    const auto flat = [rows](const Tensor &t, int64_t n) { return plain(t.detach()).reshape({rows, n}).contiguous(); };
    const Tensor t = flat(teacher, K), i = flat(indices, K);
    const Maybe l = lse ? Maybe(flat(*lse, 1)) : Maybe(), w = weight ? Maybe(flat(*weight, 1)) : Maybe();
    if (graph) return DistillTopk::apply(z, t, i, l, w, T);
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::distill_topk_loss", "").typed<decltype(distill_topk_loss)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(z, t, i, l, w, T);
}

// ---- relative position bias ----------------------------------------------------------------------------------------------
struct BiasSizes {
    int64_t B, H, T, S;
    int type, m;
    std::vector<int> first;
};

bool whole_planes(const Tensor &t) {
    return t.numel() == 0 || ((t.size(3) == 1 || t.stride(3) == 1) && (t.size(2) == 1 || t.stride(2) == t.size(3)) && t.stride(0) >= 0 && t.stride(1) >= 0);
}

// one for each of the batch
void offsets_fit(const Tensor &offsets, int64_t B, c10::Device device) {
    TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) == B && offsets.device() == device && offsets.is_contiguous() &&
                          (offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong),
                      "offset must be a number, or a contiguous int32 or int64 tensor with one for each of the batch on ", device, ", got ", offsets.scalar_type(), " ", offsets.sizes());
}

BiasSizes bias_sizes(const char *name, const Tensor &x, const Tensor &offsets, at::IntArrayRef first) {
    on_gpu(name, x);
    TORCH_CHECK_VALUE(x.dim() == 4, name, " must be [batch, heads, queries, keys], got ", x.sizes());
    TORCH_CHECK_VALUE(whole_planes(x), name, ": a head's queries and keys must be contiguous");
    if (offsets.numel()) offsets_fit(offsets, x.size(0), x.device());
    BiasSizes s = {x.size(0), x.size(1), x.size(2), x.size(3), type_code(x.scalar_type()), (int)first.size() + 1, {}};
    for (const int64_t f : first) s.first.push_back((int)std::clamp<int64_t>(f, -1, INT32_MAX));  // (what is none stays none)
    return s;
}

// `first`: the first distances of the buckets of a direction but the nearest
Tensor relative_bias_fwd(const Tensor &scores, const Tensor &table, const Maybe &each, int64_t offset, at::IntArrayRef first, bool both) {
    const Tensor offsets = given(each);
    const BiasSizes s = bias_sizes("scores", scores, offsets, first);
    TORCH_CHECK_VALUE(table.scalar_type() == at::kFloat && table.device() == scores.device() && table.is_contiguous() && table.dim() == 2 && table.size(0) == (both ? 2 : 1) * s.m && table.size(1) == s.H,
                      "table must be a contiguous float32 tensor [", (both ? 2 : 1) * s.m, ", ", s.H, "] on ", scores.device(), ", got ", table.scalar_type(), " ", table.sizes(), " on ", table.device());
    const c10::DeviceGuard guard(scores.device());
    Tensor out = at::empty(scores.sizes(), scores.options());
    check(library().relative_bias_fwd(memory(scores), scores.stride(0), scores.stride(1), floats(table), memory(out), s.B, s.H, s.T, s.S, s.first.data(), s.m, both, offset, memory(offsets),
                                      offsets.defined() && offsets.scalar_type() == at::kInt ? 4 : 8, s.type, stream_of(scores)),
          "hgq_relative_bias_fwd");
    return out;
}

Tensor relative_bias_bwd(const Tensor &dy, const Maybe &each, int64_t offset, at::IntArrayRef first, bool both) {
    const Tensor offsets = given(each);
    const BiasSizes s = bias_sizes("the scores' gradient", dy, offsets, first);
    const c10::DeviceGuard guard(dy.device());
    Tensor dtable = at::empty({(both ? 2 : 1) * s.m, s.H}, dy.options().dtype(at::kFloat));
    const Workspace<float> ws(library().relative_bias_bwd_workspace(s.B, s.H, s.T, s.S, s.m, both));
    check(lib.relative_bias_bwd(memory(dy), dy.stride(0), dy.stride(1), floats(dtable), ws.get(), s.B, s.H, s.T, s.S, s.first.data(), s.m, both, offset, memory(offsets),
                                offsets.defined() && offsets.scalar_type() == at::kInt ? 4 : 8, s.type, stream_of(dy)),
          "hgq_relative_bias_bwd");
    return dtable;
}

const auto &bias_op() {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::relative_bias_fwd", "").typed<decltype(relative_bias_fwd)>();
    return op;
}

// with a head's queries and keys in one piece
Tensor planes(const Tensor &t) {
    if (t.dim() == 4 && whole_planes(t) && !t.is_neg()) return t;
    return t.contiguous().resolve_neg();
}

struct RelativeBias : torch::autograd::Function<RelativeBias> {
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &scores, const Tensor &table, const Maybe &offsets, int64_t offset, std::vector<int64_t> first, bool both) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({given(offsets)});
        ctx->saved_data["offset"] = offset, ctx->saved_data["first"] = first, ctx->saved_data["both"] = both;
        return bias_op().call(scores, table, offsets, offset, first, both);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::relative_bias_bwd", "").typed<decltype(relative_bias_bwd)>();
        torch::autograd::variable_list out(6), table(1);
        if (ctx->needs_input_grad(0)) out[0] = grads[0];
        if (ctx->needs_input_grad(1)) {
            {
                at::AutoDispatchBelowADInplaceOrView below;
                const Tensor offsets = ctx->get_saved_variables()[0];
                table[0] = op.call(planes(grads[0]), offsets.defined() ? Maybe(offsets) : Maybe(), ctx->saved_data["offset"].toInt(), ctx->saved_data["first"].toIntVector(), ctx->saved_data["both"].toBool());
            }
            once_only(table, {grads[0]}, "relative_bias");
            out[1] = table[0];
        }
        return out;
    }
};

Tensor relative_bias(const Tensor &scores, const Tensor &table, std::vector<int64_t> first, bool both, int64_t offset, const std::optional<Tensor> &offsets) {
    TORCH_CHECK_VALUE(scores.dim() == 3 || scores.dim() == 4, "scores must be [heads, queries, keys] or [batch, heads, queries, keys], got ", scores.sizes());
    if (offsets) offsets_fit(*offsets, scores.dim() == 4 ? scores.size(0) : 1, scores.device());  // (one without elements is none to the operators, not to a caller)
    const bool graph = differentiated(scores) || differentiated(table);
    if (graph) accumulates_here("scores", scores), accumulates_here("table", table);
    const Tensor x = planes(scores.dim() == 3 ? scores.unsqueeze(0) : scores);
    Tensor out;
    if (graph) {
        out = RelativeBias::apply(x, plain(table.contiguous()), offsets, offset, first, both);
    } else {
        at::AutoDispatchBelowADInplaceOrView below;
        out = bias_op().call(x, plain(table.contiguous()), offsets, offset, first, both);
    }
    return scores.dim() == 3 ? out.squeeze(0) : out;
}

// ---- norms around a residual sum -----------------------------------------------------------------------------------------
struct ResidualSizes {
    int64_t rows, C;
    int type;
};

ResidualSizes residual_sizes(const Tensor &x, const Tensor &u, const Tensor &gate, const Tensor &post, const Tensor &pre, int64_t P) {
    on_gpu("x", x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., channels], got ", x.sizes());
    TORCH_CHECK_VALUE(x.is_contiguous(), "x must be contiguous");
    const int64_t C = x.size(-1), rows = x.numel() / C;
    TORCH_CHECK_VALUE((u.dim() == 1 && u.numel() == 0) || (u.sizes() == x.sizes() && u.scalar_type() == x.scalar_type() && u.device() == x.device() && u.is_contiguous()), "update must be contiguous and like x, got ",
                      u.scalar_type(), " ", u.sizes(), " on ", u.device());
    TORCH_CHECK_VALUE(P >= 1 && rows % P == 0, "rows of a gate");
    TORCH_CHECK_VALUE(gate.numel() == 0 || ((rows == 0 || gate.numel() == rows / P * C) && gate.scalar_type() == x.scalar_type() && gate.device() == x.device() && gate.is_contiguous()),
                      "gate must be contiguous, of x's type, and have an element for each of x or each of a sample's channels, got ", gate.scalar_type(), " ", gate.sizes(), " on ", gate.device());
    numbers("post_gamma", post, C, x), numbers("pre_gamma", pre, C, x);
    return {rows, C, type_code(x.scalar_type())};
}

// y (with an update) and h, and the norms' factors where they are wanted
void residual_forward(const Tensor &x, const Tensor &u, const Tensor &gate, const Tensor &post, const Tensor &pre, int64_t P, double scale, double epsilon, int64_t act, Tensor &y, Tensor &h,
                      Tensor *r) {
    const ResidualSizes s = residual_sizes(x, u, gate, post, pre, P);
    const c10::DeviceGuard guard(x.device());
    const bool update = u.sizes() == x.sizes();
    if (update) y = whole_like(x);
    h = whole_like(x);
    if (r) *r = vector_like((update ? 2 : 1) * s.rows, x);
    float *r_y = r ? floats(*r) : nullptr, *r_u = r_y && update ? r_y + s.rows : nullptr;
    check(library().residual_norm_fwd(memory(x), memory(u), memory(gate), floats(post), floats(pre), update ? memory(y) : nullptr, memory(h), r_u, r_y, s.rows, P, s.C, (float)scale, (float)epsilon,
                                      (int)act, s.type, stream_of(x)),
          "hgq_residual_norm_fwd");
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_fwd(const Tensor &x, const Maybe &u, const Maybe &gate, const Maybe &post, const Maybe &pre, int64_t P, double scale, double epsilon, int64_t act) {
    Tensor y, h, r;
    residual_forward(x, given(u), given(gate), given(post), given(pre), P, scale, epsilon, act, y, h, &r);
    return {y.defined() ? y : at::empty({0}, x.options()), h, r};
}

std::vector<Tensor> residual_norm_values(const Tensor &x, const Maybe &u, const Maybe &gate, const Maybe &post, const Maybe &pre, int64_t P, double scale, double epsilon, int64_t act) {
    Tensor y, h;
    residual_forward(x, given(u), given(gate), given(post), given(pre), P, scale, epsilon, act, y, h, nullptr);
    if (!y.defined()) return {h};
    return {y, h};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> residual_norm_bwd(const Maybe &maybe_dy, const Maybe &maybe_dh, const Tensor &x, const Maybe &maybe_u, const Maybe &maybe_gate,
                                                                     const Maybe &maybe_post, const Maybe &maybe_pre, const Tensor &r, int64_t P, double scale, double epsilon, int64_t act, bool need_dx, bool need_du, bool need_dgate,
                                                                     bool need_dpost, bool need_dpre) {
    const Tensor dy = given(maybe_dy), dh = given(maybe_dh), u = given(maybe_u), gate = given(maybe_gate), post = given(maybe_post), pre = given(maybe_pre);
    const ResidualSizes s = residual_sizes(x, u, gate, post, pre, P);
    for (const Tensor *g : {&dy, &dh})
        TORCH_CHECK_VALUE(g->numel() == 0 || (g->sizes() == x.sizes() && g->scalar_type() == x.scalar_type() && g->device() == x.device() && g->is_contiguous()), "gradients must be contiguous and like x");
    const bool update = u.sizes() == x.sizes();
    TORCH_CHECK_VALUE(r.numel() == (update ? 2 : 1) * s.rows && r.scalar_type() == at::kFloat && r.device() == x.device() && r.is_contiguous(), "r must be what the forward call left");
    const c10::DeviceGuard guard(x.device());
    need_dgate = need_dgate && gate.defined();
    const bool all = need_dx && need_du && update && need_dgate;
    const Tensor none = all ? Tensor() : at::empty({0}, x.options());
    Tensor dx = need_dx ? whole_like(x) : none, du = need_du && update ? whole_like(x) : none, dgate = !need_dgate ? none : s.rows ? whole_like(gate) : at::zeros_like(gate), dpost = vector_like(need_dpost ? s.C : 0, x),
           dpre = vector_like(need_dpre ? s.C : 0, x);
    const Workspace<float> ws(library().residual_norm_bwd_workspace(s.rows, P, s.C, s.type));
    const float *r_y = floats(r), *r_u = r_y && update ? r_y + s.rows : nullptr;
    check(lib.residual_norm_bwd(memory(dy), memory(dh), memory(x), memory(u), s.rows ? memory(gate) : nullptr, floats(post), floats(pre), r_u, r_y, memory(dx), memory(du), s.rows ? memory(dgate) : nullptr, floats(dpost), floats(dpre),
                                ws.get(), s.rows, P, s.C, (float)scale, (float)epsilon, (int)act, s.type, stream_of(x)),
          "hgq_residual_norm_bwd");
    return {dx, du, dgate, dpost, dpre};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Maybe &u, const Maybe &gate, const Maybe &post, const Maybe &pre, int64_t P,
                                                  double scale, double epsilon, int64_t act) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::residual_norm_fwd", "").typed<decltype(residual_norm_fwd)>();
        at::AutoDispatchBelowADInplaceOrView below;
        auto [y, h, r] = op.call(x, u, gate, post, pre, P, scale, epsilon, act);
        ctx->save_for_backward({x, given(u), given(gate), given(post), given(pre), r});
        ctx->saved_data["P"] = P, ctx->saved_data["scale"] = scale, ctx->saved_data["epsilon"] = epsilon, ctx->saved_data["act"] = act;
        ctx->set_materialize_grads(false);
        if (!u) return {h};
        return {y, h};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, const torch::autograd::variable_list &grads) {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::residual_norm_bwd", "").typed<decltype(residual_norm_bwd)>();
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0];
        const bool update = grads.size() == 2;
        torch::autograd::variable_list out(9);
        const Tensor &gy = update ? grads[0] : Tensor(), &gh = grads[update ? 1 : 0];
        if (!gy.defined() && !gh.defined()) return out;
        bool need[5];  // (what was not given is no input of the node)
        for (int k = 0, input = 0; k < 5; ++k) need[k] = saved[k].defined() && ctx->needs_input_grad(input++);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            const auto there = [](const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); };
            const auto whole = [](const Tensor &g) { return g.defined() ? Maybe(plain(g.contiguous())) : Maybe(); };
            const auto [dx, du, dgate, dpost, dpre] = op.call(whole(gy), whole(gh), x, there(saved[1]), there(saved[2]), there(saved[3]), there(saved[4]), saved[5], ctx->saved_data["P"].toInt(),
                                                              ctx->saved_data["scale"].toDouble(), ctx->saved_data["epsilon"].toDouble(), ctx->saved_data["act"].toInt(), need[0], need[1], need[2],
                                                              need[3], need[4]);
            const Tensor *all[] = {&dx, &du, &dgate, &dpost, &dpre};
            for (int k = 0; k < 5; ++k)
                if (need[k]) out[k] = *all[k];
        }
        once_only(out, {gy, gh, saved[0], saved[1], saved[2], saved[3], saved[4]}, "residual_norm");
        return out;
    }
};

// {y, h}; without an update {h}
std::vector<Tensor> residual_norm(const Tensor &x, const std::optional<Tensor> &u, const std::optional<Tensor> &gate, const std::optional<Tensor> &post, const std::optional<Tensor> &pre,
                                  double scale, double epsilon, int64_t act) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., channels], got ", x.sizes());
    const int64_t C = x.size(-1), rows = x.numel() / C;
    for (const auto &[name, t] : {std::make_pair("post_gamma", &post), std::make_pair("pre_gamma", &pre)})
        TORCH_CHECK_VALUE(!*t || ((*t)->dim() == 1 && (*t)->numel() == C), name, " must be a vector with an element per channel");
    TORCH_CHECK_VALUE(!u || u->sizes() == x.sizes(), "update must be like x, got ", u->sizes(), " for ", x.sizes());
    int64_t P = 1;
    if (gate && gate->sizes() != x.sizes()) {
        bool fits = gate->dim() >= 1 && gate->size(-1) == C;
        if (gate->dim() == 1) {  // one row for all
            P = rows;
        } else {  // one for each sample
            fits = fits && x.dim() >= 2 && gate->size(0) == x.size(0) && (gate->dim() == 2 || gate->dim() == x.dim());
            for (int64_t d = 1; d + 1 < gate->dim() && fits; ++d) fits = gate->size(d) == 1;
            P = x.dim() >= 2 && x.size(0) ? rows / x.size(0) : 1;
        }
        TORCH_CHECK_VALUE(fits, "gate must be like x, [batch, channels] or [channels], got ", gate->sizes(), " for ", x.sizes());
        if (P < 1) P = 1;
    }
    const char *names[] = {"update", "gate", "post_gamma", "pre_gamma"};
    const std::optional<Tensor> *rest[] = {&u, &gate, &post, &pre};
    bool graph = differentiated(x);
    for (const auto *t : rest) graph = graph || (*t && differentiated(**t));
    if (graph) {
        accumulates_here("x", x);
        for (int k = 0; k < 4; ++k)
            if (*rest[k]) accumulates_here(names[k], **rest[k]);
    }
    const auto whole = [](const Maybe &t) { return t ? Maybe(plain(t->contiguous())) : Maybe(); };
    const Tensor rows_of_x = plain(x.contiguous());
    const Maybe in_u = whole(u), in_gate = whole(gate), in_post = whole(post), in_pre = whole(pre);
    if (graph) return ResidualNorm::apply(rows_of_x, in_u, in_gate, in_post, in_pre, P, scale, epsilon, act);
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::residual_norm_values", "").typed<decltype(residual_norm_values)>();
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(rows_of_x, in_u, in_gate, in_post, in_pre, P, scale, epsilon, act);
}

// ---- the global norm -------------------------------------------------------------------------------------------------
Tensor global_norm(at::TensorList tensors) {
    TORCH_CHECK_VALUE(!tensors.empty(), "at least one tensor is expected");
    const Tensor &first = tensors[0];
    TORCH_CHECK_VALUE(first.is_cuda(), "tensors must be on a GPU (there is no CPU implementation), got device ", first.device());
    const c10::DeviceGuard guard(first.device());
    std::vector<hgq_adamw_item> items(tensors.size());  // (zeros)
    std::vector<Tensor> held;
    for (size_t k = 0; k < tensors.size(); ++k) {
        const Tensor &t = tensors[k];
        const int type = type_code(t.scalar_type());
        TORCH_CHECK_VALUE(type >= 0, "tensors must be float32, bfloat16 or float16, got ", t.scalar_type());
        TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.device() == first.device(), "tensors must be dense and on one device, got ", t.layout(), " on ", t.device());
        items[k].n = t.numel(), items[k].type = type;
        if (!items[k].n) continue;
        if (!t.is_contiguous()) held.push_back(t.detach().contiguous());
        items[k].g = t.is_contiguous() ? t.const_data_ptr() : held.back().const_data_ptr();
    }
    Tensor out = at::empty({}, first.options().dtype(at::kFloat));
    const Workspace<double> parts(library().global_norm_parts(items.data(), (int)items.size()));
    check(lib.global_norm(items.data(), (int)items.size(), parts.get(), out.data_ptr<float>(), stream_of(first)), "hgq_global_norm");
    return out;
}

// ---- an AdamW run's variables ----------------------------------------------------------------------------------------
constexpr float INF = std::numeric_limits<float>::infinity();

// The descriptors of an optimizer's variables: moments, place and type once; variable, gradient and limits at every step.
class AdamwVariables {
public:
    AdamwVariables(const py::sequence &params, const py::list &moments, int state_bits) : params_(params), bits_(state_bits) {  // (a copy of the list)
        for (const auto &m : moments) moments_.push_back(THPVariable_Unpack(m.ptr()));
        int64_t at = 0;
        for (const auto &p : params) {
            const Tensor &t = THPVariable_Unpack(p.ptr());
            hgq_adamw_item it = {};
            it.type = type_code(t.scalar_type()), it.first = at, it.lo = -INF, it.hi = INF;
            char *m = (char *)moments_[0].data_ptr(), *v = (char *)moments_[bits_ == 8 ? 2 : 1].data_ptr();
            if (bits_ == 8) {
                it.m = m + at, it.v = v + at;
                it.m_scale = (uint8_t *)moments_[1].data_ptr() + at / HGQ_ADAMW_BLOCK, it.v_scale = (uint8_t *)moments_[3].data_ptr() + at / HGQ_ADAMW_BLOCK;
            } else {
                it.m = m + 4 * at, it.v = v + 4 * at;
            }
            items_.push_back(it), sizes_.push_back(t.numel()), types_.push_back(t.scalar_type()), decay_.push_back(0);
            at += (t.numel() + HGQ_ADAMW_BLOCK - 1) / HGQ_ADAMW_BLOCK * HGQ_ADAMW_BLOCK;
            device_ = t.device();
        }
        side_ = py::reinterpret_steal<py::object>(PyUnicode_InternFromString("_hgq_side"));
        constraint_ = py::reinterpret_steal<py::object>(PyUnicode_InternFromString("constraint"));
        regularizer_ = py::reinterpret_steal<py::object>(PyUnicode_InternFromString("regularizer"));
    }

    void set_decay(int64_t k, float decay) { decay_.at(k) = decay; }

    // Variables and gradients of a step.  Returns the indices of the variables that have more to say - gradient pieces, a constraint, a
    // regularizer - which the caller sets by `limits` and `pieces`; None: there is no gradient at all.
    py::object gather() {
        HANDLE_TH_ERRORS
        const at::NoGradGuard no_grad;
        held_.clear();
        py::list special;
        bool any = false;
        for (size_t k = 0; k < items_.size(); ++k) {
            hgq_adamw_item &it = items_[k];
            PyObject *p = PyTuple_GET_ITEM(params_.ptr(), (Py_ssize_t)k);
            const Tensor &t = THPVariable_Unpack(p);
            const Tensor &g = t.grad();
            PyObject **dict = _PyObject_GetDictPtr(p);
            PyObject *own = dict ? *dict : nullptr;
            PyObject *side = own ? PyDict_GetItem(own, side_.ptr()) : nullptr;
            const bool pieces = side && PyObject_IsTrue(side) == 1;
            it.n = 0;
            if (sizes_[k] == 0 || (!g.defined() && !pieces)) continue;
            TORCH_CHECK_VALUE(t.device() == device_ && t.scalar_type() == types_[k] && t.numel() == sizes_[k] && t.is_contiguous() && !t.is_neg(),
                              "variables must stay contiguous, on ", device_, ", and of their size and type");
            it.w = t.data_ptr(), it.g = nullptr;
            if (g.defined()) {
                TORCH_CHECK_VALUE(g.layout() == at::kStrided, "gradient must be dense");
                TORCH_CHECK_VALUE(g.device() == device_ && g.scalar_type() == types_[k] && g.numel() == sizes_[k], "gradient must be like its variable, got ",
                                  g.scalar_type(), " ", g.sizes(), " on ", g.device());
                if (g.is_contiguous() && !g.is_neg()) {
                    it.g = g.data_ptr();
                } else {
                    held_.push_back(g.contiguous().resolve_neg());
                    it.g = held_.back().data_ptr();
                }
            }
            it.n = sizes_[k], it.l1 = 0, it.lo = -INF, it.hi = INF, it.decay = decay_[k];
            for (int s = 0; s < HGQ_SGD_SIDES; ++s) it.side[s] = it.side_scale[s] = nullptr;
            any = true;
            PyObject *c = own ? PyDict_GetItem(own, constraint_.ptr()) : nullptr, *r = own ? PyDict_GetItem(own, regularizer_.ptr()) : nullptr;
            if (pieces || (c && c != Py_None) || (r && r != Py_None)) special.append((int64_t)k);
        }
        if (!any) return py::none();
        return special;
        END_HANDLE_TH_ERRORS_PYBIND
    }

    void limits(int64_t k, float l1, float lo, float hi) {
        hgq_adamw_item &it = items_.at(k);
        it.l1 = l1, it.lo = lo, it.hi = hi;
    }

    // further gradient pieces of variable k: (scale or None, gradient) pairs
    void pieces(int64_t k, const py::list &pairs) {
        HANDLE_TH_ERRORS
        const at::NoGradGuard no_grad;
        hgq_adamw_item &it = items_.at(k);
        TORCH_CHECK_VALUE(pairs.size() <= HGQ_SGD_SIDES, "at most ", HGQ_SGD_SIDES, " side gradients per variable");
        for (size_t s = 0; s < pairs.size(); ++s) {
            const py::tuple pair = pairs[s].cast<py::tuple>();
            const Tensor &d = THPVariable_Unpack(pair[1].ptr());
            TORCH_CHECK_VALUE(d.device() == device_ && d.scalar_type() == at::kFloat && d.numel() == sizes_[k] && d.layout() == at::kStrided,
                              "a side gradient must be a dense float32 tensor of its variable's size on ", device_);
            held_.push_back(d.contiguous().resolve_neg());
            it.side[s] = held_.back().data_ptr<float>();
            if (pair[0].is_none()) continue;
            const Tensor &c = THPVariable_Unpack(pair[0].ptr());
            TORCH_CHECK_VALUE(c.device() == device_ && c.scalar_type() == at::kFloat && c.numel() == 1, "a side-gradient scale is one float32 on the GPU");
            held_.push_back(c);
            it.side_scale[s] = c.data_ptr<float>();
        }
        END_HANDLE_TH_ERRORS_PYBIND
    }

    // The update of what `gather` found.  clipnorm 0: no clipping; norm_out, sum_out: None, or one float32 each
    void step(const py::handle &state, double beta_1, double beta_2, double epsilon, double clipnorm, const py::handle &norm_out, uint64_t seed,
              const py::list &terms, const py::handle &sum_out) {
        HANDLE_TH_ERRORS
        const Tensor &st = THPVariable_Unpack(state.ptr());
        const float *ptrs[HGQ_SUM_BATCH];
        TORCH_CHECK_VALUE(terms.size() <= HGQ_SUM_BATCH, "at most ", HGQ_SUM_BATCH, " terms ride along with the update");
        for (size_t t = 0; t < terms.size(); ++t) ptrs[t] = scalar(terms[t], "every term");
        float *norm = norm_out.is_none() ? nullptr : scalar(norm_out, "norm_out"), *sum = terms.size() ? scalar(sum_out, "sum_out") : nullptr;
        const int n_terms = (int)terms.size(), count = (int)items_.size();
        {
            const py::gil_scoped_release others;
            const c10::DeviceGuard guard(device_);
            void *stream = stream_of(st);
            const int64_t n = clipnorm > 0 ? library().global_norm_parts(items_.data(), count) : 0;
            const Workspace<double> parts(n);
            if (n > 0) check(lib.global_norm(items_.data(), count, parts.get(), nullptr, stream), "hgq_global_norm");
            check(library().adamw_update_multi(items_.data(), count, bits_, (hgq_adamw_state *)st.data_ptr(), beta_1, beta_2, (float)epsilon,
                                               n > 0 ? (float)clipnorm : 0.0f, parts.get(), n, norm, seed, ptrs, n_terms, sum,
                                               stream),
                  "hgq_adamw_update_multi");
        }
        held_.clear();  // (the allocator hands this memory to later work of the same stream only)
        END_HANDLE_TH_ERRORS_PYBIND
    }

private:
    float *scalar(const py::handle &h, const char *what) const {
        const Tensor &t = THPVariable_Unpack(h.ptr());
        TORCH_CHECK_VALUE(t.device() == device_ && t.scalar_type() == at::kFloat && t.numel() == 1, what, " must be one float32 on ", device_);
        return t.data_ptr<float>();
    }

    const py::tuple params_;
    std::vector<Tensor> moments_, held_;
    std::vector<hgq_adamw_item> items_;
    std::vector<int64_t> sizes_;
    std::vector<at::ScalarType> types_;
    std::vector<float> decay_;
    c10::Device device_ = c10::Device(c10::DeviceType::CPU);
    int bits_;
    py::object side_, constraint_, regularizer_;
};

void bind(const py::dict &entries, const py::object &error) {
    library_error = error.inc_ref().ptr();
    auto at = [&](const char *name) { return (void *)entries[name].cast<uintptr_t>(); };
    lib.last_error = (decltype(lib.last_error))at("hgq_last_error");
    lib.global_norm_parts = (decltype(lib.global_norm_parts))at("hgq_global_norm_parts");
    lib.global_norm = (decltype(lib.global_norm))at("hgq_global_norm");
    lib.adamw_update_multi = (decltype(lib.adamw_update_multi))at("hgq_adamw_update_multi");
    lib.group_norm_fwd_workspace = (decltype(lib.group_norm_fwd_workspace))at("hgq_group_norm_fwd_workspace");
    lib.group_norm_fwd = (decltype(lib.group_norm_fwd))at("hgq_group_norm_fwd");
    lib.group_norm_bwd_workspace = (decltype(lib.group_norm_bwd_workspace))at("hgq_group_norm_bwd_workspace");
    lib.group_norm_bwd = (decltype(lib.group_norm_bwd))at("hgq_group_norm_bwd");
    lib.distill_topk_workspace = (decltype(lib.distill_topk_workspace))at("hgq_distill_topk_workspace");
    lib.distill_topk_fwd = (decltype(lib.distill_topk_fwd))at("hgq_distill_topk_fwd");
    lib.distill_topk_bwd = (decltype(lib.distill_topk_bwd))at("hgq_distill_topk_bwd");
    lib.relative_bias_fwd = (decltype(lib.relative_bias_fwd))at("hgq_relative_bias_fwd");
    lib.relative_bias_bwd_workspace = (decltype(lib.relative_bias_bwd_workspace))at("hgq_relative_bias_bwd_workspace");
    lib.relative_bias_bwd = (decltype(lib.relative_bias_bwd))at("hgq_relative_bias_bwd");
    lib.residual_norm_fwd = (decltype(lib.residual_norm_fwd))at("hgq_residual_norm_fwd");
    lib.residual_norm_bwd_workspace = (decltype(lib.residual_norm_bwd_workspace))at("hgq_residual_norm_bwd_workspace");
    lib.residual_norm_bwd = (decltype(lib.residual_norm_bwd))at("hgq_residual_norm_bwd");
    bound = true;
}

Tensor tensor_of(const py::handle &h, const char *what) {
    TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), what, " must be a tensor, got ", py::str(py::type::of(h)).cast<std::string>());
    return THPVariable_Unpack(h.ptr());
}

std::optional<Tensor> tensor_or_none(const py::handle &h, const char *what) {
    if (h.is_none()) return std::nullopt;
    return tensor_of(h, what);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(hgq, m) {
    m.def("group_norm_fwd(Tensor x, Tensor gamma, Tensor beta, int groups, float epsilon, int act) -> (Tensor, Tensor)");
    m.def("group_norm_bwd(Tensor dy, Tensor x, Tensor gamma, Tensor beta, Tensor stats, int groups, int act, bool need_dx, bool need_dgamma, bool need_dbeta) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("global_norm(Tensor[] tensors) -> Tensor");
    m.def("distill_topk_loss(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, Tensor? teacher_lse, Tensor? sample_weight, float temperature) -> Tensor");
    m.def("distill_topk_fwd(Tensor logits, Tensor teacher_logits, Tensor teacher_indices, Tensor? teacher_lse, Tensor? sample_weight, float temperature) -> (Tensor, Tensor, Tensor)");
    m.def("distill_topk_bwd(Tensor upstream, Tensor logits, Tensor teacher_logits, Tensor teacher_indices, Tensor? teacher_lse, Tensor? sample_weight, Tensor stats, float temperature) "
          "-> Tensor");
    m.def("distill_topk_bwd_(Tensor upstream, Tensor logits, Tensor teacher_logits, Tensor teacher_indices, Tensor? teacher_lse, Tensor? sample_weight, Tensor stats, float temperature, "
          "Tensor(a!) dlogits) -> ()");
    m.def("relative_bias_fwd(Tensor scores, Tensor table, Tensor? offsets, int offset, int[] first, bool both) -> Tensor");
    m.def("relative_bias_bwd(Tensor dout, Tensor? offsets, int offset, int[] first, bool both) -> Tensor");
    m.def("residual_norm_values(Tensor x, Tensor? update, Tensor? gate, Tensor? post_gamma, Tensor? pre_gamma, int gate_rows, float scale, float epsilon, int act) -> Tensor[]");
    m.def("residual_norm_fwd(Tensor x, Tensor? update, Tensor? gate, Tensor? post_gamma, Tensor? pre_gamma, int gate_rows, float scale, float epsilon, int act) -> (Tensor, Tensor, Tensor)");
    m.def("residual_norm_bwd(Tensor? dy, Tensor? dh, Tensor x, Tensor? update, Tensor? gate, Tensor? post_gamma, Tensor? pre_gamma, Tensor r, int gate_rows, float scale, float epsilon, int act, "
          "bool need_dx, bool need_dupdate, bool need_dgate, bool need_dpost, bool need_dpre) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

// (CPU tensors reach the checks, which say that there is no CPU implementation)
TORCH_LIBRARY_IMPL(hgq, CUDA, m) {
    m.impl("group_norm_fwd", group_norm_fwd);
    m.impl("group_norm_bwd", group_norm_bwd);
    m.impl("global_norm", global_norm);
    m.impl("distill_topk_loss", distill_topk_loss);
    m.impl("distill_topk_fwd", distill_topk_fwd);
    m.impl("distill_topk_bwd", distill_topk_bwd);
    m.impl("distill_topk_bwd_", distill_topk_bwd_);
    m.impl("relative_bias_fwd", relative_bias_fwd);
    m.impl("relative_bias_bwd", relative_bias_bwd);
    m.impl("residual_norm_values", residual_norm_values);
    m.impl("residual_norm_fwd", residual_norm_fwd);
    m.impl("residual_norm_bwd", residual_norm_bwd);
}
TORCH_LIBRARY_IMPL(hgq, CPU, m) {
    m.impl("group_norm_fwd", group_norm_fwd);
    m.impl("group_norm_bwd", group_norm_bwd);
    m.impl("global_norm", global_norm);
    m.impl("distill_topk_loss", distill_topk_loss);
    m.impl("distill_topk_fwd", distill_topk_fwd);
    m.impl("distill_topk_bwd", distill_topk_bwd);
    m.impl("distill_topk_bwd_", distill_topk_bwd_);
    m.impl("relative_bias_fwd", relative_bias_fwd);
    m.impl("relative_bias_bwd", relative_bias_bwd);
    m.impl("residual_norm_values", residual_norm_values);
    m.impl("residual_norm_fwd", residual_norm_fwd);
    m.impl("residual_norm_bwd", residual_norm_bwd);
}

PYBIND11_MODULE(_host, m) {
    m.def("bind", &bind);
    m.def("accumulates_elsewhere", [](const py::handle &t) { return accumulates_elsewhere(tensor_of(t, "a variable")); });
    m.def("group_norm", [](const py::handle &x, int64_t groups, const py::handle &gamma, const py::handle &beta, double epsilon, int64_t act) {
        HANDLE_TH_ERRORS
        std::optional<Tensor> ga, be;
        if (!gamma.is_none()) ga = tensor_of(gamma, "gamma");
        if (!beta.is_none()) be = tensor_of(beta, "beta");
        const Tensor input = tensor_of(x, "x");
        Tensor y;
        {
            const py::gil_scoped_release others;
            y = group_norm(input, groups, ga, be, epsilon, act);
        }
        return py::reinterpret_steal<py::object>(THPVariable_Wrap(y));
        END_HANDLE_TH_ERRORS_PYBIND
    });
    m.def("global_norm", [](const py::sequence &tensors) {
        HANDLE_TH_ERRORS
        std::vector<Tensor> list;
        list.reserve(tensors.size());
        for (const auto &t : tensors)
            if (!t.is_none()) list.push_back(tensor_of(t, "every entry"));
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("hgq::global_norm", "").typed<Tensor(at::TensorList)>();
        TORCH_CHECK_VALUE(!list.empty(), "at least one tensor is expected");
        Tensor norm;
        {
            const py::gil_scoped_release others;
            at::AutoDispatchBelowADInplaceOrView below;  // (a number: not differentiable)
            norm = op.call(list);
        }
        return py::reinterpret_steal<py::object>(THPVariable_Wrap(norm));
        END_HANDLE_TH_ERRORS_PYBIND
    });
    m.def("distill_topk", [](const py::handle &logits, const py::handle &teacher, const py::handle &indices, double T, const py::handle &lse, const py::handle &weight) {
        HANDLE_TH_ERRORS
        const Tensor z = tensor_of(logits, "logits"), t = tensor_of(teacher, "teacher_logits"), i = tensor_of(indices, "teacher_indices");
        const auto l = tensor_or_none(lse, "teacher_lse"), w = tensor_or_none(weight, "sample_weight");
        Tensor loss;
        {
            const py::gil_scoped_release others;
            loss = distill_topk(z, t, i, T, l, w);
        }
        return py::reinterpret_steal<py::object>(THPVariable_Wrap(loss));
        END_HANDLE_TH_ERRORS_PYBIND
    });
    m.def("relative_bias", [](const py::handle &scores, const py::handle &table, const std::vector<int64_t> &first, bool both, int64_t offset, const py::handle &offsets) {
        HANDLE_TH_ERRORS
        const Tensor x = tensor_of(scores, "scores"), t = tensor_of(table, "table");
        const auto o = tensor_or_none(offsets, "offset");
        Tensor out;
        {
            const py::gil_scoped_release others;
            out = relative_bias(x, t, first, both, offset, o);
        }
        return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
        END_HANDLE_TH_ERRORS_PYBIND
    });
    m.def("residual_norm", [](const py::handle &x, const py::handle &update, const py::handle &gate, const py::handle &post, const py::handle &pre, double scale, double epsilon, int64_t act) {
        HANDLE_TH_ERRORS
        const Tensor input = tensor_of(x, "x");
        const auto u = tensor_or_none(update, "update"), g = tensor_or_none(gate, "gate"), po = tensor_or_none(post, "post_gamma"), pr = tensor_or_none(pre, "pre_gamma");
        std::vector<Tensor> out;
        {
            const py::gil_scoped_release others;
            out = residual_norm(input, u, g, po, pr, scale, epsilon, act);
        }
        py::tuple t(out.size());
        for (size_t k = 0; k < out.size(); ++k) t[k] = py::reinterpret_steal<py::object>(THPVariable_Wrap(out[k]));
        return py::object(t);
        END_HANDLE_TH_ERRORS_PYBIND
    });
    py::class_<AdamwVariables>(m, "AdamwVariables")
        .def(py::init<const py::sequence &, const py::list &, int>())
        .def("set_decay", &AdamwVariables::set_decay)
        .def("gather", &AdamwVariables::gather)
        .def("limits", &AdamwVariables::limits)
        .def("pieces", &AdamwVariables::pieces)
        .def("step", &AdamwVariables::step);
}
