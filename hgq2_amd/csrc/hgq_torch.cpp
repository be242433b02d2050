// The host side of the operators whose calls are short beside what Python costs around them: group normalisation with its autograd
// node (a backward pass in Python waits for the interpreter on the engine's thread: 118 us for two launches of 10 us each), the
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
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

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
    bound = true;
}

Tensor tensor_of(const py::handle &h, const char *what) {
    TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), what, " must be a tensor, got ", py::str(py::type::of(h)).cast<std::string>());
    return THPVariable_Unpack(h.ptr());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(hgq, m) {
    m.def("group_norm_fwd(Tensor x, Tensor gamma, Tensor beta, int groups, float epsilon, int act) -> (Tensor, Tensor)");
    m.def("group_norm_bwd(Tensor dy, Tensor x, Tensor gamma, Tensor beta, Tensor stats, int groups, int act, bool need_dx, bool need_dgamma, bool need_dbeta) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("global_norm(Tensor[] tensors) -> Tensor");
}

// (CPU tensors reach the checks, which say that there is no CPU implementation)
TORCH_LIBRARY_IMPL(hgq, CUDA, m) {
    m.impl("group_norm_fwd", group_norm_fwd);
    m.impl("group_norm_bwd", group_norm_bwd);
    m.impl("global_norm", global_norm);
}
TORCH_LIBRARY_IMPL(hgq, CPU, m) {
    m.impl("group_norm_fwd", group_norm_fwd);
    m.impl("group_norm_bwd", group_norm_bwd);
    m.impl("global_norm", global_norm);
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
    py::class_<AdamwVariables>(m, "AdamwVariables")
        .def(py::init<const py::sequence &, const py::list &, int>())
        .def("set_decay", &AdamwVariables::set_decay)
        .def("gather", &AdamwVariables::gather)
        .def("limits", &AdamwVariables::limits)
        .def("pieces", &AdamwVariables::pieces)
        .def("step", &AdamwVariables::step);
}
