// torch's side of the dense operators: argument checks, output and workspace tensors, autograd nodes, over the
// C ABI of libgat_mi355.so (include/gat_mi355.h).  In C++ because the smallest of these calls take a few
// microseconds on the GPU: an autograd node in Python costs ten times that (the engine's thread has to take
// the interpreter's lock and run the backward there).  gat_amd/dense.py has the documentation.
#include <ATen/TracerMode.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/gat_mi355.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// The library's entry points, looked up in the file the Python package loads
struct Api {
#define ENTRY(name) decltype(&gatmi_##name) name = nullptr;
#define ENTRIES                                                                           \
    ENTRY(last_error) ENTRY(linear_fwd_workspace_bytes) ENTRY(linear_fwd)                 \
    ENTRY(linear_bwd_workspace_bytes_of) ENTRY(linear_bwd) ENTRY(group_norm_workspace_bytes) \
    ENTRY(group_norm_fwd) ENTRY(group_norm_bwd) ENTRY(embedding_fwd)                      \
    ENTRY(embedding_bwd_workspace_bytes) ENTRY(embedding_bwd) ENTRY(dropout)
    ENTRIES
#undef ENTRY
    bool loaded = false;
} api;

void load(const std::string &path) {
    void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(h, "cannot load ", path, ": ", dlerror());
#define ENTRY(name)                                                                       \
    api.name = reinterpret_cast<decltype(api.name)>(dlsym(h, "gatmi_" #name));            \
    TORCH_CHECK(api.name, path, " has no gatmi_" #name);
    ENTRIES
#undef ENTRY
    api.loaded = true;
}

void check(int code, const char *what) {
    TORCH_CHECK(code == 0, what, " failed (code ", code, "): ", api.last_error());
}

// The kernels run on raw pointers, out of sight of what transforms or records torch's operators: a forward-mode
// tangent would be dropped, and a trace would hold an empty tensor where the result was.  (vmap and torch.func's
// wrapped tensors have no pointer and raise by themselves.)
void plain_call(const char *name, std::initializer_list<const Tensor *> operands) {
    TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(), "gat_amd.", name, " cannot be recorded by torch.jit.trace");
    for (const Tensor *t : operands)
        TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "gat_amd.", name,
                    " has no forward-mode derivative (an operand carries a tangent)");
}
const Tensor *maybe(const MaybeTensor &t) { return t ? &*t : nullptr; }

int dtype_code(const char *name, const Tensor &x) {
    TORCH_CHECK(api.loaded, "gat_amd: the library is not loaded");
    TORCH_CHECK(x.is_cuda(), "gat_amd.", name, " runs on the GPU only (no CPU fallback)");
    switch (x.scalar_type()) {
    case at::kFloat: return GATMI_F32;
    case at::kBFloat16: return GATMI_BF16;
    case at::kHalf: return GATMI_F16;
    default: TORCH_CHECK_TYPE(false, name, ": tensors must be float32, bfloat16 or float16, got ", x.scalar_type());
    }
    return -1;
}
void same(const char *name, const Tensor &x, const Tensor &t) {
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, ": all tensors must be ", x.scalar_type(), ", got ",
                     t.scalar_type());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, ": tensors on ", x.device(), " and ", t.device());
}
void same(const char *name, const Tensor &x, const MaybeTensor &t) {
    if (t) same(name, x, *t);
}
void check_act(const char *name, int64_t act) {
    TORCH_CHECK_VALUE(act >= GATMI_ACT_NONE && act <= GATMI_ACT_GELU, name, ": unknown activation code ", act);
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes_like(size_t n, const Tensor &t) {
    return n ? at::empty({(int64_t)n}, t.options().dtype(at::kByte)) : Tensor();
}
Tensor contiguous(const MaybeTensor &t) { return t ? t->contiguous() : Tensor(); }

// What a backward returns under create_graph: the gradients, with a second derivative that raises
variable_list once(const char *name, variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list live;
    for (auto &g : grads)
        if (g.defined()) live.push_back(g.detach().requires_grad_(true));
    auto refuse = std::make_shared<torch::autograd::DelayedError>(
        std::string(name) + ": the second derivative is not implemented", (int64_t)live.size());
    live = (*refuse)(std::move(live));
    size_t i = 0;
    for (auto &g : grads)
        if (g.defined()) g = live[i++];
    return grads;
}

// ---- linear ------------------------------------------------------------------------------
gatmi_linear linear_desc(const Tensor &x, const Tensor &w, int dtype, int64_t act) {
    gatmi_linear d;
    const int64_t k = x.size(-1);
    d.rows = x.numel() / k;
    d.in_features = (int32_t)k;
    d.out_features = (int32_t)w.size(0);
    d.dtype = dtype;
    d.act = (int32_t)act;
    return d;
}

// (y, slope); slope only when `keep` and the activation has one
std::pair<Tensor, Tensor> linear_run(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, int dtype,
                                     int64_t act, bool keep) {
    const gatmi_linear d = linear_desc(x, w, dtype, act);
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    Tensor y = at::empty(shape, x.options()), slope;
    if (keep && act != GATMI_ACT_NONE)
        slope = at::empty(shape, x.options().dtype(dtype == GATMI_F32 ? at::kFloat : at::kShort));
    const size_t need = api.linear_fwd_workspace_bytes(&d);
    Tensor ws = bytes_like(need, x);
    check(api.linear_fwd(&d, ptr(x), ptr(w), ptr(b), ptr(r), ptr(y), ptr(slope), ptr(ws), need, stream_of(x)),
          "gatmi_linear_fwd");
    return {y, slope};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const MaybeTensor &b_,
                          const MaybeTensor &r_, int64_t dtype, int64_t act, bool keep) {
        const Tensor x = x_.contiguous(), w = w_.contiguous();
        auto [y, slope] = linear_run(x, w, contiguous(b_), contiguous(r_), (int)dtype, act, keep);
        if (keep) ctx->save_for_backward({x, w, slope});       // (a gradient of the residual alone needs none)
        else ctx->save_for_backward({Tensor(), Tensor(), Tensor()});
        ctx->saved_data["bias"] = b_.has_value();
        ctx->saved_data["residual"] = r_.has_value();
        ctx->saved_data["dtype"] = dtype;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(7);
        if (!grads[0].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
        // edges are numbered over the tensors that were given
        const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
        const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = has_b && ctx->needs_input_grad(2);
        if (has_r && ctx->needs_input_grad(2 + has_b)) out[3] = grads[0];
        if (nx || nw || nb) {
            at::AutoDispatchBelowADInplaceOrView below;
            c10::DeviceGuard guard(x.device());
            const gatmi_linear d = linear_desc(x, w, (int)ctx->saved_data["dtype"].toInt(), ctx->saved_data["act"].toInt());
            const Tensor gy = grads[0].contiguous();
            if (nx) out[0] = at::empty(x.sizes(), x.options());
            if (nw) out[1] = at::empty(w.sizes(), w.options());
            if (nb) out[2] = at::empty({w.size(0)}, w.options());
            const size_t need = api.linear_bwd_workspace_bytes_of(&d, nx, nw, nb);
            Tensor ws = bytes_like(need, x);
            check(api.linear_bwd(&d, ptr(x), ptr(w), ptr(slope), ptr(gy), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws),
                                 need, stream_of(x)),
                  "gatmi_linear_bwd");
        }
        return once("linear_act", out);
    }
};

Tensor linear_act(const Tensor &x, const Tensor &w, const MaybeTensor &b, int64_t act, const MaybeTensor &r) {
    const char *me = "linear_act";
    plain_call(me, {&x, &w, maybe(b), maybe(r)});
    const int dtype = dtype_code(me, x);
    same(me, x, w), same(me, x, b), same(me, x, r);
    check_act(me, act);
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.numel() > 0, me,
                      ": x must be [..., in] and weight [out, in], got ", x.sizes(), " and ", w.sizes());
    TORCH_CHECK_VALUE(w.size(0) <= 65536 && w.size(1) <= 65536, me, " covers up to 65536 features, got weight ", w.sizes());
    TORCH_CHECK_VALUE(!b || (b->dim() == 1 && b->size(0) == w.size(0)), me, ": bias must be [", w.size(0), "], got ",
                      b ? b->sizes() : at::IntArrayRef());
    if (r) {
        auto shape = x.sizes().vec();
        shape.back() = w.size(0);
        TORCH_CHECK_VALUE(r->sizes() == at::IntArrayRef(shape), me, ": residual must be ", at::IntArrayRef(shape), ", got ",
                          r->sizes());
    }
    c10::DeviceGuard guard(x.device());
    const bool grad = at::GradMode::is_enabled();
    const bool keep = grad && (x.requires_grad() || w.requires_grad() || (b && b->requires_grad()));
    if (keep || (grad && r && r->requires_grad())) return LinearFn::apply(x, w, b, r, (int64_t)dtype, act, keep);
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_run(x.contiguous(), w.contiguous(), contiguous(b), contiguous(r), dtype, act, false).first;
}

// ---- group norm ----------------------------------------------------------------------------
gatmi_group_norm group_norm_desc(const Tensor &x, const Tensor &w, const Tensor &b, int64_t groups, int dtype,
                                 int64_t act, double eps) {
    gatmi_group_norm d;
    memset(&d, 0, sizeof(d));
    d.batch = x.size(0);
    d.length = 1;
    for (int64_t i = 1; i + 1 < x.dim(); ++i) d.length *= x.size(i);
    if (d.length == 0) d.length = 1;       // no samples either (checked)
    d.groups = (int32_t)groups;
    d.width = (int32_t)(x.size(-1) / groups);
    d.dtype = dtype;
    d.act = (int32_t)act;
    d.eps = (float)eps;
    d.weight = ptr(w);
    d.bias = ptr(b);
    return d;
}

std::pair<Tensor, Tensor> group_norm_run(const Tensor &x, const Tensor &w, const Tensor &b, int64_t groups, int dtype,
                                         int64_t act, double eps, bool keep) {
    const gatmi_group_norm d = group_norm_desc(x, w, b, groups, dtype, act, eps);
    Tensor y = at::empty(x.sizes(), x.options()), stats, ws;
    size_t need = 0;
    if (keep || d.length > 1 || d.width > 2048) {      // the one-pass form can do without
        stats = at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat));
        need = api.group_norm_workspace_bytes(&d);
        ws = bytes_like(need, x);
    }
    float *mean = static_cast<float *>(ptr(stats));
    check(api.group_norm_fwd(&d, ptr(x), ptr(y), mean, mean ? mean + x.size(0) * groups : nullptr, ptr(ws), need,
                             stream_of(x)),
          "gatmi_group_norm_fwd");
    return {y, stats};
}

struct GroupNormFn : torch::autograd::Function<GroupNormFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const Tensor &b_, int64_t groups,
                          int64_t dtype, int64_t act, double eps) {
        const Tensor x = x_.contiguous(), w = w_.contiguous(), b = b_.contiguous();
        auto [y, stats] = group_norm_run(x, w, b, groups, (int)dtype, act, eps, true);
        ctx->save_for_backward({x, w, b, stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["dtype"] = dtype;
        ctx->saved_data["act"] = act;
        ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(7);
        if (!grads[0].defined()) return out;
        at::AutoDispatchBelowADInplaceOrView below;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        c10::DeviceGuard guard(x.device());
        const gatmi_group_norm d = group_norm_desc(x, w, b, groups, (int)ctx->saved_data["dtype"].toInt(),
                                                   ctx->saved_data["act"].toInt(), ctx->saved_data["eps"].toDouble());
        const Tensor gy = grads[0].contiguous();
        out[0] = at::empty(x.sizes(), x.options());
        out[1] = at::empty(w.sizes(), w.options());
        out[2] = at::empty(b.sizes(), b.options());
        const size_t need = api.group_norm_workspace_bytes(&d);
        Tensor ws = bytes_like(need, x);
        float *mean = static_cast<float *>(ptr(stats));
        check(api.group_norm_bwd(&d, ptr(x), ptr(gy), mean, mean + x.size(0) * groups, ptr(out[0]), ptr(out[1]),
                                 ptr(out[2]), ptr(ws), need, stream_of(x)),
              "gatmi_group_norm_bwd");
        return once("group_norm_act", out);
    }
};

Tensor group_norm_act(const Tensor &x, int64_t groups, const Tensor &w, const Tensor &b, double eps, int64_t act) {
    const char *me = "group_norm_act";
    plain_call(me, {&x, &w, &b});
    const int dtype = dtype_code(me, x);
    same(me, x, w), same(me, x, b);
    check_act(me, act);
    TORCH_CHECK_VALUE(x.dim() >= 2 && groups >= 1 && x.size(-1) >= 1 && x.size(-1) % groups == 0, me,
                      ": x must be [N, ..., C] with C a multiple of ", groups, " groups, got ", x.sizes());
    const int64_t c = x.size(-1);
    TORCH_CHECK_VALUE(c <= GATMI_GROUP_NORM_MAX_CHANNELS, me, " covers up to ", GATMI_GROUP_NORM_MAX_CHANNELS,
                      " channels, got ", c);
    TORCH_CHECK_VALUE(w.dim() == 1 && b.dim() == 1 && w.size(0) == c && b.size(0) == c, me, ": weight and bias must be [", c,
                      "], got ", w.sizes(), ", ", b.sizes());
    TORCH_CHECK_VALUE(x.size(0) == 0 || x.numel() > 0, me, ": samples without positions, ", x.sizes());
    TORCH_CHECK_VALUE(eps >= 0.0, me, ": eps must not be negative, got ", eps);
    c10::DeviceGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || b.requires_grad()))
        return GroupNormFn::apply(x, w, b, groups, (int64_t)dtype, act, eps);
    at::AutoDispatchBelowADInplaceOrView below;
    return group_norm_run(x.contiguous(), w.contiguous(), b.contiguous(), groups, dtype, act, eps, false).first;
}

// ---- embedding ----------------------------------------------------------------------------
Tensor embedding_run(const Tensor &ids, const Tensor &table, double scale, int dtype) {
    auto shape = ids.sizes().vec();
    shape.push_back(table.size(1));
    Tensor y = at::empty(shape, table.options());
    check(api.embedding_fwd(dtype, ids.numel(), table.size(0), table.size(1), (float)scale,
                            static_cast<const int64_t *>(ptr(ids)), ptr(table), ptr(y), stream_of(table)),
          "gatmi_embedding_fwd");
    return y;
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &ids_, const Tensor &table, double scale, int64_t dtype) {
        const Tensor ids = ids_.contiguous();
        ctx->save_for_backward({ids});
        ctx->saved_data["dtype"] = dtype;
        ctx->saved_data["vocab"] = table.size(0);
        ctx->saved_data["dim"] = table.size(1);
        ctx->saved_data["scale"] = scale;
        return embedding_run(ids, table.contiguous(), scale, (int)dtype);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor ids = ctx->get_saved_variables()[0];
        const int64_t vocab = ctx->saved_data["vocab"].toInt(), dim = ctx->saved_data["dim"].toInt(), n = ids.numel();
        c10::DeviceGuard guard(ids.device());
        const Tensor gy = grads[0].contiguous();
        out[1] = at::empty({vocab, dim}, gy.options());
        const size_t need = api.embedding_bwd_workspace_bytes(n, vocab, dim);
        Tensor ws = bytes_like(need, ids);
        check(api.embedding_bwd((int)ctx->saved_data["dtype"].toInt(), n, vocab, dim,
                                (float)ctx->saved_data["scale"].toDouble(), static_cast<const int64_t *>(ptr(ids)), ptr(gy),
                                ptr(out[1]), ptr(ws), need, stream_of(ids)),
              "gatmi_embedding_bwd");
        return once("embedding", out);
    }
};

Tensor embedding(const Tensor &ids, const Tensor &table, double scale) {
    const char *me = "embedding";
    plain_call(me, {&table});
    const int dtype = dtype_code(me, table);
    TORCH_CHECK_VALUE(ids.device() == table.device(), me, ": ids on ", ids.device(), ", table on ", table.device());
    TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong, me, ": ids must be int64, got ", ids.scalar_type());
    TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) >= 1, me, ": table must be [entries, dim], got ", table.sizes());
    c10::DeviceGuard guard(table.device());
    if (at::GradMode::is_enabled() && table.requires_grad()) return EmbeddingFn::apply(ids, table, scale, (int64_t)dtype);
    at::AutoDispatchBelowADInplaceOrView below;
    return embedding_run(ids.contiguous(), table.contiguous(), scale, dtype);
}

// ---- dropout ------------------------------------------------------------------------------
// seed_dev: the seed is read there (and left in `used`); else `seed`
Tensor dropout_run(const Tensor &x, const Tensor &r, double p, uint64_t seed, const Tensor &seed_dev, const Tensor &used,
                   int dtype) {
    Tensor y = at::empty(x.sizes(), x.options());
    const int64_t cols = x.size(-1);
    check(api.dropout(dtype, cols ? x.numel() / cols : 0, cols ? cols : 1, (float)p, seed,
                      static_cast<const uint64_t *>(ptr(seed_dev)), static_cast<uint64_t *>(ptr(used)), ptr(x), ptr(r),
                      ptr(y), stream_of(x)),
          "gatmi_dropout");
    return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &r, double p, int64_t seed,
                          const MaybeTensor &seed_dev, int64_t dtype) {
        Tensor used;       // the seed this call drew from, for a backward after the caller's has moved on
        if (seed_dev) used = at::empty({1}, seed_dev->options());
        Tensor y = dropout_run(x.contiguous(), contiguous(r), p, (uint64_t)seed, seed_dev ? *seed_dev : Tensor(), used,
                               (int)dtype);
        ctx->save_for_backward({used});
        ctx->saved_data["residual"] = r.has_value();
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["dtype"] = dtype;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
        if (ctx->needs_input_grad(0)) {
            at::AutoDispatchBelowADInplaceOrView below;
            c10::DeviceGuard guard(grads[0].device());
            out[0] = dropout_run(grads[0].contiguous(), Tensor(), ctx->saved_data["p"].toDouble(),
                                 (uint64_t)ctx->saved_data["seed"].toInt(), ctx->get_saved_variables()[0], Tensor(),
                                 (int)ctx->saved_data["dtype"].toInt());
        }
        return once("dropout", out);
    }
};

Tensor dropout(const Tensor &x, double p, bool training, uint64_t seed, MaybeTensor seed_dev, int64_t step,
               const MaybeTensor &r) {
    const char *me = "dropout";
    if ((training && p != 0.0) || r) plain_call(me, {&x, maybe(r)});      // (otherwise x is handed back)
    const int dtype = dtype_code(me, x);
    same(me, x, r);
    TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0 && (float)p < 1.f, me, ": p must be in [0, 1), got ", p);
    TORCH_CHECK_VALUE(x.dim() >= 1, me, ": x must have at least one axis");
    TORCH_CHECK_VALUE(!r || r->sizes() == x.sizes(), me, ": residual must be ", x.sizes(), ", got ",
                      r ? r->sizes() : at::IntArrayRef());
    TORCH_CHECK_VALUE(!seed_dev || (seed_dev->scalar_type() == at::kLong && seed_dev->numel() == 1 &&
                                    seed_dev->device() == x.device()),
                      me, ": a seed tensor is one int64 on ", x.device());
    if (!training) p = 0.0;
    if (p == 0.0 && !r) return x;
    c10::DeviceGuard guard(x.device());
    if (seed_dev && p > 0.0) {
        at::AutoDispatchBelowADInplaceOrView below;
        const_cast<Tensor &>(*seed_dev).add_(step);
    }
    const bool grad = at::GradMode::is_enabled();
    if (grad && (x.requires_grad() || (r && r->requires_grad())))
        return DropoutFn::apply(x, r, p, (int64_t)seed, seed_dev, (int64_t)dtype);
    at::AutoDispatchBelowADInplaceOrView below;
    return dropout_run(x.contiguous(), contiguous(r), p, seed, seed_dev ? *seed_dev : Tensor(), Tensor(), dtype);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("load", &load);
    m.def("linear_act", &linear_act);
    m.def("group_norm_act", &group_norm_act);
    m.def("embedding", &embedding);
    m.def("dropout", &dropout);
}
