// torch.ops.cmvae_amd.{set_attention, group_norm_act, adamw_step, adamw_state_values}: the argument checks, allocations
// and autograd nodes of these operators, over the C entry points of libcmvae_hip.so.
//
// Unlike the other ops of the namespace (cmvae_amd/registry.py, in Python over ctypes) these are called many times per step
// on small tensors, where the host is what takes the time: a forward + backward of a small group norm took 117 us with its
// autograd node in Python — the engine runs every backward pass on a thread of its own, which finds the interpreter's caches
// cold — for 20 us of kernels.
//
// The library's path is handed in by cmvae_amd/_lib.py (`_use_library`), so that CMVAE_HIP_LIB holds here too.  Workspaces
// come from torch's caching allocator, per call: a captured graph owns its own.
#include <ATen/ATen.h>
#include <ATen/TensorUtils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <dlfcn.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/cmvae_abi.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
    decltype(&cmvae_last_error) last_error;
    decltype(&cmvae_set_attention_workspace_bytes) sa_ws;
    decltype(&cmvae_set_attention_fwd) sa_fwd;
    decltype(&cmvae_set_attention_bwd) sa_bwd;
    decltype(&cmvae_group_norm_workspace_bytes) gn_ws;
    decltype(&cmvae_group_norm_fwd) gn_fwd;
    decltype(&cmvae_group_norm_bwd) gn_bwd;
    decltype(&cmvae_adamw_step) adamw;
    decltype(&cmvae_adamw_state_values) adamw_values;
} lib = {};

void use_library(std::string path) {
    void* h = dlopen(path.c_str(), RTLD_NOW);
    TORCH_CHECK(h, "cmvae_amd: ", dlerror());
    auto sym = [&](auto& fn, const char* name) {
        fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(h, name));
        TORCH_CHECK(fn, "cmvae_amd: ", path, " has no symbol ", name);
    };
    sym(lib.last_error, "cmvae_last_error");
    sym(lib.sa_ws, "cmvae_set_attention_workspace_bytes");
    sym(lib.sa_fwd, "cmvae_set_attention_fwd");
    sym(lib.sa_bwd, "cmvae_set_attention_bwd");
    sym(lib.gn_ws, "cmvae_group_norm_workspace_bytes");
    sym(lib.gn_fwd, "cmvae_group_norm_fwd");
    sym(lib.gn_bwd, "cmvae_group_norm_bwd");
    sym(lib.adamw, "cmvae_adamw_step");
    sym(lib.adamw_values, "cmvae_adamw_state_values");
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: ", lib.last_error()); }

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? CMVAE_F32 : t == at::kBFloat16 ? CMVAE_BF16 : t == at::kHalf ? CMVAE_F16 : -1;
}

void* ptr(const optional<Tensor>& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
bool given(const optional<Tensor>& t) { return t.has_value() && t->defined(); }

Tensor workspace(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Gradients that cannot be differentiated again say so when that is tried: under create_graph they get a node that throws,
// between them and what they depend on.  `of` has to hold a tensor that autograd knows for every input that wanted a gradient: a
// copy made inside of Function::forward is none (grad mode is off there), and with a constant incoming gradient nothing
// would be left to throw.  So inputs are copied, where they have to be, before Function::apply.
variable_list once(variable_list grads, const variable_list& of, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    const size_t n = grads.size();
    grads.insert(grads.end(), of.begin(), of.end());
    auto err = std::make_shared<torch::autograd::DelayedError>(
        std::string("cmvae_amd ") + what + ": differentiable once; its gradient was differentiated", (int64_t)grads.size());
    variable_list out = (*err)(std::move(grads));
    out.resize(n);
    return out;
}

// ------------------------------------------------------------------------------------------------ set attention
// t with adjacent channels and rows that start at multiples of 16 bytes under 2^22 elements apart (a copy if it has not)
Tensor rows16(const Tensor& t) {
    const int64_t per = 16 / t.element_size();
    auto s = t.strides();
    if (s[3] != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 || s[0] % per || s[1] % per || s[2] % per || s[1] >= (1 << 22))
        return t.clone(at::MemoryFormat::Contiguous);
    return t;
}

void strides3(int64_t (&out)[3], const Tensor& t) {
    for (int i = 0; i < 3; ++i) out[i] = t.stride(i);
}

struct SetAttentionArgs {
    double scale;
    bool causal, residual;
};

cmvae_set_attn describe(const Tensor& q, const Tensor& k, const Tensor& v, const SetAttentionArgs& a, void* q_len, void* k_len) {
    cmvae_set_attn d = {};
    d.dtype = dtype_code(q.scalar_type());
    d.B = (int32_t)q.size(0); d.Sq = (int32_t)q.size(1); d.H = (int32_t)q.size(2); d.D = (int32_t)q.size(3);
    d.Sk = (int32_t)k.size(1); d.Hkv = (int32_t)k.size(2);
    d.causal = a.causal; d.residual = a.residual; d.scale = (float)a.scale;
    d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr();
    strides3(d.q_stride, q); strides3(d.k_stride, k); strides3(d.v_stride, v);
    d.q_len = (const int32_t*)q_len; d.k_len = (const int32_t*)k_len;
    return d;
}

class SetAttention : public torch::autograd::Function<SetAttention> {
 public:
    // q, k, v as rows16() leaves them
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal,
                          const optional<Tensor>& q_len, const optional<Tensor>& k_len, bool residual, bool save) {
        c10::DeviceGuard guard(q.device());
        const SetAttentionArgs a = {scale, causal, residual};
        const Tensor o = at::empty(q.sizes(), q.options());
        Tensor attn = o, low, lse;
        if (save) {
            lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
            if (residual) attn = at::empty(q.sizes(), q.options());
            if (q.scalar_type() != at::kFloat) low = at::empty(q.sizes(), q.options());
        }
        if (o.numel()) {
            cmvae_set_attn d = describe(q, k, v, a, ptr(q_len), ptr(k_len));
            d.o = o.data_ptr();
            d.attn = save && residual ? attn.data_ptr() : nullptr;
            d.attn_low = ptr(low);
            d.lse = (float*)ptr(lse);
            const size_t n = lib.sa_ws(&d, 0);
            const Tensor ws = workspace(n, q);
            check(lib.sa_fwd(&d, ptr(ws), n, stream_of(q)), "cmvae_set_attention_fwd");
        }
        if (save) {
            ctx->saved_data["scale"] = scale;
            ctx->saved_data["causal"] = causal;
            ctx->saved_data["residual"] = residual;
            ctx->save_for_backward({q, k, v, attn, lse, given(q_len) ? *q_len : Tensor(), given(k_len) ? *k_len : Tensor(), low});
        }
        return o;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &attn = s[3], &lse = s[4];
        const SetAttentionArgs a = {ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(),
                                    ctx->saved_data["residual"].toBool()};
        Tensor dq, dk, dv;
        {
            at::NoGradGuard no_grad;
            c10::DeviceGuard guard(q.device());
            dq = at::empty(q.sizes(), q.options());
            dk = at::empty(k.sizes(), k.options());
            dv = at::empty(k.sizes(), k.options());
            if (dq.numel() == 0) {
                dk.zero_();
                dv.zero_();
            } else {
                const Tensor go = rows16(g[0]), delta = at::empty(lse.sizes(), lse.options());
                cmvae_set_attn d = describe(q, k, v, a, ptr(s[5]), ptr(s[6]));
                d.dO = go.data_ptr();
                strides3(d.dO_stride, go);
                d.o = d.attn = attn.data_ptr();
                d.attn_low = ptr(s[7]);
                d.lse = (float*)lse.data_ptr(); d.delta = (float*)delta.data_ptr();
                d.dq = dq.data_ptr(); d.dk = dk.data_ptr(); d.dv = dv.data_ptr();
                const size_t n = lib.sa_ws(&d, 1);
                const Tensor ws = workspace(n, q);
                check(lib.sa_bwd(&d, ptr(ws), n, stream_of(q)), "cmvae_set_attention_bwd");
            }
        }
        variable_list out = once({dq, dk, dv}, {g[0], q, k, v}, "set_attention");
        out.resize(9);
        return out;
    }
};

Tensor set_attention(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, const optional<Tensor>& q_len,
                     const optional<Tensor>& k_len, bool residual) {
    const std::pair<const Tensor*, const char*> ts[] = {{&q, "q"}, {&k, "k"}, {&v, "v"}};
    for (const auto& [t, n] : ts) {
        TORCH_CHECK(t->is_cuda(), "cmvae_amd set_attention: ", n, " must be a GPU tensor (there is no CPU path)");
        TORCH_CHECK(dtype_code(t->scalar_type()) >= 0 && t->scalar_type() == q.scalar_type() && t->device() == q.device(),
                    "cmvae_amd set_attention: q, k, v must share one device and one of float32, bfloat16, float16; ", n, " is ",
                    t->scalar_type(), " on ", t->device());
        TORCH_CHECK(t->dim() == 4, "cmvae_amd set_attention: ", n, " must be [batch, rows, heads, channels], got ", t->sizes());
    }
    const int64_t B = q.size(0), H = q.size(2), D = q.size(3), Hkv = k.size(2);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D && Hkv >= 1 && H >= 1 && H % Hkv == 0,
                "cmvae_amd set_attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(),
                " do not fit (equal batch and channels, k and v alike, query heads a multiple of key heads)");
    TORCH_CHECK(D == 64 || D == 128, "cmvae_amd set_attention: heads of 64 or 128 channels are supported, got ", D);
    TORCH_CHECK(scale >= 1e-30 && scale <= 1e30, "cmvae_amd set_attention: scale must be a positive finite number, got ", scale);
    TORCH_CHECK(B < (1 << 30) && q.size(1) < (1 << 30) && k.size(1) < (1 << 30) && H < (1 << 30),
                "cmvae_amd set_attention: more than 2^30 batch entries, rows or heads");
    const std::pair<const optional<Tensor>*, const char*> ls[] = {{&q_len, "q_len"}, {&k_len, "k_len"}};
    for (const auto& [t, n] : ls)
        if (given(*t))
            TORCH_CHECK((*t)->device() == q.device() && (*t)->scalar_type() == at::kInt && (*t)->dim() == 1 && (*t)->size(0) == B &&
                            (*t)->is_contiguous(),
                        "cmvae_amd set_attention: ", n, " must be a dense int32 tensor of shape [", B, "] beside q");
    const bool save = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    return SetAttention::apply(rows16(q), rows16(k), rows16(v), scale, causal, q_len, k_len, residual, save);
}

// ------------------------------------------------------------------------------------------------ group norm
std::vector<int64_t> sizes3(const Tensor& x) {
    int64_t P = 1;
    for (int64_t i = 1; i + 1 < x.dim(); ++i) P *= x.size(i);
    return {x.size(0), P, x.size(-1)};
}

// [N, ..., C] as [N, P, C] with adjacent channels (a copy where strides do not allow it)
Tensor rows3(const Tensor& x) {
    const Tensor r = x.dim() == 3 ? x : x.reshape(sizes3(x));
    return r.stride(2) == 1 ? r : r.contiguous();
}

// x, or a dense copy of it where rows3() would make one
Tensor viewable(const Tensor& x) {
    if (x.is_contiguous() || (x.dim() == 3 && x.stride(2) == 1)) return x;
    const auto st = at::detail::computeStride(x.sizes(), x.strides(), sizes3(x));
    return st && (*st)[2] == 1 ? x : x.contiguous();
}

void strides2(int64_t (&out)[2], const Tensor& t) {
    for (int i = 0; i < 2; ++i) out[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

cmvae_group_norm describe(const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int64_t act) {
    cmvae_group_norm d = {};
    const Tensor& ref = w.defined() ? w : b;
    d.dtype = dtype_code(x.scalar_type());
    d.wdtype = ref.defined() ? dtype_code(ref.scalar_type()) : CMVAE_F32;
    d.act = (int32_t)act;
    d.N = (int32_t)x.size(0); d.P = (int32_t)x.size(1); d.C = (int32_t)x.size(2); d.G = (int32_t)groups;
    d.eps = (float)eps;
    d.x = x.data_ptr(); d.weight = ptr(w); d.bias = ptr(b);
    strides2(d.x_stride, x);
    return d;
}

class GroupNormAct : public torch::autograd::Function<GroupNormAct> {
 public:
    // x0 as viewable() leaves it, weight and bias dense
    static Tensor forward(AutogradContext* ctx, const Tensor& x0, int64_t groups, const optional<Tensor>& weight,
                          const optional<Tensor>& bias, double eps, int64_t act, bool save) {
        c10::DeviceGuard guard(x0.device());
        const Tensor x = rows3(x0);
        const Tensor w = given(weight) ? *weight : Tensor(), b = given(bias) ? *bias : Tensor();
        const Tensor y = at::empty(x0.sizes(), x.options());
        Tensor stats;
        if (save) stats = at::empty({x.size(0), groups, 4}, x.options().dtype(at::kFloat));
        if (y.numel()) {
            cmvae_group_norm d = describe(x, groups, w, b, eps, act);
            d.y = y.data_ptr();
            d.stats = (float*)ptr(stats);
            const size_t n = lib.gn_ws(&d, 0);
            const Tensor ws = workspace(n, x);
            check(lib.gn_fwd(&d, ptr(ws), n, stream_of(x)), "cmvae_group_norm_fwd");
        }
        if (save) {
            ctx->saved_data["groups"] = groups;
            ctx->saved_data["eps"] = eps;
            ctx->saved_data["act"] = act;
            ctx->saved_data["parameters"] = (given(weight) && weight->requires_grad()) || (given(bias) && bias->requires_grad());
            ctx->save_for_backward({x0, w, b, stats});
        }
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &x0 = s[0], &w = s[1], &b = s[2], &stats = s[3];
        Tensor dx, dw, db;
        {
            at::NoGradGuard no_grad;
            c10::DeviceGuard guard(x0.device());
            const Tensor x = rows3(x0);
            dx = at::empty(x0.sizes(), x0.options());
            if (ctx->saved_data["parameters"].toBool()) {
                if (w.defined()) dw = at::empty(w.sizes(), w.options());
                if (b.defined()) db = at::empty(b.sizes(), b.options());
            }
            if (dx.numel() == 0) {
                if (dw.defined()) dw.zero_();
                if (db.defined()) db.zero_();
            } else {
                const Tensor dy = rows3(g[0]);
                cmvae_group_norm d = describe(x, ctx->saved_data["groups"].toInt(), w, b, ctx->saved_data["eps"].toDouble(),
                                              ctx->saved_data["act"].toInt());
                d.dy = dy.data_ptr();
                strides2(d.dy_stride, dy);
                d.stats = (float*)stats.data_ptr();
                d.dx = dx.data_ptr(); d.dweight = ptr(dw); d.dbias = ptr(db);
                const size_t n = lib.gn_ws(&d, 1);
                const Tensor ws = workspace(n, x);
                check(lib.gn_bwd(&d, ptr(ws), n, stream_of(x)), "cmvae_group_norm_bwd");
            }
        }
        variable_list out = once({dx, dw, db}, {g[0], x0, w, b}, "group_norm_act");
        return {out[0], Tensor(), out[1], out[2], Tensor(), Tensor(), Tensor()};
    }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps,
                      int64_t act) {
    TORCH_CHECK(x.is_cuda(), "cmvae_amd group_norm_act: x must be a GPU tensor (there is no CPU path)");
    TORCH_CHECK(dtype_code(x.scalar_type()) >= 0 && x.dim() >= 2,
                "cmvae_amd group_norm_act: x must be a float32, bfloat16 or float16 tensor [N, ..., C], got ", x.scalar_type(), " ",
                x.sizes());
    const int64_t C = x.size(-1);
    TORCH_CHECK(groups >= 1 && C >= 1 && C % groups == 0, "cmvae_amd group_norm_act: ", groups, " groups of ", C, " channels");
    TORCH_CHECK(act >= 0 && act <= 3, "cmvae_amd group_norm_act: activation ", act);
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "cmvae_amd group_norm_act: eps must be finite and not negative, got ", eps);
    TORCH_CHECK(x.size(0) < (1LL << 31) && x.numel() / std::max<int64_t>(1, x.size(0) * C) <= (1 << 30) && C <= (1 << 24),
                "cmvae_amd group_norm_act: x of shape ", x.sizes(), " is too large");
    const std::pair<const optional<Tensor>*, const char*> ps[] = {{&weight, "weight"}, {&bias, "bias"}};
    for (const auto& [t, n] : ps)
        if (given(*t))
            TORCH_CHECK((*t)->device() == x.device() && (*t)->dim() == 1 && (*t)->size(0) == C &&
                            ((*t)->scalar_type() == at::kFloat || (*t)->scalar_type() == x.scalar_type()),
                        "cmvae_amd group_norm_act: ", n, " must be a [", C, "] tensor beside x, of float32 or its type");
    TORCH_CHECK(!given(weight) || !given(bias) || weight->scalar_type() == bias->scalar_type(),
                "cmvae_amd group_norm_act: weight and bias are of different types");
    const bool save = at::GradMode::is_enabled() && (x.requires_grad() || (given(weight) && weight->requires_grad()) ||
                                                     (given(bias) && bias->requires_grad()));
    auto dense = [](const optional<Tensor>& t) { return given(t) ? optional<Tensor>(t->contiguous()) : optional<Tensor>(); };
    return GroupNormAct::apply(viewable(x), groups, dense(weight), dense(bias), eps, act, save);
}

// ------------------------------------------------------------------------------------------------ AdamW
constexpr int64_t BLOCK = 256;

// checked states: their width in bits
int states(const Tensor& m, const Tensor& v, const optional<Tensor>& scales) {
    const std::pair<const Tensor*, const char*> ts[] = {{&m, "exp_avg"}, {&v, "exp_avg_sq"}};
    for (const auto& [t, n] : ts)
        TORCH_CHECK(t->is_cuda() && t->dim() == 1 && t->is_contiguous(), "cmvae_amd adamw: ", n,
                    " must be a flat GPU tensor (there is no CPU path)");
    TORCH_CHECK(m.numel() == v.numel() && m.device() == v.device() && m.numel() % BLOCK == 0,
                "cmvae_amd adamw: exp_avg and exp_avg_sq must have one length, a multiple of ", BLOCK, ", and one device");
    if (!given(scales)) {
        TORCH_CHECK(m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat,
                    "cmvae_amd adamw: states without scales must be float32");
        return 32;
    }
    TORCH_CHECK(m.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kByte,
                "cmvae_amd adamw: 8-bit states are float8_e4m3fn (exp_avg) and uint8 (exp_avg_sq)");
    TORCH_CHECK(scales->device() == m.device() && scales->scalar_type() == at::kFloat && scales->dim() == 2 && scales->size(0) == 2 &&
                    scales->size(1) == m.numel() / BLOCK && scales->is_contiguous(),
                "cmvae_amd adamw: scales must be a dense float32 tensor [2, ", m.numel() / BLOCK, "] beside the states");
    return 8;
}

void adamw_step(at::TensorList params, const c10::List<optional<Tensor>>& grads, const Tensor& exp_avg, const Tensor& exp_avg_sq,
                const optional<Tensor>& scales, int64_t step, const optional<Tensor>& step_dev, double lr, double beta1,
                double beta2, double eps, double weight_decay) {
    const int bits = states(exp_avg, exp_avg_sq, scales);
    TORCH_CHECK(params.size() == grads.size(), "cmvae_amd adamw: ", params.size(), " parameters and ", grads.size(), " gradients");
    TORCH_CHECK(!given(step_dev) || (step_dev->device() == exp_avg.device() && step_dev->scalar_type() == at::kLong &&
                                     step_dev->numel() == 1),
                "cmvae_amd adamw: step must be a number or an int64 tensor of one value beside the states");
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(exp_avg.device());
    std::vector<cmvae_adamw_tensor> table;
    std::vector<Tensor> keep;
    // what the launch writes, and what it reads only: a workgroup may read before or after another one writes
    std::vector<std::pair<uintptr_t, uintptr_t>> spans, reads;
    spans.reserve(params.size() + 3);
    reads.reserve(params.size() + 1);
    auto span = [](const Tensor& t) {
        const auto first = reinterpret_cast<uintptr_t>(t.data_ptr());
        return std::make_pair(first, first + t.numel() * t.element_size());
    };
    auto written = [&](const Tensor& t) {
        if (t.numel()) spans.push_back(span(t));
    };
    written(exp_avg);
    written(exp_avg_sq);
    if (given(scales)) written(*scales);
    table.reserve(params.size());
    int64_t at = 0;
    for (size_t i = 0; i < params.size(); ++i) {
        const Tensor& p = params[i];
        const int64_t n = p.numel(), here = at;
        at += (n + BLOCK - 1) / BLOCK * BLOCK;
        const optional<Tensor> og = grads.get(i);
        if (!given(og)) continue;
        Tensor g = *og;
        const int code = dtype_code(p.scalar_type());
        TORCH_CHECK(code >= 0 && g.scalar_type() == p.scalar_type() && p.device() == exp_avg.device() && g.device() == p.device() &&
                        g.sizes() == p.sizes(),
                    "cmvae_amd adamw: a parameter ", p.scalar_type(), " ", p.sizes(), " on ", p.device(), " with a gradient ",
                    g.scalar_type(), " ", g.sizes(), " on ", g.device(),
                    " (float32, bfloat16 or float16, alike, on the states' device)");
        TORCH_CHECK(p.is_contiguous() || (p.dim() == 4 && p.is_contiguous(at::MemoryFormat::ChannelsLast)),
                    "cmvae_amd adamw: a parameter of shape ", p.sizes(), " has strides ", p.strides(), ": it must be dense");
        if (g.strides() != p.strides()) {
            g = at::empty_like(p).copy_(g);
            keep.push_back(g);
        }
        if (n == 0) continue;
        written(p);
        if (g.data_ptr() != p.data_ptr()) reads.push_back(span(g));       // its own parameter: one thread reads both, then writes
        table.push_back({p.data_ptr(), g.data_ptr(), n, here, code});
    }
    if (given(step_dev)) reads.push_back(span(*step_dev));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        TORCH_CHECK(spans[i].first >= spans[i - 1].second, "cmvae_amd adamw: a parameter appears twice, or parameters and states overlap");
    for (const auto& r : reads) {
        const auto after = std::lower_bound(spans.begin(), spans.end(), std::make_pair(r.second, uintptr_t(0)));
        TORCH_CHECK(after == spans.begin() || std::prev(after)->second <= r.first,
                    "cmvae_amd adamw: a gradient or the step count overlaps a parameter or a state that the step writes");
    }
    TORCH_CHECK(at == exp_avg.numel(), "cmvae_amd adamw: the parameters take ", at, " state values, the states hold ",
                exp_avg.numel());
    check(lib.adamw(table.data(), (int)table.size(), bits, exp_avg.data_ptr(), exp_avg_sq.data_ptr(), (float*)ptr(scales),
                    exp_avg.numel(), step, (const int64_t*)ptr(step_dev), lr, beta1, beta2, eps, weight_decay, stream_of(exp_avg)),
          "cmvae_adamw_step");
    for (size_t i = 0; i < params.size(); ++i)
        if (given(grads.get(i)) && !params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
}

std::tuple<Tensor, Tensor> adamw_state_values(const Tensor& exp_avg, const Tensor& exp_avg_sq, const optional<Tensor>& scales) {
    TORCH_CHECK(states(exp_avg, exp_avg_sq, scales) == 8, "cmvae_amd adamw: states in 32 bits are their values");
    c10::DeviceGuard guard(exp_avg.device());
    const Tensor m = at::empty({exp_avg.numel()}, exp_avg.options().dtype(at::kFloat)), v = at::empty_like(m);
    check(lib.adamw_values(exp_avg.data_ptr(), exp_avg_sq.data_ptr(), (const float*)ptr(scales), exp_avg.numel(),
                           (float*)m.data_ptr(), (float*)v.data_ptr(), stream_of(exp_avg)),
          "cmvae_adamw_state_values");
    return {m, v};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cmvae_amd, m) {
    m.def("_use_library(str path) -> ()", use_library);
    m.def("set_attention(Tensor q, Tensor k, Tensor v, float scale, bool causal, Tensor? q_len, Tensor? k_len, bool residual)"
          " -> Tensor", set_attention);
    m.def("group_norm_act(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act) -> Tensor", group_norm_act);
    m.def("adamw_step(Tensor(a!)[] params, Tensor?[] grads, Tensor(b!) exp_avg, Tensor(c!) exp_avg_sq, Tensor(d!)? scales, int step, "
          "Tensor? step_dev, float lr, float beta1, float beta2, float eps, float weight_decay) -> ()", adamw_step);
    m.def("adamw_state_values(Tensor exp_avg, Tensor exp_avg_sq, Tensor? scales) -> (Tensor, Tensor)", adamw_state_values);
}
