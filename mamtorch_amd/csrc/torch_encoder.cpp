// torch operators of an encoder layer around the MAM layers (namespace mamtorch_kernel_encoder): tensor checks, outputs, workspace and the
// current stream for the C ABI of libmam_hip.so, and the autograd formulas.  No kernels here.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <vector>

#include "../../include/mam_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::vector<Tensor> Tensors;
typedef c10::optional<Tensor> MaybeTensor;

void *current_stream(const Tensor &t) { return static_cast<void *>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }

void check_rc(int rc, const char *what)
{
    TORCH_CHECK(rc == MAM_OK, what, " failed: ", mam_error_string(rc), " (", mam_last_error(), ")");
}

int type_of(const Tensor &t, const char *name)
{
    TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
    switch (t.scalar_type()) {
        case at::kFloat: return MAM_F32;
        case at::kBFloat16: return MAM_BF16;
        case at::kHalf: return MAM_F16;
        default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
    return -1;
}

void check_like(const Tensor &t, const Tensor &x, const char *name)
{
    TORCH_CHECK(t.device() == x.device(), name, " is on a different device");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the operand's type ", x.scalar_type(), ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == x.sizes(), name, " must have the operand's shape ", x.sizes(), ", got ", t.sizes());
}

bool has(const MaybeTensor &t) { return t.has_value() && t->defined(); }
const void *ptr(const MaybeTensor &t) { return has(t) ? t->data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace_for(size_t bytes, const Tensor &like)
{
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

// A tensor as rows of its last dimension: the tensor itself where its rows are a stride apart, else a copy.
struct Rows { Tensor t; int64_t n, c, ld; };
Rows rows_of(const Tensor &x, const char *name)
{
    TORCH_CHECK(x.dim() >= 1, name, " must have at least one dimension");
    const int64_t c = x.size(-1), n = c ? x.numel() / c : 0;
    if (x.is_contiguous() || x.numel() == 0) return {x, n, c, c};
    const bool unit = c == 1 || x.stride(-1) == 1;
    int64_t ld = 0, next = 0;      // stride of a row, and what the next outer dimension's must be
    bool even = unit;
    for (int64_t i = x.dim() - 2; even && i >= 0; --i) {
        if (x.size(i) == 1) continue;
        if (!ld) ld = x.stride(i);
        else even = x.stride(i) == next;
        next = x.stride(i) * x.size(i);
    }
    if (even && (!ld || ld >= c)) return {x, n, c, ld ? ld : c};
    return {x.contiguous(), n, c, c};
}

int weight_type(const Tensor &x, int type, const MaybeTensor &weight, const MaybeTensor &bias, int64_t c)
{
    int w = type;
    const Tensor *first = nullptr;
    for (const MaybeTensor *t : {&weight, &bias}) {
        const char *name = t == &weight ? "weight" : "bias";
        if (!has(*t)) continue;
        TORCH_CHECK((*t)->device() == x.device(), name, " is on a different device");
        const int got = type_of(**t, name);
        TORCH_CHECK(got == type || got == MAM_F32, name, " must be float32 or of the operand's type");
        TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == c && (*t)->is_contiguous(), name, " must be a contiguous vector of ", c, " elements");
        TORCH_CHECK(!first || first->scalar_type() == (*t)->scalar_type(), "weight and bias must be of one type");
        first = &**t;
        w = got;
    }
    return w;
}

mam_dropout_t dropout_of(const Tensor &x, double p, double scale, int64_t seed, int64_t offset, const MaybeTensor &step)
{
    TORCH_CHECK(p >= 0 && p <= 1, "p must be between 0 and 1, got ", p);
    if (has(step)) {
        TORCH_CHECK(step->device() == x.device(), "step is on a different device");
        TORCH_CHECK(step->scalar_type() == at::kLong && step->numel() == 1, "step must be one int64 element");
    }
    mam_dropout_t d{};
    d.p = p;
    d.scale = static_cast<float>(scale);
    d.seed = static_cast<uint64_t>(seed);
    d.offset = static_cast<uint64_t>(offset);
    d.step = has(step) ? step->data_ptr<int64_t>() : nullptr;
    return d;
}

// ---- kernels' side ----
Tensors layer_norm_cuda(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps, bool with_stats)
{
    const int type = type_of(x, "x");
    const Rows r = rows_of(x, "x");
    const int w = weight_type(x, type, weight, bias, r.c);
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options());
    const auto stats = x.options().dtype(at::kFloat);
    Tensor mean = at::empty({with_stats ? r.n : 0}, stats), rstd = at::empty({with_stats ? r.n : 0}, stats);
    check_rc(mam_layer_norm(r.t.data_ptr(), r.ld, ptr(weight), ptr(bias), eps, y.data_ptr(), with_stats ? mean.data_ptr<float>() : nullptr,
                            with_stats ? rstd.data_ptr<float>() : nullptr, r.n, r.c, type, w, current_stream(x)),
             "mam_layer_norm");
    return {y, mean, rstd};
}

struct WeightGrads { Tensor dw, db, ws; };
WeightGrads weight_grads(const Tensor &x, int type, int64_t n, int64_t c, int w, bool want_dw, bool want_db)
{
    WeightGrads g;
    const auto options = x.options().dtype(w == MAM_F32 ? at::kFloat : w == MAM_BF16 ? at::kBFloat16 : at::kHalf);
    if (want_dw) g.dw = at::empty({c}, options);
    if (want_db) g.db = at::empty({c}, options);
    if (want_dw || want_db) g.ws = workspace_for(mam_layer_norm_backward_workspace(n, c, type), x);
    return g;
}

Tensor or_empty(const Tensor &t, const Tensor &like) { return t.defined() ? t : at::empty({0}, like.options()); }

void check_stats(const Tensor &t, const Tensor &x, int64_t n, const char *name)
{
    TORCH_CHECK(t.device() == x.device() && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name,
                " must be a contiguous float32 vector of ", n, " rows on the operand's device");
}

// wanted: the gradients of x, weight, bias
Tensors layer_norm_backward_cuda(const Tensor &dy, const Tensor &x, const MaybeTensor &weight, const Tensor &mean, const Tensor &rstd,
                                 bool want_dx, bool want_dw, bool want_db, bool weight_is_float)
{
    const int type = type_of(x, "x");
    check_like(dy, x, "grad");
    const Rows r = rows_of(x, "x"), g = rows_of(dy, "grad");
    int w = weight_type(x, type, weight, c10::nullopt, r.c);
    if (!has(weight)) w = weight_is_float ? MAM_F32 : type;
    check_stats(mean, x, r.n, "mean");
    check_stats(rstd, x, r.n, "rstd");
    const c10::DeviceGuard guard(x.device());
    Tensor dx;
    if (want_dx) dx = at::empty(x.sizes(), x.options());
    const WeightGrads grads = weight_grads(x, type, r.n, r.c, w, want_dw, want_db);
    check_rc(mam_layer_norm_backward(g.t.data_ptr(), g.ld, r.t.data_ptr(), r.ld, ptr(weight), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                                     out_ptr(dx), out_ptr(grads.dw), out_ptr(grads.db), r.n, r.c, type, w, out_ptr(grads.ws),
                                     grads.ws.defined() ? grads.ws.numel() : 0, current_stream(x)),
             "mam_layer_norm_backward");
    return {or_empty(dx, x), or_empty(grads.dw, x), or_empty(grads.db, x)};
}

Tensor dropout_cuda(const Tensor &x, const MaybeTensor &residual, double p, double scale, int64_t seed, int64_t offset, const MaybeTensor &step)
{
    const int type = type_of(x, "x");
    if (has(residual)) check_like(*residual, x, "residual");
    const mam_dropout_t d = dropout_of(x, p, scale, seed, offset, step);
    const c10::DeviceGuard guard(x.device());
    const Tensor from = x.contiguous();
    Tensor add;
    if (has(residual)) add = residual->contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    check_rc(mam_dropout(from.data_ptr(), out_ptr(add), y.data_ptr(), x.numel(), type, &d, current_stream(x)), "mam_dropout");
    return y;
}

Tensors add_dropout_layer_norm_cuda(const Tensor &x, const Tensor &residual, const MaybeTensor &weight, const MaybeTensor &bias, double p,
                                    double scale, int64_t seed, int64_t offset, double eps, const MaybeTensor &step, bool with_stats)
{
    const int type = type_of(x, "x");
    check_like(residual, x, "residual");
    const Rows r = rows_of(x, "x"), add = rows_of(residual, "residual");
    const int w = weight_type(x, type, weight, bias, r.c);
    const mam_dropout_t d = dropout_of(x, p, scale, seed, offset, step);
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options()), s = at::empty(x.sizes(), x.options());
    const auto stats = x.options().dtype(at::kFloat);
    Tensor mean = at::empty({with_stats ? r.n : 0}, stats), rstd = at::empty({with_stats ? r.n : 0}, stats);
    check_rc(mam_add_dropout_layer_norm(r.t.data_ptr(), r.ld, add.t.data_ptr(), add.ld, &d, ptr(weight), ptr(bias), eps, y.data_ptr(),
                                        s.data_ptr(), with_stats ? mean.data_ptr<float>() : nullptr,
                                        with_stats ? rstd.data_ptr<float>() : nullptr, r.n, r.c, type, w, current_stream(x)),
             "mam_add_dropout_layer_norm");
    return {y, s, mean, rstd};
}

// wanted: the gradients of x, residual, weight, bias
Tensors add_dropout_layer_norm_backward_cuda(const Tensor &dy, const MaybeTensor &ds, const Tensor &s, const MaybeTensor &weight,
                                             const Tensor &mean, const Tensor &rstd, double p, double scale, int64_t seed, int64_t offset,
                                             const MaybeTensor &step, bool want_dx, bool want_residual, bool want_dw, bool want_db,
                                             bool weight_is_float)
{
    const int type = type_of(s, "s");
    check_like(dy, s, "grad");
    if (has(ds)) check_like(*ds, s, "the gradient of the sum");
    TORCH_CHECK(s.is_contiguous(), "s must be contiguous");
    const Rows r = rows_of(s, "s"), g = rows_of(dy, "grad");
    Rows more{};
    if (has(ds)) more = rows_of(*ds, "the gradient of the sum");
    int w = weight_type(s, type, weight, c10::nullopt, r.c);
    if (!has(weight)) w = weight_is_float ? MAM_F32 : type;
    check_stats(mean, s, r.n, "mean");
    check_stats(rstd, s, r.n, "rstd");
    const mam_dropout_t d = dropout_of(s, p, scale, seed, offset, step);
    const c10::DeviceGuard guard(s.device());
    Tensor dx, dr;
    if (want_dx) dx = at::empty(s.sizes(), s.options());
    if (want_residual) dr = at::empty(s.sizes(), s.options());
    const WeightGrads grads = weight_grads(s, type, r.n, r.c, w, want_dw, want_db);
    check_rc(mam_add_dropout_layer_norm_backward(g.t.data_ptr(), g.ld, out_ptr(more.t), more.ld, s.data_ptr(), ptr(weight),
                                                 mean.data_ptr<float>(), rstd.data_ptr<float>(), &d, out_ptr(dr), out_ptr(dx),
                                                 out_ptr(grads.dw), out_ptr(grads.db), r.n, r.c, type, w, out_ptr(grads.ws),
                                                 grads.ws.defined() ? grads.ws.numel() : 0, current_stream(s)),
             "mam_add_dropout_layer_norm_backward");
    return {or_empty(dx, s), or_empty(dr, s), or_empty(grads.dw, s), or_empty(grads.db, s)};
}

// A tensor with elements next to each other in its last dimension: itself, or a copy.
Tensor unit_last(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

struct AttentionCall {
    mam_diff_attention_t a;
    Tensor q, k, v, mask;           // what the pointers belong to
};

AttentionCall attention_call(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale, bool causal,
                             const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask)
{
    AttentionCall c{};
    mam_diff_attention_t &a = c.a;
    a.type = type_of(q, "q");
    for (const Tensor *t : {&k, &v}) {
        const char *name = t == &k ? "k" : "v";
        TORCH_CHECK(t->device() == q.device(), name, " is on a different device");
        TORCH_CHECK(t->scalar_type() == q.scalar_type(), name, " must have q's type ", q.scalar_type(), ", got ", t->scalar_type());
    }
    TORCH_CHECK(q.dim() == 5 && q.size(3) == 2, "q must be (batch, queries, heads, 2, head size), got ", q.sizes());
    TORCH_CHECK(k.dim() == 5 && k.size(3) == 2, "k must be (batch, keys, key heads, 2, head size), got ", k.sizes());
    TORCH_CHECK(v.dim() == 4, "v must be (batch, keys, key heads, value size), got ", v.sizes());
    a.B = q.size(0); a.Lq = q.size(1); a.H = q.size(2); a.D = q.size(4);
    a.Lk = k.size(1); a.Hkv = k.size(2); a.Dv = v.size(3);
    TORCH_CHECK(k.size(0) == a.B && v.size(0) == a.B && v.size(1) == a.Lk && v.size(2) == a.Hkv && k.size(4) == a.D,
                "q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not match");
    TORCH_CHECK(a.H == 0 || (a.Hkv > 0 && a.H % a.Hkv == 0), "the ", a.Hkv, " key heads must divide the ", a.H, " query heads");
    TORCH_CHECK(a.D >= 1 && a.D <= 128 && a.Dv >= 1 && a.Dv <= 256, "head sizes are 1 to 128 and value sizes 1 to 256, got ", a.D, " and ", a.Dv);
    TORCH_CHECK(lam.device() == q.device(), "lam is on a different device");
    a.lam_type = type_of(lam, "lam");
    TORCH_CHECK(a.lam_type == a.type || a.lam_type == MAM_F32, "lam must be float32 or of q's type");
    TORCH_CHECK(lam.dim() == 1 && lam.size(0) == a.H && lam.is_contiguous(), "lam must be a contiguous vector of ", a.H, " heads");
    TORCH_CHECK(scale > 0 && scale <= 1e30, "scale must be positive and finite, got ", scale);
    for (const MaybeTensor *t : {&lengths, &starts}) {
        const char *name = t == &lengths ? "lengths" : "starts";
        if (!has(*t)) continue;
        TORCH_CHECK((*t)->device() == q.device(), name, " is on a different device");
        TORCH_CHECK((*t)->scalar_type() == at::kInt && (*t)->dim() == 1 && (*t)->size(0) == a.B && (*t)->is_contiguous(), name,
                    " must be a contiguous int32 vector of ", a.B, " requests");
    }
    TORCH_CHECK(!has(starts) || causal, "starts is for causal calls");
    if (has(key_mask)) {
        TORCH_CHECK(key_mask->device() == q.device(), "key_mask is on a different device");
        TORCH_CHECK(key_mask->scalar_type() == at::kBool && key_mask->dim() == 2 && key_mask->size(0) == a.B && key_mask->size(1) == a.Lk,
                    "key_mask must be a bool tensor of (", a.B, ", ", a.Lk, ")");
        c.mask = unit_last(*key_mask);
        a.key_mask = static_cast<const unsigned char *>(c.mask.data_ptr());
        a.mask_stride = c.mask.stride(0);
    }
    c.q = unit_last(q);
    c.k = unit_last(k);
    c.v = unit_last(v);
    a.q = c.q.data_ptr(); a.k = c.k.data_ptr(); a.v = c.v.data_ptr(); a.lam = lam.data_ptr();
    for (int i = 0; i < 4; ++i) {
        a.q_stride[i] = c.q.stride(i);
        a.k_stride[i] = c.k.stride(i);
        if (i < 3) a.v_stride[i] = c.v.stride(i);
    }
    a.lengths = has(lengths) ? lengths->data_ptr<int32_t>() : nullptr;
    a.starts = has(starts) ? starts->data_ptr<int32_t>() : nullptr;
    a.scale = scale;
    a.causal = causal;
    return c;
}

Tensors diff_attention_cuda(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale, bool causal,
                            const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask, bool with_sums)
{
    const c10::DeviceGuard guard(q.device());
    const AttentionCall c = attention_call(q, k, v, lam, scale, causal, lengths, starts, key_mask);
    const mam_diff_attention_t &a = c.a;
    Tensor out = at::empty({a.B, a.Lq, a.H, a.Dv}, q.options());
    const int64_t planes = a.type == MAM_F32 ? 1 : 2;
    Tensor kept = with_sums ? at::empty({planes, a.B, a.Lq, a.H, a.Dv}, q.options().dtype(at::kFloat)) : at::empty({0}, q.options().dtype(at::kFloat));
    Tensor lse = with_sums ? at::empty({2, a.B, a.H, a.Lq}, q.options().dtype(at::kFloat)) : at::empty({0}, q.options().dtype(at::kFloat));
    const Tensor ws = workspace_for(mam_diff_attention_workspace(&a), q);
    check_rc(mam_diff_attention(&a, out.data_ptr(), with_sums ? kept.data_ptr<float>() : nullptr, with_sums ? lse.data_ptr<float>() : nullptr,
                                out_ptr(ws), ws.defined() ? ws.numel() : 0, current_stream(q)),
             "mam_diff_attention");
    return {out, kept, lse};
}

// wanted: the gradients of q, of k and v, of lam
Tensors diff_attention_backward_cuda(const Tensor &grad, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, const Tensor &out,
                                     const Tensor &kept, const Tensor &lse, double scale, bool causal, const MaybeTensor &lengths,
                                     const MaybeTensor &starts, const MaybeTensor &key_mask, bool want_q, bool want_kv, bool want_lam)
{
    const c10::DeviceGuard guard(q.device());
    const AttentionCall c = attention_call(q, k, v, lam, scale, causal, lengths, starts, key_mask);
    const mam_diff_attention_t &a = c.a;
    TORCH_CHECK(out.sizes() == at::IntArrayRef({a.B, a.Lq, a.H, a.Dv}), "out has the wrong shape");
    check_like(out, grad, "out");
    TORCH_CHECK(out.device() == q.device() && out.scalar_type() == q.scalar_type(), "out must have q's type and device");
    TORCH_CHECK(out.is_contiguous(), "out must be contiguous");
    const int64_t planes = a.type == MAM_F32 ? 1 : 2;
    TORCH_CHECK(kept.device() == q.device() && kept.scalar_type() == at::kFloat && kept.is_contiguous() &&
                    kept.sizes() == at::IntArrayRef({planes, a.B, a.Lq, a.H, a.Dv}),
                "kept must be a contiguous float32 tensor of ", planes, " planes like out");
    TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                    lse.sizes() == at::IntArrayRef({2, a.B, a.H, a.Lq}),
                "lse must be a contiguous float32 tensor of (2, batch, heads, queries)");
    const Tensor g = unit_last(grad);
    const int64_t strides[3] = {g.stride(0), g.stride(1), g.stride(2)};
    Tensor dq, dk, dv, dlam;
    if (want_q) dq = at::empty({a.B, a.Lq, a.H, 2, a.D}, q.options());
    if (want_kv) {
        dk = at::empty({a.B, a.Lk, a.Hkv, 2, a.D}, q.options());
        dv = at::empty({a.B, a.Lk, a.Hkv, a.Dv}, q.options());
    }
    if (want_lam) dlam = at::empty({a.H}, lam.options());
    const Tensor ws = workspace_for(mam_diff_attention_backward_workspace(&a), q);
    check_rc(mam_diff_attention_backward(&a, g.data_ptr(), strides, out.data_ptr(), kept.data_ptr<float>(), lse.data_ptr<float>(), out_ptr(dq),
                                         out_ptr(dk), out_ptr(dv), out_ptr(dlam), out_ptr(ws), ws.defined() ? ws.numel() : 0, current_stream(q)),
             "mam_diff_attention_backward");
    return {or_empty(dq, q), or_empty(dk, q), or_empty(dv, q), or_empty(dlam, lam)};
}

// ---- autograd ----
template <class Signature>
c10::TypedOperatorHandle<Signature> find(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool wants(const MaybeTensor &t) { return t.has_value() && wants(*t); }
template <class... T>
bool recording(const T &...t)
{
    return at::GradMode::is_enabled() && (wants(t) || ...);
}
Tensor or_none(const MaybeTensor &t) { return has(t) ? *t : Tensor(); }
MaybeTensor maybe(const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
bool is_float(const MaybeTensor &a, const MaybeTensor &b)
{
    return (has(a) && a->scalar_type() == at::kFloat) || (has(b) && b->scalar_type() == at::kFloat);
}

Tensors norm_below(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps, bool with_stats)
{
    static const auto op = find<Tensors(const Tensor &, const MaybeTensor &, const MaybeTensor &, double, bool)>(
        "mamtorch_kernel_encoder::layer_norm");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, weight, bias, eps, with_stats);
}

struct Norm : public Function<Norm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps)
    {
        Tensors out = norm_below(x, weight, bias, eps, true);
        ctx->saved_data["dx"] = x.requires_grad();
        ctx->saved_data["dw"] = wants(weight);
        ctx->saved_data["db"] = wants(bias);
        ctx->saved_data["float"] = is_float(weight, bias);
        ctx->save_for_backward({x, or_none(weight), out[1], out[2]});
        ctx->mark_non_differentiable({out[1], out[2]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        static const auto op = find<Tensors(const Tensor &, const Tensor &, const MaybeTensor &, const Tensor &, const Tensor &, bool, bool, bool,
                                            bool)>("mamtorch_kernel_encoder::layer_norm_backward");
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const variable_list s = ctx->get_saved_variables();
        const bool dx = ctx->saved_data["dx"].toBool(), dw = ctx->saved_data["dw"].toBool(), db = ctx->saved_data["db"].toBool();
        const Tensors g = op.call(grads[0], s[0], maybe(s[1]), s[2], s[3], dx, dw, db, ctx->saved_data["float"].toBool());
        if (dx) out[0] = g[0];
        if (dw) out[1] = g[1];
        if (db) out[2] = g[2];
        return out;
    }
};

Tensors layer_norm_autograd(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps, bool with_stats)
{
    return recording(x, weight, bias) ? Norm::apply(x, weight, bias, eps) : norm_below(x, weight, bias, eps, with_stats);
}

Tensor dropout_below(const Tensor &x, const MaybeTensor &residual, double p, double scale, int64_t seed, int64_t offset, const MaybeTensor &step)
{
    static const auto op = find<Tensor(const Tensor &, const MaybeTensor &, double, double, int64_t, int64_t, const MaybeTensor &)>(
        "mamtorch_kernel_encoder::dropout");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, residual, p, scale, seed, offset, step);
}

struct Drop : public Function<Drop> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &residual, double p, double scale, int64_t seed,
                          int64_t offset, const MaybeTensor &step)
    {
        ctx->saved_data["p"] = p;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["x"] = x.requires_grad();
        ctx->saved_data["residual"] = wants(residual);
        ctx->save_for_backward({or_none(step)});
        return dropout_below(x, residual, p, scale, seed, offset, step);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list out(7);
        if (ctx->saved_data["x"].toBool()) {
            static const auto op = find<Tensor(const Tensor &, const MaybeTensor &, double, double, int64_t, int64_t, const MaybeTensor &)>(
                "mamtorch_kernel_encoder::dropout");
            out[0] = op.call(grads[0], c10::nullopt, ctx->saved_data["p"].toDouble(), ctx->saved_data["scale"].toDouble(),
                             ctx->saved_data["seed"].toInt(), ctx->saved_data["offset"].toInt(), maybe(ctx->get_saved_variables()[0]));
        }
        if (ctx->saved_data["residual"].toBool()) out[1] = grads[0];
        return out;
    }
};

Tensor dropout_autograd(const Tensor &x, const MaybeTensor &residual, double p, double scale, int64_t seed, int64_t offset,
                        const MaybeTensor &step)
{
    return recording(x, residual) ? Drop::apply(x, residual, p, scale, seed, offset, step)
                                  : dropout_below(x, residual, p, scale, seed, offset, step);
}

Tensors join_below(const Tensor &x, const Tensor &residual, const MaybeTensor &weight, const MaybeTensor &bias, double p, double scale,
                   int64_t seed, int64_t offset, double eps, const MaybeTensor &step, bool with_stats)
{
    static const auto op = find<Tensors(const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &, double, double, int64_t, int64_t,
                                        double, const MaybeTensor &, bool)>("mamtorch_kernel_encoder::add_dropout_layer_norm");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, residual, weight, bias, p, scale, seed, offset, eps, step, with_stats);
}

struct Join : public Function<Join> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &residual, const MaybeTensor &weight,
                                 const MaybeTensor &bias, double p, double scale, int64_t seed, int64_t offset, double eps,
                                 const MaybeTensor &step)
    {
        Tensors out = join_below(x, residual, weight, bias, p, scale, seed, offset, eps, step, true);
        ctx->saved_data["p"] = p;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["x"] = x.requires_grad();
        ctx->saved_data["residual"] = residual.requires_grad();
        ctx->saved_data["dw"] = wants(weight);
        ctx->saved_data["db"] = wants(bias);
        ctx->saved_data["float"] = is_float(weight, bias);
        ctx->save_for_backward({out[1], or_none(weight), out[2], out[3], or_none(step)});
        ctx->mark_non_differentiable({out[2], out[3]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        static const auto op =
            find<Tensors(const Tensor &, const MaybeTensor &, const Tensor &, const MaybeTensor &, const Tensor &, const Tensor &, double, double,
                         int64_t, int64_t, const MaybeTensor &, bool, bool, bool, bool, bool)>(
                "mamtorch_kernel_encoder::add_dropout_layer_norm_backward");
        static const auto drop = find<Tensor(const Tensor &, const MaybeTensor &, double, double, int64_t, int64_t, const MaybeTensor &)>(
            "mamtorch_kernel_encoder::dropout");
        variable_list out(10);
        const bool x = ctx->saved_data["x"].toBool(), residual = ctx->saved_data["residual"].toBool();
        const bool dw = ctx->saved_data["dw"].toBool(), db = ctx->saved_data["db"].toBool();
        const double p = ctx->saved_data["p"].toDouble(), scale = ctx->saved_data["scale"].toDouble();
        const int64_t seed = ctx->saved_data["seed"].toInt(), offset = ctx->saved_data["offset"].toInt();
        const variable_list s = ctx->get_saved_variables();
        if (!grads[0].defined()) {              // only the sum was used further on
            if (!grads[1].defined()) return out;
            if (x) out[0] = drop.call(grads[1], c10::nullopt, p, scale, seed, offset, maybe(s[4]));
            if (residual) out[1] = grads[1];
            return out;
        }
        const Tensors g = op.call(grads[0], maybe(grads[1]), s[0], maybe(s[1]), s[2], s[3], p, scale, seed, offset, maybe(s[4]), x, residual, dw,
                                  db, ctx->saved_data["float"].toBool());
        if (x) out[0] = g[0];
        if (residual) out[1] = g[1];
        if (dw) out[2] = g[2];
        if (db) out[3] = g[3];
        return out;
    }
};

Tensors add_dropout_layer_norm_autograd(const Tensor &x, const Tensor &residual, const MaybeTensor &weight, const MaybeTensor &bias, double p,
                                        double scale, int64_t seed, int64_t offset, double eps, const MaybeTensor &step, bool with_stats)
{
    return recording(x, residual, weight, bias) ? Join::apply(x, residual, weight, bias, p, scale, seed, offset, eps, step)
                                                : join_below(x, residual, weight, bias, p, scale, seed, offset, eps, step, with_stats);
}

typedef Tensors AttentionSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, double, bool, const MaybeTensor &,
                                   const MaybeTensor &, const MaybeTensor &, bool);
typedef Tensors AttentionBackwardSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                           const Tensor &, const Tensor &, double, bool, const MaybeTensor &, const MaybeTensor &,
                                           const MaybeTensor &, bool, bool, bool);

Tensors attention_below(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale, bool causal,
                        const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask, bool with_sums)
{
    static const auto op = find<AttentionSignature>("mamtorch_kernel_encoder::diff_attention");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(q, k, v, lam, scale, causal, lengths, starts, key_mask, with_sums);
}

struct Attention : public Function<Attention> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale,
                                 bool causal, const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask)
    {
        Tensors out = attention_below(q, k, v, lam, scale, causal, lengths, starts, key_mask, true);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["q"] = q.requires_grad();
        ctx->saved_data["k"] = k.requires_grad();
        ctx->saved_data["v"] = v.requires_grad();
        ctx->saved_data["lam"] = lam.requires_grad();
        ctx->save_for_backward({q, k, v, lam, out[0], out[1], out[2], or_none(lengths), or_none(starts), or_none(key_mask)});
        ctx->mark_non_differentiable({out[1], out[2]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        static const auto op = find<AttentionBackwardSignature>("mamtorch_kernel_encoder::diff_attention_backward");
        variable_list out(9);
        if (!grads[0].defined()) return out;
        const variable_list s = ctx->get_saved_variables();
        const bool q = ctx->saved_data["q"].toBool(), k = ctx->saved_data["k"].toBool(), v = ctx->saved_data["v"].toBool();
        const bool lam = ctx->saved_data["lam"].toBool();
        const Tensors g = op.call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["scale"].toDouble(),
                                  ctx->saved_data["causal"].toBool(), maybe(s[7]), maybe(s[8]), maybe(s[9]), q, k || v, lam);
        if (q) out[0] = g[0];
        if (k) out[1] = g[1];
        if (v) out[2] = g[2];
        if (lam) out[3] = g[3];
        return out;
    }
};

Tensors diff_attention_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale, bool causal,
                                const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask, bool with_sums)
{
    return recording(q, k, v, lam) ? Attention::apply(q, k, v, lam, scale, causal, lengths, starts, key_mask)
                                   : attention_below(q, k, v, lam, scale, causal, lengths, starts, key_mask, with_sums);
}

}  // namespace

TORCH_LIBRARY(mamtorch_kernel_encoder, m)
{
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool with_stats) -> Tensor[]");
    m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, bool want_x, bool want_weight, "
          "bool want_bias, bool weight_is_float) -> Tensor[]");
    m.def("dropout(Tensor x, Tensor? residual, float p, float scale, int seed, int offset, Tensor? step) -> Tensor");
    m.def("add_dropout_layer_norm(Tensor x, Tensor residual, Tensor? weight, Tensor? bias, float p, float scale, int seed, int offset, "
          "float eps, Tensor? step, bool with_stats) -> Tensor[]");
    m.def("add_dropout_layer_norm_backward(Tensor grad, Tensor? grad_sum, Tensor s, Tensor? weight, Tensor mean, Tensor rstd, float p, "
          "float scale, int seed, int offset, Tensor? step, bool want_x, bool want_residual, bool want_weight, bool want_bias, "
          "bool weight_is_float) -> Tensor[]");
    m.def("diff_attention(Tensor q, Tensor k, Tensor v, Tensor lam, float scale, bool causal, Tensor? lengths, Tensor? starts, "
          "Tensor? key_mask, bool with_sums) -> Tensor[]");
    m.def("diff_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor lam, Tensor out, Tensor kept, Tensor lse, float scale, "
          "bool causal, Tensor? lengths, Tensor? starts, Tensor? key_mask, bool want_q, bool want_kv, bool want_lam) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(mamtorch_kernel_encoder, CUDA, m)
{
    m.impl("diff_attention", &diff_attention_cuda);
    m.impl("diff_attention_backward", &diff_attention_backward_cuda);
    m.impl("layer_norm", &layer_norm_cuda);
    m.impl("layer_norm_backward", &layer_norm_backward_cuda);
    m.impl("dropout", &dropout_cuda);
    m.impl("add_dropout_layer_norm", &add_dropout_layer_norm_cuda);
    m.impl("add_dropout_layer_norm_backward", &add_dropout_layer_norm_backward_cuda);
}

TORCH_LIBRARY_IMPL(mamtorch_kernel_encoder, Autograd, m)
{
    m.impl("layer_norm", &layer_norm_autograd);
    m.impl("dropout", &dropout_autograd);
    m.impl("add_dropout_layer_norm", &add_dropout_layer_norm_autograd);
    m.impl("diff_attention", &diff_attention_autograd);
}
