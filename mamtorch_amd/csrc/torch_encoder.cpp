// torch operators of an encoder layer around the MAM layers (namespace mamtorch_kernel_encoder): tensor checks, outputs, workspace and the
// current stream for the C ABI of libmam_hip.so, and the autograd formulas.  No kernels here.
#include "torch_encoder.h"

#include "mam_rows.h"

namespace {

// A tensor as rows of its last dimension: the tensor itself where its rows are a stride apart, else a copy.
struct Rows { Tensor t; int64_t n, c, ld; };
Rows rows_of(const Tensor &x, const char *name)
{
    TORCH_CHECK(x.dim() >= 1, name, " must have at least one dimension");
    const int64_t c = x.size(-1), n = c ? x.numel() / c : 0;
    if (x.is_contiguous() || x.numel() == 0) return {x, n, c, c};
    const int64_t ld = mam::row_stride(x.sizes().data(), x.strides().data(), x.dim());
    if (ld >= 0) return {x, n, c, ld};
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
    TORCH_CHECK(static_cast<float>(scale) > 0 && scale <= 1e30, "scale must be positive and finite in float32, got ", scale);
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
    const Tensor ws = workspace_for(with_sums ? 0 : mam_diff_attention_workspace(&a), q);
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
bool is_float(const MaybeTensor &a, const MaybeTensor &b)
{
    return (has(a) && a->scalar_type() == at::kFloat) || (has(b) && b->scalar_type() == at::kFloat);
}

typedef Tensors NormSignature(const Tensor &, const MaybeTensor &, const MaybeTensor &, double, bool);
typedef Tensors NormBackwardSignature(const Tensor &, const Tensor &, const MaybeTensor &, const Tensor &, const Tensor &, bool, bool, bool, bool);

struct NormNode : public GradNode {
    bool weight_is_float = false;
    std::string name() const override { return "LayerNormBackward"; }
    variable_list apply(variable_list &&grads) override
    {
        static const auto op = find<NormBackwardSignature>("mamtorch_kernel_encoder::layer_norm_backward");
        variable_list out(3);
        if (!grads[0].defined()) return out;
        check_saved();
        const bool dx = task_should_compute_output(0), dw = task_should_compute_output(1), db = task_should_compute_output(2);
        Tensors g;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(grads[0], take(0), maybe(take(1)), take(2), take(3), dx, dw, db, weight_is_float);
        }
        if (dx) out[0] = g[0];
        if (dw) out[1] = g[1];
        if (db) out[2] = g[2];
        check_differentiated_once(grads, out);
        return out;
    }
};

Tensors layer_norm_autograd(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps, bool with_stats)
{
    static const auto op = find<NormSignature>("mamtorch_kernel_encoder::layer_norm");
    check_no_tangent("layer_norm", x, weight, bias);
    const bool record = recording(x, weight, bias);
    Tensors out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(x, weight, bias, eps, with_stats || record);
    }
    if (!record) return out;
    const auto node = node_of<NormNode>(x, or_none(weight), or_none(bias));
    node->weight_is_float = is_float(weight, bias);
    for (const Tensor &t : {x, or_none(weight), out[1], out[2]}) node->save(t);
    torch::autograd::set_history(out[0], node);
    return out;
}

typedef Tensor DropSignature(const Tensor &, const MaybeTensor &, double, double, int64_t, int64_t, const MaybeTensor &);

struct DropNode : public GradNode {
    double p = 0, scale = 0;
    int64_t seed = 0, offset = 0;
    bool stepped = false;
    std::string name() const override { return "CounterDropoutBackward"; }
    variable_list apply(variable_list &&grads) override
    {
        static const auto op = find<DropSignature>("mamtorch_kernel_encoder::dropout");
        variable_list out(2);
        if (!grads[0].defined()) return out;
        if (stepped) check_saved();
        if (task_should_compute_output(0))
            out[0] = op.call(grads[0], c10::nullopt, p, scale, seed, offset, stepped ? MaybeTensor(take(0)) : MaybeTensor());
        if (task_should_compute_output(1)) out[1] = grads[0];
        return out;
    }
};

Tensor dropout_autograd(const Tensor &x, const MaybeTensor &residual, double p, double scale, int64_t seed, int64_t offset,
                        const MaybeTensor &step)
{
    static const auto op = find<DropSignature>("mamtorch_kernel_encoder::dropout");
    check_no_tangent("dropout", x, residual);
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(x, residual, p, scale, seed, offset, step);
    }
    if (!recording(x, residual)) return out;
    const auto node = node_of<DropNode>(x, or_none(residual));
    node->p = p;
    node->scale = scale;
    node->seed = seed;
    node->offset = offset;
    node->stepped = has(step);
    if (has(step)) node->save(*step);
    torch::autograd::set_history(out, node);
    return out;
}

typedef Tensors JoinSignature(const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &, double, double, int64_t, int64_t, double,
                              const MaybeTensor &, bool);
typedef Tensors JoinBackwardSignature(const Tensor &, const MaybeTensor &, const Tensor &, const MaybeTensor &, const Tensor &, const Tensor &,
                                      double, double, int64_t, int64_t, const MaybeTensor &, bool, bool, bool, bool, bool);

struct JoinNode : public GradNode {
    double p = 0, scale = 0;
    int64_t seed = 0, offset = 0;
    bool weight_is_float = false;
    std::string name() const override { return "AddDropoutLayerNormBackward"; }
    variable_list apply(variable_list &&grads) override
    {
        static const auto op = find<JoinBackwardSignature>("mamtorch_kernel_encoder::add_dropout_layer_norm_backward");
        static const auto drop = find<DropSignature>("mamtorch_kernel_encoder::dropout");
        variable_list out(4);
        const bool x = task_should_compute_output(0), residual = task_should_compute_output(1);
        const bool dw = task_should_compute_output(2), db = task_should_compute_output(3);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        check_saved();
        if (!grads[0].defined()) {              // only the sum was used further on
            if (x) out[0] = drop.call(grads[1], c10::nullopt, p, scale, seed, offset, maybe(take(4)));
            if (residual) out[1] = grads[1];
            return out;
        }
        Tensors g;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(grads[0], maybe(grads[1]), take(0), maybe(take(1)), take(2), take(3), p, scale, seed, offset, maybe(take(4)), x, residual,
                        dw, db, weight_is_float);
        }
        if (x) out[0] = g[0];
        if (residual) out[1] = g[1];
        if (dw) out[2] = g[2];
        if (db) out[3] = g[3];
        check_differentiated_once(grads, out);
        return out;
    }
};

Tensors add_dropout_layer_norm_autograd(const Tensor &x, const Tensor &residual, const MaybeTensor &weight, const MaybeTensor &bias, double p,
                                        double scale, int64_t seed, int64_t offset, double eps, const MaybeTensor &step, bool with_stats)
{
    static const auto op = find<JoinSignature>("mamtorch_kernel_encoder::add_dropout_layer_norm");
    check_no_tangent("add_dropout_layer_norm", x, residual, weight, bias);
    const bool record = recording(x, residual, weight, bias);
    Tensors out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(x, residual, weight, bias, p, scale, seed, offset, eps, step, with_stats || record);
    }
    if (!record) return out;
    const auto node = node_of<JoinNode>(x, residual, or_none(weight), or_none(bias));
    node->p = p;
    node->scale = scale;
    node->seed = seed;
    node->offset = offset;
    node->weight_is_float = is_float(weight, bias);
    torch::autograd::set_history(out[0], node);
    torch::autograd::set_history(out[1], node);
    node->save_output(out[1]);
    for (const Tensor &t : {or_none(weight), out[2], out[3], or_none(step)}) node->save(t);
    return out;
}

typedef Tensors AttentionSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, double, bool, const MaybeTensor &,
                                   const MaybeTensor &, const MaybeTensor &, bool);
typedef Tensors AttentionBackwardSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                           const Tensor &, const Tensor &, double, bool, const MaybeTensor &, const MaybeTensor &,
                                           const MaybeTensor &, bool, bool, bool);

struct AttentionNode : public GradNode {
    double scale = 0;
    bool causal = false;
    std::string name() const override { return "DiffAttentionBackward"; }
    variable_list apply(variable_list &&grads) override
    {
        static const auto op = find<AttentionBackwardSignature>("mamtorch_kernel_encoder::diff_attention_backward");
        variable_list out(4);
        if (!grads[0].defined()) return out;
        check_saved();
        const bool q = task_should_compute_output(0), k = task_should_compute_output(1), v = task_should_compute_output(2);
        const bool lam = task_should_compute_output(3);
        Tensors g;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(grads[0], take(0), take(1), take(2), take(3), take(4), take(5), take(6), scale, causal, maybe(take(7)), maybe(take(8)),
                        maybe(take(9)), q, k || v, lam);
        }
        if (q) out[0] = g[0];
        if (k) out[1] = g[1];
        if (v) out[2] = g[2];
        if (lam) out[3] = g[3];
        check_differentiated_once(grads, out);
        return out;
    }
};

Tensors diff_attention_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lam, double scale, bool causal,
                                const MaybeTensor &lengths, const MaybeTensor &starts, const MaybeTensor &key_mask, bool with_sums)
{
    static const auto op = find<AttentionSignature>("mamtorch_kernel_encoder::diff_attention");
    check_no_tangent("diff_attention", q, k, v, lam);
    const bool record = recording(q, k, v, lam);
    Tensors out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(q, k, v, lam, scale, causal, lengths, starts, key_mask, with_sums || record);
    }
    if (!record) return out;
    const auto node = node_of<AttentionNode>(q, k, v, lam);
    node->scale = scale;
    node->causal = causal;
    torch::autograd::set_history(out[0], node);
    for (const Tensor &t : {q, k, v, lam}) node->save(t);
    node->save_output(out[0]);
    for (const Tensor &t : {out[1], out[2], or_none(lengths), or_none(starts), or_none(key_mask)}) node->save(t);
    return out;
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
