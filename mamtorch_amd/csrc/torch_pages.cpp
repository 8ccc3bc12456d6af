// torch operators of differential attention with positions and of its paged cache (namespace mamtorch_kernel_encoder): norms with rotation and their gradient, the
// pages' bookkeeping, attention over pages.  Tensor checks, outputs, workspaces and the current stream for the C ABI of libmam_hip.so.  No kernels here.
#include "torch_encoder.h"

namespace {

typedef std::tuple<Tensor, Tensor> Pair;

// Tensors that a call changes: what has saved one of them for a backward pass is told so.
void changed(const Tensor &t)
{
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_whole(const Tensor &t, const Tensor &like, at::IntArrayRef sizes, const char *name)
{
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " is on a different device");
    TORCH_CHECK(t.scalar_type() == at::kInt && t.sizes() == sizes && t.is_contiguous(), name, " must be a contiguous int32 tensor of ", sizes, ", got ",
                t.scalar_type(), " of ", t.sizes());
}
const int32_t *ints(const MaybeTensor &t) { return has(t) ? t->data_ptr<int32_t>() : nullptr; }

// ---- norms with rotation ----
struct RotateCall {
    mam_norm_rotate_t a;
    Tensor q, k;                // what the pointers belong to
};

void check_heads(const Tensor &q, const Tensor &k)
{
    TORCH_CHECK(q.dim() == 5 && k.dim() == 5, "q and k must be (batch, tokens, heads, maps, head size), got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3) && k.size(4) == q.size(4), "q ", q.sizes(), " and k ", k.sizes(),
                " do not match");
    TORCH_CHECK(k.device() == q.device(), "k is on a different device");
    TORCH_CHECK(k.scalar_type() == q.scalar_type(), "k must have q's type ", q.scalar_type(), ", got ", k.scalar_type());
}

RotateCall rotate_call(const Tensor &q, const Tensor &k, const MaybeTensor &q_weight, const MaybeTensor &k_weight, const MaybeTensor &frequencies,
                       const MaybeTensor &positions, double eps, bool norm, bool interleaved)
{
    RotateCall c{};
    mam_norm_rotate_t &a = c.a;
    a.type = type_of(q, "q");
    check_heads(q, k);
    a.B = q.size(0); a.L = q.size(1); a.H = q.size(2); a.Hkv = k.size(2); a.M = q.size(3); a.D = q.size(4);
    TORCH_CHECK(a.D >= 1 && a.D <= 128, "head sizes are 1 to 128, got ", a.D);
    a.weight_type = a.type;
    const Tensor *first = nullptr;
    for (const MaybeTensor *t : {&q_weight, &k_weight}) {
        const char *name = t == &q_weight ? "q_weight" : "k_weight";
        if (!has(*t)) continue;
        TORCH_CHECK(norm, name, " is for calls with a norm");
        TORCH_CHECK((*t)->device() == q.device(), name, " is on a different device");
        const int got = type_of(**t, name);
        TORCH_CHECK(got == a.type || got == MAM_F32, name, " must be float32 or of q's type");
        TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == a.D && (*t)->is_contiguous(), name, " must be a contiguous vector of ", a.D, " elements");
        TORCH_CHECK(!first || first->scalar_type() == (*t)->scalar_type(), "q_weight and k_weight must be of one type");
        first = &**t;
        a.weight_type = got;
    }
    if (has(frequencies)) {
        TORCH_CHECK(frequencies->device() == q.device(), "frequencies is on a different device");
        TORCH_CHECK(frequencies->scalar_type() == at::kDouble && frequencies->dim() == 1 && frequencies->is_contiguous() && 2 * frequencies->size(0) <= a.D,
                    "frequencies must be a contiguous float64 vector of at most ", a.D / 2, " pairs, got ", frequencies->scalar_type(), " of ",
                    frequencies->sizes());
        a.frequencies = frequencies->data_ptr<double>();
        a.pairs = frequencies->size(0);
    }
    if (has(positions)) {
        TORCH_CHECK(positions->device() == q.device(), "positions is on a different device");
        TORCH_CHECK(positions->scalar_type() == at::kInt && positions->dim() == 2 && positions->size(0) == a.B && positions->size(1) == a.L,
                    "positions must be an int32 tensor of (", a.B, ", ", a.L, "), got ", positions->scalar_type(), " of ", positions->sizes());
        a.positions = positions->data_ptr<int32_t>();
        a.position_stride[0] = positions->stride(0);
        a.position_stride[1] = positions->stride(1);
    }
    TORCH_CHECK(!norm || (eps >= 0 && eps <= 1e30), "eps must not be negative, and finite, got ", eps);
    c.q = unit_last(q);
    c.k = unit_last(k);
    a.q = c.q.data_ptr();
    a.k = c.k.data_ptr();
    a.q_weight = ptr(q_weight);
    a.k_weight = ptr(k_weight);
    for (int i = 0; i < 4; ++i) {
        a.q_stride[i] = c.q.stride(i);
        a.k_stride[i] = c.k.stride(i);
    }
    a.eps = eps;
    a.norm = norm;
    a.interleaved = interleaved;
    return c;
}

Pair norm_rotate_cuda(const Tensor &q, const Tensor &k, const MaybeTensor &q_weight, const MaybeTensor &k_weight, const MaybeTensor &frequencies,
                      const MaybeTensor &positions, double eps, bool norm, bool interleaved)
{
    const c10::DeviceGuard guard(q.device());
    const RotateCall c = rotate_call(q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved);
    Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
    check_rc(mam_norm_rotate(&c.a, q_out.data_ptr(), k_out.data_ptr(), current_stream(q)), "mam_norm_rotate");
    return {q_out, k_out};
}

// wanted: the gradients of q, k and their weights; a gradient of an output that is not there is zero
Tensors norm_rotate_backward_cuda(const MaybeTensor &q_grad, const MaybeTensor &k_grad, const Tensor &q, const Tensor &k, const MaybeTensor &q_weight,
                                  const MaybeTensor &k_weight, const MaybeTensor &frequencies, const MaybeTensor &positions, double eps, bool norm,
                                  bool interleaved, bool want_q, bool want_k, bool want_q_weight, bool want_k_weight)
{
    const c10::DeviceGuard guard(q.device());
    const RotateCall c = rotate_call(q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved);
    Tensor g[2];
    int64_t strides[2][4] = {};
    for (int i = 0; i < 2; ++i) {
        const MaybeTensor &grad = i ? k_grad : q_grad;
        TORCH_CHECK(has(grad) || !(i ? want_k || want_k_weight : want_q || want_q_weight), "a gradient that is wanted needs its output's");
        if (!has(grad)) continue;
        check_like(*grad, i ? k : q, i ? "k_grad" : "q_grad");
        g[i] = unit_last(*grad);
        for (int n = 0; n < 4; ++n) strides[i][n] = g[i].stride(n);
    }
    const bool weights = want_q_weight || want_k_weight;
    TORCH_CHECK(!weights || norm, "there is no norm whose weights have gradients");
    const auto options = q.options().dtype(c.a.weight_type == MAM_F32 ? at::kFloat : q.scalar_type());
    Tensor dq, dk, dqw, dkw;
    if (want_q) dq = at::empty(q.sizes(), q.options());
    if (want_k) dk = at::empty(k.sizes(), k.options());
    if (want_q_weight) dqw = at::empty({c.a.D}, options);
    if (want_k_weight) dkw = at::empty({c.a.D}, options);
    const Tensor ws = workspace_for(weights ? mam_norm_rotate_backward_workspace(&c.a) : 0, q);
    check_rc(mam_norm_rotate_backward(&c.a, out_ptr(g[0]), strides[0], out_ptr(g[1]), strides[1], out_ptr(dq), out_ptr(dk), out_ptr(dqw), out_ptr(dkw),
                                      out_ptr(ws), ws.defined() ? ws.numel() : 0, current_stream(q)),
             "mam_norm_rotate_backward");
    return {or_empty(dq, q), or_empty(dk, q), or_empty(dqw, q), or_empty(dkw, q)};
}

typedef Pair RotateSignature(const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, double, bool,
                             bool);
typedef Tensors RotateBackwardSignature(const MaybeTensor &, const MaybeTensor &, const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &,
                                        const MaybeTensor &, const MaybeTensor &, double, bool, bool, bool, bool, bool, bool);

struct RotateNode : public GradNode {
    double eps = 0;
    bool norm = true, interleaved = false;
    std::string name() const override { return "NormRotateBackward"; }
    variable_list apply(variable_list &&grads) override
    {
        static const auto op = find<RotateBackwardSignature>("mamtorch_kernel_encoder::norm_rotate_backward");
        variable_list out(4);
        const bool from_q = grads[0].defined(), from_k = grads[1].defined();
        if (!from_q && !from_k) return out;
        check_saved();
        const bool q = from_q && task_should_compute_output(0), k = from_k && task_should_compute_output(1);
        const bool qw = from_q && task_should_compute_output(2), kw = from_k && task_should_compute_output(3);
        Tensors g;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            g = op.call(maybe(grads[0]), maybe(grads[1]), take(0), take(1), maybe(take(2)), maybe(take(3)), maybe(take(4)), maybe(take(5)), eps, norm,
                        interleaved, q, k, qw, kw);
        }
        if (q) out[0] = g[0];
        if (k) out[1] = g[1];
        if (qw) out[2] = g[2];
        if (kw) out[3] = g[3];
        check_differentiated_once(grads, out);
        return out;
    }
};

Pair norm_rotate_autograd(const Tensor &q, const Tensor &k, const MaybeTensor &q_weight, const MaybeTensor &k_weight, const MaybeTensor &frequencies,
                          const MaybeTensor &positions, double eps, bool norm, bool interleaved)
{
    static const auto op = find<RotateSignature>("mamtorch_kernel_encoder::norm_rotate");
    check_no_tangent("norm_rotate", q, k, q_weight, k_weight);
    TORCH_CHECK_NOT_IMPLEMENTED(!wants(frequencies), "norm_rotate has no gradient of the frequencies");
    Pair out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = op.call(q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved);
    }
    if (!recording(q, k, q_weight, k_weight)) return out;
    const auto node = node_of<RotateNode>(q, k, or_none(q_weight), or_none(k_weight));
    node->eps = eps;
    node->norm = norm;
    node->interleaved = interleaved;
    for (const Tensor &t : {q, k, or_none(q_weight), or_none(k_weight), or_none(frequencies), or_none(positions)}) node->save(t);
    torch::autograd::set_history(std::get<0>(out), node);
    torch::autograd::set_history(std::get<1>(out), node);
    return out;
}

// ---- pages ----
mam_pages_t pages_of(const Tensor &k, const Tensor &v, const MaybeTensor &table, const MaybeTensor &lengths, const MaybeTensor &counts)
{
    mam_pages_t p{};
    p.type = type_of(k, "k_pages");
    TORCH_CHECK(v.device() == k.device(), "v_pages is on a different device");
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), "v_pages must have k_pages's type ", k.scalar_type(), ", got ", v.scalar_type());
    TORCH_CHECK(k.dim() == 5 && k.size(3) == 2 && k.is_contiguous(), "k_pages must be a contiguous (pages, key heads, page size, 2, head size), got ", k.sizes());
    TORCH_CHECK(v.dim() == 4 && v.is_contiguous(), "v_pages must be a contiguous (pages, key heads, page size, value size), got ", v.sizes());
    p.P = k.size(0); p.Hkv = k.size(1); p.S = k.size(2); p.D = k.size(4); p.Dv = v.size(3);
    TORCH_CHECK(v.size(0) == p.P && v.size(1) == p.Hkv && v.size(2) == p.S, "k_pages ", k.sizes(), " and v_pages ", v.sizes(), " do not match");
    TORCH_CHECK(p.S >= 16 && p.S % 16 == 0, "a page holds a multiple of 16 tokens, got ", p.S);
    TORCH_CHECK(p.D >= 1 && p.D <= 128 && p.Dv >= 1 && p.Dv <= 256, "head sizes are 1 to 128 and value sizes 1 to 256, got ", p.D, " and ", p.Dv);
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    if (!has(table)) return p;
    TORCH_CHECK(table->dim() == 2, "table must be (batch, slots), got ", table->sizes());
    p.B = table->size(0);
    p.slots = table->size(1);
    check_whole(*table, k, {p.B, p.slots}, "table");
    check_whole(*lengths, k, {p.B}, "lengths");
    if (has(counts)) check_whole(*counts, k, {p.B}, "counts");
    p.table = ints(table);
    p.lengths = ints(lengths);
    p.counts = ints(counts);
    return p;
}

Tensor norm_rotate_append_cuda(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
                               const Tensor &lengths, const MaybeTensor &counts, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                               const MaybeTensor &frequencies, const MaybeTensor &positions, double eps, bool norm, bool interleaved)
{
    const c10::DeviceGuard guard(q.device());
    const RotateCall c = rotate_call(q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved);
    TORCH_CHECK(c.a.M == 2, "q must be (batch, tokens, heads, 2, head size), got ", q.sizes());
    const mam_pages_t p = pages_of(k_pages, v_pages, table, lengths, counts);
    TORCH_CHECK(k_pages.device() == q.device(), "k_pages is on a different device");
    TORCH_CHECK(p.type == c.a.type, "k_pages must have q's type ", q.scalar_type(), ", got ", k_pages.scalar_type());
    TORCH_CHECK(v.device() == q.device(), "v is on a different device");
    TORCH_CHECK(v.scalar_type() == q.scalar_type(), "v must have q's type ", q.scalar_type(), ", got ", v.scalar_type());
    TORCH_CHECK(v.dim() == 4 && v.size(0) == c.a.B && v.size(1) == c.a.L && v.size(2) == c.a.Hkv, "k ", k.sizes(), " and v ", v.sizes(), " do not match");
    TORCH_CHECK(p.Hkv == c.a.Hkv && p.D == c.a.D && p.Dv == v.size(3), "the pages, ", k_pages.sizes(), " and ", v_pages.sizes(), ", are for other keys than ",
                k.sizes(), " and ", v.sizes());
    TORCH_CHECK(p.B == c.a.B, "the table is for ", p.B, " requests, got ", c.a.B);
    const Tensor vs = unit_last(v);
    const int64_t strides[3] = {vs.stride(0), vs.stride(1), vs.stride(2)};
    Tensor out = at::empty(q.sizes(), q.options());
    check_rc(mam_norm_rotate_append(&c.a, vs.data_ptr(), strides, &p, out.data_ptr(), current_stream(q)), "mam_norm_rotate_append");
    changed(k_pages);
    changed(v_pages);
    return out;
}

struct Book { int64_t B, slots, P; };
Book book_of(const Tensor &table, const Tensor &lengths, const Tensor &refs, const Tensor &more, const char *name)
{
    TORCH_CHECK(table.is_cuda(), "table must be on the GPU");
    TORCH_CHECK(table.dim() == 2, "table must be (batch, slots), got ", table.sizes());
    TORCH_CHECK(refs.dim() == 1, "refs must be (pages), got ", refs.sizes());
    const Book b{table.size(0), table.size(1), refs.size(0)};
    check_whole(table, table, {b.B, b.slots}, "table");
    check_whole(lengths, table, {b.B}, "lengths");
    check_whole(refs, table, {b.P}, "refs");
    check_whole(more, table, {b.B}, name);
    return b;
}

Pair pages_extend_cuda(const Tensor &table, const Tensor &lengths, const Tensor &refs, const Tensor &counts, int64_t page_size)
{
    const c10::DeviceGuard guard(table.device());
    const Book b = book_of(table, lengths, refs, counts, "counts");
    Tensor granted = at::empty({b.B}, table.options()), copies = at::empty({b.B, 2}, table.options());
    const Tensor ws = workspace_for(mam_pages_extend_workspace(b.B, b.slots, b.P), table);
    check_rc(mam_pages_extend(table.data_ptr<int32_t>(), ints(lengths), refs.data_ptr<int32_t>(), ints(counts), granted.data_ptr<int32_t>(),
                              copies.data_ptr<int32_t>(), b.B, b.slots, b.P, page_size, out_ptr(ws), ws.defined() ? ws.numel() : 0, current_stream(table)),
             "mam_pages_extend");
    changed(table);
    changed(refs);
    return {granted, copies};
}

void pages_fork_cuda(const Tensor &table, const Tensor &lengths, const Tensor &refs, const Tensor &sources, int64_t page_size)
{
    const c10::DeviceGuard guard(table.device());
    const Book b = book_of(table, lengths, refs, sources, "sources");
    check_rc(mam_pages_fork(table.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), refs.data_ptr<int32_t>(), ints(sources), b.B, b.slots, b.P, page_size,
                            current_stream(table)),
             "mam_pages_fork");
    for (const Tensor *t : {&table, &lengths, &refs}) changed(*t);
}

void pages_trim_cuda(const Tensor &table, const Tensor &lengths, const Tensor &refs, const Tensor &ends, int64_t page_size)
{
    const c10::DeviceGuard guard(table.device());
    const Book b = book_of(table, lengths, refs, ends, "ends");
    check_rc(mam_pages_trim(table.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), refs.data_ptr<int32_t>(), ints(ends), b.B, b.slots, b.P, page_size,
                            current_stream(table)),
             "mam_pages_trim");
    for (const Tensor *t : {&table, &lengths, &refs}) changed(*t);
}

void pages_copy_cuda(const Tensor &k_pages, const Tensor &v_pages, const Tensor &copies)
{
    const c10::DeviceGuard guard(k_pages.device());
    const mam_pages_t p = pages_of(k_pages, v_pages, c10::nullopt, c10::nullopt, c10::nullopt);
    TORCH_CHECK(copies.dim() == 2 && copies.size(1) == 2, "copies must be (pairs, 2), got ", copies.sizes());
    check_whole(copies, k_pages, {copies.size(0), 2}, "copies");
    check_rc(mam_pages_copy(&p, ints(copies), copies.size(0), current_stream(k_pages)), "mam_pages_copy");
    changed(k_pages);
    changed(v_pages);
}

void pages_compact_cuda(const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lengths, const Tensor &path, const MaybeTensor &counts)
{
    const c10::DeviceGuard guard(k_pages.device());
    const mam_pages_t p = pages_of(k_pages, v_pages, table, lengths, counts);
    TORCH_CHECK(path.dim() == 2 && path.size(0) == p.B, "path must be (", p.B, ", tokens), got ", path.sizes());
    check_whole(path, k_pages, {p.B, path.size(1)}, "path");
    check_rc(mam_pages_compact(&p, ints(path), path.size(1), current_stream(k_pages)), "mam_pages_compact");
    changed(k_pages);
    changed(v_pages);
}

Pair draft_tree_cuda(const Tensor &parents, const MaybeTensor &lengths)
{
    TORCH_CHECK(parents.is_cuda(), "parents must be on the GPU");
    const c10::DeviceGuard guard(parents.device());
    TORCH_CHECK(parents.dim() == 2 && parents.size(1) <= 64, "parents must be (batch, tokens) with 64 tokens at most, got ", parents.sizes());
    const int64_t b = parents.size(0), n = parents.size(1);
    check_whole(parents, parents, {b, n}, "parents");
    if (has(lengths)) check_whole(*lengths, parents, {b}, "lengths");
    Tensor masks = at::empty({b, n}, parents.options().dtype(at::kLong)), positions = at::empty({b, n}, parents.options());
    check_rc(mam_draft_tree(ints(parents), ints(lengths), masks.data_ptr<int64_t>(), positions.data_ptr<int32_t>(), b, n, current_stream(parents)),
             "mam_draft_tree");
    return {masks, positions};
}

Tensor diff_attention_pages_cuda(const Tensor &q, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lengths, const Tensor &lam,
                                 double scale, const MaybeTensor &counts, const MaybeTensor &masks)
{
    const c10::DeviceGuard guard(q.device());
    mam_diff_attention_pages_t a{};
    const int type = type_of(q, "q");
    a.pages = pages_of(k_pages, v_pages, table, lengths, counts);
    const mam_pages_t &p = a.pages;
    TORCH_CHECK(k_pages.device() == q.device(), "k_pages is on a different device");
    TORCH_CHECK(p.type == type, "k_pages must have q's type ", q.scalar_type(), ", got ", k_pages.scalar_type());
    TORCH_CHECK(q.dim() == 5 && q.size(3) == 2, "q must be (batch, tokens, heads, 2, head size), got ", q.sizes());
    a.N = q.size(1);
    a.H = q.size(2);
    TORCH_CHECK(q.size(4) == p.D, "q ", q.sizes(), " and k_pages ", k_pages.sizes(), " do not match");
    TORCH_CHECK(q.size(0) == p.B, "the table is for ", p.B, " requests, got ", q.size(0));
    TORCH_CHECK(a.H == 0 || (p.Hkv > 0 && a.H % p.Hkv == 0), "the ", p.Hkv, " key heads must divide the ", a.H, " query heads");
    TORCH_CHECK(lam.device() == q.device(), "lam is on a different device");
    a.lam_type = type_of(lam, "lam");
    TORCH_CHECK(a.lam_type == type || a.lam_type == MAM_F32, "lam must be float32 or of q's type");
    TORCH_CHECK(lam.dim() == 1 && lam.size(0) == a.H && lam.is_contiguous(), "lam must be a contiguous vector of ", a.H, " heads");
    TORCH_CHECK(static_cast<float>(scale) > 0 && scale <= 1e30, "scale must be positive and finite in float32, got ", scale);
    if (has(masks)) {
        TORCH_CHECK(a.N <= 64, "a tree has 64 tokens at most, got ", a.N);
        TORCH_CHECK(masks->device() == q.device(), "masks is on a different device");
        TORCH_CHECK(masks->scalar_type() == at::kLong && masks->dim() == 2 && masks->size(0) == p.B && masks->size(1) == a.N && masks->is_contiguous(),
                    "masks must be a contiguous int64 tensor of (", p.B, ", ", a.N, ")");
        a.masks = masks->data_ptr<int64_t>();
    }
    const Tensor qs = unit_last(q);
    a.q = qs.data_ptr();
    a.lam = lam.data_ptr();
    for (int i = 0; i < 4; ++i) a.q_stride[i] = qs.stride(i);
    a.scale = scale;
    Tensor out = at::empty({p.B, a.N, a.H, p.Dv}, q.options());
    const Tensor ws = workspace_for(mam_diff_attention_pages_workspace(&a), q);
    check_rc(mam_diff_attention_pages(&a, out.data_ptr(), out_ptr(ws), ws.defined() ? ws.numel() : 0, current_stream(q)), "mam_diff_attention_pages");
    return out;
}

// Serving's operators have no gradient; a graph that leaves them out without a word would be wrong.
void check_serving(bool record, const char *name)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!record, name, " has no gradient: call it under torch.no_grad()");
}

typedef Tensor AppendSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                               const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, double, bool, bool);

Tensor norm_rotate_append_autograd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
                                   const Tensor &lengths, const MaybeTensor &counts, const MaybeTensor &q_weight, const MaybeTensor &k_weight,
                                   const MaybeTensor &frequencies, const MaybeTensor &positions, double eps, bool norm, bool interleaved)
{
    static const auto op = find<AppendSignature>("mamtorch_kernel_encoder::norm_rotate_append");
    check_no_tangent("norm_rotate_append", q, k, v, k_pages, v_pages, q_weight, k_weight);
    check_serving(recording(q, k, v, k_pages, v_pages, q_weight, k_weight), "norm_rotate_append");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(q, k, v, k_pages, v_pages, table, lengths, counts, q_weight, k_weight, frequencies, positions, eps, norm, interleaved);
}

typedef void CopySignature(const Tensor &, const Tensor &, const Tensor &);

void pages_copy_autograd(const Tensor &k_pages, const Tensor &v_pages, const Tensor &copies)
{
    static const auto op = find<CopySignature>("mamtorch_kernel_encoder::pages_copy");
    check_serving(recording(k_pages, v_pages), "pages_copy");
    at::AutoDispatchBelowADInplaceOrView below;
    op.call(k_pages, v_pages, copies);
}

typedef void CompactSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const MaybeTensor &);

void pages_compact_autograd(const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lengths, const Tensor &path,
                            const MaybeTensor &counts)
{
    static const auto op = find<CompactSignature>("mamtorch_kernel_encoder::pages_compact");
    check_serving(recording(k_pages, v_pages), "pages_compact");
    at::AutoDispatchBelowADInplaceOrView below;
    op.call(k_pages, v_pages, table, lengths, path, counts);
}

typedef Tensor PagesSignature(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &, double, const MaybeTensor &,
                              const MaybeTensor &);

Tensor diff_attention_pages_autograd(const Tensor &q, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table, const Tensor &lengths,
                                     const Tensor &lam, double scale, const MaybeTensor &counts, const MaybeTensor &masks)
{
    static const auto op = find<PagesSignature>("mamtorch_kernel_encoder::diff_attention_pages");
    check_no_tangent("diff_attention_pages", q, k_pages, v_pages, lam);
    check_serving(recording(q, k_pages, v_pages, lam), "diff_attention_pages");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(q, k_pages, v_pages, table, lengths, lam, scale, counts, masks);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mamtorch_kernel_encoder, m)
{
    m.def("norm_rotate(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? frequencies, Tensor? positions, float eps, bool norm, "
          "bool interleaved) -> (Tensor, Tensor)");
    m.def("norm_rotate_backward(Tensor? q_grad, Tensor? k_grad, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? frequencies, "
          "Tensor? positions, float eps, bool norm, bool interleaved, bool want_q, bool want_k, bool want_q_weight, bool want_k_weight) -> Tensor[]");
    m.def("norm_rotate_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor table, Tensor lengths, Tensor? counts, "
          "Tensor? q_weight, Tensor? k_weight, Tensor? frequencies, Tensor? positions, float eps, bool norm, bool interleaved) -> Tensor");
    m.def("pages_extend(Tensor(a!) table, Tensor lengths, Tensor(b!) refs, Tensor counts, int page_size) -> (Tensor, Tensor)");
    m.def("pages_fork(Tensor(a!) table, Tensor(b!) lengths, Tensor(c!) refs, Tensor sources, int page_size) -> ()");
    m.def("pages_trim(Tensor(a!) table, Tensor(b!) lengths, Tensor(c!) refs, Tensor ends, int page_size) -> ()");
    m.def("pages_copy(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor copies) -> ()");
    m.def("pages_compact(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor table, Tensor lengths, Tensor path, Tensor? counts) -> ()");
    m.def("draft_tree(Tensor parents, Tensor? lengths) -> (Tensor, Tensor)");
    m.def("diff_attention_pages(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor lengths, Tensor lam, float scale, Tensor? counts, "
          "Tensor? masks) -> Tensor");
}

TORCH_LIBRARY_IMPL(mamtorch_kernel_encoder, CUDA, m)
{
    m.impl("norm_rotate", &norm_rotate_cuda);
    m.impl("norm_rotate_backward", &norm_rotate_backward_cuda);
    m.impl("norm_rotate_append", &norm_rotate_append_cuda);
    m.impl("pages_extend", &pages_extend_cuda);
    m.impl("pages_fork", &pages_fork_cuda);
    m.impl("pages_trim", &pages_trim_cuda);
    m.impl("pages_copy", &pages_copy_cuda);
    m.impl("pages_compact", &pages_compact_cuda);
    m.impl("draft_tree", &draft_tree_cuda);
    m.impl("diff_attention_pages", &diff_attention_pages_cuda);
}

TORCH_LIBRARY_IMPL(mamtorch_kernel_encoder, Autograd, m)
{
    m.impl("norm_rotate", &norm_rotate_autograd);
    m.impl("norm_rotate_append", &norm_rotate_append_autograd);
    m.impl("diff_attention_pages", &diff_attention_pages_autograd);
    m.impl("pages_copy", &pages_copy_autograd);
    m.impl("pages_compact", &pages_compact_autograd);
    // whole numbers alone: nothing for autograd to look at
    for (const char *name : {"pages_extend", "pages_fork", "pages_trim", "draft_tree"}) m.impl(name, torch::CppFunction::makeFallthrough());
}
