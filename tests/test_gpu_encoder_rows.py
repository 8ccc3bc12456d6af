"""GPU tests of norms and joins whose operands or gradients have rows of stride 0: broadcast tensors and the gradients of sums."""
import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]
B, L, C = 5, 7, 72
# what of (B, L, C) there is, and what sums give it such a gradient
SHAPES = {"batch": (1, L, C), "tokens": (B, 1, C), "rows": (1, 1, C)}
SUMS = {"batch": 0, "tokens": 1, "rows": (0, 1)}


def _make(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _weights():
    return 1 + _make((C,), torch.float32, 1, 0.2), _make((C,), torch.float32, 2, 0.2)


def _flat(t):
    return t.expand(B, L, C).reshape(B * L, C)


def _leaf(t):
    """(B, L, C) on the GPU with the strides of a broadcast, as a leaf of its own."""
    wide = t.to(DEV).expand(B, L, C).detach()
    assert t.shape == (B, L, C) or 0 in wide.stride()
    return wide.requires_grad_(True)


def _check_gradients(got, x, dy, more, w, b, keep, dtype, what):
    """got: gradients of x, (residual,) weight, bias, for x as normalised, the norm's gradient dy and the sum's own `more`."""
    _, xh, rstd = ref.norm(x, w, b, 1e-5)
    dx, dw, db = ref.norm_backward(dy, xh, rstd, w)
    bound, bound_w, bound_b = ref.norm_backward_bound(x, dy, xh, rstd, w, dx, dw, db, dtype, torch.float32)
    if keep is not None:        # as the joins' own tests have it: one more sum, and the factor's and the product's roundings behind the dropout
        dx = dx + more.double()
        bound = bound + (ref.UNIT[dtype] + 2 * ref.F32) * (dx.abs() + more.double().abs())
        ref.assert_within(got.pop(0).reshape(B * L, C), dx * keep, bound * keep + (ref.UNIT[dtype] + 4 * ref.F32) * (dx * keep).abs() + ref.TINY[dtype],
                          what + " behind the dropout")
    ref.assert_within(got[0].reshape(B * L, C), dx, bound, what + " dx")
    ref.assert_within(got[1], dw, bound_w, what + " dw")
    ref.assert_within(got[2], db, bound_b, what + " db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", SHAPES)
def test_norm_of_a_broadcast_operand(kind, dtype):
    x, dy, (w, b) = _make(SHAPES[kind], dtype, 3), _make((B, L, C), dtype, 4), _weights()
    leaves = [_leaf(x), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    y = enc.layer_norm(*leaves)
    want, xh, rstd = ref.norm(_flat(x), w, b, 1e-5)
    ref.assert_within(y.reshape(B * L, C), want, ref.norm_bound(_flat(x), xh, rstd, w, b, want, dtype), kind)
    _check_gradients(list(torch.autograd.grad(y, leaves, dy.to(DEV))), _flat(x), _flat(dy), None, w, b, None, dtype, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", SUMS)
def test_gradients_of_a_norm_that_is_summed(kind, dtype):
    x, dy, (w, b) = _make((B, L, C), dtype, 5), _make(SHAPES[kind], dtype, 6), _weights()
    leaves = [x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    total = enc.layer_norm(*leaves).sum(SUMS[kind])
    grads = torch.autograd.grad(total, leaves, dy.to(DEV).reshape(total.shape))
    _check_gradients(list(grads), _flat(x), _flat(dy), None, w, b, None, dtype, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", SHAPES)
@pytest.mark.parametrize("which", ["x", "residual"])
def test_join_of_a_broadcast_operand(which, kind, dtype):
    x, r = (_make(SHAPES[kind] if which == name else (B, L, C), dtype, n) for n, name in ((7, "x"), (8, "residual")))
    dy, (w, b), p = _make((B, L, C), dtype, 9), _weights(), 0.25
    leaves = [_leaf(x), _leaf(r), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    y, s = enc.add_dropout_layer_norm(*leaves, p, 21, 22)
    s_want = ref.dropped(_flat(x), p, 21, 22, _flat(r))
    assert torch.equal(s.reshape(B * L, C).cpu(), s_want)
    want, xh, rstd = ref.norm(s_want, w, b, 1e-5)
    ref.assert_within(y.reshape(B * L, C), want, ref.norm_bound(s_want, xh, rstd, w, b, want, dtype), kind)
    keep = ref.keep_mask((B * L, C), p, 21, 22).double() / (1 - p)
    _check_gradients(list(torch.autograd.grad(y, leaves, dy.to(DEV))), s_want, _flat(dy), torch.zeros(B * L, C), w, b, keep, dtype, kind)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", SUMS)
@pytest.mark.parametrize("summed", ["y", "s", "both"])
def test_gradients_of_a_join_that_is_summed(summed, kind, dtype):
    x, r, (w, b), p = _make((B, L, C), dtype, 10), _make((B, L, C), dtype, 11), _weights(), 0.25
    dy, ds = (_make(SHAPES[kind] if summed in (name, "both") else (B, L, C), dtype, n) for n, name in ((12, "y"), (13, "s")))
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, r, w, b)]
    outs = list(enc.add_dropout_layer_norm(*leaves, p, 21, 22))
    for n, name in enumerate("ys"):
        if summed in (name, "both"):
            outs[n] = outs[n].sum(SUMS[kind])
    grads = torch.autograd.grad(outs, leaves, [t.to(DEV).reshape(o.shape) for o, t in zip(outs, (dy, ds))])
    keep = ref.keep_mask((B * L, C), p, 21, 22).double() / (1 - p)
    _check_gradients(list(grads), ref.dropped(_flat(x), p, 21, 22, _flat(r)), _flat(dy), _flat(ds), w, b, keep, dtype, kind)


def test_dropout_of_a_broadcast_operand():
    x, r = _make((1, 1, C), torch.float32, 14), _make((B, 1, C), torch.float32, 15)
    xg, rg = _leaf(x), _leaf(r)
    y = enc.dropout(xg, 0.3, 5, 6, residual=rg)
    assert torch.equal(y.cpu(), ref.dropped(x.expand(B, L, C), 0.3, 5, 6, r.expand(B, L, C)))
    total = enc.dropout(xg, 0.3, 5, 6).sum(1)
    dy = _make((B, C), torch.float32, 16)
    dx, = torch.autograd.grad(total, xg, dy.to(DEV))
    assert torch.equal(dx.cpu(), ref.dropped(dy[:, None].expand(B, L, C), 0.3, 5, 6))
