"""GPU tests of layer norm, counter-based dropout and their join against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(n, c, dtype, seed, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, generator=g) * (0.5 + torch.rand(c, generator=g)) + offset * torch.randn(c, generator=g)
    return x.to(dtype), (1 + 0.2 * torch.randn(c, generator=g)), 0.2 * torch.randn(c, generator=g), torch.randn(n, c, generator=g).to(dtype)


def _check_norm(x, w, b, dy, eps, x_gpu=None, dy_gpu=None):
    dtype = x.dtype
    xg = (x.to(DEV) if x_gpu is None else x_gpu).requires_grad_(True)
    wg, bg = (None if t is None else t.to(DEV).requires_grad_(True) for t in (w, b))
    y = enc.layer_norm(xg, wg, bg, eps)
    inputs = [t for t in (xg, wg, bg) if t is not None]
    grads = dict(zip([n for n, t in (("x", xg), ("w", wg), ("b", bg)) if t is not None],
                     torch.autograd.grad(y, inputs, dy.to(DEV) if dy_gpu is None else dy_gpu)))
    want, xh, rstd = ref.norm(x, w, b, eps)
    what = "%s %s" % (tuple(x.shape), dtype)
    ref.assert_within(y, want, ref.norm_bound(x, xh, rstd, w, b, want, dtype), what + " y")
    dx, dw, db = ref.norm_backward(dy, xh, rstd, w)
    bounds = ref.norm_backward_bound(x, dy, xh, rstd, w, dx, dw, db, dtype, dtype if w is None else w.dtype)
    assert grads["x"].dtype == dtype
    ref.assert_within(grads["x"], dx, bounds[0], what + " dx")
    if w is not None:
        assert grads["w"].dtype == w.dtype
        ref.assert_within(grads["w"], dw, bounds[1], what + " dw")
    if b is not None:
        ref.assert_within(grads["b"], db, bounds[2], what + " db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, c", [(1, 1), (3, 2), (5, 63), (64, 64), (33, 127), (17, 128), (40, 129), (9, 256), (7, 257), (197, 768), (1030, 768),
                                  (50, 1001), (12, 1024), (12, 1025), (31, 2048), (5, 4096), (6, 4097), (3, 9001), (4, 16384), (3, 16385),
                                  (70, 20001), (2100, 40)])
def test_norm_and_gradients(n, c, dtype):
    x, w, b, dy = _rows(n, c, dtype, seed=n + c)
    _check_norm(x, w.to(dtype), b.to(dtype), dy, 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("has_weight, has_bias", [(True, False), (False, True), (False, False), (True, True)])
def test_norm_with_32_bit_weights_or_without(has_weight, has_bias, dtype):
    x, w, b, dy = _rows(37, 193, dtype, seed=3)
    _check_norm(x, w if has_weight else None, b.to(dtype if not has_weight else torch.float32) if has_bias else None, dy, 1e-3)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_strided_rows_and_of_other_orders(dtype):
    x, w, b, dy = _rows(24, 100, dtype, seed=4)
    wide = torch.zeros(24, 131, dtype=dtype)
    wide[:, 7:107] = x
    wide_dy = torch.zeros(24, 333, dtype=dtype)
    wide_dy[:, 101:201] = dy
    _check_norm(x, w, b, dy, 1e-5, wide.to(DEV)[:, 7:107].detach(), wide_dy.to(DEV)[:, 101:201])
    # columns a row apart (no unit stride), and outer dimensions in another order
    _check_norm(x, w, b, dy, 1e-5, x.to(DEV).T.contiguous().T.detach(), dy.to(DEV))
    x3 = x.view(4, 6, 100).to(DEV).transpose(0, 1).contiguous().transpose(0, 1).detach()
    y = enc.layer_norm(x3, w.to(DEV), b.to(DEV))
    assert torch.equal(y.reshape(24, 100), enc.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV)))


def test_norm_of_rows_that_are_far_from_zero_or_constant():
    # the variance is that of what is left after the mean: 1 part in 4096 beside it keeps its digits
    x, w, b, dy = _rows(16, 768, torch.float32, seed=5)
    _check_norm(x + 4096.0, w, b, dy, 1e-5)
    y = enc.layer_norm(torch.full((3, 77), 5.0, device=DEV), None, None, 1e-5)
    assert torch.equal(y, torch.zeros_like(y))


def test_norm_of_infinities_stays_in_its_row():
    x, w, b, _ = _rows(9, 300, torch.float32, seed=6)
    x[4, 7] = float("inf")
    x[6, 8] = float("nan")
    y = enc.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV)).cpu()
    assert y[[4, 6]].isnan().any(1).all() and y[[0, 1, 2, 3, 5, 7, 8]].isfinite().all()


def test_norm_of_nothing():
    w = torch.ones(12, device=DEV, requires_grad=True)
    x = torch.empty(0, 12, device=DEV, requires_grad=True)
    y = enc.layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 12) and torch.equal(dw, torch.zeros_like(dw))
    assert enc.layer_norm(torch.empty(5, 0, device=DEV)).shape == (5, 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 511, 4096, 8191, 100001])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.0, 1.0])
def test_dropout_bits_and_gradient(n, p, dtype):
    g = torch.Generator().manual_seed(n)
    x, r, dy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    seed, offset = -n * 0x123456789ABCDEF, 2 ** 40 + n
    xg, rg = x.to(DEV).requires_grad_(True), r.to(DEV).requires_grad_(True)
    y = enc.dropout(xg, p, seed, offset)
    assert torch.equal(y.cpu(), ref.dropped(x, p, seed, offset))
    assert torch.equal(torch.autograd.grad(y, xg, dy.to(DEV))[0].cpu(), ref.dropped(dy, p, seed, offset))
    y = enc.dropout(xg, p, seed, offset, residual=rg)
    assert torch.equal(y.cpu(), ref.dropped(x, p, seed, offset, r))
    dx, dr = torch.autograd.grad(y, (xg, rg), dy.to(DEV))
    assert torch.equal(dx.cpu(), ref.dropped(dy, p, seed, offset)) and torch.equal(dr.cpu(), dy)


def test_dropout_of_views_follows_the_elements_order():
    x = torch.randn(6, 50, generator=torch.Generator().manual_seed(1))
    want = ref.dropped(x, 0.3, 5, 6)
    assert torch.equal(enc.dropout(x.to(DEV).T.contiguous().T, 0.3, 5, 6).cpu(), want)
    wide = torch.zeros(6, 53, device=DEV)
    wide[:, 1:51] = x.to(DEV)
    assert torch.equal(enc.dropout(wide[:, 1:51], 0.3, 5, 6).cpu(), want)
    flat = torch.zeros(301, device=DEV)
    flat[1:] = x.to(DEV).view(-1)           # 4-byte aligned
    assert torch.equal(enc.dropout(flat[1:], 0.3, 5, 6).cpu().view(6, 50), want)


def test_dropped_elements_are_zero_whatever_they_hold():
    x = torch.full((4096,), float("nan"), device=DEV)
    x[::2] = float("inf")
    keep = ref.keep_mask((4096,), 0.5, 9, 0)
    y = enc.dropout(x, 0.5, 9).cpu()
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum()))) and not y[keep].isfinite().any()
    # and their share is p, to five standard deviations of 2^20 draws
    ones = enc.dropout(torch.ones(2 ** 20, device=DEV), 0.1, 77, 3, scale=1.0)
    assert abs(ones.mean().item() - 0.9) < 5 * (0.09 / 2 ** 20) ** 0.5


def test_a_step_on_the_device_is_added_to_the_offset():
    x = torch.randn(1000, generator=torch.Generator().manual_seed(2))
    xg, step = x.to(DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    graph, warm = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(warm):
        enc.dropout(xg, 0.4, 11, 7, step=step)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = enc.dropout(xg, 0.4, 11, 7, step=step)
        step += 1
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), ref.dropped(x, 0.4, 11, 7 + k))
    assert step.item() == 4
    # a step that moved between the forward and the backward is an error and no other mask
    xg.requires_grad_(True)
    out = enc.dropout(xg, 0.4, 11, 7, step=step)
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, c, p", [(1, 1, 0.5), (5, 63, 0.1), (37, 130, 0.25), (64, 128, 0.0), (197, 768, 0.1), (30, 1001, 0.5), (11, 1026, 1.0),
                                     (12, 4099, 0.1), (3, 9002, 0.3), (5, 16387, 0.1)])
def test_join_and_gradients(n, c, p, dtype):
    x, w, b, dy = _rows(n, c, dtype, seed=n + c)
    r, _, _, ds = _rows(n, c, dtype, seed=n + c + 1)
    seed, offset = 2 ** 63 + n, c
    xg, rg, wg, bg = (t.to(DEV).requires_grad_(True) for t in (x, r, w, b))
    y, s = enc.add_dropout_layer_norm(xg, rg, wg, bg, p, seed, offset)
    s_want = ref.dropped(x, p, seed, offset, r)
    assert torch.equal(s.cpu(), s_want)
    want, xh, rstd = ref.norm(s_want, w, b, 1e-5)
    ref.assert_within(y, want, ref.norm_bound(s_want, xh, rstd, w, b, want, dtype), "y")
    keep = ref.keep_mask((n, c), p, seed, offset).double() * (1 / (1 - p) if p < 1 else 0)
    for with_ds in (True, False):
        outs, grads = ([y, s], [dy.to(DEV), ds.to(DEV)]) if with_ds else ([y], [dy.to(DEV)])
        dx, dr, dw, db = torch.autograd.grad(outs, (xg, rg, wg, bg), grads, retain_graph=True)
        more = ds.double() if with_ds else torch.zeros(n, c).double()
        grad, wantw, wantb = ref.norm_backward(dy, xh, rstd, w)
        bound, boundw, boundb = ref.norm_backward_bound(s_want, dy, xh, rstd, w, grad, wantw, wantb, dtype, torch.float32)
        bound = bound + (ref.UNIT[dtype] + 2 * ref.F32) * ((grad + more).abs() + more.abs())
        ref.assert_within(dr, grad + more, bound, "residual's gradient")
        # the factor is fp32: one more rounding of it, of the product, and of the result
        ref.assert_within(dx, (grad + more) * keep, bound * keep + (ref.UNIT[dtype] + 4 * ref.F32) * ((grad + more) * keep).abs() + ref.TINY[dtype],
                          "gradient behind the dropout")
        ref.assert_within(dw, wantw, boundw, "dw")
        ref.assert_within(db, wantb, boundb, "db")
    # only the sum is used further on
    dx, dr = torch.autograd.grad(s, (xg, rg), ds.to(DEV))
    assert torch.equal(dr.cpu(), ds) and torch.equal(dx.cpu(), ref.dropped(ds, p, seed, offset))


def test_two_calls_give_the_same_bits():
    x, w, b, dy = _rows(3000, 770, torch.bfloat16, seed=8)
    r = torch.randn(3000, 770, generator=torch.Generator().manual_seed(9)).bfloat16()
    xg, rg, wg, bg = (t.to(DEV).requires_grad_(True) for t in (x, r, w, b))
    runs = []
    for _ in range(2):
        y, s = enc.add_dropout_layer_norm(xg, rg, wg, bg, 0.1, 1, 2)
        runs.append([y, s, *torch.autograd.grad(y, (xg, rg, wg, bg), dy.to(DEV))])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_calls_on_another_stream_wait_for_nobody_and_are_right():
    x, w, b, _ = _rows(500, 768, torch.float32, seed=10)
    xg, wg, bg = x.to(DEV), w.to(DEV), b.to(DEV)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        y = enc.layer_norm(xg, wg, bg)
        z = enc.dropout(y, 0.2, 3, 4)
    other.synchronize()
    assert torch.equal(z.cpu(), ref.dropped(y.cpu(), 0.2, 3, 4))
    assert torch.equal(y, enc.layer_norm(xg, wg, bg))


def test_refusals():
    x, w = torch.randn(4, 6, device=DEV), torch.ones(6, device=DEV)
    bad = [lambda: enc.layer_norm(x.double(), w.double()), lambda: enc.layer_norm(x, torch.ones(5, device=DEV)),
           lambda: enc.layer_norm(x, w.half()), lambda: enc.layer_norm(x.half(), w, w.half()), lambda: enc.layer_norm(x, w.cpu()),
           lambda: enc.dropout(x, 1.5, 1), lambda: enc.dropout(x, -0.1, 1), lambda: enc.dropout(x, float("nan"), 1),
           lambda: enc.dropout(x, 0.1, 1, residual=x[:2]), lambda: enc.dropout(x, 0.1, 1, residual=x.half()),
           lambda: enc.dropout(x, 0.1, 1, step=torch.zeros(2, dtype=torch.int64, device=DEV)),
           lambda: enc.dropout(x, 0.1, 1, step=torch.zeros(1, dtype=torch.int64)),
           lambda: enc.add_dropout_layer_norm(x, x[:, :5], w), lambda: enc.add_dropout_layer_norm(x, x, w, p=2.0),
           lambda: enc.layer_norm(torch.tensor(1.0, device=DEV))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises((NotImplementedError, RuntimeError)):
        enc.layer_norm(x.cpu(), w.cpu())


def test_opcheck():
    x, w, b, dy = _rows(6, 20, torch.float32, seed=11)
    x, w, b = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    ops = torch.ops.mamtorch_kernel_encoder
    torch.library.opcheck(ops.layer_norm, (x, w, b, 1e-5, True), test_utils=tests)
    torch.library.opcheck(ops.dropout, (x, None, 0.1, 1.1, 5, 6, None), test_utils=tests)
    torch.library.opcheck(ops.add_dropout_layer_norm, (x, x, w, b, 0.1, 1.1, 5, 6, 1e-5, None, True), test_utils=tests)
    _, mean, rstd = ops.layer_norm(x.detach(), None, None, 1e-5, True)
    torch.library.opcheck(ops.layer_norm_backward, (dy.to(DEV), x.detach(), w.detach(), mean, rstd, True, True, True, True),
                          test_utils=("test_schema", "test_faketensor"))
