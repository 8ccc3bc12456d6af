"""GPU tests of how the encoder operators stand in a graph: outputs unused, second derivatives, tangents, saved tensors, transforms."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder


def _leaf(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV).requires_grad_(True)


def _norm(x):
    return enc.layer_norm(x, torch.ones(x.shape[-1], device=DEV), None)


def _join(x):
    return enc.add_dropout_layer_norm(x, torch.ones_like(x), None, None, 0.5, 3, 4)[0]


def _attention(x):
    q = x.reshape(2, 3, 2, 2, 16)
    return enc.diff_attention(q, q, x.reshape(2, 3, 2, 32), torch.full((2,), 0.5, device=DEV))


CALLS = [_norm, _join, _attention]


@pytest.mark.parametrize("call", CALLS)
def test_a_second_derivative_is_an_error(call):
    x = _leaf(6, 64)
    g, = torch.autograd.grad(call(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.sum(), x)
    # A graph for the gradient that nobody differentiates is harmless and changes nothing.
    plain, = torch.autograd.grad(call(x).square().sum(), x)
    assert torch.equal(g.detach(), plain)


def test_dropout_is_linear_and_can_be_differentiated_twice():
    x = _leaf(6, 64)
    y = enc.dropout(x, 0.5, 3, 4)
    g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)       # 2 f^2 x with the factors f of 0 and 2
    h, = torch.autograd.grad(g.sum(), x)
    assert torch.equal(h, 2 * torch.where(y != 0, 4.0, 0.0))


@pytest.mark.parametrize("call", CALLS + [lambda x: enc.dropout(x, 0.5, 3, 4)])
@pytest.mark.parametrize("wants", [False, True])
def test_a_tangent_is_refused(call, wants):
    x = _leaf(6, 64).detach().requires_grad_(wants)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)


@pytest.mark.parametrize("call", CALLS)
def test_a_graph_is_walked_once_unless_it_is_kept(call):
    x = _leaf(6, 64)
    y = call(x).sum()
    first, = torch.autograd.grad(y, x, retain_graph=True)
    second, = torch.autograd.grad(y, x)
    assert torch.equal(first, second)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x)


@pytest.mark.parametrize("call", CALLS)
def test_a_saved_operand_that_was_changed_is_noticed(call):
    x = _leaf(6, 64)
    t = x * 1
    y = call(t)
    if call is _join:
        # The join keeps its sum and not its operands.
        t.add_(1)
        want, = torch.autograd.grad(_join(x).sum(), x)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want)
        return
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_join_with_one_output_used():
    x, r = _leaf(6, 64), _leaf(6, 64, seed=1)
    y, s = enc.add_dropout_layer_norm(x, r, None, None, 0.5, 3, 4)
    dy = torch.randn(6, 64, device=DEV)
    gx, gr = torch.autograd.grad(s, (x, r), dy, retain_graph=True)
    assert torch.equal(gr, dy) and torch.equal(gx, enc.dropout(dy, 0.5, 3, 4))
    zero = torch.zeros_like(dy)
    both = torch.autograd.grad((y, s), (x, r), (dy, zero), retain_graph=True)
    for a, b in zip(torch.autograd.grad(y, (x, r), dy), both):
        assert torch.equal(a, b)


@pytest.mark.parametrize("call", CALLS)
def test_functional_gradients(call):
    x = _leaf(6, 64)
    want, = torch.autograd.grad(call(x).square().sum(), x)
    assert torch.equal(torch.func.grad(lambda t: call(t).square().sum())(x.detach()), want)


def test_no_graph_where_none_is_asked_for():
    x = _leaf(6, 64)
    with torch.no_grad():
        assert not any(call(x).requires_grad for call in CALLS)
    assert not any(call(x.detach()).requires_grad for call in CALLS)
    assert all(call(x).requires_grad for call in CALLS)
