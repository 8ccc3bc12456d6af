"""GPU tests of differential attention where a 16-bit type's range is what could fail: weights of the second map far above 1, gradients far from 1."""
import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder


def _flat_and_peaked(queries, heads, keys, lam, dtype):
    """A first map that is flat over all keys and a second one that is all but 1 at the first key; the same for every query and head."""
    g = torch.Generator().manual_seed(keys)
    q, k = torch.zeros(1, 1, 1, 2, 8, dtype=dtype), torch.zeros(1, keys, 1, 2, 8, dtype=dtype)
    q[..., 1, 0] = 4.0
    k[:, 0, :, 1, 0] = 5.0
    v, dout = torch.randn(1, keys, 1, 8, generator=g).to(dtype), torch.randn(1, 1, 1, 8, generator=g).to(dtype)
    want = ref.Attention(q, k, v, torch.full((1,), lam, dtype=dtype), torch.ones(1, 1, keys, dtype=torch.bool), 1.0)
    wide = lambda t, n: t.expand(-1, n, heads, *t.shape[3:]).contiguous().to(DEV)        # noqa: E731
    return (wide(q, queries), wide(k, keys), wide(v, keys), torch.full((heads,), lam, dtype=dtype, device=DEV)), wide(dout, queries), want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lam", [20.0, -20.0, 1000.0, 20000.0])
# 640 tiles of 16 queries, more than are split over the keys; and a few queries that are
@pytest.mark.parametrize("queries, heads", [(256, 40), (3, 2)])
def test_a_large_weight_of_the_second_map(queries, heads, lam, dtype):
    gpu, _, want = _flat_and_peaked(queries, heads, 8192, lam, dtype)
    out = enc.diff_attention(*gpu, scale=1.0)
    ref.assert_within(out, want.out.expand(1, queries, heads, 8), want.out_bound.expand(1, queries, heads, 8), "out")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lam", [20.0, -20.0, 1000.0, 20000.0])
def test_a_large_weight_of_the_second_map_in_training(lam, dtype):
    gpu, dout, want = _flat_and_peaked(20, 2, 8192, lam, dtype)
    gpu[0].requires_grad_(True)
    out = enc.diff_attention(*gpu, scale=1.0)
    ref.assert_within(out, want.out.expand(1, 20, 2, 8), want.out_bound.expand(1, 20, 2, 8), "out")
    # the first map's score gradients sum to nothing over equal keys, the second's weigh the one key against the rest: finite, and 0 in what q does not reach
    dq, = torch.autograd.grad(out, gpu[0], dout)
    assert dq.isfinite().all() and torch.equal(dq[..., 1:], torch.zeros_like(dq[..., 1:]))


def _check_scaled_gradients(operands, up, scale, bounds):
    """Gradients are linear in dout: those of 2^up dout0 are those of dout0 times 2^up, with what a rounding of the result to its type costs there."""
    q, k, v, lam, dout = operands
    dtype, dout0 = q.dtype, (dout.double() * 2.0 ** -up).to(q.dtype)
    assert torch.equal(dout0.double() * 2.0 ** up, dout.double()) and dout.isfinite().all()
    want = ref.Attention(q, k, v, lam, torch.ones(q.shape[0], q.shape[1], k.shape[1], dtype=torch.bool), scale, dout0)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
    grads = torch.autograd.grad(enc.diff_attention(*leaves, scale=scale), leaves, dout.to(DEV))
    for name, got in zip(("dq", "dk", "dv", "dlam"), grads):
        if name in bounds:
            exact = getattr(want, name) * 2.0 ** up
            bound = (getattr(want, name + "_bound") - ref.TINY[got.dtype] + bounds[name]) * 2.0 ** up + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
            assert name == "dlam" or (exact.abs() < 60000).all()       # fp16 holds them
            assert dtype != torch.float16 or name == "dlam" or bound.median() < exact.abs().median()     # and the bound says something
            ref.assert_within(got, exact, bound, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wide", [-5, 5])
def test_gradients_of_small_incoming_gradients(wide, dtype):
    # 2000 keys and a dout of 2^-15: gradients of scores of 1e-7.  With wide queries (keys) dk (dq) is well above its type's smallest numbers.
    g = torch.Generator().manual_seed(41)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)        # noqa: E731
    q, k, v = make(1, 500, 2, 2, 64) * 2.0 ** wide, make(1, 2000, 1, 2, 64) * 2.0 ** -wide, make(1, 2000, 1, 128)
    lam, dout = torch.tensor([0.3, 0.7]), (make(1, 500, 2, 128).double() * 2.0 ** -15).to(dtype)
    # In fp16 a score's gradient is off by half the spacing of subnormal numbers, 2^-25, where dout's rows (sums of 2^6 to 2^8) are brought to 2^3: 2^-21 in
    # units of dout0, for every term of dq (over the keys) and dk (over both heads' queries).
    tiny = 0.125 * (2.0 ** -21 if dtype == torch.float16 else 0.0)
    bounds = {"dq": tiny * k.double().abs().sum((1, 2))[:, None, None]} if wide < 0 else {"dk": tiny * q.double().abs().sum((1, 2))[:, None, None]}
    _check_scaled_gradients((q, k, v, lam, dout), -15, 0.125, bounds)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_of_large_incoming_gradients(dtype):
    # a dout of 2^13 and values of 4: gradients of scores past 65504, gradients of q, k and v well within it
    g = torch.Generator().manual_seed(42)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)        # noqa: E731
    q, k, v, dout = make(1, 40, 2, 2, 64), make(1, 8, 1, 2, 64), 4 * make(1, 8, 1, 128), 2.0 ** 13 * make(1, 40, 2, 128).clamp(-4, 4)
    _check_scaled_gradients((q, k, v, torch.tensor([0.3, 0.7]), dout), 13, 2.0 ** -6, {"dq": 0.0, "dk": 0.0, "dv": 0.0, "dlam": 0.0})
