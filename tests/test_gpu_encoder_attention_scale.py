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
