"""GPU tests of differential attention on operands that are no ordinary numbers, at sizes of each of its forward kernels."""
import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# (batch, queries, keys, heads, key heads, d, dv): keys split over workgroups and waves, over the waves of one workgroup, tiles of many rows over
# split keys, and the kernels that pass over all keys
SIZES = [(2, 1, 3000, 4, 2, 64, 128), (2, 3, 600, 4, 2, 128, 256), (1, 4, 40, 2, 2, 32, 64), (1, 60, 700, 2, 1, 64, 128), (2, 40, 100, 4, 2, 64, 128),
         (1, 150, 130, 2, 2, 128, 256)]


def _operands(b, lq, lk, h, hk, d, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)        # noqa: E731
    return make(b, lq, h, 2, d), make(b, lk, hk, 2, d), make(b, lk, hk, dv), (0.2 + 0.6 * torch.rand(h, generator=g)).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_a_query_with_nan_is_nan_and_alone_in_it(sizes, dtype):
    q, k, v, lam = _operands(*sizes, dtype, seed=sum(sizes))
    plain = enc.diff_attention(q, k, v, lam)
    at = (sizes[0] - 1, sizes[1] // 2, 1)
    for maps in ((0,), (1,), (0, 1)):
        for bad in (slice(None), slice(3, 4)):          # the whole query, one element of it
            q2 = q.clone()
            for m in maps:
                q2[at + (m, bad)] = float("nan")
            out = enc.diff_attention(q2, k, v, lam)
            assert out[at].isnan().all(), (maps, bad)
            out[at] = plain[at]
            assert torch.equal(out, plain), (maps, bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_a_query_with_nan_that_sees_no_key_is_zeros(sizes, dtype):
    q, k, v, lam = _operands(*sizes, dtype, seed=sum(sizes))
    lengths = torch.full((sizes[0],), sizes[2], dtype=torch.int32, device=DEV)
    lengths[-1] = 0
    q[-1] = float("nan")
    out = enc.diff_attention(q, k, v, lam, lengths=lengths)
    assert torch.equal(out[-1], torch.zeros_like(out[-1])) and out[:-1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_a_key_with_nan_reaches_every_query_of_its_heads(sizes, dtype):
    q, k, v, lam = _operands(*sizes, dtype, seed=sum(sizes))
    plain = enc.diff_attention(q, k, v, lam)
    k[0, sizes[2] - 1, 0, 1] = float("nan")
    out, group = enc.diff_attention(q, k, v, lam), sizes[3] // sizes[4]
    assert out[0, :, :group].isnan().all()
    out[0, :, :group] = plain[0, :, :group]
    assert torch.equal(out, plain)
