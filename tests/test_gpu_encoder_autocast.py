"""GPU tests of the encoder layer under autocast: the attention in 16 bits, the residual stream and the MAM layers in float32."""
import pytest
import torch

import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder


def _layer(**kwargs):
    torch.manual_seed(0)
    return mt.nn.MAMEncoderLayer(hidden=96, intermediate=160, heads=3, **kwargs).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_layer_under_autocast_is_its_parts(dtype):
    layer = _layer(p=0.25, seed=3).train()
    x = torch.randn(2, 37, 96, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype):
        y = layer(x)
        a = layer.attention(layer.norm1(x))
    assert a.dtype == dtype and y.dtype == torch.float32
    norm = layer.norm2
    h, s = enc.add_dropout_layer_norm(a.float(), x, norm.weight, norm.bias, 0.25, 6, 0, norm.eps)
    want = enc.dropout(layer.output(layer.act(layer.intermediate(h))), 0.25, 7, 0, s)
    assert torch.equal(y, want)
    y.square().mean().backward()
    assert x.grad.isfinite().all()
    for name, p in layer.named_parameters():
        assert p.grad.dtype == torch.float32 and p.grad.isfinite().all() and p.grad.any(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens_over_a_cache_under_autocast(dtype):
    attention = _layer(causal=True).attention.eval()
    x = torch.randn(2, 12, 96, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype):
        want = attention(x)
        cache = attention.cache(2, 12)
        parts = [attention(x[:, :7], cache=cache)] + [attention(x[:, i:i + 1], cache=cache) for i in range(7, 12)]
    assert cache.k.dtype == dtype
    # the projections' and the result's roundings to the type, each of a sum of at most 96 terms, through the head's norm
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    assert (torch.cat(parts, 1).float() - want.float()).abs().max() <= 16 * unit * want.float().abs().max()
