"""GPU tests of the encoder modules: the layer against the same layer of torch's operations, its training, its cache."""
import copy

import pytest
import torch
import torch.nn.functional as F

import encoder_reference as ref
import mamtorch
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _layer(init=0, **kwargs):
    torch.manual_seed(init)
    return mamtorch.nn.MAMEncoderLayer(hidden=96, intermediate=160, heads=3, **kwargs).to(DEV)


def _by_parts(layer, x, seen=None, masks=None):
    """The layer with torch's norm and a softmax that is written out; its MAM layers are its own.  masks: of the two dropouts."""
    att = layer.attention
    y = F.layer_norm(x, (x.shape[-1],), layer.norm1.weight, layer.norm1.bias, layer.norm1.eps)
    b, n = x.shape[:2]
    q, k, v = (f(y).view(b, n, *s).transpose(1, 2) for f, s in ((att.query, (3, 2, 16)), (att.key, (att.kv_heads, 2, 16)), (att.value, (att.kv_heads, 32))))
    k, v = (t.repeat_interleave(att.heads // att.kv_heads, 1) for t in (k, v))
    scores = torch.stack([torch.matmul(q[..., m, :], k[..., m, :].transpose(-1, -2).contiguous()) for m in (0, 1)]) / 4.0
    if seen is not None:
        scores = scores.masked_fill(~seen[:, None], -float("inf"))
    p = torch.softmax(scores, -1)
    a = torch.matmul(p[0] - att.lambdas()[None, :, None, None] * p[1], v).transpose(1, 2)
    a = F.layer_norm(a, (32,), att.norm.weight, att.norm.bias, att.norm.eps) * (1 - att.lambda_init)
    a = att.output(a.reshape(b, n, 96))
    s = x + (a if masks is None else a * masks[0])
    y = F.layer_norm(s, (96,), layer.norm2.weight, layer.norm2.bias, layer.norm2.eps)
    h = layer.output(layer.act(layer.intermediate(y)))
    return s + (h if masks is None else h * masks[1])


def _close(got, want, what):
    # sums of up to 160 products of unit size in fp32, through two norms
    off = (got - want).abs().max() / want.abs().max()
    assert off < 2e-4, (what, off.item())


@pytest.mark.parametrize("causal, kv_heads", [(False, 3), (True, 1)])
def test_layer_and_gradients_against_its_parts(causal, kv_heads):
    layer = _layer(causal=causal, kv_heads=kv_heads)
    x = torch.randn(2, 37, 96, device=DEV, requires_grad=True)
    seen = ref.seen_keys(2, 37, 37, causal=True).to(DEV) if causal else None
    other, x2 = copy.deepcopy(layer), x.detach().clone().requires_grad_(True)
    y, want = layer(x), _by_parts(other, x2, seen)
    # a MAM layer's picks may differ where two products are equal to the last bits: compare outputs, and gradients as a whole
    _close(y, want, "layer")
    dy = torch.randn_like(y)
    y.backward(dy)
    want.backward(dy)
    # what the attention contributes, whose gradient passes no pick
    for name in ("attention.output.bias", "output.bias"):
        got, ref_grad = (dict(m.named_parameters())[name].grad for m in (layer, other))
        assert (got - ref_grad).norm() / ref_grad.norm() < 2e-2, name
    for name, p in layer.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), name


def test_training_draws_new_masks_and_takes_them_up_again():
    layer = _layer(p=0.25, seed=7).train()
    x = torch.randn(2, 9, 96, device=DEV)
    masks = [[ref.keep_mask((2, 9, 96), 0.25, 14 + n, call).to(DEV) / 0.75 for n in (0, 1)] for call in (0, 1)]
    first, second = layer(x), layer(x)
    _close(first, _by_parts(layer, x, masks=masks[0]), "first call")
    _close(second, _by_parts(layer, x, masks=masks[1]), "second call")
    state = layer.state_dict()
    third = layer(x)
    other = _layer(init=1, p=0.25).train()
    other.dropout1.seed, other.dropout2.seed = layer.dropout1.seed, layer.dropout2.seed
    other.load_state_dict(state)
    assert torch.equal(other(x), third)
    layer.eval()
    assert torch.equal(layer(x), layer(x))


@pytest.mark.parametrize("kv_heads", [3, 1])
def test_tokens_one_by_one_give_what_the_prompt_gives(kv_heads):
    layer = _layer(causal=True, kv_heads=kv_heads).eval()
    x = torch.randn(3, 20, 96, device=DEV)
    with torch.no_grad():
        want = layer(x)
        cache = layer.attention.cache(3, 24)
        cache.k.fill_(float("nan"))
        cache.v.fill_(float("nan"))
        parts = [layer(x[:, :13], cache=cache)] + [layer(x[:, i:i + 1], cache=cache) for i in range(13, 20)]
    _close(torch.cat(parts, 1), want, "tokens")
    assert cache.lengths.tolist() == [20] * 3
    with pytest.raises(ValueError, match="do not fit"):
        cache.append(cache.k[:, :5], cache.v[:, :5])
    with pytest.raises(ValueError, match="lengths of its own"):
        layer(x[:, :1], cache=cache, lengths=cache.lengths)


def test_padded_requests_do_not_see_their_padding():
    layer = _layer().eval()
    x = torch.randn(2, 30, 96, device=DEV)
    lengths = torch.tensor([30, 11], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        y = layer(x, lengths=lengths)
        _close(y[1, :11], layer(x[1:, :11])[0], "shorter request")
        _close(layer(x, key_mask=torch.arange(30, device=DEV) < lengths[:, None]), y, "as a mask")


def test_a_few_steps_of_training_learn():
    layer = _layer(p=0.1, seed=3).train()
    optimizer = torch.optim.Adam(layer.parameters(), 1e-3)
    x = torch.randn(4, 16, 96, device=DEV)
    target = torch.randn(4, 16, 96, device=DEV)
    losses = []
    for _ in range(30):
        optimizer.zero_grad()
        loss = F.mse_loss(layer(x), target)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert sum(losses[-5:]) < 0.8 * sum(losses[:5]), losses


def test_weight_dropout_by_counter_masks_weight_and_gradient():
    torch.manual_seed(0)
    layer = mt.nn.FullyConnected(50, 20, wdrop_rate=0.3, wdrop_seed=11).to(DEV).train()
    plain = mt.nn.FullyConnected(50, 20).to(DEV).train()
    x = torch.randn(8, 50, device=DEV)
    for call in range(2):
        keep = ref.keep_mask((20, 50), 0.3, 11, call).to(DEV)
        with torch.no_grad():
            plain.weight.copy_(torch.where(keep, layer.weight, torch.zeros_like(layer.weight)))
            plain.bias.copy_(layer.bias)
        layer.weight.grad = plain.weight.grad = None
        y, want = layer(x), plain(x)
        assert torch.equal(y, want)
        y.sum().backward()
        want.sum().backward()
        assert torch.equal(layer.weight.grad, torch.where(keep, plain.weight.grad, torch.zeros_like(plain.weight.grad)))
    layer.eval()
    assert layer(x).isfinite().all()


def test_modules_refuse_what_they_do_not_cover():
    with pytest.raises(ValueError):
        mt.nn.DiffAttention(100, 3)
    with pytest.raises(ValueError):
        mt.nn.DiffAttention(96, 3, kv_heads=2)
    with pytest.raises(ValueError):
        mt.nn.Dropout(1.5)
    norm = mt.nn.LayerNorm(12).to(DEV)
    x = torch.randn(5, 12, device=DEV)
    torch.testing.assert_close(norm(x), F.layer_norm(x, (12,)), rtol=1e-5, atol=1e-5)
    with pytest.raises(RuntimeError):
        norm(torch.randn(5, 13, device=DEV))
