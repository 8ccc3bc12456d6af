"""GPU tests of gradients through the encoder modules: every parameter's and x's, against the same module of elementary operations in 64 bits."""
import copy

import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN, HEADS = 96, 3


def _norm(x, module):
    centred = x - x.mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred ** 2).mean(-1, keepdim=True) + module.eps) * module.weight
    return y if module.bias is None else y + module.bias


def _attention(module, x, seen):
    b, n = x.shape[:2]
    group = module.heads // module.kv_heads
    rows = lambda f, h, *s: (x @ f.weight.T + f.bias).view(b, n, h, *s).transpose(1, 2).repeat_interleave(module.heads // h, 1)  # noqa: E731
    q, k = rows(module.query, module.heads, 2, module.head_size), rows(module.key, module.kv_heads, 2, module.head_size)
    v = rows(module.value, module.kv_heads, module.value_size)
    assert k.shape[1] == module.kv_heads * group
    scores = torch.einsum("bhimd,bhjmd->mbhij", q, k) * module.head_size ** -0.5
    p = torch.softmax(scores.masked_fill(~seen[:, None], -float("inf")), -1)
    q1, k1, q2, k2 = module.lambda_vectors
    lam = torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + module.lambda_init
    out = torch.matmul(p[0] - lam[:, None, None] * p[1], v).transpose(1, 2)
    out = _norm(out, module.norm) * (1 - module.lambda_init)
    return out.reshape(b, n, module.hidden) @ module.output.weight.T + module.output.bias


def _compare(got, want, names):
    # Sums of at most 96 products or 148 rows in fp32 and a chain of two norms, a softmax and three products before and after them: each step errs by
    # at most a few hundred units of 2^-24 of its largest term, 2^-24 * 200 * 10 steps = 1.2e-4, and a gradient is compared with its own largest element.
    # That of a key's bias is 0 (a constant added to a row's scores changes nothing): its terms are those of the key's weight without x.
    sizes = {name: b.abs().max() for name, b in zip(names, want)}
    for name, a, b in zip(names, got, want):
        off = (a.double().cpu() - b).abs().max() / sizes[name.replace("key.bias", "key.weight")]
        assert off < 1.2e-4, (name, off.item())


def _leaves(module, x):
    names, params = zip(*[(n, p) for n, p in module.named_parameters()])
    return ["y", "x", *names], [x, *params]


@pytest.mark.parametrize("causal, kv_heads, depth", [(False, 3, 1), (True, 1, 4), (True, 3, 12)])
def test_attention_module(causal, kv_heads, depth):
    torch.manual_seed(depth)
    module = mt.nn.DiffAttention(HIDDEN, HEADS, kv_heads, depth, causal)
    for p in (module.norm.weight, module.norm.bias):        # away from ones and zeros
        torch.nn.init.normal_(p)
    wide, x, dy = copy.deepcopy(module).double(), torch.randn(4, 37, HIDDEN), torch.randn(4, 37, HIDDEN)
    module = module.to(DEV)
    names, leaves = _leaves(module, x.to(DEV).requires_grad_(True))
    y = module(leaves[0])
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy.to(DEV))]
    _, leaves = _leaves(wide, x.double().requires_grad_(True))
    y = _attention(wide, leaves[0], ref.seen_keys(4, 37, 37, causal=causal))
    _compare(got, [y.detach(), *torch.autograd.grad(y, leaves, dy.double())], names)


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_attention_half_of_a_layer(p):
    torch.manual_seed(1)
    layer = mt.nn.MAMEncoderLayer(HIDDEN, 40, HEADS, p=p, seed=9)
    wide, x, dy, ds = copy.deepcopy(layer).double(), *(torch.randn(4, 37, HIDDEN) for _ in range(3))
    lengths = torch.tensor([37, 20, 1, 30], dtype=torch.int32)
    layer = layer.to(DEV)
    parts = lambda m: [m.norm1.weight, m.norm1.bias, m.norm2.weight, m.norm2.bias, *m.attention.parameters()]       # noqa: E731
    x1 = x.to(DEV).requires_grad_(True)
    a = layer.attention(layer.norm1(x1), lengths.to(DEV))
    norm = layer.norm2
    y, s = mt.kernel.encoder.add_dropout_layer_norm(a, x1, norm.weight, norm.bias, p, layer.dropout1.seed or 0, 5, norm.eps)
    got = [y.detach(), s.detach(), *torch.autograd.grad((y, s), [x1, *parts(layer)], (dy.to(DEV), ds.to(DEV)))]
    x2 = x.double().requires_grad_(True)
    seen = ref.seen_keys(4, 37, 37, lengths=lengths)
    keep = ref.keep_mask(x.shape, p, 18, 5).double() / (1 - p)
    s = x2 + _attention(wide.attention, _norm(x2, wide.norm1), seen) * keep
    y = _norm(s, wide.norm2)
    want = [y.detach(), s.detach(), *torch.autograd.grad((y, s), [x2, *parts(wide)], (dy.double(), ds.double()))]
    _compare(got, want, ["y", "s", "x", "norm1.weight", "norm1.bias", "norm2.weight", "norm2.bias", *dict(wide.attention.named_parameters())])
