"""GPU tests of the encoder layer with norms, rotation and paged caches as a server and a training loop use them: what requests get in pages against one pass over their
whole sequences, drafts and forks among them, and gradients of every parameter through the rotation."""
import copy

import pytest
import torch

import mamtorch_amd as mt
import pages_reference as pref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _layers(count=2, init=0, kv_heads=3, **more):
    torch.manual_seed(init)
    more = {"causal": True, "qk_norm": True, "rotary": 12, **more}
    layers = torch.nn.ModuleList(mt.nn.MAMEncoderLayer(96, 128, 3, kv_heads=kv_heads, depth=n + 1, **more) for n in range(count))
    for layer in layers:
        if more["qk_norm"]:
            with torch.no_grad():
                layer.attention.query_norm.add_(0.3 * torch.randn(16))
                layer.attention.key_norm.add_(0.3 * torch.randn(16))
    return layers.to(DEV).eval()


def _run(layers, x, caches=None):
    for n, layer in enumerate(layers):
        x = layer(x, cache=None if caches is None else caches[n])
    return x


def _close(got, want, what):
    # fp32 throughout: sums of up to 128 terms in another order, through two layers whose norms keep errors at the size of their inputs: some hundred units of 2^-24
    assert got.shape == want.shape, what
    if not got.numel():
        return
    off = (got - want).abs().max() / want.abs().max()
    assert off <= 2e-5, (what, float(off))


def _table(layers, batch, pages, page=16, most=None):
    table = mt.nn.PageTable(batch, pages, page, most, device=DEV)
    caches = [layer.attention.pages(table) for layer in layers]
    for c in caches:                    # what nobody has put there is not used
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    return table, caches


@pytest.mark.parametrize("kv_heads", [3, 1])
@pytest.mark.parametrize("more", [{}, {"qk_norm": False}, {"rotary": 0}, {"qk_norm": False, "rotary": 0}])
@torch.no_grad()
def test_requests_of_different_lengths_in_pages(kv_heads, more):
    layers = _layers(kv_heads=kv_heads, **more)
    x = torch.randn(3, 60, 96, device=DEV)
    want = _run(layers, x)
    table, caches = _table(layers, 3, 16)
    # prompts of different lengths in one padded batch, then tokens, some of them for some requests
    prompts = torch.tensor([13, 1, 37], dtype=torch.int32, device=DEV)
    assert torch.equal(table.begin(prompts), prompts)
    y = _run(layers, x[:, :37], caches)
    for b, n in enumerate(prompts.tolist()):
        _close(y[b, :n], want[b, :n], "prompt %d" % b)
    table.accept()
    lengths = prompts.tolist()
    for step in range(8):
        counts = [1, 2, int(step % 2)]
        n = max(counts)
        new = torch.stack([x[b, length:length + n] for b, length in enumerate(lengths)])
        table.begin(torch.tensor(counts, dtype=torch.int32, device=DEV))
        y = _run(layers, new, caches)
        for b, (length, count) in enumerate(zip(lengths, counts)):
            _close(y[b, :count], want[b, length:length + count], "step %d, request %d" % (step, b))
        table.accept()
        lengths = [length + count for length, count in zip(lengths, counts)]
    assert table.lengths.tolist() == lengths
    table.trim(0)
    assert not table.refs.any() and (table.table == -1).all()


@torch.no_grad()
def test_drafted_trees_and_what_is_taken_over():
    layers = _layers()
    b, n = 3, 6
    x = torch.randn(b, 40, 96, device=DEV)
    table, caches = _table(layers, b, 24)
    lengths = torch.tensor([20, 15, 3], dtype=torch.int32, device=DEV)
    table.begin(lengths)
    _run(layers, x[:, :20], caches)
    table.accept()
    sequences = [x[i, :length] for i, length in enumerate(lengths.tolist())]
    parents = [[-1, 0, 0, 1, 2, 2], [-1, -1, 1, 2, 3, 4], [-1, 0, 1, 2, 1, 0]]
    paths, accepted = [[0, 2, 5], [1, 2, 2], [0, 1, 4]], [3, 2, 3]
    for step in range(4):
        drafts = torch.randn(b, n, 96, device=DEV)
        table.begin(parents=torch.tensor(parents, dtype=torch.int32, device=DEV))
        y = _run(layers, drafts, caches)
        for i in range(b):
            seen = pref.tree(parents[i])
            for t in range(n):
                line = [u for u in range(n) if seen[t, u]]
                whole = _run(layers, torch.cat((sequences[i], drafts[i, line]))[None])
                _close(y[i, t], whole[0, -1], "step %d, request %d, token %d" % (step, i, t))
        table.accept(torch.tensor(paths, dtype=torch.int32, device=DEV), torch.tensor(accepted, dtype=torch.int32, device=DEV))
        sequences = [torch.cat((s, d[p[:a]])) for s, d, p, a in zip(sequences, drafts, paths, accepted)]
    assert table.lengths.tolist() == [len(s) for s in sequences]


@torch.no_grad()
def test_forked_requests_go_their_own_ways():
    layers = _layers()
    x = torch.randn(4, 30, 96, device=DEV)
    table, caches = _table(layers, 4, 16)
    table.begin(torch.tensor([21, 0, 0, 0], dtype=torch.int32, device=DEV))
    _run(layers, x[:, :21], caches)
    table.accept()
    table.fork(torch.tensor([0, 0, 0, 0], dtype=torch.int32, device=DEV))
    assert int((table.refs > 0).sum()) == 2             # one prompt's pages
    sequences = [x[0, :21]] * 4
    for step in range(20):
        new = torch.randn(4, 1, 96, device=DEV)
        table.begin(1)
        y = _run(layers, new, caches)
        sequences = [torch.cat((s, t)) for s, t in zip(sequences, new)]
        for i in range(4):
            _close(y[i, 0], _run(layers, sequences[i][None])[0, -1], "step %d, beam %d" % (step, i))
        table.accept()
        if step % 3 == 1:
            sources = [(step + i * i) % 4 for i in range(4)]
            table.fork(torch.tensor(sources, dtype=torch.int32, device=DEV))
            sequences = [sequences[s] for s in sources]


@torch.no_grad()
def test_requests_without_room_are_told_and_harm_nobody():
    layers = _layers(1)
    x = torch.randn(2, 40, 96, device=DEV)
    table, caches = _table(layers, 2, 3, most=64)
    assert table.begin(20).tolist() == [20, 0]
    y = _run(layers, x[:, :20], caches)
    assert torch.isfinite(y).all()
    _close(y[0], _run(layers, x[:1, :20])[0], "the one with room")
    table.accept()
    assert table.lengths.tolist() == [20, 0]
    assert table.begin(torch.tensor([1, 10], dtype=torch.int32, device=DEV)).tolist() == [1, 10]
    table.accept(counts=5)                                              # no more than there was room for
    assert table.lengths.tolist() == [21, 5]


@torch.no_grad()
def test_a_captured_step_serves_as_an_eager_one():
    layers = _layers()
    new = torch.randn(3, 1, 96, device=DEV)
    sources = torch.tensor([2, 1, 2], dtype=torch.int32, device=DEV)

    def start():
        table, caches = _table(layers, 3, 30)
        for c in caches:
            c.k.fill_(0.5)
            c.v.fill_(0.5)
        table.begin(torch.tensor([5, 18, 31], dtype=torch.int32, device=DEV))
        table.accept()
        return table, caches

    def step(table, caches):
        table.begin(1)
        y = _run(layers, new, caches)
        table.accept()
        return y

    eager = start()
    step(*start())                                                      # lazily set up before the capture
    torch.cuda.synchronize()
    captured = start()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*captured)
    for turn in range(40):
        if turn % 7 == 3:                                               # forks between the replays: the graph copies the pages
            for table, _ in (eager, captured):
                table.fork(sources)
        new.normal_()
        want = step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn
        assert torch.equal(eager[0].table, captured[0].table) and torch.equal(eager[0].lengths, captured[0].lengths)


@torch.no_grad()
def test_rotated_tokens_over_the_dense_cache():
    layers = _layers()
    x = torch.randn(2, 20, 96, device=DEV)
    want = _run(layers, x)
    caches = [layer.attention.cache(2, 20) for layer in layers]
    parts = [_run(layers, x[:, :7], caches)] + [_run(layers, x[:, i:i + 1], caches) for i in range(7, 20)]
    _close(torch.cat(parts, 1), want, "dense cache")


@torch.no_grad()
def test_under_autocast_pages_are_16_bits():
    layers = _layers(1)
    x = torch.randn(2, 30, 96, device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        want = _run(layers, x)
        table, caches = _table(layers, 2, 16)
        assert caches[0].k.dtype == torch.bfloat16
        table.begin(29)
        first = _run(layers, x[:, :29], caches)
        table.accept()
        table.begin(1)
        y = torch.cat((first, _run(layers, x[:, 29:], caches)), 1)
    # queries, keys, probabilities, results rounded to 8 bits on both ways, in another order: some units of 2^-8 of the largest value
    assert (y - want).abs().max() <= 8 * 2.0 ** -8 * want.abs().max()


def test_gradients_of_every_parameter_against_64_bits():
    # the module's attention by its formulas in 64 bits, norms and rotation among them
    torch.manual_seed(3)
    attention = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=10).to(DEV)
    with torch.no_grad():
        for p in (attention.query_norm, attention.key_norm):
            p.add_(0.3 * torch.randn_like(p))
    x = torch.randn(2, 11, 96, device=DEV, requires_grad=True)
    dy = torch.randn(2, 11, 96, device=DEV)
    grads = torch.autograd.grad(attention(x), [x, *attention.parameters()], dy)

    wide = copy.deepcopy(attention).double()
    z = x.detach().double().requires_grad_(True)
    b, n, h, d = 2, 11, 3, 16
    places = torch.arange(n, device=DEV).expand(b, n)

    def heads(linear, weight):
        t = linear(z).view(b, n, h, 2, d)
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * weight
        angle = places.double()[..., None, None, None] * wide.frequencies
        pairs = torch.complex(t[..., :5], t[..., 5:10]) * torch.polar(torch.ones_like(angle), angle)
        return torch.cat((pairs.real, pairs.imag, t[..., 10:]), -1).permute(3, 0, 2, 1, 4)

    q, k = heads(wide.query, wide.query_norm), heads(wide.key, wide.key_norm)
    v = wide.value(z).view(b, n, h, 2 * d).permute(0, 2, 1, 3)
    hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
    p = torch.softmax((q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(hidden, -float("inf")), -1)
    q1, k1, q2, k2 = wide.lambda_vectors
    lam = torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + wide.lambda_init
    out = ((p[0] - lam[:, None, None] * p[1]) @ v).transpose(1, 2)
    out = torch.nn.functional.layer_norm(out, (2 * d,), wide.norm.weight, wide.norm.bias, wide.norm.eps) * (1 - wide.lambda_init)
    want = torch.autograd.grad(wide.output(out.reshape(b, n, 96)), [z, *wide.parameters()], dy.double())
    names = ["x"] + [name for name, _ in attention.named_parameters()]
    for name, got, ref in zip(names, grads, want):
        # sums of up to 96 terms in fp32, four products deep: some hundred units of 2^-24 of the largest value (the key's bias has no gradient but what norms and turns leave)
        assert (got - ref).abs().max() <= 5e-5 * max(float(ref.abs().max()), 1e-3), (name, float((got - ref).abs().max()), float(ref.abs().max()))


def test_modules_move_copy_and_load():
    layer = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=True)
    assert layer.frequencies.device.type == "cpu"
    layer.to(DEV)
    assert layer.frequencies.device.type == "cuda" and layer.frequencies.dtype == torch.float64
    other = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=True).to(DEV)
    other.load_state_dict(layer.state_dict())
    x = torch.randn(2, 5, 96, device=DEV)
    assert torch.equal(other(x), layer(x)) and torch.equal(copy.deepcopy(layer)(x), layer(x))
    half = copy.deepcopy(layer).half()
    assert half(x.half()).dtype == torch.float16 and half.frequencies.dtype == torch.float64
    plain = mt.nn.DiffAttention(96, 3, causal=True).to(DEV)
    for name in ("qk_norm", "rotary", "base", "frequencies", "qk_eps"):         # a module that was saved whole before it had these
        plain.__dict__.pop(name, None)
    assert torch.isfinite(plain(x)).all()
