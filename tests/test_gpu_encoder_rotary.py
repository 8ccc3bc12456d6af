"""GPU tests of norms of queries and keys with the position rotation: results and gradients against 64 bits, strides, places, refusals."""
import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt
import pages_reference as pref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _default(b, n):
    return torch.arange(n, dtype=torch.int32).expand(b, n)


def _check(q, k, wq, wk, f, pos, dtype, what, grads=True, **more):
    """Against 64 bits on what the CPU's tensors hold; the GPU's have their strides."""
    b, n = q.shape[:2]
    on = lambda t: None if t is None else t.to(DEV)                                     # noqa: E731
    leaves = [t if t is None else (t.to(DEV) if t.is_contiguous() else t).requires_grad_(grads) for t in (q, k, wq, wk)]
    y, z = enc.norm_rotate(*leaves, on(f), pos if pos is None or pos.is_cuda else pos.to(DEV), **more)
    places = _default(b, n) if pos is None else pos.cpu()
    more = {m: v for m, v in more.items() if m in ("eps", "norm", "interleaved")}
    dy, dz = _make(q.shape, dtype, 100), _make(k.shape, dtype, 101)
    got = []
    if grads:
        wanted = [t for t in leaves if t is not None and t.numel()]
        got = list(torch.autograd.grad([y, z], wanted, [dy.to(DEV), dz.to(DEV)], allow_unused=True))
    for name, x, w, out, g in (("q", q, wq, y, dy), ("k", k, wk, z, dz)):
        want = pref.Rotation(x.detach().cpu(), None if w is None else w.detach().cpu(), places, f, dy=g, **more)
        ref.assert_within(out, want.y, want.y_bound, "%s %s" % (what, name))
        if grads and x.numel():
            ref.assert_within(got[0 if name == "q" else len([t for t in (q,) if t.numel()])], want.dx, want.dx_bound, "%s d%s" % (what, name))
            if w is not None:
                at = len([t for t in (q, k) if t.numel()]) + (0 if name == "q" else int(wq is not None))
                ref.assert_within(got[at], want.dw, want.dw_bound, "%s d%s weight" % (what, name))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d, turned", [(64, 64), (128, 128), (80, 60), (33, 32), (96, 20), (7, 2), (1, 0), (2, 2), (127, 126), (40, 0)])
def test_sizes_of_heads(d, turned, interleaved, dtype):
    f = enc.rotary_frequencies(turned) if turned else None
    q, k = _make((2, 5, 4, 2, d), dtype, 1), _make((2, 5, 2, 2, d), dtype, 2, 3.0)
    wq, wk = (1 + _make((d,), torch.float32, n, 0.3) for n in (3, 4))
    _check(q, k, wq, wk, f, None, dtype, "d %d" % d, interleaved=interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, n, h, hk", [(1, 1, 1, 1), (1, 1, 16, 4), (3, 1, 6, 6), (1, 197, 6, 6), (5, 37, 8, 1), (1, 2100, 2, 1), (0, 4, 2, 2), (2, 0, 2, 2), (2, 3, 0, 2), (2, 3, 2, 0)])
def test_sizes_of_calls(b, n, h, hk, dtype):
    d = 64
    q, k = _make((b, n, h, 2, d), dtype, 5), _make((b, n, hk, 2, d), dtype, 6)
    wq, wk = ((1 + _make((d,), dtype, n, 0.3)) for n in (7, 8))
    if q.numel() and k.numel():
        _check(q, k, wq, wk, enc.rotary_frequencies(d), None, dtype, "%d x %d" % (b, n))
    else:
        _check(q, k, wq, wk, enc.rotary_frequencies(d), None, dtype, "%d x %d" % (b, n), grads=False)
        leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, wq, wk)]
        y, z = enc.norm_rotate(*leaves, enc.rotary_frequencies(d, device=DEV))
        for g, t in zip(torch.autograd.grad([y, z], leaves, [torch.ones_like(y), torch.ones_like(z)]), leaves):
            assert g.shape == t.shape and (t.numel() == 0 or torch.isfinite(g).all())
        grads = torch.autograd.grad(enc.norm_rotate(*leaves, enc.rotary_frequencies(d, device=DEV)), leaves, [torch.ones_like(y), torch.ones_like(z)])
        assert (q.numel() > 0) == bool(grads[2].any()) and (k.numel() > 0) == bool(grads[3].any())


@pytest.mark.parametrize("dtype", TYPES)
def test_a_workgroup_that_takes_tokens_again(dtype):
    # more tokens than the backward's workgroups hold in one turn
    q, k = _make((4, 4099, 2, 2, 32), dtype, 9), _make((4, 4099, 1, 2, 32), dtype, 10)
    wq, wk = ((1 + _make((32,), torch.float32, n, 0.3)) for n in (11, 12))
    _check(q, k, wq, wk, enc.rotary_frequencies(32), None, dtype, "many tokens")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("base", [10000.0, 1.0])
def test_places_far_out(base, dtype):
    # fp32 angles would be off by 2^-24 of a million radians and more
    places = torch.tensor([[0, 1, -1, 999999, 1000000, 2 ** 31 - 1, -2 ** 31, 500000]], dtype=torch.int32)
    q, k = _make((1, 8, 2, 2, 64), dtype, 13), _make((1, 8, 1, 2, 64), dtype, 14)
    _check(q, k, None, None, enc.rotary_frequencies(64, base), places, dtype, "far")


@pytest.mark.parametrize("dtype", TYPES)
def test_rotation_alone_and_norm_alone(dtype):
    q, k = _make((2, 9, 4, 2, 48), dtype, 15), _make((2, 9, 2, 2, 48), dtype, 16)
    w = 1 + _make((48,), torch.float32, 17, 0.3)
    _check(q, k, None, None, enc.rotary_frequencies(48), None, dtype, "rotation", norm=False)
    _check(q, k, w, w.clone(), None, None, dtype, "norm", eps=0.3)
    _check(q, k, w, None, enc.rotary_frequencies(24), None, dtype, "one weight")
    _check(q, k, None, None, None, None, dtype, "neither", norm=False)
    with torch.no_grad():
        y, z = enc.norm_rotate(q.to(DEV), k.to(DEV), norm=False)
    assert torch.equal(y.cpu(), q) and torch.equal(z.cpu(), k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_operands_and_places(offset, dtype):
    b, n, h, hk, d = 3, 11, 4, 2, 40
    wide = _make((b, n, (h + hk) * 2 * d + 7), dtype, 18).to(DEV)
    q = wide[..., offset:offset + h * 2 * d].unflatten(-1, (h, 2, d)).detach()
    k = wide[..., offset + h * 2 * d:offset + (h + hk) * 2 * d].unflatten(-1, (hk, 2, d)).detach()
    assert not q.is_contiguous() and not k.is_contiguous()
    wq, wk = (1 + _make((d,), torch.float32, n, 0.3) for n in (19, 20))
    places = torch.randint(0, 5000, (n, b), generator=torch.Generator().manual_seed(21), dtype=torch.int32).to(DEV).t()
    _check(q, k, wq, wk, enc.rotary_frequencies(d), places, dtype, "views")
    # heads before tokens, maps apart; one position for all tokens of a request
    q = _make((b, h, n, d, 2), dtype, 22).to(DEV).permute(0, 2, 1, 4, 3)
    k = _make((2, b, hk, n, d), dtype, 23).to(DEV).permute(1, 3, 2, 0, 4)
    _check(q.detach(), k.detach(), wq, wk, enc.rotary_frequencies(d), torch.tensor([[5], [70000], [9]], dtype=torch.int32).to(DEV).expand(b, n), dtype, "permuted")


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_operands_and_gradients_of_sums(dtype):
    b, n, h, hk, d = 2, 6, 4, 2, 64
    q, k = _make((1, 1, h, 2, d), dtype, 24), _make((b, n, 1, 2, d), dtype, 25)
    f = enc.rotary_frequencies(d)
    qw, kw = q.to(DEV).expand(b, n, h, 2, d).detach(), k.to(DEV).expand(b, n, hk, 2, d).detach()
    assert 0 in qw.stride() and 0 in kw.stride()
    _check(qw, kw, None, None, f, None, dtype, "broadcast")
    leaf = _make((b, n, h, 2, d), dtype, 26)
    x = leaf.to(DEV).requires_grad_(True)
    y, _ = enc.norm_rotate(x, kw.detach(), None, None, f.to(DEV))
    g = _make((b, h, 2, d), dtype, 27)
    dx, = torch.autograd.grad(y.sum(1), x, g.to(DEV))
    want = pref.Rotation(leaf, None, _default(b, n), f, dy=g[:, None].expand(b, n, h, 2, d))
    ref.assert_within(dx, want.dx, want.dx_bound, "gradient of a sum")


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_output_alone_is_differentiated(which):
    d, f = 64, enc.rotary_frequencies(64)
    q, k = _make((2, 5, 4, 2, d), torch.float32, 28), _make((2, 5, 2, 2, d), torch.float32, 29)
    w = 1 + _make((d,), torch.float32, 30, 0.3)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, w, w.clone())]
    outs = enc.norm_rotate(*leaves, f.to(DEV))
    at = "qk".index(which)
    x = (q, k)[at]
    dy = _make(x.shape, torch.float32, 31)
    grads = torch.autograd.grad(outs[at], leaves, dy.to(DEV), allow_unused=True)
    want = pref.Rotation(x, w, _default(2, 5), f, dy=dy)
    ref.assert_within(grads[at], want.dx, want.dx_bound, "dx")
    ref.assert_within(grads[2 + at], want.dw, want.dw_bound, "dw")
    assert grads[1 - at] is None and grads[3 - at] is None


def test_gradients_against_differences():
    # in fp32: a central difference of step e errs by 2^-24 |loss| / e and e^2 times the third derivative
    q, k = _make((1, 3, 2, 2, 8), torch.float32, 32), _make((1, 3, 1, 2, 8), torch.float32, 33)
    w, f = 1 + _make((8,), torch.float32, 34, 0.3), enc.rotary_frequencies(8, 10.0).to(DEV)
    dy, dz = (_make(t.shape, torch.float32, n).to(DEV).double() for n, t in ((35, q), (36, k)))
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, w, w.clone())]

    def loss(*at):
        y, z = enc.norm_rotate(*at, f)
        return (y.double() * dy).sum() + (z.double() * dz).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    e = 2.0 ** -8
    for n, (t, g) in enumerate(zip(leaves, grads)):
        for i in range(0, t.numel(), 5):
            step = torch.zeros(t.numel(), device=DEV)
            step[i] = e
            sides = [loss(*[(u + s * step.view(t.shape)).detach() if m == n else u.detach() for m, u in enumerate(leaves)]) for s in (1, -1)]
            assert abs(float((sides[0] - sides[1]) / (2 * e)) - float(g.reshape(-1)[i])) <= 2e-3 * (1 + abs(float(g.reshape(-1)[i])))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_infinities_and_nan(dtype):
    q = _make((1, 4, 1, 2, 64), dtype, 37)
    q[0, 0] = 0
    q[0, 1, 0, 0, 5] = float("inf")
    q[0, 2, 0, 1, 3] = float("nan")
    y, _ = enc.norm_rotate(q.to(DEV), q.to(DEV), None, None, enc.rotary_frequencies(64, device=DEV))
    y = y.cpu()
    assert not y[0, 0].any()                                    # 0 / sqrt(eps)
    assert torch.isnan(y[0, 1, 0, 0]).any() and torch.isfinite(y[0, 1, 0, 1]).all()      # inf / inf in its own row alone
    assert torch.isnan(y[0, 2, 0, 1]).all() and torch.isfinite(y[0, 2, 0, 0]).all()
    assert torch.isfinite(y[0, 3]).all()


def test_same_bits_on_every_call():
    q, k = _make((4, 300, 4, 2, 64), torch.bfloat16, 38).to(DEV), _make((4, 300, 2, 2, 64), torch.bfloat16, 39).to(DEV)
    w, f = (1 + _make((64,), torch.float32, 40, 0.3)).to(DEV), enc.rotary_frequencies(64, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, w, w.detach().clone())]
    runs = []
    for _ in range(3):
        outs = enc.norm_rotate(*leaves, f)
        runs.append([*outs, *torch.autograd.grad(outs, leaves, [o.detach() for o in outs])])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_captured_and_replayed_with_its_gradients():
    q, k = _make((2, 50, 4, 2, 64), torch.float32, 41).to(DEV), _make((2, 50, 2, 2, 64), torch.float32, 42).to(DEV)
    w, f = (1 + _make((64,), torch.float32, 43, 0.3)).to(DEV), enc.rotary_frequencies(64, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, w, w.detach().clone())]
    g = [_make(t.shape, torch.float32, 44).to(DEV) for t in (q, k)]

    def step():
        outs = enc.norm_rotate(*leaves, f)
        return [*[o.detach() for o in outs], *torch.autograd.grad(outs, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(4):
        with torch.no_grad():
            for t in leaves:
                t.add_(0.01 * n)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), n


def test_second_derivatives_and_tangents_are_errors():
    q = _make((1, 3, 2, 2, 16), torch.float32, 45).to(DEV).requires_grad_(True)
    k = _make((1, 3, 2, 2, 16), torch.float32, 46).to(DEV)
    y, _ = enc.norm_rotate(q, k, None, None, enc.rotary_frequencies(16, device=DEV))
    dq, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        dq.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.detach(), torch.ones_like(q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            enc.norm_rotate(dual, k)
    y, _ = enc.norm_rotate(q, k)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()


def test_refusals():
    make = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=DEV)     # noqa: E731
    q, k, w, f = make(2, 3, 4, 2, 16), make(2, 3, 2, 2, 16), make(16), enc.rotary_frequencies(16, device=DEV)
    for bad, text in (
            (dict(k=make(2, 4, 2, 2, 16)), "do not match"), (dict(k=make(2, 3, 2, 2, 8)), "do not match"), (dict(k=make(2, 3, 2, 16)), "must be"),
            (dict(k=k.half()), "must have q's type"), (dict(k=k.cpu()), "different device"), (dict(q=make(2, 3, 4, 2, 129), k=make(2, 3, 2, 2, 129)), "1 to 128"),
            (dict(q=q.double(), k=k.double()), "must be float32"), (dict(q_weight=make(8)), "contiguous vector"), (dict(q_weight=w.half()), "of q's type"),
            (dict(q_weight=w, norm=False), "with a norm"), (dict(q_weight=make(32)[::2]), "contiguous vector"), (dict(frequencies=f.float()), "float64"),
            (dict(frequencies=enc.rotary_frequencies(18, device=DEV)), "pairs"), (dict(frequencies=f.cpu()), "different device"),
            (dict(positions=make(2, 3, t=torch.long)), "int32"), (dict(positions=make(3, 2, t=torch.int32)), "int32"), (dict(eps=-1.0), "eps"),
            (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(frequencies=f.clone().requires_grad_(True)), "frequencies")):
        with pytest.raises(RuntimeError, match=text):
            enc.norm_rotate(**{**dict(q=q, k=k), **bad})
    with pytest.raises(RuntimeError, match="one type"):
        enc.norm_rotate(q.half(), k.half(), w.half(), w)
    with pytest.raises(ValueError, match="pairs"):
        enc.rotary_frequencies(7)
    with pytest.raises((RuntimeError, NotImplementedError)):
        enc.norm_rotate(q.cpu(), k.cpu())
