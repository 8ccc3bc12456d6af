"""GPU tests of differential attention and its gradients against the definition in 64 bits."""
import ctypes

import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _operands(b, lq, lk, h, hk, d, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)        # noqa: E731
    return make(b, lq, h, 2, d), make(b, lk, hk, 2, d), make(b, lk, hk, dv), (0.2 + 0.6 * torch.rand(h, generator=g)).to(dtype), make(b, lq, h, dv)


def _check(q, k, v, lam, dout, gpu=None, scale=None, backward=True, **limits):
    seen = ref.seen_keys(q.shape[0], q.shape[1], k.shape[1], **limits)
    want = ref.Attention(q, k, v, lam, seen, scale, dout if backward else None)
    on_gpu = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in limits.items()}
    if gpu is None:
        gpu = [t.to(DEV) for t in (q, k, v, lam)]
    out = enc.diff_attention(*gpu, scale=scale, **on_gpu)           # what serving calls
    assert out.dtype == q.dtype
    ref.assert_within(out, want.out, want.out_bound, "out")
    if not backward:
        return
    leaves = [t.detach().requires_grad_(True) for t in gpu]
    out = enc.diff_attention(*leaves, scale=scale, **on_gpu)
    ref.assert_within(out, want.out, want.out_bound, "out of the training forward")
    dq, dk, dv, dlam = torch.autograd.grad(out, leaves, dout.to(DEV))
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv), ("dlam", dlam)):
        ref.assert_within(got, getattr(want, name), getattr(want, name + "_bound"), name)


SIZES = [(1, 1, 1, 1, 1, 1, 1), (2, 1, 7, 3, 3, 5, 9), (1, 5, 33, 2, 1, 32, 64), (2, 33, 31, 4, 2, 16, 24), (1, 128, 128, 2, 2, 64, 128),
         (3, 197, 197, 3, 3, 64, 128), (2, 65, 130, 6, 2, 48, 64), (1, 70, 257, 4, 1, 80, 160), (2, 130, 67, 2, 2, 128, 256), (1, 40, 100, 3, 1, 128, 96),
         (1, 300, 301, 2, 1, 63, 127), (1, 17, 64, 8, 1, 128, 33)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_all_keys(sizes, dtype):
    _check(*_operands(*sizes, dtype, seed=sum(sizes)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_causal_and_lengths(sizes, dtype):
    b, lq, lk = sizes[:3]
    lengths = torch.tensor([lk - i * (lk // 2) // max(1, b - 1) if b > 1 else max(0, lk - 3) for i in range(b)], dtype=torch.int32)
    _check(*_operands(*sizes, dtype, seed=sum(sizes) + 1), causal=True)            # more queries than keys: the first see nothing
    _check(*_operands(*sizes, dtype, seed=sum(sizes) + 2), causal=True, lengths=lengths, starts=lengths - lq)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_see_nothing(dtype):
    q, k, v, lam, dout = _operands(4, 40, 70, 4, 2, 32, 64, dtype, seed=5)
    lengths = torch.tensor([0, 70, -5, 1000], dtype=torch.int32)           # clamped to 0 .. 70
    _check(q, k, v, lam, dout, lengths=lengths)
    mask = torch.zeros(4, 70, dtype=torch.bool)
    mask[1, ::3] = True
    mask[2, 69] = True
    _check(q, k, v, lam, dout, key_mask=mask)
    _check(q, k, v, lam, dout, key_mask=mask, causal=True, starts=torch.tensor([-100, 2 ** 31 - 1, -2 ** 31, 30], dtype=torch.int32),
           lengths=torch.tensor([70, 65, 70, 70], dtype=torch.int32))
    out = enc.diff_attention(*(t.to(DEV) for t in (q, k, v, lam)), lengths=lengths.to(DEV))
    assert torch.equal(out[0], torch.zeros_like(out[0])) and torch.equal(out[2], torch.zeros_like(out[2]))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_masked_places_hold_does_not_matter(dtype):
    q, k, v, lam, dout = _operands(2, 37, 90, 4, 2, 48, 80, dtype, seed=6)
    lengths = torch.tensor([61, 90], dtype=torch.int32)
    mask = torch.ones(2, 90, dtype=torch.bool)
    mask[0, 3:9] = False
    mask[1, 80:] = False
    lowest = torch.finfo(dtype).min
    for bad in (float("nan"), float("inf"), lowest):
        k2, v2 = k.clone(), v.clone()
        for b, s in ((0, slice(61, 90)), (0, slice(3, 9)), (1, slice(80, 90))):
            k2[b, s] = bad
            v2[b, s] = bad
        _check(q, k2, v2, lam, dout, lengths=lengths, key_mask=mask)
        # keys that a causal limit hides from all queries
        k2, v2 = k.clone(), v.clone()
        k2[:, 47:] = bad
        v2[:, 47:] = bad
        _check(q, k2, v2, lam, dout, causal=True, starts=torch.full((2,), 10, dtype=torch.int32))


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_permuted_operands(dtype):
    q, k, v, lam, dout = _operands(2, 50, 60, 4, 2, 24, 40, dtype, seed=7)
    # heads before tokens, maps first, a cache with room behind, one projection split in views at odd offsets
    qg = q.permute(3, 0, 2, 1, 4).contiguous().to(DEV).permute(1, 3, 2, 0, 4)
    cache = torch.full((2, 90, 2, 2, 24), float("nan"), dtype=dtype)
    cache[:, :60] = k
    wide = torch.zeros(2, 60, 2 * 40 + 3, dtype=dtype)
    wide[:, :, 1:81] = v.reshape(2, 60, 80)
    vg = wide.to(DEV)[:, :, 1:81].unflatten(-1, (2, 40))
    gpu = [qg, cache.to(DEV)[:, :60], vg, lam.to(DEV)]
    _check(q, k, v, lam, dout, gpu=gpu)
    _check(q, k, v, lam, dout, gpu=[qg.transpose(-1, -2).contiguous().transpose(-1, -2), *gpu[1:]], backward=False)
    # a gradient that is a broadcast value
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
    grads = torch.autograd.grad(enc.diff_attention(*leaves).sum(), leaves)
    want = ref.Attention(q, k, v, lam, ref.seen_keys(2, 50, 60), None, torch.ones_like(dout))
    for name, got in zip(("dq", "dk", "dv", "dlam"), grads):
        ref.assert_within(got, getattr(want, name), getattr(want, name + "_bound"), name)
    # one key and value for all requests: its gradient is the requests' sum
    one_k, one_v = (t[:1].to(DEV).requires_grad_(True) for t in (k, v))
    dk, dv = torch.autograd.grad(enc.diff_attention(leaves[0], one_k.expand(2, -1, -1, -1, -1), one_v.expand(2, -1, -1, -1), leaves[3]), (one_k, one_v),
                                 dout.to(DEV))
    want = ref.Attention(q, k[:1].expand_as(k), v[:1].expand_as(v), lam, ref.seen_keys(2, 50, 60), None, dout)
    for name, got in (("dk", dk), ("dv", dv)):
        sums, bound = (t.sum(0, keepdim=True) for t in (getattr(want, name), getattr(want, name + "_bound")))
        ref.assert_within(got, sums, bound + ref.UNIT[dtype] * sums.abs(), name + " of a broadcast operand")


def test_large_scores_keep_their_softmax():
    # scores of several hundred: only differences to the row's maximum enter the exponentials
    for dtype in TYPES:
        q, k, v, lam, dout = _operands(1, 70, 200, 2, 2, 64, 64, dtype, seed=8)
        _check(q * 8, k * 8, v, lam, dout)
        _check(q, k, v, lam, dout, scale=1e-6)


def test_many_small_probabilities_beside_a_large_one():
    # each of 4095 keys has about 2^-15 of the first one's probability: subnormal in fp16, and their sum counts
    for dtype in TYPES:
        q = torch.zeros(1, 1, 1, 2, 8, dtype=dtype)
        q[..., 0] = 1.0
        k = torch.zeros(1, 4096, 1, 2, 8, dtype=dtype)
        k[0, 0, :, :, 0] = 15 * 0.6931471805599453
        v = torch.zeros(1, 4096, 1, 4, dtype=dtype)
        v[0, 1:, :, 0] = 1.0
        v[0, 0, :, 1] = 1.0
        _check(q, k, v, torch.zeros(1, dtype=dtype), None, scale=1.0, backward=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, lq, lk, h, hk, d, dv", [(3, 1, 1000, 4, 1, 64, 128), (1, 1, 5000, 8, 2, 128, 256), (2, 4, 777, 4, 4, 32, 64),
                                                     (1, 2, 4097, 6, 2, 80, 80), (2, 16, 1500, 2, 2, 64, 64), (1, 1, 3000, 40, 1, 64, 128),
                                                     (1, 30, 2500, 1, 1, 64, 128), (5, 1, 0, 2, 1, 16, 16)])
def test_few_queries_over_long_keys(b, lq, lk, h, hk, d, dv, dtype):
    q, k, v, lam, _ = _operands(b, lq, lk, h, hk, d, dv, dtype, seed=lk)
    lengths = torch.tensor([max(0, lk - 700 * i) for i in range(b)], dtype=torch.int32)
    _check(q, k, v, lam, None, backward=False)
    _check(q, k, v, lam, None, backward=False, lengths=lengths)
    _check(q, k, v, lam, None, backward=False, lengths=lengths, causal=True, starts=lengths - lq)
    mask = torch.rand(b, lk, generator=torch.Generator().manual_seed(lk)) < 0.5
    _check(q, k, v, lam, None, backward=False, key_mask=mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b, lq, lk, h, hk, d, dv", [(1, 200, 600, 4, 2, 64, 128), (2, 513, 520, 2, 2, 32, 64), (2, 100, 1100, 2, 1, 128, 256),
                                                     (1, 37, 2049, 3, 1, 50, 33)])
def test_many_queries_of_few_requests(b, lq, lk, h, hk, d, dv, dtype):
    q, k, v, lam, _ = _operands(b, lq, lk, h, hk, d, dv, dtype, seed=lk + 1)
    lengths = torch.tensor([max(0, lk - 300 * i) for i in range(b)], dtype=torch.int32)
    _check(q, k, v, lam, None, backward=False)
    _check(q, k, v, lam, None, backward=False, causal=True)
    _check(q, k, v, lam, None, backward=False, lengths=lengths, causal=True, starts=lengths - lq)
    mask = torch.rand(b, lk, generator=torch.Generator().manual_seed(lk)) < 0.5
    _check(q, k, v, lam, None, backward=False, key_mask=mask, causal=True)


def test_lam_in_32_bits_beside_16_bit_operands():
    q, k, v, lam, dout = _operands(2, 30, 40, 4, 2, 32, 64, torch.bfloat16, seed=9)
    _check(q, k, v, lam.float(), dout)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_lam_does_not_go_through_rounded_probabilities(dtype):
    # Products of 16-bit operands are exact and sums fp32, so an fp32 dlam is off by what a probability is: its score's sum of 16 products
    # and the exponential, (16 + 4) 2^-24 of sum |q k| / 4 (at most 12 here) times log2(e) and as much for the sums, below 2^-15; a probability
    # in bf16 is off by 2^-9.
    q, k, v, lam, dout = _operands(1, 2, 8, 8, 8, 16, 32, dtype, seed=31)
    leaf = lam.float().to(DEV).requires_grad_(True)
    dlam, = torch.autograd.grad(enc.diff_attention(q.to(DEV), k.to(DEV), v.to(DEV), leaf), leaf, dout.to(DEV))
    p2 = torch.softmax(torch.einsum("bihd,bjhd->bhij", q[..., 1, :].double(), k[..., 1, :].double()) / 4, -1)
    terms = p2 * torch.einsum("bihc,bjhc->bhij", dout.double(), v.double())
    ref.assert_within(dlam, -terms.sum((0, 2, 3)), 2.0 ** -15 * terms.abs().sum((0, 2, 3)), "dlam")


def test_gradients_agree_with_differences():
    q, k, v, lam, dout = _operands(1, 9, 12, 2, 1, 8, 8, torch.float32, seed=10)
    gpu = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
    grads = torch.autograd.grad(enc.diff_attention(*gpu, causal=True), gpu, dout.to(DEV))
    h = 1e-2
    for n, (t, grad) in enumerate(zip(gpu, grads)):
        g = torch.Generator().manual_seed(n)
        way = torch.randn(t.shape, generator=g).to(DEV)
        way /= way.norm()
        f = lambda s: (enc.diff_attention(*(u.detach() + (s * way if i == n else 0) for i, u in enumerate(gpu)), causal=True).double().cpu()  # noqa: E731
                       * dout.double()).sum().item()
        # Richardson's step takes the h^2 term away; what is left is h^4 and the outputs' 1e-6 rounding over h
        slope = (8 * (f(h) - f(-h)) - (f(2 * h) - f(-2 * h))) / (12 * h)
        assert abs(slope - (grad * way).double().sum().item()) < 2e-3


def test_two_calls_give_the_same_bits():
    q, k, v, lam, dout = _operands(2, 150, 300, 4, 2, 64, 128, torch.bfloat16, seed=11)
    runs = []
    for _ in range(2):
        leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
        out = enc.diff_attention(*leaves)
        runs.append([out, *torch.autograd.grad(out, leaves, dout.to(DEV)), enc.diff_attention(*[t.detach()[:, :1] if i == 0 else t.detach()
                                                                                                 for i, t in enumerate(leaves)])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_request_does_not_depend_on_the_others():
    q, k, v, lam, _ = _operands(3, 20, 500, 4, 2, 64, 128, torch.float16, seed=12)
    gpu = [t.to(DEV) for t in (q, k, v, lam)]
    mixed = [gpu[0].clone(), gpu[1].clone(), gpu[2].clone(), gpu[3]]
    for t in mixed[:3]:
        t[0] = float("nan")
    assert torch.equal(enc.diff_attention(*gpu)[1:], enc.diff_attention(*mixed)[1:])


def test_only_some_gradients():
    q, k, v, lam, dout = _operands(1, 20, 30, 2, 2, 16, 16, torch.float32, seed=13)
    full = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
    want = torch.autograd.grad(enc.diff_attention(*full), full, dout.to(DEV))
    for n in range(4):
        some = [t.to(DEV).requires_grad_(i == n) for i, t in enumerate((q, k, v, lam))]
        assert torch.equal(torch.autograd.grad(enc.diff_attention(*some), some[n], dout.to(DEV))[0], want[n])


def test_nothing_to_do():
    for b, lq, lk, h, hk in ((0, 3, 4, 2, 1), (2, 0, 4, 2, 1), (2, 3, 0, 2, 1), (2, 3, 4, 0, 0), (2, 3, 4, 0, 1)):
        q, k, v, lam, dout = _operands(b, lq, lk, h, hk, 8, 16, torch.float32, seed=14)
        leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, lam)]
        out = enc.diff_attention(*leaves)
        grads = torch.autograd.grad(out, leaves, dout.to(DEV))
        assert out.shape == dout.shape and torch.equal(out, torch.zeros_like(out))
        assert all(torch.equal(g, torch.zeros_like(t)) for g, t in zip(grads, leaves))


def test_a_captured_call_replays():
    q, k, v, lam, _ = (t.to(DEV) for t in _operands(2, 1, 900, 4, 2, 64, 128, torch.bfloat16, seed=15))
    lengths = torch.tensor([900, 450], dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        enc.diff_attention(q, k, v, lam, lengths=lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = enc.diff_attention(q, k, v, lam, lengths=lengths)
    for n in (900, 1, 0, 333):
        lengths[0] = n
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, enc.diff_attention(q, k, v, lam, lengths=lengths))


def test_refusals():
    q, k, v, lam, _ = (t.to(DEV) for t in _operands(2, 3, 4, 4, 2, 8, 16, torch.float32, seed=16))
    ints = torch.zeros(2, dtype=torch.int32, device=DEV)
    mask = torch.ones(2, 4, dtype=torch.bool, device=DEV)
    big = torch.zeros(2, 3, 4, 2, 129, device=DEV)
    bad = [lambda: enc.diff_attention(q.double(), k.double(), v.double(), lam.double()), lambda: enc.diff_attention(q.half(), k, v, lam),
           lambda: enc.diff_attention(q, k[:1], v, lam), lambda: enc.diff_attention(q, k, v[:, :3], lam), lambda: enc.diff_attention(q, k[..., :7], v, lam),
           lambda: enc.diff_attention(q[:, :, :3], k, v, lam[:3]), lambda: enc.diff_attention(q, k, v, lam[:3]), lambda: enc.diff_attention(q, k, v, lam.half()),
           lambda: enc.diff_attention(q[:, :, :, :1], k, v, lam), lambda: enc.diff_attention(q[0], k[0], v[0], lam),
           lambda: enc.diff_attention(big, big[:, :, :2], torch.zeros(2, 3, 2, 16, device=DEV), lam),
           lambda: enc.diff_attention(q, k, torch.zeros(2, 4, 2, 257, device=DEV), lam),
           lambda: enc.diff_attention(q, k, v, lam, scale=0.0), lambda: enc.diff_attention(q, k, v, lam, scale=-1.0),
           lambda: enc.diff_attention(q, k, v, lam, scale=float("nan")), lambda: enc.diff_attention(q, k, v, lam, scale=float("inf")),
           lambda: enc.diff_attention(q, k, v, lam, lengths=ints.long()), lambda: enc.diff_attention(q, k, v, lam, lengths=ints[:1]),
           lambda: enc.diff_attention(q, k, v, lam, lengths=ints.cpu()), lambda: enc.diff_attention(q, k, v, lam, starts=ints),
           lambda: enc.diff_attention(q, k, v, lam, key_mask=mask.byte()), lambda: enc.diff_attention(q, k, v, lam, key_mask=mask[:, :3]),
           lambda: enc.diff_attention(q, k, v, lam.cpu())]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


def test_c_entry_wants_what_the_backward_reads_together():
    from mamtorch_amd import capi
    # 600 keys are split over workgroups, 6 are not
    q, k, v, lam, _ = (t.to(DEV) for t in _operands(1, 2, 600, 1, 1, 8, 16, torch.float32, seed=17))
    for keys in (600, 6):
        a = capi.DiffAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), q.stride()[:4], k.stride()[:4], v.stride()[:3],
                               B=1, Lq=2, Lk=keys, H=1, Hkv=1, D=8, Dv=16, scale=1.0, type=0, lam_type=0)
        need = capi.lib().mam_diff_attention_workspace(ctypes.byref(a))
        assert (need > 0) == (keys == 600)
        ws = torch.empty(max(1, need), dtype=torch.uint8, device=DEV)
        out, kept, lse = torch.zeros(1, 2, 1, 16, device=DEV), torch.zeros(1, 2, 1, 16, device=DEV), torch.zeros(2, 1, 1, 2, device=DEV)
        stream = torch.cuda.current_stream().cuda_stream
        for which in ((kept.data_ptr(), None), (None, lse.data_ptr())):
            assert capi.lib().mam_diff_attention(ctypes.byref(a), out.data_ptr(), *which, ws.data_ptr(), need, stream) == -1    # invalid argument
        if need:
            assert capi.lib().mam_diff_attention(ctypes.byref(a), out.data_ptr(), None, None, None, 0, stream) == -3            # no workspace
        torch.cuda.synchronize()
        assert not out.any() and not kept.any() and not lse.any()


def test_opcheck():
    q, k, v, lam, dout = (t.to(DEV) for t in _operands(2, 3, 4, 4, 2, 8, 16, torch.float32, seed=17))
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    ops = torch.ops.mamtorch_kernel_encoder
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    torch.library.opcheck(ops.diff_attention, (*leaves, 0.5, True, None, None, None, True), test_utils=tests)
    plain = [t.detach() for t in leaves]
    out, out2, lse = ops.diff_attention(*plain, 0.5, True, None, None, None, True)
    torch.library.opcheck(ops.diff_attention_backward, (dout, *plain, out, out2, lse, 0.5, True, None, None, None, True, True, True),
                          test_utils=("test_schema", "test_faketensor"))
