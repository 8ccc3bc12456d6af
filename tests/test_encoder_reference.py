"""CPU tests of the encoder operators' oracle, schemas, shapes and refusals on the host."""
import ctypes

import numpy as np
import pytest
import torch

import encoder_reference as ref
from mamtorch_amd import capi


def test_generator_gives_the_published_words():
    # the answers that the generator's authors publish for all-zero and all-one input
    assert ref.random_words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.random_words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_words_of_elements_are_those_of_their_counters():
    seed, offset = 0x0123456789ABCDEF, 0xFEDCBA9876543210
    for first in (0, 5, 2 ** 34 - 3):       # the low word of the group's number wraps
        words = ref.element_words(first, 11, seed, offset)
        for i in range(11):
            g = (first + i) // 4
            want = ref.random_words([g & 0xFFFFFFFF, g >> 32, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
            assert int(words[i]) == want[(first + i) % 4]


def test_norm_gradients_agree_with_differences():
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = (torch.randn(*s, generator=g).double() for s in ((3, 7), (7,), (7,), (3, 7)))
    f = lambda x, w, b: (ref.norm(x, w, b, 1e-5)[0] * dy).sum()     # noqa: E731
    _, xh, rstd = ref.norm(x, w, b, 1e-5)
    dx, dw, db = ref.norm_backward(dy, xh, rstd, w)
    h = 1e-6
    for t, grad in ((x, dx), (w, dw), (b, db)):
        for i in range(t.numel()):
            at = t.reshape(-1)[i].item()
            t.reshape(-1)[i] = at + h
            up = f(x, w, b)
            t.reshape(-1)[i] = at - h
            down = f(x, w, b)
            t.reshape(-1)[i] = at
            # the difference quotient errs by h^2 of the third derivative and by 1e-16 / h
            assert abs((up - down) / (2 * h) - grad.reshape(-1)[i]) < 1e-8


def test_the_c_entry_points_refuse_what_they_do_not_cover():
    l, one = capi.lib(), ctypes.c_void_p(256)
    drop = capi.Dropout(p=0.1, scale=1.0)
    call = l.mam_dropout
    assert call(one, None, one, -1, capi.F32, drop, None) == -1
    assert call(one, None, one, 4, 7, drop, None) == -1
    assert call(one, None, one, 4, capi.F32, None, None) == -1
    assert call(None, None, one, 4, capi.F32, drop, None) == -1
    assert call(one, None, one, 4, capi.F32, capi.Dropout(p=1.5), None) == -1
    assert call(one, None, one, 4, capi.F32, capi.Dropout(p=float("nan")), None) == -1
    assert call(None, None, None, 0, capi.F32, drop, None) == 0         # nothing to do
    norm = l.mam_layer_norm
    assert norm(one, 8, None, None, 1e-5, one, None, None, 4, -1, capi.F32, capi.F32, None) == -1
    assert norm(one, 7, None, None, 1e-5, one, None, None, 4, 8, capi.F32, capi.F32, None) == -1
    assert norm(one, 8, None, None, 1e-5, one, None, None, 4, 8, capi.F32, capi.BF16, None) == -1
    assert norm(one, 2 ** 31, None, None, 1e-5, one, None, None, 4, 2 ** 31, capi.F32, capi.F32, None) == -2
    assert norm(None, 8, None, None, 1e-5, None, None, None, 0, 8, capi.F32, capi.F32, None) == 0
    need = l.mam_layer_norm_backward_workspace(100, 8, capi.F32)
    assert need > 0 and l.mam_layer_norm_backward_workspace(0, 8, capi.F32) == 0
    back = l.mam_layer_norm_backward
    assert back(one, 8, one, 8, None, one, one, one, one, one, 100, 8, capi.F32, capi.F32, one, need - 1, None) == -3
    assert back(one, 8, one, 8, None, None, one, one, None, None, 100, 8, capi.F32, capi.F32, None, 0, None) == -1


def test_fake_kernels_propagate_shapes_and_types():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.mamtorch_kernel_encoder
    with FakeTensorMode():
        x = torch.empty(3, 5, 12, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(12, device="cuda")
        y, mean, rstd = ops.layer_norm(x, w, w, 1e-5, True)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (15,) and mean.dtype == torch.float32
        dx, dw, db = ops.layer_norm_backward(x, x, w, mean, rstd, True, True, False, True)
        assert dx.shape == x.shape and dw.shape == (12,) and dw.dtype == torch.float32 and db.numel() == 0
        assert ops.dropout(x, x, 0.1, 1.0, 1, 2, None).shape == x.shape
        y, s, mean, _ = ops.add_dropout_layer_norm(x, x, None, None, 0.1, 1.0, 1, 2, 1e-5, None, False)
        assert y.shape == s.shape == x.shape and mean.numel() == 0


def test_attention_gradients_agree_with_differences():
    g = torch.Generator().manual_seed(1)
    q, k, v, lam, dout = (torch.randn(*s, generator=g).double() for s in ((2, 3, 4, 2, 5), (2, 6, 2, 2, 5), (2, 6, 2, 7), (4,), (2, 3, 4, 7)))
    ref.UNIT[torch.float64], ref.TINY[torch.float64] = 2.0 ** -53, 0.0
    seen = ref.seen_keys(2, 3, 6, causal=True, lengths=torch.tensor([6, 2]), starts=torch.tensor([2, -1]))
    assert seen[1, 0].sum() == 0 and seen[0, 0].sum() == 3
    want = ref.Attention(q, k, v, lam, seen, None, dout)
    f = lambda: (ref.Attention(q, k, v, lam, seen).out * dout).sum().item()         # noqa: E731
    h = 1e-6
    for t, grad in ((q, want.dq), (k, want.dk), (v, want.dv), (lam, want.dlam)):
        flat, grad = t.reshape(-1), grad.reshape(-1)
        for i in range(0, t.numel(), 7):
            at = flat[i].item()
            flat[i] = at + h
            up = f()
            flat[i] = at - h
            down = f()
            flat[i] = at
            assert abs((up - down) / (2 * h) - grad[i].item()) < 1e-7


def test_the_attention_entry_points_refuse_what_they_do_not_cover():
    l = capi.lib()

    def call(**changes):
        a = capi.DiffAttention(q=256, k=256, v=256, lam=256, B=1, Lq=2, Lk=2, H=2, Hkv=1, D=8, Dv=8, scale=1.0)
        for n, v in changes.items():
            setattr(a, n, v)
        one = ctypes.c_void_p(256)
        forward = l.mam_diff_attention(a, None if changes.get("no_out") else one, None, None, None, 0, None)
        strides = (ctypes.c_int64 * 3)(16, 8, 8)
        backward = l.mam_diff_attention_backward(a, one, strides, None if changes.get("no_out") else one, one, one, one, one, one, one, None, 0, None)
        return forward, backward

    assert call(B=-1) == call(Lk=-1) == call(Hkv=0) == call(H=3, Hkv=2) == call(type=9) == call(lam_type=1) == (-1, -1)
    assert call(scale=0.0) == call(scale=float("nan")) == call(scale=float("inf")) == call(scale=-2.0) == (-1, -1)
    assert call(D=129) == call(D=0) == call(Dv=257) == call(B=2 ** 31) == call(Lq=2 ** 30) == (-2, -2)
    assert call(q=None) == call(k=None) == call(v=None) == call(lam=None) == call(no_out=True) == (-1, -1)
    assert call(B=0)[0] == 0
    a = capi.DiffAttention(q=256, k=256, v=256, lam=256, B=1, Lq=2, Lk=2, H=2, Hkv=1, D=8, Dv=8, scale=1.0)
    assert l.mam_diff_attention_backward_workspace(a) == 5 * 4 * 4
    assert l.mam_diff_attention(None, None, None, None, None, 0, None) == -1
