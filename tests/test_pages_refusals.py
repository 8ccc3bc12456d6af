"""CPU tests of refusals of the rotation's, the pages' and the paged attention's C entry points, and of the modules' arguments."""
import ctypes

import pytest
import torch

import mamtorch_amd as mt
from mamtorch_amd import capi

ONE = ctypes.c_void_p(256)
STRIDES = (ctypes.c_int64 * 4)(16, 16, 8, 8)


def _rotate(**changes):
    a = capi.NormRotate(q=256, k=256, frequencies=256, B=1, L=2, H=2, Hkv=1, M=2, D=8, pairs=4, eps=1e-6, norm=1)
    for n, v in changes.items():
        setattr(a, n, v)
    return a


def _pages(**changes):
    p = capi.Pages(k=256, v=256, table=256, lengths=256, P=4, S=16, Hkv=1, D=8, Dv=8, B=1, slots=4)
    for n, v in changes.items():
        setattr(p, n, v)
    return p


def _attention(pages=None, **changes):
    a = capi.DiffAttentionPages(q=256, lam=256, N=2, H=2, scale=1.0, pages=pages or _pages())
    for n, v in changes.items():
        setattr(a, n, v)
    return a


def _refused(rc, code, text):
    assert rc == code, (rc, capi.lib().mam_last_error())
    assert text in capi.lib().mam_last_error(), capi.lib().mam_last_error()


@pytest.mark.parametrize("changes, code, text", [
    (dict(type=3), -1, b"unknown element type"), (dict(type=1, weight_type=2), -1, b"weights"), (dict(B=-1), -1, b"negative"), (dict(D=129), -2, b"head sizes"),
    (dict(D=0, pairs=0), -2, b"head sizes"), (dict(pairs=5), -1, b"pairs"), (dict(pairs=-1), -1, b"pairs"), (dict(frequencies=None), -1, b"null"),
    (dict(eps=-1.0), -1, b"eps"), (dict(eps=float("nan")), -1, b"eps"), (dict(eps=float("inf")), -1, b"eps"), (dict(q=None), -1, b"null"), (dict(k=None), -1, b"null"),
    (dict(H=1 << 21), -2, b"heads"), (dict(M=65), -2, b"heads"), (dict(B=1 << 20, L=1 << 12), -2, b"2^31"), (dict(L=1 << 40), -2, b"2^31")])
def test_rotation(changes, code, text):
    l, a = capi.lib(), _rotate(**changes)
    _refused(l.mam_norm_rotate(a, ONE, ONE, None), code, text)
    _refused(l.mam_norm_rotate_backward(a, ONE, STRIDES, ONE, STRIDES, ONE, ONE, ONE, ONE, ONE, 1 << 30, None), code, text)
    _refused(l.mam_norm_rotate_append(a, ONE, STRIDES, _pages(), ONE, None), code, text)
    assert l.mam_norm_rotate_backward_workspace(a) == 0


def test_rotation_needs_what_it_writes_and_reads():
    l = capi.lib()
    _refused(l.mam_norm_rotate(_rotate(), None, ONE, None), -1, b"null")
    _refused(l.mam_norm_rotate(_rotate(), ONE, None, None), -1, b"null")
    _refused(l.mam_norm_rotate(None, ONE, ONE, None), -1, b"null")
    _refused(l.mam_norm_rotate_backward(_rotate(), None, STRIDES, ONE, STRIDES, ONE, None, None, None, None, 0, None), -1, b"null")
    _refused(l.mam_norm_rotate_backward(_rotate(), ONE, None, ONE, STRIDES, ONE, None, None, None, None, 0, None), -1, b"null")
    _refused(l.mam_norm_rotate_backward(_rotate(norm=0), ONE, STRIDES, ONE, STRIDES, None, None, ONE, None, ONE, 1 << 20, None), -1, b"no norm")
    need = l.mam_norm_rotate_backward_workspace(_rotate())
    assert need > 0
    _refused(l.mam_norm_rotate_backward(_rotate(), ONE, STRIDES, ONE, STRIDES, ONE, ONE, ONE, ONE, ONE, need - 1, None), -3, b"workspace")
    assert l.mam_norm_rotate(_rotate(B=0, q=None, k=None), None, None, None) == 0


PAGES = [
    (dict(type=7), -1, b"unknown element type"), (dict(S=24), -2, b"multiple of 16"), (dict(S=0), -2, b"multiple of 16"), (dict(P=-1), -1, b"negative"),
    (dict(D=129), -2, b"head sizes"), (dict(Dv=257), -2, b"head sizes"), (dict(Dv=0), -2, b"head sizes"), (dict(table=None), -1, b"null"),
    (dict(lengths=None), -1, b"null"), (dict(k=264), -1, b"16 bytes"), (dict(v=258), -1, b"16 bytes"), (dict(slots=1 << 26), -2, b"too large"),
    (dict(P=1 << 30), -2, b"too large"), (dict(S=1 << 21), -2, b"too large")]


@pytest.mark.parametrize("changes, code, text", PAGES)
def test_pages(changes, code, text):
    l, p = capi.lib(), _pages(**changes)
    _refused(l.mam_norm_rotate_append(_rotate(), ONE, STRIDES, p, ONE, None), code, text)
    _refused(l.mam_pages_copy(p, ONE, 1, None), code, text)
    _refused(l.mam_pages_compact(p, ONE, 1, None), code, text)
    _refused(l.mam_diff_attention_pages(_attention(p), ONE, None, 0, None), code, text)
    assert l.mam_diff_attention_pages_workspace(_attention(p)) == 0


def test_pages_for_other_keys():
    l = capi.lib()
    for changes in (dict(type=1), dict(B=2), dict(Hkv=2), dict(D=16)):
        _refused(l.mam_norm_rotate_append(_rotate(), ONE, STRIDES, _pages(**changes), ONE, None), -1, b"other keys")
    _refused(l.mam_norm_rotate_append(_rotate(M=1), ONE, STRIDES, _pages(), ONE, None), -1, b"other keys")
    _refused(l.mam_norm_rotate_append(_rotate(), None, STRIDES, _pages(), ONE, None), -1, b"null")
    _refused(l.mam_norm_rotate_append(_rotate(), ONE, STRIDES, _pages(), None, None), -1, b"null")
    _refused(l.mam_norm_rotate_append(_rotate(), ONE, STRIDES, _pages(k=None), ONE, None), -1, b"null")
    _refused(l.mam_pages_copy(_pages(), None, 1, None), -1, b"null")
    _refused(l.mam_pages_copy(_pages(), ONE, -1, None), -1, b"negative")
    _refused(l.mam_pages_compact(_pages(), None, 1, None), -1, b"null")
    _refused(l.mam_pages_compact(_pages(), ONE, 1 << 30, None), -2, b"too long")


@pytest.mark.parametrize("sizes, code, text", [
    ((-1, 4, 4, 16), -1, b"negative"), ((1, -4, 4, 16), -1, b"negative"), ((1, 4, 4, 8), -2, b"multiple of 16"), ((4097, 4, 4, 16), -2, b"4096"),
    ((1, 1 << 29, 4, 16), -2, b"too large"), ((4096, 1 << 20, 4, 16), -2, b"too large"), ((1, 4, 1 << 30, 16), -2, b"too large")])
def test_bookkeeping(sizes, code, text):
    l = capi.lib()
    _refused(l.mam_pages_extend(ONE, ONE, ONE, ONE, ONE, ONE, *sizes, ONE, 1 << 40, None), code, text)
    _refused(l.mam_pages_fork(ONE, ONE, ONE, ONE, *sizes, None), code, text)
    _refused(l.mam_pages_trim(ONE, ONE, ONE, ONE, *sizes, None), code, text)


def test_bookkeeping_needs_what_it_reads():
    l, sizes = capi.lib(), (2, 4, 8, 16)
    for gone in range(6):
        args = [None if n == gone else ONE for n in range(6)]
        _refused(l.mam_pages_extend(*args, *sizes, ONE, 1 << 20, None), -1, b"null")
    for call in (l.mam_pages_fork, l.mam_pages_trim):
        for gone in range(4):
            _refused(call(*[None if n == gone else ONE for n in range(4)], *sizes, None), -1, b"null")
    assert l.mam_pages_extend_workspace(2, 4, 8) == 4 * 8 and l.mam_pages_extend_workspace(2, 4, 800) == 4 * 10
    _refused(l.mam_pages_extend(ONE, ONE, ONE, ONE, ONE, ONE, *sizes, ONE, 31, None), -3, b"workspace")
    assert l.mam_pages_extend(None, None, None, None, None, None, 0, 4, 8, 16, None, 0, None) == 0
    _refused(l.mam_draft_tree(ONE, None, ONE, ONE, 1, 65, None), -2, b"64 tokens")
    _refused(l.mam_draft_tree(None, None, ONE, ONE, 1, 4, None), -1, b"null")
    _refused(l.mam_draft_tree(ONE, None, ONE, ONE, -1, 4, None), -1, b"negative")
    assert l.mam_draft_tree(None, None, None, None, 0, 4, None) == 0


@pytest.mark.parametrize("changes, code, text", [
    (dict(H=3, pages=_pages(Hkv=2)), -1, b"divide"), (dict(N=65, masks=256), -2, b"64 tokens"), (dict(scale=0.0), -1, b"scale"), (dict(scale=1e-300), -1, b"scale"),
    (dict(scale=float("nan")), -1, b"scale"), (dict(lam_type=1), -1, b"lam"), (dict(N=-1), -1, b"negative"), (dict(q=None), -1, b"null"), (dict(lam=None), -1, b"null"),
    (dict(N=1 << 40), -2, b"2^29"), (dict(pages=_pages(k=None)), -1, b"null")])
def test_attention(changes, code, text):
    l, a = capi.lib(), _attention(**changes)
    _refused(l.mam_diff_attention_pages(a, ONE, None, 0, None), code, text)


def test_attention_over_more_pages_than_it_counts():
    l = capi.lib()
    _refused(l.mam_diff_attention_pages(_attention(_pages(P=1 << 28, Hkv=2, S=128)), ONE, None, 0, None), -2, b"too many pages")


def test_attention_needs_its_workspace():
    l = capi.lib()
    a = _attention(_pages(slots=1024, P=1024, S=64))
    need = l.mam_diff_attention_pages_workspace(a)
    assert need > 0
    _refused(l.mam_diff_attention_pages(a, ONE, ONE, need - 1, None), -3, b"workspace")
    assert l.mam_diff_attention_pages(_attention(N=0), None, None, 0, None) == 0


def test_modules():
    with pytest.raises(ValueError, match="multiple of 16"):
        mt.nn.PageTable(2, 8, page_size=24)
    for rotary in (-2, 3, 18):
        with pytest.raises(ValueError, match="rotary"):
            mt.nn.DiffAttention(64, 2, causal=True, rotary=rotary)
    layer = mt.nn.DiffAttention(64, 2, rotary=True, qk_norm=True)
    assert layer.rotary == 16 and layer.frequencies.dtype == torch.float64 and layer.query_norm.shape == (16,)
    assert layer.half().frequencies.dtype == torch.float64            # no buffer that a cast rounds
    assert "frequencies" not in layer.state_dict()
    table = mt.nn.PageTable(2, 8, 16)
    pages = layer.pages(table)
    assert table.table.shape == (2, 8) and table.caches == [pages] and pages.k.dtype == torch.float16
    with pytest.raises(ValueError, match="causal"):
        layer(torch.zeros(2, 1, 64, dtype=torch.float16), cache=pages)
    with pytest.raises(ValueError, match="no step"):
        table.accept()
    with pytest.raises(ValueError, match="counts or parents"):
        table.begin()
    with pytest.raises(ValueError, match="no step"):
        pages.attend(torch.zeros(2, 1, 2, 2, 16), torch.zeros(2))
    with pytest.raises((RuntimeError, NotImplementedError)):
        table.begin(1)                                                # tensors on the CPU: no fallback
    plain = mt.nn.DiffAttention(64, 2)
    assert sorted(plain.state_dict()) == sorted(n for n in layer.state_dict() if n not in ("query_norm", "key_norm"))
