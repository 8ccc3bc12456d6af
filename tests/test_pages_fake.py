"""CPU tests of the rotation's and the pages' operators under fake tensors: shapes, types, and the refusals that the operators themselves have."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mamtorch_amd as mt

enc = mt.kernel.encoder
I32 = torch.int32


@pytest.fixture(autouse=True)
def _fake():
    with FakeTensorMode():
        yield


def make(*shape, t=torch.float32):
    return torch.empty(*shape, dtype=t, device="cuda")


def _rotate(**changes):
    return {**dict(q=make(2, 3, 4, 2, 16), k=make(2, 3, 2, 2, 16)), **changes}


def _append(**changes):
    return {**dict(q=make(2, 3, 4, 2, 16), k=make(2, 3, 2, 2, 16), v=make(2, 3, 2, 8), k_pages=make(8, 2, 16, 2, 16), v_pages=make(8, 2, 16, 8), table=make(2, 4, t=I32),
                   lengths=make(2, t=I32)), **changes}


def _attend(**changes):
    return {**dict(q=make(2, 3, 4, 2, 16), k_pages=make(8, 2, 16, 2, 16), v_pages=make(8, 2, 16, 8), table=make(2, 4, t=I32), lengths=make(2, t=I32), lam=make(4)), **changes}


def _book(name):
    def of(**changes):
        return {**{"table": make(2, 4, t=I32), "lengths": make(2, t=I32), "refs": make(8, t=I32), name: make(2, t=I32), "page_size": 16}, **changes}
    return of


def _copy(**changes):
    return {**dict(k_pages=make(8, 2, 16, 2, 16), v_pages=make(8, 2, 16, 8), copies=make(5, 2, t=I32)), **changes}


def _compact(**changes):
    return {**dict(k_pages=make(8, 2, 16, 2, 16), v_pages=make(8, 2, 16, 8), table=make(2, 4, t=I32), lengths=make(2, t=I32), path=make(2, 5, t=I32)), **changes}


def _tree(**changes):
    return {**dict(parents=make(2, 5, t=I32)), **changes}


def test_shapes_and_types():
    for t in (torch.float32, torch.bfloat16, torch.float16):
        q, k = enc.norm_rotate(**_rotate(q=make(2, 3, 4, 2, 16, t=t), k=make(2, 3, 2, 2, 16, t=t), q_weight=make(16), frequencies=make(8, t=torch.float64), positions=make(2, 3, t=I32)))
        assert q.shape == (2, 3, 4, 2, 16) and k.shape == (2, 3, 2, 2, 16) and q.dtype == k.dtype == t
        pages = dict(k_pages=make(8, 2, 16, 2, 16, t=t), v_pages=make(8, 2, 16, 8, t=t))
        y = enc.norm_rotate_append(**_append(q=q, k=k, v=make(2, 3, 2, 8, t=t), **pages, counts=make(2, t=I32)))
        assert y.shape == q.shape and y.dtype == t
        out = enc.diff_attention_pages(**_attend(q=q, **pages, masks=make(2, 3, t=torch.long)))
        assert out.shape == (2, 3, 4, 8) and out.dtype == t
    dy, w = make(2, 3, 4, 2, 16), make(16)
    grads = torch.ops.mamtorch_kernel_encoder.norm_rotate_backward(dy, None, dy, make(2, 3, 2, 2, 16), w, w, None, None, 1e-6, True, False, True, False, True, False)
    assert [g.shape for g in grads] == [dy.shape, (0,), w.shape, (0,)]
    granted, copies = enc.pages_extend(**_book("counts")())
    assert granted.shape == (2,) and copies.shape == (2, 2) and granted.dtype == copies.dtype == I32
    masks, positions = enc.draft_tree(**_tree(lengths=make(2, t=I32)))
    assert masks.shape == positions.shape == (2, 5) and masks.dtype == torch.long and positions.dtype == I32
    assert enc.pages_fork(**_book("sources")()) is None and enc.pages_trim(**_book("ends")()) is None
    assert enc.pages_copy(**_copy()) is None and enc.pages_compact(**_compact(counts=make(2, t=I32))) is None
    pages = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=True, device="cuda")
    table = mt.nn.PageTable(2, 8, 16, device="cuda")
    cache = pages.pages(table)
    with torch.no_grad():
        table.begin(parents=make(2, 5, t=I32))
        assert pages(make(2, 5, 96), cache=cache).shape == (2, 5, 96)
        table.accept(make(2, 5, t=I32))


def _refused(call, make_args, **changes):
    with pytest.raises((RuntimeError, NotImplementedError)):
        call(**make_args(**changes))


def test_refusals_of_the_rotation():
    for bad in (dict(k=make(2, 3, 2, 1, 16)), dict(k=make(2, 4, 2, 2, 16)), dict(k=make(2, 3, 2, 2, 8)), dict(k=make(2, 3, 2, 2, 16, t=torch.half)), dict(q=make(2, 3, 4, 16)),
                dict(q=make(2, 3, 4, 2, 129), k=make(2, 3, 4, 2, 129)), dict(q=make(2, 3, 4, 2, 16, t=torch.double), k=make(2, 3, 2, 2, 16, t=torch.double)), dict(q_weight=make(8)),
                dict(q_weight=make(16, t=torch.half)), dict(q_weight=make(16), norm=False), dict(frequencies=make(8)), dict(frequencies=make(9, t=torch.double)),
                dict(positions=make(2, 4, t=I32)), dict(positions=make(2, 3, t=torch.long))):
        _refused(enc.norm_rotate, _rotate, **bad)


def test_refusals_of_the_append():
    for bad in (dict(q=make(2, 3, 4, 2, 16, t=torch.half)), dict(k=make(2, 3, 1, 2, 16)), dict(v=make(2, 3, 2, 9)), dict(v=make(2, 3, 2, 8, t=torch.half)), dict(v=make(2, 2, 2, 8)),
                dict(k_pages=make(8, 2, 24, 2, 16), v_pages=make(8, 2, 24, 8)), dict(v_pages=make(7, 2, 16, 8)), dict(k_pages=make(8, 2, 16, 2, 16, t=torch.half), v_pages=make(8, 2, 16, 8, t=torch.half)),
                dict(table=make(3, 4, t=I32), lengths=make(3, t=I32)), dict(lengths=make(3, t=I32)), dict(counts=make(2, t=torch.long)), dict(q=make(2, 3, 4, 1, 16), k=make(2, 3, 2, 1, 16)),
                dict(positions=make(2, 2, t=I32)), dict(k_pages=make(8, 2, 16, 2, 24))):
        _refused(enc.norm_rotate_append, _append, **bad)


def test_refusals_of_the_attention():
    for bad in (dict(q=make(2, 3, 4, 2, 64)), dict(q=make(3, 3, 4, 2, 16)), dict(q=make(2, 3, 4, 2, 16, t=torch.half)), dict(q=make(2, 3, 3, 2, 16), lam=make(3)), dict(q=make(2, 3, 4, 1, 16)),
                dict(q=make(2, 3, 4, 16)), dict(lam=make(3)), dict(lam=make(4, t=torch.half)), dict(lam=make(1, 4)), dict(masks=make(2, 3, t=I32)), dict(masks=make(3, 3, t=torch.long)),
                dict(q=make(2, 65, 4, 2, 16), masks=make(2, 65, t=torch.long)), dict(counts=make(3, t=I32)), dict(table=make(3, 4, t=I32), lengths=make(3, t=I32)), dict(lengths=make(2)),
                dict(scale=0.0), dict(scale=float("inf")), dict(v_pages=make(8, 2, 16, 257)), dict(k_pages=make(8, 2, 24, 2, 16), v_pages=make(8, 2, 24, 8))):
        _refused(enc.diff_attention_pages, _attend, **bad)


@pytest.mark.parametrize("call, name", [(enc.pages_extend, "counts"), (enc.pages_fork, "sources"), (enc.pages_trim, "ends")])
def test_refusals_of_the_bookkeeping(call, name):
    for bad in (dict(table=make(2, 4, t=torch.long)), dict(table=make(8, t=I32)), dict(lengths=make(3, t=I32)), dict(lengths=make(2)), dict(refs=make(8)), dict(refs=make(2, 4, t=I32)),
                {name: make(3, t=I32)}, {name: make(2, t=torch.long)}, dict(page_size=24), dict(page_size=0), dict(table=make(4097, 4, t=I32), lengths=make(4097, t=I32), **{name: make(4097, t=I32)})):
        _refused(call, _book(name), **bad)


def test_refusals_of_copies_and_trees():
    for bad in (dict(copies=make(5, 3, t=I32)), dict(copies=make(5, 2, t=torch.long)), dict(copies=make(10, t=I32)), dict(v_pages=make(8, 1, 16, 8)), dict(v_pages=make(8, 2, 16, 8, t=torch.half))):
        _refused(enc.pages_copy, _copy, **bad)
    for bad in (dict(path=make(3, 5, t=I32)), dict(path=make(2, 5, t=torch.long)), dict(path=make(2, t=I32)), dict(counts=make(3, t=I32)), dict(lengths=make(1, t=I32))):
        _refused(enc.pages_compact, _compact, **bad)
    for bad in (dict(parents=make(2, 65, t=I32)), dict(parents=make(2, 5, t=torch.long)), dict(parents=make(5, t=I32)), dict(lengths=make(3, t=I32)), dict(lengths=make(2, t=torch.long))):
        _refused(enc.draft_tree, _tree, **bad)
