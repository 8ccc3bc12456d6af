"""GPU tests of the rotation's and the pages' operators against their registered forms, and of the modules compiled."""
import pytest
import torch

import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ops = torch.ops.mamtorch_kernel_encoder
enc = mt.kernel.encoder
FORMS = ("test_schema", "test_faketensor")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_opcheck(dtype):
    make = lambda *s: torch.randn(*s, device=DEV).to(dtype)     # noqa: E731
    q, k, v, lam = make(2, 3, 4, 2, 16), make(2, 3, 2, 2, 16), make(2, 3, 2, 8), make(4)
    w, f, places = torch.randn(16, device=DEV), enc.rotary_frequencies(12, device=DEV), _ints([[0, 1, 2], [7, 9, 8]])
    kp, vp, table, lengths, refs = make(8, 2, 16, 2, 16), make(8, 2, 16, 8), _ints([[2, 1, -1], [0, -1, -1]]), _ints([20, 5]), _ints([1, 1, 1, 0, 0, 0, 0, 0])
    counts, masks = _ints([3, 1]), torch.tensor([[1, 3, 5], [1, 2, 4]], device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, w, w)]
    torch.library.opcheck(ops.norm_rotate, (*leaves, f, places, 1e-6, True, False), test_utils=FORMS + ("test_autograd_registration",))
    for wants in ((True, True, True, True), (True, False, False, True)):
        torch.library.opcheck(ops.norm_rotate_backward, (q, k, q, k, w, w, f, places, 1e-6, True, True, *wants), test_utils=FORMS)
    torch.library.opcheck(ops.norm_rotate_append, (q, k, v, kp, vp, table, lengths, counts, w, w, f, places, 1e-6, True, False), test_utils=FORMS)
    torch.library.opcheck(ops.pages_extend, (table, lengths, refs, counts, 16), test_utils=FORMS)
    torch.library.opcheck(ops.pages_fork, (table, lengths, refs, _ints([1, 1]), 16), test_utils=FORMS)
    torch.library.opcheck(ops.pages_trim, (table, lengths, refs, _ints([4, 4]), 16), test_utils=FORMS)
    torch.library.opcheck(ops.pages_copy, (kp, vp, _ints([[0, 3], [-1, -1]])), test_utils=FORMS)
    torch.library.opcheck(ops.pages_compact, (kp, vp, table, lengths, _ints([[0, 2, 2], [1, 2, 3]]), counts), test_utils=FORMS)
    torch.library.opcheck(ops.draft_tree, (_ints([[-1, 0, 0], [-1, 0, 1]]), lengths), test_utils=FORMS)
    torch.library.opcheck(ops.diff_attention_pages, (q, kp, vp, table, lengths, lam, 0.25, counts, masks), test_utils=FORMS)


def test_compiled_training():
    torch.manual_seed(0)
    module = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=12).to(DEV)
    x = torch.randn(2, 20, 96, device=DEV, requires_grad=True)
    torch._dynamo.reset()
    compiled = torch.compile(module, backend="eager", fullgraph=True)
    for call in (module, compiled):
        y = call(x)
        grads = torch.autograd.grad(y.square().sum(), [x, *module.parameters()])
        if call is module:
            want = [y, *grads]
        else:
            assert all(torch.equal(a, b) for a, b in zip(want, [y, *grads]))


@torch.no_grad()
def test_compiled_serving():
    torch.manual_seed(0)
    module = mt.nn.DiffAttention(96, 3, causal=True, qk_norm=True, rotary=12).to(DEV)
    x = torch.randn(2, 20, 96, device=DEV)
    torch._dynamo.reset()
    outs = []
    for call in (module, torch.compile(module, backend="eager", fullgraph=True)):
        table = mt.nn.PageTable(2, 12, 16, device=DEV)
        pages = module.pages(table)
        pages.k.zero_(), pages.v.zero_()
        out = []
        for begin, end in ((0, 17), (17, 18), (18, 19)):
            table.begin(end - begin)
            out.append(call(x[:, begin:end], cache=pages))
            table.accept()
        table.begin(parents=_ints([[-1, 0, 0, 2]] * 2))
        out.append(call(x[:, :4], cache=pages))
        outs.append(out + [pages.k, pages.v])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
