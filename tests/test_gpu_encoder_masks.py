"""GPU tests of masks under recomputation and capture: the gradient belongs to the mask of the output, and steps differ."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import encoder_reference as ref
import mamtorch_amd as mt

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _step(n=0):
    return torch.full((1,), n, dtype=torch.int64, device=DEV)


def _modules(step):
    """What draws masks, each over x of (3, 5, 96)."""
    torch.manual_seed(0)
    layer = mt.nn.MAMEncoderLayer(hidden=96, intermediate=160, heads=3, p=0.4, seed=5, step=step, wdrop_rate=0.3, wdrop_seed=6)
    return {"dropout": mt.nn.Dropout(0.4, 5, step), "fullyconnected": mt.nn.FullyConnected(96, 64, wdrop_rate=0.3, wdrop_seed=6, wdrop_step=step),
            "layer": layer}


def _inputs():
    return torch.randn(3, 5, 96, generator=torch.Generator().manual_seed(1)).to(DEV)


def _run(module, how, x):
    x = x.detach().requires_grad_(True)
    y = how(lambda t: module(t).square(), x)
    leaves = [x, *module.parameters()]
    return [y.detach(), *torch.autograd.grad(y.sum(), leaves)]


def _plain(call, x):
    return call(x)


def _again(call, x):
    return checkpoint(call, x, use_reentrant=False)


def _close(got, want):
    for a, b in zip(got, want):         # the same kernels on the same numbers; the order of a gradient's sums may differ
        assert (a - b).abs().max() <= 1e-5 * b.abs().max().clamp(min=1e-6)


@pytest.mark.parametrize("name", ["dropout", "fullyconnected", "layer"])
def test_gradients_of_a_recomputed_forward_are_those_of_its_mask(name):
    step, x = _step(7), _inputs()
    module = _modules(step)[name].to(DEV).train()
    want = _run(module, _plain, x)
    got = _run(module, _again, x)
    _close(got, want)
    step += 1
    other = _run(module, _plain, x)
    assert (other[0].sqrt() - want[0].sqrt()).abs().max() > 0.1         # another step, another mask
    if name == "dropout":
        keep = ref.keep_mask(x.shape, 0.4, 5, 8).to(DEV)
        assert torch.equal(other[0] != 0, keep & (x != 0))
    # the reentrant form gives gradients by backward() only
    for p in module.parameters():
        p.grad = None
    x = x.requires_grad_(True)
    y = checkpoint(lambda t: module(t).square(), x, use_reentrant=True)
    y.sum().backward()
    _close([y.detach(), x.grad, *(p.grad for p in module.parameters())], other)


@pytest.mark.parametrize("name", ["dropout", "fullyconnected", "layer"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_masks_numbered_by_calls_refuse_a_recomputed_forward(name, reentrant):
    module = _modules(None)[name].to(DEV).train()
    # the square needs its input again, so that the module runs again (dropout alone keeps no tensor and would not)
    y = checkpoint(lambda x: module(x).square(), _inputs().requires_grad_(True), use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="in a backward pass"):
        y.sum().backward()
    module.eval()           # no masks: computing again is right
    if name != "dropout":
        _close(_run(module, _again, _inputs()), _run(module, _plain, _inputs()))


@pytest.mark.parametrize("name", ["dropout", "layer"])
def test_replays_of_a_captured_step_draw_new_masks(name):
    step, x = _step(), _inputs().requires_grad_(True)
    module = _modules(step)[name].to(DEV).train()
    dy = torch.randn(3, 5, 96, generator=torch.Generator().manual_seed(2)).to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(module(x), x, dy)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = module(x)
        dx, = torch.autograd.grad(y, x, dy)
        step += 1
    eager, seen = copy.deepcopy(module), []
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        word = _step(n)
        for m in eager.modules():
            for attribute in ("step", "wdrop_step"):
                if getattr(m, attribute, None) is not None:
                    setattr(m, attribute, word)
        want = eager(x)
        _close([y.detach(), dx], [want.detach(), *torch.autograd.grad(want, x, dy)])
        seen.append(y.detach().clone())
    assert step.item() == 4 and all((a - b).abs().max() > 0.1 for a, b in zip(seen, seen[1:]))


@pytest.mark.parametrize("name", ["dropout", "fullyconnected", "layer"])
def test_masks_numbered_by_calls_refuse_capture(name):
    module, x = _modules(None)[name].to(DEV).train(), _inputs()
    module(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="under graph capture"):
        with torch.cuda.graph(graph):
            x.add_(0.0)
            module(x)
    torch.cuda.synchronize()
    module(x)


@pytest.mark.parametrize("name", ["dropout", "fullyconnected", "layer"])
def test_compiled_modules_draw_the_same_masks(name):
    x = _inputs()
    counted = _modules(None)[name].to(DEV).train()
    other = copy.deepcopy(counted)
    torch._dynamo.reset()
    compiled = torch.compile(counted, backend="eager")
    for _ in range(3):
        _close([compiled(x).detach()], [other(x).detach()])
    # computed again in a backward pass, with the check in the compiled code
    y = checkpoint(lambda t: compiled(t).square(), x.requires_grad_(True), use_reentrant=False)
    with pytest.raises(RuntimeError, match="in a backward pass"):
        y.sum().backward()


@pytest.mark.parametrize("name", ["dropout", "fullyconnected", "layer"])
def test_modules_with_a_step_compile_as_a_whole(name):
    step, x = _step(3), _inputs()
    module = _modules(step)[name].to(DEV).train()
    torch._dynamo.reset()
    compiled = torch.compile(lambda t: module(t).square(), backend="eager", fullgraph=True)
    for _ in range(2):
        want = _run(module, _plain, x)
        x1 = x.detach().requires_grad_(True)
        for call in (compiled, lambda t: checkpoint(compiled, t, use_reentrant=False)):
            y = call(x1)
            _close([y.detach(), *torch.autograd.grad(y.sum(), [x1, *module.parameters()])], want)
        step += 1
