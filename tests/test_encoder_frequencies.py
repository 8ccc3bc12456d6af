"""The rotation's frequencies stand where a module's input does, however the module came there."""
import copy
import pickle

import pytest
import torch

import mamtorch_amd as mt

MORE = {"causal": True, "qk_norm": True, "rotary": 12}


def _module(device=None):
    torch.manual_seed(0)
    return mt.nn.DiffAttention(96, 3, device=device, **MORE)


def _right(f, device):
    # formed where they stand: powers differ in the last of their 53 bits between devices
    return f.device.type == device and f.dtype == torch.float64 and torch.equal(f, mt.kernel.encoder.rotary_frequencies(12, device=f.device))


def test_parameters_that_are_assigned_bring_the_frequencies_along():
    made, layer = _module(), mt.nn.MAMEncoderLayer(96, 128, 3, device="meta", **MORE)
    empty = _module("meta")
    assert empty.frequencies.device.type == "meta"
    empty.load_state_dict(made.state_dict(), assign=True)
    assert _right(empty.frequencies, "cpu")
    layer.load_state_dict(mt.nn.MAMEncoderLayer(96, 128, 3, **MORE).state_dict(), assign=True)
    assert _right(layer.attention.frequencies, "cpu")
    for again in (copy.deepcopy(empty), pickle.loads(pickle.dumps(empty))):
        again.load_state_dict(_module("meta").state_dict(), assign=True)
        assert again.frequencies.device.type == "meta" and _right(empty.frequencies, "cpu")
    plain = mt.nn.DiffAttention(96, 3)
    plain.load_state_dict(plain.state_dict())
    assert plain.frequencies is None


def test_a_replica_that_has_another_devices_frequencies(monkeypatch):
    seen = []

    def norm_rotate(q, k, q_weight, k_weight, frequencies, *rest):
        seen.append(frequencies)
        return q, k

    monkeypatch.setattr(mt.kernel.encoder, "norm_rotate", norm_rotate)
    monkeypatch.setattr(mt.kernel.encoder, "diff_attention", lambda q, k, v, *rest, **more: v)
    monkeypatch.setattr(mt.kernel.encoder, "layer_norm", lambda x, *rest: x)
    module = _module()
    module(torch.randn(2, 5, 96))
    assert seen.pop() is module.frequencies
    replica = module._replicate_for_data_parallel()         # shares what is neither parameter nor buffer
    for name, child in module._modules.items():
        setattr(replica, name, child)
    for name, p in module._parameters.items():
        setattr(replica, name, p)
    replica.frequencies = module.frequencies.to("meta")
    replica(torch.randn(2, 5, 96))
    assert _right(seen.pop(), "cpu")


@pytest.mark.gpu
@torch.no_grad()
def test_frequencies_of_another_device():
    module = _module().to("cuda:0")
    x = torch.randn(2, 20, 96, device="cuda:0")
    other = copy.deepcopy(module)
    other.frequencies = other.frequencies.cpu()
    assert torch.equal(module(x), other(x))
    outs = []
    for m in (module, other):
        table = mt.nn.PageTable(2, 8, 16, device="cuda:0")
        pages = m.pages(table)
        table.begin(20)
        outs.append(m(x, cache=pages))
    assert torch.equal(*outs)
    empty = _module("meta")
    empty.load_state_dict(module.state_dict(), assign=True)
    assert _right(empty.frequencies, "cuda") and torch.equal(empty(x), module(x))
