"""CPU tests of what numbers the masks of the modules that form them from counters."""
import io

import pytest
import torch

import mamtorch_amd as mt


def _dropout():
    module = mt.nn.Dropout(0.5, 3)
    return module, module.next_offset


def _fullyconnected():
    module = mt.nn.FullyConnected(6, 4, wdrop_rate=0.5, wdrop_seed=3).train()
    return module, module._dropped_weight


@pytest.mark.parametrize("make", [_dropout, _fullyconnected])
def test_a_counted_mask_is_refused_in_a_backward_pass(make):
    module, draw = make()
    x = torch.ones(2, requires_grad=True)
    y = x * 2
    y.register_hook(lambda g: draw() and None)
    with pytest.raises(RuntimeError, match="in a backward pass.*step"):
        y.sum().backward()


@pytest.mark.parametrize("make", [_dropout, _fullyconnected])
def test_a_counted_mask_is_refused_in_a_replica(make):
    module, _ = make()
    replica = module._replicate_for_data_parallel()
    replica.weight = getattr(module, "weight", None)
    with pytest.raises(RuntimeError, match="in a replica.*step"):
        replica.next_offset() if isinstance(replica, mt.nn.Dropout) else replica._dropped_weight()


def test_calls_number_the_masks_where_nothing_else_does():
    module = mt.nn.Dropout(0.5, 3)
    assert [module.next_offset() for _ in range(3)] == [0, 1, 2] and module.get_extra_state()["calls"] == 3
    module.step = torch.zeros(1, dtype=torch.int64)
    assert [module.next_offset() for _ in range(3)] == [0, 0, 0] and module.get_extra_state()["calls"] == 3


def _keys(layer):
    return [layer.dropout1.seed, layer.dropout2.seed]


def _layer(**kwargs):
    return mt.nn.MAMEncoderLayer(hidden=24, intermediate=40, heads=2, **kwargs)


def test_modules_without_a_seed_take_one_of_their_own():
    torch.manual_seed(0)
    layers = [_layer(p=0.1) for _ in range(3)]
    drops = [mt.nn.Dropout(), mt.nn.Dropout()]
    keys = [k for layer in layers for k in _keys(layer)] + [d.seed for d in drops]
    assert len(set(keys)) == 8
    torch.manual_seed(0)
    assert _keys(_layer(p=0.1)) == keys[:2]


def test_a_module_that_drops_nothing_draws_nothing():
    torch.manual_seed(0)
    before = torch.random.get_rng_state()
    module = mt.nn.Dropout(0.0)
    assert torch.equal(torch.random.get_rng_state(), before) and module.seed is None
    module.p = 0.5
    module.next_offset()
    other = mt.nn.Dropout(0.0)
    other.next_offset()
    assert module.seed is not None and module.seed != other.seed


def test_layers_of_one_seed_differ_by_depth():
    keys = [k for depth in range(1, 13) for k in _keys(_layer(p=0.1, seed=7, depth=depth))]
    assert len(set(keys)) == 24 and keys[:2] == [14, 15]


def test_a_drawn_seed_is_taken_up_with_the_state_and_a_given_one_kept():
    layer = _layer(p=0.1)
    layer.dropout1.next_offset()
    other, given = _layer(p=0.1), _layer(p=0.1, seed=7)
    for to in (other, given):
        to.load_state_dict(layer.state_dict())
        assert to.dropout1.calls == 1 and to.dropout2.calls == 0
    assert _keys(other) == _keys(layer) and _keys(given) == [14, 15]
    other.load_state_dict(given.state_dict())
    assert _keys(other) == [14, 15]
    state = layer.state_dict()
    state["dropout1._extra_state"] = {"calls": 4}           # as it was before seeds were part of it
    keys = _keys(other)
    other.load_state_dict(state)
    assert other.dropout1.calls == 4 and other.dropout1.seed == keys[0]


def test_weights_of_a_layer_have_masks_of_their_own():
    layers = [_layer(p=0.1, seed=7, depth=depth, wdrop_rate=0.5, wdrop_seed=14) for depth in (1, 2)]
    keys = [k & 2 ** 64 - 1 for layer in layers for k in (*_keys(layer), layer.intermediate.wdrop_seed, layer.output.wdrop_seed)]
    assert len(set(keys)) == 8
    assert _layer(wdrop_rate=0.5).output.wdrop_seed is None


def test_a_module_that_was_saved_whole_before_it_had_a_seed_still_trains(monkeypatch):
    module = mt.nn.FullyConnected(6, 4, wdrop_rate=0.5)
    for name in ("wdrop_seed", "wdrop_step", "wdrop_calls"):
        del module.__dict__[name]
    file = io.BytesIO()
    torch.save(module, file)
    file.seek(0)
    module = torch.load(file, weights_only=False).train()
    monkeypatch.setattr(mt.kernel.v4, "apply_keep", lambda w, keep: w * keep)
    assert module._dropped_weight().shape == (4, 6) and sorted(module.state_dict()) == ["bias", "weight"]


def test_calls_of_a_weights_dropout_are_part_of_the_state():
    make = lambda **kwargs: torch.nn.Sequential(mt.nn.FullyConnected(6, 4, **kwargs), torch.nn.ReLU())      # noqa: E731
    counted, other, plain = make(wdrop_rate=0.5, wdrop_seed=3), make(wdrop_rate=0.5, wdrop_seed=3), make()
    counted[0].wdrop_calls = 5
    state = counted.state_dict()
    assert sorted(state) == ["0.bias", "0.wdrop_calls", "0.weight"] and sorted(plain.state_dict()) == ["0.bias", "0.weight"]
    other.load_state_dict(state)
    assert other[0].wdrop_calls == 5 and torch.equal(other[0].weight, counted[0].weight)
    other.load_state_dict(plain.state_dict())               # a state without it
    assert other[0].wdrop_calls == 5 and torch.equal(other[0].weight, plain[0].weight)
    plain.load_state_dict(state)                            # a layer without a seed
    assert "0.wdrop_calls" in state
    with pytest.raises(RuntimeError, match="Unexpected"):
        other.load_state_dict({**state, "0.wdrop_call": torch.tensor(1)})


def test_a_dropout_that_was_saved_whole_before_it_had_a_step_still_draws():
    module = mt.nn.Dropout(0.5, 3)
    for name in ("step", "seed_given"):
        del module.__dict__[name]
    file = io.BytesIO()
    torch.save(module, file)
    file.seek(0)
    module = torch.load(file, weights_only=False).train()
    assert module.next_offset() == 0 and module.step is None
    module.load_state_dict(mt.nn.Dropout(0.5, 8).state_dict())
    assert module.seed == 3 and module.calls == 0
