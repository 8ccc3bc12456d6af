"""CPU tests of what numbers the masks of the modules that form them from counters."""
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
