"""CPU tests of the row stride that the norms hand to their kernels, on a host-only program."""
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_row_stride_is_where_the_rows_stand(tmp_path):
    exe = str(tmp_path / "rows_host")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", os.path.join(ROOT, "tests", "rows_host.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout[-2000:]


@pytest.mark.parametrize("reduce, strides", [(lambda y: y.sum(0), (0, 8, 1)), (lambda y: y.sum(1), (8, 0, 1)), (lambda y: y.sum((0, 1)), (0, 0, 1))])
def test_gradients_of_sums_have_rows_of_stride_0(reduce, strides):
    # why such strides are ordinary: what autograd hands to the backward of whatever was summed
    y = torch.zeros(4, 6, 8, requires_grad=True)
    seen = []
    y.register_hook(lambda g: seen.append(g.stride()))
    out = reduce(y)
    (out * torch.randn(out.shape)).sum().backward()
    assert seen == [strides]
