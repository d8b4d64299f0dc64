"""The dims and bases that rope_axes passes on are those of the call (CPU: the launch is left out and its arguments read)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from selas_b200 import _lib, ops
from selas_b200._lib import FluxB200Error

X = torch.zeros(1, 2, 3, 64)
IDS = torch.zeros(3, 2)


@pytest.fixture
def sent(monkeypatch):
    """A call's (bases, dims) as the kernel gets them."""
    packed = []
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_launch", lambda index, entry, flops, nbytes, args: packed.append(args))

    def call(dims, theta):
        ops.rope_axes(X, IDS, dims, theta)
        a = _lib.FbRopeArgs.from_buffer_copy(packed.pop())
        return list(a.theta[:a.axes]), list(a.axes_dim[:a.axes])

    return call


def test_a_base_that_changes_in_place_is_read_again(sent):
    """A tensor or array as the base, alone or one per axis: the call uses the value it has now."""
    one, other = torch.tensor(10000.0), torch.tensor(500.0)
    assert sent((24, 40), one) == ([1e4, 1e4], [24, 40])
    assert sent((24, 40), (one, other)) == ([1e4, 500.0], [24, 40])
    one.fill_(777.0)
    other.fill_(3.0)
    assert sent((24, 40), one) == ([777.0, 777.0], [24, 40])
    assert sent((24, 40), (one, other)) == ([777.0, 3.0], [24, 40])
    assert sent((24, 40), np.array(2.5)) == ([2.5, 2.5], [24, 40])


def test_dims_that_change_in_place_are_read_again(sent):
    dims = (torch.tensor(24), torch.tensor(40))
    assert sent(dims, 1e4) == ([1e4, 1e4], [24, 40])
    dims[0].fill_(32)
    dims[1].fill_(32)
    assert sent(dims, 1e4) == ([1e4, 1e4], [32, 32])
    assert sent(torch.tensor([20, 44]), 1e4) == sent([20, 44], 10000) == sent(np.array([20, 44]), np.float32(1e4)) == ([1e4, 1e4], [20, 44])


@pytest.mark.parametrize("dims,theta", [((24.5, 39.5), 1e4), (64, 1e4), (("a", "b"), 1e4), ((24, 40), "base"), ((24, 40), None),
                                        ((24, 40), torch.ones(2)), ((float("nan"), 40), 1e4)])
def test_what_is_no_number_is_refused(sent, dims, theta):
    with pytest.raises(FluxB200Error, match="whole numbers"):
        sent(dims, theta)
