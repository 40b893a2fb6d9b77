"""A rotation's table is made on the device that is asked for, whatever the default device."""

from __future__ import annotations

import copy
import io

import pytest
import torch

from foldforge_b200 import kernels
from foldforge_b200.engine.modules import QKNorm


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_tables_under_another_default_device(device):
    want = kernels.rotary_table([1.0, 0.1], [1, 0], device="cpu")
    with torch.device(device):
        got = kernels.rotary_table([1.0, 0.1], [1, 0], device="cpu")
        table = QKNorm(8, frequencies=[1.0, 0.1], axes=[1, 0]).table(torch.device("cpu"))
    for t in (got, table):
        assert torch.equal(t.quarters, want.quarters) and torch.equal(t.pair_axes, want.pair_axes) and t.axes == 2


def test_a_stored_module_leaves_its_tables_behind():
    """Loaded onto another device, a table kept under its old one would be refused beside q and k."""
    norm = QKNorm(8, frequencies=[1.0, 0.1], axes=[1, 0])
    norm.table(torch.device("cpu"))
    with io.BytesIO() as f:
        torch.save(norm, f)
        f.seek(0)
        loaded = torch.load(f, map_location="meta", weights_only=False)
    for other in (loaded, copy.deepcopy(norm)):
        assert other._tables == {} and other.frequencies == norm.frequencies and other.q_weight is not norm.q_weight
        assert other.table(torch.device("cpu")).quarters.device.type == "cpu"
    assert len(norm._tables) == 1
