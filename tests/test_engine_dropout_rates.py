"""Dropout of a whole model at the ops' own rates, without a GPU."""

from __future__ import annotations

import pytest
import torch

from foldforge_b200.engine import training
from foldforge_b200.engine.evoformer import EvoformerBlock
from foldforge_b200.engine.modules import PairformerBlock, PairformerConfig, Transition
from foldforge_b200.engine.pairformer import pairformer_block


def dropping(model):
    return [n for n, m in model.named_modules() if getattr(m, "dropout", 0) > 0]


@pytest.mark.parametrize("make", [lambda: EvoformerBlock(), lambda: pairformer_block(d_pair=16, triangle_model="af3"),
                                  lambda: PairformerBlock(PairformerConfig(d_pair=16, d_hidden_tri_multi=16, d_single=0))])
def test_a_model_whose_ops_have_no_rate_is_told_so(make):
    """The factories and the engine's blocks give their ops no rate: without one nothing would be dropped."""
    model = make()
    with pytest.raises(ValueError, match="rate"):
        training.set_dropout(model)
    assert dropping(model) == []
    names = training.set_dropout(model, 0.2)
    assert names and dropping(model) == names
    with pytest.raises(ValueError, match="rate"):
        training.set_dropout(model)
    assert dropping(model) == names  # a call that is refused changes nothing
    assert training.set_dropout(model, 0.0) == names and dropping(model) == []


def test_ops_with_and_without_a_rate():
    model = torch.nn.ModuleList([PairformerBlock(PairformerConfig(d_pair=16, d_hidden_tri_multi=16, d_single=0, p_drop=p)) for p in (0.25, 0.0)])
    names = training.set_dropout(model)
    assert len(names) == 8 and dropping(model) == names[:4]
    assert training.set_dropout(Transition(8)) == []  # nothing to drop


def test_an_op_of_another_kind_keeps_its_own_rate():
    """A module of the user's that takes dropout in its own way decides what no rate means."""

    class Op(torch.nn.Module):
        def set_dropout(self, p=None):
            self.dropout = 0.3 if p is None else p

    op = Op()
    assert training.set_dropout(op) == [""] and op.dropout == 0.3
