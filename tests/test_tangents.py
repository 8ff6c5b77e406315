"""The check that refuses tensors with a forward-mode tangent."""
import pytest
import torch

from stof.ops import StofError, _refuse_tangents


def test_tangents_are_noticed_inside_a_level_only():
    fw = torch.autograd.forward_ad
    x = torch.zeros(3)
    _refuse_tangents(x, None)
    with fw.dual_level():
        _refuse_tangents(x, None)
        with pytest.raises(StofError, match="tangent"):
            _refuse_tangents(None, x, fw.make_dual(x, x))
        _refuse_tangents(torch.zeros(2, dtype=torch.int8))
    _refuse_tangents(x)
