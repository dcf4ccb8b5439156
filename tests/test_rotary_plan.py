"""CPU tests of Rotary plans as tuples: a plan of one position a token is its three values, as it is unpacked and packed."""

import copy
import pickle

import pytest
import torch

from fa2.rotary import Rotary, rotary_plan


@pytest.mark.parametrize("plan", [rotary_plan(32, device="cpu"), rotary_plan(32, interleaved=True, device="cpu")._replace(scale=1.5),
                                  Rotary(torch.ones(8, dtype=torch.float64)), Rotary(torch.ones(8, dtype=torch.float64), True, 2.0, None)])
def test_one_position_a_token(plan):
    freqs, interleaved, scale = plan
    assert freqs is plan.freqs and interleaved is plan.interleaved and scale is plan.scale and plan.axes is None
    assert plan._fields == ("freqs", "interleaved", "scale") and isinstance(plan, (tuple, Rotary))
    again = Rotary(*plan)
    assert type(again) is type(plan) and again.freqs is freqs and again[1:] == plan[1:]
    assert repr(plan).startswith("Rotary(freqs=")
    for other in (copy.copy(plan), copy.deepcopy(plan), pickle.loads(pickle.dumps(plan)), plan._replace(scale=3.0)):
        assert type(other) is type(plan) and torch.equal(other.freqs, freqs) and other.interleaved is interleaved and other.axes is None
    with pytest.raises((TypeError, ValueError)):
        plan._replace(nothing=1)


def test_several_axes():
    """... and one of several axes has them beside those."""
    axes = [0, 1, 2, 0] * 4
    plan = rotary_plan(32, axes=axes, device="cpu")
    for other in (plan, copy.copy(plan), pickle.loads(pickle.dumps(plan)), plan._replace(scale=3.0), type(plan)(*plan),
                  Rotary(plan.freqs, plan.interleaved, plan.scale, plan.axes), Rotary(plan.freqs, axes=plan.axes),
                  rotary_plan(32, device="cpu")._replace(axes=plan.axes), torch.utils._pytree.tree_map(lambda x: x, plan)):
        assert other.axes.tolist() == axes and torch.equal(other.freqs, plan.freqs) and other.interleaved is False
    assert plan._replace(scale=3.0).scale == 3.0 and plan._replace(axes=None).axes is None
