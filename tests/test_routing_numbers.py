"""Arguments of the routing calls that are no plain numbers: read at every call, or refused with the package's error.  No GPU."""
import numpy as np
import pytest
import torch

from mgpt_b200 import MoeError, routing

HOW = dict(score="sigmoid", bias=None, groups=4, top_groups=2, group_top=2, renormalise=True, scale=1.5)


def _argument(**how):
    how = HOW | how
    return routing._routing(8, how["score"], how["bias"], how["groups"], how["top_groups"], how["group_top"], how["renormalise"], how["scale"], None)


def test_numbers_that_change_in_place():
    scale, groups, on = torch.tensor(2.0), np.array(4), torch.tensor(True)
    for value in (2.0, 3.0, -0.0, 0.0):
        scale.fill_(value)
        got = _argument(scale=scale).scale
        assert got == value and np.signbit(got) == np.signbit(value)
    for value in (4, 2):
        groups[...] = value
        r = _argument(groups=groups, top_groups=None)
        assert (r.groups, r.top_groups) == (value, value)
    for value in (True, False):
        on.fill_(value)
        assert _argument(renormalise=on).renormalise == value


@pytest.mark.parametrize("like", [dict(scale=np.float32(1.5)), dict(groups=np.int64(4)), dict(scale=torch.tensor(1.5)), dict(renormalise=1), dict(top_groups=np.int32(2))])
def test_numbers_of_other_types(like):
    assert bytes(_argument(**like)) == bytes(_argument())


@pytest.mark.parametrize("bad", [dict(groups=1.5), dict(groups=None), dict(top_groups=2.0), dict(group_top="2"), dict(scale=None), dict(scale="x"), dict(scale=[1.0]), dict(scale=10 ** 400),
                                 dict(scale=torch.zeros(2)), dict(renormalise=torch.zeros(2)), dict(score=None), dict(score=3), dict(score=["sigmoid"]), dict(groups=2 ** 40)])
def test_refusals(bad):
    with pytest.raises(MoeError):
        _argument(**bad)
