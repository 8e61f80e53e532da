"""CPU: the rotary entry points' plain arguments, which are checked and converted once per value."""
import numpy as np
import pytest
import torch

import v1t_amd
from v1t_amd import lib as L
from v1t_amd import positions

Q, AT = torch.zeros(2, 5, 4, 16), torch.zeros(5, 2, dtype=torch.int32)


@pytest.fixture
def turns(monkeypatch):
    """What each launch would turn by."""
    seen = []
    monkeypatch.setattr(positions, "_launch", lambda turn, at, pairs: seen.append(turn))
    monkeypatch.setattr(L, "require_cuda", lambda *a: None)
    return seen


@pytest.mark.parametrize("call", ["rotary", "rotary_"])
@pytest.mark.parametrize("base", ["fp32", "numpy", "fp64"])
def test_a_base_that_changes_in_place(turns, call, base):
    """The rates are those of the base's value at the call."""
    base = {"fp32": torch.tensor(100.0), "numpy": np.array(100.0), "fp64": torch.tensor([100.0], dtype=torch.float64)}[base]
    getattr(v1t_amd, call)(Q, AT, sections=(3, 4), base=base)
    base.fill_(10000.0) if isinstance(base, torch.Tensor) else base.fill(10000.0)
    getattr(v1t_amd, call)(Q, AT, sections=(3, 4), base=base)
    assert [t.base for t in turns] == [100.0, 10000.0]


def test_flags_that_change_in_place(turns):
    flag = torch.tensor(False)
    v1t_amd.rotary(Q, AT, sections=(3, 4), shared=flag, inverse=flag)
    flag.fill_(True)
    v1t_amd.rotary(Q, AT, sections=(3, 4), shared=flag, inverse=flag)
    assert [(t.shared, t.inverse) for t in turns] == [(0, 0), (1, 1)]


def test_sections_of_any_kind(turns):
    for sections in ((3, 4), [3, 4], np.array([3, 4]), torch.tensor([3, 4])):
        v1t_amd.rotary(Q, AT, sections=sections)
    assert all(t is turns[0] and t.sections == (3, 4) for t in turns)


@pytest.mark.parametrize("layout", [["pairs"], {"pairs": 0}, None])
def test_a_layout_that_is_no_name(layout):
    with pytest.raises(ValueError, match="layout"):
        v1t_amd.rotary(Q, AT, sections=(3, 4), layout=layout)


def test_the_way_back(turns):
    """A backward pass turns by the same angles, negated; back again by the first ones."""
    for shared in (False, True):
        for layout in ("pairs", "halves"):
            there = positions._turn((3, 4), 50.0, layout, shared, False)
            back = positions._back(there)
            assert back._replace(inverse=0, array=None) == there._replace(array=None) and back.inverse == 1 and positions._back(back) is there
