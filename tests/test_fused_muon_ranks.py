"""CPU: what a step of a data-parallel rank - the core and its mice in one call - sends to the kernels under FusedMuon, with the library replaced by a recorder."""
import math

import pytest
import torch

import v1t_amd
from v1t_amd import lib as L
from v1t_amd.synthetic import sensorium_config

LOAD = L.load


class Recorder:
    def __init__(self):
        self.adam, self.muon = [], []

    def v1t_adamw_multi(self, rs, n, *a):
        self.adam.append([(r.p, r.n, r.lr, r.l1, r.step) for r in rs[:n]])
        return 0

    def v1t_muon_step(self, rs, n, momentum, *a):
        self.muon.append([(r.p, r.g, r.m, r.rows, r.cols, r.lr, r.decay, r.l1) for r in rs[:n]])
        return 0

    def v1t_orthogonalize_ws_bytes(self, rows, cols, n):
        return 256


@pytest.fixture
def library(monkeypatch):
    recorder = Recorder()
    monkeypatch.setattr(L, "load", lambda: recorder)
    monkeypatch.setattr(L, "stream", lambda: 0)
    v1t_amd.muon._workspace_bytes.cache_clear()
    yield recorder
    v1t_amd.muon._workspace_bytes.cache_clear()


def step(library, together, l1=0.003):
    """One step of a rank with two mice: in one call, as behind an exchange of gradients, or the core alone and then its mice."""
    args, ds = sensorium_config({"A": 10, "B": 12}, input_shape=(1, 36, 64), resize_image=0, num_blocks=2, emb_dim=64, mlp_dim=128)
    torch.manual_seed(0)
    with pytest.MonkeyPatch.context() as real:  # the model's own plan is made by the library
        real.setattr(L, "load", LOAD)
        model = v1t_amd.Model(args, ds)
        opt = v1t_amd.FusedMuon.for_model(model, lr=1e-3, core_lr=2e-3, muon_lr=0.05, weight_decay=0.1)
        core = model.core._arena
        core.ensure()
        mice = []
        for m in ("A", "B"):
            a = model.mouse_arena(m)
            a.ensure()
            mice.append((a, [(o, n, c, opt.group_lr(g)) for o, n, c, g in model.mouse_step_ranges(m)]))
        opt.matrices()
    item = (core, [(0, core.param_floats, l1, opt.group_lr("core"))])
    if together:
        opt.step_arenas([item] + mice)
    else:
        opt.step_arena(*item)
        opt.step_arenas(mice)
    return model, opt, core, [a for a, _ in mice]


@pytest.mark.parametrize("together", [True, False])
def test_every_number_is_stepped_once(library, together):
    model, opt, core, mice = step(library, together)
    base = core.data.data_ptr()
    (matrices,) = library.muon
    rest, of_mice = library.adam
    spans = sorted([((p - base) // 4, rows * cols) for p, _, _, rows, cols, *_ in matrices] + [((p - base) // 4, n) for p, n, *_ in rest])
    end = 0
    for at, n in spans:
        assert at == end
        end += n
    assert end == core.param_floats
    assert [(((p - base) // 4), rows, cols) for p, _, _, rows, cols, *_ in matrices] == opt.matrices() and len(matrices) == 2 * 6
    m, _ = core.moments()
    for p, g, mom, rows, cols, lr, decay, l1 in matrices:
        assert g - core.grad.data_ptr() == mom - m.data_ptr() == p - base and l1 == pytest.approx(0.003)
        assert lr == pytest.approx(0.05 * math.sqrt(max(1.0, rows / cols)), rel=1e-6) and decay == pytest.approx(1 - 0.05 * 0.1, rel=1e-6)
    assert all(lr == pytest.approx(2e-3) and n == 1 for *_, lr, _, n in rest)
    ends = [(a.data.data_ptr(), a.data.data_ptr() + 4 * a.param_floats) for a in mice]
    assert sum(n for _, n, *_ in of_mice) == sum(a.param_floats for a in mice) and all(any(x <= p < y for x, y in ends) for p, *_ in of_mice)
    assert core.step == 1 and all(a.step == 1 for a in mice)


def test_both_ways_are_one(library):
    a = step(library, True)
    together = (library.muon, library.adam)
    library.muon, library.adam = [], []
    b = step(library, False)
    shift = lambda model, rows: [tuple(r[3:]) for r in rows]
    assert [shift(a, r) for r in together[0]] == [shift(b, r) for r in library.muon]
    assert [[tuple(r[1:]) for r in rs] for rs in together[1]] == [[tuple(r[1:]) for r in rs] for rs in library.adam]


def test_a_range_that_ends_inside_a_matrix_is_refused(library):
    _, opt, core, _ = step(library, True)
    off, rows, cols = opt.matrices()[1]
    with pytest.raises(RuntimeError, match="inside a matrix"):
        opt.step_arena(core, [(0, off + rows * cols // 2, 0.0, 2e-3)])
