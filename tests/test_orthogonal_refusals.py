"""CPU: what the orthogonalisation and the momentum step refuse, before any launch."""
import ctypes as C
import math

import pytest
import torch

import v1t_amd
from v1t_amd import lib as L

U = torch.zeros(4, 6)


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(updates=torch.zeros(3))), (ValueError, dict(updates=torch.zeros(1, 2, 3, 4))), (ValueError, dict(updates=[U, torch.zeros(3)])),
    (TypeError, dict(updates=U.double())), (TypeError, dict(updates=[U, U.bfloat16()])), (ValueError, dict(steps=-1)), (ValueError, dict(steps=33)),
    (ValueError, dict(coefficients=(1.0, 2.0))), (ValueError, dict(coefficients=[(1.0, 2.0, 3.0)] * 2)), (ValueError, dict(eps=-1.0)),
    (ValueError, dict(eps=math.nan)), (ValueError, dict(eps=math.inf)), (RuntimeError, dict(updates=U.clone().requires_grad_())),
    (RuntimeError, dict()),  # nothing wrong but the device
])
def test_orthogonalize_refusals(error, change):
    arguments = dict(updates=U) | change
    with pytest.raises(error):
        v1t_amd.orthogonalize(arguments.pop("updates"), **arguments)


def test_sizes_that_do_not_fit_32_bits():
    """2^32 + 5 columns are not 5."""
    wide = torch.zeros(1).expand(1, 2**32 + 5)
    with pytest.raises(ValueError, match="at most"):
        v1t_amd.orthogonalize(wide)
    wide = torch.empty(1, 2**32 + 5, device="meta")
    with pytest.raises(ValueError, match="at most"):
        v1t_amd.muon_step([wide], [wide], [wide], lr=0.1)
    from v1t_amd import muon

    for shape in ((40000, 40000), (1, 2**22 + 1), (2**31, 2), (2**16, 2**15 + 1)):
        with pytest.raises(ValueError, match="at most"):
            muon._workspace_bytes((shape,))


def test_nothing_to_do():
    assert v1t_amd.orthogonalize([]) == []
    v1t_amd.muon_step([], [], [], lr=0.1)
    empty = torch.zeros(0, 3)
    v1t_amd.muon_step([empty], [empty.clone()], [empty.clone()], lr=0.1)


def three(shape=(4, 6)):
    return [torch.zeros(shape) for _ in range(3)]


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(grads=[])), (ValueError, dict(lr=[0.1, 0.2])), (ValueError, dict(lr=math.nan)), (ValueError, dict(momentum=math.inf)),
    (ValueError, dict(weight_decay=math.nan)), (ValueError, dict(l1=math.nan)), (ValueError, dict(eps=-1e-3)), (ValueError, dict(steps=40)),
    (ValueError, dict(params=[torch.zeros(6)])), (TypeError, dict(grads=[torch.zeros(4, 6).double()])), (ValueError, dict(moments=[torch.zeros(6, 4)])),
    (ValueError, dict(moments=[torch.zeros(6, 4).t()])), (RuntimeError, dict()),
])
def test_muon_step_refusals(error, change):
    p, g, m = three()
    arguments = dict(params=[p], grads=[g], moments=[m], lr=0.1) | change
    with pytest.raises(error):
        v1t_amd.muon_step(**arguments)


def test_muon_step_refuses_shared_memory():
    p, g, m = three()
    buffer = torch.zeros(60)
    for params, grads, moments in (([p], [p], [m]), ([p], [g], [g]), ([p, p], [g, g.clone()], [m, m.clone()]),
                                   ([buffer[:24].view(4, 6)], [g], [buffer[20:44].view(4, 6)])):
        with pytest.raises(ValueError, match="share memory"):
            v1t_amd.muon_step(params, grads, moments, lr=0.1)


def ints(*v):
    return (C.c_int * len(v))(*v)


def test_c_entry_refusals():
    lib = L.load()
    size = lib.v1t_orthogonalize_ws_bytes
    assert size(ints(400, 700), ints(600, 500), 2) > size(ints(400), ints(600), 1) > size(ints(4), ints(6), 1) > 0
    assert size(None, None, 0) >= 0 and size(None, None, 1) == -1 and size(ints(4), ints(6), -1) == -1
    assert size(ints(0), ints(6), 1) == -1 and size(ints(4), ints(-6), 1) == -1
    assert size(ints(40000), ints(40000), 1) == -2 and size(ints(1), ints(1 << 23), 1) == -2
    units = (L.Matrix * 1)(L.Matrix(4096, 4096, 6, 1, 4, 6))  # never dereferenced: every call below is refused
    co = (C.c_float * 3)(3.4445, -4.775, 2.0315)

    def call(units=units, n=1, dtype=2, steps=1, co=co, eps=1e-7, ws=4096, ws_bytes=1 << 30):
        return lib.v1t_orthogonalize(units, n, dtype, steps, co, eps, ws, ws_bytes, None)

    bad = [dict(units=None), dict(n=-1), dict(dtype=3), dict(dtype=-1), dict(steps=-1), dict(steps=33), dict(co=None), dict(eps=-1.0), dict(eps=math.nan),
           dict(ws=4097), dict(co=(C.c_float * 3)(math.nan, 0, 0)), dict(co=(C.c_float * 3)(200.0, 0, 0)), dict(co=(C.c_float * 3)(0, 0, 130.0)),
           dict(steps=3, co=(C.c_float * 9)(6, 0, 0, 6, 0, 0, 6, 0, 0)), dict(units=(L.Matrix * 1)(L.Matrix(None, 4096, 6, 1, 4, 6))),
           dict(units=(L.Matrix * 1)(L.Matrix(4096, None, 6, 1, 4, 6))), dict(units=(L.Matrix * 1)(L.Matrix(4096, 4096, 6, 1, 0, 6)))]
    for change in bad:
        assert call(**change) == -1, change
    assert call(ws=None) == -4 and call(ws_bytes=64) == -4
    assert call(n=0) == 0
    ranges = (L.MuonRange * 1)(L.MuonRange(4096, 4096, 4096, 4, 6, 0.1, 1.0, 0.0, 0))

    def step(units=ranges, n=1, momentum=0.9, steps=1, co=co, eps=1e-7, ws=4096, ws_bytes=1 << 30):
        return lib.v1t_muon_step(units, n, momentum, 1, steps, co, eps, 0, ws, ws_bytes, None)

    for change in (dict(units=None), dict(n=-1), dict(momentum=math.nan), dict(steps=33), dict(co=None), dict(eps=-1.0),
                   dict(units=(L.MuonRange * 1)(L.MuonRange(None, 4096, 4096, 4, 6, 0.1, 1.0, 0.0, 0)))):
        assert step(**change) == -1, change
    assert step(ws_bytes=64) == -4 and step(n=0) == 0


def test_coefficients_that_grow_are_refused_by_name():
    # numbers that stay below 128 (the default ones, plain cubic steps) pass the check; the bound is over all singular values in [0, 1]
    lib = L.load()
    units = (L.Matrix * 1)(L.Matrix(4096, 4096, 6, 1, 4, 6))
    for ok in ((3.4445, -4.775, 2.0315), (1.5, -0.5, 0.0), (1.0, 0.0, 0.0)):
        assert lib.v1t_orthogonalize(units, 1, 2, 5, (C.c_float * 15)(*(ok * 5)), 1e-7, None, 0, None) == -4  # past the check: no workspace


def small(**over):
    from v1t_amd.synthetic import sensorium_config

    args, ds = sensorium_config({"A": 10}, **{**dict(input_shape=(1, 36, 64), resize_image=0, num_blocks=1, emb_dim=64, mlp_dim=128), **over})
    return v1t_amd.Model(args, ds), args, ds


def test_fused_muon_refusals():
    from v1t_amd.trainer import Trainer

    model, args, ds = small()
    with pytest.raises(ValueError, match="positive"):
        v1t_amd.FusedMuon.for_model(model, lr=1e-3, core_lr=0.0)
    with pytest.raises(ValueError, match="finite"):
        v1t_amd.FusedMuon.for_model(model, lr=1e-3, muon_lr=math.nan)
    with pytest.raises(ValueError, match="steps"):
        v1t_amd.FusedMuon.for_model(model, lr=1e-3, steps=99)
    args.optimizer = "lamb"
    with pytest.raises(NotImplementedError, match="lamb"):
        Trainer(args, model, ds)
    muon = v1t_amd.FusedMuon.for_model(model, lr=1e-3)
    adam = v1t_amd.FusedAdamW.for_model(model, lr=1e-3)
    for a, b in ((muon, adam), (adam, muon)):
        with pytest.raises(ValueError, match="other optimizer"):
            a.load_state_dict(b.state_dict())
    # every attention and MLP matrix of the core, q, k and v apart; no table, no BehaviorMLP
    assert [(r, c) for _, r, c in muon.matrices()] == [(256, 64)] * 3 + [(64, 256), (128, 64), (64, 128)]


def test_fused_muon_restores_its_rates():
    """The matrices' rate is muon_lr where the core's is core_lr, also for an optimizer that was made with other rates than its checkpoint's."""
    model, _, _ = small()
    saved = v1t_amd.FusedMuon.for_model(model, lr=1e-3, core_lr=2e-3, muon_lr=0.05)
    saved.param_groups[[g["name"] for g in saved.param_groups].index("core")]["lr"] = 5e-4  # a scheduler's quarter
    other = v1t_amd.FusedMuon.for_model(model, lr=1e-3, core_lr=1e-3, muon_lr=0.01)
    other.load_state_dict(saved.state_dict())
    (group,) = [g for g in other.param_groups if "muon" in g]
    assert group["name"] == "core" and group["lr"] == 5e-4 and group["muon"] == {"lr": 0.05, "core_lr": 2e-3}
    group["muon"]["lr"] = 1.0
    assert [g["muon"]["lr"] for g in saved.param_groups if "muon" in g] == [0.05]  # a copy


def test_rotary_core_refusals():
    with pytest.raises(ValueError, match="head dim 3"):
        small(rotary=True, emb_dim=3, num_heads=1)
    with pytest.raises(NotImplementedError, match="use_lsa"):
        small(rotary=True, use_lsa=True)
    with pytest.raises(ValueError, match="rotary_base"):
        small(rotary=True, rotary_base=-1.0)
    model, _, _ = small(rotary=True)
    at = model.core.rotary_positions()
    assert at.shape == (1654, 2) and at[0].tolist() == [0, 0] and at[1].tolist() == [0, 0] and at[58].tolist() == [1, 0] and at[-1].tolist() == [28, 56]
    lib = L.load()
    sections = ints(16, 16)
    for positions, sec, axes, base in ((4096, None, 2, 100.0), (4096, sections, 0, 100.0), (4096, sections, 5, 100.0), (4096, sections, 2, 0.0), (4096, sections, 2, math.nan),
                                       (4096, ints(17, 16), 2, 100.0), (4096, ints(-1, 3), 2, 100.0), (4096, ints(0, 0), 2, 100.0)):
        assert lib.v1t_vit_set_rotary(model.core._plan, positions, sec, axes, base) == -1
    assert lib.v1t_vit_set_rotary(None, 4096, sections, 2, 100.0) == -1
    assert lib.v1t_vit_set_rotary(model.core._plan, None, None, 0, 0.0) == 0
