"""GPU: cores with rotary positions (args.rotary) against the oracle, and trained by FusedMuon. Tolerances are those of the same comparisons without the rotation
(test_gpu_parity.py): it adds one bf16 rounding of q and k to the projection's own."""
import math

import numpy as np
import pytest
import torch

import v1t_amd
from oracle import v1t_oracle as O
from oracle import weights as W
from tests.helpers import assert_close, check_rel
from v1t_amd.synthetic import default_args, make_ds

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Y_RTOL, Y_ATOL, G_TOL = 1e-3, 1e-6, 1.2e-2


def build(cfg, sd, **more):
    args = default_args(
        input_shape=cfg.input_shape, resize_image=0, num_blocks=cfg.num_blocks, emb_dim=cfg.emb_dim, mlp_dim=cfg.mlp_dim, num_heads=cfg.num_heads,
        behavior_mode=cfg.behavior_mode, use_lsa=cfg.use_lsa, patch_stride=cfg.patch_stride, p_dropout=cfg.p_dropout, t_dropout=cfg.t_dropout,
        core=cfg.core, pos_emb=cfg.pos_emb, rotary=cfg.rotary, rotary_base=cfg.rotary_base, **more)
    args.output_shapes = {m: (cfg.num_neurons[m],) for m in cfg.mouse_ids}
    model = v1t_amd.Model(args, make_ds(cfg.num_neurons))
    r = model.load_state_dict(sd, strict=False)
    assert not r.unexpected_keys and set(r.missing_keys) <= {"image_cropper.grid", "elu1.one"}, r
    return model.to(DEV), args


def forward(model, batch, mouse="A", **kw):
    b = {k: v.to(DEV) for k, v in batch.items()}
    return model(inputs=b["image"], mouse_id=mouse, behaviors=b["behavior"], pupil_centers=b["pupil_center"], **kw)[0]


def config(**over):
    return O.Config(**{**dict(num_blocks=2, emb_dim=64, mlp_dim=96, num_heads=2, mouse_ids=("A",), num_neurons={"A": 64}, p_dropout=0.0, t_dropout=0.0, rotary=True), **over})


CASES = {
    "head64": config(), "head155": config(emb_dim=155, patch_stride=2, num_heads=4), "head33": config(emb_dim=33, num_heads=1, patch_stride=2),
    "base": config(patch_stride=2, rotary_base=10000.0),
    "cct": config(core="cct", emb_dim=160, num_heads=4, patch_stride=1), "cct_alone": config(core="cct", emb_dim=160, num_heads=4, pos_emb="none"),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_core_against_the_oracle(name):
    from v1t_amd.losses import elu1_poisson_loss

    cfg, B = CASES[name], 2
    sd = W.make_state_dict(cfg, 77)
    batch = W.make_batch(cfg, "A", B, 77)
    model, _ = build(cfg, sd)
    model.train(False)
    u = forward(model, batch, activate=False)
    loss, _ = elu1_poisson_loss(u, batch["response"].to(DEV), 4500.0, B)
    loss.backward()
    sdd = {k: (v.clone().requires_grad_(True) if v.is_floating_point() else v) for k, v in sd.items()}
    want, _, y = O.total_loss(cfg, sdd, batch, "A", 4500.0)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-4 * abs(float(want.detach()))
    with torch.no_grad():
        assert_close(f"rotary.{name}.y", forward(model, batch).cpu().numpy(), y.detach().numpy(), Y_RTOL, Y_ATOL)
    n = 0
    for k, p in model.named_parameters():
        ref = sdd[k].grad if k in sdd else None
        if ref is None or p.grad is None or float(ref.abs().max()) == 0.0:
            continue
        check_rel(f"rotary.{name}.grad.{k}", p.grad.detach().cpu().reshape(ref.shape), ref, G_TOL)
        n += 1
    assert n >= 20


def test_it_matters_and_off_is_off():
    """The rotation changes the prediction; a core built without it is bit for bit what it was, also beside one with it."""
    cfg = config(patch_stride=2)
    sd = {k: (v * 8 if "qkv" in k else v) for k, v in W.make_state_dict(cfg, 5).items()}
    batch = W.make_batch(cfg, "A", 2, 5)
    with torch.no_grad():
        on = forward(build(cfg, sd)[0].train(False), batch)
        plain = O.Config(**{**cfg.__dict__, "rotary": False})
        off_model = build(plain, sd)[0].train(False)
        off = forward(off_model, batch)
        forward(build(cfg, sd)[0].train(False), batch)
        assert torch.equal(forward(off_model, batch), off)
    assert float((on - off).abs().max()) > 1e-3 * float(off.abs().max())
    assert not off_model.core.rotary


def test_kept_probabilities_are_the_turned_ones():
    """What the rollout reads: the probabilities of the last forward's q and k, against the oracle's record."""
    from v1t_amd.rollout import attention_probabilities

    cfg = config(patch_stride=2)
    sd = W.make_state_dict(cfg, 6)
    batch = W.make_batch(cfg, "A", 2, 6)
    model, _ = build(cfg, sd)
    model.train(False)
    record = []
    with torch.no_grad():
        O.vit_tokens(cfg, sd, batch["image"], "A", batch["behavior"], batch["pupil_center"], record=record)
        b = {k: v.to(DEV) for k, v in batch.items()}
        got = attention_probabilities(model.core, b["image"], b["behavior"], b["pupil_center"], "A")
    want = torch.stack(record, dim=1)
    assert_close("rotary.probabilities", got.cpu().reshape(want.shape).numpy(), want.numpy(), 1e-2, 1e-5)


def trainer(cfg, sd, native=True, **more):
    from v1t_amd.trainer import Trainer

    model, args = build(cfg, sd, **more)
    args.batch_size = 4
    tr = Trainer(args, model, make_ds(cfg.num_neurons))
    tr.native = native
    return tr, model


def batches(cfg, seed):
    return {m: {k: v.to(DEV) for k, v in W.make_batch(cfg, m, 4, seed).items()} for m in cfg.mouse_ids}


MICE = dict(mouse_ids=("A", "B"), num_neurons={"A": 64, "B": 50}, patch_stride=2)


@pytest.mark.parametrize("name", ["vit", "cct"])
def test_trained_together(name):
    """A rotary core stepped by FusedMuon through the Trainer: each step's core matrices against the momentum step in 64 bits on the gradients that the step had, everything
    else against AdamW's; the loss stays finite."""
    cfg = config(**MICE) if name == "vit" else config(core="cct", emb_dim=160, num_heads=4, pos_emb="none", **{k: v for k, v in MICE.items() if k != "patch_stride"})
    tr, model = trainer(cfg, W.make_state_dict(cfg, 8), optimizer="muon", muon_lr=0.01)
    opt, core = tr.opt, model.core
    assert isinstance(opt, v1t_amd.FusedMuon)
    seen = {}
    step = opt.step_arena

    def watched(arena, ranges, zero_grad=True):
        if arena is core._arena:
            seen["g"], seen["p"] = arena.grad.clone(), arena.data.clone()
            m, v = arena.moments()
            seen["m"], seen["v"], seen["ranges"] = m.clone(), v.clone(), list(ranges)
        return step(arena, ranges, zero_grad)

    opt.step_arena = watched
    for n in range(3):
        out = tr.train_step(batches(cfg, 20 + n))
        assert math.isfinite(float(out["loss"]))
        arena = core._arena
        ((start, size, l1, lr),) = seen["ranges"]
        assert (start, size) == (0, arena.param_floats) and l1 == 2 * float(core.reg_scale) and lr == tr.core_lr  # once per mouse
        adam = torch.ones(arena.param_floats, dtype=torch.bool, device=DEV)
        assert len(opt.matrices()) == 12
        for off, rows, cols in opt.matrices():
            part = slice(off, off + rows * cols)
            adam[part] = False
            p, g, m = (seen[k][part].view(rows, cols).double() for k in "pgm")
            g = g + l1 * torch.sign(p)
            m = 0.95 * m + g
            x = g + 0.95 * m
            flip, x = rows > cols, x / (x.norm() + 1e-7)
            x = x.t() if flip else x
            for _ in range(5):
                s = x @ x.t()
                x = 3.4445 * x + (-4.7750 * s + 2.0315 * s @ s) @ x
            o = x.t() if flip else x
            scale = 0.01 * math.sqrt(max(1.0, rows / cols))
            size_o = float(o.norm()) / math.sqrt(o.numel())
            assert float((arena.exp_avg[part].view(rows, cols).double() - m).abs().max()) <= 4e-6 * float(m.abs().max())
            # the rounding of p, and the update within 2e-3 of its root mean square: few samples leave singular values near zero, where fp32 itself is off
            off_by = (arena.data[part].view(rows, cols).double() - (p - scale * o)).abs()
            assert bool((off_by <= 2**-23 * p.abs() + 2e-3 * scale * size_o).all())
            assert bool((arena.exp_avg_sq[part] == 0).all())
        p, g, m, v = (seen[k][:arena.param_floats][adam].double() for k in "pgmv")
        b1, b2 = opt.betas
        g = g + l1 * torch.sign(p)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        want = p - lr * (m / (1 - b1 ** (n + 1))) / ((v / (1 - b2 ** (n + 1))).sqrt() + opt.eps)
        assert torch.allclose(arena.data[:arena.param_floats][adam].double(), want, rtol=1e-5, atol=1e-3 * lr)
        assert bool((arena.grad[:arena.param_floats] == 0).all())


def test_native_step_equals_autograd_step():
    """The native step and the autograd path of the same rotary core and optimizer."""
    cfg = config(**MICE)
    sd = W.make_state_dict(cfg, 9)
    after = []
    for native in (True, False):
        tr, model = trainer(cfg, sd, native, optimizer="muon")
        tr.eps_override = {m: torch.zeros(4, cfg.num_neurons[m], 2, device=DEV) for m in cfg.mouse_ids}
        if not native:
            for m in cfg.mouse_ids:
                ro = model.readouts[m]
                orig = ro.forward
                ro.forward = (lambda inputs, sample=None, shifts=None, eps=None, _o=orig, _e=tr.eps_override[m]: _o(inputs, sample=sample, shifts=shifts, eps=_e))
        tr.train_step(batches(cfg, 30))
        assert (tr.last_step_path == "native") == native
        after.append(model.core._arena.exp_avg.clone())
    # the momentum is the gradient on the first step: float atomics and launch order apart, the same
    for off, rows, cols in tr.opt.matrices():
        a, b = (x[off:off + rows * cols] for x in after)
        assert float((a - b).abs().max()) <= 1e-2 * float(b.abs().max())


def test_reference_loop_and_checkpoint(tmp_path):
    """FusedMuon.for_model in a loop of one's own: step / zero_grad, a checkpoint written and read back, the next step the same."""
    from v1t_amd import checkpoint

    cfg = config(**MICE)
    sd = W.make_state_dict(cfg, 10)

    def run(model, opt, seed):
        model.train(True)
        for m, b in batches(cfg, seed).items():
            y = model(inputs=b["image"], mouse_id=m, behaviors=b["behavior"], pupil_centers=b["pupil_center"])[0]
            (y - b["response"]).square().mean().backward()
        opt.step()
        opt.zero_grad()

    model, _ = build(cfg, sd)
    opt = v1t_amd.FusedMuon.for_model(model, lr=1e-3, core_lr=2e-3, muon_lr=0.05)
    run(model, opt, 1)
    checkpoint.write(str(tmp_path), model, opt, epoch=1, value=0.5)
    other, _ = build(cfg, sd)
    again = v1t_amd.FusedMuon.for_model(other, lr=1e-3, core_lr=2e-3, muon_lr=0.05)
    checkpoint.read(str(tmp_path), other, again)
    a, b = model.core._arena, other.core._arena
    assert torch.equal(a.data, b.data) and torch.equal(a.exp_avg, b.exp_avg) and a.step == b.step == 1
    g = torch.randn(a.total, device=DEV)
    for arena, o in ((a, opt), (b, again)):
        arena.attach_grads(force=True)
        arena.grad.copy_(g)
        o.step_arena(arena, [(0, arena.param_floats, 0.0, 2e-3)])
    assert torch.equal(a.data, b.data)
    plain = v1t_amd.FusedAdamW.for_model(other, lr=1e-3)
    with pytest.raises(ValueError, match="other optimizer"):
        checkpoint.read(str(tmp_path), other, plain)


def test_frozen_core_is_not_stepped():
    cfg = config(**MICE)
    model, _ = build(cfg, W.make_state_dict(cfg, 11))
    model.core.freeze()
    opt = v1t_amd.FusedMuon.for_model(model, lr=1e-3)
    before = model.core._arena.data.clone() if model.core._arena.data is not None else None
    model.train(True)
    for m, b in batches(cfg, 2).items():
        model(inputs=b["image"], mouse_id=m, behaviors=b["behavior"], pupil_centers=b["pupil_center"])[0].square().mean().backward()
    before = model.core._arena.data.clone() if before is None else before
    opt.step()
    assert torch.equal(model.core._arena.data, before)
