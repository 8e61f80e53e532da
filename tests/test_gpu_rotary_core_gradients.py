"""GPU: every parameter's gradient through cores with rotary positions against the oracle, under the three bounds of the other gradient checks (largest error, 2-norm, cosine): an
angle's sign, a pair or an axis that is wrong in the backward pass moves all entries a little, and the largest one need not tell."""
import pytest
import torch

import v1t_amd
from oracle import v1t_oracle as O
from oracle import weights as W
from tests.helpers import check_grad
from v1t_amd.losses import elu1_poisson_loss
from v1t_amd.synthetic import default_args, make_ds

pytestmark = pytest.mark.gpu
DEV, G_TOL = "cuda:0", 1.2e-2


def config(**over):
    return O.Config(**{**dict(num_blocks=2, emb_dim=64, mlp_dim=96, num_heads=2, mouse_ids=("A",), num_neurons={"A": 64}, p_dropout=0.0, t_dropout=0.0, rotary=True), **over})


CASES = {
    "head64": config(), "head155": config(emb_dim=155, patch_stride=2, num_heads=4), "head33": config(emb_dim=33, num_heads=1, patch_stride=2),
    "base": config(patch_stride=2, rotary_base=10000.0), "cct": config(core="cct", emb_dim=160, num_heads=4, patch_stride=1),
    "cct_alone": config(core="cct", emb_dim=160, num_heads=4, pos_emb="none"),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_gradients(name):
    cfg = CASES[name]
    sd, batch = W.make_state_dict(cfg, 78), W.make_batch(cfg, "A", 2, 78)
    args = default_args(
        input_shape=cfg.input_shape, resize_image=0, num_blocks=cfg.num_blocks, emb_dim=cfg.emb_dim, mlp_dim=cfg.mlp_dim, num_heads=cfg.num_heads,
        behavior_mode=cfg.behavior_mode, patch_stride=cfg.patch_stride, p_dropout=0.0, t_dropout=0.0, core=cfg.core, pos_emb=cfg.pos_emb, rotary=True, rotary_base=cfg.rotary_base)
    args.output_shapes = {"A": (64,)}
    model = v1t_amd.Model(args, make_ds(cfg.num_neurons))
    model.load_state_dict(sd, strict=False)
    model = model.to(DEV).train(False)
    b = {k: v.to(DEV) for k, v in batch.items()}
    u = model(inputs=b["image"], mouse_id="A", behaviors=b["behavior"], pupil_centers=b["pupil_center"], activate=False)[0]
    elu1_poisson_loss(u, b["response"], 4500.0, 2)[0].backward()
    sdd = {k: (v.clone().requires_grad_(True) if v.is_floating_point() else v) for k, v in sd.items()}
    O.total_loss(cfg, sdd, batch, "A", 4500.0)[0].backward()
    n = 0
    for k, p in model.named_parameters():
        ref = sdd[k].grad if k in sdd else None
        if ref is None or p.grad is None or float(ref.abs().max()) == 0.0:
            continue
        check_grad(f"rotary gradients.{name}.{k}", p.grad.detach().cpu().reshape(ref.shape), ref, G_TOL)
        n += "qkv" in k or "to_q" in k
    assert n >= 2
