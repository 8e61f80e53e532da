"""GPU: the readout's gradient with respect to the core's map is summed in a fixed order - the same bits in every pass - and so is everything that the core's backward makes of it
before the first atomic."""
import numpy as np
import pytest
import torch

from oracle import weights as W
from tests.helpers import build_native_model, check_rel_bulk
from v1t_amd import lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def taps(grid, h, w):
    """The kernels' cells and weights, operation by operation in 32 bits: (B, N, 4) each; a tap outside the map has the cell h * w. The compiler may take
    px - floor(px) = X (w - 1) - floor(px) as one fused operation, without px's own rounding: half a step of a number below w, w 2^-24. A weight, the product of two numbers of at
    most one, is off by at most (w + h) 2^-24."""
    px, py = (grid[..., 0] + 1) * 0.5 * (w - 1), (grid[..., 1] + 1) * 0.5 * (h - 1)
    fx, fy = px.floor(), py.floor()
    ax, ay = px - fx, py - fy
    cell, wt = [], []
    for k in range(4):
        x, y = fx.long() + (k & 1), fy.long() + (k >> 1)
        inside = (x >= 0) & (x < w) & (y >= 0) & (y < h)
        cell.append(torch.where(inside, y * w + x, h * w))
        wt.append((ax if k & 1 else 1 - ax) * (ay if k >> 1 else 1 - ay) * inside)
    return torch.stack(cell, -1), torch.stack(wt, -1)


def places(kind, B, N, h, w, g):
    at = torch.rand(B, N, 2, generator=g, device=DEV) * 2.2 - 1.1  # some outside
    if kind == "one":      # every neuron between the same four cells
        at = 0.31 + 1e-3 * at
    elif kind == "few":    # a third of them on a few spots each
        spots = torch.rand(5, 2, generator=g, device=DEV) * 1.8 - 0.9
        at[:, ::3] = spots[torch.randint(0, 5, (at[:, ::3].shape[1],), generator=g, device=DEV)] + 1e-4 * at[:, ::3]
    elif kind == "nowhere":
        at += 9.0
    return at


@pytest.mark.parametrize("B,C,h,w,N", [(2, 155, 29, 57, 8000), (1, 1, 1, 1, 1), (3, 64, 5, 7, 15), (2, 65, 3, 2, 16), (1, 160, 64, 64, 333), (2, 256, 4, 4, 2049), (1, 40, 15, 29, 9001),
                                       (33, 63, 2, 3, 7), (1, 155, 29, 57, 20000)])
@pytest.mark.parametrize("kind", ["spread", "one", "few", "nowhere"])
def test_the_same_sum_every_time(B, C, h, w, N, kind):
    lib, g = L.load(), torch.Generator(device=DEV).manual_seed(N + C)
    FS, DP = (C + 31) // 32 * 32, C + 5  # rows of the map with numbers behind their channels
    grid, gout = places(kind, B, N, h, w, g), torch.randn(B, N, generator=g, device=DEV)
    feat, z = torch.randn(N, FS, generator=g, device=DEV), torch.randn(B, h * w, DP, generator=g, device=DEV)
    start = torch.randn(B, h * w, DP, generator=g, device=DEV)
    dgrid, dfeat, dbias = torch.empty_like(grid), torch.zeros_like(feat), torch.zeros(N, device=DEV)
    nbytes = lib.v1t_gaussian2d_backward_ws_bytes(B, h, w, N)
    got = []
    for i in range(4):
        dz = start.clone()
        ws = torch.full((nbytes,), (0, 255, 85, 1)[i], dtype=torch.uint8, device=DEV)  # nothing of it may be read before it is written
        for parts in ((7,), (7,), (1, 4, 2), (1, 2, 4))[i]:
            L.check(lib.v1t_gaussian2d_backward_parts(z.data_ptr(), h * w * DP, DP, B, C, h, w, N, grid.data_ptr(), feat.data_ptr(), FS, gout.data_ptr(), dz.data_ptr(), h * w * DP, DP,
                                                      dgrid.data_ptr(), dfeat.data_ptr(), dbias.data_ptr(), ws.data_ptr(), nbytes, parts, L.stream()))
        got.append(dz)
    assert all(torch.equal(got[0], x) for x in got)
    assert torch.equal(got[0][:, :, C:], start[:, :, C:])
    cell, wt = taps(grid, h, w)
    want, size, n = start[:, :, :C].double(), start[:, :, :C].double().abs(), torch.zeros(B, h * w + 1, device=DEV, dtype=torch.float64)
    loose = torch.zeros_like(want)
    for b in range(B):
        to = torch.zeros(3, h * w + 1, C, dtype=torch.float64, device=DEV)
        for k in range(4):
            t = (wt[b, :, k].double() * gout[b].double())[:, None] * feat[:, :C].double()
            to[0].index_add_(0, cell[b, :, k], t)
            to[1].index_add_(0, cell[b, :, k], t.abs())
            to[2].index_add_(0, cell[b, :, k], gout[b].double().abs()[:, None] * feat[:, :C].double().abs())
            n[b].index_add_(0, cell[b, :, k], torch.ones(N, dtype=torch.float64, device=DEV))
        want[b] += to[0, :-1]
        size[b] += to[1, :-1]
        loose[b] = to[2, :-1]
    # n products of three factors and n + 1 sums, each rounded once, of what the terms' sizes add up to; and the weights' own error
    off = (got[0][:, :, :C].double() - want).abs()
    assert bool((off <= (n[:, :-1, None] + 4) * 2**-24 * size + (h + w) * 2**-24 * loose).all())


@pytest.mark.parametrize("sd", ["fresh", "sharp"])
def test_a_backward_pass_repeats_itself(sd):
    """The default core under 8000 neurons, fresh and with the outlier channels of trained weights: d loss / d image, behind every block's bf16 roundings, is the same in eight
    passes. Parameter gradients end in fp32 atomics: their last bits differ, and no more."""
    from v1t_amd.losses import elu1_poisson_loss

    cfg = W.config_c2({"A": 8000})
    state = (W.make_state_dict if sd == "fresh" else W.make_sharp_state_dict)(cfg, 1234)
    batch = {k: v.to(DEV) for k, v in W.make_batch(cfg, "A", 2, 1234).items()}
    model, _ = build_native_model(cfg, state, torch.device(DEV))
    model.train(False)

    def run():
        model.zero_grad(set_to_none=True)
        image = batch["image"].clone().requires_grad_()
        u = model(inputs=image, mouse_id="A", behaviors=batch["behavior"], pupil_centers=batch["pupil_center"], activate=False)[0]
        loss, _ = elu1_poisson_loss(u, batch["response"], 4500.0, 2)
        (loss + model.regularizer("A")).backward()
        return image.grad, {k: p.grad.detach().clone() for k, p in model.named_parameters() if p.grad is not None}

    image, grads = run()
    assert float(image.abs().max()) > 0 and len(grads) > 20
    for i in range(7):
        again, others = run()
        assert torch.equal(again, image), i
        for k in grads:
            check_rel_bulk(f"pass {i} repeats the first: {k} [{sd}]", others[k], grads[k], 1e-5, 1e-4)
