"""GPU: the orthogonalised update and the momentum step against the formula in 64 bits.

Tolerance, of the 2-norm of the difference over that of the result: the kernel holds its operands to 22 bits and sums in fp32, where fp32 arithmetic holds both to 24. Its
roundings are at most four times those of the formula evaluated in fp32, whose own error is measured on the same input - it is what the input's small singular values make
of 2^-24 - and is zero by luck on the smallest ones: 15 products of 2^-22 each, four times over, are added (1.5e-5). A single value may be off by 64 times that of the root
mean square. Rounding the result to 16 bits adds half a step, eps / 2."""
import math

import pytest
import torch

import v1t_amd
from v1t_amd.muon import COEFFICIENTS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def formula(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=torch.float64):
    x = u.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = (x / (x.norm() + eps)).to(dtype)  # the norm in 64 bits: its square may leave fp32's range
    for k in range(steps):
        a, b, c = coefficients if isinstance(coefficients[0], float) else coefficients[k]
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if flip else x


def close(got, u, **kw):
    want = formula(u, **kw)
    norm = float(want.norm())
    if norm == 0:
        assert bool((got == 0).all())
        return
    plain = float((formula(u, dtype=torch.float32, **kw).double() - want).norm()) / norm
    allowed = 4 * plain + 15 * 4 * 2**-22
    off = got.double() - want
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    assert float(off.norm()) / norm <= allowed + half, (float(off.norm()) / norm, allowed, half)
    rms = norm / math.sqrt(want.numel())
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert bool((off.abs() <= 64 * allowed * rms + half * want.abs() * (1 + 64 * allowed) + tiny).all())


def update(rows, cols, seed=0, kind="gauss"):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + cols)
    if kind == "gauss":
        return torch.randn(rows, cols, device=DEV, generator=g)
    u = torch.randn(rows, 3, device=DEV, generator=g) @ torch.randn(3, cols, device=DEV, generator=g)  # a few strong directions over weak ones
    return u + 0.03 * torch.randn(rows, cols, device=DEV, generator=g)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (31, 33), (32, 32), (33, 31), (64, 155), (155, 64), (65, 64), (155, 620), (620, 155), (200, 200), (129, 257), (1, 1000), (1000, 1),
          (300, 1000), (128, 128), (97, 4096), (64, 448), (64, 449), (449, 60), (31, 1024), (1025, 32), (96, 192), (90, 193), (192, 96), (65, 160), (24, 500)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_matrix(rows, cols, dtype):
    u = update(rows, cols).to(dtype)
    before = u.clone()
    o = v1t_amd.orthogonalize(u)
    assert o.shape == u.shape and o.dtype == dtype and o.is_contiguous() and torch.equal(u, before)
    close(o, u)


@pytest.mark.parametrize("kind", ["gauss", "few"])
def test_a_list_of_all_shapes_is_each_alone(kind):
    """More units than one table launch holds, small and large ones mixed; the same bits every time."""
    us = [update(r, c, i, kind) for i in range(2) for r, c in SHAPES]
    for u, o in zip(us, v1t_amd.orthogonalize(us)):
        close(o, u)
    again = v1t_amd.orthogonalize(us)
    assert all(torch.equal(a, b) for a, b in zip(again, v1t_amd.orthogonalize(us)))


def test_large_tiles():
    us = [update(1100, 1203, i) for i in range(6)] + [update(1301, 700)]  # enough tiles for the larger ones
    for u, o in zip(us, v1t_amd.orthogonalize(us)):
        close(o, u)
    u = update(2950, 3010, 1, "few")
    close(v1t_amd.orthogonalize(u), u)


@pytest.mark.parametrize("count,rows,cols", [(1, 100, 20000), (1, 1600, 1660), (1, 1800, 1900), (4, 1300, 1300), (2, 1000, 1900), (1, 2300, 2360), (5, 1800, 1860), (1, 4001, 4100)])
def test_tiles_and_pieces(count, rows, cols):
    """Symmetric products in tiles of 64 in 16 pieces, of 64 with pieces beside whole ones, of 128 in pieces, of 128 with pieces beside, of two kinds, of 192 in pieces,
    of 192 with pieces behind whole ones, of 192 whole; the same bits every time."""
    us = [update(rows, cols, i) for i in range(count)]
    os = v1t_amd.orthogonalize(us)
    for u, o in zip(us, os):
        close(o, u)
    assert all(torch.equal(a, b) for a, b in zip(os, v1t_amd.orthogonalize(us)))


@pytest.mark.parametrize("rows,cols", [(700, 2900), (2900, 700), (1000, 8100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("steps", [1, 2, 4, 5])
def test_steps_in_pairs(rows, cols, dtype, steps):
    """Long matrices, whose steps go two at a time: one, two, two pairs, and a step left over."""
    u = update(rows, cols, kind="few").to(dtype)
    close(v1t_amd.orthogonalize(u, steps=steps), u, steps=steps)


def test_pairs_that_would_leave_the_planes_range():
    """12 * 12 at zero is more than a pair's matrix may hold: such steps go one by one, also where the sizes would have them in pairs."""
    u, co = update(700, 2900), [(12.0, -20.0, 9.0), (12.0, -2.0, 0.0)]
    close(v1t_amd.orthogonalize(u, steps=2, coefficients=co), u, steps=2, coefficients=co)
    close(v1t_amd.orthogonalize(u), u)  # and the usual ones again


def test_stack_strides_and_views():
    stack = torch.stack([update(40, 50, i) for i in range(5)])
    o = v1t_amd.orthogonalize(stack)
    assert o.shape == stack.shape and torch.equal(o, torch.stack(v1t_amd.orthogonalize(list(stack))))
    assert torch.equal(v1t_amd.orthogonalize(stack.transpose(0, 1).contiguous().transpose(0, 1)), o)
    big = update(90, 120)
    for view in (big.t(), big[::2, 1::3], big[3:50, 5:100], big[:1].expand(4, -1), big[:, :1].expand(-1, 5)):
        assert torch.equal(v1t_amd.orthogonalize(view), v1t_amd.orthogonalize(view.contiguous()))
        close(v1t_amd.orthogonalize(view), view)
    assert v1t_amd.orthogonalize(torch.zeros(0, 5, device=DEV)).shape == (0, 5)
    assert v1t_amd.orthogonalize(torch.zeros(0, 5, 4, device=DEV)).shape == (0, 5, 4)
    some = v1t_amd.orthogonalize([big, torch.zeros(3, 0, device=DEV)])
    assert some[1].shape == (3, 0) and torch.equal(some[0], v1t_amd.orthogonalize(big))


@pytest.mark.parametrize("steps,coefficients", [(0, COEFFICIENTS), (1, COEFFICIENTS), (2, COEFFICIENTS), (7, (1.5, -0.5, 0.0)), (3, [(3.0, -3.0, 1.0), (2.0, -1.0, 0.0), (1.0, 0.25, -0.25)])])
def test_other_steps_and_coefficients(steps, coefficients):
    for r, c in ((20, 30), (155, 100)):
        u = update(r, c)
        close(v1t_amd.orthogonalize(u, steps=steps, coefficients=coefficients), u, steps=steps, coefficients=coefficients)


def test_it_orthogonalises():
    """Singular values end where five steps take a value of at least 0.01 of the norm: between 0.65 and 1.25."""
    u = update(100, 260)
    s = torch.linalg.svdvals(v1t_amd.orthogonalize(u).double().cpu())
    assert 0.65 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4, 1e30])
def test_scale(scale):
    """Without eps the result does not depend on the update's scale, also where its square leaves fp32's range."""
    u = update(50, 70)
    o = v1t_amd.orthogonalize(u * scale, eps=0.0)
    close(o, u * scale, eps=0.0)


@pytest.mark.parametrize("rows,cols", [(50, 70), (20, 500), (90, 100), (155, 620), (400, 170), (700, 2900)])
@pytest.mark.parametrize("scale", [1e-9, 1e-11, 1e-15, 1e-25])
def test_eps_that_outweighs_the_norm(rows, cols, scale):
    """The iterate is a polynomial of a small number then, as exact as any other; beside a matrix of the usual size."""
    u = update(rows, cols)
    o, other = v1t_amd.orthogonalize([u * scale, u])
    close(o, u * scale)
    close(other, u)
    for steps, co in ((0, COEFFICIENTS), (1, COEFFICIENTS), (4, COEFFICIENTS), (3, [(0.5, 0.25, 0.25), (1.0, 0.0, -1.0), (8.0, -3.0, 0.0)])):
        close(v1t_amd.orthogonalize(u * scale, steps=steps, coefficients=co), u * scale, steps=steps, coefficients=co)


def test_zeros_nan_and_infinity_stay_in_their_matrix():
    us = [update(33, 40, i) for i in range(4)]
    clean = v1t_amd.orthogonalize(us)
    us[1] = torch.zeros(33, 40, device=DEV)
    us[2][5, 6] = math.nan
    us[3][5, 6] = math.inf
    o = v1t_amd.orthogonalize(us)
    assert torch.equal(o[0], clean[0]) and bool((o[1] == 0).all())
    assert bool(torch.isnan(o[2]).all()) and not bool(torch.isfinite(o[3]).any())
    assert bool(torch.isnan(v1t_amd.orthogonalize(torch.zeros(3, 4, device=DEV), eps=0.0)).all())  # 0 / 0


def test_what_lies_behind_the_result_is_untouched():
    """Results of odd sizes side by side in one buffer: the C entry, with guards between."""
    import ctypes as C
    from v1t_amd import lib as L

    lib, shapes = L.load(), [(33, 47), (47, 33), (5, 5)]
    us = [update(r, c) for r, c in shapes]
    buffer = torch.full((8000,), 7.0, device=DEV)
    offsets = [100, 2000, 4001]
    units = (L.Matrix * 3)(*[L.Matrix(u.data_ptr(), buffer.data_ptr() + 4 * o, u.shape[1], 1, *u.shape) for u, o in zip(us, offsets)])
    co = (C.c_float * 15)(*(COEFFICIENTS * 5))
    size = lib.v1t_orthogonalize_ws_bytes((C.c_int * 3)(33, 47, 5), (C.c_int * 3)(47, 33, 5), 3)
    ws = torch.full((size + 4096,), 255, dtype=torch.uint8, device=DEV)  # NaN everywhere: nothing of it may be read before it is written
    L.check(lib.v1t_orthogonalize(units, 3, 2, 5, co, 1e-7, ws.data_ptr(), size, L.stream()))
    kept = torch.ones(8000, dtype=torch.bool, device=DEV)
    for u, o in zip(us, offsets):
        close(buffer[o:o + u.numel()].view_as(u), u)
        kept[o:o + u.numel()] = False
    assert bool((buffer[kept] == 7.0).all()) and bool((ws[size:] == 255).all())


# ---- the momentum step
def reference_step(p, g, m, lr, mu, nesterov, decay, l1, **kw):
    """64 bits; the orthogonalised update as the kernel's own inputs make it"""
    p, g, m = p.double(), g.double(), m.double()
    g = g + l1 * torch.sign(p)
    m = mu * m + g
    u = g + mu * m if nesterov else m
    rows, cols = p.shape[0], p.numel() // p.shape[0]
    o = formula(u.reshape(rows, cols), **kw)
    return (1 - lr * decay) * p - lr * math.sqrt(max(1.0, rows / cols)) * o.view_as(p), m


def check_step(p, m, want_p, want_m, before, lr):
    """The momentum: three fp32 roundings. The parameter: its own rounding and the update's error, at most 2e-4 of the root mean square of a matrix whose singular
    values are near one (the bound above at the fp32 error of such updates, below 2e-6)."""
    assert bool(((m.double() - want_m).abs() <= 4 * 2**-24 * (want_m.abs() + before.abs() + 10)).all())
    rows, cols = p.shape[0], p.numel() // p.shape[0]
    size = lr * math.sqrt(max(1.0, rows / cols)) / math.sqrt(max(rows, cols))
    off = (p.double() - want_p).abs()
    assert bool((off <= 3 * 2**-24 * (want_p.abs() + 5 * size) + 64 * 2.5e-5 * size).all()), float(off.max() / size)


@pytest.mark.parametrize("nesterov,decay,l1", [(True, 0.0, 0.0), (True, 0.1, 0.003), (False, 0.1, 0.0)])
def test_muon_step(nesterov, decay, l1):
    shapes = [(155, 64), (64, 155), (155, 620), (3, 5), (16, 2, 3, 3), (130, 1)]
    gen = torch.Generator(device=DEV).manual_seed(3)
    ps, gs, ms = ([torch.randn(s, device=DEV, generator=gen) for s in shapes] for _ in range(3))
    ps[0][0] = 0.0  # sign(0) = 0
    lrs = [0.02 * (i + 1) for i in range(len(shapes))]
    want = [reference_step(p, g, m, lr, 0.9, nesterov, decay, l1) for p, g, m, lr in zip(ps, gs, ms, lrs)]
    kept, before = [g.clone() for g in gs], [m.clone() for m in ms]
    v1t_amd.muon_step(ps, gs, ms, lr=lrs, momentum=0.9, nesterov=nesterov, weight_decay=decay, l1=l1)
    for p, m, (wp, wm), b, lr in zip(ps, ms, want, before, lrs):
        check_step(p, m, wp, wm, b, lr)
    assert all(torch.equal(g, k) for g, k in zip(gs, kept))
    v1t_amd.muon_step(ps, gs, ms, lr=0.01, zero_grad=True)
    assert all(bool((g == 0).all()) for g in gs)


def test_muon_step_captured_and_replayed():
    """Replays between eager work, against the same steps run eagerly, bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    shapes = [(155, 64), (170, 200)] * 30  # two table launches
    ps, gs, ms = ([torch.randn(s, device=DEV, generator=gen) for s in shapes] for _ in range(3))
    qs, ns = [p.clone() for p in ps], [m.clone() for m in ms]
    v1t_amd.muon_step([p.clone() for p in ps], gs, [m.clone() for m in ms], lr=0.02)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v1t_amd.muon_step(ps, gs, ms, lr=0.02, weight_decay=0.1)
    with torch.cuda.graph(other):
        o = v1t_amd.orthogonalize(gs)
    for _ in range(3):
        for g in gs:
            g.normal_(generator=gen)
        v1t_amd.muon_step(qs, gs, ns, lr=0.02, weight_decay=0.1)
        want = v1t_amd.orthogonalize(gs)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps + ms + o, qs + ns + want))


@pytest.mark.parametrize("trans", [False, True])
def test_the_longest(trans):
    """2^31 - 2^22 elements: byte offsets past 2^32. The iterates in 64 bits are Q X with Q of the short side, so that some columns stand for all. Gaussian rows are all but
    orthogonal: every singular value is near 1 / sqrt(511) and ends near one, 23 times as large, as do the roundings of 15 products (and half a step of the result's type)."""
    m, n = 511, 1 << 22
    g = torch.Generator(device=DEV).manual_seed(11)
    u = torch.randn((n, m) if trans else (m, n), device=DEV, generator=g, dtype=torch.bfloat16)
    o = v1t_amd.orthogonalize(u)
    x, y = (u.t(), o.t()) if trans else (u, o)
    gram = torch.zeros(m, m, dtype=torch.float64, device=DEV)
    for c in range(0, n, 1 << 18):
        part = x[:, c:c + (1 << 18)].double().contiguous()
        gram += part @ part.t().contiguous()
    norm = gram.trace().sqrt()
    q = torch.eye(m, dtype=torch.float64, device=DEV) / norm
    a, b, c = COEFFICIENTS
    for _ in range(5):
        s = q @ gram @ q.t()
        q = (a * torch.eye(m, dtype=torch.float64, device=DEV) + b * s + c * (s @ s)) @ q
    for at in (0, 1 << 20, (1 << 21) + 12345, n - 300):
        want, got = q @ x[:, at:at + 300].double().contiguous(), y[:, at:at + 300].double()
        assert float((got - want).norm() / want.norm()) <= 2**-8 + 23 * 15 * 4 * 2**-22


def test_the_widest():
    """32768 x 65536 with one number in each row, in columns of their own: the singular values are the numbers', the result has one in each row's place, too. Two steps,
    each a few roundings of 2^-22 of the value and its factors."""
    m, n = 1 << 15, 1 << 16
    g = torch.Generator(device=DEV).manual_seed(12)
    cols, d = torch.randperm(n, device=DEV, generator=g)[:m], torch.rand(m, device=DEV, generator=g) + 0.5
    u = torch.zeros(m, n, device=DEV)
    rows = torch.arange(m, device=DEV)
    u[rows, cols] = d
    s = d.double() / d.double().norm()
    o = v1t_amd.orthogonalize(u, steps=2)
    a, b, c = COEFFICIENTS
    for _ in range(2):
        s = a * s + b * s**3 + c * s**5
    got = o[rows, cols].double()
    assert float(((got - s) / s).abs().max()) <= 2 * 8 * 2**-22 + 1e-7 / float(d.norm())
    o[rows, cols] = 0.0
    assert not bool(o.any())


def test_two_streams_at_once():
    us = [update(300, 200, i) for i in range(4)]
    want = v1t_amd.orthogonalize(us)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = v1t_amd.orthogonalize(us)
    b = v1t_amd.orthogonalize(us)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) and torch.equal(z, y) for x, z, y in zip(a, b, want))


def test_versions_are_counted():
    p = torch.randn(4, 6, device=DEV, requires_grad=True)
    y = (p * p).sum()
    with torch.no_grad():
        v1t_amd.muon_step([p], [torch.randn(4, 6, device=DEV)], [torch.zeros(4, 6, device=DEV)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
