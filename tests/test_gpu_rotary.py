"""GPU: the rotary positions against the formula in 64 bits.

Tolerances: the reduced angle is rounded to 32 bits (at most 2^-26 of a turn = 9.4e-8 rad) and its sine and cosine to 2 units in the last place (2^-23); two
products and a sum round at 2^-24 each: every output is within (|x0| + |x1|) * 4e-7 of the formula before its rounding to 16 bits, which adds half a step
(eps / 2 of the value)."""
import math

import pytest
import torch

import v1t_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def turned(x, at, sections, base, layout, shared, inverse=False):
    """The definition in 64 bits on the CPU, and the bound of its fp32 evaluation before the last rounding."""
    x, at = x.detach().cpu().double(), at.cpu().double()
    pairs = sum(sections)
    y, bound = x.clone(), torch.zeros_like(x)
    j = 0
    for a, s in enumerate(sections):
        for i in range(s):
            angle = at[..., a] * base ** -(j / pairs if shared else i / s)
            angle = (-angle if inverse else angle)[..., None]
            i0, i1 = (2 * j, 2 * j + 1) if layout == "pairs" else (j, pairs + j)
            y[..., i0] = x[..., i0] * angle.cos() - x[..., i1] * angle.sin()
            y[..., i1] = x[..., i0] * angle.sin() + x[..., i1] * angle.cos()
            bound[..., i0] = bound[..., i1] = 4e-7 * (x[..., i0].abs() + x[..., i1].abs())
            j += 1
    return y, bound


def close(got, want, bound):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # half a step below the smallest normal number
    allowed = bound + (want.abs() + bound) * half + tiny
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), f"off by {float((off - allowed).max())} more than the bound"


def positions(shape, far=0, kind=torch.int32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-3, 60, shape, generator=g) + far).to(kind).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("B,T,H,K,D,sections,shared,far", [
    (1, 1, 1, 1, 2, (1,), False, 0),
    (3, 1, 16, 4, 128, (16, 24, 24), True, 900000),
    (2, 7, 4, 4, 155, (38, 38), False, 0),
    (2, 33, 6, 3, 91, (11, 15, 15), False, 5),
    (1, 130, 2, 1, 64, (5, 0, 9), True, 0),
    (5, 3, 1, 2, 13, (3, 2), False, 0),
    (1, 2, 3, 3, 512, (100, 56, 50, 50), True, 12),
    (70, 2, 2, 2, 24, (6, 6), False, 0),
])
def test_against_the_formula(dtype, layout, B, T, H, K, D, sections, shared, far):
    g = torch.Generator().manual_seed(B * T + D)
    q, k = (torch.randn(B, T, h, D, generator=g).to(dtype).to(DEV) for h in (H, K))
    for at in (positions((T, len(sections)), far), positions((B, T, len(sections)), far, torch.int64, 1)):
        arguments = dict(sections=sections, base=500.0, layout=layout, shared=shared)
        yq, yk = v1t_amd.rotary(q, at, k=k, **arguments)
        for x, y in ((q, yq), (k, yk)):
            close(y, *turned(x, at, sections, 500.0, layout, shared))
            assert torch.equal(y[..., 2 * sum(sections):], x[..., 2 * sum(sections):])
        alone = v1t_amd.rotary(q, at, **arguments)
        assert torch.equal(alone, yq)
        back = v1t_amd.rotary(q, at, inverse=True, **arguments)
        close(back, *turned(q, at, sections, 500.0, layout, shared, inverse=True))
        a, b = q.clone(), k.clone()
        v1t_amd.rotary_(a, at, k=b, **arguments)
        assert torch.equal(a, yq) and torch.equal(b, yk)


def test_fractional_and_far_positions():
    q = torch.randn(4, 2, 8, device=DEV)
    at = torch.tensor([[0.25], [-7.5], [16777215.0], [0.0]], device=DEV)
    y = v1t_amd.rotary(q, at, sections=(4,))
    close(y, *turned(q, at, (4,), 10000.0, "pairs", False))
    assert torch.equal(y[3], q[3])
    at = torch.tensor([[2**31 + 12345], [-(2**40) - 1], [2**52 + 1], [1]], device=DEV)
    # the rate and its product with the position round at 2^-53 of the angle each: 2^31 * 2^-52 = 4.8e-7 rad beside the 4e-7 of the bound, in the
    # kernel and in the formula (a factor of 3.4); at 2^52 only the magnitude holds
    y = v1t_amd.rotary(q, at, sections=(4,))
    r0, r1 = (x[..., 0].square() + x[..., 1].square() for x in (q, y))
    assert torch.allclose(r0, r1, rtol=2e-6, atol=1e-6)
    want, bound = turned(q[:1], at[:1], (4,), 10000.0, "pairs", False)
    close(y[:1], want, 3.4 * bound)


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_views_of_a_packed_projection(offset, layout):
    """q and k as views with every alignment; what lies between and behind them is not touched."""
    B, T, H, D, W = 2, 9, 3, 20, 26
    buffer = torch.randn(B, T, 3, H, W, device=DEV).to(torch.bfloat16)
    at, sections = positions((T, 2)), (4, 4)
    q, k = buffer[:, :, 0, :, offset:offset + D], buffer[:, :, 1, :, offset:offset + D]
    yq, yk = v1t_amd.rotary(q, at, k=k, sections=sections, layout=layout)
    close(yq, *turned(q, at, sections, 10000.0, layout, False))
    before = buffer.clone()
    v1t_amd.rotary_(q, at, k=k, sections=sections, layout=layout)
    assert torch.equal(q, yq) and torch.equal(k, yk)
    buffer[:, :, :2, :, offset:offset + D] = before[:, :, :2, :, offset:offset + D]
    assert torch.equal(buffer, before)


def test_other_strides():
    q = torch.randn(6, 3, 5, 16, device=DEV)
    at = positions((5, 2))
    want = v1t_amd.rotary(q.permute(0, 2, 1, 3).contiguous(), at, sections=(4, 4))
    assert torch.equal(v1t_amd.rotary(q.permute(0, 2, 1, 3), at, sections=(4, 4)), want)  # heads before tokens
    assert torch.equal(v1t_amd.rotary(q.permute(0, 2, 1, 3).transpose(-1, -2).contiguous().transpose(-1, -2), at, sections=(4, 4)), want)  # features not last in memory
    wide = torch.zeros(5, 4, device=DEV, dtype=torch.int32)
    wide[:, ::2] = at
    assert torch.equal(v1t_amd.rotary(q.permute(0, 2, 1, 3), wide[:, ::2], sections=(4, 4)), want)
    one = torch.randn(1, 5, 3, 16, device=DEV)
    assert torch.equal(v1t_amd.rotary(one.expand(4, -1, -1, -1), at, sections=(4, 4))[3], v1t_amd.rotary(one, at, sections=(4, 4))[0])
    assert v1t_amd.rotary(q[:, :, :0].permute(0, 2, 1, 3), at[:0], sections=(4, 4)).shape == (6, 0, 3, 16)
    same_place = at[:1].expand(5, -1)
    assert torch.equal(v1t_amd.rotary(q.permute(0, 2, 1, 3), same_place, sections=(4, 4)), v1t_amd.rotary(q.permute(0, 2, 1, 3), same_place.contiguous(), sections=(4, 4)))


def test_nan_stays_in_its_pair():
    q = torch.randn(1, 3, 2, 12, device=DEV)
    at = positions((3, 1))
    clean = v1t_amd.rotary(q, at, sections=(5,))
    q[0, 1, 0, 4] = math.nan
    q[0, 2, 1, 11] = math.inf
    y = v1t_amd.rotary(q, at, sections=(5,))
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[0, 1, 0, 4:6] = True
    want[0, 2, 1, 11] = True
    assert torch.equal(bad, want)
    assert torch.equal(y[~want], clean[~want])


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_gradients(layout):
    """The gradient is the formula's (the opposite turn), and agrees with central differences of the operator itself: f is linear in x, so a difference over
    a step of 1 is exact but for the roundings of the two sums (64 values, each within 4e-7 * 8 of the formula)."""
    q = torch.randn(2, 3, 4, 11, device=DEV, requires_grad=True)
    k = torch.randn(2, 3, 1, 11, device=DEV, requires_grad=True)
    at, arguments = positions((3, 2)), dict(sections=(3, 2), base=50.0, layout=layout)
    yq, yk = v1t_amd.rotary(q, at, k=k, **arguments)
    wq, wk = torch.randn_like(yq), torch.randn_like(yk)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (wq, wk), retain_graph=True)
    for w, d in ((wq, dq), (wk, dk)):
        close(d, *turned(w, at, (3, 2), 50.0, layout, False, inverse=True))
    (only,) = torch.autograd.grad(yk, k, wk, retain_graph=True)
    assert torch.equal(only, dk)
    broadcast = torch.autograd.grad(yq.sum(), q)[0]  # an expanded gradient
    close(broadcast, *turned(torch.ones_like(yq), at, (3, 2), 50.0, layout, False, inverse=True))
    with torch.no_grad():
        for i in range(q.numel()):
            step = torch.zeros_like(q).view(-1)
            step[i] = 1.0
            plus, minus = (v1t_amd.rotary(q + s * step.view_as(q), at, **arguments) for s in (1.0, -1.0))
            slope = float((wq.double() * (plus.double() - minus.double())).sum() / 2)
            assert abs(slope - float(dq.reshape(-1)[i])) < 64 * 8 * 4e-7


def test_second_derivative():
    q = torch.randn(3, 2, 8, device=DEV, requires_grad=True)
    w = torch.randn(3, 2, 8, device=DEV, requires_grad=True)
    at = positions((3, 1))
    (d,) = torch.autograd.grad(v1t_amd.rotary(q, at, sections=(4,)), q, w, create_graph=True)
    v = torch.randn_like(d)
    (dw,) = torch.autograd.grad(d, w, v)
    close(dw, *turned(v, at, (4,), 10000.0, "pairs", False))


def test_captured_and_replayed_beside_eager_work():
    q, k = (torch.randn(4, 29, h, 64, device=DEV, dtype=torch.bfloat16) for h in (4, 2))
    at, arguments = positions((29, 2)), dict(sections=(16, 16))
    v1t_amd.rotary(q, at, k=k, **arguments)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yq, yk = v1t_amd.rotary(q, at, k=k, **arguments)
    for n in range(3):
        q.normal_(), k.normal_()
        at += n
        wq, wk = v1t_amd.rotary(q, at, k=k, **arguments)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(yq, wq) and torch.equal(yk, wk)


def test_backward_captured_beside_an_eager_graph_of_the_same_leaf():
    """Refused while the eager graph lives (the captured backward would wait on the eager pass's stream); captured and right once it is dropped."""
    q = torch.randn(2, 5, 3, 16, device=DEV, requires_grad=True)
    at, arguments = positions((5, 1)), dict(sections=(6,))
    eager = v1t_amd.rotary(q, at, **arguments)
    w = torch.randn_like(eager)
    want = torch.autograd.grad(eager, q, w, retain_graph=True)[0]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive on another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            v1t_amd.rotary(q, at, **arguments)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (d,) = torch.autograd.grad(v1t_amd.rotary(q, at, **arguments), q, w)
    for _ in range(3):
        d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(d, want)
    assert torch.equal(torch.autograd.grad(v1t_amd.rotary(q, at, **arguments), q, w)[0], want)


def test_another_stream():
    q = torch.randn(64, 100, 4, 64, device=DEV)
    at = positions((100, 2))
    want = v1t_amd.rotary(q, at, sections=(16, 16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = v1t_amd.rotary(q, at, sections=(16, 16))
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,sections", [(6, (3,)), (14, (4, 3))])
def test_many_sequences_with_positions_of_their_own(D, sections):
    """More sequences than a launch has workgroups along one dimension: a workgroup goes over several, each with its own angles."""
    g = torch.Generator().manual_seed(9)
    q = torch.randn(140000, 2, 3, D, generator=g).to(DEV)
    at = positions((140000, 2, len(sections)), seed=2)
    y = v1t_amd.rotary(q, at, sections=sections)
    close(y, *turned(q, at, sections, 10000.0, "pairs", False))
    assert torch.equal(v1t_amd.rotary_(q.clone(), at, sections=sections), y)


def test_offsets_past_32_bits():
    """A cache of 2^31 + elements: the last sequence lies behind the first 4 GB."""
    big = torch.empty(3, 1100, 1000, 1000, dtype=torch.bfloat16, device=DEV)
    assert big.numel() > 2**31
    q = big[:, -40:, -2:, -64:]
    q.copy_(torch.randn(3, 40, 2, 64, device=DEV))
    at = positions((40, 1), 7)
    want = v1t_amd.rotary(q.contiguous(), at, sections=(32,))
    v1t_amd.rotary_(q, at, sections=(32,))
    assert torch.equal(q, want)


def test_version_counter_sees_the_write():
    q = torch.randn(3, 2, 8, device=DEV)
    w = torch.randn(3, 2, 8, device=DEV, requires_grad=True)
    y = (q * w).sum()
    v1t_amd.rotary_(q, positions((3, 1)), sections=(4,))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@pytest.mark.parametrize("D", [11, 16])
def test_results_may_be_changed_in_place(D):
    q = torch.randn(2, 3, 4, D, device=DEV, requires_grad=True)
    k = torch.randn(2, 3, 1, D, device=DEV, requires_grad=True)
    at = positions((3, 1))
    yq, yk = v1t_amd.rotary(q, at, k=k, sections=(5,))
    yq.mul_(2.0)
    w = torch.randn(2, 3, 4, D, device=DEV)
    (d,) = torch.autograd.grad((yq * w).sum() + yk.sum(), q)
    close(d, *turned(2 * w, at, (5,), 10000.0, "pairs", False, inverse=True))
    assert yq.untyped_storage().nbytes() >= 24 * ((D + 7) // 8 * 8) * 4  # the room is the result's own


def test_the_c_entry_without_room():
    """y rows of exactly D features: nothing behind a row's features is written, in any order of the rows."""
    import ctypes as C
    from v1t_amd import lib as L

    for D, room in ((11, 0), (11, 11), (11, 13), (21, 0), (3, 3)):
        B, T, H = 2, 5, 3
        x = torch.randn(B, T, H, D, device=DEV, dtype=torch.bfloat16)
        gap = 2 if room > D else 0
        buffer = torch.full((B * T * H * (D + gap) + 64,), 7.0, device=DEV, dtype=torch.bfloat16)
        y = buffer[32:-32].view(B, T, H, D + gap)
        at = positions((T, 1))
        op = (L.RotaryOperand * 1)(L.RotaryOperand(x.data_ptr(), y.data_ptr(), *x.stride()[:3], *y.stride()[:3], H, room))
        L.check(L.load().v1t_rotary(op, 1, 0, B, T, D, (C.c_int * 1)(1), 1, 10.0, 0, 0, 0, at.data_ptr(), 0, 0, 1, 1, L.stream()))
        close(y[..., :D], *turned(x, at, (1,), 10.0, "pairs", False))
        assert bool((buffer[:32] == 7.0).all()) and bool((buffer[-32:] == 7.0).all()) and bool((y[..., D:] == 7.0).all())
