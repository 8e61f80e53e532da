"""GPU: orthogonalised updates that come out exactly, number by number, and the precision that the two planes leave.

Exact: a matrix with one number 1 or -1 in each of 4^k of its rows and nothing else has the norm 2^k, so X holds 2^-k, X X^T 4^-k where two rows share a column, and
with (a, b, c) = (1, -1, 1) a row whose column is shared by n of them becomes 2^-k (1 - n 4^-k + n^2 16^-k): with k <= 5 every number on the way has at most 20 bits (22 are
held) and every sum less than 24, whatever its order. A number in another place, or one that was read before it was there, is not a rounding."""
import math

import pytest
import torch

import v1t_amd
from v1t_amd.muon import COEFFICIENTS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def sparse(rows, cols, seed):
    """(matrix, its image under one step of (1, -1, 1)); rows <= cols"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = min(5, int(math.log(rows, 4) + 1e-9))
    at = torch.randperm(rows, device=DEV, generator=g)[:4**k]
    col = torch.randint(0, max(1, min(cols, 4**k // 3)), (4**k,), device=DEV, generator=g)
    col = torch.randperm(cols, device=DEV, generator=g)[col]  # about three rows a column, the columns all over the matrix
    sign = torch.randint(0, 2, (4**k,), device=DEV, generator=g).double() * 2 - 1
    n = torch.bincount(col, minlength=cols)[col].double()
    u, want = torch.zeros(2, rows, cols, dtype=torch.float64, device=DEV)
    u[at, col] = sign
    want[at, col] = sign * 2.0**-k * (1 - n * 4.0**-k + n * n * 16.0**-k)
    return u.float(), want.float()


# matrices whose planes fit a CU's LDS, tiles of 64, 128 and 192, whole, in pieces and both, steps in pairs
@pytest.mark.parametrize("count,rows,cols", [(3, 20, 50), (2, 64, 155), (1, 90, 193), (4, 155, 620), (1, 300, 1000), (1, 100, 20000), (1, 1600, 1660), (1, 1800, 1900),
                                             (4, 1300, 1300), (2, 1000, 1900), (1, 2300, 2360), (1, 4001, 4100), (12, 777, 1301), (1, 700, 2900), (1, 1024, 8192)])
@pytest.mark.parametrize("trans", [False, True])
def test_every_number_in_its_place(count, rows, cols, trans):
    made = [sparse(rows, cols, 7 * i + rows) for i in range(count)]
    us, wants = [u.t().contiguous() if trans else u for u, _ in made], [w.t() if trans else w for _, w in made]
    for coefficients in ([(1.0, -1.0, 1.0)], [(1.0, -1.0, 1.0), (1.0, 0.0, 0.0)], [(1.0, 0.0, 0.0), (1.0, -1.0, 1.0)]):
        for o, w in zip(v1t_amd.orthogonalize(us, steps=len(coefficients), coefficients=coefficients, eps=0.0), wants):
            assert torch.equal(o, w)


# ---- what is lost
def planes(x, exponent):
    hi = (x * 2.0**exponent).half()
    lo = (x * 2.0**exponent - hi.double()).half()
    return hi.double() * 2.0**-exponent, lo.double() * 2.0**-exponent


def held(u, eps=1e-7, exponent=13):
    """The steps in 64 bits, but for what the kernel holds: X, A and S as two fp16 planes of 2^13 times the number (2.8 is the largest of any, under the usual coefficients) and
    products without lo lo."""
    def product(p, q):
        (ph, pl), (qh, ql) = p, q
        return ph @ qh + ph @ ql + pl @ qh

    x = u.double()
    flip = x.shape[0] > x.shape[1]
    x = planes((x.t() if flip else x) / (x.norm() + eps), exponent)
    a, b, c = COEFFICIENTS
    for k in range(5):
        g = planes(product(x, [y.t() for y in x]), exponent)
        s = planes(b * sum(g) + c * product(g, [y.t() for y in g]), exponent)
        new = a * sum(x) + product(s, x)
        x = planes(new, exponent)
    return new.t() if flip else new


def formula(u, dtype, eps=1e-7):
    x = u.double()
    flip = x.shape[0] > x.shape[1]
    x = ((x.t() if flip else x) / (x.norm() + eps)).to(dtype)
    a, b, c = COEFFICIENTS
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if flip else x


def allowed(u):
    """(the result in 64 bits, the error's 2-norm over the result's): what the planes cost, as `held` has it, and what sums in fp32 cost, as the formula in fp32 has it - each
    an error of random signs, so the kernel's own may be another draw of the same size: twice both. Planes of two bits less would take four times the first."""
    want = formula(u, torch.float64)
    off = lambda x: float((x.double() - want).norm() / want.norm())
    return want, 2 * (off(held(u)) + off(formula(u, torch.float32)))


def gradient(rows, cols, seed):
    """Directions of many strengths, as in a weight's gradient"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    fall = lambda n: (torch.arange(n, device=DEV) + 1.0) ** -0.3
    return fall(rows)[:, None] * torch.randn(rows, cols, device=DEV, generator=g) * fall(cols)


@pytest.mark.parametrize("rows,cols", [(64, 155), (155, 64), (90, 193), (155, 620), (488, 155), (777, 1301), (2048, 2048)])
def test_no_bit_less_than_the_planes_hold(rows, cols):
    u = gradient(rows, cols, rows + cols)
    want, bound = allowed(u)
    got = float((v1t_amd.orthogonalize(u).double() - want).norm() / want.norm())
    assert got <= bound, (got, bound)


@pytest.mark.parametrize("scale", [1e-3, 1e-5, 1e-7])
@pytest.mark.parametrize("rows,cols", [(64, 155), (155, 620), (488, 155)])
def test_rows_far_below_the_others(rows, cols, scale):
    """The planes have one exponent per matrix: such a row keeps fewer of its bits, as `held` has it, and costs the others none."""
    u = gradient(rows, cols, 3)
    u[5] *= scale
    want, bound = allowed(u)
    got, model, plain = (x.double() - want for x in (v1t_amd.orthogonalize(u), held(u), formula(u, torch.float32)))
    assert float(got.norm() / want.norm()) <= bound
    assert float(got[5].norm()) <= 2 * float(model[5].norm() + plain[5].norm())


def test_the_momentum_step_to_the_same_bits():
    """With a momentum of a half, m and U are one rounding each, fused or not: U is known to the bit. The parameter: the rate's rounding, its product's and the sum's."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    shapes = [(155, 64), (155, 620), (488, 155)]
    ps, ms = ([torch.randn(s, device=DEV, generator=gen) for s in shapes] for _ in range(2))
    gs = [gradient(*s, i) for i, s in enumerate(shapes)]
    before = [p.double() for p in ps]
    after = [(0.5 * m.double() + g.double()).float() for g, m in zip(gs, ms)]
    us = [(0.5 * m.double() + g.double()).float() for g, m in zip(gs, after)]
    v1t_amd.muon_step(ps, gs, ms, lr=0.02, momentum=0.5)
    assert all(torch.equal(m, a) for m, a in zip(ms, after))
    for p, b, u in zip(ps, before, us):
        want, bound = allowed(u)
        step = 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * want
        off = float((p.double() - (b - step)).norm())
        assert off <= (bound + 2 * 2**-24) * float(step.norm()) + 2**-24 * float(p.double().norm()), (off, bound)
