"""GPU: orthogonalised updates that come out exactly, number by number.

Exact: a matrix with one number 1 or -1 in each of 4^k of its rows and nothing else has the norm 2^k, so X holds 2^-k, X X^T 4^-k where two rows share a column, and
with (a, b, c) = (1, -1, 1) a row whose column is shared by n of them becomes 2^-k (1 - n 4^-k + n^2 16^-k): with k <= 5 every number on the way has at most 20 bits (22 are
held) and every sum less than 24, whatever its order. A number in another place, or one that was read before it was there, is not a rounding."""
import math

import pytest
import torch

import v1t_amd

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
