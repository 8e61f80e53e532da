"""CPU: what the rotary entry points refuse, before any launch."""
import ctypes as C

import pytest
import torch

import v1t_amd
from v1t_amd import lib as L

Q = torch.zeros(2, 5, 4, 16)
AT = torch.zeros(5, 2, dtype=torch.int32)


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(sections=())), (ValueError, dict(sections=(1, 1, 1, 1, 1))), (ValueError, dict(sections=(-1, 3))), (ValueError, dict(sections=(0, 0))),
    (ValueError, dict(sections=(5, 4))), (ValueError, dict(sections=(4, 4, 0))), (ValueError, dict(layout="whole")), (ValueError, dict(base=0.0)),
    (ValueError, dict(base=float("nan"))), (ValueError, dict(base=float("inf"))), (ValueError, dict(q=torch.zeros(5, 16))),
    (ValueError, dict(q=torch.zeros(2, 5, 0, 16))), (ValueError, dict(k=torch.zeros(2, 6, 4, 16))), (ValueError, dict(k=torch.zeros(2, 5, 4, 18))),
    (ValueError, dict(k=torch.zeros(5, 4, 16))), (TypeError, dict(k=torch.zeros(2, 5, 4, 16, dtype=torch.bfloat16))),
    (TypeError, dict(q=torch.zeros(2, 5, 4, 16, dtype=torch.float64))), (TypeError, dict(positions=AT.to(torch.int16))),
    (ValueError, dict(positions=torch.zeros(5, 3, dtype=torch.int32))), (ValueError, dict(positions=torch.zeros(3, 5, 2, dtype=torch.int32))),
    (ValueError, dict(positions=torch.zeros(5, dtype=torch.int32))), (ValueError, dict(positions=torch.zeros(5, 2, requires_grad=True))),
    (RuntimeError, dict()),  # nothing wrong but the device: there is no CPU path
])
@pytest.mark.parametrize("call", ["rotary", "rotary_"])
def test_refusals(call, error, change):
    arguments = dict(q=Q, positions=AT, sections=(3, 4), **{}) | change
    with pytest.raises(error):
        getattr(v1t_amd, call)(arguments.pop("q"), arguments.pop("positions"), **arguments)


def test_too_many_pairs():
    with pytest.raises(ValueError, match="256"):
        v1t_amd.rotary(torch.zeros(1, 1, 600), torch.zeros(1, 1, dtype=torch.int32), sections=(257,))


@pytest.mark.parametrize("call", ["rotary", "rotary_"])
@pytest.mark.parametrize("shape", [(2**32 + 1, 1, 8), (2**32 + 1, 1, 1, 8), (1, 2**32 + 1, 8), (1, 1, 2**32 + 8)])
def test_sizes_that_do_not_fit_32_bits(call, shape):
    """2^32 + 1 tokens are not one."""
    with pytest.raises(ValueError, match="less than"):
        getattr(v1t_amd, call)(torch.zeros(1).expand(shape), torch.zeros(1, 1, dtype=torch.int32).expand(shape[-3], 1), sections=(4,))


def test_in_place_refusals():
    at = dict(positions=AT, sections=(3, 4))
    with pytest.raises(RuntimeError, match="requires grad"):
        v1t_amd.rotary_(Q.clone().requires_grad_(), **at)
    with pytest.raises(ValueError, match="unit stride"):
        v1t_amd.rotary_(torch.zeros(2, 5, 4, 32)[..., ::2], **at)
    with pytest.raises(ValueError, match="expanded"):
        v1t_amd.rotary_(torch.zeros(1, 5, 4, 16).expand(2, -1, -1, -1), **at)
    with pytest.raises(ValueError, match="expanded"):
        v1t_amd.rotary_(torch.zeros(400).as_strided((2, 5, 4, 16), (160, 32, 8, 1)), **at)  # heads overlap
    q = Q.clone()
    with pytest.raises(ValueError, match="share"):
        v1t_amd.rotary_(q, k=q, **at)
    packed = torch.zeros(2, 5, 12, 16)
    with pytest.raises(ValueError, match="share"):
        v1t_amd.rotary_(packed[:, :, :4], k=packed[:, :, 3:7], **at)
    with pytest.raises(RuntimeError, match="GPU"):  # apart: only the device is refused
        v1t_amd.rotary_(packed[:, :, :4], k=packed[:, :, 4:8], **at)


def test_c_entry_refusals():
    lib = L.load()
    ops = (L.RotaryOperand * 2)()
    for o in ops:
        o.x, o.y, o.heads = 4096, 4096, 4  # never dereferenced: every call below is refused or empty
    sec = (C.c_int * 5)(3, 4, 0, 0, 0)

    def call(ops=ops, n_ops=2, dtype=0, B=1, T=1, D=16, sections=sec, n_axes=2, base=100.0, positions=4096, position_type=0):
        return lib.v1t_rotary(ops, n_ops, dtype, B, T, D, sections, n_axes, base, 0, 0, 0, positions, position_type, 0, 2, 1, None)

    bad = [dict(ops=None), dict(n_ops=0), dict(n_ops=3), dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(T=-1), dict(D=0), dict(D=13), dict(sections=None),
           dict(n_axes=0), dict(n_axes=5), dict(base=0.0), dict(base=-1.0), dict(base=float("nan")), dict(base=float("inf")), dict(positions=None),
           dict(position_type=3), dict(sections=(C.c_int * 2)(-1, 4)), dict(sections=(C.c_int * 2)(0, 0))]
    for change in bad:
        assert call(**change) == -1, change
    assert call(D=1024, sections=(C.c_int * 2)(200, 57)) == -2  # more pairs than a kernel argument holds
    assert call(B=0) == 0 and call(T=0) == 0  # nothing to do
    assert call(D=2048, T=(1 << 31) - 1, sections=(C.c_int * 2)(100, 100)) == -2  # a launch of more than 2^32 threads
    ops[1].heads = 0
    assert call() == -1
