"""CPU: views that hold their numbers with the other sign (`z.conj().imag`), whose raw memory is not what they stand for."""
import ctypes as C

import pytest
import torch

import v1t_amd
from v1t_amd import lib as L
from v1t_amd import muon, positions


def negated(*shape, dtype=torch.float32):
    x = torch.view_as_complex(torch.randn(*shape, 2, dtype=dtype)).conj().imag
    assert x.is_neg()
    return x


def read(x):
    """The numbers as a kernel reads them: from memory, by strides."""
    flat = (C.c_float * (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())))).from_address(x.data_ptr())
    return torch.frombuffer(flat, dtype=torch.float32).as_strided(x.shape, x.stride()).clone()


@pytest.fixture
def launched(monkeypatch):
    seen = []

    def launch(turn, at, pairs):
        seen.append([read(at)] + [read(x) for x, _ in pairs])
        for _, y in pairs:
            y.zero_()
    monkeypatch.setattr(positions, "_launch", launch)
    monkeypatch.setattr(muon, "_orthogonalize", lambda pairs, *a: seen.append([read(u) for u, _ in pairs]))
    monkeypatch.setattr(L, "require_cuda", lambda *a: None)
    monkeypatch.setattr(L, "leaves_in_capture", lambda *a: None)
    return seen


@pytest.mark.parametrize("contiguous", [False, True])
def test_rotary_reads_their_numbers(launched, contiguous):
    q, k, at = negated(2, 5, 4, 16), negated(2, 5, 2, 16), negated(5, 2)
    if contiguous:
        q, k, at = (torch._neg_view(x.clone().resolve_neg().neg()) for x in (q, k, at))
    v1t_amd.rotary(q, at, k=k, sections=(3, 4))
    for got, want in zip(launched[0], (at, q, k)):
        assert torch.equal(got, want)


def test_the_gradients_too(launched):
    q = torch.randn(2, 5, 4, 16, requires_grad=True)
    y = v1t_amd.rotary(q, torch.zeros(5, 2), sections=(3, 4))
    g = torch._neg_view(torch.randn(2, 5, 4, 16))
    torch.autograd.grad(y, q, g)
    assert torch.equal(launched[1][1], g)


def test_in_place_they_are_refused():
    q, at = torch._neg_view(torch.randn(2, 5, 4, 16)), torch.zeros(5, 2)
    with pytest.raises(ValueError, match="negates"):
        v1t_amd.rotary_(q, at, sections=(3, 4))
    with pytest.raises(ValueError, match="negates"):
        v1t_amd.rotary_(torch.randn(2, 5, 4, 16), at, k=q, sections=(3, 4))
    for i in range(3):
        p = [torch.randn(4, 6) for _ in range(3)]
        p[i] = torch._neg_view(p[i])
        with pytest.raises(ValueError, match="negate"):
            v1t_amd.muon_step(*([x] for x in p), lr=0.1)


def test_positions_in_place(launched):
    at = negated(5, 2)
    v1t_amd.rotary_(torch.randn(2, 5, 4, 16), at, sections=(3, 4))
    assert torch.equal(launched[0][0], at)


def test_orthogonalize_reads_their_numbers(launched):
    us = [negated(4, 6), torch.randn(4, 6), torch._neg_view(torch.randn(3, 2))]
    v1t_amd.orthogonalize(us)
    assert all(torch.equal(a, b) for a, b in zip(launched[0], us))
