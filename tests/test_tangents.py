"""CPU: operators that read and write raw pointers refuse tensors that carry a tangent (forward-mode differentiation), which they would lose."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import v1t_amd
from v1t_amd import lib as L
from v1t_amd import positions

Q, AT = torch.zeros(2, 5, 4, 16), torch.zeros(5, 2)


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


def fresh(*shape):
    return torch.zeros(shape or (4, 6))


CALLS = {
    "rotary q": lambda d: v1t_amd.rotary(d(Q.clone()), AT, sections=(3, 4)),
    "rotary q of two": lambda d: v1t_amd.rotary(d(Q.clone()), AT, k=Q, sections=(3, 4)),
    "rotary k": lambda d: v1t_amd.rotary(Q, AT, k=d(Q.clone()), sections=(3, 4)),
    "rotary positions": lambda d: v1t_amd.rotary(Q, d(AT.clone()), sections=(3, 4)),
    "rotary_ q": lambda d: v1t_amd.rotary_(d(Q.clone()), AT, sections=(3, 4)),
    "rotary_ k": lambda d: v1t_amd.rotary_(Q.clone(), AT, k=d(Q.clone()), sections=(3, 4)),
    "orthogonalize": lambda d: v1t_amd.orthogonalize(d(fresh())),
    "orthogonalize stack": lambda d: v1t_amd.orthogonalize(d(fresh(3, 4, 6))),
    "orthogonalize list": lambda d: v1t_amd.orthogonalize([fresh(), d(fresh(2, 2))]),
    "muon_step parameter": lambda d: v1t_amd.muon_step([d(fresh())], [fresh()], [fresh()], lr=0.1),
    "muon_step gradient": lambda d: v1t_amd.muon_step([fresh()], [d(fresh())], [fresh()], lr=0.1),
    "muon_step momentum": lambda d: v1t_amd.muon_step([fresh()], [fresh()], [d(fresh())], lr=0.1),
}


@pytest.mark.parametrize("call", sorted(CALLS))
def test_a_tangent_is_refused(call):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            CALLS[call](dual)
        with pytest.raises(RuntimeError, match="GPU"):  # beside a level that these tensors have no part in, only the device is wrong
            CALLS[call](lambda x: x)
    with pytest.raises(RuntimeError, match="GPU"):
        CALLS[call](lambda x: x)


def test_a_tangent_in_the_backward_pass_is_refused(monkeypatch):
    """Its gradients may be the dual ones."""
    monkeypatch.setattr(positions, "_launch", lambda turn, at, pairs: [y.zero_() for _, y in pairs])
    monkeypatch.setattr(L, "require_cuda", lambda *a: None)
    monkeypatch.setattr(L, "leaves_in_capture", lambda *a: None)
    q, k = (Q.clone().requires_grad_() for _ in range(2))
    yq, yk = v1t_amd.rotary(q, AT, k=k, sections=(3, 4))
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.autograd.grad((yq, yk), (q, k), (torch.ones_like(yq), dual(torch.ones_like(yk))))
    yq, yk = v1t_amd.rotary(q, AT, k=k, sections=(3, 4))
    assert all(g.shape == Q.shape for g in torch.autograd.grad((yq, yk), (q, k), (torch.ones_like(yq), torch.ones_like(yk))))
