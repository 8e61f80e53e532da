"""CPU: what autograd makes of `rotary`, with the launch replaced by the formula."""
import pytest
import torch

import v1t_amd
from v1t_amd import lib as L
from v1t_amd import positions


@pytest.fixture(autouse=True)
def formula(monkeypatch):
    def launch(turn, at, pairs):
        s = torch.cat([torch.full((n,), a) for a, n in enumerate(turn.sections)])
        i = torch.cat([torch.arange(n) / n for n in turn.sections]).double()
        angle = at.double()[:, s] * turn.base**-i * (-1 if turn.inverse else 1)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        for x, y in pairs:
            z, p = x.detach().double().clone(), turn.pairs
            z[..., 0:2 * p:2], z[..., 1:2 * p:2] = x.double()[..., 0:2 * p:2] * c - x.double()[..., 1:2 * p:2] * s, x.double()[..., 0:2 * p:2] * s + x.double()[..., 1:2 * p:2] * c
            y.copy_(z)
    monkeypatch.setattr(positions, "_launch", launch)
    monkeypatch.setattr(L, "require_cuda", lambda *a: None)
    monkeypatch.setattr(L, "stream_of", lambda device: 7)


AT = torch.arange(10).view(5, 2)


@pytest.mark.parametrize("qg,kg", [(True, True), (True, False), (False, True), (False, False)])
def test_a_result_requires_grad_where_its_input_does(qg, kg):
    q, k = torch.randn(2, 5, 4, 16, requires_grad=qg), torch.randn(2, 5, 2, 16, requires_grad=kg)
    yq, yk = v1t_amd.rotary(q, AT, k=k, sections=(3, 4))
    assert (yq.requires_grad, yk.requires_grad) == (qg, kg)
    back = {}
    for y, x in ((yq, q), (yk, k)):
        if x.requires_grad:
            g = torch.randn_like(y)
            (back[x],) = torch.autograd.grad(y, x, g, retain_graph=True)
            assert torch.allclose(back[x], v1t_amd.rotary(g, AT, sections=(3, 4), inverse=True))
    if qg or kg:
        (yq.sum() + yk.sum()).backward()
        assert (q.grad is not None, k.grad is not None) == (qg, kg)
        if not (qg and kg):
            other = yk if qg else yq
            other.add_(1.0)  # a plain tensor: free to be changed


@pytest.mark.parametrize("qg,kg", [(True, True), (True, False), (False, True)])
def test_second_derivatives(qg, kg):
    q, k = torch.randn(5, 1, 8, requires_grad=qg), torch.randn(5, 2, 8, requires_grad=kg)
    yq, yk = v1t_amd.rotary(q, AT, k=k, sections=(1, 2))
    xs = [x for x in (q, k) if x.requires_grad]
    gs = torch.autograd.grad((yq**3).sum() + (yk**3).sum(), xs, create_graph=True)
    v = [torch.randn_like(g) for g in gs]
    hv = torch.autograd.grad(gs, xs, v)
    for x, g, w in zip(xs, hv, v):  # R^T diag(6 y) R v
        turned = lambda z, inverse=False: v1t_amd.rotary(z, AT, sections=(1, 2), inverse=inverse)
        want = turned(6 * turned(x.detach()) * turned(w), True)
        assert torch.allclose(g, want, atol=1e-5)


def test_a_leaf_of_k_alone_is_marked(monkeypatch):
    """Whichever of the two requires grad, its leaf is watched for captures."""
    k = torch.randn(5, 2, 8, requires_grad=True)
    _, yk = v1t_amd.rotary(torch.randn(5, 1, 8), AT, k=k, sections=(1, 2))
    (node,) = [n for n, _ in yk.grad_fn.next_functions if hasattr(n, "variable")]
    assert node.variable is k and node.metadata["v1t_stream"] == 7
