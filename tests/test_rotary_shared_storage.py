"""q and k as views of one buffer, turned in place: whether they share an element, against the sets of their elements; and the values."""
import itertools
import random

import pytest
import torch

import v1t_amd
from v1t_amd.positions import _apart


def elements(x):
    return {x.storage_offset() + sum(i * s for i, s in zip(at, x.stride())) for at in itertools.product(*map(range, x.shape))}


def test_never_taken_for_apart():
    rng, buffer, apart = random.Random(3), torch.zeros(300), 0
    for _ in range(4000):
        shape = [rng.randint(1, 3) for _ in range(rng.choice((2, 3)))] + [rng.choice((2, 4))]
        views = []
        for _ in range(2):
            sizes = shape[:-2] + [rng.randint(1, 3), shape[-1]]
            strides = [rng.choice((2, 3, 4, 6, 8, 12, 16, 24, 48)) for _ in sizes[:-1]] + [1]
            offset = rng.randint(0, 40)
            if offset + sum((n - 1) * s for n, s in zip(sizes, strides)) < 300:
                views.append(buffer.as_strided(sizes, strides, offset))
        if len(views) == 2 and _apart(*views):
            assert not elements(views[0]) & elements(views[1]), [(v.shape, v.stride(), v.storage_offset()) for v in views]
            apart += 1
    assert apart > 500


PACKED = {
    "side by side": lambda x: (x[:, :, :4], x[:, :, 4:6]),
    "in turn": lambda x: (x[:, :, ::2], x[:, :, 1::2]),
    "in turn, one head of k": lambda x: (x[:, :, ::2], x[:, :, 3:4]),
    "by halves of a row": lambda x: (x[..., :8], x[..., 8:]),
    "sequences apart": lambda x: (x[:1], x[1:2]),
}


@pytest.mark.parametrize("name", sorted(PACKED))
def test_packed_views_are_apart(name):
    q, k = PACKED[name](torch.zeros(2, 5, 8, 16))
    assert not elements(q) & elements(k)
    for a, b in ((q, k), (k, q)):
        with pytest.raises(RuntimeError, match="GPU"):  # only the device is wrong
            v1t_amd.rotary_(a, torch.zeros(5, 2, dtype=torch.int32), k=b, sections=(2, 2))


@pytest.mark.parametrize("views", [lambda x: (x[:, :, :4], x[:, :, 3:5]), lambda x: (x[..., :8], x[..., 7:15]), lambda x: (x[:, :, ::2], x[:, :, 2:3]), lambda x: (x, x)])
def test_shared_elements_are_refused(views):
    q, k = views(torch.zeros(2, 5, 8, 16))
    with pytest.raises(ValueError, match="share elements"):
        v1t_amd.rotary_(q, torch.zeros(5, 2, dtype=torch.int32), k=k, sections=(1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("name", sorted(PACKED))
def test_turned_where_they_lie(name, layout):
    g = torch.Generator(device="cuda:0").manual_seed(5)
    x = torch.randn(2, 5, 8, 16, device="cuda:0", generator=g)
    at = torch.arange(10, dtype=torch.int32, device="cuda:0").view(5, 2)
    want, before = x.clone(), x.clone()
    q, k = PACKED[name](want)
    yq, yk = v1t_amd.rotary(q.contiguous(), at, k=k.contiguous(), sections=(1, 2), layout=layout)
    q.copy_(yq)
    k.copy_(yk)
    q, k = PACKED[name](x)
    v1t_amd.rotary_(q, at, k=k, sections=(1, 2), layout=layout)
    assert torch.equal(x, want) and not torch.equal(x, before)
