"""Dropout from the counter-based generator: the mask bit for bit, the values to their type's rounding."""
import math

import numpy as np
import pytest
import torch

from oracle import operators as P
from gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from flashdp4review_b200.core import ops
    return ops


def mask(x, s):
    return torch.from_numpy(P.keep_mask(x.numel(), s.p, s.seed, s.stream_id, s.step, s.offset)).view(x.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 2056, 100003])
@pytest.mark.parametrize("residual", [False, True])
def test_values_and_mask(ops, dtype, n, residual):
    gen = torch.Generator().manual_seed(n)
    x, r = torch.randn(n, generator=gen).to(dtype), torch.randn(n, generator=gen).to(dtype)
    s = ops.DropoutSpec(p=0.3, seed=0xFEDCBA9876543210, stream_id=3, step=11)
    got = ops.dropout(x.to(dev()), s, residual=r.to(dev()) if residual else None).cpu().double()
    keep = mask(x, s)
    want = torch.where(keep, x.double() / 0.7, 0.0) + (r.double() if residual else 0.0)
    # one fp32 product with a factor rounded to fp32, one fp32 sum, one rounding to the type
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 4 * 2.0 ** -24 * (x.double().abs() / 0.7 + want.abs()) + 2.0 ** -25
    assert ((got - want).abs() <= tol).all()
    if not residual:
        assert torch.equal(got != 0, keep & (x != 0))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -32, 1e-4, 0.1, 0.25, 0.5, 0.9, 1 - 2.0 ** -32, 1.0])
def test_every_probability(ops, p):
    """p = 0 keeps all, p = 1 drops all, and between them an element on the border is decided by its lower 16 bits."""
    x = torch.ones(400003)
    s = ops.DropoutSpec(p=p, seed=12345, stream_id=1, step=1)
    got = ops.dropout(x.to(dev()), s).cpu() != 0
    assert torch.equal(got, mask(x, s))
    if p in (0.0, 1.0):
        assert bool(got.all()) == (p == 0.0) and bool(got.any()) == (p == 0.0)
    share = 1 - got.double().mean().item()
    assert abs(share - p) <= 5 * math.sqrt(p * (1 - p) / x.numel()) + 1e-9


def test_ties_are_decided_by_the_second_draw(ops):
    """Two thresholds that differ in the lower 16 bits only give masks that differ, in a few elements."""
    x = torch.ones(1 << 22)
    a, b = (ops.DropoutSpec(p=(0x3333 * 65536 + lo) / 2 ** 32, seed=5, stream_id=2, step=3) for lo in (1, 65535))
    ka, kb = (ops.dropout(x.to(dev()), s).cpu() != 0 for s in (a, b))
    assert torch.equal(ka, mask(x, a)) and torch.equal(kb, mask(x, b))
    differ = int((ka != kb).sum())
    assert 0 < differ < 200 and bool((ka | ~kb).all())        # the higher threshold drops more; 64 expected


def test_streams_steps_offsets(ops):
    x = torch.ones(4096, device=dev())
    base = dict(p=0.5, seed=1, stream_id=1, step=1)
    m0 = ops.dropout(x, ops.DropoutSpec(**base))
    assert torch.equal(m0, ops.dropout(x, ops.DropoutSpec(**base)))
    for change in (dict(seed=2), dict(seed=1 << 32 | 1), dict(stream_id=2), dict(step=2)):
        other = ops.dropout(x, ops.DropoutSpec(**{**base, **change}))
        assert 0.4 < (other != m0).float().mean().item() < 0.6, change
    shifted = ops.dropout(x[:2048], ops.DropoutSpec(**base, offset=256))
    assert torch.equal(shifted, m0[2048:])
    far = ops.DropoutSpec(**base, offset=(1 << 60) - 1)
    assert torch.equal(ops.dropout(x[:8], far).cpu() != 0, mask(x[:8].cpu(), far))


def test_infinities_in_dropped_places(ops):
    x = torch.full((4096,), math.inf, device=dev(), dtype=torch.bfloat16)
    x[::2] = math.nan
    s = ops.DropoutSpec(p=0.5, seed=9, stream_id=1, step=1)
    y, keep = ops.dropout(x, s), mask(x.cpu(), s).to(dev())
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    r = torch.arange(4096, device=dev()).to(torch.bfloat16)
    assert torch.equal(ops.dropout(x, s, residual=r)[~keep], r[~keep])


def test_in_place_views_and_alignment(ops):
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(64, 50, generator=gen).to(torch.bfloat16).to(dev())
    s = ops.DropoutSpec(p=0.2, seed=4, stream_id=1, step=1)
    want = ops.dropout(x, s)
    t = x.t().contiguous().t()
    assert torch.equal(ops.dropout(t, s), want)                          # numbered by position, not by storage
    off = torch.zeros(x.numel() + 3, dtype=x.dtype, device=dev())[3:].view(64, 50).copy_(x)
    assert off.data_ptr() % 16 != 0 and torch.equal(ops.dropout(off, s), want)
    r = x.clone()
    both = ops.dropout(x, s, residual=x)
    assert torch.equal(ops.dropout(x, s, residual=r, out=r), both) and torch.equal(r, both)
    z = x.clone()
    assert ops.dropout(z, s, out=z).data_ptr() == z.data_ptr() and torch.equal(z, want)
    assert ops.dropout(x[:0], s).shape == (0, 50)


def test_backward_is_the_same_mask(ops):
    gen = torch.Generator().manual_seed(3)
    g = torch.randn(10, 33, generator=gen).to(dev())
    s = ops.DropoutSpec(p=0.4, seed=8, stream_id=1, step=1)
    dx = ops.dropout_backward(g, s)
    assert torch.equal(dx != 0, ops.dropout(torch.ones_like(g), s) != 0)


def test_more_than_2_32_elements(ops):
    """In place; what stands for any stretch is what a tensor of its length draws with the stretch's first group as offset."""
    n = 2 ** 32 + 24
    base = dict(p=0.3, seed=11, stream_id=4, step=9)
    x = torch.ones(n, dtype=torch.float16, device=dev())
    assert ops.dropout(x, ops.DropoutSpec(**base), out=x) is not None
    ones = torch.ones(4104, dtype=torch.float16, device=dev())
    for start in (0, 2 ** 31 - 2048, 2 ** 32 - 4096, n - 4104):
        assert torch.equal(x[start:start + 4104], ops.dropout(ones, ops.DropoutSpec(**base, offset=start // 8)))


def test_two_streams_at_once(ops):
    x = torch.randn(3, 1 << 20, device=dev())
    specs = [ops.DropoutSpec(p=0.25, seed=s) for s in range(3)]
    want = [ops.dropout(x[i], specs[i]) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got.append(ops.dropout(x[i], specs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
