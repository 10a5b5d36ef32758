"""Group norm, channels last, against float64: forward, input gradient, per-sample-clipped parameter gradients.

Tolerances.  A stored result is off by at most half a step of its type (finfo.eps / 2 of its value).  What comes before that is
fp32: a result passes through fewer than 64 roundings in a row -- a thread's chain of at most 4 + T / (chunks * rows at a time) additions, the
chunks' chain, a dozen operations of the formula, and at the sizes here never more -- each at most 2^-24 of the sum of
the magnitudes that it is made of, which the oracle returns: 2^-18 of that in all.  The fast exponential and reciprocal
(2^-21 relative, for every type) are inside the same 2^-18.  Where a relu's argument is within 2^-16 of zero its slope may come out as
either of 0 and 1; sums may then miss those terms.
"""
import math

import pytest
import torch

from oracle import dp_oracle as O
from oracle import operators as P
from gpu_util import dev

pytestmark = pytest.mark.gpu
FP32 = 2.0 ** -18


@pytest.fixture(scope="module")
def ops():
    from flashdp4review_b200.core import ops
    return ops


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, mag, dtype, extra=None):
    got = got.detach().double().cpu()
    tol = half_step(dtype) * want.abs() + FP32 * mag + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    if extra is not None:
        tol = tol + extra
    bad = (got - want).abs() > tol
    assert not bad.any(), ((got - want).abs() / tol).max()


def case(B, T, C, dtype, seed, mean=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, T, C, generator=gen) * 1.3 + torch.randn(C, generator=gen) * mean).to(dtype)
    dy = (torch.randn(B, T, C, generator=gen) * 0.1 * torch.exp(torch.randn(B, 1, 1, generator=gen))).to(dtype)
    return x, dy, 1 + 0.2 * torch.randn(C, generator=gen), 0.2 * torch.randn(C, generator=gen)


def check(ops, x, dy, gamma, beta, G, act, spec=None, eps=1e-5, pdtype=torch.float32):
    B, T, C = x.shape
    dtype = x.dtype
    keep = None if spec is None else torch.from_numpy(P.keep_mask(x.numel(), spec.p, spec.seed, spec.stream_id, spec.step, spec.offset)).view(x.shape)
    p = 0.0 if spec is None else spec.p
    w = None if gamma is None else gamma.to(pdtype)
    b = None if beta is None else beta.to(pdtype)
    y, mean, rstd, xhat, z = P.group_norm(x, w, b, G, eps, act, keep, p)
    scale = 1.0 if spec is None else 1 / (1 - p) if p < 1 else 0.0
    xd, dyd = x.to(dev()), dy.to(dev())
    wd, bd = (None, None) if w is None else (w.to(dev()), b.to(dev()))
    gy, st = ops.group_norm_forward(xd, wd, bd, G, eps, activation=act, dropout=spec)
    # what z is made of: the difference x - mean (rounded against x and the mean), times rstd * gamma, and beta.  The mean is
    # a number p of the data plus the mean of x - p, whose roundings are relative to the mean of |x - p| <= std + |p - mean|: over the
    # threads' several p two standard deviations, which times rstd is 2 -- also where x and the mean are next to zero.
    by = lambda a: a.repeat_interleave(C // G, 1)[:, None]
    big = ((x.double().abs() + by(mean.abs())) * by(rstd) + 2) * (1 if w is None else w.double().abs()) + (0 if b is None else b.double().abs())
    close(gy, y, big * 1.13 * scale * (1 if keep is None else keep), dtype)
    close(st["mean"], mean, x.double().abs().amax((1, 2))[:, None].expand(B, G), torch.float32)
    close(st["rstd"], rstd, rstd * (1 + (mean * rstd).square()), torch.float32)
    clip = 0.7 * P.clipped_mean(P.group_norm_backward(dy, w, rstd, xhat, z, G, act, keep, p)["dgamma"][0], 1e9, 1.0)[1].median().item() + 1e-30
    res = ops.dp_group_norm_backward(dyd, xd, wd, bd, st["mean"], st["rstd"], G, clip, 1.0, activation=act, dropout=spec, return_norms=True)
    want = P.group_norm_backward(dy, w, rstd, xhat, z, G, act, keep, p)
    # rounding of xhat reaches the slope: |gz| moves by at most |act''| <= 1.13 of the rounding of z
    slope_err = FP32 * big * dy.double().abs() * scale if act is not None else torch.zeros_like(big)
    border = torch.zeros_like(big)
    if act == "relu":
        border = (z.abs() < 2.0 ** -16) * dy.double().abs() * scale
    gmul = 1 if w is None else w.double().abs()
    n = T * C // G
    grp = lambda a: by(a.reshape(B, T, G, C // G).sum((1, 3)) / n)
    lost = slope_err + border
    xerr = FP32 * ((x.double().abs() + by(mean.abs())) * by(rstd) + 2)       # of xhat
    u, gz = want["gz"] * gmul, want["gz"].abs()
    extra = by(rstd) * (lost * gmul + grp(lost * gmul) + xhat.abs() * grp(lost * gmul * xhat.abs() + u.abs() * xerr) + xerr * grp((u * xhat).abs()))
    close(res[0], want["dx"][0], want["dx"][1], dtype, extra)
    if w is None:
        assert res[1] is None and res[2] is None
        return
    for got, norms, name, more in ((res[1], res[3], "dgamma", (lost * xhat.abs() + gz * xerr).sum(1)), (res[2], res[4], "dbeta", lost.sum(1))):
        per, mag = want[name]
        mean_, n_ = P.clipped_mean(per, clip, 1.0)
        err = FP32 * mag + more                                              # of the per-sample gradient, element by element
        nerr = err.square().sum(1).sqrt() + FP32 * n_
        assert ((norms.double().cpu() - n_).abs() <= nerr + 1e-30).all()
        f = torch.from_numpy(O.clip_factor(n_.numpy(), clip, 1.0))
        # factor: relative error at most that of the norm; then B sums
        rel = torch.where(n_ > 0, nerr / n_.clamp(min=1e-30), 0.0) + FP32
        tol = ((err * f[:, None]) + (per.abs() * (f * rel)[:, None])).sum(0) / B
        close(got, mean_, torch.zeros_like(mean_), pdtype, tol + 1e-30)


SHAPES = [(2, 1, 32, 4), (3, 5, 64, 32), (1, 7, 8, 1), (4, 64, 128, 32), (2, 200, 320, 32), (3, 33, 90, 6), (2, 50, 7, 7),
          (1, 3, 2056, 8), (2, 9, 4096, 32), (1, 2, 8192, 1), (2, 1000, 48, 1), (5, 17, 1026, 2), (300, 4, 16, 2), (1, 4099, 24, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_float64(ops, shape, dtype):
    B, T, C, G = shape
    check(ops, *case(B, T, C, dtype, seed=B * 7919 + T * 31 + C), G, None)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 50, 64, 8), (2, 21, 30, 5)])
def test_activations(ops, act, dtype, shape):
    B, T, C, G = shape
    check(ops, *case(B, T, C, dtype, seed=5), G, act)


@pytest.mark.parametrize("p", [0.1, 0.5, 1.0, 0.0])
@pytest.mark.parametrize("shape", [(3, 40, 64, 8), (2, 21, 30, 5)])
def test_dropout_behind_it(ops, p, shape):
    B, T, C, G = shape
    spec = ops.DropoutSpec(p=p, seed=0x123456789ABCDEF0, stream_id=9, step=4, offset=77)
    x, dy, gamma, beta = case(B, T, C, torch.bfloat16, seed=6)
    check(ops, x, dy, gamma, beta, G, "silu", spec)
    # the mask is that of the operator on its own
    y, _ = ops.group_norm_forward(x.to(dev()), gamma.to(dev()), (beta + 5).to(dev()), G, dropout=spec)
    if p < 1:
        assert torch.equal(y != 0, ops.dropout(torch.ones_like(y), spec) != 0)


@pytest.mark.parametrize("pdtype", [torch.float32, torch.bfloat16, torch.float16])
def test_parameter_types_and_no_parameters(ops, pdtype):
    x, dy, gamma, beta = case(3, 30, 64, torch.bfloat16, seed=8)
    check(ops, x, dy, gamma, beta, 8, "silu", pdtype=pdtype)
    check(ops, x, dy, None, None, 8, "silu")


@pytest.mark.parametrize("offset", [30.0, 1000.0])
def test_a_mean_far_from_zero(ops, offset):
    """Deviations are taken about numbers of the data, not about zero: the variance keeps its digits."""
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(2, 300, 64, generator=gen) + offset)
    x[0, 0] = -3 * offset                     # ... and the first row is not like the others
    check(ops, x, torch.randn(2, 300, 64, generator=gen), torch.ones(64), torch.zeros(64), 8, None)


def test_equal_numbers_have_no_spread(ops):
    x = torch.full((2, 40, 32), 7.25, dtype=torch.bfloat16, device=dev())
    y, st = ops.group_norm_forward(x, torch.ones(32, device=dev()), torch.full((32,), 0.5, device=dev()), 4)
    assert torch.equal(y, torch.full_like(y, 0.5))
    assert torch.allclose(st["rstd"], torch.full_like(st["rstd"], 1e-5 ** -0.5), rtol=1e-6)


def test_a_sample_that_is_not_finite_stays_alone(ops):
    x, dy, gamma, beta = (t.to(dev()) for t in case(4, 50, 64, torch.bfloat16, seed=9))
    y0, st0 = ops.group_norm_forward(x, gamma, beta, 8, activation="silu")
    dx0 = ops.dp_group_norm_backward(dy, x, gamma, beta, st0["mean"], st0["rstd"], 8, 1.0, 1.0, activation="silu")[0]
    x2 = x.clone()
    x2[1, 3, 5], x2[2, 0, 0] = math.nan, math.inf
    y, st = ops.group_norm_forward(x2, gamma, beta, 8, activation="silu")
    dx, _, _, ng, nb = ops.dp_group_norm_backward(dy, x2, gamma, beta, st["mean"], st["rstd"], 8, 1.0, 1.0, activation="silu", return_norms=True)
    for b in (0, 3):
        assert torch.equal(y[b], y0[b]) and torch.equal(dx[b], dx0[b])
    assert torch.isinf(ng[1:3]).all() and torch.isfinite(ng[[0, 3]]).all()


def test_views_and_unaligned_storage(ops):
    """Inputs that are not contiguous, or not on a 16-byte boundary, give what a fresh copy gives."""
    x, dy, gamma, beta = (t.to(dev()) for t in case(3, 40, 64, torch.bfloat16, seed=10))
    big = torch.zeros(3 * 40 * 64 + 1, dtype=x.dtype, device=dev())
    off = big[1:].view(3, 40, 64).copy_(x)
    assert off.data_ptr() % 16 != 0
    strided = x.transpose(0, 1).contiguous().transpose(0, 1)
    want = ops.group_norm_forward(x, gamma, beta, 8, activation="gelu")[0]
    for v in (off, strided):
        y, st = ops.group_norm_forward(v, gamma, beta, 8, activation="gelu")
        assert (y.float() - want.float()).abs().max() <= 2 ** -8 * want.float().abs().max()
        a = ops.dp_group_norm_backward(dy, v, gamma, beta, st["mean"], st["rstd"], 8, 1.0, 1.0, activation="gelu")
        b = ops.dp_group_norm_backward(dy, x, gamma, beta, st["mean"], st["rstd"], 8, 1.0, 1.0, activation="gelu")
        for u, v2 in zip(a, b):
            assert (u.float() - v2.float()).abs().max() <= 2 ** -8 * v2.float().abs().max() + 1e-12


def test_noise_divisor_and_repeatability(ops):
    x, dy, gamma, beta = (t.to(dev()) for t in case(4, 100, 64, torch.bfloat16, seed=11))
    _, st = ops.group_norm_forward(x, gamma, beta, 8)
    args = (dy, x, gamma, beta, st["mean"], st["rstd"], 8, 1.0, 1.0)
    ns = ops.NoiseSpec(std=0.5, seed=77, param_id=5, param_id2=6, step=2)
    r0, r1, r2 = (ops.dp_group_norm_backward(*args, noise=n, batch_divisor=4) for n in (None, ns, ns))
    r8 = ops.dp_group_norm_backward(*args, batch_divisor=8)
    for a, b in zip(r1, r2):
        assert torch.equal(a, b)
    assert torch.equal(r0[0], r1[0])
    assert torch.equal(r0[1], 2 * r8[1]) and torch.equal(r0[2], 2 * r8[2])
    for k, pid in ((1, 5), (2, 6)):
        z = torch.from_numpy(O.gaussian_noise(64, 0.5, 77, pid, 2))
        assert ((r1[k] - r0[k]).double().cpu() - z).abs().max() < 3e-6


def test_many_chunks_and_many_samples(ops):
    """Statistics put together by a launch of their own (more than 64 chunks a sample), and more samples than the clipped sum keeps
    factors of in shared memory."""
    check(ops, *case(1, 9001, 96, torch.bfloat16, seed=3), 6, "silu")
    check(ops, *case(1, 9001, 96, torch.float32, seed=4), 6, None)
    B, T, C, G = 9000, 2, 8, 2
    x, dy, w, b = case(B, T, C, torch.float32, seed=5)
    y, mean, rstd, xhat, z = P.group_norm(x, w, b, G, 1e-5, None, None, 0.0)
    _, st = ops.group_norm_forward(x.to(dev()), w.to(dev()), b.to(dev()), G)
    res = ops.dp_group_norm_backward(dy.to(dev()), x.to(dev()), w.to(dev()), b.to(dev()), st["mean"], st["rstd"], G, 0.1, 1.0, return_norms=True)
    want = P.group_norm_backward(dy, w, rstd, xhat, z, G, None, None, 0.0)
    xerr = FP32 * ((x.double().abs() + mean.abs().repeat_interleave(C // G, 1)[:, None]) * rstd.repeat_interleave(C // G, 1)[:, None] + 2)
    for got, norms, name, more in ((res[1], res[3], "dgamma", (dy.double().abs() * xerr).sum(1)), (res[2], res[4], "dbeta", 0.0)):
        per, mag = want[name]
        mean_, n_ = P.clipped_mean(per, 0.1, 1.0)
        err = FP32 * mag + more
        nerr = err.square().sum(1).sqrt() + FP32 * n_
        assert ((norms.double().cpu() - n_).abs() <= nerr + 1e-30).all()
        f = torch.from_numpy(O.clip_factor(n_.numpy(), 0.1, 1.0))
        # the sum over the samples is a chain of at most B additions, each off by 2^-24 of the magnitudes so far
        tol = (err * f[:, None] + per.abs() * (f * (nerr / n_.clamp(min=1e-30) + FP32 + B * 2.0 ** -24))[:, None]).sum(0) / B
        close(got, mean_, torch.zeros_like(mean_), torch.float32, tol)


def test_more_than_2_31_elements(ops):
    """Samples of 512 equal stretches: their statistics and the sums of the backward are a stretch's (times 512), and every stretch
    of a result has the same bits.  A thread's chain has fewer than 4096 rows (2^21 in at least 222 chunks and three row classes),
    so sums are off by at most 2^-12 of their magnitudes, and the variance, which two of them make, by 2^-11."""
    B, T, C, G, N = 2, 4096, 520, 8, 512
    x, dy, w, b = case(B, T, C, torch.bfloat16, seed=6)
    big_x, big_dy = x.to(dev()).repeat(1, N, 1), dy.to(dev()).repeat(1, N, 1)
    assert big_x.numel() > 2 ** 31
    y, st = ops.group_norm_forward(big_x, w.to(dev()), b.to(dev()), G, activation="silu")
    got = y.view(B, N, T, C)
    assert all(torch.equal(got[:, i], got[:, 0]) for i in range(1, N))
    want, mean, rstd, xhat, z = P.group_norm(x, w, b, G, 1e-5, "silu", None, 0.0)
    by = lambda a: a.repeat_interleave(C // G, 1)[:, None]
    lost = 2.0 ** -11
    zerr = lost * (((x.double().abs() + by(mean.abs())) * by(rstd) + 2) * w.double().abs() + b.double().abs())
    close(got[:, 0], want, 1.13 * zerr / FP32, torch.bfloat16)
    del y, got
    res = ops.dp_group_norm_backward(big_dy, big_x, w.to(dev()), b.to(dev()), st["mean"], st["rstd"], G, 1e30, 1.0, activation="silu")
    got = res[0].view(B, N, T, C)
    assert all(torch.equal(got[:, i], got[:, 0]) for i in range(1, N))
    back = P.group_norm_backward(dy, w, rstd, xhat, z, G, "silu", None, 0.0)
    gerr = 1.13 * zerr * dy.double().abs() + lost * back["gz"].abs()          # of gz: |act''| <= 1.13
    grp = lambda a: by(a.reshape(B, T, G, C // G).sum((1, 3)) / (T * C // G))
    gmul = w.double().abs()
    xerr = lost * ((x.double().abs() + by(mean.abs())) * by(rstd) + 2)
    u = back["gz"].abs() * gmul
    extra = by(rstd) * (gerr * gmul + grp(gerr * gmul) + xhat.abs() * grp(gerr * gmul * xhat.abs() + u * xerr) + xerr * grp(u * xhat.abs()))
    close(got[:, 0], back["dx"][0], back["dx"][1] * lost / FP32, torch.bfloat16, extra)
    for g, name, more in ((res[1], "dgamma", (gerr * xhat.abs() + back["gz"].abs() * xerr).sum(1)), (res[2], "dbeta", gerr.sum(1))):
        per, mag = back[name]
        close(g, N * per.mean(0), torch.zeros(C), torch.float32, N * (lost * mag + more).mean(0))


def test_a_variance_beyond_fp32(ops):
    """Finite numbers whose squared deviations overflow: rstd is 0 and the output the bias, as torch's; the other groups and samples
    are as they would be."""
    gen = torch.Generator().manual_seed(12)
    for B, T, C in ((3, 40, 64), (6, 400, 512)):              # both passes in one kernel; a kernel a pass
        x = torch.randn(B, T, C, generator=gen)
        gamma, beta = torch.rand(C, generator=gen) + 0.5, torch.randn(C, generator=gen)
        y0, st0 = ops.group_norm_forward(x.to(dev()), gamma.to(dev()), beta.to(dev()), 8)
        x[1, :, :C // 8] *= 1e25
        x[0, 3, C // 8] = 1e30                              # (one such number is enough)
        y, st = ops.group_norm_forward(x.to(dev()), gamma.to(dev()), beta.to(dev()), 8)
        assert (st["rstd"][1, 0] == 0).all() and (st["rstd"][0, 1] == 0).all()
        cg = C // 8
        assert torch.equal(y[1, :, :cg], beta[:cg].to(dev()).expand(T, cg)) and torch.equal(y[0, :, cg:2 * cg], beta[cg:2 * cg].to(dev()).expand(T, cg))
        assert torch.equal(y[2], y0[2]) and torch.equal(y[1, :, cg:], y0[1, :, cg:]) and torch.equal(y[0, :, :cg], y0[0, :, :cg])
        assert torch.equal(y[0, :, 2 * cg:], y0[0, :, 2 * cg:])
        dx, dg, db = ops.dp_group_norm_backward(torch.full_like(y, 1e-2), x.to(dev()), gamma.to(dev()), beta.to(dev()), st["mean"], st["rstd"], 8, 1.0, 1.0)
        assert (dx[1, :, :cg] == 0).all() and all(torch.isfinite(t).all() for t in (dx, dg, db))


# ---- tensors that take a kernel a pass -------------------------------------------------------------------------------------
def launches(call):
    from flashdp4review_b200 import _lib
    lib = _lib.load()
    before = lib.fdp_launch_count()
    res = call()
    return lib.fdp_launch_count() - before, res


def takes_a_kernel_a_pass(ops, x, w, b, G, act, spec):
    """(and not clusters: one launch forward, two backward; nor statistics put together by a launch of their own)"""
    n, (_, st) = launches(lambda: ops.group_norm_forward(x, w, b, G, activation=act, dropout=spec))
    m, _ = launches(lambda: ops.dp_group_norm_backward(x, x, w, b, st["mean"], st["rstd"], G, 1.0, 1.0, activation=act, dropout=spec))
    return n == 2 and m == 3


# A thread's chain there is of at most 22 rows, a sample has at most 64 chunks, eight of which a thread adds up at most, then eight
# threads': fewer than the 64 roundings in a row that the tolerances count.
GRID = [(6, 400, 512, 8, torch.bfloat16), (8, 1600, 90, 6, torch.float16), (8, 1600, 91, 7, torch.bfloat16), (8, 40, 4104, 8, torch.bfloat16),
        (8, 600, 130, 5, torch.float32), (8, 600, 132, 4, torch.float32), (8, 1600, 90, 90, torch.bfloat16), (8, 40, 4101, 3, torch.float16)]


@pytest.mark.parametrize("act,p", [(None, 0.0), ("gelu_tanh", 0.3), ("silu", 0.0)])
@pytest.mark.parametrize("shape", GRID)
def test_a_kernel_a_pass(ops, shape, act, p):
    """Several samples of more than 2 MB together, with whole vectors, rows that are only even, odd rows, and rows of more columns than
    a block has threads; clipping that bites on some of the samples."""
    B, T, C, G, dtype = shape
    spec = ops.DropoutSpec(p=p, seed=11, stream_id=2, step=3) if p else None
    x, dy, gamma, beta = case(B, T, C, dtype, seed=B + T + C)
    assert takes_a_kernel_a_pass(ops, x.to(dev()), gamma.to(dev()), beta.to(dev()), G, act, spec)
    check(ops, x, dy, gamma, beta, G, act, spec)


@pytest.mark.parametrize("dropped", [False, True])
def test_a_kernel_a_pass_on_unaligned_storage(ops, dropped):
    """What an aligned copy gives, each within its roundings of float64: numbers one by one in place of vectors."""
    x, dy, gamma, beta = case(6, 400, 512, torch.bfloat16, seed=21)
    spec = ops.DropoutSpec(p=0.2, seed=5) if dropped else None
    # a view off 16 bytes stays one through .to() and .contiguous() on its own device
    off = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=dev())[1:].view(t.shape).copy_(t)
    xo, do = off(x), off(dy)
    assert xo.data_ptr() % 16 and takes_a_kernel_a_pass(ops, xo, gamma.to(dev()), beta.to(dev()), 8, "silu", spec)

    class Off:
        """a tensor whose copy on the device is off 16 bytes"""
        def __init__(self, host, there):
            self.host, self.there = host, there

        def __getattr__(self, name):
            return getattr(self.host, name)

        def to(self, *_):
            return self.there

    check(ops, Off(x, xo), Off(dy, do), gamma, beta, 8, "silu", spec)


@pytest.mark.parametrize("shape", [(6, 400, 512, 8), (4, 64, 128, 32)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_parts_of_a_backward(ops, shape, p):
    """Without the input's gradient, or without the parameters', the rest has the same bits."""
    B, T, C, G = shape
    x, dy, gamma, beta = (t.to(dev()) for t in case(B, T, C, torch.bfloat16, seed=22))
    spec = ops.DropoutSpec(p=p, seed=5) if p else None
    _, st = ops.group_norm_forward(x, gamma, beta, G, activation="gelu", dropout=spec)
    back = lambda **k: ops.dp_group_norm_backward(dy, x, gamma, beta, st["mean"], st["rstd"], G, 0.5, 1.0, activation="gelu", dropout=spec, return_norms=True, **k)
    whole, no_dx, no_dw = back(), back(need_dx=False), back(need_dw=False)
    assert no_dx[0] is None and all(torch.equal(a, b) for a, b in zip(whole[1:], no_dx[1:]))
    assert torch.equal(no_dw[0], whole[0]) and no_dw[1:] == (None,) * 4


def test_many_samples_in_a_kernel_a_pass(ops):
    """More samples than the clipped sum keeps factors of in shared memory, of more than 2 MB together."""
    B, T, C, G = 9000, 8, 16, 2
    x, dy, w, b = case(B, T, C, torch.float32, seed=25)
    y, mean, rstd, xhat, z = P.group_norm(x, w, b, G, 1e-5, None, None, 0.0)
    n, (_, st) = launches(lambda: ops.group_norm_forward(x.to(dev()), w.to(dev()), b.to(dev()), G))
    assert n == 2
    res = ops.dp_group_norm_backward(dy.to(dev()), x.to(dev()), w.to(dev()), b.to(dev()), st["mean"], st["rstd"], G, 0.2, 1.0, return_norms=True)
    want = P.group_norm_backward(dy, w, rstd, xhat, z, G, None, None, 0.0)
    xerr = FP32 * ((x.double().abs() + mean.abs().repeat_interleave(C // G, 1)[:, None]) * rstd.repeat_interleave(C // G, 1)[:, None] + 2)
    for got, norms, name, more in ((res[1], res[3], "dgamma", (dy.double().abs() * xerr).sum(1)), (res[2], res[4], "dbeta", 0.0)):
        per, mag = want[name]
        mean_, n_ = P.clipped_mean(per, 0.2, 1.0)
        assert 0 < (n_ > 0.2).sum() < B
        err = FP32 * mag + more
        nerr = err.square().sum(1).sqrt() + FP32 * n_
        assert ((norms.double().cpu() - n_).abs() <= nerr + 1e-30).all()
        f = torch.from_numpy(O.clip_factor(n_.numpy(), 0.2, 1.0))
        # the sum over the samples is a chain of at most B additions, each off by 2^-24 of the magnitudes so far
        tol = (err * f[:, None] + per.abs() * (f * (nerr / n_.clamp(min=1e-30) + FP32 + B * 2.0 ** -24))[:, None]).sum(0) / B
        close(got, mean_, torch.zeros_like(mean_), torch.float32, tol)
