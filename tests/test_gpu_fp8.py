"""Products in e4m3 with a scale for each block of 128: quantisation bit for bit, products against float64.

Tolerance of a product: products of two e4m3 numbers are exact in fp32, and so are powers of two as scales.  One matrix
instruction adds 32 products to the accumulator, each cut off at no less than 24 bits below the largest of them, which is at most
the sum of all magnitudes: products lose 33 * 2^-24 of what their own instruction adds, 33 * 2^-24 of the sum over all; the accumulator
one bit of its last place, 2^-23 of the sum, in each of four instructions for every 128 numbers, of which at most 8 * 128 go by for an
fp32 output before an accumulator starts anew (and is added with one rounding); then the bias's and the last rounding.
(48 + 8 * blocks) * 2^-24 of the sum of all magnitudes, at most 8 blocks and one more a chain for fp32, and half a step of the output type.
"""
import math

import pytest
import torch

from oracle import operators as P
from gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from flashdp4review_b200.core import ops
    return ops


def wide(gen, r, c, dtype):
    """numbers over many orders of magnitude, with rows and blocks of their own size"""
    x = torch.randn(r, c, generator=gen) * torch.exp(2 * torch.randn(r, 1, generator=gen)) * torch.exp(torch.randn(1, c, generator=gen))
    return x.to(dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 8), (17, 127), (16, 128), (33, 129), (5, 1000), (40, 640), (130, 513)])
def test_quantisation(ops, dtype, shape):
    gen = torch.Generator().manual_seed(shape[0] * 1000 + shape[1])
    x = wide(gen, *shape, dtype)
    if shape[0] > 2 and shape[1] > 100:
        x[0] = 0.0
        x[1, 3], x[1, 50], x[2, 77] = math.nan, math.inf, -math.inf
        x[2, :20] = 448.0                              # the largest number stays itself ...
        x[min(4, shape[0] - 1), 7] = 449.0 if dtype != torch.bfloat16 else 452.0       # ... and what is above it moves the scale
    q, s = ops.fp8_quantize(x.to(dev()))
    v, scale = P.e4m3_blocks(x, 1)
    assert torch.equal(s.cpu().double(), scale)
    assert q.shape == x.shape and same(q.float().cpu().double(), v)
    w8 = ops.fp8_quantize_weight(x.to(dev()))
    v, scale = P.e4m3_blocks(x, 128)
    assert torch.equal(w8.scales.cpu().double(), scale)
    assert same(w8.values.float().cpu().double(), v) and same(w8.values_t.float().cpu().double(), v.t())


def test_smallest_and_largest_numbers(ops):
    x = torch.zeros(6, 256)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[3, 1] = 1e-45, 3.4e38, 2.0 ** -126, 448 * 2.0 ** 10, 2.0 ** -20
    x[4, :128], x[4, 128:] = 1e-38, 1e30
    q, s = ops.fp8_quantize(x.to(dev()))
    v, scale = P.e4m3_blocks(x, 1)
    assert torch.equal(s.cpu().double(), scale) and torch.equal(q.float().cpu().double(), v)


def check(ops, M, N, K, dtype, out_dtype=None, bias=True, layout="out_in", seed=0):
    gen = torch.Generator().manual_seed(seed + M * 7 + N * 3 + K)
    x = wide(gen, M, K, torch.float32).clamp(-300, 300).to(dtype)
    w = (torch.randn(N, K, generator=gen) * 0.05).to(dtype)
    b = torch.randn(N, generator=gen).to(dtype) if bias else None
    g = (torch.randn(M, N, generator=gen) * 1e-2).to(dtype)
    stored = w if layout == "out_in" else w.t().contiguous()
    w8 = ops.fp8_quantize_weight(stored.to(dev()), layout)
    y = ops.fp8_linear_forward(x.to(dev()), w8, None if b is None else b.to(dev()), out_dtype=out_dtype)
    dx = ops.fp8_linear_input_grad(g.to(dev()), w8, out_dtype=out_dtype)
    xq, gq = (P.e4m3_stands_for(t, 1).to(dev()) for t in (x, g))
    wq = P.e4m3_stands_for(w, 128).to(dev())
    t = out_dtype or dtype
    for got, a, m, extra, k in ((y, xq, wq.t(), 0.0 if b is None else b.double().to(dev()), K), (dx, gq, wq, 0.0, N)):
        assert got.dtype == t
        want = a @ m + extra
        mag = a.abs() @ m.abs() + (extra.abs() if b is not None and got is y else 0.0)
        blocks = -(-k // 128)
        lost = 48 + (8 * blocks if t != torch.float32 else 8 * min(blocks, 8) + blocks / 8)
        tol = torch.finfo(t).eps / 2 * want.abs() + lost * 2.0 ** -24 * mag + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        err = (got.double() - want).abs()
        assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 64, 64), (1, 1, 1), (5, 7, 9), (3, 130, 2000), (128, 128, 128), (129, 257, 255), (300, 1000, 999),
                                   (1000, 96, 4096), (512, 768, 768), (64, 4096, 200), (17, 24, 16385)])
def test_products(ops, dtype, shape):
    check(ops, *shape, dtype)


@pytest.mark.parametrize("shape", [(2560, 2048, 384), (2500, 2041, 130), (2561, 2056, 1024), (20000, 256, 640), (300, 20001, 129)])
@pytest.mark.parametrize("out", [None, torch.float32])
def test_products_of_many_tiles(ops, shape, out):
    check(ops, *shape, torch.bfloat16, out_dtype=out, bias=out is None)


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
def test_both_layouts_and_leading_axes(ops, layout):
    check(ops, 200, 300, 400, torch.bfloat16, layout=layout)
    x = torch.randn(2, 5, 3, 64, device=dev())
    w8 = ops.fp8_quantize_weight(torch.randn(32, 64, device=dev()))
    y = ops.fp8_linear_forward(x, w8)
    assert y.shape == (2, 5, 3, 32) and torch.equal(y.view(30, 32), ops.fp8_linear_forward(x.view(30, 64), w8))
    t = x.transpose(0, 2)
    assert torch.equal(ops.fp8_linear_forward(t, w8), y.transpose(0, 2))


@pytest.mark.parametrize("M", [256, 4096])
def test_rows_stay_apart(ops, M):
    """No number of a row depends on another row: with all the other rows changed, and with NaNs in them, a row's bits are the
    same.  (Per-sample clipping bounds what a sample contributes only if nothing else carries it.)"""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(M, 640, generator=gen).to(torch.bfloat16).to(dev())
    w8 = ops.fp8_quantize_weight((torch.randn(1280, 640, generator=gen) * 0.05).to(torch.bfloat16).to(dev()))
    y = ops.fp8_linear_forward(x, w8)
    x2 = x * 1000
    x2[::3] = math.nan
    x2[7], x2[100] = x[7], x[100]
    y2 = ops.fp8_linear_forward(x2, w8)
    assert torch.equal(y[7], y2[7]) and torch.equal(y[100], y2[100]) and torch.isnan(y2[0]).all()


def test_repeated_calls_give_the_same_bits(ops):
    gen = torch.Generator().manual_seed(5)
    for M, N, K in ((64, 768, 4096), (3000, 2100, 500)):
        x = torch.randn(M, K, generator=gen).to(dev())
        w8 = ops.fp8_quantize_weight(torch.randn(N, K, generator=gen).to(dev()))
        a = ops.fp8_linear_forward(x, w8)
        for _ in range(3):
            assert torch.equal(a, ops.fp8_linear_forward(x, w8))


@pytest.mark.parametrize("N,K", [(64, 2056), (2056, 128), (2057, 128)])
def test_more_than_2_31_elements(ops, N, K):
    """Rows at the end of an operand or a result with more than 2^31 numbers are what they are by themselves (in tiles and orders of
    accumulation that may be others: 48 + 8 a K block roundings at most on either side)."""
    M, last = 2 ** 20 + 136, 300
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(4096, K, generator=gen).to(torch.bfloat16).to(dev()).repeat(257, 1)[:M]
    x[-last:] = torch.randn(last, K, generator=gen).to(torch.bfloat16).to(dev())
    w = torch.randn(N, K, generator=gen).to(torch.bfloat16).to(dev())
    w8 = ops.fp8_quantize_weight(w)
    assert x.numel() > 2 ** 31 or M * N > 2 ** 31
    y = ops.fp8_linear_forward(x, w8)
    few = ops.fp8_linear_forward(x[-last:], w8, out_dtype=torch.float32)
    mag = ops.fp8_linear_forward(x[-last:].abs(), ops.fp8_quantize_weight(w.abs()), out_dtype=torch.float32)
    tol = torch.finfo(torch.bfloat16).eps / 2 * few.abs() + 2 * (48 + 8 * -(-K // 128)) * 2.0 ** -24 * mag * 1.01
    assert ((y[-last:].float() - few).abs() <= tol).all()
    assert torch.equal(y[4096 * 254:4096 * 255], y[:4096])      # (of the 256th stretch 164 rows are among the last)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_long_contraction(ops, dtype):
    """262144 numbers in one accumulator, without a cut along them (144 tiles of 128 x 128).  Numbers that e4m3 holds exactly, so the
    quantisation loses nothing; the first blocks are much larger than the others, so that what comes after them is cut off.  An accumulator runs
    for 128 blocks at most, 512 instructions each off by a unit in the last place, 2^-23: with 16-bit outputs too the sum is off by less
    than 2^-14 of the magnitudes for that (and 48 roundings of the rest; 2^-24 for each of the 16 sums after), then by half a step."""
    M = N = 1536
    K = 1 << 18
    gen = torch.Generator(device=dev()).manual_seed(7)
    some = lambda r: (torch.randint(8, 16, (r, K), device=dev(), generator=gen) / 8.0).to(dtype)
    x, w = some(M), some(N)
    x[:, :128] *= 2.0 ** 12
    x *= 2.0 ** -8
    w *= 2.0 ** -8
    y = ops.fp8_linear_forward(x, ops.fp8_quantize_weight(w))
    want = x[:64].double() @ w.double().t()
    assert torch.isfinite(y).all()
    tol = torch.finfo(dtype).eps / 2 * want + (2.0 ** -14 + 64 * 2.0 ** -24) * want
    err = (y[:64].double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()
    # roundings to the output's type go both ways; what is cut off goes one: the mean of 98304 relative errors shows it alone
    assert ((y[:64].double() - want) / want).mean().abs() <= 2.0 ** -14
