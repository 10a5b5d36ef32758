"""The operators' formulas and refusals, without a GPU."""
import ctypes

import pytest
import torch

from flashdp4review_b200 import _lib, core
from flashdp4review_b200.core import ops
from oracle import operators as P


def test_gradient_against_differences():
    """The formulas that the kernels are held to, against central differences of the forward formula (CPU, float64)."""
    gen = torch.Generator().manual_seed(1)
    x, dy = torch.randn(2, 5, 6, generator=gen).double(), torch.randn(2, 5, 6, generator=gen).double()
    gamma, beta = torch.randn(6, generator=gen).double(), torch.randn(6, generator=gen).double()
    keep = torch.rand(2, 5, 6, generator=gen) > 0.3
    for act in (None, "silu", "gelu", "gelu_tanh"):
        _, _, rstd, xhat, z = P.group_norm(x, gamma, beta, 3, 1e-5, act, keep, 0.3)
        got = P.group_norm_backward(dy, gamma, rstd, xhat, z, 3, act, keep, 0.3)["dx"][0]
        f = lambda v: (P.group_norm(v, gamma, beta, 3, 1e-5, act, keep, 0.3)[0] * dy).sum()
        h = 1e-5
        for i in ((0, 0, 0), (1, 4, 5), (0, 2, 3)):
            a, b = x.clone(), x.clone()
            a[i] += h
            b[i] -= h
            assert abs((f(a) - f(b)) / (2 * h) - got[i]) < 1e-6


# ---- refusals: before anything is launched, so without a GPU -------------------------------------------------------------
PTR, ODD = 8192, 8196          # not looked at by a call that is refused


def _drop(p=0.1, offset=0):
    return ctypes.byref(_lib.DropoutParams(p, 1, offset, 1, 1, None))


def _dp(std=0.0):
    return ctypes.byref(_lib.DPParams(1.0, 1.0, std, 0, 1, 1, 2, 1, 0, 1, None))


@pytest.mark.parametrize("change,status", [
    (dict(x=None), "ARG"), (dict(y=None), "ARG"), (dict(dtype=3), "DTYPE"), (dict(drop=None), "ARG"), (dict(drop=-0.1), "ARG"),
    (dict(drop=1.1), "ARG"), (dict(drop=float("nan")), "ARG"), (dict(offset=1 << 60), "ARG"), (dict(n=0, x=None), "OK"),
    (dict(y=PTR + 16), "ARG"), (dict(y=PTR - 36), "ARG"), (dict(res=PTR + 4100, y=PTR + 4096), "ARG")])
def test_dropout_entry_refuses(change, status):
    a = dict(x=PTR, res=None, y=PTR, n=10, dtype=0, drop=0.1, offset=0) | change
    d = None if a["drop"] is None else _drop(a["drop"], a["offset"])
    assert _lib.load().fdp_dropout(a["x"], a["res"], a["y"], a["n"], a["dtype"], d, None) == getattr(_lib, "FDP_OK" if status == "OK" else "FDP_ERR_" + status)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), "ARG"), (dict(gamma=None), "ARG"), (dict(beta=None), "ARG"), (dict(mean=None), "ARG"), (dict(B=0), "ARG"), (dict(T=-1), "ARG"),
    (dict(C=0), "ARG"), (dict(G=0), "ARG"), (dict(act=5), "ARG"), (dict(act=-1), "ARG"), (dict(dtype=7), "DTYPE"), (dict(pdt=3), "DTYPE"),
    (dict(G=3), "SHAPE"), (dict(C=8200, G=8), "SHAPE"), (dict(B=1 << 16, T=1 << 16), "SHAPE"), (dict(B=1 << 25, T=1, C=512), "SHAPE"),
    (dict(p=2.0), "ARG")])
def test_group_norm_entries_refuse(change, status):
    a = dict(x=PTR, gamma=PTR, beta=PTR, mean=PTR, B=2, T=4, C=16, G=4, act=0, dtype=0, pdt=0, p=0.1) | change
    want = getattr(_lib, "FDP_ERR_" + status)
    lib = _lib.load()
    shape = (a["B"], a["T"], a["C"], a["G"])
    assert lib.fdp_group_norm_fwd(a["x"], a["gamma"], a["beta"], PTR, a["mean"], PTR, *shape, 1e-5, a["act"], a["dtype"], a["pdt"], _drop(a["p"]),
                                  PTR, 1 << 40, None) == want
    assert lib.fdp_group_norm_bwd(PTR, a["x"], a["gamma"], a["beta"], a["mean"], PTR, PTR, PTR, PTR, None, None, *shape, a["act"], a["dtype"],
                                  a["pdt"], _drop(a["p"]), _dp(), PTR, 1 << 40, None) == want


def test_group_norm_backward_refuses_what_it_cannot_write():
    lib, shape = _lib.load(), (2, 4, 16, 4)
    rest = (*shape, 0, 0, 0, None)
    call = lambda g, dx, dg, db, p=_dp(): lib.fdp_group_norm_bwd(PTR, PTR, g, g, PTR, PTR, dx, dg, db, None, None, *rest, p, PTR, 1 << 40, None)
    assert call(PTR, None, None, None) == _lib.FDP_ERR_ARG           # nothing asked for
    assert call(PTR, PTR, PTR, None) == _lib.FDP_ERR_ARG             # one of the pair
    assert call(None, PTR, PTR, PTR) == _lib.FDP_ERR_ARG             # gradients of parameters that are not there
    assert call(PTR, PTR, PTR, PTR, None) == _lib.FDP_ERR_ARG
    assert call(PTR, PTR, PTR, PTR, _dp(-1.0)) == _lib.FDP_ERR_ARG
    for n in (lib.fdp_group_norm_fwd_workspace_bytes, lib.fdp_group_norm_bwd_workspace_bytes):
        assert n(*shape) > 0 and n(0, 4, 16, 4) == 0 and n(2, 4, 16, 0) == 0 and n(2, 4, 16, 3) == 0


@pytest.mark.parametrize("change,status", [
    (dict(x=None), "ARG"), (dict(w=None), "ARG"), (dict(e=None), "ARG"), (dict(y=None), "ARG"), (dict(rows=0), "ARG"), (dict(n=0), "ARG"),
    (dict(k=-5), "ARG"), (dict(dtype=9), "DTYPE"), (dict(out=-1), "DTYPE"), (dict(w=ODD), "ALIGN"), (dict(e=ODD), "ALIGN"),
    (dict(rows=1 << 30, n=1 << 30), "SHAPE"), (dict(k=(1 << 30) + 1), "SHAPE")])
def test_fp8_entries_refuse(change, status):
    a = dict(x=PTR, w=PTR, e=PTR, y=PTR, rows=4, n=8, k=16, dtype=0, out=0) | change
    assert _lib.load().fdp_fp8_matmul(a["x"], a["w"], a["e"], None, a["y"], a["rows"], a["n"], a["k"], a["dtype"], a["out"], PTR, 1 << 50,
                                      None) == getattr(_lib, "FDP_ERR_" + status)


def test_fp8_quantisers_refuse():
    lib = _lib.load()
    assert lib.fdp_fp8_quantize(None, PTR, PTR, 4, 8, 0, None) == _lib.FDP_ERR_ARG
    assert lib.fdp_fp8_quantize(PTR, ODD, PTR, 4, 8, 0, None) == _lib.FDP_ERR_ALIGN
    assert lib.fdp_fp8_quantize(PTR, PTR, PTR, 4, 8, 5, None) == _lib.FDP_ERR_DTYPE
    assert lib.fdp_fp8_quantize(PTR, PTR, PTR, 1 << 30, 1 << 20, 0, None) == _lib.FDP_ERR_SHAPE
    assert lib.fdp_fp8_quantize_weight(PTR, PTR, PTR, PTR, None, PTR, 4, 8, 0, None) == _lib.FDP_ERR_ARG
    assert lib.fdp_fp8_quantize_weight(PTR, PTR, ODD, PTR, PTR, PTR, 4, 8, 0, None) == _lib.FDP_ERR_ALIGN
    assert [lib.fdp_fp8_pitch(n) for n in (0, 1, 16, 17)] == [0, 16, 16, 32]
    assert [lib.fdp_fp8_exponent_bytes(*s) for s in ((0, 1), (1, 1), (128, 512), (129, 513))] == [0, 512, 512, 2048]
    assert lib.fdp_fp8_matmul_workspace_bytes(1, 1, 1) > 0 and lib.fdp_fp8_matmul_workspace_bytes(1, 0, 1) == 0


def test_operators_refuse():
    x = torch.zeros(2, 4, 16)
    w = torch.ones(16)
    for call in (lambda: core.dropout(x, core.DropoutSpec()), lambda: core.group_norm_forward(x, w, w, 4), lambda: core.fp8_quantize(x),
                 lambda: core.fp8_quantize_weight(x[0])):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    for bad in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(offset=-1), dict(offset=1 << 60)):
        with pytest.raises(ValueError):
            ops._drop(core.DropoutSpec(**bad))
    for counter in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="step counter"):
            ops._drop(core.DropoutSpec(step_device=counter))
    with pytest.raises(ValueError, match="activation"):
        ops._activation("swish")
    for args in ((x, w, w, 3), (x, w, w, 0), (x, w, None, 4)):
        with pytest.raises(ValueError):
            ops._group_norm_args(*args)
    for args in ((x[0, 0], w, w, 4), (x[:0], w, w, 4)):
        with pytest.raises(RuntimeError):
            ops._group_norm_args(*args)


def test_sizes_beyond_32_bits_are_refused():
    """(not taken modulo 2^32, as a size that fits)"""
    host, n = _lib.host(), (1 << 32) + 8
    one = torch.zeros(1, 1)
    w = torch.zeros(16, 16).to(torch.float8_e4m3fn)
    for call in (lambda: host.fp8_quantize(one.expand(n, 16), 0), lambda: host.fp8_quantize(one.expand(4, n), 0),
                 lambda: host.fp8_quantize_weight(one.expand(n, 16), 0), lambda: host.fp8_quantize_weight(one.expand(16, n), 0),
                 lambda: host.fp8_matmul(one.expand(n, 16), w, torch.zeros(512, dtype=torch.uint8), None, 0, 0),
                 lambda: host.group_norm_fwd(one.expand(2, n), None, None, 1, 8, 1e-5, 0, 0, 0, None),
                 lambda: host.group_norm_fwd(one.expand(n, 8), None, None, 1, 8, 1e-5, 0, 0, 0, None)):
        with pytest.raises(RuntimeError, match="too many"):
            call()


def test_products_in_8_bits_are_chosen_by_size():
    from flashdp4review_b200 import runtime
    assert not runtime.fp8_products() and not ops.fp8_product_ok(torch.bfloat16, 4096, 1024, 1024)
    runtime.set_fp8_products(True)
    try:
        assert ops.fp8_product_ok(torch.bfloat16, 128, 64, 64) and ops.fp8_product_ok(torch.float32, 1000, 999, 65)
        assert not ops.fp8_product_ok(torch.bfloat16, 127, 64, 64) and not ops.fp8_product_ok(torch.bfloat16, 128, 63, 64)
        assert not ops.fp8_product_ok(torch.float64, 128, 64, 64)
        runtime.set_input_grad_impl("library")
        assert not ops.fp8_product_ok(torch.bfloat16, 128, 64, 64)
    finally:
        runtime.set_input_grad_impl("auto")
        runtime.set_fp8_products(False)


def test_quantisation_formula():
    """What the oracle calls e4m3 is torch's, for every number of its range and every border between two."""
    v = torch.arange(-4480, 4481).double() / 10
    small = torch.arange(-400, 401).double() / 2 ** 12
    for t in (v, small):
        got = P.e4m3_blocks(torch.cat([t, torch.tensor([448.0])])[:, None].expand(-1, 128), 1)
        per_row = P.e4m3_blocks(torch.stack([t, torch.full_like(t, 448.0)], 1), 1)
        assert torch.equal(per_row[1], torch.ones_like(per_row[1]))
        assert torch.equal(per_row[0][:, 0], t.float().to(torch.float8_e4m3fn).double())
        assert torch.isfinite(got[0]).all()
