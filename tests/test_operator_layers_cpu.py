"""The layers of the operators around a stand-in for the kernels, without a GPU: what they do to tensors, masks and graphs."""
import ctypes

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

import flashdp4review_b200 as fdp
from flashdp4review_b200 import _lib, runtime
from flashdp4review_b200.core import ops
from flashdp4review_b200.layers import _common
from oracle import operators as P


@pytest.fixture
def on_cpu(monkeypatch):
    """dropout by its formula, with the operator's manner of taking and returning tensors"""
    def dropout(input, spec, residual=None, out=None):
        assert residual is None or (residual.shape == input.shape and residual.dtype == input.dtype)
        assert out is None or (out.shape == input.shape and out.is_contiguous())
        keep = torch.from_numpy(P.keep_mask(input.numel(), spec.p, spec.seed, spec.stream_id, spec.step, spec.offset)).view(input.shape)
        y = torch.where(keep, input / (1 - spec.p), 0.0).contiguous()
        y = y if residual is None else y + residual
        return y if out is None else out.copy_(y)

    monkeypatch.setattr(ops, "dropout", dropout)
    monkeypatch.setattr(ops, "dropout_backward", lambda g, spec: dropout(g, spec))


def stored(fmt):
    x = torch.randn(4, 6, 5, 7, generator=torch.Generator().manual_seed(1))
    if fmt == "channels_last":
        return x.contiguous(memory_format=torch.channels_last)
    return x.transpose(1, 3) if fmt == "transposed" else x[:, :, ::2] if fmt == "strided" else x


@pytest.fixture
def counter(monkeypatch):
    """A step counter that the stand-in reads as the kernels do: when they run."""
    c = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(_common, "_counter_of", lambda x: c)

    def dropout(input, spec, residual=None, out=None):
        step = spec.step + int(spec.step_device)
        keep = torch.from_numpy(P.keep_mask(input.numel(), spec.p, spec.seed, spec.stream_id, step, spec.offset)).view(input.shape)
        y = torch.where(keep, input / (1 - spec.p), 0.0).contiguous()
        return y if out is None else out.copy_(y)

    monkeypatch.setattr(ops, "dropout", dropout)
    monkeypatch.setattr(ops, "dropout_backward", lambda g, spec: dropout(g, spec))
    return c


class Two(nn.Module):
    """a dropout of something that needs no gradient, and one that does"""

    def __init__(self):
        super().__init__()
        self.first, self.second = fdp.DPDropout(0.5), fdp.DPDropout(0.5)
        self.a, self.b = nn.Parameter(torch.ones(1000)), nn.Parameter(torch.ones(1000))

    def forward(self, x):
        return self.second(self.first(x) * self.a) * self.b


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_recomputed_pass_draws_its_own_step(counter, reentrant):
    """With the counter on and moved between a checkpoint's passes, the second draws what the first one drew; the gradient of a
    factor behind the dropouts is the output."""
    m = Two()
    x = torch.ones(1000, requires_grad=reentrant)
    for k in range(3):
        m.zero_grad()
        torch.manual_seed(5)                     # (the same seeds in every turn: what is done with is not found again)
        y = checkpoint(m, x, use_reentrant=reentrant)
        counter.add_(1)
        y.sum().backward()
        assert torch.equal(m.b.grad, y.detach()) and torch.equal(m.a.grad, y.detach()) and 100 < (y != 0).sum() < 400
    a, b = (checkpoint(m, x, use_reentrant=reentrant) for _ in range(2))       # two graphs at once
    counter.add_(1)
    for y in (b, a):
        m.zero_grad()
        y.sum().backward(retain_graph=True)
        assert torch.equal(m.b.grad, y.detach())
        m.zero_grad()
        y.sum().backward()                       # (and a graph twice)
        assert torch.equal(m.b.grad, y.detach())
    assert not torch.equal(a, b)


def test_a_recomputed_pass_that_cannot_be_told_apart_is_refused(counter):
    m = Two()
    x = torch.ones(1000)
    graphs = []
    for _ in range(2):
        torch.manual_seed(5)
        graphs.append(checkpoint(m, x, use_reentrant=False))
        counter.add_(1)
    with pytest.raises(RuntimeError, match="same seed"):
        graphs[0].sum().backward()


def test_steps_are_forgotten_with_their_graphs(counter):
    m = Two()
    x = torch.ones(1000, requires_grad=True)
    before = len(_common._drawn)
    for _ in range(5):
        m(x).sum().backward()
    assert len(_common._drawn) == before


def test_a_first_pass_that_is_no_longer_known_is_refused(counter, monkeypatch):
    """Passes without a graph are kept in a bounded number: a checkpoint whose first pass was dropped does not draw another mask."""
    monkeypatch.setattr(_common, "_GRAPHLESS_MOST", 2)
    monkeypatch.setattr(_common, "_forgotten", False)
    _common._graphless.clear()
    m = Two()
    x = torch.ones(1000, requires_grad=True)
    y = checkpoint(m, x, use_reentrant=True)
    y.sum().backward()                           # (its two dropouts are the two that are kept)
    y = checkpoint(m, x, use_reentrant=True)
    with torch.no_grad():
        for _ in range(3):
            m.first(x)
    assert len(_common._graphless) == 2
    with pytest.raises(RuntimeError, match="no longer known"):
        y.sum().backward()


def numbers_of(spec, elements):
    """which groups of which streams a call draws"""
    return {(spec.seed, spec.stream_id, spec.offset + g) for g in range((elements + 7) // 8)}


@pytest.mark.parametrize("sizes", [(10 * 64, 6 * 64), (6 * 64, 10 * 64), (24, 24, 8), (12, 12), (5, 3), (13, 13, 13), (64, 32, 96, 64), (1, 1)])
def test_ranks_never_share_a_draw(sizes):
    """Whatever the sizes of their shards, and with one seed in all of them."""
    drawn = []
    try:
        for rank, n in enumerate(sizes):
            fdp.set_data_parallel(rank, len(sizes))
            torch.manual_seed(7)
            drawn.append(numbers_of(_common.dropout_spec(0.5, 3, torch.empty(n)), n))
    finally:
        fdp.set_data_parallel(0, 1)
    for i, a in enumerate(drawn):
        for b in drawn[:i]:
            assert not a & b
    if len(set(sizes)) == 1 and sizes[0] % 8 == 0:
        torch.manual_seed(7)
        assert set().union(*drawn) == numbers_of(_common.dropout_spec(0.5, 3, torch.empty(sum(sizes))), sum(sizes))


@pytest.mark.parametrize("fmt", ["contiguous", "channels_last", "transposed", "strided"])
@pytest.mark.parametrize("residual", [False, True])
def test_an_output_may_be_modified_in_place(on_cpu, fmt, residual):
    """What nn.Dropout's output takes: sums into it, activations in place; with the gradients of the same thing not in place."""
    m = fdp.DPDropout(0.4)
    x, r = stored(fmt).requires_grad_(), torch.randn_like(stored(fmt))
    args = (r,) if residual else ()

    def run(change):
        torch.manual_seed(3)
        x.grad = None
        y = change(m(x, *args))
        y.square().sum().backward()
        return y.detach(), x.grad

    pairs = [(lambda y: y.add_(r), lambda y: y + r), (lambda y: y.relu_(), lambda y: y.relu()), (lambda y: F.silu(y, inplace=True), F.silu)]
    for inplace, plain in pairs:
        for a, b in zip(run(inplace), run(plain)):
            assert torch.equal(a, b)
    y = m(x, *args)
    y += 1.0
    assert not y._is_view() and (fmt == "strided" or y.stride() == x.stride())


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("case", ["dtype", "shape", "number"])
def test_a_residual_of_another_type_or_shape(on_cpu, training, case):
    """The sum that evaluation gives, in training behind the dropout."""
    m = fdp.DPDropout(0.3).train(training)
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(4, 6, generator=gen).to(torch.bfloat16 if case == "dtype" else torch.float32).requires_grad_()
    r = torch.randn({"dtype": (4, 6), "shape": (6,), "number": ()}[case], generator=gen).requires_grad_()
    torch.manual_seed(1)
    y = m(x, r)
    torch.manual_seed(1)
    assert torch.equal(y, m(x) + r) and y.dtype == torch.float32 and y.shape == (4, 6)
    y.sum().backward()
    assert x.grad.dtype == x.dtype and torch.equal(r.grad, torch.full(r.shape, 24.0 / max(1, r.numel())))


@pytest.mark.parametrize("view", [False, True])
def test_a_leaf_is_refused_before_it_is_overwritten(on_cpu, view):
    """In place on what autograd does not let be modified: an error, and the numbers stay."""
    m = fdp.DPDropout(0.5, inplace=True)
    leaf = torch.ones(4, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="in-place|inplace"):
        m(leaf[:2] if view else leaf)
    assert torch.equal(leaf, torch.ones(4, 8))
    parts = (torch.ones(4, 8, requires_grad=True) * 1).unbind(0)
    with pytest.raises(RuntimeError, match="in-place|inplace"):
        m(parts[0])
    assert torch.equal(parts[0], torch.ones(8))
    with torch.no_grad():
        assert m(leaf) is leaf and (leaf == 0).any()


def test_group_norm_norms_come_with_their_gradients():
    """The norms are by-products of the clipped gradients: a call that asks for norms alone is refused, not left unanswered."""
    lib, at = _lib.load(), 8192              # (not looked at by a call that is refused)
    p = _lib.DPParams(1.0, 1.0, 0.0, 0, 1, 1, 2, 1, 0, 1, None)
    for ng, nb in ((at, at), (at, None), (None, at)):
        assert lib.fdp_group_norm_bwd(at, at, at, at, at, at, at, None, None, ng, nb, 2, 4, 16, 4, 0, 0, 0, None, ctypes.byref(p), at, 1 << 40,
                                      None) == _lib.FDP_ERR_ARG


def test_a_dropout_takes_no_parameter_id():
    """The noise of a model's parameters is a function of their ids, in construction order: dropouts in between do not move them."""
    a = runtime.next_param_id()
    drops = [fdp.DPDropout(0.5) for _ in range(3)]
    assert runtime.next_param_id() == a + 1 and len({d._stream_id for d in drops}) == 3


def test_a_kept_graph_is_not_taken_for_a_later_one(counter):
    """Run again once, kept, and run again after another pass under its seed: refused, since the steps differ."""
    m = Two()
    x = torch.ones(1000, requires_grad=True)
    torch.manual_seed(5)
    y = checkpoint(m, x, use_reentrant=False)
    y.sum().backward(retain_graph=True)
    counter.add_(1)
    torch.manual_seed(5)
    other = checkpoint(m, x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="same seed"):
        y.sum().backward()
    del other
    m.zero_grad()
    y.sum().backward()
    assert torch.equal(m.b.grad, y.detach())
