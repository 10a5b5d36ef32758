"""The layers of the operators on the device where their manners could differ from those of the layers they stand for."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

import flashdp4review_b200 as fdp
from gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpoint_under_a_counter_that_moves(reentrant):
    """use_device_noise_step on and advance_noise_step between a checkpointed forward and its backward: the gradients are those of the
    pass without a checkpoint."""
    torch.manual_seed(4)
    block = nn.Sequential(fdp.DPDropout(0.4), fdp.DPGroupNorm(4, 32, activation="gelu", dropout=0.4, channels_last=True, noise_multiplier=0.0),
                          fdp.DPLinear(32, 32, noise_multiplier=0.0), fdp.DPDropout(0.4)).to(dev())
    x = torch.randn(3, 20, 32, device=dev(), requires_grad=reentrant)
    fdp.use_device_noise_step(True)
    try:
        counter = fdp.runtime.device_noise_counter()
        res = []
        for again in (False, True):
            counter.fill_(7)
            torch.manual_seed(9)
            x.grad = None
            block.zero_grad()
            y = checkpoint(block, x, use_reentrant=reentrant) if again else block(x)
            fdp.advance_noise_step()
            y.square().sum().backward()
            res.append([y.detach()] + [p.grad.clone() for p in block.parameters()] + ([x.grad] if reentrant else []))
        for a, b in zip(*res):
            assert torch.equal(a, b)
    finally:
        fdp.use_device_noise_step(False)


def test_unequal_shards_are_dropped_independently():
    """One seed, shards of ten and six samples: no sample of the second is dropped as one of the first."""
    m = fdp.DPDropout(0.5)
    masks = []
    try:
        for rank, n in ((0, 10), (1, 6)):
            fdp.set_data_parallel(rank, 2)
            torch.manual_seed(7)
            masks.append(m(torch.ones(n, 64, device=dev())))
    finally:
        fdp.set_data_parallel(0, 1)
    assert not any(torch.equal(a, b) for a in masks[0] for b in masks[1])


@pytest.mark.parametrize("shape", [(4, 32, 5, 6), (4, 32, 15), (4, 32), (2, 32, 3, 4, 5), (4, 32, 1), (4, 32, 1, 1), (1, 32, 5, 6)])
@pytest.mark.parametrize("fmt", ["contiguous", "channels_last", "transposed", "strided"])
def test_group_norm_keeps_the_memory_order(shape, fmt):
    """nn.GroupNorm's: output and input gradient of a contiguous input are contiguous, those of one in a channels-last format are
    in that format, those of any other contiguous; same numbers."""
    x = torch.randn(shape, device=dev())
    axes = len(shape) - 2
    if fmt == "channels_last":
        if axes < 2:
            pytest.skip("no such format")
        x = x.contiguous(memory_format=torch.channels_last if axes == 2 else torch.channels_last_3d)
    elif fmt == "transposed":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif fmt == "strided":
        x = torch.randn(shape[:-1] + (2 * shape[-1],), device=dev())[..., ::2]
    torch.manual_seed(1)
    m = fdp.DPGroupNorm(8, 32, activation="silu", C=1e6, noise_multiplier=0.0).to(dev())
    with torch.no_grad():
        m.weight.normal_(1.0, 0.2)
        m.bias.normal_(0.0, 0.2)
    a, b = (x.detach().requires_grad_() for _ in range(2))
    # (what is in front of the layer sees the gradient as it leaves it; a leaf would be given strides of its own)
    seen = []
    ha, hb = a.view_as(a), b.view_as(b)
    ha.register_hook(seen.append)
    y, want = m(ha), F.silu(F.group_norm(hb, 8, m.weight, m.bias))
    g = torch.randn(shape, device=dev())
    # 2^8 roundings of fp32 of the largest, generously for both
    assert (y - want).abs().max() <= 2.0 ** -16 * want.abs().max()
    gb, = torch.autograd.grad(want, b, g)
    y.backward(g)
    assert (a.grad - gb).abs().max() <= 2.0 ** -14 * gb.abs().max()
    if fmt == "channels_last":
        form = torch.channels_last if axes == 2 else torch.channels_last_3d
        assert y.is_contiguous(memory_format=form) and seen[0].is_contiguous(memory_format=form)
    else:
        assert y.is_contiguous() and seen[0].is_contiguous()
        assert y.view(shape[0], -1).shape == (shape[0], y.numel() // shape[0])
    z = m(x.detach())
    z += 1.0                                       # and both may be changed in place
    y = m(a * 1.0)
    y.mul_(2.0).sum().backward()


@pytest.mark.parametrize("fmt", ["contiguous", "channels_last", "transposed"])
def test_a_dropout_may_be_modified_in_place(fmt):
    x = torch.randn(4, 6, 5, 7, device=dev())
    x = x.contiguous(memory_format=torch.channels_last) if fmt == "channels_last" else x.transpose(1, 3) if fmt == "transposed" else x
    x.requires_grad_()
    m, r = fdp.DPDropout(0.3), torch.randn_like(x)
    res = []
    for inplace in (True, False):
        torch.manual_seed(2)
        x.grad = None
        y = m(x)
        assert y.stride() == x.stride()
        y = F.relu(y.add_(r), inplace=True) if inplace else F.relu(y + r)
        y.square().sum().backward()
        res.append((y.detach(), x.grad))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


def test_a_16_bit_branch_onto_an_fp32_residual():
    """Under autocast: the branch leaves a product in 16 bits, the residual stream is fp32."""
    lin, drop = fdp.DPLinear(128, 128, noise_multiplier=0.0).to(dev()), fdp.DPDropout(0.3)
    x = torch.randn(4, 50, 128, device=dev(), requires_grad=True)
    for training in (True, False):
        drop.train(training)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = lin(x)
            torch.manual_seed(3)
            y = drop(h, x)
            torch.manual_seed(3)
            want = drop(h) + x
        assert y.dtype == torch.float32 and torch.equal(y, want)
        y.sum().backward()


@pytest.fixture
def fp8():
    fdp.set_fp8_products(True)
    yield
    fdp.set_fp8_products(False)


def test_layers_beside_the_8_bit_products_keep_their_nodes(fp8):
    """The switch sends a layer to the Function class only for a call that runs in 8 bits."""
    few, many = torch.randn(2, 20, 192, device=dev(), requires_grad=True), torch.randn(2, 100, 192, device=dev(), requires_grad=True)
    lin, conv, ln = fdp.DPLinear(192, 256).to(dev()), fdp.DPConv1D(256, 192).to(dev()), fdp.DPLayerNorm(192).to(dev())
    fdp.set_fp8_products(False)
    native = [type(m(few).grad_fn).__name__ for m in (lin, ln)] + [type(conv(few).grad_fn.next_functions[0][0]).__name__]
    fdp.set_fp8_products(True)
    now = [type(m(few).grad_fn).__name__ for m in (lin, ln)] + [type(conv(few).grad_fn.next_functions[0][0]).__name__]
    assert now == native and not any("Func" in n and "Backward" in n and n.startswith("_DP") for n in now)
    assert type(ln(many).grad_fn).__name__ == native[1]
    assert type(lin(many).grad_fn).__name__ == "_DPLinearFuncBackward"


@pytest.mark.parametrize("shape", [(64, 64), (192, 256), (63, 256), (100, 100)])
def test_mixed_types_are_answered_or_refused_as_without_8_bits(shape):
    """A 16-bit input of a layer with fp32 weights, outside autocast."""
    m = fdp.DPLinear(shape[0], shape[1], noise_multiplier=0.0).to(dev())
    c = fdp.DPConv1D(shape[1], shape[0], noise_multiplier=0.0).to(dev())
    x = torch.randn(200, shape[0], device=dev(), dtype=torch.bfloat16)
    for layer in (m, c):
        answers = []
        for on in (False, True):
            fdp.set_fp8_products(on)
            try:
                answers.append(layer(x).dtype)
            except RuntimeError as e:
                answers.append("refused")
            finally:
                fdp.set_fp8_products(False)
        assert answers[0] == answers[1]


@pytest.mark.parametrize("kind", ["linear", "conv1d"])
@pytest.mark.parametrize("n_in,n_out", [(192, 256), (199, 250)])
def test_the_8_bit_weight_is_a_saved_tensor(fp8, kind, n_in, n_out):
    """Seen and moved by saved-tensor hooks (here to the host and back), let go of by the backward, and kept only where an input
    gradient will ask for it."""
    m = (fdp.DPLinear(n_in, n_out, noise_multiplier=0.0) if kind == "linear" else fdp.DPConv1D(n_out, n_in, noise_multiplier=0.0)).to(dev())
    x = torch.randn(2, 100, n_in, device=dev(), requires_grad=True)
    g = torch.randn(2, 100, n_out, device=dev())
    m(x).backward(g)
    want, x.grad = x.grad, None
    packed = []

    def pack(t):
        packed.append(t.dtype)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(dev())):
        y = m(x)
    assert packed.count(torch.float8_e4m3fn) == 1
    y.backward(g)
    assert torch.equal(x.grad, want)
    packed.clear()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(dev())):
        m(x.detach())
    assert torch.float8_e4m3fn not in packed


def test_the_8_bit_weight_does_not_outlive_its_backward(fp8):
    m = fdp.DPLinear(4096, 4096, noise_multiplier=0.0).to(dev())
    x = torch.randn(256, 4096, device=dev(), requires_grad=True)
    torch.autograd.grad(m(x).sum(), [x])                  # (what the library allocates once)
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    y = m(x)
    loss = y.sum()
    dx, = torch.autograd.grad(loss, [x])
    held = torch.cuda.memory_allocated() - start
    assert held < y.numel() * 4 + dx.numel() * 4 + (1 << 20)          # output and gradient, not the 16 MB of a weight in 8 bits


def test_group_norm_gradients_through_the_reducer():
    """A group norm's gradients in the buckets of the data-parallel reducer are those without it, accumulated and started anew."""
    from flashdp4review_b200.distributed import DPGradReducer

    def make():
        torch.manual_seed(1)
        return nn.Sequential(fdp.DPGroupNorm(4, 32, activation="silu", channels_last=True, C=0.3, noise_multiplier=0.0),
                             fdp.DPLinear(32, 50, C=0.3, noise_multiplier=0.0)).to(dev())

    x, g = torch.randn(4, 6, 32, device=dev()), torch.randn(4, 6, 50, device=dev()) * 0.1
    plain, model = make(), make()
    plain(x).backward(g)
    red = DPGradReducer(model, bucket_bytes=1 << 12, grad_as_bucket_view=True)
    for again in (False, True):
        model(x).backward(g)
        red.finish()
        for p, q in zip(model.parameters(), plain.parameters()):
            assert p.grad.data_ptr() == red._views[id(p)].data_ptr() and torch.equal(p.grad, q.grad)
        red.zero_grad()
    red.remove()


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_captured_checkpoint(reentrant):
    """A checkpointed dropout in a captured step whose counter moves before the backward: in every replay the gradient of a factor behind
    it is the output, and every replay draws anew."""
    m = fdp.DPDropout(0.5)
    fdp.use_device_noise_step(True)
    try:
        x, w = (torch.ones(1000, device=dev(), requires_grad=True) for _ in range(2))

        def step():
            y = checkpoint(lambda t: m(t) * w, x, use_reentrant=reentrant)
            fdp.advance_noise_step()
            y.sum().backward()
            return y.detach()

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        w.grad = x.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        seen = []
        for _ in range(2):
            w.grad.zero_()
            x.grad.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(w.grad, y) and torch.equal(x.grad, y)
            seen.append(y.clone())
        assert not torch.equal(*seen)
    finally:
        fdp.use_device_noise_step(False)
