"""The layers of the operators on the device where their manners could differ from those of the layers they stand for."""
import pytest
import torch
import torch.nn as nn
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
