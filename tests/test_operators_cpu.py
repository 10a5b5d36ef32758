"""The operators' formulas and refusals, without a GPU."""
import torch

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
