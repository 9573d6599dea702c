"""Rows of one value that is no short binary fraction: their sums round, and the layer norm of such a
row is beta up to a bound that follows from the sums' depth.

The kernels add a row up in chains of at most 16 elements per lane (rows longer than 16384: cols /
1024 and 8 more), 6 additions across a wave and 16 across waves: D in all. The first mean is off by
(D + 1) 2^-24 of the value (the division rounds too). The differences from it are exact and equal;
their mean, the correction, is off by (D + 2) 2^-24 of itself, and subtracting it rounds once. With
rstd <= 1 / sqrt(epsilon), |y - beta| <= |gamma| |x| (D + 1) (D + 3) 2^-48 / sqrt(epsilon), and y
rounds once; four products' and rstd's own rounding change that by less than a hundredth."""
import math

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1, 3, 7, 100, 784, 1537, 4096, 4099, 16384, 16385, 50001])
@pytest.mark.parametrize("epsilon", [1e-5, 1e-12])
def test_constant_rows_are_beta(cols, epsilon):
    from distributed_tensorflow_amd.ops import hip
    gen = torch.Generator().manual_seed(cols)
    values = torch.cat([torch.tensor([0.1, 1 / 3, 1234.567, -98765.4, 1e-8, 7.5, 0.0]),
                        torch.randn(40, generator=gen) * 100])
    gamma = torch.randn(cols, generator=gen).cuda()
    beta = torch.randn(cols, generator=gen).cuda()
    x = values.cuda().unsqueeze(1).expand(-1, cols).contiguous()
    y, mean, rstd = hip.layer_norm(x, gamma, beta, epsilon, want_stats=True)
    depth = max(16, math.ceil(cols / 1024) + 8) + 22
    size = x.double().abs() * (depth + 1) * (depth + 3) * 2.0 ** -48 / math.sqrt(epsilon)
    off = (y.double() - beta.double()).abs()
    limit = 1.01 * size * gamma.double().abs()
    assert (off <= limit + 2.0 ** -24 * (beta.double().abs() + limit)).all()
    assert ((mean.double().cpu() - values.double()).abs()
            <= values.double().abs() * (2.0 ** -24 + (depth + 3) ** 2 * 2.0 ** -48)).all()
    assert torch.isfinite(rstd).all()
