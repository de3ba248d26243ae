"""The gates of the norms of rows, value by value, for arguments of any size (tests/block_oracle.py).

Steps of 2^-24 of a value in 32 bits: the exponential 2, 1 + e and its reciprocal 2, their product and the argument's 2, the norm of
a row of 64 equal values 6 (squares, six sums of two equals that are exact, mean, root, reciprocal, product), weight and gate 2: 14,
and a gradient's slope 4 more, of the size of its terms, and its factors 2: 20. A result in 16 bits is rounded once more.
"""

import pytest
import torch

from block_oracle import gate as exact_gate

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24
ROUNDING = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize('activation', ['sigmoid', 'silu'])
@pytest.mark.parametrize('dtype, reach', [(torch.float32, 80.0), (torch.bfloat16, 80.0), (torch.float16, 8.0)])
def test_gates_of_any_size(dtype, reach, activation):
    from cuju_amd import layers
    z = torch.linspace(-reach, reach, 64 * 500, dtype=torch.float64).to(dtype).view(500, 64).cuda()
    x = torch.ones(500, 64, dtype=dtype, device='cuda')
    weight, gate = torch.full((64,), 0.5, device='cuda'), z.clone().requires_grad_()
    y = layers.rms_norm(x, weight, gate, epsilon=0.0, activation=activation)
    factor, slope = exact_gate(z.double(), activation)
    exact = 0.5 * factor
    # float16 ends at 2^-24: half of that is its least step's rounding.
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    error = (y.detach().double() - exact).abs()
    assert bool((error <= (14 * STEP + ROUNDING[dtype]) * exact.abs() + least).all()), float((error / exact.abs()).nan_to_num(0).max())
    found, = torch.autograd.grad(y, gate, torch.ones_like(y))
    s = torch.sigmoid(z.double())
    terms = 0.5 * (s * torch.sigmoid(-z.double()) if activation == 'sigmoid' else s * (1 + z.double().abs() * torch.sigmoid(-z.double())))
    slope = s * torch.sigmoid(-z.double()) if activation == 'sigmoid' else s * (1 + z.double() * torch.sigmoid(-z.double()))
    error = (found.double() - 0.5 * slope).abs()
    assert bool((error <= 20 * STEP * terms + ROUNDING[dtype] * 0.5 * slope.abs() + least).all()), float((error / terms).max())


@pytest.mark.parametrize('activation', ['sigmoid', 'silu'])
def test_gates_at_the_ends(activation):
    # Where the exponential leaves 32 bits, and arguments that are not finite.
    from cuju_amd import layers
    z = torch.tensor([[-3e38, -200.0, -104.0, 104.0, 200.0, 3e38, float('inf'), float('nan')]], device='cuda', requires_grad=True)
    x = torch.ones_like(z)
    y = layers.rms_norm(x, None, z, epsilon=0.0, activation=activation)
    found, = torch.autograd.grad(y, z, torch.ones_like(y))
    wanted = exact_gate(z.detach().double(), activation)[0]
    torch.testing.assert_close(y.detach().double()[:, :6], wanted[:, :6], rtol=14 * STEP, atol=2.0 ** -126)
    assert y[0, 6].item() == (1.0 if activation == 'sigmoid' else float('inf')) and bool(y[0, 7].isnan())
    assert bool((found[0, :3].abs() <= 2.0 ** -120).all()) and bool(found[0, 7].isnan())
    torch.testing.assert_close(found[0, 3:6], torch.full((3,), 0.0 if activation == 'sigmoid' else 1.0, device='cuda'), rtol=0, atol=2.0 ** -120)
