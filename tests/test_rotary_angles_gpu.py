"""Cosines and sines of ``rotary_axes`` by themselves: rows (1, 0) turn into (cos, sin).

Bound with u = 2^-23, an ulp relative to a value at least: sincospi is within 2 ulp, and putting back what the fraction of
a turn lost in float32 rounds once, half an ulp: 2.5 u |value|, also near a zero.  What is put back is below
pi 2^-25 and off by 2^-22 of itself, 2^-45.  The kernel's turns and the float64 angle are each off by at most
2^-51 of the angle."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('far', [64, 4096, 1 << 20, 1 << 26])
@pytest.mark.parametrize('theta', [1e6, 10.0])
def test_cosines_and_sines_near_zero(pkg, device, far, theta):
    half, tokens = 64, 4096
    gen = torch.Generator().manual_seed(far)
    positions = torch.randint(0, far, (1, 1, tokens), generator=gen)
    rows = torch.zeros(1, tokens, 1, 2 * half, device=device)
    rows[..., :half] = 1.0
    out = pkg.rotary_axes(rows, None, positions.to(device), (half,), theta=theta)[0].cpu().double()[0, :, 0]
    angle = positions[0, 0, :, None].double() * theta ** -(torch.arange(half, dtype=torch.float64) / half)
    want = torch.cat([angle.cos(), angle.sin()], -1)
    tol = 2.5 * 2.0 ** -23 * want.abs() + 2.0 ** -45 + torch.cat([angle, angle], -1) * 2.0 ** -50
    over = ((out - want).abs() - tol).max().item()
    assert over <= 0, f'off by {over:.3e} more than the bound'
