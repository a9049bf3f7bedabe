"""The angles of the rotary embedding in float32."""

import math

import numpy as np
import pytest
import torch

from _paged import EPS24
from mfattn.kernels import rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("near", [0.0, 0.25, 0.5, 0.75, 0.125, 0.375, 0.9999999])
@pytest.mark.parametrize("off", [1e-7, 3e-6, 1e-3, 0.02])
def test_sine_and_cosine_have_float32s_relative_accuracy(near, off, device):
    """Beside every multiple of a quarter turn, where a sine or cosine is small.

    Half steps of float32, relative: the fraction of a turn 1, sin and cos 4, the magnitude 1,
    the product 1, the sum (with a zero) 1: at most 8."""
    freqs = [2 * math.pi * (near + s * off * (1 + i / 16)) for s in (1, -1) for i in range(16)]
    rot = rotary.Rotary(64, frequencies=freqs)
    x = torch.zeros(2, 1, 64, device=device)
    x[0, :, :32] = 1.0                       # u = 1, w = 0: (cos, sin)
    x[1, :, 32:] = 1.0                       # u = 0, w = 1: (-sin, cos)
    y, _ = rotary.rotate(x, None, rot, torch.ones(2, dtype=torch.int32, device=device))
    a = np.array(freqs, dtype=np.longdouble)
    c, s = torch.from_numpy(np.cos(a).astype(np.float64)), torch.from_numpy(np.sin(a).astype(np.float64))
    y = y.double().cpu()[:, 0]
    for got, want in ((y[0, :32], c), (y[0, 32:], s), (y[1, :32], -s), (y[1, 32:], c)):
        # a frequency in 64 bits is off by 2^-53 of it, an angle's fraction by 2^-65 turns
        absolute = 2.0 ** -52 * abs(torch.from_numpy(a.astype(np.float64)))
        assert ((got - want).abs() - (8 * EPS24 * want.abs() + absolute)).max() <= 0


def test_error_does_not_exceed_a_chain_of_float32_operations(device):
    """Root mean square against float64, beside cos and sin rounded once from float64 angles."""
    rot = rotary.Rotary(64, theta=1e6)
    g = torch.Generator(device=device).manual_seed(2)
    for low, high in ((0, 4096), (90000, 131000), (2 ** 31 - 5000, 2 ** 31 - 1)):
        pos = torch.randint(low, high, (4000,), generator=g, device=device, dtype=torch.int32)
        x = torch.randn(4000, 4, 64, generator=g, device=device)
        got, _ = rotary.rotate(x, None, rot, pos)
        # turns in 64-bit integers: float64 angles lose what matters at 2^31
        turn = 2 * np.longdouble("3.14159265358979323846264338327950288")
        steps = torch.tensor([int(np.longdouble(f) / turn * 2 ** 62) for f in rot.frequencies],
                             dtype=torch.int64, device=device)
        turns = (pos.long()[:, None] * steps) & (2 ** 62 - 1)
        angle = (turns.double() * (2 * math.pi * 2.0 ** -62))[:, None]
        c, s = torch.cos(angle), torch.sin(angle)
        u, w = x[..., :32], x[..., 32:]
        want = torch.cat((u.double() * c - w.double() * s, w.double() * c + u.double() * s), -1)
        c, s = c.float(), s.float()
        plain = torch.cat((u * c - w * s, w * c + u * s), -1)
        own, other = ((y.double() - want).square().mean().sqrt().item() for y in (got, plain))
        print(f"positions {low} .. {high}: {own:.3e}, plain {other:.3e}", flush=True)
        # (frequencies of 62 bits here, times positions of 31)
        assert own <= 1.05 * other + 2.0 ** -31 * 2 * math.pi
