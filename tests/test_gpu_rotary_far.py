import math

import numpy as np
import pytest
import torch

import d2conv3d_b200 as d2c

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("base", [100.0, 10000.0, 500000.0])
@pytest.mark.parametrize("far", [1 << 20, 1 << 27, 1 << 36])
def test_what_a_far_position_costs(far, base):
    """Angles against extended precision (64 bits of significand): p * 2^-50 radians at most, besides float32's own roundings: the angle
    in half turns, 2 pi 2^-25; sin and cos, 2 u; products and sum, 3 u."""
    torch.manual_seed(0)
    n, half = 60, 20
    p = torch.randint(far // 2, far, (n, 3))
    x = torch.randn(1, n, 2, 6 * half, device="cuda")
    y = d2c.rotary_embedding_3d(x, p.cuda(), (2 * half,) * 3, base=base)[0].double().cpu().numpy()
    x = x[0].double().cpu().numpy()
    step = np.longdouble(base) ** (-np.arange(half, dtype=np.longdouble) / half)
    for axis in range(3):
        angle = p[:, axis].numpy().astype(np.longdouble)[:, None] * step
        c, s = np.cos(angle).astype(np.float64)[:, None], np.sin(angle).astype(np.float64)[:, None]
        at = slice(2 * half * axis, 2 * half * axis + half), slice(2 * half * axis + half, 2 * half * (axis + 1))
        u, v = x[..., at[0]], x[..., at[1]]
        bound = (np.abs(u) + np.abs(v)) * (2 * math.pi * U / 2 + 5 * U + far * 2.0 ** -50)
        assert (np.abs(y[..., at[0]] - (u * c - v * s)) <= bound).all() and (np.abs(y[..., at[1]] - (u * s + v * c)) <= bound).all()
