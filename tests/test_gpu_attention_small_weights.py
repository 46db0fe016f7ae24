"""Cross attention where most of a row's weights are far below its largest: they are small, but there are many of them."""
import pytest
import torch

import d2conv3d_b200 as d2c

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def in_parts():
    before = d2c.get_math_mode()
    d2c.set_math_mode("bf16x3")            # float32: whatever the size of the call
    yield
    d2c.set_math_mode(before)


@pytest.mark.parametrize("gap", [8.0, 11.0, 14.0, 17.0])
@pytest.mark.parametrize("keys,d", [(1000, 64), (12960, 64), (12960, 128), (51360, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_one_key_above_many_alike(dtype, keys, d, gap):
    """One key scores `gap` nats above all others, which are alike; values 1 for them and 0 for it, so that the result is the share that
    the others have: keys e^-gap / (1 + keys e^-gap), 4e-5 and more.  A weight is off by half a step of fp16's smallest numbers, 2^-25,
    against a largest one of 2^7 at least: 2^-32 e^gap of itself; the rest is roundings of a few 2^-23 (float32: two parts; the scores, 1e-6 of
    gap at most; a chain of truncated sums, 72 2^-23) and half a step of the result, and of P (float16)."""
    q = torch.ones(1, 300, 1, d, device="cuda", dtype=dtype)
    k = torch.zeros(1, keys, 1, d, device="cuda", dtype=dtype)
    v = torch.ones(1, keys, 1, d, device="cuda", dtype=dtype)
    for at in (0, 200, keys - 1):                                        # in the first tile, a later one, the last one
        kk, vv = k.clone(), v.clone()
        kk[0, at] = gap / d ** 0.5                                       # scale * q . k = d^-1/2 * d * gap d^-1/2
        vv[0, at] = 0
        s = float(kk[0, at, 0, 0].double()) * d ** 0.5
        share = (keys - 1) * torch.exp(torch.tensor(-s, dtype=torch.float64))
        want = float(share / (1 + share))
        half = torch.finfo(dtype).eps / 2
        rounding = 2.0 ** -16.8 + 2.0 ** -20 * gap if dtype == torch.float32 else 2 * half + 2.0 ** -16.8
        bound = want * (2.0 ** -32 * torch.exp(torch.tensor(s)).item() + rounding) + torch.finfo(dtype).smallest_normal * half * 2
        with torch.no_grad():
            o = d2c.cross_attention(q, kk, vv)
        off = float((o.double() - want).abs().max())
        assert off <= bound, f"key {at}: off by {off / want:.2e}, allowed {bound / want:.2e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("keys,lq", [(300, 140), (3000, 20), (300, 1)])
def test_a_first_tile_that_scores_minus_infinity(dtype, keys, lq):
    """Keys whose scores are all -inf weigh nothing, wherever they are, and what follows may lie far below zero."""
    torch.manual_seed(0)
    q = torch.rand(1, lq, 2, 64, device="cuda").to(dtype) + 1
    k, v = (torch.randn(1, keys, 2, 64, device="cuda").to(dtype) for _ in range(2))
    k[..., 1] = -200                       # scores of about -37 nats, 2^-54: beyond what fp16 holds
    k[:, :150, :, 0] = -float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = d2c.cross_attention(*leaves)
    rest = d2c.cross_attention(q, k[:, 150:], v[:, 150:])
    want = torch.softmax(torch.einsum("bihd,bjhd->bhij", q.double(), k[:, 150:].double()) / 8, -1)
    want = torch.einsum("bhij,bjhd->bihd", want, v[:, 150:].double())
    # P and the result are rounded by half a step each; P against values whose signs are not alike
    bound = torch.finfo(dtype).eps * 2 * v.abs().max().double()
    assert (o.double() - want).abs().max() <= bound and (rest.double() - want).abs().max() <= bound


def test_rows_without_weights_beside_rows_that_grow():
    """Products beyond the type's range are -inf for the queries that meet them so, through two tiles, while the other queries' scores
    grow from tile to tile."""
    torch.manual_seed(1)
    dtype = torch.bfloat16
    q = torch.rand(1, 140, 1, 64, device="cuda").to(dtype) + 1
    k, v = (torch.randn(1, 600, 1, 64, device="cuda").to(dtype) for _ in range(2))
    q[:, ::2, :, 0], q[:, 1::2, :, 0] = 1e20, 1e-20
    k[:, :300, :, 0], k[:, 300:, :, 0] = -1e20, 0
    k[..., 1] = torch.linspace(-200, 0, 600, device="cuda").to(dtype).view(1, -1, 1)
    with torch.no_grad():
        o = d2c.cross_attention(q, k, v)
    want = torch.softmax(torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) / 8, -1)
    want = torch.einsum("bhij,bjhd->bihd", want, v.double())
    assert (o.double() - want).abs().max() <= torch.finfo(dtype).eps * 2 * v.abs().max().double()
