import pytest
import torch

import d2conv3d_b200 as d2c
from tests._tokens import assert_within, rotary_oracle, rounded

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def grid_positions(grid, step=(1, 1, 1)):
    axes = [(torch.arange(n, dtype=torch.float64) + 0.5) * s - 0.5 for n, s in zip(grid, step)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(1, -1, 3)


def check(x, positions, where, axis_dims, base=10000.0, interleaved=False, step=None):
    leaf = x.detach().requires_grad_()
    y = d2c.rotary_embedding_3d(leaf, positions, axis_dims, base=base, interleaved=interleaved, grid_step=step)
    assert y.is_contiguous() and y.dtype == x.dtype
    g = torch.randn(x.shape, device="cuda").to(x.dtype)
    gx = torch.autograd.grad(y, leaf, g)[0]
    want, bound = rotary_oracle(x, where, axis_dims, base, interleaved)
    assert_within(y, want, rounded(want, bound, x.dtype), "y")
    want, bound = rotary_oracle(g, where, axis_dims, base, interleaved, inverse=True)
    assert_within(gx, want, rounded(want, bound, x.dtype), "gx")


# every vector width (multiples of 8, 4, 2 and odd halves), sections left out, channels that stay, one token, one head
@pytest.mark.parametrize("dim,axes", [(64, (16, 24, 24)), (32, (8, 12, 12)), (128, (44, 42, 42)), (80, (26, 26, 26)), (2, (0, 2, 0)),
                                      (6, (2, 2, 2)), (64, (0, 32, 32)), (64, (0, 0, 0)), (30, (10, 6, 8)), (512, (160, 176, 176))])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_grid(dim, axes, dtype, interleaved):
    torch.manual_seed(dim)
    for b, grid, heads in ((1, (1, 1, 1), 1), (2, (3, 5, 7), 3), (1, (2, 9, 4), 8)):
        x = torch.randn(b, grid[0] * grid[1] * grid[2], heads, dim, device="cuda").to(dtype)
        check(x, grid, grid_positions(grid).expand(b, -1, -1), axes, interleaved=interleaved)


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("shared", [False, True])
def test_positions_of_their_own(ptype, shared):
    torch.manual_seed(1)
    b, n = 3, 50
    p = torch.randint(-1000, 200000, (n, 3) if shared else (b, n, 3))
    p = p.to(ptype) if ptype != torch.float32 else p.float() / 8 + 0.3
    x = torch.randn(b, n, 4, 64, device="cuda")
    check(x, p.cuda(), p.double().expand(b, n, 3), (16, 24, 24))
    check(x[:1], p.cuda() if shared else p[:1].cuda(), (p if shared else p[0]).double()[None], (16, 24, 24))


def test_far_positions():
    p = torch.tensor([[1 << 40, (1 << 45) + 7, 123456789012]])
    x = torch.randn(1, 1, 2, 48, device="cuda")
    check(x, p.cuda(), p[None], (16, 16, 16), base=100.0)


def test_grid_step_shares_a_frame():
    # cells of a level of twice the stride sit between two of the finer level's
    x = torch.randn(1, 6, 1, 32, device="cuda")
    check(x, (1, 2, 3), grid_positions((1, 2, 3), (1, 2, 2.5)), (8, 12, 12), step=(1, 2, 2.5))


@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(interleaved):
    torch.manual_seed(2)
    qkv = torch.randn(2, 30, 3, 4, 64, device="cuda").bfloat16()
    grid = (2, 3, 5)
    for x in (qkv[:, :, 1], qkv[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2), qkv[:, :, 2, :, 3:63],
              qkv[:, :, 2, :, ::2], qkv[:, :, 0, :1].expand(2, 30, 4, 64)):
        axes = (8, 12, 12) if x.shape[-1] < 64 else (16, 24, 24)
        check(x, grid, grid_positions(grid).expand(2, -1, -1), axes, interleaved=interleaved)
    flat = torch.randn(1 + 30 * 64, device="cuda").half()          # a start that is not aligned to a pair
    check(flat[1:].view(1, 30, 1, 64), grid, grid_positions(grid), (16, 24, 24), interleaved=interleaved)


def test_channels_that_stay_keep_their_bits():
    x = torch.full((1, 4, 2, 32), float("nan"), device="cuda")
    x[..., :24] = 1
    x[..., 30] = float("inf")
    y = d2c.rotary_embedding_3d(x, (1, 2, 2), (8, 8, 8))
    assert torch.isfinite(y[..., :24]).all()
    assert y[..., 24:30].isnan().all() and (y[..., 30] == float("inf")).all()


def test_empty_and_more_tokens_than_blocks():
    assert d2c.rotary_embedding_3d(torch.zeros(2, 0, 3, 8, device="cuda"), (0, 5, 5), (2, 2, 2)).shape == (2, 0, 3, 8)
    x = torch.randn(1, 4 * 300 * 40, 1, 8, device="cuda")
    check(x, (4, 300, 40), grid_positions((4, 300, 40)), (4, 2, 2))


def test_strides_that_pass_32_bits():
    base = torch.zeros((1 << 31) + 4096, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((2, 4, 2, 32), ((1 << 31) + 64, 64, 32, 1))
    x.normal_()
    assert torch.equal(d2c.rotary_embedding_3d(x, (1, 2, 2), (8, 12, 12)),
                       d2c.rotary_embedding_3d(x.contiguous(), (1, 2, 2), (8, 12, 12)))


def test_refusals():
    x = torch.zeros(1, 4, 2, 32, device="cuda")
    for axes in ((8, 12, 14), (7, 12, 12), (-2, 2, 2)):
        with pytest.raises(RuntimeError, match="axis_dims"):
            d2c.rotary_embedding_3d(x, (1, 2, 2), axes)
    with pytest.raises(RuntimeError, match="positions for"):
        d2c.rotary_embedding_3d(x, (1, 2, 3), (8, 12, 12))
    with pytest.raises(RuntimeError, match="positions must be"):
        d2c.rotary_embedding_3d(x, torch.zeros(5, 3, device="cuda"), (8, 12, 12))
    with pytest.raises(RuntimeError, match="int32, int64 or float32"):
        d2c.rotary_embedding_3d(x, torch.zeros(4, 3, device="cuda").double(), (8, 12, 12))
    with pytest.raises(RuntimeError, match="not differentiable in positions"):
        d2c.rotary_embedding_3d(x, torch.zeros(4, 3, device="cuda", requires_grad=True), (8, 12, 12))
    with pytest.raises(RuntimeError, match="expected positions on"):
        d2c.rotary_embedding_3d(x, torch.zeros(4, 3), (8, 12, 12))
    with pytest.raises(RuntimeError, match="even number of channels"):
        d2c.rotary_embedding_3d(x[..., :31], (1, 2, 2), (8, 12, 10))
    with pytest.raises(RuntimeError, match="not implemented"):
        d2c.rotary_embedding_3d(x.double(), (1, 2, 2), (8, 12, 12))
