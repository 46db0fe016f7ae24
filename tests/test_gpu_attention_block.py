"""The token operators as they are used together: norm, projection, rotary positions, attention, projection."""
import os
import subprocess
import sys

import pytest
import torch

import d2conv3d_b200 as d2c
from d2conv3d_b200.decoder import Decoder, pyramid_shapes

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def plain_block(m, x, context, lengths):
    """The same block in 64-bit tensor operations."""
    def norm(t, n):
        t = t.flatten(2).mT
        h = (t - t.mean(-1, keepdim=True)) / (t.var(-1, unbiased=False, keepdim=True) + n.eps).sqrt()
        return h * n.weight + n.bias

    def rotate(t, grid, step):
        axes = [(torch.arange(n, device=t.device, dtype=torch.float64) + 0.5) * s - 0.5 for n, s in zip(grid, step)]
        p = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)
        out, c0 = [], 0
        for a, n in enumerate(m.axis_dims):
            f = 10000.0 ** (-torch.arange(0, n, 2, device=t.device, dtype=torch.float64) / n)
            w = (p[:, a, None] * f)[None, :, None]
            u, v = t[..., c0:c0 + n // 2], t[..., c0 + n // 2:c0 + n]
            out += [u * w.cos() - v * w.sin(), u * w.sin() + v * w.cos()]
            c0 += n
        return torch.cat(out + [t[..., c0:]], -1)

    b = x.shape[0]
    q = m.to_q(norm(x, m.norm)).view(b, -1, m.heads, m.head_dim)
    k, v = m.to_kv(norm(context, m.context_norm)).view(b, -1, 2, m.kv_heads, m.head_dim).unbind(2)
    q = rotate(q, x.shape[2:], [c / s for c, s in zip(context.shape[2:], x.shape[2:])])
    k = rotate(k, context.shape[2:], (1, 1, 1))
    k, v = (t.repeat_interleave(m.heads // m.kv_heads, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) / m.head_dim ** 0.5
    if lengths is not None:
        s = s.masked_fill(torch.arange(k.shape[1], device=s.device) >= lengths.view(-1, 1, 1, 1), -torch.inf)
    o = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v)
    return x + m.to_out(o.flatten(2)).mT.reshape(x.shape)


@pytest.mark.parametrize("kv_heads,ragged", [(4, False), (2, True)])
def test_block_and_its_gradients(kv_heads, ragged):
    torch.manual_seed(0)
    m = d2c.CrossAttention3d(48, 80, heads=4, kv_heads=kv_heads, head_dim=32).cuda()
    x, context = torch.randn(2, 48, 2, 5, 7, device="cuda"), torch.randn(2, 80, 2, 9, 13, device="cuda")
    n = torch.tensor([234, 150], device="cuda") if ragged else None
    ins = [t.requires_grad_() for t in (x, context)] + list(m.parameters())
    y = m(x, context, n)
    g = torch.randn_like(y)
    grads = torch.autograd.grad(y, ins, g)
    m64 = d2c.CrossAttention3d(48, 80, heads=4, kv_heads=kv_heads, head_dim=32).cuda().double()
    m64.load_state_dict(m.state_dict())
    ins64 = [t.detach().double().requires_grad_() for t in (x, context)] + list(m64.parameters())
    y64 = plain_block(m64, ins64[0], ins64[1], n)
    want = torch.autograd.grad(y64, ins64, g.double())
    # fp32 throughout, chains of 234 keys and 80 channels: a few hundred u = 6e-8 of each tensor's scale
    for got, ref in zip((y,) + grads, (y64,) + want):
        assert (got.double() - ref).abs().max() <= 3e-5 * ref.abs().max()


def test_predictor_norm_of_a_deformable_layer():
    torch.manual_seed(1)
    layer = d2c.MDConv3d(64, 64, 3, padding=1, init="random", norm_type="LayerNorm3d").cuda()
    torch.nn.init.normal_(layer.deform_params.weight, std=0.02)
    x = torch.randn(1, 64, 3, 8, 9, device="cuda", requires_grad=True)
    y = layer(x)
    grads = torch.autograd.grad(y.square().sum(), [x, layer.norm.weight, layer.norm.bias])
    assert all(torch.isfinite(t).all() and t.abs().max() > 0 for t in grads)
    # the norm is what the predictor sees
    h = torch.nn.functional.layer_norm(x.detach().movedim(1, -1), (64,), layer.norm.weight, layer.norm.bias).movedim(-1, 1)
    assert (layer.norm(x) - h).abs().max() <= 1e-5


@pytest.mark.parametrize("train", [False, True])
def test_decoder_with_the_attention_bridge(train):
    torch.manual_seed(2)
    widths = (64, 64, 64, 128)
    net = Decoder(widths=widths, channels=128, offset_groups=2, bridge="cross_attention").cuda()
    pyramid = [torch.randn(s, device="cuda").relu_() for s in pyramid_shapes(1, 2, 64, 96, widths)]
    if not train:
        with torch.no_grad():
            y = net(*pyramid)
        assert y.shape == (1, 2, 2, 64, 96) and torch.isfinite(y).all()
        return
    y = net(*pyramid)
    y.square().mean().backward()
    for name, p in net.gc.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().max() > 0, name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_under_autocast(dtype):
    torch.manual_seed(3)
    m = d2c.CrossAttention3d(48, 80, heads=2, head_dim=64).cuda()
    x, context = torch.randn(2, 48, 2, 5, 7, device="cuda", requires_grad=True), torch.randn(2, 80, 2, 9, 13, device="cuda")
    full = m(x, context)
    with torch.autocast("cuda", dtype):
        y = m(x, context)
        y16 = m(x.to(dtype), context.to(dtype))
    # rounding of tokens, projections, probabilities and outputs: a dozen half steps of 16 bits
    for got in (y, y16):
        assert (got - full).abs().max() <= 12 * torch.finfo(dtype).eps / 2 * full.abs().max()
    y.square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())


FIRST_CALL_CAPTURED = """
import torch
import d2conv3d_b200 as d2c
mode = "bf16x3" if "%(dtype)s" == "float32" else "auto"
d2c.set_math_mode(mode)
def make(*s):
    return torch.randn(*s, device="cuda").to(torch.%(dtype)s).requires_grad_()
x, w, q, k, g = make(2, 64, 90), make(64), make(1, 90, 2, 64), make(1, 200, 2, 64), make(1, 90, 2, 64).detach()
one, gn = make(1, 1, 2, 64), make(2, 90, 64).detach()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def step():
    y = d2c.layer_norm(x, w, layout="tokens")
    r = d2c.rotary_embedding_3d(q, (1, 9, 10), (16, 24, 24))
    o = d2c.cross_attention(r, k, k)
    return (y, o, d2c.cross_attention(one.detach(), k.detach(), k.detach())) + torch.autograd.grad((y, o), (x, w, q, k), (gn, g))
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
"""


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_first_calls_of_a_process_are_captured(dtype):
    # whatever a first call sets up must not disturb a capture
    p = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED % {"dtype": dtype}], capture_output=True, text=True, timeout=240, cwd=ROOT)
    assert p.returncode == 0, p.stderr[-2000:]
