import pytest
import torch

import d2conv3d_b200 as d2c
from tests._tokens import assert_within, layer_norm_oracle, rounded

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def run(x, w, b, g, layout, eps=1e-5):
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = d2c.layer_norm(*leaves, eps=eps, layout=layout)
    live = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, live, g))
    return y.detach(), [next(grads) if t is not None else None for t in leaves]


def check(x, w, b, g, layout, eps=1e-5):
    y, (gx, gw, gb) = run(x, w, b, g, layout, eps)
    first = layout != "channels_last"
    gg = g
    if layout == "tokens":
        gg = g.mT.reshape(x.shape)
    want = layer_norm_oracle(x, w, b, gg, eps, 1 if first else -1)
    if layout == "tokens":
        want["y"] = tuple(t.flatten(2).mT for t in want["y"])
    assert_within(y, want["y"][0], rounded(*want["y"], x.dtype), "y")
    assert_within(gx, want["gx"][0], rounded(*want["gx"], x.dtype), "gx")
    for got, key, p in ((gw, "gw", w), (gb, "gb", b)):
        if p is not None:
            assert got.dtype == p.dtype
            assert_within(got, want[key][0], rounded(*want[key], p.dtype), key)


def data(shape, out, c, dtype, pdtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=gen) * 1.5 + 0.5).to(dtype).cuda()
    w = (torch.randn(c, generator=gen) * 0.3 + 1).to(pdtype).cuda()
    b = (torch.randn(c, generator=gen) * 0.3).to(pdtype).cuda()
    return x, w, b, torch.randn(out, generator=gen).to(dtype).cuda()


# one channel, fewer than a vector, every group size's edge, odd widths, wider than a block's registers
@pytest.mark.parametrize("c", [1, 3, 8, 64, 65, 255, 256, 512, 1000, 1024, 1032, 2048, 4097, 8192, 8200])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(c, dtype):
    for rows in (1, 5, 77):
        check(*data((rows, c), (rows, c), c, dtype, dtype, c + rows), "channels_last")


@pytest.mark.parametrize("layout", ["channels_first", "tokens"])
@pytest.mark.parametrize("c", [1, 7, 64, 72, 144, 256, 520, 1024, 2048, 2052])
@pytest.mark.parametrize("dtype", TYPES)
def test_volumes(c, dtype, layout):
    for b, dims in ((1, (1, 1, 1)), (2, (2, 3, 5)), (1, (2, 7, 10)), (3, (1, 4, 33))):
        n = dims[0] * dims[1] * dims[2]
        out = (b, n, c) if layout == "tokens" else (b, c) + dims
        check(*data((b, c) + dims, out, c, dtype, dtype, c + n), layout)


@pytest.mark.parametrize("layout", ["channels_last", "channels_first", "tokens"])
def test_many_positions(layout):
    c, b, dims = 96, 2, (4, 31, 50)
    n = dims[0] * dims[1] * dims[2]
    shape = (b, n, c) if layout == "channels_last" else (b, c) + dims
    out = (b, c) + dims if layout == "channels_first" else (b, n, c)
    check(*data(shape, out, c, torch.bfloat16, torch.float32, 3), layout)


@pytest.mark.parametrize("with_w,with_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("layout", ["channels_last", "channels_first"])
def test_optional_parameters(with_w, with_b, layout):
    shape = (3, 5, 40) if layout == "channels_last" else (3, 40, 2, 3, 4)
    x, w, b, g = data(shape, shape, 40, torch.float16, torch.float32, 9)
    check(x, w if with_w else None, b if with_b else None, g, layout)


def test_strided_unaligned_and_4d_inputs():
    base = torch.randn(6, 9, 80, device="cuda", dtype=torch.bfloat16)
    g = torch.randn(6, 9, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(65, device="cuda", dtype=torch.bfloat16)
    check(base[:, :, 3:67], w[1:], w[:64], g, "channels_last")
    check(base.transpose(0, 1)[..., :64], w[1:], w[:64], g.transpose(0, 1), "channels_last")
    flat = torch.randn(1 + 4 * 64 * 30, device="cuda", dtype=torch.float16)
    check(flat[1:].view(4, 64, 30), w[1:].half(), w[:64].half(), torch.randn(4, 64, 30, device="cuda").half(), "channels_first")


def test_only_some_gradients():
    x, w, b, g = data((2, 33, 2, 3, 4), (2, 33, 2, 3, 4), 33, torch.float32, torch.float32, 4)
    _, full = run(x, w, b, g, "channels_first")
    for need in range(3):
        leaves = [t.clone().requires_grad_(i == need) for i, t in enumerate((x, w, b))]
        y = d2c.layer_norm(*leaves, layout="channels_first")
        got = torch.autograd.grad(y, leaves[need], g)[0]
        assert torch.equal(got, full[need])


def test_far_from_zero_and_constant_rows():
    # a mean 1000 times the spread: sums of squares would lose the variance
    x = (torch.randn(7, 384) + 1000).cuda()
    w, b = torch.ones(384).cuda(), torch.zeros(384).cuda()
    check(x, w, b, torch.randn(7, 384).cuda(), "channels_last")
    check(x.t().reshape(1, 384, 7), w, b, torch.randn(1, 384, 7).cuda(), "channels_first")
    y = d2c.layer_norm(torch.full((3, 256), 5.0, device="cuda"), w[:256], b[:256] + 2)
    assert torch.equal(y, torch.full_like(y, 2.0))


def test_nan_stays_in_its_position():
    for layout, shape in (("channels_last", (4, 9, 64)), ("channels_first", (4, 64, 9)), ("tokens", (4, 64, 9))):
        x = torch.randn(shape, device="cuda")
        clean = d2c.layer_norm(x, layout=layout)
        at = (2, 5, 7) if layout == "channels_last" else (2, 7, 5)
        x[at] = float("nan")
        y = d2c.layer_norm(x, layout=layout)
        rows = y if layout != "channels_first" else y.mT
        cleans = clean if layout != "channels_first" else clean.mT
        assert rows[2, 5].isnan().all()
        rows[2, 5] = cleans[2, 5]
        assert torch.equal(rows, cleans)


def test_empty():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = d2c.layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 8) and torch.equal(w.grad, torch.zeros_like(w))
    assert d2c.layer_norm(torch.zeros(2, 8, 0, 4, device="cuda"), layout="tokens").shape == (2, 0, 8)


def test_same_bits_every_time_and_no_second_derivative():
    x, w, b, g = data((2, 8000, 256), (2, 8000, 256), 256, torch.bfloat16, torch.float32, 5)
    first = run(x, w, b, g, "channels_last")
    for _ in range(3):
        again = run(x, w, b, g, "channels_last")
        assert torch.equal(first[0], again[0]) and all(torch.equal(p, q) for p, q in zip(first[1], again[1]))
    leaf = torch.randn(4, 8, device="cuda", requires_grad=True)
    gx = torch.autograd.grad(d2c.layer_norm(leaf).square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="twice"):
        gx.sum().backward()


def test_gradient_by_differences():
    torch.manual_seed(0)
    x, w = torch.randn(2, 6, 5, device="cuda"), torch.randn(6, device="cuda")
    g = torch.randn(2, 6, 5, device="cuda")
    leaf = x.clone().requires_grad_()
    gx = torch.autograd.grad(d2c.layer_norm(leaf, w, layout="channels_first"), leaf, g)[0]

    def f(t):
        m = t.double().mean(1, keepdim=True)
        h = (t.double() - m) / ((t.double() - m).square().mean(1, keepdim=True) + 1e-5).sqrt()
        return float((h * w.double().view(1, 6, 1) * g.double()).sum())

    for _ in range(5):
        step = torch.randn_like(x).double() * 1e-5
        diff = (f(x.double() + step) - f(x.double() - step)) / 2
        assert abs(diff - float((gx.double() * step).sum())) <= 1e-4 * float((gx.double() * step).abs().sum()) + 1e-9


def test_refusals():
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(RuntimeError, match="not implemented"):
        d2c.layer_norm(x.double())
    with pytest.raises(RuntimeError, match=r"must be \[8\]"):
        d2c.layer_norm(x, torch.ones(7, device="cuda"))
    with pytest.raises(RuntimeError, match="float32 or of the input's type"):
        d2c.layer_norm(x, torch.ones(8, device="cuda").half())
    with pytest.raises(RuntimeError, match="same type"):
        d2c.layer_norm(x.half(), torch.ones(8, device="cuda").half(), torch.ones(8, device="cuda"))
    with pytest.raises(RuntimeError, match="expected weight on"):
        d2c.layer_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="dimensions"):
        d2c.layer_norm(x[0], layout="channels_first")
    with pytest.raises(RuntimeError, match="channels"):
        d2c.layer_norm(torch.zeros(3, 0, device="cuda"))


def test_captured_and_on_another_stream():
    x, w, b, g = data((1, 64, 2, 9, 11), (1, 198, 64), 64, torch.bfloat16, torch.float32, 6)
    want = run(x, w, b, g, "tokens")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, g, "tokens")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = d2c.layer_norm(*leaves, layout="tokens")
        grads = torch.autograd.grad(y, leaves, g)
    with torch.no_grad():
        leaves[0].copy_(x * 2)
    graph.replay()
    want = run(x * 2, w, b, g, "tokens")
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(grads, want[1]))


def test_more_elements_than_32_bits_count():
    c, n = 64, (1 << 25) + 3                                # 2^31 + 192 elements
    x = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16)
    tail = torch.randn(5, c, device="cuda").bfloat16()
    x[-5:] = tail
    assert torch.equal(d2c.layer_norm(x)[-5:], d2c.layer_norm(tail))
    del x
    v = torch.zeros(65600, 512, 64, device="cuda", dtype=torch.bfloat16)
    v[-1] = torch.randn(512, 64, device="cuda").bfloat16()
    got = d2c.layer_norm(v, layout="channels_first")[-1:]
    want = layer_norm_oracle(v[-1:], None, None, torch.zeros_like(v[-1:]), 1e-5, 1)["y"]
    assert_within(got, want[0], rounded(*want, torch.bfloat16), "last clip")
