import math

import pytest
import torch

import d2conv3d_b200 as d2c
from tests._tokens import U, assert_within, attention_oracle, half, rounded

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(b, lq, lk, hq, hkv, d, dtype, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    t = lambda *s, std=1.0: (torch.randn(s, generator=gen) * std).to(dtype).cuda()  # noqa: E731
    return t(b, lq, hq, d, std=spread), t(b, lk, hkv, d, std=spread), t(b, lk, hkv, d), t(b, lq, hq, d)


def run(q, k, v, g, lengths=None, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = d2c.cross_attention(*leaves, key_lengths=lengths, scale=scale)
    return (o.detach(),) + torch.autograd.grad(o, leaves, g)


# fp32 by math mode: (half a step of the probabilities, what the operands' rounding takes from a product).  "bf16x3", the mode of split
# operands, which "auto" takes for large calls: hi + lo fp16
# parts keep a factor to 2^-22 (half a step of the second part, 2^-11 of at most 2^-11), and lo lo, at most 2^-22, is left out.
# "bf16": each factor to 2^-9.
FP32_MODES = {"fp32": (U, 0.0), "bf16x3": (2.0 ** -22, 3 * 2.0 ** -22), "bf16": (2.0 ** -9, 2.0 ** -8 + 2.0 ** -18)}


def check(q, k, v, g, lengths=None, scale=None):
    before = d2c.get_math_mode()
    for mode in FP32_MODES if q.dtype == torch.float32 else ("auto",):
        p_half, product = FP32_MODES[mode] if q.dtype == torch.float32 else (half(q.dtype), 0.0)
        try:
            d2c.set_math_mode(mode)
            got = run(q, k, v, g, lengths, scale)
            with torch.no_grad():
                served = d2c.cross_attention(q, k, v, lengths, scale)
        finally:
            d2c.set_math_mode(before)
        want = attention_oracle(q, k, v, g, lengths, 1 / math.sqrt(q.shape[-1]) if scale is None else scale, p_half, product)
        for name, t in zip(("o", "gq", "gk", "gv"), got):
            assert t.dtype == q.dtype
            assert_within(t, want[name][0], rounded(*want[name], q.dtype), f"{name} {mode}")
        assert torch.equal(served, got[0])


# lengths from one to several tiles, on both sides of the tiles' edges
LENGTHS = [(1, 1), (1, 7), (2, 64), (3, 129), (16, 200), (17, 33), (63, 65), (64, 128), (65, 127), (127, 1), (128, 256), (129, 300),
           (200, 5), (257, 130), (300, 513)]


@pytest.mark.parametrize("lq,lk", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths(lq, lk, dtype):
    check(*make(2, lq, lk, 2, 2, 64, dtype, lq + lk))


@pytest.mark.parametrize("d", [1, 5, 8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 120, 127, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_widths(d, dtype):
    check(*make(1, 70, 150, 2, 1, d, dtype, d))
    check(*make(1, 2, 150, 2, 1, d, dtype, d))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (6, 1), (8, 8), (16, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_shared_heads(hq, hkv, dtype):
    check(*make(2, 1, 300, hq, hkv, 64, dtype, hq))
    check(*make(1, 140, 190, hq, hkv, 32, dtype, hq))


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_with_nan_behind_the_lengths(dtype, itype):
    # lengths at and around tile edges, none at all, all of them, and values outside 0 .. Lk
    lens = [0, 1, 64, 127, 128, 129, 300, -3, 1000]
    for lq in (1, 5, 140):
        q, k, v, g = make(len(lens), lq, 300, 4, 2, 64, dtype, lq)
        n = torch.tensor(lens, dtype=itype, device="cuda")
        want = run(q, k, v, g, n)
        for i, m in enumerate(lens):
            m = min(max(m, 0), 300)
            k[i, m:], v[i, m:] = float("nan"), float("inf")
        check_q = run(q, k, v, g, n)
        for a, b in zip(want, check_q):
            assert torch.equal(a, b)
        assert (want[0][0] == 0).all() and (want[1][0] == 0).all()
        for i, m in enumerate(lens):
            m = min(max(m, 0), 300)
            assert (want[2][i, m:] == 0).all() and (want[3][i, m:] == 0).all()
            k[i, m:], v[i, m:] = 0, 0
        check(q, k, v, g, n)


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_rows_and_scales(dtype):
    q, k, v, g = make(1, 130, 260, 2, 2, 64, dtype, 3, spread=3.0)
    check(q, k, v, g)
    check(q, k, v, g, scale=0.01)
    check(q, k, v, g, scale=-0.05)
    check(q, k, v, g, scale=0.0)


def test_scores_far_apart():
    # one key far above all others in a late tile: what was summed before it vanishes; far below: adds nothing
    q, k, v, g = make(1, 70, 400, 1, 1, 64, torch.bfloat16, 4)
    q[:] = 1
    for at, size in ((390, 30.0), (5, 30.0), (200, -30.0)):
        kk = k.clone()
        kk[0, at] = size
        check(q, kk, v, g)
    o = d2c.cross_attention(q, kk, v)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_small_gradients(dtype):
    # under 16-bit loss scales gradients are small: they must not vanish in intermediate roundings
    q, k, v, g = make(1, 150, 700, 2, 1, 64, dtype, 5)
    g = g * (2.0 ** -7 if dtype == torch.float16 else 2.0 ** -20)
    check(q, k, v, g)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    torch.manual_seed(6)
    b, lq, lk, h, d = 2, 66, 140, 2, 64
    q = torch.randn(b, h, lq, d, device="cuda").to(dtype).transpose(1, 2)
    kv = torch.randn(b, lk, 2, h, d, device="cuda").to(dtype)
    g = torch.randn(b, h, lq, d, device="cuda").to(dtype).transpose(1, 2)
    check(q, kv[:, :, 0], kv[:, :, 1], g)
    check(q[:, :1], kv[:, :, 0], kv[:, :, 1], g[:, :1])
    odd = torch.randn(b, lk, h, d + 3, device="cuda").to(dtype)
    check(q, odd[..., 1:65], odd[..., 3:], g)                    # rows that are not 16-byte aligned
    check(q[:, :1], odd[..., 1:65], odd[..., 3:], g[:, :1])
    check(q[..., ::2], kv[:, :, 0, :, ::2], kv[:, :, 1, :, 1::2], g[..., ::2])
    one = torch.randn(b, lk, 1, d, device="cuda").to(dtype).expand(b, lk, h, d)
    check(q, one, one, g)
    check(q, kv[:, :, 0], kv[:, :, 0], g)                        # keys that are values
    check(q, kv[:, :, 0], kv[:, :, 1], g[:, :1, :1].expand(b, lq, h, d))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_keys_few_queries_and_the_reverse(dtype):
    # shares of the long axis that are joined afterwards
    check(*make(1, 20, 4001, 1, 1, 64, dtype, 7))
    check(*make(1, 1, 20011, 2, 1, 32, dtype, 8))
    check(*make(1, 3000, 40, 2, 1, 64, dtype, 9))


def test_large_fp32_calls_take_split_operands():
    q, k, v, g = make(1, 600, 1000, 2, 1, 64, torch.float32, 21)
    auto = run(q, k, v, g)
    for mode, same in (("bf16x3", True), ("fp32", False)):
        try:
            d2c.set_math_mode(mode)
            other = run(q, k, v, g)
        finally:
            d2c.set_math_mode("auto")
        assert all(torch.equal(a, b) for a, b in zip(auto, other)) == same


def test_gradient_by_differences():
    torch.manual_seed(0)
    q, k, v, g = make(1, 9, 21, 2, 1, 16, torch.float32, 1)
    grads = run(q, k, v, g)[1:]
    n = 2

    def f(q, k, v):
        s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(n, 2)) / 4
        return float((torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.repeat_interleave(n, 2)) * g.double()).sum())

    at = [t.double() for t in (q, k, v)]
    for i, grad in enumerate(grads):
        step = torch.randn_like(at[i]) * 1e-5
        up = [t + step if j == i else t for j, t in enumerate(at)]
        down = [t - step if j == i else t for j, t in enumerate(at)]
        diff = (f(*up) - f(*down)) / 2
        assert abs(diff - float((grad.double() * step).sum())) <= 1e-4 * float((grad.double() * step).abs().sum())


def test_empty():
    k = torch.randn(2, 5, 2, 64, device="cuda", requires_grad=True)
    q = torch.randn(2, 3, 4, 64, device="cuda", requires_grad=True)
    o = d2c.cross_attention(q, k[:, :0], k[:, :0])
    assert torch.equal(o, torch.zeros_like(o))
    gq, gk = torch.autograd.grad(o.sum(), (q, k))
    assert (gq == 0).all() and (gk == 0).all()
    o = d2c.cross_attention(q[:, :0], k, k)
    assert o.shape == (2, 0, 4, 64) and (torch.autograd.grad(o.sum(), k)[0] == 0).all()
    assert d2c.cross_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 64)


@pytest.mark.parametrize("big,small", [(1e30, 1e-30), (3e38, 1.0), (1e-38, 1e-3)])
def test_fp32_beyond_the_range_of_16_bits(big, small):
    # operands are scaled by powers of two before they are split: nothing overflows, nothing vanishes
    q, k, v, g = make(2, 300, 400, 2, 1, 64, torch.float32, 22)
    d2c.set_math_mode("bf16x3")
    try:
        check(q, k, v, g)
        plain = run(q, k, v, g)
        big, small = 2.0 ** min(127, round(math.log2(big))), 2.0 ** round(math.log2(small))   # 2^128 is not a float32
        if big > 2.0 ** 100:
            v = v / 64
            plain = (plain[0] / 64, plain[1] / 64, plain[2] / 64, plain[3])
        o = run(q, k, v * big, g)[0]
        if big < 2.0 ** -100:
            # below fp32's normal range: v is scaled to 1 at most, not to 2^14, so that its parts end at 2^-25 of that, and the result
            # is a multiple of 2^-149 on either side
            assert (o.double() - plain[0].double() * big).abs().max() <= big * v.abs().max() * 2.0 ** -22 + 2.0 ** -148
        else:
            assert torch.equal(o, plain[0] * big)
        gv = run(q, k, v, g * small)[3]
        assert torch.equal(gv, plain[3] * small)
        if 1e-30 < small < 1:
            assert torch.equal(run(q * small, k / small, v, g)[0], plain[0])
    finally:
        d2c.set_math_mode("auto")


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time(dtype):
    q, k, v, g = make(2, 333, 1500, 4, 2, 64, dtype, 11)
    n = torch.tensor([1500, 777], device="cuda")
    first = run(q, k, v, g, n)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run(q, k, v, g, n)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [1, 200])
def test_captured_replayed_and_on_another_stream(dtype, lq):
    q, k, v, g = make(1, lq, 500, 2, 2, 64, dtype, 12)
    n = torch.tensor([400], device="cuda", dtype=torch.int32)
    want = run(q, k, v, g, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, g, n)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    graphs, outs = [], []
    for _ in range(2):                                           # two graphs side by side: neither uses the other's memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = d2c.cross_attention(*leaves, key_lengths=n)
            outs.append((o,) + torch.autograd.grad(o, leaves, g))
        graphs.append(graph)
    n.fill_(77)                                                  # lengths are read when the graph runs
    want = run(q, k, v, g, n)
    streams = [torch.cuda.Stream() for _ in graphs]
    for graph, s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_saved_tensors_are_checked_and_no_second_derivative():
    q, k, v, g = make(1, 9, 21, 2, 1, 16, torch.float32, 1)
    q.requires_grad_()
    o = d2c.cross_attention(q, k, v)
    k.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o, q, g)
    gq = torch.autograd.grad(d2c.cross_attention(q, k, v), q, g, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="twice"):
        gq.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_that_pass_32_bits(dtype):
    # the second clip starts past 2^31 elements; so do the last keys of a long one
    far = (1 << 31) + 128
    base = torch.empty(far + (1 << 20), device="cuda", dtype=dtype)
    k = base.as_strided((2, 150, 1, 64), (far, 64, 64, 1))
    k.normal_()
    q, _, _, g = make(2, 130, 1, 2, 1, 64, dtype, 13)
    for lq in (1, 130):
        a, b = run(q[:, :lq], k, k, g[:, :lq]), run(q[:, :lq], k.contiguous(), k.contiguous(), g[:, :lq])
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    step = (1 << 31) // 140
    step -= step % 64
    k = base.as_strided((1, 140, 1, 64), (0, step, 64, 1))
    k.normal_()
    for lq in (1, 130):
        a, b = run(q[:1, :lq], k, k, g[:1, :lq]), run(q[:1, :lq], k.contiguous(), k.contiguous(), g[:1, :lq])
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_more_heads_than_a_grid_dimension(dtype):
    q, k, v, g = make(2, 17, 40, 1, 1, 16, dtype, 14)
    if dtype == torch.float32:
        d2c.set_math_mode("bf16x3")
    try:
        want = run(q, k, v, g)
        many = [t.repeat(35000, 1, 1, 1) for t in (q, k, v, g)]
        for a, b in zip(run(*many), want):
            assert torch.equal(a[-2:], b) and torch.equal(a[:2], b)
    finally:
        d2c.set_math_mode("auto")


def test_refusals():
    q, k, v, _ = make(2, 3, 5, 4, 2, 64, torch.float32)
    for args, text in (((q.double(), k.double(), v.double()), "not implemented"), ((q, k.half(), v), "same type"),
                       ((q, k, v[:, :4]), "does not match key"), ((q, k[:1], v[:1]), "does not match query"),
                       ((q, k[..., :32], v[..., :32]), "does not match query"), ((q[0], k, v), "ndimension"),
                       ((q[:, :, :3], k, v), "cannot share"), ((q, k.cpu(), v), "expected key on")):
        with pytest.raises(RuntimeError, match=text):
            d2c.cross_attention(*args)
    for n, text in ((torch.ones(3, device="cuda", dtype=torch.int32), "must be"), (torch.ones(2, device="cuda"), "int32 or int64"),
                    (torch.ones(2, dtype=torch.int32), "expected key_lengths on")):
        with pytest.raises(RuntimeError, match=text):
            d2c.cross_attention(q, k, v, n)
    wide = torch.zeros(1, 2, 1, 136, device="cuda")
    with pytest.raises(RuntimeError, match="1 to 128"):
        d2c.cross_attention(wide, wide, wide)


@pytest.mark.parametrize("keys", [32768, 262144])
def test_fp32_gradients_of_many_keys(keys):
    # Probabilities of about 1 / keys: the score gradients are far below the bound that their scale is taken from.  Values and gradients
    # of +-1 give that bound its largest distance.  Scores of std 8 * 2^-5 * 2^-3: p keys is 1 within some per cent.
    # Tolerance, 2-norm: a chain of at most 72 products whose sums are truncated to 24 bits, each by at most 2^-23 of the result: 2^-16.8;
    # the second parts of dS: scaled by 2^8 (15 - ilogb(255)), dS has rms 8 * 2^8 / keys, at 2^18 keys 2^-7, and a step of 2^-24 leaves
    # 2^-25.8 of it: 2^-18.8.  Together 1.1e-5 (a scale that is smaller by 2^3 alone leaves 2^-15.8, 1.8e-5).
    gen = torch.Generator().manual_seed(7)
    sign = lambda *s: (torch.randint(0, 2, s, generator=gen) * 2 - 1).float().cuda()  # noqa: E731
    n, d = max(6, 2 ** 20 // keys), 64
    q = (torch.randn(1, n, 1, d, generator=gen) / 32).cuda()
    k = torch.randn(1, keys, 1, d, generator=gen).cuda()
    v, g = sign(1, keys, 1, d), sign(1, n, 1, d)
    got = run(q, k, v, g)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    p = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", leaves[0], leaves[1]) * d ** -0.5, -1)
    o = torch.einsum("bhqk,bkhd->bqhd", p, leaves[2])
    want = (o.detach(),) + torch.autograd.grad(o, leaves, g.double())
    for name, a, e in zip(("o", "grad_q", "grad_k", "grad_v"), got, want):
        assert float((a.double() - e).norm() / e.norm()) <= 1.1e-5, name


def test_fp32_gradients_of_many_keys_in_parts():
    before = d2c.get_math_mode()
    try:
        d2c.set_math_mode("bf16x3")        # whatever "auto" takes for so many keys
        test_fp32_gradients_of_many_keys(262144)
    finally:
        d2c.set_math_mode(before)
