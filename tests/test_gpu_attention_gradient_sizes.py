"""Gradients of cross attention where the queries' incoming gradients differ in size by many powers of two, as a segmentation loss gives
them (voxels that are certain, and those at a border): every query's and every key's row has to be right against its own size."""
import pytest
import torch

import d2conv3d_b200 as d2c

pytestmark = pytest.mark.gpu


def gradients(q, k, v, g):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(d2c.cross_attention(*leaves), leaves, g)


def rows(q, k, v, g):
    """{gradient: (value in 64 bits, bound of the 2-norm of each row's error)}; heads alike in number.

    What a product's operands lose: 22 bits of each are kept and lo lo is left out, 3 * 2^-22 (float32 in parts; nothing in float16).  Its
    signs are not alike, so that a sum of products is off by that much of the 2-norm of its terms: e_s, e_dp.  A probability is off by
    e_s, by its exponential's 2^-22, by the rounding of lse (2^-24 of it) and of itself (half a step of its parts: 2^-22, or 2^-11), dS
    by the last too.  delta is formed from the rounded o: half a step of it, the same for all keys of a query: it meets sum p k whole.
    Independent errors add up in the 2-norm; 4 of those are allowed.  A sum on the tensor cores is truncated at each of at most 72
    products of a chain by 2^-23 of its size: that of the result, or of its terms' 2-norm where they cancel."""
    half = torch.finfo(q.dtype).eps / 2
    parts = q.dtype == torch.float32
    lost, step = (3 * 2.0 ** -22, 2.0 ** -22) if parts else (0.0, half)
    q, k, v, g = (t.detach().double().transpose(1, 2) for t in (q, k, v, g))
    scale = q.shape[-1] ** -0.5
    s = q @ k.mT * scale
    p = torch.softmax(s, -1)
    o = p @ v
    dp = g @ v.mT
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_p = lost * (q.square() @ k.square().mT).sqrt() * scale + 2.0 ** -22 + torch.logsumexp(s, -1, keepdim=True).abs() * 2.0 ** -24 + step
    e_dp = lost * (g.square() @ v.square().mT).sqrt() + 2.0 ** -22 * dp.abs()
    e_delta = half * (g * o).norm(dim=-1, keepdim=True) * 2 + 2.0 ** -22 * delta.abs()
    e_ds = ds.abs() * (e_p + step) + p * e_dp
    chain = 72 * 2.0 ** -23

    def bound(value, e, w, x, along=0.0):
        """value = w x, w off by e."""
        terms = lambda t: (t.square() @ x.square().sum(-1, keepdim=True)).sqrt()  # noqa: E731
        size = torch.maximum(value.norm(dim=-1, keepdim=True), terms(w))
        off = 4 * (terms(e) + lost * terms(w)) + chain * size + along + half * value.norm(dim=-1, keepdim=True)
        smallest = torch.finfo(torch.float32 if parts else torch.float16)
        return (value.transpose(1, 2), (off + smallest.smallest_normal * smallest.eps * x.shape[-1] ** 0.5)[..., 0].transpose(1, 2))

    e_key = ((p * e_delta).square().mT @ q.square().sum(-1, keepdim=True)).sqrt() * 4
    return {"grad_q": bound(ds @ k * scale, e_ds * scale, ds * scale, k, e_delta * (p @ k).norm(dim=-1, keepdim=True) * scale),
            "grad_k": bound(ds.mT @ q * scale, e_ds.mT * scale, ds.mT * scale, q, e_key * scale),
            "grad_v": bound(p.mT @ g, (p * e_p).mT, p.mT, g)}


def check(q, k, v, g, names=("grad_q", "grad_k", "grad_v")):
    got, want = dict(zip(("grad_q", "grad_k", "grad_v"), gradients(q, k, v, g))), rows(q, k, v, g)
    for name in names:
        value, bound = want[name]
        off = (got[name].double() - value).norm(dim=-1)
        at = int((off / bound).argmax())
        row = float(value.norm(dim=-1).flatten()[at])
        assert (off <= bound).all(), f"{name}: row {at} is off by {float(off.flatten()[at]) / row:.2e}, allowed {float(bound.flatten()[at]) / row:.2e}"


def make(lq, lk, d, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(1, n, 2, d, generator=gen).cuda().to(dtype) for n in (lq, lk, lk, lq))


@pytest.fixture(autouse=True)
def in_parts():
    before = d2c.get_math_mode()
    d2c.set_math_mode("bf16x3")            # whatever the size of the call
    yield
    d2c.set_math_mode(before)


def sizes(kind, lq, dtype):
    """A factor for each query's gradient; float16 holds fewer of them."""
    gen = torch.Generator().manual_seed(9)
    top = 12 if dtype == torch.float16 else 0
    if kind == "one_above":
        s = torch.full((lq,), -14.0 if dtype == torch.float16 else -24.0)
        s[lq // 3] = 0
    else:
        low = -14.0 if dtype == torch.float16 else {"spread_20": -20.0, "spread_60": -60.0}[kind]
        s = (torch.rand(lq, generator=gen) * low).floor()
    return torch.exp2(s + top).cuda().view(1, -1, 1, 1)


@pytest.mark.parametrize("kind", ["one_above", "spread_20", "spread_60"])
@pytest.mark.parametrize("lk,d", [(3240, 64), (3240, 128), (3240, 40), (12960, 64), (200, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_queries_of_unlike_sizes(dtype, lk, d, kind):
    q, k, v, g = make(300, lk, d, dtype)
    check(q, k, v, (g.float() * sizes(kind, 300, dtype)).to(dtype))


@pytest.mark.parametrize("keys", [65536, 262144])
def test_many_keys(keys):
    q, k, v, g = make(130, keys, 64, torch.float32, 1)
    check(q, k, v, g * sizes("spread_20", 130, torch.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_keys_that_only_small_gradients_reach(dtype, d):
    """Two regions: a query's own region scores 2 a^2 / sqrt(d) = 36 nats above the other, so that the other region's keys get less than
    2^-50 of it; the second region's gradients are 2^-30 (float16: 2^-13) of the first's."""
    q, k, v, g = make(400, 700, d, dtype, 2)
    a = (18.0 * d ** 0.5) ** 0.5
    for t in (q, k):
        t[:, ::2, :, 0], t[:, 1::2, :, 0] = a, -a
    big = 2.0 ** 12 if dtype == torch.float16 else 1.0
    g = g.float() * big
    g[:, 1::2] *= 2.0 ** (-13 if dtype == torch.float16 else -30)
    check(q, k, v, g.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_probabilities_that_grow_along_the_keys(dtype, d):
    """Every tile's scores lie above the last's: what a row was scaled to is taken back tile after tile."""
    q, k, v, g = make(140, 1500, d, dtype, 3)
    q[..., 0] = 1
    k[..., 0] = torch.linspace(-30, 30, 1500, device="cuda").to(dtype).view(1, -1, 1) * (d / 64) ** 0.5
    check(q, k, v, g, names=("grad_q",))
    check(k.flip(1), q, q, k, names=("grad_k", "grad_v"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("d,at", [(64, 100), (64, 3000), (128, 100)])
def test_a_large_value_that_nobody_looks_at(dtype, d, at):
    """A key 36 nats below the others whose value is 2^14 times theirs: it adds nothing to any score gradient."""
    q, k, v, g = make(300, 3240, d, dtype, 6)
    q[..., 0] = 6
    k[..., 0] = 0
    k[:, at, :, 0] = -6 * d ** 0.5
    v[:, at] *= 2.0 ** 14
    check(q, k, v, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_queries_without_a_gradient(dtype):
    """Masked queries: zero gradients give zero rows and change nothing else."""
    q, k, v, g = make(300, 500, 64, dtype, 4)
    g[:, 100:290] = 0
    got = gradients(q, k, v, g)
    assert (got[0][:, 100:290] == 0).all()
    check(q, k, v, g, names=("grad_k", "grad_v"))
    none = gradients(q, k, v, torch.zeros_like(g))
    assert all((t == 0).all() for t in none)


@pytest.mark.parametrize("keys", [65536, 65537, 200000])
def test_the_default_mode_takes_parts_for_any_number_of_keys(keys):
    """No edge at some number of keys: the calls just above one were four times slower."""
    q, k, v, g = make(130, keys, 64, torch.float32, 5)
    want = gradients(q, k, v, g)
    d2c.set_math_mode("auto")
    assert all(torch.equal(a, b) for a, b in zip(gradients(q, k, v, g), want))
    check(q, k, v, g)
