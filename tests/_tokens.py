"""Oracles of the token operators in 64 bits, each with an element-wise bound of what the kernels' arithmetic may be off by.

u = 2^-24 is half a step of fp32, half(t) half a step of a result's type (its last rounding).  Bounds count the operations of the
kernels' longest chains; sums are fp32 over at most a few hundred terms a thread, then over threads."""
import math

import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what):
    got, want, bound = got.detach().double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    excess = ((got - want).abs() / bound.clamp_min(1e-300)).nan_to_num(0.0)
    worst = float(excess.max()) if excess.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} times what its arithmetic may be off by"


def rounded(want, bound, dtype):
    """The bound with the last rounding: half a step of the value that the kernel had (subnormal steps below the normal range)."""
    return bound * (1 + half(dtype)) + want.abs() * half(dtype) + torch.finfo(dtype).smallest_normal * half(dtype) * 2


def layer_norm_oracle(x, w, b, g, eps, axis):
    """x, g with channels on `axis`: {y, gx, gw, gb: (value, bound)} before the last rounding."""
    x, g = x.detach().double().cpu(), g.detach().double().cpu()
    n = x.shape[axis]
    shape = [1] * x.dim()
    shape[axis] = n
    wv = torch.ones(shape, dtype=torch.float64) if w is None else w.detach().double().cpu().view(shape)
    bv = torch.zeros(shape, dtype=torch.float64) if b is None else b.detach().double().cpu().view(shape)
    mean = x.mean(axis, keepdim=True)
    var = (x - mean).square().mean(axis, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (x - mean) * r
    # a sum of n terms: at most 128 additions follow one another (32 a thread, tree or up to 64 groups)
    dmean = 130 * U * x.abs().mean(axis, keepdim=True)
    # relative error of r: half of that of var + eps (the mean's error enters squared), of the root and the division
    drel = 80 * U + (dmean * r) ** 2
    dh = dmean * r + h.abs() * drel + 3 * U * (x.abs() + mean.abs()) * r
    out = {"y": (h * wv + bv, dh * wv.abs() + 2 * U * (h * wv).abs() + U * bv.abs())}
    gw = g * wv
    m1, m2 = gw.mean(axis, keepdim=True), (gw * h).mean(axis, keepdim=True)
    d1 = 130 * U * gw.abs().mean(axis, keepdim=True)
    d2 = 130 * U * (gw * h).abs().mean(axis, keepdim=True) + (gw.abs() * dh).mean(axis, keepdim=True)
    inner = gw - m1 - h * m2
    gx = r * inner
    out["gx"] = (gx, r * (d1 + h.abs() * d2 + dh * m2.abs() + 6 * U * (gw.abs() + m1.abs() + (h * m2).abs())) + gx.abs() * (drel + 2 * U))
    sums = [a for a in range(x.dim()) if a != axis % x.dim()]
    count = x.numel() // n
    chain = min(count, 4096) + 600                           # additions in a row: a block's positions, then the blocks
    out["gw"] = ((g * h).sum(sums), (g.abs() * dh).sum(sums) + chain * U * (g * h).abs().sum(sums))
    out["gb"] = (g.sum(sums), chain * U * g.abs().sum(sums))
    return out


def rotary_oracle(x, positions, axis_dims, base, interleaved, inverse=False):
    """positions [B, L, 3] in 64 bits.  Returns value and bound."""
    x = x.detach().double().cpu()
    positions = positions.double().cpu()
    out, size = x.clone(), torch.zeros_like(x)
    c0 = 0
    for axis, n in enumerate(axis_dims):
        for i in range(n // 2):
            angle = positions[..., axis] * base ** (-2.0 * i / n) * (-1 if inverse else 1)
            c, s = angle.cos()[..., None], angle.sin()[..., None]
            a, b = (c0 + 2 * i, c0 + 2 * i + 1) if interleaved else (c0 + i, c0 + i + n // 2)
            out[..., a] = x[..., a] * c - x[..., b] * s
            out[..., b] = x[..., a] * s + x[..., b] * c
            size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
        c0 += n
    # the angle in turns is rounded to fp32 (2 pi 2^-25 of a half turn's angle), sin and cos to 2 u, products and sum 2 u; the
    # 64-bit product of position and frequency is off by a few 2^-53 of itself
    far = float(positions.abs().max()) if positions.numel() else 0.0
    return out, size * (2 * math.pi * U / 2 + 5 * U + far * 2 * math.pi * 2.0 ** -50)


def attention_oracle(q, k, v, g, lengths, scale, p_half, product=0.0):
    """{o, gq, gk, gv: (value, bound before the last rounding)}.  p_half: half a step of the type that probabilities and score
    gradients are rounded to before they are multiplied (u where they stay in fp32).  product: what the operands' rounding
    takes from a product, relative to its size (fp32 tensors whose products run on tensor cores)."""
    dtype = q.dtype
    q, k, v, g = (t.detach().double().cpu() for t in (q, k, v, g))
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    n = Hq // Hkv
    lens = [Lk] * B if lengths is None else [min(max(int(x), 0), Lk) for x in lengths.cpu()]
    val = {key: torch.zeros_like(t) for key, t in (("o", q), ("gq", q), ("gk", k), ("gv", v))}
    err = {key: torch.zeros_like(t) for key, t in val.items()}
    for b in range(B):
        m = lens[b]
        for h in range(Hq):
            Q, K, V, G = q[b, :, h], k[b, :m, h // n], v[b, :m, h // n], g[b, :, h]
            if m == 0:
                continue
            s = Q @ K.T * scale
            p = torch.softmax(s, -1)
            o = p @ V
            # a score: D products added in fp32 (tensor cores may truncate: twice u), scaled; its exponential and the row's sum
            ds = ((2 * D + 8) * U + product) * (Q.abs() @ K.abs().T) * abs(scale)
            # parts below fp16's normal range are off by up to 2^-25 of what they were scaled to: 2^14 for the largest element
            low = 2.0 ** -38 if product else 0.0
            ds = ds + low * Q.abs().max() * K.abs().max() * D * abs(scale)
            rel = 2 * ds.max(-1, keepdim=True).values + (s.abs().max() * 4 + 16) * U + (m / 64 + 64) * 2 * U
            chain = (m / 8 + 64) * 2 * U                                 # additions along the keys
            val["o"][b, :, h] = o
            p_low = 2.0 ** -25 if p_half > U else 0.0                    # a probability against the row's largest
            err["o"][b, :, h] = (p * (rel + 2 * p_half + product + chain)) @ V.abs() + 4 * U * o.abs() + p_low * V.abs().sum(0)
            dp = G @ V.T
            delta = (G * o).sum(-1, keepdim=True)
            e_delta = (G.abs() * (err["o"][b, :, h] + half(dtype) * o.abs())).sum(-1, keepdim=True) + 2 * D * U * (G * o).abs().sum(-1, keepdim=True)
            e_dp = ((2 * D + 4) * U + product) * (G.abs() @ V.abs().T)
            d = p * (dp - delta)
            e_d = p * ((dp - delta).abs() * (rel + 2 * p_half + 4 * U) + (e_dp + e_delta) * (1 + rel + p_half))
            if p_half > U:
                e_d = e_d + 2.0 ** -38 * D * G.abs().max() * V.abs().max()
            rows = (Lq / 8 + 64) * 2 * U * n                             # additions along the queries
            val["gq"][b, :, h] = d @ K * scale
            err["gq"][b, :, h] = ((e_d + d.abs() * (chain + product)) @ K.abs()) * abs(scale)
            val["gk"][b, :m, h // n] += d.T @ Q * scale
            err["gk"][b, :m, h // n] += ((e_d + d.abs() * (rows + product)).T @ Q.abs()) * abs(scale)
            val["gv"][b, :m, h // n] += p.T @ G
            err["gv"][b, :m, h // n] += (p * (rel + 2 * p_half + product + rows)).T @ G.abs()
    return {key: (val[key], err[key]) for key in val}
