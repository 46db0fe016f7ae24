"""Performance cases of the token operators: layer norm, rotary positions over (time, height, width), and cross attention
between the tokens of two pyramid levels.

A case is a dict of plain values.  `prepare` makes what the program has in hand before the call, `run` makes the call:
the framework's operators where `own` is true, otherwise the same formulas in elementary tensor operations in 32 bits.
A training step returns the output and the gradients of every input and parameter.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def _norm(name, layout, dtype, b, c, dims, train):
    return dict(name=name, kind="norm", layout=layout, dtype=dtype, b=b, c=c, d=dims[0], h=dims[1], w=dims[2], train=train)


def _rotary(name, dtype, b, dims, heads, dim, axes, positions, interleaved, train):
    return dict(name=name, kind="rotary", dtype=dtype, b=b, d=dims[0], h=dims[1], w=dims[2], heads=heads, dim=dim, at=axes[0],
                ah=axes[1], aw=axes[2], positions=positions, interleaved=interleaved, train=train)


def _attend(name, dtype, b, lq, lk, hq, hkv, dim, ragged, train):
    return dict(name=name, kind="attend", dtype=dtype, b=b, lq=lq, lk=lk, hq=hq, hkv=hkv, dim=dim, ragged=ragged, train=train)


def listed():
    return [
        # token rows of one frame of the coarsest pyramid level of a 480 x 854 clip: launches and host time
        _norm("norm_frame", "channels_last", "bfloat16", 1, 256, (1, 15, 27), False),
        # the predictor's input norm in a refine block at stride 8 (odd width), the training scripts' two clips
        _norm("norm_volume_train", "channels_first", "float32", 2, 256, (8, 60, 107), True),
        # a stage-4 feature volume turned into the keys' token rows before their projection
        _norm("norm_tokens_train", "tokens", "bfloat16", 2, 1024, (8, 30, 54), True),
        # token rows of the stage-4 level between attention blocks, under fp16 autocast
        _norm("norm_rows_train", "channels_last", "float16", 4, 512, (8, 30, 54), True),
        # queries of one frame at stride 32, serving
        _rotary("rotary_frame", "bfloat16", 1, (1, 15, 27), 4, 64, (16, 24, 24), "grid", False, False),
        # keys of the stage-4 level, two clips, training in fp32
        _rotary("rotary_train", "float32", 2, (8, 30, 54), 8, 64, (16, 24, 24), "grid", False, True),
        # queries of the stride-4 level with positions of their own (crops of a long video), neighbouring pairs
        _rotary("rotary_positions", "bfloat16", 1, (8, 120, 214), 8, 32, (8, 12, 12), "tensor", True, False),
        # one pooled query of each head against the stage-4 states of a clip, grouped heads: serving, latency counts
        _attend("attend_one", "bfloat16", 1, 1, 12960, 8, 2, 64, False, False),
        # one frame of the stride-32 level against four clips' states of unlike lengths, serving in fp16
        _attend("attend_frame", "float16", 4, 405, 12960, 8, 8, 64, True, False),
        # the bridge of the decoder in training: stride-32 tokens look at the stage-4 level of two clips
        _attend("attend_train", "bfloat16", 2, 3240, 12960, 4, 4, 64, True, True),
        # the same on a shorter clip in fp32, the type that the rest of the network trains in
        _attend("attend_train_fp32", "float32", 1, 1215, 3240, 4, 4, 64, False, True),
        # the stride-8 level of a clip looks at its stage-4 level, wide heads shared by two
        _attend("attend_wide", "bfloat16", 1, 51360, 12960, 4, 2, 128, False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _volume(rng, most):
    """Clip sizes D, H, W of at most `most` voxels: up to 16 frames, up to the stride-4 level of a 480 x 854 clip."""
    while True:
        d, h, w = _log(rng, 1, 16), _log(rng, 1, 120), _log(rng, 1, 214)
        if d * h * w <= most:
            return d, h, w


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attend", "attend"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    train = rng.random() < 0.6
    if kind == "norm":
        c = rng.choice([64, 128, 256, 512, 1024, 2048, _log(rng, 16, 2048)])
        b = _log(rng, 1, 4)
        dims = _volume(rng, max(1, min(205440, (1 << 27) // (b * c))))
        return _norm("", rng.choice(["channels_last", "channels_first", "tokens"]), dtype, b, c, dims, train)
    if kind == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128])
        heads, b = _log(rng, 1, 16), _log(rng, 1, 4)
        dims = _volume(rng, max(1, min(205440, (1 << 27) // (b * heads * dim))))
        part = 2 * (dim // 6)
        axes = rng.choice([(dim - 2 * part, part, part), (part, part, part), (0, dim // 2, dim // 2)])
        return _rotary("", dtype, b, dims, heads, dim, axes, rng.choice(["grid", "tensor"]), rng.random() < 0.5, train)
    dim = rng.choice([32, 64, 64, 128, 8 * rng.randint(2, 16)])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 1, 2, 4])
    b = _log(rng, 1, 4)
    most = 1.2e9 if train else 2.4e9              # scores in all; the largest listed case has 2.66e9
    if dtype == "float32":
        most /= 8
    while True:
        # with one or two keys the gradients of queries and keys are differences of equal numbers: no training on those
        lq, lk = rng.choice([1, _log(rng, 2, 51360), _log(rng, 32, 51360)]), _log(rng, 32 if train else 1, 51360)
        if b * hq * lq * lk <= most and b * lk * hkv * dim <= 1 << 27:
            break
    return _attend("", dtype, b, lq, lk, hq, hkv, dim, rng.random() < 0.5, train)


def _lengths(case):
    """Valid keys of each clip of a ragged batch: from all of them down to about half."""
    b, lk = case["b"], case["lk"]
    return [max(1, lk - (lk * i) // (2 * b) - (i * 7) % 13) for i in range(b)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 1000003 + 17)
    dtype = _TYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, std=1.0, mean=0.0, leaf=False, kind=dtype):
        t = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).mul_(std).add_(mean).to(kind)
        return t.requires_grad_() if leaf and train else t

    state = dict(case=case)
    if case["kind"] == "norm":
        b, c, dims = case["b"], case["c"], (case["d"], case["h"], case["w"])
        n = dims[0] * dims[1] * dims[2]
        shape = (b, n, c) if case["layout"] == "channels_last" else (b, c) + dims
        out = (b, c) + dims if case["layout"] == "channels_first" else (b, n, c)
        # features behind an activation lie off zero
        state.update(x=normal(*shape, std=1.3, mean=0.4, leaf=True), weight=normal(c, std=0.2, mean=1.0, leaf=True),
                     bias=normal(c, std=0.2, leaf=True))
        if train:
            state["g"] = normal(*out, std=0.5)
    elif case["kind"] == "rotary":
        b, n = case["b"], case["d"] * case["h"] * case["w"]
        state["x"] = normal(b, n, case["heads"], case["dim"], leaf=True)
        if case["positions"] == "grid":
            state["positions"] = (case["d"], case["h"], case["w"])
        else:
            # clips start anywhere in their videos, crops anywhere in their frames
            start = torch.randint(0, 100000, (b, 1, 3), generator=gen, device=dev)
            state["positions"] = (_grid(case, dev) + start).to(torch.int32)
        if train:
            state["g"] = normal(*state["x"].shape, std=0.5)
    else:
        b, lq, lk, hq, hkv, dim = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "dim"))
        state.update(q=normal(b, lq, hq, dim, std=1.2, leaf=True), k=normal(b, lk, hkv, dim, std=1.2, leaf=True),
                     v=normal(b, lk, hkv, dim, leaf=True), lengths=None)
        if case["ragged"]:
            order = torch.randperm(b, generator=gen, device=dev)
            state["lengths"] = torch.tensor(_lengths(case), device=dev, dtype=torch.int32)[order]
        if train:
            state["g"] = normal(b, lq, hq, dim, std=0.5)
    return state


def _grid(case, dev):
    """Positions [D*H*W, 3] of a clip's voxels in row-major order."""
    axes = [torch.arange(case[k], device=dev) for k in ("d", "h", "w")]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _rows(t, layout):
    """Channels last: [B, positions, C]."""
    return t if layout == "channels_last" else t.flatten(2).transpose(1, 2)


def _plain_norm(s):
    case, layout = s["case"], s["case"]["layout"]
    x, w, b = _rows(s["x"].detach(), layout).float(), s["weight"].detach().float(), s["bias"].detach().float()
    centred = x - x.mean(-1, keepdim=True)
    r = (centred.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    h = centred * r
    y = h * w + b

    def back(t):
        return t if layout == "channels_last" else t.transpose(1, 2).reshape(s["x"].shape)

    dtype = s["x"].dtype
    out = {"y": (back(y) if layout == "channels_first" else y).to(dtype).contiguous()}
    if case["train"]:
        g = (_rows(s["g"], layout) if layout == "channels_first" else s["g"]).float()
        gh = g * w
        gx = r * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True))
        out.update(gx=back(gx).to(dtype).contiguous(), gw=(g * h).sum((0, 1), dtype=torch.float64).to(dtype),
                   gb=g.sum((0, 1), dtype=torch.float64).to(dtype))
    return out


def _turned(x, sections, interleaved, sign):
    """x [B, L, H, D] with every section's pairs turned; sections: (first channel, channels, cos, sin)."""
    x = x.float()

    def turn(part, cos, sin):
        if interleaved:
            u, v = part[..., 0::2], part[..., 1::2]
        else:
            u, v = part.chunk(2, -1)
        a, b = u * cos - v * sin * sign, u * sin * sign + v * cos
        return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)

    parts = [turn(x[..., c0:c0 + n], cos, sin) for c0, n, cos, sin in sections]
    end = sections[-1][0] + sections[-1][1]
    return torch.cat(parts + [x[..., end:]], -1)


def _plain_rotary(s):
    case, x = s["case"], s["x"].detach()
    p = _grid(case, x.device) if case["positions"] == "grid" else s["positions"]
    p = p.to(torch.float64)
    p = p[None] if p.dim() == 2 else p

    def section(axis, c0, n):
        # far positions: the angle in 64 bits
        freq = torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=x.device),
                         -torch.arange(0, n, 2, dtype=torch.float64, device=x.device) / n)
        angle = p[..., axis, None, None] * freq
        return c0, n, angle.cos().float(), angle.sin().float()

    at, ah, aw = case["at"], case["ah"], case["aw"]
    sections = [section(a, c0, n) for a, c0, n in ((0, 0, at), (1, at, ah), (2, at + ah, aw)) if n]
    out = {"y": _turned(x, sections, case["interleaved"], 1.0).to(x.dtype)}
    if case["train"]:
        out["gx"] = _turned(s["g"], sections, case["interleaved"], -1.0).to(x.dtype)
    return out


def _plain_attend(s):
    case = s["case"]
    b, lq, lk, hq, hkv, dim = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "dim"))
    n = hq // hkv
    dtype, scale = s["q"].dtype, 1.0 / math.sqrt(dim)

    def by_kv_head(t):                              # [B, Lq, Hq, D] -> [B, Hkv, n * Lq, D]
        return t.detach().float().view(b, lq, hkv, n, dim).permute(0, 2, 3, 1, 4).reshape(b, hkv, n * lq, dim)

    def by_token(t):
        return t.view(b, hkv, n, lq, dim).permute(0, 3, 1, 2, 4).reshape(b, lq, hq, dim)

    q = by_kv_head(s["q"])
    k, v = (s[t].detach().float().transpose(1, 2) for t in ("k", "v"))
    p = (q * scale) @ k.transpose(2, 3)
    if s["lengths"] is not None:
        behind = torch.arange(lk, device=q.device)[None] >= s["lengths"][:, None]
        p.masked_fill_(behind[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = p @ v
    out = {"o": by_token(o).to(dtype)}
    if case["train"]:
        g = by_kv_head(s["g"])
        gv = p.transpose(2, 3) @ g
        ds = g @ v.transpose(2, 3)
        ds.sub_((g * o).sum(-1, keepdim=True)).mul_(p)
        gq = (ds @ k) * scale
        gk = (ds.transpose(2, 3) @ q) * scale
        out.update(gq=by_token(gq).to(dtype), gk=gk.transpose(1, 2).to(dtype), gv=gv.transpose(1, 2).to(dtype))
    return out


# ---- the framework's operators --------------------------------------------------------------------------------------


def _own(s):
    import d2conv3d_b200 as d2c
    case = s["case"]
    if case["kind"] == "norm":
        leaves = (s["x"], s["weight"], s["bias"])
        y = d2c.layer_norm(*leaves, eps=1e-5, layout=case["layout"])
        names = ("y", "gx", "gw", "gb")
    elif case["kind"] == "rotary":
        leaves = (s["x"],)
        y = d2c.rotary_embedding_3d(s["x"], s["positions"], (case["at"], case["ah"], case["aw"]),
                                    interleaved=case["interleaved"])
        names = ("y", "gx")
    else:
        leaves = (s["q"], s["k"], s["v"])
        y = d2c.cross_attention(*leaves, key_lengths=s["lengths"])
        names = ("o", "gq", "gk", "gv")
    grads = torch.autograd.grad(y, leaves, s["g"]) if case["train"] else ()
    return dict(zip(names, (y.detach(),) + tuple(grads)))


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attend": _plain_attend}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    size = _BYTES[case["dtype"]]
    passes = 5 if case["train"] else 2              # tensors as large as the input: x, y; and g, gx, x again for its gradient
    if case["kind"] == "norm":
        n = case["b"] * case["d"] * case["h"] * case["w"] * case["c"]
        return {"bytes": passes * size * n, "flops": (20 if case["train"] else 8) * n}
    if case["kind"] == "rotary":
        n = case["b"] * case["d"] * case["h"] * case["w"] * case["heads"] * case["dim"]
        return {"bytes": (4 if case["train"] else 2) * size * n, "flops": (6 if case["train"] else 3) * n}
    b, lq, lk, hq, hkv, dim = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "dim"))
    keys = sum(_lengths(case)) if case["ragged"] else b * lk
    q, kv = b * lq * hq * dim, keys * hkv * dim
    tensors = (4 * q + 4 * kv) if case["train"] else (2 * q + 2 * kv)
    return {"bytes": size * tensors, "flops": (14 if case["train"] else 4) * lq * keys * hq * dim}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------


def _exact_norm(s):
    case = s["case"]
    first = case["layout"] != "channels_last"
    axis = 1 if first else -1
    x, w, b = (s[k].detach().double() for k in ("x", "weight", "bias"))
    shape = (1, -1, 1, 1, 1) if first else (1, 1, -1)
    var, mean = torch.var_mean(x, axis, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w.view(shape) + b.view(shape)
    tokens = case["layout"] == "tokens"
    out = {"y": y.flatten(2).mT if tokens else y}
    if case["train"]:
        g = s["g"].double()
        g = g.mT.reshape(x.shape) if tokens else g
        sums = [a for a in range(x.dim()) if a != axis % x.dim()]
        unit = (x - mean) / torch.sqrt(var + 1e-5)
        inner = g * w.view(shape)
        # dy/dx of a unit vector: what lies along 1 and along the vector itself is taken out
        gx = inner - inner.mean(axis, keepdim=True) - unit * (inner * unit).mean(axis, keepdim=True)
        out.update(gx=gx / torch.sqrt(var + 1e-5), gw=(g * unit).sum(sums), gb=g.sum(sums))
    return out


def _exact_rotary(s):
    case, x = s["case"], s["x"].detach().double()
    n = (case["at"], case["ah"], case["aw"])
    p = _grid(case, x.device)[None] if case["positions"] == "grid" else s["positions"]
    phases, places = [], []
    for axis, size in enumerate(n):
        for i in range(size // 2):
            phases.append(p[..., axis].double() * 10000.0 ** (-2.0 * i / size))
            c0 = sum(n[:axis])
            places.append((c0 + 2 * i, c0 + 2 * i + 1) if case["interleaved"] else (c0 + i, c0 + i + size // 2))
    wave = torch.stack(phases, -1)[:, :, None]
    wave = torch.complex(wave.cos(), wave.sin())
    re, im = ([pair[j] for pair in places] for j in (0, 1))

    def turn(t, w):
        z = torch.complex(t[..., re], t[..., im]) * w
        y = t.clone()
        y[..., re], y[..., im] = z.real, z.imag
        return y

    out = {"y": turn(x, wave)}
    if case["train"]:
        out["gx"] = turn(s["g"].double(), wave.conj())
    return out


def _exact_attend(s):
    case = s["case"]
    n = case["hq"] // case["hkv"]
    q, k, v = (s[t].detach().double() for t in ("q", "k", "v"))
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if case["train"] else []
    rows = max(1, (1 << 30) // case["lk"])
    for b in range(case["b"]):
        keys = case["lk"] if s["lengths"] is None else int(s["lengths"][b])
        for h in range(case["hq"]):
            kk, vv = k[b, :keys, h // n], v[b, :keys, h // n]
            for r in range(0, case["lq"], rows):
                at = slice(r, r + rows)
                p = torch.softmax(q[b, at, h] @ kk.T / math.sqrt(case["dim"]), -1)
                o[b, at, h] = p @ vv
                if case["train"]:
                    g = s["g"][b, at, h].double()
                    d = g @ vv.T
                    d = p * (d - (p * d).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
                    grads[0][b, at, h] = d @ kk
                    grads[1][b, :keys, h // n] += d.T @ q[b, at, h]
                    grads[2][b, :keys, h // n] += p.T @ g
    return dict(zip(("o", "gq", "gk", "gv"), [o] + grads))


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attend": _exact_attend}[case["kind"]](state)
