"""Saved-tensor hooks decide what a backward gets back: another layout gives the same gradients, another tensor is refused."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

import d2conv3d_b200 as d2c

pytestmark = pytest.mark.gpu


def other_layout(t):
    """The same values with the last dimension's elements apart, behind an odd offset."""
    wide = torch.zeros(t.numel() * 3 + 1, dtype=t.dtype, device=t.device)
    return wide[1:].view(*t.shape, 3)[..., 0].copy_(t) if t.dim() else t.clone()


def last_dimensions_swapped(t):
    return t.mT.contiguous().mT if t.dim() > 1 else t.clone()


def kept(t):
    return t


HOOKS = {"kept": lambda: saved_tensors_hooks(kept, kept), "save_on_cpu": save_on_cpu,
         "dense": lambda: saved_tensors_hooks(lambda t: t.contiguous().clone(), kept),
         "apart": lambda: saved_tensors_hooks(other_layout, kept), "swapped": lambda: saved_tensors_hooks(kept, last_dimensions_swapped)}


def norm(dtype, layout):
    x = torch.randn(2, 40, 3, 4, 5, device="cuda").to(dtype)
    x = x.movedim(1, -1).requires_grad_() if layout == "channels_last" else x.requires_grad_()
    leaves = [x] + [torch.randn(40, device="cuda").requires_grad_() for _ in range(2)]
    return leaves, lambda: d2c.layer_norm(*leaves, layout=layout)


def rotary(dtype, layout):
    x = torch.randn(2, 50, 3, 32, device="cuda").to(dtype).requires_grad_()
    where = torch.randint(0, 1000, (2, 3, 50), device="cuda").mT
    return [x], lambda: d2c.rotary_embedding_3d(x, where, (8, 12, 12))


def attention(dtype, layout):
    """Strided views, as a block's fused projection of keys and values gives them."""
    lq = 3 if layout == "few" else 150
    q = torch.randn(2, 4, lq, 64, device="cuda").to(dtype).requires_grad_()
    kv = torch.randn(2, 300, 2, 2, 64, device="cuda").to(dtype).requires_grad_()
    n = torch.tensor([300, 170, 5, 5], device="cuda")[::2]
    return [q, kv], lambda: d2c.cross_attention(q.transpose(1, 2), kv[:, :, 0], kv[:, :, 1], key_lengths=n)


def layer(dtype, kind):
    from d2conv3d_b200.dconv_native import modules
    cls, kw = {"offsets": (modules.MDConv3d, dict(init="random", fused_head=False)), "head": (modules.MDConv3d, dict(init="random")),
               "field": (modules.XYZSizeConditionedMDConv3d, dict(init="random", fused_head=False))}[kind]
    m = cls(64, 64, 3, padding=1, **kw).cuda()
    x = torch.randn(1, 64, 3, 6, 7, device="cuda", requires_grad=True)
    return [x] + list(m.parameters()), lambda: m(x)


def conv1d(dtype, _):
    x = torch.randn(2, 8, 33, device="cuda", requires_grad=True)
    off, w = torch.randn(2, 3, 33, device="cuda", requires_grad=True), torch.randn(6, 8, 3, device="cuda", requires_grad=True)
    return [x, off, w], lambda: d2c.dconv_native._ops.deform_conv1d(x, off, None, w, None, 1, 1, 1, 1, 1)


def depthwise(dtype, _):
    m = d2c.DepthwiseConv3d(16, 16, 3, padding=1, groups=16).cuda().to(dtype)
    x = torch.randn(2, 16, 4, 6, 8, device="cuda").to(dtype).requires_grad_()
    return [x] + list(m.parameters()), lambda: m(x)


def act_group_norm(dtype, _):
    x = torch.randn(2, 16, 4, 6, 8, device="cuda", requires_grad=True)
    w, b = (torch.randn(16, device="cuda", requires_grad=True) for _ in range(2))
    return [x, w, b], lambda: d2c._lib.act_group_norm(x, w, b, 1)


CASES = [(norm, "channels_last"), (norm, "channels_first"), (norm, "tokens"), (rotary, ""), (attention, "many"), (attention, "few")]
IDS = ["norm_rows", "norm_volume", "norm_tokens", "rotary", "attention", "attention_few"]
CONVOLUTIONS = [(layer, "offsets"), (layer, "head"), (layer, "field"), (conv1d, ""), (depthwise, ""), (act_group_norm, "")]
CONVOLUTION_IDS = ["offsets", "head", "field", "conv1d", "depthwise", "act_group_norm"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_gradients_do_not_depend_on_the_layout_that_comes_back(case, dtype):
    torch.manual_seed(0)
    leaves, call = case[0](dtype, case[1])
    y = call()
    g = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, g)
    for name, hooks in HOOKS.items():
        with hooks():
            y = call()
        for a, b in zip(torch.autograd.grad(y, leaves, g), want):
            assert torch.equal(a, b), name


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("change", ["size", "type", "device"])
def test_another_tensor_is_refused(case, change):
    torch.manual_seed(0)
    leaves, call = case[0](torch.float32, case[1])
    back = {"size": lambda t: t[:1], "type": lambda t: t.double(), "device": lambda t: t.cpu()}[change]
    with saved_tensors_hooks(kept, back):
        y = call()
    with pytest.raises(RuntimeError, match="saved tensor came back"):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.parametrize("case", CONVOLUTIONS, ids=CONVOLUTION_IDS)
def test_convolutions_take_the_layout_that_comes_back(case):
    torch.manual_seed(0)
    leaves, call = case[0](torch.float32, case[1])
    with torch.no_grad():
        g = torch.randn_like(call())
    want = torch.autograd.grad(call(), leaves, g)
    for name, hooks in HOOKS.items():
        with hooks():
            y = call()
        for a, b in zip(torch.autograd.grad(y, leaves, g), want):
            # the gradients of a deformable layer's input are sums by atomics: fp32 sums of some hundred terms in another order
            assert (a - b).abs().max() <= 1e-5 * b.abs().max(), name


@pytest.mark.parametrize("case", CONVOLUTIONS, ids=CONVOLUTION_IDS)
@pytest.mark.parametrize("change", ["size", "type", "device"])
def test_convolutions_refuse_another_tensor(case, change):
    torch.manual_seed(0)
    leaves, call = case[0](torch.float32, case[1])
    back = {"size": lambda t: t[:1], "type": lambda t: t.double(), "device": lambda t: t.cpu()}[change]
    with saved_tensors_hooks(kept, lambda t: back(t) if t.numel() != t[:1].numel() or change != "size" else t.flatten()):
        y = call()
    with pytest.raises(RuntimeError, match="came back"):
        torch.autograd.grad(y, leaves, torch.ones_like(y))
