"""Forward-mode derivatives are refused, not dropped: the operators have none."""
import pytest
import torch
from torch.autograd import forward_ad

import d2conv3d_b200 as d2c


def duals(count, at, *shape):
    """`count` tensors, the one at `at` with a tangent."""
    ts = [torch.randn(shape) for _ in range(count)]
    ts[at] = forward_ad.make_dual(ts[at], torch.ones(shape))
    return ts


def test_token_operators():
    with forward_ad.dual_level():
        x = duals(1, 0, 1, 4, 2, 8)[0]
        w = duals(2, 1, 8)
        for call in (lambda: d2c.layer_norm(x), lambda: d2c.layer_norm(torch.randn(4, 8), *w),
                     lambda: d2c.rotary_embedding_3d(x, (1, 2, 2), (4, 2, 2)),
                     *(lambda i=i: d2c.cross_attention(*duals(3, i, 1, 4, 2, 8)) for i in range(3))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            d2c.layer_norm(x)


def test_a_primal_passes_the_check():
    with forward_ad.dual_level():
        x = forward_ad.unpack_dual(duals(1, 0, 1, 4, 2, 8)[0]).primal
        with pytest.raises(RuntimeError, match="is_cuda"):
            d2c.layer_norm(x)


def test_convolutions():
    with forward_ad.dual_level():
        x, w, off = torch.randn(1, 8, 3, 5, 5), torch.randn(8, 8, 3, 3, 3), torch.zeros(1, 81, 3, 5, 5)
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        native = d2c._lib.native()
        three = (1, 1, 1)
        for i in range(3):
            t = [x, off, w]
            t[i] = dual(t[i])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                native.deform_conv3d(t[0], t[1], None, t[2], None, three, three, three, 1, 1, False)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                native.deform_conv3d_head(t[0], t[1], t[2], None, -1, -1, 0, 0, three, three, three, 1, 1, None)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            native.dyn_dilated_conv3d(x, dual(torch.ones(1, 1, 3, 5, 5)), None, w, None, 0, three, three, three, 1, 1, False)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            native.deform_conv1d(dual(torch.randn(1, 8, 9)), torch.zeros(1, 3, 9), None, torch.randn(8, 8, 3), None, 1, 1, 1, 1, 1, False)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            native.depthwise_conv3d(dual(x), torch.randn(8, 1, 3, 3, 3), None, three, three, three)
