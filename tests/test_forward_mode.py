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
