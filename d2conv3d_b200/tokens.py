"""Token operators and the modules made of them: layer norm over the channels of a position, rotary positions on the
(time, height, width) grid, and cross attention between the tokens of two pyramid levels.

All of them run as the library's own kernels on CUDA tensors in float32, float16 or bfloat16, forward and backward; there is
no eager stand-in.  Arithmetic, statistics and sums are fp32, a 16-bit result is rounded once.  Every call gives the same bits
for the same inputs (no atomics), launches on the current stream of the tensors' device and can be captured into a CUDA graph.
"""
import math

import torch
import torch.nn as nn

from . import _lib

_NO_GRID, _UNIT_STEP = (0, 0, 0), (1.0, 1.0, 1.0)
_LAYOUTS = {"channels_last": 0, "channels_first": 1, "tokens": 2}


def layer_norm(input, weight=None, bias=None, eps=1e-5, layout="channels_last"):
    """Layer norm over the channels of every position: (x - mean) / sqrt(var + eps) * weight + bias, biased variance.

    layout   "channels_last":  input [..., C], normalised over its last dimension; the result has the input's shape
             "channels_first": input [B, C, *spatial], normalised over dimension 1; the result has the input's shape
             "tokens":         input [B, C, *spatial], the result is token rows [B, positions, C]
    weight, bias: [C], both float32 or both of the input's type, either may be None.  Differentiable in all three."""
    try:
        code = _LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"unexpected layout '{layout}': one of {sorted(_LAYOUTS)}") from None
    return _lib.native().layer_norm(input, weight, bias, eps, code)


def rotary_embedding_3d(x, positions, axis_dims, base=10000.0, interleaved=False, grid_step=None):
    """Turns pairs of a head's channels by angles that grow with a token's time, height and width.

    x          [B, L, H, D] with any strides; the result is contiguous
    positions  (T, H, W): the tokens are this volume's voxels in row-major order; or a tensor [L, 3] / [B, L, 3] of
               (time, height, width), int32, int64 or float32.  Angles are formed in 64 bits: a position p costs up to
               p * 2^-50 radians, which float32's own rounding (2^-23) hides up to p = 2^27
    axis_dims  channels that time, height and width turn: even, in this order from the first channel on; channels behind
               their sum stay as they are
    base       pair i of an axis with n channels turns by position * base^(-2 i / n)
    interleaved  pairs are neighbouring channels (2i, 2i + 1) instead of (i, i + n / 2)
    grid_step  with a grid: cell size on each axis, position = (index + 1/2) * step - 1/2, so that the levels of a pyramid
               share one frame; 1 if None
    Differentiable in x."""
    if len(axis_dims) != 3:
        raise ValueError(f"axis_dims must have three entries, got {axis_dims}")
    if torch.is_tensor(positions):
        if grid_step is not None:
            raise ValueError("grid_step goes with a grid, not with positions of its own")
        return _lib.native().rotary_embedding_3d(x, positions, _NO_GRID, _UNIT_STEP, axis_dims, base, interleaved)
    step = _UNIT_STEP if grid_step is None else grid_step
    if len(positions) != 3 or len(step) != 3:
        raise ValueError("a grid and its steps have three entries")
    return _lib.native().rotary_embedding_3d(x, None, positions, step, axis_dims, base, interleaved)


def cross_attention(query, key, value, key_lengths=None, scale=None):
    """softmax(scale * query key^T) value for every head, the keys of another length than the queries.

    query        [B, Lq, Hq, D], key and value [B, Lk, Hkv, D], D <= 128; any strides; Hq a multiple of Hkv, neighbouring
                 query heads share a key head
    key_lengths  [B] int32 or int64: keys of a clip behind its length are not looked at, whatever they hold (their gradients
                 are zero); a clip without keys gives zeros.  Values are clamped to 0 .. Lk.
    scale        1 / sqrt(D) if None
    The result is [B, Lq, Hq, D], contiguous.  Differentiable in query, key and value."""
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, query.shape[-1]))
    return _lib.native().cross_attention(query, key, value, key_lengths, scale)


class LayerNorm3d(nn.Module):
    """Layer norm over the channels of every voxel of a volume [B, C, D, H, W]; with tokens=True the result is [B, D*H*W, C]."""

    def __init__(self, channels, eps=1e-5, tokens=False):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))
        self.eps = eps
        self.tokens = tokens

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps, "tokens" if self.tokens else "channels_first")


def default_axis_dims(dim):
    """A head's channels shared out to time, height and width, as evenly as even numbers allow."""
    part = 2 * (dim // 6)
    return dim - dim % 2 - 2 * part, part, part


class CrossAttention3d(nn.Module):
    """Pre-norm cross attention between two volumes: every voxel of x [B, channels, D, H, W] looks at all voxels of context
    [B, context_channels, D', H', W'], and the result is added to x.  Rotary positions are in the context's voxels, so that
    the two levels share one frame.  context_lengths: as key_lengths of cross_attention, in row-major voxels (clips whose
    last frames are padding)."""

    def __init__(self, channels, context_channels, heads=4, kv_heads=None, head_dim=64, axis_dims=None):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads or heads, head_dim
        self.axis_dims = tuple(axis_dims) if axis_dims is not None else default_axis_dims(head_dim)
        self.norm = LayerNorm3d(channels, tokens=True)
        self.context_norm = LayerNorm3d(context_channels, tokens=True)
        self.to_q = nn.Linear(channels, heads * head_dim, bias=False)
        self.to_kv = nn.Linear(context_channels, 2 * self.kv_heads * head_dim, bias=False)
        self.to_out = nn.Linear(heads * head_dim, channels)

    def forward(self, x, context, context_lengths=None):
        b, grid, from_grid = x.shape[0], x.shape[2:], context.shape[2:]
        q = self.to_q(self.norm(x)).view(b, -1, self.heads, self.head_dim)
        kv = self.to_kv(self.context_norm(context)).view(b, -1, 2, self.kv_heads, self.head_dim)
        step = [m / n for n, m in zip(grid, from_grid)]
        q = rotary_embedding_3d(q, tuple(grid), self.axis_dims, grid_step=step)
        k = rotary_embedding_3d(kv[:, :, 0], tuple(from_grid), self.axis_dims)
        o = cross_attention(q, k, kv[:, :, 1], context_lengths)
        return x + self.to_out(o.flatten(2)).transpose(1, 2).reshape(x.shape)
