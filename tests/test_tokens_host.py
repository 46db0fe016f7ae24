"""Token operators without a GPU: refusals, the C ABI's checks, and the modules that use them."""
import ctypes

import pytest
import torch

import d2conv3d_b200 as d2c
from d2conv3d_b200 import _lib, tokens
from d2conv3d_b200.dconv_native import modules
from d2conv3d_b200.decoder import CrossAttentionBridge3d, Decoder


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="is_cuda"):
        d2c.layer_norm(x)
    with pytest.raises(RuntimeError, match="is_cuda"):
        d2c.rotary_embedding_3d(x, (1, 2, 2), (2, 2, 4))
    with pytest.raises(RuntimeError, match="is_cuda"):
        d2c.cross_attention(x, x, x)


def test_python_arguments():
    x = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="layout"):
        d2c.layer_norm(x, layout="channels")
    with pytest.raises(ValueError, match="axis_dims"):
        d2c.rotary_embedding_3d(x, (1, 2, 2), (4, 4))
    with pytest.raises(ValueError, match="grid"):
        d2c.rotary_embedding_3d(x, (2, 2), (4, 2, 2))
    with pytest.raises(ValueError, match="grid_step"):
        d2c.rotary_embedding_3d(x, torch.zeros(4, 3), (4, 2, 2), grid_step=(1, 1, 1))


class NormDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("param_dtype", ctypes.c_int32), ("layout", ctypes.c_int32), ("batch", ctypes.c_int32),
                ("channels", ctypes.c_int32), ("positions", ctypes.c_int64), ("eps", ctypes.c_float)]


class RotaryDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("dtype", "batch", "length", "heads", "dim")] + \
               [("strides", ctypes.c_int64 * 3), ("axis_dims", ctypes.c_int32 * 3), ("interleaved", ctypes.c_int32),
                ("inverse", ctypes.c_int32), ("pos_kind", ctypes.c_int32), ("grid", ctypes.c_int32 * 3),
                ("grid_step", ctypes.c_double * 3), ("pos_batch_stride", ctypes.c_int64), ("base", ctypes.c_double)]


class AttentionDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("dtype", "batch", "queries", "keys", "q_heads", "kv_heads", "dim", "lengths_i64")] + \
               [("scale", ctypes.c_float)] + [(n, ctypes.c_int64 * 3) for n in ("q", "k", "v", "g")]


def test_c_abi_checks_sizes_before_anything_is_launched():
    L = _lib.lib()

    def norm(**kw):
        f = dict(dtype=0, param_dtype=0, layout=0, batch=1, channels=8, positions=4, eps=1e-5)
        f.update(kw)
        return L.d2c_layer_norm_check(ctypes.byref(NormDesc(**f)))

    assert norm() == 0 and norm(dtype=3, param_dtype=0) == 0 and norm(layout=2) == 0
    assert norm(dtype=1) == -2 and norm(dtype=0, param_dtype=3) == -2 and norm(layout=3) == -10
    assert norm(batch=0) == -3 and norm(channels=0) == -3 and norm(positions=0) == -3
    assert norm(positions=1 << 50, channels=1 << 20) == -9
    assert L.d2c_layer_norm_check(None) == -1

    def rotary(axis=(4, 2, 2), grid=(1, 2, 2), **kw):
        f = dict(dtype=0, batch=1, length=4, heads=1, dim=8, base=1e4)
        f.update(kw)
        d = RotaryDesc(**f)
        d.axis_dims[:] = axis
        d.grid[:] = grid
        d.grid_step[:] = (1.0, 1.0, 1.0)
        return L.d2c_rotary_check(ctypes.byref(d))

    assert rotary() == 0 and rotary(axis=(0, 0, 0)) == 0
    assert rotary(axis=(4, 4, 2)) == -3 and rotary(axis=(3, 2, 2)) == -3 and rotary(dim=7) == -3 and rotary(dim=514) == -3
    assert rotary(grid=(1, 2, 3)) == -3 and rotary(grid=(0, 2, 2)) == -3 and rotary(pos_kind=4) == -10 and rotary(base=0.0) == -3

    def attention(**kw):
        f = dict(dtype=3, batch=1, queries=4, keys=4, q_heads=4, kv_heads=2, dim=64, scale=1.0)
        f.update(kw)
        return L.d2c_attention_check(ctypes.byref(AttentionDesc(**f)))

    assert attention() == 0
    assert attention(dtype=1) == -2 and attention(kv_heads=3) == -4 and attention(dim=129) == -3 and attention(dim=0) == -3
    assert attention(queries=0) == -3 and attention(keys=0) == -3
    assert attention(queries=1 << 30, q_heads=4) == -9 and attention(keys=(1 << 30) + 1, kv_heads=1) == -9
    assert attention(batch=1 << 20, q_heads=8, kv_heads=8) == 0
    assert L.d2c_status_string(-13) != b"unknown status"


def test_convolutions_refuse_the_token_types():
    d = _lib.ConvDesc(3, 1, 8, 8, 4, 6, 6, 3, 3, 3, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 2)
    od = (ctypes.c_int64 * 4)(2 * 81, 4, 6, 6)
    assert _lib.lib().d2c_deform_conv3d_check(ctypes.byref(d), od, None) == -2


def test_default_axis_dims():
    for dim in range(2, 130):
        n = tokens.default_axis_dims(dim)
        assert all(a >= 0 and a % 2 == 0 for a in n) and sum(n) == dim - dim % 2


def test_modules_that_use_them():
    layer = modules.MDConv3d(8, 8, 3, padding=1, norm_type="LayerNorm3d")
    assert isinstance(layer.norm, d2c.LayerNorm3d) and layer.norm.weight.shape == (8,)
    net = Decoder(widths=(8, 16, 32, 64), channels=32, conv=None, bridge="cross_attention")
    assert isinstance(net.gc, CrossAttentionBridge3d)
    with pytest.raises(ValueError, match="bridge"):
        Decoder(widths=(8, 16, 32, 64), channels=32, conv=None, bridge="none")
    # what was there keeps its parameters
    assert set(k.split(".")[0] for k in Decoder(widths=(8, 16, 32, 64), channels=32, conv=None).state_dict()) == \
        {"gc", "convG1", "convG2", "rf3", "rf2", "rf1", "pred"}
