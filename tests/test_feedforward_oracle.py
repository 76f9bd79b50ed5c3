"""The plain forms that the feed-forward operators are compared with, and what
the entry points refuse before they touch a device.  CPU only."""
from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

import feedforward_ref as R
from conftest import ROOT
import train_station_amd as T
from train_station_amd._ffi import LinearShape, gradtrack, hip, last_error

EINVAL, EWORKSPACE = 100001, 100003


def test_packed_values_hold_their_bounds():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((7, 333)) * 10.0 ** rng.integers(-30, 30, (7, 333))
    codes, scales = R.pack8(x)
    assert codes.shape == (7, 384) and scales.shape == (3, 7, 4)
    v = R.unpack8(codes, scales, 333)
    k = scales.transpose(1, 0, 2).reshape(7, -1).repeat(32, 1)[:, :333].astype(int) - 127
    assert np.all(np.abs(v - x) <= np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** (k - 10.0)))
    assert not codes[:, 333:].any()
    # the smallest scale: half of it would not hold the block's largest
    top = np.abs(np.pad(x, ((0, 0), (0, 51)))).reshape(7, -1, 32).max(2)
    ks = scales.transpose(1, 0, 2).reshape(7, -1).astype(int) - 127
    assert np.all(top <= 448 * 2.0 ** ks) and np.all((top > 448 * 2.0 ** (ks - 1.0)) | (ks == -117))


def test_codes_are_exact_at_their_own_values():
    x = np.resize(R.e4m3_values()[:127], (127, 32))
    x[:, 0] = 448.0  # the scale of every block is 1
    codes, scales = R.pack8(x)
    assert np.all(scales[0, :, 0] == 127) and np.array_equal(R.unpack8(codes, scales, 32), x)


@pytest.mark.parametrize("name", ["none", "silu", "gelu_tanh"])
def test_layer_gradients_are_the_differences(name):
    rng = np.random.default_rng(1)
    x, w, b = rng.standard_normal((5, 7)), rng.standard_normal((7, 6)), rng.standard_normal(6)
    go, t = rng.standard_normal((5, 6)), 1e-6
    y, z = R.linear(x, w, b, name, None)
    dx, dw, db = R.linear_grads(x, w, z, name, go)
    loss = lambda x, w, b: (R.linear(x, w, b, name, None)[0] * go).sum()  # noqa: E731
    for a, g, at in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        d = rng.standard_normal(a.shape)
        args = [x, w, b]
        lo, hi = list(args), list(args)
        lo[at], hi[at] = a - t * d, a + t * d
        assert abs((loss(*hi) - loss(*lo)) / (2 * t) - (g * d).sum()) < 1e-7 * (1 + np.abs(g * d).sum())


def test_norm_gradients_are_the_differences():
    rng = np.random.default_rng(2)
    h, w, go, t = rng.standard_normal((4, 9)), rng.standard_normal(9), rng.standard_normal((4, 9)), 1e-6
    dh, dw = R.rms_norm_grads(h, w, go, 1e-3)
    for a, g, f in ((h, dh, lambda a: R.rms_norm(a, w, 1e-3)), (w, dw, lambda a: R.rms_norm(h, a, 1e-3))):
        d = rng.standard_normal(a.shape)
        diff = ((f(a + t * d) - f(a - t * d)) * go).sum() / (2 * t)
        assert abs(diff - (g * d).sum()) < 1e-7 * (1 + np.abs(g * d).sum())


# ---- refusals (before any launch) -------------------------------------------------

P = 0x10000  # stands for a device pointer: nothing here gets as far as reading it


def linear(shape=(4, 8, 16), x=P, w=P, act=0, y=P, codes=None, scales=None, ws=None, floats=1 << 40):
    s = LinearShape(*shape)
    return hip.ts_hip_linear(ctypes.byref(s), x, w, None, act, None, y, None, codes, scales, ws, floats, None)


def backward(shape=(4, 8, 16), x=P, codes=None, scales=None, w=P, act=0, slope=None, go=P, dx=P, ws=P, floats=1 << 40):
    s = LinearShape(*shape)
    return hip.ts_hip_linear_backward(ctypes.byref(s), x, codes, scales, w, None, act, slope, go, dx, None, None, ws, floats,
                                      None)


def test_layer_entries_refuse():
    assert linear(act=4) == EINVAL and linear(act=-1) == EINVAL
    assert linear(x=None) == EINVAL and linear(w=None) == EINVAL and linear(y=None) == EINVAL
    assert linear(codes=P) == EINVAL and linear(scales=P) == EINVAL
    assert linear(shape=(1 << 24, 8, 8)) == EINVAL and linear(shape=(1 << 22, 8, 1 << 22)) == EINVAL
    assert linear(shape=(0, 8, 16)) == 0  # nothing to do
    assert hip.ts_hip_linear(None, P, P, None, 0, None, P, None, None, None, None, 0, None) == EINVAL
    assert backward(act=7) == EINVAL and backward(go=None) == EINVAL and backward(codes=P) == EINVAL
    assert backward(act=2, slope=None) == EINVAL  # neither the slopes nor what to compute them from
    assert backward(ws=None) == EINVAL and backward(floats=0) == EWORKSPACE
    assert backward(dx=None) == 0


@pytest.mark.parametrize("shape", [(0, 4096, 16), (4, 4096, 0), (0, 4096, 4096), (4, 0, 4096), (4096, 0, 16), (4, 16, 0),
                                   (0, 16, 4096), (0, 0, 0), (4096, 4096, 0), (0, 1 << 20, 1 << 10)])
def test_workspaces_of_empty_layers(shape):
    """No product, so nothing for one: dz (batch x fan_out) at most."""
    s = LinearShape(*shape)
    assert hip.ts_hip_linear_workspace_floats(ctypes.byref(s)) == 0
    dz = -(-shape[0] * shape[2] // 64) * 64
    parts = -(-shape[0] // 512) * shape[2] if shape[0] > 1024 else 0
    assert hip.ts_hip_linear_backward_workspace_floats(ctypes.byref(s)) == dz + -(-parts // 64) * 64
    if shape[0] == 0:
        assert linear(shape=shape, floats=0) == 0 and backward(shape=shape, dx=None, floats=0) == 0
    assert linear(shape=(shape[0], shape[1], 0), floats=0) == 0


def test_packed_layer_refuses():
    def call(batch=4, k=8, n=16, act=0, y=P, xc=P, ws=P):
        return hip.ts_hip_linear_packed(xc, P, ws, P, batch, k, n, None, act, None, y, None, 1 << 40, None)

    assert call(act=9) == EINVAL and call(y=None) == EINVAL and call(xc=None) == EINVAL and call(ws=None) == EINVAL
    assert call(batch=1 << 24) == EINVAL and call(batch=0) == 0


def test_norm_entries_refuse():
    f = hip.ts_hip_rms_norm
    assert f(None, None, P, 4, 8, 1e-6, None, P, None) == EINVAL
    assert f(P, None, None, 4, 8, 1e-6, None, P, None) == EINVAL
    assert f(P, None, P, 4, 8, 1e-6, None, None, None) == EINVAL
    assert f(P, P, P, 4, 8, 1e-6, None, P, None) == EINVAL  # a residual without h
    assert f(P, None, P, 4, 8, 1e-6, P, P, None) == EINVAL  # h without a residual
    assert f(None, None, None, 0, 8, 1e-6, None, None, None) == 0
    assert hip.ts_hip_rms_norm_packed(P, None, P, 4, 8, 1e-6, None, P, None, None) == EINVAL
    b = hip.ts_hip_rms_norm_backward
    assert b(P, P, None, 4, 8, 1e-6, P, None, None, 0, None, None) == EINVAL
    assert b(P, P, P, 4, 8, 1e-6, None, P, None, 0, None, None) == EWORKSPACE
    assert b(P, P, P, 4, 8, 1e-6, None, None, None, 0, None, None) == 0
    assert hip.ts_hip_pack8(None, 4, 8, P, P, None) == EINVAL and hip.ts_hip_pack8(P, 4, 8, P, None, None) == EINVAL
    assert hip.ts_hip_unpack8(P, P, 4, 8, None, None) == EINVAL


class Array:
    def __init__(self, **kw):
        self.__cuda_array_interface__ = dict(dict(shape=(2, 3), typestr="<f4", data=(P, False), version=3), **kw)


def test_device_arrays_are_checked():
    for bad, what in ((np.zeros(3, np.float32), "no device memory"), (Array(typestr="<f2"), "type <f2"),
                      (Array(strides=(16, 4)), "not contiguous"), (Array(strides=(4, 8)), "not contiguous")):
        with pytest.raises(T.TsError, match=what):
            T.Tensor.from_device(bad)
    codes, scales = Array(typestr="|u1", shape=(2, 128)), Array(typestr="|u1", shape=(1, 2, 4))
    for c, s, cols in ((codes, scales, 129), (codes, scales, -1), (codes, Array(typestr="|u1", shape=(2, 1, 4)), 100),
                       (Array(typestr="|u1", shape=(128,)), scales, 100), (Array(), scales, 100)):
        with pytest.raises(T.TsError):
            T.Packed8.from_device(c, s, cols)


@pytest.mark.parametrize("shape", [(1 << 62,), (1 << 32, 1 << 32), (1 << 31, 1 << 31, 4), (3, (1 << 62) + 1), (1 << 64,), (-1,),
                                   (1 << 40, 1 << 40, 1 << 40)])
def test_shapes_whose_size_wraps_are_refused(shape):
    with pytest.raises(T.TsError, match="larger than any memory|no shape"):
        T.Tensor.from_device(Array(shape=shape))
    dims = (ctypes.c_size_t * len(shape))(*shape)
    if all(0 <= d < 1 << 64 for d in shape):
        released = []
        release = ctypes.CFUNCTYPE(None, ctypes.c_void_p)(released.append)
        assert not gradtrack.ts_tensor_from_device(P, dims, len(shape), release, 7) and released == [7]


def test_an_array_that_will_not_be_shared_is_an_error_of_the_library():
    class Kept:  # as torch's tensors that require grad
        @property
        def __cuda_array_interface__(self):
            raise RuntimeError("use detach()")

    with pytest.raises(T.TsError, match=r"exposes no device memory: use detach\(\)"):
        T.Tensor.from_device(Kept())


def test_arrays_that_may_not_be_written_are_refused():
    with pytest.raises(T.TsError, match="read-only"):
        T.Tensor.from_device(Array(shape=(0, 3), data=(P, True)))
    with pytest.raises(T.TsError, match="masked"):
        T.Tensor.from_device(Array(shape=(0, 3), mask=object()))
    # codes and scales are read only
    codes, scales = Array(typestr="|u1", shape=(0, 128), data=(P, True)), Array(typestr="|u1", shape=(1, 0, 4), data=(P, True))
    assert T.Packed8.from_device(codes, scales, 100).shape == (0, 100)


def test_memory_is_given_back_once_whatever_allocation_fails(tmp_path):
    lib, here = ROOT / "train-station_amd", ROOT / "tests" / "release_calls.cpp"
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{ROOT / 'include'}", "-o", tmp_path / "p", here, f"-L{lib}", "-lts_gradtrack",
                    "-lts_hip", f"-Wl,-rpath,{lib}", "-Wl,-rpath,/opt/rocm/lib"], check=True)
    got = subprocess.run([tmp_path / "p"], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr


def test_empty_shapes_of_long_sides_are_empty():
    t = T.Tensor.from_device(Array(shape=(1 << 62, 0, 1 << 62), data=(0, False)))
    assert t.size() == 0


@pytest.mark.parametrize("rows,cols", [(1 << 57, 128), (1 << 56, 256), (1, (1 << 64) - 1), (1, (1 << 64) - 127), (3, 1 << 63),
                                       ((1 << 57) + 1, 128)])
def test_packed_sizes_that_wrap_are_refused(rows, cols):
    assert not gradtrack.ts_packed8_from_device(P, P, rows, cols, None, None)
    assert "larger than any memory" in last_error()


def test_names_are_checked():
    t = object.__new__(T.Tensor)
    t._h = None
    with pytest.raises(T.TsError, match="unknown activation 'gelu'"):
        t.linear(t, activation="gelu")
    with pytest.raises(T.TsError, match="unknown checkpoint '4bit'"):
        t.linear(t, checkpoint="4bit")
