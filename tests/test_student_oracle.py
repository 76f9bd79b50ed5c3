"""A student's operators without a device: the plain forms the device is compared with
against differences and torch, and what the entries refuse."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import student_ref as R
import train_station_amd as T
from conftest import normal
from train_station_amd._ffi import gradtrack, hip, last_error

EINVAL, EWORKSPACE = 100001, 100003
P = 1 << 20  # an address that is never read: every call here ends on the host
INF = np.inf


def test_block8_is_torch_s_rounding():
    x = normal((130, 300), 1) * np.float32(30)
    for tiles in (False, True):
        codes, scales = R.block8(x, tiles)
        q = np.zeros((130, 384))
        q[:, :300] = x
        by = scales.T[np.arange(130) // (128 if tiles else 1)].repeat(128, 1)
        want = torch.from_numpy((q / by).astype(np.float32)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        assert np.mean(codes != want) < 1e-4  # (the quotients' own rounding at a border)
        # half a step of the largest binade, 16, is the most a value of its size is off
        assert np.max(np.abs(R.unblock8(codes, scales, 300, tiles) - x) / by[:, :300]) <= 16.01


@pytest.mark.parametrize("bias", [False, True])
def test_layer_norm_is_torch_s_and_its_gradients_differences(bias):
    h, w = normal((4, 9), 1).astype(np.float64) + 3, normal((9,), 2).astype(np.float64)
    b = normal((9,), 3).astype(np.float64) if bias else None
    go = normal((4, 9), 4).astype(np.float64)
    want = torch.nn.functional.layer_norm(torch.from_numpy(h), (9,), torch.from_numpy(w),
                                          None if b is None else torch.from_numpy(b), 1e-5).numpy()
    assert np.allclose(R.layer_norm(h, w, b, 1e-5), want, rtol=1e-12, atol=1e-13)
    dh, dw, db = R.layer_norm_grads(h, w, go, 1e-5)
    step = 1e-6
    f = lambda h, w, c: (go * (R.layer_norm(h, w, None, 1e-5) + c)).sum()  # noqa: E731
    for i in np.ndindex(4, 9):
        e = np.zeros_like(h)
        e[i] = step
        assert abs((f(h + e, w, 0) - f(h - e, w, 0)) / (2 * step) - dh[i]) < 1e-7
    for j in range(9):
        e = np.zeros(9)
        e[j] = step
        assert abs((f(h, w + e, 0) - f(h, w - e, 0)) / (2 * step) - dw[j]) < 1e-7
        assert abs((f(h, w, e) - f(h, w, -e)) / (2 * step) - db[j]) < 1e-7


def distillation_case(rows, vocab, kept, seed=0):
    rng = np.random.default_rng(seed)
    z = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    idx = rng.integers(-1, vocab, (rows, kept)).astype(np.int32)
    teacher = (rng.standard_normal((rows, kept)) * 2).astype(np.float32)
    labels = rng.integers(-1, vocab, rows).astype(np.int32)
    return z, idx, teacher, labels, rng.random(rows).astype(np.float32)


@pytest.mark.parametrize("t,hard", [(1.0, 0.0), (2.0, 0.3), (1.0, 1.0), (0.5, 0.5)])
def test_distillation_s_gradient_is_its_differences(t, hard):
    z, idx, teacher, labels, w = distillation_case(4, 6, 5)
    idx[1], idx[2, 1] = -1, idx[2, 0]  # a row of none, an index twice
    idx[3], labels[3] = -1, -1
    z = z.astype(np.float64)
    loss, dz, _, _ = R.distillation(z, idx, teacher, t, labels, hard, w)
    step = 1e-6
    for i in np.ndindex(*z.shape):
        e = np.zeros_like(z)
        e[i] = step
        up, down = (R.distillation(z + s * e, idx, teacher, t, labels, hard, w)[0] for s in (1, -1))
        assert abs((up - down) / (2 * step) - dz[i]) < 1e-7
    assert not dz[3].any()


def test_distillation_against_torch():
    z, idx, teacher, labels, _ = distillation_case(5, 40, 4)
    idx = np.abs(idx)
    Z = torch.from_numpy(z).double().requires_grad_(True)
    q = torch.softmax(torch.from_numpy(teacher).double() / 2, 1)
    logp = torch.log_softmax(Z / 2, 1).gather(1, torch.from_numpy(idx).long())
    kl = (q * (q.log() - logp)).sum(1).mean() * 4
    has = torch.from_numpy(labels >= 0)
    ce = torch.nn.functional.cross_entropy(Z, torch.from_numpy(labels).long(), ignore_index=-1, reduction="sum") / 5
    assert has.any()
    (0.7 * kl + 0.3 * ce).backward()
    loss, dz, _, _ = R.distillation(z, idx, teacher, 2.0, labels, 0.3)
    assert abs(loss - (0.7 * kl + 0.3 * ce).item()) < 1e-6 and np.allclose(dz, Z.grad.numpy(), atol=1e-7)


# ---- refusals ---------------------------------------------------------------------------


def test_layer_norm_entries_refuse():
    f = hip.ts_hip_layer_norm
    assert f(None, None, P, P, 4, 8, 1e-5, None, P, None) == EINVAL
    assert f(P, None, None, P, 4, 8, 1e-5, None, P, None) == EINVAL
    assert f(P, None, P, P, 4, 8, 1e-5, None, None, None) == EINVAL
    assert f(P, P, P, P, 4, 8, 1e-5, None, P, None) == EINVAL  # a residual without h
    assert f(P, None, P, P, 4, 8, 1e-5, P, P, None) == EINVAL  # h without a residual
    assert f(P, None, P, P, 1 << 31, 8, 1e-5, None, P, None) == EINVAL
    assert f(None, None, None, None, 0, 8, 1e-5, None, None, None) == 0
    g = hip.ts_hip_layer_norm_block8
    assert g(P, None, P, P, 4, 8, 1e-5, None, P, None, None) == EINVAL
    assert g(P, None, P, P, 4, 8, 1e-5, None, None, P, None) == EINVAL
    b = hip.ts_hip_layer_norm_backward
    assert b(P, P, None, 4, 8, 1e-5, P, None, None, None, 0, None, None) == EINVAL
    assert b(P, P, P, 4, 8, 1e-5, None, P, None, None, 0, None, None) == EWORKSPACE
    assert b(P, P, P, 4, 8, 1e-5, None, None, P, P, 1, None, None) == EWORKSPACE
    assert b(P, P, P, 4, 8, 1e-5, None, None, None, None, 0, None, None) == 0


def test_block8_entries_refuse():
    assert hip.ts_hip_block8(None, 4, 8, 0, P, P, None) == EINVAL and hip.ts_hip_block8(P, 4, 8, 0, P, None, None) == EINVAL
    assert hip.ts_hip_unblock8(P, P, 4, 8, 0, None, None) == EINVAL
    assert [hip.ts_hip_block8_scale_rows(n, 1) for n in (0, 1, 128, 129)] == [0, 1, 1, 2]
    assert hip.ts_hip_block8_scale_rows(129, 0) == 129

    def call(batch=4, k=8, n=16, act=0, y=P, xc=P, xs=P, wc=P, ws=P):
        return hip.ts_hip_linear_block8(xc, xs, wc, ws, batch, k, n, None, act, None, y, None)

    assert call(act=9) == EINVAL and call(y=None) == EINVAL and call(xc=None) == EINVAL and call(ws=None) == EINVAL
    assert call(xs=None) == EINVAL and call(wc=None) == EINVAL
    assert call(batch=1 << 24) == EINVAL and call(batch=0) == 0 and call(n=0) == 0


def test_distillation_entry_refuses():
    def call(rows=4, vocab=8, kept=2, t=1.0, hard=0.5, z=P, idx=P, teacher=P, labels=P, loss=P, bad=P, work=P, floats=1 << 40):
        return hip.ts_hip_distillation(z, rows, vocab, idx, teacher, kept, t, labels, hard, None, None, loss, P, bad, work, floats,
                                       None, None)

    for bad in (dict(t=0.0), dict(t=-1.0), dict(t=np.nan), dict(t=INF), dict(t=1e-30), dict(hard=-0.1), dict(hard=1.1),
                dict(hard=np.nan), dict(kept=1025), dict(labels=None), dict(z=None), dict(idx=None), dict(teacher=None),
                dict(loss=None), dict(bad=None), dict(vocab=(1 << 28) + 1), dict(rows=1 << 31)):
        assert call(**bad) == EINVAL, bad
    assert call(work=None) == EWORKSPACE and call(floats=1) == EWORKSPACE


class Array:
    def __init__(self, **kw):
        self.__cuda_array_interface__ = dict(dict(shape=(2, 3), typestr="<f4", data=(P, False), version=3), **kw)


def test_device_arrays_are_checked():
    codes, scales = Array(typestr="|u1", shape=(2, 128)), Array(shape=(1, 2))
    for c, s, cols, tiles in ((codes, scales, 129, False), (codes, scales, -1, False), (codes, scales, 100, True),
                              (codes, Array(shape=(2, 1)), 100, False), (Array(typestr="|u1", shape=(128,)), scales, 100, False),
                              (Array(typestr="|u1", shape=()), scales, 100, True), (codes, Array(typestr="|u1", shape=(1, 2)), 100, False),
                              (Array(shape=(2, 128)), scales, 100, False)):
        with pytest.raises(T.TsError):
            T.Block8.from_device(c, s, cols, tiles)
    with pytest.raises(T.TsError, match="type <f4"):
        T.Indices.from_device(Array())
    with pytest.raises(T.TsError, match="not contiguous"):
        T.Indices.from_device(Array(typestr="<i4", strides=(4, 8)))
    empty = T.Block8.from_device(Array(typestr="|u1", shape=(0, 128), data=(P, True)), Array(shape=(1, 0), data=(P, True)), 100)
    assert empty.shape == (0, 100) and not empty.tiles and empty.pitch == 128


def test_indices_are_whole_numbers_of_32_bits():
    for bad in ([1.5], [1 << 31], [-(1 << 31) - 1], np.array([2 ** 40], np.uint64)):
        with pytest.raises(T.TsError, match="Indices"):
            T.Indices.from_slice(bad, (1,))
    with pytest.raises(T.TsError, match="doesn't match shape"):
        T.Indices.from_slice([1, 2], (3,))
    assert T.Indices.from_slice([], (0, 5)).shape == (0, 5)


@pytest.mark.parametrize("rows,cols", [(1 << 57, 128), (1, (1 << 64) - 1), (1, (1 << 64) - 127), (3, 1 << 63)])
@pytest.mark.parametrize("tiles", [0, 1])
def test_block8_sizes_that_wrap_are_refused(rows, cols, tiles):
    assert not gradtrack.ts_block8_from_device(P, P, rows, cols, tiles, None, None)
    assert "larger than any memory" in last_error()


@pytest.mark.parametrize("shape", [(1 << 63,), (1 << 32, 1 << 32), (3, (1 << 62) + 1), (1 << 40, 1 << 40, 1 << 40)])
def test_indices_sizes_that_wrap_are_refused(shape):
    dims = (ctypes.c_size_t * len(shape))(*shape)
    released = []
    release = ctypes.CFUNCTYPE(None, ctypes.c_void_p)(released.append)
    assert not gradtrack.ts_indices_from_device(P, dims, len(shape), release, 7) and released == [7]
    assert "larger than any memory" in last_error()


def test_null_handles_are_errors():
    for call in (lambda: gradtrack.ts_tensor_layer_norm(None, None, None, 1e-5), lambda: gradtrack.ts_tensor_block8(None, 0),
                 lambda: gradtrack.ts_block8_unpack(None), lambda: gradtrack.ts_block8_linear(None, None, None, 0, None),
                 lambda: gradtrack.ts_tensor_distillation(None, None, None, 1.0, None, 0.0, None),
                 lambda: gradtrack.ts_indices_device_ptr(None)):
        assert not call() and "NULL" in last_error()


# ---- logic of handles without a device: empty tensors have no memory -------------------------


def empty(*shape):
    return T.Tensor.from_device(Array(shape=shape, data=(0, False)))


def indices(*shape):
    return T.Indices.from_slice([], shape)


def test_arguments_of_the_handles_are_checked():
    x, w = empty(0, 8), empty(0)
    for call, what in ((lambda: x.layer_norm(w), r"weight \[0\] for rows of 8"),
                       (lambda: empty(0, 0).layer_norm(w, empty(0, 1)), r"bias \[0, 1\] for rows of 0"),
                       (lambda: empty(0, 0).add_layer_norm(x, w), r"residual \[0, 8\] added to \[0, 0\]"),
                       (lambda: empty(0, 0).layer_norm(w, eps=-1.0), "eps must not be negative"),
                       (lambda: empty(0, 0).layer_norm(w, eps=float("nan")), "eps must not be negative"),
                       (lambda: empty(2, 0, 0).layer_norm_block8(w), "requires a matrix"),
                       (lambda: empty(0).block8(), "requires a matrix")):
        with pytest.raises(T.TsError, match=what):
            call()
    z, i, t = empty(0, 9), indices(0, 4), empty(0, 4)
    for call, what in ((lambda: empty(0).distillation(i, t), "requires a matrix"),
                       (lambda: empty(2, 0).distillation(indices(2, 0), empty(2, 0)), "no columns"),
                       (lambda: z.distillation(indices(0), t), "indices"), (lambda: z.distillation(i, empty(0, 5)), "teacher"),
                       (lambda: z.distillation(indices(0, 1025), empty(0, 1025)), "at most 1024"),
                       (lambda: z.distillation(i, t, 0.0), "temperature"), (lambda: z.distillation(i, t, float("nan")), "temperature"),
                       (lambda: z.distillation(i, t, -1.0), "temperature"), (lambda: z.distillation(i, t, INF), "temperature"),
                       (lambda: z.distillation(i, t, hard=0.5), "no labels"), (lambda: z.distillation(i, t, hard=1.5), "share"),
                       (lambda: z.distillation(i, t, hard=float("nan")), "share"),
                       (lambda: z.distillation(i, t, labels=indices(0, 1), hard=0.5), "labels"),
                       (lambda: z.distillation(i, t, weights=empty(0, 1)), "weights")):
        with pytest.raises(T.TsError, match=what):
            call()
    rows = T.Block8.from_device(Array(typestr="|u1", shape=(0, 128)), Array(shape=(1, 0)), 100)
    tiles = T.Block8.from_device(Array(typestr="|u1", shape=(0, 128)), Array(shape=(1, 0)), 100, tiles=True)
    with pytest.raises(T.TsError, match="a scale per row"):
        rows.linear(rows)
    with pytest.raises(T.TsError, match="a scale per row"):
        tiles.linear(tiles)
    with pytest.raises(T.TsError, match="Inner dimensions"):
        rows.linear(T.Block8.from_device(Array(typestr="|u1", shape=(0, 128)), Array(shape=(1, 0)), 99, tiles=True))
    with pytest.raises(T.TsError, match="unknown activation 'gelu'"):
        rows.linear(tiles, activation="gelu")
