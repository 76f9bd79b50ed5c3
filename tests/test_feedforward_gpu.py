"""A feed-forward block's operators on the device against their plain forms in
64 bits (feedforward_ref.py, which derives the tolerances)."""
from __future__ import annotations

import numpy as np
import pytest

import feedforward_ref as R
from conftest import normal
from gpu_util import Dev, T, hip, hip_check, sync

pytestmark = pytest.mark.gpu


class DeviceArray:
    """A device buffer as other libraries expose theirs."""

    def __init__(self, a, offset=0):
        self.host = np.ascontiguousarray(a)
        words = np.zeros(max((self.host.nbytes + 3) // 4, 1), np.float32)
        words.view(np.uint8)[: self.host.nbytes] = self.host.reshape(-1).view(np.uint8)
        self.dev = Dev.of(words, offset)
        kind = "<f4" if self.host.dtype == np.float32 else "|u1"
        self.__cuda_array_interface__ = dict(shape=self.host.shape, typestr=kind, data=(self.dev.ptr, False), version=2)

    def get(self):
        return self.dev.get().view(np.uint8)[: self.host.nbytes].view(self.host.dtype).reshape(self.host.shape)


def tensor(a):
    return T.Tensor.from_slice(np.ascontiguousarray(a, np.float32), a.shape)


def packed(a):
    """A Packed8 of the plain form's codes."""
    codes, scales = R.pack8(a)
    return T.Packed8.from_device(DeviceArray(codes), DeviceArray(scales), a.shape[1])


def parts(p):
    """codes and scales of a Packed8, on the host."""
    T.synchronize()
    rows, pitch = p.shape[0], p.pitch
    codes, scales = np.empty((rows, pitch), np.uint8), np.empty((pitch // 128, rows, 4), np.uint8)
    hip_check(hip.ts_hip_memcpy_bytes(codes.ctypes.data, p.codes_ptr(), codes.nbytes, 1, None), "codes")
    hip_check(hip.ts_hip_memcpy_bytes(scales.ctypes.data, p.scales_ptr(), scales.nbytes, 1, None), "scales")
    sync()
    return codes, scales


def assert_within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want) / bound
    assert np.all(off <= 1), f"{what}: {np.nanmax(off):.3g} of its bound at {np.unravel_index(np.nanargmax(off), off.shape)}"


# ---- values in 8 bits ---------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 127), (4, 128), (3, 129), (70, 1003), (1, 5000)])
def test_pack8(rows, cols):
    rng = np.random.default_rng(rows * cols)
    x = (rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-38, 37, (rows, 1))).astype(np.float32)
    x[rng.random((rows, cols)) < 0.1] = 0.0
    p = tensor(x).pack8()
    assert p.shape == (rows, cols) and p.pitch == R.pitch_of(cols)
    codes, scales = parts(p)
    want = R.pack8(x)
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])
    assert np.array_equal(p.unpack().data(), R.unpack8(*want, cols).astype(np.float32))


def test_pack8_borders():
    """Every code, every border between two, their neighbours, at the smallest, middle and largest scales."""
    v = R.e4m3_values()[:127]
    mid = (v[1:] + v[:-1]) / 2
    base = np.r_[v, mid, -v, -mid].astype(np.float32)
    line = np.r_[base, np.nextafter(base, np.float32(np.inf)), np.nextafter(base, np.float32(-np.inf))]
    line = np.clip(line, -448, 448)
    line = np.resize(line, -(-line.size // 31) * 31).reshape(-1, 31)
    blocks = np.concatenate([line, np.full((line.shape[0], 1), 448.0)], 1).reshape(1, -1)
    x = np.concatenate([blocks * 2.0 ** k for k in (-117, -60, 0, 60, 119)]).astype(np.float32)
    codes, scales = parts(tensor(x).pack8())
    want = R.pack8(x)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


def test_pack8_what_no_code_holds():
    x = np.zeros((4, 64), np.float32)
    x[0, :3] = [np.inf, -np.inf, 1.0]
    x[1, :3] = [np.nan, 2.0, -np.nan]
    x[2, :2] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    x[3, :3] = [1e-45, 2.0 ** -127, 2.0 ** -126]
    codes, scales = parts(tensor(x).pack8())
    want = R.pack8(x)
    assert np.array_equal(scales, want[1])
    nan = (want[0] & 127) == 127  # either of the two NaN codes
    assert nan.sum() == 2 and np.all((codes[nan] & 127) == 127) and np.array_equal(codes[~nan], want[0][~nan])
    assert scales[0, 0, 0] == 246 and codes[0, 0] == 0x7e and codes[0, 1] == 0xfe


# ---- norm -----------------------------------------------------------------------------

NORMS = [(1, 1), (1, 4096), (3, 7), (5, 256), (6, 257), (9, 512), (4, 1003), (130, 784), (7, 1025), (3, 2048), (2, 4095),
         (5, 4097), (2, 8192), (3, 8193), (2, 16384), (3, 16385), (2, 40001), (700, 64)]


def norm_case(rows, cols, residual, eps=1e-6):
    x, r = normal((rows, cols), 1), normal((rows, cols), 2) * 3 if residual else None
    w = (1 + 0.2 * normal((cols,), 3)).astype(np.float32)
    h = x if r is None else (x + r).astype(np.float32)
    return x, r, w, h


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(rows, cols, residual):
    x, r, w, h = norm_case(rows, cols, residual)
    go = normal((rows, cols), 4)
    X, W = tensor(x).with_requires_grad(), tensor(w).with_requires_grad()
    Rs = tensor(r).with_requires_grad() if residual else None
    if residual:
        y, stream = X.add_rms_norm(Rs, W, 1e-6)
        assert np.array_equal(stream.data(), h)
    else:
        y = X.rms_norm(W, 1e-6)
    want = R.rms_norm(h, w, 1e-6)
    assert_within(y.data(), want, 4 * R.U * np.abs(want) + 1e-40, "y")
    y.backward(tensor(go))
    dh, dw = R.rms_norm_grads(h, w, go, 1e-6)
    s = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(1, keepdims=True) + 1e-6)
    g = np.abs(go.astype(np.float64) * w)
    back = np.abs(h) * s ** 3 * np.abs((go.astype(np.float64) * w * h).mean(1, keepdims=True))
    assert_within(X.grad_by_value().data(), dh, 4 * R.U * (s * g + back) + 1e-40, "dx")
    if residual:
        assert np.array_equal(Rs.grad_by_value().data(), X.grad_by_value().data())
    # a rounding each of r and h r, one of each part (the long rows': one a row) and one at the end
    steps = 5 + (rows if cols > 16384 else 0)
    assert_within(W.grad_by_value().data(), dw, steps * R.U * np.abs(go * h * s).sum(0) + 1e-40, "dweight")
    T.clear_gradients()


@pytest.mark.parametrize("rows,cols", [(600, 8192), (600, 8200), (300, 16383), (1100, 4100), (1500, 1030)])
def test_rms_norm_sums_many_rows(rows, cols):
    """Weight gradients where each workgroup adds several rows, within the bounds of one."""
    test_rms_norm(rows, cols, True)


@pytest.mark.parametrize("rows,cols", [(1, 16385), (3, 40001), (300, 16390), (700, 20003)])
@pytest.mark.parametrize("need", ["both", "weight", "x"])
def test_long_rows_weight_gradients_are_summed_in_64_bits(rows, cols, need):
    x, _, w, h = norm_case(rows, cols, False)
    go = np.abs(normal((rows, cols), 4)) * np.sign(x)  # every term of a sum of one sign
    X, W = tensor(x), tensor(w)
    for t in (X, W) if need == "both" else (W,) if need == "weight" else (X,):
        t.with_requires_grad()
    X.rms_norm(W, 1e-6).backward(tensor(go))
    dh, dw = R.rms_norm_grads(h, w, go, 1e-6)
    s = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(1, keepdims=True) + 1e-6)
    if need != "x":
        assert_within(W.grad_by_value().data(), dw, 5 * R.U * np.abs(go * h * s).sum(0) + 1e-40, "dweight")
    if need != "weight":
        g = np.abs(go.astype(np.float64) * w)
        back = np.abs(h) * s ** 3 * np.abs((go.astype(np.float64) * w * h).mean(1, keepdims=True))
        assert_within(X.grad_by_value().data(), dh, 4 * R.U * (s * g + back) + 1e-40, "dx")
    T.clear_gradients()


def test_long_rows_weight_gradients_keep_what_fp32_sums_lose():
    rows, cols = 40 * 256 + 1, 16388
    go = np.zeros((rows, cols), np.float32)
    go[::256] = 0.9 * 2.0 ** -25  # of rows that one workgroup of 256 takes in turn; beside 1, nothing in fp32
    go[0] = 1.0
    W = tensor(np.ones(cols, np.float32)).with_requires_grad()
    T.Tensor.ones((rows, cols)).rms_norm(W, 0.0).backward(tensor(go))
    want = go[::256].astype(np.float64).sum(0)
    assert_within(W.grad_by_value().data(), want, 5 * R.U * want, "dweight")
    T.clear_gradients()


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_packed(rows, cols, residual):
    x, r, w, h = norm_case(rows, cols, residual)
    if residual:
        p, stream = tensor(x).add_rms_norm_packed(tensor(r), tensor(w), 1e-6)
        assert np.array_equal(stream.data(), h)
    else:
        p = tensor(x).rms_norm_packed(tensor(w), 1e-6)
    codes, scales = parts(p)
    want = R.pack8(R.rms_norm(h, w, 1e-6))
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


def test_norm_of_more_rows_than_a_launch_has_workgroups():
    rows, cols = (1 << 23) + 5, 3
    x, w = normal((rows, cols), 1), normal((cols,), 2)
    X = tensor(x)
    y = X.rms_norm(tensor(w)).data()
    want = R.rms_norm(x, w, 1e-6)
    assert_within(y, want, 4 * R.U * np.abs(want) + 1e-40, "y")
    del X


def test_packed_norm_of_zero_rows_pads_with_zeros():
    x = normal((3, 40), 1)
    x[1] = 0.0
    codes, scales = parts(tensor(x).rms_norm_packed(tensor(np.ones(40, np.float32)), 0.0))
    assert np.all((codes[1, :40] & 127) == 127)  # 0 / 0
    assert not codes[:, 40:].any()


@pytest.mark.parametrize("rows,cols", [(1, 5), (128, 784), (700, 64), (3000, 1000)])
def test_norm_backward_with_and_without_a_ticket(rows, cols):
    """The same sums by one launch and by two, to the last place, and the ticket zero again."""
    h, go = Dev.of(normal((rows, cols), 1)), Dev.of(normal((rows, cols), 2))
    w, ticket = Dev.of(normal((cols,), 3)), Dev.of(np.zeros(1, np.float32))
    floats = hip.ts_hip_rms_norm_backward_workspace_floats(rows, cols)
    work, got = Dev(floats), []
    for t in (None, ticket.ptr, ticket.ptr):
        dh, dw = Dev(rows * cols), Dev(cols)
        hip_check(hip.ts_hip_rms_norm_backward(h.ptr, w.ptr, go.ptr, rows, cols, 1e-6, dh.ptr, dw.ptr, work.ptr, floats, t,
                                               None))
        got.append((dh.get(), dw.get()))
    assert not ticket.get().view(np.uint32).any()
    for dh, dw in got[1:]:
        assert np.array_equal(dh, got[0][0]) and np.allclose(dw, got[0][1], rtol=2e-7, atol=0)


def test_norm_of_zero_and_tiny_and_huge_rows():
    x = np.zeros((4, 40), np.float32)
    x[1], x[2], x[3, 5] = 1e-30, 1e30, np.nan
    w = np.ones(40, np.float32)
    y = tensor(x).rms_norm(tensor(w), 1e-6).data()
    assert not y[0].any() and np.isnan(y[3]).all()
    assert_within(y[1:3], R.rms_norm(x[1:3].astype(np.float64), w, 1e-6), np.abs(y[1:3]) * 4 * R.U + 1e-44, "y")
    z = tensor(x[:1]).rms_norm(tensor(w), 0.0).data()  # 0 / 0
    assert np.isnan(z).all()


# rows whose r, r^3 or sums leave fp32's range while their norm and its gradients stay inside
FAR_ROWS = [1e-42, 1e-38, 1e-30, 1e-20, 1e-12, 1.0, 1e12, 1e18, 1e20, 1e22, 1e30, 3e37]
FAR_COLS = [1, 40, 300, 1000, 1500, 4000, 8000, 16384, 20000]


def far_case(cols):
    """A row of each size and a constant one beside it, small rows' gradients small enough for theirs."""
    size = np.repeat(np.asarray(FAR_ROWS), 2)[:, None]
    h = normal((size.size, cols), 1).astype(np.float64)
    h[1::2] = 1.0
    go = normal((size.size, cols), 2) * np.sqrt(np.minimum(size, 1.0))
    w = (1 + 0.2 * normal((cols,), 3)).astype(np.float32)
    return (np.clip(h, -6, 6) * size).astype(np.float32), w, go.astype(np.float32)


@pytest.mark.parametrize("cols", FAR_COLS)
def test_norm_of_tiny_and_huge_rows_without_eps(cols):
    h, w, _ = far_case(cols)
    h = np.r_[h, np.full((1, cols), 3.3e38, np.float32), np.full((1, cols), 1e-45, np.float32)]
    want = R.rms_norm(h, w, 0.0)
    assert_within(tensor(h).rms_norm(tensor(w), 0.0).data(), want, 4 * R.U * np.abs(want) + 1e-40, "y")
    codes, scales = parts(tensor(h).rms_norm_packed(tensor(w), 0.0))
    packed_want = R.pack8(want)
    assert np.array_equal(scales, packed_want[1]) and np.array_equal(codes, packed_want[0])


@pytest.mark.parametrize("cols", FAR_COLS)
def test_norm_gradients_of_tiny_and_huge_rows(cols):
    h, w, go = far_case(cols)
    X, W = tensor(h).with_requires_grad(), tensor(w).with_requires_grad()
    X.rms_norm(W, 0.0).backward(tensor(go))
    dh, dw = R.rms_norm_grads(h, w, go, 0.0)
    s = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(1, keepdims=True))
    g = np.abs(go.astype(np.float64) * w)
    back = np.abs(h) * s ** 3 * np.abs((go.astype(np.float64) * w * h).mean(1, keepdims=True))
    assert_within(X.grad_by_value().data(), dh, 4 * R.U * (s * g + back) + 1e-40, "dx")
    steps = 5 + (len(h) if cols > 16384 else 0)
    assert_within(W.grad_by_value().data(), dw, steps * R.U * np.abs(go * h * s).sum(0) + 1e-40, "dweight")
    T.clear_gradients()


def test_norm_gradients_accumulate_and_pass_through_the_sum():
    x, r, w, h = norm_case(6, 96, True)
    X, Rs, W = (tensor(a).with_requires_grad() for a in (x, r, w))
    y, stream = X.add_rms_norm(Rs, W, 1e-6)
    loss = y.mul_tensor(y).add_tensor(stream).sum()
    loss.backward()
    yv = R.rms_norm(h, w, 1e-6)
    dh, dw = R.rms_norm_grads(h, w, 2 * yv, 1e-6)
    assert np.allclose(X.grad_by_value().data(), dh + 1, rtol=1e-5, atol=1e-5)
    assert np.allclose(Rs.grad_by_value().data(), dh + 1, rtol=1e-5, atol=1e-5)
    assert np.allclose(W.grad_by_value().data(), dw, rtol=1e-5, atol=1e-4)
    T.clear_gradients()


def test_norm_of_more_axes_and_of_nothing():
    x, w = normal((2, 3, 5), 1), normal((5,), 2)
    X = tensor(x).with_requires_grad()
    y = X.rms_norm(tensor(w))
    assert y.shape == (2, 3, 5)
    want = R.rms_norm(x.reshape(6, 5), w, 1e-6).reshape(2, 3, 5)
    assert_within(y.data(), want, 4 * R.U * np.abs(want) + 1e-40, "y")
    y.backward(tensor(np.ones((2, 3, 5), np.float32)))
    assert X.grad_by_value().shape == (2, 3, 5)
    E, W = T.Tensor.zeros((0, 5)).with_requires_grad(), tensor(w).with_requires_grad()
    y = E.rms_norm(W)
    assert y.shape == (0, 5)
    y.backward(T.Tensor.zeros((0, 5)))
    assert not W.grad_by_value().data().any()
    T.clear_gradients()


# ---- layers ---------------------------------------------------------------------------

LAYERS = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (16, 32, 128), (33, 65, 31), (64, 784, 10), (128, 129, 130), (2, 1000, 3),
          (257, 40, 300), (1, 513, 65), (300, 17, 33)]


def layer_case(m, k, n, bias, residual, seed=0):
    x, w = normal((m, k), seed + 1), normal((k, n), seed + 2, k ** -0.5)
    b = normal((n,), seed + 3, 0.1) if bias else None
    r = normal((m, n), seed + 4) if residual else None
    return x, w, b, r, normal((m, n), seed + 5, 1 / m)


def check_layer(m, k, n, name, bias, residual, checkpoint, seed=0):
    x, w, b, r, go = layer_case(m, k, n, bias, residual, seed)
    X, W = tensor(x).with_requires_grad(), tensor(w).with_requires_grad()
    B = tensor(b).with_requires_grad() if bias else None
    Rs = tensor(r).with_requires_grad() if residual else None
    y = X.linear(W, bias=B, activation=name, residual=Rs, checkpoint=checkpoint)
    want, z = R.linear(x, w, b, name, r)
    assert_within(y.data(), want, R.linear_bound(x, w, b, name, r, z), "y")
    y.backward(tensor(go))
    kept = x if checkpoint == "full" else R.unpack8(*R.pack8(x), k)
    z = R.linear(kept, w, b, "none", None)[0]
    dx, dw, db = R.linear_grads(kept, w, z, name, go)
    ex, ew, eb = R.linear_grads_bound(kept, w, b, z, name, go)
    if name == "relu":  # an input within rounding of zero takes either slope: its whole gradient
        turn = np.abs(go) * ~R.relu_safe(x, w, b, kept)
        ex, ew, eb = ex + turn @ np.abs(w).T, ew + np.abs(kept).T @ turn, eb + turn.sum(0)
    assert_within(X.grad_by_value().data(), dx, ex, "dx")
    assert_within(W.grad_by_value().data(), dw, ew, "dweight")
    if bias:
        assert_within(B.grad_by_value().data(), db, eb, "dbias")
    if residual:
        assert np.array_equal(Rs.grad_by_value().data(), go)
    T.clear_gradients()


@pytest.mark.parametrize("m,k,n", LAYERS)
@pytest.mark.parametrize("checkpoint", ["full", "8bit"])
@pytest.mark.parametrize("name,bias,residual", [("none", False, False), ("relu", True, False), ("silu", True, True),
                                                ("gelu_tanh", False, True)])
def test_linear(m, k, n, name, bias, residual, checkpoint):
    check_layer(m, k, n, name, bias, residual, checkpoint)


# products large enough for the bf16 cores: every one of the three, some of them, odd sizes, k past a block's end
LARGE = [(1024, 1024, 1024), (1000, 777, 1531), (129, 8000, 1000), (1003, 129, 8191), (5000, 640, 260), (257, 4100, 1025)]


@pytest.mark.parametrize("m,k,n", LARGE)
@pytest.mark.parametrize("name,bias,residual,checkpoint", [("none", False, True, "full"), ("silu", True, False, "8bit"),
                                                           ("gelu_tanh", True, True, "full"), ("relu", True, False, "8bit")])
def test_linear_large(m, k, n, name, bias, residual, checkpoint):
    check_layer(m, k, n, name, bias, residual, checkpoint)


# long sums of few tiles, shared by workgroups: each product in turn, on either kind of instructions
@pytest.mark.parametrize("m,k,n", [(8200, 20, 30), (3, 5003, 40), (40, 33, 4100), (260, 8200, 500), (500, 300, 9000),
                                   (9000, 400, 310)])
@pytest.mark.parametrize("name,bias,residual,checkpoint", [("silu", True, True, "full"), ("gelu_tanh", True, False, "8bit")])
def test_linear_long(m, k, n, name, bias, residual, checkpoint):
    check_layer(m, k, n, name, bias, residual, checkpoint)


# few rows beside a large weight, which is read as it lies: one tile of rows and several, odd sizes of
# everything but the weight's rows, k past a stage's end, k in one part and in eight
STREAMS = [(17, 5003, 6404), (64, 4096, 2052), (65, 2501, 3244), (128, 2000, 2060), (129, 1531, 2604), (512, 1001, 1000),
           (300, 130, 12900), (250, 16001, 132), (200, 2046, 2750)]


@pytest.mark.parametrize("m,k,n", STREAMS)
@pytest.mark.parametrize("name,bias,residual,checkpoint", [("silu", True, True, "full"), ("gelu_tanh", True, False, "8bit"),
                                                           ("none", False, True, "8bit")])
def test_linear_beside_a_large_weight(m, k, n, name, bias, residual, checkpoint):
    check_layer(m, k, n, name, bias, residual, checkpoint)


# weights read as they lie by a row or a few, and large results of few k
@pytest.mark.parametrize("m,k,n", [(1, 4100, 3000), (2, 3001, 4004), (9, 4097, 3004), (31, 2048, 6004), (33, 2500, 2504),
                                   (4000, 1, 3100), (3501, 17, 2003)])
@pytest.mark.parametrize("name,bias,residual,checkpoint", [("silu", True, True, "full"), ("gelu_tanh", True, False, "8bit")])
def test_linear_of_few_rows_or_inputs(m, k, n, name, bias, residual, checkpoint):
    check_layer(m, k, n, name, bias, residual, checkpoint)


def test_linear_of_no_inputs_and_many_rows():
    b, w = normal((3100,), 1), T.Tensor.zeros((0, 3100))
    assert np.array_equal(T.Tensor.zeros((4000, 0)).linear(w, bias=tensor(b)).data(), np.tile(b, (4000, 1)))


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_linear_of_a_weight_at_any_address(offset):
    m, k, n = 100, 2052, 2604
    x, w, b, r, go = layer_case(m, k, n, True, True)
    W = T.Tensor.from_device(DeviceArray(w, offset)).with_requires_grad()
    X = tensor(x).with_requires_grad()
    y = X.linear(W, bias=tensor(b), activation="silu", residual=tensor(r))
    want, z = R.linear(x, w, b, "silu", r)
    assert_within(y.data(), want, R.linear_bound(x, w, b, "silu", r, z), "y")
    y.backward(tensor(go))
    z = R.linear(x, w, b, "none", None)[0]
    dx, dw, _ = R.linear_grads(x, w, z, "silu", go)
    ex, ew, _ = R.linear_grads_bound(x, w, b, z, "silu", go)
    assert_within(X.grad_by_value().data(), dx, ex, "dx")
    assert_within(W.grad_by_value().data(), dw, ew, "dweight")
    T.clear_gradients()


def test_linear_beside_a_large_weight_that_is_not_finite():
    m, k, n = 40, 4100, 4000
    x, w = normal((m, k), 1), normal((k, n), 2)
    w[4099, 7], w[0, 200], x[3, 5] = np.inf, np.nan, -np.inf
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
    got = tensor(x).linear(tensor(w)).data()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    bound = R.product_bound(*(np.where(np.isfinite(a), a, 0) for a in (x, w)))
    assert fine.any() and np.all(np.abs(got[fine] - want[fine]) <= bound[fine])


def test_linear_large_keeps_small_values_beside_large_ones():
    """Pieces are exact whatever else a row holds: magnitudes over sixty binades, and the smallest of fp32."""
    m, k, n = 600, 1100, 1200
    x, w, b, r, go = layer_case(m, k, n, False, False)
    rng = np.random.default_rng(1)
    x = (x * 2.0 ** rng.integers(-30, 31, x.shape)).astype(np.float32)
    w = (w * 2.0 ** rng.integers(-30, 31, w.shape)).astype(np.float32)
    x[5] *= np.float32(2.0 ** -100)
    got = tensor(x).linear(tensor(w)).data()
    want = R.linear(x, w, None, "none", None)[0]
    assert_within(got, want, R.product_bound(x, w) + 1e-37, "y")


def test_linear_large_with_values_that_are_not_finite():
    m, k, n = 900, 1030, 1000
    x, w, b, r, go = layer_case(m, k, n, True, False)
    x[3, 5], x[300, 1], x[301, 2], x[899, 1029] = np.nan, np.inf, -np.inf, 3e38
    w[1029] = np.abs(w[1029]) + 2.0  # a sum past fp32's range
    w[7, 999] = np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64) + b
        limit = np.where(np.abs(want) > np.finfo(np.float32).max, np.sign(want) * np.inf, want)
    got = tensor(x).linear(tensor(w), bias=tensor(b)).data()
    assert np.array_equal(np.isnan(got), np.isnan(limit))
    assert np.array_equal(np.isinf(got), np.isinf(limit)) and np.array_equal(got[np.isinf(got)], limit[np.isinf(limit)])
    fine = np.isfinite(limit)
    bound = R.product_bound(np.nan_to_num(x, posinf=0, neginf=0), np.nan_to_num(w, posinf=0)) + R.U * np.abs(np.nan_to_num(want))
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine])


@pytest.mark.parametrize("checkpoint", ["full", "8bit"])
def test_linear_gradient_is_the_difference(checkpoint):
    """Along a random direction of every input, by the device's own forward values."""
    m, k, n, t = 24, 40, 33, 2.0 ** -7
    x, w, b, r, _ = layer_case(m, k, n, True, True)
    x = R.unpack8(*R.pack8(x), k).astype(np.float32)  # its checkpoint is itself
    go = normal((m, n), 9)
    leaves = [tensor(a).with_requires_grad() for a in (x, w, b, r)]
    X, W, B, Rs = leaves
    X.linear(W, bias=B, activation="gelu_tanh", residual=Rs, checkpoint=checkpoint).backward(tensor(go))
    for at, (a, leaf) in enumerate(zip((x, w, b, r), leaves)):
        d = normal(a.shape, 20 + at)
        ends = []
        for s in (-t, t):
            args = [x, w, b, r]
            args[at] = (a + np.float32(s) * d).astype(np.float32)
            A = [tensor(v) for v in args]
            ends.append(A[0].linear(A[1], bias=A[2], activation="gelu_tanh", residual=A[3]).data().astype(np.float64))
        diff = ((ends[1] - ends[0]) * go).sum() / (2 * t)
        slope = (leaf.grad_by_value().data().astype(np.float64) * d).sum()
        # rounding of the values over the step, and t^2 of a third derivative of order 1 of each output
        scale = np.abs(go).sum()
        assert abs(diff - slope) <= scale * (16 * R.U * 8 / t) + np.abs(go).sum() * t * t * 2 * np.abs(d).max() ** 3, at
    T.clear_gradients()


@pytest.mark.parametrize("batch,fan_in,fan_out", [(1 << 21, 1, 3), (1000003, 2, 17)])
def test_bias_gradients_of_many_rows_are_summed_in_64_bits(batch, fan_in, fan_out):
    go = np.abs(normal((batch, fan_out), 1))
    B = tensor(np.zeros(fan_out, np.float32)).with_requires_grad()
    X, W = T.Tensor.zeros((batch, fan_in)), T.Tensor.zeros((fan_in, fan_out))
    X.linear(W, bias=B).backward(tensor(go))
    want = go.astype(np.float64).sum(0)
    # a rounding of each part, and one of their sum
    assert_within(B.grad_by_value().data(), want, 2.01 * R.U * want, "dbias")
    T.clear_gradients()


@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (33, 65, 31), (9000, 20, 30), (1000, 777, 1531), (64, 4096, 2052), (3, 5003, 40)])
@pytest.mark.parametrize("checkpoint", ["full", "8bit"])
def test_relu_passes_nothing_on_where_it_is_zero(m, k, n, checkpoint):
    """Infinities and NaN of the output's gradient at places that relu holds back, as for Tensor.relu."""
    x, w, b, _, go = layer_case(m, k, n, True, False)
    kept = x if checkpoint == "full" else R.unpack8(*R.pack8(x), k)
    z = R.linear(kept, w, b, "none", None)[0]
    safe = R.relu_safe(x, w, b, kept)
    go = np.where(safe, go, 0).astype(np.float32)
    off = safe & (z < 0)
    sent = go.copy()
    sent[off] = np.resize(np.float32([np.inf, -np.inf, np.nan, 1.0]), off.sum())
    assert not np.isfinite(sent).all()
    X, W, B = (tensor(a).with_requires_grad() for a in (x, w, b))
    X.linear(W, bias=B, activation="relu", checkpoint=checkpoint).backward(tensor(sent))
    dx, dw, db = R.linear_grads(kept, w, z, "relu", go)
    ex, ew, eb = R.linear_grads_bound(kept, w, b, z, "relu", np.where(off, 0, go))
    assert_within(X.grad_by_value().data(), dx, ex, "dx")
    assert_within(W.grad_by_value().data(), dw, ew, "dweight")
    assert_within(B.grad_by_value().data(), db, eb, "dbias")
    T.clear_gradients()


def test_linear_grads_for_some_inputs_only():
    x, w, b, r, go = layer_case(12, 20, 9, True, True)
    for need in range(16):
        ts = [tensor(a) for a in (x, w, b, r)]
        for i, t in enumerate(ts):
            if need >> i & 1:
                t.with_requires_grad()
        y = ts[0].linear(ts[1], bias=ts[2], activation="silu", residual=ts[3], checkpoint="8bit" if need & 2 else "full")
        assert y.requires_grad() == bool(need)
        if need:
            y.backward(tensor(go))
        for i, t in enumerate(ts):
            g = t.grad_by_value()
            assert (g is not None) == bool(need >> i & 1), (need, i)
        T.clear_gradients()
    with T.NoGradTrack():
        assert not tensor(x).with_requires_grad().linear(tensor(w)).requires_grad()


@pytest.mark.parametrize("shape", [(0, 5, 3), (4, 0, 3), (4, 5, 0)])
@pytest.mark.parametrize("checkpoint", ["full", "8bit"])
def test_linear_of_nothing(shape, checkpoint):
    m, k, n = shape
    X, W = T.Tensor.zeros((m, k)).with_requires_grad(), T.Tensor.zeros((k, n)).with_requires_grad()
    b = normal((n,), 1)
    B = tensor(b).with_requires_grad()
    y = X.linear(W, bias=B, activation="silu", checkpoint=checkpoint)
    assert y.shape == (m, n)
    want = np.tile(R.act(b.astype(np.float64), "silu"), (m, 1))
    assert_within(y.data(), want, 20 * R.U * np.abs(want) + 1e-40, "y")
    y.backward(T.Tensor.ones((m, n)))
    assert W.grad_by_value().shape == (k, n) and not W.grad_by_value().data().any()
    want = m * R.act_slope(b.astype(np.float64), "silu")
    assert_within(B.grad_by_value().data(), want, 40 * R.U * np.abs(want) + 1e-40, "dbias")
    if m * k:
        assert not X.grad_by_value().data().any()
    T.clear_gradients()


# sizes past which sums are shared by workgroups and weights are read as they lie, beside a zero
@pytest.mark.parametrize("shape", [(0, 4096, 16), (0, 4096, 4096), (4, 0, 4096), (4, 4096, 0), (2100, 0, 300)])
@pytest.mark.parametrize("checkpoint", ["full", "8bit"])
def test_linear_of_nothing_beside_a_long_side(shape, checkpoint):
    m, k, n = shape
    x, w, b, go = np.zeros((m, k), np.float32), np.zeros((k, n), np.float32), normal((n,), 1), np.ones((m, n), np.float32)
    X, W, B = (tensor(a).with_requires_grad() for a in (x, w, b))
    y = X.linear(W, bias=B, activation="silu", checkpoint=checkpoint)
    want, z = R.linear(x, w, b, "silu", None)
    assert_within(y.data(), want, R.linear_bound(x, w, b, "silu", None, z), "y")
    y.backward(tensor(go))
    dx, dw, db = R.linear_grads(x, w, z, "silu", go)
    eb = R.linear_grads_bound(x, w, b, z, "silu", go)[2]
    assert np.array_equal(X.grad_by_value().data(), dx) and np.array_equal(W.grad_by_value().data(), dw)
    assert_within(B.grad_by_value().data(), db, eb, "dbias")
    T.clear_gradients()


def test_linear_of_more_axes():
    x, w = normal((2, 3, 5), 1), normal((5, 4), 2)
    X = tensor(x).with_requires_grad()
    y = X.linear(tensor(w), activation="relu")
    assert y.shape == (2, 3, 4)
    y.backward(T.Tensor.ones((2, 3, 4)))
    assert X.grad_by_value().shape == (2, 3, 5)
    T.clear_gradients()


def far_values():
    return np.r_[np.linspace(-100, 100, 801), [-1e20, 1e20, -1e38, 1e38, -88.7, 88.7, -104, -0.0, 1e-30, -1e-42]]


@pytest.mark.parametrize("name", ["relu", "silu", "gelu_tanh"])
def test_activations_and_slopes_far_out(name):
    z = far_values().astype(np.float32)
    X, W = tensor(z.reshape(-1, 1)).with_requires_grad(), tensor(np.ones((1, 1), np.float32))
    y = X.linear(W, activation=name)
    zz = z.astype(np.float64).reshape(-1, 1)
    with np.errstate(over="ignore", invalid="ignore"):
        want, slope = R.act(zz, name), np.nan_to_num(R.act_slope(zz, name))
    # an exponential, a reciprocal and the cubic, each relative: the cubic's error enters times |v|, which is below 110
    # wherever the result is not the limit
    assert_within(y.data(), want, 16 * R.U * np.abs(want) * (1 + np.minimum(np.abs(zz) ** 3, 110)) + 1e-43, "y")
    y.backward(T.Tensor.ones((z.size, 1)))
    g = X.grad_by_value().data()
    near = (np.abs(zz) < 20).reshape(-1)
    assert np.all(np.isfinite(g))
    assert_within(g[near], slope[near], 64 * R.U * np.maximum(np.abs(slope[near]), 1), "slope")
    far = ~near
    assert np.allclose(g[far], (zz[far] > 0).astype(float), atol=1e-6)
    T.clear_gradients()


def test_linear_with_values_that_are_not_finite():
    x, w, b, r, go = layer_case(40, 70, 50, True, False)
    x[3, 5], x[7, 1], x[8, 2] = np.nan, np.inf, -np.inf
    y = tensor(x).linear(tensor(w), bias=tensor(b)).data()
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w + b
    assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(np.isinf(y), np.isinf(want))
    assert np.array_equal(y[np.isinf(y)] > 0, want[np.isinf(want)] > 0)
    rest = np.isfinite(want).all(1)
    assert_within(y[rest], want[rest], R.linear_bound(x[rest], w, b, "none", None, want[rest]), "y")


# ---- layers in 8 bits -------------------------------------------------------------------


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 8, 8), (1, 4096, 512), (2, 33, 5), (5, 127, 19), (16, 128, 64), (17, 129, 65),
                                   (33, 1531, 31), (70, 300, 77), (200, 640, 130), (1024, 1024, 1024), (1999, 1531, 777),
                                   (129, 8000, 1000), (5000, 100, 2050)])
@pytest.mark.parametrize("name,bias,residual", [("none", False, False), ("relu", True, False), ("silu", True, True),
                                                ("gelu_tanh", False, True)])
def test_linear_packed(m, k, n, name, bias, residual):
    x, w, b, r, _ = layer_case(m, k, n, bias, residual)
    w = np.ascontiguousarray(w.T)
    xq, wq = (R.unpack8(*R.pack8(a), k) for a in (x, w))
    y = packed(x).linear(packed(w), bias=tensor(b) if bias else None, activation=name,
                         residual=tensor(r) if residual else None)
    want, z = R.linear(xq, wq.T, b, name, r)
    assert_within(y.data(), want, R.linear_bound(xq, wq.T, b, name, r, z), "y")


def test_linear_packed_scales_of_every_size():
    """Blocks from the smallest scale to the largest, the products' exponents in range."""
    m, n, k = 9, 20, 32 * 40
    rng = np.random.default_rng(3)
    e = rng.integers(-110, 111, (40,))
    x = (rng.standard_normal((m, k)) * 2.0 ** np.repeat(e, 32)).astype(np.float32)
    w = (rng.standard_normal((n, k)) * 2.0 ** np.repeat(-e, 32)).astype(np.float32)
    xq, wq = (R.unpack8(*R.pack8(a), k) for a in (x, w))
    y = packed(x).linear(packed(w))
    want = xq @ wq.T
    assert_within(y.data(), want, R.product_bound(xq, wq.T), "y")


def test_linear_packed_nan_codes_and_nothing():
    x, w = normal((4, 50), 1), normal((6, 50), 2)
    x[2, 7] = np.nan
    y = tensor(x).pack8().linear(tensor(w).pack8()).data()
    assert np.isnan(y[2]).all() and np.isfinite(np.delete(y, 2, 0)).all()
    b = normal((6,), 3)
    y = T.Tensor.zeros((4, 0)).pack8().linear(T.Tensor.zeros((6, 0)).pack8(), bias=tensor(b)).data()
    assert np.array_equal(y, np.tile(b, (4, 1)))
    assert T.Tensor.zeros((0, 5)).pack8().linear(tensor(w[:, :5]).pack8()).shape == (0, 6)


# ---- the rest ---------------------------------------------------------------------------


def test_refusals():
    x, w = tensor(normal((4, 6), 1)), tensor(normal((6, 5), 2))
    v5, v6 = tensor(normal((5,), 3)), tensor(normal((6,), 4))
    r = tensor(normal((4, 5), 5))
    for call, what in ((lambda: x.linear(x), "Inner dimensions must match"), (lambda: x.linear(v6), "weight matrix"),
                       (lambda: x.linear(w, bias=v6), "bias"), (lambda: x.linear(w, residual=x), "residual"),
                       (lambda: x.rms_norm(v5), "weight"), (lambda: x.add_rms_norm(r, v6), "residual"),
                       (lambda: x.rms_norm(v6, -1.0), "eps"), (lambda: x.rms_norm(v6, float("nan")), "eps"),
                       (lambda: v6.pack8(), "matrix"), (lambda: v6.rms_norm_packed(v6), "matrix"),
                       (lambda: x.pack8().linear(r.pack8()), "Inner dimensions must match"),
                       (lambda: x.pack8().linear(x.pack8(), bias=v5), "bias")):
        with pytest.raises(T.TsError, match=what):
            call()


def test_device_memory_is_used_in_place_and_given_back():
    import gc

    a = DeviceArray(normal((8, 16), 1))
    t = T.Tensor.from_device(a)
    assert t.device_ptr() == a.dev.ptr and np.array_equal(t.data(), a.host)
    t.fill(2.0)
    T.synchronize()
    assert np.array_equal(a.get(), np.full((8, 16), 2.0, np.float32))
    from train_station_amd import tensor as module

    held = len(module._lent)
    w = tensor(normal((16, 4), 2)).with_requires_grad()
    y = t.linear(w)
    del t
    gc.collect()
    assert len(module._lent) == held  # the recorded layer reads it in its backward pass
    y.backward(T.Tensor.ones((8, 4)))
    assert np.allclose(w.grad_by_value().data(), 16.0)
    T.clear_gradients()
    del y
    gc.collect()
    assert len(module._lent) == held - 1
    host = np.zeros((2, 3), np.float32)

    class Host:
        __cuda_array_interface__ = dict(shape=(2, 3), typestr="<f4", data=(host.ctypes.data, False), version=2)

    class Past(Host):  # more than the allocation holds
        __cuda_array_interface__ = dict(shape=(1 << 40,), typestr="<f4", data=(a.dev.ptr, False), version=2)

    for bad in (Host(), Past()):
        with pytest.raises(T.TsError, match="device memory"):
            T.Tensor.from_device(bad)
    assert len(module._lent) == held - 1


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("rows,cols", [(3, 5), (64, 8), (40, 300), (700, 64)])
def test_every_operation_takes_memory_at_any_address(rows, cols, offset):
    """The framework's operations over a caller's memory, as over its own: only the order of a sum may differ."""
    x, y, w = np.abs(normal((rows, cols), 1)) + 0.1, normal((rows, cols), 2), normal((cols, 24), 3)
    v, go = normal((cols,), 4), normal((rows, 24), 5)

    def run(place):
        X, Y, W, V, G = (place(a) for a in (x, y, w, v, go))
        out = [X.add_tensor(Y), X.sub_tensor(Y), Y.mul_tensor(X), Y.div_tensor(X), X.add_tensor(V), X.exp(), X.log(), X.sqrt(),
               Y.tanh(), Y.sigmoid(), Y.relu(), Y.leaky_relu(0.1), X.pow_scalar(1.5), X.add_scalar(2.0), Y.softmax(1), Y.softmax(0),
               X.sum(), X.mean(), X.sum_dims([0]), X.sum_dims([1]), X.mean_dims([0, 1]), Y.t().contiguous(), Y.clone(),
               Y.matmul(W), Y.t().matmul(G), G.t().matmul(Y), Y.matmul(X.t()), Y.rms_norm(V), Y.pack8().unpack(),
               Y.linear(W, activation="silu", residual=G), T.Tensor.from_binary(Y.to_binary()), T.Tensor.from_json(Y.to_json())]
        got = [t.data() for t in out]
        # a layer's step: gradients, the optimizer on the caller's parameters
        B = place(np.zeros(24, np.float32))
        for p in (W, B):
            p.with_requires_grad()
        opt = T.Adam.with_learning_rate(1e-2)
        opt.add_parameters([W, B])
        loss = G.mul_tensor(G).mean()  # of the gradient that the products read
        Y.matmul(W).add_tensor(B).backward(G)
        got += [W.grad_by_value().data(), B.grad_by_value().data(), loss.data()]
        opt.step([W, B])
        opt.zero_grad([W, B])
        T.clear_gradients()
        X.fill(3.0)
        return got + [W.data(), B.data(), X.data()]

    own = run(tensor)
    lent = run(lambda a: T.Tensor.from_device(DeviceArray(np.ascontiguousarray(a, np.float32), offset)))
    for n, (a, b) in enumerate(zip(own, lent)):
        assert a.shape == b.shape and np.allclose(a, b, rtol=2e-6, atol=2e-5), n


@pytest.mark.parametrize("order", ["synchronize", "stream"])
def test_lent_memory_may_be_written_again_once_the_library_is_waited_for(order):
    """What was computed from it has the values it held then, read or not by the time it is written."""
    x, w = normal((48, 32), 1), normal((32, 24), 2)
    go = np.abs(normal((48, 24), 3))

    def values(t, g, W):
        y = t.matmul(W)
        m = t.mul_scalar(2.0).add_scalar(1.0)
        W.with_requires_grad()
        s = g.mul_scalar(3.0).sum()
        out = [y, y.relu(), t.matmul(W).add_tensor(y).sum(), m, m.mul_tensor(m).mean(), t.sum(), t.t().contiguous(), t.exp(),
               t.softmax(1), t.sum_dims([0]), t.linear(W), t.clone(), s]
        return out

    want = [v.data() for v in values(tensor(x), tensor(go), tensor(w))]
    a, b, c = DeviceArray(x), DeviceArray(go), DeviceArray(w)
    got = values(*(T.Tensor.from_device(v) for v in (a, b, c)))
    if order == "synchronize":
        T.synchronize()
    else:  # as an event recorded there would
        hip_check(hip.ts_hip_stream_synchronize(T.stream()), "ts_hip_stream_synchronize")
    for v in (a, b, c):
        v.dev.put(np.full(v.host.size, 7.0, np.float32))
    for n, (g, v) in enumerate(zip(got, want)):
        assert np.array_equal(g.data(), v), n
    T.clear_gradients()


def test_gradients_outlive_the_lent_memory_of_the_one_they_came_from():
    """A residual's gradient is the output's own; it stays when the caller writes that memory again, and adds up."""
    x, w, r = normal((20, 16), 1), normal((16, 12), 2), normal((20, 12), 3)
    X, Rs, W = tensor(x), tensor(r).with_requires_grad(), tensor(w)
    A = tensor(r).with_requires_grad()
    first, second = normal((20, 12), 4), normal((20, 12), 5)
    lent = DeviceArray(first)
    g = T.Tensor.from_device(lent)
    y = X.linear(W, residual=Rs).add_tensor(A)
    y.backward(g)
    T.synchronize()
    lent.dev.put(second)
    for t in (Rs, A, y):
        assert np.array_equal(t.grad_by_value().data(), first)
    X.linear(W, residual=Rs).add_tensor(A).backward(g)
    T.synchronize()
    lent.dev.put(np.zeros_like(second))
    for t in (Rs, A):
        assert np.array_equal(t.grad_by_value().data(), first + second)
    T.clear_gradients()


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("m,k,n", [(64, 8, 8), (32, 784, 128), (64, 40, 64)])
def test_a_sum_beside_a_weights_gradient_takes_memory_at_any_address(m, k, n, offset):
    """A gradient over a caller's memory whose sum waits: the weight gradient's launch forms it where it can."""
    x, w, go = normal((m, k), 1), normal((k, n), 2), normal((m, n), 3)
    W, B = tensor(w).with_requires_grad(), tensor(np.zeros(n, np.float32)).with_requires_grad()
    g = T.Tensor.from_device(DeviceArray(go, offset))
    total = g.mul_scalar(2.0).sum()
    tensor(x).matmul(W).add_tensor(B).backward(g)
    g64 = go.astype(np.float64)
    assert abs(total.value() - 2 * g64.sum()) <= m * n * R.U * 2 * np.abs(g64).sum()
    assert_within(W.grad_by_value().data(), x.T.astype(np.float64) @ g64, R.product_bound(x.T, go), "dweight")
    assert_within(B.grad_by_value().data(), g64.sum(0), m * R.U * np.abs(g64).sum(0), "dbias")
    T.clear_gradients()


def test_memory_of_another_device_is_refused():
    import ctypes

    count = ctypes.c_int()
    hip_check(hip.ts_hip_get_device_count(ctypes.byref(count)), "ts_hip_get_device_count")
    a = DeviceArray(normal((8, 16), 1))
    assert hip.ts_hip_check_device_range(a.dev.ptr, a.host.nbytes) == 0
    if count.value < 2:
        pytest.skip("one device")
    hip_check(hip.ts_hip_set_device(1), "ts_hip_set_device")
    try:
        assert hip.ts_hip_check_device_range(a.dev.ptr, a.host.nbytes) != 0
        with pytest.raises(T.TsError, match="device memory"):
            T.Tensor.from_device(a)
    finally:
        hip_check(hip.ts_hip_set_device(0), "ts_hip_set_device")


def block_parameters(d=48, f=80, seed=0):
    return [tensor(a).with_requires_grad() for a in (np.ones(d, np.float32), normal((d, f), seed + 1, d ** -0.5),
                                                     np.zeros(f, np.float32), normal((f, d), seed + 2, f ** -0.5),
                                                     np.zeros(d, np.float32))]


def block_step(ps, opt, x, r, t):
    norm, w1, b1, w2, b2 = ps
    h, stream = x.add_rms_norm(r, norm)
    y = h.linear(w1, bias=b1, activation="silu", checkpoint="8bit").linear(w2, bias=b2, residual=stream, checkpoint="8bit")
    d = y.sub_tensor(t)
    loss = d.mul_tensor(d).mean()
    loss.backward()
    opt.step(ps)
    opt.zero_grad(ps)
    T.clear_gradients()
    return loss


@pytest.mark.parametrize("batch,d,f", [(32, 48, 80), (1100, 520, 1400)])
def test_block_trains_and_replays_as_it_runs(batch, d, f):
    """A block's step recorded and replayed, with eager work between the replays, has the eager steps' bits."""
    x, r, t = (tensor(normal((batch, d), s)) for s in (5, 6, 7))
    lr = 1e-2 if d < 100 else 1e-3
    eager, opt = block_parameters(d, f), T.Adam.with_learning_rate(lr)
    opt.add_parameters(eager)
    losses = [block_step(eager, opt, x, r, t).value() for _ in range(7)]
    assert losses[-1] < (0.7 if d < 100 else 0.95) * losses[0]
    ps, opt2 = block_parameters(d, f), T.Adam.with_learning_rate(lr)
    opt2.add_parameters(ps)
    block_step(ps, opt2, x, r, t)
    with T.StepGraph.record() as g:
        block_step(ps, opt2, x, r, t)
    for n in (1, 2, 1):
        g.replay(n)
        T.synchronize()
        tensor(normal((16, d), 9)).linear(ps[1]).sum().value()
    block_step(ps, opt2, x, r, t)
    block_step(ps, opt2, x, r, t)
    for a, b in zip(eager, ps):
        assert np.array_equal(a.data(), b.data())
    g.free()


def test_a_stack_of_blocks_by_leaves_has_the_stacks_gradients():
    """Each block's input a leaf of its own, its gradient passed on to the block below: every node runs once."""
    depth, batch, d, f = 4, 24, 48, 80
    stack = [block_parameters(d, f, 10 * i) for i in range(depth)]
    x, go = normal((batch, d), 5), normal((batch, d), 6)

    def block(ps, h):
        norm, w1, b1, w2, b2 = ps
        y = h.rms_norm(norm).linear(w1, bias=b1, activation="silu")
        return y.linear(w2, bias=b2, residual=h)

    def grads(first):
        g = [first.grad_by_value().data()] + [p.grad_by_value().data() for ps in stack for p in ps]
        for ps in stack:
            for p in ps:
                p.zero_grad()
        T.clear_gradients()
        return g

    X = tensor(x).with_requires_grad()
    h = X
    for ps in stack:
        h = block(ps, h)
    h.backward(tensor(go))
    whole = grads(X)

    leaves, outs = [tensor(x).with_requires_grad()], []
    for ps in stack:
        outs.append(block(ps, leaves[-1]))
        with T.NoGradTrack():
            leaves.append(outs[-1].clone())
        leaves[-1].with_requires_grad()
    g = tensor(go)
    for leaf, y in zip(reversed(leaves[:-1]), reversed(outs)):
        y.backward(g)
        g = leaf.grad_by_value()
    for a, b in zip(grads(leaves[0]), whole):
        assert np.linalg.norm(a - b) <= 1e-5 * np.linalg.norm(b)


def test_a_recorded_step_keeps_the_device_memory_it_reads():
    import gc

    from train_station_amd import tensor as module

    held = len(module._lent)
    a, w = normal((24, 20), 1), normal((20, 12), 2)
    lent = T.Tensor.from_device(DeviceArray(a))
    W = tensor(w).with_requires_grad()
    opt = T.Adam.with_learning_rate(1e-3)
    opt.add_parameters([W])
    with T.StepGraph.record() as g:
        loss = lent.linear(W, activation="silu").sum()
        loss.backward()
        opt.step([W])
        opt.zero_grad([W])
        T.clear_gradients()
    del lent
    gc.collect()
    assert len(module._lent) == held + 1
    want = [R.linear(a, w, None, "silu", None)[0].sum()]
    g.replay(1)
    assert abs(loss.value() - want[0]) < 1e-3 * np.abs(want[0]) + 1e-3
    g.replay(2)
    T.synchronize()
    del loss
    g.free()
    gc.collect()
    assert len(module._lent) == held


def test_equal_calls_give_equal_bits():
    outs = []
    for m, k, n in 2 * [(150, 260, 190)] + 2 * [(1100, 1030, 900)]:
        x, w, b, r, go = layer_case(m, k, n, True, True)
        X, W, B = (tensor(a).with_requires_grad() for a in (x, w, b))
        y = X.linear(W, bias=B, activation="gelu_tanh", residual=tensor(r), checkpoint="8bit")
        y.backward(tensor(go))
        outs.append([y.data()] + [t.grad_by_value().data() for t in (X, W, B)])
        T.clear_gradients()
    for first, second in (outs[:2], outs[2:]):
        for a, b in zip(first, second):
            assert np.array_equal(a, b)


def test_example_trains_and_serves():
    """The example block: its loss falls, and in 8 bits it is within what its three roundings of 2^-4 a value,
    averaged over the sums, come to."""
    import importlib.util

    from conftest import ROOT

    spec = importlib.util.spec_from_file_location("feedforward_block", ROOT / "examples" / "feedforward_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, off = example.main(width=96, hidden=160, batch=40, steps=12)
    assert losses[-1] < 0.8 * losses[0] and np.all(np.isfinite(losses))
    assert 0 < off < 2.0 ** -4
