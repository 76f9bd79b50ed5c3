"""A student's operators on the device against their plain forms in 64 bits
(student_ref.py, which derives the tolerances)."""
from __future__ import annotations

import numpy as np
import pytest

import student_ref as R
from conftest import normal
from gpu_util import Dev, T, ZeroIndex, hip, hip_check, sync
from test_feedforward_gpu import DeviceArray, assert_within, tensor

pytestmark = pytest.mark.gpu
EPS = 1e-5


class IndexArray:
    """A device buffer of 32-bit whole numbers as other libraries expose theirs."""

    def __init__(self, a, offset=0):
        self.host = np.ascontiguousarray(a, np.int32)
        self.dev = Dev.of(self.host.view(np.float32).reshape(-1), offset)
        self.__cuda_array_interface__ = dict(shape=self.host.shape, typestr="<i4", data=(self.dev.ptr, False), version=2)


def indices(a):
    a = np.asarray(a, np.int32)
    return T.Indices.from_slice(a, a.shape)


def blocks(a, tiles=False):
    """A Block8 of the plain form's codes, and its values in 64 bits."""
    codes, scales = R.block8(a, tiles)
    return (T.Block8.from_device(DeviceArray(codes), DeviceArray(scales), a.shape[1], tiles),
            R.block8_values(codes, scales, a.shape[1], tiles))


def parts(p):
    """codes and scales of a Block8, on the host."""
    T.synchronize()
    rows, pitch = p.shape[0], p.pitch
    codes = np.empty((rows, pitch), np.uint8)
    scales = np.empty((pitch // 128, R.scale_rows(rows, p.tiles)), np.float32)
    hip_check(hip.ts_hip_memcpy_bytes(codes.ctypes.data, p.codes_ptr(), codes.nbytes, 1, None), "codes")
    hip_check(hip.ts_hip_memcpy_bytes(scales.ctypes.data, p.scales_ptr(), scales.nbytes, 1, None), "scales")
    sync()
    return codes, scales


# ---- values in 8 bits ---------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 127), (3, 128), (2, 129), (127, 5), (128, 130), (129, 256), (300, 1003), (1, 5000)])
@pytest.mark.parametrize("tiles", [False, True])
def test_block8(rows, cols, tiles):
    rng = np.random.default_rng(rows * cols)
    x = (rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-38, 37, (rows, 1))).astype(np.float32)
    x[rng.random((rows, cols)) < 0.1] = 0.0
    p = tensor(x).block8(tiles)
    assert p.shape == (rows, cols) and p.pitch == R.pitch_of(cols) and p.tiles == tiles
    codes, scales = parts(p)
    want = R.block8(x, tiles)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])
    assert np.array_equal(p.unpack().data(), R.unblock8(*want, cols, tiles))


@pytest.mark.parametrize("tiles", [False, True])
def test_block8_borders_and_what_no_code_holds(tiles):
    """Every code, every border between two and their neighbours, at small, middle and large scales; infinities and NaN."""
    v = R.e4m3_values()[:127]
    base = np.r_[v, (v[1:] + v[:-1]) / 2].astype(np.float32)
    base = np.r_[base, np.nextafter(base, np.float32(np.inf)), np.nextafter(base, np.float32(-np.inf))]
    base = np.resize(np.clip(np.r_[base, -base], -448, 448), 127 * 12).reshape(-1, 127)
    rows = [np.c_[base, np.full(len(base), 448.0)] * 2.0 ** k for k in (-108, -60, 0, 60, 119)]
    odd = np.zeros((4, 128))
    odd[0, :3] = [np.inf, -np.inf, 1.0]
    odd[1, :3] = [np.nan, 2.0, -3.0]
    odd[2, :2] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    odd[3, :3] = [1e-45, 2.0 ** -127, 2.0 ** -126]
    x = np.concatenate([odd, *rows]).astype(np.float32)
    if tiles:  # a block each: 127 rows of zeros after every one
        apart = np.zeros((len(x) * 128, 128), np.float32)
        apart[::128] = x
        x = apart
    codes, scales = parts(tensor(x).block8(tiles))
    want = R.block8(x, tiles)
    assert np.array_equal(scales, want[1])
    nan = (want[0] & 127) == 127  # either of the two NaN codes
    assert nan.sum() == 1 and np.all((codes[nan] & 127) == 127) and np.array_equal(codes[~nan], want[0][~nan])
    assert codes[0, 0] == 0x7e and codes[0, 1] == 0xfe and np.all(np.isfinite(scales))


@pytest.mark.parametrize("tiles", [False, True])
def test_block8_of_values_within_a_rounding_of_a_border(tiles):
    """Their fp32 rounding is the border itself, at every border and for scales of many bits: the code is the value's own."""
    v = R.e4m3_values()[:127]
    border = (v[1:] + v[:-1]) / 2
    x = np.zeros((40, 3 * 128), np.float32)
    for row, top in zip(x, np.random.default_rng(3).uniform(1, 2, len(x)).astype(np.float32)):
        near = (border * (np.float64(top) / 448)).astype(np.float32)
        near = np.r_[near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf))]
        row.reshape(3, 128)[:, 0] = top
        row.reshape(3, 128)[:, 1:] = np.resize(near, (3, 127)) * np.resize([1, -1], 127)
    if tiles:
        x = np.concatenate([x, np.zeros((127 * len(x), x.shape[1]), np.float32)]).reshape(128, len(x), -1).swapaxes(0, 1).reshape(-1, x.shape[1])
    codes, scales = parts(tensor(x).block8(tiles))
    want = R.block8(x, tiles)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


def test_block8_of_nothing_and_of_a_view():
    assert T.Tensor.zeros((0, 5)).block8().shape == (0, 5) and T.Tensor.zeros((5, 0)).block8(True).unpack().shape == (5, 0)
    x = normal((40, 300), 1)
    codes, scales = parts(tensor(x).t().block8())
    want = R.block8(np.ascontiguousarray(x.T))
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])


# ---- layers in 8 bits -----------------------------------------------------------------

LAYERS = [(1, 1, 1), (1, 128, 128), (3, 5, 7), (16, 130, 128), (17, 65, 31), (33, 784, 10), (128, 129, 130), (2, 1000, 3),
          (257, 40, 300), (1, 513, 129), (300, 17, 33), (128, 128, 128), (129, 1000, 257), (200, 2000, 260), (1, 4096, 1000),
          (500, 300, 700), (1000, 1003, 1029), (20, 2000, 2100), (20, 1200, 8200), (500, 1100, 700), (29, 130, 17000)]


@pytest.mark.parametrize("m,k,n", LAYERS)
@pytest.mark.parametrize("act,bias,residual", [("none", False, False), ("relu", True, True), ("silu", True, False),
                                               ("gelu_tanh", False, True)])
def test_block8_linear(m, k, n, act, bias, residual):
    x, xv = blocks(normal((m, k), 1) * np.float32(3))
    w, wv = blocks(normal((n, k), 2, k ** -0.5), True)
    b = normal((n,), 3, 0.1) if bias else None
    r = normal((m, n), 4) if residual else None
    y = x.linear(w, tensor(b) if bias else None, act, tensor(r) if residual else None)
    want, bound = R.linear(xv, wv, b, act, r)
    assert_within(y.data(), want, bound, "y")


@pytest.mark.parametrize("m,k,n", [(64, 200, 8200), (8255, 100, 65), (1003, 1, 900), (2000, 150, 2101), (2011, 1153, 2080),
                                   (2975, 130, 2801), (3001, 700, 2820),
                                   (2050, 2200, 2050), (1100, 2300, 1100), (70, 2190, 8200),
                                   (33, 300, 8300), (64, 140, 33000), (8200, 300, 33), (33000, 140, 64)])
def test_block8_linear_by_tiles(m, k, n):
    """Each size of tile, with edges within it, one and several blocks of columns."""
    x, xv = blocks(normal((m, k), 1))
    w, wv = blocks(normal((n, k), 2, k ** -0.5), True)
    b, r = normal((n,), 3, 0.1), normal((m, n), 4)
    want, bound = R.linear(xv, wv, b, "silu", r)
    assert_within(x.linear(w, tensor(b), "silu", tensor(r)).data(), want, bound, "y")


@pytest.mark.parametrize("m,k,n", [(1, 300, 140), (150, 300, 300), (1500, 900, 800)])
def test_block8_linear_of_far_scales_and_odd_codes(m, k, n):
    """Rows and tiles of sizes far apart, and every row its own: a wrong row's or block's scale shows."""
    rng = np.random.default_rng(5)
    x = normal((m, k), 1) * (2.0 ** rng.integers(-30, 30, (m, 1))) * 2.0 ** (rng.integers(-3, 3, -(-k // 128)).repeat(128)[:k])
    w = normal((n, k), 2) * (2.0 ** rng.integers(-20, 20, -(-n // 128))).repeat(128)[:n, None]
    (X, xv), (W, wv) = blocks(x.astype(np.float32)), blocks(w.astype(np.float32), True)
    want, bound = R.linear(xv, wv, None, "none", None)
    assert_within(X.linear(W).data(), want, bound, "y")


@pytest.mark.parametrize("m,n", [(3, 5), (400, 300)])
def test_block8_linear_of_nothing_and_of_nan(m, n):
    b, r = normal((n,), 3), normal((m, n), 4)
    X, W = T.Tensor.zeros((m, 0)).block8(), T.Tensor.zeros((n, 0)).block8(True)
    assert np.array_equal(X.linear(W, tensor(b), "relu", tensor(r)).data(), np.maximum(b, 0) + r)
    assert T.Tensor.zeros((0, 5)).block8().linear(T.Tensor.ones((4, 5)).block8(True)).shape == (0, 4)
    large = T.Tensor.zeros((1100, 0)).block8().linear(T.Tensor.zeros((1030, 0)).block8(True)).data()
    assert large.shape == (1100, 1030) and not large.any()
    x, w = normal((m, 1200), 1), normal((n, 1200), 2)
    x[1, 700] = np.nan
    y = tensor(x).block8().linear(tensor(w).block8(True)).data()
    assert np.isnan(y[1]).all() and np.isfinite(np.delete(y, 1, 0)).all()


def test_block8_linear_over_a_caller_s_memory_at_any_offset_of_16_bytes():
    x, w = normal((140, 200), 1), normal((150, 200), 2)
    (cx, sx), (cw, sw) = R.block8(x), R.block8(w, True)
    X = T.Block8.from_device(DeviceArray(cx, 4), DeviceArray(sx, 1), 200)
    W = T.Block8.from_device(DeviceArray(cw, 8), DeviceArray(sw, 3), 200, tiles=True)
    want, bound = R.linear(R.block8_values(cx, sx, 200), R.block8_values(cw, sw, 200, True), None, "none", None)
    assert_within(X.linear(W).data(), want, bound, "y")
    with pytest.raises(T.TsError, match="16-byte"):
        T.Block8.from_device(DeviceArray(cx, 1), DeviceArray(sx), 200)
    with pytest.raises(T.TsError, match="one allocation"):
        small = DeviceArray(sx[:, :1])
        small.__cuda_array_interface__["shape"] = (2, 1 << 20)
        big = DeviceArray(cx)
        big.__cuda_array_interface__["shape"] = (1 << 20, 256)
        T.Block8.from_device(big, small, 200)


# ---- layer norm -----------------------------------------------------------------------

NORMS = [(1, 1), (1, 4096), (3, 7), (5, 256), (6, 257), (9, 512), (4, 1003), (130, 784), (7, 1025), (3, 2048), (2, 4095),
         (5, 4097), (2, 8192), (3, 8193), (2, 16384), (3, 16385), (2, 40001), (700, 64)]


def norm_case(rows, cols, residual, bias, far=0.0):
    x, r = normal((rows, cols), 1) + np.float32(far), normal((rows, cols), 2) * 3 if residual else None
    w = (1 + 0.2 * normal((cols,), 3)).astype(np.float32)
    b = normal((cols,), 5, 0.5) if bias else None
    return x, r, w, b, x if r is None else (x + r).astype(np.float32)


def check_layer_norm(rows, cols, residual, bias, far=0.0, eps=EPS):
    x, r, w, b, h = norm_case(rows, cols, residual, bias, far)
    go = normal((rows, cols), 4)
    X, W = tensor(x).with_requires_grad(), tensor(w).with_requires_grad()
    B = tensor(b).with_requires_grad() if bias else None
    Rs = tensor(r).with_requires_grad() if residual else None
    if residual:
        y, stream = X.add_layer_norm(Rs, W, B, eps)
        assert np.array_equal(stream.data(), h)
    else:
        y = X.layer_norm(W, B, eps)
    assert_within(y.data(), R.layer_norm(h, w, b, eps), R.layer_norm_bound(h, w, b, eps), "y")
    y.backward(tensor(go))
    want, bound = R.layer_norm_grads(h, w, go, eps), R.layer_norm_grads_bound(h, w, go, eps)
    assert_within(X.grad_by_value().data(), want[0], bound[0], "dx")
    if residual:
        assert np.array_equal(Rs.grad_by_value().data(), X.grad_by_value().data())
    assert_within(W.grad_by_value().data(), want[1], bound[1], "dweight")
    if bias:
        assert_within(B.grad_by_value().data(), want[2], bound[2], "dbias")
    T.clear_gradients()


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("residual,bias", [(False, True), (True, False), (True, True)])
def test_layer_norm(rows, cols, residual, bias):
    check_layer_norm(rows, cols, residual, bias)


@pytest.mark.parametrize("rows,cols", [(600, 8192), (600, 8200), (300, 16383), (1100, 4100), (1500, 1030), (300, 16390), (70, 40001),
                                       (2100, 255), (2101, 510), (2102, 1021), (1025, 2047),
                                       (9000, 128), (5001, 60), (4099, 127), (3001, 5), (2, 3)])
def test_layer_norm_sums_many_rows(rows, cols):
    check_layer_norm(rows, cols, True, True)


@pytest.mark.parametrize("far", [1.0, 1e3, -1e6, 3e7])
@pytest.mark.parametrize("cols", [40, 1000, 5000, 20000])
def test_layer_norm_of_rows_far_from_zero(cols, far):
    check_layer_norm(3, cols, False, True, far)


FAR_ROWS = [1e-42, 1e-38, 1e-30, 1e-20, 1e-12, 1.0, 1e12, 1e18, 1e20, 1e30, 3e37]


@pytest.mark.parametrize("cols", [2, 40, 300, 1500, 4000, 8000, 16384, 20000])
def test_layer_norm_of_tiny_and_huge_rows_without_eps(cols):
    size = np.asarray(FAR_ROWS)[:, None]
    h = normal((size.size, cols), 1).astype(np.float64)
    h[:, 0], h[:, 1] = 1.0, -1.0  # no constant row, of any size
    h = (np.clip(h, -6, 6) * size).astype(np.float32)
    go = (normal((size.size, cols), 2) * np.sqrt(np.minimum(size, 1.0))).astype(np.float32)
    w = (1 + 0.2 * normal((cols,), 3)).astype(np.float32)
    X, W = tensor(h).with_requires_grad(), tensor(w).with_requires_grad()
    y = X.layer_norm(W, None, 0.0)
    assert_within(y.data(), R.layer_norm(h, w, None, 0.0), R.layer_norm_bound(h, w, None, 0.0), "y")
    y.backward(tensor(go))
    want, bound = R.layer_norm_grads(h, w, go, 0.0), R.layer_norm_grads_bound(h, w, go, 0.0)
    assert_within(X.grad_by_value().data(), want[0], bound[0], "dx")
    assert_within(W.grad_by_value().data(), want[1], bound[1], "dweight")
    T.clear_gradients()


def test_layer_norm_of_constant_rows_and_of_what_is_not_finite():
    low = np.finfo(np.float32).min
    x = normal((7, 300), 1)
    x[0], x[1], x[2] = 0.0, low, 1e30
    x[3, 5], x[4, 0], x[5, 7] = np.nan, np.inf, -np.inf
    b, w = normal((300,), 2), normal((300,), 3)
    X, W, B = (tensor(a).with_requires_grad() for a in (x, w, b))
    y = X.layer_norm(W, B)
    for r in range(3):  # (h - mean) r is 0
        assert np.array_equal(y.data()[r], b)
    assert np.isnan(y.data()[3:6]).all() and np.isfinite(y.data()[6]).all()
    y.backward(tensor(np.ones_like(x)))
    assert np.isfinite(X.grad_by_value().data()[:3]).all() and np.isnan(W.grad_by_value().data()).all()
    assert np.array_equal(B.grad_by_value().data(), np.full(300, 7, np.float32))
    assert np.isnan(tensor(x[:1]).layer_norm(tensor(w), None, 0.0).data()).all()  # 0 / 0
    T.clear_gradients()


@pytest.mark.parametrize("cols", [40, 1200, 20000])
@pytest.mark.parametrize("need", ["x", "weight", "bias", "weight bias", "x bias"])
def test_layer_norm_gradients_that_are_asked_for(cols, need):
    x, _, w, b, h = norm_case(33, cols, False, True)
    go = normal((33, cols), 4)
    leaves = dict(x=tensor(x), weight=tensor(w), bias=tensor(b))
    for k in need.split():
        leaves[k].with_requires_grad()
    leaves["x"].layer_norm(leaves["weight"], leaves["bias"]).backward(tensor(go))
    for k, want, bound in zip(leaves, R.layer_norm_grads(h, w, go, EPS), R.layer_norm_grads_bound(h, w, go, EPS)):
        got = leaves[k].grad_by_value()
        assert (got is not None) == (k in need.split())
        if got is not None:
            assert_within(got.data(), want, bound, k)
    T.clear_gradients()


def test_layer_norm_keeps_what_fp32_sums_lose():
    rows, cols = 40 * 256 + 1, 16388
    go = np.zeros((rows, cols), np.float32)
    go[::256] = 0.9 * 2.0 ** -25  # of rows that one workgroup of 256 takes in turn; beside 1, nothing in fp32
    go[0] = 1.0
    B = tensor(np.zeros(cols, np.float32)).with_requires_grad()
    T.Tensor.ones((rows, cols)).layer_norm(T.Tensor.ones((cols,)), B).backward(tensor(go))
    want = go[::256].astype(np.float64).sum(0)
    assert_within(B.grad_by_value().data(), want, 3 * R.U * want, "dbias")
    T.clear_gradients()


@pytest.mark.parametrize("rows,cols", [(1, 5), (128, 784), (700, 64), (3000, 1000)])
def test_layer_norm_backward_with_and_without_a_ticket(rows, cols):
    """The same sums by one launch and by two, to the last place, and the ticket zero again."""
    h, go = Dev.of(normal((rows, cols), 1)), Dev.of(normal((rows, cols), 2))
    w, ticket = Dev.of(normal((cols,), 3)), Dev.of(np.zeros(1, np.float32))
    floats = hip.ts_hip_layer_norm_backward_workspace_floats(rows, cols)
    work, got = Dev(floats), []
    for t in (None, ticket.ptr, ticket.ptr):
        dh, dw, db = Dev(rows * cols), Dev(cols), Dev(cols)
        hip_check(hip.ts_hip_layer_norm_backward(h.ptr, w.ptr, go.ptr, rows, cols, EPS, dh.ptr, dw.ptr, db.ptr, work.ptr, floats,
                                                 t, None))
        got.append((dh.get(), dw.get(), db.get()))
    assert not ticket.get().view(np.uint32).any()
    for dh, dw, db in got[1:]:
        assert np.array_equal(dh, got[0][0])
        # (the parts in another order of f64 sums: the last place)
        assert np.allclose(dw, got[0][1], rtol=2e-7, atol=0) and np.allclose(db, got[0][2], rtol=2e-7, atol=0)


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("residual,bias", [(False, False), (True, True)])
def test_layer_norm_block8(rows, cols, residual, bias):
    x, r, w, b, h = norm_case(rows, cols, residual, bias)
    X, W, B = tensor(x), tensor(w), tensor(b) if bias else None
    if residual:
        p, stream = X.add_layer_norm_block8(tensor(r), W, B)
        assert np.array_equal(stream.data(), h)
    else:
        p = X.layer_norm_block8(W, B)
    codes, scales = parts(p)
    want = R.block8(R.layer_norm(h, w, b, EPS))
    # (a row of one column and no bias is 0 / sqrt(eps): the mean's last bit is of no size)
    assert np.allclose(scales, want[1], rtol=2 * R.U, atol=0) and np.array_equal(codes, want[0])


def test_layer_norm_block8_of_many_values():
    """A code each on y's own side of its border, of three million."""
    x, r, w, b, h = norm_case(700, 4096, True, True)
    codes, scales = parts(tensor(x).add_layer_norm_block8(tensor(r), tensor(w), tensor(b))[0])
    want = R.block8(R.layer_norm(h, w, b, EPS))
    assert np.allclose(scales, want[1], rtol=2 * R.U, atol=0) and np.array_equal(codes, want[0])


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 6, 255, 257, 258, 509, 1021, 1022, 1026, 2047, 4094, 4099, 8189, 8194, 12289, 16381, 16386])
def test_layer_norm_entries_at_any_address(cols):
    """Rows that end within a quad, 4 bytes from any boundary, the sum in place of either input; nothing past the last row."""
    rows = 5
    x, r, w, b, h = norm_case(rows, cols, True, True)
    go = normal((rows, cols), 4)
    y_want, y_bound = R.layer_norm(h, w, b, EPS), R.layer_norm_bound(h, w, b, EPS)
    W, B, G = Dev.of(w, 1), Dev.of(b, 2), Dev.of(go, 3)
    past = np.full(3, 7.0, np.float32)

    def room(a, offset):
        return Dev.of(np.r_[np.asarray(a, np.float32).ravel(), past], offset)

    def of(d):
        a = d.get()
        assert np.array_equal(a[-3:], past)
        return a[:-3]

    for place in ("x", "residual", "apart"):
        X, Rs, Y = room(x, 1), room(r, 3), room(np.full(rows * cols, 7.0), 2)
        H = dict(x=X, residual=Rs, apart=room(np.zeros(rows * cols), 2))[place]
        hip_check(hip.ts_hip_layer_norm(X.ptr, Rs.ptr, W.ptr, B.ptr, rows, cols, EPS, H.ptr, Y.ptr, None))
        assert np.array_equal(of(H).reshape(rows, cols), h)
        assert_within(of(Y).reshape(rows, cols), y_want, y_bound, "y")
        of(X), of(Rs)
    floats = hip.ts_hip_layer_norm_backward_workspace_floats(rows, cols)
    work, ticket = Dev(floats), Dev.of(np.zeros(1, np.float32))
    dh, dw, db = room(np.full(rows * cols, 7.0), 1), room(np.full(cols, 7.0), 2), room(np.full(cols, 7.0), 3)
    hip_check(hip.ts_hip_layer_norm_backward(H.ptr, W.ptr, G.ptr, rows, cols, EPS, dh.ptr, dw.ptr, db.ptr, work.ptr, floats, ticket.ptr, None))
    want, bound = R.layer_norm_grads(h, w, go, EPS), R.layer_norm_grads_bound(h, w, go, EPS)
    for got, shape, a, e, what in zip((dh, dw, db), ((rows, cols), (cols,), (cols,)), want, bound, ("dh", "dweight", "dbias")):
        assert_within(of(got).reshape(shape), a, e, what)


def test_layer_norm_block8_pads_rows_of_nan_with_zeros():
    x = normal((3, 40), 1)
    x[1] = np.nan
    codes, _ = parts(tensor(x).layer_norm_block8(tensor(np.ones(40, np.float32)), tensor(np.ones(40, np.float32))))
    assert np.all((codes[1, :40] & 127) == 127) and not codes[:, 40:].any()


def test_layer_norm_of_more_rows_than_a_launch_has_workgroups():
    rows, cols = (1 << 23) + 5, 3
    x, w, b = normal((rows, cols), 1), normal((cols,), 2), normal((cols,), 3)
    y = tensor(x).layer_norm(tensor(w), tensor(b)).data()
    assert_within(y, R.layer_norm(x, w, b, EPS), R.layer_norm_bound(x, w, b, EPS), "y")


def test_layer_norm_gradients_accumulate_and_pass_through_the_sum():
    x, r, w, b, h = norm_case(6, 96, True, True)
    X, Rs, W, B = (tensor(a).with_requires_grad() for a in (x, r, w, b))
    y, stream = X.add_layer_norm(Rs, W, B)
    y.mul_tensor(y).add_tensor(stream).sum().backward()
    dh, dw, db = R.layer_norm_grads(h, w, 2 * R.layer_norm(h, w, b, EPS), EPS)
    for t, want in ((X, dh + 1), (Rs, dh + 1), (W, dw), (B, db)):
        assert np.allclose(t.grad_by_value().data(), want, rtol=1e-5, atol=1e-4)
    T.clear_gradients()


def test_layer_norm_of_more_axes_of_nothing_of_itself_and_without_gradients():
    x, w, b = normal((2, 3, 5), 1), normal((5,), 2), normal((5,), 3)
    X = tensor(x).with_requires_grad()
    y = X.layer_norm(tensor(w), tensor(b))
    assert_within(y.data().reshape(6, 5), R.layer_norm(x.reshape(6, 5), w, b, EPS), R.layer_norm_bound(x.reshape(6, 5), w, b, EPS), "y")
    y.backward(T.Tensor.ones((2, 3, 5)))
    assert X.grad_by_value().shape == (2, 3, 5)
    T.clear_gradients()
    E, W, B = T.Tensor.zeros((0, 5)).with_requires_grad(), tensor(w).with_requires_grad(), tensor(b).with_requires_grad()
    y = E.layer_norm(W, B)
    y.backward(T.Tensor.zeros((0, 5)))
    assert y.shape == (0, 5) and not W.grad_by_value().data().any() and not B.grad_by_value().data().any()
    T.clear_gradients()
    X = tensor(x).with_requires_grad()
    y, h = X.add_layer_norm(X, tensor(w))  # x twice
    y.backward(T.Tensor.ones((2, 3, 5)))
    dh, _, _ = R.layer_norm_grads((x + x).reshape(6, 5), w, np.ones((6, 5)), EPS)
    assert np.allclose(X.grad_by_value().data().reshape(6, 5), 2 * dh, rtol=1e-4, atol=1e-5)
    T.clear_gradients()
    with T.NoGradTrack():
        assert not X.layer_norm(tensor(w)).requires_grad() and not X.add_layer_norm(X, tensor(w))[1].requires_grad()


# ---- distillation ---------------------------------------------------------------------


def distill_case(rows, vocab, kept, seed=0):
    """Logits and lists of every kind: entries missing, given twice, of -inf, rows of none, labels among the entries and none."""
    rng = np.random.default_rng(seed)
    z = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    idx = rng.integers(0, vocab, (rows, kept)).astype(np.int32)
    teacher = (rng.standard_normal((rows, kept)) * 3).astype(np.float32)
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    w = (rng.random(rows) + 0.1).astype(np.float32)
    for r in range(rows):
        kind = r % 9
        if kind == 1:
            idx[r, rng.random(kept) < 0.5] = -1
        elif kind == 2:
            idx[r] = idx[r, 0]  # one column, all of them
        elif kind == 3:
            labels[r] = -1
        elif kind == 4:
            idx[r] = -1 - (np.arange(kept) % 3)
        elif kind == 5:
            teacher[r, rng.random(kept) < 0.5] = -np.inf
            labels[r] = idx[r, -1]
        elif kind == 6:
            masked = rng.random(vocab) < 0.3
            masked[idx[r]] = masked[labels[r]] = False
            z[r, masked] = -np.inf if r % 2 else np.finfo(np.float32).min
        elif kind == 7:
            idx[r], labels[r], z[r, 0] = -1, -1, np.nan
        elif kind == 8:
            w[r], z[r, 0] = 0.0, np.inf
    return z, idx, teacher, labels, w


def check_distillation(rows, vocab, kept, t, hard, weighted, seed=0, case=None):
    z, idx, teacher, labels, w = case or distill_case(rows, vocab, kept, seed)
    if not weighted and (case is None):
        z[8::9, 0] = 0.0
    want, dz, bound, bz = R.distillation(z, idx, teacher, t, labels, hard, w if weighted else None)
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(indices(idx), tensor(teacher), t, indices(labels) if hard else None, hard, tensor(w) if weighted else None)
    assert loss.shape == (1,)
    assert_within(loss.data(), np.array([want]), bound, "loss")
    loss.backward()
    assert_within(Z.grad_by_value().data(), dz, bz, "dz")
    T.clear_gradients()
    with T.NoGradTrack():  # without its gradient: the same bits
        again = Z.distillation(indices(idx), tensor(teacher), t, indices(labels) if hard else None, hard,
                               tensor(w) if weighted else None)
    assert not again.requires_grad() and np.array_equal(again.data(), loss.data())


# by rows (a wave, waves, long rows) and by segments (few rows of many columns)
DISTILL = [(1, 1, 1), (3, 7, 2), (19, 10, 3), (9, 255, 10), (10, 257, 5), (37, 1000, 64), (9, 1025, 300), (11, 4095, 20), (9, 4096, 8),
           (130, 1003, 17), (5000, 33, 4), (6000, 1029, 9), (70, 2047, 200), (41, 2048, 40), (9, 1500, 7), (9, 2049, 64), (27, 5001, 10), (3, 50001, 20), (2, 66000, 9), (30, 131071, 12), (10, 50001, 100), (2, 131072, 1024), (1, 300001, 5),
           (140, 4101, 30), (150, 8193, 9), (135, 16385, 33), (129, 32768, 70), (131, 40003, 11), (129, 65537, 20), (129, 131100, 40)]


@pytest.mark.parametrize("rows,vocab,kept", DISTILL)
@pytest.mark.parametrize("t,hard,weighted", [(1.0, 0.0, False), (2.0, 0.4, True)])
def test_distillation(rows, vocab, kept, t, hard, weighted):
    check_distillation(rows, vocab, kept, t, hard, weighted)


@pytest.mark.parametrize("rows,vocab,kept", [(27, 300, 6), (4, 60000, 12), (20, 9000, 12), (140, 9001, 12), (260, 33001, 12), (130, 70001, 5)])
@pytest.mark.parametrize("t,hard,weighted", [(1.0, 0.5, True), (0.5, 0.5, False), (3.0, 1.0, True), (1.0, 1.0, False), (10.0, 0.0, True),
                                             (2.0, 0.5, True), (4.0, 0.3, False), (1.5, 0.2, True)])
def test_distillation_s_shares_and_temperatures(rows, vocab, kept, t, hard, weighted):
    check_distillation(rows, vocab, kept, t, hard, weighted)


@pytest.mark.parametrize("rows,vocab", [(6, 50), (6, 60000), (6, 6000), (140, 6000)])
def test_distillation_without_entries(rows, vocab):
    z = normal((rows, vocab), 1)
    labels = np.arange(rows, dtype=np.int32)
    none = np.zeros((rows, 0), np.int32), np.zeros((rows, 0), np.float32)
    check_distillation(rows, vocab, 0, 2.0, 0.25, False, case=(z, *none, labels, None))
    check_distillation(rows, vocab, 0, 2.0, 0.0, False, case=(z, *none, labels, None))
    Z = T.Tensor.zeros((0, vocab)).with_requires_grad()
    loss = Z.distillation(T.Indices.from_slice([], (0, 4)), T.Tensor.zeros((0, 4)))
    loss.backward()
    assert loss.value() == 0.0 and Z.grad_by_value().shape == (0, vocab)
    T.clear_gradients()


@pytest.mark.parametrize("rows,vocab", [(4, 700), (4, 70000), (4, 7000), (132, 7000)])
def test_distillation_where_the_student_gives_no_chance(rows, vocab):
    """A column of -inf that the teacher asks for: the loss is infinite, the gradient p - q."""
    z = normal((rows, vocab), 1)
    idx, teacher = np.tile(np.array([3, 5], np.int32), (rows, 1)), np.zeros((rows, 2), np.float32)
    z[1, 3] = -np.inf
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(indices(idx), tensor(teacher))
    assert loss.value() == np.inf
    loss.backward()
    g = Z.grad_by_value().data()
    _, dz, _, bz = R.distillation(z, idx, teacher)
    assert_within(g, dz, bz, "dz")
    # asked of it with no weight, or of a row of nothing but -inf: nothing, and NaN in that row alone
    teacher[1, 0] = -np.inf
    assert np.isfinite(tensor(z).distillation(indices(idx), tensor(teacher)).value())
    z[2] = -np.inf
    Z = tensor(z).with_requires_grad()
    Z.distillation(indices(idx), tensor(teacher)).backward()
    g = Z.grad_by_value().data()
    assert np.isnan(g[2]).all() and np.isfinite(np.delete(g, 2, 0)).all()
    T.clear_gradients()


@pytest.mark.parametrize("rows,vocab", [(6, 3), (6, 1001), (6, 60001), (6, 6001), (132, 6001), (131, 33001), (130, 70001)])
@pytest.mark.parametrize("t,hard", [(1.0, 0.0), (2.0, 0.5), (1.5, 0.5)])
def test_distillation_of_logits_that_are_no_numbers(rows, vocab, t, hard):
    """A NaN anywhere in a row, or an infinity, makes the loss NaN and that row's gradient, no other's."""
    z = normal((rows, vocab), 1)
    idx, teacher, labels = np.zeros((rows, 1), np.int32), np.zeros((rows, 1), np.float32), np.zeros(rows, np.int32)
    for at, what in ((0, np.nan), (vocab - 1, np.nan), (vocab // 2, np.nan), (slice(None), np.nan), (vocab - 1, np.inf)):
        bad = z.copy()
        bad[1, at] = what
        Z = tensor(bad).with_requires_grad()
        loss = Z.distillation(indices(idx), tensor(teacher), t, indices(labels), hard)
        assert np.isnan(loss.value())
        loss.backward()
        g = Z.grad_by_value().data()
        assert np.isnan(g[1]).all() and np.isfinite(np.delete(g, 1, 0)).all()
        T.clear_gradients()


@pytest.mark.parametrize("rows,vocab", [(5, 90), (5, 60000), (5, 6000), (133, 6000)])
def test_distillation_s_gradient_is_scaled_and_asked_for_again(rows, vocab):
    z, idx, teacher, labels, w = distill_case(rows, vocab, 7)
    z[7::9, 0] = 0.0
    args = (indices(idx), tensor(teacher), 2.0, indices(labels), 0.3, tensor(w))
    _, dz, _, bz = R.distillation(z, idx, teacher, 2.0, labels, 0.3, w)
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(*args)
    loss.backward()
    first = Z.grad_by_value().data()
    Z.zero_grad()
    loss.backward(tensor(np.array([2.5], np.float32)))  # accumulates on the graph's own: 1 + 2.5
    assert_within(Z.grad_by_value().data(), 3.5 * dz, 3.5 * bz + 4 * R.U * np.abs(3.5 * dz), "dz again")
    T.clear_gradients()
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(*args)
    loss.mul_scalar(-0.5).backward()
    assert_within(Z.grad_by_value().data(), -0.5 * dz, 0.5 * bz + R.U * np.abs(dz), "dz scaled")
    T.clear_gradients()
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(*args)
    loss.backward()
    Z.grad_view().fill(0.0)  # what was handed out is the caller's
    T.clear_gradients()
    loss = Z.distillation(*args)
    T.set_fusion(False)
    try:
        loss.backward()
    finally:
        T.set_fusion(True)
    assert_within(Z.grad_by_value().data(), dz, bz, "dz without fusion")
    assert np.allclose(first, Z.grad_by_value().data(), rtol=1e-6, atol=1e-9)
    T.clear_gradients()


@pytest.mark.parametrize("rows,vocab", [(40, 90), (5, 60000), (5, 6000), (133, 6000)])
def test_distillation_reports_entries_outside_the_vocabulary(rows, vocab):
    z, teacher = normal((rows, vocab), 1), np.zeros((rows, 3), np.float32)
    idx, labels = np.zeros((rows, 3), np.int32), np.zeros(rows, np.int32)
    idx[2, 1], idx[4, 0] = vocab, np.iinfo(np.int32).max
    Z = tensor(z).with_requires_grad()
    loss = Z.distillation(indices(idx), tensor(teacher))
    with pytest.raises(T.TsError, match="entry 7 is outside the vocabulary"):
        T.synchronize()
    T.synchronize()  # said once
    loss.backward()
    labels[3] = vocab
    tensor(z).distillation(indices(np.zeros_like(idx)), tensor(teacher), 1.0, indices(labels), 0.5)
    with pytest.raises(T.TsError, match="label of row 3 is outside the vocabulary"):
        T.synchronize()
    # what is left: as if they were not there
    idx[2, 1] = idx[4, 0] = -1
    _, dz, _, bz = R.distillation(z, idx, teacher)
    assert_within(Z.grad_by_value().data(), dz, bz, "dz")
    T.clear_gradients()


def test_distillation_over_a_caller_s_memory_at_any_address():
    for rows, vocab in ((12, 4999), (140, 4999), (30, 1), (30, 2), (31, 3), (30, 5), (25, 31), (25, 33), (33, 993), (9, 1000), (9, 4065),
                        (10, 8161), (140, 16353), (140, 32737), (140, 32736), (131, 65505), (3, 61441), (3, 61409)):
        for offset in (1, 2, 3, 5, 30):
            check_at_an_address(rows, vocab, offset)


def check_at_an_address(rows, vocab, offset):
    z, idx, teacher, labels, w = distill_case(rows, vocab, 9)
    z[7::9, 0] = 0.0
    Z = T.Tensor.from_device(DeviceArray(z, offset)).with_requires_grad()
    loss = Z.distillation(T.Indices.from_device(IndexArray(idx, 1)), T.Tensor.from_device(DeviceArray(teacher, 3)), 1.5,
                          T.Indices.from_device(IndexArray(labels, 2)), 0.5, T.Tensor.from_device(DeviceArray(w, 1)))
    want, dz, bound, bz = R.distillation(z, idx, teacher, 1.5, labels, 0.5, w)
    assert_within(loss.data(), np.array([want]), bound, "loss")
    loss.backward()
    assert_within(Z.grad_by_value().data(), dz, bz, "dz")
    T.clear_gradients()


def test_indices_are_in_one_allocation():
    with pytest.raises(T.TsError, match="one allocation"):
        far = IndexArray(np.zeros((3, 4), np.int32))
        far.__cuda_array_interface__["shape"] = (1 << 30,)
        T.Indices.from_device(far)


def test_distillation_of_far_logits():
    """Logits of 1e30, and all of them the type's lowest: nothing leaves fp32 on the way."""
    low = np.finfo(np.float32).min
    for rows, vocab in ((4, 600), (4, 60000), (4, 6000), (140, 6000)):
        z = np.full((rows, vocab), low, np.float32)
        z[1] = 1e30
        z[2, ::2] = -low
        z[3] = normal((vocab,), 1) + np.float32(1e6)
        idx, teacher = np.tile(np.array([2, 4], np.int32), (rows, 1)), np.full((rows, 2), low, np.float32)
        want, dz, bound, bz = R.distillation(z, idx, teacher, 0.5)
        Z = tensor(z).with_requires_grad()
        loss = Z.distillation(indices(idx), tensor(teacher), 0.5)
        loss.backward()
        assert_within(Z.grad_by_value().data(), dz, bz, "dz")
        assert_within(loss.data(), np.array([want]), bound, "loss")
        T.clear_gradients()


def test_distillation_entry_by_itself():
    """The C entry with a device gradient of the loss, by one launch and by two, and equal bits from equal calls."""
    ticket = Dev.of(np.zeros(1, np.float32))
    for rows, vocab in ((33, 500), (9, 60000), (20, 9000), (140, 9000), (1100, 4200)):
        z, idx, teacher, labels, w = distill_case(rows, vocab, 11)
        z[7::9, 0] = 0.0
        dev = [Dev.of(z), Dev.of(idx.view(np.float32)), Dev.of(teacher), Dev.of(labels.view(np.float32)), Dev.of(w),
               Dev.of(np.array([3.0], np.float32))]
        floats, bad, got = hip.ts_hip_distillation_workspace_floats(rows, vocab), ZeroIndex(), []
        work = Dev(floats)
        for one in (None, ticket.ptr, ticket.ptr, None):
            loss, out = Dev(1), Dev(rows * vocab + 2)
            out.put(np.full(rows * vocab + 2, 7.0, np.float32))
            hip_check(hip.ts_hip_distillation(dev[0].ptr, rows, vocab, dev[1].ptr, dev[2].ptr, 11, 2.0, dev[3].ptr, 0.5, dev[4].ptr,
                                              dev[5].ptr, loss.ptr, out.ptr, bad.ptr, work.ptr, floats, one, None))
            got.append((loss.get(), out.get()))
        want, dz, bound, bz = R.distillation(z, idx, teacher, 2.0, labels, 0.5, w)
        assert_within(got[0][0], np.array([want]), bound, "loss")
        assert_within(got[0][1][:-2].reshape(rows, vocab), 3 * dz, 3 * bz + 2 * R.U * np.abs(3 * dz), "dz")
        assert np.all(got[0][1][-2:] == 7.0) and bad.value() is None
        assert not ticket.get().view(np.uint32).any()
        assert all(np.array_equal(g[1], got[0][1]) for g in got) and got[1][0] == got[2][0] and got[3][0] == got[0][0]
        assert abs(got[1][0] - got[0][0]) <= 2 * R.U * abs(want)  # (the parts in another order of f64 sums)


@pytest.mark.parametrize("rows,vocab", [(33, 500), (40, 9000), (9, 60000)])
def test_distillation_entry_has_its_loss_where_its_gradient_is_held_back(rows, vocab):
    z, idx, teacher, labels, w = distill_case(rows, vocab, 11)
    z[7::9, 0] = 0.0
    dev = [Dev.of(z), Dev.of(idx.view(np.float32)), Dev.of(teacher), Dev.of(labels.view(np.float32)), Dev.of(w),
           Dev.of(np.zeros(1, np.float32))]
    floats, bad = hip.ts_hip_distillation_workspace_floats(rows, vocab), ZeroIndex()
    work, loss, out = Dev(floats), Dev(1), Dev(rows * vocab)
    out.put(np.full(rows * vocab, 7.0, np.float32))
    hip_check(hip.ts_hip_distillation(dev[0].ptr, rows, vocab, dev[1].ptr, dev[2].ptr, 11, 2.0, dev[3].ptr, 0.5, dev[4].ptr,
                                      dev[5].ptr, loss.ptr, out.ptr, bad.ptr, work.ptr, floats, None, None))
    want, _, bound, _ = R.distillation(z, idx, teacher, 2.0, labels, 0.5, w)
    assert_within(loss.get(), np.array([want]), bound, "loss")
    assert not out.get().any()


# ---- together ---------------------------------------------------------------------------


def student(d, f, vocab):
    """A block and a head: norm weights and biases, two layers, the head."""
    return [tensor(a).with_requires_grad() for a in (
        1 + 0.1 * normal((d,), 1), 0.1 * normal((d,), 2), normal((d, f), 3, d ** -0.5), normal((f, d), 4, f ** -0.5),
        1 + 0.1 * normal((d,), 5), 0.1 * normal((d,), 6), normal((d, vocab), 7, d ** -0.5))]


def logits_of(ps, x, r):
    g1, b1, w1, w2, g2, b2, head = ps
    y, h = x.add_layer_norm(r, g1, b1)
    y, _ = y.linear(w1, activation="silu").linear(w2).add_layer_norm(h, g2, b2)
    return y.linear(head)


def student_step(ps, opt, x, r, lists):
    loss = logits_of(ps, x, r).distillation(*lists)
    loss.backward()
    opt.step(ps)
    opt.zero_grad(ps)
    T.clear_gradients()
    return loss


@pytest.mark.parametrize("batch,d,f,vocab", [(6, 40, 56, 90), (150, 256, 300, 5003), (4, 64, 96, 50000)])
def test_a_student_trains_and_replays_as_it_runs(batch, d, f, vocab):
    """A student's step recorded and replayed, with eager work between the replays, has the eager steps' bits."""
    _, idx, teacher, labels, w = distill_case(batch, vocab, 5)
    lists = (indices(idx), tensor(teacher), 2.0, indices(labels), 0.3, tensor(w))
    x, r = tensor(normal((batch, d), 8)), tensor(normal((batch, d), 9))
    eager, opt = student(d, f, vocab), T.Adam.with_learning_rate(1e-3)
    opt.add_parameters(eager)
    losses = [student_step(eager, opt, x, r, lists).value() for _ in range(7)]
    assert all(np.isfinite(losses))
    ps, opt2 = student(d, f, vocab), T.Adam.with_learning_rate(1e-3)
    opt2.add_parameters(ps)
    student_step(ps, opt2, x, r, lists)
    with T.StepGraph.record() as g:
        kept = student_step(ps, opt2, x, r, lists)
    for n, at in ((1, 1), (2, 3), (1, 4)):
        g.replay(n)
        T.synchronize()
        assert kept.value() == np.float32(losses[at])
        logits_of(ps, x, r).distillation(*lists).value()
        T.clear_gradients()
    student_step(ps, opt2, x, r, lists)
    student_step(ps, opt2, x, r, lists)
    for a, b in zip(eager, ps):
        assert np.array_equal(a.data(), b.data())
    g.free()


def test_a_student_s_gradients_are_the_plain_ones():
    batch, d, f, vocab = 9, 24, 32, 50
    z, idx, teacher, labels, w = distill_case(batch, vocab, 5)
    ps = student(d, f, vocab)
    x, r = normal((batch, d), 8), normal((batch, d), 9)
    loss = logits_of(ps, tensor(x), tensor(r)).distillation(indices(idx), tensor(teacher), 2.0, indices(labels), 0.3, tensor(w))
    loss.backward()
    g1, b1, w1, w2, g2, b2, head = (p.data().astype(np.float64) for p in ps)
    h = x.astype(np.float64) + r
    y1 = R.layer_norm(h, g1, b1, EPS)
    z1 = y1 @ w1
    a1 = R.act(z1, "silu")
    h2 = a1 @ w2 + h
    y2 = R.layer_norm(h2, g2, b2, EPS)
    want, dz, _, _ = R.distillation(y2 @ head, idx, teacher, 2.0, labels, 0.3, w)
    dh2, dg2, db2 = R.layer_norm_grads(h2, g2, dz @ head.T, EPS)
    s = 1 / (1 + np.exp(-z1))
    dz1 = (dh2 @ w2.T) * s * (1 + z1 * (1 - s))
    _, dg1, db1 = R.layer_norm_grads(h, g1, dz1 @ w1.T, EPS)
    assert abs(loss.value() - want) < 1e-5 * abs(want)
    for p, g in zip(ps, (dg1, db1, y1.T @ dz1, a1.T @ dh2, dg2, db2, y2.T @ dz)):
        assert np.linalg.norm(p.grad_by_value().data() - g) < 2e-6 * np.linalg.norm(g) + 1e-9
    T.clear_gradients()


@pytest.mark.parametrize("batch,d,f,vocab", [(1, 256, 384, 1000), (5, 200, 300, 777), (300, 512, 640, 1500)])
def test_a_student_serves_in_8_bits(batch, d, f, vocab):
    """The same block from 8-bit values: each operator's output is the plain form's of what it was given."""
    g1, b1, w1, w2, g2, b2, head = (p.data() for p in student(d, f, vocab))
    x, r = normal((batch, d), 8), normal((batch, d), 9)
    weights = [tensor(np.ascontiguousarray(w.T)).block8(tiles=True) for w in (w1, w2, head)]
    values = [R.block8_values(*R.block8(np.ascontiguousarray(w.T), True), w.shape[0], True) for w in (w1, w2, head)]

    def given(p):
        return R.block8_values(*parts(p), p.shape[1])

    p, h = tensor(x).add_layer_norm_block8(tensor(r), tensor(g1), tensor(b1))
    a = p.linear(weights[0], activation="silu")
    want, bound = R.linear(given(p), values[0], None, "silu", None)
    assert_within(a.data(), want, bound, "hidden")
    q = a.block8()
    y = q.linear(weights[1], residual=h)
    want, bound = R.linear(given(q), values[1], None, "none", h.data())
    assert_within(y.data(), want, bound, "stream")
    p2 = y.layer_norm_block8(tensor(g2), tensor(b2))
    out = p2.linear(weights[2])
    want, bound = R.linear(given(p2), values[2], None, "none", None)
    assert_within(out.data(), want, bound, "logits")
    # and it is the student's, as far as 8 bits go: a code is off by 2^-4 at most, four layers' together by less than 0.15 of the rms
    full = logits_of([tensor(v) for v in (g1, b1, w1, w2, g2, b2, head)], tensor(x), tensor(r)).data()
    assert np.sqrt(np.mean((out.data() - full) ** 2)) < 0.15 * np.sqrt(np.mean(full ** 2))


def test_calls_of_two_threads_keep_their_results():
    import threading

    x, w, b = tensor(normal((130, 784), 1)), tensor(normal((784,), 2)), tensor(normal((784,), 3))
    z, idx, teacher, labels, wt = distill_case(27, 500, 4)
    z[7::9, 0] = 0.0
    lists = (tensor(z), indices(idx), tensor(teacher), 2.0, indices(labels), 0.5, tensor(wt))
    want = x.layer_norm(w, b).data(), lists[0].distillation(*lists[1:]).value()
    wrong = []

    def work():
        for _ in range(20):
            y, loss = x.layer_norm(w, b), lists[0].distillation(*lists[1:])
            if not np.array_equal(y.data(), want[0]) or loss.value() != want[1]:
                wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
