"""The operators of a pre-norm feed-forward block, each as one pass: what is
measured, its plain form in elementary torch operations, and the same from the
definitions in 64 bits.

A case is a dict of plain values whose "kind" picks the operator:

* ``norm``          h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight,
                    forward and backward (training)
* ``norm_packed``   the same forward with y in 8 bits (serving)
* ``linear``        act(x W + bias) + residual, forward and backward, from an
                    input kept in full or as its 8-bit checkpoint (training)
* ``linear_packed`` act(x W^T + bias) + residual of an input and weights in 8
                    bits (serving)

8 bits: e4m3 values with a power-of-two scale for each 32 columns of a row, the
smallest that keeps the block's largest magnitude within 448 (from 2^-117 to
2^119).  Rows are padded with zeros to a multiple of 128 columns; the scales of
128 columns, one byte each (the exponent plus 127), stand together and go row
by row: codes [rows, pitch], scales [pitch / 128, rows, 4].
"""
from __future__ import annotations

import math

import torch

own = False  # True: run() calls this framework's operators, False: the plain forms

EPS = 1e-6


def listed():
    return [
        # one row, as a served token passes a norm: launch and host time
        dict(name="norm_packed_token", kind="norm_packed", rows=1, cols=4096, residual=True),
        # a prompt's rows on their way to a product in 8 bits
        dict(name="norm_packed_rows", kind="norm_packed", rows=8192, cols=4096, residual=True),
        # no size divides anything: rows that end inside a block of 32
        dict(name="norm_packed_odd", kind="norm_packed", rows=3000, cols=1003, residual=False),
        # a small model's training step
        dict(name="norm_small", kind="norm", rows=128, cols=784, residual=True),
        # the residual stream of a wide model, memory traffic alone
        dict(name="norm_rows", kind="norm", rows=8192, cols=4096, residual=True),
        # one token through a wide layer: the weights' bytes
        dict(name="linear_packed_token", kind="linear_packed", batch=1, fan_in=4096, fan_out=4096, act="silu", bias=True,
             residual=False),
        # a ragged batch over sizes that nothing divides
        dict(name="linear_packed_odd", kind="linear_packed", batch=1999, fan_in=1531, fan_out=777, act="gelu_tanh",
             bias=True, residual=True),
        # a prompt through a wide layer: matrix products alone
        dict(name="linear_packed_rows", kind="linear_packed", batch=8192, fan_in=4096, fan_out=4096, act="none",
             bias=True, residual=True),
        # the first layer of a small classifier, its input kept in full
        dict(name="linear_small", kind="linear", batch=128, fan_in=784, fan_out=128, act="silu", bias=True,
             residual=False, checkpoint="full"),
        # one hidden layer of an ordinary network
        dict(name="linear_mid", kind="linear", batch=2048, fan_in=1024, fan_out=4096, act="silu", bias=True,
             residual=False, checkpoint="8bit"),
        # a projection back to the residual stream with sizes that nothing divides
        dict(name="linear_odd", kind="linear", batch=3000, fan_in=1003, fan_out=2050, act="none", bias=False,
             residual=True, checkpoint="8bit"),
        # a wide layer over a large batch, the largest call
        dict(name="linear_wide", kind="linear", batch=8192, fan_in=4096, fan_out=4096, act="gelu_tanh", bias=True,
             residual=True, checkpoint="8bit"),
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of lo..hi, every second one rounded to
    a multiple of 32 (16 below 64), the others as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        m = 32 if v >= 64 else 16
        v = (v + m // 2) // m * m
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["norm", "norm_packed", "linear", "linear", "linear_packed", "linear_packed"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if kind in ("norm", "norm_packed"):
        cols = _size(rng, 8, 16384)
        return dict(kind=kind, rows=_size(rng, 1, min(16384, (1 << 25) // cols)), cols=cols, residual=flag())
    while True:
        m, k, n = _size(rng, 1, 8192), _size(rng, 8, 8192), _size(rng, 8, 8192)
        if m * k * n <= 8192 * 4096 * 4096:
            break
    case = dict(kind=kind, batch=m, fan_in=k, fan_out=n, bias=flag(), residual=flag())
    if kind == "linear":
        return dict(case, act=rng.choice(["none", "silu", "gelu_tanh"]), checkpoint=rng.choice(["full", "8bit", "8bit"]))
    return dict(case, act=rng.choice(["none", "relu", "silu", "gelu_tanh"]))


# ---- inputs ---------------------------------------------------------------------


def _inputs(case, seed):
    """The pass's values as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale

    def stream(rows, cols):
        """A residual stream's rows: a few columns far larger than the others."""
        big = torch.rand(cols, generator=g, device="cuda") < 1 / 64
        return normal(rows, cols) * torch.where(big, 20.0, 1.0)

    if case["kind"] in ("norm", "norm_packed"):
        r, c = case["rows"], case["cols"]
        d = dict(x=normal(r, c), weight=1 + normal(c, scale=0.2))
        if case["residual"]:
            d["residual"] = stream(r, c)
        if case["kind"] == "norm":
            d["go"] = normal(r, c)
        return d
    m, k, n = case["batch"], case["fan_in"], case["fan_out"]
    if case["kind"] == "linear":
        d = dict(x=normal(m, k), weight=normal(k, n, scale=k ** -0.5), go=normal(m, n, scale=1 / m))
    else:
        d = dict(zip(("xc", "xs"), _pack_inputs(stream(m, k))))
        d.update(zip(("wc", "ws"), _pack_inputs(normal(n, k, scale=k ** -0.5))))
    if case["bias"]:
        d["bias"] = normal(n, scale=0.1)
    if case["residual"]:
        d["residual"] = normal(m, n)
    return d


def _blocks(v):
    """Rows padded with zeros to whole groups of 128 columns, as [rows, blocks, 32]."""
    rows, cols = v.shape
    out = torch.zeros(rows, (cols + 127) // 128 * 128, dtype=v.dtype, device=v.device)
    out[:, :cols] = v
    return out.view(rows, -1, 32)


def _by_group(scale):
    """[rows, blocks] as the scales stand: [blocks / 4, rows, 4]."""
    return scale.view(scale.shape[0], -1, 4).transpose(0, 1).contiguous()


def _pow2(k):
    """2^k in 64 bits, exactly (exp2, pow and ldexp round on the GPU)."""
    return (k.to(torch.int64) + 1023 << 52).view(torch.float64)


def _pack_inputs(x):
    """What packing gave earlier: codes and scale exponents in bytes."""
    b = _blocks(x)
    m, e = torch.frexp(b.abs().amax(2))
    k = torch.where(m > 0, e - torch.where(m <= 0.875, 9, 8), -117).clamp(-117, 119)
    codes = (b * _pow2(-k).float()[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(x.shape[0], -1), _by_group((k + 127).to(torch.uint8))


class _Span:
    """What torch needs to read a device buffer of the framework in place."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner  # kept: the buffer is its
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


def _view(t):
    return torch.as_tensor(_Span(t, t.device_ptr(), t.shape, "<f4"), device="cuda")


def _packed_view(p):
    rows, pitch = p.shape[0], p.pitch
    codes = torch.as_tensor(_Span(p, p.codes_ptr(), (rows, pitch), "|u1"), device="cuda")
    scales = torch.as_tensor(_Span(p, p.scales_ptr(), (pitch // 128, rows, 4), "|u1"), device="cuda")
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # handles on the same memory
        import train_station_amd as T

        torch.cuda.current_stream().synchronize()
        h = {k: T.Tensor.from_device(v) for k, v in s.items() if v.dtype == torch.float32}
        if case["kind"] == "linear_packed":
            h["x"] = T.Packed8.from_device(s["xc"], s["xs"], case["fan_in"])
            h["weight"] = T.Packed8.from_device(s["wc"], s["ws"], case["fan_in"])
        if case["kind"] in ("norm", "linear"):
            for k in ("x", "weight", "bias", "residual"):
                if k in h:
                    h[k].with_requires_grad()
        s["own"] = h
    s["case"] = case
    return s


# ---- one pass with the framework's operators ----------------------------------------
# A pass is queued on the library's own stream, as a program's next call follows
# it there.  The tensors returned are views of the library's buffers: read them
# after torch.cuda.synchronize() (or on the library's stream), and before they are
# let go, since the next pass may then write their memory.


def _run_own(s):
    import train_station_amd as T

    case, h = s["case"], s["own"]
    kind, r, b = case["kind"], h.get("residual"), h.get("bias")
    if kind == "norm_packed":
        if r is None:
            return _packed_view(h["x"].rms_norm_packed(h["weight"], EPS))
        packed, stream = h["x"].add_rms_norm_packed(r, h["weight"], EPS)
        return dict(_packed_view(packed), h=_view(stream))
    if kind == "linear_packed":
        return _view(h["x"].linear(h["weight"], bias=b, activation=case["act"], residual=r))
    out = {}
    if kind == "norm":
        if r is None:
            y = h["x"].rms_norm(h["weight"], EPS)
        else:
            y, stream = h["x"].add_rms_norm(r, h["weight"], EPS)
            out["h"] = _view(stream)
    else:
        y = h["x"].linear(h["weight"], bias=b, activation=case["act"], residual=r, checkpoint=case["checkpoint"])
    y.backward(h["go"])
    out["y"] = _view(y)
    for k in ("x", "weight", "bias", "residual"):
        if k in h:
            out["d" + k] = _view(h[k].grad_view())
            h[k].zero_grad()
    T.clear_gradients()
    return out


# ---- the plain forms -----------------------------------------------------------------


def _pack_plain(y):
    """64-bit rows to 8 bits: (codes, scales) as the values they stand for."""
    b = _blocks(y)
    need = b.abs().amax(2) / 448
    k = torch.ceil(torch.log2(need)).nan_to_num(neginf=-117.0).clamp(-117, 119)
    k = torch.where(_pow2(k - 1) >= need, k - 1, torch.where(_pow2(k) < need, k + 1, k)).clamp(-117, 119)
    q = b * _pow2(-k)[:, :, None]
    step = _pow2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    q = (torch.round(q / step) * step).clamp(-448, 448)
    return {"codes": q.view(y.shape[0], -1).to(torch.float8_e4m3fn),
            "scales": (_by_group(k) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)}


def _values(codes, scales, cols):
    """The 32-bit values that codes and scale bytes stand for."""
    v = codes.view(torch.float8_e4m3fn).to(torch.float32).view(codes.shape[0], -1, 32)
    k = scales.transpose(0, 1).reshape(codes.shape[0], -1).to(torch.int32) - 127
    return (v * _pow2(k).float()[:, :, None]).view(codes.shape[0], -1)[:, :cols]


def _checkpoint(x):
    """x as its 8-bit checkpoint gives it back."""
    b = _blocks(x)
    need = b.abs().amax(2) / 448  # (the quotient's rounding never crosses a power of two: 448 is 7 of them)
    k = torch.ceil(torch.log2(need.double())).nan_to_num(neginf=-117.0).clamp(-117, 119)
    q = b * _pow2(-k).float()[:, :, None]
    step = _pow2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6).double())) - 3).float()
    q = (torch.round(q / step) * step).clamp(-448, 448)
    return (q * _pow2(k).float()[:, :, None]).view(x.shape[0], -1)[:, : x.shape[1]].contiguous()


_G1, _G2 = 2 * math.sqrt(2 / math.pi), 0.044715


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    v = z if act == "silu" else _G1 * (z + _G2 * z * z * z)
    return z / (1 + torch.exp(-v))


def _act_slope(z, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    s = 1 / (1 + torch.exp(-_G1 * (z + _G2 * z * z * z)))
    return s + z * s * (1 - s) * (_G1 * (1 + 3 * _G2 * z * z))


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind, r, b = case["kind"], s.get("residual"), s.get("bias")
    if kind in ("norm", "norm_packed"):
        h = s["x"] if r is None else s["x"] + r
        stream = {} if r is None else {"h": h}
        if kind == "norm_packed":  # 64 bits: a rounding to 8 takes either side of a border
            d = h.double()
            y = d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) * s["weight"].double()
            return dict(_pack_plain(y), **stream)
        scale = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        unit = h * scale
        gw = s["go"] * s["weight"]
        dx = scale * (gw - unit * (gw * unit).mean(1, keepdim=True))
        out = dict(y=unit * s["weight"], dx=dx, dweight=(s["go"] * unit).sum(0), **stream)
        return out if r is None else dict(out, dresidual=dx)
    if kind == "linear_packed":
        z = _values(s["xc"], s["xs"], case["fan_in"]) @ _values(s["wc"], s["ws"], case["fan_in"]).t()
        z = z if b is None else z + b
        y = _act(z, case["act"])
        return y if r is None else y + r
    x, w, go = s["x"], s["weight"], s["go"]
    z = x @ w if b is None else x @ w + b
    y = _act(z, case["act"])
    kept = _checkpoint(x) if case["checkpoint"] == "8bit" else x
    dz = go
    if case["act"] != "none":
        if case["checkpoint"] == "8bit":  # the layer once more, from what was kept
            z = kept @ w if b is None else kept @ w + b
        dz = go * _act_slope(z, case["act"])
    out = dict(y=y if r is None else y + r, dx=dz @ w.t(), dweight=kept.t() @ dz)
    if b is not None:
        out["dbias"] = dz.sum(0)
    if r is not None:
        out["dresidual"] = go
    return out


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_packed"):
        n, c = case["rows"] * case["cols"], case["cols"]
        add = 1 if case["residual"] else 0
        if kind == "norm_packed":  # x, residual read; h and 1 1/32 bytes a value written
            return dict(bytes=4 * n * (1 + 2 * add) + n * 33 / 32 + 4 * c, flops=6 * n)
        # x, residual, go read; y, h and one gradient written
        return dict(bytes=4 * n * (4 + 2 * add) + 12 * c, flops=16 * n)
    m, k, n = case["batch"], case["fan_in"], case["fan_out"]
    bias, res = (n if case["bias"] else 0), (m * n if case["residual"] else 0)
    if kind == "linear_packed":
        return dict(bytes=(m + n) * k * 33 / 32 + 4 * (m * n + bias + res), flops=2 * m * k * n)
    products = 4 if case["checkpoint"] == "8bit" and case["act"] != "none" else 3
    return dict(bytes=4 * (2 * m * k + 2 * k * n + 2 * m * n + 2 * bias + res), flops=2 * products * m * k * n)


# ---- the same in 64 bits ---------------------------------------------------------------


def _two_to(k):
    """2^k for whole k, from a table of exact values."""
    return torch.tensor([2.0 ** i for i in range(-1000, 1001)], dtype=torch.float64, device=k.device)[k.long() + 1000]


def _round8(y):
    """64-bit values to 8 bits: the quotients by their block's scale, rounded, and the scales' exponents."""
    b = _blocks(y)
    mant, e = torch.frexp(b.abs().amax(2))  # largest = mant 2^e, mant in [1/2, 1); 448 = 7/8 2^9
    k = torch.where(mant > 0, torch.where(mant > 7 / 8, e - 8, e - 9), -117).clamp(-117, 119)
    q = b * _two_to(-k)[:, :, None]
    _, qe = torch.frexp(q)
    unit = torch.where(q == 0, -5, qe).clamp(min=-5) - 4  # four significant bits, none below 2^-9
    q = torch.round(q * _two_to(-unit)) * _two_to(unit)
    return torch.clamp(q, -448, 448), k


def exact(case, seed):
    v = {k: (x.double() if x.dtype == torch.float32 else x) for k, x in _inputs(case, seed).items()}
    kind, r, b = case["kind"], v.get("residual"), v.get("bias")
    if kind in ("norm", "norm_packed"):
        # the stream is kept in 32 bits and normalised as it is kept
        h = v["x"] if r is None else (v["x"] + r).float().double()
        if kind == "norm":
            h.requires_grad_(True)
            v["weight"].requires_grad_(True)
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * v["weight"]
        out = {} if r is None else {"h": h.detach()}
        if kind == "norm_packed":
            q, k = _round8(y)
            return dict(out, codes=q.view(q.shape[0], -1), scales=_by_group(_two_to(k)))
        y.backward(v["go"])
        out.update(y=y.detach(), dx=h.grad, dweight=v["weight"].grad)
        return out if r is None else dict(out, dresidual=h.grad)
    act = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
           "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]

    def layer(x, w):
        z = act(x @ w + (0 if b is None else b))
        return z if r is None else z + r

    if kind == "linear_packed":
        def wide(codes, scales):
            q = codes.view(torch.float8_e4m3fn).double().view(codes.shape[0], -1, 32)
            k = scales.permute(1, 0, 2).reshape(codes.shape[0], -1, 1).int() - 127
            return (q * _two_to(k)).view(codes.shape[0], -1)

        return layer(wide(v["xc"], v["xs"]), wide(v["wc"], v["ws"]).t().contiguous())
    x, w, m = v["x"], v["weight"], case["batch"]
    kept = x
    if case["checkpoint"] == "8bit":
        q, k = _round8(x)
        kept = (q * _two_to(k)[:, :, None]).view(m, -1)[:, : case["fan_in"]].contiguous()
    y = layer(x, w)
    leaves = {"dx": kept.requires_grad_(True), "dweight": w.requires_grad_(True)}
    if b is not None:
        leaves["dbias"] = b.requires_grad_(True)
    if r is not None:
        leaves["dresidual"] = r.requires_grad_(True)
    layer(kept, w).backward(v["go"])
    return dict({k: t.grad for k, t in leaves.items()}, y=y.detach())
