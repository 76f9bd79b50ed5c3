"""The operators that train a student from a larger teacher and serve it in 8 bits,
each as one pass: what is measured, its plain form in elementary torch
operations, and the same from the definitions in 64 bits.

A case is a dict of plain values whose "kind" picks the operator:

* ``layer_norm``         h = x + residual; y = (h - mean(h)) / sqrt(var(h) + eps) *
                         weight + bias over the rows, forward and backward (training)
* ``layer_norm_block8``  the same forward with y in 8 bits (serving)
* ``block8_linear``      act(x W^T + bias) + residual of an input and weights in 8
                         bits (serving)
* ``distillation``       a student's loss against a teacher's top logits and the true
                         labels, with the gradient of every logit (training)

8 bits: e4m3 codes with one 32-bit scale for each block of 128 columns, of one row
(an input) or of 128 rows (a weight): the block's largest magnitude over 448.
Rows are padded with zeros to a multiple of 128 columns:
codes [rows, pitch], scales [pitch / 128, rows or rows / 128].

The loss of logits z, a row of them at a time, T the temperature, a the share of the
labels: with q the softmax of the teacher's kept logits over T, p the softmax of all
of the row over T and s that of the row itself,
  weight ((1 - a) T^2 sum of q (log q - log p) - a log s[label]),
summed over the rows.  An entry of index -1 is none, and a row of none has no first
term; a label of -1 is none, and its row has no second term.
"""
from __future__ import annotations

import math

import torch

own = False  # True: run() calls this framework's operators, False: the plain forms

EPS = 1e-5


def listed():
    return [
        # a small model's training step
        dict(name="layer_norm_small", kind="layer_norm", rows=128, cols=784, residual=True, bias=True),
        # no size divides anything, no stream beside it
        dict(name="layer_norm_odd", kind="layer_norm", rows=3000, cols=1003, residual=False, bias=False),
        # the residual stream of a wide model, memory traffic alone
        dict(name="layer_norm_rows", kind="layer_norm", rows=8192, cols=4096, residual=True, bias=True),
        # one row, as a served token passes a norm: launch and host time
        dict(name="layer_norm_block8_token", kind="layer_norm_block8", rows=1, cols=4096, residual=True, bias=True),
        # a prompt's rows on their way to a product in 8 bits
        dict(name="layer_norm_block8_rows", kind="layer_norm_block8", rows=8192, cols=4096, residual=True, bias=True),
        # one token through a wide layer: the weights' bytes
        dict(name="block8_linear_token", kind="block8_linear", batch=1, fan_in=4096, fan_out=4096, act="silu", bias=True,
             residual=False),
        # a ragged batch over sizes that nothing divides
        dict(name="block8_linear_odd", kind="block8_linear", batch=1999, fan_in=1531, fan_out=777, act="gelu_tanh",
             bias=True, residual=True),
        # a prompt through a wide layer: matrix products alone
        dict(name="block8_linear_rows", kind="block8_linear", batch=8192, fan_in=4096, fan_out=4096, act="none",
             bias=True, residual=True),
        # a small classifier taught by a larger one that keeps a few classes a row
        dict(name="distillation_small", kind="distillation", rows=128, vocab=1000, kept=10, temperature=2.0, hard=0.5,
             ragged=False, weights=False),
        # a few positions over a large vocabulary: rows too few to fill the chip one by one
        dict(name="distillation_few", kind="distillation", rows=8, vocab=131072, kept=64, temperature=1.0, hard=0.0,
             ragged=False, weights=False),
        # a padded batch over a vocabulary that nothing divides, lists of the teacher's of several lengths
        dict(name="distillation_odd", kind="distillation", rows=999, vocab=50001, kept=50, temperature=2.0, hard=0.3,
             ragged=True, weights=True),
        # a long batch over an ordinary vocabulary, the largest call
        dict(name="distillation_rows", kind="distillation", rows=8192, vocab=32768, kept=128, temperature=1.0, hard=0.5,
             ragged=False, weights=True),
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
    kind = rng.choice(["layer_norm", "layer_norm_block8", "block8_linear", "block8_linear", "distillation", "distillation"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if kind in ("layer_norm", "layer_norm_block8"):
        cols = _size(rng, 8, 16384)
        return dict(kind=kind, rows=_size(rng, 1, min(16384, (1 << 25) // cols)), cols=cols, residual=flag(), bias=flag())
    if kind == "distillation":
        vocab = _size(rng, 10, 131072)
        return dict(kind=kind, rows=_size(rng, 1, min(8192, (1 << 28) // vocab)), vocab=vocab,
                    kept=_size(rng, 1, min(256, vocab)), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                    hard=rng.choice([0.0, 0.0, 0.3, 0.5]), ragged=flag(), weights=flag())
    while True:
        m, k, n = _size(rng, 1, 8192), _size(rng, 8, 8192), _size(rng, 8, 8192)
        if m * k * n <= 8192 * 4096 * 4096:
            break
    return dict(kind=kind, batch=m, fan_in=k, fan_out=n, act=rng.choice(["none", "relu", "silu", "gelu_tanh"]), bias=flag(),
                residual=flag())


# ---- inputs ---------------------------------------------------------------------


def _inputs(case, seed):
    """The pass's values as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale

    def stream(rows, cols):
        """A residual stream's rows: a few columns far larger than the others, and away from zero."""
        big = torch.rand(cols, generator=g, device="cuda") < 1 / 64
        return normal(rows, cols) * torch.where(big, 20.0, 1.0) + normal(cols, scale=0.5)

    kind = case["kind"]
    if kind in ("layer_norm", "layer_norm_block8"):
        r, c = case["rows"], case["cols"]
        d = dict(x=normal(r, c), weight=1 + normal(c, scale=0.2))
        if case["bias"]:
            d["bias"] = normal(c, scale=0.1)
        if case["residual"]:
            d["residual"] = stream(r, c)
        if kind == "layer_norm":
            d["go"] = normal(r, c)
        return d
    if kind == "distillation":
        r, v, k = case["rows"], case["vocab"], case["kept"]
        # the teacher's k best of a row, best first, all different; the student has learned a part of it
        start = torch.randint(v, (r, 1), generator=g, device="cuda")
        indices = (torch.randperm(v, generator=g, device="cuda")[:k] + start) % v
        teacher = 12.0 - 6 * torch.rand(r, k, generator=g, device="cuda").sort(1).values
        logits = normal(r, v, scale=2.0)
        logits.scatter_(1, indices, 0.7 * teacher + normal(r, k))
        labels = indices[:, 0].clone()
        if case["ragged"]:  # a teacher's list ends where its mass does
            length = torch.randint(1, k + 1, (r, 1), generator=g, device="cuda")
            indices = torch.where(torch.arange(k, device="cuda") < length, indices, -1)
        d = dict(logits=logits, teacher=teacher)
        if case["weights"]:  # a padded batch: its last rows hold nothing, the others share the loss
            full = max(1, r - r // 16)
            d["weights"] = torch.zeros(r, device="cuda")
            d["weights"][:full] = 1.0 / full
            indices[full:] = -1
            labels[full:] = -1
        d.update(indices=indices.int(), labels=labels.int())
        return d
    m, k, n = case["batch"], case["fan_in"], case["fan_out"]
    d = dict(zip(("xc", "xs"), _pack_inputs(stream(m, k), 1)))
    d.update(zip(("wc", "ws"), _pack_inputs(normal(n, k, scale=k ** -0.5), 128)))
    if case["bias"]:
        d["bias"] = normal(n, scale=0.1)
    if case["residual"]:
        d["residual"] = normal(m, n)
    return d


def _blocks(v, high=1):
    """A matrix in blocks of `high` rows and 128 columns, padded with zeros: [row blocks, high, column blocks, 128]."""
    rows, cols = v.shape
    out = torch.zeros(-(-rows // high) * high, (cols + 127) // 128 * 128, dtype=v.dtype, device=v.device)
    out[:rows, :cols] = v
    return out.view(out.shape[0] // high, high, -1, 128)


def _pow2(k):
    """2^k in 64 bits, exactly (exp2, pow and ldexp round on the GPU)."""
    return (k.to(torch.int64) + 1023 << 52).view(torch.float64)


def _pack_inputs(x, high):
    """What packing gave earlier: codes, and a scale for each 128 columns of `high` rows."""
    b = _blocks(x, high)
    scale = b.abs().amax((1, 3)).clamp(min=2.0 ** -100) / 448
    codes = (b * (1 / scale)[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(b.shape[0] * high, -1)[: x.shape[0]].contiguous(), scale.t().contiguous()


class _Span:
    """What torch needs to read a device buffer of the framework in place."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner  # kept: the buffer is its
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


def _view(t):
    return torch.as_tensor(_Span(t, t.device_ptr(), t.shape, "<f4"), device="cuda")


def _block8_view(p):
    rows, pitch = p.shape[0], p.pitch
    codes = torch.as_tensor(_Span(p, p.codes_ptr(), (rows, pitch), "|u1"), device="cuda")
    scales = torch.as_tensor(_Span(p, p.scales_ptr(), (pitch // 128, rows), "<f4"), device="cuda")
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # handles on the same memory
        import train_station_amd as T

        torch.cuda.current_stream().synchronize()
        h = {k: T.Tensor.from_device(v) for k, v in s.items() if v.dtype == torch.float32 and k not in ("xs", "ws")}
        if case["kind"] == "block8_linear":
            h["x"] = T.Block8.from_device(s["xc"], s["xs"], case["fan_in"])
            h["weight"] = T.Block8.from_device(s["wc"], s["ws"], case["fan_in"], tiles=True)
        if case["kind"] == "distillation":
            h["indices"] = T.Indices.from_device(s["indices"])
            h["labels"] = T.Indices.from_device(s["labels"])
        for k in {"layer_norm": ("x", "weight", "bias", "residual"), "distillation": ("logits",)}.get(case["kind"], ()):
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
    if kind == "layer_norm_block8":
        if r is None:
            return _block8_view(h["x"].layer_norm_block8(h["weight"], b, EPS))
        packed, stream = h["x"].add_layer_norm_block8(r, h["weight"], b, EPS)
        return dict(_block8_view(packed), h=_view(stream))
    if kind == "block8_linear":
        return _view(h["x"].linear(h["weight"], bias=b, activation=case["act"], residual=r))
    out = {}
    if kind == "distillation":
        labels = h["labels"] if case["hard"] else None
        y = h["logits"].distillation(h["indices"], h["teacher"], temperature=case["temperature"], labels=labels,
                                     hard=case["hard"], weights=h.get("weights"))
        y.backward()
        out["loss"] = _view(y)
    else:
        if r is None:
            y = h["x"].layer_norm(h["weight"], b, EPS)
        else:
            y, stream = h["x"].add_layer_norm(r, h["weight"], b, EPS)
            out["h"] = _view(stream)
        y.backward(h["go"])
        out["y"] = _view(y)
    for k in ("x", "weight", "bias", "residual", "logits"):
        if k in h:
            out["d" + k] = _view(h[k].grad_view())
            h[k].zero_grad()
    T.clear_gradients()
    return out


# ---- the plain forms -----------------------------------------------------------------


def _block8_plain(y):
    """64-bit rows to 8 bits: (codes, scales) as the values they stand for."""
    b = _blocks(y)
    scale = b.abs().amax((1, 3)).clamp(min=2.0 ** -100) / 448
    q = b / scale[:, None, :, None]
    step = _pow2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    q = (torch.round(q / step) * step).clamp(-448, 448)
    return {"codes": q.view(y.shape[0], -1).to(torch.float8_e4m3fn), "scales": scale.t().contiguous().float()}


def _values(codes, scales, cols, high):
    """The 32-bit values that codes and scales stand for."""
    rows = codes.shape[0]
    by = scales.t().repeat_interleave(high, 0)[:rows]
    return (codes.view(torch.float8_e4m3fn).to(torch.float32).view(rows, -1, 128) * by[:, :, None]).view(rows, -1)[:, :cols]


_G1, _G2 = 2 * math.sqrt(2 / math.pi), 0.044715


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    v = z if act == "silu" else _G1 * (z + _G2 * z * z * z)
    return z / (1 + torch.exp(-v))


def _distillation_plain(case, s):
    z, idx, t, a = s["logits"], s["indices"].long(), case["temperature"], case["hard"]
    rows = z.shape[0]
    w = s["weights"] if "weights" in s else torch.full((rows,), 1.0 / rows, device=z.device)
    live = idx >= 0
    at = idx.clamp(min=0)
    top = torch.where(live, s["teacher"], float("-inf"))
    best = top.amax(1, keepdim=True)
    e = torch.exp((top - torch.where(live.any(1, keepdim=True), best, torch.zeros_like(best))) / t)
    q = e / torch.where(live.any(1, keepdim=True), e.sum(1, keepdim=True), torch.ones_like(best))
    m = z.amax(1, keepdim=True)
    d = (z - m) / t
    p = torch.exp(d)
    total = p.sum(1, keepdim=True)
    p = p / total
    log_p = torch.gather(d, 1, at) - torch.log(total)
    loss = (1 - a) * t * t * torch.where(q > 0, q * (torch.log(q) - log_p), torch.zeros_like(q)).sum(1)
    soft = (1 - a) * t * w * live.any(1)
    grad = soft[:, None] * p
    grad.scatter_add_(1, at, -soft[:, None] * q)
    if a:
        label = s["labels"].long()
        has = label >= 0
        at = label.clamp(min=0)[:, None]
        if t != 1:
            d = z - m
            p = torch.exp(d)
            total = p.sum(1, keepdim=True)
            p = p / total
        loss = loss + torch.where(has, a * (torch.log(total) - torch.gather(d, 1, at))[:, 0], torch.zeros_like(w))
        hard = a * w * has
        grad += hard[:, None] * p
        grad.scatter_add_(1, at, -hard[:, None])
    return {"loss": (w * loss).sum().reshape(1), "dlogits": grad}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind, r, b = case["kind"], s.get("residual"), s.get("bias")
    if kind == "distillation":
        return _distillation_plain(case, s)
    if kind == "block8_linear":
        z = _values(s["xc"], s["xs"], case["fan_in"], 1) @ _values(s["wc"], s["ws"], case["fan_in"], 128).t()
        z = z if b is None else z + b
        y = _act(z, case["act"])
        return y if r is None else y + r
    h = s["x"] if r is None else s["x"] + r
    stream = {} if r is None else {"h": h}
    if kind == "layer_norm_block8":  # 64 bits: a rounding to 8 takes either side of a border
        d = h.double()
        d = d - d.mean(1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) * s["weight"].double()
        return dict(_block8_plain(y if b is None else y + b.double()), **stream)
    d = h - h.mean(1, keepdim=True)
    scale = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    unit = d * scale
    y = unit * s["weight"]
    gw = s["go"] * s["weight"]
    dx = scale * (gw - gw.mean(1, keepdim=True) - unit * (gw * unit).mean(1, keepdim=True))
    out = dict(y=y if b is None else y + b, dx=dx, dweight=(s["go"] * unit).sum(0), **stream)
    if b is not None:
        out["dbias"] = s["go"].sum(0)
    return out if r is None else dict(out, dresidual=dx)


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("layer_norm", "layer_norm_block8"):
        n, c = case["rows"] * case["cols"], case["cols"]
        add, bias = 1 if case["residual"] else 0, 1 if case["bias"] else 0
        if kind == "layer_norm_block8":  # x, residual read; h, a byte a value and 4 for each 128 written
            return dict(bytes=4 * n * (1 + 2 * add) + n * 33 / 32 + 4 * c * (1 + bias), flops=9 * n)
        # x, residual, go read; y, h and one gradient written
        return dict(bytes=4 * n * (4 + 2 * add) + 8 * c * (1 + bias) + 4 * c, flops=24 * n)
    if kind == "distillation":
        n, r = case["rows"] * case["vocab"], case["rows"]
        softmaxes = 2 if case["hard"] and case["temperature"] != 1 else 1
        # logits read, their gradients written; the lists, labels and weights
        return dict(bytes=8 * n + 8 * r * case["kept"] + 8 * r, flops=8 * n * softmaxes)
    m, k, n = case["batch"], case["fan_in"], case["fan_out"]
    bias, res = (n if case["bias"] else 0), (m * n if case["residual"] else 0)
    return dict(bytes=m * k * 33 / 32 + n * k + 4 * (m * n + bias + res), flops=2 * m * k * n)


# ---- the same in 64 bits ---------------------------------------------------------------


def _round8(y):
    """64-bit rows to 8 bits: the quotients by their block's scale, rounded, and the scales."""
    b = _blocks(y)
    scale = b.abs().amax((1, 3)).clamp(min=2.0 ** -100) / 448
    q = b / scale[:, None, :, None]
    _, e = torch.frexp(q)
    e = torch.where(q == 0, -5, e).clamp(min=-5) - 4  # four significant bits, none below 2^-9
    unit = torch.tensor([2.0 ** i for i in range(-9, 12)], dtype=torch.float64, device=q.device)[e.long() + 9]
    return torch.clamp(torch.round(q / unit) * unit, -448, 448).view(y.shape[0], -1), scale.t()


def _distillation_exact(case, v):
    z, t, a = v["logits"].requires_grad_(True), case["temperature"], case["hard"]
    rows, idx = z.shape[0], v["indices"].long()
    w = v["weights"] if "weights" in v else torch.full((rows,), 1.0 / rows, device=z.device, dtype=torch.float64)
    some = (idx >= 0).any(1)
    q = torch.zeros_like(v["teacher"])
    q[some] = torch.softmax((v["teacher"] / t).masked_fill(idx < 0, float("-inf"))[some], 1)
    log_p = torch.log_softmax(z / t, 1).gather(1, idx.clamp(min=0))
    loss = (1 - a) * t * t * (w * (torch.xlogy(q, q) - q * log_p).sum(1)).sum()
    if a:
        kept = v["labels"] >= 0
        picked = torch.log_softmax(z, 1).gather(1, v["labels"].long().clamp(min=0)[:, None])[:, 0]
        loss = loss - a * (w * picked)[kept].sum()
    loss.backward()
    return {"loss": loss.detach().reshape(1), "dlogits": z.grad}


def exact(case, seed):
    v = {k: (x.double() if x.dtype == torch.float32 else x) for k, x in _inputs(case, seed).items()}
    kind, r, b = case["kind"], v.get("residual"), v.get("bias")
    if kind == "distillation":
        return _distillation_exact(case, v)
    if kind == "block8_linear":
        def wide(codes, scales, high):
            q = codes.view(torch.float8_e4m3fn).double()
            by = torch.arange(q.shape[0], device=q.device) // high
            return q * scales[:, by].t().repeat_interleave(128, 1)

        act = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
               "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]
        z = act(wide(v["xc"], v["xs"], 1) @ wide(v["wc"], v["ws"], 128).t().contiguous() + (0 if b is None else b))
        return z if r is None else z + r
    # the stream is kept in 32 bits and normalised as it is kept
    h = v["x"] if r is None else (v["x"] + r).float().double()
    if kind == "layer_norm":
        leaves = {"dx": h, "dweight": v["weight"], "dbias": b}
        leaves = {k: t.requires_grad_(True) for k, t in leaves.items() if t is not None}
    var, mean = torch.var_mean(h, 1, unbiased=False, keepdim=True)
    y = (h - mean) * torch.rsqrt(var + EPS) * v["weight"] + (0 if b is None else b)
    out = {} if r is None else {"h": h.detach()}
    if kind == "layer_norm_block8":
        q, scale = _round8(y)
        return dict(out, codes=q, scales=scale)
    y.backward(v["go"])
    out.update({k: t.grad for k, t in leaves.items()}, y=y.detach())
    return out if r is None else dict(out, dresidual=h.grad)
