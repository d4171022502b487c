"""The feed-forward half of a decoder block as timed cases: RMS norm with the
residual's addition, products of 8-bit matrices, and gated feed-forward layers
in fp32 (with their gradient) and in 8 bits.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU from
the seed alone, ``run`` is one pass, in elementary torch operations or, where
``own`` is true, by the C ABI's entry points on the same buffers.  ``exact``
gives the same results in float64, ``work`` the bytes and operations that a
pass cannot do without (each input read once, each output written once).

An 8-bit matrix (rows, cols) is held in groups of 128 neighbouring elements of
a row: E4M3 numbers that share one scale 2^e, held as the byte e + 127.  e is
the smallest number with amax <= 448 * 2^e, at least -119; elements are rounded
to the nearest number, ties to the even one; a group of zeros has the byte 127.
Codes lie as (rows, ceil(cols / 128) * 128) bytes, zero behind a row's end, and
scales as (rows, ceil(cols / 512) * 4), 127 behind a row's last group.  Outputs
in 8 bits are returned as what they hold: codes and scales as the numbers that
torch's float8_e4m3fn and float8_e8m0fnu give them.
"""

from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # A step of a serving batch: eight tokens' sums and normed rows, for the next 8-bit product.
        dict(name="norm8_step", kind="norm8", rows=8, d=4096, residual=True),
        # A prompt's rows, an odd number of them.
        dict(name="norm8_prompt", kind="norm8", rows=8191, d=4096, residual=True),
        # The norm of a training step, in fp32, with what its backward needs.
        dict(name="norm_train", kind="norm", rows=8192, d=1024, residual=True),
        # Its gradient, with the gradient that passes the norm by added.
        dict(name="norm_grad", kind="norm_grad", rows=8192, d=1024, residual=True),
        # One token of one request: latency and the weights' bytes.
        dict(name="product8_step", kind="product8", n=1, m=4096, k=4096, bias=True, residual=True),
        # A serving batch, a wide projection.
        dict(name="product8_batch", kind="product8", n=37, m=16384, k=4096, bias=True, residual=False),
        # A prompt: a large product.
        dict(name="product8_prompt", kind="product8", n=4096, m=4096, k=4096, bias=False, residual=True),
        # A serving batch through a gated layer of an odd width.
        dict(name="gated8_step", kind="gated8", n=16, d=4096, hidden=10923, act="silu", bias=False),
        # A prompt through a gated layer.
        dict(name="gated8_prompt", kind="gated8", n=4096, d=4096, hidden=8192, act="silu", bias=True),
        # The forward pass of a training step.
        dict(name="gated_train", kind="gated", n=8192, d=1024, hidden=4096, act="gelu", bias=True),
        # The backward pass of a small layer, odd sizes.
        dict(name="gated_grad_small", kind="gated_grad", n=200, d=257, hidden=685, act="silu", bias=True),
        # The backward pass of a training step.
        dict(name="gated_grad", kind="gated_grad", n=8192, d=1024, hidden=2730, act="silu", bias=True),
    ]


# ---- drawn cases: the same ranges ----


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choices(("norm8", "norm", "norm_grad", "product8", "gated8", "gated", "gated_grad"), weights=(2, 1, 2, 4, 3, 2, 2))[0]
    if kind.startswith("norm"):
        d = 4 * _log_int(rng, 16, 4096)
        return dict(kind=kind, rows=_log_int(rng, 1, min(16384, (1 << (24 if kind == "norm_grad" else 25)) // d)), d=d,
                    residual=rng.random() < 0.7)
    few = rng.random() < 0.5
    if kind == "product8":
        k, m = _log_int(rng, 64, 16384), _log_int(rng, 64, 16384)
        n = _log_int(rng, 1, 64) if few else _log_int(rng, 65, max(65, min(8192, (1 << 36) // (k * m))))
        return dict(kind=kind, n=n, m=m, k=k, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    act, bias = rng.choice(("silu", "gelu")), rng.random() < 0.6
    if kind == "gated8":
        d, hidden = _log_int(rng, 64, 8192), _log_int(rng, 64, 16384)
        n = _log_int(rng, 1, 64) if few else _log_int(rng, 65, max(65, min(8192, (1 << 36) // (d * hidden))))
        return dict(kind=kind, n=n, d=d, hidden=hidden, act=act, bias=bias)
    d, hidden = _log_int(rng, 32, 4096), _log_int(rng, 32, 8192)
    return dict(kind=kind, n=_log_int(rng, 1, max(1, min(8192, (1 << (35 if kind == "gated" else 34)) // (d * hidden)))), d=d, hidden=hidden,
                act=act, bias=bias)


# ---- inputs ----


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise(x):
    """Codes and scales of x (rows, cols)."""
    rows, cols = x.shape
    groups, kept = -(-cols // 128), -(-cols // 512) * 4
    group = torch.zeros((rows, groups * 128), device="cuda")
    group[:, :cols] = x
    group = group.unflatten(1, (groups, 128))
    amax = group.abs().amax(-1, keepdim=True)
    # amax = f * 2^x with 1 <= f < 2: e is x - 8 where f <= 1.75, else x - 7.
    byte = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=8)
    byte = torch.where(amax > 0, byte, torch.full_like(byte, 127))
    codes = (group * ((254 - byte) << 23).view(torch.float32)).to(torch.float8_e4m3fn).view(torch.uint8).flatten(1)
    scales = torch.full((rows, kept), 127, device="cuda", dtype=torch.uint8)
    scales[:, :groups] = byte[..., 0].to(torch.uint8)
    return codes, scales


def _activations(g, rows, cols):
    """Normed rows: a few channels are far larger than the others."""
    return _normal(g, rows, cols) * torch.exp(0.5 * _normal(g, cols))


def prepare(case, seed):
    g, c = torch.Generator(device="cuda").manual_seed(int(seed)), case
    kind = c["kind"]
    st = dict(kind=kind, act=c.get("act"))
    if kind.startswith("norm"):
        rows, d = c["rows"], c["d"]
        st["x"] = _activations(g, rows, d)
        st["residual"] = _normal(g, rows, d) if c["residual"] else None
        st["gamma"], st["eps"] = 1 + 0.2 * _normal(g, d), 2.0 ** -17  # held in 32 bits as it is
        if kind == "norm_grad":
            st["dy"] = 0.1 * _normal(g, rows, d)
            st["rstd"] = (1 / torch.sqrt(st["x"].double().square().mean(-1) + st["eps"])).float()
        return st
    if kind in ("product8", "gated8"):
        k = c["k"] if kind == "product8" else c["d"]
        m = c["m"] if kind == "product8" else 2 * c["hidden"]
        st["k"], st["hidden"] = k, c.get("hidden")
        st["a"] = _quantise(_activations(g, c["n"], k))
        st["w"] = _quantise(_normal(g, m, k) / math.sqrt(k))
        st["bias"] = 0.1 * _normal(g, m) if c["bias"] else None
        st["residual"] = _normal(g, c["n"], m) if c.get("residual") else None
        return st
    n, d, hidden = c["n"], c["d"], c["hidden"]
    st["x"] = _activations(g, n, d)
    st["w"] = _normal(g, d, 2 * hidden) / math.sqrt(d)  # the gate's columns, then the other projection's
    st["bias"] = 0.1 * _normal(g, 2 * hidden) if c["bias"] else None
    if kind == "gated_grad":
        st["w_down"], st["dy"] = _normal(g, hidden, d) / math.sqrt(hidden), _normal(g, n, d)
        st["h"], st["pre"] = _plain_gated(st)  # the forward's, which a training step has
    return st


# ---- the plain forms ----


def _plain_norm(st):
    x, residual = st["x"], st["residual"]
    s = x if residual is None else x + residual
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + st["eps"])
    y = s * rstd * st["gamma"]
    return dict(y=y, rstd=rstd[:, 0], **({} if residual is None else dict(sum=s)))


def _plain_norm8(st):
    x, residual = st["x"], st["residual"]
    s = x if residual is None else x + residual
    # In 64 bits: the border between two codes is not to move with the order of a sum.
    wide = s.double()
    rstd = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + st["eps"])
    codes, scales = _quantise((wide * rstd * st["gamma"].double()).float())
    return dict(**_held(codes, scales), **({} if residual is None else dict(sum=s)))


def _plain_norm_grad(st):
    x, dy, rstd = st["x"], st["dy"], st["rstd"][:, None]
    xhat, g = x * rstd, dy * st["gamma"]
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if st["residual"] is not None:
        dx = dx + st["residual"]
    return dict(dx=dx, dgamma=(dy * xhat).sum(0))


def _held(codes, scales):
    return dict(codes=codes.view(torch.float8_e4m3fn), scales=scales.view(torch.float8_e8m0fnu))


def _values(operand, cols):
    """What codes and scales stand for, (rows, cols)."""
    codes, scales = operand
    v = codes.view(torch.float8_e4m3fn).to(torch.float32).unflatten(1, (-1, 128))
    size = (scales[:, :v.shape[1]].int() << 23).view(torch.float32)
    return (v * size[..., None]).flatten(1)[:, :cols]


def _plain_product8(st):
    y = torch.matmul(_values(st["a"], st["k"]), _values(st["w"], st["k"]).t())
    if st["bias"] is not None:
        y = y + st["bias"]
    return y if st["residual"] is None else y + st["residual"]


def _activation(act, x):
    """Its value and slope."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-x))
        return x * s, s * (1 + x * (1 - s))
    t = torch.tanh(0.8 * x)
    return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.4 * x * (1 - t * t)


def _gate(act, pre):
    gate, up = pre.chunk(2, -1)
    return _activation(act, gate)[0] * up


def _plain_gated8(st):
    pre = torch.matmul(_values(st["a"], st["k"]), _values(st["w"], st["k"]).t())
    return _held(*_quantise(_gate(st["act"], pre if st["bias"] is None else pre + st["bias"])))


def _plain_gated(st):
    pre = torch.matmul(st["x"], st["w"])
    if st["bias"] is not None:
        pre = pre + st["bias"]
    return _gate(st["act"], pre), pre


def _plain_gated_grad(st):
    x, w, dy = st["x"], st["w"], st["dy"]
    gate, up = st["pre"].chunk(2, -1)
    value, slope = _activation(st["act"], gate)
    dh = torch.matmul(dy, st["w_down"].t())
    dpre = torch.cat((dh * up * slope, dh * value), -1)
    out = dict(dx=torch.matmul(dpre, w.t()), dw=torch.matmul(x.t(), dpre), dw_down=torch.matmul(st["h"].t(), dy))
    if st["bias"] is not None:
        out["dbias"] = dpre.sum(0)
    return out


# ---- the framework's entry points ----


def _own_run(st):
    from ember_amd import capi
    L, kind = capi.lib(), st["kind"]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rows8 = lambda pair, cols: capi.Rows8View(at(pair[0]), at(pair[1]), pair[0].shape[0], cols)  # noqa: E731

    def new8(rows, cols):
        return new(rows, -(-cols // 128) * 128, dtype=torch.uint8), new(rows, -(-cols // 512) * 4, dtype=torch.uint8)

    act = dict(gelu=1, silu=2).get(st["act"], 0)
    if kind.startswith("norm"):
        x, residual, gamma = st["x"], st["residual"], st["gamma"]
        rows, d = x.shape
        if kind == "norm_grad":
            dx, dgamma = torch.empty_like(x), torch.empty_like(gamma)
            capi.check(L.rmsnorm_bwd(at(x), at(gamma), at(st["rstd"]), at(st["dy"]), at(residual), at(dx), at(dgamma), rows, d), "rmsnorm_bwd")
            return dict(dx=dx, dgamma=dgamma)
        out = {} if residual is None else dict(sum=torch.empty_like(x))
        if kind == "norm":
            y, rstd = torch.empty_like(x), new(rows)
            capi.check(L.rmsnorm_fwd(at(x), at(residual), at(gamma), at(out.get("sum")), at(y), at(rstd), rows, d, st["eps"]), "rmsnorm_fwd")
            return dict(y=y, rstd=rstd, **out)
        y = new8(rows, d)
        capi.check(L.rmsnorm_fwd8(at(x), at(residual), at(gamma), at(out.get("sum")), rows8(y, d), st["eps"]), "rmsnorm_fwd8")
        return dict(**_held(*y), **out)
    if kind == "product8":
        out = new(st["a"][0].shape[0], st["w"][0].shape[0])
        capi.check(L.linear8_fwd(rows8(st["a"], st["k"]), rows8(st["w"], st["k"]), at(st["bias"]), at(st["residual"]), at(out), 0), "linear8_fwd")
        return out
    if kind == "gated8":
        h = new8(st["a"][0].shape[0], st["hidden"])
        capi.check(L.gated8_fwd(rows8(st["a"], st["k"]), rows8(st["w"], st["k"]), at(st["bias"]), rows8(h, st["hidden"]), act), "gated8_fwd")
        return _held(*h)
    x, w = st["x"], st["w"]
    n, d, hidden = *x.shape, w.shape[1] // 2
    if kind == "gated":
        h, pre = new(n, hidden), new(n, 2 * hidden)
        capi.check(L.gated_fwd(at(x), at(w), at(st["bias"]), at(h), at(pre), n, hidden, d, act), "gated_fwd")
        return h, pre
    dpre, dy = new(n, 2 * hidden), at(st["dy"])
    out = dict(dx=new(n, d), dw=new(d, 2 * hidden), dw_down=new(hidden, d))
    capi.check(L.gated_bwd(dy, at(st["w_down"]), at(st["pre"]), at(dpre), n, hidden, d, act), "gated_bwd")
    capi.check(L.gemm_ex(at(dpre), at(w), at(out["dx"]), 1, n, d, 2 * hidden, 0, 1, None, None, None, 0), "gemm_ex")
    capi.check(L.gemm_ex(at(x), at(dpre), at(out["dw"]), 1, d, 2 * hidden, n, 1, 0, None, None, None, 0), "gemm_ex")
    capi.check(L.gemm_ex(at(st["h"]), dy, at(out["dw_down"]), 1, hidden, d, n, 1, 0, None, None, None, 0), "gemm_ex")
    if st["bias"] is not None:
        out["dbias"] = new(2 * hidden)
        capi.check(L.col_sum(at(dpre), at(out["dbias"]), n, 2 * hidden), "col_sum")
    return out


def run(st):
    if own:
        return _own_run(st)
    return dict(norm=_plain_norm, norm8=_plain_norm8, norm_grad=_plain_norm_grad, product8=_plain_product8, gated8=_plain_gated8,
                gated=_plain_gated, gated_grad=_plain_gated_grad)[st["kind"]](st)


# ---- the same in float64 ----


def _exact_values(operand, cols):
    """Decoded from the bits: sign, four bits of exponent, three of fraction."""
    codes, scales = operand[0].double(), operand[1].double()
    sign, rest = 1 - 2 * torch.floor(codes / 128), codes % 128
    exponent, fraction = torch.floor(rest / 8), rest % 8
    size = torch.where(exponent > 0, (1 + fraction / 8) * 2.0 ** (exponent - 7), fraction * 2.0 ** -9)
    return (sign * size * torch.repeat_interleave(2.0 ** (scales - 127), 128, 1)[:, :codes.shape[1]])[:, :cols]


def _exact_round(x):
    """x (rows, cols) in 8 bits: codes' values and scales, padded as they lie."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % 512)).unflatten(1, (-1, 128))
    amax = x.abs().amax(-1, keepdim=True)
    step = 2.0 ** torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448)) / 448)).clamp(min=-119)
    size = (x / step).abs()
    # Numbers of one exponent are an eighth of its power of two apart, those below 2^-6 2^-9.
    ulp = 2.0 ** (torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    codes = (torch.sign(x) * torch.round(size / ulp) * ulp).flatten(1)
    return dict(codes=codes[:, :-(-cols // 128) * 128].contiguous(), scales=step[..., 0].contiguous())


def _exact_slope(act, x):
    if act == "silu":
        return torch.sigmoid(x) + x * torch.sigmoid(x) * torch.sigmoid(-x)
    return 0.5 * (1 + torch.tanh(0.8 * x)) + 0.4 * x / torch.cosh(0.8 * x).square()


def _exact_act(act, x):
    return x * torch.sigmoid(x) if act == "silu" else x * torch.sigmoid(1.6 * x)  # (1 + tanh z) / 2 = sigmoid(2 z)


def exact(case, seed):
    st = prepare(case, seed)
    kind, act = st["kind"], st["act"]
    wide = lambda name: None if st[name] is None else st[name].double()  # noqa: E731
    if kind.startswith("norm"):
        x, residual, gamma = wide("x"), wide("residual"), wide("gamma")
        if kind == "norm_grad":
            rstd, g = wide("rstd")[:, None], wide("dy") * gamma
            dx = rstd * g - rstd.pow(3) * x * (g * x).sum(-1, keepdim=True) / x.shape[1]
            return dict(dx=dx if residual is None else dx + residual, dgamma=torch.einsum("rd,rd,r->d", wide("dy"), x, rstd[:, 0]))
        s = x if residual is None else x + residual
        if kind == "norm8" and residual is not None:
            s = s.float().double()  # the sum that is stored is the one that is normed
        out = {} if residual is None else dict(sum=s)
        norm = torch.sqrt((s * s).sum(-1) / s.shape[1] + st["eps"])
        y = s / norm[:, None] * gamma
        return dict(**_exact_round(y), **out) if kind == "norm8" else dict(y=y, rstd=1 / norm, **out)
    if kind in ("product8", "gated8"):
        y = torch.matmul(_exact_values(st["a"], st["k"]), _exact_values(st["w"], st["k"]).t().contiguous())
        y = y if st["bias"] is None else y + wide("bias")
        if kind == "product8":
            return y if st["residual"] is None else y + wide("residual")
        return _exact_round(_exact_act(act, y[:, :st["hidden"]]) * y[:, st["hidden"]:])
    x, w = wide("x"), wide("w")
    hidden = w.shape[1] // 2
    if kind == "gated":
        pre = torch.matmul(x, w)
        pre = pre if st["bias"] is None else pre + wide("bias")
        return _exact_act(act, pre[:, :hidden]) * pre[:, hidden:], pre
    # From the forward's pre and h that the call is given, as they are.
    gate, up, dy = wide("pre")[:, :hidden], wide("pre")[:, hidden:], wide("dy")
    dh = torch.matmul(dy, wide("w_down").t().contiguous())
    d_gate, d_up = dh * up * _exact_slope(act, gate), dh * _exact_act(act, gate)
    out = dict(dx=torch.matmul(d_gate, w[:, :hidden].t().contiguous()) + torch.matmul(d_up, w[:, hidden:].t().contiguous()),
               dw=torch.cat([torch.matmul(x.t().contiguous(), d) for d in (d_gate, d_up)], 1),
               dw_down=torch.matmul(wide("h").t().contiguous(), dy))
    if st["bias"] is not None:
        out["dbias"] = torch.cat((d_gate.sum(0), d_up.sum(0)))
    return out


# ---- what a pass cannot do without ----


def work(case):
    c, kind = case, case["kind"]
    if kind.startswith("norm"):
        n, more = c["rows"] * c["d"], c["residual"]
        if kind == "norm_grad":
            return dict(bytes=(16 if more else 12) * n + 4 * c["rows"] + 8 * c["d"], flops=9 * n)
        return dict(bytes=n * (4 + (8 if more else 0) + (4 if kind == "norm" else 129 / 128)) + 4 * c["d"], flops=6 * n)
    n = c["n"]
    if kind == "product8":
        m, k = c["m"], c["k"]
        return dict(bytes=(n + m) * k * 129 / 128 + 4 * n * m * (2 if c["residual"] else 1), flops=2 * n * m * k)
    d, hidden = c["d"], c["hidden"]
    if kind == "gated8":
        return dict(bytes=((n + 2 * hidden) * d + n * hidden) * 129 / 128, flops=4 * n * hidden * d)
    if kind == "gated":
        return dict(bytes=4 * (n * d + 2 * d * hidden + 3 * n * hidden), flops=4 * n * d * hidden)
    return dict(bytes=4 * (3 * n * d + 3 * n * hidden + 6 * d * hidden), flops=12 * n * d * hidden)
