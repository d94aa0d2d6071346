"""The operators of an MX-quantised feed-forward block, as measured cases.

Four operators around the quantiser and the MX GEMM: the norms of a residual stream, a GEMM with
bias, activation and residual in its epilogue, a gated feed-forward projection, and the backward
pass of its activation. ``own`` selects the library's entry points; otherwise the same results are
computed with elementary torch operations in 32 bits. ``exact`` computes them in 64 bits.

Conventions of every case: bf16 tensors are row-major; an MX tensor is one byte per element with one
UE8M0 scale per 32 elements of a row, the scales in tiles of 128 rows x 4 scale columns (512 bytes,
scale (r, s) at byte (r % 32) * 16 + (r / 32 % 4) * 4 + s % 4), rows and scale columns padded to
whole tiles with zero bytes. MX results are returned as float8 tensors, which stand for themselves.
"""

import math
import os
import sys

import torch

own = False

FMT = {"e4m3": (torch.float8_e4m3fn, 8, 448.0), "e5m2": (torch.float8_e5m2, 15, 57344.0)}


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one generated token: the norms between two blocks, feeding the next GEMM
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 8192, "post": True,
         "gate": "vector", "out": "e4m3"},
        # a prompt or a training batch through the same norms
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "cols": 8192, "post": True,
         "gate": "vector", "out": "e4m3"},
        # a ragged batch with a gate per token (a conditioned block), result kept in bf16
        {"name": "norm_ragged_bf16", "op": "norm", "rows": 1037, "cols": 5152, "post": False,
         "gate": "token", "out": "bf16"},
        # training: the gradient of the norms of a batch
        {"name": "norm_backward", "op": "norm_bwd", "rows": 8192, "cols": 4096, "post": True,
         "gate": "vector"},
        # one generated token: the down projection onto the residual stream
        {"name": "linear_token", "op": "linear", "m": 1, "n": 8192, "k": 28672, "act": "none",
         "bias": False, "residual": True, "out": "bf16", "at": "e4m3", "bt": "e4m3"},
        # a ragged batch of sequences through an ungated feed-forward layer with biases
        {"name": "linear_ragged", "op": "linear", "m": 200, "n": 4128, "k": 2080, "act": "gelu",
         "bias": True, "residual": False, "out": "e4m3", "at": "e4m3", "bt": "e4m3"},
        # a prompt or batch: the down projection, bias and residual added
        {"name": "linear_prefill", "op": "linear", "m": 4096, "n": 8192, "k": 28672,
         "act": "none", "bias": True, "residual": True, "out": "bf16", "at": "e4m3",
         "bt": "e4m3"},
        # one generated token: gate and up projections, quantised for the down projection
        {"name": "gated_token", "op": "gated", "m": 1, "f": 28672, "k": 8192, "act": "silu",
         "out": "e4m3", "save": False},
        # a small batch of generated tokens
        {"name": "gated_batch", "op": "gated", "m": 48, "f": 10240, "k": 4096,
         "act": "gelu_tanh", "out": "bf16", "save": False},
        # training, forward: the projections are kept for the backward pass
        {"name": "gated_train", "op": "gated", "m": 4096, "f": 28672, "k": 8192, "act": "silu",
         "out": "e4m3", "save": True},
        # training, backward: gradients of the block's input and of both weights, ragged batch
        {"name": "gated_backward", "op": "gated_bwd", "m": 2000, "f": 10240, "k": 4096,
         "act": "silu", "gt": "e5m2"},
        # training, backward of an ungated layer's activation, with the bias gradient
        {"name": "act_backward", "op": "act_bwd", "rows": 4096, "cols": 16384, "act": "gelu",
         "gt": "e5m2"},
    ]


def draw(rng):
    def span(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
        return int(min(hi, max(lo, step * round(v / step))))

    op = rng.choice(["norm", "norm_bwd", "linear", "linear", "gated", "gated", "gated_bwd",
                     "act_bwd"])
    if op == "norm":
        out = rng.choice(["e4m3", "e5m2", "bf16"])
        return {"op": op, "rows": span(1, 8192), "cols": span(64, 8192, 32),
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "vector", "token"]),
                "out": out}
    if op == "norm_bwd":
        return {"op": op, "rows": span(8, 8192), "cols": span(64, 4096, 32),
                "post": rng.random() < 0.5, "gate": rng.choice(["none", "vector", "token"])}
    if op == "linear":
        out = rng.choice(["bf16", "e4m3"])
        return {"op": op, "m": span(1, 4096), "n": span(128, 8192, 32 if out == "e4m3" else 8),
                "k": span(128, 16384, 32),
                "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "out": out,
                "at": rng.choice(["e4m3", "e5m2"]), "bt": "e4m3"}
    if op == "gated":
        out = rng.choice(["bf16", "e4m3"])
        return {"op": op, "m": span(1, 4096), "f": span(128, 10240, 32), "k": span(128, 8192, 32),
                "act": rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), "out": out,
                "save": rng.random() < 0.5}
    if op == "gated_bwd":
        return {"op": op, "m": span(32, 4096), "f": span(128, 8192, 32),
                "k": span(128, 4096, 32), "act": rng.choice(["silu", "gelu", "gelu_tanh"]),
                "gt": rng.choice(["e4m3", "e5m2"])}
    return {"op": op, "rows": span(1, 4096), "cols": span(64, 16384, 32),
            "act": rng.choice(["relu", "silu", "gelu", "gelu_tanh"]),
            "gt": rng.choice(["e4m3", "e5m2"])}


def _tile_bytes(rows, blocks):
    return 512 * -(-rows // 128) * -(-blocks // 4)


def _mx_bytes(rows, cols):
    return rows * cols + rows * cols // 32


def work(case):
    c, op = case, case["op"]
    if op == "norm":
        n = c["rows"] * c["cols"]
        gate = {"none": 0, "vector": 2 * c["cols"], "token": 2 * n}[c["gate"]]
        out = 2 * n if c["out"] == "bf16" else _mx_bytes(c["rows"], c["cols"])
        return {"bytes": 6 * n + gate + out + 2 * c["cols"] * (2 if c["post"] else 1) +
                4 * c["rows"], "flops": 12 * n}
    if op == "norm_bwd":
        n = c["rows"] * c["cols"]
        gate = {"none": 0, "vector": 6 * c["cols"], "token": 4 * n}[c["gate"]]
        return {"bytes": 12 * n + gate + c["cols"] * (12 if c["post"] else 6) + 8 * c["rows"],
                "flops": 24 * n}
    if op == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        out = 2 * m * n if c["out"] == "bf16" else _mx_bytes(m, n)
        return {"bytes": _mx_bytes(m, k) + _mx_bytes(n, k) + out +
                (2 * m * n if c["residual"] else 0) + (2 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "gated":
        m, f, k = c["m"], c["f"], c["k"]
        out = 2 * m * f if c["out"] == "bf16" else _mx_bytes(m, f)
        return {"bytes": _mx_bytes(m, k) + 2 * _mx_bytes(f, k) + out +
                (4 * m * f if c["save"] else 0), "flops": 4 * m * f * k}
    if op == "gated_bwd":
        m, f, k = c["m"], c["f"], c["k"]
        return {"bytes": 6 * m * f + _mx_bytes(m, k) + _mx_bytes(2 * f, k) + 2 * m * k + 4 * f * k,
                "flops": 8 * m * f * k}
    n = c["rows"] * c["cols"]
    return {"bytes": 4 * n + 2 * _mx_bytes(c["rows"], c["cols"]) + 4 * c["cols"], "flops": 20 * n}


# ---- inputs -----------------------------------------------------------------------------------
def _normal(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _stream(g, rows, cols):
    """A residual stream: unit values with a few channels an order of magnitude larger."""
    x = _normal(g, rows, cols)
    x[:, ::97] *= 12.0
    return x.to(torch.bfloat16)


def _operand(g, rows, cols, fmt, std=1.0, pad=None):
    """A random MX operand [rows, cols]; with `pad`, the columns from `pad` on hold zeros."""
    v = _normal(g, rows, cols, std=std)
    if pad is not None:
        v[:, pad:] = 0
    return _quantise(v, fmt)


def prepare(case, seed):
    c, op = case, case["op"]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}
    bf = torch.bfloat16
    if op in ("norm", "norm_bwd"):
        rows, cols = c["rows"], c["cols"]
        s["y"] = _normal(g, rows, cols, std=0.7).to(bf)
        s["w"] = (1 + 0.1 * _normal(g, cols)).to(bf)
        s["w_post"] = (1 + 0.1 * _normal(g, cols)).to(bf) if c["post"] else None
        s["gate"] = {"none": None, "vector": lambda: _normal(g, cols, std=0.5).to(bf),
                     "token": lambda: _normal(g, rows, cols, std=0.5).to(bf)}[c["gate"]]
        s["gate"] = s["gate"]() if s["gate"] is not None else None
        s["scale"] = 0.5
        if op == "norm":
            s["x"] = _stream(g, rows, cols)
        else:  # what the forward pass left behind, and the gradients that arrive
            s["x_out"] = _stream(g, rows, cols)
            s["dn"] = _normal(g, rows, cols, std=0.1).to(bf)
            s["dx_out"] = _normal(g, rows, cols, std=0.1).to(bf)
            s["rstd"] = torch.rsqrt(s["x_out"].double().square().mean(1) + 1e-6).float()
            s["rstd_post"] = torch.rsqrt(s["y"].double().square().mean(1) + 1e-6).float() \
                if c["post"] else None
    elif op == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s["a"], s["sfa"] = _operand(g, m, k, c["at"])
        s["b"], s["sfb"] = _operand(g, n, k, c["bt"], std=k ** -0.5)
        s["bias"] = _normal(g, n, std=0.5).to(bf) if c["bias"] else None
        s["residual"] = _stream(g, m, n) if c["residual"] else None
    elif op == "gated":
        m, f, k = c["m"], c["f"], c["k"]
        s["a"], s["sfa"] = _operand(g, m, k, "e4m3")
        s["wg"], s["sfg"] = _operand(g, f, k, "e4m3", std=k ** -0.5)
        s["wu"], s["sfu"] = _operand(g, f, k, "e4m3", std=k ** -0.5)
    elif op == "gated_bwd":
        m, f, k = c["m"], c["f"], c["k"]
        s["gate"], s["up"] = _normal(g, m, f).to(bf), _normal(g, m, f).to(bf)
        s["dh"] = _normal(g, m, f, std=0.05).to(bf)
        # the input transposed, quantised along the tokens (padded to whole blocks), and both
        # weights transposed, quantised along the features
        s["xt"], s["sfxt"] = _operand(g, k, -(-m // 32) * 32, "e4m3", pad=m)
        s["wt"], s["sfwt"] = _operand(g, k, 2 * f, "e4m3", std=k ** -0.5)
    else:
        rows, cols = c["rows"], c["cols"]
        s["pre"] = _normal(g, rows, cols).to(bf)
        s["dh"] = _normal(g, rows, cols, std=0.05).to(bf)
    return s


# ---- plain form -------------------------------------------------------------------------------
def _block(sf):
    """Row-major scales [rows, blocks] (uint8) to the tiled layout, padded with zeros."""
    rows, blocks = sf.shape
    R, S = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros((R * 128, S * 4), dtype=torch.uint8, device=sf.device)
    full[:rows, :blocks] = sf
    return full.view(R, 4, 32, S, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _unblock(sf, rows, blocks):
    R, S = -(-rows // 128), -(-blocks // 4)
    return sf.view(torch.uint8).view(R, S, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(
        R * 128, S * 4)[:rows, :blocks]


def _quantise(v, fmt):
    """f32 [rows, cols] to (float8 [rows, cols], scales in the tiled layout)."""
    kind, emax, top = FMT[fmt]
    rows, cols = v.shape
    b = v.view(rows, cols // 32, 32)
    amax = b.abs().amax(2)
    code = ((amax.view(torch.int32) >> 23) & 255).sub(emax).clamp_(min=0)
    inv = torch.ldexp(torch.ones_like(amax), 127 - code)
    q = (b * inv.unsqueeze(2)).clamp_(-top, top).to(kind).view(rows, cols)
    return q, _block(code.to(torch.uint8)).view(torch.float8_e8m0fnu)


def _value(q, sf):
    """The f32 values an MX operand stands for."""
    rows, cols = q.shape
    code = _unblock(sf, rows, cols // 32).to(torch.int32)
    scale = torch.ldexp(torch.ones(code.shape, device=q.device), code - 127)
    return (q.float().view(rows, cols // 32, 32) * scale.unsqueeze(2)).view(rows, cols)


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def _act_grad(v, act):
    if act == "relu":
        return (v > 0).float()
    if act == "silu":
        t = torch.sigmoid(v)
        return t * (1 + v * (1 - t))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + \
            v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    return torch.ones_like(v)


def _plain_norm(s):
    c = s["case"]
    x, y = s["x"].float(), s["y"].float()
    rp = None
    if c["post"]:
        rp = torch.rsqrt(y.square().mean(1) + 1e-6)
        y = y * rp.unsqueeze(1) * s["w_post"].float()
    if s["gate"] is not None:
        y = y * s["gate"].float()
    xo = (x + s["scale"] * y).to(torch.bfloat16)
    x = xo.float()
    r = torch.rsqrt(x.square().mean(1) + 1e-6)
    n = x * r.unsqueeze(1) * s["w"].float()
    n = n.to(torch.bfloat16) if c["out"] == "bf16" else _quantise(n, c["out"])
    return xo, n, (r, rp)


def _plain_norm_bwd(s):
    x, y, w = s["x_out"].float(), s["y"].float(), s["w"].float()
    dn, r = s["dn"].float(), s["rstd"].unsqueeze(1)
    a = dn * w
    dx = s["dx_out"].float() + r * a - x * r ** 3 * (a * x).mean(1, keepdim=True)
    dw = (dn * x * r).sum(0)
    p, yh = y, None
    if s["w_post"] is not None:
        yh = y * s["rstd_post"].unsqueeze(1)
        p = yh * s["w_post"].float()
    dg, dp = None, s["scale"] * dx
    if s["gate"] is not None:
        dg = s["scale"] * p * dx
        dg = dg.sum(0) if s["gate"].dim() == 1 else dg.to(torch.bfloat16)
        dp = dp * s["gate"].float()
    dy, dwp = dp, None
    if s["w_post"] is not None:
        b, rp = dp * s["w_post"].float(), s["rstd_post"].unsqueeze(1)
        dy = rp * (b - yh * (b * yh).mean(1, keepdim=True))
        dwp = (dp * yh).sum(0)
    return dx.to(torch.bfloat16), dw, dy.to(torch.bfloat16), dwp, dg


def _plain_linear(s):
    c = s["case"]
    v = _value(s["a"], s["sfa"]) @ _value(s["b"], s["sfb"]).t()
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, c["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(torch.bfloat16) if c["out"] == "bf16" else _quantise(v, c["out"])


def _plain_gated(s):
    c = s["case"]
    a = _value(s["a"], s["sfa"])
    gate, up = a @ _value(s["wg"], s["sfg"]).t(), a @ _value(s["wu"], s["sfu"]).t()
    h = _act(gate, c["act"]) * up
    h = h.to(torch.bfloat16) if c["out"] == "bf16" else _quantise(h, c["out"])
    return (h, (gate.to(torch.bfloat16), up.to(torch.bfloat16))) if c["save"] else h


def _transposed(v, fmt):
    """f32 [rows, cols] to the MX operand [cols, rows padded to whole blocks]."""
    rows, cols = v.shape
    t = torch.zeros((cols, -(-rows // 32) * 32), device=v.device)
    t[:, :rows] = v.t()
    return _quantise(t, fmt)


def _plain_gated_bwd(s):
    c = s["case"]
    dh, gate, up = s["dh"].float(), s["gate"].float(), s["up"].float()
    d = torch.cat([dh * up * _act_grad(gate, c["act"]), dh * _act(gate, c["act"])], 1)
    dx = _value(*_quantise(d, c["gt"])) @ _value(s["wt"], s["sfwt"]).t()
    dw = _value(*_transposed(d, c["gt"])) @ _value(s["xt"], s["sfxt"]).t()
    return dx.to(torch.bfloat16), dw.to(torch.bfloat16)


def _plain_act_bwd(s):
    c = s["case"]
    d = s["dh"].float() * _act_grad(s["pre"].float(), c["act"])
    return _quantise(d, c["gt"]), _transposed(d, c["gt"]), d.sum(0)


# ---- the library's entry points ----------------------------------------------------------------
def _lib():
    if "ptxstd" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "ptx-std_b200"))
    import ptxstd
    return ptxstd


def _f8(pair, fmt):
    return pair[0].view(FMT[fmt][0]), pair[1].view(torch.float8_e8m0fnu)


def _u8(t):
    return t.view(torch.uint8)


def _own(s):
    P, c, op = _lib(), s["case"], s["case"]["op"]
    if op == "norm":
        fmt = None if c["out"] == "bf16" else c["out"]
        xo, n, stats = P.rmsnorm_residual(s["x"], s["w"], y=s["y"], w_post=s["w_post"],
                                          gate=s["gate"], scale=s["scale"], eps=1e-6,
                                          elem_type=fmt)
        return xo, (n if fmt is None else _f8(n, fmt)), stats
    if op == "norm_bwd":
        return P.rmsnorm_residual_backward(
            s["dn"], s["x_out"], s["w"], (s["rstd"], s["rstd_post"]), dx_out=s["dx_out"],
            y=s["y"], w_post=s["w_post"], gate=s["gate"], scale=s["scale"])
    if op == "linear":
        fmt = None if c["out"] == "bf16" else c["out"]
        r = P.gemm_mx_epilogue(_u8(s["a"]), c["at"], _u8(s["sfa"]), _u8(s["b"]), c["bt"],
                               _u8(s["sfb"]), bias=s["bias"], act=c["act"],
                               residual=s["residual"], elem_type=fmt)
        return r if fmt is None else _f8(r, fmt)
    if op == "gated":
        fmt = None if c["out"] == "bf16" else c["out"]
        r = P.gemm_mx_gated(_u8(s["a"]), "e4m3", _u8(s["sfa"]), _u8(s["wg"]), _u8(s["sfg"]),
                            _u8(s["wu"]), _u8(s["sfu"]), "e4m3", act=c["act"], elem_type=fmt,
                            save=c["save"])
        h, kept = r if c["save"] else (r, None)
        h = h if fmt is None else _f8(h, fmt)
        return (h, kept) if c["save"] else h
    if op == "gated_bwd":
        return P.gemm_mx_gated_backward(s["dh"], s["gate"], s["up"], _u8(s["xt"]), "e4m3",
                                        _u8(s["sfxt"]), _u8(s["wt"]), "e4m3", _u8(s["sfwt"]),
                                        act=c["act"], elem_type=c["gt"])
    row, col, db = P.act_backward_mx(s["dh"], s["pre"], act=c["act"], elem_type=c["gt"],
                                     bias_grad=True)
    return _f8(row, c["gt"]), _f8(col, c["gt"]), db


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "linear": _plain_linear,
            "gated": _plain_gated, "gated_bwd": _plain_gated_bwd,
            "act_bwd": _plain_act_bwd}[state["case"]["op"]](state)


# ---- 64 bits ----------------------------------------------------------------------------------
def _at(rows, blocks, device):
    """Byte of scale (r, s) in the tiled layout, [rows, blocks]."""
    r = torch.arange(rows, device=device).unsqueeze(1)
    s = torch.arange(blocks, device=device).unsqueeze(0)
    tile = (r // 128) * -(-blocks // 4) + s // 4
    return tile * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + s % 4


def _value64(q, sf):
    rows, cols = q.shape
    scale = sf.double()[_at(rows, cols // 32, q.device)]
    return q.double() * scale.repeat_interleave(32, 1)


def _quantise64(v, fmt):
    kind, emax, top = FMT[fmt]
    rows, cols = v.shape
    amax = v.abs().reshape(rows, cols // 32, 32).amax(2)
    exponent = torch.frexp(amax)[1] - 1  # floor(log2) of a positive value
    code = torch.where(amax > 0, exponent + 127 - emax, 0).clamp(0, 254)
    each = torch.exp2((127 - code).double()).repeat_interleave(32, 1)
    q = (v * each).clamp(-top, top)
    # the nearest value with the format's fraction bits, ties to even, subnormals included
    bits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    step = torch.exp2((torch.frexp(q)[1] - 1).clamp(min=low).double() - bits)
    q = (torch.round(q / step) * step).clamp(-top, top)
    sf = torch.zeros(_tile_bytes(rows, cols // 32), dtype=torch.uint8, device=v.device)
    sf[_at(rows, cols // 32, v.device)] = code.to(torch.uint8)
    return q, torch.exp2(sf.double() - 127)


def _act64(v, act):
    """The activation and its derivative."""
    if act == "relu":
        return torch.relu(v), (v > 0).double()
    if act == "silu":
        t = 1 / (1 + torch.exp(-v))
        return v * t, t + v * t * (1 - t)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(8 / math.pi)
        t = 1 / (1 + torch.exp(-k * (v + 0.044715 * v * v * v)))
        return v * t, t + v * t * (1 - t) * k * (1 + 0.134145 * v * v)
    return v, torch.ones_like(v)


def exact(case, seed):
    s, c, op = prepare(case, seed), case, case["op"]
    d = {k: v.double() for k, v in s.items()
         if isinstance(v, torch.Tensor) and v.dtype in (torch.bfloat16, torch.float32)}
    if op == "norm":
        y = d["y"]
        rp = None
        if "w_post" in d:
            rp = 1 / (y.pow(2).mean(1) + 1e-6).sqrt()
            y = y * rp[:, None] * d["w_post"]
        xo = (d["x"] + 0.5 * d.get("gate", 1.0) * y).to(torch.bfloat16).double()
        r = 1 / (xo.pow(2).mean(1) + 1e-6).sqrt()
        n = xo * r[:, None] * d["w"]
        return xo, (n if c["out"] == "bf16" else _quantise64(n, c["out"])), (r, rp)
    if op == "norm_bwd":
        xh, a = d["x_out"] * d["rstd"][:, None], d["dn"] * d["w"]
        dx = d["dx_out"] + d["rstd"][:, None] * (a - xh * (a * xh).mean(1)[:, None])
        yh = d["y"] * d["rstd_post"][:, None] if c["post"] else d["y"]
        p = yh * d["w_post"] if c["post"] else yh
        dg = 0.5 * p * dx if c["gate"] != "none" else None
        b = 0.5 * dx * d.get("gate", 1.0)
        dwp = None
        dy = b
        if c["post"]:
            dwp = (b * yh).sum(0)
            b = b * d["w_post"]
            dy = d["rstd_post"][:, None] * (b - yh * (b * yh).mean(1)[:, None])
        return dx, (d["dn"] * xh).sum(0), dy, dwp, dg.sum(0) if c["gate"] == "vector" else dg
    if op == "linear":
        v = torch.matmul(_value64(s["a"], s["sfa"]), _value64(s["b"], s["sfb"]).T)
        v = _act64(v + d["bias"] if c["bias"] else v, c["act"])[0]
        v = v + d["residual"] if c["residual"] else v
        return v if c["out"] == "bf16" else _quantise64(v, c["out"])
    if op == "gated":
        a = _value64(s["a"], s["sfa"])
        gate = torch.matmul(a, _value64(s["wg"], s["sfg"]).T)
        up = torch.matmul(a, _value64(s["wu"], s["sfu"]).T)
        h = _act64(gate, c["act"])[0] * up
        h = h if c["out"] == "bf16" else _quantise64(h, c["out"])
        return (h, (gate, up)) if c["save"] else h

    def both(v):
        rows, cols = v.shape
        t = torch.zeros((cols, -(-rows // 32) * 32), device=v.device, dtype=torch.float64)
        t[:, :rows] = v.T
        return _quantise64(v, c["gt"]), _quantise64(t, c["gt"])

    if op == "gated_bwd":
        f, df = _act64(d["gate"], c["act"])
        grads = torch.hstack((d["dh"] * d["up"] * df, d["dh"] * f))
        row, col = both(grads)

        def stood(pair):
            rows, cols = pair[0].shape
            scale = pair[1][_at(rows, cols // 32, pair[0].device)]
            return pair[0] * scale.repeat_interleave(32, 1)

        return (torch.matmul(stood(row), _value64(s["wt"], s["sfwt"]).T),
                torch.matmul(stood(col), _value64(s["xt"], s["sfxt"]).T))
    grads = d["dh"] * _act64(d["pre"], c["act"])[1]
    row, col = both(grads)
    return row, col, grads.sum(0)
