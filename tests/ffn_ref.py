"""Plain 64-bit restatements of the feed-forward operators (torch, any device) and the interval
checks their tests use.

A kernel computes a value v within a derived bound d of the exact one and rounds it once; rounding
is monotone, so the stored result has to lie between the roundings of (exact - d) and (exact + d).
That holds for bf16 and for MX codes alike (where a block's scale, too, has to lie between the
scales of its two bounds), saturation included, with no further allowance.
"""

import math

import torch

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
EMAX = {"e4m3": 8, "e5m2": 15}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
MANT = {"e4m3": 3, "e5m2": 2}
LOW = {"e4m3": -6, "e5m2": -14}


def sf_offsets(rows, blocks, device="cpu"):
    r = torch.arange(rows, device=device)[:, None]
    s = torch.arange(blocks, device=device)[None, :]
    return ((r // 128) * (-(-blocks // 4)) + s // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + \
        s % 4


def sf_rowmajor(sf, rows, blocks):
    """(codes [rows, blocks], the padding bytes) of a padded blocked scale tensor."""
    at = sf_offsets(rows, blocks, sf.device)
    mask = torch.ones(sf.numel(), dtype=torch.bool, device=sf.device)
    mask[at.reshape(-1)] = False
    return sf[at], sf[mask]


def dequant(q, sf, fmt):
    """f64 values of an E4M3 / E5M2 operand with padded blocked scales."""
    rows, cols = q.shape
    code, _ = sf_rowmajor(sf, rows, cols // 32)
    v = q.view(F8[fmt]).double().view(rows, cols // 32, 32)
    s = torch.where(code == 255, torch.nan, torch.exp2(code.double() - 127))
    return (v * s[:, :, None]).view(rows, cols)


def act(x, kind):
    if kind == "relu":
        return x.clamp(min=0)
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return x * 0.5 * torch.erfc(-x / math.sqrt(2))
    if kind == "gelu_tanh":
        return x * torch.sigmoid(math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3))
    return x


def act_grad(x, kind):
    x = x.detach().clone().requires_grad_(True)
    y = act(x, kind)
    if kind == "relu":
        return (x > 0).double()
    return torch.autograd.grad(y.sum(), x)[0]


def _round(x, fmt):
    """x (f64) to the format's values, nearest even, saturating."""
    e = torch.frexp(x)[1] - 1
    step = torch.exp2(e.clamp(min=LOW[fmt]).double() - MANT[fmt])
    return (torch.round(x / step) * step).clamp(-TOP[fmt], TOP[fmt])


def scale_code(amax, fmt):
    e = torch.frexp(amax)[1] - 1
    return torch.where(amax > 0, (e + 127).clamp(0, 254) - EMAX[fmt], 0).clamp(min=0)


def check_bf16(got, ref, d, what=""):
    """got is the bf16 rounding of a value within d of ref."""
    assert got.dtype == torch.bfloat16 and got.shape == ref.shape
    g = got.double()
    lo = (ref - d).to(torch.bfloat16).double()
    hi = (ref + d).to(torch.bfloat16).double()
    bad = ~((g >= lo) & (g <= hi))
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(), g[bad][:4].tolist(),
                           ref[bad][:4].tolist())


def check_mx(q, sf, ref, d, fmt, padded=True, what=""):
    """(q, sf) is the MX quantisation of values within d of ref; the padding bytes are zero."""
    rows, cols = ref.shape
    blocks = cols // 32
    if padded:
        code, rest = sf_rowmajor(sf, rows, blocks)
        assert not rest.any(), f"{what}: scale padding written"
    else:
        code = sf.view(rows, blocks)
    d = d.expand_as(ref) if isinstance(d, torch.Tensor) else torch.full_like(ref, d)
    b = ref.abs().view(rows, blocks, 32)
    db = d.reshape(rows, blocks, 32)
    lo = scale_code((b - db).clamp(min=0).amax(2), fmt)
    hi = scale_code((b + db).amax(2), fmt)
    c = code.long()
    bad = (c < lo) | (c > hi)
    assert not bad.any(), (what, "scale", bad.nonzero()[:4].tolist(), c[bad][:4].tolist(),
                           lo[bad][:4].tolist())
    inv = torch.exp2((127 - c).double()).repeat_interleave(32, 1)
    v = q.view(F8[fmt]).double()
    low, high = _round((ref - d) * inv, fmt), _round((ref + d) * inv, fmt)
    bad = ~((v >= low) & (v <= high))
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(), v[bad][:4].tolist(),
                           (ref * inv)[bad][:4].tolist())


def gemm(a, b):
    """(a b^T, sum |a b|) in f64."""
    return a @ b.t(), a.abs() @ b.abs().t()


def acc_bound(mag, K):
    """The tensor cores' f32 accumulation: each K = 32 step rounds or truncates the running sum
    and its own partial sum to 24 significant bits (2^-23 of at most sum |a b| each)."""
    return mag * ((K // 32 + 1) * 2.0 ** -22)


def norm_forward(x, y, w_post, gate, scale, eps):
    """(x + scale gate p, magnitude of its terms, ry) in f64, before the bf16 rounding."""
    p, ry = y, None
    if w_post is not None:
        ry = 1 / (y.square().mean(1) + eps).sqrt()
        p = y * ry[:, None] * w_post
    p = p * scale * (gate if gate is not None else 1.0)
    return x + p, x.abs() + p.abs(), ry


def norm_result(xo, w, eps):
    r = 1 / (xo.square().mean(1) + eps).sqrt()
    return xo * r[:, None] * w, r


def norm_backward(dn, du, xo, w, rx, y, w_post, ry, gate, scale):
    """The gradients in f64 and the magnitudes of their terms."""
    rx = rx[:, None]
    a = dn * w
    mean = (a * xo).mean(1, keepdim=True)
    mean_mag = (a * xo).abs().mean(1, keepdim=True)
    dx = rx * a - xo * rx ** 3 * mean
    mag = (rx * a).abs() + xo.abs() * rx ** 3 * mean_mag
    if du is not None:
        dx, mag = dx + du, mag + du.abs()
    out = {"dx": (dx, mag), "dw": ((dn * xo * rx).sum(0), (dn * xo * rx).abs().sum(0))}
    if y is None:
        return out
    yh = y * ry[:, None] if w_post is not None else y
    p = yh * w_post if w_post is not None else yh
    g = gate if gate is not None else 1.0
    if gate is not None:
        dg, dg_mag = scale * p * dx, (scale * p).abs() * mag
        out["dgate"] = (dg.sum(0), dg_mag.sum(0)) if gate.dim() == 1 else (dg, dg_mag)
    dp, dp_mag = scale * g * dx, (abs(scale) * (g.abs() if gate is not None else 1.0)) * mag
    if w_post is None:
        out["dy"] = (dp, dp_mag)
        return out
    out["dw_post"] = ((dp * yh).sum(0), (dp_mag * yh.abs()).sum(0))
    b, b_mag = dp * w_post, dp_mag * w_post.abs()
    m = (b * yh).mean(1, keepdim=True)
    m_mag = (b_mag * yh.abs()).mean(1, keepdim=True)
    r = ry[:, None]
    out["dy"] = (r * (b - yh * m), r * (b_mag + yh.abs() * m_mag))
    return out
