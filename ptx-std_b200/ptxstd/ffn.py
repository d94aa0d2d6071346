"""Feed-forward operators around the MX GEMM over CUDA tensors (torch supplies memory/streams).

Norms of a residual stream, a GEMM with bias, activation and residual in its epilogue, a gated
projection, and the backward passes. MX tensors are (payload, scales) pairs as from
``quantize_mx``: payload [rows, cols] uint8, scales a flat uint8 tensor in the blocked layout,
padded to whole tiles of 128 rows x 4 scale columns (``sf_numel``; the padding that these operators
write is zero, the padding that they read may hold anything).

Inputs have to be contiguous and on the current CUDA device.
"""

from __future__ import annotations

from . import _torch, check, lib
from .kernels import MX_E4M3, MX_E5M2, _mx_type

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def sf_numel(rows: int, cols: int) -> int:
    """Bytes of the padded blocked scale tensor of an MX operand [rows, cols]."""
    return -(-rows // 128) * -(-cols // 128) * 512


def _act(act) -> int:
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"unknown activation {act!r} (one of {sorted(ACTS)})")
    return code


def _out_type(t) -> int:
    code = _mx_type(t)
    if code not in (MX_E4M3, MX_E5M2):
        raise ValueError("these operators write MX results as e4m3 or e5m2")
    return code


def _want(t, name: str, dtype, shape) -> None:
    """Type and shape of one argument (None passes)."""
    if t is None:
        return
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _want_mx(q, sf, name: str, cols: int | None = None) -> tuple[int, int]:
    """An MX operand's (rows, cols), with its type, width and scale size checked."""
    torch = _torch()
    if q.dtype is not torch.uint8 or sf.dtype is not torch.uint8 or q.dim() != 2:
        raise TypeError(f"{name}: expected a 2-D uint8 payload and uint8 scales")
    rows, k = q.shape
    if cols is not None and k != cols:
        raise ValueError(f"{name}: K mismatch ({k}, expected {cols})")
    if sf.numel() != sf_numel(rows, k):
        raise ValueError(f"{name}: the blocked scales of [{rows}, {k}] have {sf_numel(rows, k)} "
                         f"bytes, got {sf.numel()}")
    return rows, k


def _ins(*tensors) -> list[int]:
    """Device pointers of the inputs (0 for None), each contiguous and on the current device."""
    out = []
    dev = None
    for t in tensors:
        if t is None:
            out.append(0)
            continue
        d = t.get_device()
        if d != dev:
            if d < 0:
                raise TypeError("expected a CUDA tensor")
            dev = _torch().cuda.current_device()
            if d != dev:
                raise ValueError(f"tensor on cuda:{d}, but the current device is cuda:{dev}")
        if not t.is_contiguous():
            raise ValueError("expected a contiguous tensor")
        out.append(t.data_ptr())
    return out


def _outs(*tensors) -> list[int]:
    """Device pointers of tensors allocated here."""
    return [0 if t is None else t.data_ptr() for t in tensors]


def _handle(stream, like) -> int:
    """The cudaStream_t of `stream`, or of the current stream of the tensor's device."""
    if stream is not None:
        return stream.cuda_stream
    return _torch()._C._cuda_getCurrentRawStream(like.get_device())


def _new(rows: int, cols: int, dtype, device):
    """An uninitialised [rows, cols] tensor (empty_strided is the cheapest of torch's calls)."""
    return _torch().empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _new1(n: int, dtype, device):
    return _torch().empty_strided((n,), (1,), dtype=dtype, device=device)


def _mx_empty(rows: int, cols: int, device):
    u8 = _torch().uint8
    return _new(rows, cols, u8, device), _new1(sf_numel(rows, cols), u8, device)


def rmsnorm_residual(x, w, y=None, w_post=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                     elem_type=None, sf_layout: int = 1, stream=None):
    """x' = bf16(x + scale * gate * p), p = rmsnorm(y) * w_post (y without w_post); the result
    n = rmsnorm(x') * w, as bf16 or, with an elem_type ("e4m3", "e5m2"), as an MX operand with
    blocked (sf_layout 1, padded) or row-major (0) scales.

    x, y bf16 [rows, cols]; w, w_post bf16 [cols]; gate bf16 [cols] or [rows, cols]. Returns
    (x', n or (q, sf), (rstd, rstd_post)); the f32 [rows] statistics are what the backward pass
    takes, rstd_post None without w_post. Without y, x' is x itself."""
    torch = _torch()
    if x.dtype is not torch.bfloat16 or x.dim() != 2:
        raise TypeError("expected a 2-D bfloat16 tensor")
    rows, cols = x.shape
    bf = torch.bfloat16
    _want(w, "w", bf, (cols,))
    _want(y, "y", bf, (rows, cols))
    _want(w_post, "w_post", bf, (cols,))
    if y is None and (w_post is not None or gate is not None):
        raise ValueError("w_post and gate belong to y")
    gate_rows = 1
    if gate is not None and gate.dim() == 2:
        _want(gate, "gate", bf, (rows, cols))
        gate_rows = rows
    else:
        _want(gate, "gate", bf, (cols,))
    t = None if elem_type is None else _out_type(elem_type)
    px, py, pwp, pg, pw = _ins(x, y, w_post, gate, w)
    dev, s = x.device, _handle(stream, x)
    x_out = torch.empty_like(x) if y is not None else None
    n = q = sf = None
    if t is None:
        n = torch.empty_like(x)
    elif sf_layout == 1:
        q, sf = _mx_empty(rows, cols, dev)
    else:
        q = _new(rows, cols, torch.uint8, dev)
        sf = _new(rows, cols // 32, torch.uint8, dev)
    rstd = _new1(rows, torch.float32, dev)
    rstd_post = _new1(rows, torch.float32, dev) if w_post is not None else None
    pxo, pn, pq, psf, pr, prp = _outs(x_out, n, q, sf, rstd, rstd_post)
    check(lib().ptxstd_rmsnorm_residual(px, py, pwp, pg, gate_rows, scale, pw, eps, rows, cols,
                                        pxo, pn, t or 0, pq, psf, sf_layout, pr, prp, s),
          "rmsnorm_residual")
    return (x if x_out is None else x_out), (n if t is None else (q, sf)), (rstd, rstd_post)


def rmsnorm_residual_backward(dn, x_out, w, stats, dx_out=None, y=None, w_post=None, gate=None,
                              scale: float = 1.0, stream=None):
    """Gradient of rmsnorm_residual, from dn (bf16, of n) and dx_out (bf16, of x' by other paths,
    or None). x_out and stats are what the forward pass returned, the rest what it was given.

    Returns (dx bf16, dw f32, dy bf16, dw_post f32, dgate), None where there was no such input;
    dgate is f32 [cols] for a [cols] gate and bf16 [rows, cols] for one per row."""
    torch = _torch()
    if dn.dtype is not torch.bfloat16 or dn.dim() != 2:
        raise TypeError("expected a 2-D bfloat16 tensor")
    rows, cols = dn.shape
    bf, f32, dev = torch.bfloat16, torch.float32, dn.device
    rstd, rstd_post = stats
    _want(x_out, "x_out", bf, (rows, cols))
    _want(dx_out, "dx_out", bf, (rows, cols))
    _want(y, "y", bf, (rows, cols))
    _want(w, "w", bf, (cols,))
    _want(w_post, "w_post", bf, (cols,))
    _want(rstd, "rstd", f32, (rows,))
    _want(rstd_post, "rstd_post", f32, (rows,))
    if y is None and (w_post is not None or gate is not None):
        raise ValueError("w_post and gate belong to y")
    if (w_post is None) != (rstd_post is None):
        raise ValueError("w_post and its statistics belong together")
    per_row = gate is not None and gate.dim() == 2
    _want(gate, "gate", bf, (rows, cols) if per_row else (cols,))
    if per_row and rows == 1:  # one row: the gradient of a [cols] gate, given back as bf16 [1, cols]
        got = rmsnorm_residual_backward(dn, x_out, w, stats, dx_out, y, w_post, gate.view(cols),
                                        scale, stream)
        return (*got[:4], got[4].to(bf).view(1, cols))
    pdn, pdu, px, pw, pr, py, pwp, prp, pg = _ins(dn, dx_out, x_out, w, rstd, y, w_post, rstd_post,
                                                  gate)
    s = _handle(stream, dn)
    dx = torch.empty_like(dn)
    dw = _new1(cols, f32, dev)
    dy = torch.empty_like(dn) if y is not None else None
    dwp = _new1(cols, f32, dev) if w_post is not None else None
    dg = None
    if gate is not None:
        dg = torch.empty_like(gate) if per_row else _new1(cols, f32, dev)
    nbytes = lib().ptxstd_rmsnorm_residual_backward_workspace_bytes(rows, cols)
    ws = _new1(max(16, nbytes), torch.uint8, dev)
    pdx, pdw, pdy, pdwp, pdg, pws = _outs(dx, dw, dy, dwp, dg, ws)
    check(lib().ptxstd_rmsnorm_residual_backward(
        pdn, pdu, px, pw, pr, py, pwp, prp, pg, rows if per_row else 1, scale, rows, cols, pdx,
        pdw, pdy, pdwp, pdg, pws, nbytes, s), "rmsnorm_residual_backward")
    return dx, dw, dy, dwp, dg


def gemm_mx_epilogue(a, a_type, sfa, b, b_type, sfb, bias=None, act="none", residual=None,
                     elem_type=None, save_pre: bool = False, stream=None):
    """act(a @ b^T + bias) + residual of MX operands a [M, K], b [N, K] (any M >= 1, K % 32 == 0,
    N % 8 == 0): bf16 [M, N] or, with an elem_type (N % 32 == 0), an MX operand (q, sf). bias bf16
    [N], residual bf16 [M, N]. With save_pre the result is (result, pre), pre = a @ b^T + bias in
    bf16 for act_backward_mx."""
    torch = _torch()
    ta, tb, f = _mx_type(a_type), _mx_type(b_type), _act(act)
    M, K = _want_mx(a, sfa, "a")
    N, _ = _want_mx(b, sfb, "b", K)
    _want(bias, "bias", torch.bfloat16, (N,))
    _want(residual, "residual", torch.bfloat16, (M, N))
    t = 0 if elem_type is None else _out_type(elem_type)
    pa, psa, pb, psb, pbias, pres = _ins(a, sfa, b, sfb, bias, residual)
    dev, s = a.device, _handle(stream, a)
    c = q = sf = None
    if elem_type is None:
        c = _new(M, N, torch.bfloat16, dev)
    else:
        q, sf = _mx_empty(M, N, dev)
    pre = _new(M, N, torch.bfloat16, dev) if save_pre else None
    pc, ppre, pq, psf = _outs(c, pre, q, sf)
    check(lib().ptxstd_gemm_mx_epilogue(pa, ta, psa, pb, tb, psb, pbias, f, pres, pc, ppre, t, pq,
                                        psf, M, N, K, s), "gemm_mx_epilogue")
    r = c if elem_type is None else (q, sf)
    return (r, pre) if save_pre else r


def gemm_mx_gated(a, a_type, sfa, w_gate, sf_gate, w_up, sf_up, w_type, act="silu", elem_type=None,
                  save: bool = False, stream=None):
    """act(a @ w_gate^T) * (a @ w_up^T) of MX operands a [M, K], w_gate and w_up [F, K] in one
    kernel (any M >= 1, K % 32 == 0, F % 8 == 0): bf16 [M, F] or, with an elem_type (F % 32 == 0),
    an MX operand (q, sf). With save the result is (h, (gate, up)), the two projections in bf16
    for the backward pass."""
    torch = _torch()
    ta, tw, f = _mx_type(a_type), _mx_type(w_type), _act(act)
    M, K = _want_mx(a, sfa, "a")
    F, _ = _want_mx(w_gate, sf_gate, "w_gate", K)
    if _want_mx(w_up, sf_up, "w_up", K)[0] != F:
        raise ValueError("w_gate and w_up have different numbers of rows")
    t = 0 if elem_type is None else _out_type(elem_type)
    pa, psa, pg, psg, pu, psu = _ins(a, sfa, w_gate, sf_gate, w_up, sf_up)
    dev, s = a.device, _handle(stream, a)
    h = q = sf = gate = up = None
    if elem_type is None:
        h = _new(M, F, torch.bfloat16, dev)
    else:
        q, sf = _mx_empty(M, F, dev)
    if save:
        gate, up = _new(M, F, torch.bfloat16, dev), _new(M, F, torch.bfloat16, dev)
    ph, pgate, pup, pq, psf = _outs(h, gate, up, q, sf)
    check(lib().ptxstd_gemm_mx_gated(pa, ta, psa, pg, psg, pu, psu, tw, f, ph, pgate, pup, t, pq,
                                     psf, M, F, K, s), "gemm_mx_gated")
    r = h if elem_type is None else (q, sf)
    return (r, (gate, up)) if save else r


def act_backward_mx(dh, gate, up=None, act="silu", elem_type="e5m2", bias_grad: bool = False,
                    stream=None):
    """D = [dh * up * act'(gate) | dh * act(gate)] (D = dh * act'(gate) without up), quantised along
    its rows and along its columns in one pass: ((q [rows, W], sf), (qt [W, R], sft)), R = rows
    rounded up to 32. dh, gate, up bf16 [rows, cols], cols % 32 == 0. With bias_grad the column sums
    of D (f32 [W]) come third."""
    torch = _torch()
    f, t = _act(act), _out_type(elem_type)
    if dh.dtype is not torch.bfloat16 or dh.dim() != 2:
        raise TypeError("expected a 2-D bfloat16 tensor")
    rows, cols = dh.shape
    _want(gate, "gate", torch.bfloat16, (rows, cols))
    _want(up, "up", torch.bfloat16, (rows, cols))
    pdh, pg, pu = _ins(dh, gate, up)
    dev, s = dh.device, _handle(stream, dh)
    W, R = cols * (1 if up is None else 2), -(-rows // 32) * 32
    q, sf = _mx_empty(rows, W, dev)
    qt, sft = _mx_empty(W, R, dev)
    db = ws = None
    nbytes = 0
    if bias_grad:
        db = _new1(W, torch.float32, dev)
        nbytes = lib().ptxstd_act_backward_mx_workspace_bytes(rows, cols, up is not None, 1)
        ws = _new1(max(16, nbytes), torch.uint8, dev)
    pq, psf, pqt, psft, pdb, pws = _outs(q, sf, qt, sft, db, ws)
    check(lib().ptxstd_act_backward_mx(f, pdh, pg, pu, rows, cols, t, pq, psf, pqt, psft, pdb, pws,
                                       nbytes, s), "act_backward_mx")
    return ((q, sf), (qt, sft), db) if bias_grad else ((q, sf), (qt, sft))


def quantize_mx_t(x, elem_type, stream=None):
    """bf16 [rows, cols] (cols % 8 == 0) -> the transposed MX operand (payload [cols, R], padded
    blocked scales), blocks of 32 along the rows of x, R = rows rounded up to 32 (zeros there)."""
    torch = _torch()
    if x.dtype is not torch.bfloat16 or x.dim() != 2:
        raise TypeError("expected a 2-D bfloat16 tensor")
    t = _out_type(elem_type)
    rows, cols = x.shape
    (px,) = _ins(x)
    qt, sft = _mx_empty(cols, -(-rows // 32) * 32, x.device)
    check(lib().ptxstd_quantize_mx_t(px, rows, cols, t, *_outs(qt, sft), _handle(stream, x)),
          "quantize_mx_t")
    return qt, sft


def gemm_mx_gated_backward(dh, gate, up, xt, x_type, sfxt, wt, w_type, sfwt, act="silu",
                           elem_type="e5m2", stream=None):
    """Backward pass of gemm_mx_gated: (dx bf16 [M, K], dw bf16 [2 F, K], gate rows first).

    dh, gate, up bf16 [M, F]; xt [K, R] the input transposed and quantised along the tokens
    (quantize_mx_t); wt [K, 2 F] both weights transposed and quantised along the features (gate
    features first). Three kernels: act_backward_mx with `elem_type`, then dx = D wt^T and
    dw = D^T xt^T."""
    (q, sf), (qt, sft) = act_backward_mx(dh, gate, up, act, elem_type, stream=stream)
    dx = gemm_mx_epilogue(q, elem_type, sf, wt, w_type, sfwt, stream=stream)
    dw = gemm_mx_epilogue(qt, elem_type, sft, xt, x_type, sfxt, stream=stream)
    return dx, dw
