"""Feed-forward operators around the MX GEMM over CUDA tensors (torch supplies memory/streams).

Norms of a residual stream, a GEMM with bias, activation and residual in its epilogue, a gated
projection, and the backward passes. MX tensors are (payload, scales) pairs as from
``quantize_mx``: payload [rows, cols] uint8, scales a flat uint8 tensor in the blocked layout,
padded to whole tiles of 128 rows x 4 scale columns (``sf_numel``; the padding that these operators
write is zero, the padding that they read may hold anything).

Inputs have to be contiguous and on the current CUDA device.
"""

from __future__ import annotations

import os

from . import HERE, lib
from .kernels import MX_E4M3, MX_E5M2, _mx_type

ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_OUT = {None: -1, "e4m3": MX_E4M3, "e5m2": MX_E5M2}

_module = None


def _ext():
    """The extension module with the argument checks, allocations and C calls (ptxstd/_ffn.so, from
    build.py); it raises if it or libptxstd.so is missing."""
    global _module
    if _module is None:
        lib()
        if not os.path.exists(os.path.join(HERE, "_ffn.so")):
            raise OSError(f"{HERE}/_ffn.so is missing: run `python ptx-std_b200/build.py` first")
        import torch  # noqa: F401  (its libraries resolve the module's symbols)

        from . import _ffn
        _module = _ffn
    return _module


def sf_numel(rows: int, cols: int) -> int:
    """Bytes of the padded blocked scale tensor of an MX operand [rows, cols]."""
    return -(-rows // 128) * -(-cols // 128) * 512


def _act(act) -> int:
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"unknown activation {act!r} (one of {sorted(ACTS)})")
    return code


def _out_type(t) -> int:
    """The result's type: -1 for None (bf16), else the code of e4m3 or e5m2."""
    code = _OUT.get(t)
    if code is None:
        code = _mx_type(t)
        if code not in (MX_E4M3, MX_E5M2):
            raise ValueError("these operators write MX results as e4m3 or e5m2")
    return code


def rmsnorm_residual(x, w, y=None, w_post=None, gate=None, scale: float = 1.0, eps: float = 1e-6,
                     elem_type=None, sf_layout: int = 1, stream=None):
    """x' = bf16(x + scale * gate * p), p = rmsnorm(y) * w_post (y without w_post); the result
    n = rmsnorm(x') * w, as bf16 or, with an elem_type ("e4m3", "e5m2"), as an MX operand with
    blocked (sf_layout 1, padded) or row-major (0) scales.

    x, y bf16 [rows, cols]; w, w_post bf16 [cols]; gate bf16 [cols] or [rows, cols]. Returns
    (x', n or (q, sf), (rstd, rstd_post)); the f32 [rows] statistics are what the backward pass
    takes, rstd_post None without w_post. Without y, x' is x itself."""
    return _ext().rmsnorm_residual(x, w, y, w_post, gate, scale, eps, _out_type(elem_type),
                                   sf_layout, stream)


def rmsnorm_residual_backward(dn, x_out, w, stats, dx_out=None, y=None, w_post=None, gate=None,
                              scale: float = 1.0, stream=None):
    """Gradient of rmsnorm_residual, from dn (bf16, of n) and dx_out (bf16, of x' by other paths,
    or None). x_out and stats are what the forward pass returned, the rest what it was given.

    Returns (dx bf16, dw f32, dy bf16, dw_post f32, dgate), None where there was no such input;
    dgate is f32 [cols] for a [cols] gate and bf16 [rows, cols] for one per row."""
    rstd, rstd_post = stats
    return _ext().rmsnorm_residual_backward(dn, x_out, w, rstd, rstd_post, dx_out, y, w_post, gate,
                                            scale, stream)


def gemm_mx_epilogue(a, a_type, sfa, b, b_type, sfb, bias=None, act="none", residual=None,
                     elem_type=None, save_pre: bool = False, stream=None):
    """act(a @ b^T + bias) + residual of MX operands a [M, K], b [N, K] (any M >= 1, K % 32 == 0,
    N % 8 == 0): bf16 [M, N] or, with an elem_type (N % 32 == 0), an MX operand (q, sf). bias bf16
    [N], residual bf16 [M, N]. With save_pre the result is (result, pre), pre = a @ b^T + bias in
    bf16 for act_backward_mx."""
    return _ext().gemm_mx_epilogue(a, _mx_type(a_type), sfa, b, _mx_type(b_type), sfb, bias,
                                   _act(act), residual, _out_type(elem_type), save_pre, stream)


def gemm_mx_gated(a, a_type, sfa, w_gate, sf_gate, w_up, sf_up, w_type, act="silu", elem_type=None,
                  save: bool = False, stream=None):
    """act(a @ w_gate^T) * (a @ w_up^T) of MX operands a [M, K], w_gate and w_up [F, K] in one
    kernel (any M >= 1, K % 32 == 0, F % 8 == 0): bf16 [M, F] or, with an elem_type (F % 32 == 0),
    an MX operand (q, sf). With save the result is (h, (gate, up)), the two projections in bf16
    for the backward pass."""
    return _ext().gemm_mx_gated(a, _mx_type(a_type), sfa, w_gate, sf_gate, w_up, sf_up,
                                _mx_type(w_type), _act(act), _out_type(elem_type), save, stream)


def act_backward_mx(dh, gate, up=None, act="silu", elem_type="e5m2", bias_grad: bool = False,
                    stream=None):
    """D = [dh * up * act'(gate) | dh * act(gate)] (D = dh * act'(gate) without up), quantised along
    its rows and along its columns in one pass: ((q [rows, W], sf), (qt [W, R], sft)), R = rows
    rounded up to 32. dh, gate, up bf16 [rows, cols], cols % 32 == 0. With bias_grad the column sums
    of D (f32 [W]) come third."""
    return _ext().act_backward_mx(dh, gate, up, _act(act), _out_type(elem_type), bias_grad, stream)


def quantize_mx_t(x, elem_type, stream=None):
    """bf16 [rows, cols] (cols % 8 == 0) -> the transposed MX operand (payload [cols, R], padded
    blocked scales), blocks of 32 along the rows of x, R = rows rounded up to 32 (zeros there)."""
    return _ext().quantize_mx_t(x, _out_type(elem_type), stream)


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
