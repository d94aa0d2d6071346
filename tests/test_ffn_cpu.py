"""Host side of the feed-forward operators without a GPU: refusals, workspace sizes, and the 64-bit
restatements themselves against finite differences."""

import ctypes as C

import pytest
import torch

import ffn_ref as R


def _mx(rows, cols):
    from ptxstd.ffn import sf_numel
    return (torch.zeros((rows, cols), dtype=torch.uint8),
            torch.zeros(sf_numel(rows, cols), dtype=torch.uint8))


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_c_refusals(ptxstd_lib):
    """EINVAL before any CUDA call: sizes, types, missing and misaligned pointers."""
    L, E = ptxstd_lib.lib(), ptxstd_lib.EINVAL
    p = 4096

    def epilogue(a=p, at=0, sfa=p, b=p, bt=0, sfb=p, bias=0, act=0, res=0, c=p, pre=0, ot=0, q=0,
                 sfq=0, M=16, N=64, K=64):
        return L.ptxstd_gemm_mx_epilogue(a, at, sfa, b, bt, sfb, bias, act, res, c, pre, ot, q, sfq,
                                         M, N, K, None)

    for kw in (dict(M=0), dict(M=-1), dict(N=60), dict(K=48), dict(K=0), dict(M=1 << 31),
               dict(at=2), dict(bt=6), dict(act=5), dict(act=-1), dict(c=0), dict(a=0), dict(sfb=0),
               dict(a=p + 8), dict(c=p + 2), dict(bias=p + 4), dict(res=p + 8), dict(pre=p + 8),
               dict(q=p), dict(q=p, sfq=p, N=40), dict(q=p, sfq=p, ot=3), dict(q=p, sfq=p + 4)):
        assert epilogue(**kw) == E, kw

    def gated(a=p, at=0, wg=p, sfg=p, wu=p, wt=0, act=2, h=p, gate=0, up=0, ot=0, q=0, sfq=0, M=16,
              F=64, K=64):
        return L.ptxstd_gemm_mx_gated(a, at, p, wg, sfg, wu, p, wt, act, h, gate, up, ot, q, sfq, M,
                                      F, K, None)

    for kw in (dict(M=0), dict(F=4), dict(K=16), dict(gate=p), dict(up=p), dict(h=0), dict(wg=0),
               dict(wu=p + 1), dict(act=9), dict(wt=2), dict(q=p, sfq=p, F=72), dict(q=p),
               dict(q=p, sfq=p, ot=5)):
        assert gated(**kw) == E, kw

    def back(act=2, dh=p, gate=p, up=0, rows=8, cols=64, t=0, q=p, sf=p, qt=p, sft=p, db=0, ws=0,
             nb=0):
        return L.ptxstd_act_backward_mx(act, dh, gate, up, rows, cols, t, q, sf, qt, sft, db, ws, nb,
                                        None)

    for kw in (dict(rows=0), dict(cols=40), dict(t=3), dict(act=7), dict(dh=0), dict(gate=p + 2),
               dict(q=0), dict(sft=0), dict(db=p), dict(db=p, ws=p, nb=511),
               dict(db=p, ws=p, nb=1023, up=p), dict(up=p + 8)):
        assert back(**kw) == E, kw
    assert L.ptxstd_quantize_mx_t(p, 8, 12, 0, p, p, None) == E
    assert L.ptxstd_quantize_mx_t(p, 0, 16, 0, p, p, None) == E
    assert L.ptxstd_quantize_mx_t(p, 8, 16, 4, p, p, None) == E
    assert L.ptxstd_quantize_mx_t(p + 2, 8, 16, 0, p, p, None) == E
    assert L.ptxstd_quantize_mx(p, 8, 32, 0, p, p, 3, None) == E

    def norm(x=p, y=p, wp=0, g=0, gr=1, w=p, eps=1e-6, rows=8, cols=64, xo=p, n=p, ot=0, q=0, sf=0,
             lay=1, r=0, rp=0):
        return L.ptxstd_rmsnorm_residual(x, y, wp, g, gr, 1.0, w, eps, rows, cols, xo, n, ot, q, sf,
                                         lay, r, rp, None)

    for kw in (dict(rows=0), dict(cols=0), dict(cols=12), dict(cols=32776), dict(eps=-1.0),
               dict(eps=float("nan")), dict(x=0), dict(w=0), dict(n=0), dict(y=0), dict(xo=0),
               dict(y=0, xo=0, wp=p), dict(y=0, xo=0, g=p), dict(rp=p), dict(g=p, gr=3),
               dict(q=p, sf=p, cols=40), dict(q=p), dict(q=p, sf=p, lay=2), dict(q=p, sf=p, ot=3),
               dict(x=p + 8), dict(g=p + 2), dict(r=p + 4)):
        assert norm(**kw) == E, kw

    def nback(dn=p, du=0, x=p, w=p, r=p, y=p, wp=0, rp=0, g=0, gr=1, rows=8, cols=64, dx=p, dw=p,
              dy=p, dwp=0, dg=0, ws=p, nb=1 << 20):
        return L.ptxstd_rmsnorm_residual_backward(dn, du, x, w, r, y, wp, rp, g, gr, 1.0, rows, cols,
                                                  dx, dw, dy, dwp, dg, ws, nb, None)

    for kw in (dict(rows=0), dict(cols=20), dict(cols=16392), dict(dn=0), dict(r=0), dict(ws=0),
               dict(nb=8 * 2 * 64 * 4 - 1), dict(dy=0), dict(y=0), dict(y=0, dy=0, wp=p),
               dict(wp=p), dict(wp=p, rp=p), dict(g=p), dict(g=p, dg=p, gr=2), dict(dx=p + 8)):
        assert nback(**kw) == E, kw


def test_workspace_sizes(ptxstd_lib):
    L = ptxstd_lib.lib()
    f = L.ptxstd_act_backward_mx_workspace_bytes
    assert f(1, 64, 0, 1) == 512 and f(129, 64, 1, 1) == 2048
    assert f(129, 64, 1, 0) == 0 and f(0, 64, 0, 1) == 0
    g = L.ptxstd_rmsnorm_residual_backward_workspace_bytes
    assert g(1, 64) == 2 * 64 * 4 and g(8, 64) == 8 * 2 * 64 * 4
    assert g(0, 64) == 0 and g(8, 16392) == 0
    assert g(1 << 20, 8192) < 64 << 20


def test_wrapper_refusals(ptxstd_lib):
    """Shape and type errors come before any device call."""
    P = ptxstd_lib
    a, sfa = _mx(5, 64)
    b, sfb = _mx(32, 64)
    with pytest.raises(ValueError, match="K mismatch"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, *(_mx(32, 96)[0], "e4m3", _mx(32, 96)[1]))
    with pytest.raises(ValueError, match="blocked scales"):
        P.gemm_mx_epilogue(a, "e4m3", sfa[:-1], b, "e4m3", sfb)
    with pytest.raises(ValueError, match="unknown activation"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, act="tanh")
    with pytest.raises(ValueError, match="unknown MX element type"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e8m0", sfb)
    with pytest.raises(ValueError, match="bias"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, bias=_bf(31))
    with pytest.raises(TypeError, match="residual"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, residual=torch.zeros(5, 32))
    with pytest.raises(ValueError, match="e4m3 or e5m2"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, elem_type="e2m1")
    with pytest.raises(TypeError, match="CUDA"):
        P.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb)
    with pytest.raises(ValueError, match="different numbers of rows"):
        P.gemm_mx_gated(a, "e4m3", sfa, b, sfb, *_mx(64, 64), "e4m3")
    with pytest.raises(TypeError):
        P.gemm_mx_gated(a.float(), "e4m3", sfa, b, sfb, b, sfb, "e4m3")
    with pytest.raises(ValueError, match="up"):
        P.act_backward_mx(_bf(4, 64), _bf(4, 64), _bf(4, 32))
    with pytest.raises(TypeError):
        P.act_backward_mx(torch.zeros(4, 64), _bf(4, 64))
    with pytest.raises(TypeError):
        P.quantize_mx_t(torch.zeros(4, 64), "e4m3")
    with pytest.raises(ValueError, match="e4m3 or e5m2"):
        P.quantize_mx_t(_bf(4, 64), "e3m2")
    x, w = _bf(4, 64), _bf(64)
    with pytest.raises(ValueError, match="belong to y"):
        P.rmsnorm_residual(x, w, gate=w)
    with pytest.raises(ValueError, match="gate"):
        P.rmsnorm_residual(x, w, y=x, gate=_bf(3, 64))
    with pytest.raises(ValueError, match="w_post"):
        P.rmsnorm_residual(x, w, y=x, w_post=_bf(32))
    with pytest.raises(TypeError):
        P.rmsnorm_residual(x.float(), w)
    r = torch.zeros(4)
    with pytest.raises(ValueError, match="belong together"):
        P.rmsnorm_residual_backward(x, x, w, (r, None), y=x, w_post=w)
    with pytest.raises(ValueError, match="rstd"):
        P.rmsnorm_residual_backward(x, x, w, (r[:3], None))
    with pytest.raises(TypeError, match="CUDA"):
        P.rmsnorm_residual_backward(x, x, w, (r, None))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "vector", "row"])
def test_norm_gradient_formula(post, gate):
    """The restated gradient against central differences of the restated forward pass (f64: a step
    of 1e-6 leaves an error of about 1e-9)."""
    g = torch.Generator().manual_seed(7)
    rows, cols = 3, 16
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, y, w, wp = n(rows, cols), n(rows, cols), n(cols), n(cols) if post else None
    gt = {"none": None, "vector": n(cols), "row": n(rows, cols)}[gate]
    dn, du, s, eps = n(rows, cols), n(rows, cols), 0.7, 1e-6

    def loss(x, y, w, wp, gt):
        xo, _, _ = R.norm_forward(x, y, wp, gt, s, eps)
        return (R.norm_result(xo, w, eps)[0] * dn).sum() + (xo * du).sum()

    xo, _, ry = R.norm_forward(x, y, wp, gt, s, eps)
    rx = R.norm_result(xo, w, eps)[1]
    got = R.norm_backward(dn, du, xo, w, rx, y, wp, ry, gt, s)
    args = dict(x=x, y=y, w=w, wp=wp, gt=gt)
    for name, key in (("x", "dx"), ("y", "dy"), ("w", "dw"), ("wp", "dw_post"), ("gt", "dgate")):
        if args[name] is None:
            continue
        v, h = n(*args[name].shape), 1e-6
        d = (loss(**{**args, name: args[name] + h * v}) -
             loss(**{**args, name: args[name] - h * v})) / (2 * h)
        assert abs(float(d - (got[key][0] * v).sum())) < 1e-6 * (1 + abs(float(d))), name


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu", "gelu_tanh", "none"])
def test_act_gradient_formula(kind):
    x = torch.linspace(-6, 6, 401, dtype=torch.float64) + 1e-3
    h = 1e-6
    d = (R.act(x + h, kind) - R.act(x - h, kind)) / (2 * h)
    want = torch.ones_like(x) if kind == "none" else R.act_grad(x, kind)
    assert (d - want).abs().max() < 1e-8


def test_rounding_restatement():
    """The f64 element rounding equals torch's float8 casts on every exactly representable f32 and
    on ties, below saturation."""
    for fmt in ("e4m3", "e5m2"):
        codes = torch.arange(256, dtype=torch.uint8).view(R.F8[fmt]).float()
        v = codes[codes.isfinite()].sort().values
        x = torch.cat([v, (v[1:] + v[:-1]) / 2, (v[1:] * 0.7 + v[:-1] * 0.3)])
        assert torch.equal(R._round(x.double(), fmt).float(), x.to(R.F8[fmt]).float())
    assert C.sizeof(C.c_void_p) == 8


def test_no_non_coherent_loads_under_programmatic_launch():
    """A kernel launched with programmatic stream serialisation runs beside the one before it, which
    may still be writing what this one reads after griddepcontrol.wait (a bias, a gate, a weight
    vector). ld.global.nc asks for memory that nothing writes while the kernel runs, and the compiler
    may move such a load above the wait."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "ptx-std_b200", "csrc")
    for name in ("norm.cu", "act_backward.cu", "gemm_mx_fused.cu", "reduce.cuh", "mx_block.cuh",
                 "epilogue.cuh", "common.cuh"):
        with open(os.path.join(csrc, name)) as f:
            code = re.sub(r"//.*", "", f.read())
        assert not re.search(r"__ldg|global\.nc|__restrict__", code), name


def test_the_library_builds_without_torch(ptxstd_lib, monkeypatch, capsys):
    """The C library needs nvcc only; where torch is not installed the Python extension module is left
    out, with a word, and the build of the library still succeeds."""
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location(
        "ptxstd_build_test", os.path.join(root, "ptx-std_b200", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    before = os.path.getmtime(build.MODULE)
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec",
                        lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build_module(force=True) is None
    assert "torch" in capsys.readouterr().err
    assert os.path.getmtime(build.MODULE) == before
