"""The feed-forward operators on a B200 against their 64-bit restatements (ffn_ref).

Every stored value is held to an interval: the rounding of (exact - d) .. (exact + d). d counts the
f32 arithmetic only: the tensor cores' accumulation (ffn_ref.acc_bound), and 2^-19 of a value for
the chain of at most a dozen f32 operations and fast exponentials behind it (each within 2^-22).
"""

import ctypes as C
import math

import numpy as np
import pytest
import torch

import ffn_ref as R

pytestmark = pytest.mark.gpu

CHAIN = 2.0 ** -19


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bf(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _mx(g, rows, cols, fmt="e4m3", std=1.0):
    import ptxstd
    return ptxstd.quantize_mx(_bf(g, rows, cols, std=std), fmt, sf_layout=2)


def _ok():
    import ptxstd
    torch.cuda.synchronize()
    code, detail = ptxstd.last_device_error()
    assert code == 0, (code, hex(detail))


def _pad_nan(sf, rows, cols):
    """The same scales with NaN codes in the padding (which operators must not let through)."""
    sf = sf.clone()
    at = R.sf_offsets(rows, cols // 32, sf.device).reshape(-1)
    keep = sf[at].clone()
    sf.fill_(255)
    sf[at] = keep
    return sf


# ---- padded scales ------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (129, 160), (128, 128), (300, 416)])
def test_quantize_padded_layout(cuda, oracle, rows, cols):
    g = _gen(rows)
    x = _bf(g, rows, cols)
    import ptxstd
    for fmt, t in (("e4m3", oracle.E4M3), ("e2m1", oracle.E2M1)):
        q, sf = ptxstd.quantize_mx(x, fmt, sf_layout=2)
        oq, osf = oracle.quantize_mx(x.view(torch.int16).cpu().numpy().view(np.uint16), t)
        code, rest = R.sf_rowmajor(sf, rows, cols // 32)
        assert np.array_equal(q.cpu().numpy(), oq) and np.array_equal(code.cpu().numpy(), osf)
        assert not rest.any()


# ---- GEMM with an epilogue ----------------------------------------------------------------------
def _linear_case(M, N, K, act="none", bias=False, residual=False, out=None, at="e4m3", bt="e4m3",
                 pre=False, seed=0):
    import ptxstd
    g = _gen(seed + M + 3 * N + 7 * K)
    a, sfa = _mx(g, M, K, at)
    b, sfb = _mx(g, N, K, bt, std=K ** -0.5)
    sfa, sfb = _pad_nan(sfa, M, K), _pad_nan(sfb, N, K)
    bi = _bf(g, N) if bias else None
    re = _bf(g, M, N, std=4.0) if residual else None
    r = ptxstd.gemm_mx_epilogue(a, at, sfa, b, bt, sfb, bias=bi, act=act, residual=re,
                                elem_type=out, save_pre=pre)
    _ok()
    ref, mag = R.gemm(R.dequant(a, sfa, at), R.dequant(b, sfb, bt))
    d = R.acc_bound(mag, K)
    if bias:
        ref, d = ref + bi.double(), d + CHAIN * bi.double().abs()
    if pre:
        r, p = r
        R.check_bf16(p, ref, d + CHAIN * ref.abs(), "pre")
    # every activation here is at most 1.13-Lipschitz; |act(x)| <= |x|
    v = R.act(ref, act)
    d = 1.13 * d + CHAIN * ref.abs()
    if residual:
        v, d = v + re.double(), d + CHAIN * re.double().abs()
    if out is None:
        R.check_bf16(r, v, d, "c")
    else:
        R.check_mx(*r, v, d, out, what="c")


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 64, 65, 127, 128, 129, 200, 255, 256, 257, 511])
@pytest.mark.parametrize("N,K", [(8, 32), (136, 416), (384, 1056)])
def test_linear_sizes(cuda, M, N, K):
    _linear_case(M, N, K, bias=True, residual=True)


@pytest.mark.parametrize("M", [3, 130, 700])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_linear_activations(cuda, M, act):
    _linear_case(M, 288, 512, act=act, bias=True, pre=True)
    _linear_case(M, 288, 512, act=act, bias=True, residual=True, out="e4m3", pre=True)


@pytest.mark.parametrize("M,N,K", [(1, 32, 64), (33, 160, 96), (129, 4128, 2080), (256, 96, 4096),
                                   (300, 32, 160), (513, 1184, 1504)])
@pytest.mark.parametrize("out", ["e4m3", "e5m2"])
def test_linear_mx_result(cuda, M, N, K, out):
    _linear_case(M, N, K, out=out, at="e5m2", residual=True)


@pytest.mark.parametrize("M", [7, 290])
@pytest.mark.parametrize("at,bt", [("e5m2", "e4m3"), ("e2m3", "e3m2"), ("e2m1", "e4m3"),
                                   ("e4m3", "e2m1")])
def test_linear_element_types(cuda, oracle, M, at, bt):
    """Every kind of payload, held to the oracle's f64 product of the decoded operands."""
    import ptxstd
    N, K = 72, 160
    g = _gen(M)
    T = {"e4m3": oracle.E4M3, "e5m2": oracle.E5M2, "e2m3": oracle.E2M3, "e3m2": oracle.E3M2,
         "e2m1": oracle.E2M1}
    xa, xb = _bf(g, M, K), _bf(g, N, K)
    a, sfa = ptxstd.quantize_mx(xa, at, sf_layout=2)
    b, sfb = ptxstd.quantize_mx(xb, bt, sf_layout=2)
    c = ptxstd.gemm_mx_epilogue(a, at, sfa, b, bt, sfb)
    _ok()
    np16 = lambda t: t.view(torch.int16).cpu().numpy().view(np.uint16)  # noqa: E731
    oa, osa = oracle.quantize_mx(np16(xa), T[at])
    ob, osb = oracle.quantize_mx(np16(xb), T[bt])
    r, col = np.meshgrid(np.arange(M), np.arange(N), indexing="ij")
    ref, mag = oracle.gemm_mx_ref(oa, T[at], osa, ob, T[bt], osb, r.ravel(), col.ravel())
    ref, mag = (torch.from_numpy(np.asarray(v, dtype=np.float64)).view(M, N) for v in (ref, mag))
    R.check_bf16(c.cpu(), ref, R.acc_bound(mag, K))


@pytest.mark.parametrize("M", [4, 300])
def test_linear_both_results_and_residual_in_place(cuda, M):
    """d_c and d_q of one call agree; the residual may be the output; guard bytes stay."""
    import ptxstd
    N, K = 160, 224
    g = _gen(M)
    a, sfa = _mx(g, M, K)
    b, sfb = _mx(g, N, K, std=K ** -0.5)
    res = _bf(g, M, N)
    want = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, residual=res)
    wq, wsf = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, residual=res,
                                      elem_type="e4m3")
    guard = 4096
    c = torch.full((M * N + guard,), 7.0, dtype=torch.bfloat16, device="cuda")
    c[:M * N] = res.reshape(-1)
    q = torch.full((M * N + guard,), 77, dtype=torch.uint8, device="cuda")
    sf = torch.full((wsf.numel() + guard,), 77, dtype=torch.uint8, device="cuda")
    L = ptxstd.lib()
    st = L.ptxstd_gemm_mx_epilogue(a.data_ptr(), 0, sfa.data_ptr(), b.data_ptr(), 0, sfb.data_ptr(),
                                   None, 0, c.data_ptr(), c.data_ptr(), None, 0, q.data_ptr(),
                                   sf.data_ptr(), M, N, K, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    _ok()
    assert torch.equal(c[:M * N].view(M, N), want) and (c[M * N:] == 7).all()
    assert torch.equal(q[:M * N].view(M, N), wq) and (q[M * N:] == 77).all()
    assert torch.equal(sf[:wsf.numel()], wsf) and (sf[wsf.numel():] == 77).all()


@pytest.mark.parametrize("M", [20, 400])
def test_nan_and_infinity_stay_in_their_row(cuda, M):
    """A NaN scale in one row of A reaches that row of the result only, in bf16 and as MX codes
    (scale 255, elements NaN); infinite biases give infinite columns."""
    import ptxstd
    N, K = 96, 256
    g = _gen(3)
    a, sfa = _mx(g, M, K)
    b, sfb = _mx(g, N, K)
    clean = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb)
    bad = sfa.clone()
    bad[R.sf_offsets(M, K // 32)[13, 5]] = 255
    c = ptxstd.gemm_mx_epilogue(a, "e4m3", bad, b, "e4m3", sfb)
    q, sf = ptxstd.gemm_mx_epilogue(a, "e4m3", bad, b, "e4m3", sfb, elem_type="e4m3")
    bias = torch.zeros(N, dtype=torch.bfloat16, device="cuda")
    bias[5] = -math.inf
    ci = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, bias=bias)
    _ok()
    rows = torch.arange(M, device="cuda") != 13
    assert c[13].isnan().all() and torch.equal(c[rows], clean[rows])
    code, rest = R.sf_rowmajor(sf, M, N // 32)
    assert (code[13] == 255).all() and (code[rows] != 255).all() and not rest.any()
    assert ((q[13] & 127) == 127).all()
    cols = torch.arange(N, device="cuda") != 5
    assert (ci[:, 5] == -math.inf).all() and torch.equal(ci[:, cols], clean[:, cols])


def test_linear_long_k(cuda):
    """The down projection of one token and of a few (a long K, split over a cluster)."""
    _linear_case(1, 1024, 28672, residual=True)
    _linear_case(16, 264, 28672 - 32, bias=True)


# ---- gated projection ---------------------------------------------------------------------------
def _gated_case(M, F, K, act="silu", out=None, save=False, seed=0):
    import ptxstd
    g = _gen(seed + M + 3 * F + 7 * K)
    a, sfa = _mx(g, M, K)
    wg, sfg = _mx(g, F, K, std=K ** -0.5)
    wu, sfu = _mx(g, F, K, std=K ** -0.5)
    sfa, sfg, sfu = _pad_nan(sfa, M, K), _pad_nan(sfg, F, K), _pad_nan(sfu, F, K)
    r = ptxstd.gemm_mx_gated(a, "e4m3", sfa, wg, sfg, wu, sfu, "e4m3", act=act, elem_type=out,
                             save=save)
    _ok()
    av = R.dequant(a, sfa, "e4m3")
    gate, gm = R.gemm(av, R.dequant(wg, sfg, "e4m3"))
    up, um = R.gemm(av, R.dequant(wu, sfu, "e4m3"))
    dg, du = R.acc_bound(gm, K), R.acc_bound(um, K)
    if save:
        r, (sg, su) = r
        R.check_bf16(sg, gate, dg, "gate")
        R.check_bf16(su, up, du, "up")
    f = R.act(gate, act)
    df = 1.13 * dg + CHAIN * gate.abs()
    d = f.abs() * du + up.abs() * df + df * du + CHAIN * (f * up).abs()
    if out is None:
        R.check_bf16(r, f * up, d, "h")
    else:
        R.check_mx(*r, f * up, d, out, what="h")


@pytest.mark.parametrize("M", [1, 16, 31, 100, 128, 129, 250, 256, 257, 600])
@pytest.mark.parametrize("F,K", [(32, 32), (160, 224), (416, 1056)])
def test_gated_sizes(cuda, M, F, K):
    _gated_case(M, F, K, save=True)
    _gated_case(M, F, K, out="e4m3", save=M % 2 == 0)


@pytest.mark.parametrize("M", [9, 300])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh"])
def test_gated_activations(cuda, M, act):
    _gated_case(M, 128, 256, act=act)
    _gated_case(M, 128, 256, act=act, out="e5m2")


@pytest.mark.parametrize("M", [6, 270])
def test_gated_features_of_eight(cuda, M):
    _gated_case(M, 8, 64)
    _gated_case(M, 200, 96, save=True)


@pytest.mark.parametrize("M", [5, 300])
def test_gated_both_results(cuda, M):
    """d_h and d_q of one call, with the projections beside them (C ABI): as the separate calls."""
    import ptxstd
    F, K = 160, 224
    g = _gen(M)
    a, sfa = _mx(g, M, K)
    wg, sfg = _mx(g, F, K, std=K ** -0.5)
    wu, sfu = _mx(g, F, K, std=K ** -0.5)
    ops = (a, "e4m3", sfa, wg, sfg, wu, sfu, "e4m3")
    h, (gate, up) = ptxstd.gemm_mx_gated(*ops, save=True)
    q, sf = ptxstd.gemm_mx_gated(*ops, elem_type="e5m2")
    got = [torch.empty_like(t) for t in (h, gate, up, q, sf)]
    p = [t.data_ptr() for t in got]
    assert ptxstd.lib().ptxstd_gemm_mx_gated(
        a.data_ptr(), 0, sfa.data_ptr(), wg.data_ptr(), sfg.data_ptr(), wu.data_ptr(),
        sfu.data_ptr(), 0, 2, p[0], p[1], p[2], 1, p[3], p[4], M, F, K,
        torch.cuda.current_stream().cuda_stream) == 0
    _ok()
    for u, v in zip(got, (h, gate, up, q, sf)):
        assert torch.equal(u, v)


# ---- gradient of the activation, transposing quantiser ------------------------------------------
def _t(v):
    rows, cols = v.shape
    out = torch.zeros((cols, -(-rows // 32) * 32), dtype=v.dtype, device=v.device)
    out[:, :rows] = v.t()
    return out


@pytest.mark.parametrize("rows,cols", [(1, 32), (31, 64), (32, 96), (129, 160), (300, 416),
                                       (128, 2080)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_act_backward(cuda, rows, cols, gated, fmt):
    import ptxstd
    g = _gen(rows + cols)
    for act in ("silu", "gelu", "gelu_tanh", "relu", "none"):
        dh, gate = _bf(g, rows, cols, std=0.1), _bf(g, rows, cols, std=2.0)
        up = _bf(g, rows, cols) if gated else None
        row, col, db = ptxstd.act_backward_mx(dh, gate, up, act=act, elem_type=fmt, bias_grad=True)
        row2, col2 = ptxstd.act_backward_mx(dh, gate, up, act=act, elem_type=fmt)
        _ok()
        x = gate.double()
        df = torch.ones_like(x) if act == "none" else R.act_grad(x, act)
        d = dh.double() * df
        # f' is a sum of terms up to 1.2 in size, each within CHAIN
        e = 4 * CHAIN * dh.double().abs()
        if gated:
            u, f = up.double(), dh.double() * R.act(x, act)
            d, e = torch.cat([d * u, f], 1), torch.cat([e * u.abs(), e * x.abs()], 1)
        R.check_mx(*row, d, e, fmt, what=f"{act} rows")
        R.check_mx(*col, _t(d), _t(e), fmt, what=f"{act} columns")
        lim = e.sum(0) + d.abs().sum(0) * 2.0 ** -18
        assert ((db.double() - d.sum(0)).abs() <= lim).all()
        for p, q in zip(row + col, row2 + col2):
            assert torch.equal(p, q)


@pytest.mark.parametrize("rows,cols", [(1, 32), (129, 160)])
def test_act_backward_into_given_memory(cuda, rows, cols):
    """Outputs at 16-byte boundaries that are not 32-byte ones, with guards around (C ABI)."""
    import ptxstd
    g = _gen(rows)
    dh, gate, up = _bf(g, rows, cols), _bf(g, rows, cols), _bf(g, rows, cols)
    row, col = ptxstd.act_backward_mx(dh, gate, up, act="gelu")
    want = [*row, *col]
    buf = [torch.full((t.numel() + 96,), 77, dtype=torch.uint8, device="cuda") for t in want]
    assert ptxstd.lib().ptxstd_act_backward_mx(
        3, dh.data_ptr(), gate.data_ptr(), up.data_ptr(), rows, cols, 1,
        *[b.data_ptr() + 48 for b in buf], None, None, 0,
        torch.cuda.current_stream().cuda_stream) == 0
    xt = ptxstd.quantize_mx_t(dh, "e4m3")
    want += xt
    buf += [torch.full((t.numel() + 96,), 77, dtype=torch.uint8, device="cuda") for t in xt]
    assert ptxstd.lib().ptxstd_quantize_mx_t(
        dh.data_ptr(), rows, cols, 0, buf[4].data_ptr() + 48, buf[5].data_ptr() + 48,
        torch.cuda.current_stream().cuda_stream) == 0
    _ok()
    for b, t in zip(buf, want):
        assert torch.equal(b[48:-48], t.reshape(-1))
        assert (b[:48] == 77).all() and (b[-48:] == 77).all()


@pytest.mark.parametrize("rows,cols", [(1, 8), (32, 32), (33, 72), (200, 264), (1000, 136)])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantize_transposed(cuda, rows, cols, fmt):
    """Bit-exact: bf16 values times powers of two have one rounding."""
    import ptxstd
    x = _bf(_gen(rows), rows, cols, std=3.0)
    x[0, 0] = 0
    qt, sft = ptxstd.quantize_mx_t(x, fmt)
    _ok()
    R.check_mx(qt, sft, _t(x.double()), 0.0, fmt)
    if rows % 32 == 0:
        q, sf = ptxstd.quantize_mx(x.t().contiguous(), fmt, sf_layout=2)
        assert torch.equal(q, qt) and torch.equal(sf, sft)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_quantisers_agree_on_special_values(cuda, fmt):
    """NaN, infinities, subnormals, zeros, saturation: the transposing quantiser and the norm's and
    the GEMM's block quantiser give the codes of quantize_mx."""
    import ptxstd
    x = _bf(_gen(4), 128, 64, std=3.0)
    x[0, 0], x[33, 1], x[40, 2] = math.nan, math.inf, -math.inf
    x[:32, 3] = 0
    x[:32, 4] = torch.arange(32, device="cuda").to(torch.bfloat16) * 2.0 ** -130
    x[:32, 5] = torch.linspace(400, 500, 32, device="cuda").to(torch.bfloat16)
    x[:32, 6] = 3.3e38
    x[:32, 7] = 2.0 ** -126
    x[:32, 8] = -0.0
    qt, sft = ptxstd.quantize_mx_t(x, fmt)
    q, sf = ptxstd.quantize_mx(x.t().contiguous(), fmt, sf_layout=2)
    _ok()
    assert torch.equal(sft, sf) and torch.equal(qt, q)
    # D = dh exactly (no activation): rows quantised from registers
    (r, rsf), (c, csf) = ptxstd.act_backward_mx(x, torch.zeros_like(x), act="none", elem_type=fmt)
    q, sf = ptxstd.quantize_mx(x, fmt, sf_layout=2)
    _ok()
    assert torch.equal(rsf, sf) and torch.equal(r, q)
    assert torch.equal(csf, sft) and torch.equal(c, qt)


@pytest.mark.parametrize("M", [5, 300])
def test_gated_element_types(cuda, M):
    """FP6 and FP4 weights: equal to the products of the linear kernel with the same operands."""
    import ptxstd
    F, K = 96, 160
    g = _gen(M)
    a, sfa = _mx(g, M, K, "e5m2")
    for wt in ("e2m3", "e2m1"):
        wg, sfg = _mx(g, F, K, wt)
        wu, sfu = _mx(g, F, K, wt)
        h, (gate, up) = ptxstd.gemm_mx_gated(a, "e5m2", sfa, wg, sfg, wu, sfu, wt, act="none",
                                             save=True)
        lg = ptxstd.gemm_mx_epilogue(a, "e5m2", sfa, wg, wt, sfg)
        lu = ptxstd.gemm_mx_epilogue(a, "e5m2", sfa, wu, wt, sfu)
        _ok()
        # both accumulate the same products in f32; the tilings may differ, so one bf16 step
        for p, q in ((gate, lg), (up, lu)):
            assert ((p.double() - q.double()).abs() <= 2.0 ** -7 * q.double().abs() + 1e-30).all()
        R.check_bf16(h, gate.double() * up.double(), 2.0 ** -7 * (gate.double() * up.double()).abs())


def test_activation_extremes(cuda):
    """Saturated, tiny and infinite pre-activations: no NaN where the limit is finite."""
    import ptxstd
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 90.0, -90.0, 1e4, -1e4, 1e20, -1e20,
                      3e38, -3e38] + [0.5] * 18, device="cuda").to(torch.bfloat16)
    gate = v.repeat(4, 1)
    dh = torch.ones_like(gate)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        (q, sf), _ = ptxstd.act_backward_mx(dh, gate, act=act, elem_type="e4m3")
        _ok()
        got = R.dequant(q, sf, "e4m3")
        want = torch.where(gate.double() > 20, 1.0, 0.0)
        big = gate.double().abs() > 20
        assert torch.equal(got[big], want[big]), act
        assert got.isfinite().all()


# ---- norms --------------------------------------------------------------------------------------
def _norm_inputs(rows, cols, post, gate, seed=0):
    g = _gen(seed + rows + cols)
    x, y = _bf(g, rows, cols, std=2.0), _bf(g, rows, cols, std=0.7)
    x[:, ::17] *= 8
    w = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(torch.bfloat16)
    wp = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(torch.bfloat16) if post \
        else None
    gt = {"none": None, "vector": _bf(g, cols), "row": _bf(g, rows, cols)}[gate]
    return g, x, y, w, wp, gt


def _d(t):
    return None if t is None else t.double()


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 8192), (3, 256), (5, 480), (130, 1024),
                                       (7, 1056), (300, 2080), (2, 16384 + 32), (2, 32768)])
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "vector"), (True, "row"),
                                       (False, "vector")])
def test_norm_forward(cuda, rows, cols, post, gate):
    import ptxstd
    _, x, y, w, wp, gt = _norm_inputs(rows, cols, post, gate)
    eps, s = 1e-5, 0.5
    for fmt, layout in ((None, 1), ("e4m3", 1), ("e5m2", 0)):
        xo, n, (r, rp) = ptxstd.rmsnorm_residual(x, w, y=y, w_post=wp, gate=gt, scale=s, eps=eps,
                                                 elem_type=fmt, sf_layout=layout)
        _ok()
        ref, mag, ry = R.norm_forward(_d(x), _d(y), _d(wp), _d(gt), s, eps)
        R.check_bf16(xo, ref, CHAIN * mag, "x'")
        ref, rx = R.norm_result(xo.double(), _d(w), eps)
        assert ((r.double() - rx).abs() <= CHAIN * rx).all()
        assert (rp is None) == (not post)
        if post:
            assert ((rp.double() - ry).abs() <= CHAIN * ry).all()
        if fmt is None:
            R.check_bf16(n, ref, CHAIN * ref.abs(), "n")
        else:
            R.check_mx(*n, ref, CHAIN * ref.abs(), fmt, padded=layout == 1, what="n")


@pytest.mark.parametrize("rows,cols", [(592, 1056), (1037, 5152), (1500, 2048), (3000, 4096 + 32),
                                       (1600, 8192), (12000, 1056), (3100, 4064)])
@pytest.mark.parametrize("post,gate", [(True, "vector"), (True, "row"), (False, "row"),
                                       (False, "none")])
def test_norm_forward_many_rows(cuda, rows, cols, post, gate):
    """Enough rows for several per block; repeated and back to back, so that blocks of consecutive
    calls share SMs."""
    import ptxstd
    _, x, y, w, wp, gt = _norm_inputs(rows, cols, post, gate)
    eps, s = 1e-6, 0.5
    args = dict(y=y, w_post=wp, gate=gt, scale=s, eps=eps, elem_type="e4m3")
    runs = [ptxstd.rmsnorm_residual(x, w, **args) for _ in range(20)]
    _ok()
    for r in runs[1:]:
        for p, q in zip(_flat(runs[0]), _flat(r)):
            assert torch.equal(p, q)
    xo, n, (r, rp) = runs[0]
    ref, mag, _ = R.norm_forward(_d(x), _d(y), _d(wp), _d(gt), s, eps)
    R.check_bf16(xo, ref, CHAIN * mag, "x'")
    ref, rx = R.norm_result(xo.double(), _d(w), eps)
    assert ((r.double() - rx).abs() <= CHAIN * rx).all()
    R.check_mx(*n, ref, CHAIN * ref.abs(), "e4m3", what="n")
    plain = ptxstd.rmsnorm_residual(x, w)[1]
    _ok()
    ref = R.norm_result(_d(x), _d(w), 1e-6)[0]
    R.check_bf16(plain, ref, CHAIN * ref.abs(), "plain")


@pytest.mark.parametrize("rows,cols", [(3000, 1056), (1100, 8192), (2000, 4096)])
@pytest.mark.parametrize("gate", ["vector", "row"])
def test_norm_backward_many_rows(cuda, rows, cols, gate):
    import ptxstd
    g, xo, y, w, wp, gt = _norm_inputs(rows, cols, True, gate)
    dn, du = _bf(g, rows, cols, std=0.3), _bf(g, rows, cols, std=0.3)
    rx = torch.rsqrt(xo.double().square().mean(1) + 1e-6).float()
    ry = torch.rsqrt(y.double().square().mean(1) + 1e-6).float()
    runs = [ptxstd.rmsnorm_residual_backward(dn, xo, w, (rx, ry), dx_out=du, y=y, w_post=wp,
                                             gate=gt, scale=0.5) for _ in range(20)]
    _ok()
    for r in runs[1:]:
        for p, q in zip(runs[0], r):
            assert torch.equal(p, q)
    dx, dw, dy, dwp, dg = runs[0]
    ref = R.norm_backward(_d(dn), _d(du), _d(xo), _d(w), _d(rx), _d(y), _d(wp), _d(ry), _d(gt),
                          0.5)
    R.check_bf16(dx, ref["dx"][0], CHAIN * ref["dx"][1], "dx")
    R.check_bf16(dy, ref["dy"][0], 4 * CHAIN * ref["dy"][1], "dy")
    terms = CHAIN + (rows / 148 + 200) * 2.0 ** -24
    for name, got in (("dw", dw), ("dw_post", dwp)):
        assert ((got.double() - ref[name][0]).abs() <= 4 * terms * ref[name][1]).all(), name


def test_norm_without_branch(cuda):
    """No y: x' is x; columns that are not a multiple of 32 in bf16; a zero row stays zero."""
    import ptxstd
    _, x, _, w, _, _ = _norm_inputs(70, 40, False, "none")
    x[3] = 0
    xo, n, (r, rp) = ptxstd.rmsnorm_residual(x, w, eps=1e-6)
    _ok()
    assert xo is x and rp is None and not n[3].any() and float(r[3]) == pytest.approx(1e3, rel=1e-5)
    R.check_bf16(n, R.norm_result(_d(x), _d(w), 1e-6)[0], CHAIN * 200.0, "n")
    with pytest.raises(ptxstd.PtxStdError):
        ptxstd.rmsnorm_residual(x, w, elem_type="e4m3")  # 40 % 32
    # NaN stays in its row
    x[5, 7] = math.nan
    n2 = ptxstd.rmsnorm_residual(x, w, eps=1e-6)[1]
    keep = torch.arange(70, device="cuda") != 5
    assert n2[5].isnan().all() and torch.equal(n2[keep], n[keep])


def test_norm_in_place(cuda):
    """x' may be written over x (C ABI)."""
    import ptxstd
    _, x, y, w, wp, gt = _norm_inputs(9, 512, True, "vector")
    want = ptxstd.rmsnorm_residual(x, w, y=y, w_post=wp, gate=gt, scale=2.0)
    n = torch.empty_like(x)
    st = ptxstd.lib().ptxstd_rmsnorm_residual(
        x.data_ptr(), y.data_ptr(), wp.data_ptr(), gt.data_ptr(), 1, 2.0, w.data_ptr(), 1e-6, 9,
        512, x.data_ptr(), n.data_ptr(), 0, None, None, 1, None, None,
        torch.cuda.current_stream().cuda_stream)
    assert st == 0
    _ok()
    assert torch.equal(x, want[0]) and torch.equal(n, want[1])


@pytest.mark.parametrize("rows,cols", [(3100, 4064), (1600, 8192), (500, 1056)])
def test_norm_in_place_many_rows(cuda, rows, cols):
    """x' over x, n in both forms at once (C ABI): as the separate calls give them."""
    import ptxstd
    _, x, y, w, wp, gt = _norm_inputs(rows, cols, True, "row")
    args = dict(y=y, w_post=wp, gate=gt, scale=2.0)
    xo, n, _ = ptxstd.rmsnorm_residual(x, w, **args)
    (q, sf) = ptxstd.rmsnorm_residual(x, w, elem_type="e4m3", **args)[1]
    n2, q2, sf2 = torch.empty_like(n), torch.empty_like(q), torch.empty_like(sf)
    st = ptxstd.lib().ptxstd_rmsnorm_residual(
        x.data_ptr(), y.data_ptr(), wp.data_ptr(), gt.data_ptr(), rows, 2.0, w.data_ptr(), 1e-6,
        rows, cols, x.data_ptr(), n2.data_ptr(), 0, q2.data_ptr(), sf2.data_ptr(), 1, None, None,
        torch.cuda.current_stream().cuda_stream)
    assert st == 0
    _ok()
    for p, r in ((x, xo), (n2, n), (q2, q), (sf2, sf)):
        assert torch.equal(p, r)


@pytest.mark.parametrize("rows,cols", [(40, 480), (700, 4096), (300, 8192), (5, 8192 + 32)])
def test_norm_backward_in_place(cuda, rows, cols):
    """dx may be written over dx_out (C ABI)."""
    import ptxstd
    g, xo, y, w, wp, gt = _norm_inputs(rows, cols, True, "vector")
    dn, du = _bf(g, rows, cols), _bf(g, rows, cols)
    _, _, st = ptxstd.rmsnorm_residual(xo, w, y=y, w_post=wp, gate=gt)
    want = ptxstd.rmsnorm_residual_backward(dn, xo, w, st, dx_out=du, y=y, w_post=wp, gate=gt)
    got = [du] + [torch.empty_like(t) for t in want[1:]]
    L = ptxstd.lib()
    nb = L.ptxstd_rmsnorm_residual_backward_workspace_bytes(rows, cols)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    ptr = [t.data_ptr() for t in (dn, du, xo, w, st[0], y, wp, st[1], gt)]
    assert L.ptxstd_rmsnorm_residual_backward(
        *ptr, 1, 1.0, rows, cols, *[t.data_ptr() for t in got], ws.data_ptr(), nb,
        torch.cuda.current_stream().cuda_stream) == 0
    _ok()
    for p, r in zip(got, want):
        assert torch.equal(p, r)


@pytest.mark.parametrize("rows,cols", [(1, 32), (2, 40), (5, 480), (300, 1056), (1200, 256),
                                       (9, 4096 + 32), (160, 8192), (5, 8192 + 32), (3, 16384)])
@pytest.mark.parametrize("post,gate,du", [(False, "none", True), (True, "vector", True),
                                          (True, "row", False), (False, "row", True)])
def test_norm_backward(cuda, rows, cols, post, gate, du):
    import ptxstd
    g, xo, y, w, wp, gt = _norm_inputs(rows, cols, post, gate)
    dn = _bf(g, rows, cols, std=0.3)
    dxo = _bf(g, rows, cols, std=0.3) if du else None
    rx = torch.rsqrt(xo.double().square().mean(1) + 1e-6).float()
    ry = torch.rsqrt(y.double().square().mean(1) + 1e-6).float() if post else None
    dx, dw, dy, dwp, dg = ptxstd.rmsnorm_residual_backward(
        dn, xo, w, (rx, ry), dx_out=dxo, y=y, w_post=wp, gate=gt, scale=0.5)
    again = ptxstd.rmsnorm_residual_backward(
        dn, xo, w, (rx, ry), dx_out=dxo, y=y, w_post=wp, gate=gt, scale=0.5)
    _ok()
    ref = R.norm_backward(_d(dn), _d(dxo), _d(xo), _d(w), _d(rx), _d(y), _d(wp), _d(ry), _d(gt),
                          0.5)
    # the f32 sums over a row add at most 32 terms per thread, then over at most 512 threads in a
    # tree: 41 roundings of 2^-24, under CHAIN of the terms' magnitudes; column sums over at most
    # rows / CTAs + CTAs / 8 + 8 terms, 2^-24 each
    R.check_bf16(dx, ref["dx"][0], CHAIN * ref["dx"][1], "dx")
    R.check_bf16(dy, ref["dy"][0], 4 * CHAIN * ref["dy"][1], "dy")
    terms = CHAIN + (rows / 148 + 200) * 2.0 ** -24
    for name, got in (("dw", dw), ("dw_post", dwp)):
        if got is None:
            assert name not in ref
            continue
        assert got.dtype == torch.float32
        assert ((got.double() - ref[name][0]).abs() <= 4 * terms * ref[name][1]).all(), name
    if gate == "vector":
        assert dg.dtype == torch.float32
        assert ((dg.double() - ref["dgate"][0]).abs() <= 4 * terms * ref["dgate"][1]).all()
    elif gate == "row":
        if rows == 1:  # through the column sum, then rounded
            ref["dgate"] = (ref["dgate"][0].view(1, -1), ref["dgate"][1].view(1, -1))
        R.check_bf16(dg, ref["dgate"][0], 4 * CHAIN * ref["dgate"][1], "dgate")
    else:
        assert dg is None
    for p, q in zip((dx, dw, dy, dwp, dg), again):
        assert p is q is None or torch.equal(p, q)


@pytest.mark.parametrize("rows,cols", [(70, 480), (330, 1056), (300, 8192), (3, 8192 + 32)])
@pytest.mark.parametrize("px,py", [(50, 50), (-50, -50), (50, -50), (-50, 50), (0, 50), (-50, 0)])
@pytest.mark.parametrize("gate", ["vector", "row"])
def test_norm_backward_of_large_and_tiny_rows(cuda, rows, cols, px, py, gate):
    """Rows around 2^50 and 2^-50, whose norms are exact in f32 and whose cubed factors are not
    representable in it. The tolerances are those of test_norm_backward: powers of two change no
    rounding, and every product of the formulas, with the factors next to their rows, stays between
    2^-126 and 2^127 (at most |t x'| summed: 2^(100 + 13 + 10)). A sum's terms below the others by
    more than 2^24 only lose what CHAIN allows of the magnitudes."""
    import ptxstd
    g, xo, y, w, wp, gt = _norm_inputs(rows, cols, True, gate)
    xo, y = xo * 2.0 ** px, y * 2.0 ** py
    dn, du = _bf(g, rows, cols, std=0.3), _bf(g, rows, cols, std=0.3)
    rx = torch.rsqrt(xo.double().square().mean(1)).float()
    ry = torch.rsqrt(y.double().square().mean(1)).float()
    for dxo in (None, du):
        dx, dw, dy, dwp, dg = ptxstd.rmsnorm_residual_backward(
            dn, xo, w, (rx, ry), dx_out=dxo, y=y, w_post=wp, gate=gt, scale=0.5)
        _ok()
        ref = R.norm_backward(_d(dn), _d(dxo), _d(xo), _d(w), _d(rx), _d(y), _d(wp), _d(ry),
                              _d(gt), 0.5)
        R.check_bf16(dx, ref["dx"][0], CHAIN * ref["dx"][1], "dx")
        R.check_bf16(dy, ref["dy"][0], 4 * CHAIN * ref["dy"][1], "dy")
        terms = CHAIN + (rows / 148 + 200) * 2.0 ** -24
        for name, got in (("dw", dw), ("dw_post", dwp)):
            assert ((got.double() - ref[name][0]).abs() <= 4 * terms * ref[name][1]).all(), name
        if gate == "row":
            R.check_bf16(dg, ref["dgate"][0], 4 * CHAIN * ref["dgate"][1], "dgate")
        else:
            lim = 4 * terms * ref["dgate"][1]
            assert ((dg.double() - ref["dgate"][0]).abs() <= lim).all()


def test_norm_gradient_against_differences(cuda):
    """The kernels' gradients along a direction against the central difference of the 64-bit
    forward pass: they differ by the gradients' bf16 rounding, 2^-8 of each entry."""
    import ptxstd
    rows, cols, s, eps = 4, 512, 0.5, 1e-6
    g, x, y, w, wp, gt = _norm_inputs(rows, cols, True, "vector")
    dn, du = _bf(g, rows, cols, std=0.3), _bf(g, rows, cols, std=0.3)
    # the stored x' is the point of expansion, so start from an x for which x' needs no rounding
    p, _, ry = R.norm_forward(torch.zeros_like(_d(x)), _d(y), _d(wp), _d(gt), s, eps)
    xo = x
    x64 = _d(xo) - p
    rx = R.norm_result(_d(xo), _d(w), eps)[1]
    got = ptxstd.rmsnorm_residual_backward(dn, xo, w, (rx.float(), ry.float()), dx_out=du, y=y,
                                           w_post=wp, gate=gt, scale=s)
    args = [x64, _d(w), _d(y), _d(wp), _d(gt)]

    def loss(x, w, y, wp, gt):
        o = R.norm_forward(x, y, wp, gt, s, eps)[0]
        return (R.norm_result(o, w, eps)[0] * _d(dn)).sum() + (o * _d(du)).sum()

    for k in range(5):
        v = torch.randn(args[k].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-6
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * v, args[k] - h * v
        d = float(loss(*up) - loss(*down)) / (2 * h)
        e = float((got[k].double() * v).sum())
        assert abs(d - e) <= 2.0 ** -8 * float((got[k].double() * v).abs().sum()) + 1e-4 * abs(d)


# ---- together -----------------------------------------------------------------------------------
class Block:
    """norm -> gated projection -> down projection onto the residual stream, and its backward."""

    def __init__(self, M, D, F, seed=1):
        import ptxstd
        g = _gen(seed)
        self.P, self.M, self.D, self.F = ptxstd, M, D, F
        self.x, self.y = _bf(g, M, D, std=2.0), _bf(g, M, D)
        self.w, self.wp, self.gate = _bf(g, D), _bf(g, D), _bf(g, D)
        self.wg = _bf(g, F, D, std=D ** -0.5)
        self.wu = _bf(g, F, D, std=D ** -0.5)
        self.wd = _bf(g, D, F, std=F ** -0.5)
        q = lambda t: ptxstd.quantize_mx(t, "e4m3", sf_layout=2)  # noqa: E731
        self.qg, self.qu, self.qd = q(self.wg), q(self.wu), q(self.wd)
        self.gut = q(torch.cat([self.wg, self.wu]).t().contiguous())
        self.dt = q(self.wd.t().contiguous())
        self.dout = _bf(g, M, D, std=0.1)

    def forward(self):
        P = self.P
        xo, n, st = P.rmsnorm_residual(self.x, self.w, y=self.y, w_post=self.wp, gate=self.gate,
                                       scale=0.5, elem_type="e4m3")
        h, (g, u) = P.gemm_mx_gated(n[0], "e4m3", n[1], self.qg[0], self.qg[1], self.qu[0],
                                    self.qu[1], "e4m3", elem_type="e4m3", save=True)
        out = P.gemm_mx_epilogue(h[0], "e4m3", h[1], self.qd[0], "e4m3", self.qd[1], residual=xo)
        return xo, n, st, h, g, u, out

    def backward(self, xo, n, st, h, g, u, out):
        P = self.P
        dq, dsf = P.quantize_mx(self.dout, "e5m2", sf_layout=2)
        dh = P.gemm_mx_epilogue(dq, "e5m2", dsf, self.dt[0], "e4m3", self.dt[1])
        nb = P.rmsnorm_residual(xo, self.w)[1]
        nt, sfnt = P.quantize_mx_t(nb, "e4m3")
        dn, dw = P.gemm_mx_gated_backward(dh, g, u, nt, "e4m3", sfnt, self.gut[0], "e4m3",
                                          self.gut[1])
        return (dh, dn, dw) + P.rmsnorm_residual_backward(
            dn, xo, self.w, st, dx_out=self.dout, y=self.y, w_post=self.wp, gate=self.gate,
            scale=0.5)


def _flat(v):
    return [t for x in v for t in (_flat(x) if isinstance(x, (tuple, list)) else [x])
            if t is not None]


@pytest.mark.parametrize("M", [1, 40, 333])
def test_block_stage_by_stage(cuda, M):
    """A whole feed-forward block forward and backward, launched without a wait in between; every
    stage is then held to its restatement on the stage's own stored inputs."""
    b = Block(M, 256, 416)
    f = b.forward()
    xo, n, st, h, g, u, out = f
    dh, dn, dw, dx, dnw, dy, dwp, dgate = b.backward(*f)
    _ok()
    D, F = b.D, b.F
    a = R.dequant(*n, "e4m3")
    gate, gm = R.gemm(a, R.dequant(*b.qg, "e4m3"))
    R.check_bf16(g, gate, R.acc_bound(gm, D), "gate")
    c, cm = R.gemm(R.dequant(*h, "e4m3"), R.dequant(*b.qd, "e4m3"))
    R.check_bf16(out, c + _d(xo), R.acc_bound(cm, F) + CHAIN * _d(xo).abs(), "out")
    # backward: the quantised gradient follows from the stored dh, gate, up
    (q, sf), (qt, sft) = b.P.act_backward_mx(dh, g, u)
    c, cm = R.gemm(R.dequant(q, sf, "e5m2"), R.dequant(*b.gut, "e4m3"))
    R.check_bf16(dn, c, R.acc_bound(cm, 2 * F), "dn")
    nt = b.P.quantize_mx_t(b.P.rmsnorm_residual(xo, b.w)[1], "e4m3")
    c, cm = R.gemm(R.dequant(qt, sft, "e5m2"), R.dequant(*nt, "e4m3"))
    R.check_bf16(dw, c, R.acc_bound(cm, -(-M // 32) * 32), "dw")
    ref = R.norm_backward(_d(dn), _d(b.dout), _d(xo), _d(b.w), _d(st[0]), _d(b.y), _d(b.wp),
                          _d(st[1]), _d(b.gate), 0.5)
    R.check_bf16(dx, ref["dx"][0], CHAIN * ref["dx"][1], "dx")
    R.check_bf16(dy, ref["dy"][0], 4 * CHAIN * ref["dy"][1], "dy")


@pytest.mark.parametrize("M", [1, 40, 333])
def test_training_step_as_documented(cuda, M):
    """The calls of the documented training step (n and h in bf16, then both quantisers), with the down
    projection's weight gradient; that one and dh held to their restatement on the stored operands."""
    import ptxstd
    b = Block(M, 256, 416, seed=31)
    x1, n, stats = ptxstd.rmsnorm_residual(b.x, b.w, y=b.y, w_post=b.wp, gate=b.gate, scale=0.5)
    q, sf = ptxstd.quantize_mx(n, "e4m3", sf_layout=2)
    h, kept = ptxstd.gemm_mx_gated(q, "e4m3", sf, *b.qg, *b.qu, "e4m3", save=True)
    hq, hsf = ptxstd.quantize_mx(h, "e4m3", sf_layout=2)
    out = ptxstd.gemm_mx_epilogue(hq, "e4m3", hsf, b.qd[0], "e4m3", b.qd[1], residual=x1)
    dq, dsf = ptxstd.quantize_mx(b.dout, "e5m2", sf_layout=2)
    dh = ptxstd.gemm_mx_epilogue(dq, "e5m2", dsf, b.dt[0], "e4m3", b.dt[1])
    dqt, dsft = ptxstd.quantize_mx_t(b.dout, "e5m2")
    ht, hsft = ptxstd.quantize_mx_t(h, "e4m3")
    dwd = ptxstd.gemm_mx_epilogue(dqt, "e5m2", dsft, ht, "e4m3", hsft)
    nt, sfnt = ptxstd.quantize_mx_t(n, "e4m3")
    dn, dwgu = ptxstd.gemm_mx_gated_backward(dh, *kept, nt, "e4m3", sfnt, b.gut[0], "e4m3",
                                             b.gut[1])
    dx, dw, dy, dwp, dg = ptxstd.rmsnorm_residual_backward(
        dn, x1, b.w, stats, dx_out=b.dout, y=b.y, w_post=b.wp, gate=b.gate, scale=0.5)
    _ok()
    assert out.shape == dx.shape == dy.shape == (M, b.D) and dwd.shape == (b.D, b.F)
    assert dwgu.shape == (2 * b.F, b.D) and dw.shape == dwp.shape == dg.shape == (b.D,)
    R.check_mx(dqt, dsft, _t(_d(b.dout)), 0.0, "e5m2", what="dout^T")
    R.check_mx(ht, hsft, _t(_d(h)), 0.0, "e4m3", what="h^T")
    rows = dqt.shape[1]
    c, cm = R.gemm(R.dequant(dqt, dsft, "e5m2"), R.dequant(ht, hsft, "e4m3"))
    R.check_bf16(dwd, c, R.acc_bound(cm, rows), "dwd")
    c, cm = R.gemm(R.dequant(dq, dsf, "e5m2"), R.dequant(*b.dt, "e4m3"))
    R.check_bf16(dh, c, R.acc_bound(cm, b.D), "dh")


def test_block_gradients_follow_the_exact_ones(cuda):
    """End to end against autograd of the unquantised block in 64 bits. A check of signs and factors,
    not of rounding: E4M3 / E5M2 operands carry up to 2^-4 and 2^-3 of relative rounding each
    (and 2^-3 where a block saturates), independent over the entries of each product, so the
    gradients keep a cosine well above 0.99 to the exact ones and a norm within 5 %."""
    b = Block(256, 256, 512, seed=5)
    f = b.forward()
    dh, dn, dw, dx, dnw, dy, dwp, dgate = b.backward(*f)
    _ok()
    v = {k: _d(getattr(b, k)).requires_grad_(True)
         for k in ("x", "y", "w", "wp", "gate", "wg", "wu", "wd")}
    xo = R.norm_forward(v["x"], v["y"], v["wp"], v["gate"], 0.5, 1e-6)[0]
    n = R.norm_result(xo, v["w"], 1e-6)[0]
    out = xo + (R.act(n @ v["wg"].t(), "silu") * (n @ v["wu"].t())) @ v["wd"].t()
    out.backward(_d(b.dout))
    want = {"dx": v["x"].grad, "dy": v["y"].grad, "dw": v["w"].grad, "dwp": v["wp"].grad,
            "dgate": v["gate"].grad, "dwgu": torch.cat([v["wg"].grad, v["wu"].grad])}
    got = {"dx": dx, "dy": dy, "dw": dnw, "dwp": dwp, "dgate": dgate, "dwgu": dw}
    for k, w in want.items():
        p, q = got[k].double().reshape(-1), w.reshape(-1)
        cos = float(p @ q / (p.norm() * q.norm()))
        assert cos > 0.99 and abs(float(p.norm() / q.norm()) - 1) < 0.05, (k, cos)


@pytest.mark.parametrize("M", [3, 300])
def test_captured_and_replayed(cuda, M):
    """Forward and backward captured into one CUDA graph; replays on changed inputs equal eager
    calls on them, bit for bit."""
    b = Block(M, 256, 416, seed=9)
    b.backward(*b.forward())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            f = b.forward()
            r = b.backward(*f)
    torch.cuda.current_stream().wait_stream(s)
    for k in range(2):
        b.x.copy_(_bf(_gen(50 + k), M, b.D, std=2.0))
        b.dout.copy_(_bf(_gen(60 + k), M, b.D, std=0.1))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in _flat((f, r))]
        ef = b.forward()
        eager = _flat((ef, b.backward(*ef)))
        _ok()
        for p, q in zip(replayed, eager):
            assert torch.equal(p, q)


def test_two_streams_at_once(cuda):
    """Blocks of both kernels (few rows, many rows) running on two streams give the results that
    they give alone."""
    blocks = [Block(5, 512, 1024, seed=3), Block(300, 512, 1024, seed=4),
              Block(140, 512, 1024, seed=6)]
    alone = []
    for b in blocks:
        f = b.forward()
        alone.append([t.clone() for t in _flat((f, b.backward(*f)))])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    got = [None] * len(blocks)
    for _ in range(5):
        for i, (b, s) in enumerate(zip(blocks, streams)):
            with torch.cuda.stream(s):
                f = b.forward()
                got[i] = _flat((f, b.backward(*f)))
    _ok()
    for want, have in zip(alone, got):
        for p, q in zip(want, have):
            assert torch.equal(p, q)


# ---- offsets past 32 bits -------------------------------------------------------------------------
def _tiled(block, rows):
    """`block` repeated over `rows` rows (contiguous)."""
    reps = -(-rows // block.shape[0])
    return block.repeat(reps, 1)[:rows].contiguous()


def test_norm_offsets_past_32_bits(cuda):
    """2.2e9 elements: the last rows (byte and element offsets past 2^32 and 2^31) against the
    restatement, the column sums against those of the repeated block."""
    import ptxstd
    period, reps, cols = 1024, 262, 8192
    rows = period * reps
    assert rows * cols > 1 << 31
    g = _gen(1)
    xb, yb, dnb = (_bf(g, period, cols, std=s) for s in (2.0, 0.7, 0.3))
    w, wp, gt = (_bf(g, cols) for _ in range(3))
    x, y = _tiled(xb, rows), _tiled(yb, rows)
    xo, (q, sf), st = ptxstd.rmsnorm_residual(x, w, y=y, w_post=wp, gate=gt, scale=0.5,
                                              elem_type="e4m3")
    _ok()
    tail = slice(rows - 256, rows)
    ref, mag, _ = R.norm_forward(_d(x[tail]), _d(y[tail]), _d(wp), _d(gt), 0.5, 1e-6)
    R.check_bf16(xo[tail], ref, CHAIN * mag, "x'")
    ref, _ = R.norm_result(_d(xo[tail]), _d(w), 1e-6)
    R.check_mx(q[tail], sf[-2 * 64 * 512:], ref, CHAIN * ref.abs(), "e4m3", what="n")
    del q, sf, x
    dn = _tiled(dnb, rows)
    dx, dw, dy, dwp, dg = ptxstd.rmsnorm_residual_backward(dn, xo, w, st, y=y, w_post=wp, gate=gt,
                                                           scale=0.5)
    _ok()
    ref = R.norm_backward(_d(dn[tail]), None, _d(xo[tail]), _d(w), _d(st[0][tail]), _d(y[tail]),
                          _d(wp), _d(st[1][tail]), _d(gt), 0.5)
    R.check_bf16(dx[tail], ref["dx"][0], CHAIN * ref["dx"][1], "dx")
    R.check_bf16(dy[tail], ref["dy"][0], 4 * CHAIN * ref["dy"][1], "dy")
    one = R.norm_backward(_d(dnb), None, _d(xo[:period]), _d(w), _d(st[0][:period]), _d(yb), _d(wp),
                          _d(st[1][:period]), _d(gt), 0.5)
    terms = CHAIN + (rows / 148 + 200) * 2.0 ** -24
    for name, got in (("dw", dw), ("dw_post", dwp), ("dgate", dg)):
        want, mag = one[name][0] * reps, one[name][1] * reps
        assert ((got.double() - want).abs() <= 4 * terms * mag).all(), name


def test_act_backward_offsets_past_32_bits(cuda):
    """The last 128 rows of 2.2e9 elements equal a call on those rows alone, bit for bit, in both
    operands (tiles do not depend on one another)."""
    import ptxstd
    cols, rows = 16384, 128 * 1056
    assert rows * cols > 1 << 31
    g = _gen(2)
    dh, gate = _tiled(_bf(g, 640, cols, std=0.1), rows), _tiled(_bf(g, 896, cols, std=2.0), rows)
    (q, sf), (qt, sft) = ptxstd.act_backward_mx(dh, gate, act="silu", elem_type="e4m3")
    a, b = dh[-128:].contiguous(), gate[-128:].contiguous()
    (q1, sf1), (qt1, sft1) = ptxstd.act_backward_mx(a, b, act="silu", elem_type="e4m3")
    _ok()
    assert torch.equal(q[-128:], q1) and torch.equal(qt[:, -128:], qt1)
    assert torch.equal(sf[-sf1.numel():], sf1)
    # the transposed scales: the last of each row tile's 512-byte tiles
    assert torch.equal(sft.view(cols // 128, -1, 512)[:, -1], sft1.view(cols // 128, 512))


def test_linear_offsets_past_32_bits(cuda):
    """A result of 2.2e9 elements with a residual: its first and last rows."""
    import ptxstd
    M, N, K = 270336, 8192, 64
    assert M * N > 1 << 31
    g = _gen(3)
    a, sfa = _mx(g, M, K)
    b, sfb = _mx(g, N, K, std=K ** -0.5)
    res = _tiled(_bf(g, 1024, N), M)
    c = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, residual=res)
    _ok()
    bv = R.dequant(b, sfb, "e4m3")
    for rows, tiles in ((slice(0, 256), slice(0, 2 * 512)), (slice(M - 256, M), slice(-2 * 512, None))):
        ref, mag = R.gemm(R.dequant(a[rows], sfa[tiles], "e4m3"), bv)
        r = _d(res[rows])
        R.check_bf16(c[rows], ref + r, R.acc_bound(mag, K) + CHAIN * (ref.abs() + r.abs()), "c")


def test_two_host_threads_at_once(cuda):
    """Concurrent calls from two threads, each on a stream of its own."""
    import threading
    blocks = [Block(3, 512, 1024, seed=21), Block(300, 512, 1024, seed=22)]
    want = [_flat((f, b.backward(*f))) for b in blocks for f in [b.forward()]]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    f = blocks[i].forward()
                    got[i] = _flat((f, blocks[i].backward(*f)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    _ok()
    assert not errors
    for p, q in zip(want, got):
        assert len(p) == len(q) and all(torch.equal(u, v) for u, v in zip(p, q))


def test_first_calls_are_captured(cuda):
    """In a new process the first call of every operator may be one under graph capture."""
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = sys.argv[1:]
import torch
import test_ffn_gpu as T
b = T.Block(300, 256, 512)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    f = b.forward()
    r = T._flat((f, b.backward(*f)))
g.replay()
torch.cuda.synchronize()
f = b.forward()
e = T._flat((f, b.backward(*f)))
T._ok()
assert len(r) == len(e) and all(torch.equal(p, q) for p, q in zip(r, e))
"""
    r = subprocess.run([sys.executable, "-c", code] + sys.path, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_stream_argument(cuda):
    """Calls on a stream that is not the current one: right results, with the caller's own work on
    the current stream reusing freed memory meanwhile."""
    import ptxstd
    rows, cols = 2000, 4096
    g, xo, y, w, wp, gt = _norm_inputs(rows, cols, True, "vector")
    dn = _bf(g, rows, cols)
    rx = torch.rsqrt(xo.double().square().mean(1) + 1e-6).float()
    ry = torch.rsqrt(y.double().square().mean(1) + 1e-6).float()
    args = dict(y=y, w_post=wp, gate=gt, scale=0.5)
    want = ptxstd.rmsnorm_residual_backward(dn, xo, w, (rx, ry), **args)
    want_db = ptxstd.act_backward_mx(dn, xo, act="gelu", bias_grad=True)[2]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(10):
        got = ptxstd.rmsnorm_residual_backward(dn, xo, w, (rx, ry), stream=s, **args)
        db = ptxstd.act_backward_mx(dn, xo, act="gelu", bias_grad=True, stream=s)[2]
        for _ in range(4):  # takes any block the calls gave back to the current stream
            torch.full((8 << 20,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for p, q in zip(want, got):
            assert torch.equal(p, q)
        assert torch.equal(db, want_db)
    _ok()


def test_beside_the_other_gemms(cuda):
    """The operators on one stream while the framework's other tensor-core kernels, which take all
    of an SM's TMEM, run on another: everything finishes with the results it has alone."""
    import ptxstd
    b1, b2 = Block(7, 512, 1024, seed=11), Block(400, 512, 1024, seed=12)
    want = [[t.clone() for t in _flat(b.forward())] for b in (b1, b2)]
    g = _gen(5)
    a, sfa = ptxstd.quantize_mx(_bf(g, 512, 1024), "e4m3", sf_layout=1)
    x = _bf(g, 16, 2048)
    w4, sf4 = ptxstd.quantize_nvfp4(_bf(g, 1024, 2048, std=0.02), 0.02 / 448, sf_layout=1)
    c0 = ptxstd.gemm_mx(a, "e4m3", sfa, a, "e4m3", sfa).clone()
    y0 = ptxstd.gemm_decode(x, w4, sf4, 0.02 / 448).clone()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            got = [_flat(b.forward()) for b in (b1, b2)]
        with torch.cuda.stream(s2):
            c = ptxstd.gemm_mx(a, "e4m3", sfa, a, "e4m3", sfa)
            y = ptxstd.gemm_decode(x, w4, sf4, 0.02 / 448)
    _ok()
    assert torch.equal(c, c0) and torch.equal(y, y0)
    for p, q in zip(want, got):
        for u, v in zip(p, q):
            assert torch.equal(u, v)


def test_vectors_written_by_the_call_before(cuda):
    """Weight, gate and bias vectors that the previous call of the stream writes, into the buffer that
    the calls before it read: with programmatic launch all of them may be resident at once. Without a
    wait in between, every result is that of calls which are waited for."""
    import ptxstd
    D, K = 8192, 64
    g = _gen(17)
    b, sfb = _mx(g, D, K, std=K ** -0.5)
    tokens = [_mx(g, 1, K) for _ in range(2)]
    buf = torch.zeros(D, dtype=torch.bfloat16, device="cuda")
    rows = (1600, 300, 3)  # the ring, a row per block with two vectors per thread and with one
    x, y = _bf(g, rows[0], D, std=2.0), _bf(g, rows[0], D, std=0.7)
    dn = _bf(g, rows[0], D, std=0.3)
    rx = torch.rsqrt(x.double().square().mean(1) + 1e-6).float()
    ry = torch.rsqrt(y.double().square().mean(1) + 1e-6).float()
    wide, narrow = _mx(g, 2048, K), _mx(g, 5, K)
    L = ptxstd.lib()

    def write(i):
        a, sfa = tokens[i]
        assert L.ptxstd_gemm_mx_epilogue(
            a.data_ptr(), 0, sfa.data_ptr(), b.data_ptr(), 0, sfb.data_ptr(), None, 0, None,
            buf.data_ptr(), None, 0, None, None, 1, D, K,
            torch.cuda.current_stream().cuda_stream) == 0

    def reads():
        for r in rows:
            yield lambda r=r: ptxstd.rmsnorm_residual(x[:r], buf, y=y[:r], w_post=buf, gate=buf)[:2]
        for r in rows[1:]:
            for c in (1024, 4096, D):  # registers, the ring
                part = [t[:r, :c].contiguous() for t in (dn, x, y)]
                yield lambda r=r, c=c, part=part: ptxstd.rmsnorm_residual_backward(
                    part[0], part[1], buf[:c], (rx[:r], ry[:r]), y=part[2], w_post=buf[:c],
                    gate=buf[:c])
        for a, sfa in (wide, narrow):
            yield lambda a=a, sfa=sfa: ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb,
                                                               bias=buf)

    for read in reads():
        want = []
        for i in range(2):
            write(i)
            torch.cuda.synchronize()
            want.append(read())
            torch.cuda.synchronize()
        got = []
        for k in range(20):
            write(k % 2)
            got.append(read())
        _ok()
        assert not torch.equal(_flat([want[0]])[0], _flat([want[1]])[0])
        for k, r in enumerate(got):
            for p, q in zip(_flat([want[k % 2]]), _flat([r])):
                assert torch.equal(p, q), k


def test_out_of_memory_is_torchs_error(cuda):
    """A result that does not fit raises torch.OutOfMemoryError, as every torch allocation does (here
    under a limit of this process's own, well below the 8.6 GB asked for), and the next call works."""
    import ptxstd
    rows = 65536
    g = _gen(1)
    a, sfa = _mx(g, rows, 32)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.02)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, a, "e4m3", sfa)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    ptxstd.gemm_mx_epilogue(a[:128], "e4m3", sfa[:512], a[:256], "e4m3", sfa[:1024])
    _ok()


def test_device_refusals(cuda):
    import ptxstd
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        ptxstd.rmsnorm_residual(x, w)
    with pytest.raises(ValueError, match="contiguous"):
        ptxstd.rmsnorm_residual(torch.zeros((64, 4), dtype=torch.bfloat16, device="cuda").t(),
                                w.cuda())
    flat = torch.zeros(4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ptxstd.PtxStdError):  # 2-byte offset: not 16-byte aligned
        ptxstd.rmsnorm_residual(flat[1:257].view(4, 64), w.cuda())
    assert C.sizeof(C.c_void_p) == 8


# ---- the activations over all of bf16 -----------------------------------------------------------
def _every_bf16():
    """Every finite bf16 value, in order."""
    x = torch.arange(1 << 16, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    return x[x.float().isfinite()].float().sort().values.to(torch.bfloat16)


def _value_bounds(x, act):
    """(f, f', bound of f, bound of f') in f64, the bounds relative to the values' own terms.

    The exponential's argument z, at most 128 in size where its result is in range, passes at most
    eight roundings to f32, those of the constants included: 8 * 128 * 2^-24 * ln 2 < 4.3e-5 of the
    result. The exponential, the reciprocal, the polynomial and at most eight further operations
    add less than 2^-19: 2^-14 = 6.1e-5 in all. Where the logistic function is below 2^-128, or the
    density below 2^-126, zero may stand for it (asked a factor of two before). 2^-148: f32's
    subnormals."""
    rel, a, zero = 2.0 ** -14, x.abs(), torch.zeros_like(x)
    if act in ("none", "relu"):
        return R.act(x, act), torch.ones_like(x) if act == "none" else (x > 0).double(), zero, zero
    if act == "gelu":
        phi = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        cdf = 0.5 * torch.erfc(-x / math.sqrt(2))
        f, df = x * cdf, cdf + x * phi
        terms, out_of_range, sharp = cdf + a * phi, phi < 2.0 ** -125, zero
        lost, lost_f = torch.minimum(cdf, 1 - cdf) + a * phi, torch.where(x < 0, f.abs(), zero)
    else:
        k, c = (math.sqrt(8 / math.pi), 0.044715) if act == "gelu_tanh" else (1.0, 0.0)
        u, du = k * (x + c * x ** 3), k * (1 + 3 * c * x * x)
        t, s = torch.sigmoid(u), torch.sigmoid(-u)
        inner = torch.where(t * s == 0, zero, a * t * s * du)
        f, df = x * t, t + x.sign() * inner
        terms, out_of_range = t + inner, t < 2.0 ** -127
        lost, lost_f = terms, f.abs()
        # above zero the factor 1 - t has the absolute rounding of a value next to 1, at most 2^-22
        # with the reciprocal's; below 2^-24 it is zero
        sharp = torch.where((x > 0) & (s > 2.0 ** -26), a * du * 2.0 ** -22, zero) + \
            torch.where((x > 0) & (s < 2.0 ** -22), inner, zero)
    return f, df, rel * f.abs() + torch.where(out_of_range, lost_f, zero) + 2.0 ** -148, \
        rel * terms + sharp + torch.where(out_of_range, lost, zero) + 2.0 ** -148


@pytest.mark.parametrize("M", [1, 1100])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activation_of_every_bf16(cuda, act, M):
    """Zero operands, so that the bias is the pre-activation exactly: act(x) for every finite bf16,
    held to its own size and not to x's. M: the kernel for few rows and the one for many."""
    import ptxstd
    x = _every_bf16()
    N = x.numel()
    a, sfa = ptxstd.quantize_mx(torch.zeros(M, 32, dtype=torch.bfloat16, device="cuda"), "e4m3",
                                sf_layout=2)
    b, sfb = ptxstd.quantize_mx(torch.zeros(N, 32, dtype=torch.bfloat16, device="cuda"), "e4m3",
                                sf_layout=2)
    c = ptxstd.gemm_mx_epilogue(a, "e4m3", sfa, b, "e4m3", sfb, bias=x, act=act)
    _ok()
    f, _, d, _ = _value_bounds(x.double(), act)
    R.check_bf16(c[0], f, d, act)
    assert (c == c[0]).all()


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activation_gradient_of_every_bf16(cuda, act):
    """One row with dh = 1: the f32 column sums are act'(x) itself; and the products' 8-bit blocks of
    32 neighbouring values."""
    import ptxstd
    x = _every_bf16()
    gate = x.view(1, -1)
    row, _, db = ptxstd.act_backward_mx(torch.ones_like(gate), gate, act=act, elem_type="e4m3",
                                        bias_grad=True)
    _ok()
    _, df, _, d = _value_bounds(x.double(), act)
    bad = (db.double() - df).abs() > d
    assert not bad.any(), (act, x[bad][:5].tolist(), db[bad][:5].tolist(), df[bad][:5].tolist(),
                           d[bad][:5].tolist())
    R.check_mx(*row, df.view(1, -1), d.view(1, -1), "e4m3", what=act)
