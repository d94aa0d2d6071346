"""Host-side argument checks of the Python bindings: shape and type errors are raised before any
device call, so they hold on a CPU-only host."""

import pytest


def test_gemm_mx_shape_checks(ptxstd_lib):
    import torch

    import ptxstd
    a = torch.zeros((256, 128), dtype=torch.uint8)
    sfa = torch.zeros(256 * 128 // 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="K mismatch"):
        ptxstd.gemm_mx(a, "e2m3", sfa, torch.zeros((256, 64), dtype=torch.uint8), "e2m3", sfa)
    with pytest.raises(ValueError, match="one UE8M0 per 32"):
        ptxstd.gemm_mx(a, "e2m3", sfa[:-1], a, "e2m3", sfa)
    with pytest.raises(ValueError, match="unknown MX element type"):
        ptxstd.gemm_mx(a, "e9m9", sfa, a, "e2m3", sfa)
    with pytest.raises(ValueError, match="unknown MX element type"):
        ptxstd.gemm_mx(a, 2, sfa, a, "e2m3", sfa)   # 2 is not a tcgen05 element-type code


def test_quantize_mx_input_checks(ptxstd_lib):
    import torch

    import ptxstd
    with pytest.raises(TypeError):
        ptxstd.quantize_mx(torch.zeros((128, 128), dtype=torch.float32), "e4m3")
    with pytest.raises(TypeError):
        ptxstd.quantize_mx(torch.zeros(128, dtype=torch.bfloat16), "e4m3")


def test_cp_unpack_shape_checks(ptxstd_lib):
    import torch

    import ptxstd
    with pytest.raises(ValueError):
        ptxstd.tcgen05_cp_unpack(torch.zeros((100, 32), dtype=torch.uint8), "e2m3")
    with pytest.raises(ValueError):
        ptxstd.tcgen05_cp_unpack(torch.zeros((128, 16), dtype=torch.uint8), "e2m1")
    with pytest.raises(ValueError, match="FP6"):
        ptxstd.tcgen05_cp_unpack(torch.zeros((128, 32), dtype=torch.uint8), "e4m3")


def test_mx_type_names(ptxstd_lib):
    import ptxstd
    from ptxstd import kernels
    assert kernels.MX_TYPES == {"e4m3": 0, "e5m2": 1, "e2m3": 3, "e3m2": 4, "e2m1": 5}
    assert (ptxstd.MX_E4M3, ptxstd.MX_E5M2, ptxstd.MX_E2M3, ptxstd.MX_E3M2,
            ptxstd.MX_E2M1) == (0, 1, 3, 4, 5)


def test_gemm_schedule_setting(ptxstd_lib):
    """The tile-schedule setting round-trips and rejects unknown values (no device needed)."""
    import ptxstd
    assert ptxstd.get_gemm_schedule() == ptxstd.SCHEDULE_PERSISTENT
    try:
        ptxstd.set_gemm_schedule(ptxstd.SCHEDULE_DYNAMIC)
        assert ptxstd.get_gemm_schedule() == ptxstd.SCHEDULE_DYNAMIC
        with pytest.raises(ptxstd.PtxStdError):
            ptxstd.set_gemm_schedule(2)
        assert ptxstd.get_gemm_schedule() == ptxstd.SCHEDULE_DYNAMIC
    finally:
        ptxstd.set_gemm_schedule(ptxstd.SCHEDULE_PERSISTENT)


@pytest.mark.parametrize("rows,cols,layout,need", [(1, 32, 2, 512), (129, 160, 2, 2 * 2 * 512),
                                                   (128, 128, 1, 512), (5, 96, 0, 15)])
def test_quantize_mx_given_outputs_have_room(ptxstd_lib, rows, cols, layout, need):
    """The padded layout clears and writes whole tiles, more than rows * cols / 32 bytes: a pair made
    for another layout is refused before the call. What is large enough gets as far as the check
    for device memory."""
    import torch

    import ptxstd
    x = torch.zeros((rows, cols), dtype=torch.bfloat16)

    def call(nq, nsf):
        out = (torch.zeros(nq, dtype=torch.uint8), torch.zeros(nsf, dtype=torch.uint8))
        ptxstd.quantize_mx(x, "e4m3", sf_layout=layout, out=out)

    with pytest.raises(ValueError, match="sf: too small"):
        call(rows * cols, need - 1)
    with pytest.raises(ValueError, match="q: too small"):
        call(rows * cols - 1, need)
    with pytest.raises(TypeError, match="CUDA"):
        call(rows * cols, need)
    with pytest.raises(ValueError, match="sf: on"):
        ptxstd.quantize_mx(x, "e4m3", sf_layout=layout,
                           out=(torch.zeros(rows * cols, dtype=torch.uint8),
                                torch.zeros(need, dtype=torch.uint8, device="meta")))


def test_given_outputs_have_room(ptxstd_lib):
    """The same for every other call that writes into a tensor it is given."""
    import torch

    import ptxstd
    x = torch.zeros((128, 256), dtype=torch.bfloat16)
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    c = torch.zeros(128 * 128 - 1, dtype=torch.bfloat16)
    calls = {
        "mxfp8": lambda: ptxstd.quantize_mxfp8(x, out=(u8(128, 256), u8(128 * 8 - 1))),
        "nvfp4": lambda: ptxstd.quantize_nvfp4(x, 1.0, out=(u8(128, 127), u8(128, 16))),
        "fp8": lambda: ptxstd.gemm_fp8(u8(128, 64), u8(128, 64), out=c),
        "gemm_mxfp8": lambda: ptxstd.gemm_mxfp8(u8(128, 64), u8(256), u8(128, 64), u8(256), out=c),
        "gemm_mx": lambda: ptxstd.gemm_mx(u8(128, 64), 0, u8(256), u8(128, 64), 0, u8(256), out=c),
        "sparse": lambda: ptxstd.gemm_mxfp8_sparse(u8(128, 32), u8(128, 8), u8(128), u8(128, 64),
                                                   u8(128), out=c),
        "gemm_nvfp4": lambda: ptxstd.gemm_nvfp4(u8(128, 32), u8(512), 1.0, u8(128, 32), u8(512),
                                                1.0, out=c),
        "decode": lambda: ptxstd.gemm_decode(x[:16, :64], u8(128, 32), u8(512), 1.0, out=c[:2047],
                                             workspace=(0, 0)),
    }
    for name, call in calls.items():
        with pytest.raises(ValueError, match="too small"):
            call()
            pytest.fail(name)


def test_given_outputs_of_the_sharded_gemms_have_room(ptxstd_lib):
    """A communicator that was never set up: the refusals come before any call on it."""
    import torch

    from ptxstd.dist import Dist
    d = Dist.__new__(Dist)
    d.world, d.rank, d.handle, d._p2p, d._ws = 2, 0, None, None, {}
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    a, w = torch.zeros((256, 32), dtype=torch.uint8), torch.zeros((128, 32), dtype=torch.uint8)
    sf = torch.zeros(1024, dtype=torch.uint8)
    c = torch.zeros(256 * 128 - 1, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="too small"):
        d.gemm_nvfp4(a, sf, 1.0, w, sf, 1.0, 256, out=c)
    with pytest.raises(ValueError, match="too small"):
        d.gemm_decode(x, w, sf, 1.0, 256, out=c[:4 * 256 - 1])
    with pytest.raises(ValueError, match="too small"):
        d.gemm_decode_p2p(x, w, sf, 1.0, 256, out=c[:4 * 256 - 1])
