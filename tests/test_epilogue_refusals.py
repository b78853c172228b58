"""What the 8-bit row operators and the epilogue products refuse, on the
host-check build: -1 and the reason on stderr, before any device work (a call
that passes the checks ends at "no device" there)."""
import ctypes as C

import pytest

from lattice_amd.bindings import (KcmmError, KcmmGemmEpilogue, ACT_NONE, ACT_SILU)

P = 1 << 20     # an aligned address; nothing is read from it
STEP = 1 << 33  # buffers this far apart overlap nothing


def at(i):
    return P + i * STEP


@pytest.fixture
def refused(hostcheck_lib, capfd):
    def check(fn, *args, why, **kw):
        capfd.readouterr()
        with pytest.raises(KcmmError):
            getattr(hostcheck_lib, fn)(*args, **kw)
        said = capfd.readouterr().err
        assert why in said and said.startswith("kcmm_"), said
    return check


NORM = dict(x_ptr=at(0), residual_ptr=at(1), w_ptr=at(2), hidden_ptr=at(3), codes_ptr=at(4),
            scales_ptr=at(5), rows=4, hidden_size=64, eps=1e-5)


@pytest.mark.parametrize("change,why", [
    ({}, "no device"),
    (dict(residual_ptr=0, hidden_ptr=0), "no device"),
    (dict(hidden_ptr=at(0)), "no device"),
    (dict(hidden_ptr=at(1)), "no device"),
    (dict(eps=0.0), "no device"),
    (dict(rows=1 << 20), "no device"),
    (dict(x_ptr=0), "null"), (dict(w_ptr=0), "null"), (dict(codes_ptr=0), "null"),
    (dict(scales_ptr=0), "null"), (dict(residual_ptr=0), "both or neither"),
    (dict(hidden_ptr=0), "both or neither"),
    (dict(rows=0), "rows"), (dict(rows=(1 << 20) + 1), "rows"),
    (dict(hidden_size=0), "multiple of 8"), (dict(hidden_size=60), "multiple of 8"),
    (dict(hidden_size=(1 << 24) + 8), "multiple of 8"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(x_ptr=at(0) + 8), "aligned"), (dict(codes_ptr=at(4) + 8), "aligned"),
    (dict(w_ptr=at(2) + 2), "aligned"), (dict(scales_ptr=at(5) + 2), "aligned"),
    (dict(scales_ptr=at(5) + 4), "no device"),
    (dict(hidden_ptr=at(0) + 16), "overlaps"), (dict(hidden_ptr=at(1) + 128), "overlaps"),
    (dict(hidden_ptr=at(2)), "overlaps"), (dict(codes_ptr=at(0)), "overlaps"),
    (dict(codes_ptr=at(1) + 256), "overlaps"), (dict(codes_ptr=at(3) + 496), "overlaps"),
    (dict(codes_ptr=at(2) + 112), "overlaps"), (dict(scales_ptr=at(4) + 240), "overlaps"),
    (dict(scales_ptr=at(0)), "overlaps"), (dict(scales_ptr=at(3)), "overlaps"),
    (dict(codes_ptr=at(3) + 512), "no device"),
])
def test_add_rmsnorm(refused, change, why):
    refused("add_rmsnorm_fp8", why=why, **{**NORM, **change})


@pytest.mark.parametrize("fn,x,width", [("quant_rows_fp8", "x_ptr", 1), ("silu_mul_fp8", "gate_up_ptr", 2)])
@pytest.mark.parametrize("change,why", [
    ({}, "no device"), (dict(x=0), "null"), (dict(codes_ptr=0), "null"), (dict(scales_ptr=0), "null"),
    (dict(rows=0), "rows"), (dict(cols=12), "multiple of 8"), (dict(cols=0), "multiple of 8"),
    (dict(x=at(0) + 4), "aligned"), (dict(codes_ptr=at(0)), "overlaps"),
    (dict(scales_ptr=at(1) + 240), "overlaps"), (dict(end=-16), "overlaps"), (dict(end=0), "no device"),
])
def test_row_codes(refused, fn, x, width, change, why):
    a = {x: change.get("x", at(0)), "codes_ptr": at(1), "scales_ptr": at(2), "rows": 4,
         "intermediate" if width == 2 else "cols": change.get("cols", 64)}
    a.update({k: v for k, v in change.items() if k in a})
    if "end" in change:     # codes right behind x, or into its last bytes
        a["codes_ptr"] = at(0) + 4 * 64 * 2 * width + change["end"]
    refused(fn, why=why, **a)


GEMM = dict(y_ptr=at(4), m=4, n=48, k=64, bias_ptr=at(5), residual_ptr=at(6), activation=ACT_SILU)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("change,why", [
    ({}, "no device"),
    (dict(bias_ptr=0, residual_ptr=0, activation=ACT_NONE), "no device"),
    (dict(residual_ptr=at(4)), "no device"),
    (dict(n=1), "no device"), (dict(n=49), "no device"), (dict(k=16), "no device"),
    (dict(y_ptr=0), "null"), (dict(x_ptr=0), "null"), (dict(w_ptr=0), "null"),
    (dict(m=0), "m, n > 0"), (dict(n=0), "m, n > 0"), (dict(k=0), "multiple of"),
    (dict(k=12), "multiple of"), (dict(k=(1 << 24) + 16), "2^24"),
    (dict(activation=-1), "activation"), (dict(activation=5), "activation"),
    (dict(x_ptr=at(0) + 8), "aligned"), (dict(w_ptr=at(1) + 2), "aligned"),
    (dict(y_ptr=at(4) + 1), "aligned"), (dict(bias_ptr=at(5) + 1), "aligned"),
    (dict(residual_ptr=at(6) + 1), "aligned"),
    (dict(y_ptr=at(4) + 2, bias_ptr=at(5) + 2, residual_ptr=at(6) + 2), "no device"),
    (dict(y_ptr=at(0)), "overlaps"), (dict(y_ptr=at(1) + 16), "overlaps"),
    (dict(y_ptr=at(5)), "overlaps"), (dict(residual_ptr=at(4) + 16), "overlaps"),
    (dict(y_ptr=at(6) - 16), "overlaps"),
    (dict(m=1 << 20, k=1 << 12), "too large"), (dict(n=1 << 20, k=1 << 12), "too large"),
    (dict(m=1 << 16, n=1 << 15), "too large"),
    (dict(m=(1 << 20) + 1), "too large"), (dict(n=(1 << 22) + 1), "too large"),
    (dict(m=1 << 20), "no device"), (dict(n=1 << 22), "no device"),
])
def test_products(refused, fp8, change, why):
    a = {"x_ptr": at(0), "w_ptr": at(1), **GEMM, **change}
    if fp8:
        a.update(x8_ptr=a.pop("x_ptr"), w8_ptr=a.pop("w_ptr"), xscale_ptr=at(2), wscale_ptr=at(3))
    refused("gemm_fp8" if fp8 else "gemm_bf16_epi", why=why, **a)


@pytest.mark.parametrize("change,why", [(dict(xscale_ptr=0), "null"), (dict(wscale_ptr=0), "null"),
                                        (dict(k=8), "multiple of 16"),
                                        (dict(xscale_ptr=at(2) + 2), "aligned"),
                                        (dict(wscale_ptr=at(3) + 1), "aligned"),
                                        (dict(xscale_ptr=at(2) + 4, wscale_ptr=at(3) + 4), "no device"),
                                        (dict(y_ptr=at(2)), "overlaps"),
                                        (dict(y_ptr=at(3) + 16), "overlaps")])
def test_fp8_products(refused, change, why):
    refused("gemm_fp8", why=why, **{"x8_ptr": at(0), "xscale_ptr": at(2), "w8_ptr": at(1),
                                    "wscale_ptr": at(3), **GEMM, **change})


def test_no_epilogue(hostcheck_lib, capfd):
    """A NULL epilogue is none; the struct's layout is the header's."""
    assert hostcheck_lib.lib.kcmm_gemm_bf16_epi_on_stream(at(0), at(1), at(2), None, 4, 48, 8, 0) == -1
    assert "no device" in capfd.readouterr().err
    assert C.sizeof(KcmmGemmEpilogue) == 24 and KcmmGemmEpilogue.activation.offset == 16
