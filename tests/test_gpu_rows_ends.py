"""Rows as e4m3 codes at the ends of their range: SwiGLU gates so negative that e^-g
is past fp32, norms of nothing."""
import numpy as np
import pytest

from tests import e4m3 as E
from tests.test_gpu_quant_rows import Outputs, check_rows, dev16

pytestmark = pytest.mark.gpu


def silu_rows(torch, lib, gate, up):
    rows, inter = gate.shape
    gu = np.ascontiguousarray(np.concatenate([gate, up], axis=1))
    bits = (gu.view(np.uint32) >> 16).astype(np.uint16)
    xd = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).cuda()
    o = Outputs(torch, rows, inter)
    lib.silu_mul_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), rows, inter,
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return o.get()


@pytest.mark.parametrize("inter", [64, 4096, 33000])
def test_gates_past_the_exponential_s_range(gpu_lib, inter):
    """silu(g) = g e^g is a normal number down to g = -91 or so and none below -103,
    but a large up makes values of some size of it all the same: a row of such gates
    has its scale and codes.  REL: |g| < 171, 171 log2(e) + 10 roundings of 2^-24 at
    the most, less than 2^-15."""
    import torch
    rng = np.random.default_rng(inter)
    g = E.bf16(np.stack([rng.uniform(lo, hi, inter) for lo, hi in
                         ((-100, -88.75), (-130, -88.75), (-170, -140), (-92, 3))]))
    u = E.bf16(rng.uniform(-1, 1, (4, inter)) * np.array([3e38, 3e38, 3e38, 3e38])[:, None])
    u[3] /= 2.0 ** 10                   # (values of ordinary gates stay below infinity)
    codes, scales = silu_rows(torch, gpu_lib, g, u)
    d = g.astype(np.float64)
    check_rows(codes, scales, d / (1 + np.exp(-d)) * u, 2.0 ** -15)
    assert np.all(scales[:2] < 1) and np.all((codes[:3] & 0x7f).max(axis=1) > 0x40)


def test_far_gates_and_ups_that_are_not_finite(gpu_lib):
    """A finite gate times an infinite up is infinite (the code of 448, the other
    sign), however far the gate; NaN where the formula has it."""
    import torch
    rng = np.random.default_rng(3)
    g = E.bf16(rng.standard_normal((2, 64)))
    u = E.bf16(rng.standard_normal((2, 64)))
    g[0, :5] = [-89, -95, -120, -600, -1e30]
    u[0, :5] = [np.inf, -np.inf, np.inf, -np.inf, np.inf]
    g[1, :4] = [-np.inf, -100, np.nan, -1e38]
    u[1, :4] = [1, np.nan, 1, 3e38]
    codes, scales = silu_rows(torch, gpu_lib, g, u)
    assert list(codes[0, :5]) == [0xfe, 0x7e, 0xfe, 0x7e, 0xfe]
    assert np.all((codes[1, :3] & 0x7f) == 0x7f) and (codes[1, 3] & 0x7f) == 0
    d = g.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        v = d / (1 + np.exp(-d)) * u
    v[0, :5] = v[1, :4] = 0
    codes[0, :5] = codes[1, :4] = 0
    check_rows(codes, scales, v, 2.0 ** -17)


@pytest.mark.parametrize("cols", [64, 4096, 33000])
def test_norm_of_zeros_without_eps(gpu_lib, cols):
    """0 / 0: NaN codes and scale 1 in that row, nothing in the others."""
    import torch
    x = E.bf16(np.random.default_rng(cols).standard_normal((3, cols)))
    x[1] = 0
    xd, wd = dev16(torch, x), dev16(torch, np.ones(cols))
    o = Outputs(torch, 3, cols)
    gpu_lib.add_rmsnorm_fp8(xd.data_ptr(), 0, wd.data_ptr(), 0, o.c.data_ptr(), o.s.data_ptr(), 3, cols,
                            0.0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = o.get()
    assert np.all((codes[1] & 0x7f) == 0x7f) and scales[1] == 1
    _, v = E.add_rmsnorm(x[::2], None, np.ones(cols), 0.0)
    check_rows(codes[::2], scales[::2], v, 2.0 ** -18 + cols / 1024 * 2.0 ** -24)
