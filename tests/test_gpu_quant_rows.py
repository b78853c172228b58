"""Rows as e4m3 codes with scales (kcmm_add_rmsnorm_fp8, kcmm_quant_rows_fp8,
kcmm_silu_mul_fp8) on the GPU against plain forms.

quant has no arithmetic but the fp32 quotient: bit for bit.  norm and silu
compute v in fp32: hidden is bit for bit (one fp32 addition, one rounding);
the scale is relative REL off, and a code is the nearest to v / scale up to
the same, so that code * scale is within half an e4m3 step of v (2^-4 of it,
or 2^-10 of the scale among the subnormals) and REL.  REL of the norm: at most
8 * 4 products a lane and 6 + 16 more additions, 54 roundings of 2^-24, halved
by the square root, and 6 roundings after it: 33 * 2^-24 < 2^-18.  Rows past
32768 columns add 8 * cols / 8192 products a lane.  REL of silu: the
exponential of g is off by its argument's rounding, |g| <= 64 here, times
log2(e), 2^-24 relative each, and the instruction's and four more roundings:
< 100 * 2^-24 < 2^-17."""
import numpy as np
import pytest

from tests import e4m3 as E

pytestmark = pytest.mark.gpu

EPS = 1e-5


def dev16(torch, values):
    return torch.from_numpy(E.bf16_bits(values).view(np.int16)).view(torch.bfloat16).cuda()


def host16(t):
    import torch
    return E.bf16_values(t.cpu().view(torch.int16).numpy().view(np.uint16))


class Outputs:
    """Output buffers with guard bytes behind them."""

    def __init__(self, torch, rows, cols):
        self.shape = rows, cols
        self.c = torch.full((rows * cols + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.s = torch.full((rows + 16,), -7.0, dtype=torch.float32, device="cuda")

    def get(self):
        rows, cols = self.shape
        c, s = self.c.cpu().numpy(), self.s.cpu().numpy()
        assert np.all(c[rows * cols:] == 0xA5) and np.all(s[rows:] == -7.0)
        return c[:rows * cols].reshape(rows, cols), s[:rows]


def check_rows(codes, scales, v, rel):
    a = np.abs(v).max(axis=1)
    want = np.where(a > 0, np.maximum(a / E.E4M3_MAX, 2.0 ** -126), 1.0)
    assert np.all(np.abs(scales - want) <= (rel + 2.0 ** -23) * want)
    got = E.e4m3_values()[codes] * scales[:, None].astype(np.float64)
    tol = np.maximum(E.E4M3_HALF * np.abs(v), 2.0 ** -10 * scales[:, None])
    tol = tol * (1 + 2.0 ** -20) + 2 * rel * np.abs(v)
    assert np.all(np.abs(got - v) <= tol), np.max(np.abs(got - v) / tol)


def norm_case(torch, lib, rows, cols, residual, seed=0, in_place=None, x=None, eps=EPS):
    rng = np.random.default_rng([seed, rows, cols])
    if x is None:
        x = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal(cols))
    x = E.bf16(x)
    r = E.bf16(3 * rng.standard_normal((rows, cols))) if residual else None
    w = E.bf16(1 + 0.3 * rng.standard_normal(cols))
    xd, wd = dev16(torch, x), dev16(torch, w)
    rd = dev16(torch, r) if residual else None
    hd = {None: torch.zeros_like(xd), "x": xd, "r": rd}[in_place] if residual else None
    o = Outputs(torch, rows, cols)
    lib.add_rmsnorm_fp8(xd.data_ptr(), rd.data_ptr() if residual else 0, wd.data_ptr(),
                        hd.data_ptr() if residual else 0, o.c.data_ptr(), o.s.data_ptr(), rows,
                        cols, eps, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    h, v = E.add_rmsnorm(x, r, w, eps)
    if residual:
        assert np.array_equal(host16(hd).view(np.uint32), h.view(np.uint32))
    codes, scales = o.get()
    check_rows(codes, scales, v, 2.0 ** -18 + cols / 1024 * 2.0 ** -24)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 64), (5, 512), (1, 520), (7, 1024), (2, 1032),
                                       (9, 2048), (4, 2816), (1, 4096), (65, 4096), (3, 5128),
                                       (6, 8192), (2, 14336), (3, 16384), (2, 28672), (2, 32768),
                                       (3, 32776), (1, 70000), (2051, 1024), (1030, 4096),
                                       (600, 8192)])
def test_add_rmsnorm(gpu_lib, rows, cols, residual):
    import torch
    norm_case(torch, gpu_lib, rows, cols, residual)


@pytest.mark.parametrize("cols", [1024, 4096, 40000])
@pytest.mark.parametrize("in_place", ["x", "r"])
def test_add_rmsnorm_in_place(gpu_lib, cols, in_place):
    import torch
    norm_case(torch, gpu_lib, 5, cols, True, in_place=in_place)


@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-20, 1e18])
def test_add_rmsnorm_small_and_large_rows(gpu_lib, size):
    """All-zero rows (scale 1, codes 0), rows far below eps, rows whose sum of
    squares is past fp32."""
    import torch
    x = size * np.random.default_rng(1).standard_normal((4, 4096))
    norm_case(torch, gpu_lib, 4, 4096, False, x=x)


@pytest.mark.parametrize("cols", [512, 4096, 33000])
@pytest.mark.parametrize("size", [1e-30, 1e-17, 1e25, 3e37])
def test_add_rmsnorm_without_eps(gpu_lib, size, cols):
    """Squares far outside fp32 and no eps to hide them: the rows' sizes drop out."""
    import torch
    x = size * np.random.default_rng(2).standard_normal((5, cols))
    norm_case(torch, gpu_lib, 5, cols, False, x=x, eps=0.0)


@pytest.mark.parametrize("rows,cols", [(1, 8), (2, 72), (1, 512), (130, 1032), (5, 2048), (64, 4096),
                                       (3, 14336), (2, 32768), (2, 32776), (1111, 2048),
                                       (4100, 264), (1, 131072)])
@pytest.mark.parametrize("size", [1.0, 3e38, 1e-36, 1e-39])
def test_quant_rows_bit_for_bit(gpu_lib, rows, cols, size):
    """size 1e-36 and 1e-39: scales below 2^-80, and where a / 448 is raised to 2^-126."""
    import torch
    rng = np.random.default_rng([rows, cols])
    x = rng.uniform(-1, 1, (rows, cols)) * np.exp2(-rng.integers(0, 24, (rows, cols)))
    x = E.bf16(size * x)
    x[rows // 2] = 0
    xd = dev16(torch, x)
    o = Outputs(torch, rows, cols)
    gpu_lib.quant_rows_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), rows, cols,
                           torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = o.get()
    want = E.row_scale(x)
    assert np.array_equal(scales, want)
    assert np.array_equal(codes, E.e4m3_codes(x / want[:, None]))


@pytest.mark.parametrize("cols", [64, 4096, 33000])
def test_quant_rows_not_finite(gpu_lib, cols):
    """Infinities and NaN: no part of the scale; +-448 and NaN among the codes."""
    import torch
    x = E.bf16(np.random.default_rng(3).standard_normal((6, cols)))
    x[0, 5], x[1, 7], x[2, 3], x[2, 4] = np.inf, -np.inf, np.nan, np.inf
    x[3] = np.nan
    x[4] = -np.inf
    bits = (x.view(np.uint32) >> 16).astype(np.uint16)
    xd = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).cuda()
    o = Outputs(torch, 6, cols)
    gpu_lib.quant_rows_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), 6, cols,
                           torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = o.get()
    assert np.array_equal(scales, E.row_scale(x))
    want = E.e4m3_codes(x / scales[:, None])
    nan = np.isnan(x)
    assert np.array_equal(codes[~nan], want[~nan]) and np.all((codes[nan] & 0x7f) == 0x7f)


def test_norm_not_finite(gpu_lib):
    """A NaN makes its whole row NaN (scale 1: no finite value); an infinity
    makes the other columns 0 and itself NaN; the other rows do not notice."""
    import torch
    rng = np.random.default_rng(5)
    x = E.bf16(rng.standard_normal((3, 512)))
    clean = x.copy()
    x[0, 9], x[2, 11] = np.nan, np.inf
    bits = (x.view(np.uint32) >> 16).astype(np.uint16)
    xd = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).cuda()
    wd = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    o = Outputs(torch, 3, 512)
    gpu_lib.add_rmsnorm_fp8(xd.data_ptr(), 0, wd.data_ptr(), 0, o.c.data_ptr(), o.s.data_ptr(), 3,
                            512, EPS, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = o.get()
    assert np.all((codes[0] & 0x7f) == 0x7f) and scales[0] == 1
    assert scales[2] == 1 and (codes[2, 11] & 0x7f) == 0x7f
    assert np.all((np.delete(codes[2], 11) & 0x7f) == 0)
    _, v = E.add_rmsnorm(clean[1:2], None, np.ones(512), EPS)
    check_rows(codes[1:2], scales[1:2], v, 2.0 ** -18)


@pytest.mark.parametrize("rows,inter", [(1, 8), (3, 264), (64, 2816), (5, 8192), (2, 14336),
                                        (2, 28672), (2, 32776), (300, 1024), (1500, 2816)])
def test_silu_mul(gpu_lib, rows, inter):
    import torch
    rng = np.random.default_rng([rows, inter])
    gu = rng.standard_normal((rows, 2 * inter)) * 4
    gu[0, :inter // 2] *= 4          # gates to about +-64
    gu = E.bf16(np.clip(gu, -64, 64))
    xd = dev16(torch, gu)
    o = Outputs(torch, rows, inter)
    gpu_lib.silu_mul_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), rows, inter,
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    g, u = gu[:, :inter].astype(np.float64), gu[:, inter:].astype(np.float64)
    codes, scales = o.get()
    check_rows(codes, scales, g / (1 + np.exp(-g)) * u, 2.0 ** -17)


@pytest.mark.parametrize("inter", [64, 8192, 33000])
def test_silu_mul_not_finite(gpu_lib, inter):
    """Gates whose exponential overflows or vanishes, infinities and NaN: as the
    formula has them in fp32 (silu(-inf) is NaN), the rest of the row as ever."""
    import torch
    rng = np.random.default_rng(inter)
    g = E.bf16(rng.standard_normal((4, inter)))
    u = E.bf16(rng.standard_normal((4, inter)))
    g[0, :6], u[0, :6] = [-200, -100, -89, 100, 200, -88], 1.0
    g[1, :4], u[1, :4] = [np.inf, -np.inf, np.nan, 2.0], [1.0, 1.0, 1.0, -np.inf]
    g[2], u[2] = -300, 1.0                    # every value vanishes
    gu = np.concatenate([g, u], axis=1)
    bits = (np.ascontiguousarray(gu).view(np.uint32) >> 16).astype(np.uint16)
    xd = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).cuda()
    o = Outputs(torch, 4, inter)
    gpu_lib.silu_mul_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), 4, inter,
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    codes, scales = o.get()
    with np.errstate(over="ignore", invalid="ignore"):
        d = g.astype(np.float64)
        v = d / (1 + np.exp(-d)) * u
    v[0, 0] = v[0, 1] = 0                     # e^100 is past fp32
    v[2] = 0
    assert scales[2] == 1 and np.all((codes[2] & 0x7f) == 0)
    assert (codes[1, 0], codes[1, 3]) == (0x7e, 0xfe) and np.all((codes[1, 1:3] & 0x7f) == 0x7f)
    v[1, :4] = 0
    codes[1, :4] = 0
    check_rows(codes, scales, v, 2.0 ** -17)


def test_silu_mul_at_the_exponent_s_end(gpu_lib):
    """Gates whose 1 / (1 + e^-g) is below the normal numbers while g times it is
    not, with ups that make values of some size of it.  REL as above: |g| < 89 in
    the place of 64, 89 log2(e) + 5 < 135 roundings of 2^-24, less than 2^-16."""
    import torch
    rng = np.random.default_rng(12)
    inter = 512
    g = E.bf16(rng.uniform(-88.5, -85, (2, inter)))
    u = E.bf16(rng.standard_normal((2, inter)) * 1e36)
    xd = dev16(torch, np.concatenate([g, u], axis=1))
    o = Outputs(torch, 2, inter)
    gpu_lib.silu_mul_fp8(xd.data_ptr(), o.c.data_ptr(), o.s.data_ptr(), 2, inter,
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    d = g.astype(np.float64)
    codes, scales = o.get()
    check_rows(codes, scales, d / (1 + np.exp(-d)) * u, 2.0 ** -16)


def test_rows_past_four_gib(gpu_lib):
    """Element offsets above 2^31 (byte offsets above 2^32): the rows written
    near the end are quantised, and only with their own values."""
    import torch
    rows, cols = 70_000, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(8)
    at = [0, 40_000, rows - 1]
    v = E.bf16(rng.standard_normal((3, cols)))
    x[torch.tensor(at, device="cuda")] = dev16(torch, v)
    codes = torch.full((rows, cols), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(rows, dtype=torch.float32, device="cuda")
    gpu_lib.quant_rows_fp8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, cols,
                           torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = E.row_scale(v)
    assert np.array_equal(codes[torch.tensor(at, device="cuda")].cpu().numpy(),
                          E.e4m3_codes(v / want[:, None]))
    s = scales.cpu().numpy()
    assert np.array_equal(s[at], want) and np.all(np.delete(s, at) == 1)
    assert int((codes != 0).any(1).sum()) == 3
