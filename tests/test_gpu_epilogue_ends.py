"""The ends of the epilogue products' ranges on the GPU: activations whose
results are far below their arguments, scales near the ends of fp32."""
import numpy as np
import pytest

from lattice_amd.bindings import ACT_GELU, ACT_GELU_TANH, ACT_NONE, ACT_SILU
from tests import e4m3 as E
from tests.test_gpu_gemm_epi import call

pytestmark = pytest.mark.gpu


def activated(torch, lib, z, act):
    """act of the bf16 values z by a product whose other operand is 1."""
    x, w = np.zeros((len(z), 16)), np.zeros((24, 16))
    x[:, 3], w[:, 3] = z, 1
    got = call(torch, lib, x, w, act=act)
    assert np.array_equal(got, np.broadcast_to(got[:, :1], got.shape))
    return got[:, 0].astype(np.float64)


def store_and_roundings(y):
    """Half a step of bf16 (2^-134 below the normal numbers), and 2^-15 of y: an
    exponent of at most 104 = 150 ln 2 whose value four roundings of 2^-24 went into,
    with ten more of y's own, is 426 * 2^-24 off, and a fit 2^-21.  y / z below the
    normal numbers of fp32 is 2^-150 off besides, half of its least step, and y by |z| <
    100 times that, less than 2^-143."""
    return np.maximum(E.BF16_HALF * np.abs(y), 2.0 ** -134) + 2.0 ** -15 * np.abs(y) + 2.0 ** -143


def test_gelu_of_the_lower_tail(gpu_lib):
    """z Phi(z) for z of -2 to where nothing is left of it, against fp64 relative
    to the result: 1 - erf has none of its bits there."""
    import torch
    z = np.unique(E.bf16(np.linspace(-14.5, -2, 1500))).astype(np.float64)
    y = E.activation(z, 2)
    assert np.abs(y).min() < 2.0 ** -134 and np.abs(y).max() > 0.04
    got = activated(torch, gpu_lib, z, ACT_GELU)
    assert np.all(np.abs(got - y) <= store_and_roundings(y))


def test_gelu_everywhere_else(gpu_lib):
    import torch
    z = np.unique(E.bf16(np.concatenate([np.linspace(-2, 6, 1500), [-1e-30, -1e-5, 0, 1e-36, 1e-9,
                                                                   30, 1e4, 1e30, 3e38]])))
    y = E.activation(z.astype(np.float64), 2)
    got = activated(torch, gpu_lib, z, ACT_GELU)
    assert np.all(np.abs(got - y) <= store_and_roundings(y))


def test_gelu_of_infinities(gpu_lib):
    """inf Phi(inf) = inf; -inf Phi(-inf) is the product of an infinity and 0."""
    import torch
    bias = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0], device="cuda").bfloat16()
    x, w = (torch.zeros(n, 16, device="cuda").bfloat16() for n in (3, 4))
    y = torch.zeros(3, 4, device="cuda").bfloat16()
    gpu_lib.gemm_bf16_epi(x.data_ptr(), w.data_ptr(), y.data_ptr(), 3, 4, 16, bias_ptr=bias.data_ptr(),
                          activation=ACT_GELU, stream_ptr=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = y.float().cpu().numpy()
    assert np.all(got[:, 0] == np.inf) and np.all(np.isnan(got[:, 1:3])) and np.all(got[:, 3] == 0.83984375)


@pytest.mark.parametrize("act,low,high", [(ACT_SILU, -99, -86), (ACT_GELU_TANH, -10.45, -9.8)])
def test_results_below_the_normal_numbers(gpu_lib, act, low, high):
    """z sigmoid(t) of less than 2^-126: bf16 has it down to 2^-133.  Its t is off by
    at most five roundings of 99 * 2^-24, so y by 2^-15 with eight more of its own; and
    by 2^-143, see above."""
    import torch
    z = np.unique(E.bf16(np.linspace(low, high, 600))).astype(np.float64)
    t = z if act == ACT_SILU else np.sqrt(8 / np.pi) * (z + 0.044715 * z ** 3)
    y = z / (1 + np.exp(-t))
    assert t.min() > -99.5 and np.abs(y).min() < 2.0 ** -132 and np.abs(y).max() > 2.0 ** -126
    got = activated(torch, gpu_lib, z, act)
    assert np.all(np.abs(got - y) <= store_and_roundings(y))


@pytest.mark.parametrize("tile,splits", [(None, 1), (9, 1), (9, 2), (100, 1), (100, 2)])
@pytest.mark.parametrize("m,n,k", [(3, 41, 272), (300, 264, 1024)])
def test_scales_whose_product_alone_is_ordinary(gpu_lib, tunables, m, n, k, tile, splits):
    """Tokens of any size (scales 2^-126 .. 2^119, as the row quantisers make them)
    against weights that bring them back: sum xscale wscale is a whole number
    times a power of two that fp32 has, sum xscale alone is past it or below it.
    Bit for bit, as every sum is exact in fp32."""
    import torch
    if tile is not None:
        tunables.setenv("KCMM_EPI_TILE", str(tile))
        tunables.setenv("KCMM_GEMM_SPLITS", str(splits))
    rng = np.random.default_rng([m, n, k])
    for unit, xe, we in ((1.0, rng.integers(100, 120, m), rng.integers(-110, -90, n)),
                         (2.0 ** -9, rng.integers(-126, -100, m), rng.integers(100, 120, n)),
                         (1.0, rng.integers(100, 120, m), np.full(n, -149))):
        x = unit * rng.integers(-3, 4, (m, k)).astype(np.float64)
        w = unit * rng.integers(-3, 4, (n, k)).astype(np.float64)
        xs, ws = np.exp2(xe.astype(np.float64)), np.exp2(we.astype(np.float64))
        bias = E.bf16(rng.integers(-100, 101, n))
        y, s = E.product(x, w, None, None, None, None, ACT_NONE)
        assert s.max() < 2 ** 14 * unit * unit
        y = y * (xs[:, None] * ws)                      # exact: powers of two
        for b in (None, bias):
            got = call(torch, gpu_lib, x, w, xs, ws, b)
            z = E.f32(y) if b is None else E.f32(E.f32(y) + b)
            assert np.array_equal(got, E.bf16(z)), (unit, b is None)
