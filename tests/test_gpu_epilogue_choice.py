"""What an epilogue product launches, and the 256-row tiles in all their forms:
the heights of their token tiles, two heights at once, K splits."""
import numpy as np
import pytest

from lattice_amd.bindings import ACT_NONE
from tests import e4m3 as E
from tests.test_gpu_gemm_epi import call

pytestmark = pytest.mark.gpu


def captured(torch, lib, m, n, k, fp8):
    """(grid, block) of what a captured product launches; nothing runs."""
    from tests.test_gpu_graph import _captured_kernels
    x, w = (torch.empty(r * k, dtype=torch.uint8 if fp8 else torch.bfloat16, device="cuda") for r in (m, n))
    s = torch.empty(max(m, n), dtype=torch.float32, device="cuda")
    y = torch.empty(m * n, dtype=torch.bfloat16, device="cuda")

    def run(st):
        if fp8:
            lib.gemm_fp8(x.data_ptr(), s.data_ptr(), w.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k,
                         stream_ptr=st)
        else:
            lib.gemm_bf16_epi(x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k, stream_ptr=st)

    torch.cuda.synchronize()
    return _captured_kernels(run)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(200, 512, 4096), (128, 4096, 4096), (104, 28672, 2048),
                                   (777, 1000, 1040)])
def test_other_products_variables_choose_nothing_here(gpu_lib, tunables, m, n, k, fp8):
    """KCMM_GEMM_SPLITS and KCMM_GEMM_TILE are the other products' while
    KCMM_EPI_TILE is not set, also where they name a split or a tile that the
    256-row tiles cannot have."""
    import torch
    usual = captured(torch, gpu_lib, m, n, k, fp8)
    for name, values in (("KCMM_GEMM_SPLITS", "1 2 3 8"), ("KCMM_GEMM_TILE", "0 101 104 112")):
        for v in values.split():
            tunables.setenv(name, v)
            assert captured(torch, gpu_lib, m, n, k, fp8) == usual, (name, v)
        tunables.delenv(name)


def whole_numbers(torch, lib, m, n, k, fp8):
    rng = np.random.default_rng([m, n, k, fp8])
    x = rng.integers(-3, 4, (m, k)).astype(np.float32)
    w = rng.integers(-3, 4, (n, k)).astype(np.float32)
    bias = E.bf16(rng.integers(-100, 101, n))
    res = E.bf16(rng.integers(-100, 101, (m, n)))
    xs = ws = None
    z = x @ w.T                                       # exact: below 2^24
    assert 9 * k < 2 ** 20
    if fp8:
        xs, ws = np.exp2(rng.integers(-1, 2, m)), np.exp2(rng.integers(-1, 2, n))
        z = z * E.f32(xs)[:, None] * E.f32(ws)
    got = call(torch, lib, x.astype(np.float64) if fp8 else x, w.astype(np.float64) if fp8 else w, xs, ws,
               bias, res, ACT_NONE)
    return np.array_equal(got, E.bf16(z + bias + res))


# 100 + 10 * (height of the last half of the weight tiles) + height, in 64 tokens
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heights", [101, 102, 103, 104, 112, 113, 114, 121, 123, 124, 132, 134, 141, 143])
def test_every_height_of_the_256_row_tiles(gpu_lib, tunables, heights, fp8):
    """Each height alone and with another for the last half of the weight tiles:
    an odd number of weight tiles the last of which ends inside, one weight tile (no
    second height), tokens of less than a tile, of whole ones, of a ragged last one."""
    import torch
    tunables.setenv("KCMM_EPI_TILE", "100")
    tunables.setenv("KCMM_GEMM_TILE", str(heights))
    for m, n, k in [(1, 520, 144), (63, 1283, 272), (256, 513, 1040), (385, 1283, 400), (701, 1100, 272),
                    (130, 200, 2064), (1025, 770, 64)]:
        assert whole_numbers(torch, gpu_lib, m, n, k, fp8), (m, n, k)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(449, 34547, 384), (1115, 23342, 736)])
def test_two_heights_where_they_are_chosen(gpu_lib, m, n, k, fp8):
    """Whole rounds of high tiles and a last one of lower tiles.  bf16: the 256-row
    kernel with more workgroups than tiles of any one height make."""
    import torch
    if not fp8:
        (grid, block), = captured(torch, gpu_lib, m, n, k, fp8)
        tiles = -(-n // 256)
        assert block[0] == 512 and grid[0] not in [tiles * -(-m // (64 * h)) for h in (1, 2, 3, 4)]
    assert whole_numbers(torch, gpu_lib, m, n, k, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
@pytest.mark.parametrize("m,n,lines", [(130, 300, 32), (300, 513, 35), (70, 1025, 44)])
def test_k_splits_of_the_256_row_tiles(gpu_lib, tunables, m, n, lines, splits, fp8):
    """K in 1 to 8 shares (of 35 lines, asked for as 40, the last share is shorter;
    44 lines end inside the last): bit for bit on whole numbers, and K
    is shared.  A sum of 2^16 that 2^-9 is added to line by line stays 2^16, whose
    steps are 2^-7; in a share of its own the small ones are a sum that it does not lose."""
    import torch
    tunables.setenv("KCMM_EPI_TILE", "100")
    tunables.setenv("KCMM_GEMM_SPLITS", str(splits))
    per = 128 if fp8 else 64
    k = lines * per - (16 if lines == 44 else 0)
    assert whole_numbers(torch, gpu_lib, m, n, k, fp8)
    x, w = np.zeros((m, k)), np.zeros((n, k))
    x[:, 0] = w[:, 0] = 256
    x[:, per::per], w[:, per::per] = 2.0 ** -4, 2.0 ** -5
    xs, ws = (np.ones(m), np.ones(n)) if fp8 else (None, None)
    got = call(torch, gpu_lib, x, w, xs, ws, None, np.full((m, n), -2.0 ** 16))
    small = lines - -(-lines // splits)               # lines of the shares after the first
    # each of at most 7 shares is added to 2^16 with a rounding to 2^-7
    assert np.all(np.abs(got - small * 2.0 ** -9) <= 7 * 2.0 ** -8)
    assert np.all((got > 0) == (splits > 1))
