"""What an epilogue product launches."""
import pytest

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
