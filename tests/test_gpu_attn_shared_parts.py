"""Decode attention of groups that share a prefix (kcmm_paged_attn_decode_shared):
the parts of a long prefix and their join, for every number of query heads a kv
head, against fp64 under the tolerance of test_gpu_attn_shared."""
import pytest

from lattice_amd.bindings import KV_BF16, KV_F16, KV_FP8
from tests.test_gpu_attn_shared import check

pytestmark = pytest.mark.gpu


# the page types and head widths whose parts are joined
SPLIT = [(KV_BF16, 128), (KV_F16, 128), (KV_FP8, 128), (KV_BF16, 64), (KV_F16, 64)]


@pytest.mark.parametrize("dtype,d", SPLIT)
@pytest.mark.parametrize("group", range(1, 17))
def test_heads_of_a_kv_head(gpu_lib, dtype, group, d):
    """Every width of the join's rows (group * d / 4 of its 256 threads): a few
    parts, and more than it takes at a time."""
    import torch
    check(torch, gpu_lib, dtype, 2 * group, 2, d, 16, [[(100, 133), (100, 101), (100, 164)], [(37, 70)]],
          seed=group)
    check(torch, gpu_lib, dtype, group, 1, d, 16, [[(2100, 2100 + 40 * i) for i in range(3)], [(0, 5)]], seed=group)
