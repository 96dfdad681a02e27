"""Which kernel a 4-bit product's plan names for results whose columns are no whole 16-byte pieces (no GPU needed)."""
import pytest

from iree_b200 import dispatch_gen as dg


@pytest.mark.parametrize("M", [17, 300])
def test_plans_of_part_pieces_do_not_store_by_tma(M):
    for N, n_offset in ((100, 0), (70, 8), (1, 0)):
        assert dg.plan_w4a16("part", M, N, 256, ldo=320, n_offset=n_offset).dispatches[-1].export == "b200_w4a16_gemm"
    assert dg.plan_w4a16("whole", M, 104, 256, ldo=320, n_offset=8).dispatches[-1].export == "b200_w4a16_gemm_wt"
