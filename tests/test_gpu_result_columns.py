"""Results whose last columns are a part of a 16-byte piece, in rows that are whole pieces apart: what stands behind the last column
is somebody else's."""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import BF16, F16, check_experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("N", [1, 7, 70, 127, 129, 250, 260])
@pytest.mark.parametrize("counts", [[64], [64, 130, 63], [300, 90]])
def test_experts_tensor_products_leave_what_is_behind_their_columns(ctx, counts, N, kind):
    """Tiles of 64 and of 256 rows with whole pieces of 64 rows, which are stored by TMA where that writes N columns only."""
    check_experts(ctx, kind, counts, N, 160, 32, True, spare=2, variant=ib.W4A16_EXPERTS_TENSOR, pad_out=-N % 8)
    check_experts(ctx, kind, counts, N, 160, 32, True, spare=2, variant=ib.W4A16_EXPERTS_TENSOR, pad_out=-N % 8 + 24)
