"""Results whose last columns are a part of a 16-byte piece, in rows that are whole pieces apart: what stands behind the last column
is somebody else's."""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import BF16, F16, check_experts, free, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("N", [1, 7, 70, 127, 129, 250, 260])
@pytest.mark.parametrize("counts", [[64], [64, 130, 63], [300, 90]])
def test_experts_tensor_products_leave_what_is_behind_their_columns(ctx, counts, N, kind):
    """Tiles of 64 and of 256 rows with whole pieces of 64 rows, which are stored by TMA where that writes N columns only."""
    check_experts(ctx, kind, counts, N, 160, 32, True, spare=2, variant=ib.W4A16_EXPERTS_TENSOR, pad_out=-N % 8)
    check_experts(ctx, kind, counts, N, 160, 32, True, spare=2, variant=ib.W4A16_EXPERTS_TENSOR, pad_out=-N % 8 + 24)


@pytest.mark.parametrize("M", [17, 64, 300])
@pytest.mark.parametrize("N, off", [(70, 0), (100, 8), (129, 16), (261, 0), (264, 8)])
def test_w4a16_column_blocks_leave_their_neighbours(ctx, M, N, off):
    """A rank's columns in a wider result: AUTO takes the TMA-storing kernel only for whole 16-byte pieces, which refuses others."""
    rng = np.random.default_rng([M, N])
    K, ldo = 256, 320
    a = rng.integers(-2, 3, (M, K)).astype(np.float16)
    q = rng.integers(0, 16, (N, K))
    wq, scales = (q[:, 0::2] | (q[:, 1::2] << 4)).astype(np.uint8), np.full((N, K // 128), 0.25, np.float16)
    want = (a.astype(np.float64) @ np.where(q >= 8, q - 16, q).T * 0.25).astype(np.float16)
    da, dw, ds = (upload(ctx, v) for v in (a, wq, scales))
    do = upload(ctx, np.full((M, ldo), 7.0, np.float16))
    ws = ctx.w4a16_workspace(N)
    p = ib.W4A16Params(M, N, K, 128, ldo, off, ib.W4A16_AUTO, 0)
    variant, tile_n = ctx.w4a16_prepare(p, da, dw, ds, do, ws)
    assert variant == (ib.W4A16_GEMM if N % 8 else ib.W4A16_GEMM_WT)
    ctx.w4a16_run(p, da, dw, ds, do, ws, variant, tile_n)
    got = do.download(np.float16, (M, ldo))
    ctx.workspace_status(ws)
    assert (got[:, off:off + N] == want).all() and (got[:, :off] == 7).all() and (got[:, off + N:] == 7).all()
    if N % 8:
        wt = ib.W4A16Params(M, N, K, 128, ldo, off, ib.W4A16_GEMM_WT, 0)
        with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
            ctx.w4a16_prepare(wt, da, dw, ds, do, ws)
        with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
            ctx.w4a16_run(wt, da, dw, ds, do, ws, ib.W4A16_GEMM_WT, 128)
    free(da, dw, ds, do, ws)
