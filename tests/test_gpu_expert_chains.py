"""Chains of the expert layer's calls and matrix-vector products that are launched early."""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import BF16, free, to_bits, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True])
def test_scales_written_two_dispatches_ahead(ctx, recorded):
    """combine (writes the scales) -> combine (of something else) -> matrix-vector product, dispatch overlap on: only the middle
    call is 'the dispatch ahead', so the product may not have fetched scales before the first one was done."""
    rng = np.random.default_rng(17)
    N, K, group, slots = 28672, 2048, 32, 8
    groups = K // group
    wq = upload(ctx, rng.integers(0, 256, (N, K // 2), dtype=np.uint8))
    a = upload(ctx, to_bits(rng.standard_normal((1, K)), BF16))
    rows = upload(ctx, to_bits(rng.uniform(0.001, 0.01, (N * slots, groups)), BF16))
    position = upload(ctx, rng.permutation(N * slots).astype(np.int32))
    weights, scales, out = ctx.alloc(4 * N * slots), ctx.alloc(2 * N * groups), ctx.alloc(2 * N)
    other, first = ctx.alloc(2 * 64), upload(ctx, np.zeros(1, np.int32))
    p_scales = ib.ExpertRowsParams(BF16, N, slots, 8, 0, groups, groups, groups)
    p_other = ib.ExpertRowsParams(BF16, 1, 1, 8, 0, 64, 64, 64)
    p = ib.W4A16MatvecParams(BF16, 1, N, K, group, K, N)

    def chain():
        ctx.expert_combine(p_scales, rows, weights, position, scales)
        ctx.expert_combine(p_other, rows, weights, first, other)
        ctx.w4a16_matvec(p, a, wq, scales, None, out)

    ctx.set_dispatch_overlap(True)
    graph = None
    try:
        if recorded:
            ctx.begin_graph()
            chain()
            graph = ctx.end_graph()
        for turn in range(6):
            factors = (rng.standard_normal((N, slots)) * 4.0 ** turn).astype(np.float32)
            weights.upload(factors)
            graph.execute() if recorded else chain()
            got = out.download(np.uint16, (N,))
            ctx.synchronize()
            out.fill(0)
            ctx.w4a16_matvec(p, a, wq, scales, None, out)     # the scales are there now
            assert (got == out.download(np.uint16, (N,))).all(), turn
    finally:
        ctx.set_dispatch_overlap(False)
        if graph:
            graph.release()
    free(wq, a, rows, position, weights, scales, out, other, first)
