"""Chains of the expert layer's calls and matrix-vector products that are launched early."""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import BF16, F16, free, make_ids, plain_dispatch, to_bits, upload

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


@pytest.mark.parametrize("reserved", [0, 100, 146])
def test_a_recorded_dispatch_of_many_slots(ctx, reserved):
    """Count, scan and route as one recording, replayed on other ids with one workspace; also with most SMs left free."""
    rng = np.random.default_rng(reserved)
    T, k, E, D = 3001, 7, 200, 40
    P = T * k
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, D, D)
    x = rng.integers(0, 65536, (T, D)).astype(np.uint16)
    dx, di = upload(ctx, x), ctx.alloc(4 * P)
    doff, dpos, dord, dr = ctx.alloc(4 * (E + 1)), ctx.alloc(4 * P), ctx.alloc(4 * P), ctx.alloc(2 * P * D)
    ws = ctx.expert_dispatch_workspace(p)
    ctx.set_reserved_sms(reserved)
    try:
        ctx.begin_graph()
        ctx.expert_dispatch(p, di, dx, doff, dpos, dord, dr, ws)
        ctx.expert_dispatch(p, di, dx, doff, dpos, dord, dr, ws)
        graph = ctx.end_graph()
    finally:
        ctx.set_reserved_sms(0)
    for turn in range(4):
        ids = make_ids(rng, T, k, -20 * (turn % 2), E + 20) if turn else np.full((T, k), 199, np.int32)
        di.upload(ids)
        ws.fill(0xFF)
        graph.execute()
        offsets, position, order = plain_dispatch(ids, E, 0)
        assert (doff.download(np.int32, (E + 1,)) == offsets).all()
        assert (dpos.download(np.int32, (T, k)) == position).all() and (dord.download(np.int32, (P,)) == order).all()
        kept = order[order >= 0]
        assert (dr.download(np.uint16, (P, D))[:kept.size] == x[kept // k]).all()
    graph.release()
    free(dx, di, doff, dpos, dord, dr, ws)


def test_prepare_is_refused_while_a_graph_is_recorded(ctx):
    """... by the tensor-core variant, which would have to copy; what was recorded before and after still runs."""
    rng = np.random.default_rng(2)
    E, rows, N, K = 2, 40, 64, 128
    da, dw = upload(ctx, to_bits(rng.integers(-2, 3, (rows, K)), F16)), upload(ctx, rng.integers(0, 256, (E, N, K // 2), dtype=np.uint8))
    ds, doff = upload(ctx, to_bits(np.full((E, N, 1), 0.5), F16)), upload(ctx, np.array([0, 11, 40], np.int32))
    first, second = ctx.alloc(2 * rows * N).fill(0), ctx.alloc(2 * rows * N).fill(0)
    tensor = ib.W4A16ExpertsParams(F16, E, rows, N, K, 128, K, N, ib.W4A16_EXPERTS_TENSOR)
    stream = ib.W4A16ExpertsParams(F16, E, rows, N, K, 128, K, N, ib.W4A16_EXPERTS_STREAM)
    ws = ctx.w4a16_experts_workspace(tensor)
    ctx.w4a16_experts_prepare(tensor, da, dw, first, ws)
    ctx.begin_graph()
    ctx.w4a16_experts_run(tensor, da, dw, ds, None, doff, first, ws, ib.W4A16_EXPERTS_TENSOR)
    with pytest.raises(ib.IreeB200Error, match="FAILED_PRECONDITION"):
        ctx.w4a16_experts(tensor, da, dw, ds, None, doff, first, ws)
    ctx.w4a16_experts(stream, da, dw, ds, None, doff, second, ws)
    graph = ctx.end_graph()
    graph.execute()
    a, b = first.download(np.uint16, (rows, N)), second.download(np.uint16, (rows, N))
    ctx.workspace_status(ws)
    assert a.any() and (a == b).all()
    graph.release()
    free(da, dw, ds, doff, first, second, ws)
