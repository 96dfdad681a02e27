"""Every way through the 4-bit products' kernels, in numbers that all roundings before the last one hold exactly: whole
activations up to 2, scales that are powers of two and zero points whose distance from a nibble has few digits, so that a sum is a
whole number of steps below 2^24 and one wrong weight, scale, zero point or element of K shows.

Where weights are rounded (tensor-core products), they are compared with a product of weights rounded the same way: half a step of
round16((q - z)) s; what is left to allow for is the f32 sum, (K / 16 + 1) truncations of 2^-23 of W = sum |a w|, and half a step of
the result."""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import (BF16, F16, HALF_STEP, Weights, free, offsets_of, plain_dispatch, run_experts, run_matvec, to_bits,
                               to_f64, upload)

pytestmark = pytest.mark.gpu

STREAM, TENSOR = ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR


def exact_weights(rng, kind, E, N, K, group, zeros):
    """`zeros`: None, "whole" (0..15), "halves" (steps of 1/2) or "large" (up to 110); w is exact in the kind's type."""
    w = Weights(rng, kind, E, N, K, group, zeros is not None)
    s = 2.0 ** rng.integers(-4, 0, w.scales.shape)
    w.scales = to_bits(s, kind)
    if zeros is None:
        w.w = np.where(w.q >= 8, w.q - 16, w.q) * np.repeat(s, group, axis=-1)
    else:
        z = {"whole": rng.integers(0, 16, s.shape), "halves": rng.integers(0, 31, s.shape) / 2.0, "large": rng.integers(60, 111, s.shape)}[zeros]
        w.zeros = to_bits(z, kind)
        w.w = (w.q - np.repeat(z, group, axis=-1)) * np.repeat(s, group, axis=-1)
    return w


def whole_rows(rng, rows, K, kind):
    """Few activations other than 0, so that sums stay below 2^24 steps and results below f16's largest number."""
    a = rng.integers(-2, 3, (rows, K)) * (rng.random((rows, K)) < min(1.0, 300 / K))
    return a.astype(np.float64)


def check_exact_experts(ctx, kind, counts, N, K, group, zeros, variant, seed=0, spare=0, shift=0, **layout):
    rng = np.random.default_rng([seed, kind, N, K, group, len(counts)])
    w = exact_weights(rng, kind, len(counts), N, K, group, zeros)
    a = whole_rows(rng, sum(counts) + spare, K, kind)
    got = run_shifted(ctx, kind, counts, len(a), w, group, to_bits(a, kind), variant, shift, **layout)
    off = offsets_of(counts)
    for e in range(len(counts)):
        if counts[e]:
            exact = a[off[e]:off[e + 1]] @ w.w[e].T
            assert np.abs(exact).max() < 60000
            assert (got[off[e]:off[e + 1]] == to_bits(exact, kind)).all(), e


def run_shifted(ctx, kind, counts, rows, w, group, a_bits, variant, shift, **layout):
    """run_experts, or the same with scales and zero points `shift` elements into their buffers (2-byte boundaries will do)."""
    if not shift:
        return run_experts(ctx, kind, counts, rows, w, group, a_bits, variant, **layout)
    E, N, K = len(counts), w.wq.shape[1], a_bits.shape[1]
    ldo = N + layout.get("pad_out", 0)
    da, dw, doff = (upload(ctx, v) for v in (a_bits, w.wq, offsets_of(counts)))
    ds, dz = (v if v is None else upload(ctx, np.concatenate([np.full(shift, 0x7FFF, np.uint16), v.reshape(-1)])) for v in (w.scales, w.zeros))
    do = ctx.alloc(2 * rows * ldo).fill(0)
    p = ib.W4A16ExpertsParams(kind, E, rows, N, K, group, K, ldo, variant)
    ws = ctx.w4a16_experts_workspace(p)
    ctx.w4a16_experts(p, da, dw, ds.ptr + 2 * shift, dz and dz.ptr + 2 * shift, doff, do, ws)
    got = do.download(np.uint16, (rows, ldo))[:, :N]
    ctx.workspace_status(ws)
    free(da, dw, doff, ds, dz, do, ws)
    return got


SHAPES = [  # N, K, group: K / group a multiple of 8, of 4, of 2, odd; K inside a chunk of 128; groups of any multiple of 32
    (70, 256, 32), (70, 768, 32), (70, 512, 64), (33, 1024, 128), (70, 128, 32), (70, 1408, 32), (70, 384, 64), (70, 640, 128),
    (70, 96, 32), (70, 1376, 32), (70, 4128, 32), (33, 11008, 128), (33, 11008, 64), (70, 480, 96), (70, 480, 160), (70, 1536, 256),
    (20, 4032, 64), (20, 2112, 192),
]


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("zeros", [None, "whole", "halves", "large"])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("N, K, group", SHAPES)
def test_weights_scales_and_zero_points_of_every_layout(ctx, N, K, group, kind, zeros, shift):
    pad = -N % 8
    check_exact_experts(ctx, kind, [3, 0, 8], N, K, group, zeros, STREAM, shift=shift)
    check_exact_experts(ctx, kind, [9, 16, 40], N, K, group, zeros, STREAM, shift=shift)
    check_exact_experts(ctx, kind, [5, 0, 50], N, K, group, zeros, TENSOR, shift=shift, pad_out=pad)
    check_exact_experts(ctx, kind, [150, 300], N, K, group, zeros, TENSOR, shift=shift, pad_out=pad)


@pytest.mark.parametrize("zeros", [None, "whole"])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("N, K, group", SHAPES)
@pytest.mark.parametrize("M", [1, 8, 16])
def test_matvec_of_every_layout(ctx, M, N, K, group, kind, zeros):
    rng = np.random.default_rng([M, N, K, group, kind])
    w = exact_weights(rng, kind, 1, N, K, group, zeros)
    a = whole_rows(rng, M, K, kind)
    assert (run_matvec(ctx, kind, to_bits(a, kind), w, group) == to_bits(a @ w.w[0].T, kind)).all()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("counts, N, K", [([700, 0, 300], 128 * 60 - 24, 384), ([513, 1], 128 * 80, 160), ([40, 60, 1, 0, 64], 128 * 90 - 8, 256)])
def test_several_tiles_per_block(ctx, kind, counts, N, K):
    """300, 320 and 450 tiles of the 256-row and the 64-row kernel: accumulators handed over, rings carried on from tile to tile."""
    check_exact_experts(ctx, kind, counts, N, K, 32, "whole", TENSOR)


def test_several_tiles_per_block_with_reserved_sms(ctx):
    ctx.set_reserved_sms(130)
    try:
        check_exact_experts(ctx, F16, [300, 70], 128 * 11, 512, 64, "whole", TENSOR)
        check_exact_experts(ctx, BF16, [30, 7, 0, 11], 128 * 11, 512, 32, "whole", TENSOR)
        check_exact_experts(ctx, BF16, [30, 7, 0, 11], 1500, 512, 32, None, STREAM)
        check_exact_experts(ctx, F16, [3, 1, 0, 5], 1500, 512, 128, None, STREAM)
    finally:
        ctx.set_reserved_sms(0)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("group", [32, 1 << 20])
def test_the_longest_rows(ctx, kind, group):
    for variant in (STREAM, TENSOR):
        check_exact_experts(ctx, kind, [2, 17], 8, 1 << 20, group, "whole", variant)


@pytest.mark.parametrize("zeros", ["none", "whole", "fractional", "large"])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("counts, N, K, group", [([20, 0, 33], 72, 4128, 32), ([20, 0, 33], 72, 512, 32), ([150, 100], 136, 1408, 64), ([9, 60], 40, 1024, 128)])
def test_tensor_products_of_weights_rounded_once(ctx, kind, counts, N, K, group, zeros):
    rng = np.random.default_rng([kind, N, K, group])
    E = len(counts)
    w = Weights(rng, kind, E, N, K, group, zeros != "none", integer_zeros=zeros == "whole")
    if zeros == "large":
        w.zeros = to_bits(rng.uniform(60, 130, w.zeros.shape), kind)
    s = np.repeat(to_f64(w.scales, kind), group, axis=-1)
    if zeros == "none":
        q = np.where(w.q >= 8, w.q - 16.0, w.q)
    else:
        q = to_f64(to_bits(w.q - np.repeat(to_f64(w.zeros, kind), group, axis=-1), kind), kind)
    rounded = to_f64(to_bits(q * s, kind), kind)
    a_bits = to_bits(rng.standard_normal((sum(counts), K)), kind)
    got = to_f64(run_experts(ctx, kind, counts, sum(counts), w, group, a_bits, TENSOR), kind)
    a, off = to_f64(a_bits, kind), offsets_of(counts)
    for e in range(E):
        part = a[off[e]:off[e + 1]]
        exact, W = part @ rounded[e].T, np.abs(part) @ np.abs(rounded[e]).T
        tol = HALF_STEP[kind] * np.abs(exact) + 2.0 ** -25 + (K / 16 + 1) * 2.0 ** -23 * W
        assert (np.abs(got[off[e]:off[e + 1]] - exact) <= tol).all(), e


@pytest.mark.parametrize("variant", [0, STREAM, TENSOR])
def test_a_rank_that_owns_a_part_of_the_experts(ctx, variant):
    """8 of 64 experts: rows for all slots, of which an eighth is used. AUTO goes by the rows there are room for."""
    rng = np.random.default_rng(21)
    T, k, E, first, D, N = 64, 8, 8, 16, 256, 96
    P = T * k
    ids = np.stack([rng.permutation(64)[:k] for _ in range(T)]).astype(np.int32)
    offsets, position, order = plain_dispatch(ids, E, first)
    w = exact_weights(rng, BF16, E, N, D, 64, "whole")
    x = whole_rows(rng, T, D, BF16)
    dx, di, dw, ds, dz = (upload(ctx, v) for v in (to_bits(x, BF16), ids, w.wq, w.scales, w.zeros))
    doff, dpos, dord = (ctx.alloc(4 * n) for n in (E + 1, P, P))
    dr, do = ctx.alloc(2 * P * D).fill(0xFF), ctx.alloc(2 * P * N).fill(0x5A)
    p = ib.ExpertRowsParams(BF16, T, k, E, first, D, D, D)
    pe = ib.W4A16ExpertsParams(BF16, E, P, N, D, 64, D, N, variant)
    ws = ctx.w4a16_experts_workspace(pe)
    chosen = ctx.w4a16_experts_prepare(pe, dr, dw, do, ws)
    assert chosen == (variant or TENSOR)
    ctx.expert_dispatch(p, di, dx, doff, dpos, dord, dr, None)
    ctx.w4a16_experts_run(pe, dr, dw, ds, dz, doff, do, ws, chosen)
    got = do.download(np.uint16, (P, N))
    ctx.workspace_status(ws)
    used = offsets[E]
    assert 0 < used < P // 4
    for e in range(E):
        rows = order[offsets[e]:offsets[e + 1]]
        assert (got[offsets[e]:offsets[e + 1]] == to_bits(x[rows // k] @ w.w[e].T, BF16)).all()
    assert (got[used:] == 0x5A5A).all()
    free(dx, di, dw, ds, dz, doff, dpos, dord, dr, do, ws)


@pytest.mark.parametrize("variant, rows", [(STREAM, 40), (STREAM, 300), (TENSOR, 200), (TENSOR, 2000)])
def test_the_same_bits_every_time(ctx, variant, rows):
    rng = np.random.default_rng(rows)
    E, N, K, kind = 8, 1408, 2048, BF16
    counts = rng.multinomial(rows, np.ones(E) / E)
    w = Weights(rng, kind, E, N, K, 64, True)
    da, dw, ds, dz, doff = (upload(ctx, v) for v in (to_bits(rng.standard_normal((rows, K)), kind), w.wq, w.scales, w.zeros, offsets_of(counts)))
    p = ib.W4A16ExpertsParams(kind, E, rows, N, K, 64, K, N, variant)
    outs = [ctx.alloc(2 * rows * N) for _ in range(12)]
    spaces = [ctx.w4a16_experts_workspace(p) for _ in outs]
    for o, ws in zip(outs, spaces):
        ctx.w4a16_experts_prepare(p, da, dw, o, ws)
    for o, ws in zip(outs, spaces):
        ctx.w4a16_experts_run(p, da, dw, ds, dz, doff, o, ws, variant)
    first = outs[0].download(np.uint16, (rows, N))
    for o, ws in zip(outs, spaces):
        assert (o.download(np.uint16, (rows, N)) == first).all()
        ctx.workspace_status(ws)
    free(da, dw, ds, dz, doff, *outs, *spaces)
