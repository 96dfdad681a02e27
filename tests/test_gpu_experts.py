"""4-bit matrix-vector products and the expert layer on the GPU, against plain forms in 64 bits.

Tolerances. A result is rounded once to its type: half a step, eps / 2 relative (f16 2^-11, bf16 2^-8), and 2^-25 absolute
where f16 has no more digits. Sums are f32: a block of up to 128 values passes through at most 8 matrix instructions and
as many for the sums of the activations, each off by at most a truncation (2^-23) of what it holds, which Q = sum |a| (q' + z')
bounds (q' the stored nibble, z' the zero point; f16 holds both 64, bf16 128 higher): 16 * 2^-23 * s Q in all. Adding the blocks and
the warps' parts rounds (K / 32 + 16) times to 2^-24 of W = sum |a w|.
"""
import numpy as np
import pytest

import iree_b200 as ib
from iree_b200 import workloads

pytestmark = pytest.mark.gpu

F16, BF16 = ib.KIND_F16, ib.KIND_BF16
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def to_bits(x, kind):
    """f32 array -> 16-bit patterns, round to nearest even."""
    x = np.asarray(x, np.float32)
    if kind == F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    rounded = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def to_f64(bits, kind):
    bits = np.asarray(bits, np.uint16)
    if kind == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def nan_bits(kind):
    return np.uint16(0x7E00 if kind == F16 else 0x7FC0)


class Weights:
    """[E, N, K] weights: stored nibbles, scales, zero points, and what they stand for in 64 bits."""

    def __init__(self, rng, kind, E, N, K, group, zeros, integer_zeros=True):
        self.q = rng.integers(0, 16, (E, N, K))
        self.wq = (self.q[..., 0::2] | (self.q[..., 1::2] << 4)).astype(np.uint8)
        self.scales = to_bits(rng.uniform(0.005, 0.05, (E, N, K // group)), kind)
        self.zeros = None
        s = np.repeat(to_f64(self.scales, kind), group, axis=-1)
        if zeros:
            z = rng.integers(0, 16, (E, N, K // group)) if integer_zeros else rng.uniform(0, 15, (E, N, K // group))
            self.zeros = to_bits(z, kind)
            z = np.repeat(to_f64(self.zeros, kind), group, axis=-1)
            self.w = (self.q - z) * s
            self.magnitude = (self.q + z + (256 if kind == BF16 else 128)) * s
        else:
            self.w = np.where(self.q >= 8, self.q - 16, self.q) * s
            self.magnitude = ((self.q ^ 8) + 8.0 + (256 if kind == BF16 else 128)) * s


def product_tolerance(a, w, magnitude, exact, kind, least=2.0 ** -25):
    K = a.shape[-1]
    Q, W = np.abs(a) @ magnitude.T, np.abs(a) @ np.abs(w).T
    return HALF_STEP[kind] * np.abs(exact) + least + 16 * 2.0 ** -23 * Q + (K / 32 + 16) * 2.0 ** -24 * W


def upload(ctx, x):
    return ctx.to_device(np.ascontiguousarray(x)) if x is not None else None


def free(*buffers):
    for b in buffers:
        if b is not None:
            b.free()


def run_matvec(ctx, kind, a_bits, weights, group, pad_a=0, pad_out=0, offset=0):
    """a_bits [M, K]; rows `pad_a` elements further apart, activations and result `offset` elements into their buffers."""
    M, K = a_bits.shape
    N = weights.wq.shape[1]
    lda, ldo = K + pad_a, N + pad_out
    host = np.full(offset + M * lda, nan_bits(kind), np.uint16)
    host[offset:].reshape(M, lda)[:, :K] = a_bits
    da, dw, ds, dz = (upload(ctx, x) for x in (host, weights.wq, weights.scales, weights.zeros))
    out = np.full(offset + M * ldo + 8, 0x5A5A, np.uint16)
    do = upload(ctx, out)
    p = ib.W4A16MatvecParams(kind, M, N, K, group, lda, ldo)
    ctx.w4a16_matvec(p, da.ptr + 2 * offset, dw, ds, dz, do.ptr + 2 * offset)
    got = do.download(np.uint16, out.shape)
    free(da, dw, ds, dz, do)
    body = got[offset:offset + M * ldo].reshape(M, ldo)
    assert (got[:offset] == 0x5A5A).all() and (got[offset + M * ldo:] == 0x5A5A).all()
    assert (body[:, N:] == 0x5A5A).all()      # nothing between the rows is written
    return body[:, :N]


def check_matvec(ctx, kind, M, N, K, group, zeros, seed=0, integer_zeros=True, **layout):
    rng = np.random.default_rng([seed, kind, M, N, K, group, int(zeros)])
    a = to_bits(rng.standard_normal((M, K)) * np.where(rng.random(K) < 0.01, 12, 1), kind)
    w = Weights(rng, kind, 1, N, K, group, zeros, integer_zeros)
    a64 = to_f64(a, kind)
    exact = a64 @ w.w[0].T
    got = to_f64(run_matvec(ctx, kind, a, w, group, **layout), kind)
    assert (np.abs(got - exact) <= product_tolerance(a64, w.w[0], w.magnitude[0], exact, kind)).all()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M, N, K, group", [
    (1, 1, 32, 32), (1, 17, 64, 64), (2, 75, 160, 32), (3, 1003, 1376, 32), (7, 250, 480, 96), (8, 333, 512, 128),
    (9, 160, 192, 64), (16, 300, 1024, 256), (5, 40, 8320, 128), (16, 70, 4224, 64), (11, 19, 8224, 32), (1, 2400, 4096, 128),
    (2, 5, 65536, 64), (12, 33, 40960, 128),
])
def test_matvec(ctx, kind, zeros, M, N, K, group):
    check_matvec(ctx, kind, M, N, K, group, zeros)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("layout", [dict(pad_a=8), dict(pad_a=3), dict(offset=1), dict(pad_out=5, offset=3), dict(pad_a=8, pad_out=8, offset=8)])
@pytest.mark.parametrize("M", [4, 13])
def test_matvec_pitches_and_alignments(ctx, kind, layout, M):
    check_matvec(ctx, kind, M, 90, 416, 32, True, **layout)


@pytest.mark.parametrize("M", [2, 16])
def test_matvec_more_rows_than_a_cta_holds_at_once(ctx, M):
    check_matvec(ctx, BF16, M, 148 * 530, 96, 32, True)     # over 512 weight rows per CTA


@pytest.mark.parametrize("kind", [F16, BF16])
def test_matvec_fractional_zero_points(ctx, kind):
    check_matvec(ctx, kind, 6, 130, 512, 64, True, integer_zeros=False)


@pytest.mark.parametrize("kind", [F16, BF16])
def test_matvec_small_and_large_activations(ctx, kind):
    """Activations down to the smallest f16 value (1e-30 in bf16) and up to thousands."""
    rng = np.random.default_rng(5)
    K, N = 256, 48
    w = Weights(rng, kind, 1, N, K, 128, True)
    for scale in (2.0 ** -24 if kind == F16 else 1e-30, 2.0 ** -14, 900.0):
        a = to_bits(rng.integers(-15, 16, (4, K)) * scale, kind)
        a64 = to_f64(a, kind)
        exact = a64 @ w.w[0].T
        got = to_f64(run_matvec(ctx, kind, a, w, 128), kind)
        # bf16 has f32's range: nothing absolute is lost there. (The term is left out, not taken off the sum: at 1e-30, 64
        # bits that hold 2^-25 keep nothing of the others, 2^-25 * 2^-53 being 2^-78.)
        tol = product_tolerance(a64, w.w[0], w.magnitude[0], exact, kind, 0.0 if kind == BF16 else 2.0 ** -25)
        ok = np.abs(got - exact) <= tol
        assert (ok | (np.abs(exact) > 65504)).all()


def test_matvec_infinity_and_nan_stay_in_their_row(ctx):
    rng = np.random.default_rng(6)
    w = Weights(rng, F16, 1, 64, 256, 128, False)
    a = to_bits(rng.standard_normal((5, 256)), F16)
    clean = run_matvec(ctx, F16, a, w, 128)
    a[1, 7] = 0x7C00
    a[3, 100] = 0x7E00
    got = run_matvec(ctx, F16, a, w, 128)
    for m in (0, 2, 4):
        assert (got[m] == clean[m]).all()
    assert not np.isfinite(to_f64(got[1], F16)).any() and np.isnan(to_f64(got[3], F16)).all()


def test_matvec_agrees_with_the_signed_product(ctx):
    """The symmetric form of the same weights through iree_b200_w4a16 (decode kernel): one f16 step apart at most."""
    from iree_b200.w4a16 import w4a16_numpy
    a, wq, s = workloads.c4_w4a16(8, N=512, K=4096, seed=3)
    want = w4a16_numpy(ctx, a, wq, s).astype(np.float64)
    w = Weights.__new__(Weights)
    w.wq, w.scales, w.zeros = wq[None], s.view(np.uint16)[None], None
    got = run_matvec(ctx, F16, a.view(np.uint16), w, 128).view(np.float16).astype(np.float64)
    assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(want) + 2e-3).all()


# ---- rows to experts and back ------------------------------------------------------------------------------------------------


def plain_dispatch(ids, E, first):
    flat = ids.reshape(-1).astype(np.int64) - first
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(E + 1))
    position = np.empty(flat.size, np.int64)
    position[order] = np.arange(flat.size)
    position[key == E] = -1
    return offsets, position.reshape(ids.shape), np.where(key[order] < E, order, -1)


def make_ids(rng, T, k, lo, hi):
    return rng.integers(lo, hi, (T, k)).astype(np.int32)


ROUTES = [  # tokens, slots, experts, first, width, pad_tokens, pad_rows, offset
    (0, 2, 5, 0, 64, 0, 0, 0), (1, 1, 1, 0, 8, 0, 0, 0), (1, 8, 64, 0, 4096, 0, 0, 0), (3, 2, 4, 4, 20, 0, 0, 0),
    (37, 6, 60, 0, 100, 4, 12, 0), (64, 2, 8, 0, 513, 0, 0, 0), (300, 4, 16, 16, 256, 8, 8, 8), (65, 3, 7, 0, 40, 1, 0, 1),
    (1000, 8, 128, 0, 24, 0, 0, 0), (1025, 8, 256, 0, 72, 0, 0, 0), (5000, 2, 1024, 0, 16, 0, 0, 0), (9001, 1, 3, -1, 9, 0, 0, 0),
    (40, 256, 33, 0, 8, 0, 0, 0), (33, 255, 9, 0, 12, 0, 0, 0),
]


@pytest.mark.parametrize("T, k, E, first, D, pad_t, pad_r, offset", ROUTES)
def test_dispatch(ctx, T, k, E, first, D, pad_t, pad_r, offset):
    rng = np.random.default_rng([T, k, E])
    ids = make_ids(rng, T, k, first - 2, first + E + 2)      # some outside on either side
    P, tp, rp = T * k, D + pad_t, D + pad_r
    x = rng.integers(0, 65536, (T, D)).astype(np.uint16)
    host = np.zeros(offset + max(T * tp, 1), np.uint16)
    host[offset:offset + T * tp].reshape(T, tp)[:, :D] = x
    dx, di = upload(ctx, host), upload(ctx, ids if ids.size else np.zeros(1, np.int32))
    doff, dpos, dord = (ctx.alloc(max(4 * n, 4)).fill(0x77) for n in (E + 1, P, P))
    rows0 = np.full(offset + P * rp + 8, 0x5A5A, np.uint16)
    dr = upload(ctx, rows0)
    p = ib.ExpertRowsParams(F16, T, k, E, first, D, tp, rp)
    ws = ctx.expert_dispatch_workspace(p)
    ctx.expert_dispatch(p, di, dx.ptr + 2 * offset, doff, dpos, dord, dr.ptr + 2 * offset, ws)
    offsets, position, order = plain_dispatch(ids, E, first)
    assert (doff.download(np.int32, (E + 1,)) == offsets).all()
    if P:
        assert (dpos.download(np.int32, (T, k)) == position).all()
        assert (dord.download(np.int32, (P,)) == order).all()
    got = dr.download(np.uint16, rows0.shape)
    want = rows0.copy()
    kept = order[order >= 0]
    want[offset:offset + P * rp].reshape(P, rp)[:kept.size, :D] = x[kept // k]
    assert (got == want).all()
    free(dx, di, doff, dpos, dord, dr, ws)


def test_dispatch_of_one_popular_expert_and_of_none(ctx):
    for ids, kept in ((np.full((2100, 4), 5, np.int32), 8400), (np.full((2100, 4), -1, np.int32), 0),
                      (np.full((3, 2), 2 ** 31 - 1, np.int32), 0)):
        T, k = ids.shape
        p = ib.ExpertRowsParams(BF16, T, k, 8, 0, 8, 8, 8)
        x = np.arange(T * 8).astype(np.uint16).reshape(T, 8)
        dx, di = upload(ctx, x), upload(ctx, ids)
        doff, dpos, dord, dr = ctx.alloc(36), ctx.alloc(4 * T * k), ctx.alloc(4 * T * k), ctx.alloc(16 * T * k).fill(0)
        ws = ctx.expert_dispatch_workspace(p)
        ctx.expert_dispatch(p, di, dx, doff, dpos, dord, dr, ws)
        assert doff.download(np.int32, (9,))[-1] == kept
        assert (dord.download(np.int32, (T * k,)) == np.where(np.arange(T * k) < kept, np.arange(T * k), -1)).all()
        if kept:
            assert (dr.download(np.uint16, (T, k, 8)) == x[:, None]).all()
        free(dx, di, doff, dpos, dord, dr, ws)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("T, k, E, first, D, pad_t, pad_r, offset", [r for r in ROUTES if r[0]])
def test_combine_and_gradients(ctx, kind, T, k, E, first, D, pad_t, pad_r, offset):
    rng = np.random.default_rng([T, k, E, 1])
    P, tp, rp = T * k, D + pad_t, D + pad_r
    _, position, order = plain_dispatch(make_ids(rng, T, k, first - 1, first + E + 1), E, first)
    position = position.astype(np.int32)
    there = position >= 0
    rows = np.full((P, rp), nan_bits(kind), np.uint16)       # rows behind the last one, and the gaps, are NaN
    kept = int(there.sum())
    rows[:kept, :D] = to_bits(rng.standard_normal((kept, D)), kind)
    weights = rng.standard_normal((T, k)).astype(np.float32)
    weights[~there] = np.inf                                 # a dropped slot's weight is not looked at
    dout = to_bits(rng.standard_normal((T, D)), kind)
    dout_host = np.full((T, tp), nan_bits(kind), np.uint16)
    dout_host[:, :D] = dout

    def shifted(x):
        return upload(ctx, np.concatenate([np.zeros(offset, np.uint16), x.reshape(-1), np.zeros(8, np.uint16)]))

    dr, dd = shifted(rows), shifted(dout_host)
    dw, dp = upload(ctx, weights), upload(ctx, position)
    do = shifted(np.full((T, tp), 0x5A5A, np.uint16))
    dg = shifted(np.full((P, rp), 0x5A5A, np.uint16))
    dx = shifted(np.full((T, tp), 0x5A5A, np.uint16))
    ddw = ctx.alloc(4 * P).fill(0x55)
    p = ib.ExpertRowsParams(kind, T, k, E, first, D, tp, rp)
    o = 2 * offset
    ctx.expert_combine(p, dr.ptr + o, dw, dp, do.ptr + o)
    ctx.expert_dispatch_backward(p, dr.ptr + o, dp, dx.ptr + o)
    ctx.expert_combine_backward(p, dd.ptr + o, dr.ptr + o, dw, dp, dg.ptr + o, ddw)

    picked = np.where(there[..., None], to_f64(rows[:, :D], kind)[np.maximum(position, 0)], 0.0)
    w64 = np.where(there, weights.astype(np.float64), 0.0)
    half = HALF_STEP[kind]

    def read(buf, n, pitch):
        return buf.download(np.uint16, (offset + n * pitch + 8,))[offset:offset + n * pitch].reshape(n, pitch)

    got = read(do, T, tp)
    exact = (picked * w64[..., None]).sum(1)
    tol = half * np.abs(exact) + 2.0 ** -25 + k * 2.0 ** -24 * np.abs(picked * w64[..., None]).sum(1)
    assert (np.abs(to_f64(got[:, :D], kind) - exact) <= tol).all() and (got[:, D:] == 0x5A5A).all()
    got = read(dx, T, tp)
    exact = picked.sum(1)
    tol = half * np.abs(exact) + 2.0 ** -25 + k * 2.0 ** -24 * np.abs(picked).sum(1)
    assert (np.abs(to_f64(got[:, :D], kind) - exact) <= tol).all() and (got[:, D:] == 0x5A5A).all()
    # gradients of the combine
    d64 = to_f64(dout, kind)
    got = read(dg, P, rp)
    slot = order[:kept]
    exact = w64.reshape(-1)[slot][:, None] * d64[slot // k]
    tol = half * np.abs(exact) + 2.0 ** -25 + 2.0 ** -24 * np.abs(exact)
    assert (np.abs(to_f64(got[:kept, :D], kind) - exact) <= tol).all()
    assert (got[kept:] == 0x5A5A).all() and (got[:, D:] == 0x5A5A).all()
    exact = (picked * d64[:, None]).sum(2)
    tol = (D / 32 + 16) * 2.0 ** -24 * np.abs(picked * d64[:, None]).sum(2)
    got = ddw.download(np.float32, (T, k)).astype(np.float64)
    assert (np.abs(got - exact) <= tol).all() and (got[~there] == 0).all()
    free(dr, dd, dw, dp, do, dg, dx, ddw)


def test_combine_gradients_against_differences(ctx):
    """<dout, out(rows + h u) - out(rows - h u)> / 2h against <drows, u>, and the same for the weights: out is linear in
    either, so in numbers that all roundings hold exactly the two are equal."""
    rng = np.random.default_rng(9)
    T, k, E, D = 6, 3, 4, 32
    _, position, _ = plain_dispatch(make_ids(rng, T, k, 0, E), E, 0)
    P = T * k
    rows, u = rng.integers(-4, 5, (2, P, D)).astype(np.float32)
    weights, v = rng.integers(-2, 3, (2, T, k)).astype(np.float32)
    dout = rng.integers(-3, 4, (T, D)).astype(np.float32)
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, D, D)
    dp = upload(ctx, position.astype(np.int32))

    def out(r, w):
        dr, dw, do = upload(ctx, to_bits(r, F16)), upload(ctx, w.astype(np.float32)), ctx.alloc(2 * T * D)
        ctx.expert_combine(p, dr, dw, dp, do)
        y = to_f64(do.download(np.uint16, (T, D)), F16)
        free(dr, dw, do)
        return y

    dr, dw, dd = upload(ctx, to_bits(rows, F16)), upload(ctx, weights), upload(ctx, to_bits(dout, F16))
    dg, ddw = ctx.alloc(2 * P * D), ctx.alloc(4 * P)
    ctx.expert_combine_backward(p, dd, dr, dw, dp, dg, ddw)
    drows, dweights = to_f64(dg.download(np.uint16, (P, D)), F16), ddw.download(np.float32, (T, k))
    assert (dout * (out(rows + u, weights) - out(rows - u, weights))).sum() / 2 == (drows * u).sum()
    assert (dout * (out(rows, weights + v) - out(rows, weights - v))).sum() / 2 == (dweights * v).sum()
    free(dp, dr, dw, dd, dg, ddw)


# ---- the experts' products ------------------------------------------------------------------------------------------------------


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def run_experts(ctx, kind, counts, rows, weights, group, a_bits, variant=0, pad_a=0, pad_out=0, offset=0):
    E, N = weights.wq.shape[:2]
    K = a_bits.shape[1]
    lda, ldo = K + pad_a, N + pad_out
    host = np.full(offset + rows * lda, nan_bits(kind), np.uint16)
    host[offset:].reshape(rows, lda)[:, :K] = a_bits
    da, dw, ds, dz, doff = (upload(ctx, x) for x in (host, weights.wq, weights.scales, weights.zeros, offsets_of(counts)))
    do = upload(ctx, np.full(offset + rows * ldo + 8, 0x5A5A, np.uint16))
    p = ib.W4A16ExpertsParams(kind, E, rows, N, K, group, lda, ldo, variant)
    ws = ctx.w4a16_experts_workspace(p)
    ctx.w4a16_experts(p, da.ptr + 2 * offset, dw, ds, dz, doff, do.ptr + 2 * offset, ws)
    got = do.download(np.uint16, (offset + rows * ldo + 8,))
    ctx.workspace_status(ws)
    free(da, dw, ds, dz, doff, do, ws)
    body = got[offset:offset + rows * ldo].reshape(rows, ldo)
    assert (got[offset + rows * ldo:] == 0x5A5A).all() and (body[:, N:] == 0x5A5A).all()
    assert (body[sum(counts):] == 0x5A5A).all()             # rows behind the last one are left as they were
    return body[:, :N]


def experts_tolerance(a, w, magnitude, exact, kind, variant):
    """TENSOR rounds a weight to the kind's type (half a step of |w|; q - z is exact for whole zero points) and adds K / 16
    products of 16 in f32, each off by at most 2^-23 of W so far; AUTO may be either."""
    tol = product_tolerance(a, w, magnitude, exact, kind)
    if variant == ib.W4A16_EXPERTS_STREAM:
        return tol
    W = np.abs(a) @ np.abs(w).T
    tensor = HALF_STEP[kind] * (np.abs(exact) + 1.01 * W) + 2.0 ** -25 + (a.shape[-1] / 16 + 1) * 2.0 ** -23 * W
    return tensor if variant == ib.W4A16_EXPERTS_TENSOR else np.maximum(tol, tensor)


def check_experts(ctx, kind, counts, N, K, group, zeros, spare=0, variant=0, seed=0, **layout):
    rng = np.random.default_rng([seed, kind, N, K, group, int(zeros), sum(counts)])
    E, rows = len(counts), sum(counts) + spare
    w = Weights(rng, kind, E, N, K, group, zeros)
    a = to_bits(rng.standard_normal((rows, K)), kind)
    a[sum(counts):] = nan_bits(kind)
    got = to_f64(run_experts(ctx, kind, counts, rows, w, group, a, variant, **layout), kind)
    a64, off = to_f64(a, kind), offsets_of(counts)
    for e in range(E):
        part = a64[off[e]:off[e + 1]]
        exact = part @ w.w[e].T
        tol = experts_tolerance(part, w.w[e], w.magnitude[e], exact, kind, variant)
        assert (np.abs(got[off[e]:off[e + 1]] - exact) <= tol).all(), e


EXPERT_SHAPES = [  # rows per expert, N, K, group
    ([1], 40, 64, 32), ([0, 3, 0, 1, 9], 75, 160, 32), ([2, 0, 0, 30], 130, 256, 64), ([0] * 70 + [5] + [0] * 9, 33, 128, 128),
    ([5, 14], 7, 32, 32), ([17, 1, 8, 16], 96, 480, 96), ([1] * 300, 20, 64, 64), ([100, 2], 200, 1024, 128), ([3, 4, 5, 6], 1003, 4128, 32),
]


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("counts, N, K, group", EXPERT_SHAPES)
def test_experts(ctx, variant, kind, zeros, counts, N, K, group):
    pad = -N % 8 if variant == ib.W4A16_EXPERTS_TENSOR else 0     # its result pitch is a multiple of 8
    check_experts(ctx, kind, counts, N, K, group, zeros, spare=3, variant=variant, pad_out=pad)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("counts", [[256], [257], [255, 64, 128], [600, 0, 1], [16, 17, 63, 64, 65, 66], [1025, 31]])
def test_experts_tensor_tiles(ctx, kind, counts):
    """Part tiles of every kind: whole and part pieces of 64 rows, parts of 16 and more rows, N that ends inside a tile."""
    check_experts(ctx, kind, counts, 200, 384, 64, True, variant=ib.W4A16_EXPERTS_TENSOR)


@pytest.mark.parametrize("layout", [dict(pad_a=8, pad_out=8), dict(pad_a=1), dict(offset=1), dict(pad_out=3), dict(pad_a=8, offset=8)])
@pytest.mark.parametrize("counts", [[4, 0, 21], [40, 70, 30]])
def test_experts_pitches_and_alignments(ctx, layout, counts):
    check_experts(ctx, BF16, counts, 72, 320, 64, True, spare=2, **layout)


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
def test_experts_without_rows(ctx, variant):
    check_experts(ctx, F16, [0, 0, 0], 64, 128, 128, False, spare=5, variant=variant)


def test_experts_tensor_refuses_what_its_copies_cannot_reach(ctx):
    rng = np.random.default_rng(3)
    w = Weights(rng, F16, 2, 24, 64, 32, False)
    a = to_bits(rng.standard_normal((8, 64)), F16)
    for layout in (dict(pad_a=1), dict(pad_out=1), dict(offset=4)):
        with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
            run_experts(ctx, F16, [4, 4], 8, w, 32, a, variant=ib.W4A16_EXPERTS_TENSOR, **layout)


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
def test_experts_whose_weights_pass_four_gigabytes(ctx, variant):
    """The last expert's weights and scales start 7.4 GB and 0.23 GB into their arrays."""
    import torch
    rng = np.random.default_rng(8)
    E, N, K, group, kind = 64, 28672, 8192, 128, F16
    counts = [2] + [0] * (E - 2) + [21]
    rows = sum(counts)
    wq = torch.full((E, N, K // 2), 0x77, dtype=torch.uint8, device="cuda")
    scales = torch.full((E, N, K // group), 0.0625, dtype=torch.float16, device="cuda")
    last = torch.from_numpy(rng.integers(0, 256, (N, K // 2), dtype=np.uint8))
    wq[-1].copy_(last)
    scales[-1] = 0.03125
    a = torch.from_numpy(rng.integers(-2, 3, (rows, K)).astype(np.float16)).cuda()
    out = torch.zeros(rows, N, dtype=torch.float16, device="cuda")
    offsets = torch.from_numpy(offsets_of(counts)).cuda()
    torch.cuda.synchronize()
    p = ib.W4A16ExpertsParams(kind, E, rows, N, K, group, K, N, variant)
    ws = ctx.w4a16_experts_workspace(p)
    ctx.w4a16_experts(p, a, wq, scales, None, offsets, out, ws)
    ctx.synchronize()
    ctx.workspace_status(ws)
    # whole numbers times powers of two: every step before the last rounding is exact
    pick = rng.integers(0, N, 200)
    q = np.stack([last.numpy()[pick] & 15, last.numpy()[pick] >> 4], axis=-1).reshape(len(pick), K).astype(np.float64)
    q[q >= 8] -= 16
    a64, got = a.cpu().numpy().astype(np.float64), out.cpu().numpy()
    assert (got[2:][:, pick] == (a64[2:] @ q.T * 0.03125).astype(np.float16)).all()
    assert (got[:2] == (a64[:2].sum(1, keepdims=True) * 7 * 0.0625).astype(np.float16)).all()
    ws.free()


def test_rows_that_pass_four_gigabytes(ctx):
    """2^20 rows of 2200: the last ones start 4.6 GB into their array."""
    import torch
    T, k, E, D = 1 << 19, 2, 16, 2200
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-9, 10, (T, D), generator=g, device="cuda", dtype=torch.int16).to(torch.float16)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    offsets, position, order = torch.zeros(E + 1, **i32), torch.zeros(T, k, **i32), torch.zeros(T * k, **i32)
    rows, out = torch.zeros(T * k, D, dtype=torch.float16, device="cuda"), torch.zeros(T, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, D, D)
    ws = ctx.expert_dispatch_workspace(p)
    ctx.expert_dispatch(p, ids, x, offsets, position, order, rows, ws)
    ctx.expert_dispatch_backward(p, rows, position, out)
    ctx.synchronize()
    want = torch.sort(ids.reshape(-1).long(), stable=True).indices
    assert (order.long() == want).all() and (position.reshape(-1)[want] == torch.arange(T * k, device="cuda")).all()
    for lo in range(0, T * k, 1 << 17):       # in parts: the comparison's own memory
        assert (rows[lo:lo + (1 << 17)] == x[want[lo:lo + (1 << 17)] // k]).all()
    assert (out == x + x).all()
    ws.free()


def test_experts_tensor_refuses_a_workspace_of_other_operands(ctx):
    """run() on a workspace that was never prepared, or for another result: nothing is computed and the status says so."""
    rng = np.random.default_rng(4)
    E, rows, N, K = 2, 40, 64, 128
    w = Weights(rng, F16, E, N, K, 128, False)
    da, dw, ds, doff = (upload(ctx, v) for v in (to_bits(rng.standard_normal((rows, K)), F16), w.wq, w.scales, offsets_of([18, 22])))
    do, other = (ctx.alloc(2 * rows * N).fill(0x5A) for _ in range(2))
    p = ib.W4A16ExpertsParams(F16, E, rows, N, K, 128, K, N, ib.W4A16_EXPERTS_TENSOR)
    fresh, ready = ctx.w4a16_experts_workspace(p), ctx.w4a16_experts_workspace(p)
    assert ctx.w4a16_experts_prepare(p, da, dw, do, ready) == ib.W4A16_EXPERTS_TENSOR
    for ws, out in ((fresh, do), (ready, other)):
        ctx.w4a16_experts_run(p, da, dw, ds, None, doff, out, ws, ib.W4A16_EXPERTS_TENSOR)
        with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
            ctx.workspace_status(ws)
        assert (out.download(np.uint8, (2 * rows * N,)) == 0x5A).all()
    free(da, dw, ds, doff, do, other, fresh, ready)


def test_arrays_of_another_kind_are_refused(ctx):
    """Host arrays, elements of another size and tensors elsewhere would be read as something they are not."""
    import torch
    p = ib.ExpertRowsParams(F16, 2, 2, 4, 0, 8, 8, 8)
    t = dict(ids=torch.zeros(2, 2, dtype=torch.int32), x=torch.zeros(2, 8, dtype=torch.float16), offsets=torch.zeros(5, dtype=torch.int32),
             position=torch.zeros(2, 2, dtype=torch.int32), order=torch.zeros(4, dtype=torch.int32), rows=torch.zeros(4, 8, dtype=torch.float16))
    good = [v.cuda() for v in t.values()]
    torch.cuda.synchronize()
    ctx.expert_dispatch(p, *good, None)
    ctx.synchronize()
    for i, v in enumerate(t.values()):
        for bad in (v, v.numpy(), good[i].to(torch.float64 if v.is_floating_point() else torch.int64)):
            with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
                ctx.expert_dispatch(p, *good[:i], bad, *good[i + 1:], None)


def test_arrays_with_gaps_are_refused(ctx):
    """Tables, weights and scales have no pitch; rows have one, but adjacent elements."""
    import torch
    T, k, E, D = 3, 2, 4, 16
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, 2 * D, 3 * D)
    i32, half = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.float16, device="cuda")
    ids = torch.tensor([[1, 0], [3, 9], [2, 2]], **i32)
    x = torch.arange(T * 2 * D, **half).reshape(T, 2 * D)[:, :D]
    offsets, position, order = torch.zeros(E + 1, **i32), torch.zeros(T, k, **i32), torch.zeros(T * k, **i32)
    rows = torch.zeros(T * k, 3 * D, **half)[:, :D]
    torch.cuda.synchronize()
    good = [ids, x, offsets, position, order, rows]
    ctx.expert_dispatch(p, *good, None)
    ctx.synchronize()
    assert position.tolist() == [[1, 0], [4, -1], [2, 3]]
    assert (rows[:5] == x[torch.tensor([0, 0, 2, 2, 1], device="cuda")]).all()
    for i, v in enumerate(good):
        # the same shape, but every other element; for rows also with whole planes between them
        gaps = torch.zeros(*v.shape, 2, dtype=v.dtype, device="cuda")[..., 0]
        planes = torch.zeros(2, *v.shape, dtype=v.dtype, device="cuda")[:, :1]
        for bad in (gaps, planes):
            with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
                ctx.expert_dispatch(p, *good[:i], bad, *good[i + 1:], None)
    weights = torch.ones(T, 2 * k, device="cuda")[:, :k]
    out = torch.zeros(T, 2 * D, **half)[:, :D]
    with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT"):
        ctx.expert_combine(p, rows, weights, position, out)
    ctx.expert_combine(p, rows, weights.contiguous(), position, out)
    ctx.synchronize()
    assert (out == x * torch.tensor([[2], [1], [2]], **half)).all()


def layer_buffers(ctx, rng, T, k, E, D, H, group, kind):
    x = to_bits(rng.standard_normal((T, D)), kind)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    weights = rng.random((T, k)).astype(np.float32)
    return x, ids, weights


@pytest.mark.parametrize("T", [24, 200])
def test_expert_layer_as_one_recorded_graph(ctx, T):
    """dispatch -> experts (up) -> experts (down) -> combine, recorded once and replayed on new tokens and new routing, early
    launches on and off; against the same layer in 64 bits with the middle rounded as the calls round it."""
    rng = np.random.default_rng(11)
    kind, k, E, D, H, group = BF16, 2, 8, 128, 192, 64
    P = T * k
    up, down = Weights(rng, kind, E, H, D, group, True), Weights(rng, kind, E, D, H, group, False)
    dup = [upload(ctx, v) for v in (up.wq, up.scales, up.zeros)]
    ddn = [upload(ctx, v) for v in (down.wq, down.scales)]
    dx, di, dw = ctx.alloc(2 * T * D), ctx.alloc(4 * P), ctx.alloc(4 * P)
    doff, dpos, dord = ctx.alloc(4 * (E + 1)), ctx.alloc(4 * P), ctx.alloc(4 * P)
    dr, dh, dy, do = ctx.alloc(2 * P * D), ctx.alloc(2 * P * H), ctx.alloc(2 * P * D), ctx.alloc(2 * T * D)
    pr = ib.ExpertRowsParams(kind, T, k, E, 0, D, D, D)
    p1 = ib.W4A16ExpertsParams(kind, E, P, H, D, group, D, H, 0)
    p2 = ib.W4A16ExpertsParams(kind, E, P, D, H, group, H, D, 0)
    ws, ws1, ws2 = ctx.expert_dispatch_workspace(pr), ctx.w4a16_experts_workspace(p1), ctx.w4a16_experts_workspace(p2)
    v1 = ctx.w4a16_experts_prepare(p1, dr, dup[0], dh, ws1)
    v2 = ctx.w4a16_experts_prepare(p2, dh, ddn[0], dy, ws2)

    def layer():
        ctx.expert_dispatch(pr, di, dx, doff, dpos, dord, dr, ws)
        ctx.w4a16_experts_run(p1, dr, dup[0], dup[1], dup[2], doff, dh, ws1, v1)
        ctx.w4a16_experts_run(p2, dh, ddn[0], ddn[1], None, doff, dy, ws2, v2)
        ctx.expert_combine(pr, dy, dw, dpos, do)

    graphs = []
    for overlap in (False, True):
        ctx.set_dispatch_overlap(overlap)
        ctx.begin_graph()
        layer()
        graphs.append(ctx.end_graph())
    try:
        for turn in range(4):
            x, ids, weights = layer_buffers(ctx, rng, T, k, E, D, H, group, kind)
            dropped = rng.random((T, k)) < 0.1
            ids[dropped] = -1
            dx.upload(x), di.upload(ids), dw.upload(weights)
            do.fill(0x5A)
            if turn == 3:
                layer()          # the last turn without a graph, early launches on
            else:
                graphs[turn % 2].execute()
            got = to_f64(do.download(np.uint16, (T, D)), kind)
            _, position, _ = plain_dispatch(ids, E, 0)
            want, bound = np.zeros((T, D)), np.full((T, D), 2.0 ** -25)
            for t in range(T):
                for j in range(k):
                    e = ids[t, j]
                    if e < 0:
                        continue
                    xe = to_f64(x[t], kind)
                    h64 = up.w[e] @ xe
                    h_tol = experts_tolerance(xe[None], up.w[e], up.magnitude[e], h64[None], kind, 0)[0]
                    y64 = down.w[e] @ h64
                    y_tol = experts_tolerance(h64[None], down.w[e], down.magnitude[e], y64[None], kind, 0)[0] * 1.01 + 1.01 * np.abs(down.w[e]) @ h_tol
                    want[t] += weights[t, j] * y64
                    bound[t] += weights[t, j] * (y_tol + k * 2.0 ** -24 * np.abs(y64))
            bound += HALF_STEP[kind] * (np.abs(want) + bound)
            assert (np.abs(got - want) <= bound).all(), turn
    finally:
        ctx.set_dispatch_overlap(False)
        for g in graphs:
            g.release()
    free(*dup, *ddn, dx, di, dw, doff, dpos, dord, dr, dh, dy, do, ws, ws1, ws2)


def test_results_do_not_depend_on_timing(ctx):
    """The same call fifty times on a busy stream: the same bits."""
    rng = np.random.default_rng(13)
    kind, M, N, K = F16, 16, 700, 2048
    w = Weights(rng, kind, 1, N, K, 128, True)
    a = to_bits(rng.standard_normal((M, K)), kind)
    da, dw, ds, dz = (upload(ctx, v) for v in (a, w.wq, w.scales, w.zeros))
    outs = [ctx.alloc(2 * M * N) for _ in range(50)]
    p = ib.W4A16MatvecParams(kind, M, N, K, 128, K, N)
    for o in outs:
        ctx.w4a16_matvec(p, da, dw, ds, dz, o)
    first = outs[0].download(np.uint16, (M, N))
    for o in outs[1:]:
        assert (o.download(np.uint16, (M, N)) == first).all()
    free(da, dw, ds, dz, *outs)
