"""4-bit products at the ends of their types' ranges, against 64 bits. Tolerances as in test_gpu_experts, and where bf16 sums
leave f32's normal numbers: the streaming kernels hold them 2^-15 times their value, so each of the (K / 32 + 16) additions is
off by at most half of 2^-149, 2^-135 of the value, and the result by half a step of bf16's last digit, 2^-134. (Products and
sums of activations are whole multiples of 2^-133 2^-15 = 2^-148 there, and exact.)"""
import numpy as np
import pytest

import iree_b200 as ib
from .test_gpu_experts import BF16, F16, Weights, offsets_of, product_tolerance, run_experts, run_matvec, to_bits, to_f64

pytestmark = pytest.mark.gpu

BF16_MAX = (2 - 2.0 ** -7) * 2.0 ** 127


def scaled_weights(rng, kind, E, N, K, group, zeros, factor):
    w = Weights(rng, kind, E, N, K, group, zeros)
    before = to_f64(w.scales, kind)
    w.scales = to_bits(before * factor, kind)
    ratio = np.repeat(to_f64(w.scales, kind) / before, group, axis=-1)
    w.w, w.magnitude = w.w * ratio, w.magnitude * ratio
    return w


def check_both(ctx, a64, w, group):
    """The matrix-vector product and the streamed experts' product of one expert."""
    M, K = a64.shape
    a = to_bits(a64, BF16)
    a64 = to_f64(a, BF16)
    exact = a64 @ w.w[0].T
    assert np.isfinite(exact).all() and (np.abs(exact) <= BF16_MAX).all()
    tol = product_tolerance(a64, w.w[0], w.magnitude[0], exact, BF16, 2.0 ** -134 + (K / 32 + 16) * 2.0 ** -135)
    got = to_f64(run_matvec(ctx, BF16, a, w, group), BF16)
    assert (np.abs(got - exact) <= tol).all()
    got = to_f64(run_experts(ctx, BF16, [M], M, w, group, a, ib.W4A16_EXPERTS_STREAM), BF16)
    assert (np.abs(got - exact) <= tol).all()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 12])
def test_bf16_activations_near_the_largest(ctx, M, group, zeros):
    """One activation of 3e36, and whole rows of the largest one: the sums that a result needs pass f32's range unscaled."""
    rng = np.random.default_rng([M, group, int(zeros)])
    K, N = 512, 70
    w = scaled_weights(rng, BF16, 1, N, K, group, zeros, 2.0 ** -14)
    a = rng.standard_normal((M, K))
    a[0, 5] = 3e36
    check_both(ctx, a, w, group)
    check_both(ctx, np.full((M, K), BF16_MAX), w, group)
    check_both(ctx, np.where(rng.random((M, K)) < 0.5, -BF16_MAX, BF16_MAX), w, group)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("scale", [2.0 ** -133, 2.0 ** -126, 2.0 ** -120, 2.0 ** -110])
def test_bf16_activations_near_the_smallest(ctx, scale, group, zeros):
    rng = np.random.default_rng([group, int(zeros)])
    K, N = 256, 48
    for factor in (1.0, 2.0 ** 10):
        w = scaled_weights(rng, BF16, 1, N, K, group, zeros, factor)
        check_both(ctx, rng.integers(-15, 16, (9, K)) * scale, w, group)


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("K, group", [(32, 32), (160, 32), (224, 32), (192, 64), (288, 96)])
@pytest.mark.parametrize("counts", [[5, 20], [150, 3]])
def test_weights_that_do_not_exist_are_not_formed(ctx, counts, K, group, kind, variant):
    """K that ends inside a chunk of 128: what stands behind it is stored nibble 0 by the reading, and 0 - zero point times the
    last scale is an infinity here, while the weights that there are are -scale or 0. Whole numbers times one scale: exact."""
    rng = np.random.default_rng([K, group, kind])
    E, N, scale = len(counts), 40, 6000.0 if kind == F16 else 3e37
    unit = 2.0 ** -6 if kind == F16 else 2.0 ** -30
    w = Weights(rng, kind, E, N, K, group, True)
    w.q = rng.integers(14, 16, (E, N, K))
    w.wq = (w.q[..., 0::2] | (w.q[..., 1::2] << 4)).astype(np.uint8)
    w.scales, w.zeros = to_bits(np.full(w.scales.shape, scale), kind), to_bits(np.full(w.scales.shape, 15.0), kind)
    s = to_f64(w.scales, kind)[0, 0, 0]
    a = rng.integers(-1, 2, (sum(counts), K)) * unit
    got = run_experts(ctx, kind, counts, sum(counts), w, group, to_bits(a, kind), variant)
    off = offsets_of(counts)
    for e in range(E):
        exact = a[off[e]:off[e + 1]] @ ((w.q[e] - 15) * s).T      # whole numbers up to 288, times one number of 11 bits
        assert (got[off[e]:off[e + 1]] == to_bits(exact, kind)).all()


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("step", [2.0 ** -14, 2.0 ** -18, 2.0 ** -24])
def test_f16_scales_without_a_leading_digit(ctx, step, zeros, variant):
    """Scales down to f16's smallest number, whole zero points: whole multiples of 2^-24, which 16 bits hold; the sums are whole
    multiples of the scale too."""
    rng = np.random.default_rng([int(-np.log2(step)), int(zeros)])
    counts, N, K, group = [20, 70], 40, 256, 64
    w = Weights(rng, F16, 2, N, K, group, zeros)
    times = rng.integers(1, 4, w.scales.shape)
    s = np.repeat(times * step, group, axis=-1)
    w.scales = to_bits(times * step, F16)
    q = w.q - np.repeat(to_f64(w.zeros, F16), group, axis=-1) if zeros else np.where(w.q >= 8, w.q - 16, w.q)
    a = rng.integers(-2, 3, (sum(counts), K)).astype(np.float64)
    got = run_experts(ctx, F16, counts, sum(counts), w, group, to_bits(a, F16), variant)
    off = offsets_of(counts)
    for e in range(2):
        assert (to_f64(got[off[e]:off[e + 1]], F16) == to_f64(to_bits(a[off[e]:off[e + 1]] @ (q[e] * s[e]).T, F16), F16)).all()


@pytest.mark.parametrize("variant", [ib.W4A16_EXPERTS_STREAM, ib.W4A16_EXPERTS_TENSOR])
@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("counts", [[7, 30], [200, 101]])
def test_what_is_not_finite_stays_in_its_row_and_column(ctx, counts, kind, variant):
    rng = np.random.default_rng(19)
    N, K, group, rows = 72, 320, 64, sum(counts)
    w = Weights(rng, kind, 2, N, K, group, True)
    a = to_bits(rng.standard_normal((rows, K)), kind)
    clean = run_experts(ctx, kind, counts, rows, w, group, a, variant)
    inf, nan = (0x7C00, 0x7E00) if kind == F16 else (0x7F80, 0x7FC0)
    a[2, 7], a[counts[0] - 1, 100], a[rows - 1, K - 1] = inf, nan, inf
    w.scales[0, 5, 1], w.zeros[1, 70, 4] = nan, nan
    got = run_experts(ctx, kind, counts, rows, w, group, a, variant)
    bad = np.zeros((rows, N), bool)
    bad[[2, counts[0] - 1, rows - 1]] = True
    bad[:counts[0], 5] = bad[counts[0]:, 70] = True
    assert (got[~bad] == clean[~bad]).all() and not np.isfinite(to_f64(got[bad], kind)).any()
