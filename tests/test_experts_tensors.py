"""What the expert layer's Python calls refuse in torch tensors: another size or row pitch than the parameters give. Tensors of the
CPU stand in for the device's (a context without a device takes them for its own and refuses at the very end)."""
import pytest
import torch

import iree_b200 as ib

F16, BF16 = ib.KIND_F16, ib.KIND_BF16
HALF, I32, F32, U8 = torch.float16, torch.int32, torch.float32, torch.uint8


@pytest.fixture
def ctx(built):
    c = ib.Context.__new__(ib.Context)
    c.handle, c.ordinal = None, -1
    return c


def refusal(call, params, arrays, *more):
    with pytest.raises(ib.IreeB200Error, match="INVALID_ARGUMENT") as e:
        call(params, *arrays, *more)
    return str(e.value)


def check(call, params, good, bad, more=()):
    """Every array of `good` is let through; each of `bad`, (index, tensor), in its place is not."""
    assert "context" in refusal(call, params, good, *more)
    for i, x in bad:
        message = refusal(call, params, good[:i] + [x] + good[i + 1:], *more)
        assert "parameters say" in message, (i, tuple(x.shape), message)


def strided(rows, width, pitch, dtype=HALF):
    return torch.zeros(rows, pitch, dtype=dtype)[:, :width]


@pytest.mark.parametrize("M, N, K, group, lda, ldo", [(3, 40, 128, 32, 128, 40), (3, 40, 128, 64, 136, 48), (1, 40, 128, 128, 500, 900)])
def test_matvec(ctx, M, N, K, group, lda, ldo):
    p = ib.W4A16MatvecParams(F16, M, N, K, group, lda, ldo)
    scales = torch.zeros(N, K // group, dtype=HALF)
    good = [strided(M, K, lda), torch.zeros(N, K // 2, dtype=U8), scales, scales.clone(), strided(M, N, ldo)]
    bad = [(1, torch.zeros(N - 1, K // 2, dtype=U8)), (1, torch.zeros(N, K, dtype=U8)),
           (2, torch.zeros(N, K // group // 2, dtype=HALF)), (2, torch.zeros(N, 2 * K // group, dtype=HALF)),
           (3, torch.zeros(N, 0, dtype=HALF)),
           (0, torch.zeros(M, K - 32, dtype=HALF)), (0, strided(M, K - 8, lda)), (4, strided(M, N - 1, ldo))]
    if M > 1:
        bad += [(0, strided(M - 1, K, lda)), (0, strided(M, K, lda + 8)), (0, strided(M, K, 2 * lda)),
                (4, torch.zeros(M, ldo + 8, dtype=HALF)), (4, strided(M, N, ldo + 8)),
                (4, torch.zeros(1, N, dtype=HALF).expand(M, N))]
    check(ctx.w4a16_matvec, p, good, bad)
    assert "context" in refusal(ctx.w4a16_matvec, p, good[:3] + [None] + good[4:])


@pytest.mark.parametrize("run", [False, True])
def test_experts(ctx, run):
    E, P, N, K, group, lda, ldo = 3, 10, 24, 64, 32, 72, 32
    p = ib.W4A16ExpertsParams(F16, E, P, N, K, group, lda, ldo, ib.W4A16_EXPERTS_STREAM)
    scales = torch.zeros(E, N, K // group, dtype=HALF)
    good = [strided(P, K, lda), torch.zeros(E, N, K // 2, dtype=U8), scales, scales.clone(), torch.zeros(E + 1, dtype=I32),
            strided(P, N, ldo), torch.zeros(512, dtype=U8)]
    bad = [(0, strided(P - 1, K, lda)), (0, strided(P, K, K + 16)), (1, torch.zeros(E - 1, N, K // 2, dtype=U8)),
           (2, torch.zeros(N, K // group, dtype=HALF)), (3, torch.zeros(E, N, K // group + 1, dtype=HALF)),
           (4, torch.zeros(E, dtype=I32)), (5, strided(P, N, N + 16)), (5, strided(P - 1, N, ldo)),
           (6, torch.zeros(511, dtype=U8))]
    if run:
        check(ctx.w4a16_experts_run, p, good, bad, (ib.W4A16_EXPERTS_STREAM,))
    else:
        check(ctx.w4a16_experts, p, good, bad)
        take = {0: 0, 1: 1, 5: 2, 6: 3}
        check(ctx.w4a16_experts_prepare, p, [good[i] for i in take], [(take[i], x) for i, x in bad if i in take])


@pytest.mark.parametrize("T, k, D, tp, rp", [(5, 2, 16, 16, 16), (5, 2, 16, 24, 40), (1, 1, 16, 16, 16)])
def test_rows(ctx, T, k, D, tp, rp):
    E, P = 4, T * k
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, tp, rp)
    ids, weights, order = torch.zeros(T, k, dtype=I32), torch.zeros(T, k), torch.zeros(P, dtype=I32)
    x, rows, offsets = strided(T, D, tp), strided(P, D, rp), torch.zeros(E + 1, dtype=I32)
    small_x, small_rows, small_table = strided(T, D - 1, tp), strided(P, D - 1, rp), torch.zeros(T, 0, dtype=I32)
    tables = [small_table, torch.zeros(P - 1, dtype=I32)]
    if T > 1:
        tables += [torch.zeros(T, k + 1, dtype=I32), torch.zeros(T - 1, k, dtype=I32)]

    def bad_rows(i, rows_there, pitch):
        found = [(i, strided(rows_there, D - 1, pitch)), (i, torch.zeros(rows_there * D - 1, dtype=HALF))]
        if rows_there > 1:
            found += [(i, strided(rows_there - 1, D, pitch)), (i, strided(rows_there, D, pitch + 8))]
        return found

    def bad_tables(*at):
        return [(i, t) for i in at for t in tables]

    def bad_weights(*at):
        return [(i, t.to(F32)) for i in at for t in tables]

    check(ctx.expert_dispatch, p, [ids, x, offsets, ids.clone(), order, rows],
          bad_tables(0, 3) + bad_rows(1, T, tp) + bad_rows(5, P, rp) + [(2, torch.zeros(E, dtype=I32)), (4, torch.zeros(P - 1, dtype=I32))],
          (None,))
    check(ctx.expert_dispatch_backward, p, [rows, ids, x], bad_tables(1) + bad_rows(0, P, rp) + bad_rows(2, T, tp))
    check(ctx.expert_combine, p, [rows, weights, ids, x],
          bad_tables(2) + bad_weights(1) + bad_rows(0, P, rp) + bad_rows(3, T, tp))
    check(ctx.expert_combine_backward, p, [x, rows, weights, ids, strided(P, D, rp), weights.clone()],
          bad_tables(3) + bad_weights(2, 5) + bad_rows(0, T, tp) + bad_rows(1, P, rp) + bad_rows(4, P, rp))


def test_what_is_larger_or_cut_otherwise_is_taken(ctx):
    """Buffers for more rows than a call uses, rows split over dimensions, tables of one dimension, and nothing at all."""
    T, k, D, E = 5, 2, 16, 4
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, D, D)
    weights, ids = torch.zeros(T + 3, k), torch.zeros(T * k, dtype=I32)
    for rows in (torch.zeros(T * k + 7, D, dtype=HALF), torch.zeros(T, k, D, dtype=HALF), torch.zeros(T * k, 4, 4, dtype=HALF),
                 torch.zeros(T * k * D, dtype=HALF), torch.zeros(T * k + 7, 4, 4, dtype=HALF)):
        for out in (torch.zeros(T, D, dtype=HALF), torch.zeros(T + 1, 2, 8, dtype=HALF)):
            assert "context" in refusal(ctx.expert_combine, p, [rows, weights, ids, out])
    none = ib.ExpertRowsParams(F16, 0, k, E, 0, D, D, D)
    empty = torch.zeros(0, D, dtype=HALF)
    assert "context" in refusal(ctx.expert_dispatch, none, [torch.zeros(0, k, dtype=I32), empty, torch.zeros(E + 1, dtype=I32),
                                                            torch.zeros(0, k, dtype=I32), torch.zeros(0, dtype=I32), empty], None)
    narrow = ib.ExpertRowsParams(F16, T, k, E, 0, 0, 8, 8)
    assert "context" in refusal(ctx.expert_dispatch, narrow, [ids, torch.zeros(T, 0, dtype=HALF), torch.zeros(E + 1, dtype=I32),
                                                              ids, ids, torch.zeros(T * k, 0, dtype=HALF)], None)


def test_device_buffers_hold_what_the_parameters_say(ctx):
    made = []

    def buffer(nbytes):
        b = ib.DeviceBuffer.__new__(ib.DeviceBuffer)
        b.ctx, b.nbytes, b.ptr = ctx, nbytes, (len(made) + 1) << 20
        made.append(b)
        return b

    M, N, K = 2, 8, 64
    p = ib.W4A16MatvecParams(F16, M, N, K, 32, K, N)
    sizes = [2 * M * K, N * K // 2, 2 * N * 2, 2 * N * 2, 2 * M * N]
    assert "context" in refusal(ctx.w4a16_matvec, p, [buffer(n) for n in sizes])
    assert "context" in refusal(ctx.w4a16_matvec, p, [buffer(n + 5) for n in sizes])
    for i in range(5):
        message = refusal(ctx.w4a16_matvec, p, [buffer(n - (j == i)) for j, n in enumerate(sizes)])
        assert "buffer of" in message
    rows = ib.ExpertRowsParams(F16, 9000, 1, 4, 0, 8, 8, 8)
    sizes = [4 * 9000, 16 * 9000, 20, 4 * 9000, 4 * 9000, 16 * 9000, 149 * 16]
    assert "context" in refusal(ctx.expert_dispatch, rows, [buffer(n) for n in sizes])
    for i in range(7):
        assert "buffer of" in refusal(ctx.expert_dispatch, rows, [buffer(n - (j == i)) for j, n in enumerate(sizes)])
