"""The largest sizes of the expert layer's calls: what is refused (no GPU needed), and the widest rows that are not."""
import ctypes as C

import pytest

import iree_b200 as ib
from iree_b200.runtime import library

WIDEST = (1 << 31) - 1 - 4096
P = 1 << 20


def refused(name, params, *args):
    return getattr(library(), "iree_b200_" + name)(None, C.addressof(params), *args), library().iree_b200_last_error().decode()


@pytest.mark.parametrize("width", [WIDEST + 1, (1 << 31) - 256, (1 << 31) - 1])
def test_rows_that_end_beyond_31_bits(built, width):
    p = ib.ExpertRowsParams(ib.KIND_F16, 1, 1, 4, 0, width, width, width)
    for name, args in (("expert_dispatch", (P, P, P, P, P, P, None)), ("expert_dispatch_backward", (P, P, P << 9)),
                       ("expert_combine", (P, P, P, P << 9)), ("expert_combine_backward", (P, P, P, P, P << 9, P))):
        status, message = refused(name, p, *args)
        assert status == 11 and "wide" in message


def test_tensor_tiles_that_end_beyond_31_bits(built):
    """One expert of almost 2^31 weight rows: AUTO streams it, TENSOR refuses."""
    largest = (1 << 31) - 1 - 256
    for N, fits in ((largest - 7 & ~7, True), (largest + 1, False), ((1 << 31) - 8, False)):
        ldo = (N + 7) & ~7
        run = ib.W4A16ExpertsParams(ib.KIND_F16, 1, 9, N, 32, 32, 32, ldo, ib.W4A16_EXPERTS_TENSOR)
        status, message = refused("w4a16_experts_run", run, P, P, P, None, P, P, P, ib.W4A16_EXPERTS_TENSOR)
        assert status == 3 and ("context" in message) == fits and ("experts * N" in message) != fits


@pytest.mark.gpu
@pytest.mark.parametrize("width", [WIDEST, WIDEST - 3, WIDEST - 7])
def test_the_widest_rows(ctx, width):
    """2^31 - 4097 elements and the next widths of whole 8- and 16-byte pieces, one row each way."""
    import torch
    half = dict(dtype=torch.float16, device="cuda")
    x, rows, out = torch.ones(1, width, **half), torch.zeros(1, width, **half), torch.zeros(1, width, **half)
    for at in (0, 1, width // 2, width - 9, width - 1):
        x[0, at] = 3
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, offsets, position, order = torch.zeros(1, 1, **i32), torch.zeros(2, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32)
    weights = torch.full((1, 1), 2.0, device="cuda")
    torch.cuda.synchronize()
    p = ib.ExpertRowsParams(ib.KIND_F16, 1, 1, 1, 0, width, width, width)
    ctx.expert_dispatch(p, ids, x, offsets, position, order, rows, None)
    ctx.expert_combine(p, rows, weights, position, out)
    ctx.synchronize()
    assert offsets.tolist() == [0, 1] and torch.equal(rows, x) and torch.equal(out, x + x)
    ctx.expert_dispatch_backward(p, rows, position, out)
    ctx.synchronize()
    assert torch.equal(out, x)
