"""The dispatch stream in the caller's hands: order against torch's work without a synchronisation, and between two streams."""
import ctypes as C

import numpy as np
import pytest

import iree_b200 as ib

F16 = ib.KIND_F16


def test_set_stream_needs_a_device(built):
    assert ib.library().iree_hal_b200_device_set_stream(C.c_void_p(None), C.c_void_p(1)) == 3


@pytest.fixture
def streams(built):
    """A context of its own, so that other tests keep their stream."""
    c = ib.Context(0)
    yield c
    c.set_stream(None)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("side", [False, True])
@pytest.mark.parametrize("recorded", [False, True])
def test_calls_are_in_order_with_torch(streams, side, recorded):
    """Inputs that torch is still writing, a result that torch reads at once, and buffers that torch hands out again; on the
    default stream and on another one."""
    import torch
    ctx = streams
    T, k, E, D = 512, 4, 16, 1024
    p = ib.ExpertRowsParams(F16, T, k, E, 0, D, D, D)
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    assert ctx.stream != stream.cuda_stream
    ctx.set_stream(stream)
    assert ctx.stream == (stream.cuda_stream or 1)
    generator = torch.Generator(device="cuda").manual_seed(5)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        i32 = dict(dtype=torch.int32, device="cuda")
        x, ids = torch.zeros(T, D, dtype=torch.float16, device="cuda"), torch.zeros(T, k, **i32)
        tables = torch.zeros(E + 1, **i32), torch.zeros(T, k, **i32), torch.zeros(T * k, **i32)
        rows, out = torch.zeros(T * k, D, dtype=torch.float16, device="cuda"), torch.zeros(T, D, dtype=torch.float16, device="cuda")

        def calls(ids, x, rows, out):
            ctx.expert_dispatch(p, ids, x, *tables, rows, None)
            ctx.expert_dispatch_backward(p, rows, tables[1], out)

        if recorded:
            ctx.begin_graph()
            calls(ids, x, rows, out)
            graph = ctx.end_graph()
        wrong = []
        for _ in range(8):
            new_x = torch.randint(-8, 9, (T, D), generator=generator, device="cuda").to(torch.float16)
            new_ids = torch.randint(0, E, (T, k), generator=generator, **i32)
            (big @ big).sum()                                # what the stream is busy with when the calls are made
            if recorded:
                x.copy_(new_x), ids.copy_(new_ids)
                graph.execute()
                wrong.append((out != 4 * new_x).any())
            else:
                fresh = torch.empty_like(rows), torch.empty_like(out)
                calls(new_ids, new_x, *fresh)
                wrong.append((fresh[1] != 4 * new_x).any())
        assert not torch.stack(wrong).any()
    if recorded:
        graph.release()


@pytest.mark.gpu
def test_work_queued_before_the_switch_is_waited_for(streams):
    import torch
    ctx = streams
    rng = np.random.default_rng(1)
    N, K = 28672, 4096
    wq, scales = ctx.to_device(rng.integers(0, 256, (N, K // 2), dtype=np.uint8)), ctx.to_device(np.full((N, K // 128), 0.01, np.float16))
    a = ctx.to_device(rng.integers(-3, 4, (1, K)).astype(np.float16))
    y, z = ctx.alloc(2 * N), ctx.alloc(2 * N)
    p = ib.W4A16MatvecParams(F16, 1, N, K, 128, K, N)
    copy = ib.ExpertRowsParams(F16, 1, 1, 1, 0, N, N, N)
    one, zero = ctx.to_device(np.ones(1, np.float32)), ctx.to_device(np.zeros(1, np.int32))
    other = torch.cuda.Stream()
    for stream in (other, None, other, torch.cuda.default_stream()):
        y.fill(0), z.fill(0)
        for _ in range(20):
            ctx.w4a16_matvec(p, a, wq, scales, None, y)
        ctx.set_stream(stream)
        ctx.expert_combine(copy, y, one, zero, z)
        got = z.download(np.uint16, (N,))
        assert (got == y.download(np.uint16, (N,))).all() and got.any()
    for b in (wq, scales, a, y, z, one, zero):
        b.free()
