"""What the expert layer's calls refuse, decided before any device is touched (no GPU needed)."""
import ctypes as C

import pytest

import iree_b200 as ib
from iree_b200.runtime import library

OK_PTR = 1 << 20   # an address the calls only look at (alignment); nothing is dispatched without a context


def status(name, params, *args):
    f = getattr(library(), "iree_b200_" + name)
    return f(None, C.addressof(params), *args)


def message():
    return library().iree_b200_last_error().decode()


def matvec(kind=ib.KIND_F16, M=1, N=64, K=128, group=128, lda=None, ldo=None):
    return ib.W4A16MatvecParams(kind, M, N, K, group, K if lda is None else lda, N if ldo is None else ldo)


def experts(kind=ib.KIND_F16, E=4, rows=8, N=64, K=128, group=128, lda=None, ldo=None, variant=0):
    return ib.W4A16ExpertsParams(kind, E, rows, N, K, group, K if lda is None else lda, N if ldo is None else ldo, variant)


def rows(kind=ib.KIND_F16, tokens=4, slots=2, E=4, first=0, width=64, tp=None, rp=None):
    return ib.ExpertRowsParams(kind, tokens, slots, E, first, width, width if tp is None else tp, width if rp is None else rp)


@pytest.mark.parametrize("params, code, words", [
    (matvec(kind=ib.KIND_I8), 12, "kind"), (matvec(M=-1), 3, "negative"), (matvec(N=-1, ldo=0), 3, "negative"),
    (matvec(K=0, lda=0), 3, "group"), (matvec(K=100), 3, "group"), (matvec(K=96, group=48), 3, "group"), (matvec(group=0), 3, "group"),
    (matvec(group=-32), 3, "group"), (matvec(lda=127), 3, "pitch"), (matvec(ldo=63), 3, "pitch"), (matvec(M=17), 11, "rows"),
    (matvec(K=(1 << 20) + 32, group=32), 11, "K is"),
])
def test_matvec_parameters(built, params, code, words):
    assert status("w4a16_matvec", params, OK_PTR, OK_PTR, OK_PTR, None, OK_PTR) == code and words in message()


@pytest.mark.parametrize("ptrs, words", [
    ((None, OK_PTR, OK_PTR, None, OK_PTR), "NULL"), ((OK_PTR, None, OK_PTR, None, OK_PTR), "NULL"),
    ((OK_PTR, OK_PTR, None, None, OK_PTR), "NULL"), ((OK_PTR, OK_PTR, OK_PTR, None, None), "NULL"),
    ((OK_PTR, OK_PTR + 8, OK_PTR, None, OK_PTR), "16-byte"), ((OK_PTR + 1, OK_PTR, OK_PTR, None, OK_PTR), "2-byte"),
    ((OK_PTR, OK_PTR, OK_PTR + 1, None, OK_PTR), "2-byte"), ((OK_PTR, OK_PTR, OK_PTR, OK_PTR + 1, OK_PTR), "2-byte"),
    ((OK_PTR, OK_PTR, OK_PTR, None, OK_PTR + 1), "2-byte"), ((OK_PTR, OK_PTR, OK_PTR, OK_PTR, OK_PTR), "context"),
])
def test_product_pointers(built, ptrs, words):
    assert status("w4a16_matvec", matvec(), *ptrs) == 3 and words in message()
    a, w, s, z, o = ptrs
    assert status("w4a16_experts_run", experts(), a, w, s, z, OK_PTR, o, OK_PTR, 1) == 3 and words in message()


@pytest.mark.parametrize("params, code, words", [
    (experts(kind=ib.KIND_I8), 12, "kind"), (experts(E=0), 11, "experts"), (experts(E=1025), 11, "experts"),
    (experts(rows=-1), 3, "negative"), (experts(K=64), 3, "group"), (experts(lda=64), 3, "pitch"), (experts(variant=9), 3, "variant"),
])
def test_experts_parameters(built, params, code, words):
    assert status("w4a16_experts", params, OK_PTR, OK_PTR, OK_PTR, None, OK_PTR, OK_PTR, OK_PTR) == code and words in message()
    out = C.c_int32()
    assert library().iree_b200_w4a16_experts_prepare(None, C.byref(params), C.c_void_p(OK_PTR), C.c_void_p(OK_PTR), C.c_void_p(OK_PTR),
                                                     C.c_void_p(OK_PTR), C.byref(out)) == code


def test_experts_offsets(built):
    for offsets in (None, OK_PTR + 2):
        assert status("w4a16_experts_run", experts(), OK_PTR, OK_PTR, OK_PTR, None, offsets, OK_PTR, OK_PTR, 1) == 3
        assert "offsets" in message()


@pytest.mark.parametrize("params, code, words", [
    (rows(kind=ib.KIND_I8), 12, "kind"), (rows(tokens=-1), 3, "negative"), (rows(width=-1, tp=0, rp=0), 3, "negative"),
    (rows(slots=0), 11, "slots"), (rows(slots=257), 11, "slots"), (rows(E=0), 11, "experts"), (rows(E=1025), 11, "experts"),
    (rows(tokens=1 << 30, slots=2), 11, "31 bits"), (rows(tp=63), 3, "pitch"), (rows(rp=63), 3, "pitch"),
])
def test_rows_parameters(built, params, code, words):
    p, other = OK_PTR, OK_PTR + 4096
    for name, args in (("expert_dispatch", (p, p, p, p, p, p, p)), ("expert_dispatch_backward", (p, p, other)),
                       ("expert_combine", (p, p, p, other)), ("expert_combine_backward", (p, p, p, p, other, p))):
        assert status(name, params, *args) == code and words in message(), name
    assert library().iree_b200_expert_dispatch_workspace_bytes(C.byref(params)) == 0


@pytest.mark.parametrize("name, count, elements, tables, optional", [
    ("expert_dispatch", 7, (1, 5), (0, 2, 3, 4, 6), (6,)), ("expert_dispatch_backward", 3, (0, 2), (1,), ()),
    ("expert_combine", 4, (0, 3), (1, 2), ()), ("expert_combine_backward", 6, (0, 1, 4), (2, 3, 5), ()),
])
def test_rows_pointers(built, name, count, elements, tables, optional):
    good = [OK_PTR + 4096 * i for i in range(count)]
    assert status(name, rows(), *good) == 3 and "context" in message()
    for i in range(count):
        args = list(good)
        args[i] = None
        assert status(name, rows(), *args) == 3 and ("NULL" in message())
        assert ("context" in message()) == (i in optional)
    for i in elements:
        args = list(good)
        args[i] += 1
        assert status(name, rows(), *args) == 3 and "2-byte" in message()
    for i in tables:
        args = list(good)
        args[i] += 2
        assert status(name, rows(), *args) == 3 and "4-byte" in message()


def test_overlapping_results_are_refused(built):
    p, q = OK_PTR, OK_PTR + 4096
    assert status("expert_combine", rows(), p, q, q, p) == 3 and "overlap" in message()
    assert status("expert_dispatch_backward", rows(), p, q, p) == 3 and "overlap" in message()
    assert status("expert_combine_backward", rows(), q, p, q, q, p, q) == 3 and "overlap" in message()
    assert status("expert_combine_backward", rows(), p, q, q, q, p, q) == 3 and "overlap" in message()


def test_a_large_dispatch_needs_its_workspace(built):
    big = rows(tokens=8193, slots=1, E=16)
    need = library().iree_b200_expert_dispatch_workspace_bytes(C.byref(big))
    assert need >= 16 * 4
    p = OK_PTR
    assert status("expert_dispatch", big, p, p, p, p, p, p, None) == 3 and "workspace" in message()
    assert library().iree_b200_expert_dispatch_workspace_bytes(C.byref(rows(tokens=8192, slots=1))) == 0


def test_experts_tensor_variant(built):
    """Alignment and pitches of the tensor-core variant, its workspace, and run() without prepare()'s variant."""
    P = OK_PTR
    t = ib.W4A16_EXPERTS_TENSOR

    def run(params, a=P, w=P, o=P, ws=P, variant=t):
        return status("w4a16_experts_run", params, a, w, P, None, P, o, ws, variant)

    assert run(experts()) == 3 and "context" in message()
    assert run(experts(), variant=0) == 9 and "prepare" in message()
    assert run(experts(), variant=7) == 9
    for bad in (dict(a=P + 8), dict(o=P + 8)):
        assert run(experts(), **bad) == 3 and "16-byte" in message()
    assert run(experts(lda=129)) == 3 and run(experts(ldo=65)) == 3 and run(experts(E=1024, N=1 << 22, ldo=1 << 22)) == 3
    for ws in (None, P + 64):
        assert run(experts(), ws=ws) == 3 and "workspace" in message()
        out = C.c_int32()
        assert library().iree_b200_w4a16_experts_prepare(None, C.byref(experts(variant=t)), C.c_void_p(P), C.c_void_p(P),
                                                         C.c_void_p(P), C.c_void_p(ws), C.byref(out)) == 3
        assert "workspace" in message()
