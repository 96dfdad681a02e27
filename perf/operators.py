"""The expert-layer operators as measured work: 4-bit matrix-vector products, tokens sorted by expert and back, and the
experts' 4-bit products.

``run`` computes an operator in its plain form, or (``own``) through the framework's entry points. Sizes are this
repository's W4A16 configurations (11008 x 4096 and 28672 x 8192 weights) where they apply, else generic ones.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_contexts = {}


def listed():
    return [
        # one token through a projection of the 11008 x 4096 layer, finest groups, zero points: what decoding waits for
        dict(name="matvec_1_token", op="matvec", type="bf16", M=1, N=11008, K=4096, group=32, zeros=True),
        # a small odd projection for a few tokens: latency
        dict(name="matvec_small_odd", op="matvec", type="f16", M=3, N=1003, K=1376, group=32, zeros=False),
        # a decoding batch of 16 through the largest layer
        dict(name="matvec_batch_16", op="matvec", type="f16", M=16, N=28672, K=8192, group=128, zeros=True),
        # routing of a decoding batch
        dict(name="dispatch_decode", op="dispatch", type="bf16", tokens=8, slots=2, experts=8, width=4096, drop=0.0),
        # routing of a long prompt batch over many experts, the end of the batch being padding
        dict(name="dispatch_prompt", op="dispatch", type="bf16", tokens=8192, slots=8, experts=64, width=2048, drop=0.06),
        # the experts' first product for a decoding batch: weights are read once, by few rows each
        dict(name="experts_decode", op="experts", type="f16", tokens=4, slots=2, experts=8, N=11008, K=4096, group=128, zeros=False, drop=0.0),
        # many small experts, a chunk of tokens
        dict(name="experts_chunk", op="experts", type="bf16", tokens=250, slots=4, experts=32, N=1408, K=2048, group=64, zeros=True, drop=0.1),
        # the experts' first product for a prompt: bound by the tensor cores
        dict(name="experts_prompt", op="experts", type="f16", tokens=4096, slots=2, experts=8, N=11008, K=4096, group=128, zeros=True, drop=0.0),
        # back to token order for a decoding batch
        dict(name="combine_decode", op="combine", type="f16", tokens=16, slots=8, experts=64, width=2048, drop=0.0),
        # back to token order for a prompt
        dict(name="combine_prompt", op="combine", type="bf16", tokens=8192, slots=2, experts=8, width=4096, drop=0.0),
        # training: the gradients of a combine over many slots
        dict(name="combine_grad", op="combine_grad", type="bf16", tokens=4096, slots=8, experts=64, width=2048, drop=0.0),
        # training: the gradient of a dispatch whose rows are not a whole number of 16-byte pieces
        dict(name="dispatch_grad", op="dispatch_grad", type="f16", tokens=4095, slots=4, experts=16, width=2044, drop=0.03),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "dispatch", "experts", "experts", "combine", "combine_grad", "dispatch_grad"])
    c = dict(op=op, type=rng.choice(["f16", "bf16"]))
    if op in ("matvec", "experts"):
        group = rng.choice([32, 64, 128])
        if op == "matvec":
            c.update(M=rng.randint(1, 16), N=_log(rng, 64, 28672), K=group * max(1, _log(rng, 256, 8192) // group))
        else:
            slots = rng.choice([1, 2, 4, 6])
            experts = rng.choice([8, 16, 32])
            N = _log(rng, 64, 11008)
            K = group * max(1, _log(rng, 256, 4096) // group)
            while experts * N * K > 8 * 11008 * 4096:
                N = max(64, N // 2)
            c.update(tokens=max(1, _log(rng, 1, 8192) // slots), slots=slots, experts=experts, N=N, K=K, drop=rng.choice([0.0, 0.1]))
        c.update(group=group, zeros=rng.random() < 0.5)
        return c
    slots = rng.randint(1, 8)
    width = _log(rng, 64, 4096)
    width = width if rng.random() < 0.3 else max(8, width // 8 * 8)
    tokens = _log(rng, 1, 8192)
    while tokens * slots * width > 4096 * 8 * 2048:
        tokens //= 2
    c.update(tokens=tokens, slots=slots, experts=rng.choice([8, 16, 60, 128, 256]), width=width, drop=rng.choice([0.0, 0.05]))
    return c


def _routing(case, g):
    """Router decisions of a batch: distinct experts for each token, some experts more popular than others, the tokens
    at the end of the batch padding (no expert)."""
    T, k, E = case["tokens"], case["slots"], case["experts"]
    score = torch.rand(T, E, generator=g, device="cuda") + 0.3 * torch.rand(1, E, generator=g, device="cuda")
    ids = score.topk(k, dim=1).indices.to(torch.int32)
    kept = T - int(T * case["drop"])
    ids[kept:] = -1
    weights = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), dim=1)
    return ids, weights


def _sorted(ids, E):
    """What the dispatch says of the ids: counts before each expert, each slot's row (-1: none), each row's slot (-1)."""
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order], torch.arange(E + 1, device=ids.device))
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=ids.device)
    position = torch.where(key < E, place, torch.full_like(place, -1)).reshape(ids.shape)
    order = torch.where(key[order] < E, order, torch.full_like(order, -1))
    return offsets.to(torch.int32), position.to(torch.int32), order.to(torch.int32)


def _activations(g, rows, width, dt):
    """Hidden states: unit variance, a few channels an order of magnitude larger."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    big = torch.rand(1, width, generator=g, device="cuda") < 0.004
    return torch.where(big, x * 12, x).to(dt)


def _weights(g, experts, N, K, group, zeros, dt):
    wq = torch.randint(0, 256, (experts, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(experts, N, K // group, generator=g, device="cuda") * 0.045 + 0.005).to(dt)
    z = torch.randint(4, 12, (experts, N, K // group), generator=g, device="cuda").to(dt) if zeros else None
    return wq, s, z


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    dt = _TYPES[case["type"]]
    s = dict(case=case, op=case["op"])
    if case["op"] == "matvec":
        s["a"] = _activations(g, case["M"], case["K"], dt)
        s["wq"], s["scales"], s["zeros"] = _weights(g, 1, case["N"], case["K"], case["group"], case["zeros"], dt)
        s["out"] = torch.zeros(case["M"], case["N"], dtype=dt, device="cuda")
        return s
    T, k, E = case["tokens"], case["slots"], case["experts"]
    P = T * k
    s["ids"], s["weights"] = _routing(case, g)
    offsets, position, order = _sorted(s["ids"], E)
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "dispatch":
        D = case["width"]
        s["x"] = _activations(g, T, D, dt)
        s["offsets"], s["position"], s["order"] = torch.zeros(E + 1, **i32), torch.zeros(T, k, **i32), torch.zeros(P, **i32)
        s["rows"] = torch.zeros(P, D, dtype=dt, device="cuda")
        return s
    s["offsets"], s["position"], s["order"] = offsets, position, order
    if case["op"] == "experts":
        s["rows"] = _activations(g, P, case["K"], dt)
        s["wq"], s["scales"], s["zeros"] = _weights(g, E, case["N"], case["K"], case["group"], case["zeros"], dt)
        s["out"] = torch.zeros(P, case["N"], dtype=dt, device="cuda")
        # the batch's shape as the host knows it: experts with rows, most rows of one of them
        counts = (offsets[1:] - offsets[:-1]).cpu()
        s["active"] = counts.nonzero().reshape(-1).cuda()
        s["most"] = max(1, int(counts.max()))
        return s
    D = case["width"]
    s["rows"] = _activations(g, P, D, dt)
    if case["op"] == "combine":
        s["out"] = torch.zeros(T, D, dtype=dt, device="cuda")
    elif case["op"] == "combine_grad":
        s["dout"] = torch.randn(T, D, generator=g, device="cuda").to(dt)
        s["drows"] = torch.zeros(P, D, dtype=dt, device="cuda")
        s["dweights"] = torch.zeros(T, k, device="cuda")
    else:
        s["dx"] = torch.zeros(T, D, dtype=dt, device="cuda")
    return s


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["op"]](state)


# ---- plain forms ----------------------------------------------------------------------------------------------------------


def _dequantised(wq, scales, zeros, group):
    """[..., N, K/2] bytes -> [..., N, K] f32; element 2i in the low nibble of byte i."""
    q = torch.stack((wq & 15, wq >> 4), dim=-1).flatten(-2).to(torch.float32)
    q = q.unflatten(-1, (-1, group))
    if zeros is None:
        q = q - 16.0 * (q >= 8)
    else:
        q = q - zeros.to(torch.float32).unsqueeze(-1)
    return (q * scales.to(torch.float32).unsqueeze(-1)).flatten(-2)


def _plain_matvec(s):
    w = _dequantised(s["wq"][0], s["scales"][0], None if s["zeros"] is None else s["zeros"][0], s["case"]["group"])
    return (s["a"].to(torch.float32) @ w.t()).to(s["a"].dtype)


def _plain_dispatch(s):
    T, k = s["ids"].shape
    offsets, position, order = _sorted(s["ids"], s["case"]["experts"])
    token = order.clamp(min=0).to(torch.int64) // k
    rows = torch.where((order >= 0).unsqueeze(1), s["x"][token], torch.zeros((), dtype=s["x"].dtype, device="cuda"))
    return dict(offsets=offsets, position=position, order=order, rows=rows)


def _plain_experts(s):
    act, most, rows, offsets = s["active"], s["most"], s["rows"], s["offsets"].to(torch.int64)
    w = _dequantised(s["wq"][act], s["scales"][act], None if s["zeros"] is None else s["zeros"][act], s["case"]["group"])
    at = offsets[act].unsqueeze(1) + torch.arange(most, device="cuda")
    y = torch.bmm(rows.to(torch.float32)[at.clamp(max=rows.shape[0] - 1)], w.transpose(1, 2))
    row = torch.arange(rows.shape[0], device="cuda")
    which = (torch.searchsorted(offsets[act], row, right=True) - 1).clamp(min=0)
    y = y[which, (row - offsets[act][which]).clamp(max=most - 1)].to(rows.dtype)
    return torch.where((row < offsets[-1]).unsqueeze(1), y, torch.zeros((), dtype=rows.dtype, device="cuda"))


def _slots(s, rows):
    """[T, k, D] f32: each slot's row, zeros where it has none; and where it has one."""
    there = s["position"] >= 0
    picked = rows[s["position"].clamp(min=0).to(torch.int64)].to(torch.float32)
    return torch.where(there.unsqueeze(2), picked, torch.zeros((), device="cuda")), there


def _plain_combine(s):
    picked, _ = _slots(s, s["rows"])
    return (picked * s["weights"].unsqueeze(2)).sum(1).to(s["rows"].dtype)


def _plain_combine_grad(s):
    picked, there = _slots(s, s["rows"])
    dout = s["dout"].to(torch.float32).unsqueeze(1)
    dweights = (picked * dout).sum(2)
    k = s["ids"].shape[1]
    order = s["order"].to(torch.int64)
    slot = order.clamp(min=0)
    drows = (s["weights"].reshape(-1)[slot].unsqueeze(1) * s["dout"].to(torch.float32)[slot // k]).to(s["rows"].dtype)
    drows = torch.where((order >= 0).unsqueeze(1), drows, torch.zeros((), dtype=drows.dtype, device="cuda"))
    return dict(drows=drows, dweights=torch.where(there, dweights, torch.zeros((), device="cuda")))


def _plain_dispatch_grad(s):
    picked, _ = _slots(s, s["rows"])
    return picked.sum(1).to(s["rows"].dtype)


_PLAIN = dict(matvec=_plain_matvec, dispatch=_plain_dispatch, experts=_plain_experts, combine=_plain_combine,
              combine_grad=_plain_combine_grad, dispatch_grad=_plain_dispatch_grad)


# ---- through the framework --------------------------------------------------------------------------------------------------


def _context():
    """One per device and stream: its work is queued on torch's current stream, in order with whoever makes the inputs and
    reads the results."""
    import iree_b200
    device, stream = torch.cuda.current_device(), torch.cuda.current_stream()
    key = device, stream.cuda_stream
    if key not in _contexts:
        _contexts[key] = iree_b200.Context(device)
        _contexts[key].set_stream(stream)
    return _contexts[key]


def _run_own(s):
    """The calls of a program that keeps its context, parameter blocks, workspaces and (experts) prepared maps from call to
    call; they are made on a state's first pass, for the stream that is current then."""
    import iree_b200 as ib
    if "ctx" not in s:
        s["ctx"] = _context()
    ctx, case, op = s["ctx"], s["case"], s["op"]
    kind = ib.KIND_F16 if case["type"] == "f16" else ib.KIND_BF16
    if op == "matvec":
        if "p" not in s:
            s["p"] = ib.W4A16MatvecParams(kind, case["M"], case["N"], case["K"], case["group"], case["K"], case["N"])
        ctx.w4a16_matvec(s["p"], s["a"], s["wq"], s["scales"], s["zeros"], s["out"])
        return s["out"]
    if op == "experts":
        if "p" not in s:
            s["p"] = ib.W4A16ExpertsParams(kind, case["experts"], s["rows"].shape[0], case["N"], case["K"], case["group"],
                                           case["K"], case["N"], ib.W4A16_EXPERTS_AUTO)
            s["ws"] = ctx.w4a16_experts_workspace(s["p"])
            s["variant"] = ctx.w4a16_experts_prepare(s["p"], s["rows"], s["wq"], s["out"], s["ws"])
        ctx.w4a16_experts_run(s["p"], s["rows"], s["wq"], s["scales"], s["zeros"], s["offsets"], s["out"], s["ws"], s["variant"])
        return s["out"]
    if "p" not in s:
        s["p"] = ib.ExpertRowsParams(kind, case["tokens"], case["slots"], case["experts"], 0, case["width"], case["width"],
                                     case["width"])
    if op == "dispatch":
        if "ws" not in s:
            s["ws"] = ctx.expert_dispatch_workspace(s["p"])
        ctx.expert_dispatch(s["p"], s["ids"], s["x"], s["offsets"], s["position"], s["order"], s["rows"], s["ws"])
        return dict(offsets=s["offsets"], position=s["position"], order=s["order"], rows=s["rows"])
    if op == "combine":
        ctx.expert_combine(s["p"], s["rows"], s["weights"], s["position"], s["out"])
        return s["out"]
    if op == "combine_grad":
        ctx.expert_combine_backward(s["p"], s["dout"], s["rows"], s["weights"], s["position"], s["drows"], s["dweights"])
        return dict(drows=s["drows"], dweights=s["dweights"])
    ctx.expert_dispatch_backward(s["p"], s["rows"], s["position"], s["dx"])
    return s["dx"]


# ---- what a pass cannot do without, and its value in 64 bits ------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "matvec":
        M, N, K = case["M"], case["N"], case["K"]
        per_group = 4 if case["zeros"] else 2
        return dict(bytes=N * K / 2 + N * (K // case["group"]) * per_group + 2 * M * K + 2 * M * N, flops=2.0 * M * N * K)
    T, k, E = case["tokens"], case["slots"], case["experts"]
    kept = (T - int(T * case["drop"])) * k
    if op == "experts":
        N, K = case["N"], case["K"]
        active = E * (1 - (1 - min(1.0, k / E)) ** (kept // k))
        per_expert = N * K / 2 + N * (K // case["group"]) * (4 if case["zeros"] else 2)
        return dict(bytes=active * per_expert + 2 * kept * (K + N) + 4 * (E + 1), flops=2.0 * kept * N * K)
    D = case["width"]
    if op == "dispatch":
        return dict(bytes=12 * T * k + 4 * (E + 1) + 2 * kept // k * D + 2 * kept * D, flops=0.0)
    if op == "combine":
        return dict(bytes=8 * T * k + 2 * kept * D + 2 * T * D, flops=2.0 * kept * D)
    if op == "combine_grad":
        return dict(bytes=12 * T * k + 4 * kept * D + 2 * T * D, flops=3.0 * kept * D)
    return dict(bytes=4 * T * k + 2 * kept * D + 2 * T * D, flops=1.0 * kept * D)


def _exact_weights(wq, scales, zeros, group):
    b = wq.to(torch.int64)
    q = torch.empty(b.shape[0], b.shape[1] * 2, dtype=torch.float64, device=b.device)
    low, high = b % 16, b // 16
    if zeros is None:
        low, high = (low + 8) % 16 - 8, (high + 8) % 16 - 8
    q[:, 0::2], q[:, 1::2] = low.double(), high.double()
    if zeros is not None:
        q -= zeros.double().repeat_interleave(group, dim=1)
    return q * scales.double().repeat_interleave(group, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "matvec":
        w = _exact_weights(s["wq"][0], s["scales"][0], None if s["zeros"] is None else s["zeros"][0], case["group"])
        return torch.einsum("mk,nk->mn", s["a"].double(), w)
    if op == "experts":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        bounds = s["offsets"].tolist()
        for e in range(case["experts"]):
            lo, hi = bounds[e], bounds[e + 1]
            if hi > lo:
                z = None if s["zeros"] is None else s["zeros"][e]
                out[lo:hi] = s["rows"][lo:hi].double() @ _exact_weights(s["wq"][e], s["scales"][e], z, case["group"]).t()
        return out
    if op == "dispatch":
        rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for e in range(case["experts"]):  # whole numbers have to be equal anyway; the rows are copies
            t = torch.nonzero(s["ids"] == e)[:, 0]
            rows[at:at + t.numel()] = s["x"][t].double()
            at += t.numel()
        return dict(offsets=None, position=None, order=None, rows=rows)
    T, k, D = case["tokens"], case["slots"], case["width"]
    position = s["position"].to(torch.int64)
    out = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    if op == "combine_grad":
        drows = torch.zeros(T * k, D, dtype=torch.float64, device="cuda")
        dweights = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        t = torch.nonzero(position[:, j] >= 0).reshape(-1)
        p = position[t, j]
        r = s["rows"][p].double()
        if op == "combine":
            out[t] += r * s["weights"][t, j].double().unsqueeze(1)
        elif op == "dispatch_grad":
            out[t] += r
        else:
            d = s["dout"][t].double()
            dweights[t, j] = torch.einsum("td,td->t", r, d)
            drows[p] = d * s["weights"][t, j].double().unsqueeze(1)
    return dict(drows=drows, dweights=dweights) if op == "combine_grad" else out
