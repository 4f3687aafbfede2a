"""Cases of the optimizer step beside the reduction: the global norm of many gradient tensors and the AdamW step with
states in 32 or in 8 bits, each on gradients that may still lie as several vectors (the local one and one per peer, as a
scatter-reduce round leaves them).

A case's tensors lie one behind the other in flat buffers, as a sharded optimizer keeps them: `tensors` of them with
`total` elements together, sizes spread over a factor of 400, each starting at a multiple of `align` elements. The first two
thirds have weight decay. Padding is zero and stays zero."""
import functools
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
BLOCK = 256  # elements that share the scale of an 8-bit state
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM = 3e-4, 0.9, 0.95, 1e-8, 0.1, 1.0
LOSS_SCALE = 1024.0  # of gradients in f16
Mi = 1 << 20


def _norm(name, tensors, total, grad, peers=0, align=256):
    return {"name": name, "op": "norm", "tensors": tensors, "total": total, "grad": grad, "peers": peers, "align": align, "overflow": False}


def _adamw(name, bits, tensors, total, grad, param="f32", copy="none", peers=0, clip=False, device=False, align=256, step=1000):
    return {"name": name, "op": "adamw", "bits": bits, "tensors": tensors, "total": total, "grad": grad, "param": param, "copy": copy,
            "peers": peers, "clip": clip, "device": device, "align": align, "step": step, "overflow": False}


def listed():
    return [
        # the gradients of one small layer: nothing but latency
        _norm("norm-small", 3, 1003, "f32"),
        # clipping before the step: all gradients of a model, in the type of its activations
        _norm("norm-model-bf16", 290, 64 * Mi, "bf16"),
        # last round of a radix-4 scatter-reduce over a shard: three peers' vectors folded, the fold written, its norm taken
        _norm("norm-fold4-f32", 40, 16 * Mi + 5, "f32", peers=3, align=1),
        # biases and norm weights alone
        _adamw("adamw32-small", 32, 24, 20011, "f32", step=1),
        # mixed precision with a clipped step that a graph may hold: step number and rate live on the device
        _adamw("adamw32-model-clip", 32, 290, 64 * Mi, "bf16", copy="bf16", clip=True, device=True),
        # the largest: one flat shard, everything in 32 bits
        _adamw("adamw32-shard-256Mi", 32, 1, 256 * Mi, "f32"),
        # no clipping: the step takes the four vectors of the last scatter-reduce round itself
        _adamw("adamw32-fold4", 32, 40, 32 * Mi + 9, "f32", copy="bf16", peers=3, align=1),
        # parameters in half precision, loss-scaled gradients, tensors packed without padding
        _adamw("adamw32-f16-packed", 32, 150, 8 * Mi + 77, "f16", param="f16", clip=True, align=1),
        _adamw("adamw8-small", 8, 24, 20011, "f32", step=1),
        _adamw("adamw8-model-clip", 8, 290, 64 * Mi, "bf16", copy="bf16", clip=True, device=True),
        _adamw("adamw8-shard-256Mi", 8, 1, 256 * Mi, "f32"),
        # parameters kept in bf16 alone, two ranks
        _adamw("adamw8-bf16-fold2", 8, 97, 24 * Mi + 3, "bf16", param="bf16", peers=1),
    ]


def draw(rng):
    spread = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))  # noqa: E731
    total = spread(1000, 64 * Mi)
    tensors = min(spread(1, 600), max(1, total // 64))
    grad, peers = rng.choice(("f32", "bf16", "f16")), rng.choice((0, 0, 1, 3, 7))
    if rng.random() < 0.35:
        c = _norm("", tensors, total, grad, peers, rng.choice((1, 256)))
        c["overflow"] = rng.random() < 0.15
    else:
        bits, param = rng.choice((32, 8)), rng.choice(("f32", "f32", "f32", "bf16", "f16"))
        copy = rng.choice(("none", "bf16", "f16")) if param == "f32" else "none"
        clip = rng.random() < 0.5
        c = _adamw("", bits, tensors, total, grad, param, copy, peers, clip, rng.random() < 0.4,
                   256 if bits == 8 else rng.choice((1, 256)), spread(1, 100000))
        c["overflow"] = clip and rng.random() < 0.15
    del c["name"]
    return c


def sizes_of(case):
    """Sizes of the case's tensors, and where each starts in the flat buffers; the last entry is the buffers' length."""
    n, total, align = case["tensors"], case["total"], case["align"]
    w = [math.exp(6.0 * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    sizes = [max(1, int((total - n) * x / sum(w))) for x in w]
    sizes[max(range(n), key=sizes.__getitem__)] += total - sum(sizes)
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + -(-s // align) * align)
    return sizes, starts


def decayed_of(case):
    """How many of the tensors, from the first, have weight decay."""
    return -(-2 * case["tensors"] // 3)


def grad_scale_of(case):
    return 1.0 / ((1 + case["peers"]) * (LOSS_SCALE if case["grad"] == "f16" else 1.0))


def quantize(x, positive):
    """Codes (e4m3) and one power-of-two scale per BLOCK elements: the smallest that keeps the block's largest magnitude at 448
    or below. `positive`: what is above zero stays above zero."""
    x = x.view(-1, BLOCK)
    e = (((x.abs().amax(1).view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_(min=1)
    y = x * ((254 - e) << 23).view(torch.float32)[:, None]
    if positive:
        y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).view(-1), (e << 23).view(torch.float32)


def dequantize(codes, scale):
    return (codes.view(-1, BLOCK).float() * scale[:, None]).view(-1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 7919 + 17)
    rand = lambda n: torch.rand(n, generator=gen, device=DEVICE)  # noqa: E731
    randn = lambda n: torch.randn(n, generator=gen, device=DEVICE)  # noqa: E731
    sizes, starts = sizes_of(case)
    n = starts[-1]
    # gradients of a tensor are of one magnitude, those of different tensors are not
    sigma = torch.zeros(2 * len(sizes), device=DEVICE)
    sigma[::2] = 10.0 ** (rand(len(sizes)) * 3 - 5)
    count = torch.tensor([x for i, s in enumerate(sizes) for x in (s, starts[i + 1] - starts[i] - s)], device=DEVICE)
    sigma = torch.repeat_interleave(sigma, count, output_size=n)
    used = (sigma > 0).float()
    lead = LOSS_SCALE if case["grad"] == "f16" else 1.0
    pitch = -(-n // 64) * 64
    grads = torch.zeros(1 + case["peers"], pitch, dtype=TYPES[case["grad"]], device=DEVICE)
    for row in grads:
        row[:n] = randn(n) * sigma * lead
    if case["overflow"]:
        grads[-1, starts[len(sizes) // 2]] = math.inf
    state = {"case": case, "grads": grads, "n": n, "grad_scale": grad_scale_of(case)}
    if case["op"] == "norm":
        state["stats"] = torch.zeros(2, dtype=torch.float64, device=DEVICE)
        if case["peers"]:
            state["folded"] = torch.zeros(n, dtype=grads.dtype, device=DEVICE)
    else:
        state["param"] = (randn(n) * 0.02 * used).to(TYPES[case["param"]])
        avg, sq = randn(n) * sigma * 0.3, sigma * sigma * (0.2 + rand(n))
        if case["bits"] == 8:
            state["avg"], state["avg_scale"] = quantize(avg, False)
            state["sq"], state["sq_scale"] = quantize(sq.sqrt(), True)
        else:
            state["avg"], state["sq"] = avg, sq
        if case["copy"] != "none":
            state["copy"] = state["param"].to(TYPES[case["copy"]])
        if case["clip"]:  # what the norm of this gradient gave
            g = grads[:, :n].double().sum(0)
            state["stats"] = torch.stack([g.square().sum(), (~torch.isfinite(g)).sum().double()])
            del g
        if case["device"]:  # the rate's 8 bytes, then the number of steps done
            state["clock"] = torch.tensor([0, case["step"] - 1], dtype=torch.int64, device=DEVICE)
            state["clock"][:1].view(torch.float64).fill_(LR)
        state["step"] = case["step"]
        state["decayed"] = starts[decayed_of(case)]
    if own:
        # the plan a user's program lays out once for its tensors
        state["plan"], state["args"] = _plan(state, sizes, starts)
    return state


# ---- the framework's operators -------------------------------------------------------------------------------------

def _plan(state, sizes, starts):
    from xccl_amd import mc
    from xccl_amd.types import BFLOAT16, Dt, Status
    kind = {"f32": Dt.FLOAT32, "bf16": BFLOAT16, "f16": Dt.FLOAT16, "none": Dt.UNSUPPORTED}
    case, grads = state["case"], state["grads"]
    if mc.xccl_mem_component_init() != Status.OK:
        raise RuntimeError("the ROCm component is not loaded")
    adamw = case["op"] == "adamw"
    layout = mc.StepLayout(grad_dtype=kind[case["grad"]], param_dtype=kind[case["param"] if adamw else "none"],
                           copy_dtype=kind[case["copy"] if adamw else "none"], state_bits=case["bits"] if adamw else 0,
                           n_peers=case["peers"], peer_stride=grads.stride(0) * grads.element_size())
    at = lambda name, start: state[name].data_ptr() + start * state[name].element_size() if name in state else None  # noqa: E731
    table = []
    for i, (size, start) in enumerate(zip(sizes, starts)):
        table.append(mc.StepTensor(
            grad=at("grads", start), peers=at("grads", start + grads.stride(0)) if case["peers"] else None, folded=at("folded", start),
            param=at("param", start), copy=at("copy", start), exp_avg=at("avg", start), exp_avg_sq=at("sq", start),
            exp_avg_scale=at("avg_scale", start // BLOCK), exp_avg_sq_scale=at("sq_scale", start // BLOCK), size=size,
            weight_decay=DECAY if adamw and i < decayed_of(case) else 0.0))
    args = None
    if adamw:
        args = mc.AdamwArgs(lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, grad_scale=state["grad_scale"], max_norm=MAX_NORM if case["clip"] else 0.0,
                            step=case["step"], stats=at("stats", 0), clock=at("clock", 0))
    return mc.StepPlan(layout, table), args


def _run_own(state):
    from xccl_amd import mc
    from xccl_amd.types import MemType, Status
    stream = mc.Stream(torch.cuda.current_stream().cuda_stream)
    if state["case"]["op"] == "norm":
        status, _ = mc.xccl_mem_component_grad_norm_nb(state["plan"].handle, state["stats"].data_ptr(), MemType.ROCM, stream, False)
    else:
        state["args"].step = state["step"]
        status, _ = mc.xccl_mem_component_adamw_nb(state["plan"].handle, state["args"], MemType.ROCM, stream, False)
    if status != Status.OK:
        raise RuntimeError(str(status))


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _folded(state):
    g = state["grads"][:, :state["n"]]
    return functools.reduce(lambda a, p: p.float() + a, g[1:], g[0].float())


def _plain_norm(state):
    a = _folded(state)
    if "folded" in state:
        state["folded"].copy_(a)
        a = state["folded"]
    state["stats"][0] = a.double().square().sum()
    state["stats"][1] = (~torch.isfinite(a)).sum()


def _plain_adamw(state):
    case = state["case"]
    scale, keep, lr, t = state["grad_scale"], None, LR, state["step"]
    if case["clip"]:
        scale = scale * torch.clamp(MAX_NORM / (state["stats"][0].sqrt() * scale + 1e-6), max=1.0)
        keep = state["stats"][1] == 0
    if case["device"]:
        lr, t = state["clock"][:1].view(torch.float64)[0], (state["clock"][1] + 1).double()
    c1, c2 = 1.0 - BETA1 ** t, (1.0 - BETA2 ** t) ** 0.5
    f32 = lambda x: x.float() if isinstance(x, torch.Tensor) else x  # noqa: E731
    g = _folded(state) * f32(scale)
    eight = case["bits"] == 8
    avg, sq = state["avg"], state["sq"]
    if eight:
        avg, sq = dequantize(avg, state["avg_scale"]), dequantize(sq, state["sq_scale"]).square()
    avg = avg * BETA1 + g * (1.0 - BETA1)
    sq = sq * BETA2 + (g * (1.0 - BETA2)) * g
    root = sq.sqrt()
    p = state["param"].float()
    k = state["decayed"]
    kept = torch.cat([p[:k] * f32(1.0 - lr * DECAY), p[k:]])
    p = kept - f32(lr / c1) * (avg / (root * f32(1.0 / c2) + EPS))
    new = {"param": p}
    if "copy" in state:
        new["copy"] = p
    if eight:
        new["avg"], new["avg_scale"] = quantize(avg, False)
        new["sq"], new["sq_scale"] = quantize(root, True)
    else:
        new["avg"], new["sq"] = avg, sq
    pick = lambda x, old: x if keep is None else torch.where(keep, x.to(old.dtype).view(old.dtype), old)  # noqa: E731
    list(map(lambda name: state[name].copy_(pick(new[name], state[name])), new))
    if case["device"]:
        state["clock"][1] += 1 if keep is None else keep


def run(state):
    if own:
        _run_own(state)
    elif state["case"]["op"] == "norm":
        _plain_norm(state)
    else:
        _plain_adamw(state)
    if state["case"]["op"] == "adamw":
        state["step"] += 1
    out = {name: state[name] for name in ("folded", "param", "copy", "avg", "avg_scale", "sq", "sq_scale") if name in state}
    if state["case"]["op"] == "norm":
        out["stats"] = state["stats"]
    if "clock" in state:
        out["steps"] = state["clock"][1:]
    return out


def work(case):
    n, grad = case["total"], BYTES[case["grad"]] * (1 + case["peers"])
    if case["op"] == "norm":
        return {"bytes": n * (grad + (BYTES[case["grad"]] if case["peers"] else 0)), "flops": n * (case["peers"] + 2)}
    states = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    skipped = case["overflow"]
    return {"bytes": 16 if skipped else n * (grad + 2 * BYTES[case["param"]] + BYTES[case["copy"]] + states),
            "flops": 0 if skipped else n * (case["peers"] + (16 if case["bits"] == 32 else 24))}


# ---- from the definition, in 64 bits -------------------------------------------------------------------------------

def _to_e4m3(y):
    """The nearest e4m3 value, ties to even, of numbers up to 448 in magnitude."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    sizes, starts = sizes_of(case)
    n, wide = state["n"], torch.float64
    a = torch.zeros(n, dtype=wide, device=DEVICE)
    for row in state["grads"]:
        a += row[:n].to(wide)
    if case["op"] == "norm":
        if case["peers"]:  # the norm is that of the fold as written, rounded: it has no value in 64 bits of its own
            return {"folded": a, "stats": None}
        return {"stats": torch.stack([(a * a).sum(), torch.isfinite(a).logical_not().sum().to(wide)])}
    # which of two neighbouring scales a block gets is a border
    out = {"avg_scale": None, "sq_scale": None, "steps": None}
    if case["clip"] and bool(state["stats"][1] != 0):  # skipped: what was there stays, bit for bit
        return {name: None for name in ("param", "copy", "avg", "avg_scale", "sq", "sq_scale", "steps")}
    scale = state["grad_scale"]
    if case["clip"]:
        norm = float(state["stats"][0]) ** 0.5 * scale
        scale *= min(1.0, MAX_NORM / (norm + 1e-6))
    m, v, p = state["avg"].to(wide), state["sq"].to(wide), state["param"].to(wide)
    if case["bits"] == 8:
        m *= state["avg_scale"].to(wide).repeat_interleave(BLOCK)
        v *= state["sq_scale"].to(wide).repeat_interleave(BLOCK)
        v *= v.clone()
    a *= scale
    m.mul_(BETA1).add_(a, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(a, a, value=1 - BETA2)
    t = case["step"]
    for i, start in enumerate(starts[:-1]):
        s = slice(start, start + sizes[i])
        if i < decayed_of(case):
            p[s] -= LR * DECAY * p[s]
    p -= LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out["param"] = p
    if "copy" in state:
        out["copy"] = p
    if case["bits"] == 32:
        out["avg"], out["sq"] = m, v
    else:
        for name, x in (("avg", m), ("sq", v.sqrt())):
            largest = x.view(-1, BLOCK).abs().amax(1).clamp(min=2.0 ** -110)
            unit = torch.exp2(torch.ceil(torch.log2(largest / 448.0)))
            y = _to_e4m3(x / unit.repeat_interleave(BLOCK))
            if name == "sq":
                y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
            out[name] = y
    return out
