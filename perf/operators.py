"""What is measured of the matrix optimizer's operators: their cases, their plain forms and their values in 64 bits.

* ``momentum``: ``fairscale_amd.optim.momentum_pass`` over a list of gradients (unscale, moving average, Nesterov
  look-ahead, norm of each matrix, overflow flag);
* ``orthogonalize``: ``fairscale_amd.optim.orthogonalize`` over a list of matrices or batches of matrices;
* ``step``: ``fairscale_amd.optim.Muon.step`` over a list of parameters (all of it: momentum, orthogonalisation, update).

A case says its list as text, ``"4*4096x4096 2*8:64x512"``: four matrices of 4096 x 4096 and two batches of eight.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MOMENTUM = 0.95
LR = 2e-3
WEIGHT_DECAY = 0.1
GRAD_SCALE = 1024.0  # the loss scale of the fp16 gradients

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_LARGEST = "4*4096x4096 2*11008x4096 4096x11008"


def _shapes(text):
    """``"2*8:64x512 7x5"`` -> [(8, 64, 512), (8, 64, 512), (7, 5)]."""
    got = []
    for word in text.split():
        count, _, shape = word.rpartition("*")
        batch, _, matrix = shape.rpartition(":")
        rows, cols = matrix.split("x")
        got += [((int(batch),) if batch else ()) + (int(rows), int(cols))] * int(count or 1)
    return got


def listed():
    return [
        # one small adapter's matrices: a pass that is all latency
        {"name": "momentum_small_fp32", "op": "momentum", "list": "64x768 768x64", "type": "fp32", "nesterov": True},
        # a ragged list of odd sizes, fp16 gradients that carry a loss scale
        {"name": "momentum_ragged_fp16", "op": "momentum", "list": "1001x777 33x2049 513x4097 255x257 1x1000 1999x3", "type": "fp16", "nesterov": False},
        # the matrices of one layer of the 7B list (hidden 4096, FFN 11008)
        {"name": "momentum_layer_bf16", "op": "momentum", "list": _LARGEST, "type": "bf16", "nesterov": True},
        # one matrix of a small model: launches and latency
        {"name": "orth_small_fp32", "op": "orthogonalize", "list": "64x256", "type": "fp32"},
        # a projection taken head by head: 32 matrices of head size 128
        {"name": "orth_heads_bf16", "op": "orthogonalize", "list": "32:128x4096", "type": "bf16"},
        # odd sizes, wide and tall, in one list
        {"name": "orth_ragged_fp16", "op": "orthogonalize", "list": "1000x1777 2049x333 7x5 257x1023 129x4097", "type": "fp16"},
        # one square matrix of the 7B list: few tiles, long inner products
        {"name": "orth_4096_bf16", "op": "orthogonalize", "list": "4096x4096", "type": "bf16"},
        # the feed-forward matrices of the 13B shard's model, to fp32 accuracy
        {"name": "orth_ffn_fp32", "op": "orthogonalize", "list": "5120x13824", "type": "fp32"},
        # six attention blocks of the GPT-2-small list: fp32 masters, scaled fp16 gradients, fp16 copies
        {"name": "step_gpt2_mixed", "op": "step", "list": "6*768x2304 6*768x768", "precision": "mixed", "type": "fp16", "nesterov": True},
        # a tiny fp32 model, tall, wide and thin matrices
        {"name": "step_small_full", "op": "step", "list": "96x96 3*32x96 40x10 1x64", "precision": "full", "type": "fp32", "nesterov": True},
        # eight experts' matrices as one parameter, bf16 with fp32 momentum
        {"name": "step_experts_bf16", "op": "step", "list": "8:1024x2816 8:2816x1024", "precision": "memory_efficient", "type": "bf16", "nesterov": True},
        # one layer of the 7B list, fp16 parameters and gradients
        {"name": "step_layer_fp16", "op": "step", "list": _LARGEST, "precision": "memory_efficient", "type": "fp16", "nesterov": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["momentum", "orthogonalize", "step"])
    case = {"op": op}
    if op == "step":
        case["precision"], case["type"] = rng.choice([("full", "fp32"), ("mixed", "fp16"), ("memory_efficient", "fp16"), ("memory_efficient", "bf16")])
    else:
        case["type"] = rng.choice(["fp32", "fp16", "bf16"])
    if op != "orthogonalize":
        case["nesterov"] = rng.random() < 0.75
    words, flops, elements = [], 0.0, 0
    for _ in range(rng.randint(1, 8)):
        short = _log_uniform(rng, 1, 4096)
        long = min(16384, _log_uniform(rng, short, 6 * short + 64))
        batch = _log_uniform(rng, 2, 32) if short <= 1024 and rng.random() < 0.3 else 1
        rows, cols = (short, long) if rng.random() < 0.6 else (long, short)
        flops += batch * _orth_flops(rows, cols)
        elements += batch * rows * cols
        if words and (flops > 8e12 or elements > 1.5e8):
            break
        words.append(("%d:" % batch if batch > 1 else "") + "%dx%d" % (rows, cols))
    case["list"] = " ".join(words)
    return case


def _orth_flops(rows, cols):
    """Of one matrix, with every symmetric product counted once: the iteration on the matrix itself, or on its Gram
    matrix with one product at either end, whichever is less."""
    s, l = min(rows, cols), max(rows, cols)
    return float(min(STEPS * (3 * s * s * l + s**3), 3 * s * s * l + (4 * STEPS - 3) * s**3))


def work(case):
    shapes = _shapes(case["list"])
    elements = sum(math.prod(s) for s in shapes)
    size = 4 if case["type"] == "fp32" else 2
    orth = sum((s[0] if len(s) == 3 else 1) * _orth_flops(*s[-2:]) for s in shapes)
    if case["op"] == "momentum":  # gradient and momentum read, momentum and update written
        return {"bytes": elements * (2 * size + 8), "flops": 10 * elements}
    if case["op"] == "orthogonalize":
        return {"bytes": elements * 2 * size, "flops": orth}
    master = {"full": 8, "mixed": 8 + 2, "memory_efficient": 4}[case["precision"]]  # parameter read and written, copy written
    return {"bytes": elements * (size + 8 + master), "flops": orth + 10 * elements}


def _matrix(shape, generator):
    """Values like a layer's gradient: noise, and a few directions that stand out of it."""
    rows, cols = shape[-2:]
    noise = torch.randn(shape, generator=generator, device="cuda")
    few = min(4, rows, cols)
    left = torch.randn((*shape[:-1], few), generator=generator, device="cuda")
    right = torch.randn((*shape[:-2], few, cols), generator=generator, device="cuda")
    return noise + torch.matmul(left, right) * (1.0 / math.sqrt(max(rows, cols)))


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    shapes, dtype = _shapes(case["list"]), _TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "orthogonalize":
        state["matrices"] = [(_matrix(s, generator) * 1e-3 * (8.0 if dtype == torch.float16 else 1.0)).to(dtype) for s in shapes]
        return state
    scale = GRAD_SCALE if dtype == torch.float16 else 1.0
    state["scale"] = scale
    state["grads"] = [(_matrix(s, generator) * 1e-3 * scale).to(dtype) for s in shapes]
    state["momenta"] = [_matrix(s, generator) * 2e-4 for s in shapes]
    if case["op"] == "step":
        stored = torch.float32 if case["precision"] == "full" else dtype
        params = [torch.randn(s, generator=generator, device="cuda") * 0.02 for s in shapes]
        state["params"] = [torch.nn.Parameter(p.to(stored)) for p in params]
        state["masters"] = [p.detach().float() for p in state["params"]] if case["precision"] == "mixed" else None
        for p, g in zip(state["params"], state["grads"]):
            p.grad = g
    return state


# ---- the plain form: elementary torch operations in 32 bits, rounded once at the end

def _plain_momentum(grad, buf, scale, nesterov):
    """Updates ``buf`` in place; returns the update in fp32."""
    r = grad.float() / scale
    buf.add_((r - buf) * (1.0 - MOMENTUM))
    return r + (buf - r) * MOMENTUM if nesterov else buf


def _plain_orthogonalize(update):
    a, b, c = COEFFICIENTS
    x = update.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1).contiguous() if tall else x
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    x = (x.double() / norm).float()
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-2, -1) if tall else x


def _plain_step(case, master, param, grad, buf, scale):
    update = _plain_orthogonalize(_plain_momentum(grad, buf, scale, case["nesterov"]))
    rows, cols = update.shape[-2:]
    p = param.detach().float() if master is None else master
    p = p * (1.0 - LR * WEIGHT_DECAY) - update * (LR * 0.2 * math.sqrt(max(rows, cols)))
    param.data.copy_(p)
    if master is not None:
        master.copy_(p)


def _run_plain(state):
    case = state["case"]
    if case["op"] == "orthogonalize":
        return [_plain_orthogonalize(m).to(m.dtype) for m in state["matrices"]]
    if case["op"] == "momentum":
        updates = [_plain_momentum(g, m, state["scale"], case["nesterov"]).to(g.dtype) for g, m in zip(state["grads"], state["momenta"])]
        norms = torch.stack([u.double().square().sum().sqrt().float() for u in updates])
        found = torch.stack([torch.logical_not(torch.isfinite(u).all()) for u in updates]).any().float().reshape(1)
        return {"updates": updates, "momenta": state["momenta"], "norms": norms, "found_inf": found}
    masters = state["masters"] or [None] * len(state["params"])
    [_plain_step(case, w, p, g, m, state["scale"]) for w, p, g, m in zip(masters, state["params"], state["grads"], state["momenta"])]
    return {"params": [p.detach() for p in state["params"]], "masters": state["masters"], "momenta": state["momenta"]}


# ---- the framework's operators

def _optimizer(state):
    """The optimizer a training program keeps, resumed with the momentum at hand."""
    from fairscale_amd.optim import Muon, Precision

    if "optimizer" not in state:
        precision = {"full": Precision.FULL_PRECISION, "mixed": Precision.MIXED_PRECISION,
                     "memory_efficient": Precision.MEMORY_EFFICIENT_MIXED_PRECISION}[state["case"]["precision"]]
        state["optimizer"] = optimizer = Muon(state["params"], lr=LR, weight_decay=WEIGHT_DECAY, momentum=MOMENTUM,
                                              nesterov=state["case"]["nesterov"], ns_coefficients=COEFFICIENTS, eps=EPS,
                                              ns_steps=STEPS, adjust_lr_fn="match_rms_adamw", precision=precision)
        for p, m in zip(state["params"], state["momenta"]):
            optimizer.state[p]["momentum_buffer"] = m
    return state["optimizer"]


def _run_own(state):
    from fairscale_amd.optim import momentum_pass, orthogonalize

    case = state["case"]
    if case["op"] == "orthogonalize":
        return orthogonalize(state["matrices"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if case["op"] == "momentum":
        got = momentum_pass(state["grads"], state["momenta"], MOMENTUM, nesterov=case["nesterov"], scale=state["scale"])
        return {"updates": got.updates, "momenta": state["momenta"], "norms": got.norms, "found_inf": got.found_inf}
    optimizer = _optimizer(state)
    optimizer.step(scale=state["scale"])
    masters = [w.detach() for w in optimizer.fp32_param_groups[0]["params"]] if case["precision"] == "mixed" else None
    return {"params": [p.detach() for p in state["params"]], "masters": masters,
            "momenta": [optimizer.state[p]["momentum_buffer"] for p in state["params"]]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits, on the right side of the matrix where the plain form works on the left

def _exact_orthogonal(update):
    a, b, c = COEFFICIENTS
    wide = update.shape[-2] < update.shape[-1]
    y = update.transpose(-2, -1).contiguous() if wide else update
    y = y / torch.linalg.vector_norm(y, dim=(-2, -1), keepdim=True).clamp(min=EPS)
    eye = torch.eye(y.shape[-1], dtype=torch.float64, device=y.device)
    for _ in range(STEPS):
        gram = y.transpose(-2, -1).contiguous().matmul(y)
        y = y.matmul(a * eye + gram.matmul(b * eye + c * gram))
    return y.transpose(-2, -1) if wide else y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return [_exact_orthogonal(m.double()) for m in state["matrices"]]
    out = {"updates": [], "momenta": [], "params": [], "masters": []}
    for k, (g, m) in enumerate(zip(state["grads"], state["momenta"])):
        grad = g.double() / state["scale"]
        buf = MOMENTUM * m.double() + (1.0 - MOMENTUM) * grad
        update = (1.0 - MOMENTUM) * grad + MOMENTUM * buf if case["nesterov"] else buf
        out["momenta"].append(buf)
        out["updates"].append(update)
        if case["op"] == "step":
            p = (state["masters"][k] if state["masters"] else state["params"][k]).detach().double()
            factor = LR * 0.2 * math.sqrt(max(p.shape[-2:]))
            p = p - LR * WEIGHT_DECAY * p - factor * _exact_orthogonal(update)
            out["params"].append(p)
            out["masters"].append(p)
    if case["op"] == "momentum":
        return {"updates": out["updates"], "momenta": out["momenta"], "norms": torch.stack([u.square().sum().sqrt() for u in out["updates"]]),
                "found_inf": None}
    return {"params": out["params"], "masters": out["masters"] if state["masters"] else None, "momenta": out["momenta"]}
