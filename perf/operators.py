"""What the distillation and 8-bit operators are measured on: cases, inputs, a plain form of each operator, and its
definition in 64 bits.

``own`` selects what ``run`` calls: False, the plain forms below (elementary torch operations); True, the framework's
operators (``steptronoss_b200.ops``).  Shapes are those of the Qwen3 configurations in ``playground/`` (8B: hidden 4096,
qkv 6144, gate + up 24576; 1.7B: hidden 2048, gate + up 12288; vocabulary 151936) and generic odd ones.
"""
import math

import torch

own = False

VOCAB = 151936
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a teacher's top 64 on the eight answer tokens of a short sequence: latency counts
        dict(name="distill_step_8_tokens", op="distill_grad", T=8, V=VOCAB, K=64, dtype="bf16", temperature=1.0),
        # a packed training sequence of 4096 tokens, logits already computed, loss and gradient in one pass
        dict(name="distill_pack_4096", op="distill_grad", T=4096, V=VOCAB, K=64, dtype="bf16", temperature=1.0),
        # fp32 logits of an odd vocabulary through autograd, softened, with a gradient that differs from token to token
        dict(name="distill_autograd_odd", op="distill", T=777, V=50257, K=20, dtype="fp32", temperature=2.0),
        # the training step of a student's LM head: hidden states in, loss, dL/dh and dL/dW out
        dict(name="distill_linear_4096", op="distill_linear", T=4096, V=VOCAB, K=64, H=2048, temperature=1.0),
        # one token through an 8-bit qkv projection
        dict(name="int8_gemm_1", op="int8_gemm", M=1, N=6144, K=4096),
        # a decode batch through the gate + up projection
        dict(name="int8_gemm_48", op="int8_gemm", M=48, N=24576, K=4096),
        # a packed sequence of 8192 tokens through the gate + up projection of a frozen model
        dict(name="int8_gemm_8192", op="int8_gemm", M=8192, N=24576, K=4096),
        # bf16 tokens quantised on the fly, nothing a multiple of anything
        dict(name="int8_linear_ragged", op="int8_linear", M=1333, N=5001, K=2050),
        # residual add, norm and e4m3 blocks for four tokens of a decode step
        dict(name="norm_e4m3_4", op="norm_e4m3", T=4, H=4096),
        # the same for a pack of 16384 tokens
        dict(name="norm_e4m3_16384", op="norm_e4m3", T=16384, H=4096),
        # the start of a frozen model's FFN at decode: residual add, norm to int8, gate + up product
        dict(name="norm_int8_linear_16", op="norm_int8_linear", T=16, H=2048, N=12288),
        # the same with a hidden size that no vector width divides
        dict(name="norm_int8_linear_odd", op="norm_int8_linear", T=515, H=1990, N=2051),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["distill_grad", "distill", "distill_linear", "int8_gemm", "int8_linear", "norm_e4m3",
                     "norm_int8_linear"])
    if op.startswith("distill"):
        V = _log(rng, 1000, VOCAB)
        case = dict(op=op, T=_log(rng, 1, 4096), V=V, K=_log(rng, 1, 256), temperature=rng.choice([1.0, 0.5, 2.0, 4.0]))
        if op == "distill_linear":
            case["H"] = 64 * rng.randint(2, 32)
            case["V"] = (V + 7) // 8 * 8
        else:
            case["dtype"] = rng.choice(["bf16", "bf16", "fp32"])
            if case["dtype"] == "fp32":
                case["T"] = min(case["T"], 2048)
        return case
    if op.startswith("int8"):
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 200, 24576), _log(rng, 100, 12288)
            if M * N * K <= 8192 * 24576 * 4096:
                return dict(op=op, M=M, N=N, K=K)
    if op == "norm_e4m3":
        return dict(op=op, T=_log(rng, 1, 16384), H=128 * rng.randint(4, 64) if rng.random() < 0.6 else 4096)
    return dict(op=op, T=_log(rng, 1, 4096), H=_log(rng, 200, 8192), N=_log(rng, 200, 12288))


# ---------------------------------------------------------------------------------------------------------- inputs
def _pitched(q):
    """8-bit rows whose pitch is a multiple of 16 bytes, as a program lays its weights out once."""
    rows, K = q.shape
    buf = torch.zeros((rows, (K + 15) // 16 * 16), dtype=q.dtype, device=q.device)
    buf[:, :K] = q
    return buf[:, :K]


def _int8_weight(g, N, K):
    w = torch.randn(N, K, device="cuda", generator=g) * 0.02
    scale = w.abs().amax(1) / 127
    return _pitched((w / scale[:, None]).round().to(torch.int8)), scale


def _tokens(g, rows, width):
    """Hidden states: a few channels much larger than the others, as transformers have them."""
    x = torch.randn(rows, width, device="cuda", generator=g)
    channel = torch.ones(width, device="cuda")
    channel[torch.randint(0, width, (max(1, width // 256),), device="cuda", generator=g)] = 8.0
    return (x * channel).to(torch.bfloat16)


def _teacher(g, scores, K):
    """Top-K ids and log-probabilities of a teacher that mostly agrees with `scores`; shorter rows end in -inf, some
    rows (padding, prompt) have no entry at all."""
    T, V = scores.shape
    t = torch.randn(T, V, device="cuda", generator=g)
    t.add_(scores.float(), alpha=0.9)
    logp, ids = t.topk(K, dim=1)
    logp = logp - t.logsumexp(1, keepdim=True)
    keep = torch.randint(1, K + 1, (T, 1), device="cuda", generator=g)
    keep = torch.where(torch.rand(T, 1, device="cuda", generator=g) < 0.75, K, keep)
    keep[torch.rand(T, 1, device="cuda", generator=g) < 0.02] = 0
    keep[0] = K
    gone = torch.arange(K, device="cuda")[None] >= keep
    return ids.masked_fill(gone, 0), logp.masked_fill(gone, -math.inf)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, state = case["op"], {"op": case["op"]}
    if op in ("distill_grad", "distill"):
        T, V = case["T"], case["V"]
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        logits = torch.randn(T, V, device="cuda", generator=g, dtype=dtype).mul_(2.5)
        state["ids"], state["teacher"] = _teacher(g, logits, case["K"])
        state["logits"] = logits.requires_grad_(op == "distill")
        state["weights"] = torch.rand(T, device="cuda", generator=g) / T
        state["temperature"] = case["temperature"]
    elif op == "distill_linear":
        T, V, H = case["T"], case["V"], case["H"]
        h = torch.randn(T, H, device="cuda", generator=g, dtype=torch.bfloat16)
        w = torch.randn(V, H, device="cuda", generator=g, dtype=torch.bfloat16).mul_(2.5 / math.sqrt(H))
        state["ids"], state["teacher"] = _teacher(g, h @ w.t(), case["K"])
        state["h"], state["w"] = h.requires_grad_(True), w.requires_grad_(True)
        state["weights"] = torch.rand(T, device="cuda", generator=g) / T
        state["temperature"] = case["temperature"]
    elif op == "int8_gemm":
        x = torch.randn(case["M"], case["K"], device="cuda", generator=g)
        state["sx"] = x.abs().amax(1) / 127
        state["xq"] = _pitched((x / state["sx"][:, None]).round().to(torch.int8))
        state["wq"], state["sw"] = _int8_weight(g, case["N"], case["K"])
    elif op == "int8_linear":
        state["x"] = _tokens(g, case["M"], case["K"])
        state["wq"], state["sw"] = _int8_weight(g, case["N"], case["K"])
    else:
        state["x"], state["delta"] = _tokens(g, case["T"], case["H"]), _tokens(g, case["T"], case["H"])
        state["gain"] = (1 + 0.1 * torch.randn(case["H"], device="cuda", generator=g)).to(torch.bfloat16)
        if op == "norm_int8_linear":
            state["wq"], state["sw"] = _int8_weight(g, case["N"], case["H"])
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_distill(s, state):
    """Loss per token and its gradient with respect to the fp32 logits `s`, for a weight of one."""
    ids, temperature = state["ids"], state["temperature"]
    s = s / temperature
    m = s.amax(1, keepdim=True)
    e = (s - m).exp()
    total = e.sum(1, keepdim=True)
    t = state["teacher"].float() / temperature
    tm = t.amax(1, keepdim=True)
    some = tm > -math.inf
    te = torch.where(some, (t - tm).exp(), 0.0)
    tsum = torch.where(some, te.sum(1, keepdim=True), 1.0)
    q = te / tsum
    logq = t - tm - tsum.log()
    logp = s.gather(1, ids) - m - total.log()
    loss = torch.where(q > 0, q * (logq - logp), 0.0).sum(1)
    grad = torch.where(some, e / total, 0.0).scatter_add_(1, ids, -q) / temperature
    return loss, grad


def _plain_quantised(y):
    scale = y.abs().amax(1) / 127
    scale = torch.where(scale > 0, scale, 1.0)
    return (y / scale[:, None]).round(), scale


def _plain_product(xq, sx, wq, sw):
    """The sums pass 2^24, so they are taken in 64 bits; the result is bf16."""
    dot = xq.double() @ wq.double().t()
    return (dot.float() * sx[:, None] * sw[None]).to(torch.bfloat16)


def _plain_norm(state):
    s = (state["x"].float() + state["delta"].float()).to(torch.bfloat16)
    f = s.float()
    return s, f * torch.rsqrt(f.square().mean(1, keepdim=True) + EPS) * state["gain"].float()


def _plain(state):
    op = state["op"]
    if op in ("distill_grad", "distill"):
        logits = state["logits"].detach()
        loss, grad = _plain_distill(logits.float(), state)
        return {"loss": loss, "grad": (grad * state["weights"][:, None]).to(logits.dtype)}
    if op == "distill_linear":
        h, w = state["h"].detach().float(), state["w"].detach().float()
        loss, grad = _plain_distill(h @ w.t(), state)
        grad = grad * state["weights"][:, None]
        return {"total": (loss * state["weights"]).sum(), "loss": loss, "dh": (grad @ w).to(torch.bfloat16),
                "dw": (grad.t() @ h).to(torch.bfloat16)}
    if op == "int8_gemm":
        return _plain_product(state["xq"], state["sx"], state["wq"], state["sw"])
    if op == "int8_linear":
        q, scale = _plain_quantised(state["x"].float())
        return _plain_product(q, scale, state["wq"], state["sw"])
    s, y = _plain_norm(state)
    if op == "norm_e4m3":
        blocks = y.view(y.shape[0], -1, 128)
        scale = blocks.abs().amax(2) / 448
        scale = torch.where(scale > 0, scale, 1.0)
        q = (blocks / scale[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        return {"s": s, "q": q.view(y.shape), "scale": scale}
    q, scale = _plain_quantised(y)
    return {"s": s, "y": _plain_product(q, scale, state["wq"], state["sw"])}


def _own(state):
    from steptronoss_b200 import ops

    op = state["op"]
    if op == "distill_grad":
        loss, grad = ops.topk_distillation_loss_and_grad(state["logits"], state["ids"], state["teacher"],
                                                         state["weights"], state["temperature"])
        return {"loss": loss, "grad": grad}
    if op == "distill":
        loss = ops.topk_distillation(state["logits"], state["ids"], state["teacher"], state["temperature"])
        (grad,) = torch.autograd.grad(loss, state["logits"], state["weights"])
        return {"loss": loss.detach(), "grad": grad}
    if op == "distill_linear":
        total, loss = ops.fused_linear_topk_distillation(state["h"], state["w"], state["ids"], state["teacher"],
                                                         state["weights"], state["temperature"])
        dh, dw = torch.autograd.grad(total, [state["h"], state["w"]])
        return {"total": total.detach(), "loss": loss, "dh": dh, "dw": dw}
    if op == "int8_gemm":
        return ops.gemm_int8(state["xq"], state["sx"], state["wq"], state["sw"])
    if op == "int8_linear":
        return ops.linear_int8(state["x"], state["wq"], state["sw"])
    if op == "norm_e4m3":
        s, q, scale = ops.add_rmsnorm_quant(state["x"], state["delta"], state["gain"], EPS, fmt="e4m3_1x128")
        return {"s": s, "q": q, "scale": scale}
    s, q, scale = ops.add_rmsnorm_quant(state["x"], state["delta"], state["gain"], EPS, fmt="int8")
    return {"s": s, "y": ops.gemm_int8(q, scale, state["wq"], state["sw"])}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------- sizes
def work(case):
    op = case["op"]
    if op.startswith("distill"):
        T, V = case["T"], case["V"]
        side = T * case["K"] * (8 + 4) + 4 * T + 4 * T      # teacher entries, weights, loss
        if op == "distill_linear":
            H = case["H"]
            return {"bytes": 2 * 2 * (T * H + V * H) + side, "flops": 6 * T * V * H}
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * size * T * V + side, "flops": 6 * T * V}
    if op.startswith("int8"):
        M, N, K = case["M"], case["N"], case["K"]
        tokens = M * K + 4 * M if op == "int8_gemm" else 2 * M * K
        return {"bytes": tokens + N * K + 4 * N + 2 * M * N, "flops": 2 * M * N * K}
    T, H = case["T"], case["H"]
    if op == "norm_e4m3":
        return {"bytes": 7 * T * H + 4 * T * (H // 128) + 2 * H, "flops": 8 * T * H}
    N = case["N"]
    return {"bytes": 6 * T * H + 2 * H + N * H + 4 * N + 2 * T * N, "flops": 2 * T * N * H + 8 * T * H}


# ---------------------------------------------------------------------------------------------------------- 64 bits
def _exact_distill(logits, state):
    """sum_j q_j log(q_j / p_j) with q = softmax of the teacher's entries and p = softmax of the logits, both at the
    temperature, and its derivative (p - q) / temperature, for `logits` in 64 bits."""
    tau = state["temperature"]
    logp = torch.log_softmax(logits / tau, dim=1)
    teacher = state["teacher"].double() / tau
    has = torch.isfinite(teacher).any(1)
    logq = torch.log_softmax(torch.where(has[:, None], teacher, 0.0), dim=1)
    q = torch.where(has[:, None], logq.exp(), 0.0)
    terms = q * (logq - torch.gather(logp, 1, state["ids"]))
    loss = torch.where(q > 0, terms, torch.zeros_like(terms)).sum(1)
    grad = logp.exp_().mul_(has[:, None])
    grad.scatter_add_(1, state["ids"], q.neg())
    return loss, grad.div_(tau).mul_(state["weights"].double()[:, None])


def _exact_int8(v):
    top = v.abs().max(dim=1).values
    scale = torch.where(top > 0, top / 127.0, torch.ones_like(top))
    return torch.round(v / scale.unsqueeze(1)), scale


def _exact_product(q, scale, state):
    w = state["wq"].double() * state["sw"].double().unsqueeze(1)
    return torch.matmul(q * scale.unsqueeze(1), w.transpose(0, 1))


def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    if op in ("distill_grad", "distill"):
        loss, grad = _exact_distill(state["logits"].detach().double(), state)
        return {"loss": loss, "grad": grad}
    if op == "distill_linear":
        h, w = state["h"].detach().double(), state["w"].detach().double()
        loss, grad = _exact_distill(torch.matmul(h, w.transpose(0, 1)), state)
        return {"total": torch.dot(loss, state["weights"].double()), "loss": loss, "dh": torch.matmul(grad, w),
                "dw": torch.matmul(grad.transpose(0, 1), h)}
    if op == "int8_gemm":
        return _exact_product(state["xq"].double(), state["sx"].double(), state)
    if op == "int8_linear":
        return _exact_product(*_exact_int8(state["x"].double()), state)
    # the norm is taken of the residual stream as it is stored, in bf16
    s = (state["x"].double() + state["delta"].double()).to(torch.bfloat16).double()
    y = s / torch.sqrt(s.pow(2).sum(1, keepdim=True) / case["H"] + EPS) * state["gain"].double()
    if op == "norm_int8_linear":
        return {"s": s, "y": _exact_product(*_exact_int8(y), state)}
    top = y.reshape(case["T"], case["H"] // 128, 128).abs().max(dim=2).values
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    q = (y / scale.repeat_interleave(128, dim=1)).to(torch.float8_e4m3fn)
    return {"s": s, "q": q.double(), "scale": scale}
