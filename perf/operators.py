"""Cases for three operators of a language model's training step on the `ocl` device, with their plain forms:

* the softmax cross entropy of a linear layer over a large vocabulary, with its gradients
  (pytorch_vulkan_b200.functional.linear_cross_entropy);
* the AdamW step over many tensors, with states in 32 bits and in 8 bits (pytorch_vulkan_b200.optim.AdamW);
* the learned relative position bias by buckets of the distance, with its gradient
  (pytorch_vulkan_b200.functional.relative_position_bias).

Where `own` is false the operators are computed from elementary torch operations on the CUDA device; where it is true by the
framework, whose tensors live on its own device, `ocl`: the same values, moved there once by prepare().
"""
import ctypes
import math
import os

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_BLOCK = 256  # elements of one scale of the 8-bit states


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the classifier of the default ResNet-50 workload: 64 images, 2048 features, 1000 classes, exact fp32
        {"name": "loss_classes_fp32", "op": "loss", "N": 64, "D": 2048, "V": 1000, "dtype": "fp32", "bias": True, "train": True, "ignored": 0.0, "smooth": 0.0},
        # scoring one token while serving: only the loss, the smallest call
        {"name": "loss_token_fp16", "op": "loss", "N": 1, "D": 2048, "V": 32768, "dtype": "fp16", "bias": False, "train": False, "ignored": 0.0, "smooth": 0.0},
        # an ordinary fine-tuning step: odd sizes, prompt tokens that are not scored, smoothed labels
        {"name": "loss_odd_bf16", "op": "loss", "N": 4095, "D": 1000, "V": 49999, "dtype": "bf16", "bias": False, "train": True, "ignored": 0.3, "smooth": 0.1},
        # a small language model in fp32
        {"name": "loss_fp32", "op": "loss", "N": 2048, "D": 768, "V": 32768, "dtype": "fp32", "bias": False, "train": True, "ignored": 0.05, "smooth": 0.0},
        # a large language model's last layer over a batch of 8192 tokens
        {"name": "loss_large_bf16", "op": "loss", "N": 8192, "D": 4096, "V": 131072, "dtype": "bf16", "bias": False, "train": True, "ignored": 0.05, "smooth": 0.0},
        # a small network of a few dozen tensors: launches count
        {"name": "adamw_small_fp32", "op": "adamw", "layers": 2, "width": 64, "head": 10, "dtype": "fp32", "bits": 32, "step": 3},
        # a ViT-B sized network in fp32
        {"name": "adamw_vit_fp32", "op": "adamw", "layers": 16, "width": 640, "head": 1000, "dtype": "fp32", "bits": 32, "step": 1000},
        # 8-bit states: a small network of odd tensors, and a 350M parameter language model in bf16
        {"name": "adamw8_small_fp32", "op": "adamw", "layers": 3, "width": 190, "head": 1001, "dtype": "fp32", "bits": 8, "step": 10},
        {"name": "adamw8_lm_bf16", "op": "adamw", "layers": 24, "width": 1024, "head": 50001, "dtype": "bf16", "bits": 8, "step": 2000},
        # one new token against a cache, causal
        {"name": "bias_token_fp16", "op": "bias", "H": 32, "Lq": 1, "Lk": 4099, "buckets": 32, "far": 128, "both": False, "dtype": "fp16", "train": False},
        # ViT-B/16's 197 tokens and 12 heads, with the gradient
        {"name": "bias_vit_fp32", "op": "bias", "H": 12, "Lq": 197, "Lk": 197, "buckets": 32, "far": 128, "both": True, "dtype": "fp32", "train": True},
        # a long sequence
        {"name": "bias_long_bf16", "op": "bias", "H": 16, "Lq": 4096, "Lk": 4096, "buckets": 64, "far": 1024, "both": True, "dtype": "bf16", "train": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["loss", "loss", "adamw", "bias"])
    if op == "loss":
        dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        most = 1.0e12 if dtype != "fp32" else 1.0e11  # N V D
        while True:
            N, D, V = _log_int(rng, 1, 8192), _log_int(rng, 32, 4096), _log_int(rng, 10, 131072)
            if rng.random() < 0.7:
                D = max(8, D // 8 * 8)
            if N * D * V <= most:
                break
        return {"op": "loss", "N": N, "D": D, "V": V, "dtype": dtype, "bias": rng.random() < 0.3, "train": rng.random() < 0.75,
                "ignored": rng.choice([0.0, 0.1, 0.5]), "smooth": rng.choice([0.0, 0.0, 0.1])}
    if op == "adamw":
        width = _log_int(rng, 16, 800)
        layers = max(1, min(_log_int(rng, 1, 24), int(1.2e8 / (12 * width * width))))
        bits = rng.choice([8, 32])
        dtype = rng.choice(["fp32", "bf16", "fp16"]) if bits == 8 else "fp32"
        return {"op": "adamw", "layers": layers, "width": width, "head": _log_int(rng, 2, 20000), "dtype": dtype, "bits": bits, "step": _log_int(rng, 1, 10000)}
    while True:
        H, Lq, Lk = rng.randint(1, 32), rng.choice([1, _log_int(rng, 2, 4096), _log_int(rng, 2, 4096)]), _log_int(rng, 2, 8192)
        if H * Lq * Lk <= 2.6e8:
            break
    buckets = 4 * rng.randint(2, 32)
    return {"op": "bias", "H": H, "Lq": min(Lq, Lk), "Lk": Lk, "buckets": buckets, "far": buckets * rng.choice([1, 2, 4, 16]), "both": rng.random() < 0.5,
            "dtype": rng.choice(["fp32", "bf16", "fp16"]), "train": rng.random() < 0.7}


def _shapes(case):
    """The tensors of a transformer of this size, as a model's parameters() gives them."""
    D, L = case["width"], case["layers"]
    layer = [(D,), (D,), (D, D), (D, D), (D, D), (D, D), (D,), (D,), (D,), (4 * D, D), (4 * D,), (D, 4 * D), (D,)]
    return layer * L + [(D,), (case["head"], D), (case["head"],)]


def work(case):
    if case["op"] == "loss":
        N, D, V, s = case["N"], case["D"], case["V"], _SIZE[case["dtype"]]
        tensors = (N * D + V * D + (V if case["bias"] else 0)) * s
        if case["train"]:
            return {"bytes": 2 * tensors + 8 * N + 4, "flops": 6 * N * V * D}
        return {"bytes": tensors + 12 * N, "flops": 2 * N * V * D}
    if case["op"] == "adamw":
        n, s = sum(math.prod(x) for x in _shapes(case)), _SIZE[case["dtype"]]
        if case["bits"] == 32:
            return {"bytes": n * (3 * s + 16), "flops": 12 * n}
        # codes and scales read and written, and the moments that they stand for written as fp32
        return {"bytes": n * (3 * s + 4 + 16 / _BLOCK + 8), "flops": 20 * n}
    cells = case["H"] * case["Lq"] * case["Lk"]
    return {"bytes": cells * _SIZE[case["dtype"]] * (2 if case["train"] else 1), "flops": cells * (1 if case["train"] else 0)}


# -------------------------------------------------------------------------------------------------------------- prepare
def _hand(t):
    """`t` on the device of the program that calls: CUDA's for the plain form, the framework's for its own."""
    if not own or t is None:
        return t
    import pytorch_vulkan_b200 as pkg

    lib = ctypes.CDLL(os.path.join(os.path.dirname(pkg.__file__), "lib", "libpvb2.so"))
    lib.pvb2_memcpy_async.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]
    t = t.contiguous()
    out = torch.empty(t.shape, dtype=t.dtype, device="ocl")
    torch.cuda.synchronize()
    if t.numel() and lib.pvb2_memcpy_async(out.data_ptr(), t.data_ptr(), t.numel() * t.element_size(), 2, None):
        raise RuntimeError("copy to the ocl device failed")
    torch.cuda.synchronize()
    return out


def _loss_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, D, V, dt = case["N"], case["D"], case["V"], _DTYPES[case["dtype"]]
    w = torch.randn(V, D, device="cuda", generator=g).mul_(1.0 / math.sqrt(D)).to(dt)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    # normalised hidden states, half of which already point at their token, as in a model that has learned something
    sure = torch.rand(N, 1, device="cuda", generator=g).sub_(0.5).clamp_(min=0).mul_(16.0)
    x = (torch.randn(N, D, device="cuda", generator=g) + sure * w[t].float()).to(dt)
    b = torch.randn(V, device="cuda", generator=g).mul_(0.1).to(dt) if case["bias"] else None
    t[torch.rand(N, device="cuda", generator=g) < case["ignored"]] = -100
    return x, w, b, t


def _adamw_inputs(case, seed):
    """Flat buffers of the parameters, gradients and moments, each tensor at a multiple of the block, with zeros between."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, places, at = _DTYPES[case["dtype"]], [], 0
    for s in _shapes(case):
        places.append((at, math.prod(s), s))
        at += -(-math.prod(s) // _BLOCK) * _BLOCK
    ends = torch.tensor([[a, n] for a, n, _ in places], device="cuda")
    marks = torch.zeros(at + 1, dtype=torch.int32, device="cuda")
    marks[ends[:, 0]] += 1
    marks.index_add_(0, ends.sum(1), -torch.ones(len(places), dtype=torch.int32, device="cuda"))
    inside = marks.cumsum(0, dtype=torch.int32)[:at] > 0
    # the size of the gradients differs from block to block, as it does from row to row of a weight
    size = torch.exp(torch.randn(at // _BLOCK, 1, device="cuda", generator=g)).mul_(1e-3).expand(-1, _BLOCK).reshape(-1)
    rand = lambda: torch.randn(at, device="cuda", generator=g).mul_(inside)  # noqa: E731
    p, grad = rand().mul_(0.02).to(dt), rand().mul_(size).to(dt)
    m, u = rand().mul_(size).mul_(0.3), rand().mul_(0.2).exp_().mul_(size).mul_(inside)
    return places, p, grad, m, u


def prepare(case, seed):
    if case["op"] == "loss":
        x, w, b, t = (_hand(v) for v in _loss_inputs(case, seed))
        if own:
            torch.ocl.set_math_mode(1)  # fp32 products, as the plain form's
            for v in (x, w, b):
                if v is not None and case["train"]:
                    v.requires_grad_()
        return {"case": case, "x": x, "w": w, "b": b, "t": t}
    if case["op"] == "adamw":
        places, p, grad, m, u = _adamw_inputs(case, seed)
        state = {"case": case, "step": case["step"]}
        if case["bits"] == 8:
            cm, sm = _encode(m, 3)
            cu, su = _encode(u, 4)
            held = {"p": p, "g": grad, "cm": cm, "sm": sm, "cu": cu, "su": su}
        else:
            held = {"p": p, "g": grad, "m": m, "v": u.square_()}
        state.update({k: _hand(v) for k, v in held.items()})
        if own:
            state.update(_optimizer(state, places))
        return state
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    table = torch.randn(case["buckets"], case["H"], device="cuda", generator=g).to(dt)
    grad = torch.randn(1, case["H"], case["Lq"], case["Lk"], device="cuda", generator=g).mul_(1e-2).to(dt) if case["train"] else None
    table, grad = _hand(table), _hand(grad)
    if own and case["train"]:
        table.requires_grad_()
    return {"case": case, "table": table, "grad": grad}


def _optimizer(state, places):
    """The optimizer that a program resumes from a checkpoint: its parameters, gradients and state are views of the flat buffers."""
    view = lambda t, a, n, s: t[a:a + n].view(s)  # noqa: E731
    params = [view(state["p"], *q) for q in places]
    for p, q in zip(params, places):
        p.grad = view(state["g"], *q)
    step = lambda: torch.full((), float(state["step"] - 1), device="ocl")  # noqa: E731
    from pytorch_vulkan_b200.optim import AdamW

    opt = AdamW(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=state["case"]["bits"])
    if state["case"]["bits"] == 32:
        for p, q in zip(params, places):
            opt.state[p] = {"step": step(), "exp_avg": view(state["m"], *q), "exp_avg_sq": view(state["v"], *q)}
        return {"opt": opt}
    m, v = torch.zeros(state["p"].shape, device="ocl"), torch.zeros(state["p"].shape, device="ocl")
    for p, (a, n, s) in zip(params, places):
        blocks = slice(a // _BLOCK, a // _BLOCK + -(-n // _BLOCK))
        opt.state[p] = {"step": step(), "exp_avg_code": state["cm"][a:a + n], "exp_avg_scale": state["sm"][blocks],
                        "exp_avg_rms_code": state["cu"][a:a + n], "exp_avg_rms_scale": state["su"][blocks]}
    return {"opt": opt, "m": m, "v": v, "ms": [view(m, *q) for q in places], "vs": [view(v, *q) for q in places]}


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if own:
        return {"loss": _own_loss, "adamw": _own_adamw, "bias": _own_bias}[case["op"]](case, state)
    return {"loss": _plain_loss, "adamw": _plain_adamw, "bias": _plain_bias}[case["op"]](case, state)


def _own_loss(case, s):
    from pytorch_vulkan_b200.functional import linear_cross_entropy

    loss = linear_cross_entropy(s["x"], s["w"], s["t"], s["b"], reduction="mean" if case["train"] else "none", label_smoothing=case["smooth"])
    if not case["train"]:
        return [loss]
    grads = torch.autograd.grad(loss, [v for v in (s["x"], s["w"], s["b"]) if v is not None])
    return [loss.detach(), *grads]


def _own_adamw(case, s):
    s["opt"].step()
    if case["bits"] == 8:
        s["opt"].write_state_values(s["ms"], s["vs"])
    return [s["p"], s["m"], s["v"]]


def _own_bias(case, s):
    from pytorch_vulkan_b200.functional import relative_position_bias

    bias = relative_position_bias(s["table"], case["Lq"], case["Lk"], bidirectional=case["both"], max_distance=case["far"], q_offset=case["Lk"] - case["Lq"])
    if not case["train"]:
        return [bias]
    return [bias.detach(), *torch.autograd.grad(bias, [s["table"]], [s["grad"]])]


def _plain_loss(case, s):
    x, w, t, V = s["x"].float(), s["w"].float(), s["t"], case["V"]
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"].float()
    counts = t != -100
    at = torch.where(counts, t, 0)[:, None]
    e = z.amax(1, keepdim=True)
    smooth = z.mean(1) if case["smooth"] else 0.0
    zt = z.gather(1, at)[:, 0]
    z -= e
    z.exp_()
    total = z.sum(1, keepdim=True)
    lse = (e + total.log())[:, 0]
    loss = torch.where(counts, lse - (1 - case["smooth"]) * zt - case["smooth"] * smooth, 0.0)
    if not case["train"]:
        return [loss]
    n = counts.sum().float()
    z /= total
    if case["smooth"]:
        z -= case["smooth"] / V
    z.scatter_add_(1, at, torch.full_like(at, -(1 - case["smooth"]), dtype=torch.float32))
    z *= torch.where(counts, 1.0 / n, 0.0)[:, None]
    grads = [z @ w, z.t() @ x] + ([z.sum(0)] if s["b"] is not None else [])
    return [loss.sum() / n] + [g.to(s["x"].dtype) for g in grads]


def _encode(y, mantissa):
    """Codes and scales of the 8-bit states: in blocks of 256 elements y = s c, c a number with a 4-bit exponent (bias 15) and
    `mantissa` bits of mantissa, s such that the block's largest |y| takes the largest code. Signed with 3 bits of mantissa;
    with 4 there is no sign, and what is positive never gets code 0."""
    y = y.view(-1, _BLOCK)
    top = 2.0 - 2.0 ** -mantissa
    s = y.abs().amax(1, keepdim=True) * torch.tensor(1.0 / top, device=y.device)
    r = torch.where(s > 0, y / s, 0.0)
    bits = (r.abs() * 2.0 ** -112).view(torch.int32)
    drop = 23 - mantissa
    code = torch.clamp((bits + (2 ** (drop - 1) - 1) + ((bits >> drop) & 1)) >> drop, max=16 * 2 ** mantissa - 1)
    code = torch.where(r < 0, code | 128, code) if mantissa == 3 else torch.where((y > 0) & (code == 0), 1, code)
    return code.to(torch.uint8).view(-1), s.view(-1)


def _decode(code, s, mantissa):
    code = code.to(torch.int32).view(-1, _BLOCK)
    top = code & 127 if mantissa == 3 else code
    y = (top << (23 - mantissa)).view(torch.float32) * 2.0 ** 112 * s[:, None]
    return (torch.where(code > 127, -y, y) if mantissa == 3 else y).view(-1)


def _plain_adamw(case, s):
    lr, b1, b2, eps, decay = 1e-3, 0.9, 0.999, 1e-8, 0.01
    g = s["g"].float()
    if case["bits"] == 8:
        m = _decode(s["cm"], s["sm"], 3)
        v = _decode(s["cu"], s["su"], 4).square_()
    else:
        m, v = s["m"], s["v"]
    # each product and sum rounds by itself: the codes go by these values
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_(g.square().mul_(1 - b2))
    u = v.sqrt()
    p = s["p"].float() * (1 - lr * decay)
    denominator = u * (1 / math.sqrt(1 - b2 ** s["step"])) + eps
    p -= (m / denominator) * (lr / (1 - b1 ** s["step"]))
    s["p"].copy_(p)
    s["step"] += 1
    if case["bits"] == 32:
        return [s["p"], m, v]
    s["cm"], s["sm"] = _encode(m, 3)
    s["cu"], s["su"] = _encode(u, 4)
    return [s["p"], _decode(s["cm"], s["sm"], 3), _decode(s["cu"], s["su"], 4).square_()]


def _plain_bias(case, s):
    Lq, Lk, H = case["Lq"], case["Lk"], case["H"]
    # row 0 of the table for the distance -(Lq - 1 + offset), and so on: a distance is a diagonal of the scores
    rel = torch.arange(Lq + Lk - 1, device="cuda") - (Lq - 1 + Lk - Lq)
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    far = rel.abs() if case["both"] else (-rel).clamp(min=0)
    exact_to = n // 2
    # in 64 bits, with a slack far below the step from one distance to the next, so that a distance on a border is not below it
    steps = torch.log(far.clamp(min=1).double() / exact_to) / math.log(case["far"] / exact_to) * (n - exact_to)
    bucket = torch.where(far < exact_to, far, (exact_to + torch.floor(steps + 1e-9).long()).clamp(max=n - 1))
    if case["both"]:
        bucket = bucket + n * (rel > 0)
    by_distance = s["table"].float()[bucket]
    cell = torch.arange(Lk, device="cuda")[None, :] - torch.arange(Lq, device="cuda")[:, None] + (Lq - 1)
    bias = by_distance.t()[:, cell].to(s["table"].dtype)[None]
    if not case["train"]:
        return [bias]
    # rows upside down and one element longer each than the view that is summed: diagonals become columns
    g = torch.nn.functional.pad(s["grad"][0].float().flip(1), (0, Lq)).reshape(H, -1)
    g = g[:, : Lq * (Lq + Lk - 1)].view(H, Lq, Lq + Lk - 1).sum(1, dtype=torch.float64)
    table = torch.zeros(case["buckets"], H, dtype=torch.float64, device="cuda").index_add_(0, bucket, g.t().contiguous())
    return [bias, table.to(s["table"].dtype)]


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "loss":
        x, w, b, t = _loss_inputs(case, seed)
        w64, V, e = w.double(), case["V"], case["smooth"]
        dx, dw = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(w64)
        db, losses, scored = torch.zeros(V, dtype=torch.float64, device="cuda"), [], int((t >= 0).sum())
        for a in range(0, case["N"], 1024):
            xa, ta = x[a:a + 1024].double(), t[a:a + 1024]
            z = torch.addmm(b.double(), xa, w64.t()) if b is not None else xa @ w64.t()
            logp = z - torch.logsumexp(z, 1, keepdim=True)
            goal = torch.full_like(z, e / V)
            goal[torch.arange(len(ta), device="cuda"), ta.clamp(min=0)] += 1 - e
            losses.append(-(goal * logp).nan_to_num_(0.0).sum(1) * (ta >= 0))
            if case["train"]:
                d = (logp.exp() - goal) * ((ta >= 0).double() / max(scored, 1))[:, None]
                dx[a:a + 1024] = d @ w64
                dw += d.t() @ xa
                db += d.sum(0)
        losses = torch.cat(losses)
        if not case["train"]:
            return [losses]
        return [losses.sum() / scored, dx, dw] + ([db] if b is not None else [])
    if case["op"] == "adamw":
        _, p, grad, m, u = _adamw_inputs(case, seed)
        lr, b1, b2, k, v = 1e-3, 0.9, 0.999, case["step"], None
        if case["bits"] == 8:
            # the step begins from what the codes hold
            m, u = (_decode(*_encode(y, bits), bits) for y, bits in ((m, 3), (u, 4)))
        v = u.square().double() if case["bits"] == 8 else u.square_().double()
        m = b1 * m.double() + (1 - b1) * grad.double()
        v = b2 * v + (1 - b2) * grad.double() ** 2
        hat = m / (1 - b1 ** k) / (torch.sqrt(v / (1 - b2 ** k)) + 1e-8)
        p = p.double() - lr * 0.01 * p.double() - lr * hat
        # a moment that lies on the border of two codes takes the one or the other by its last bit in 32 bits: there is no
        # value in 64 bits that it ought to be
        return [p, m, v] if case["bits"] == 32 else [p, None, None]
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randn(case["buckets"], case["H"], device="cuda", generator=g).to(_DTYPES[case["dtype"]]).double()
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    first = n // 2

    def bucket(rel):
        d = abs(rel) if case["both"] else max(-rel, 0)
        at = d
        if d >= first:
            # floor(log(d / first) / log(far / first) * (n - first)) by whole numbers
            at = math.floor((math.log(d) - math.log(first)) / (math.log(case["far"]) - math.log(first)) * (n - first))
            while at + 1 <= n - first and (d ** (n - first)) * first ** (at + 1) >= case["far"] ** (at + 1) * first ** (n - first):
                at += 1
            while at > 0 and (d ** (n - first)) * first ** at < case["far"] ** at * first ** (n - first):
                at -= 1
            at = min(first + at, n - 1)
        return at + (n if case["both"] and rel > 0 else 0)

    Lq, Lk = case["Lq"], case["Lk"]
    of = [bucket(rel) for rel in range(-(Lk - 1), Lq)]
    which = torch.tensor(of, device="cuda")
    rows = torch.stack([which[Lq - 1 - i:Lq - 1 - i + Lk] for i in range(Lq)])
    bias = torch.empty(1, case["H"], Lq, Lk, dtype=torch.float64, device="cuda")
    for h in range(case["H"]):
        bias[0, h] = table[:, h][rows]
    if not case["train"]:
        return [bias]
    grad = torch.randn(1, case["H"], Lq, Lk, device="cuda", generator=g).mul_(1e-2).to(_DTYPES[case["dtype"]])[0]
    sums = torch.zeros(case["buckets"], case["H"], dtype=torch.float64, device="cuda")
    for k in sorted(set(of)):
        lo, hi = of.index(k), len(of) - 1 - of[::-1].index(k)
        # the diagonals of one bucket are neighbours: between two shifted triangles
        part = torch.triu(torch.tril(grad, hi - (Lq - 1)), lo - (Lq - 1))
        sums[k] = part.sum((1, 2), dtype=torch.float64)
    return [bias, sums]
