"""Cases for four operators of a language model on the `ocl` device, with their plain forms:

* the root-mean-square norm with the residual's addition, its gradients, and its output in 8 bits with scales
  (pytorch_vulkan_b200.functional.rms_norm, rms_norm_8bit);
* the linear layer in 8-bit floating point with a scale for each block of 128 (pytorch_vulkan_b200.functional.linear_8bit);
* log probabilities of given tokens with entropy, gradient and top alternatives
  (pytorch_vulkan_b200.functional.token_log_probs);
* the gradients' global norm over many tensors, and clipping to it (pytorch_vulkan_b200.optim.clip_grad_norm_).

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
_GROUP = 128  # elements of one scale
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of a language model between two layers: the smallest call
        {"name": "norm_token_bf16", "op": "norm", "rows": 1, "D": 4096, "dtype": "bf16", "residual": True, "mode": "serve"},
        # ViT-B/16's 197 tokens of 64 images, with gradients
        {"name": "norm_vit_fp32", "op": "norm", "rows": 12608, "D": 768, "dtype": "fp32", "residual": False, "mode": "train"},
        # a training step over 8192 tokens, with the residual stream
        {"name": "norm_train_bf16", "op": "norm", "rows": 8192, "D": 4096, "dtype": "bf16", "residual": True, "mode": "train"},
        # a prompt on its way into a layer in 8 bits; the last group of a row is short
        {"name": "norm8_odd_fp16", "op": "norm", "rows": 2047, "D": 5000, "dtype": "fp16", "residual": True, "mode": "8bit"},
        # a linear layer on one new token
        {"name": "linear8_token_bf16", "op": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16", "bias": False},
        # a short ragged batch, a last block of 104 inputs, with a bias
        {"name": "linear8_odd_fp16", "op": "linear", "M": 300, "N": 5001, "K": 1000, "dtype": "fp16", "bias": True},
        # a large layer over 8192 tokens
        {"name": "linear8_large_bf16", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16", "bias": False},
        # the answer's next token with its 20 best alternatives
        {"name": "logp_token_fp32", "op": "logp", "N": 1, "V": 32768, "dtype": "fp32", "top": 20, "train": False, "ignored": 0.0},
        # scoring a batch of answers, an odd vocabulary, prompt tokens that are not scored
        {"name": "logp_score_bf16", "op": "logp", "N": 4095, "V": 49999, "dtype": "bf16", "top": 5, "train": False, "ignored": 0.3},
        # a policy-gradient step with an entropy term over 8192 tokens
        {"name": "logp_train_bf16", "op": "logp", "N": 8192, "V": 131072, "dtype": "bf16", "top": 0, "train": True, "ignored": 0.1},
        # a small network of a few dozen tensors: launches count
        {"name": "clip_small_fp32", "op": "clip", "layers": 2, "width": 64, "head": 10, "dtype": "fp32", "most": 0.5},
        # a 350M parameter language model
        {"name": "clip_lm_bf16", "op": "clip", "layers": 24, "width": 1024, "head": 50001, "dtype": "bf16", "most": 0.5},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "logp", "logp", "clip"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    while op == "norm":
        rows, D = _log_int(rng, 1, 16384), _log_int(rng, 16, 16384)
        if rng.random() < 0.7:
            D = D // 8 * 8
        if rows * D <= 3.3e7:
            return {"op": op, "rows": rows, "D": D, "dtype": dtype, "residual": rng.random() < 0.7, "mode": rng.choice(["serve", "train", "train", "8bit"])}
    while op == "linear":
        M, N, K = rng.choice([rng.randint(1, 16), _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)]), _log_int(rng, 16, 16384), _log_int(rng, 32, 16384)
        if rng.random() < 0.7:
            N, K = N // 16 * 16, K // 32 * 32
        if M * N * K <= 5.4e11:
            return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype, "bias": rng.random() < 0.3}
    while op == "logp":
        N, V = _log_int(rng, 1, 8192), _log_int(rng, 10, 262144)
        if rng.random() < 0.6:
            V = max(16, V // 8 * 8)
        if N * V <= (1.0e9 if dtype != "fp32" else 5.0e8):
            train = rng.random() < 0.5
            return {"op": op, "N": N, "V": V, "dtype": dtype, "top": 0 if train else rng.choice([0, 1, 5, min(20, V), min(32, V)]), "train": train,
                    "ignored": rng.choice([0.0, 0.1, 0.5])}
    width = _log_int(rng, 16, 1024)
    layers = max(1, min(_log_int(rng, 1, 24), int(2.5e8 / (12 * width * width))))
    return {"op": op, "layers": layers, "width": width, "head": _log_int(rng, 2, 40000), "dtype": dtype, "most": rng.choice([0.01, 0.5, 1.0e6])}


def _shapes(case):
    """The tensors of a transformer of this size, as a model's parameters() gives them."""
    D, L = case["width"], case["layers"]
    layer = [(D,), (D,), (D, D), (D, D), (D, D), (D, D), (D,), (D,), (D,), (4 * D, D), (4 * D,), (D, 4 * D), (D,)]
    return layer * L + [(D,), (case["head"], D), (case["head"],)]


def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        cells, add = case["rows"] * case["D"], 2 if case["residual"] else 1
        if case["mode"] == "8bit":  # the codes are written and read, and the values that they stand for are written
            scales = 8 * case["rows"] * -(-case["D"] // _GROUP)
            return {"bytes": cells * (add * s + (s if add == 2 else 0) + 6) + scales + case["D"] * s, "flops": 7 * cells}
        if case["mode"] == "serve":
            return {"bytes": cells * 2 * add * s + case["D"] * s, "flops": 5 * cells}
        # x, residual, y, sum, their gradients; both terms of a sum have the same gradient
        return {"bytes": cells * s * (3 * add + 1) + 2 * case["D"] * s, "flops": 15 * cells}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        blocks = -(-K // _GROUP)
        return {"bytes": M * K + N * K + 4 * blocks * (M + -(-N // _GROUP)) + M * N * s + (N * s if case["bias"] else 0), "flops": 2 * M * N * K}
    if case["op"] == "logp":
        cells = case["N"] * case["V"]
        return {"bytes": cells * s * (2 if case["train"] else 1) + case["N"] * (16 + 12 * case["top"]), "flops": cells * (12 if case["train"] else 6)}
    n = sum(math.prod(x) for x in _shapes(case))
    return {"bytes": 2 * n * s + 4, "flops": 3 * n}


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


def _hand_codes(t):
    """Codes with their rows on 16-byte boundaries, as functional.quantize_8bit lays them out."""
    K = t.shape[1]
    wide = torch.nn.functional.pad(t, (0, -K % 16))
    return _hand(wide)[:, :K]


def _norm_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, D, dt = case["rows"], case["D"], _DTYPES[case["dtype"]]
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    # hidden states: rows of different size, some features far larger than the others
    feature = torch.where(torch.rand(D, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    size = torch.exp(0.5 * rand(rows, 1))
    x = (rand(rows, D) * (0.5 if case["residual"] else feature * size)).to(dt)
    r = (rand(rows, D) * feature * size).to(dt) if case["residual"] else None
    w = (1 + 0.1 * rand(D)).to(dt)
    train = case["mode"] == "train"
    gy = (1e-2 * rand(rows, D)).to(dt) if train else None
    gs = (1e-2 * rand(rows, D)).to(dt) if train and case["residual"] else None
    return x, r, w, gy, gs


def _linear_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, N, K = case["M"], case["N"], case["K"]
    blocks = -(-K // _GROUP)
    x = torch.randn(M, K, device="cuda", generator=g)
    x *= torch.where(torch.rand(K, device="cuda", generator=g) < 0.01, 20.0, 1.0)
    x = torch.nn.functional.pad(x, (0, blocks * _GROUP - K)).view(M, blocks, _GROUP)
    xs = x.abs().amax(2) / 448.0
    xc = (x / xs[:, :, None]).view(M, -1)[:, :K].to(torch.float8_e4m3fn).view(torch.uint8)
    w = torch.randn(N, K, device="cuda", generator=g).mul_(1.0 / math.sqrt(K))
    tall = -(-N // _GROUP)
    w = torch.nn.functional.pad(w, (0, blocks * _GROUP - K, 0, tall * _GROUP - N)).view(tall, _GROUP, blocks, _GROUP)
    ws = w.abs().amax((1, 3)) / 448.0
    wc = (w / ws[:, None, :, None]).view(tall * _GROUP, -1)[:N, :K].to(torch.float8_e4m3fn).view(torch.uint8)
    b = torch.randn(N, device="cuda", generator=g).mul_(0.1).to(_DTYPES[case["dtype"]]) if case["bias"] else None
    return xc, xs, wc, ws, b


def _logp_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    N, V = case["N"], case["V"]
    t = torch.randint(0, V, (N, 1), device="cuda", generator=g)
    # logits of a model that is sure of some tokens and not of others
    z = torch.randn(N, V, device="cuda", generator=g).mul_(1 + 2 * torch.rand(N, 1, device="cuda", generator=g))
    z.scatter_add_(1, t, 15 * torch.rand(N, 1, device="cuda", generator=g))
    z = z.to(_DTYPES[case["dtype"]])
    t = t[:, 0].clone()
    t[torch.rand(N, device="cuda", generator=g) < case["ignored"]] = -100
    gl, ge = (torch.randn(N, device="cuda", generator=g), 0.01 * torch.rand(N, device="cuda", generator=g)) if case["train"] else (None, None)
    return z, t, gl, ge


def _clip_inputs(case, seed):
    """A flat buffer of the gradients, each tensor at a multiple of 128 elements, with zeros between, and the tensors' places."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    places, at = [], 0
    for s in _shapes(case):
        places.append((at, math.prod(s), s))
        at += -(-math.prod(s) // _GROUP) * _GROUP
    ends = torch.tensor([[a, n] for a, n, _ in places], device="cuda")
    marks = torch.zeros(at + 1, dtype=torch.int32, device="cuda")
    marks[ends[:, 0]] += 1
    marks.index_add_(0, ends.sum(1), -torch.ones(len(places), dtype=torch.int32, device="cuda"))
    inside = marks.cumsum(0, dtype=torch.int32)[:at] > 0
    # the size of the gradients differs from block to block, as it does from row to row of a weight
    size = torch.exp(torch.randn(at // _GROUP, 1, device="cuda", generator=g)).mul_(1e-3).expand(-1, _GROUP).reshape(-1)
    return places, torch.randn(at, device="cuda", generator=g).mul_(inside).mul_(size).to(_DTYPES[case["dtype"]])


def prepare(case, seed):
    if case["op"] == "norm":
        x, r, w, gy, gs = (_hand(v) for v in _norm_inputs(case, seed))
        if own and case["mode"] == "train":
            for v in (x, r, w):
                if v is not None:
                    v.requires_grad_()
        return {"case": case, "x": x, "r": r, "w": w, "gy": gy, "gs": gs}
    if case["op"] == "linear":
        xc, xs, wc, ws, b = _linear_inputs(case, seed)
        return {"case": case, "xc": _hand_codes(xc), "xs": _hand(xs), "wc": _hand_codes(wc), "ws": _hand(ws), "b": _hand(b)}
    if case["op"] == "logp":
        z, t, gl, ge = (_hand(v) for v in _logp_inputs(case, seed))
        if own and case["train"]:
            z.requires_grad_()
        return {"case": case, "z": z, "t": t, "gl": gl, "ge": ge}
    places, grad = _clip_inputs(case, seed)
    state = {"case": case, "g": _hand(grad)}
    if own:
        state["params"] = []
        for a, n, s in places:
            p = torch.zeros(s, dtype=grad.dtype, device="ocl", requires_grad=True)
            p.grad = state["g"][a:a + n].view(s)
            state["params"].append(p)
    return state


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    case = state["case"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "logp": _own_logp, "clip": _own_clip}[case["op"]](case, state)
    return {"norm": _plain_norm, "linear": _plain_linear, "logp": _plain_logp, "clip": _plain_clip}[case["op"]](case, state)


def _own_norm(case, s):
    from pytorch_vulkan_b200 import functional

    if case["mode"] == "8bit":
        codes, scales, *total = functional.rms_norm_8bit(s["x"], s["w"], s["r"], eps=_EPS)
        return [functional.dequantize_8bit(codes, scales), *total]
    out = functional.rms_norm(s["x"], s["w"], s["r"], eps=_EPS)
    out = list(out) if case["residual"] else [out]
    if case["mode"] == "serve":
        return out
    grads = torch.autograd.grad(out, [v for v in (s["x"], s["r"], s["w"]) if v is not None], [v for v in (s["gy"], s["gs"]) if v is not None])
    return [v.detach() for v in out] + list(grads)


def _own_linear(case, s):
    from pytorch_vulkan_b200.functional import linear_8bit

    return [linear_8bit(s["xc"], s["xs"], s["wc"], s["ws"], s["b"], dtype=_DTYPES[case["dtype"]])]


def _own_logp(case, s):
    from pytorch_vulkan_b200.functional import token_log_probs

    out = token_log_probs(s["z"], s["t"], top=case["top"])
    if not case["train"]:
        return list(out)
    return [v.detach() for v in out] + list(torch.autograd.grad(out, [s["z"]], [s["gl"], s["ge"]]))


def _own_clip(case, s):
    from pytorch_vulkan_b200.optim import clip_grad_norm_

    return [clip_grad_norm_(s["params"], case["most"]), s["g"]]


def _plain_norm(case, s):
    dt = s["x"].dtype
    # the norm is that of the sum as it is stored
    total = (s["x"].float() + s["r"].float()).to(dt) if case["residual"] else s["x"]
    h, w = total.float(), s["w"].float()
    # the mean in 64 bits: values next to the border of two codes go by its last bit in 32
    mean = h.double().square().mean(1, keepdim=True).float()
    rstd = 1.0 / torch.sqrt(mean + _EPS)
    n = h * rstd
    y = n * w
    kept = [total] if case["residual"] else []
    if case["mode"] == "8bit":
        rows, D = h.shape
        short = -D % _GROUP
        y = torch.nn.functional.pad(y, (0, short)).view(rows, -1, _GROUP)
        most = y.abs().amax(2, keepdim=True)
        # (448 as a tensor: a quotient with a number is a product with a reciprocal, rounded twice)
        top = torch.full_like(most, 448.0)
        codes = (y * torch.where(most > 2.0 ** -100, top / most, 0.0)).to(torch.float8_e4m3fn)
        scales = torch.where(most > 2.0 ** -100, most / top, 0.0)
        return [(codes.float() * scales).view(rows, -1)[:, :D], *kept]
    if case["mode"] == "serve":
        return [y.to(dt), *kept]
    g = s["gy"].float()
    gw = g * w
    dx = (gw - n * (gw * n).mean(1, keepdim=True)) * rstd
    if case["residual"]:
        dx = dx + s["gs"].float()
    dx = dx.to(dt)
    dw = (g * n).sum(0).to(dt)
    return [y.to(dt), *kept] + ([dx, dx] if case["residual"] else [dx]) + [dw]


def _plain_linear(case, s):
    M, N, K = case["M"], case["N"], case["K"]
    x = s["xc"].view(torch.float8_e4m3fn).float() * s["xs"].repeat_interleave(_GROUP, 1)[:, :K]
    w = s["wc"].view(torch.float8_e4m3fn).float() * s["ws"].repeat_interleave(_GROUP, 0)[:N].repeat_interleave(_GROUP, 1)[:, :K]
    y = x @ w.t()
    if s["b"] is not None:
        y += s["b"].float()
    return [y.to(_DTYPES[case["dtype"]])]


def _plain_logp(case, s):
    z, t, V = s["z"].float() + 0.0, s["t"], case["V"]
    scored = (t >= 0) & (t < V)
    at = torch.where(scored, t, 0)[:, None]
    most = z.amax(1, keepdim=True)
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True)
    lse = most + total.log()
    lp = torch.where(scored, z.gather(1, at)[:, 0] - lse[:, 0], 0.0)
    # log p - the largest one's, so that nothing large is subtracted
    entropy = total.log()[:, 0] - (e * (z - most)).sum(1) / total[:, 0]
    if case["train"]:
        e /= total
        z -= lse
        z += entropy[:, None]
        z *= s["ge"][:, None]
        gl = torch.where(scored, s["gl"], 0.0)[:, None]
        z += gl
        z *= e
        z.neg_()
        z.scatter_add_(1, at, gl)
        return [lp, entropy, z.to(s["z"].dtype)]
    if not case["top"]:
        return [lp, entropy]
    # equal values by their places, the lower one first
    bits = z.view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32) + (V - 1 - torch.arange(V, device=z.device))
    which = V - 1 - (torch.topk(key, case["top"], dim=1).values & 0xFFFFFFFF)
    return [lp, entropy, z.gather(1, which) - lse, which]


def _plain_clip(case, s):
    norm = s["g"].float().square().sum(dtype=torch.float64).sqrt().float()
    s["g"].copy_(s["g"].float() * torch.clamp(case["most"] / (norm + 1e-6), max=1.0))
    return [norm, s["g"]]


# ---------------------------------------------------------------------------------------------------------------- exact
def _numbers(code):
    """The numbers of e4m3 codes, from their bits."""
    c = torch.arange(256, device=code.device)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e.double() - 7))
    return torch.where(c > 127, -v, v)[code.long()]


def _exact_norm(case, seed):
    x, r, w, gy, gs = _norm_inputs(case, seed)
    total = (x.double() + r.double()).to(x.dtype) if r is not None else x
    h, w64 = total.double(), w.double()
    rstd = torch.rsqrt((h * h).sum(1, keepdim=True) / case["D"] + _EPS)
    y = h * rstd * w64
    kept = [total.double()] if r is not None else []
    if case["mode"] == "8bit":
        # a value next to the border of two codes takes the one or the other by its last bit in 32 bits, and the codes are
        # a sixteenth apart: there is no value in 64 bits that it ought to be
        return [None, *kept]
    if case["mode"] == "serve":
        return [y, *kept]
    g = gy.double()
    a = g * w64
    dx = rstd * a - h * rstd ** 3 * (a * h).sum(1, keepdim=True) / case["D"]
    if gs is not None:
        dx = dx + gs.double()
    dw = (g * h * rstd).sum(0)
    return [y, *kept] + ([dx, dx] if r is not None else [dx]) + [dw]


def _exact_linear(case, seed):
    xc, xs, wc, ws, b = _linear_inputs(case, seed)
    y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device="cuda")
    rows = torch.arange(case["N"], device="cuda") // _GROUP
    for k in range(xs.shape[1]):
        at = slice(k * _GROUP, (k + 1) * _GROUP)
        y += (_numbers(xc[:, at]) * xs[:, k, None].double()) @ (_numbers(wc[:, at]) * ws[rows, k, None].double()).t()
    return [y + b.double() if b is not None else y]


def _exact_logp(case, seed):
    z, t, gl, ge = _logp_inputs(case, seed)
    V, top = case["V"], case["top"]
    dz = torch.empty(z.shape, dtype=torch.float64, device="cuda") if case["train"] else None
    step, got = max(1, 2 ** 26 // V), []
    for a in range(0, case["N"], step):
        rows, ta = z[a:a + step].double(), t[a:a + step]
        logp = rows - torch.logsumexp(rows, 1, keepdim=True)
        p = logp.exp()
        h = -(p * logp).sum(1)
        place = torch.arange(len(ta), device="cuda")
        lp = torch.where(ta >= 0, logp[place, ta.clamp(min=0)], 0.0)
        got.append([lp, h])
        if case["train"]:
            l = torch.where(ta >= 0, gl[a:a + step].double(), 0.0)
            d = -p * (l[:, None] + ge[a:a + step].double()[:, None] * (logp + h[:, None]))
            d[place, ta.clamp(min=0)] += l
            dz[a:a + step] = d
        elif top:
            order = torch.sort(rows, dim=1, descending=True, stable=True).indices[:, :top]
            got[-1] += [logp.gather(1, order), order]
    out = [torch.cat(v) for v in zip(*got)]
    return out + [dz] if case["train"] else out


def exact(case, seed):
    if case["op"] == "norm":
        return _exact_norm(case, seed)
    if case["op"] == "linear":
        return _exact_linear(case, seed)
    if case["op"] == "logp":
        return _exact_logp(case, seed)
    _, g = _clip_inputs(case, seed)
    g = g.double()
    norm = torch.linalg.vector_norm(g)
    return [norm, g * min(1.0, case["most"] / (float(norm) + 1e-6))]
