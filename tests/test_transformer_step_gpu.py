"""A transformer layer's training step on `ocl` with the pieces together, as a
user has them: a learned relative position bias into attention, the cross
entropy of the last linear layer, and AdamW with 32-bit or 8-bit moments.

The reference is the same model in float64 on the CPU.  In exact fp32 mode all
products of the step are fp32, so that gradients are within 2^-15 of their
largest element (a few hundred roundings of 2^-24 through five products), and
the updated parameters within what that makes of an Adam update: nothing where
the gradient is not near zero, since a first step moves by lr times its sign.
"""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
B, L, H, D, V = 3, 29, 4, 32, 517
E = H * D


def parameters():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)
    return {"qkv": r(3 * E, E) / math.sqrt(E), "out": r(E, E) / math.sqrt(E), "table": r(16, H), "norm": 1 + 0.1 * r(E),
            "shift": 0.1 * r(E), "head": r(V, E) / math.sqrt(E), "bias": 0.1 * r(V)}


def inputs():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, L, E, generator=g)
    t = torch.randint(0, V, (B, L), generator=g)
    t[0, -5:] = -100  # a padded sequence
    t[2, 3] = -100
    return x, t


def buckets(n, far):
    """Of the distances i - j, one direction: keys ahead of the query take bucket 0."""
    e, at = n // 2, torch.zeros(L, L, dtype=torch.int64)
    for i in range(L):
        for j in range(i + 1):
            d = i - j
            at[i, j] = d if d < e else min(n - 1, e + int(math.log(d / e) / math.log(far / e) * (n - e) + 1e-9))
    return at


def attention_input(p, x):
    h = F.layer_norm(x, (E,), p["norm"], p["shift"])
    qkv = (h.reshape(-1, E) @ p["qkv"].t()).view(B, L, 3, H, D).permute(2, 0, 3, 1, 4)
    return qkv[0], qkv[1], qkv[2]


def features(p, x, o):
    return x + (o.transpose(1, 2).reshape(-1, E) @ p["out"].t()).view(B, L, E)


def causal():
    return torch.full((L, L), float("-inf")).triu(1)


def loss_ocl(pkg, p, x, t, mask):
    q, k, v = attention_input(p, x)
    bias = pkg.functional.relative_position_bias(p["table"], L, L, bidirectional=False, max_distance=20) + mask
    h = features(p, x, F.scaled_dot_product_attention(q, k, v, attn_mask=bias))
    return pkg.functional.linear_cross_entropy(h, p["head"], t, p["bias"], label_smoothing=0.1)


def loss_cpu(p, x, t):
    q, k, v = attention_input(p, x)
    s = q @ k.transpose(-1, -2) / math.sqrt(D) + p["table"][buckets(16, 20)].permute(2, 0, 1) + causal().double()
    h = features(p, x, torch.softmax(s, -1) @ v)
    return F.cross_entropy(F.linear(h, p["head"], p["bias"]).reshape(-1, V), t.reshape(-1), label_smoothing=0.1)


@pytest.fixture()
def step(ocl, math_fp32):
    x, t = inputs()
    ref = {k: v.double().requires_grad_() for k, v in parameters().items()}
    loss = loss_cpu(ref, x.double(), t)
    loss.backward()
    return x, t, ref, loss.item()


@pytest.mark.parametrize("bits", [32, 8])
def test_one_step(ocl, step, bits):
    x, t, ref, want = step
    p = {k: v.to(DEV).requires_grad_() for k, v in parameters().items()}
    opt = ocl.optim.AdamW(p.values(), lr=1e-3, weight_decay=0.1, state_bits=bits)
    loss = loss_ocl(ocl, p, x.to(DEV), t.to(DEV), causal().to(DEV))
    loss.backward()
    assert abs(loss.item() - want) <= 2.0 ** -18 * want
    for k, v in p.items():
        g, r = v.grad.cpu().double(), ref[k].grad
        assert (g - r).abs().max() <= 2.0 ** -15 * r.abs().max(), k
    opt.step()
    for k, v in p.items():
        g, before = ref[k].grad, ref[k].detach()
        after = before * (1 - 1e-3 * 0.1) - 1e-3 * g / (g.abs() + 1e-8)
        sure = g.abs() > 2.0 ** -13 * g.abs().max()  # else the update may turn with the gradient's error
        # lr times the share of eps and of the gradient's error in a quotient near 1, and fp32's roundings of p
        bound = 1e-3 * (2.0 ** -15 * g.abs().max() + 1e-8) / g.abs().clamp(min=1e-30) * 1e-3 + 2.0 ** -20 * (before.abs() + 1e-3)
        assert ((v.detach().cpu().double() - after).abs()[sure] <= bound[sure] + 1e-9).all(), k


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_eager_steps(ocl, step, bits):
    """Three steps replayed from a graph, and three issued one by one from the same state, bit for bit; with an eager
    graph of the same leaves alive while the step is captured."""
    x, t, _, _ = step
    results = []
    for captured in (False, True):
        p = {k: v.to(DEV).requires_grad_() for k, v in parameters().items()}
        xd, td, mask = x.to(DEV), t.to(DEV), causal().to(DEV)
        opt = ocl.optim.AdamW(p.values(), lr=1e-2, state_bits=bits)

        def run():
            opt.zero_grad(set_to_none=True)
            loss = loss_ocl(ocl, p, xd, td, mask)
            loss.backward()
            opt.step()
            return loss.detach()

        run()
        losses = []
        if captured:
            alive = loss_ocl(ocl, p, xd, td, mask)
            graph = torch.ocl.Graph()
            with graph.capture():
                held = run()
            for _ in range(3):
                graph.replay()
                losses.append(held.item())
            assert torch.isfinite(alive.cpu())
        else:
            losses = [run().item() for _ in range(3)]
        results.append((losses, [v.detach().cpu() for v in p.values()],
                        [s.cpu() for v in p.values() for s in opt.state[v].values()]))
        if captured:
            graph.reset()
    assert results[0][0] == results[1][0]
    for k in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(results[0][k], results[1][k]))
