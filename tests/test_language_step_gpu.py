"""The language model's operators together, as a user has them: a policy-gradient
step (norms with the residual stream, log probabilities and entropy, clipping,
AdamW), and serving in 8 bits (norms into layers, the next token's log
probabilities and alternatives).

The training reference is the same model in float64 on the CPU.  In exact fp32
mode all products of the step are fp32, so that gradients are within 2^-15 of
their largest element (a few hundred roundings of 2^-24 through six products).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
B, L, E, F, V = 3, 17, 96, 160, 517
U = 2.0 ** -24


def parameters():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"norm1": 1 + 0.1 * r(E), "up": r(F, E) / math.sqrt(E), "down": r(E, F) / math.sqrt(F), "norm2": 1 + 0.1 * r(E),
            "head": r(V, E) / math.sqrt(E)}


def inputs():
    g = torch.Generator().manual_seed(1)
    x, prev = torch.randn(B, L, E, generator=g), torch.randn(B, L, E, generator=g)
    t = torch.randint(0, V, (B, L), generator=g)
    t[0, :5] = -100  # a prompt
    return x, prev, t, torch.randn(B, L, generator=g)


def loss_ocl(pkg, p, x, prev, t, adv):
    f = pkg.functional
    y, stream = f.rms_norm(x, p["norm1"], prev, eps=1e-5)
    h = torch.relu(y.reshape(-1, E) @ p["up"].t()) @ p["down"].t()
    y, _ = f.rms_norm(h.view(B, L, E), p["norm2"], stream, eps=1e-5)
    logits = (y.reshape(-1, E) @ p["head"].t()).view(B, L, V)
    lp, entropy = f.token_log_probs(logits, t)
    return -(lp * adv).sum() / (B * L) - 0.05 * entropy.mean()


def loss_cpu(p, x, prev, t, adv):
    def norm(h, w):
        return h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w

    stream = x + prev
    h = torch.relu(norm(stream, p["norm1"]) @ p["up"].t()) @ p["down"].t()
    logp = torch.log_softmax(norm(h + stream, p["norm2"]) @ p["head"].t(), -1)
    lp = torch.where(t >= 0, logp.gather(-1, t.clamp(min=0)[..., None])[..., 0], 0.0)
    return -(lp * adv).sum() / (B * L) + 0.05 * (logp.exp() * logp).sum(-1).mean()


def test_policy_gradient_step(ocl, math_fp32):
    x, prev, t, adv = inputs()
    ref = {k: v.double().requires_grad_() for k, v in parameters().items()}
    want = loss_cpu(ref, x.double(), prev.double(), t, adv.double())
    want.backward()
    p = {k: v.to(DEV).requires_grad_() for k, v in parameters().items()}
    opt = ocl.optim.AdamW(p.values(), lr=1e-3, weight_decay=0.0)
    loss = loss_ocl(ocl, p, x.to(DEV), prev.to(DEV), t.to(DEV), adv.to(DEV))
    loss.backward()
    # a sum of terms of up to 10 that cancel
    assert abs(loss.item() - want.item()) <= 2.0 ** -18 * 10
    for k, v in p.items():
        g, r = v.grad.cpu().double(), ref[k].grad
        assert (g - r).abs().max() <= 2.0 ** -15 * r.abs().max(), k
    norm = math.sqrt(sum(r.grad.square().sum().item() for r in ref.values()))
    got = ocl.optim.clip_grad_norm_(p.values(), norm / 3).item()
    assert abs(got - norm) <= 2.0 ** -15 * norm
    for k, v in p.items():
        r = ref[k].grad / 3
        assert (v.grad.cpu().double() - r).abs().max() <= 2.0 ** -14 * r.abs().max(), k
    before = {k: v.detach().cpu() for k, v in p.items()}
    opt.step()
    # a first step of Adam moves by lr times the gradient's sign, where that is not near eps
    for k, v in p.items():
        sure = ref[k].grad.abs() > 2.0 ** -12 * ref[k].grad.abs().max()
        moved = (v.detach().cpu() - before[k])[sure]
        assert torch.equal(moved.sign(), -ref[k].grad[sure].sign().float())


def test_captured_steps_are_eager_steps(ocl, math_fp32):
    """Three steps replayed from a graph and three issued one by one, bit for bit, with an eager graph of the same leaves
    alive while the step is captured."""
    x, prev, t, adv = (v.to(DEV) for v in inputs())
    results = []
    for captured in (False, True):
        p = {k: v.to(DEV).requires_grad_() for k, v in parameters().items()}
        opt = ocl.optim.AdamW(p.values(), lr=1e-2)

        def run():
            opt.zero_grad(set_to_none=True)
            loss = loss_ocl(ocl, p, x, prev, t, adv)
            loss.backward()
            norm = ocl.optim.clip_grad_norm_(p.values(), 0.1)
            opt.step()
            return loss.detach(), norm

        run()
        seen = []
        if captured:
            alive = loss_ocl(ocl, p, x, prev, t, adv)
            graph = torch.ocl.Graph()
            with graph.capture():
                held = run()
            for _ in range(3):
                graph.replay()
                seen.append([v.item() for v in held])
            assert torch.isfinite(alive.cpu())
            graph.reset()
        else:
            seen = [[v.item() for v in run()] for _ in range(3)]
        results.append((seen, [v.detach().cpu() for v in p.values()]))
    assert results[0][0] == results[1][0]
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))


class Server:
    """A layer and the head in 8 bits, their weights quantised once."""

    def __init__(self, pkg):
        self.f = pkg.functional
        self.p = {k: v.to(torch.bfloat16).to(DEV) for k, v in parameters().items()}
        self.w = {k: self.f.quantize_8bit(self.p[k], block_rows=128) for k in ("up", "down", "head")}

    def __call__(self, x, prev, t, top):
        f, p, w = self.f, self.p, self.w
        codes, scales, stream = f.rms_norm_8bit(x, p["norm1"], prev)
        up = torch.relu(f.linear_8bit(codes, scales, *w["up"], dtype=torch.float32))
        down = f.linear_8bit(*f.quantize_8bit(up), *w["down"], dtype=torch.bfloat16)
        codes, scales, stream = f.rms_norm_8bit(down, p["norm2"], stream)
        logits = f.linear_8bit(codes, scales, *w["head"], dtype=torch.float32)
        return (codes, scales, stream, logits, *f.token_log_probs(logits, t, top=top))


@pytest.mark.parametrize("rows", [(1,), (B, L), (200,)], ids=["token", "batch", "many"])
def test_serving_in_8_bits(ocl, rows):
    g = torch.Generator().manual_seed(2)
    x, prev = (torch.randn(*rows, E, generator=g).to(torch.bfloat16) for _ in range(2))
    t = torch.randint(0, V, rows, generator=g)
    with torch.no_grad():
        server = Server(ocl)
        codes, scales, stream, logits, lp, entropy, tlp, tat = server(x.to(DEV), prev.to(DEV), t.to(DEV), 5)
        # the last layer, of the codes that it had
        a = ocl.functional.dequantize_8bit(codes, scales).cpu().double()
        w = ocl.functional.dequantize_8bit(*server.w["head"]).cpu().double()
    z = logits.cpu()
    assert z.shape == (*rows, V) and stream.shape == x.shape
    # one block of 96 products: 2 (128 + 1 + 4) roundings of the magnitudes' sum
    assert ((z.double() - a @ w.t()).abs() <= 2 * 133 * U * (a.abs() @ w.abs().t())).all()
    logp = torch.log_softmax(z.double(), -1)
    h = -(logp.exp() * logp).sum(-1)
    bound = U * (100 + 10 * h)
    want = logp.gather(-1, t[..., None])[..., 0]
    assert ((lp.cpu().double() - want).abs() <= bound + 3 * U * want.abs()).all()
    assert ((entropy.cpu().double() - h).abs() <= bound * (1 + h)).all()
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :5]
    assert torch.equal(tat.cpu(), order)
    assert ((tlp.cpu().double() - logp.gather(-1, order)).abs() <= bound[..., None] + 3 * U * logp.gather(-1, order).abs()).all()
    # and near the model in bf16's numbers without codes: what three layers in 8 bits leave, a tenth of the logits' size
    p = {k: v.cpu().double() for k, v in server.p.items()}
    s = (x.float() + prev.float()).to(torch.bfloat16).double()
    norm = lambda v, weight: v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight  # noqa: E731
    exact = norm(torch.relu(norm(s, p["norm1"]) @ p["up"].t()) @ p["down"].t() + s, p["norm2"]) @ p["head"].t()
    assert (z.double() - exact).norm() <= 0.1 * exact.norm()


def test_captured_serving(ocl):
    """One graph of the whole pass, replayed for new inputs: the same bits as eager."""
    g = torch.Generator().manual_seed(3)
    batches = [[torch.randn(4, E, generator=g).to(torch.bfloat16), torch.randn(4, E, generator=g).to(torch.bfloat16),
                torch.randint(0, V, (4,), generator=g)] for _ in range(3)]
    with torch.no_grad():
        server = Server(ocl)
        eager = [[v.cpu() for v in server(*(b.to(DEV) for b in batch), 3)] for batch in batches]
        held = [b.to(DEV) for b in batches[0]]
        graph = torch.ocl.Graph()
        with graph.capture():
            out = server(*held, 3)
        for batch, want in zip(batches, eager):
            for a, b in zip(held, batch):
                a.copy_(b)
            graph.replay()
            assert all(torch.equal(a.cpu(), b) for a, b in zip(out, want))


def test_on_another_stream_and_thread(ocl):
    """The operators on a stream of their own, and from two threads at once: the bits of the default stream's."""
    import threading

    g = torch.Generator().manual_seed(4)
    x, prev = (torch.randn(64, E, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    t = torch.randint(0, V, (64,), generator=g).to(DEV)
    with torch.no_grad():
        server = Server(ocl)
        want = [v.cpu() for v in server(x, prev, t, 7)]
        stream = torch.Stream(device=DEV)
        torch.ocl.synchronize()
        with stream:
            for _ in range(5):
                got = server(x, prev, t, 7)
        stream.synchronize()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
        results = {}

        def work(i):
            with torch.no_grad():
                for _ in range(20):
                    out = server(x, prev, t, 7)
                results[i] = [v.cpu() for v in out]

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(results[i], want))


@pytest.mark.parametrize("rows", [1, 130, 700])
def test_one_call_after_the_other(ocl, rows):
    """A launch may begin before the one in front of it ends: a long chain of small calls, each of which reads what the
    last one wrote and writes where an earlier one read, gives the bits of the same chain with a pause after each."""
    f = ocl.functional
    g = torch.Generator().manual_seed(rows)
    D, V = 640, 1000
    w1, ws1 = f.quantize_8bit((0.05 * torch.randn(D, D, generator=g)).to(torch.bfloat16).to("ocl"), block_rows=128)
    w2, ws2 = f.quantize_8bit((0.05 * torch.randn(V, D, generator=g)).to(torch.bfloat16).to("ocl"), block_rows=128)
    x0 = torch.randn(rows, D, generator=g).to(torch.bfloat16)
    gain = (1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to("ocl")
    tokens = torch.randint(0, V, (rows,), generator=g).to("ocl")

    def chain(pause):
        out = []
        wait = torch.ocl.synchronize if pause else (lambda: None)
        x, stream = x0.to("ocl"), x0.to("ocl")
        with torch.no_grad():
            for i in range(30):
                codes, scales, stream = f.rms_norm_8bit(x, gain, stream)
                wait()
                x = f.linear_8bit(codes, scales, w1, ws1)
                wait()
                codes, scales = f.quantize_8bit(f.rms_norm(x, gain))
                wait()
                logits = f.linear_8bit(codes, scales, w2, ws2)
                wait()
                lp, entropy, _, best = f.token_log_probs(logits, tokens, top=3)
                wait()
                x = f.dequantize_8bit(codes, scales, dtype=torch.bfloat16)
                wait()
                out.append((lp + entropy, best))
        return [(a.cpu(), b.cpu()) for a, b in out] + [(x.cpu(), stream.cpu())]

    want = chain(True)
    for _ in range(3):
        for (a, b), (c, d) in zip(chain(False), want):
            assert torch.equal(a, c) and torch.equal(b, d)
