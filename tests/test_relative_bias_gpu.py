"""Learned relative position bias on `ocl` against its definition: buckets by
whole-number arithmetic, values exact, gradients summed in float64.

A table's gradient is summed in fp32 over at most 64 rows of a diagonal, or 64
elements of a row where one bucket holds all, and in float64 beyond, then rounded once to the table's type: its error is at most
64 * 2^-24 of the sum of magnitudes and half a step of the result.
"""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def bucket(rel, buckets, both, far):
    n = buckets // 2 if both else buckets
    e = n // 2
    d = abs(rel) if both else max(-rel, 0)
    b = d
    if d >= e:
        k = 0  # the last k with d >= e (far / e)^(k / (n - e)), by whole numbers
        while k < n - 1 - e and d ** (n - e) * e ** (k + 1) >= far ** (k + 1) * e ** (n - e):
            k += 1
        b = e + k
    return b + (n if both and rel > 0 else 0)


def index(q, k, buckets, both, far, offset):
    of = {r: bucket(r, buckets, both, far) for r in range(-(q - 1) - offset, k - offset)}
    if q == 0 or k == 0:
        return torch.zeros(q, k, dtype=torch.int64)
    line = torch.tensor([of[r] for r in sorted(of)])
    return line[(torch.arange(k)[None] - torch.arange(q)[:, None]) + q - 1]


CASES = [
    # heads, q, k, buckets, both, far, offset
    (12, 197, 197, 32, True, 128, 0),     # ViT-B/16's tokens and heads
    (3, 1, 1, 32, True, 128, 0),
    (4, 1, 2051, 32, False, 128, 2050),   # one new token against a cache
    (1, 7, 1030, 16, False, 20, 1023),
    (2, 65, 33, 4, True, 2, 0),           # smallest tables, distances on every border
    (2, 40, 40, 2, False, 2, 0),
    (5, 130, 1025, 64, True, 1024, 0),    # past one column tile by one
    (2, 1025, 63, 128, True, 500, 100),
    (3, 16, 16, 8, True, 100, 1000),      # every key far behind
    (3, 16, 16, 8, False, 100, -1000),    # every key far ahead
    (1, 300, 2100, 512, False, 1 << 20, 7),
    (2, 37, 5003, 32, True, 40, 2600),    # long runs of one bucket before and behind the others
    (2, 90, 5003, 32, False, 40, 2600),
    (2, 0, 5, 8, True, 9, 0),
    (2, 5, 0, 8, True, 9, 0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_values_and_gradient(ocl, case, dtype):
    H, q, k, buckets, both, far, offset = case
    gen = torch.Generator().manual_seed(q * 31 + k)
    table = torch.randn(buckets, H, generator=gen).to(dtype)
    grad = torch.randn(1, H, q, k, generator=gen).to(dtype)
    td = table.to(DEV).requires_grad_()
    out = ocl.functional.relative_position_bias(td, q, k, bidirectional=both, max_distance=far, q_offset=offset)
    at = index(q, k, buckets, both, far, offset)
    assert out.shape == (1, H, q, k) and out.dtype == dtype
    assert torch.equal(out.detach().cpu(), table[at].permute(2, 0, 1)[None])
    (got,) = torch.autograd.grad(out, td, grad.to(DEV))
    cells = grad[0].double().reshape(H, -1).t()
    want = torch.zeros(buckets, H, dtype=torch.float64).index_add_(0, at.reshape(-1), cells)
    size = torch.zeros(buckets, H, dtype=torch.float64).index_add_(0, at.reshape(-1), cells.abs())
    bound = 64 * 2.0 ** -24 * size
    bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + (6e-8 if dtype == torch.float16 else 0)
    assert got.dtype == dtype
    assert ((got.cpu().double() - want).abs() <= bound).all()


def test_gradient_strides_and_batches(ocl):
    """The backward op takes any strides: a broadcast batch, permuted and gapped gradients, a batch to be summed."""
    H, q, k = 3, 50, 70
    gen = torch.Generator().manual_seed(0)
    at = index(q, k, 32, True, 64, 5)

    def check(gd, g):
        got = torch.ops.ocl.relative_position_bias_backward(gd, 32, True, 64, 5).cpu().double()
        cells = g.double().sum(0).reshape(H, -1).t()
        want = torch.zeros(32, H, dtype=torch.float64).index_add_(0, at.reshape(-1), cells)
        size = torch.zeros(32, H, dtype=torch.float64).index_add_(0, at.reshape(-1), g.double().abs().sum(0).reshape(H, -1).t())
        assert ((got - want).abs() <= 65 * 2.0 ** -24 * size).all()

    g = torch.randn(4, H, q, k, generator=gen)
    check(g.to(DEV), g)
    check(g[:1].to(DEV).expand(6, H, q, k), g[:1].expand(6, H, q, k))
    h = torch.randn(2, k, q, H, generator=gen)
    check(h.to(DEV).permute(0, 3, 2, 1), h.permute(0, 3, 2, 1))
    w = torch.randn(2, H, q, 2 * k + 1, generator=gen)
    check(w.to(DEV)[..., 1::2], w[..., 1::2])
    check(w.to(DEV)[..., 1:k + 1], w[..., 1:k + 1])
    check(g.to(DEV)[:0], g[:0])


def test_bias_in_attention(ocl, math_fp32):
    """Through scaled_dot_product_attention as its mask, shared by the batch, with every gradient."""
    B, H, L, D = 2, 4, 37, 32
    gen = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(B, H, L, D, generator=gen) for _ in range(4))
    table = torch.randn(16, H, generator=gen)
    dev = [x.to(DEV).requires_grad_() for x in (q, k, v, table)]
    bias = ocl.functional.relative_position_bias(dev[3], L, L, max_distance=20)
    F.scaled_dot_product_attention(*dev[:3], attn_mask=bias).backward(do.to(DEV))
    ref = [x.double().requires_grad_() for x in (q, k, v, table)]
    s = ref[0] @ ref[1].transpose(-1, -2) / math.sqrt(D) + ref[3][index(L, L, 16, True, 20, 0)].permute(2, 0, 1)
    (torch.softmax(s, -1) @ ref[2]).backward(do.double())
    for a, b in zip(dev, ref):
        # fp32 products over at most 37 and 32 terms: 1e-5 of the tensor's magnitude, as the attention tests hold
        assert (a.grad.cpu().double() - b.grad).abs().max() <= 1e-5 * b.grad.abs().max().clamp(min=1)


def test_captured_with_its_gradient(ocl):
    table = torch.randn(32, 4, generator=torch.Generator().manual_seed(2)).to(DEV).requires_grad_()
    grad = torch.randn(1, 4, 60, 60, generator=torch.Generator().manual_seed(3)).to(DEV)

    def run():
        out = ocl.functional.relative_position_bias(table, 60, 60)
        return out.detach(), torch.autograd.grad(out, table, grad)[0]

    eager = run()
    graph = torch.ocl.Graph()
    with graph.capture():
        held = run()
    for scale in (1.0, 2.0):
        with torch.no_grad():
            table.mul_(scale)
            grad.mul_(scale)
        graph.replay()
        assert torch.equal(held[0].cpu(), eager[0].cpu() * scale)
        assert torch.equal(held[1].cpu(), eager[1].cpu() * scale)
    graph.reset()


def test_refusals(ocl):
    f = ocl.functional.relative_position_bias
    t = torch.zeros(32, 4).to(DEV)
    for args, kw, match in [
        ((torch.zeros(33, 4).to(DEV), 3, 3), {}, "even number"),
        ((torch.zeros(2, 4).to(DEV), 3, 3), {}, "even number"),
        ((torch.zeros(1, 4).to(DEV), 3, 3), dict(bidirectional=False), "buckets"),
        ((torch.zeros(514, 4).to(DEV), 3, 3), {}, "buckets"),
        ((t, 3, 3), dict(max_distance=8), "max_distance"),
        ((t, 3, 3), dict(max_distance=1 << 21), "max_distance"),
        ((t, -1, 3), {}, "below zero"),
        ((t, 3, 3), dict(q_offset=1 << 40), "out of range"),
        ((t[0], 3, 3), {}, "num_buckets, heads"),
        ((t.to(torch.int32), 3, 3), {}, "fp32, fp16 or bf16"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)
    with pytest.raises((RuntimeError, NotImplementedError)):
        f(torch.zeros(32, 4), 3, 3)
    w = t.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(f(w, 3, 3).sum(), w, create_graph=True)
