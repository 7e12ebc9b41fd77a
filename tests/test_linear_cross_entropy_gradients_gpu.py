"""Gradients of functional.linear_cross_entropy where rows, vocabulary entries
or operands differ by many powers of ten, and at sizes whose tiles outnumber
the SM pairs, against the formula in float64 (on the GPU's CUDA device, for the
larger sizes' sake).

Bounds.  As in the other tests of this operator: a logit errs by e_z = (D + 8)
2^-23 |x||w|, for fp32 operands 3 2^-22 |x||w| more and 2^-39 of each operand's
largest magnitude, and 2^-23 of itself; a loss by twice the row's largest e_z and
2^-19 (1 + |z|).  A probability errs by p times that, and by 2^-13 p + 2^-27
where it was kept in 16 bits.  What the products read, G_ij = p_ij - goal_ij,
rounds to 16 bits: 2^-9 of itself in bf16, 2^-12 in fp16 (each taken as twice
that here), 3 2^-22 as two fp16 parts, and 2^-40 as least step of either fp16
kind.  For dx that is of a G without the row's own gradient g_i, which multiplies
the row afterwards: the errors of dx_i are g_i times the row's.  For dw, G_ij is
relative to the largest |g| of all rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [FP32, BF16, FP16], ids=["fp32", "bf16", "fp16"])
KEEP = pytest.mark.parametrize("keep", ["0", "2048"], ids=["formed", "kept"])
HALF = {FP32: 2.0 ** -24, BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def make(N, D, V, dtype, bias=False, ignored=0.0, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * N + 3 * D + V)
    w = (torch.randn(V, D, generator=g) / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    x = (torch.randn(N, D, generator=g) + 3 * torch.rand(N, 1, generator=g) * w[t].float()).to(dtype)
    b = (torch.randn(V, generator=g) * 0.5).to(dtype) if bias else None
    t[torch.rand(N, generator=g) < ignored] = -100
    return x, w, b, t


def run(ocl, x, w, b, t, grad=None, **kw):
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b) if v is not None]
    loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2] if b is not None else None, **kw)
    got = torch.autograd.grad(loss, leaves, grad.to(DEV) if grad is not None else None)
    return [loss.detach().cpu(), *(g.cpu() for g in got)]


def formula(x, w, b, t, gi, smooth=0.0, on="cpu"):
    """The losses of the rows, and dx, dw, db for row gradients gi (0 for rows without a loss), each with its bound."""
    dtype, (N, D), V = x.dtype, x.shape, w.shape[0]
    x, w, t, gi = x.double().to(on), w.double().to(on), t.to(on), gi.double().to(on)
    at = t.clamp(min=0)[:, None]
    z = x @ w.t()
    if b is not None:
        z += b.double().to(on)
    logp = torch.log_softmax(z, 1)
    losses = -(1 - smooth) * logp.gather(1, at)[:, 0] - smooth * logp.mean(1)
    left_out = 3 * 2.0 ** -22 if dtype == FP32 else 0.0
    least = 2.0 ** -39 if dtype == FP32 else 0.0
    xa, wa, ga = x.abs(), w.abs(), gi.abs()
    ez = least * (xa.max() * wa.sum(1) + wa.max() * xa.sum(1, keepdim=True)) + ((D + 8) * 2.0 ** -23 + left_out) * (xa @ wa.t())
    err = (2 * (ez + 2.0 ** -22 * z.abs()).max(1).values + 2.0 ** -19 * (1 + z.abs().max(1).values))[:, None]
    p = logp.exp_()
    G = p - smooth / V
    G.scatter_add_(1, at, torch.full_like(G[:, :1], smooth - 1))
    dx, dw, db = (G @ w) * gi[:, None], (G * gi[:, None]).t() @ x, gi @ G
    one = G.abs_()
    eg = p * (err + 2.0 ** -19 + 2.0 ** -22) + one * {FP32: left_out, BF16: 2.0 ** -8, FP16: 2.0 ** -11}[dtype] + 2.0 ** -22 * smooth / V
    eg.scatter_add_(1, at, torch.full_like(eg[:, :1], 2.0 ** -22))
    if dtype != FP32:
        eg += 2.0 ** -13 * p + 2.0 ** -27
    step = 0.0 if dtype == BF16 else 2.0 ** -40
    row = (eg + step) @ wa + ((V + 10) * 2.0 ** -23 + left_out) * (one @ wa) + least * wa.max() * one.sum(1, keepdim=True)
    eg, one = eg * ga[:, None] + step * ga.max(), one * ga[:, None]
    col = eg.t() @ xa + ((N + 10) * 2.0 ** -23 + left_out) * (one.t() @ xa) + least * xa.max() * one.sum(0)[:, None]
    bounds = [row * ga[:, None], col, eg.sum(0) + (N + 10) * 2.0 ** -23 * one.sum(0)]
    grads = [dx, dw, db]
    bounds = [e + HALF[dtype] * (r.abs() + e) + (2.0 ** -25 if dtype == FP16 else 1e-44) for r, e in zip(grads, bounds)]
    return losses, err[:, 0], grads, bounds


def within(got, want, bound, what):
    got = got.double().to(want.device)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, f"{what}: over its bound by {over}"


@TYPES
@KEEP
@pytest.mark.parametrize("shift", [0.0, 30.0, 200.0])
def test_whole_groups_masked_by_the_bias(ocl, monkeypatch, math_fp32, dtype, keep, shift):
    """Entries whose bias is -inf, 64 neighbours and more of them, take no part, however small the others' logits are."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    x, w, b, t = make(70, 32, 1200, dtype, bias=True)
    out = torch.zeros(1200, dtype=torch.bool)
    out[100:600] = out[700:1100] = True
    b[~out] -= shift
    b[out] = float("-inf")
    left = torch.nonzero(~out)[:, 0]
    t = left[t % len(left)]
    loss, dx, dw, db = run(ocl, x, w, b, t, reduction="sum")
    place = torch.cumsum(~out, 0) - 1
    losses, err, grads, bounds = formula(x, w[left], b[left], place[t], torch.ones(70))
    assert (loss.double() - losses.sum()).abs() <= err.sum() + 2.0 ** -23 * losses.sum()
    for a, r, e, what in zip((dx, dw[left], db[left]), grads, bounds, "xwb"):
        within(a, r, e, what)
    assert (dw[out] == 0).all() and (db[out] == 0).all()


ROWS = pytest.mark.parametrize("size", [(150, 72, 520), (20, 1000, 90), (5, 40, 600), (1500, 24, 47003)],
                               ids=["tiles", "slabs", "few", "pieces"])


@TYPES
@KEEP
@ROWS
def test_row_gradients_of_all_sizes(ocl, monkeypatch, math_fp32, size, dtype, keep):
    """reduction="none": the gradients of the rows over twelve powers of ten; each row of dx errs relative to its own."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    N = size[0]
    x, w, b, t = make(*size, dtype, bias=True)
    grad = 10.0 ** torch.linspace(0, -12, N) * torch.where(torch.arange(N) % 3 == 0, -1.0, 1.0)
    if dtype == FP16:
        grad = grad * 1e4  # so that most rows are above fp16's least number
    grad = grad[torch.randperm(N, generator=torch.Generator().manual_seed(1))].contiguous()
    losses, err, grads, bounds = formula(x, w, b, t, grad, smooth=0.1)
    got = run(ocl, x, w, b, t, grad=grad, reduction="none", label_smoothing=0.1)
    within(got[0], losses, err, "losses")
    for a, r, e, what in zip(got[1:], grads, bounds, "xwb"):
        within(a, r, e, what)


@TYPES
@KEEP
@ROWS
def test_row_gradients_that_are_no_numbers(ocl, monkeypatch, math_fp32, size, dtype, keep):
    """reduction="none": an infinite gradient, or NaN, reaches its own row of dx only; in a row without a loss nothing."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    N = size[0]
    x, w, b, t = make(*size, dtype, bias=True)
    t[4] = -100
    grad = torch.linspace(0.5, -0.25, N)
    fine = run(ocl, x, w, b, t, grad=grad, reduction="none")
    grad[4] = float("nan")
    same = run(ocl, x, w, b, t, grad=grad, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(fine, same))
    grad[1], grad[3] = float("inf"), float("nan")
    got = run(ocl, x, w, b, t, grad=grad, reduction="none")
    others = torch.ones(N, dtype=torch.bool)
    others[1] = others[3] = False
    assert torch.equal(got[1][others], fine[1][others])
    assert not torch.isfinite(got[1][1]).any() and torch.isnan(got[1][3]).all()
    assert not torch.isfinite(got[2]).any()


@KEEP
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("size", [(150, 72, 520), (20, 1000, 90), (5, 40, 600), (2100, 24, 12000)],
                         ids=["tiles", "slabs", "few", "pieces"])
def test_operands_scaled_by_powers_of_two(ocl, monkeypatch, math_fp32, size, reduction, keep):
    """x 2^k and w 2^-k have the logits of x and w, and gradients that are theirs times 2^-k and 2^k, bit for bit where
    they are no denormal numbers (an error of one rounding to such a number, 2^-150, where they are)."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    x, w, b, t = make(*size, FP32, bias=True)
    grad = torch.linspace(0.01, 0.02, size[0]) if reduction == "none" else torch.tensor(0.01)
    loss, dx, dw, db = run(ocl, x, w, b, t, grad=grad, reduction=reduction)
    for k in (96, -96):
        loss2, dx2, dw2, db2 = run(ocl, x * 2.0 ** k, w * 2.0 ** -k, b, t, grad=grad, reduction=reduction)
        assert torch.equal(loss, loss2) and torch.equal(db, db2)
        for a, a2, by in ((dx, dx2, -k), (dw, dw2, k)):
            want = a.double() * 2.0 ** by
            normal = want.abs() >= 2.0 ** -126
            assert normal.double().mean() > 0.99
            assert torch.equal(a2.double()[normal], want[normal])
            assert ((a2.double() - want).abs()[~normal] <= 2.0 ** -149).all()


def test_forward_mode_is_refused(ocl):
    """A tangent is not lost without a word."""
    import torch.autograd.forward_ad as fw

    x, w, b, t = make(12, 16, 40, FP32, bias=True)
    given = [v.to(DEV) for v in (x, w, b)]
    with fw.dual_level():
        for k in range(3):
            for requires in (False, True):
                args = [v.detach().requires_grad_(requires) for v in given]
                args[k] = fw.make_dual(args[k], torch.ones_like(given[k]))
                with pytest.raises(RuntimeError, match="jvp"):
                    ocl.functional.linear_cross_entropy(args[0], args[1], t.to(DEV), args[2])
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                    ocl.functional.linear_cross_entropy(args[0], args[1], t.to(DEV), args[2])
        table = fw.make_dual(torch.zeros(8, 2).to(DEV), torch.ones(8, 2).to(DEV))
        with pytest.raises(RuntimeError, match="jvp"):
            ocl.functional.relative_position_bias(table, 5, 5)
    want = ocl.functional.linear_cross_entropy(given[0], given[1], t.to(DEV), given[2])  # outside, as ever
    assert torch.isfinite(want.cpu())


@TYPES
@KEEP
@pytest.mark.parametrize("size", [(2304, 1160, 4608), (2310, 8192, 2310), (9000, 520, 9001), (2304, 2304, 4608)],
                         ids=lambda s: "x".join(map(str, s)))
def test_more_tiles_than_pairs(ocl, monkeypatch, math_fp32, size, dtype, keep):
    """Tiles of 256 columns that outnumber the pairs of SMs, with sums over K in several chunks, so that accumulators are
    used again with either phase; tiles in groups the last of which is narrower; and dx laid down by one piece of the
    vocabulary and added to by the next on tiles whose K is not cut."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    x, w, b, t = make(*size, dtype, bias=True, ignored=0.1)
    scored = t >= 0
    gi = scored.double() / scored.sum()
    losses, err, grads, bounds = formula(x, w, b, t, gi, smooth=0.05, on="cuda")
    got = run(ocl, x, w, b, t, label_smoothing=0.05)
    want, bound = (gi.to("cuda") * losses).sum(), (gi.to("cuda") * err).sum()
    within(got[0], want, bound + 2.0 ** -22 * want, "loss")
    for a, r, e, what in zip(got[1:], grads, bounds, "xwb"):
        within(a, r, e, what)
    torch.cuda.empty_cache()


@TYPES
@KEEP
@ROWS
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_upstream_gradients_that_are_no_numbers(ocl, monkeypatch, math_fp32, size, dtype, keep, reduction):
    """An infinite gradient of the loss, or NaN: rows without a loss have the gradient 0 all the same, and without any row
    that has one everything is 0."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    x, w, b, t = make(*size, dtype, bias=True)
    t[4], t[1] = -100, size[2]
    for bad in (float("inf"), float("-inf"), float("nan")):
        _, dx, dw, db = run(ocl, x, w, b, t, grad=torch.tensor(bad), reduction=reduction)
        assert (dx[4] == 0).all() and (dx[1] == 0).all()
        assert not torch.isfinite(dx[0]).any() and not torch.isfinite(dx[2:4]).any()
        assert not torch.isfinite(db).any()
        for g in run(ocl, x, w, b, torch.full_like(t, -100), grad=torch.tensor(bad), reduction=reduction)[1:]:
            assert (g == 0).all()


@TYPES
@KEEP
def test_losses_that_are_summed_afterwards(ocl, monkeypatch, math_fp32, dtype, keep):
    """reduction="none" and a sum or mean of the losses: one number comes back for all rows, whatever the shape."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    x, w, b, t = make(150, 72, 520, dtype, bias=True, ignored=0.2)
    for shape in ((150,), (10, 15), (1, 150), (150, 1)):
        leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
        xs, ts = leaves[0].view(*shape, 72), t.view(shape).to(DEV)
        f = lambda red: ocl.functional.linear_cross_entropy(xs, leaves[1], ts, leaves[2], reduction=red)
        want = torch.autograd.grad(f("sum"), leaves)
        got = torch.autograd.grad(f("none").sum(), leaves)
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, got))
        each = torch.autograd.grad(f("none"), leaves, torch.ones(shape).to(DEV))
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, each))
        part = torch.full(shape[:-1] + (1,), 0.5)  # rows of the batch with a gradient each: no single number
        part.view(-1)[0] = 2.0
        expanded = torch.autograd.grad(f("none"), leaves, part.to(DEV).expand(shape))
        each = torch.autograd.grad(f("none"), leaves, part.expand(shape).contiguous().to(DEV))
        assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(expanded, each))
    one = [v.to(DEV).requires_grad_() for v in (x[:1], w)]
    f = lambda red: ocl.functional.linear_cross_entropy(*one, t.clamp(min=0)[:1].to(DEV), reduction=red)
    for a, b in zip(torch.autograd.grad(f("none").sum() * 0.25, one), torch.autograd.grad(f("sum") * 0.25, one)):
        assert torch.equal(a.cpu(), b.cpu())
