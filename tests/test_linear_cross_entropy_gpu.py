"""Cross entropy of a linear layer on `ocl` (functional.linear_cross_entropy)
against F.cross_entropy of the product in float64 on the CPU.

Bounds.  A logit is a sum of D products in fp32 accumulators: its error is at
most e_z = (D + 8) u' |x||w| with u' = 2^-23 (a tensor core may cut rather than
round), plus what two fp16 parts leave of fp32 operands: each part rounds by half
of 2^-10, so that each operand is within 2^-22 of itself and the product of the
second parts, which is not formed, below 2^-22 |x||w|, 3 2^-22 in all; and scaled
so that the largest magnitude is at least 2^14, an operand's second part cannot
be nearer than half of fp16's least step, 2^-25 / 2^14 = 2^-39 of that largest.
The log of the sum of exponentials errs by at most the largest such error and
2^-20 of its own; a loss by twice that.  A probability p errs by p (2 e_z +
2^-19), and, where the forward pass kept it for 16-bit operands (a number with
12 bits of mantissa and 4 of exponent relative to the largest of 64 columns), by
half a step more: 2^-13 p, or 2^-27 of that largest (at most 1).  G is held in 16 bits (2^-9 for bf16, 2^-12 for fp16, 3 2^-22 as two of
them for fp32, both fp16 kinds scaled by 2^15 relative to the largest row's gradient), and the gradients are sums of products of G, so that each is within
|G| |w| (or |G|^T |x|) times those errors, the accumulation's, and one rounding
to its type.
"""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
HALF = {FP32: 2.0 ** -24, BF16: 2.0 ** -8, FP16: 2.0 ** -11}


@pytest.fixture(params=[1, 0], ids=["fp32math", "tf32math"])
def mode(ocl, request):
    old = torch.ocl.get_math_mode()
    torch.ocl.set_math_mode(request.param)
    yield request.param
    torch.ocl.set_math_mode(old)


def make(N, D, V, dtype, bias=False, ignored=0.0, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7 * N + 3 * D + V)
    w = (torch.randn(V, D, generator=g) / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    x = (torch.randn(N, D, generator=g) * scale + 3 * torch.rand(N, 1, generator=g) * w[t].float()).to(dtype)
    b = (torch.randn(V, generator=g) * 0.5).to(dtype) if bias else None
    t[torch.rand(N, generator=g) < ignored] = -100
    return x, w, b, t


def check(ocl, x, w, b, t, mode=1, reduction="mean", smooth=0.0, ignore=-100, grad=None, given=None):
    """`given`: the device tensors to call with, where they are other views than plain copies."""
    N, D = x.reshape(-1, x.shape[-1]).shape
    V, dtype = w.shape[0], x.dtype
    leaves = given or [v.to(DEV).requires_grad_() if v is not None else None for v in (x, w, b)]
    loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], ignore_index=ignore,
                                               reduction=reduction, label_smoothing=smooth)
    assert loss.dtype == FP32 and loss.shape == (t.shape if reduction == "none" else ())
    want_grad = torch.ones(loss.shape) if grad is None else grad
    used = [v for v in leaves if v is not None]
    got = torch.autograd.grad(loss, used, want_grad.to(DEV))

    ref = [v.double().requires_grad_() if v is not None else None for v in (x, w, b)]
    scored = ((t != ignore) & (t >= 0) & (t < V)).reshape(-1)
    # rows without a loss take no part, whatever they hold
    xr = torch.where(scored[:, None], ref[0].reshape(N, D), 0.0)
    tr = torch.where(scored, t.reshape(-1), ignore)
    z = F.linear(xr, ref[1], ref[2])
    if reduction == "none":
        per = torch.where(scored, F.cross_entropy(z, torch.where(scored, t.reshape(-1), 0), reduction="none",
                                                  label_smoothing=smooth), 0.0)
        want = per.reshape(t.shape)
        gi = want_grad.double().reshape(-1) * scored
    else:
        want = F.cross_entropy(z, tr, ignore_index=ignore, reduction=reduction, label_smoothing=smooth)
        n = scored.sum().item()
        gi = scored.double() * want_grad.double() / (max(n, 1) if reduction == "mean" else 1)
    with torch.no_grad():
        xa, wa = xr.abs(), ref[1].abs()
        left_out = 3 * 2.0 ** -22 if dtype == FP32 else 0.0
        least = 2.0 ** -39 if dtype == FP32 else 0.0
        ez = least * (xa.max() * wa.sum(1) + wa.max() * xa.sum(1, keepdim=True))
        ez = ez + ((D + 8) * 2.0 ** -23 + left_out) * (xa @ wa.t()) + (2.0 ** -22 * ref[2].abs() if b is not None else 0.0)
        ez = ez + 2.0 ** -23 * z.abs()
        err = 2 * ez.max(1).values + 2.0 ** -19 * (1 + z.abs().max(1).values)
        loss_err = err * scored
        if reduction == "none":
            bound = loss_err.reshape(t.shape)
        else:
            bound = loss_err.sum() / (max(scored.sum().item(), 1) if reduction == "mean" else 1) + 2.0 ** -23 * want.abs().nan_to_num(0.0)
    diff = (loss.detach().cpu().double() - want.detach()).abs()
    if reduction == "mean" and not scored.any():
        assert torch.isnan(loss.detach().cpu()) and torch.isnan(want)
        grads = [torch.zeros_like(v.double()) for v in (x, w, b) if v is not None]
    else:
        assert (diff <= bound).all(), (diff.max(), bound.max())
        grads = torch.autograd.grad((per * gi).sum() if reduction == "none" else want, [v for v in ref if v is not None],
                                    None if reduction == "none" else want_grad.double())
    with torch.no_grad():
        p = torch.softmax(z, 1)
        goal = torch.full_like(z, smooth / V)
        goal[torch.arange(N), torch.where(scored, t.reshape(-1), 0)] += 1 - smooth
        G = ((p - goal) * gi[:, None]).abs()
        eg = p * gi.abs()[:, None] * (err[:, None] + 2.0 ** -19) + G * {FP32: left_out, BF16: 2.0 ** -8, FP16: 2.0 ** -11}[dtype]
        eg = eg + 2.0 ** -22 * (p + goal) * gi.abs()[:, None]
        if dtype != FP32:
            eg = eg + (2.0 ** -13 * p + 2.0 ** -27) * gi.abs()[:, None]
        if dtype != BF16:  # what is below fp16's steps, scaled by 2^15
            eg = eg + (2.0 ** -25 / 2 ** 15) * gi.abs().max()
        bounds = [eg @ wa + ((V + 8) * 2.0 ** -23 + left_out) * (G @ wa) + least * wa.max() * G.sum(1, keepdim=True),
                  eg.t() @ xa + ((N + 8) * 2.0 ** -23 + left_out) * (G.t() @ xa) + least * xa.max() * G.sum(0)[:, None],
                  eg.sum(0) + 2.0 ** -23 * (N + 8) * G.sum(0)]
        bounds[0] = bounds[0].reshape(x.shape)
    for name, a, r, e, leaf in zip("xwb", got, grads, bounds, used):
        assert a.dtype == dtype and a.shape == leaf.shape
        e = e + HALF[dtype] * (r.abs() + e) + (2.0 ** -25 if dtype == FP16 else 0.0)
        d = (a.cpu().double() - r.reshape(a.shape)).abs()
        assert torch.isfinite(a.cpu()).all(), name
        assert (d <= e.reshape(a.shape) + 1e-40).all(), (name, (d - e.reshape(a.shape)).max(), d.max())
    return loss, got


SIZES = [
    (1, 1, 1), (1, 8, 2), (2, 3, 5), (127, 64, 255), (128, 64, 256), (129, 72, 257), (64, 100, 1000), (33, 513, 129),
    (300, 40, 2500), (1, 2048, 4099), (257, 65, 1025), (700, 200, 300),
    (6, 4104, 8200), (3000, 520, 24), (700, 1713, 70),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", SIZES, ids=["x".join(map(str, s)) for s in SIZES])
def test_sizes(ocl, mode, size, dtype):
    if mode == 0 and dtype != FP32:
        pytest.skip("the math mode is about fp32 operands")
    check(ocl, *make(*size, dtype), mode=mode)


FEW = [(3, 520, 900), (4, 24, 70), (5, 2048, 333), (7, 1, 9), (8, 100, 4100), (8, 4001, 300), (2, 30000, 40), (6, 8, 1)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("size", FEW, ids=["x".join(map(str, s)) for s in FEW])
def test_few_rows(ocl, math_fp32, size, dtype):
    """A token or some, as while serving: with and without gradients, smoothing, bias and rows without a loss."""
    x, w, b, t = make(*size, dtype, bias=True)
    if size[0] > 2:
        t[1] = -100
    check(ocl, x, w, b, t, reduction="none", smooth=0.2, grad=torch.linspace(-1, 1, size[0]))
    loss, _ = check(ocl, x, w, None, t)
    with torch.no_grad():
        again = ocl.functional.linear_cross_entropy(x.to(DEV), w.to(DEV), t.to(DEV))
    assert torch.equal(again.cpu(), loss.detach().cpu())
    wide = torch.cat([w, w.new_zeros(w.shape[0], 3)], 1).to(DEV)[:, :w.shape[1]].detach().requires_grad_()
    check(ocl, x, w, None, t, given=[x.to(DEV).requires_grad_(), wide, None])


def test_many_rows_and_few_classes(ocl, math_fp32):
    """More rows than are joined at once, and K cut because the tiles are few."""
    for dtype in (BF16, FP32):
        check(ocl, *make(20001, 600, 12, dtype, bias=True, ignored=0.3))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smooth", [0.0, 0.1, 1.0])
def test_reductions_smoothing_bias_and_ignored_rows(ocl, dtype, reduction, smooth):
    old = torch.ocl.get_math_mode()
    torch.ocl.set_math_mode(1)
    try:
        x, w, b, t = make(150, 48, 600, dtype, bias=True, ignored=0.3)
        g = torch.Generator().manual_seed(5)
        grad = torch.randn(150, generator=g) * torch.exp(3 * torch.randn(150, generator=g)) if reduction == "none" else torch.tensor(-0.37)
        check(ocl, x, w, b, t, reduction=reduction, smooth=smooth, grad=grad)
    finally:
        torch.ocl.set_math_mode(old)


def test_pieces_of_the_vocabulary(ocl, mode):
    """Enough entries and rows for several pieces and a short last one."""
    check(ocl, *make(1500, 24, 47003, BF16, ignored=0.1))
    check(ocl, *make(9000, 24, 9001, FP16, bias=True, seed=1))
    check(ocl, *make(2100, 24, 12000, FP32, bias=True, seed=2), mode=mode)


def test_more_rows_than_are_joined_at_once(ocl):
    x, w, b, t = make(16400, 16, 300, BF16, ignored=0.2)
    check(ocl, x, w, b, t, reduction="none")


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_rows_without_a_loss_may_hold_anything(ocl, dtype):
    old = torch.ocl.get_math_mode()
    torch.ocl.set_math_mode(1)
    try:
        x, w, b, t = make(200, 40, 500, dtype)
        t[3], t[10], t[199], t[50] = -100, 500, -1, 7
        x[3], x[10] = float("nan"), float("inf")
        check(ocl, x, w, b, t)
        check(ocl, x, w, b, t, reduction="none", grad=torch.linspace(-1, 2, 200))
        t[t == 7] = 499
        check(ocl, x, w, b, t, ignore=499)
        t[:] = -100
        check(ocl, x, w, b, t)
        check(ocl, x, w, b, t, reduction="sum")
    finally:
        torch.ocl.set_math_mode(old)


def test_vocabulary_entries_masked_by_the_bias(ocl, math_fp32):
    """A bias of -inf or of the type's lowest value takes an entry out; a row left with nothing has no finite loss."""
    for dtype in (FP32, BF16):
        x, w, b, t = make(70, 32, 700, dtype, bias=True)
        b[100:600] = float("-inf")
        b[650:] = torch.finfo(dtype).min
        t = torch.where((t >= 100) & (t < 600) | (t >= 650), t % 100, t)
        leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
        loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2], reduction="none")
        got = torch.autograd.grad(loss.sum(), leaves)
        keep = torch.cat([torch.arange(100), torch.arange(600, 650)])
        ref = [v.double().requires_grad_() for v in (x, w[keep], b[keep])]
        where = torch.where(t >= 600, t - 500, t)
        want = F.cross_entropy(F.linear(*ref), where, reduction="none")
        grads = torch.autograd.grad(want.sum(), ref)
        # the sums of the other tests' bounds at these sizes are below these (1e-5 and 2^-6 of the largest value)
        rel = 1e-5 if dtype == FP32 else 2.0 ** -6
        assert (loss.detach().cpu().double() - want.detach()).abs().max() <= 1e-5 * want.max()
        for a, r in zip((got[0].cpu(), got[1].cpu()[keep], got[2].cpu()[keep]), grads):
            assert (a.double() - r).abs().max() <= rel * r.abs().max()
        out = torch.ones(700, dtype=torch.bool)
        out[keep] = False
        assert (got[1].cpu()[out] == 0).all() and (got[2].cpu()[out] == 0).all()
    x, w, b, t = make(5, 16, 300, FP32, bias=True)
    b[:] = float("-inf")
    loss = ocl.functional.linear_cross_entropy(x.to(DEV), w.to(DEV), t.to(DEV), b.to(DEV), reduction="none")
    assert not torch.isfinite(loss.cpu()).any()


def test_extreme_logits(ocl, math_fp32):
    """Logits of +-1e4 (exponentials of either sign out of range), one entry certain."""
    for dtype in (FP32, BF16):
        x, w, b, t = make(64, 32, 400, dtype, scale=1e4)
        check(ocl, x, w, b, t, reduction="none")
        leaves = [v.to(DEV).requires_grad_() for v in (x, w)]
        loss = ocl.functional.linear_cross_entropy(*leaves, t.to(DEV))
        assert all(torch.isfinite(g.cpu()).all() for g in torch.autograd.grad(loss, leaves))


@pytest.mark.parametrize("size", [(150, 72, 520), (20, 1000, 90), (4, 40, 60)], ids=["tiles", "slabs", "few"])
def test_operands_of_extreme_magnitude(ocl, math_fp32, size):
    """fp32 operands whose scales are far from 1, in both directions, and a row far above the others."""
    x, w, b, t = make(*size, FP32, bias=True)
    for s in (1e30, 1e-30):
        check(ocl, x * s, w / s, b, t)
    check(ocl, x * 1e-25, w * 1e-20, b, t, reduction="sum")
    x[1] *= 1e4
    check(ocl, x, w, None, t, reduction="none")
    x[1] = 1e38
    t[1] = -100
    check(ocl, x, w, b, t)


def test_strides_offsets_and_shapes(ocl):
    for dtype in (BF16, FP32):
        x, w, b, t = make(6 * 20, 56, 300, dtype, bias=True)
        x3, t2 = x.view(6, 20, 56), t.view(6, 20)
        check(ocl, x3, w, b, t2)
        check(ocl, x3, w, b, t2, reduction="none")
        for views in (
            lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)]).to(DEV)[1:].view(v.shape),             # odd address
            lambda v: torch.cat([v, v.new_zeros(*v.shape[:-1], 3)], -1).to(DEV)[..., :v.shape[-1]],     # odd row stride
            lambda v: torch.cat([v, v.new_zeros(*v.shape[:-1], 8)], -1).to(DEV)[..., :v.shape[-1]],     # wider rows
            lambda v: v.transpose(0, -1).contiguous().to(DEV).transpose(0, -1),                          # columns first
            lambda v: v.repeat_interleave(2, -1).to(DEV)[..., ::2],                                      # gaps
        ):
            given = [views(v).detach().requires_grad_() for v in (x3, w)] + [b.to(DEV).requires_grad_()]
            check(ocl, x3, w, b, t2, given=given)
        one = x[:1].to(DEV).expand(120, 56).detach().requires_grad_()  # one row for all
        check(ocl, x[:1].expand(120, 56), w, None, t, given=[one, w.to(DEV).requires_grad_(), None])
    x, w, b, t = make(9, 24, 30, BF16)
    check(ocl, x[0], w, b, t[0], reduction="sum")


def test_only_some_gradients(ocl):
    x, w, b, t = make(130, 64, 700, BF16, bias=True)
    full = check(ocl, x, w, b, t)[1]
    for needs in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [v.to(DEV).requires_grad_(bool(n)) for v, n in zip((x, w, b), needs)]
        loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2])
        loss.backward()
        for leaf, n, want in zip(leaves, needs, full):
            assert (leaf.grad is not None) == bool(n)
            if n:
                assert torch.equal(leaf.grad.cpu(), want.cpu())


def test_no_rows(ocl):
    w = torch.randn(10, 8).to(DEV).requires_grad_()
    x = torch.zeros(0, 8).to(DEV).requires_grad_()
    t = torch.zeros(0, dtype=torch.int64).to(DEV)
    loss = ocl.functional.linear_cross_entropy(x, w, t, reduction="sum")
    assert loss.item() == 0
    gx, gw = torch.autograd.grad(loss, [x, w])
    assert gx.shape == (0, 8) and (gw.cpu() == 0).all()
    assert torch.isnan(ocl.functional.linear_cross_entropy(x, w, t).cpu())
    assert ocl.functional.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)


def test_same_results_every_time(ocl):
    x, w, b, t = make(1000, 136, 5000, BF16, bias=True, ignored=0.1)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    runs = []
    for _ in range(3):
        loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], t.to(DEV), leaves[2])
        runs.append([loss.detach().cpu(), *(g.cpu() for g in torch.autograd.grad(loss, leaves))])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_gradient_by_differences(ocl, math_fp32):
    """The loss along a random direction, against the gradient."""
    x, w, b, t = make(40, 30, 90, FP32, bias=True)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    f = lambda *v: ocl.functional.linear_cross_entropy(v[0], v[1], t.to(DEV), v[2], label_smoothing=0.1)
    grads = torch.autograd.grad(f(*leaves), leaves)
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=gen).to(DEV)
        h = 2.0 ** -6
        up, down = ([v.detach() + (h * s) * d if k == i else v.detach() for k, v in enumerate(leaves)] for s in (1, -1))
        slope = (f(*up).double().item() - f(*down).double().item()) / (2 * h)
        want = (grads[i].cpu().double() * d.cpu().double()).sum().item()
        # a loss of about 5 in fp32 errs by 2^-20: 2^-14 of a slope; the cubic term is h^2 of the third derivative,
        # below |d|^3 of a row's logits (a few tens here)
        assert abs(slope - want) <= 2.0 ** -13 + h * h * 30 * (1 + abs(want))


def test_captured_and_replayed(ocl):
    x, w, b, t = make(300, 64, 1100, BF16, bias=True, ignored=0.1)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    td = t.to(DEV)

    def run():
        loss = ocl.functional.linear_cross_entropy(leaves[0], leaves[1], td, leaves[2])
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    run()
    graph, other = torch.ocl.Graph(), torch.ocl.Graph()
    with graph.capture():
        held = run()
    with other.capture():  # a second graph of the same work, with its own memory
        held2 = run()
    x2, _, _, t2 = make(300, 64, 1100, BF16, bias=True, ignored=0.3, seed=9)
    for xx, tt in ((x, t), (x2, t2)):
        with torch.no_grad():
            leaves[0].copy_(xx)
        td.copy_(tt)
        graph.replay()
        other.replay()
        got, got2 = [v.cpu() for v in held], [v.cpu() for v in held2]
        want = [v.cpu() for v in run()]
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, got2))
    graph.reset()
    other.reset()


def test_on_another_stream(ocl):
    x, w, b, t = make(500, 64, 1500, BF16)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w)]
    td = t.to(DEV)
    f = lambda: ocl.functional.linear_cross_entropy(*leaves, td)
    want = [v.cpu() for v in torch.autograd.grad(f(), leaves)]
    torch.ocl.synchronize()
    stream = torch.Stream(device=DEV)
    with stream:
        got = torch.autograd.grad(f(), leaves)
    stream.synchronize()
    assert all(torch.equal(a, b.cpu()) for a, b in zip(want, got))


def test_memory_stays_bounded(ocl, monkeypatch):
    """No logits: a step that keeps nothing takes far less than N x V numbers beyond its operands and gradients."""
    N, D, V = 4096, 64, 131072
    monkeypatch.setenv("B200_CE_KEEP_MB", "0")
    x, w = torch.zeros(N, D, dtype=BF16).to(DEV).requires_grad_(), torch.zeros(V, D, dtype=BF16).to(DEV).requires_grad_()
    t = torch.zeros(N, dtype=torch.int64).to(DEV)
    torch.ocl.synchronize()
    torch.ocl.reset_peak_memory_stats()
    before = torch.ocl.memory_allocated()
    torch.autograd.grad(ocl.functional.linear_cross_entropy(x, w, t), [x, w])
    assert torch.ocl.max_memory_allocated() - before < N * V * 2 // 4


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("keep", ["0", "5", "2048"])
def test_kept_softmax(ocl, monkeypatch, math_fp32, dtype, keep):
    """Nothing, some, and all of the softmax kept for the backward pass; and a second backward pass of the same graph."""
    monkeypatch.setenv("B200_CE_KEEP_MB", keep)
    check(ocl, *make(700, 40, 9001, dtype, bias=True, ignored=0.1), smooth=0.1)
    check(ocl, *make(30, 520, 900, dtype, bias=True, ignored=0.1), reduction="none")
    check(ocl, *make(17000, 16, 1100, dtype))
    x, w, b, t = make(500, 64, 5000, dtype)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w)]
    loss = ocl.functional.linear_cross_entropy(*leaves, t.to(DEV))
    one = torch.autograd.grad(loss, leaves, retain_graph=True)
    two = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(one, two))


def test_what_is_kept_stays_in_its_budget(ocl, monkeypatch):
    N, D, V = 4096, 64, 65536
    monkeypatch.setenv("B200_CE_KEEP_MB", "100")
    x, w = torch.zeros(N, D, dtype=BF16).to(DEV).requires_grad_(), torch.zeros(V, D, dtype=BF16).to(DEV)
    t = torch.zeros(N, dtype=torch.int64).to(DEV)
    torch.ocl.synchronize()
    before = torch.ocl.memory_allocated()
    loss = ocl.functional.linear_cross_entropy(x, w, t)
    held = torch.ocl.memory_allocated() - before
    # the budget, the allocator's size class above it (a quarter), and what belongs to each row
    assert 50 << 20 < held <= 1.25 * (100 << 20) + (1 << 20)
    with torch.no_grad():
        before = torch.ocl.memory_allocated()
        kept_nothing = ocl.functional.linear_cross_entropy(x, w, t)
        assert torch.ocl.memory_allocated() - before < 1 << 20
    assert torch.equal(loss.detach().cpu(), kept_nothing.cpu())


def test_two_streams_at_once(ocl):
    """Calls that overlap on the device share nothing."""
    x, w, b, t = make(2000, 128, 6000, BF16)
    x2, _, _, t2 = make(2000, 128, 6000, BF16, seed=3)
    leaves, other = ([v.to(DEV).requires_grad_() for v in p] for p in ((x, w), (x2, w)))
    td, td2 = t.to(DEV), t2.to(DEV)
    f = lambda v, tt: torch.autograd.grad(ocl.functional.linear_cross_entropy(*v, tt), v)
    want, want2 = [g.cpu() for g in f(leaves, td)], [g.cpu() for g in f(other, td2)]
    torch.ocl.synchronize()
    streams = [torch.Stream(device=DEV) for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, (v, tt) in enumerate(((leaves, td), (other, td2))):
            with streams[k]:
                got[k] = f(v, tt)
    torch.ocl.synchronize()
    assert all(torch.equal(a, g.cpu()) for a, g in zip(want + want2, got[0] + got[1]))


def test_no_wait_ran_out(ocl):
    import ctypes
    import os

    lib = ctypes.CDLL(os.path.join(os.path.dirname(ocl.__file__), "lib", "libpvb2.so"))
    x, w, b, t = make(100, 64, 700, BF16)
    check(ocl, x, w, b, t)
    flag = ctypes.c_int(-1)
    assert lib.pvb2_linear_ce_status(ctypes.byref(flag), 0) == 0 and flag.value == 0


def test_refusals(ocl):
    f = ocl.functional.linear_cross_entropy
    x, w, t = torch.zeros(4, 8).to(DEV), torch.zeros(5, 8).to(DEV), torch.zeros(4, dtype=torch.int64).to(DEV)
    b = torch.zeros(5).to(DEV)
    for args, kw, match in [
        ((x.to(BF16), w, t), {}, "one type"),
        ((x.to(torch.int32), w.to(torch.int32), t), {}, "one type"),
        ((x[:, :7], w, t), {}, "features"),
        ((x, w[0], t), {}, "features"),
        ((x, w[:0], t), {}, "no classes"),
        ((x, w, t[:3]), {}, "target"),
        ((x, w, t.to(torch.int32)), {}, "target"),
        ((x, w, t, b[:4]), {}, "bias"),
        ((x, w, t, b.to(BF16)), {}, "bias"),
        ((x, w, t, b), dict(label_smoothing=1.5), "label smoothing"),
        ((x, w, t.cpu()), {}, "on ocl expected"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)
    with pytest.raises(ValueError, match="reduction"):
        f(x, w, t, reduction="max")
    wr = w.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(f(x, wr, t), wr, create_graph=True)
