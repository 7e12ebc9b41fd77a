"""Log probabilities of given tokens, entropy, alternatives and gradients on
`ocl` against float64.

u = 2^-24 is half a step of fp32.  An exponential of z - m carries 3 u |z - m|
and a few u; the sum of V of them over 512 threads V / 512 + 40 additions.  The
exponentials' errors weigh with p, so that |z - m| counts by its mean, which is
at most the entropy, and by its square's mean in the entropy's own sum.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
U = 2.0 ** -24


def make(N, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + N + 3 * V)
    z = torch.randn(N, V, generator=g) * (1 + 3 * torch.rand(N, 1, generator=g))
    t = torch.randint(0, V, (N,), generator=g)
    z[torch.arange(0, N, 2), t[::2]] += 12
    if N > 2:
        t[1], t[2] = -100, V
    return z.to(dtype), t, torch.randn(N, generator=g), torch.randn(N, generator=g)


class Reference:
    def __init__(self, z, t, skip_empty=False):
        z = z.double()
        self.V = z.shape[1]
        self.scored = (t >= 0) & (t < self.V)
        self.at = t.clamp(0, self.V - 1)
        m = z.amax(1, keepdim=True)
        self.empty = (m == float("-inf"))[:, 0]
        d = z - torch.where(m == float("-inf"), 0.0, m)
        e = d.exp()
        s = e.sum(1, keepdim=True).clamp(min=1e-300)
        self.logp = d - s.log()
        self.p = e / s
        mean = lambda v: torch.where(self.p > 0, self.p * v, 0.0).sum(1)  # noqa: E731
        self.H = mean(-self.logp)
        lp = self.logp.gather(1, self.at[:, None])[:, 0]
        self.lp = torch.where(self.scored, torch.where(self.empty, float("-inf"), lp), 0.0)
        base = (self.V / 256 + 90) * U
        self.bound_lse = base + 5 * U * self.H
        self.bound_H = base * (1 + self.H) + 5 * U * mean(d * d)

    def bound_lp(self, lp):
        return self.bound_lse.view(-1, *[1] * (lp.dim() - 1)) + 3 * U * lp.abs()

    def gradient(self, g, k):
        g = torch.where(self.scored, g.double(), 0.0)[:, None]
        k = k.double()[:, None]
        logp = self.logp.clamp(min=-1e300)
        want = -self.p * (g + k * (logp + self.H[:, None]))
        size = self.p * (g.abs() + k.abs() * (logp.abs() + self.H[:, None]))
        bound = size * ((self.V / 256 + 100) * U + 6 * U * (logp.abs() + self.H[:, None]))
        bound = bound + self.p * k.abs() * (self.bound_H + self.bound_lse)[:, None]
        one = torch.zeros_like(want).scatter_(1, self.at[:, None], 1.0) * g
        want = want + one
        # exponentials below fp32's normal numbers are 0
        return torch.where(self.empty[:, None], 0.0, want), bound + 2 * U * one.abs() + 2.0 ** -126 * (g.abs() + 200 * k.abs())


def near(got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape
    same = (got == want)
    assert (same | ((got - want).abs() <= bound)).all(), ((got - want).abs() / bound)[~same].max()


def best(z, top):
    """By falling logit, equal ones by their places."""
    order = torch.sort(z.float() + 0.0, dim=1, descending=True, stable=True).indices
    return order[:, :top]


SHAPES = [(1, 1), (1, 10), (3, 7), (5, 129), (2, 4096), (4, 5003), (1, 32768), (9, 50001), (1, 200003), (300, 1000), (700, 33)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_values_and_gradient(ocl, shape, dtype):
    z, t, g, k = make(*shape, dtype)
    zd = z.to(DEV).requires_grad_()
    lp, H = ocl.functional.token_log_probs(zd, t.to(DEV))
    ref = Reference(z, t)
    assert lp.dtype == H.dtype == torch.float32
    near(lp.detach(), ref.lp, ref.bound_lp(ref.lp))
    near(H.detach(), ref.H, ref.bound_H)
    (dz,) = torch.autograd.grad([lp, H], zd, [g.to(DEV), k.to(DEV)])
    want, bound = ref.gradient(g, k)
    assert dz.dtype == dtype
    eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
    near(dz, want, bound + eps * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0))
    for top in sorted({1, min(5, shape[1]), min(20, shape[1]), min(32, shape[1])}):
        with torch.no_grad():
            lp2, H2, tlp, tat = ocl.functional.token_log_probs(zd, t.to(DEV), top=top)
        assert torch.equal(lp2.cpu(), lp.detach().cpu()) and torch.equal(H2.cpu(), H.detach().cpu())
        at = best(z, top)
        assert tat.dtype == torch.int64 and torch.equal(tat.cpu(), at)
        want = ref.logp.gather(1, at)
        near(tlp, want, ref.bound_lp(want))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [40, 1000, 33333])
def test_equal_falling_and_rising_logits(ocl, dtype, V):
    """Ties go to the lower place, also between zeros of both signs; orders that keep every list busy."""
    g = torch.Generator().manual_seed(V)
    rows = [torch.zeros(V), torch.arange(V) * (50.0 / V), -torch.arange(V) * (50.0 / V), torch.randint(0, 3, (V,), generator=g).float(),
            torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0), torch.full((V,), torch.finfo(dtype).min),
            torch.where(torch.arange(V) == V - 1, 1.0, float(torch.finfo(dtype).min)),
            torch.full((V,), torch.finfo(dtype).max), torch.where(torch.arange(V) % 7 == 5, -1.0, float("-inf"))]
    z = torch.stack(rows).to(dtype)
    t = torch.full((len(rows),), V - 1)
    ref = Reference(z, t)
    for top in (1, 7, 32):
        lp, H, tlp, tat = ocl.functional.token_log_probs(z.to(DEV), t.to(DEV), top=top)
        at = best(z, top)
        assert torch.equal(tat.cpu(), at)
        near(lp, ref.lp, ref.bound_lp(ref.lp))
        near(H, ref.H, ref.bound_H)
        want = ref.logp.gather(1, at)
        near(tlp, want, ref.bound_lp(want))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [5, 1000, 70001])
def test_far_from_zero(ocl, dtype, V):
    """Rows of logits of one magnitude, alike or a step or more apart, of either sign, and what a finite mask leaves."""
    g = torch.Generator().manual_seed(V)
    most = float(torch.finfo(dtype).max)
    rows = []
    for size in (1e3, 6e4, 1e6, 1e8, 1e9, 3e9, 1e10, 2e10, 1e15, 1e20, 1e30, 1e38, 2e38):
        for sign in (-1, 1):
            v = sign * min(size, most)
            near_it = v * (1 + torch.randint(0, 3, (V,), generator=g) * 2.0 ** -20).clamp(max=most / abs(v))
            rows += [torch.full((V,), v), near_it, torch.where(torch.arange(V) % 5 == 3, torch.randn(V, generator=g), -abs(v))]
    z = torch.stack(rows).to(dtype)
    t = torch.randint(0, V, (len(rows),), generator=g)
    gl, gh = torch.randn(len(rows), generator=g), torch.randn(len(rows), generator=g)
    zd = z.to(DEV).requires_grad_()
    lp, H = ocl.functional.token_log_probs(zd, t.to(DEV))
    ref = Reference(z, t)
    near(lp.detach(), ref.lp, ref.bound_lp(ref.lp))
    near(H.detach(), ref.H, ref.bound_H)
    (dz,) = torch.autograd.grad([lp, H], zd, [gl.to(DEV), gh.to(DEV)])
    want, bound = ref.gradient(gl, gh)
    eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
    bound = torch.where(ref.p > 0, bound, 2.0 ** -126 * 300)  # (log p of -1e38 times p of 0)
    near(dz, want, bound + eps * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_masks(ocl, dtype):
    """-inf has no probability and no gradient, a row of nothing else none at all; NaN and +inf spoil their own row."""
    V = 777
    z, t, g, k = make(8, V, dtype, seed=2)
    t[:] = torch.tensor([0, 5, V - 1, 3, -100, 9, 10, 11])
    z[0, 1:] = float("-inf")           # one token is certain
    z[1, ::2] = float("-inf")
    z[2] = float("-inf")               # nothing is left
    z[4] = float("-inf")               # and no token is asked for
    z[3, 3] = float("-inf")            # the token itself is masked
    zd = z.to(DEV).requires_grad_()
    lp, H = ocl.functional.token_log_probs(zd, t.to(DEV))
    ref = Reference(z, t)
    assert lp[0].item() == 0 and H[0].item() == 0 and lp[2].item() == float("-inf") and H[2].item() == 0
    assert lp[4].item() == 0 and lp[3].item() == float("-inf")
    near(lp.detach(), ref.lp, ref.bound_lp(ref.lp.clamp(min=-1e9)))
    near(H.detach(), ref.H, ref.bound_H)
    (dz,) = torch.autograd.grad([lp, H], zd, [g.to(DEV), k.to(DEV)])
    assert torch.isfinite(dz.cpu()).all() and (dz[2].cpu() == 0).all() and (dz[4].cpu() == 0).all()
    hidden = z == float("-inf")
    hidden[3, 3] = False
    assert (dz.cpu()[hidden] == 0).all()
    want, bound = ref.gradient(g, k)
    eps = torch.finfo(dtype).eps / 2
    near(dz, want, bound + eps * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0))
    _, _, tlp, tat = ocl.functional.token_log_probs(zd.detach(), t.to(DEV), top=3)
    assert torch.equal(tat.cpu(), best(z, 3)) and (tlp[2].cpu() == float("-inf")).all()
    z[5, 700], z[6, 20] = float("nan"), float("inf")
    lp, H, tlp, tat = ocl.functional.token_log_probs(z.to(DEV), t.to(DEV), top=3)
    for row in (5, 6):
        assert lp[row].isnan() and H[row].isnan()
    near(lp[:5], ref.lp[:5], ref.bound_lp(ref.lp.clamp(min=-1e9))[:5])
    assert ((tat.cpu() >= 0) & (tat.cpu() < V)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_layouts_and_what_is_asked_for(ocl, dtype):
    """Rows that begin anywhere, transposed logits, more dimensions, no rows; one gradient of the two, one number for all."""
    z, t, g, k = make(12, 1003, dtype, seed=4)
    f = ocl.functional.token_log_probs
    zd, td = z.to(DEV), t.to(DEV)
    ref = Reference(z[:, 5:900], t.clamp(max=800))
    for view in (zd[:, 5:900], zd[:, 5:900].clone(), z.t().contiguous().to(DEV).t()[:, 5:900], zd.view(3, 4, 1003)[..., 5:900]):
        leaf = view.detach().requires_grad_()
        lp, H, tlp, tat = f(leaf, t.clamp(max=800).to(DEV).view(view.shape[:-1]), top=4)
        near(lp.detach().view(12), ref.lp, ref.bound_lp(ref.lp))
        assert torch.equal(tat.cpu().view(12, 4), best(z[:, 5:900], 4))
        eps = torch.finfo(dtype).eps / 2
        for outs, gg, kk in (([lp.sum()], torch.ones(12), torch.zeros(12)), ([H.mean()], torch.zeros(12), torch.full((12,), 1 / 12)),
                             ([lp.sum() + H.sum()], torch.ones(12), torch.ones(12))):
            (dz,) = torch.autograd.grad(outs, leaf, retain_graph=True)
            want, bound = ref.gradient(gg, kk)
            assert dz.shape == leaf.shape
            near(dz.reshape(12, 895), want, bound + eps * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0))
    assert not tlp.requires_grad
    one = f(zd[0], td[0], top=2)
    assert one[0].shape == () and one[2].shape == (2,)
    none = f(zd[:0], td[:0], top=2)
    assert none[0].shape == (0,) and none[3].shape == (0, 2)
    empty = zd[:0].detach().requires_grad_()
    assert torch.autograd.grad(f(empty, td[:0])[0].sum(), empty)[0].shape == (0, 1003)
    leaf = zd.float().detach().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(f(leaf, td)[0].sum(), leaf, create_graph=True)


def test_gradient_against_differences(ocl):
    z, t, g, k = make(3, 50, torch.float32, seed=6)
    zd = z.to(DEV).requires_grad_()
    (dz,) = torch.autograd.grad(ocl.functional.token_log_probs(zd, t.to(DEV)), zd, [g.to(DEV), k.to(DEV)])

    def value(z):
        logp = torch.log_softmax(z, 1)
        lp = torch.where((t >= 0) & (t < 50), logp.gather(1, t.clamp(0, 49)[:, None])[:, 0], 0.0)
        return (lp * g + -(logp.exp() * logp).sum(1) * k).sum().item()

    # central differences in float64 with a step of 1e-5: off by about 1e-10 and 1e-11 of the value
    for i in range(0, 150, 7):
        e = torch.zeros(150, dtype=torch.float64)
        e[i] = 1e-5
        d = (value(z.double() + e.view(3, 50)) - value(z.double() - e.view(3, 50))) / 2e-5
        assert abs(d - dz.cpu().view(-1)[i].item()) < 2e-5


def test_refusals(ocl):
    f = ocl.functional.token_log_probs
    z, t = torch.zeros(4, 20, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad in (lambda: f(z, t.int()), lambda: f(z, t[:3]), lambda: f(z.long(), t), lambda: f(z, t, top=33), lambda: f(z, t, top=21),
                lambda: f(z, t, top=-1), lambda: f(z, t.cpu()), lambda: f(z[:, :0], t), lambda: f(z.sum(), t.sum())):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(Exception):
        f(fwd.make_dual(z, torch.ones_like(z)), t)


def test_captured(ocl):
    """Two captured graphs replayed in turn: the same bits as eager."""
    z, t, g, k = (x.to(DEV) for x in make(20, 30001, torch.bfloat16))
    z.requires_grad_()

    def step():
        out = ocl.functional.token_log_probs(z, t, top=5)
        return [v.detach() for v in out] + list(torch.autograd.grad(out[:2], z, [g, k]))

    eager = [v.cpu() for v in step()]
    held = []
    for _ in range(2):
        graph = torch.ocl.Graph()
        with graph.capture():
            out = step()
        held.append((graph, out))
    for graph, out in held * 2:
        for v in out:
            v.zero_()
        graph.replay()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out, eager))


@pytest.mark.parametrize("V", [40, 3000, 50003, 131072])
@pytest.mark.parametrize("rows", [1, 200])
def test_few_tokens_are_left(ocl, V, rows):
    """A mask that leaves fewer tokens than alternatives are asked for: these, and then hidden ones by their places."""
    g = torch.Generator().manual_seed(V)
    for left in (0, 1, 3, 19, 20, 33):
        z = torch.full((rows, V), float("-inf"))
        for r in range(rows):
            z[r, torch.randperm(V, generator=g)[:left]] = torch.randn(left, generator=g)
        z = z.to(torch.bfloat16)
        t = torch.zeros(rows, dtype=torch.int64)
        _, _, tlp, tat = ocl.functional.token_log_probs(z.to(DEV), t.to(DEV), top=20)
        at = best(z, 20)
        assert torch.equal(tat.cpu(), at)
        ref = Reference(z, t)
        want = torch.where(ref.empty[:, None], float("-inf"), ref.logp.gather(1, at))
        near(tlp, want, ref.bound_lp(want.clamp(min=-1e9)))
