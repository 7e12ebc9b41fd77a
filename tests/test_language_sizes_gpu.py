"""Sizes at which the language model's kernels run their loops in their steady state: rings whose slots are filled again,
scales that are read in several runs, rows of a whole block, groups of tiles of which the last is narrower.

Tolerances as in the operators' own tests: u = 2^-24 is half a step of fp32.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def near(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off / bound).max()


class Rows:
    """Some rows' log probabilities and gradients in float64, with their tolerances (3 u |z - m| an exponential, V / 256
    + 90 additions)."""

    def __init__(self, z, t):
        z = z.double()
        self.t, self.V = t, z.shape[1]
        self.logp = torch.log_softmax(z, 1)
        self.p = self.logp.exp()
        self.H = -(self.p * self.logp).sum(1)
        self.lp = self.logp.gather(1, t[:, None])[:, 0]
        base = (self.V / 256 + 90) * U
        d = z - z.amax(1, keepdim=True)
        self.bound_lse = base + 5 * U * self.H
        self.bound_H = base * (1 + self.H) + 5 * U * (self.p * d * d).sum(1)

    def gradient(self, g, k):
        g, k = g.double()[:, None], k.double()[:, None]
        away = self.logp + self.H[:, None]
        want = -self.p * (g + k * away)
        size = self.p * (g.abs() + k.abs() * (self.logp.abs() + self.H[:, None]))
        bound = size * ((self.V / 256 + 100) * U + 6 * U * (self.logp.abs() + self.H[:, None]))
        bound = bound + self.p * k.abs() * (self.bound_H + self.bound_lse)[:, None]
        one = torch.zeros_like(want).scatter_(1, self.t[:, None], 1.0) * g
        return want + one, bound + 2 * U * one.abs() + 2.0 ** -126 * (g.abs() + 200 * k.abs())


def logits(N, V, dtype):
    g = torch.Generator().manual_seed(N + V)
    z = (torch.randn(N, V, generator=g) * (1 + 3 * torch.rand(N, 1, generator=g))).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    some = torch.randperm(N, generator=g)[:24]
    return z, t, torch.randn(N, generator=g), torch.randn(N, generator=g), some


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [20000, 20001, 66003])
@pytest.mark.parametrize("apart", [0, 5], ids=["alike", "otherwise"])
def test_gradient_of_many_long_rows(ocl, dtype, V, apart):
    """Ten and more chunks a thread; with gaps between the rows, logits and gradient lie differently."""
    N = 750
    z, t, g, k, some = logits(N, V, dtype)
    zd = torch.nn.functional.pad(z, (0, apart)).to(DEV)[:, :V].detach().requires_grad_()
    out = ocl.functional.token_log_probs(zd, t.to(DEV))
    (dz,) = torch.autograd.grad(out, zd, [g.to(DEV), k.to(DEV)])
    want, bound = Rows(z[some], t[some]).gradient(g[some], k[some])
    eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
    near(dz.cpu()[some], want, bound + eps * (want.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [148, 301])
@pytest.mark.parametrize("V", [6001, 12001, 50001, 90001])
def test_rows_of_a_block(ocl, dtype, N, V):
    """As many rows as there are SMs and more, each a block's of 128 or 256 threads."""
    z, t, _, _, some = logits(N, V, dtype)
    ref = Rows(z[some], t[some])
    zd, td = z.to(DEV), t.to(DEV)
    plain = ocl.functional.token_log_probs(zd, td)
    near(plain[0].cpu()[some], ref.lp, ref.bound_lse + 3 * U * ref.lp.abs())
    near(plain[1].cpu()[some], ref.H, ref.bound_H)
    order = torch.sort(z[some], dim=1, descending=True, stable=True).indices
    for top in (1, 20):
        lp, H, tlp, tat = ocl.functional.token_log_probs(zd, td, top=top)
        assert torch.equal(tat.cpu()[some], order[:, :top])
        want = ref.logp.gather(1, order[:, :top])
        near(tlp.cpu()[some], want, ref.bound_lse[:, None] + 3 * U * want.abs())
        near(lp.cpu()[some], ref.lp, ref.bound_lse + 3 * U * ref.lp.abs())


def operands(M, N, K):
    g = torch.Generator().manual_seed(M + 3 * N + 5 * K)
    blocks = (K + 127) // 128

    def codes(rows):
        c = torch.randint(0, 256, (rows, K), generator=g, dtype=torch.uint8)
        c[(c & 127) == 127] = 0  # the two NaNs
        return c

    return (codes(M), torch.exp(torch.randn(M, blocks, generator=g)) * 1e-2, codes(N),
            torch.exp(torch.randn((N + 127) // 128, blocks, generator=g)) * 1e-3, g)


def layer_check(y, ops, rows, outputs):
    xc, xs, wc, ws = ops[:4]
    K, blocks = xc.shape[1], xs.shape[1]
    x = xc[rows].view(torch.float8_e4m3fn).double() * xs[rows].double().repeat_interleave(128, 1)[:, :K]
    w = wc[outputs].view(torch.float8_e4m3fn).double() * ws[outputs // 128].double().repeat_interleave(128, 1)[:, :K]
    near(y.cpu()[rows][:, outputs], x @ w.t(), 2 * (128 + blocks + 4) * U * (x.abs() @ w.abs().t()))


@pytest.mark.parametrize("M", [1, 20, 50, 100])
@pytest.mark.parametrize("size", [(9600, 4500), (9501, 8500), (128, 40000)], ids=["two-runs", "three-runs", "split"])
def test_layer_of_many_blocks_a_cta(ocl, M, size):
    """More K blocks than a run of scales and than the ring of each tile width."""
    ops = operands(M, *size)
    y = ocl.functional.linear_8bit(*(t.to(DEV) for t in ops[:4]), dtype=torch.float32)
    outputs = torch.cat([torch.randperm(size[0], generator=ops[4])[:100], torch.tensor([0, size[0] - 1])])
    layer_check(y, ops, torch.arange(M), outputs)


@pytest.mark.parametrize("M", [2305, 2304 + 15 * 128 + 1])
def test_layer_with_a_narrow_last_group(ocl, M):
    """Rows' tiles go by in groups of eight, the last one of two or of one, partly empty."""
    ops = operands(M, 1301, 16400)
    y = ocl.functional.linear_8bit(*(t.to(DEV) for t in ops[:4]), dtype=torch.float32)
    rows = torch.cat([torch.randperm(M, generator=ops[4])[:60], torch.arange(2040, 2060), torch.arange(M - 20, M)])
    outputs = torch.cat([torch.randperm(1301, generator=ops[4])[:200], torch.tensor([255, 256, 1279, 1280, 1300])])
    layer_check(y, ops, rows, outputs)
    seen = y.cpu()
    assert seen.isfinite().all() and (seen != 0).all(1).any() and ((seen != 0).sum(1) > 1200).all()
