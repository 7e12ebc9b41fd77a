"""RMS norm with the residual's addition, its gradients and its 8-bit output on
`ocl`, against the formulas in float64.

u = 2^-24 is half a step of fp32.  Forward: the mean of squares, the sum with
eps, the root and the quotient round once each (the root halves what comes
before), the two products once: at most 5 u of y, then half a step of the type.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
U = 2.0 ** -24
# the smallest step of a type: half of it is a rounding's absolute part
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def rounding(want, dtype):
    return (torch.finfo(dtype).eps / 2 * want.abs() if dtype != torch.float32 else 0 * want) + TINY[dtype]


def make(rows, D, dtype, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed + 7 * rows + D)
    size = torch.exp(torch.randn(rows, 1, generator=g))
    x = (torch.randn(rows, D, generator=g) * size).to(dtype)
    r = torch.randn(rows, D, generator=g).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    gy, gs = torch.randn(rows, D, generator=g).to(dtype), torch.randn(rows, D, generator=g).to(dtype)
    return x, r, w, gy, gs


def summed(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def close(got, want, bound):
    assert got.shape == want.shape
    off = (got.double().cpu() - want).abs() - bound
    assert (off <= 0).all(), off.max()


def check_forward(y, h, w, eps):
    h64 = h.double()
    want = h64 / (h64.square().mean(-1, keepdim=True) + eps).sqrt() * (1 if w is None else w.double())
    close(y, want, 6 * U * want.abs() + rounding(want, h.dtype) * (1 + 6 * U))


def reference_gradients(h, w, gy, gs, eps):
    h, gy = h.double(), gy.double()
    D, rows = h.shape[1], h.shape[0]
    rstd = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    n, a = h * rstd, gy * (1 if w is None else w.double())
    mean = (a * n).mean(1, keepdim=True)
    dx = (a - n * mean) * rstd
    # the dot product's sum: at most D / 1024 + 100 additions one after the other; the other roundings, 8 of either term
    off = (D / 1024 + 110) * U * (a * n).abs().mean(1, keepdim=True)
    bound = rstd * (n.abs() * off + 10 * U * (a.abs() + (n * mean).abs()))
    if gs is not None:
        dx = dx + gs.double()
        bound = bound + 2 * U * (gs.double().abs() + dx.abs())
    dw = (gy * n).sum(0)
    return dx, bound, dw, (rows + 50) * U * (gy * n).abs().sum(0)


SHAPES = [(1, 1), (3, 7), (1, 4096), (5, 64), (2, 128), (33, 129), (130, 768), (65, 1000), (9, 1024), (7, 2047), (17, 2048),
          (4, 5000), (3, 8191), (3, 8192), (2, 16384), (2, 16385), (2, 32768), (1, 40000), (1200, 40), (700, 257)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
def test_values_and_gradients(ocl, shape, dtype, residual):
    x, r, w, gy, gs = make(*shape, dtype, residual=residual)
    leaves = [t.to(DEV).requires_grad_() for t in (x, r, w) if t is not None]
    xd, wd, rd = leaves[0], leaves[-1], leaves[1] if residual else None
    out = ocl.functional.rms_norm(xd, wd, rd, eps=1e-5)
    h = summed(x, r)
    if residual:
        y, s = out
        assert torch.equal(s.detach().cpu(), h)
    else:
        y = out
    assert y.dtype == dtype
    check_forward(y.detach(), h, w, 1e-5)
    with torch.no_grad():
        again = ocl.functional.rms_norm(xd, wd, rd, eps=1e-5)
        assert torch.equal((again[0] if residual else again).cpu(), y.detach().cpu())
    grads = torch.autograd.grad(list(out) if residual else [y], leaves, [gy.to(DEV)] + ([gs.to(DEV)] if residual else []))
    dx, bx, dw, bw = reference_gradients(h, w, gy, gs if residual else None, 1e-5)
    close(grads[0], dx, bx + rounding(dx, dtype) + torch.finfo(dtype).eps * bx)
    close(grads[-1], dw, bw + rounding(dw, dtype) + torch.finfo(dtype).eps * bw)
    if residual:
        assert torch.equal(grads[0].cpu(), grads[1].cpu())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_strides_orders_and_no_weight(ocl, dtype):
    """Rows apart, rows that begin off 16-byte boundaries, transposed and expanded inputs, more dimensions, no weight."""
    g = torch.Generator().manual_seed(1)
    base = torch.randn(6, 5, 300, generator=g).to(dtype)
    bd = base.to(DEV)
    f = ocl.functional.rms_norm
    w = torch.randn(128, generator=g).to(dtype)
    for view in (lambda t: t[:, :, 16:144], lambda t: t[:, :, 3:131], lambda t: t[1:, ::2, :128],
                 lambda t: t[:, 1:2, 5:133].expand(6, 9, 128), lambda t: t[0, 0, :128], lambda t: t[:, :, :128].transpose(0, 1)):
        for weight in (None, w):
            h = view(base)
            y = f(view(bd), None if weight is None else weight.to(DEV), eps=1e-6)
            check_forward(y, h.reshape(-1, 128), weight, 1e-6) if h.dim() == 2 else check_forward(y, h, weight, 1e-6)
    t = base[:, 0, :6]
    check_forward(f(t.to(DEV).t(), eps=1e-6), t.t(), None, 1e-6)
    # the second term laid out in another way than the first; upstream gradients of a sum
    a, b = base[:, 0, :128], base[:, :, 3:131].transpose(0, 1)[0]
    ad, bdd = bd[:, 0, :128].detach().requires_grad_(), bd[:, :, 3:131].transpose(0, 1)[0].detach().requires_grad_()
    y, s = f(ad, w.to(DEV), bdd)
    assert torch.equal(s.detach().cpu(), summed(a, b))
    (y.float().sum() + s.float().sum()).backward()
    dx, bound, _, _ = reference_gradients(summed(a, b), w, torch.ones(6, 128), torch.ones(6, 128), 1e-6)
    for got in (ad.grad, bdd.grad):
        close(got, dx, bound + rounding(dx, dtype) + torch.finfo(dtype).eps * bound)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 2051), (300, 1025), (2500, 2057), (9, 5001), (1210, 4099), (5, 12289), (3, 16375), (2, 16377)],
                         ids=lambda s: "-".join(map(str, s)))
def test_rows_between_boundaries(ocl, shape, dtype):
    """Odd lengths: rows that begin anywhere, operands that begin alike and not, more rows than blocks; what lies between
    the rows is not written."""
    rows, D = shape
    x, r, w, gy, gs = make(rows, D, dtype)
    f = ocl.functional.rms_norm
    h = summed(x, r)
    dx, bx, dw, bw = reference_gradients(h, w, gy, gs, 1e-6)
    for wide, at in ((D, 0), (D + 8, 8), (D + 16, 3), (D + 3, 0)):
        back = torch.full((rows, wide), float("nan"), dtype=dtype)
        back[:, at:at + D] = x
        xd = back.to(DEV)[:, at:at + D].detach().requires_grad_()
        rd, wd = r.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        y, s = f(xd, wd, rd, eps=1e-6)
        assert torch.equal(s.detach().cpu(), h)
        check_forward(y.detach(), h, w, 1e-6)
        torch.autograd.backward([y, s], [gy.to(DEV), gs.to(DEV)])
        for got, want, bound in ((xd.grad, dx, bx), (rd.grad, dx, bx), (wd.grad, dw, bw)):
            close(got, want, bound + rounding(want, dtype) + torch.finfo(dtype).eps * bound)
    # a weight that begins between boundaries
    wide = torch.cat([torch.ones(1, dtype=dtype), w]).to(DEV)
    check_forward(f(x.to(DEV), wide[1:], eps=1e-6), x, w, 1e-6)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_what_is_asked_for(ocl, dtype):
    """Only some gradients; only the sum used; a leaf that is both terms; backward twice over a kept graph."""
    x, r, w, gy, gs = make(40, 257, dtype)
    xd, rd, wd = (t.to(DEV) for t in (x, r, w))
    dx, bx, dw, bw = reference_gradients(summed(x, r), w, gy, None, 1e-6)
    for which in range(3):
        leaves = [xd.detach(), rd.detach(), wd.detach()]
        leaves[which].requires_grad_()
        y, _ = ocl.functional.rms_norm(leaves[0], leaves[2], leaves[1])
        (got,) = torch.autograd.grad(y, leaves[which], gy.to(DEV))
        want, bound = (dw, bw) if which == 2 else (dx, bx)
        close(got, want, bound + rounding(want, dtype) + torch.finfo(dtype).eps * bound)
    a = xd.detach().requires_grad_()
    _, s = ocl.functional.rms_norm(a, wd, rd)
    (got,) = torch.autograd.grad(s, a, gs.to(DEV))
    assert torch.equal(got.cpu(), gs)
    y, s = ocl.functional.rms_norm(a, wd, a)
    assert torch.equal(s.detach().cpu(), summed(x, x))
    y.backward(gy.to(DEV), retain_graph=True)
    first = a.grad.cpu()
    a.grad = None
    y.backward(gy.to(DEV))
    assert torch.equal(a.grad.cpu(), first)
    with pytest.raises(RuntimeError, match="differentiated again"):
        b = xd.float().detach().requires_grad_()
        torch.autograd.grad(ocl.functional.rms_norm(b).sum(), b, create_graph=True)


def test_gradient_against_differences(ocl):
    g = torch.Generator().manual_seed(3)
    x, w, gy = torch.randn(2, 33, generator=g), torch.randn(33, generator=g), torch.randn(2, 33, generator=g)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    dx, dw = torch.autograd.grad(ocl.functional.rms_norm(xd, wd, eps=1e-3), [xd, wd], gy.to(DEV))

    def value(x, w):
        y = x / (x.square().mean(1, keepdim=True) + 1e-3).sqrt() * w
        return (y * gy.double()).sum()

    # central differences in float64 with steps of 1e-5: off by about 1e-10 and 1e-11 of the value
    for at, got in ((0, dx), (1, dw)):
        args = [x.double(), w.double()]
        for i in range(0, args[at].numel(), 5):
            e = torch.zeros_like(args[at]).view(-1)
            e[i] = 1e-5
            e = e.view_as(args[at])
            up, down = list(args), list(args)
            up[at], down[at] = args[at] + e, args[at] - e
            assert abs((value(*up) - value(*down)).item() / 2e-5 - got.cpu().view(-1)[i].item()) < 2e-5


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_magnitudes_zeros_and_nans(ocl, dtype):
    """Rows of zeros, of the type's largest and smallest numbers; a NaN or an infinity spoils its own row alone."""
    top = torch.finfo(dtype).max
    x = torch.stack([torch.zeros(96), torch.full((96,), top), torch.full((96,), float(torch.finfo(dtype).tiny)),
                     torch.linspace(-1, 1, 96) * top, torch.ones(96), torch.ones(96)]).to(dtype)
    x[4, 3], x[5, 7] = float("nan"), float("inf")
    y = ocl.functional.rms_norm(x.to(DEV), eps=0.0 if dtype != torch.float16 else 1e-6).cpu()
    assert y[4].isnan().all() and y[5, 7].isnan() and (y[5].nan_to_num(0) == 0).all()
    if dtype == torch.float16:
        check_forward(y[:4], x[:4], None, 1e-6)
    else:
        assert y[0].isnan().all()  # 0 / 0: eps is what keeps a row of zeros
        if dtype == torch.float32:
            assert (y[1] == 0).all()  # the mean of squares is beyond fp32, as in the formula there
    assert (ocl.functional.rms_norm(torch.zeros(3, 8, dtype=dtype).to(DEV)).cpu() == 0).all()


def test_nothing(ocl):
    f = ocl.functional.rms_norm
    for shape in ((0, 16), (4, 0), (2, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[-1], device=DEV, requires_grad=True)
        y, s = f(x, w, torch.zeros(shape, device=DEV))
        assert y.shape == s.shape == torch.Size(shape)
        gx, gw = torch.autograd.grad(y, [x, w], torch.zeros(shape, device=DEV))
        assert gx.shape == torch.Size(shape) and (gw.cpu() == 0).all() and gw.shape == (shape[-1],)
        codes, scales = ocl.functional.rms_norm_8bit(x.detach(), w.detach())
        assert codes.shape == torch.Size(shape) and scales.shape == torch.Size(shape[:-1] + ((shape[-1] + 127) // 128,))


# --------------------------------------------------------------- 8-bit output
def quantized(y, tall=False):
    """Codes and scales by the definition, in fp32 operations that round once each."""
    rows, D = y.shape
    pad = torch.nn.functional.pad(y, (0, -D % 128, 0, -rows % 128 if tall else 0))
    cells = pad.view(-1, 128, pad.shape[1] // 128, 128) if tall else pad.view(-1, 1, pad.shape[1] // 128, 128)
    most = cells.abs().amax((1, 3), keepdim=True)
    ok = most > 2.0 ** -100
    top = torch.full_like(most, 448.0)  # (448 / x of a number is a product with a reciprocal in torch, rounded twice)
    codes = (cells * torch.where(ok, top / most, 0.0)).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.reshape(pad.shape)[:rows, :D], torch.where(ok, most / top, 0.0)[:, 0, :, 0]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 128), (70, 129), (4, 1000), (33, 2048), (2, 5001), (3, 9000), (1, 40000)],
                         ids=lambda s: "-".join(map(str, s)))
def test_8bit_output(ocl, shape, dtype):
    """Codes and scales bit for bit: the mean of squares is rounded from 64 bits, all else are IEEE operations."""
    x, r, w, _, _ = make(*shape, dtype, seed=5)
    codes, scales, s = ocl.functional.rms_norm_8bit(x.to(DEV), w.to(DEV), r.to(DEV), eps=1e-6)
    h = summed(x, r)
    assert torch.equal(s.cpu(), h) and codes.dtype == torch.uint8
    mean = h.double().square().mean(1, keepdim=True).float()
    # numpy's root and quotient are the IEEE ones
    rstd = np.float32(1) / np.sqrt(mean.numpy() + np.float32(1e-6))
    y = h.float() * torch.from_numpy(rstd) * w.float()
    want, want_scales = quantized(y)
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(codes.cpu(), want)
    assert codes.stride(0) % 16 == 0 or shape[0] == 1
    values = ocl.functional.dequantize_8bit(codes, scales).cpu()
    numbers = want.view(torch.float8_e4m3fn).float()
    assert torch.equal(values, numbers * want_scales.repeat_interleave(128, 1)[:, :shape[1]])
    # and near y: half a step of e4m3 is 2^-4 of the value, or 2^-10 of the smallest normal scale
    assert ((values - y).abs() <= 2.0 ** -4 * 1.001 * y.abs() + 2.0 ** -10 * want_scales.repeat_interleave(128, 1)[:, :shape[1]]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("tall", [False, True], ids=["rows", "blocks"])
def test_quantize(ocl, dtype, tall):
    g = torch.Generator().manual_seed(9)
    q, dq = ocl.functional.quantize_8bit, ocl.functional.dequantize_8bit
    for rows, D in ((1, 1), (130, 257), (256, 384), (127, 1001), (3, 70000)):
        x = (torch.randn(rows, D, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
        x[0, : D // 2] = 0
        for view, ref in ((x.to(DEV), x), (x.to(DEV)[:, D // 3:], x[:, D // 3:])):
            codes, scales = q(view, block_rows=128 if tall else 1)
            want, want_scales = quantized(ref.float(), tall)
            assert torch.equal(codes.cpu(), want) and torch.equal(scales.cpu(), want_scales)
            numbers = want.view(torch.float8_e4m3fn).float()
            up = want_scales.repeat_interleave(128, 1)[:, :ref.shape[1]]
            if tall:
                up = up.repeat_interleave(128, 0)[:rows]
            for out in TYPES:
                assert torch.equal(dq(codes, scales, dtype=out).cpu(), (numbers * up).to(out))
    # blocks of tiny numbers are 0, of infinities and NaN NaN, and no other block is touched
    x = torch.ones(2, 512)
    x[0, :128], x[0, 128], x[1, 300] = 1e-38, float("inf"), float("nan")
    if dtype == torch.float32:
        codes, scales = q(x.to(DEV))
        v = dq(codes, scales).cpu()
        assert (v[0, :128] == 0).all() and v[0, 128:256].isnan().all() and (v[0, 256:] == 1).all()
        assert (v[1, :256] == 1).all() and v[1, 256:384].isnan().all() and (v[1, 384:] == 1).all()


def test_refusals(ocl):
    f = ocl.functional
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (lambda: f.rms_norm(x, w[:7]), lambda: f.rms_norm(x, w.to(torch.bfloat16)), lambda: f.rms_norm(x, w, x[:3]),
                lambda: f.rms_norm(x, w, x.to(torch.float16)), lambda: f.rms_norm(x.long()), lambda: f.rms_norm(x, eps=-1.0),
                lambda: f.rms_norm(x, eps=float("nan")), lambda: f.rms_norm(x, torch.ones(8)), lambda: f.rms_norm(x.sum()),
                lambda: f.quantize_8bit(x[0], block_rows=128), lambda: f.dequantize_8bit(x, x),
                lambda: f.dequantize_8bit(*f.quantize_8bit(x), dtype=torch.float64),
                lambda: f.rms_norm_8bit(x.clone().requires_grad_())):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    with pytest.raises(ValueError, match="block_rows"):
        f.quantize_8bit(x, block_rows=2)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(Exception):
        f.rms_norm(fwd.make_dual(x, torch.ones_like(x)), w)


def test_captured(ocl):
    """Two captured graphs, replayed in turn, each with its own forward and backward pass."""
    x, r, w, gy, gs = (t.to(DEV) for t in make(300, 1000, torch.bfloat16))
    leaves = [t.requires_grad_() for t in (x, r, w)]

    def step():
        y, s = ocl.functional.rms_norm(x, w, r)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [gy, gs])]

    eager = [t.cpu() for t in step()]
    graphs = []
    for _ in range(2):
        graph = torch.ocl.Graph()
        with graph.capture():
            out = step()
        graphs.append((graph, out))
    for graph, out in graphs * 2:
        for t in out:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out, eager))
