"""The 8-bit layer where a row's scale times the weight's leaves fp32's normal numbers although the result is one.

Codes have 2^-9 to 448, so a block's sum of 128 products is 0 or has 2^-18 to
2^25, and the scales' product may be far below or above fp32's range while the
result is inside.  The tolerance is that of the layer at any scales, each of
128 + blocks + 4 roundings of u = 2^-24 relative to the sum of magnitudes, twice
for additions that cut; below 2^-126 each addition to the sum rounds to a
multiple of 2^-149 (half of it, and half for the scale itself).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
U = 2.0 ** -24

# one tile width of few rows each, whole and split over a cluster, and pairs of CTAs on many
SHAPES = [(1, 300, 1100), (16, 512, 4096), (20, 257, 1100), (50, 300, 1100), (100, 300, 1100), (3, 9700, 200), (900, 3001, 1100)]
IDS = ["-".join(map(str, s)) for s in SHAPES]


def codes_of(rows, K, g):
    c = torch.randint(0, 256, (rows, K), generator=g, dtype=torch.int64)
    c[(c & 127) == 127] = 0  # the two NaNs
    return c.to(torch.uint8)


def numbers(codes, scales, tall):
    v = codes.view(torch.float8_e4m3fn).double()
    s = scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]
    return v * (s.repeat_interleave(128, 0)[:codes.shape[0]] if tall else s)


def check(ocl, xc, xs, wc, ws):
    y = ocl.functional.linear_8bit(xc.to(DEV), xs.to(DEV), wc.to(DEV), ws.to(DEV), dtype=torch.float32).cpu().double()
    x, w = numbers(xc, xs, False), numbers(wc, ws, True)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    assert (size < 1e38).all()
    blocks = xs.shape[1]
    bound = 2 * (128 + blocks + 4) * U * size + blocks * 2.0 ** -149
    assert ((y - want).abs() <= bound).all(), ((y - want).abs() / bound).max()
    return want


def powers(shape, low, high, g):
    return torch.exp2(low + (high - low) * torch.rand(shape, generator=g, dtype=torch.float64)).float()


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_small_scales(ocl, shape):
    """Products of 2^-145 to 2^-120, beside rows of usual ones, of zeros and of products that vanish altogether."""
    M, N, K = shape
    g = torch.Generator().manual_seed(M + N)
    blocks = (K + 127) // 128
    xc, wc = codes_of(M, K, g), codes_of(N, K, g)
    ws = powers(((N + 127) // 128, blocks), -65, -60, g)
    xs = powers((M, blocks), -80, -60, g)
    xs[1::7] = powers((len(xs[1::7]), blocks), 50, 60, g)
    xs[2::7] = 0
    xs[3::7] = powers((len(xs[3::7]), blocks), -109, -100, g)
    xs[4::7, ::2] = 0
    xs[5::7] *= -1
    want = check(ocl, xc, xs, wc, ws)
    assert (want[0].abs().amax() > 2.0 ** -120) and (want[0].abs().amax() < 2.0 ** -80)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_large_scales(ocl, shape):
    """Products beyond fp32 before sums of 0 (which are 0, not NaN) and before tiny ones."""
    M, N, K = shape
    g = torch.Generator().manual_seed(M + N + 1)
    blocks = (K + 127) // 128
    xc, wc = codes_of(M, K, g), codes_of(N, K, g)
    xs, ws = powers((M, blocks), -3, 3, g), powers(((N + 127) // 128, blocks), -3, 3, g)
    # block 0: nothing in x
    xs[:, 0], ws[:, 0] = 2.0 ** 70, 2.0 ** 65
    xc[:, :128] = 0
    xs[::3, 0] = 2.0 ** 118
    check(ocl, xc, xs, wc, ws)
    # block 1: numbers of 2^-9 to 2^-6, products of 2^-18 to 2^-12, 128 of them
    xc[:, 128:256] = xc[:, 128:256] & 0x87
    wc[:, 128:256] = wc[:, 128:256] & 0x87
    xs[:, 1], ws[:, 1] = 2.0 ** 67, -(2.0 ** 62)
    xs[2::5, 1] = 1.0
    check(ocl, xc, xs, wc, ws)


@pytest.mark.parametrize("shape", [(1, 300, 384), (900, 3001, 384)], ids=["few", "many"])
def test_infinite_scales_beside_small_ones(ocl, shape):
    """A scale that is infinite or NaN spoils its row (or its 128 outputs) as ever, whatever the other scales are."""
    M, N, K = shape
    g = torch.Generator().manual_seed(3)
    xc, wc = codes_of(M, K, g), codes_of(N, K, g)
    xs, ws = powers((M, 3), -80, -70, g), powers(((N + 127) // 128, 3), -65, -60, g)
    ws[1, 2], xs[0, 1] = float("inf"), float("nan")
    y = ocl.functional.linear_8bit(xc.to(DEV), xs.to(DEV), wc.to(DEV), ws.to(DEV), dtype=torch.float32).cpu()
    assert y[0].isnan().all() and not y[:, 128:256].isfinite().any()
    clean = torch.ones(N, dtype=torch.bool)
    clean[128:256] = False
    assert y[1:, clean].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", [(40, 300, 333), (700, 3001, 333)], ids=["few", "many"])
def test_with_a_bias(ocl, shape, dtype):
    """Rows of small scales and of usual ones, with a bias, in every output type, and the same bits again."""
    M, N, K = shape
    g = torch.Generator().manual_seed(5)
    xc, wc = codes_of(M, K, g), codes_of(N, K, g)
    xs, ws = powers((M, 3), -75, -65, g), powers(((N + 127) // 128, 3), -70, -60, g)
    xs[::2] = powers((len(xs[::2]), 3), 50, 60, g)
    bias = torch.randn(N, generator=g).to(dtype)
    ops = [t.to(DEV) for t in (xc, xs, wc, ws, bias)]
    y = ocl.functional.linear_8bit(*ops, dtype=dtype).cpu()
    assert torch.equal(ocl.functional.linear_8bit(*ops, dtype=dtype).cpu(), y)
    x, w = numbers(xc, xs, False), numbers(wc, ws, True)
    want, size = x @ w.t() + bias.double(), x.abs() @ w.abs().t()
    bound = 2 * (128 + 3 + 4) * U * size + U * (want.abs() + bias.double().abs())
    bound = bound + (torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -25 if dtype != torch.float32 else 0)
    # (an fp16 is infinite from 65504 and half its step of 32 on)
    beyond = y.isinf() & (want.abs() + bound >= 65520) if dtype == torch.float16 else torch.zeros_like(y, dtype=torch.bool)
    assert (((y.double() - want).abs() <= bound) | beyond).all()


def test_codes_of_small_numbers(ocl):
    """quantize_8bit's own codes of numbers near 1e-28 and 1e-7: the layer of the numbers that they stand for."""
    g = torch.Generator().manual_seed(4)
    f = ocl.functional
    x, w = 1e-28 * torch.randn(40, 700, generator=g), 1e-7 * torch.randn(200, 700, generator=g)
    xc, xs = f.quantize_8bit(x.to(DEV))
    wc, ws = f.quantize_8bit(w.to(DEV), block_rows=128)
    check(ocl, xc.cpu().contiguous(), xs.cpu(), wc.cpu().contiguous(), ws.cpu())
