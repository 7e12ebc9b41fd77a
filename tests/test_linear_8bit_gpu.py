"""The linear layer in 8-bit floating point on `ocl` against the product of the
numbers that the codes stand for, in float64.

Products of two codes are exact.  u = 2^-24 is half a step of fp32.  The 128
products of a block and the blocks are summed with at most 128 + blocks + 4
roundings of u, each relative to at most the sum of magnitudes (twice that, for
additions that cut), the scales' product and the bias round once more; then
half a step of the output's type.
"""
import ctypes
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
U = 2.0 ** -24
OUT = [torch.float32, torch.bfloat16, torch.float16]


def operands(M, N, K, seed=0, lead=None):
    g = torch.Generator().manual_seed(seed + M + 3 * N + 5 * K)
    blocks = (K + 127) // 128

    def codes(rows):
        c = torch.randint(0, 256, (rows, K), generator=g, dtype=torch.int64)
        c[(c & 127) == 127] = 0  # the two NaNs
        return c.to(torch.uint8)

    xs = torch.exp(torch.randn(M, blocks, generator=g)) * 1e-2
    ws = torch.exp(torch.randn((N + 127) // 128, blocks, generator=g)) * 1e-3
    return codes(M), xs, codes(N), ws, torch.randn(N, generator=g)


def numbers(codes, scales, tall):
    v = codes.view(torch.float8_e4m3fn).double()
    s = scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]
    if tall:
        s = s.repeat_interleave(128, 0)[:codes.shape[0]]
    return v * s


def check(y, xc, xs, wc, ws, bias=None):
    dtype, blocks = y.dtype, xs.shape[1]
    x, w = numbers(xc, xs, False), numbers(wc, ws, True)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    bound = 2 * (128 + blocks + 4) * U * size
    if bias is not None:
        b = bias.to(dtype).double()
        want, bound = want + b, bound + U * (want.abs() + b.abs())
    bound = bound + (torch.finfo(dtype).eps / 2 * (want.abs() + bound) if dtype != torch.float32 else 0)
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 0)
    got = y.double().cpu()
    assert got.shape == want.shape
    fine = torch.isfinite(got) if dtype == torch.float16 else torch.ones_like(got, dtype=torch.bool)
    assert ((got - want).abs() <= bound)[fine].all(), ((got - want).abs() / bound)[fine].max()
    assert (want[~fine].abs() >= 65504).all()


# few rows (each tile width, split over a cluster and not), many rows on pairs, ends in every direction
SHAPES = [(1, 128, 128), (1, 1, 1), (1, 4096, 4096), (2, 16, 32), (7, 300, 1000), (16, 129, 513), (17, 128, 2048), (32, 1000, 160),
          (33, 257, 384), (64, 64, 4096), (65, 513, 640), (128, 256, 128), (129, 130, 16), (300, 777, 1000), (1, 40000, 256),
          (3, 128, 20000), (2048, 2048, 512), (2047, 2500, 1300), (5000, 1001, 144), (1024, 5000, 128), (600, 9000, 100)]


@pytest.mark.parametrize("dtype", OUT, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_values(ocl, shape, dtype):
    xc, xs, wc, ws, b = operands(*shape)
    bias = b if shape[0] % 2 else None
    y = ocl.functional.linear_8bit(xc.to(DEV), xs.to(DEV), wc.to(DEV), ws.to(DEV),
                                   None if bias is None else bias.to(dtype).to(DEV), dtype=dtype)
    check(y, xc, xs, wc, ws, bias)


def test_the_same_bits(ocl):
    """Sums over a cluster join in a fixed order."""
    for shape in ((1, 512, 8192), (40, 256, 4096), (700, 3000, 1024)):
        ops = [t.to(DEV) for t in operands(*shape)[:4]]
        first = ocl.functional.linear_8bit(*ops, dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(ocl.functional.linear_8bit(*ops, dtype=torch.float32).cpu(), first.cpu())


def test_layouts(ocl):
    """Rows of quantize_8bit, rows that begin anywhere, transposed and sliced operands, more dimensions, no rows."""
    f = ocl.functional
    xc, xs, wc, ws, _ = operands(24, 200, 333)
    want = f.linear_8bit(xc.to(DEV), xs.to(DEV), wc.to(DEV), ws.to(DEV), dtype=torch.float32).cpu()
    wide = torch.zeros(24, 400, dtype=torch.uint8)
    wide[:, 7:340] = xc
    tall = torch.zeros(333, 200, dtype=torch.uint8)
    tall.copy_(wc.t())
    y = f.linear_8bit(wide.to(DEV)[:, 7:340], xs.t().contiguous().to(DEV).t(), tall.to(DEV).t(), ws.to(DEV), dtype=torch.float32)
    assert torch.equal(y.cpu(), want)
    y = f.linear_8bit(xc.to(DEV).view(2, 3, 4, 333), xs.to(DEV).view(2, 3, 4, 3), wc.to(DEV), ws.to(DEV), dtype=torch.float32)
    assert torch.equal(y.cpu().view(24, 200), want)
    y = f.linear_8bit(xc[5].to(DEV), xs[5].to(DEV), wc.to(DEV), ws.to(DEV), dtype=torch.float32)
    assert y.shape == (200,)
    check(y.view(1, 200), xc[5:6], xs[5:6], wc, ws)
    assert f.linear_8bit(xc[:0].to(DEV), xs[:0].to(DEV), wc.to(DEV), ws.to(DEV)).shape == (0, 200)


def test_one_row_as_among_many(ocl):
    """A row's result does not depend on how many others there are beyond its roundings."""
    xc, xs, wc, ws, _ = operands(1500, 2048, 1024)
    ops = (wc.to(DEV), ws.to(DEV))
    for M in (1, 16, 100, 1500):
        check(ocl.functional.linear_8bit(xc[:M].to(DEV), xs[:M].to(DEV), *ops, dtype=torch.float32), xc[:M], xs[:M], wc, ws)


@pytest.mark.parametrize("M", [1, 40, 900])
def test_nan_and_infinity_stay_in_their_rows(ocl, M):
    xc, xs, wc, ws, _ = operands(M, 2304, 300)
    xs[0, 1] = float("nan")
    wc[5, 3] = 0x7F
    ws[1, 2] = float("inf")
    y = ocl.functional.linear_8bit(xc.to(DEV), xs.to(DEV), wc.to(DEV), ws.to(DEV), dtype=torch.float32).cpu()
    assert y[0].isnan().all() and y[:, 5].isnan().all() and not y[1:, 128:256].isfinite().any()
    clean = torch.ones(2304, dtype=torch.bool)
    clean[5], clean[128:256] = False, False
    assert y[1:, clean].isfinite().all()
    if M > 1:
        ws[1, 2], wc[5, 3] = 1.0, 0
        x, w = numbers(xc[1:], xs[1:], False), numbers(wc, ws, True)
        bound = 2 * (128 + 3 + 4) * U * (x.abs() @ w.abs().t())
        assert ((y[1:].double() - x @ w.t()).abs() <= bound)[:, clean].all()


def test_of_quantised_numbers(ocl):
    """The layer of a weight that was quantised once: near F.linear by what the codes' rounding does."""
    g = torch.Generator().manual_seed(4)
    f = ocl.functional
    x, w = torch.randn(50, 512, generator=g), torch.randn(300, 512, generator=g) / 512 ** 0.5
    codes, scales = f.quantize_8bit(x.to(DEV))
    wc, ws = f.quantize_8bit(w.to(DEV), block_rows=128)
    y = f.linear_8bit(codes, scales, wc, ws, dtype=torch.float32).cpu().double()
    exact = f.dequantize_8bit(codes, scales).cpu().double() @ f.dequantize_8bit(wc, ws).cpu().double().t()
    assert (y - exact).abs().max() <= 2 * (128 + 8) * U * (x.abs() @ w.abs().t()).max() * 1.2
    # 2^-4 of each factor at most, and so 2^-3 (and a little) of the sum of magnitudes
    assert ((y - x.double() @ w.double().t()).abs() <= 0.13 * (x.abs() @ w.abs().t()) + 1e-3).all()


def test_refusals(ocl):
    xc, xs, wc, ws, b = (t.to(DEV) for t in operands(4, 200, 300))
    f = ocl.functional.linear_8bit
    for bad in (lambda: f(xc.float(), xs, wc, ws), lambda: f(xc, xs[:, :2], wc, ws), lambda: f(xc, xs, wc, ws[:1]),
                lambda: f(xc, xs.to(torch.bfloat16), wc, ws), lambda: f(xc, xs, wc[:, :299], ws), lambda: f(xc, xs, wc, ws, b),
                lambda: f(xc, xs, wc, ws, b[:199], dtype=torch.float32), lambda: f(xc, xs, wc, ws, dtype=torch.float64),
                lambda: f(xc, xs, wc, ws.clone().requires_grad_()), lambda: f(xc[:, :0], xs[:, :0], wc[:, :0], ws[:, :0]),
                lambda: f(xc, xs, wc, ws, b.clone().requires_grad_(), dtype=torch.float32), lambda: f(xc, xs, wc[0], ws)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    with pytest.raises((RuntimeError, NotImplementedError)):
        f(xc.cpu(), xs.cpu(), wc.cpu(), ws.cpu())


def test_no_wait_gave_up(ocl):
    lib = ctypes.CDLL(os.path.join(os.path.dirname(ocl.__file__), "lib", "libpvb2.so"))
    torch.ocl.synchronize()
    flag = ctypes.c_int(-1)
    assert lib.pvb2_linear8_status(ctypes.byref(flag), 0) == 0 and flag.value == 0
