"""RMS norm of rows whose mean of squares lies beneath fp32's normal numbers, which counts where eps is next to nothing.

u = 2^-24 is half a step of fp32; roundings as in the norm's other tests: at most 5 u of y, then half a step of the type.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16]
IDS = ["fp32", "bf16"]
U = 2.0 ** -24


def rows_of(D, dtype):
    g = torch.Generator().manual_seed(D)
    size = torch.exp2(-torch.arange(20, 124, 4).double())[:, None]
    return (torch.randn(len(size), D, generator=g).double() * size).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("eps", [0.0, 1e-35, 1e-41], ids=str)
@pytest.mark.parametrize("D", [5, 768, 1001, 4096, 5001, 40000])
def test_small_rows(ocl, D, eps, dtype):
    x = rows_of(D, dtype)
    g = torch.Generator().manual_seed(1)
    w, gy = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype), torch.randn(x.shape, generator=g).to(dtype)
    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = ocl.functional.rms_norm(xd, wd, eps=eps)
    h = x.double()
    rstd = 1 / (h.square().mean(1, keepdim=True) + float(np.float32(eps))).sqrt()
    n = h * rstd
    want = n * w.double()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
    tiny = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    got = y.detach().cpu().double()
    assert ((got - want).abs() <= 6 * U * want.abs() + (half * want.abs() + tiny) * (1 + 6 * U)).all()
    dx, dw = torch.autograd.grad(y, [xd, wd], gy.to(DEV))
    a = gy.double() * w.double()
    mean = (a * n).mean(1, keepdim=True)
    want = (a - n * mean) * rstd
    # the dot product's sum: at most D / 1024 + 110 additions one after the other; the other roundings, 10 of either term
    bound = rstd * (n.abs() * (D / 1024 + 110) * U * (a * n).abs().mean(1, keepdim=True) + 10 * U * (a.abs() + (n * mean).abs()))
    fine = want.abs() < 1e38
    assert (((dx.cpu().double() - want).abs() <= bound + half * (want.abs() + bound)) | ~fine).all() and fine.double().mean() > 0.9
    want = (gy.double() * n).sum(0)
    bound = (len(x) + 50) * U * (gy.double() * n).abs().sum(0)
    assert ((dw.cpu().double() - want).abs() <= bound + half * (want.abs() + bound)).all()


def test_codes_of_small_rows(ocl):
    """The codes are those of y, whatever the rows' size."""
    x, y = rows_of(700, torch.float32), rows_of(700, torch.float32) * 2.0 ** 20
    a, b = (ocl.functional.dequantize_8bit(*ocl.functional.rms_norm_8bit(t.to(DEV), eps=0.0)).cpu() for t in (x, y))
    # the same rows but for powers of two: one of fp32's roundings apart, a step of the codes (2^-3) where it falls on a border
    assert ((a - b).abs() <= 2.0 ** -3 * torch.maximum(a.abs(), b.abs()) + 1e-2).all() and (a == b).double().mean() > 0.99
