"""The host side of the RMS norm, the 8-bit codes and layer, the token log
probabilities and the clipping of gradients, without a device: refusals of the
C-ABI (which come before any launch), workspace queries, calls with nothing to
do, and the Python surface."""
import ctypes
import math
import os

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "pytorch_vulkan_b200", "lib", "libpvb2.so")
F32, F64, F16, BF16 = 0, 1, 2, 3
SOME = ctypes.c_void_p(1 << 20)  # an address that nothing reads
ODD = ctypes.c_void_p((1 << 20) + 2)
I64 = ctypes.c_int64


class Norm(ctypes.Structure):
    _fields_ = [(n, I64) for n in ("rows", "D", "ldx", "ldr", "ldg", "ldc")] + [("eps", ctypes.c_double), ("dtype", ctypes.c_int32)]


class Linear(ctypes.Structure):
    _fields_ = [(n, I64) for n in ("M", "N", "K", "ldx", "ldw")] + [("dtype", ctypes.c_int32)]


class Logp(ctypes.Structure):
    _fields_ = [(n, I64) for n in ("N", "V", "ldz")] + [("dtype", ctypes.c_int32), ("top", ctypes.c_int32)]


class Grad(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("numel", I64), ("dtype", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    L.pvb2_last_error.restype = ctypes.c_char_p
    for name in ("pvb2_rms_norm_bwd_workspace_size", "pvb2_clip_grad_norm_workspace_size"):
        getattr(L, name).restype = ctypes.c_size_t
    return L


def refused(lib, status, text):
    assert status == 1 and text in lib.pvb2_last_error().decode(), (status, lib.pvb2_last_error())


def norm(**kw):
    return Norm(**{**dict(rows=8, D=64, ldx=64, ldr=64, ldg=64, ldc=64, eps=1e-6, dtype=BF16), **kw})


def norm_fwd(lib, d, x=SOME, out=SOME, sum_=SOME, r=SOME):
    return lib.pvb2_rms_norm_fwd(ctypes.byref(d), x, r, SOME, out, sum_, None, None)


def norm_8bit(lib, d, x=SOME, out=SOME, sum_=SOME, r=SOME):
    return lib.pvb2_rms_norm_8bit(ctypes.byref(d), x, r, SOME, out, SOME, sum_, None)


def test_rms_norm_refusals(lib):
    for kw, text in [(dict(dtype=F64), "fp32, fp16 or bf16"), (dict(rows=-1), "out of range"), (dict(D=-1), "out of range"),
                     (dict(D=(1 << 24) + 1), "out of range"), (dict(rows=1 << 31), "out of range"), (dict(eps=-1e-6), "eps"),
                     (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(ldx=63), "strides"), (dict(ldr=1), "strides")]:
        d = norm(**kw)
        p = ctypes.byref(d)
        refused(lib, lib.pvb2_rms_norm_fwd(p, SOME, SOME, SOME, SOME, SOME, None, None), text)
        refused(lib, lib.pvb2_rms_norm_8bit(p, SOME, SOME, SOME, SOME, SOME, SOME, None), text)
        refused(lib, lib.pvb2_rms_norm_bwd(p, SOME, SOME, SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_size_t(1 << 30), None), text)
    d = norm()
    p = ctypes.byref(d)
    for kw in (dict(x=None), dict(out=None), dict(sum_=None)):
        refused(lib, norm_fwd(lib, d, **kw), "null pointer")
        refused(lib, norm_8bit(lib, d, **kw), "null pointer")
    refused(lib, lib.pvb2_rms_norm_bwd(p, None, SOME, SOME, SOME, None, SOME, SOME, SOME, ctypes.c_size_t(1 << 30), None), "null pointer")
    refused(lib, lib.pvb2_rms_norm_bwd(p, SOME, SOME, None, SOME, None, SOME, SOME, SOME, ctypes.c_size_t(1 << 30), None), "null pointer")
    need = lib.pvb2_rms_norm_bwd_workspace_size(p)
    assert need >= 4 * 64
    refused(lib, lib.pvb2_rms_norm_bwd(p, SOME, SOME, SOME, SOME, None, SOME, SOME, SOME, ctypes.c_size_t(need - 1), None), "workspace")
    refused(lib, lib.pvb2_rms_norm_bwd(p, SOME, SOME, SOME, SOME, None, SOME, SOME, None, ctypes.c_size_t(need), None), "workspace")
    refused(lib, lib.pvb2_rms_norm_fwd(None, SOME, None, SOME, SOME, None, None, None), "no descriptor")
    # nothing to do is no error
    for kw in (dict(rows=0), dict(D=0, ldx=0, ldr=0, ldg=0, ldc=0)):
        assert lib.pvb2_rms_norm_fwd(ctypes.byref(norm(**kw)), None, None, None, None, None, None, None) == 0
    assert lib.pvb2_rms_norm_bwd(p, SOME, SOME, SOME, SOME, None, None, None, None, ctypes.c_size_t(0), None) == 0
    # shares of the weight's gradient do not grow with the rows
    assert lib.pvb2_rms_norm_bwd_workspace_size(ctypes.byref(norm(rows=1 << 24, D=4096, ldx=4096))) < 1 << 25


def test_codes_refusals(lib):
    q = lambda dtype=F32, rows=8, D=64, x=SOME, ldx=64, tall=0, codes=SOME, ldc=64, scales=SOME: lib.pvb2_quantize_8bit(  # noqa: E731
        dtype, I64(rows), I64(D), x, I64(ldx), tall, codes, I64(ldc), scales, None)
    for kw, text in [(dict(dtype=F64), "fp32, fp16 or bf16"), (dict(rows=-1), "out of range"), (dict(ldx=10), "strides"),
                     (dict(ldc=10), "strides"), (dict(x=None), "null pointer"), (dict(codes=None), "null pointer"),
                     (dict(scales=None), "null pointer"), (dict(rows=65536 * 128, tall=1), "blocks of 128")]:
        refused(lib, q(**kw), text)
    d = lambda rows=8, D=64, codes=SOME, ldc=64, scales=SOME, dtype=F32, out=SOME: lib.pvb2_dequantize_8bit(  # noqa: E731
        I64(rows), I64(D), codes, I64(ldc), scales, 0, dtype, out, None)
    for kw, text in [(dict(dtype=F64), "fp32, fp16 or bf16"), (dict(ldc=63), "strides"), (dict(out=None), "null pointer"),
                     (dict(D=-1), "out of range")]:
        refused(lib, d(**kw), text)
    assert q(rows=0, x=None, codes=None, scales=None) == 0 and d(D=0, codes=None, scales=None, out=None) == 0


def linear(lib, x=SOME, xs=SOME, w=SOME, ws=SOME, y=SOME, **kw):
    d = Linear(**{**dict(M=4, N=8, K=256, ldx=256, ldw=256, dtype=BF16), **kw})
    return lib.pvb2_linear8(ctypes.byref(d), x, xs, w, ws, None, y, None)


def test_linear_refusals(lib):
    for kw, text in [(dict(dtype=F64), "fp32, fp16 or bf16"), (dict(K=0), "out of range"), (dict(M=-1), "out of range"),
                     (dict(N=1 << 31), "out of range"), (dict(M=1 << 29, N=1 << 29), "more outputs"), (dict(ldx=255), "strides"),
                     (dict(ldw=100), "strides"), (dict(ldx=264), "16-byte"), (dict(ldw=257), "16-byte"), (dict(x=ODD), "16-byte"),
                     (dict(w=ODD), "16-byte"), (dict(x=None), "null pointer"), (dict(ws=None), "null pointer"),
                     (dict(y=None), "null pointer")]:
        refused(lib, linear(lib, **kw), text)
    assert linear(lib, M=0, x=None, xs=None, y=None) == 0 and linear(lib, N=0, w=None, ws=None, y=None) == 0


def logp_fwd(lib, z=SOME, t=SOME, lp=SOME, h=SOME, tlp=SOME, tat=SOME, **kw):
    d = Logp(**{**dict(N=4, V=100, ldz=100, dtype=BF16, top=0), **kw})
    return lib.pvb2_token_logp_fwd(ctypes.byref(d), z, t, lp, h, None, tlp, tat, None)


def logp_bwd(lib, z=SOME, t=SOME, stats=SOME, dz=SOME, **kw):
    d = Logp(**{**dict(N=4, V=100, ldz=100, dtype=BF16, top=0), **kw})
    return lib.pvb2_token_logp_bwd(ctypes.byref(d), z, t, stats, None, 0, None, 0, dz, None)


def test_token_log_probs_refusals(lib):
    for kw, text in [(dict(dtype=F64), "fp32, fp16 or bf16"), (dict(V=0), "out of range"), (dict(N=-1), "out of range"),
                     (dict(V=1 << 31, ldz=1 << 31), "out of range"), (dict(top=33), "top"), (dict(top=-1), "top"),
                     (dict(V=5, ldz=5, top=6), "top"), (dict(ldz=99), "stride")]:
        refused(lib, logp_fwd(lib, **kw), text)
        refused(lib, logp_bwd(lib, **kw), text)
    for kw in (dict(z=None), dict(t=None), dict(lp=None), dict(h=None), dict(tlp=None, top=2), dict(tat=None, top=2)):
        refused(lib, logp_fwd(lib, **kw), "null pointer")
    for kw in (dict(z=None), dict(t=None), dict(stats=None), dict(dz=None)):
        refused(lib, logp_bwd(lib, **kw), "null pointer")
    assert logp_fwd(lib, N=0, z=None, t=None, lp=None, h=None) == 0 and logp_bwd(lib, N=0, z=None, t=None, stats=None, dz=None) == 0


def clip(lib, grads, norm_type=2, scale=1, most=1.0, out=SOME, ws=SOME, ws_bytes=1 << 30):
    arr = (Grad * max(1, len(grads)))(*grads)
    return lib.pvb2_clip_grad_norm(len(grads), arr, norm_type, scale, ctypes.c_double(most), out, ws, ctypes.c_size_t(ws_bytes), None)


def test_clip_refusals(lib):
    one = lambda data=1 << 20, numel=100, dtype=F32: Grad(data, numel, dtype)  # noqa: E731
    for grads, text in [([one(dtype=F64)], "fp32, fp16 or bf16"), ([one(numel=-1)], "elements"), ([one(data=None)], "null pointer"),
                        ([one(data=(1 << 20) + 2)], "not aligned"), ([one(), one()], "twice"),
                        ([one(), one(data=(1 << 20) + 396)], "overlap"), ([one(data=(1 << 20) + 8, dtype=BF16), one()], "overlap")]:
        refused(lib, clip(lib, grads), text)
    refused(lib, clip(lib, [one()], norm_type=3), "norms")
    refused(lib, clip(lib, [one()], most=-1.0), "max_norm")
    refused(lib, clip(lib, [one()], most=math.nan), "max_norm")
    refused(lib, clip(lib, [one()], out=None), "null pointer")
    refused(lib, clip(lib, [one()], ws_bytes=7), "workspace")
    refused(lib, clip(lib, [one()], ws=None), "workspace")
    assert lib.pvb2_clip_grad_norm_workspace_size(0) == 0
    assert 8 * 132 <= lib.pvb2_clip_grad_norm_workspace_size(1) <= lib.pvb2_clip_grad_norm_workspace_size(5000) < 1 << 20


def test_python_surface():
    import pytorch_vulkan_b200 as pkg

    f = pkg.functional
    for op in ("rms_norm", "rms_norm_add", "rms_norm_8bit", "quantize_8bit", "dequantize_8bit", "linear_8bit", "token_log_probs"):
        assert hasattr(torch.ops.ocl, op)
    for name in ("rms_norm", "rms_norm_8bit", "quantize_8bit", "dequantize_8bit", "linear_8bit", "token_log_probs"):
        assert getattr(torch.ocl.functional, name).__doc__
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="block_rows"):
        f.quantize_8bit(x, block_rows=64)
    for call in (lambda: f.rms_norm(x), lambda: f.rms_norm(x, None, x), lambda: f.quantize_8bit(x),
                 lambda: f.token_log_probs(x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    p = torch.zeros(3, requires_grad=True)
    assert pkg.optim.clip_grad_norm_([p], 1.0).item() == 0.0
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="ocl expected"):
        pkg.optim.clip_grad_norm_([p], 1.0)
    for args in ((-1.0,), (1.0, 3.0), (math.nan,)):
        with pytest.raises(ValueError):
            pkg.optim.clip_grad_norm_([p], *args)


def test_launches_that_fail_say_so(lib):
    """Where there is no device every launch fails: its own error comes back, from every entry point."""
    count = ctypes.c_int(-1)
    lib.pvb2_device_count(ctypes.byref(count))
    if count.value != 0:
        pytest.skip("a launch of these addresses is for machines without a device alone")
    n, z = norm(), Logp(N=4, V=100, ldz=100, dtype=BF16, top=0)
    need = ctypes.c_size_t(1 << 30)
    calls = [
        ("launch_over", lambda: norm_fwd(lib, n)),
        ("launch_over", lambda: lib.pvb2_rms_norm_bwd(ctypes.byref(n), SOME, SOME, SOME, SOME, None, SOME, SOME, SOME, need, None)),
        ("quant_tile_kernel", lambda: lib.pvb2_quantize_8bit(F32, I64(8), I64(64), SOME, I64(64), 1, SOME, I64(64), SOME, None)),
        ("dequant_kernel", lambda: lib.pvb2_dequantize_8bit(I64(8), I64(64), SOME, I64(64), SOME, 0, F32, SOME, None)),
        ("failed", lambda: lib.pvb2_token_logp_fwd(ctypes.byref(z), SOME, SOME, SOME, SOME, None, None, None, None)),
    ]
    for what, call in calls:
        assert call() == 3, what
        text = lib.pvb2_last_error().decode()
        assert what in text and "failed" in text, (what, text)
