"""The host side of the cross entropy of a linear layer, the AdamW step and the
relative position bias, without a device: refusals of the C-ABI (which come
before any launch), workspace and memory-to-keep queries, the Python surface,
and the 8-bit codes' numbers."""
import ctypes
import os

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "pytorch_vulkan_b200", "lib", "libpvb2.so")
F32, F16, BF16, U8 = 0, 2, 3, 8
SOME = ctypes.c_void_p(1 << 20)  # an address that nothing reads


class Tensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("sizes", ctypes.c_int64 * 8), ("strides", ctypes.c_int64 * 8),
                ("ndim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class Ce(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("N", "D", "V", "ldx", "ldw", "ignore_index")] + [
        ("label_smoothing", ctypes.c_double), ("kept", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("dtype", "reduction")]


class Adam(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("param_dtype", "state_dtype", "decoupled", "maximize", "amsgrad",
                                             "increment_step")] + [
        (n, ctypes.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [
        (n, ctypes.c_void_p) for n in ("lr_device", "grad_scale", "found_inf")]


class AdamTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "max_exp_avg_sq",
                                              "exp_avg_scale", "exp_avg_sq_scale", "step")] + [("numel", ctypes.c_int64)]


class Bias(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("H", "num_buckets", "bidirectional", "dtype")] + [
        (n, ctypes.c_int64) for n in ("Lq", "Lk", "max_distance", "q_offset")]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    L.pvb2_last_error.restype = ctypes.c_char_p
    for name in ("pvb2_linear_ce_fwd_workspace_size", "pvb2_linear_ce_bwd_workspace_size", "pvb2_linear_ce_keep",
                 "pvb2_adamw_workspace_size", "pvb2_relative_bias_bwd_workspace_size"):
        getattr(L, name).restype = ctypes.c_size_t
    return L


def ce(**kw):
    d = dict(N=100, D=64, V=1000, ldx=64, ldw=64, ignore_index=-100, label_smoothing=0.0, kept=0, dtype=BF16, reduction=1)
    d.update(kw)
    return Ce(**d)


def ce_fwd(lib, d, x=SOME, w=SOME, target=SOME, out=SOME, lse=SOME, count=SOME, kept=None, ws=SOME, ws_bytes=1 << 40):
    return lib.pvb2_linear_ce_fwd(ctypes.byref(d), x, w, None, target, out, lse, count, kept, ws, ctypes.c_size_t(ws_bytes),
                                  None)


def ce_bwd(lib, d, x=SOME, w=SOME, target=SOME, lse=SOME, count=SOME, kept=None, grad=SOME, dx=SOME, dw=SOME, ws=SOME,
           ws_bytes=1 << 40):
    return lib.pvb2_linear_ce_bwd(ctypes.byref(d), x, w, None, target, lse, count, kept, grad, dx, dw, None, ws,
                                  ctypes.c_size_t(ws_bytes), None)


def refused(lib, status, text):
    assert status == 1 and text in lib.pvb2_last_error().decode(), lib.pvb2_last_error()


def test_linear_cross_entropy_refusals(lib):
    for kw, text in [
        (dict(dtype=1), "fp32, fp16 or bf16"), (dict(reduction=3), "reduction"),
        (dict(V=0), "out of range"), (dict(D=0), "out of range"), (dict(N=-1), "out of range"),
        (dict(N=1 << 24), "out of range"), (dict(ldx=63), "row strides"), (dict(ldw=10), "row strides"),
        (dict(label_smoothing=-0.1), "label smoothing"), (dict(label_smoothing=float("nan")), "label smoothing"),
        (dict(kept=100), "multiple of 256"), (dict(kept=1001), "multiple of 256"), (dict(kept=-256), "multiple of 256"),
    ]:
        d = ce(**kw)
        refused(lib, ce_fwd(lib, d), text)
        refused(lib, ce_bwd(lib, d), text)
        assert lib.pvb2_linear_ce_fwd_workspace_size(ctypes.byref(d)) == 0
        assert lib.pvb2_linear_ce_bwd_workspace_size(ctypes.byref(d)) == 0
    d = ce()
    for kw in (dict(x=None), dict(w=None), dict(target=None), dict(out=None), dict(lse=None), dict(count=None)):
        refused(lib, ce_fwd(lib, d, **kw), "null pointer")
    for kw in (dict(x=None), dict(w=None), dict(target=None), dict(lse=None), dict(count=None), dict(grad=None)):
        refused(lib, ce_bwd(lib, d, **kw), "null pointer")
    need = lib.pvb2_linear_ce_fwd_workspace_size(ctypes.byref(d))
    refused(lib, ce_fwd(lib, d, ws_bytes=need - 1), "workspace")
    refused(lib, ce_fwd(lib, d, ws=None), "workspace")
    refused(lib, ce_bwd(lib, d, ws_bytes=lib.pvb2_linear_ce_bwd_workspace_size(ctypes.byref(d)) - 1), "workspace")
    refused(lib, ce_fwd(lib, ce(kept=512)), "what is kept")
    refused(lib, ce_bwd(lib, ce(kept=512)), "missing")
    odd = ctypes.c_void_p((1 << 20) + 2)
    refused(lib, ce_fwd(lib, d, x=odd), "16-byte boundaries")
    refused(lib, ce_bwd(lib, d, w=odd), "16-byte boundaries")


def test_what_a_forward_pass_keeps(lib):
    """All classes where they fit, else a multiple of 256 of them within the budget, none below 1024."""
    def keep(budget, **kw):
        d = ce(**kw)
        n = lib.pvb2_linear_ce_keep(ctypes.byref(d), ctypes.c_size_t(budget))
        assert n <= budget + 4 * d.N + 4096 if n else d.kept == 0
        return d.kept, n

    big = dict(N=4096, V=100003, D=512, ldx=512, ldw=512)
    full, n = keep(1 << 40, **big)
    assert full == 100003 and n >= 2 * 4096 * 100003
    some, n = keep(100 << 20, **big)
    assert some % 256 == 0 and 11000 < some < 12800 and n > 90 << 20
    assert keep(4096 * 2 * 1000, **big) == (0, 0)
    assert keep(0, **big) == (0, 0)
    some32, _ = keep(100 << 20, **dict(big, dtype=F32))
    assert 6000 < some32 < 6600  # fp32 logits take twice the memory
    assert keep(1 << 30, N=0) == (0, 0)
    assert keep(1 << 30, V=7) == (7, keep(1 << 30, V=7)[1])
    assert keep(1 << 30, label_smoothing=2.0) == (0, 0)


def test_workspaces_do_not_grow_with_rows_times_classes(lib):
    for rows, classes in ((4096, 1 << 20), (1 << 20, 4096)):
        d = ce(N=rows, V=classes, D=64)
        for f in (lib.pvb2_linear_ce_fwd_workspace_size, lib.pvb2_linear_ce_bwd_workspace_size):
            assert 0 < f(ctypes.byref(d)) < rows * classes * 2 // 2


def adam(lib, d, tensors, ws=SOME, ws_bytes=1 << 30):
    arr = (AdamTensor * max(1, len(tensors)))(*tensors)
    return lib.pvb2_adamw_multi(ctypes.byref(d), len(tensors), arr, ws, ctypes.c_size_t(ws_bytes), None)


def test_adamw_refusals(lib):
    good = dict(param_dtype=F32, state_dtype=F32, decoupled=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    ptr = dict(param=1 << 20, grad=2 << 20, exp_avg=3 << 20, exp_avg_sq=4 << 20, step=5 << 20, numel=10)
    one = lambda **kw: AdamTensor(**dict(ptr, **kw))
    for kw, text in [(dict(param_dtype=1), "parameters are"), (dict(state_dtype=F16), "moments are"),
                     (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"), (dict(beta1=float("nan")), "betas"),
                     (dict(state_dtype=U8, decoupled=0), "8-bit moments"), (dict(state_dtype=U8, amsgrad=1), "8-bit moments"),
                     (dict(state_dtype=U8, grad_scale=64), "8-bit moments")]:
        refused(lib, adam(lib, Adam(**dict(good, **kw)), [one()]), text)
    d = Adam(**good)
    for kw, text in [(dict(param=None), "null pointer"), (dict(exp_avg=None), "null pointer"), (dict(step=None), "no step"),
                     (dict(numel=-1), "elements"), (dict(numel=1 << 41), "elements")]:
        refused(lib, adam(lib, d, [one(**kw)]), text)
    refused(lib, adam(lib, Adam(**dict(good, state_dtype=U8)), [one()]), "no scales")
    refused(lib, adam(lib, Adam(**dict(good, amsgrad=1)), [one()]), "running maximum")
    refused(lib, adam(lib, d, [one(), one()]), "listed twice")
    refused(lib, adam(lib, d, [one()], ws_bytes=8), "workspace")
    refused(lib, adam(lib, d, [one()], ws=None), "workspace")
    assert lib.pvb2_adamw_workspace_size(3) == 48 and lib.pvb2_adamw_workspace_size(0) == 0
    assert adam(lib, d, [], ws=None, ws_bytes=0) == 0
    arr = (AdamTensor * 1)(one(exp_avg_scale=64))
    refused(lib, lib.pvb2_adamw8_values(1, arr, None), "no scales")


def bias(**kw):
    d = dict(H=4, num_buckets=32, bidirectional=1, dtype=F32, Lq=10, Lk=12, max_distance=128, q_offset=0)
    d.update(kw)
    return Bias(**d)


def test_relative_bias_refusals(lib):
    def grad(sizes=(2, 4, 10, 12), dtype=F32):
        st = [0] * 8
        n = 1
        for i in reversed(range(4)):
            st[i], n = n, n * sizes[i]
        return Tensor(1 << 20, (ctypes.c_int64 * 8)(*sizes), (ctypes.c_int64 * 8)(*st), 4, dtype)

    for kw, text in [(dict(dtype=1), "fp32, fp16 or bf16"), (dict(num_buckets=1, bidirectional=0), "buckets"),
                     (dict(num_buckets=513, bidirectional=0), "buckets"), (dict(num_buckets=31), "even number"),
                     (dict(num_buckets=2), "even number"), (dict(max_distance=8), "max_distance"),
                     (dict(max_distance=(1 << 20) + 1), "max_distance"), (dict(H=-1), "out of range"),
                     (dict(Lq=-1), "out of range"), (dict(Lk=1 << 40), "out of range"),
                     (dict(q_offset=-(1 << 40)), "out of range")]:
        d = bias(**kw)
        refused(lib, lib.pvb2_relative_bias_fwd(ctypes.byref(d), SOME, SOME, None), text)
        refused(lib, lib.pvb2_relative_bias_bwd(ctypes.byref(d), ctypes.byref(grad()), SOME, SOME,
                                                ctypes.c_size_t(1 << 30), None), text)
    d = bias()
    refused(lib, lib.pvb2_relative_bias_fwd(ctypes.byref(d), None, SOME, None), "null pointer")
    for g in (grad((2, 3, 10, 12)), grad((2, 4, 10, 13)), grad(dtype=F16)):
        refused(lib, lib.pvb2_relative_bias_bwd(ctypes.byref(d), ctypes.byref(g), SOME, SOME, ctypes.c_size_t(1 << 30),
                                                None), "grad [B, H, Lq, Lk]")
    need = lib.pvb2_relative_bias_bwd_workspace_size(ctypes.byref(d), ctypes.c_int64(2))
    assert need > 0
    refused(lib, lib.pvb2_relative_bias_bwd(ctypes.byref(d), ctypes.byref(grad()), SOME, SOME, ctypes.c_size_t(need - 1),
                                            None), "workspace")
    # nothing to do is no error
    assert lib.pvb2_relative_bias_fwd(ctypes.byref(bias(Lq=0)), None, None, None) == 0


def test_python_surface():
    import pytorch_vulkan_b200 as pkg

    assert torch.ocl.functional is pkg.functional and torch.ocl.optim is pkg.optim
    for op in ("linear_cross_entropy", "relative_position_bias", "relative_position_bias_backward"):
        assert hasattr(torch.ops.ocl, op)
    cpu = torch.zeros(3, requires_grad=True)
    with pytest.raises(ValueError, match="ocl device expected"):
        pkg.optim.AdamW([cpu])
    with pytest.raises(ValueError, match="state_bits"):
        pkg.optim.AdamW([cpu], state_bits=16)
    with pytest.raises(ValueError, match="reduction"):
        pkg.functional.linear_cross_entropy(cpu, cpu, cpu, reduction="avg")
    with pytest.raises((RuntimeError, NotImplementedError)):
        pkg.functional.linear_cross_entropy(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))


def test_numbers_of_the_8_bit_codes():
    """What a code stands for: a sign (first moments), 4 bits of exponent with bias 15, 3 or 4 bits of mantissa."""
    for mantissa in (3, 4):
        top = 16 * 2 ** mantissa
        codes = torch.arange(top, dtype=torch.int32)
        by_bits = (codes << (23 - mantissa)).view(torch.float32) * 2.0 ** 112
        e, m = codes >> mantissa, codes & (2 ** mantissa - 1)
        one = 2 ** mantissa
        number = torch.where(e == 0, m.double() / one * 2.0 ** -14, (1 + m.double() / one) * 2.0 ** (e.double() - 15))
        assert torch.equal(by_bits.double(), number)
        assert number[-1].item() == 2 - 2.0 ** -mantissa and number[1].item() == 2.0 ** (-14 - mantissa)
        # neighbours are at most 2^-mantissa of the lower one apart: half a step is 2^-(mantissa + 1) of a number
        normal = number[one:]
        assert ((normal[1:] - normal[:-1]) <= 2.0 ** -mantissa * normal[:-1]).all()
