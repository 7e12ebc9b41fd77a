"""Clipping by the gradients' global norm on `ocl`, against float64.

Eight squares are summed in fp32 (8 roundings of u = 2^-24, half of that after
the root), those sums in float64, and the norm rounds once: 5 u.  The factor
rounds twice more, a gradient's product once, and then to its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]
U = 2.0 ** -24


def parameters(shapes, dtypes, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    params = []
    for i, s in enumerate(shapes):
        p = torch.zeros(s, dtype=dtypes[i % len(dtypes)], device=DEV, requires_grad=True)
        p.grad = (scale * torch.randn(s, generator=g)).to(p.dtype).to(DEV)
        params.append(p)
    return params


def norm_of(grads, p):
    v = torch.cat([g.double().flatten() for g in grads]) if grads else torch.zeros(1).double()
    return v.norm(p).item()


def check(params, most, p=2.0):
    before = [x.grad.cpu() for x in params]
    norm = pytest.importorskip("pytorch_vulkan_b200").optim.clip_grad_norm_(params, most, p)
    want = norm_of(before, p)
    assert norm.shape == () and norm.dtype == torch.float32
    got = norm.item()
    assert abs(got - want) <= 6 * U * want, (got, want)
    coef = min(1.0, most / (want + 1e-6))
    for x, g in zip(params, before):
        w = g.double() * coef
        if coef == 1.0:
            assert torch.equal(x.grad.cpu(), g)
            continue
        eps = torch.finfo(g.dtype).eps / 2 if g.dtype != torch.float32 else 0
        bound = w.abs() * (10 * U + eps) + (2.0 ** -25 if g.dtype == torch.float16 else 2.0 ** -134 if eps else 2.0 ** -149)
        assert ((x.grad.cpu().double() - w).abs() <= bound).all()


SHAPES = {"one": [(5,)], "few": [(64, 64), (64,), (1,), (), (33, 7), (0,), (2, 3, 4)], "odd": [(101,), (8193,), (1, 50001), (7,)],
          "large": [(3000, 1000), (1000,), (4096, 513)], "many": [(17,)] * 1300 + [(20000,)]}


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf], ids=["2", "1", "inf"])
@pytest.mark.parametrize("dtype", TYPES + ["mixed"], ids=IDS + ["mixed"])
@pytest.mark.parametrize("name", SHAPES)
def test_norm_and_gradients(ocl, name, dtype, p):
    types = TYPES if dtype == "mixed" else [dtype]
    for most in (0.3, 1e9):
        check(parameters(SHAPES[name], types), most, p)


def test_layouts(ocl):
    """Gradients in channels-last order, views off 16-byte boundaries, one tensor in place of a list, a generator."""
    g = torch.Generator().manual_seed(1)
    flat = torch.randn(5000, generator=g).to(DEV)
    params = parameters([(4, 6, 5, 7)], [torch.float32])
    params[0].grad = params[0].grad.to(memory_format=torch.channels_last)
    for at, n in ((1, 1000), (1001, 33), (1035, 3000)):
        p = torch.zeros(n, device=DEV, requires_grad=True)
        p.grad = flat[at:at + n]
        params.append(p)
    around = flat.cpu().clone()
    check(params, 1.0)
    after = flat.cpu()
    for i in (0, 1034, *range(4035, 5000)):
        assert after[i] == around[i]
    one = parameters([(300,)], [torch.bfloat16])[0]
    before = one.grad.cpu().double()
    norm = ocl.optim.clip_grad_norm_(one, 2.0).item()
    assert abs(norm - before.norm().item()) <= 6 * U * norm
    assert abs(ocl.optim.clip_grad_norm_((p for p in [one]), 1e9).item() - 2.0) < 2.0 * 2.0 ** -8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_magnitudes(ocl, dtype):
    """Squares beyond fp32's numbers, on either side."""
    for scale in (1e25, 1e-30, 1e18, 1e-12):
        params = parameters([(100,), (9, 9)], [dtype], scale)
        check(params, 1.0 if scale > 1 else 1e-35)
    params = parameters([(1000,)], [dtype], 1e-5)
    params[0].grad[3] = 1e20
    check(params, 1.0)


def test_nan_and_infinity(ocl):
    for p in (2.0, 1.0, math.inf):
        for value in (math.nan, math.inf):
            params = parameters([(1000,), (50,)], [torch.float32])
            params[0].grad[77] = value
            before = [x.grad.cpu() for x in params]
            with pytest.raises(RuntimeError, match="non-finite"):
                ocl.optim.clip_grad_norm_(params, 1.0, p, error_if_nonfinite=True)
            assert all(torch.equal(x.grad.cpu().nan_to_num(9, 9), b.nan_to_num(9, 9)) for x, b in zip(params, before))
            norm = ocl.optim.clip_grad_norm_(params, 1.0, p).item()
            after = [x.grad.cpu() for x in params]
            if math.isnan(value):
                assert math.isnan(norm) and all(a.isnan().all() for a in after)
            else:  # a factor of 0, as the formula has it
                assert norm == math.inf and after[0][77].isnan() and (after[1] == 0).all()


def test_what_it_does_to_parameters(ocl):
    """Those without a gradient are passed over; none at all gives 0; the parameters stay; autograd knows of the change."""
    params = parameters([(10,), (20,)], [torch.float32])
    params.append(torch.zeros(5, device=DEV, requires_grad=True))
    version = params[0].grad._version
    ocl.optim.clip_grad_norm_(params, 1e-3, error_if_nonfinite=True)
    assert params[2].grad is None and params[0].grad._version > version
    assert ocl.optim.clip_grad_norm_([params[2]], 1.0).item() == 0.0 and ocl.optim.clip_grad_norm_([], 1.0).item() == 0.0
    check(parameters([(30,)], [torch.float32]), 0.0)


def test_the_same_bits(ocl):
    params = parameters([(1000, 1000), (77,)] * 3, TYPES)
    first = [ocl.optim.clip_grad_norm_(params, 1e9, p).item() for p in (2.0, 1.0)]
    for _ in range(3):
        assert [ocl.optim.clip_grad_norm_(params, 1e9, p).item() for p in (2.0, 1.0)] == first


def test_refusals(ocl):
    f = ocl.optim.clip_grad_norm_
    params = parameters([(10,), (20,)], [torch.float32])
    twice = torch.zeros(20, device=DEV, requires_grad=True)
    twice.grad = params[1].grad
    wide = torch.zeros(4, 10, device=DEV, requires_grad=True)
    wide.grad = torch.ones(4, 20, device=DEV)[:, :10]
    spread = torch.zeros(4, 10, device=DEV, requires_grad=True)
    spread.grad = torch.ones(10, device=DEV).expand(4, 10)
    whole = torch.zeros(10, dtype=torch.float64, device=DEV, requires_grad=True)
    whole.grad = torch.zeros(10, dtype=torch.float64, device=DEV)
    cpu = torch.zeros(3, requires_grad=True)
    cpu.grad = torch.ones(3)
    for extra in ([params[0]], [twice], [wide], [spread], [whole], [cpu]):
        with pytest.raises((RuntimeError, ValueError)):
            f(params + extra, 1.0)
    for args in ((-1.0,), (math.nan,), (1.0, 3.0), (1.0, 0.0)):
        with pytest.raises(ValueError):
            f(params, *args)
    with pytest.raises(RuntimeError, match="not a tensor"):
        f([1.0], 1.0)


def test_captured(ocl):
    """A step of two graphs over the same gradients, replayed in turn: each forms the norm of what is there then."""
    params = parameters([(1000, 100), (513,)], [torch.float32, torch.bfloat16])
    fresh = [p.grad.clone() for p in params]
    ocl.optim.clip_grad_norm_(params, 1e9)
    held = []
    for most in (3.0, 0.5):
        graph = torch.ocl.Graph()
        with graph.capture():
            norm = ocl.optim.clip_grad_norm_(params, most)
        held.append((graph, norm, most))
    for factor in (1.0, 2.0):
        for p, g in zip(params, fresh):
            p.grad.copy_(g * factor)
        want = norm_of([p.grad.cpu() for p in params], 2.0)
        for graph, norm, most in held:
            graph.replay()
            assert abs(norm.item() - want) <= 2.0 ** -7 * want
            want = most
