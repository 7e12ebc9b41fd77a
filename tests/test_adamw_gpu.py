"""Adam / AdamW steps on `ocl`: torch.optim's fused path and
pytorch_vulkan_b200.optim.AdamW with 32-bit and 8-bit moments, against the
formula in float64 on the CPU.

Tolerances count roundings of fp32 (half a step is 2^-24 of the value): a
moment is two products and a sum on rounded coefficients (at most 5 roundings
of its larger term); the update is a root, a quotient, two products and a sum
on rounded factors (at most 12, plus the moments' own); the parameter takes
one product and one difference (3 of |p|, with the rounded factor) and, in 16
bits, one rounding to its type.  8-bit moments are compared code by code with
the formula in fp32, rounded operation by operation.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
U = 2.0 ** -24
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.99, 1e-8, 0.05
HYPER = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)


def reference(p, g, m, v, t, *, decoupled=True, maximize=False, vmax=None):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    if maximize:
        g = -g
    if decoupled:
        p = p * (1 - LR * WD)
    else:
        g = g + WD * p
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    w = v if vmax is None else torch.maximum(v, vmax.double())
    up = LR / (1 - B1 ** t) * m / ((w / (1 - B2 ** t)).sqrt() + EPS)
    return p - up, m, v, up, g, w


def close(got, want, bound, what):
    got = got.detach().cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    got, want, bound = got[fine], want[fine], bound[fine]
    over = ((got - want).abs() - bound).max().item() if want.numel() else 0.0
    assert over <= 0, f"{what}: over its bound by {over}"


def check_step(p0, g, m0, v0, t, p, m, v, dtype):
    """p, m, v after the step that began at p0, m0, v0 (CPU tensors)."""
    rp, rm, rv, up, _, _ = reference(p0, g, m0, v0, t)
    gd = g.double().abs()
    close(m, rm, 5 * U * (m0.double().abs() + gd) + 1e-44, "m")
    close(v, rv, 6 * U * rv + 1e-44, "v")
    # the update inherits m's error, up to 5 U (|m0| + |g|) / |m| of it
    spread = LR / (1 - B1 ** t) * (m0.double().abs() + gd) / ((rv / (1 - B2 ** t)).sqrt() + EPS)
    bound = 3 * U * p0.double().abs() + 12 * U * up.abs() + 5 * U * spread + 1e-44
    close(p, rp, bound + torch.finfo(dtype).eps / 2 * (rp.abs() + bound) * (dtype != torch.float32) + (6e-8 if dtype == torch.float16 else 0), "p")


def rand(shape, g, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


SHAPES = [(1,), (255,), (256,), (257,), (33, 65), (8192,), (8193,), (3, 5, 7, 11), (0,), (100, 300)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_adamw_32_bit_moments(ocl, dtype):
    gen = torch.Generator().manual_seed(1)
    ps = [rand(s, gen, 0.5, dtype) for s in SHAPES]
    dev = [p.to(DEV).requires_grad_() for p in ps]
    opt = ocl.optim.AdamW(dev, **HYPER)
    ms, vs = [torch.zeros(s) for s in SHAPES], [torch.zeros(s) for s in SHAPES]
    for t in range(1, 4):
        gs = [rand(s, gen, 0.1, dtype) for s in SHAPES]
        for d, g in zip(dev, gs):
            d.grad = g.to(DEV)
        opt.step()
        for p, g, m, v, d in zip(ps, gs, ms, vs, dev):
            s = opt.state[d]
            check_step(p, g, m, v, t, d, s["exp_avg"], s["exp_avg_sq"], dtype)
            assert s["exp_avg"].dtype == torch.float32 and s["step"].item() == t
        # the next step begins from what the device holds
        ps = [d.detach().cpu() for d in dev]
        ms, vs = ([opt.state[d][k].cpu() for d in dev] for k in ("exp_avg", "exp_avg_sq"))


def test_adamw_many_unaligned_tensors(ocl):
    """300 tensors (more than one launch takes) at odd addresses."""
    gen = torch.Generator().manual_seed(2)
    sizes = [1 + (37 * i) % 701 for i in range(300)]
    flat = {k: rand((sum(sizes) + 1,), gen, 0.3) for k in "pgmv"}
    flat["v"] = flat["v"].abs()
    held = {k: x.to(DEV) for k, x in flat.items()}
    at, params, views = 1, [], []
    opt = None
    for n in sizes:
        view = {k: held[k][at:at + n] for k in held}
        view["p"].grad = view["g"]
        params.append(view["p"])
        views.append((at, n, view))
        at += n
    opt = ocl.optim.AdamW(params, **HYPER)
    for (_, _, w), p in zip(views, params):
        opt.state[p] = {"step": torch.full((), 4.0).to(DEV), "exp_avg": w["m"], "exp_avg_sq": w["v"]}
    opt.step()
    check_step(flat["p"][1:], flat["g"][1:], flat["m"][1:], flat["v"][1:], 5, held["p"][1:], held["m"][1:], held["v"][1:],
               torch.float32)
    for k in "pmv":  # what is before the first tensor stays
        assert held[k][0].item() == flat[k][0].item()


def test_adamw_channels_last_and_other_gradient_layout(ocl):
    gen = torch.Generator().manual_seed(3)
    p0, g0 = rand((6, 5, 4, 3), gen), rand((6, 5, 4, 3), gen)
    p = p0.to(DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    opt = ocl.optim.AdamW([p], **HYPER)
    p.grad = g0.to(DEV)
    opt.step()
    zero = torch.zeros_like(p0)
    check_step(p0, g0, zero, zero, 1, p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"], torch.float32)


# ---------------------------------------------------------------- 8-bit moments
def encode(y, mantissa):
    n = y.numel()
    y = torch.nn.functional.pad(y.reshape(-1), (0, -n % 256)).view(-1, 256)
    s = y.abs().amax(1, keepdim=True) * torch.tensor(1.0 / (2.0 - 2.0 ** -mantissa))
    r = torch.where(s > 0, y / s, torch.zeros(()))
    bits = (r.abs() * 2.0 ** -112).view(torch.int32)
    drop = 23 - mantissa
    code = ((bits + (2 ** (drop - 1) - 1) + ((bits >> drop) & 1)) >> drop).clamp(max=16 * 2 ** mantissa - 1)
    code = torch.where(r < 0, code | 128, code) if mantissa == 3 else torch.where((y > 0) & (code == 0), 1, code)
    return code.to(torch.uint8).view(-1)[:n], s.view(-1)


def decode(code, s, mantissa):
    c = code.to(torch.int32)
    top = c & 127 if mantissa == 3 else c
    y = (top << (23 - mantissa)).view(torch.float32) * 2.0 ** 112 * s.repeat_interleave(256)[:c.numel()]
    return torch.where(c > 127, -y, y) if mantissa == 3 else y


def root(x):
    # the nearest fp32 number to the root: torch's fp32 root on the CPU is a vector library's and may be one off in the
    # last place; by way of float64 it is not (53 bits >= 2 * 24 + 2, so rounding twice is rounding once)
    return x.double().sqrt().float()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_adamw_8_bit_moments(ocl, dtype):
    gen = torch.Generator().manual_seed(4)
    shapes = SHAPES + [(513, 9)]
    ps = [rand(s, gen, 0.5, dtype) for s in shapes]
    dev = [p.to(DEV).requires_grad_() for p in ps]
    opt = ocl.optim.AdamW(dev, **HYPER, state_bits=8)
    states = [[torch.zeros(p.numel(), dtype=torch.uint8), torch.zeros(-(-p.numel() // 256))] * 2 for p in ps]
    f = torch.tensor  # coefficients as fp32
    for t in range(1, 5):
        # sizes that differ by element, some of them zero, one block of zeros
        gs = [(rand(s, gen) * torch.exp(4 * rand(s, gen))).to(dtype) for s in shapes]
        gs = [torch.where(g.abs() < 0.05, torch.zeros((), dtype=dtype), g) for g in gs]
        gs[5][256:512] = 0
        for d, g in zip(dev, gs):
            d.grad = g.to(DEV)
        opt.step()
        for k, (p, g, d) in enumerate(zip(ps, gs, dev)):
            if not p.numel():
                continue
            cm, sm, cu, su = states[k]
            m0, u0 = decode(cm, sm, 3), decode(cu, su, 4)
            gf = g.float().reshape(-1)
            m = m0 * f(B1) + gf * f(1 - B1)
            u = root(u0 * u0 * f(B2) + gf * gf * f(1 - B2))
            want = [*encode(m, 3), *encode(u, 4)]
            s = opt.state[d]
            got = [s[key].cpu() for key in ("exp_avg_code", "exp_avg_scale", "exp_avg_rms_code", "exp_avg_rms_scale")]
            for a, b, what in zip(got, want, ("codes of m", "scales of m", "codes of u", "scales of u")):
                assert ((a == b) | ((a != a) & (b != b))).all(), f"step {t}, tensor {k}: {what}"
            rp, rm, rv, up, _, _ = reference(p.reshape(-1), gf, m0, u0 * u0, t)
            spread = LR / (1 - B1 ** t) * (m0.double().abs() + gf.double().abs()) / ((rv / (1 - B2 ** t)).sqrt() + EPS)
            bound = 3 * U * p.double().abs().reshape(-1) + 14 * U * up.abs() + 5 * U * spread + 1e-44
            bound = bound + torch.finfo(dtype).eps / 2 * (rp.abs() + bound) * (dtype != torch.float32) + (6e-8 if dtype == torch.float16 else 0)
            close(d.reshape(-1), rp, bound, f"p of tensor {k} at step {t}")
            # a stored moment is half a step of its code off at most (below 2^-14 s the step is fixed; a root that is
            # not zero is one step off at most)
            hm, hu = decode(got[0], got[1], 3).double(), decode(got[2], got[3], 4).double()
            # (a gradient that fp16 cannot hold is infinite, and its block's moments are no numbers from then on)
            at = torch.isfinite(hm) & torch.isfinite(hu) & torch.isfinite(rm) & torch.isfinite(rv)
            assert at.all() or dtype == torch.float16
            hm, hu, rm, rv = hm[at], hu[at], rm[at], rv[at]
            step = got[1].double().repeat_interleave(256)[:at.numel()][at]
            assert ((hm - rm).abs() <= rm.abs() * 2.0 ** -4 * (1 + 1e-5) + step * 2.0 ** -18 * (1 + 1e-5) + 1e-44).all()
            step = got[3].double().repeat_interleave(256)[:at.numel()][at]
            assert ((hu - rv.sqrt()).abs() <= rv.sqrt() * 2.0 ** -5 * (1 + 1e-5) + step * 2.0 ** -18 * (1 + 1e-5) + 1e-44).all()
            assert ((hu > 0) == (u.double()[at] > 0)).all()
            states[k] = got
        ps = [d.detach().cpu() for d in dev]
    outs = [[torch.empty(p.shape).to(DEV) for p in ps] for _ in range(2)]
    opt.write_state_values(*outs)
    for k, (cm, sm, cu, su) in enumerate(states):
        if ps[k].numel():
            assert torch.allclose(outs[0][k].cpu().reshape(-1), decode(cm, sm, 3), rtol=0, atol=0, equal_nan=True)
            assert torch.allclose(outs[1][k].cpu().reshape(-1), decode(cu, su, 4).square(), rtol=0, atol=0, equal_nan=True)


def test_adamw_8_bit_extremes(ocl):
    """A block with one huge and otherwise tiny gradients, the least and the largest magnitudes, and a NaN that stays in
    its own block."""
    n = 256 * 4
    g = torch.full((n,), 1e-6)
    g[0] = 1e6
    g[256:512] = 1e-30
    g[512:768] = 1e18
    g[800] = float("nan")
    p = torch.ones(n).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], **HYPER, state_bits=8)
    p.grad = g.to(DEV)
    opt.step()
    m, v = torch.empty(n).to(DEV), torch.empty(n).to(DEV)
    opt.write_state_values([m], [v])
    want = (g * torch.tensor(1 - B1), root(g * g * torch.tensor(1 - B2)))
    for got, y, bits in ((m, want[0], 3), (v, want[1], 4)):
        ref = decode(*encode(y, bits), bits)
        ref = ref if bits == 3 else ref.square()
        assert torch.equal(got.cpu()[:768], ref[:768])
        assert torch.isnan(got.cpu()[768:]).all()
    assert torch.isfinite(p[:768].detach().cpu()).all()
    assert (v.cpu()[1:256] > 0).all()  # roots far below the block's largest stay above zero
    assert torch.isnan(p.detach().cpu()[800])


# ---------------------------------------------------------------- torch's fused optimizers
@pytest.mark.parametrize("cls", [torch.optim.AdamW, torch.optim.Adam], ids=["AdamW", "Adam"])
@pytest.mark.parametrize("amsgrad", [False, True])
@pytest.mark.parametrize("maximize", [False, True])
def test_torch_fused_optimizers(ocl, cls, amsgrad, maximize):
    gen = torch.Generator().manual_seed(5)
    ps = [rand(s, gen) for s in SHAPES]
    dev = [p.to(DEV).requires_grad_() for p in ps]
    kw = dict(HYPER, amsgrad=amsgrad, maximize=maximize)
    opt = cls(dev, fused=True, **kw)
    state = [(torch.zeros(s), torch.zeros(s), torch.zeros(s) if amsgrad else None) for s in SHAPES]
    launches = torch.ocl.kernel_launch_count()
    for t in range(1, 4):
        gs = [rand(s, gen, 0.2) for s in SHAPES]
        for d, g in zip(dev, gs):
            d.grad = g.to(DEV)
        opt.step()
        for p, g, d, (m, v, x) in zip(ps, gs, dev, state):
            rp, rm, rv, up, ge, w = reference(p, g, m, v, t, decoupled=cls is torch.optim.AdamW, maximize=maximize, vmax=x)
            s = opt.state[d]
            # Adam's gradient has a product and a sum of its own (2 roundings of its terms)
            ge = ge.abs() + WD * p.double().abs() + g.double().abs()
            close(s["exp_avg"], rm, 7 * U * (m.double().abs() + ge), "m")
            dv = 6 * U * rv + 4 * U * (1 - B2) * ge * ge
            close(s["exp_avg_sq"], rv, dv, "v")
            if amsgrad:
                close(s["max_exp_avg_sq"], w, dv + 6 * U * w, "max v")
            root = (w / (1 - B2 ** t)).sqrt() + EPS
            scale = LR / (1 - B1 ** t)
            # the update's error from v's: half of it, relative to w
            bound = 3 * U * p.double().abs() + 12 * U * up.abs() + 7 * U * scale * (m.double().abs() + ge) / root + up.abs() * dv / (2 * w + 1e-300)
            close(d, rp, 1.01 * bound, "p")
        ps = [d.detach().cpu() for d in dev]
        state = [(opt.state[d]["exp_avg"].cpu(), opt.state[d]["exp_avg_sq"].cpu(),
                  opt.state[d]["max_exp_avg_sq"].cpu() if amsgrad else None) for d in dev]
    # a step is the step counts, the factors and one launch over all tensors
    assert torch.ocl.kernel_launch_count() - launches <= 3 * (3 + 2 * len(SHAPES))


def _raw(op, p, g, m, v, step, **kw):
    args = dict(lr=LR, beta1=B1, beta2=B2, weight_decay=WD, eps=EPS, amsgrad=False, maximize=False)
    args.update(kw)
    op([p], [g], [m], [v], [], [step], **args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_fused_adamw_gradient_scale_found_inf_and_tensor_lr(ocl, dtype):
    gen = torch.Generator().manual_seed(6)
    p0, g0, m0, v0 = (rand((1000,), gen, 0.3, dtype) for _ in range(4))
    v0 = v0.abs()
    op = torch.ops.aten._fused_adamw_
    p, g, m, v = (x.to(DEV) for x in (p0, (g0.float() * 128).to(dtype), m0, v0))
    step, scale = torch.full((), 7.0).to(DEV), torch.full((), 128.0).to(DEV)
    _raw(op, p, g, m, v, step, grad_scale=scale, found_inf=torch.ones(()).to(DEV))
    for a, b in ((p, p0), (m, m0), (v, v0)):  # a step that is skipped changes nothing
        assert torch.equal(a.cpu(), b)
    _raw(op, p, g, m, v, step, grad_scale=scale, found_inf=torch.zeros(()).to(DEV), lr=torch.full((), LR).to(DEV))
    assert torch.equal(g.cpu(), g0)  # powers of two: unscaled exactly, and written back
    rp, rm, rv, up, _, _ = reference(p0, g0, m0, v0, 7)
    h = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = 6e-8 if dtype == torch.float16 else 0.0
    big = m0.double().abs() + g0.double().abs()
    close(m, rm, (5 * U + h) * big + tiny, "m")
    close(v, rv, (6 * U + h) * rv * 1.01 + tiny, "v")
    # lr as an fp32 value on the device is off by one rounding
    spread = LR / (1 - B1 ** 7) * big / ((rv / (1 - B2 ** 7)).sqrt() + EPS)
    bound = 4 * U * p0.double().abs() + 14 * U * up.abs() + 5 * U * spread
    close(p, rp, bound + h * (rp.abs() + bound) + tiny, "p")


def test_captured_step_advances_like_eager_steps(ocl):
    for bits in (32, 8):
        gen = torch.Generator().manual_seed(7)
        ps = [rand(s, gen) for s in SHAPES]
        gs = [rand(s, gen, 0.1) for s in SHAPES]
        results = []
        for captured in (False, True):
            dev = [p.to(DEV).requires_grad_() for p in ps]
            opt = ocl.optim.AdamW(dev, **HYPER, state_bits=bits)
            for d, g in zip(dev, gs):
                d.grad = g.to(DEV)
            opt.step()
            if captured:
                graph = torch.ocl.Graph()
                with graph.capture():
                    opt.step()
                for _ in range(3):
                    graph.replay()
            else:
                for _ in range(3):
                    opt.step()
            results.append([d.detach().cpu() for d in dev] + [v.cpu() for d in dev for v in opt.state[d].values()])
            if captured:
                graph.reset()
        for a, b in zip(*results):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(ocl, bits):
    gen = torch.Generator().manual_seed(8)
    ps = [rand(s, gen, 1.0, torch.bfloat16) for s in SHAPES[:5]]
    gs = [rand(s, gen, 0.1, torch.bfloat16) for s in SHAPES[:5]]

    def make(values):
        dev = [p.to(DEV).requires_grad_() for p in values]
        for d, g in zip(dev, gs):
            d.grad = g.to(DEV)
        return dev, ocl.optim.AdamW(dev, **HYPER, state_bits=bits)

    dev, opt = make(ps)
    opt.step()
    saved = opt.state_dict()
    saved = {"state": {i: {k: v.cpu().clone() for k, v in s.items()} for i, s in saved["state"].items()},
             "param_groups": saved["param_groups"]}
    dev2, opt2 = make([d.detach().cpu() for d in dev])
    opt2.load_state_dict(saved)
    opt.step()
    opt2.step()
    for a, b in zip(dev, dev2):
        assert torch.equal(a.cpu(), b.cpu())
        for k, v in opt.state[a].items():
            assert v.dtype == opt2.state[b][k].dtype and torch.equal(v.cpu(), opt2.state[b][k].cpu())
    other = ocl.optim.AdamW(dev, **HYPER, state_bits=40 - bits)
    with pytest.raises(ValueError, match="state of parameter"):
        other.load_state_dict(saved)


def test_torch_fused_with_gradients_of_another_layout(ocl):
    gen = torch.Generator().manual_seed(10)
    p0, g0 = rand((6, 5, 4, 3), gen), rand((6, 5, 4, 3), gen)
    p = p0.to(DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    opt = torch.optim.AdamW([p], fused=True, **HYPER)
    p.grad = g0.to(DEV)
    opt.step()
    zero = torch.zeros_like(p0)
    check_step(p0, g0, zero, zero, 1, p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"], torch.float32)


def test_copies_keep_their_kind_of_state(ocl):
    import copy

    p = torch.randn(300).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], state_bits=8)
    twin = copy.deepcopy(opt)
    assert twin.state_bits == 8
    q = twin.param_groups[0]["params"][0]
    p.grad, q.grad = torch.ones(300).to(DEV), torch.ones(300).to(DEV)
    opt.step()
    twin.step()
    assert torch.equal(p.detach().cpu(), q.detach().cpu()) and "exp_avg_code" in twin.state[q]


def test_closure_groups_and_parameters_without_gradient(ocl):
    a, b, c = (torch.ones(50).to(DEV).requires_grad_() for _ in range(3))
    h = torch.ones(40, dtype=torch.bfloat16).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([{"params": [a, h]}, {"params": [b, c], "lr": 0.5, "weight_decay": 0.0}], lr=0.25, weight_decay=0.0)
    assert opt.step() is None  # no gradients yet: nothing happens, and no state appears
    assert not opt.state
    c.grad = None

    def closure():
        opt.zero_grad()
        loss = (a * 2.0).sum() + (b * 3.0).sum() + (h * 1.0).sum()
        loss.backward()
        return loss

    assert opt.step(closure).item() == 50 * 2 + 50 * 3 + 40
    # a first step moves by lr times the gradient's sign
    for t, want in ((a, 0.75), (b, 0.5), (h, 0.75), (c, 1.0)):
        assert (t.detach().cpu().float() - want).abs().max() <= 1e-6
    assert c not in opt.state or not opt.state[c]


def test_refusals(ocl):
    p = torch.zeros(8).to(DEV).requires_grad_()
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=4)):
        with pytest.raises(ValueError):
            ocl.optim.AdamW([p], **bad)
    with pytest.raises(ValueError, match="twice"):
        ocl.optim.AdamW([p, p])
    with pytest.raises(ValueError, match="ocl device expected"):
        ocl.optim.AdamW([torch.zeros(3, requires_grad=True)])
    base = torch.zeros(8, 8).to(DEV)
    gap = base[:, :4]  # rows with gaps between them
    gap.grad = torch.zeros(8, 4).to(DEV)
    with pytest.raises(RuntimeError, match="gaps or overlaps"):
        ocl.optim.AdamW([gap]).step()
    q = torch.zeros(4).to(DEV)
    for kw, match in ((dict(g=torch.zeros(5).to(DEV)), "another shape"), (dict(g=torch.zeros(4)), "ocl:0"),
                      (dict(m=torch.zeros(4, dtype=torch.float16).to(DEV)), "moments"),
                      (dict(step=torch.zeros(())), "step")):
        args = dict(p=q, g=torch.zeros(4).to(DEV), m=torch.zeros(4).to(DEV), v=torch.zeros(4).to(DEV),
                    step=torch.ones(()).to(DEV))
        args.update(kw)
        with pytest.raises(RuntimeError, match=match):
            _raw(torch.ops.aten._fused_adamw_, **args)
    z = [torch.zeros(4).to(DEV) for _ in range(4)]
    with pytest.raises(RuntimeError, match="listed twice"):
        torch.ops.aten._fused_adamw_([z[0], z[0]], [z[1]] * 2, [z[2]] * 2, [z[3]] * 2, [], [torch.ones(()).to(DEV)] * 2, lr=LR,
                                     beta1=B1, beta2=B2, weight_decay=0.0, eps=EPS, amsgrad=False, maximize=False)


def test_on_another_stream(ocl):
    """The step runs on the current stream, behind what was queued there."""
    gen = torch.Generator().manual_seed(9)
    p0, g0 = rand((100003,), gen), rand((100003,), gen)
    p, g = p0.to(DEV).requires_grad_(), g0.to(DEV)
    opt = ocl.optim.AdamW([p], **HYPER)
    torch.ocl.synchronize()
    stream = torch.Stream(device=DEV)
    with stream:
        p.grad = g * 2.0
        opt.step()
    stream.synchronize()
    zero = torch.zeros_like(p0)
    s = opt.state[p]
    check_step(p0, g0 * 2, zero, zero, 1, p, s["exp_avg"], s["exp_avg_sq"], torch.float32)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_in_another_memory_order_is_refused(ocl, bits):
    """Moments lie in memory as their parameter did: after a change of its memory order they belong to other elements."""
    gen = torch.Generator().manual_seed(11)
    p0, g0 = rand((6, 5, 4, 3), gen), rand((6, 5, 4, 3), gen)
    formats = (torch.contiguous_format, torch.channels_last)
    for first, then in (formats, formats[::-1]):
        p = p0.to(DEV).contiguous(memory_format=first).requires_grad_()
        opt = ocl.optim.AdamW([p], **HYPER, state_bits=bits)
        p.grad = g0.to(DEV).contiguous(memory_format=first)
        opt.step()
        held = p.detach().cpu().clone()
        saved = opt.state_dict()
        # a program that goes on in the old order, from a checkpoint too
        q = held.to(DEV).contiguous(memory_format=first).requires_grad_()
        twin = ocl.optim.AdamW([q], **HYPER, state_bits=bits)
        twin.load_state_dict(saved)
        q.grad = g0.to(DEV)
        twin.step()
        # and one that changes it, as module.to(memory_format=...) does
        p.data = p.data.contiguous(memory_format=then)
        with pytest.raises(RuntimeError, match="does not fit"):
            opt.step()
        out = [torch.empty_like(p, memory_format=torch.preserve_format) for _ in range(2)]
        if bits == 8:
            with pytest.raises(RuntimeError, match="does not fit"):
                opt.write_state_values([out[0].detach()], [out[1].detach()])
        assert torch.equal(p.detach().cpu(), held)
        r = held.to(DEV).contiguous(memory_format=then).requires_grad_()
        other = ocl.optim.AdamW([r], **HYPER, state_bits=bits)
        r.grad = g0.to(DEV)
        with pytest.raises((RuntimeError, ValueError), match="fit"):
            other.load_state_dict(saved)
            other.step()
        # back in its order the state goes on as if nothing had been
        p.data = p.data.contiguous(memory_format=first)
        opt.step()
        assert torch.equal(p.detach().cpu(), q.detach().cpu())


def test_8_bit_moments_in_any_dense_order(ocl):
    """A channels-last parameter takes the steps that the same numbers take in a row."""
    gen = torch.Generator().manual_seed(12)
    p0 = rand((9, 8, 7, 5), gen)
    p = p0.to(DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    flat = p0.permute(0, 2, 3, 1).contiguous().view(-1).to(DEV).requires_grad_()
    one, two = (ocl.optim.AdamW([v], **HYPER, state_bits=8) for v in (p, flat))
    for _ in range(3):
        g = rand((9, 8, 7, 5), gen, 0.1)
        p.grad, flat.grad = g.to(DEV), g.permute(0, 2, 3, 1).contiguous().view(-1).to(DEV)
        one.step()
        two.step()
    assert torch.equal(p.detach().cpu().permute(0, 2, 3, 1).reshape(-1), flat.detach().cpu())
    m, v = (torch.empty_like(p, memory_format=torch.preserve_format).detach() for _ in range(2))
    mf, vf = (torch.empty_like(flat).detach() for _ in range(2))
    one.write_state_values([m], [v])
    two.write_state_values([mf], [vf])
    for a, b in ((m, mf), (v, vf)):
        assert torch.equal(a.cpu().permute(0, 2, 3, 1).reshape(-1), b.cpu())


def test_a_refused_group_is_not_added(ocl):
    p, q = torch.ones(8).to(DEV).requires_grad_(), torch.ones(8).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], **HYPER)
    for bad, match in ((dict(params=[q, q]), "twice"), (dict(params=[q, torch.ones(3, requires_grad=True)]), "ocl device expected"),
                       (dict(params=[torch.ones(3, dtype=torch.float64, device="cpu", requires_grad=True)]), "expected")):
        with pytest.raises(ValueError, match=match):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1 and opt.param_groups[0]["params"] == [p]
    q.grad = p.grad = torch.ones(8).to(DEV)
    opt.step()
    assert (q.detach().cpu() == 1).all() and (p.detach().cpu() != 1).all()
    opt.add_param_group({"params": [q]})
    opt.step()
    assert (q.detach().cpu() != 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_is_refused_changes_nothing(ocl, bits):
    gen = torch.Generator().manual_seed(13)
    ps = [rand(s, gen, 1.0, torch.bfloat16) for s in ((300,), (20, 30))]

    def make(lr, state_bits):
        dev = [p.to(DEV).requires_grad_() for p in ps]
        opt = ocl.optim.AdamW(dev, lr=lr, state_bits=state_bits)
        for d in dev:
            d.grad = torch.ones_like(d)
        opt.step()
        return opt

    opt, good = make(0.125, bits), make(0.25, bits).state_dict()
    cut = {"state": {k: dict(v) for k, v in good["state"].items()}, "param_groups": good["param_groups"]}
    key = "exp_avg_sq" if bits == 32 else "exp_avg_rms_scale"
    cut["state"][1][key] = cut["state"][1][key].reshape(-1)[:1]
    number = {"state": {k: dict(v) for k, v in good["state"].items()}, "param_groups": good["param_groups"]}
    number["state"][0]["step"] = 3
    before = {p: {k: v.cpu().clone() for k, v in s.items()} for p, s in opt.state.items()}
    for bad in (make(0.25, 40 - bits).state_dict(), cut, number):
        with pytest.raises(ValueError, match="state of parameter"):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 0.125 and set(opt.state) == set(before)
        for p, s in before.items():
            assert set(opt.state[p]) == set(s)
            for k, v in s.items():
                assert torch.equal(opt.state[p][k].cpu(), v) and opt.state[p][k].dtype == v.dtype
    seen = []
    opt.register_load_state_dict_post_hook(lambda o: seen.append({k: v.dtype for k, v in o.state[o.param_groups[0]["params"][0]].items()}))
    opt.load_state_dict(good)
    assert opt.param_groups[0]["lr"] == 0.25
    assert seen == [{k: v.dtype for k, v in good["state"][0].items()}]  # whole when a hook sees it


def test_loading_takes_no_more_memory_than_the_state(ocl):
    p = torch.zeros(1 << 22, dtype=torch.float32).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    saved = opt.state_dict()
    torch.ocl.synchronize()
    torch.ocl.reset_peak_memory_stats()
    before = torch.ocl.memory_allocated()
    opt.load_state_dict(saved)
    # two tensors of 4 MB and two of 64 KB; their fp32 form would take 16 MB each
    assert torch.ocl.max_memory_allocated() - before <= 10 << 20


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_step_is_not_captured(ocl, bits):
    """What a graph would replay of it is the zeroed state, again and again."""
    p, q = (torch.ones(300).to(DEV).requires_grad_() for _ in range(2))
    opt = ocl.optim.AdamW([p, q], **HYPER, state_bits=bits)
    p.grad = torch.ones(300).to(DEV)
    q.grad = None

    def captured():
        graph = torch.ocl.Graph()
        with graph.capture():
            opt.step()
        return graph

    with pytest.raises(RuntimeError, match="before it is captured"):
        captured()
    assert not any(opt.state.values())
    opt.step()
    q.grad = torch.ones(300).to(DEV)  # a parameter that takes part for the first time
    with pytest.raises(RuntimeError, match="before it is captured"):
        captured()
    opt.step()
    graph = captured()
    graph.replay()
    graph.replay()
    assert opt.state[p]["step"].item() == 4 and opt.state[q]["step"].item() == 3
    graph.reset()


@pytest.mark.parametrize("bits", [32, 8])
def test_lookups_that_run_python(ocl, bits):
    """A parameter's hash is Python code, in which gradients and states of others may go away: a state that was found
    before stays alive until the step is done, and a parameter whose gradient went is left as it is."""
    import gc

    at_last = []

    class Leaf(torch.nn.Parameter):
        def __hash__(self):
            if at_last and self is params[3]:
                at_last.pop()()
            return super().__hash__()

    params = []
    params.extend(Leaf(torch.ones(70000 + i).to(DEV)) for i in range(4))
    opt = ocl.optim.AdamW(params, **HYPER, state_bits=bits)
    for p in params:
        p.grad = torch.full_like(p, 2.0)
    opt.step()
    outs = [[torch.zeros(p.shape).to(DEV) for p in params] for _ in range(2)]

    def drop():
        for p in params[:3]:
            del opt.state[p]
        params[0].grad = None
        params[1].grad = params[1].grad * 1.0
        gc.collect()
        # whatever was freed is written over
        junk = [torch.full((70000 + i,), float("nan")).to(DEV) for i in range(4) for _ in range(6)]
        del junk

    if bits == 8:
        kept = dict(opt.state)
        at_last.append(drop)
        opt.write_state_values(*outs)
        for m, v in zip(*outs):  # (1 - B1) 2 and (1 - B2) 4 to half a step of their codes, twice that for a square
            assert ((m.cpu() / (2 * (1 - B1)) - 1).abs() <= 2.0 ** -4).all()
            assert ((v.cpu() / (4 * (1 - B2)) - 1).abs() <= 2.0 ** -3).all()
        opt.state.update(kept)
        del kept
        for p in params:
            p.grad = torch.full_like(p, 2.0)
    before = [p.detach().cpu().clone() for p in params]
    at_last.append(drop)
    opt.step()
    assert torch.equal(params[0].detach().cpu(), before[0])
    for p, b in zip(params[1:], before[1:]):
        after = p.detach().cpu()
        assert torch.isfinite(after).all() and (after < b).all()
    assert list(opt.state) == params[3:]
    p = params[0]
    p.grad = torch.full_like(p, 2.0)  # its next step is a first one
    opt.step()
    assert opt.state[p]["step"].item() == 1


def test_a_refused_step_changes_nothing(ocl):
    """Of parameters of several types, one whose state does not fit: the others are not updated before the refusal."""
    a = torch.ones(300).to(DEV).requires_grad_()
    b = torch.ones(300, dtype=torch.bfloat16).to(DEV).requires_grad_()
    for bits, key in ((32, "exp_avg"), (8, "exp_avg_scale")):
        opt = ocl.optim.AdamW([a, b], **HYPER, state_bits=bits)
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        opt.step()
        held = a.detach().cpu().clone()
        opt.state[b][key] = torch.zeros(7).to(DEV)
        with pytest.raises(RuntimeError, match="does not fit"):
            opt.step()
        assert torch.equal(a.detach().cpu(), held) and opt.state[a]["step"].item() == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_could_not_be_made_is_made_again(ocl, monkeypatch, bits):
    """Memory that runs out while a state is made leaves none behind, and the next step makes it."""
    p = torch.ones(300).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], **HYPER, state_bits=bits)
    p.grad = torch.ones(300).to(DEV)
    made, zeros, zeros_like = [], torch.zeros, torch.zeros_like

    def limited(f):
        def call(*args, **kw):
            made.append(1)
            if len(made) == 2:
                raise RuntimeError("out of memory")
            return f(*args, **kw)
        return call

    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", limited(zeros))
        m.setattr(torch, "zeros_like", limited(zeros_like))
        with pytest.raises(RuntimeError, match="out of memory"):
            opt.step()
    assert (p.detach().cpu() == 1).all()
    opt.step()
    assert opt.state[p]["step"].item() == 1 and (p.detach().cpu() < 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_maximize_is_the_step_along_the_negated_gradient(ocl, bits):
    gen = torch.Generator().manual_seed(14)
    ps = [rand(s, gen) for s in SHAPES]
    up, down = ([p.to(DEV).requires_grad_() for p in ps] for _ in range(2))
    one = ocl.optim.AdamW(up, **HYPER, state_bits=bits, maximize=True)
    two = ocl.optim.AdamW(down, **HYPER, state_bits=bits)
    for _ in range(3):
        for a, b in zip(up, down):
            g = rand(a.shape, gen, 0.1)
            a.grad, b.grad = g.to(DEV), (-g).to(DEV)
        one.step()
        two.step()
    for a, b, p in zip(up, down, ps):
        assert torch.equal(a.detach().cpu(), b.detach().cpu())
        assert not p.numel() or not torch.equal(a.detach().cpu(), p)
        for k, v in one.state[a].items():
            assert torch.equal(v.cpu(), two.state[b][k].cpu())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_of_other_types_is_refused_when_it_is_loaded(ocl, bits):
    """torch's optimizers keep moments in the parameters' type: refused at once, not by the next step."""
    p = torch.ones(300, dtype=torch.bfloat16).to(DEV).requires_grad_()
    opt = ocl.optim.AdamW([p], **HYPER, state_bits=bits)
    p.grad = torch.ones_like(p)
    opt.step()
    held = {k: v.cpu().clone() for k, v in opt.state[p].items()}
    saved = opt.state_dict()
    for key in held:
        other = {"state": {0: dict(saved["state"][0])}, "param_groups": saved["param_groups"]}
        other["state"][0][key] = other["state"][0][key].cpu().to(torch.bfloat16)
        with pytest.raises(ValueError, match="state of parameter 0"):
            opt.load_state_dict(other)
        assert all(torch.equal(opt.state[p][k].cpu(), v) for k, v in held.items())
    opt.step()
    if bits == 32:
        q = torch.ones(300, dtype=torch.bfloat16).to(DEV).requires_grad_()
        theirs = torch.optim.AdamW([q], fused=True, **HYPER)
        q.grad = torch.ones_like(q)
        theirs.step()
        with pytest.raises(ValueError, match="state of parameter 0"):
            opt.load_state_dict(theirs.state_dict())
