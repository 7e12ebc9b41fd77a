"""What a log probability and an entropy can be, at most 0 and at least 0, whatever the roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "ocl:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(4000, 33), (2000, 1000), (200, 20001), (300, 6001), (3, 100003)],
                         ids=lambda s: "-".join(map(str, s)))
def test_certain_tokens(ocl, shape, dtype):
    """Rows of which one token has all of the probability, by 40 and more or because a mask leaves no other."""
    N, V = shape
    g = torch.Generator().manual_seed(N + V)
    z = 3 * torch.randn(N, V, generator=g)
    t = torch.randint(0, V, (N,), generator=g)
    z[torch.arange(N), t] = 60 + 40 * torch.rand(N, generator=g)
    at = torch.arange(V)[None, :] == t[:, None]
    z[::3] = torch.where(at, z, float("-inf"))[::3]
    z = z.to(dtype)
    lp, H, tlp, tat = ocl.functional.token_log_probs(z.to(DEV), t.to(DEV), top=2)
    lp, H, tlp = lp.cpu(), H.cpu(), tlp.cpu()
    assert torch.equal(tat[:, 0].cpu(), t) and torch.equal(tlp[:, 0], lp)
    assert (lp <= 0).all() and (tlp <= 0).all(), (lp.max(), tlp.max())
    assert (H >= 0).all(), H.min()
    # the others have V e^-40 at most of it; exponentials of 2 u and what follows, a few u of 1 (u = 2^-24)
    assert (lp > -40 * 2.0 ** -24 - V * 1e-17).all() and (H < 40 * 2.0 ** -24 + V * 1e-15).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [7, 777, 40001])
def test_a_token_that_is_masked_itself(ocl, dtype, V):
    """Its log probability is -inf, and the formula's gradient, g ([j = t] - p_j) + k (..), leaves it g alone; other
    masked logits have none, and in a row of nothing else no logit has."""
    g = torch.Generator().manual_seed(V)
    N = 40
    z = torch.randn(N, V, generator=g).to(dtype)
    t = torch.randint(1, V, (N,), generator=g)
    z[torch.arange(N), t] = float("-inf")
    z[:, 0] = float("-inf")
    z[::9] = float("-inf")
    gl, gh = torch.randn(N, generator=g), torch.randn(N, generator=g)
    zd = z.to(DEV).requires_grad_()
    out = ocl.functional.token_log_probs(zd, t.to(DEV))
    assert (out[0].detach().cpu() == float("-inf")).all()
    (dz,) = torch.autograd.grad(out, zd, [gl.to(DEV), gh.to(DEV)])
    dz = dz.cpu()
    some = torch.ones(N, dtype=torch.bool)
    some[::9] = False
    assert torch.equal(dz[torch.arange(N), t][some], gl.to(dtype)[some]) and (dz[:, 0] == 0).all() and (dz[::9] == 0).all()
