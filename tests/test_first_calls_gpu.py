"""First calls of a kernel from several threads at once: what a kernel needs set up once per device is done before any of
them launches it.  In a process of its own, where nothing has run yet."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import threading, torch
import pytorch_vulkan_b200 as pkg
from pytorch_vulkan_b200.functional import linear_cross_entropy
import torch.nn.functional as F

DEV, THREADS = "ocl:0", 8

def loss(dtype, N, D, V):
    g = torch.Generator().manual_seed(N)
    x, w = (torch.randn(n, D, generator=g).to(dtype).to(DEV) for n in (N, V))
    t = torch.randint(0, V, (N,), generator=g).to(DEV)
    return lambda: linear_cross_entropy(x, w, t)

def product():
    a = torch.ones(256, 512).to(DEV)
    return lambda: a @ a.t()

def convolution():
    a, b = torch.ones(8, 64, 14, 14).to(DEV), torch.ones(64, 64, 3, 3).to(DEV)
    return lambda: F.conv2d(a, b, padding=1)

def attention():
    q = torch.ones(2, 4, 197, 64).to(DEV)
    return lambda: F.scaled_dot_product_attention(q, q, q)

calls = [loss(torch.bfloat16, 300, 64, 3000), loss(torch.float16, 3, 64, 3000), loss(torch.float32, 300, 64, 3000),
         loss(torch.float32, 2, 1500, 500), product(), convolution(), attention()]
torch.ocl.synchronize()
for call in calls:
    barrier, results, errors = threading.Barrier(THREADS), [], []
    def work():
        barrier.wait()
        try:
            results.append(call())
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(THREADS)]
    for t in threads: t.start()
    for t in threads: t.join()
    assert not errors, errors[0]
    torch.ocl.synchronize()
    first = results[0].cpu()
    assert torch.isfinite(first).all() and all(torch.equal(first, r.cpu()) for r in results)
print("done")
"""


def test_first_calls_from_several_threads(ocl):
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", CODE], cwd=REPO, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stderr[-2000:]
