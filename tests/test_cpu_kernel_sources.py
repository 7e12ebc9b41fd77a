"""Rules of the kernels' sources that no run would show to be broken before it hangs or reads too early."""
import glob
import os
import re

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch_vulkan_b200", "csrc", "kernels")
SOURCES = sorted(glob.glob(os.path.join(KERNELS, "*.cu")) + glob.glob(os.path.join(KERNELS, "*.cuh")))


def code(path):
    """A source without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def kernels(text):
    """(name, body) of each __global__ function."""
    for m in re.finditer(r"__global__[^;{]*?(\w+)\s*\((?:[^(){}]|\([^()]*\))*\)\s*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m[1], text[m.end():at]


def overlapped():
    return [(os.path.basename(p), name, body) for p in SOURCES for name, body in kernels(code(p)) if "let_next_come()" in body]


def test_launches_that_begin_early_wait():
    found = overlapped()
    assert len(found) >= 10
    for path, name, body in found:
        assert "wait_for_last()" in body, (path, name)


def test_the_next_launch_comes_after_tensor_memory_is_had():
    """A launch that came earlier could take this block's tensor memory and hold it until this block has ended, which
    waits for it."""
    with_memory = [(p, n, b) for p, n, b in overlapped() if "tmem_alloc" in b]
    assert {n for _, n, _ in with_memory} == {"linear8_kernel", "linear8_few_kernel"}
    for path, name, body in with_memory:
        had = body.rindex("tmem_alloc")
        come = body.index("let_next_come()")
        assert had < come and "__syncthreads" in body[had:come], (path, name)


def test_arrivals_at_another_blocks_barrier_have_the_clusters_scope():
    """Without one an arrival has its own block's, in which the other block does not take part."""
    arrivals = [(os.path.basename(p), m[0]) for p in SOURCES for m in re.finditer(r"mbarrier\.arrive[\w.:]*shared::cluster\S*", code(p))]
    assert len(arrivals) >= 2
    for path, text in arrivals:
        assert re.match(r"mbarrier\.arrive(\.expect_tx)?\.(release|relaxed)\.cluster\.", text), (path, text)
