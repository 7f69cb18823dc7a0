"""Grouped products and 8-bit floating point called by several host threads at once, and for the first time in a process while a stream is captured (GPU)."""
import subprocess
import sys
import textwrap
import threading
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


class Work:
    """A thread's weights and inputs; a pass gives all its results."""

    def __init__(self, ops, seed):
        g = torch.Generator().manual_seed(seed)
        self.ops, self.n = ops, 300 + 13 * seed
        self.w, self.gated = ops.quantize_weight_fp8(torch.randn(self.n, 1640, generator=g).to(DEV)), ops.quantize_weight_fp8(torch.randn(4, 272, 640, generator=g).to(DEV), glu=True)
        self.packed = ops.pack_grouped(torch.randn(4, 136, 64, generator=g).to(torch.bfloat16).to(DEV))
        self.inputs = [(torch.randn(rows, 1640, generator=g).to(DEV), torch.randn(rows, 64, generator=g).to(torch.bfloat16).to(DEV),
                        torch.randint(-1, 4, (rows, 2), generator=g).to(torch.int32).to(DEV)) for rows in (1 + seed, 40, 150 + seed, 1100)]

    def run(self):
        ops, results = self.ops, []
        for x, few, choice in self.inputs:
            rows = x.shape[0]
            rows8, narrow8, out = ops.fp8_rows(rows, 1640, DEV), ops.fp8_rows(rows, 640, DEV), torch.empty((rows, self.n), device=DEV)
            ops.quantize_fp8(x, rows8)
            ops.gemm_fp8(rows8, self.w, out)
            room = ops.row_groups(rows, 2, 4, DEV)
            answers, units = torch.zeros((2 * rows, 136), device=DEV), torch.zeros((2 * rows, 136), device=DEV)
            total = torch.empty((rows, 136), device=DEV)
            ops.group_rows(choice, room)
            ops.gemm_grouped(few, self.packed, room, answers)
            ops.quantize_fp8(x[:, :640], narrow8)
            ops.gemm_grouped(narrow8, self.gated, room, units, swiglu="silu")
            ops.combine_groups(answers, room, torch.ones((rows, 2), device=DEV), total)
            results += [out, answers, units, total, ops.fp8_values(rows8, torch.empty_like(x))]
        return results


def test_host_threads_at_once(ops):
    """Every pass of every thread gives the bits that it gives alone; an exception in a thread is the test's."""
    threads, turns = 3, 20
    works = [Work(ops, seed) for seed in range(threads)]
    want = [w.run() for w in works]
    torch.cuda.synchronize()
    begin = threading.Barrier(threads)

    def work(i):
        done = 0
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            begin.wait(timeout=60)
            for _ in range(turns):
                assert all(torch.equal(a, b) for a, b in zip(works[i].run(), want[i]))
                done += 1
        return done

    with ThreadPoolExecutor(threads) as pool:
        assert [f.result(timeout=300) for f in [pool.submit(work, i) for i in range(threads)]] == [turns] * threads


FIRST = """
import torch
from jllm_serve_b200.csrc import ops
ops.require_device()
DEV = "cuda:0"
g = torch.Generator().manual_seed(3)
n, k = 320, 1313
w, gated = ops.quantize_weight_fp8(torch.randn(n, k, generator=g).to(DEV)), ops.quantize_weight_fp8(torch.randn(n, k, generator=g).to(DEV), glu=True)
packed = ops.pack_grouped(torch.randn(11, 152, 88, generator=g).to(torch.bfloat16).to(DEV))
experts = ops.quantize_weight_fp8(torch.randn(11, 144, 88, generator=g).to(DEV), glu=True)
steps = []
for rows, cut in ((1, 0), (20, 16128), (37, 32124), (60, 64121), (130, 128211), (130, 128214), (2500, 0)):
    x, few = torch.randn(rows, k, generator=g).to(DEV), torch.randn(rows, 88, generator=g).to(DEV)
    choice = torch.randint(-1, 11, (rows, 2), generator=g).to(torch.int32).to(DEV)
    rows8, few8, room = ops.fp8_rows(rows, k, DEV), ops.fp8_rows(rows, 88, DEV), ops.row_groups(rows, 2, 11, DEV)
    kept = [torch.zeros(shape, device=DEV, dtype=t) for shape, t in (((rows, n), torch.float32), ((rows, n // 2), torch.bfloat16), ((2 * rows, 152), torch.float32),
                                                                     ((2 * rows, 72), torch.bfloat16), ((rows, 152), torch.float32), ((rows, k), torch.float32))]
    steps.append((rows, cut, x, few.to(torch.bfloat16), few, choice, rows8, few8, room, torch.full((rows, 2), 0.5, device=DEV), kept))

def run():
    for rows, cut, x, few, few32, choice, rows8, few8, room, share, kept in steps:
        grouped = cut if cut % 10 == 1 else 0
        ops.quantize_fp8(x, rows8)
        ops.quantize_fp8(few32, few8)
        ops.gemm_fp8(rows8, w, kept[0], cut=cut)
        ops.gemm_fp8(rows8, gated, kept[1], swiglu="silu", cut=cut)
        ops.group_rows(choice, room)
        ops.gemm_grouped(few, packed, room, kept[2], cut=grouped)
        ops.gemm_grouped(few8, experts, room, kept[3], swiglu="silu", cut=grouped)
        ops.combine_groups(kept[2], room, share, kept[4])
        ops.fp8_values(rows8, kept[5])

torch.cuda.synchronize()
before = ops.launch_count
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()
assert ops.launch_count - before == 9 * len(steps)
graph.replay()
torch.cuda.synchronize()
replayed = [t.clone() for s in steps for t in s[-1]]
for s in steps:
    for t in s[-1]:
        t.zero_()
run()
torch.cuda.synchronize()
for i, (a, t) in enumerate(zip(replayed, [t for s in steps for t in s[-1]])):
    assert torch.equal(a, t) and bool(a.any()) == bool(t.any()), i
ops.check_kernel_errors()
print("first calls were captured")
"""


def test_the_first_calls_of_a_process_are_captured():
    """What the library asks the driver once (a kernel's own shared memory and its opt-in, how many clusters run at a time) it asks here while a stream is captured."""
    proc = subprocess.run([sys.executable, "-c", textwrap.dedent(FIRST)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "first calls were captured" in proc.stdout, proc.stdout[-2000:] + proc.stderr[-3000:]
