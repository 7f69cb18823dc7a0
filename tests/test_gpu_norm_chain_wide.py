"""The norms between two parts at the widest rows that one block holds (GPU), in a process of its own, since what a kernel has asked for of shared memory it keeps.

Tolerance: a row's sum of squares has 48 terms a thread and eight steps over the block, all positive: 56 halves of 2^-23, half of that behind the root; with the
products' roundings below 2^-18 of the magnitudes that are added. Twice that for each of the two norms that follow one another."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import sys
import torch
from jllm_serve_b200.csrc import ops
ops.require_device()
dim, kind = int(sys.argv[1]), getattr(torch, sys.argv[2])
g, eps, rows, dev = torch.Generator().manual_seed(dim), 1e-5, 3, "cuda:0"
x, a, b = (torch.randn(rows, dim, generator=g) for _ in range(3))
ga, gb, gp, gn = (1 + 0.1 * torch.randn(dim, generator=g) for _ in range(4))
def norm(v, gain):
    return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) * gain
for two in (False, True):
    xd, nxt = x.to(dev), torch.empty(rows, dim, dtype=kind, device=dev)
    more = dict(b=b.to(dev), gain_a=ga.to(dev), gain_b=gb.to(dev), scale=0.5) if two else {}
    ops.norm_chain(xd, a.to(dev), gp.to(dev), eps, next_out=nxt, gain_next=gn.to(dev), **more)
    ad, bd = a.double(), b.double()
    v = 0.5 * (norm(ad, ga) + norm(bd, gb)) if two else ad
    size = 0.5 * (norm(ad, ga).abs() + norm(bd, gb).abs()) if two else ad.abs()
    factor = 1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) * gp.abs()
    total = x.double() + norm(v, gp)
    off_total = 2.0 ** -17 * (x.double().abs() + size * factor)
    assert ((xd.cpu().double() - total).abs() <= off_total).all(), two
    after = 1 / torch.sqrt((total * total).mean(dim=1, keepdim=True) + eps) * gn.abs()
    want = norm(total, gn)
    slack = off_total * after + 2.0 ** -17 * want.abs()
    assert ((nxt.cpu().double() - want).abs() <= slack + (want.abs() + slack) * torch.finfo(kind).eps / 2).all(), two
print("as wide as that")
"""


@pytest.mark.parametrize("dim", [12288, 12287, 12257, 12250, 8193])
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_widest_rows(dim, kind):
    proc = subprocess.run([sys.executable, "-c", PROGRAM, str(dim), kind], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "as wide as that" in proc.stdout, proc.stderr[-2000:]
