"""Counts of groups at which grouping rows needs almost all of the shared memory that a launch has without asking (GPU): a first call in a process of its own, since what
a kernel has asked for once it keeps."""
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
pairs = int(sys.argv[1])
for groups in map(int, sys.argv[2].split(",")):
    choice = torch.randint(-1, groups, (pairs, 1), generator=torch.Generator().manual_seed(groups)).to(torch.int32)
    room = ops.row_groups(pairs, 1, groups, "cuda:0")
    ops.group_rows(choice.cuda(), room)
    key = torch.where(choice[:, 0] < 0, groups, choice[:, 0].long())
    order, asked = torch.sort(key, stable=True).indices, int((choice >= 0).sum())
    assert room.offsets[-1].item() == asked and torch.equal(room.order[:asked].cpu().long(), order[:asked]) and (room.order[asked:] == -1).all()
    assert torch.equal(room.place.cpu()[order[:asked], 0].long(), torch.arange(asked))
ops.check_kernel_errors()
print("all were grouped")
"""


@pytest.mark.parametrize("pairs,groups", [(300, "615,616,617,618,619,620"), (700, "318,319,320,321,322"), (1500, "290,291,292,293"), (30000, "291,292,293"),
                                          (300000, "349,350,351,352"), (200, "1023,1024")])
def test_counts_next_to_what_a_launch_has(pairs, groups):
    proc = subprocess.run([sys.executable, "-c", PROGRAM, str(pairs), groups], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and "all were grouped" in proc.stdout, proc.stderr[-2000:]
