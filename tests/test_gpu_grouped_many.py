"""Grouped products of hundreds of groups in the wide kernel, whose lists of groups leave its ring a stage less (GPU): every cut gives a pair's result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    yield o
    o.check_kernel_errors()


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("by_pair", [False, True])
@pytest.mark.parametrize("cut", [0, 16121, 64121, 128211])
@pytest.mark.parametrize("groups,rows,top", [(256, 700, 3), (257, 90, 8), (1024, 500, 2), (1024, 1500, 4)])
def test_many_groups(ops, kind, by_pair, cut, groups, rows, top):
    """Whole numbers, whose sums float32 has exactly; a few groups have many pairs, some none."""
    n, k = 200, 640
    g = torch.Generator().manual_seed(groups + rows)
    score = torch.rand(rows, groups, generator=g)
    score[:, :3] += 0.6
    choice = score.topk(top, dim=1).indices.to(torch.int32)
    choice[5] = -1
    m = rows * top if by_pair else rows
    a, w = torch.randint(-8, 9, (m, k), generator=g).float(), torch.randint(-8, 9, (groups, n, k), generator=g).float()
    if kind == "fp8":
        held = ops.fp8_rows(m, k, DEV)
        held.data.copy_(a.to(torch.float8_e4m3fn))
        held.scales.fill_(0.5)
        packed, factor = ops.pack_fp8(w.to(torch.float8_e4m3fn).to(DEV), torch.full((groups, 2, 5), 0.25, device=DEV)), 0.125
    else:
        held, packed, factor = a.to(torch.bfloat16).to(DEV), ops.pack_grouped(w.to(torch.bfloat16).to(DEV)), 1.0
    room = ops.row_groups(rows, top, groups, DEV)
    ops.group_rows(choice.to(DEV), room)
    flat = choice.flatten().long()
    key = torch.where(flat < 0, groups, flat)
    order = torch.sort(key, stable=True).indices[:int((flat >= 0).sum())]
    out = torch.full((rows * top, n), 5.0, device=DEV)
    ops.gemm_grouped(held, packed, room, out, by_pair=by_pair, cut=cut)
    rows_of = torch.arange(len(order)) if by_pair else order // top
    expert = flat[order]
    want = torch.empty(len(order), n)
    for e in expert.unique().tolist():
        there = expert == e
        want[there] = a[rows_of[there]] @ w[e].T * factor
    assert torch.equal(out[:len(order)].cpu(), want) and (out[len(order):] == 5).all()
