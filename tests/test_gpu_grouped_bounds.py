"""Grouped products and 8-bit floating point at the bounds of what they are given (GPU): steps that are smaller than what their groups were filled for, what lies
behind the values of a row, a part of a packed weight, two host threads at once."""
import math
import threading

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


def rnd(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + 31 * len(shape) + shape[-1]))


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("cut", [0, 16121, 128211])
@pytest.mark.parametrize("by_pair", [False, True])
def test_a_smaller_step_whose_groups_are_a_larger_ones(ops, kind, cut, by_pair):
    """Whatever the groups say: no row that the smaller step does not have is read, and none is written."""
    rows, top, groups, n, k, few = 300, 2, 5, 130, 200, 7
    room = ops.row_groups(rows, top, groups, DEV)
    ops.group_rows(torch.randint(0, groups, (rows, top), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV), room)
    part = room.first(few)
    weight = rnd(groups, n, k).to(DEV)
    have = few * top if by_pair else few
    if kind == "fp8":
        w, held = ops.quantize_weight_fp8(weight), ops.fp8_rows(have + 400, k, DEV)
        ops.quantize_fp8(torch.full((have + 400, k), math.nan, device=DEV), held)
        ops.quantize_fp8(rnd(have, k).to(DEV), held[:have])
    else:
        w, held = ops.pack_grouped(weight.to(torch.bfloat16)), torch.full((have + 400, k), math.nan, dtype=torch.bfloat16, device=DEV)
        held[:have] = rnd(have, k).to(DEV)
    out = torch.full((few * top + 400, n), 5.0, device=DEV)
    ops.gemm_grouped(held[:have], w, part, out[:few * top], by_pair=by_pair, cut=cut)
    assert out[:few * top].isfinite().all() and (out[few * top:] == 5).all()
    answers = torch.full((few * top + 700, 24), math.nan, device=DEV)
    answers[:few * top] = 1
    summed = torch.full((few, 24), 7.0, device=DEV)
    ops.combine_groups(answers[:few * top], part, torch.ones((few, top), device=DEV), summed)
    assert summed.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 5, 100, 127, 129, 500, 1003])
def test_what_is_behind_a_row_stays_and_is_not_read(ops, cols, dtype):
    """The bytes between a row's last value and the next row: not written by the rounding, and no product takes them in (they are NaN here)."""
    rows, n = 9, 70
    wide = torch.full((rows, -(-cols // 16) * 16 + 32), 0x7f, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    rows8 = ops.Fp8Rows(wide[:, :cols], torch.empty((rows, -(-cols // 512) * 4), device=DEV))
    x = rnd(rows, cols).to(dtype).to(DEV)
    ops.quantize_fp8(x, rows8)
    assert (wide.view(torch.uint8)[:, cols:] == 0x7f).all()
    room8 = ops.fp8_rows(rows, cols, DEV)
    ops.quantize_fp8(x, room8)
    assert torch.equal(room8.data.view(torch.uint8), rows8.data.view(torch.uint8)) and torch.equal(room8.scale, rows8.scale)
    weight = rnd(n, cols).to(DEV)
    w, several = ops.quantize_weight_fp8(weight), ops.quantize_weight_fp8(weight[None].expand(3, n, cols))
    alone = torch.empty((rows, n), device=DEV)
    for cut in (16121, 32121, 64121, 128211):
        ops.gemm_fp8(rows8, w, alone, cut=cut)
        assert alone.isfinite().all()
        room, out = ops.row_groups(rows, 1, 3, DEV), torch.empty((rows, n), device=DEV)
        ops.group_rows((torch.arange(rows, dtype=torch.int32) % 3)[:, None].to(DEV), room)
        ops.gemm_grouped(rows8, several, room, out, cut=cut)
        assert torch.equal(out[room.place.flatten().long()], alone)


def test_a_part_of_a_packed_weight(ops):
    n, k = 700, 1000
    w = ops.quantize_weight_fp8(rnd(n, k).to(DEV))
    for rows in (3, 60, 200):
        rows8 = ops.fp8_rows(rows, k, DEV)
        ops.quantize_fp8(rnd(rows, k).to(DEV), rows8)
        whole = torch.empty((rows, n), device=DEV)
        for cut in (16121, 128211):
            ops.gemm_fp8(rows8, w, whole, cut=cut)
            for lo, hi in ((0, 700), (128, 290), (512, 513), (640, 700)):
                out = torch.full((rows, hi - lo + 3), 9.0, device=DEV)
                ops.gemm_fp8(rows8, w.take_rows(lo, hi), out[:, :hi - lo], cut=cut)
                assert torch.equal(out[:, :hi - lo], whole[:, lo:hi]) and (out[:, hi - lo:] == 9).all()


def test_two_host_threads_at_once(ops):
    """Each with a stream, sizes and tensors of its own."""
    wrong = []

    def work(seed):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            w = ops.quantize_weight_fp8(rnd(300 + seed, 640, seed=seed).to(DEV))
            packed = ops.pack_grouped(rnd(4, 136, 64, seed=seed).to(torch.bfloat16).to(DEV))
            first = {}
            for turn in range(20):
                for rows in (1 + seed, 40, 150 + seed):
                    rows8, out = ops.fp8_rows(rows, 640, DEV), torch.empty((rows, 300 + seed), device=DEV)
                    ops.quantize_fp8(rnd(rows, 640, seed=seed).to(DEV), rows8)
                    ops.gemm_fp8(rows8, w, out)
                    room, answers = ops.row_groups(rows, 2, 4, DEV), torch.empty((2 * rows, 136), device=DEV)
                    ops.group_rows((torch.arange(2 * rows, dtype=torch.int32).view(rows, 2) % 4).to(DEV), room)
                    ops.gemm_grouped(rnd(rows, 64, seed=seed).to(torch.bfloat16).to(DEV), packed, room, answers)
                    both = torch.cat([out.flatten(), answers.flatten()]).cpu()
                    if not torch.equal(first.setdefault(rows, both), both):
                        wrong.append((seed, turn, rows))

    threads = [threading.Thread(target=work, args=(seed,)) for seed in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


def test_first_calls_inside_a_capture(ops):
    """Sizes that no call had before: what a first call asks of the driver may be asked while a stream is captured."""
    rows, n, k = 37, 1111, 1313
    x, w = rnd(rows, k).to(DEV), ops.quantize_weight_fp8(rnd(n, k).to(DEV))
    packed = ops.pack_grouped(rnd(11, 152, 88).to(torch.bfloat16).to(DEV))
    few = rnd(rows, 88).to(torch.bfloat16).to(DEV)
    choice = (torch.arange(rows * 2, dtype=torch.int32).view(rows, 2) % 11).to(DEV)
    rows8, room = ops.fp8_rows(rows, k, DEV), ops.row_groups(rows, 2, 11, DEV)
    out, answers, summed = torch.zeros((rows, n), device=DEV), torch.zeros((2 * rows, 152), device=DEV), torch.zeros((rows, 152), device=DEV)
    share = torch.full((rows, 2), 0.5, device=DEV)

    def step():
        ops.quantize_fp8(x, rows8)
        ops.gemm_fp8(rows8, w, out)
        ops.group_rows(choice, room)
        ops.gemm_grouped(few, packed, room, answers)
        ops.combine_groups(answers, room, share, summed)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    torch.cuda.synchronize()
    replayed = [t.clone() for t in (out, answers, summed)]
    for t in (out, answers, summed):
        t.zero_()
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and a.any() for a, b in zip(replayed, (out, answers, summed)))
