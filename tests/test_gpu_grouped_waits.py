"""The waits of the grouped products that are made to run out (GPU): the kernel gives up by the clock, says which wait it was, leaves nothing on its way
to memory that it has given back, and what is launched behind it is right."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_b200.csrc import ops as o
    o.require_device()
    o.check_kernel_errors()
    return o


def product(ops, kind, rows, width, dim, groups=0):
    """(call(out, cut), exact result): whole numbers whose sums stay below 2^24, so that float32 has them exactly."""
    g = torch.Generator().manual_seed(rows + width + dim)
    a = torch.randint(-8, 9, (rows, dim), generator=g).float()
    w = torch.randint(-8, 9, (max(groups, 1), width, dim), generator=g).float()
    if kind == "fp8":
        a8 = ops.fp8_rows(rows, dim, DEV)
        a8.data.copy_(a.to(torch.float8_e4m3fn))
        a8.scales.fill_(0.5)
        packed = ops.pack_fp8(w.to(torch.float8_e4m3fn).to(DEV), torch.full((w.shape[0], -(-width // 128), -(-dim // 128)), 0.25, device=DEV))
        rows_, factor = a8, 0.125
    else:
        packed, rows_, factor = ops.pack_grouped(w.to(torch.bfloat16).to(DEV)), a.to(torch.bfloat16).to(DEV), 1.0
    if not groups:
        return (lambda out, cut: ops.gemm_fp8(rows_, packed, out, cut=cut)), factor * (a.double() @ w[0].double().T).float()
    choice = torch.arange(rows, dtype=torch.int32)[:, None] % groups
    room = ops.row_groups(rows, 1, groups, DEV)
    ops.group_rows(choice.to(DEV), room)
    order = torch.sort(choice[:, 0], stable=True).indices
    want = torch.stack([factor * (a[r].double() @ w[int(choice[r, 0])].double().T) for r in order.tolist()]).float()
    return (lambda out, cut: ops.gemm_grouped(rows_, packed, room, out, cut=cut)), want


# A wait for the other roles of the block lasts twice as long as the MMAs' wait for a copy, so which wait runs out first is known: with a ring that
# holds all k blocks a stage that is not released is missed by the producer alone, behind a right result; with a shorter one the k block that would come
# next is what the MMAs miss first.
@pytest.mark.parametrize("what,cut,rows,dim,code", [
    ("copy", 32121, 20, 1024, 42), ("copy", 16111, 9, 1024, 42), ("copy", 32124, 20, 1024, 42), ("copy", 128211, 100, 1024, 42), ("copy", 64121, 60, 640, 42),
    ("release", 32111, 20, 1024, 41), ("release", 32121, 20, 1024, 42), ("release", 128211, 100, 1024, 42), ("release", 128211, 100, 256, 41),
    ("parts", 32122, 20, 1024, 43), ("parts", 16128, 16, 1024, 43), ("parts", 16114, 3, 512, 43), ("parts", 128212, 100, 512, 43),
    ("parts", 128214, 20, 640, 43), ("copy", 128212, 100, 512, 42)])
def test_a_wait_that_runs_out_returns_and_is_reported(ops, what, cut, rows, dim, code):
    run, want = product(ops, "fp8", rows, 256, dim)
    ops.gemm_grouped_starve_next(what)
    run(torch.empty(rows, 256, device=DEV), cut)
    out = torch.empty(rows, 256, device=DEV)
    run(out, cut)                                       # (launched while the starved one still waits)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError, match=rf"bounded wait ran out inside gemm_grouped \(code {code}\)"):
        ops.check_kernel_errors()
    assert torch.equal(out.cpu(), want)
    again = torch.empty(rows, 256, device=DEV)
    run(again, cut)
    torch.cuda.synchronize()
    ops.check_kernel_errors()
    assert torch.equal(again.cpu(), want)


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("what,cut", [("copy", 16121), ("copy", 128211), ("release", 32121), ("release", 128211)])
def test_groups_whose_wait_runs_out(ops, kind, what, cut):
    run, want = product(ops, kind, 40, 256, 2048, groups=3)
    ops.gemm_grouped_starve_next(what)
    run(torch.empty(40, 256, device=DEV), cut)
    out = torch.empty(40, 256, device=DEV)
    run(out, cut)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError, match="inside gemm_grouped"):
        ops.check_kernel_errors()
    assert torch.equal(out.cpu(), want)
    ops.check_kernel_errors()


def test_a_short_limit_does_not_disturb_a_product_that_misses_nothing(ops):
    run, want = product(ops, "fp8", 40, 256, 1024)
    for cut in (16121, 32124, 64111, 128211, 128212, 128214):
        out = torch.empty(40, 256, device=DEV)
        ops.gemm_grouped_starve_next("nothing", 2000)
        run(out, cut)
        ops.check_kernel_errors()
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("cut", [16121, 32124, 128211])
def test_what_the_kernel_in_front_takes_is_not_waited_for(ops, cut):
    """A row of 2^27 values takes one block some 16 ms, and lets the product's blocks begin at once: a limit of 1 ms counts from there on."""
    run, want = product(ops, "fp8", 20, 256, 1024)
    out = torch.empty(20, 256, device=DEV)
    run(out, cut)
    row, row8 = torch.ones(1, 1 << 27, dtype=torch.bfloat16, device=DEV), ops.int8_rows(1, 1 << 27, DEV)
    began, ended = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    out.zero_()
    began.record()
    ops.quantize_int8(row, row8)
    ops.gemm_grouped_starve_next("nothing", 1000)
    run(out, cut)
    ended.record()
    torch.cuda.synchronize()
    assert began.elapsed_time(ended) > 4.0
    ops.check_kernel_errors()
    assert torch.equal(out.cpu(), want)


def test_refusals(ops):
    for limit in (0, -1, 2000000):
        with pytest.raises(ops.KernelError):
            ops.gemm_grouped_starve_next("copy", limit)
    run, _ = product(ops, "fp8", 20, 256, 1024)
    ops.gemm_grouped_starve_next("parts")
    with pytest.raises(ops.KernelError):               # a block alone has nobody who could send
        run(torch.empty(20, 256, device=DEV), 32121)
    for cut in (64122, 128213, 128218, 128222, 128111, 48121, 16129, 16131, 32101):      # no kernel, no cluster, no such number of blocks
        with pytest.raises(ops.KernelError):
            run(torch.empty(20, 256, device=DEV), cut)
    run(torch.empty(20, 256, device=DEV), 32121)
    ops.check_kernel_errors()
