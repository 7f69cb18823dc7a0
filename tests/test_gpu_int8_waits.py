"""The waits of the product in 8-bit integers that are made to run out (GPU): the kernel gives up by the clock, says which wait it was, leaves
nothing on its way to memory that it has given back, and what is launched behind it is right."""
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


def product(ops, rows, width, dim):
    g = torch.Generator().manual_seed(rows + width + dim)
    a, w = (torch.randint(-127, 128, (n, dim), generator=g, dtype=torch.int8) for n in (rows, width))
    a8 = ops.int8_rows(rows, dim, DEV)
    a8.data.copy_(a)
    a8.scale.fill_(2.0 ** -7)
    packed = ops.pack_int8(w.to(DEV), torch.full((width,), 0.5, device=DEV))
    # (the scales are powers of two and the sums below 2^24, so the float32 result is the exact one)
    return a8, packed, (a.double() @ w.double().T * 2.0 ** -8).float()


# A wait for the other roles of the block lasts twice as long as the MMAs' wait for a copy, so which wait runs out first is known: with a ring
# that holds all k blocks a stage that is not released is missed by the producer alone, behind a right result; with a shorter one the k block
# that would come next is what the MMAs miss first.
@pytest.mark.parametrize("what,cut,rows,dim,code", [
    ("copy", 1, 20, 1024, 32), ("copy", 11, 20, 1024, 32), ("copy", 4, 20, 1024, 32), ("copy", 18, 100, 1024, 32), ("copy", 1, 256, 256, 32),
    ("release", 11, 20, 1024, 31), ("release", 14, 20, 1024, 31), ("release", 1, 20, 1024, 32),
    ("parts", 2, 20, 1024, 33), ("parts", 18, 100, 1024, 33), ("parts", 14, 256, 512, 33)])
def test_a_wait_that_runs_out_returns_and_is_reported(ops, what, cut, rows, dim, code):
    a8, packed, want = product(ops, rows, 256, dim)
    ops.gemm_int8_starve_next(what)
    ops.gemm_int8(a8, packed, torch.empty(rows, 256, device=DEV), cut=cut)
    out = torch.empty(rows, 256, device=DEV)
    ops.gemm_int8(a8, packed, out, cut=cut)            # (launched while the starved one still waits)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError, match=rf"bounded wait ran out inside gemm_int8 \(code {code}\)"):
        ops.check_kernel_errors()
    assert torch.equal(out.cpu(), want)
    again = torch.empty(rows, 256, device=DEV)
    ops.gemm_int8(a8, packed, again, cut=cut)
    torch.cuda.synchronize()
    ops.check_kernel_errors()
    assert torch.equal(again.cpu(), want)


def test_a_short_limit_does_not_disturb_a_product_that_misses_nothing(ops):
    a8, packed, want = product(ops, 40, 256, 1024)
    for cut in (1, 4, 11):
        out = torch.empty(40, 256, device=DEV)
        ops.gemm_int8_starve_next("nothing", 2000)
        ops.gemm_int8(a8, packed, out, cut=cut)
        ops.check_kernel_errors()
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("cut", [1, 4, 11, 12])
def test_what_the_kernel_in_front_takes_is_not_waited_for(ops, cut):
    """A row of 2^27 values takes one block some 16 ms, and lets the product's blocks begin at once: a limit of 1 ms counts from there on."""
    a8, packed, want = product(ops, 20, 256, 1024)
    out = torch.empty(20, 256, device=DEV)
    ops.gemm_int8(a8, packed, out, cut=cut)
    row, row8 = torch.ones(1, 1 << 27, dtype=torch.bfloat16, device=DEV), ops.int8_rows(1, 1 << 27, DEV)
    began, ended = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    out.zero_()
    began.record()
    ops.quantize_int8(row, row8)
    ops.gemm_int8_starve_next("nothing", 1000)
    ops.gemm_int8(a8, packed, out, cut=cut)
    ended.record()
    torch.cuda.synchronize()
    assert began.elapsed_time(ended) > 4.0
    ops.check_kernel_errors()
    assert torch.equal(out.cpu(), want)


def test_refusals(ops):
    for limit in (0, -1, 2000000):
        with pytest.raises(ops.KernelError):
            ops.gemm_int8_starve_next("copy", limit)
    a8, packed, _ = product(ops, 20, 256, 1024)
    ops.gemm_int8_starve_next("parts")
    with pytest.raises(ops.KernelError):               # a block alone has nobody who could send
        ops.gemm_int8(a8, packed, torch.empty(20, 256, device=DEV), cut=1)
    ops.gemm_int8(a8, packed, torch.empty(20, 256, device=DEV), cut=1)
    ops.check_kernel_errors()
