"""The layout of packed groups' weights and of rows in 8-bit floating point, and what is refused of them (CPU)."""
import pytest
import torch

from jllm_serve_b200.csrc import ops


def e4m3(*shape):
    g = torch.Generator().manual_seed(sum(shape))
    return (100 * torch.randn(shape, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 128, 128), (3, 129, 127), (1, 300, 500), (4, 16, 1000)])
def test_packing_goes_back(shape):
    w, scale = e4m3(*shape), torch.rand((shape[0], -(-shape[1] // 128), -(-shape[2] // 128)))
    packed = ops.pack_fp8(w, scale)
    assert packed.shape == shape[1:] and packed.groups == shape[0] and torch.equal(packed.unpack().view(torch.uint8), w.view(torch.uint8))
    G, T, KB = shape[0], -(-shape[1] // 128), -(-shape[2] // 128)
    assert packed.data.shape == (G, T, KB, 128, 128) and packed.scales.shape == (G, 16 * T, -(-KB // 4) * 4)
    for r in {0, shape[1] - 1, shape[1] // 2}:          # every eight rows have the scale of their block
        assert torch.equal(packed.scales[:, r // 8, :KB], scale[:, r // 128])
    # row r of a tile is 128 bytes, its 16-byte chunk c at chunk position c ^ (r & 7)
    r, k = shape[1] - 1, shape[2] - 1
    tile = packed.data[-1, r // 128, k // 128].view(128, 8, 16)
    assert tile[r % 128, (k % 128 // 16) ^ (r & 7), k % 16] == w.view(torch.int8)[-1, r, k]


@pytest.mark.parametrize("shape", [(1, 128, 64), (2, 130, 72), (3, 16, 8), (1, 1, 1000)])
def test_bfloat16_packing_goes_back(shape):
    w = torch.randn(shape).to(torch.bfloat16)
    packed = ops.pack_grouped(w)
    assert packed.k_blocks == -(-shape[2] // 64) and not packed.fp8 and torch.equal(packed.unpack(), w)


@pytest.mark.parametrize("hidden", [8, 24, 128, 136, 200])
def test_gate_and_up_rows_interleave_in_eights_with_their_own_scales(hidden):
    w, scale = e4m3(2, 2 * hidden, 260), torch.rand((2, -(-2 * hidden // 128), 3))
    packed = ops.pack_fp8(w, scale, glu=True)
    order = [b * 8 + i + half for b in range(hidden // 8) for half in (0, hidden) for i in range(8)]
    assert torch.equal(packed.unpack().view(torch.uint8), w[:, order].view(torch.uint8))
    for i, r in enumerate(order):
        assert torch.equal(packed.scales[:, i // 8, :3], scale[:, r // 128])


def test_a_weight_rounded_in_blocks():
    w = torch.randn(200, 300)
    w[128:, 128:256] = 0
    packed = ops.quantize_weight_fp8(w)
    scale = packed.scales[0, [0, 16], :3]
    values = packed.unpack()[0].float() * scale.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]
    # half a step of e4m3: 2^-4 of the value, or 2^-10 steps of the scale below its smallest normal value
    assert ((values - w).abs() <= w.abs() * 2.0 ** -4 * 1.0001 + scale.max() * 2.0 ** -10).all() and (values[128:, 128:256] == 0).all()
    assert packed.unpack()[0].float().abs().amax() == 448


def test_rows_begin_at_16_bytes():
    rows8 = ops.fp8_rows(3, 130, "cpu")
    assert rows8.shape == (3, 130) and rows8.data.stride(0) == 144 and rows8.scale.shape == (3, 2) and rows8.scales.shape == (3, 4)
    assert rows8[1:].shape == (2, 130) and rows8[3:].shape == (0, 130) and ops.fp8_rows(0, 5, "cpu").shape == (0, 5)


def test_refusals():
    f8, zeros = torch.float8_e4m3fn, torch.zeros
    bf = torch.bfloat16
    for call in (lambda: ops.Fp8Rows(zeros(3, 16), zeros(3, 4)),
                 lambda: ops.Fp8Rows(zeros(3, 16, dtype=f8), zeros(2, 4)),
                 lambda: ops.Fp8Rows(zeros(3, 16, dtype=f8), zeros(3, 1)),                       # scales in fours
                 lambda: ops.Fp8Rows(zeros(3, 1024, dtype=f8), zeros(3, 4)),                     # too few of them
                 lambda: ops.Fp8Rows(zeros(3, 17, dtype=f8), zeros(3, 4)),                       # rows of 17 bytes
                 lambda: ops.Fp8Rows(zeros(16, 16, dtype=f8).T[:, :8], zeros(16, 4)),
                 lambda: ops.Fp8Rows(zeros(3, 16, dtype=f8), zeros(3, 8)[:, :4]),
                 lambda: ops.fp8_rows(3, 16, "cpu")[1], lambda: ops.fp8_rows(4, 16, "cpu")[::2], lambda: ops.fp8_rows(-1, 16, "cpu"), lambda: ops.fp8_rows(1, 0, "cpu"),
                 lambda: ops.pack_fp8(zeros(3, 16), zeros(1, 1)),
                 lambda: ops.pack_fp8(zeros(3, 16, dtype=f8), zeros(2, 1)),
                 lambda: ops.pack_fp8(zeros(2, 3, 16, dtype=f8), zeros(1, 1)),
                 lambda: ops.pack_fp8(zeros(16, dtype=f8), zeros(1)),
                 lambda: ops.pack_fp8(zeros(0, 16, dtype=f8), zeros(0, 1)),
                 lambda: ops.pack_fp8(zeros(24, 16, dtype=f8), zeros(1, 1), glu=True),
                 lambda: ops.pack_grouped(zeros(2, 16, 12, dtype=bf)), lambda: ops.pack_grouped(zeros(2, 16, 16)), lambda: ops.pack_grouped(zeros(16, 16, dtype=bf)),
                 lambda: ops.pack_grouped(zeros(2, 8, 16, dtype=bf), glu=True),
                 lambda: ops.pack_grouped(zeros(ops.MOST_GROUPS + 1, 1, 8, dtype=bf)),
                 lambda: ops.quantize_weight_fp8(zeros(3, 3, dtype=torch.float16)), lambda: ops.quantize_weight_fp8(zeros(0, 3)),
                 lambda: ops.row_groups(3, 0, 4, "cpu"), lambda: ops.row_groups(-1, 1, 4, "cpu"), lambda: ops.row_groups(3, 2, 0, "cpu"),
                 lambda: ops.row_groups(3, 2, ops.MOST_GROUPS + 1, "cpu"), lambda: ops.row_groups(2 ** 30, 2, 4, "meta"), lambda: ops.row_groups(3, 2, 4, "cpu").first(4)):
        with pytest.raises(ops.KernelError):
            call()


def test_calls_are_refused_in_front_of_a_launch():
    """What does not fit together, and whatever does not lie on the current device."""
    bf, i32 = torch.bfloat16, torch.int32
    groups = ops.row_groups(4, 2, 3, "cpu")
    w8, w16 = ops.pack_fp8(e4m3(3, 32, 48), torch.ones(3, 1, 1)), ops.pack_grouped(torch.zeros(3, 32, 48, dtype=bf))
    one, glu = ops.pack_fp8(e4m3(32, 48), torch.ones(1, 1)), ops.pack_fp8(e4m3(32, 48), torch.ones(1, 1), glu=True)
    rows8, rows16, out = ops.fp8_rows(4, 48, "cpu"), torch.zeros(4, 48, dtype=bf), torch.zeros(8, 32)
    before = ops.launch_count
    for call in (lambda: ops.group_rows(torch.zeros(4, 2), groups), lambda: ops.group_rows(torch.zeros(4, 3, dtype=i32), groups),
                 lambda: ops.group_rows(torch.zeros(4, 2, dtype=i32), groups),                            # not on a GPU
                 lambda: ops.gemm_grouped(rows16, w8, groups, out), lambda: ops.gemm_grouped(rows8, w16, groups, out), lambda: ops.gemm_grouped(rows8, one, groups, out),
                 lambda: ops.gemm_grouped(rows8, w8, groups, out, by_pair=True), lambda: ops.gemm_grouped(rows8, w8, groups, out, swiglu="silu"),
                 lambda: ops.gemm_grouped(rows8, w8, groups, out), lambda: ops.gemm_grouped(rows16, w16, groups, out), lambda: ops.gemm_grouped(rows16, w16, groups, out.half()),
                 lambda: ops.gemm_fp8(rows8, w8, out), lambda: ops.gemm_fp8(rows8, one, out[:4]), lambda: ops.gemm_fp8(rows8, glu, out[:4, :16]),
                 lambda: ops.gemm_fp8(rows8, glu, out[:4, :16], swiglu=ops.GluUnits(1, 8)), lambda: ops.gemm_fp8(ops.fp8_rows(4, 40, "cpu"), one, out[:4]),
                 lambda: ops.quantize_fp8(rows16, rows8), lambda: ops.quantize_fp8(rows16.half(), rows8), lambda: ops.fp8_values(rows8, torch.zeros(4, 48)),
                 lambda: ops.combine_groups(out, groups, torch.zeros(4, 2), torch.zeros(4, 32)), lambda: ops.combine_groups(out, groups, torch.zeros(4, 2, dtype=bf), torch.zeros(4, 32))):
        with pytest.raises(ops.KernelError):
            call()
    assert ops.launch_count == before


def test_rows_of_a_packed_weight():
    w, scale = e4m3(300, 200), torch.rand(3, 2)
    packed = ops.pack_fp8(w, scale)
    part = packed.take_rows(128, 290)
    assert part.shape == (162, 200) and torch.equal(part.unpack()[0].view(torch.uint8), w[128:290].view(torch.uint8)) and torch.equal(part.scales[0, [0, 16], :2], scale[1:])
    for lo, hi in ((30, 100), (128, 128), (0, 301), (-128, 10)):
        with pytest.raises(ops.KernelError):
            packed.take_rows(lo, hi)


def test_settings_of_the_command_line(tmp_path):
    from jllm_serve_b200.cli import Settings, SettingsError
    load = lambda *args: Settings.load(list(args), env={}, cwd=tmp_path).validate()      # noqa: E731
    assert load("--weights", "fp8").get("backend.weights") == "fp8"
    for args in (("--weights", "fp4"), ("--weights", "fp8", "--dtype", "fp32")):
        with pytest.raises(SettingsError):
            load(*args)
