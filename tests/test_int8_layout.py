"""The layout of 8-bit weights and rows, and what is refused of them (CPU)."""
import pytest
import torch

from jllm_serve_b200.csrc import ops


def weight(rows, cols):
    g = torch.Generator().manual_seed(rows + cols)
    return torch.randint(-128, 128, (rows, cols), generator=g, dtype=torch.int8), torch.rand((rows,), generator=g)


@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (129, 127), (300, 500), (16, 1000)])
def test_packing_goes_back(rows, cols):
    w, scale = weight(rows, cols)
    packed = ops.pack_int8(w, scale)
    assert packed.shape == (rows, cols) and torch.equal(packed.unpack(), w) and torch.equal(packed.scale, scale)
    assert packed.data.shape == (-(-rows // 128), -(-cols // 128), 128, 128)
    # row r of a tile is 128 bytes, its 16-byte chunk c at chunk position c ^ (r & 7)
    r, k = rows - 1, cols - 1
    tile = packed.data[r // 128, k // 128].view(128, 8, 16)
    assert tile[r % 128, (k % 128 // 16) ^ (r & 7), k % 16] == w[r, k]
    assert int(packed.data.long().abs().sum()) == int(w.long().abs().sum())          # filled up with zeros


def test_gate_and_up_rows_interleave_in_eights():
    w, scale = weight(48, 20)
    packed = ops.pack_int8(w, scale, glu=True)
    order = [b * 8 + i + half for b in range(3) for half in (0, 24) for i in range(8)]
    assert torch.equal(packed.unpack(), w[order]) and torch.equal(packed.scale, scale[order])


def test_rows_begin_at_16_bytes():
    rows8 = ops.int8_rows(3, 17, "cpu")
    assert rows8.shape == (3, 17) and rows8.stride == 32 and rows8[1:].shape == (2, 17)
    assert ops.int8_rows(0, 5, "cpu").shape == (0, 5)
    one = ops.Int8Rows(torch.zeros(1, 17, dtype=torch.int8), torch.zeros(1))          # a single row's stride says nothing
    assert one.stride == 32


def test_refusals():
    zeros = torch.zeros
    for call in (lambda: ops.Int8Rows(zeros(3, 16), zeros(3)),
                 lambda: ops.Int8Rows(zeros(3, 16, dtype=torch.int8), zeros(2)),
                 lambda: ops.Int8Rows(zeros(3, 17, dtype=torch.int8), zeros(3)),                    # rows of 17 bytes
                 lambda: ops.Int8Rows(zeros(16, 16, dtype=torch.int8).T, zeros(16)),
                 lambda: ops.Int8Rows(zeros(4, 33, dtype=torch.int8)[:, 1:], zeros(4)),
                 lambda: ops.Int8Rows(zeros(3, 16, dtype=torch.int8), zeros(3, 2)[:, 0]),
                 lambda: ops.int8_rows(3, 16, "cpu")[1],
                 lambda: ops.pack_int8(zeros(3, 16), zeros(3)),
                 lambda: ops.pack_int8(zeros(3, 16, dtype=torch.int8), zeros(4)),
                 lambda: ops.pack_int8(zeros(0, 16, dtype=torch.int8), zeros(0)),
                 lambda: ops.pack_int8(zeros(24, 16, dtype=torch.int8), zeros(24), glu=True),
                 lambda: ops.pack_int8(zeros(1, ops.INT8_MAX_K + 1, dtype=torch.int8), zeros(1))):
        with pytest.raises(ops.KernelError):
            call()


def test_settings_of_the_command_line(tmp_path):
    from jllm_serve_b200.cli import Settings, SettingsError
    load = lambda *args: Settings.load(list(args), env={}, cwd=tmp_path).validate()      # noqa: E731
    assert load().get("backend.weights") == "" and load("--weights", "int8").get("backend.weights") == "int8"
    for args in (("--weights", "int4"), ("--weights", "int8", "--dtype", "fp32")):
        with pytest.raises(SettingsError):
            load(*args)
