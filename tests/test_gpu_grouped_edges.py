"""Grouped products and 8-bit floating point where they can go wrong (GPU): captured and replayed, on other streams, one behind the other on the same buffers,
matrices beyond 2^31 values, every significand of bfloat16, calls that the launchers refuse."""
import ctypes

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


class Layer:
    """A layer of experts with its buffers, as a serving program holds it."""

    def __init__(self, ops, kind, rows, top=3, groups=9, dim=256, hidden=72, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.ops, self.kind, self.rows, self.top, self.groups_n, self.dim, self.hidden = ops, kind, rows, top, groups, dim, hidden
        gu, dn = torch.randn(groups, 2 * hidden, dim, generator=g) * dim ** -0.5, torch.randn(groups, dim, hidden, generator=g) * hidden ** -0.5
        make = ops.quantize_weight_fp8 if kind == "fp8" else lambda w, glu=False: ops.pack_grouped(w.to(torch.bfloat16), glu)
        self.gate_up, self.down = make(gu.to(DEV), glu=True), make(dn.to(DEV))
        self.x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
        self.choice, self.share = torch.zeros(rows, top, dtype=torch.int32, device=DEV), torch.zeros(rows, top, device=DEV)
        self.room = ops.row_groups(rows, top, groups, DEV)
        self.units = torch.empty(rows * top, hidden, dtype=torch.float32 if kind == "fp8" else torch.bfloat16, device=DEV)
        self.answers, self.out = torch.empty(rows * top, dim, device=DEV), torch.empty(rows, dim, device=DEV)
        if kind == "fp8":
            self.x8, self.u8 = ops.fp8_rows(rows, dim, DEV), ops.fp8_rows(rows * top, hidden, DEV)

    def put(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.rows, self.dim, generator=g))
        choice = torch.rand(self.rows, self.groups_n, generator=g).topk(self.top, dim=1).indices.to(torch.int32)
        choice[torch.rand(self.rows, generator=g) < 0.15] = -1
        self.choice.copy_(choice)
        self.share.copy_(torch.rand(self.rows, self.top, generator=g))

    def run(self):
        ops, x, units = self.ops, self.x, self.units
        ops.group_rows(self.choice, self.room)
        if self.kind == "fp8":
            ops.quantize_fp8(x, self.x8)
            x = self.x8
        ops.gemm_grouped(x, self.gate_up, self.room, units, swiglu="silu")
        if self.kind == "fp8":
            ops.quantize_fp8(units, self.u8)
            units = self.u8
        ops.gemm_grouped(units, self.down, self.room, self.answers, by_pair=True)
        ops.combine_groups(self.answers, self.room, self.share, self.out)


def settled(layer, seed):
    """The layer's result with everything waited for between its calls' inputs and its end."""
    layer.put(seed)
    torch.cuda.synchronize()
    layer.run()
    torch.cuda.synchronize()
    return layer.out.clone()


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
@pytest.mark.parametrize("rows", [3, 40, 900])
def test_captured_and_replayed_with_other_choices(ops, kind, rows):
    layer = Layer(ops, kind, rows)
    want = [settled(layer, s) for s in range(4)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.run()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run()
        for s in (2, 0, 3, 1):
            layer.put(s)
            graph.replay()
            stream.synchronize()
            assert torch.equal(layer.out, want[s])
    ops.check_kernel_errors()


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
def test_two_streams_at_once(ops, kind):
    layers = [Layer(ops, kind, rows, seed=rows) for rows in (33, 500)]
    want = [settled(layer, 5) for layer in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(20):
        for layer, stream in zip(layers, streams):
            layer.out.zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                layer.run()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for layer, w in zip(layers, want):
            assert torch.equal(layer.out, w)


@pytest.mark.parametrize("kind", ["bfloat16", "fp8"])
def test_one_behind_the_other_on_the_same_buffers(ops, kind):
    """Kernels that begin before the one in front has ended wait for what they read and for what they overwrite."""
    layer = Layer(ops, kind, 64)
    want = [settled(layer, s) for s in range(3)]
    inputs = []
    for s in range(3):
        layer.put(s)
        inputs.append((layer.x.clone(), layer.choice.clone(), layer.share.clone()))
    outs = []
    for i in range(60):
        for to, frm in zip((layer.x, layer.choice, layer.share), inputs[i % 3]):
            to.copy_(frm)
        layer.run()
        outs.append(layer.out.clone())
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 3])


def test_the_same_bits_at_every_run(ops):
    """Nothing depends on which block comes first."""
    g = torch.Generator().manual_seed(3)
    a = ops.fp8_rows(24, 4096, DEV)
    ops.quantize_fp8(torch.randn(24, 4096, generator=g).to(DEV), a)
    w = ops.quantize_weight_fp8(torch.randn(512, 4096, generator=g).to(DEV))
    for cut in (0, 32124, 16128, 16121, 64121, 128211, 128212, 128214):
        outs = []
        for _ in range(8):
            out = torch.empty(24, 512, device=DEV)
            ops.gemm_fp8(a, w, out, cut=cut)
            outs.append(out)
        assert all(torch.equal(outs[0], o) for o in outs)


def test_every_significand_of_bfloat16(ops):
    """All 128 x 128 pairs of a block's largest magnitude and a value, over 26 powers of two: rounded once, half to even."""
    import tests.test_gpu_grouped as plain
    sig = torch.arange(128, 256).float()
    values = (sig[:, None] * 2.0 ** -torch.arange(26).float()[None, :]).flatten()                # 3,328 values
    for shift in (-7, 30, -100):
        rows = []
        for m in sig:
            v = values[values <= m]
            v = torch.cat([v, torch.zeros(-len(v) % 127)]).view(-1, 127)
            rows.append(torch.cat([v, m.expand(v.shape[0], 1)], dim=1))
        x = (torch.cat(rows) * 2.0 ** shift)
        x[::2] *= -1
        x = x.to(torch.bfloat16)
        q, scale = plain.plain_fp8(x.float())
        out = ops.fp8_rows(*x.shape, DEV)
        ops.quantize_fp8(x.to(DEV), out)
        assert torch.equal(out.scale.cpu(), scale) and torch.equal(out.data.cpu().double(), q)


def test_scales_of_every_significand(ops):
    """The largest magnitude over 448, rounded once: 2^18 of float32's significands."""
    m = (torch.arange(2 ** 18) * 32 + 2 ** 23 + torch.arange(2 ** 18) % 31).float() * 2.0 ** -20
    x = torch.zeros(2 ** 18, 128)
    x[:, 5] = -m
    out = ops.fp8_rows(*x.shape, DEV)
    ops.quantize_fp8(x.to(DEV), out)
    assert torch.equal(out.scale.cpu()[:, 0], (m.double() / 448).float()) and (out.data[:, 5].float() == -448).all()


def test_matrices_beyond_32_bits(ops):
    """Rows, results and answers whose places do not fit 31 bits."""
    rows, width, dim = 70016, 32768, 128          # 2.3e9 results
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(rows, dim, generator=g, device=DEV).to(torch.bfloat16)
    a = ops.fp8_rows(rows, dim, DEV)
    ops.quantize_fp8(x, a)
    w = torch.randn(width, dim, generator=g, device=DEV)
    packed = ops.quantize_weight_fp8(w)
    out = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    ops.gemm_fp8(a, packed, out)
    few = torch.tensor([0, 1, 65535, 65536, 65537, 70015])
    part = torch.empty(len(few), width, dtype=torch.bfloat16, device=DEV)
    b = ops.fp8_rows(len(few), dim, DEV)
    ops.quantize_fp8(x[few.to(DEV)], b)
    ops.gemm_fp8(b, packed, part, cut=128211)
    whole = torch.empty_like(part)
    ops.gemm_fp8(a[:128], packed, torch.empty(128, width, dtype=torch.bfloat16, device=DEV), cut=128211)
    assert torch.equal(out[few.to(DEV)], part) and whole.shape == part.shape
    # the same values as wide rows: quantised, taken back, and summed as answers
    wide = ops.fp8_rows(rows, width, DEV)
    ops.quantize_fp8(out, wide)
    back = torch.empty_like(out)
    ops.fp8_values(wide, back)
    ends = out[-2:].float()
    m = ends.view(2, -1, 128).abs().amax(dim=2, keepdim=True)
    off = (back[-2:].float().view(2, -1, 128) - ends.view(2, -1, 128)).abs()
    assert (off <= ends.view(2, -1, 128).abs() * (2.0 ** -4 + 2.0 ** -8) + m * 2.0 ** -18).all()          # half a step of e4m3, a rounding, the smallest steps
    room = ops.row_groups(rows // 2, 2, 1, DEV)
    choice = torch.zeros(rows // 2, 2, dtype=torch.int32, device=DEV)
    ops.group_rows(choice, room)
    total = torch.empty(rows // 2, width, dtype=torch.bfloat16, device=DEV)
    ops.combine_groups(out, room, torch.ones(rows // 2, 2, device=DEV), total)
    assert torch.equal(total[-1], (out[-2].float() + out[-1].float()).to(torch.bfloat16))


def test_no_rows_and_no_choices(ops):
    packed = ops.pack_grouped(torch.zeros(3, 16, 8, dtype=torch.bfloat16, device=DEV))
    room = ops.row_groups(0, 2, 3, DEV)
    ops.group_rows(torch.empty(0, 2, dtype=torch.int32, device=DEV), room)
    assert room.offsets.tolist() == [0, 0, 0, 0]
    ops.gemm_grouped(torch.empty(0, 8, dtype=torch.bfloat16, device=DEV), packed, room, torch.empty(0, 16, device=DEV))
    ops.combine_groups(torch.empty(0, 16, device=DEV), room, torch.empty(0, 2, device=DEV), torch.empty(0, 16, device=DEV))
    ops.quantize_fp8(torch.empty(0, 40, device=DEV), ops.fp8_rows(0, 40, DEV))
    room = ops.row_groups(6, 2, 3, DEV)
    ops.group_rows(torch.full((6, 2), -1, dtype=torch.int32, device=DEV), room)
    out = torch.full((6, 16), 3.0, device=DEV)
    ops.combine_groups(torch.full((12, 16), float("nan"), device=DEV), room, torch.ones(6, 2, device=DEV), out, accumulate=True)
    assert (out == 3).all()
    ops.combine_groups(torch.full((12, 16), float("nan"), device=DEV), room, torch.ones(6, 2, device=DEV), out)
    assert (out == 0).all()


def test_the_same_expert_twice(ops):
    """A row may ask an expert with two of its choices: two pairs."""
    choice = torch.tensor([[1, 1], [0, 1], [1, -1]], dtype=torch.int32)
    room = ops.row_groups(3, 2, 2, DEV)
    ops.group_rows(choice.to(DEV), room)
    assert room.order.tolist() == [2, 0, 1, 3, 4, -1] and room.place.tolist() == [[1, 2], [0, 3], [4, -1]] and room.offsets.tolist() == [0, 1, 5]


def test_what_the_launcher_refuses(ops):
    """The library's own checks, for whoever calls it without the ones in front (no launch is made)."""
    lib = ops.library()
    a, w = ops.fp8_rows(4, 256, DEV), ops.quantize_weight_fp8(torch.ones(64, 256, device=DEV))
    out = torch.zeros(4, 64, device=DEV)
    room = ops.row_groups(4, 1, 1, DEV)

    def call(rows=a, weight=w, groups=0, by_pair=0, bias=0, ldo=64, accumulate=0, word=0, cut=0):
        return lib.jllm_gemm_grouped(rows if isinstance(rows, int) else rows.view, weight if isinstance(weight, int) else weight.view, groups, by_pair, bias, 0, out.data_ptr(), 0,
                                     ldo, accumulate, word, cut, 0)

    def changed(view, **fields):
        copy = type(view).from_buffer_copy(view)
        for name, value in fields.items():
            setattr(copy, name, value)
        call.keep = copy
        return ctypes.addressof(copy)
    assert call() == 0
    for bad in (dict(ldo=63), dict(accumulate=3), dict(word=1), dict(cut=7), dict(groups=room.view, accumulate=1), dict(groups=room.view, bias=out.data_ptr())):
        assert call(**bad) != 0, bad
    for fields in (dict(cols=255), dict(rows=-1), dict(scale=0), dict(scale_ld=3), dict(scale_ld=0), dict(stride=100), dict(stride=264), dict(data=a.data.data_ptr() + 8)):
        assert call(rows=changed(a._view, **fields)) != 0, fields
    for fields in (dict(cols=128), dict(groups=2), dict(k_blocks=3), dict(rows=0), dict(scale_ld=1), dict(data=w.data.data_ptr() + 8), dict(scale=0)):
        assert call(weight=changed(w._view, **fields)) != 0, fields
    for fields in (dict(rows=5), dict(groups=2), dict(top=2 ** 30)):
        assert call(groups=changed(room._view, **fields)) != 0, fields
    for fields in (dict(groups=0), dict(groups=1025), dict(top=0), dict(rows=-1), dict(rows=2 ** 30, top=2)):
        assert lib.jllm_group_rows(out.data_ptr(), 2, changed(room._view, **fields), 0) != 0, fields
    assert lib.jllm_combine_groups(out.data_ptr(), 0, 63, room.view, out.data_ptr(), 1, out.data_ptr(), 0, 64, 64, 0, 0) != 0
    assert lib.jllm_quantize_fp8(out.data_ptr(), 0, 255, a.view, 0) != 0 and lib.jllm_fp8_values(changed(a._view, scale_ld=1), out.data_ptr(), 0, 256, 0) != 0
    torch.cuda.synchronize()


def test_tensors_elsewhere_are_refused(ops):
    """Rows, weights or results on the host beside others on the GPU."""
    w = ops.quantize_weight_fp8(torch.ones(64, 256, device=DEV))
    a, out = ops.fp8_rows(4, 256, DEV), torch.zeros(4, 64, device=DEV)
    before = ops.launch_count
    for call in (lambda: ops.gemm_fp8(ops.fp8_rows(4, 256, "cpu"), w, out), lambda: ops.gemm_fp8(a, w, out.cpu()), lambda: ops.quantize_fp8(torch.zeros(4, 256), a),
                 lambda: ops.gemm_fp8(a, w, out, torch.zeros(64)), lambda: ops.fp8_values(a, torch.zeros(4, 256)),
                 lambda: ops.Fp8Rows(a.data, a.scales.cpu())):
        with pytest.raises(ops.KernelError):
            call()
    assert ops.launch_count == before
