"""A product right behind the packing of its weight (GPU): it does not begin before the packing has ended."""
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


def early_launches(graph):
    """Of a captured graph, how many launches may begin before what is in front of them has ended."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    answer = runtime.cudaGraphGetEdges_v2(graph, 4096)
    assert int(answer[0]) == 0
    edges = answer[3][:answer[4]]
    assert len(edges) >= 1
    return sum(int(edge.type) != 0 for edge in edges)


@pytest.mark.parametrize("n,k,glu", [(96, 200, False), (272, 700, True), (4096, 1920, False)])
def test_a_product_right_behind_its_weights_packing(ops, n, k, glu):
    g = torch.Generator().manual_seed(n)
    data, scale = (100 * torch.randn(n, k, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV), torch.rand(-(-n // 128), -(-k // 128), generator=g).to(DEV)
    rows8, bf16 = ops.fp8_rows(5, k, DEV), torch.randn(5, k, generator=g).to(DEV)
    out = torch.empty(5, n // 2 if glu else n, device=DEV)
    ops.quantize_fp8(bf16, rows8)
    weight = ops.pack_fp8(data, scale, glu)
    torch.cuda.synchronize()
    ops.gemm_fp8(rows8, weight, out, swiglu=glu)
    want = out.clone()
    for _ in range(20):
        ops.gemm_fp8(rows8, ops.pack_fp8(data, scale, glu), out.zero_(), swiglu=glu)
        assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        weight = ops.pack_fp8(data, scale, glu)
        ops.gemm_fp8(rows8, weight, out, swiglu=glu)
    assert early_launches(graph.raw_cuda_graph()) == 0
    with_rows = torch.cuda.CUDAGraph(keep_graph=True)          # (behind a kernel of this library it does begin early, and so is seen)
    with torch.cuda.graph(with_rows):
        ops.quantize_fp8(bf16, rows8)
        ops.gemm_fp8(rows8, weight, out, swiglu=glu)
    assert early_launches(with_rows.raw_cuda_graph()) == 1
    out.zero_()
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
