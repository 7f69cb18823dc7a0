"""Every product that a model of 8-bit floating point runs, in its steps (GPU): each against 64 bits from its own inputs, the weights rounded from the model's
file by the definition. What the products get from one another does not blur it, so a scale of one block that is wrong shows.

Tolerances as in `test_gpu_grouped.py`: a sum's additions, the biases' and the sum's with what was there, a rounding to the result's type."""
import pytest
import torch

from tests.plain import qwen3_plain as plain
from tests.test_gpu_grouped import ULP, plain_e4m3, plain_fp8, product_slack, units_and_slack, values_of
from tests.tiny import TINY_A, TINY_B, TINY_C, TINY_E, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu


def weight_values(w):
    """float64 values of a float32 weight rounded in blocks of 128 x 128."""
    n, k = w.shape
    blocks = torch.nn.functional.pad(w.double(), (0, -k % 128, 0, -n % 128)).unflatten(0, (-1, 128)).unflatten(-1, (-1, 128))
    scale = (blocks.abs().amax(dim=(1, 3), keepdim=True).clamp(min=2.0 ** -100) / 448).float().double()
    return (plain_e4m3(blocks / scale) * scale).flatten(2).flatten(0, 1)[:n, :k]


@pytest.mark.parametrize("config,seed", [(TINY_A, 3), (TINY_B, 5), (TINY_C, 7), (TINY_E, 6)])
def test_every_product_of_a_models_steps(config, seed, tmp_path, monkeypatch):
    from jllm_serve_b200.csrc import ops
    from jllm_serve_b200.engine import Engine, Segment
    from jllm_serve_b200.parts.linear import Fp8Linear
    folder = make_model_folder(config, seed, tmp_path)
    _, weights = plain.load_plain(folder)
    tokens = random_tokens(60, config["vocab_size"], seed)
    seen, forward = [], Fp8Linear.forward

    def watched(self, a, out, accumulate=False, swiglu=False, relu2=False):
        before = out.clone() if accumulate else None
        forward(self, a, out, accumulate, swiglu, relu2)
        seen.append((self, a.clone(), out.clone(), before, bool(swiglu)))
    monkeypatch.setattr(Fp8Linear, "forward", watched)
    with Engine(folder, weights="fp8", page_size=8, max_tokens_cached=512, max_batch_tokens=64, max_running=2, ctx=128, cuda_graphs=False) as engine:
        want = {}
        for l, block in enumerate(engine.runner.model.blocks):
            for linear, names in ((block.mixer.qkv, ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj")), (block.mixer.out, ("self_attn.o_proj",)),
                                  (block.feed_forward.gate_up, ("mlp.gate_proj", "mlp.up_proj")), (block.feed_forward.down, ("mlp.down_proj",))):
                names = [f"model.layers.{l}.{n}" for n in names]
                bias = [weights[n + ".bias"] for n in names if n + ".bias" in weights]
                want[id(linear)] = names, weight_values(torch.cat([weights[n + ".weight"] for n in names])), torch.cat(bias).double() if bias else None
        seen.clear()
        for lo, hi in ((0, 47), (47, 59), (59, 60)):
            engine.runner.step([Segment("r", tokens[lo:hi], lo, list(range(hi - lo)))])
        torch.cuda.synchronize()
        ops.check_kernel_errors()
    assert len(seen) == 3 * 4 * config["num_hidden_layers"]
    for linear, a, out, before, gated in seen:
        names, w, bias = want[id(linear)]
        assert (linear.bias is None) == (bias is None)
        x = values_of(*plain_fp8(a.float().cpu()))
        result, slack = x @ w.T, product_slack(x, w, -(-w.shape[1] // 128))
        if gated:
            result, slack = units_and_slack(result, slack)
        for more in (bias, None if before is None else before.cpu().double()):
            if more is not None:
                result = result + more
                slack = slack + ULP * result.abs()
        off = (out.cpu().double() - result).abs()
        bound = slack + (result.abs() + slack) * torch.finfo(out.dtype).eps / 2
        assert (off <= bound).all(), (names, float((off - bound).max()))
