"""Models whose layers' products run in 8-bit floating point (GPU): the engine against the plain implementation with the same rounding of weights and rows,
generation with and without replayed steps, and what is refused."""
import pytest
import torch

from tests.plain import qwen3_plain as plain
from tests.tiny import TINY_A, TINY_B, TINY_C, TINY_E, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu


def e4m3(x):
    """float32 -> the nearest e4m3 value, half to even."""
    _, exponent = torch.frexp(x.abs())
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def row_values(v):
    """The values that the rows of v stand for, a scale for each 128 of them."""
    blocks = torch.nn.functional.pad(v, (0, -v.shape[-1] % 128)).unflatten(-1, (-1, 128))
    scale = blocks.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -100) / 448.0
    return (e4m3(blocks / scale) * scale).flatten(-2)[..., :v.shape[-1]]


def weight_values(w):
    n, k = w.shape
    blocks = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).unflatten(0, (-1, 128)).unflatten(-1, (-1, 128))
    scale = blocks.abs().amax(dim=(1, 3), keepdim=True).clamp(min=2.0 ** -100) / 448.0
    return (e4m3(blocks / scale) * scale).flatten(2).flatten(0, 1)[:n, :k]


def plain_logits(monkeypatch, cfg, weights, tokens):
    """The plain forward pass with every layer product in 8 bits (queries, keys and values, gate and up stacked as the engine stacks them); the head
    (and a tied embedding) as it is."""
    whole = plain.linear
    layers = {id(t): name for name, t in weights.items() if "layers." in name}
    stacks = (("q_proj.weight", "k_proj.weight", "v_proj.weight"), ("gate_proj.weight", "up_proj.weight"))

    def stacked(name, w):
        for stack in stacks:
            for part in stack:
                if name.endswith(part):
                    tensors = [weights[name.replace(part, other)] for other in stack]
                    lo = sum(t.shape[0] for t in tensors[:stack.index(part)])
                    return weight_values(torch.cat(tensors))[lo:lo + w.shape[0]]
        return weight_values(w)

    def linear(x, w, b=None):
        return whole(row_values(x), stacked(layers[id(w)], w), b) if id(w) in layers else whole(x, w, b)
    with monkeypatch.context() as m:
        m.setattr(plain, "linear", linear)
        return plain.forward(cfg, weights, list(tokens))


@pytest.mark.parametrize("config,seed", [(TINY_A, 3), (TINY_B, 5), (TINY_C, 7), (TINY_E, 6)])
def test_logits_follow_the_plain_rounding(config, seed, tmp_path, monkeypatch):
    """The engine rounds to bfloat16 in front of the 8 bits where the plain form does not. A value that moves by d crosses an edge of its 8 bits with
    probability d / step, and then moves by a step: step 2^-3 to 2^-4 of the value, mean d about 2^-10 of it, so each product's rows are off by sqrt(step
    d) = 1%; sixteen products one behind the other: 4%. Held to twice that."""
    from jllm_serve_b200.engine import Engine, Segment
    from jllm_serve_b200.parts.linear import Fp8Linear
    folder = make_model_folder(config, seed, tmp_path)
    cfg, weights = plain.load_plain(folder)
    tokens = random_tokens(75, config["vocab_size"], seed)
    want = plain_logits(monkeypatch, cfg, weights, tokens)
    with Engine(folder, weights="fp8", page_size=8, max_tokens_cached=512, max_batch_tokens=64, max_running=2, ctx=128) as engine:
        assert all(isinstance(p, Fp8Linear) for b in engine.runner.model.blocks
                   for p in (b.mixer.qkv, b.mixer.out, b.feed_forward.gate_up, b.feed_forward.down))
        got = []
        for lo, hi in ((0, 50), (50, 67)):           # portions of a prompt, then single tokens (captured and replayed)
            got.append(engine.runner.step([Segment("r", tokens[lo:hi], lo, list(range(hi - lo)))]).clone())
        for i in range(67, 75):
            got.append(engine.runner.step([Segment("r", tokens[i:i + 1], i, [0])]).clone())
        got = torch.cat(got).cpu()
        from jllm_serve_b200.csrc import ops
        ops.check_kernel_errors()
    off = (got - want).norm(dim=1) / want.norm(dim=1)
    print(f"off by {off.mean():.4f} in the mean, {off.max():.4f} at most")
    assert got.shape == want.shape and float(off.max()) <= 0.08, off


def test_generation_with_and_without_replayed_steps(tmp_path):
    from jllm_serve_b200.engine import Engine
    from jllm_serve_b200.sampling import SamplingParams
    folder = make_model_folder(TINY_B, 5, tmp_path)
    prompts = [random_tokens(n, TINY_B["vocab_size"], 40 + n) for n in (9, 33, 70)]
    got = []
    for graphs in (True, False):
        with Engine(folder, weights="fp8", page_size=8, max_tokens_cached=512, max_batch_tokens=64, chunk=32, max_running=4, ctx=256, cuda_graphs=graphs) as engine:
            assert "weights=fp8" in engine.runner.describe()
            got.append([r.tokens for r in engine.generate(prompts, SamplingParams.greedy_params(12, ignore_eos=True))])
    assert got[0] == got[1] and all(len(t) == 12 for t in got[0])


def test_a_layer_that_reads_anothers_cache():
    """Its product is the query rows of the packed weight alone."""
    from jllm_serve_b200.csrc import ops
    from jllm_serve_b200.parts.base import Runtime
    from jllm_serve_b200.parts.linear import Fp8Linear
    g = torch.Generator().manual_seed(2)
    w, bias = torch.randn(300, 96, generator=g).to("cuda:0"), torch.randn(300, generator=g).to("cuda:0")
    whole = Fp8Linear(w, bias, Runtime(torch.device("cuda:0"), torch.bfloat16, 64, 32, 16, "fp8"))
    x = torch.randn(20, 96, generator=g).to("cuda:0")
    a = torch.empty(20, 300, device="cuda:0")
    whole.forward(x, a)
    for lo, hi in ((0, 70), (128, 300), (0, 300)):
        b = torch.empty(20, hi - lo, device="cuda:0")
        whole.rows(lo, hi).forward(x, b)
        assert torch.equal(a[:, lo:hi], b)
    with pytest.raises(ops.KernelError):
        whole.rows(30, 100)


def test_refusals(tmp_path):
    from jllm_serve_b200.engine import Engine
    from tests.movivik_cases import MOVIVIK_A
    folder = make_model_folder(TINY_A, 3, tmp_path)
    with pytest.raises(ValueError):
        Engine(folder, max_tokens_cached=128, ctx=64, dtype="float32", weights="fp8")
    with pytest.raises(ValueError, match="8-bit floating point"):
        Engine(config=MOVIVIK_A, seed=1, weights="fp8", max_tokens_cached=128, ctx=64)
