"""Models whose layers' products run in 8-bit integers (GPU): the engine against the plain implementation with the same rounding of weights
and rows, generation with and without replayed steps, and what is refused."""
import copy

import pytest
import torch

from tests.plain import qwen3_plain as plain
from tests.tiny import TINY_A, TINY_B, TINY_C, TINY_E, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu


def to_values(v):
    """The values that the rows of v stand for in 8 bits."""
    m = v.abs().amax(dim=-1, keepdim=True)
    return torch.round(v * (127.0 / m)).clamp(-127, 127) * (m / 127.0)


def plain_logits(monkeypatch, cfg, weights, tokens):
    """The plain forward pass with every layer product in 8 bits; the head (and a tied embedding) as it is."""
    whole = plain.linear
    layers = {id(t) for name, t in weights.items() if "layers." in name}

    def linear(x, w, b=None):
        return whole(to_values(x), to_values(w), b) if id(w) in layers else whole(x, w, b)
    with monkeypatch.context() as m:
        m.setattr(plain, "linear", linear)
        return plain.forward(cfg, weights, list(tokens))


@pytest.mark.parametrize("config,seed", [(TINY_A, 3), (TINY_B, 5), (TINY_C, 7), (TINY_E, 6)])
def test_logits_follow_the_plain_rounding(config, seed, tmp_path, monkeypatch):
    """The engine rounds to bfloat16 between the products where the plain form does not. A value of a row that moves by d crosses an edge of
    its 8 bits with probability d / step, and then moves by a step: step about 3.2 sigma / 127, mean d about 2^-9 / 4 of the value, so
    each product's rows are off by sqrt(step d) = 0.4% of sigma; sixteen products one behind the other: 1.6%. Held to three times that."""
    from jllm_serve_b200.engine import Engine, Segment
    from jllm_serve_b200.parts.linear import Int8Linear
    folder = make_model_folder(config, seed, tmp_path)
    cfg, weights = plain.load_plain(folder)
    tokens = random_tokens(75, config["vocab_size"], seed)
    want = plain_logits(monkeypatch, cfg, weights, tokens)
    with Engine(folder, weights="int8", page_size=8, max_tokens_cached=512, max_batch_tokens=64, max_running=2, ctx=128) as engine:
        assert all(isinstance(p, Int8Linear) for b in engine.runner.model.blocks
                   for p in (b.mixer.qkv, b.mixer.out, b.feed_forward.gate_up, b.feed_forward.down))
        got = []
        for lo, hi in ((0, 50), (50, 67)):           # portions of a prompt, then single tokens (captured and replayed)
            got.append(engine.runner.step([Segment("r", tokens[lo:hi], lo, list(range(hi - lo)))]).clone())
        for i in range(67, 75):
            got.append(engine.runner.step([Segment("r", tokens[i:i + 1], i, [0])]).clone())
        got = torch.cat(got).cpu()
        from jllm_serve_b200.csrc import ops
        ops.check_kernel_errors()
    assert got.shape == want.shape
    off = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(off.max()) <= 0.05, off


def test_generation_with_and_without_replayed_steps(tmp_path):
    from jllm_serve_b200.engine import Engine
    from jllm_serve_b200.sampling import SamplingParams
    folder = make_model_folder(TINY_B, 5, tmp_path)
    prompts = [random_tokens(n, TINY_B["vocab_size"], 40 + n) for n in (9, 33, 70)]
    got = []
    for graphs in (True, False):
        with Engine(folder, weights="int8", page_size=8, max_tokens_cached=512, max_batch_tokens=64, chunk=32, max_running=4, ctx=256,
                    cuda_graphs=graphs) as engine:
            assert "weights=int8" in engine.runner.describe()
            got.append([r.tokens for r in engine.generate(prompts, SamplingParams.greedy_params(12, ignore_eos=True))])
    assert got[0] == got[1] and all(len(t) == 12 for t in got[0])


def test_a_hidden_width_that_does_not_come_in_eights(tmp_path, monkeypatch):
    """Gate and up are then one plain product, and the gating a launch of its own."""
    from jllm_serve_b200.engine import Engine, Segment
    config = copy.deepcopy(TINY_A)
    config["intermediate_size"] = 130
    folder = make_model_folder(config, 3, tmp_path)
    cfg, weights = plain.load_plain(folder)
    tokens = random_tokens(40, config["vocab_size"], 1)
    want = plain_logits(monkeypatch, cfg, weights, tokens)
    with Engine(folder, weights="int8", page_size=8, max_tokens_cached=128, max_batch_tokens=64, max_running=2, ctx=64) as engine:
        got = engine.runner.step([Segment("r", tokens, 0, list(range(40)))]).cpu()
    assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) <= 0.05


def test_a_layer_that_reads_anothers_cache(tmp_path):
    """Its product is the query rows of the packed weight alone."""
    from jllm_serve_b200.parts.base import Runtime
    from jllm_serve_b200.parts.linear import Int8Linear
    g = torch.Generator().manual_seed(2)
    w = torch.randn(300, 96, generator=g).to("cuda:0")
    bias = torch.randn(300, generator=g).to("cuda:0")
    rt = Runtime(torch.device("cuda:0"), torch.bfloat16, 64, 32, 16, "int8")
    whole = Int8Linear(w, bias, rt)
    x = torch.randn(20, 96, generator=g).to("cuda:0")
    a, b = torch.empty(20, 300, device="cuda:0"), torch.empty(20, 70, device="cuda:0")
    whole.forward(x, a)
    whole.rows(30, 100).forward(x, b)
    assert torch.equal(a[:, 30:100], b)


def test_refusals(tmp_path):
    from jllm_serve_b200.engine import Engine
    from tests.movivik_cases import MOVIVIK_A
    folder = make_model_folder(TINY_A, 3, tmp_path)
    for kw in (dict(dtype="float32", weights="int8"), dict(weights="int4")):
        with pytest.raises(ValueError):
            Engine(folder, max_tokens_cached=128, ctx=64, **kw)
    with pytest.raises(ValueError, match="8-bit"):
        Engine(config=MOVIVIK_A, seed=1, weights="int8", max_tokens_cached=128, ctx=64)
