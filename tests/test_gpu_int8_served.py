"""A layer of a served width in 8-bit integers (GPU): prompts of several hundred rows in one step, which the products take in groups of tokens,
alone, two beside one another and beside a decoding request. Every operator that the steps call is looked at by itself: its output from the
inputs that the model gave it, against the plain form with the kernels' own roundings."""
import pytest
import torch

from tests.test_gpu_int8 import check_norm, plain_int8, same
from tests.tiny import make_model_folder, random_tokens

pytestmark = pytest.mark.gpu

# the layer of the benchmark's model: 4,096 wide, 32 heads of 128 over 8, 12,288 hidden units
SERVED = dict(model_type="qwen3", architectures=["Qwen3ForCausalLM"], hidden_size=4096, num_hidden_layers=1, num_attention_heads=32,
              num_key_value_heads=8, head_dim=128, intermediate_size=12288, vocab_size=509, rope_theta=1000000.0, rms_norm_eps=1e-6,
              tie_word_embeddings=False, attention_bias=False, use_sliding_window=False, max_position_embeddings=4096, hidden_act="silu")


class Watched:
    """The 8-bit operators of `ops`, each call followed by its check; `seen` counts the rows that each was called with."""

    def __init__(self, ops, monkeypatch):
        self.seen = []
        for name in ("gemm_int8", "quantize_int8", "add_rmsnorm_int8"):
            monkeypatch.setattr(ops, name, self.watch(name, getattr(ops, name), getattr(self, name)))

    def watch(self, name, call, check):
        def run(*args, **kw):
            check(call, *args, **kw)
            self.seen.append((name, args[0].shape[0]))
        return run

    def gemm_int8(self, call, a, w, out, bias=None, accumulate=False, swiglu=False):
        old = out.clone()
        call(a, w, out, bias, accumulate, swiglu)
        assert bias is None
        v = (a.data.double() @ w.unpack().double().T).float() * a.scale[:, None] * w.scale[None, :]
        if not swiglu:
            assert torch.equal(out, (v + old.float() if accumulate else v).to(out.dtype))
            return
        gate, up = v.double().view(v.shape[0], -1, 2, 8).unbind(2)
        want = (gate * torch.sigmoid(gate) * up).reshape(v.shape[0], -1)
        # (a fast exponential's error, and the rounding to bfloat16)
        assert torch.allclose(out.double(), want, rtol=2.0 ** -8, atol=1e-6 * float(want.abs().max()))

    def quantize_int8(self, call, x, out):
        call(x, out)
        q, scale = plain_int8(x.float().cpu())
        assert torch.equal(out.data.cpu(), q) and same(out.scale.cpu(), scale)

    def add_rmsnorm_int8(self, call, x, gain, eps, out, y=None):
        total = x if y is None else x + y.float()
        total = total.clone()
        call(x, gain, eps, out, y=y)
        assert torch.equal(x, total)
        check_norm(out, total.cpu(), gain.cpu(), eps, x.shape[1])


def test_every_operator_of_a_prompts_steps(tmp_path, monkeypatch):
    from jllm_serve_b200.csrc import ops
    from jllm_serve_b200.engine import Engine, Segment
    folder = make_model_folder(SERVED, 4, tmp_path)
    a, b = random_tokens(640, 509, 1), random_tokens(330, 509, 2)
    with Engine(folder, weights="int8", page_size=16, max_tokens_cached=2048, max_batch_tokens=1024, max_running=4, ctx=1024) as engine:
        watched = Watched(ops, monkeypatch)
        for segments in ([Segment("a", a[:601], 0, list(range(601)))],                                           # one prompt: three groups of tokens
                         [Segment("a", a[601:602], 601, [0]), Segment("b", b[:300], 0, list(range(300)))],
                         [Segment("a", a[602:632], 602, [29]), Segment("b", b[300:], 300, [29])]):
            rows = sum(len(s.tokens) for s in segments)
            logits = engine.runner.step(segments)
            ops.check_kernel_errors()
            assert torch.isfinite(logits).all()
            # both norms, the attention's result and the units, four products
            assert sorted(watched.seen) == sorted([("add_rmsnorm_int8", rows)] * 2 + [("quantize_int8", rows)] * 2 + [("gemm_int8", rows)] * 4)
            watched.seen.clear()
