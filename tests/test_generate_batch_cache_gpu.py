"""Batched greedy generation with the caches held in 4 bits (lsx_model_generate_batch_cache) against a plain
forward pass of the same checkpoint in 64 bits whose cache is rounded the same way."""
import json
import struct

import numpy as np
import pytest

import cache_reference as ref
import laplacesscissors_b200 as lsx
from conftest import GOLDEN
from laplacesscissors_b200 import LsxError, synth

pytestmark = pytest.mark.gpu


class PlainModel:
    """A Qwen3-layout checkpoint (tied head) in 64 bits, one sequence, its decode steps over a rounded cache."""

    def __init__(self, root):
        self.config = json.loads((root / "config.json").read_text())
        self.w = {}
        for path in sorted(root.glob("*.safetensors")):
            raw = path.read_bytes()
            size = struct.unpack("<Q", raw[:8])[0]
            for name, about in json.loads(raw[8:8 + size]).items():
                if name == "__metadata__":
                    continue
                a, b = about["data_offsets"]
                data = raw[8 + size + a:8 + size + b]
                x = np.frombuffer(data, np.float32) if about["dtype"] == "F32" else \
                    (np.frombuffer(data, np.uint16).astype(np.uint32) << 16).view(np.float32)
                self.w[name] = x.reshape(about["shape"]).astype(np.float64)

    def norm(self, x, gain):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.config["rms_norm_eps"]) * gain

    def rope(self, x, positions):
        half = x.shape[-1] // 2
        angle = positions[:, None] * self.config["rope_theta"] ** (-np.arange(half) / half)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * c - b * s, b * c + a * s], -1)

    def logits(self, tokens, exact):
        """Logits of positions exact .. of a sequence whose first `exact` positions went through at once."""
        c, w = self.config, self.w
        H, K, D, n = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], len(tokens)
        x = w["model.embed_tokens.weight"][tokens]
        at = np.arange(n)
        for i in range(c["num_hidden_layers"]):
            p = f"model.layers.{i}."
            h = self.norm(x, w[p + "input_layernorm.weight"])
            q, k, v = ((h @ w[p + f"self_attn.{m}_proj.weight"].T).reshape(n, -1, D) for m in "qkv")
            q = self.rope(self.norm(q, w[p + "self_attn.q_norm.weight"]), at)
            k = self.rope(self.norm(k, w[p + "self_attn.k_norm.weight"]), at)
            held = [ref.dequantise(*ref.quantise(a.astype(np.float32))) for a in (k, v)]
            out = np.zeros((n, H, D))
            for row in range(n):
                keys, values = (k, v) if row < exact else held
                for head in range(H):
                    z = keys[:row + 1, head * K // H] @ q[row, head] / np.sqrt(D)
                    e = np.exp(z - z.max())
                    out[row, head] = e / e.sum() @ values[:row + 1, head * K // H]
            x = x + out.reshape(n, -1) @ w[p + "self_attn.o_proj.weight"].T
            h = self.norm(x, w[p + "post_attention_layernorm.weight"])
            gate, up = (h @ w[p + f"mlp.{m}_proj.weight"].T for m in ("gate", "up"))
            x = x + (gate / (1 + np.exp(-gate)) * up) @ w[p + "mlp.down_proj.weight"].T
        return self.norm(x, w["model.norm.weight"])[exact:] @ w["model.embed_tokens.weight"].T


@pytest.mark.parametrize("P,maximum", [(2, 9), (9, 7), (17, 30)])
def test_tokens_follow_a_rounded_cache(gpu, P, maximum):
    root = GOLDEN / "tiny_qwen3"
    model, plain = lsx.Model.load(root, gpu, 64), PlainModel(root)
    prompts = np.stack([synth.prompt_tokens(60 + b, P, 512) for b in range(5)])
    tokens = model.generate_batch(prompts, maximum, cache_bits=4)
    assert tokens.shape == (5, maximum)
    for prompt, made in zip(prompts, tokens):
        z = plain.logits(np.concatenate([prompt, made[:-1]]).astype(int), P - 1)
        # The decoder's f32 leaves 1e-3 (the other decode tests' rule).  An element of the cache next to a border may take
        # the next level: one score moves by |q| s / sqrt(D), some 2 * 0.3 / 8, the output by that share of one value,
        # below 0.1 of a unit row, and a logit by less than 1e-2.
        short = z.max(1) - z[np.arange(maximum), made]
        assert (short < 1e-2).all(), short.max()
    assert np.array_equal(model.generate_batch(prompts, maximum, cache_bits=4), tokens)


def test_the_default_is_f32_and_the_caches_alternate(gpu):
    model = lsx.Model.load(GOLDEN / "tiny_qwen3", gpu, 64)
    prompts = np.stack([synth.prompt_tokens(70 + b, 12, 512) for b in range(3)])
    first, rounded = model.generate_batch(prompts, 5), model.generate_batch(prompts, 5, cache_bits=4)
    assert np.array_equal(model.generate_batch(prompts, 5, cache_bits=32), first)
    assert np.array_equal(model.generate_batch(prompts, 5, cache_bits=4), rounded)
    for bits in (0, 8, 16, -1):
        with pytest.raises((LsxError, OverflowError)):
            model.generate_batch(prompts, 5, cache_bits=bits)


def test_wide_heads_and_many_pages(gpu):
    """Qwen3-4B widths: the two caches' tokens agree where the prompt's last step leaves no doubt."""
    root = synth.cached_checkpoint("QWEN3_4B", seed=13, layers=2, vocab=8192)
    model = lsx.Model.load(root, gpu, 400)
    prompts = np.stack([synth.prompt_tokens(80 + b, 333, 8192) for b in range(4)])
    rounded = model.generate_batch(prompts, 3, cache_bits=4)
    _, _, margin, _ = model.score_batch(prompts, rounded[:, :1])
    assert (margin[:, 0] > -0.5).all(), margin  # rounding moves logits of standard deviation 1 by tenths


@pytest.mark.parametrize("P,maximum", [(125, 9), (187, 9)])
def test_every_step_over_pages(gpu, P, maximum):
    """Heads of 128, prompts over several pages and steps that pass a border of theirs: each token is the one of the plain
    model over a rounded cache, or as good as it."""
    root = synth.cached_checkpoint("QWEN3_4B", seed=13, layers=2, vocab=8192)
    model, plain = lsx.Model.load(root, gpu, 400), PlainModel(root)
    prompts = np.stack([synth.prompt_tokens(90 + b, P, 8192) for b in range(2)])
    tokens = model.generate_batch(prompts, maximum, cache_bits=4)
    for prompt, made in zip(prompts, tokens):
        z = plain.logits(np.concatenate([prompt, made[:-1]]).astype(int), P - 1)
        # as above; here a level moves one score among a hundred or more by 2 * 0.4 / 11, the output by a thousandth of a unit
        # row and less, and some hundred elements of the cache may lie that near to a border: 1e-2 of a logit at most
        short = z.max(1) - z[np.arange(maximum), made]
        assert (short < 1e-2).all(), short
