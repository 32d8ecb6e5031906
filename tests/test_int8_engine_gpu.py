"""The engine with 8-bit matrices and an 8-bit cache, against a plain decoder whose matrices, tokens and cached rows go
through the same codes in 64 bits."""

import numpy as np
import pytest
import torch

import cuttings
import plain_llama
from plain_llama import PlainLlama, TINY_WEIGHTS, tiny_configs

pytestmark = pytest.mark.gpu
MODES = [dict(linear_dtype="int8"), dict(kv_cache_dtype="int8"), dict(linear_dtype="int8", kv_cache_dtype="int8")]


def held(x, dims):
    """The values that 8-bit codes with one scale over ``dims`` stand for: scale and code by the definition's float32 steps
    (matrices of bfloat16 numbers have quotients that are exact halves, which the scale's rounding decides)."""
    x32 = x.float()
    s = x32.abs().amax(dims, keepdim=True) * (1 / 127)
    return torch.where(s > 0, torch.round(x32 / s).clamp(-127, 127).double() * s.double(), 0.0)


class Plain8(PlainLlama):
    """Every prompt is one portion, so a page's scale is that of all the tokens in it."""

    def __init__(self, folder, page_size, linears, cache):
        super().__init__(folder, torch.float64)
        self.page_size, self.linears, self.cache = page_size, linears, cache
        if linears:
            self.w = {n: held(t, 1) if ".layers." in n and t.dim() == 2 else t for n, t in self.w.items()}

    def rows(self, x):  # tokens on their way into a product
        return held(x, 1) if self.linears else x

    def paged(self, x):  # [T, heads, hd]
        if not self.cache:
            return x
        return torch.cat([held(p, (0, 2)) for p in x.split(self.page_size)])

    def logits(self, token_ids):
        c, w = self.cfg, self.w
        nh, nkv = c["num_attention_heads"], c["num_key_value_heads"]
        hd, T = c["hidden_size"] // nh, len(token_ids)
        cos, sin = plain_llama.rope_tables(torch.arange(T), self.inv_freq)
        x = w["model.embed_tokens.weight"][torch.tensor(token_ids)]
        for i in range(c["num_hidden_layers"]):
            p = f"model.layers.{i}"
            h = self.rows(plain_llama.rms_norm(x, w[f"{p}.input_layernorm.weight"], c["rms_norm_eps"]))
            q, k, v = ((h @ w[f"{p}.self_attn.{n}_proj.weight"].T).view(T, m, hd) for n, m in (("q", nh), ("k", nkv), ("v", nkv)))
            q, k = (plain_llama.apply_rope(t, cos, sin) for t in (q, k))
            a = plain_llama.causal_gqa_attention(q, self.paged(k), self.paged(v)).reshape(T, -1)
            x = x + self.rows(a) @ w[f"{p}.self_attn.o_proj.weight"].T
            h = self.rows(plain_llama.rms_norm(x, w[f"{p}.post_attention_layernorm.weight"], c["rms_norm_eps"]))
            act = torch.nn.functional.silu(h @ w[f"{p}.mlp.gate_proj.weight"].T) * (h @ w[f"{p}.mlp.up_proj.weight"].T)
            x = x + self.rows(act) @ w[f"{p}.mlp.down_proj.weight"].T
        return plain_llama.lm_head(x, w, c)


def make(folder, **kw):
    from tokasaurus_b200.engine.engine import Engine

    return Engine(model=str(folder), **dict(dict(kv_cache_num_tokens=2048, allocator_sanity_checks=True), **kw))


def step_logits(eng, prompt):
    from tokasaurus_b200.engine.batch import StepEntry

    r = eng.runner
    r.cache.admit("x")
    r.cache.ensure_capacity("x", len(prompt))
    out = r.step([StepEntry("x", prompt, 0, list(range(len(prompt))))]).double().cpu()
    r.check_status()
    r.cache.free("x")
    return out


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("cfg_index", [0, 1])
def test_logits_of_whole_prompts(tiny_model_dirs, cfg_index, mode):
    folder, ps, vocab = tiny_model_dirs[cfg_index], TINY_WEIGHTS[cfg_index]["page_size"], tiny_configs()[cfg_index]["vocab_size"]
    plain = Plain8(folder, ps, "linear_dtype" in mode, "kv_cache_dtype" in mode)
    bare = PlainLlama(folder, torch.float64)
    eng = make(folder, dtype="float32", page_size=ps, **mode)
    for n in (1, 2, 17, 63, 100):
        prompt = cuttings.random_tokens(n, vocab, n)
        got, want, full = step_logits(eng, prompt), plain.logits(prompt), bare.logits(prompt)
        top = full.abs().max()
        # a number next to a half may go to the other code: a few in a thousand results, each by a code's share of a sum
        assert (got - want).abs().max() <= 0.02 * top and (got - want).pow(2).mean().sqrt() <= 0.002 * top
        # and 8 bits are near the model they stand for
        assert (got - full).pow(2).mean().sqrt() <= 0.05 * top


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cfg_index", [0, 1])
def test_generation_every_way_of_running(tiny_model_dirs, cfg_index, dtype, mode):
    """Chunked prompts beside decoding requests, with step graphs and without: tokens near the model's best."""
    folder, ps, vocab = tiny_model_dirs[cfg_index], TINY_WEIGHTS[cfg_index]["page_size"], tiny_configs()[cfg_index]["vocab_size"]
    prompts = [cuttings.random_tokens(n, vocab, 7 * n) for n in (1, 29, 64, 90)]
    plain = PlainLlama(folder, torch.float64)
    found = {}
    for graphs in (True, False):
        for most in (24, 8192):
            eng = make(folder, dtype=dtype, page_size=ps, use_cudagraphs=graphs, max_tokens_per_forward=most, **mode)
            outs = eng.generate(prompts, max_num_tokens=20, ignore_eos=True)
            assert not eng.runner.cache.requests
            for p, o in zip(prompts, outs):
                logits = plain.logits(p + o.completion_ids[:-1])[len(p) - 1:]
                top = logits.abs().max().item()
                assert len(o.completion_ids) == 20
                assert all(logits[i, t] >= logits[i].max() - 0.12 * top for i, t in enumerate(o.completion_ids))
            found[graphs, most] = [o.completion_ids for o in outs]
    for most in (24, 8192):
        if dtype == "float32":  # the same steps, recorded or not
            assert found[True, most] == found[False, most]


def test_a_decode_graph_serves_growing_contexts(tiny_model_dirs):
    """One recorded graph from the first tokens of a request to its hundredth, over pages that fill and begin."""
    folder = tiny_model_dirs[1]
    prompt = cuttings.random_tokens(3, 509, 5)
    runs = []
    for graphs in (True, False):
        eng = make(folder, dtype="float32", page_size=8, use_cudagraphs=graphs, linear_dtype="int8", kv_cache_dtype="int8")
        runs.append(eng.generate([prompt], max_num_tokens=110, ignore_eos=True)[0])
    assert runs[0].completion_ids == runs[1].completion_ids
    np.testing.assert_allclose(runs[0].logprobs, runs[1].logprobs, atol=1e-3)


def test_other_families_refuse_the_options():
    import verozen_models
    from tokasaurus_b200.config.engine_config import EngineConfig, OptionError
    from tokasaurus_b200.engine.runner import ModelRunner

    cfg = verozen_models.MODELS["d"]["config"]
    with pytest.raises(OptionError, match="dtype only"):
        ModelRunner(EngineConfig(random_weights=0, kv_cache_dtype="int8"), dict(cfg))
