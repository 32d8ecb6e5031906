"""What 8-bit serving declares on the host: options, the architectures that take them, the cache's layout and books."""

import pytest
import torch

from plain_llama import tiny_configs
from tokasaurus_b200.cache.manager import CacheManager
from tokasaurus_b200.config.engine_config import EngineConfig, OptionError, parse_overrides
from tokasaurus_b200.config.registry import known_architectures, lookup_architecture
from tokasaurus_b200.kernels.modules import int8_modules
from tokasaurus_b200.parts.attention import PagedAttention
from tokasaurus_b200.parts.base import PagedCacheNeed, QkvStage
from tokasaurus_b200.parts.int8 import Int8GatedMLP, Int8PagedAttention
from tokasaurus_b200.parts.mlp import GatedMLP
from tokasaurus_b200.parts.rope import RotaryEncoding


def build(**kw):
    arch = lookup_architecture(tiny_configs()[0])
    return arch.build_model(arch.parse_config(tiny_configs()[0]), **kw)


def test_options():
    cfg, _ = parse_overrides(["model=/m", "linear_dtype=int8", "kv_cache_dtype=int8"])
    assert cfg.finalize(128).linear_dtype == cfg.kv_cache_dtype == "int8"
    assert EngineConfig().finalize(128).linear_dtype is None
    for name in ("linear_dtype", "kv_cache_dtype"):
        with pytest.raises(OptionError, match=name):
            EngineConfig(**{name: "int4"}).finalize(128)


def test_architectures_that_take_them():
    assert lookup_architecture({"architectures": ["LlamaForCausalLM"]}).eight_bits
    assert [n for n in known_architectures() if lookup_architecture({"architectures": [n]}).eight_bits] == ["LlamaForCausalLM"]


@pytest.mark.parametrize("linears,cache", [(False, False), (True, False), (False, True), (True, True)])
def test_llama_in_parts(linears, cache):
    model = build(int8_linears=linears, int8_cache=cache)
    mixers, ffns = [b.mixer for b in model.blocks], [b.ffn for b in model.blocks]
    assert all(type(m) is (Int8PagedAttention if linears or cache else PagedAttention) for m in mixers)
    assert all(type(f) is (Int8GatedMLP if linears else GatedMLP) for f in ffns)
    assert {n.eight_bits for n in model.cache_entries().values()} == {cache}
    assert model.graph_safe and [s.name for s in model.weight_specs()] == [s.name for s in build().weight_specs()]
    sources = {s for s, _ in model.kernel_modules("bfloat16")}
    assert ("int8_product.cu" in sources) == (linears or cache) and ("attention_kv8.cu" in sources) == cache


def test_an_element_wise_stage_is_refused():
    names = dict(q_name="q", k_name="k", v_name="v", o_name="o")
    with pytest.raises(ValueError, match="stage"):
        Int8PagedAttention(64, 4, 2, 16, RotaryEncoding(16, 1e4), **names, qkv_stage=QkvStage(qk_norm_names=("a", "b")), int8_cache=True)


def test_cache_of_codes_and_scales():
    need8, need16 = PagedCacheNeed(2, 16, eight_bits=True), PagedCacheNeed(2, 16)
    m = CacheManager({0: need8, 1: need8, 2: need16}, 8, 5, 3, dtype=torch.float32, device="cpu")
    assert len(m.groups) == 2
    a, b, c = (m.layer_cache(e) for e in range(3))
    assert a.k.dtype == a.v.dtype == torch.int8 and a.k.shape == (5, 2, 8, 16) and a.k_scale.shape == a.v_scale.shape == (5, 2)
    assert a.k_scale.dtype == torch.float32 and a.k_scale.is_contiguous() and a.k.is_contiguous()
    assert len({t.data_ptr() for t in (a.k_scale, a.v_scale, b.k_scale, b.v_scale)}) == 4
    assert c.k.dtype == torch.float32 and c.k_scale is None and c.v_scale is None
    assert m.device_bytes_by_group() == [2 * 2 * 5 * 2 * (8 * 16 + 4), 1 * 2 * 5 * 2 * 8 * 16 * 4]
    assert [g.bytes_per_token(4) for g in m.groups] == [2 * 2 * 2 * 16, 1 * 2 * 2 * 16 * 4]
    books = CacheManager({0: need8}, 8, 5, 3)
    assert books.layer_cache(0).k_scale is None and books.device_bytes() == 0


def test_kernel_modules_by_head_size():
    assert int8_modules() == [("int8_product.cu", None), ("cache8.cu", None)]
    assert ("attention_kv8_tc.cu", {"TKB_HD": 128}) in int8_modules((128,)) and ("attention_kv8_tc.cu", {"TKB_HD": 256}) not in int8_modules((256,))
