"""The 8-bit MLA latent cache off the GPU: refusals and values away from the ordinary ones."""
import math

import pytest
import torch

from kimi_k3_b200.models.mla import GatedMLA, GatedMLAConfig, MLACache, QuantizedMLACache


def _cache(b=2, tokens=5, slots=12, width=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    plain = MLACache.empty(b, width, dtype=torch.float32).append(torch.randn(b, tokens, width, generator=g))
    return QuantizedMLACache.from_cache(plain, slots)


def test_gradients_are_refused_not_dropped():
    """The cache keeps no gradient: a latent or a query that needs one is refused and leaves the cache as it was."""
    cache = _cache()
    codes, offsets = cache.latent_kv.view(torch.uint8).clone(), cache.sequence_offset.clone()
    x = torch.randn(2, 3, 8, requires_grad=True)
    for call in (lambda: cache.append(x), lambda: cache.attend(x[:, :, None]),
                 lambda: cache.load(MLACache.empty(2, 8, dtype=torch.float32).append(x))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    assert torch.equal(cache.latent_kv.view(torch.uint8), codes) and torch.equal(cache.sequence_offset, offsets)
    layer = GatedMLA(GatedMLAConfig(d_model=16, num_heads=2, q_head_dim=8, v_head_dim=8, kv_latent_dim=8))
    with pytest.raises(RuntimeError, match="no backward"):
        layer(torch.randn(2, 1, 16), cache=cache, use_cache=True)
    assert torch.equal(cache.sequence_offset, offsets)
    with torch.no_grad():
        cache.append(x)
        cache.attend(x[:, :, None])
    assert cache.sequence_offset.tolist() == [8, 8]


def test_a_nan_token_reaches_only_the_queries_that_see_it():
    cache = _cache(tokens=6)
    q = torch.randn(2, 3, 4, 8, generator=torch.Generator().manual_seed(1))
    want = cache.attend(q)
    cache.scales[0, 5] = math.nan  # seen by the last query token alone
    cache.latent_kv.view(torch.uint8)[0, 5] = 0
    got = cache.attend(q)
    assert torch.isnan(got[0, 2]).all() and torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1], want[1])


def test_generation_honours_the_cache_dtype_or_refuses_it(tmp_path):
    """Without the serving decoder there is no 8-bit cache to hold; with it there is one on the CPU too."""
    from kimi_k3_b200.config.model_yaml import build_model_from_yaml
    from kimi_k3_b200.config.profiles import write_pipeline
    from kimi_k3_b200.infer import GenerationConfig, InferenceYamlConfig
    from kimi_k3_b200.infer.distributed import run_distributed_generation
    from kimi_k3_b200.parallel.config import DistributedConfig
    write_pipeline("cpu_smoke", tmp_path)
    model = build_model_from_yaml(tmp_path / "model.yaml")
    torch.save({"model_state_dict": model.state_dict(), "format_version": 1}, tmp_path / "ckpt.pt")
    iy = InferenceYamlConfig(GenerationConfig(max_new_tokens=4, device="cpu"), DistributedConfig(), None)
    args = (tmp_path / "model.yaml", tmp_path / "ckpt.pt", [5, 17, 9, 33], iy)
    with pytest.raises(ValueError, match="use_graph"):
        run_distributed_generation(*args, cache_dtype=torch.float8_e4m3fn)
    out, context = run_distributed_generation(*args, use_graph=True, cache_dtype=torch.float8_e4m3fn)
    context.close()
    states = [lc.state for lc in out.cache.layer_caches if lc.attention_type == "gated_mla"]
    assert states and all(isinstance(s, QuantizedMLACache) for s in states)


def test_positions_past_every_slot_do_not_wrap():
    cache = _cache()
    q = torch.randn(2, 3, 4, 8, generator=torch.Generator().manual_seed(2))
    ends = torch.iinfo(torch.int64)
    all_keys = cache.attend(q, query_start=torch.tensor([100, 5]))
    got = cache.attend(q, query_start=torch.tensor([ends.max, ends.max]))
    assert torch.equal(got, all_keys) and got.any()
    assert not cache.attend(q, query_start=torch.tensor([ends.min, -3])).any()
    ints = cache.attend(q, query_start=torch.full((2,), torch.iinfo(torch.int32).max, dtype=torch.int32))
    assert torch.equal(ints, all_keys)
