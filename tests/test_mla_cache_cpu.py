"""The 8-bit MLA latent cache off the GPU: its format, the cache object, the gated-MLA layer on it and the
serving decoder.  The layer's oracle rebuilds K and V from the dequantised latents."""
import math

import pytest
import torch

from kimi_k3_b200.models.mla import (ABSORBED_QUERY_LIMIT, E4M3, GatedMLA, GatedMLAConfig, MLACache, QuantizedMLACache,
                                     StaticMLACache, dequantize_latents, mla_attention, quantize_latents)


# ------------------------------------------------------------------------------------------ format
def _nearest_e4m3(v: float) -> float:
    """Round to the nearest e4m3 value, ties to even, by the definition of the format."""
    if v == 0:
        return 0.0
    e = max(math.floor(math.log2(abs(v))), -6)
    step = 2.0 ** (e - 3)
    q = abs(v) / step
    f = math.floor(q)
    n = f + (1 if q - f > 0.5 or (q - f == 0.5 and f % 2) else 0)
    return math.copysign(n * step, v)


def test_quantise_is_the_least_power_of_two_and_the_nearest_code():
    g = torch.Generator().manual_seed(0)
    rows = [torch.randn(9, generator=g) * 2.0 ** e for e in (-130, -40, -3, 0, 5, 60, 110)]
    rows += [torch.tensor([448.0] + [0.1] * 8), torch.tensor([448.5] + [0.1] * 8), torch.zeros(9)]
    x = torch.stack(rows)
    codes, scales = quantize_latents(x)
    assert codes.dtype == E4M3 and scales.dtype == torch.float32
    for row, c, s in zip(x.double().tolist(), codes.float().tolist(), scales.tolist()):
        top = max(abs(v) for v in row)
        k = -126
        while top > 448.0 * 2.0 ** k:
            k += 1
        assert s == 2.0 ** k
        assert c == [_nearest_e4m3(v / s) for v in row]


def test_non_finite_rows_and_exactness_in_bf16():
    x = torch.randn(4, 16)
    x[1, 3], x[2, 0] = math.inf, math.nan
    codes, scales = quantize_latents(x)
    assert torch.isnan(scales[1:3]).all() and not codes[1:3].float().any()
    values = dequantize_latents(codes, scales)
    assert torch.isnan(values[1:3]).all() and torch.isfinite(values[[0, 3]]).all()
    keep = values[[0, 3]]
    assert torch.equal(keep.bfloat16().float(), keep)
    # within half a step: 2^-4 relative to the element, or the smallest step of the row
    bound = torch.maximum(keep.abs() * 2.0 ** -3, scales[[0, 3], None] * 2.0 ** -9) * 0.5 + 1e-30
    assert ((keep - x[[0, 3]]).abs() <= bound).all()


# ------------------------------------------------------------------------------------------ the cache object
def test_append_ragged_single_and_overhanging_tokens():
    b, t, l, slots = 3, 4, 8, 6
    g = torch.Generator().manual_seed(1)
    c = QuantizedMLACache.zeros(b, slots, l)
    x = torch.randn(b, t, l, generator=g)
    mask = torch.tensor([[1, 1, 1, 1], [1, 1, 0, 0], [0, 0, 0, 0]], dtype=torch.bool)
    assert c.append(x, mask) is c
    assert c.sequence_offset.tolist() == [4, 2, 0]
    want = torch.zeros(b, slots, l)
    dq = dequantize_latents(*quantize_latents(x))
    want[0, :4], want[1, :2] = dq[0], dq[1, :2]
    assert torch.equal(c.read(), want)
    y = torch.randn(b, 1, l, generator=g)
    for step in range(4):  # row 0 fills up and keeps overwriting its last slot
        c.append(y + step)
    dy = [dequantize_latents(*quantize_latents(y + s))[:, 0] for s in range(4)]
    values = c.read()
    assert c.sequence_offset.tolist() == [8, 6, 4]
    assert torch.equal(values[0, 4], dy[0][0]) and torch.equal(values[0, 5], dy[3][0])
    assert torch.equal(values[1, 2:6], torch.stack([d[1] for d in dy]))
    c.append(x)  # several tokens: what overhangs is dropped
    assert torch.equal(c.read()[0], values[0])
    assert torch.equal(c.read()[2, 4:], dq[2, :2])


def test_from_cache_load_clone_reorder_and_report():
    b, l = 2, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn(b, 5, l, generator=g)
    mask = torch.tensor([[1, 1, 1, 1, 1], [1, 1, 0, 0, 0]], dtype=torch.bool)
    plain = MLACache.empty(b, l, dtype=torch.float32).append(x, mask)
    c = QuantizedMLACache.from_cache(plain, 9)
    assert c.cache_length == 9 and c.sequence_offset.tolist() == [5, 2]
    dq = dequantize_latents(*quantize_latents(x))
    assert torch.equal(c.read()[0, :5], dq[0]) and torch.equal(c.read()[1, :2], dq[1, :2]) and not c.read()[1, 2:].any()
    d = c.clone()
    d.append(torch.ones(b, 1, l))
    assert c.sequence_offset.tolist() == [5, 2] and d.sequence_offset.tolist() == [6, 3]
    r = c.reorder(torch.tensor([1, 0, 1]))
    assert r.sequence_offset.tolist() == [2, 5, 2] and torch.equal(r.read()[1], c.read()[0])
    ptr = c.latent_kv.data_ptr()
    c.load(MLACache.empty(b, l, dtype=torch.float32).append(x[:, :3], None))
    assert c.latent_kv.data_ptr() == ptr and c.sequence_offset.tolist() == [3, 3]
    assert torch.equal(c.read()[:, :3], dq[:, :3]) and not c.read()[:, 3:].any()
    # the report counts codes and scales
    from kimi_k3_b200.infer.session import cache_memory_bytes
    from kimi_k3_b200.models.backbone import HybridLayerCache
    layer = HybridLayerCache("gated_mla", c)
    assert layer.num_elements == b * 9 * l
    assert cache_memory_bytes(layer) == b * 9 * l + b * 9 * 4 + b * 8


def test_refusals():
    with pytest.raises(ValueError):
        QuantizedMLACache(torch.zeros(1, 2, 4), torch.zeros(1, 2), torch.zeros(1, dtype=torch.long))
    with pytest.raises(ValueError):
        QuantizedMLACache(torch.zeros(1, 2, 4).to(E4M3), torch.zeros(1, 3), torch.zeros(1, dtype=torch.long))
    with pytest.raises(ValueError):
        QuantizedMLACache.zeros(0, 1, 1)
    c = QuantizedMLACache.zeros(2, 3, 4)
    for bad in ((torch.zeros(1, 1, 4),), (torch.zeros(2, 1, 5),), (torch.zeros(2, 2, 4), torch.ones(2, 1, dtype=torch.bool)),
                (torch.zeros(2, 1, 4), torch.ones(2, 1))):
        with pytest.raises(ValueError):
            c.append(*bad)
    with pytest.raises(ValueError, match="shorter"):
        QuantizedMLACache.from_cache(MLACache.empty(1, 4, dtype=torch.float32).append(torch.zeros(1, 5, 4)), 4)
    with pytest.raises(ValueError, match="exceeds"):
        c.load(MLACache.empty(2, 4, dtype=torch.float32).append(torch.zeros(2, 5, 4)))
    with pytest.raises(ValueError):
        c.reorder(torch.tensor([0.0]))


# ------------------------------------------------------------------------------------------ the layer
@pytest.mark.parametrize("tokens", [1, 3, 16, 21, ABSORBED_QUERY_LIMIT, ABSORBED_QUERY_LIMIT + 5])
@pytest.mark.parametrize("ragged", [False, True])
def test_layer_on_the_quantised_cache(tokens, ragged):
    torch.manual_seed(3)
    cfg = GatedMLAConfig(d_model=24, num_heads=3, q_head_dim=8, v_head_dim=8, kv_latent_dim=16)
    layer = GatedMLA(cfg).double().eval()
    b, prompt, slots = 3, 7, 40 if tokens <= 21 else tokens + 19
    mask0 = torch.ones(b, prompt, dtype=torch.bool)
    mask0[1, 4:] = False
    with torch.no_grad():
        pre = layer(torch.randn(b, prompt, 24, dtype=torch.float64), mask0, use_cache=True).cache
        cache = QuantizedMLACache.from_cache(pre, slots)
        before = cache.sequence_offset.clone()
        x = torch.randn(b, tokens, 24, dtype=torch.float64)
        mask = None
        if ragged:
            mask = torch.arange(tokens)[None, :] < torch.tensor([tokens, max(1, tokens // 2), 1])[:, None]
        out = layer(x, mask, cache=cache, use_cache=True)
    counts = torch.full((b,), tokens) if mask is None else mask.sum(1)
    assert out.cache is cache and torch.equal(cache.sequence_offset, before + counts)
    with torch.no_grad():
        values = cache.read(torch.float64)
        q = layer.projections.project_queries(x)
        k, v = layer.projections.reconstruct_kv(values)
        live = torch.ones(b, tokens, dtype=torch.bool) if mask is None else mask
        raw = mla_attention(q, k, v, cache.valid_mask(), is_causal=True, keep_output_fp32=True, query_mask=live,
                            query_positions=before[:, None] + torch.arange(tokens))
        want, _ = layer._postprocess(raw, x)
        want = want * live[..., None]
    # the scales and the absorbed path are float64 throughout; only the order of the sums differs
    assert torch.allclose(out.hidden_states, want, rtol=0, atol=1e-12)
    # the new tokens' latents are in the cache, quantised
    lat = layer.projections.compress_kv(x)
    dq = dequantize_latents(*quantize_latents(lat), torch.float64)
    for i in range(b):
        n = int(counts[i])
        assert torch.equal(values[i, before[i]:before[i] + n], dq[i, :n])


def test_layer_with_attentions_and_diagnostics_reads_the_cache():
    torch.manual_seed(4)
    cfg = GatedMLAConfig(d_model=16, num_heads=2, q_head_dim=8, v_head_dim=8, kv_latent_dim=8)
    layer = GatedMLA(cfg).eval()
    with torch.no_grad():
        pre = layer(torch.randn(2, 5, 16), use_cache=True).cache
        x = torch.randn(2, 2, 16)
        a = layer(x, cache=QuantizedMLACache.from_cache(pre, 9))
        p = layer(x, cache=QuantizedMLACache.from_cache(pre, 9), output_attentions=True, output_diagnostics=True)
    assert torch.allclose(a.hidden_states, p.hidden_states, atol=1e-6)
    assert p.attentions.shape == (2, 2, 2, 9) and torch.allclose(p.attentions.sum(-1), torch.ones(2, 2, 2))
    assert not p.attentions[:, :, 0, 6:].any()


# ------------------------------------------------------------------------------------------ the decoder
def test_decoder_with_a_quantised_cache():
    from kimi_k3_b200 import KimiK3, kimi_k3_cpu_tiny_config
    from kimi_k3_b200.infer import GenerationConfig, GraphDecoder, graph_generate
    from kimi_k3_b200.models.backbone import HybridBackboneCache
    from kimi_k3_b200.infer.graph_decode import _static_layer
    torch.manual_seed(5)
    model = KimiK3(kimi_k3_cpu_tiny_config()).eval()
    vocab = model.config.vocab_size
    ids = torch.randint(8, vocab, (2, 6))  # past the visual placeholder ids
    cfg = GenerationConfig(max_new_tokens=5)
    dec = GraphDecoder(model, max_length=16, generation_config=cfg, cache_dtype=E4M3)
    out = dec.generate(ids)
    kinds = {type(lc.state) for lc in out.cache.layer_caches if lc.attention_type == "gated_mla"}
    assert kinds == {QuantizedMLACache}
    # the same steps by hand
    with torch.inference_mode():
        pre = model(input_ids=ids, use_cache=True, return_dict=True)
        cache = HybridBackboneCache(tuple(_static_layer(lc, 16, E4M3) for lc in pre.cache.layer_caches),
                                    pre.cache.sequence_length)
        tok, got = pre.logits[:, -1].argmax(-1), []
        for _ in range(5):
            got.append(tok)
            step = model(input_ids=tok[:, None], cache=cache, use_cache=True, return_dict=True)
            cache, tok = step.cache, step.logits[:, -1].argmax(-1)
    assert torch.equal(out.generated_ids, torch.stack(got, 1))
    again = graph_generate(model, ids, max_length=16, generation_config=cfg, cache_dtype=E4M3)
    assert torch.equal(again.generated_ids, out.generated_ids)
    plain = GraphDecoder(model, max_length=16, generation_config=cfg).generate(ids)
    assert {type(lc.state) for lc in plain.cache.layer_caches if lc.attention_type == "gated_mla"} == {StaticMLACache}
    assert out.cache_stats["memory_bytes"] < plain.cache_stats["memory_bytes"]
    with pytest.raises(ValueError, match="cache_dtype"):
        GraphDecoder(model, max_length=16, cache_dtype=torch.float16)


def test_cli_takes_the_cache_dtype():
    from kimi_k3_b200.cli import build_parser
    args = build_parser().parse_args(["infer", "--checkpoint", "c", "--prompt", "1", "--graph", "--cache-dtype", "e4m3"])
    assert args.cache_dtype == "e4m3"
    assert build_parser().parse_args(["infer", "--checkpoint", "c", "--prompt", "1"]).cache_dtype == "model"
