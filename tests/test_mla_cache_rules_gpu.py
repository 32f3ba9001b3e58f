"""The 8-bit MLA latent cache on the GPU: rules of the attention kernel and of the layer that calls it which hold at
sizes, values and states away from the ordinary ones."""
import math

import pytest
import torch

from test_mla_cache_gpu import E4M3, UNIT, check_attention, make_cache, quantise64, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [144, 272, 400, 528, 1040, 1488])
def test_last_columns_end_inside_a_warp(cuda, width, dtype):
    """Widths that end 16 or 80 columns into a block of 128, over runs of several sequences a CTA: the lanes of a warp
    that have no column left rejoin the others before the next block is read."""
    from kimi_k3_b200 import ops
    b, h, slots = 160, 6, 200
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, 1, h, width, dtype, cuda)
    lens = torch.tensor([(i * 71) % (slots + 1) for i in range(b)], device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens, scale=0.6), q, codes, scales, lens, 0.6)


def dominated(cuda, dtype, slots, first, floor=0.0, stretch=0):
    """One token outweighs each of the others by 2^18 .. 2^33 (a head each); in half of the columns its code is zero, so
    the output there is the tail alone, equal weights all of them.  160 query tokens of one sequence give every CTA whole
    walks along the cache.  Returns each head's worst error as a share of the tolerance.

    Tolerance per element: that of check_attention, plus what weights that are held to within `floor` of the largest one
    may lose: at most `stretch` tokens share a stretch with the dominating one, each with a code of the column's size."""
    from kimi_k3_b200 import ops
    width, h, tq, scale, c = 64, 32, 160, 0.5, 4.0
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn(1, slots, width, generator=g, device=cuda).abs() + 0.5
    x[..., 0] = -c
    at = 3 if first else slots // 2 + 3
    x[0, at, 0] = c
    x[0, at, 1:width // 2] = 0.0
    codes, scales = (t.float() for t in quantise64(x))
    codes = codes.to(E4M3)
    q = torch.zeros(1, 1, h, width, device=cuda)
    q[0, 0, :, 0] = torch.linspace(18.0, 33.0, h, device=cuda) * (math.log(2.0) / (2 * c * scale))
    q = q.to(dtype)
    lens = torch.tensor([slots], device=cuda)
    out = ops.mla_cache_attention(q.expand(1, tq, h, width), codes, scales, lens, query_start=lens, scale=scale)
    values = codes[0].double() * scales[0, :, None].double()
    p = torch.softmax(q[0, 0].double() @ values.T * scale, -1)  # [h, slots]
    ref, size = p @ values, p @ values.abs()
    u = UNIT[dtype]
    lost = floor * p.amax(-1, keepdim=True) * min(slots, stretch) * values.abs().amax(0)
    tol = 0.5 * u * ref.abs() + u * size + lost
    return ((out[0].double() - ref).abs() / tol).amax(dim=(0, 2)).tolist()


@pytest.mark.parametrize("slots", [4608, 32768, 131072])
@pytest.mark.parametrize("first", [True, False])
def test_one_dominating_token_and_a_flat_tail_fp32(cuda, first, slots):
    """Many equal weights round the same way at every addition: the sums along a cache keep their rounding."""
    worst = dominated(cuda, torch.float32, slots, first)
    assert max(worst) <= 1.0, worst


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slots", [4608, 32768, 131072])
@pytest.mark.parametrize("first", [True, False])
def test_one_dominating_token_and_a_flat_tail(cuda, first, slots, dtype):
    """A key's weight is held to within 2^-25 (bf16) or 2^-27 (fp16) of the largest weight of its stretch of the cache,
    8,192 tokens at most."""
    worst = dominated(cuda, dtype, slots, first, 2.0 ** (-25 if dtype == torch.bfloat16 else -27), 8192)
    assert max(worst) <= 1.0, worst


def test_more_parts_than_one_block_lists(cuda):
    """A sequence so long that its stretches outnumber the log-sums a joining block keeps at hand."""
    from kimi_k3_b200 import ops
    slots, width, h = 4_300_000, 64, 2
    g = torch.Generator(device=cuda).manual_seed(2)
    codes = torch.randint(0, 0x70, (1, slots, width), generator=g, device=cuda, dtype=torch.uint8).view(E4M3)
    scales = torch.full((1, slots), 2.0 ** -9, device=cuda)
    q = queries(1, 1, h, width, torch.bfloat16, cuda, spread=6.0)
    lens = torch.tensor([slots - 5], device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens), q, codes, scales, lens, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_past_every_slot_do_not_wrap(cuda, dtype):
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = 3, 3, 4, 768, 100
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    ends = torch.iinfo(torch.int64)
    lens = torch.tensor([100, 40, ends.max], device=cuda)  # a length past the slots is the slots
    far = torch.tensor([ends.max, ends.max - 1, 100], device=cuda)
    want = ops.mla_cache_attention(q, codes, scales, lens, query_start=torch.full_like(lens, slots))
    assert torch.equal(ops.mla_cache_attention(q, codes, scales, lens, query_start=far), want) and want.any()
    assert torch.equal(ops.mla_cache_attention(q, codes, scales, lens, query_start=far.clamp(max=2 ** 31 - 1).int()), want)
    assert not ops.mla_cache_attention(q, codes, scales, lens, query_start=torch.full_like(lens, ends.min)).any()
    before = codes.view(torch.uint8).clone()
    x = torch.randn(b, 2, width, device=cuda).to(dtype)
    ops.mla_cache_write(x, codes, scales, torch.tensor([ends.max, ends.min, slots], device=cuda))
    assert torch.equal(codes.view(torch.uint8), before)


def test_workspace_does_not_grow_with_the_row_tiles(cuda):
    """Parts of contexts are held for what the CTAs cut, two a CTA at most, however many row tiles a prompt piece makes.
    Beside the output a call holds its query parts, as many bytes as the queries rounded up to the tile's rows."""
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = 24, 60, 24, 640, 4000
    codes, scales = make_cache(b, 8, width, cuda)
    codes = codes.view(torch.uint8).repeat(1, slots // 8, 1).view(E4M3)
    scales = scales.repeat(1, slots // 8)
    q = queries(b, tq, h, width, torch.bfloat16, cuda)
    lens = torch.full((b,), slots, device=cuda)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.mla_cache_attention(q, codes, scales, lens, scale=0.6)
    used = torch.cuda.max_memory_allocated() - before
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    size = q.numel() * q.element_size()
    assert used <= 2 * size * 33 // 32 + 2 * sms * 32 * (width + 1) * 4 + (8 << 20), used
    rows = slice(0, 2)
    check_attention(out[rows], q[rows], codes[rows], scales[rows], lens[rows], 0.6)


# ------------------------------------------------------------------------------------------ the layer's choice
def _layer(cuda, width, d_model=128, heads=2):
    from kimi_k3_b200.models.mla import GatedMLA, GatedMLAConfig
    torch.manual_seed(11)
    return GatedMLA(GatedMLAConfig(d_model=d_model, num_heads=heads, q_head_dim=64, v_head_dim=64,
                                   kv_latent_dim=width)).to(cuda).eval()


@pytest.mark.parametrize("tokens", [1, 3])
def test_layer_with_a_latent_wider_than_the_attention_takes(cuda, tokens, monkeypatch):
    """Widths that the attention kernel refuses are read back and rebuilt: the layer runs, and equals its PyTorch form
    within a few fp32 roundings of the output's size."""
    from kimi_k3_b200 import ops
    from kimi_k3_b200.models.mla import QuantizedMLACache
    layer = _layer(cuda, 2176, d_model=1152, heads=18)
    assert ops.mla_cache_attention_form(torch.float32, 2176) is None
    b, prompt = 2, 37
    x0, x = torch.randn(b, prompt, 1152, device=cuda), torch.randn(b, tokens, 1152, device=cuda)
    with torch.no_grad():
        first = QuantizedMLACache.from_cache(layer(x0, use_cache=True).cache, 48)
        outs = []
        for kernels in ("1", "0"):
            monkeypatch.setenv("KIMI_K3_KERNELS", kernels)
            cache = first.clone()
            outs.append(layer(x, cache=cache, use_cache=True).hidden_states)
            assert cache.sequence_offset.tolist() == [prompt + tokens] * b
    err = (outs[0] - outs[1]).abs().max().item() / outs[1].abs().max().item()
    assert err <= 2.0 ** -11, err


def test_decoder_with_a_latent_wider_than_the_attention_takes(cuda):
    from kimi_k3_b200.config.model_yaml import build_model_config_from_mapping
    from kimi_k3_b200.config.profiles import profile_model_mapping
    from kimi_k3_b200.infer import GenerationConfig, GraphDecoder
    from kimi_k3_b200.models import KimiK3
    m = profile_model_mapping("t4_wikitext")
    m["model"].update(d_model=1152, num_heads=18, num_hybrid_groups=1, vocab_size=1000)
    m["model"]["moe"].update(latent_dim=64, shared_expert_hidden_dim=96, routed_expert_hidden_dim=128)
    m["model"]["mla"]["kv_latent_dim"] = 2176
    torch.manual_seed(5)
    model = KimiK3(build_model_config_from_mapping(m)).to(cuda).eval()
    ids = torch.randint(5, 1000, (2, 21), device=cuda)
    for use_graph in (True, False):
        out = GraphDecoder(model, max_length=40, generation_config=GenerationConfig(max_new_tokens=6), cache_dtype=E4M3,
                           use_graph=use_graph).generate(ids)
        assert out.generated_tokens == 6
        states = [lc.state for lc in out.cache.layer_caches if lc.attention_type == "gated_mla"]
        assert states and all(s.sequence_offset.tolist() == [26, 26] for s in states)


@pytest.mark.parametrize("dtype,width,tokens,attends", [
    (torch.bfloat16, 128, 64, True), (torch.bfloat16, 128, 65, False), (torch.bfloat16, 136, 8, True),
    (torch.bfloat16, 136, 9, False), (torch.float32, 128, 8, True), (torch.float32, 128, 9, False)])
def test_layer_attends_up_to_the_limit_of_the_form(cuda, dtype, width, tokens, attends, monkeypatch):
    """64 query tokens where the tensor cores attend, 8 where fp32 FMAs do; both forms against fp32 PyTorch."""
    from kimi_k3_b200.models import mla
    layer = _layer(cuda, width)
    calls = []
    attend = mla.QuantizedMLACache.attend
    monkeypatch.setattr(mla.QuantizedMLACache, "attend", lambda self, q, **kw: calls.append(q.dtype) or attend(self, q, **kw))
    b, prompt = 2, 50
    x0, x = torch.randn(b, prompt, 128, device=cuda), torch.randn(b, tokens, 128, device=cuda)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        first = mla.QuantizedMLACache.from_cache(layer(x0, use_cache=True).cache, prompt + tokens)
        out = layer(x, cache=first.clone(), use_cache=True).hidden_states.float()
        assert calls == ([dtype] if attends else [])
        monkeypatch.setenv("KIMI_K3_KERNELS", "0")
        want = layer(x, cache=first.clone(), use_cache=True).hidden_states.float()
    err = (out - want).abs().max().item() / want.abs().max().item()
    assert err <= (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -11), err


# ------------------------------------------------------------------------------------------ waits that gave up
@pytest.fixture
def status_word(cuda):
    """The device's record of waits that gave up; left clear."""
    from kimi_k3_b200.ops import _loader
    word = _loader.require().mla_cache_status_word()
    yield word
    torch.cuda.synchronize()
    word.zero_()
    torch.cuda.synchronize()


def test_check_waits_for_every_stream(cuda, status_word):
    """A record made late on a stream of its own is seen, reported once and cleared."""
    from kimi_k3_b200 import ops
    ops.mla_cache_check()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        status_word.fill_(3)
    with pytest.raises(RuntimeError, match="status 3"):
        ops.mla_cache_check(torch.device("cuda", torch.cuda.current_device()))
    ops.mla_cache_check()
    assert status_word.item() == 0


def test_decoder_checks_its_own_device(cuda, status_word, monkeypatch):
    from kimi_k3_b200 import ops
    from kimi_k3_b200.infer import GenerationConfig, GraphDecoder
    from test_decode_gpu import _small_model
    model = _small_model(cuda)
    asked, check = [], ops.mla_cache_check
    monkeypatch.setattr(ops, "mla_cache_check", lambda device=None: asked.append(device) or check(device))
    ids = torch.randint(5, 1000, (2, 9), device=cuda)
    cfg = GenerationConfig(max_new_tokens=3)
    GraphDecoder(model, max_length=16, generation_config=cfg, cache_dtype=E4M3).generate(ids)
    assert [torch.device(d) for d in asked] == [next(model.parameters()).device]
    asked.clear()
    GraphDecoder(model, max_length=16, generation_config=cfg).generate(ids)
    assert not asked


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(40, 2, 10, 640, 190), (3, 1, 6, 640, 9000), (2, 40, 24, 128, 700)],
                         ids=lambda s: "x".join(map(str, s)))
def test_results_are_nan_until_a_give_up_is_reported(cuda, status_word, shape, dtype):
    """With the record of a wait that gave up still set, rows with a key come back NaN, whole and joined ones alike; the
    check reports it, and the next call is right."""
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = shape
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([(slots, tq + 5, 65 + tq)[i % 3] for i in range(b)], device=cuda)
    status_word.fill_(2)
    assert torch.isnan(ops.mla_cache_attention(q, codes, scales, lens, scale=0.6)).all()
    with pytest.raises(RuntimeError, match="status 2"):
        ops.mla_cache_check()
    check_attention(ops.mla_cache_attention(q, codes, scales, lens, scale=0.6), q, codes, scales, lens, 0.6)
