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
