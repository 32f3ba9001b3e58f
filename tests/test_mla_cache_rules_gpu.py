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
