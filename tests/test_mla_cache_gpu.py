"""The 8-bit MLA latent cache on the GPU: writer and reader against their definition in 64 bits (equal bit for
bit), attention against a 64-bit softmax over the cache's values, at the sizes, masks and layouts where they can
go wrong, and their refusals.

Attention tolerance, per element: one rounding of the output to its type, u * |o|, plus w * A with
A = sum_t p_t scale_t |code_t|, the size of what was added up.  w allows the weights and the query as much error as
one unit of the output's type (bf16 2^-8, fp16 2^-11); fp32 results are held to 2^-16, which covers the rounding of
scores of size up to ~16 summed over the latent axis (16 * 2^-24 * a few terms' growth, through the exponential)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -16}


def quantise64(x):
    """codes (as float64 values) and scales of the rows of ``x``, by the definition."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    k = torch.full_like(top, -126.0)
    for e in range(-126, 121):  # the least exponent under which the row fits
        k = torch.where(top > 448.0 * 2.0 ** (e - 1), torch.full_like(k, max(e, -126)), k)
    v = torch.where(bad, torch.zeros_like(x), x * torch.exp2(-k))
    ulp = torch.exp2((torch.frexp(v)[1].double() - 1).clamp(min=-6) - 3)
    return torch.round(v / ulp) * ulp, torch.where(bad, torch.full_like(top, math.nan), torch.exp2(k))[..., 0]


def make_cache(b, slots, width, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(b, slots, width, generator=g, device=device)
    x *= torch.exp2(torch.randint(-3, 4, (b, slots, 1), generator=g, device=device).float())
    codes, scales = quantise64(x)
    return codes.float().to(E4M3), scales.float()


def attention64(q, codes, scales, lengths, scale, start=None):
    """contexts and sum_t p |c| in float64; keys outside a row's mask are never touched."""
    b, tq, h, width = q.shape
    out = torch.zeros(b, tq, h, width, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), codes.shape[1])
        first = int(lengths[i]) - tq if start is None else int(start[i])
        for j in range(tq):
            m = min(n, first + j + 1)
            if m <= 0:
                continue
            c = codes[i, :m].double() * scales[i, :m, None].double()
            p = torch.softmax(q[i, j].double() @ c.T * scale, -1)
            out[i, j], size[i, j] = p @ c, p @ c.abs()
    return out, size


def check_attention(out, q, codes, scales, lengths, scale, start=None):
    ref, size = attention64(q, codes, scales, lengths, scale, start)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    u = UNIT[q.dtype]
    err = (out.double() - ref).abs()
    tol = 0.5 * u * ref.abs() + u * size + 1e-30
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"error {worst:.3f} of the tolerance"


def queries(b, tq, h, width, dtype, device, seed=1, spread=1.5):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(b, tq, h, width, generator=g, device=device) * (spread / math.sqrt(width) / 2)).to(dtype)


# ------------------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [1, 8, 100, 640, 1536, 1544, 2500])
def test_write_is_exact(cuda, dtype, width):
    from kimi_k3_b200 import ops
    g = torch.Generator(device=cuda).manual_seed(width)
    b, t, slots = 5, 7, 23
    x = torch.randn(b, t, width, generator=g, device=cuda)
    x *= torch.exp2(torch.randint(-30, 12, (b, t, 1), generator=g, device=cuda).float())
    x[0, 0] = 0.0
    x[0, 1, 0] = 448.0  # the maximum is itself representable
    x[0, 2, 0] = 449.0
    x[0, 3] = 2.0 ** -24  # fp16's smallest
    if dtype != torch.float16:
        x[0, 4] *= 1e30
        x[0, 5] *= 1e-38
    x = x.to(dtype)
    x[1, 2, width // 2] = math.inf
    x[1, 3, width - 1] = math.nan
    x[1, 4, 0] = -math.inf
    codes = torch.full((b, slots, width), 7.0, device=cuda).to(E4M3)
    scales = torch.full((b, slots), 3.0, device=cuda)
    offsets = torch.tensor([0, 16, 20, -2, 4], device=cuda)  # 20: runs past the buffer; -2: before it
    counts = torch.tensor([7, 7, 7, 7, 3], device=cuda)
    ops.mla_cache_write(x, codes, scales, offsets, counts)
    want_codes, want_scales = torch.full((b, slots, width), 7.0, device=cuda).double(), torch.full_like(scales, 3.0)
    qc, qs = quantise64(x)
    for i in range(b):
        for j in range(int(counts[i])):
            s = int(offsets[i]) + j
            if 0 <= s < slots:
                want_codes[i, s], want_scales[i, s] = qc[i, j], qs[i, j].float()
    assert torch.equal(codes.double(), want_codes)
    assert torch.equal(scales.nan_to_num(nan=-1.0), want_scales.nan_to_num(nan=-1.0))
    values = ops.mla_cache_read(codes, scales, dtype=torch.float32)
    assert torch.isnan(values[1, 16 + 2:16 + 5]).all()


def test_write_strides_and_index_types(cuda):
    from kimi_k3_b200 import ops
    b, t, width, slots = 3, 5, 640, 9
    x = torch.randn(t, b, width + 8, device=cuda).bfloat16()
    want_codes, want_scales = quantise64(x[..., :width].transpose(0, 1))
    views = [x[..., :width].transpose(0, 1),                                   # rows apart, aligned
             torch.cat((x[..., :1], x[..., :width]), -1)[..., 1:].transpose(0, 1),   # misaligned rows
             x[..., :width].transpose(0, 1).transpose(1, 2).contiguous().transpose(1, 2)]  # latent axis strided
    for v in views:
        for dt in (torch.int32, torch.int64):
            # a cache inside a larger buffer, batch and slots swapped, starting off an 8-byte boundary
            codes = torch.zeros(slots, b, width + 4, dtype=torch.uint8, device=cuda)[..., 4:].transpose(0, 1).view(E4M3)
            scales = torch.zeros(slots, b, device=cuda).transpose(0, 1)
            ops.mla_cache_write(v, codes, scales, torch.tensor([0, 4, 2], dtype=dt, device=cuda))
            for i, o in enumerate((0, 4, 2)):
                assert torch.equal(codes[i, o:o + t].double(), want_codes[i])
                assert torch.equal(scales[i, o:o + t].double(), want_scales[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [1, 12, 640, 1544])
def test_read_is_exact_and_zero_past_the_length(cuda, dtype, width):
    from kimi_k3_b200 import ops
    b, slots = 4, 19
    codes, scales = make_cache(b, slots, width, cuda)
    codes.view(torch.uint8)[:, 15:] = 0x7F  # NaN codes and scales where nothing is valid
    scales[:, 15:] = math.nan
    lengths = torch.tensor([15, 0, 1, -3], device=cuda)
    for tokens in (0, 1, 19):
        out = ops.mla_cache_read(codes, scales, lengths, dtype=dtype, tokens=tokens)
        want = torch.zeros(b, tokens, width, dtype=dtype, device=cuda)
        for i in range(b):
            n = max(0, min(int(lengths[i]), tokens))
            want[i, :n] = (codes[i, :n].double() * scales[i, :n, None].double()).to(dtype)
        assert torch.equal(out, want)
    whole = ops.mla_cache_read(codes[:, :15], scales[:, :15], dtype=dtype)
    assert torch.equal(whole, (codes[:, :15].double() * scales[:, :15, None].double()).to(dtype))


# ------------------------------------------------------------------------------------------ attention
SHAPES = [  # batch, queries, heads, width, slots, lengths
    (1, 1, 1, 640, 64, [1]), (1, 1, 10, 640, 257, [257]), (3, 1, 10, 640, 300, [0, 65, 300]),
    (2, 1, 12, 768, 129, [64, 128]), (2, 1, 16, 1024, 200, [63, 200]), (3, 1, 24, 1536, 190, [190, 1, 127]),
    (2, 1, 3, 1536, 700, [700, 33]), (2, 4, 12, 768, 260, [260, 130]), (3, 3, 5, 640, 70, [2, 70, 1]),
    (2, 8, 24, 1536, 100, [100, 50]), (1, 40, 10, 640, 90, [90]), (1, 1, 7, 2048, 66, [66]), (2, 2, 3, 64, 40, [40, 9]),
    (2, 1, 4, 80, 150, [150, 149]), (2, 1, 3, 8, 50, [50, 3]), (1, 2, 2, 37, 41, [41]), (2, 1, 9, 656, 131, [131, 64]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_attention(cuda, dtype, shape):
    from kimi_k3_b200 import ops
    b, tq, h, width, slots, lengths = shape
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor(lengths, device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens, scale=0.7), q, codes, scales, lens, 0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_long_axis_is_split_and_joined(cuda, dtype):
    from kimi_k3_b200 import ops
    b, h, width, slots = 2, 5, 640, 40000
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, 1, h, width, dtype, cuda, spread=3.0)
    for lengths in ([40000, 0], [39999, 12345], [1, 64]):
        lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        out = ops.mla_cache_attention(q, codes, scales, lens)
        check_attention(out, q, codes, scales, lens, 1.0)
        assert torch.equal(out, ops.mla_cache_attention(q, codes, scales, lens))  # the joining order is fixed


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_attention_never_touches_masked_slots(cuda, dtype):
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = 3, 2, 6, 640, 200
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([130, 0, 64], device=cuda)
    want = ops.mla_cache_attention(q, codes, scales, lens)
    for i, n in enumerate(lens.tolist()):
        codes.view(torch.uint8)[i, n:] = 0x7F
        scales[i, n:] = math.nan if i else math.inf
    got = ops.mla_cache_attention(q, codes, scales, lens)
    assert torch.equal(got, want)
    assert torch.isfinite(got).all() and not got[1].any()
    # a NaN token reaches the rows that see it and no others
    scales[0, 129] = math.nan
    codes.view(torch.uint8)[0, 129] = 0
    got = ops.mla_cache_attention(q, codes, scales, lens)
    assert torch.isnan(got[0, 1]).all() and torch.equal(got[0, 0], want[0, 0]) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_query_start(cuda, dtype):
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = 4, 3, 4, 768, 100
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([100, 40, 70, 10], dtype=torch.int32, device=cuda)
    # inside the prefix; row 0 before the cache; past the length (every key is seen); no key at all
    start = torch.tensor([63, -1, 200, -3], device=cuda)
    out = ops.mla_cache_attention(q, codes, scales, lens, query_start=start, scale=0.5)
    check_attention(out, q, codes, scales, lens, 0.5, start)
    assert not out[1, 0].any() and not out[3].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_attention_extreme_values(cuda, dtype):
    """Token scales far apart, one dominating token, zero rows, zero and huge queries, a NaN query row."""
    from kimi_k3_b200 import ops
    b, h, width, slots = 2, 6, 640, 260
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(b, slots, width, generator=g, device=cuda)
    x[0] *= torch.exp2(torch.randint(-20, 6, (slots, 1), generator=g, device=cuda).float())
    x[1, 100] *= 2.0 ** 12  # a token a thousand times larger than the others
    x[1, 7:20] = 0.0
    codes, scales = (t.float() for t in quantise64(x))
    codes = codes.to(E4M3)
    q = torch.randn(b, 1, h, width, generator=g, device=cuda) * 0.05
    q[:, :, 1] = 0.0
    q[:, :, 2] *= 2.0 ** -14
    q[0, :, 3] *= 20.0
    q = q.to(dtype)
    lens = torch.tensor([260, 259], device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens, scale=0.3), q, codes, scales, lens, 0.3)
    bad = q.clone()
    bad[0, 0, 4, 5] = math.nan
    a, c = (ops.mla_cache_attention(v, codes, scales, lens, scale=0.3) for v in (q, bad))
    assert torch.isnan(c[0, 0, 4]).all()
    keep = torch.ones(b, 1, h, dtype=torch.bool, device=cuda)
    keep[0, 0, 4] = False
    assert torch.equal(a[keep], c[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_growing_maximum(cuda, dtype):
    """Scores that keep growing along the cache (every tile raises the running maximum), and falling ones."""
    from kimi_k3_b200 import ops
    width, slots, h = 640, 1000, 3
    g = torch.Generator(device=cuda).manual_seed(5)
    base = torch.randn(width, generator=g, device=cuda)
    ramp = torch.linspace(0.1, 30.0, slots, device=cuda)[:, None] * base / base.norm()
    x = torch.stack((ramp, ramp.flip(0))) + 0.02 * torch.randn(2, slots, width, generator=g, device=cuda)
    codes, scales = (t.float() for t in quantise64(x))
    codes = codes.to(E4M3)
    q = (base / base.norm() * torch.tensor([[1.0], [4.0], [0.2]], device=cuda)).expand(2, 1, h, width).to(dtype)
    lens = torch.tensor([slots, slots], device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens), q, codes, scales, lens, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_layouts(cuda, dtype):
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = 3, 2, 5, 640, 150
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([150, 20, 64], device=cuda)
    want = ops.mla_cache_attention(q, codes, scales, lens)
    check_attention(want, q, codes, scales, lens, 1.0)
    heads_first = q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)  # as a batched product leaves it
    strided = q.transpose(2, 3).contiguous().transpose(2, 3)
    shifted = torch.cat((q[..., :1], q), -1)[..., 1:]
    for v in (heads_first, strided, shifted):
        assert torch.equal(ops.mla_cache_attention(v, codes, scales, lens), want)
    swapped = codes.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E4M3)  # [slots, B, L]
    wide = torch.zeros(b, slots + 3, width + 16, dtype=torch.uint8, device=cuda)
    wide[:, 3:, 16:] = codes.view(torch.uint8)
    odd = torch.zeros(b, slots, width + 5, dtype=torch.uint8, device=cuda)
    odd[..., 5:] = codes.view(torch.uint8)
    for c in (swapped, wide[:, 3:, 16:].view(E4M3), odd[..., 5:].view(E4M3)):
        s = scales.transpose(0, 1).contiguous().transpose(0, 1)
        check_attention(ops.mla_cache_attention(q, c, s, lens), q, codes, scales, lens, 1.0)
    one = ops.mla_cache_attention(q[:1], codes[:1].expand(4, -1, -1)[:1], scales[:1], lens[:1])
    assert torch.equal(one, want[:1])
    # one prefix shared by every sequence (batch stride 0) is readable
    shared = ops.mla_cache_attention(q, codes[:1].expand(b, -1, -1), scales[:1].expand(b, -1), lens)
    check_attention(shared, q, codes[:1].expand(b, -1, -1), scales[:1].expand(b, -1), lens, 1.0)


def test_offsets_past_32_bits(cuda):
    from kimi_k3_b200 import ops
    b, slots, width, h = 3, 1_100_000, 1024, 4
    codes = torch.zeros(b, slots, width, dtype=torch.uint8, device=cuda).view(E4M3)
    scales = torch.zeros(b, slots, device=cuda)
    x = torch.randn(b, 70, width, device=cuda).bfloat16()
    ops.mla_cache_write(x, codes, scales, torch.zeros(b, dtype=torch.long, device=cuda))
    end = torch.full((b,), slots - 70, device=cuda)
    ops.mla_cache_write(x, codes, scales, end)
    qc, qs = quantise64(x)
    for at in (0, slots - 70):
        assert torch.equal(codes[:, at:at + 70].double(), qc) and torch.equal(scales[:, at:at + 70].double(), qs)
    q = queries(b, 1, h, width, torch.bfloat16, cuda)
    lens = torch.full((b,), 70, device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens), q, codes, scales, lens, 1.0)
    # the whole of it: the zero rows between the two ends take part in the softmax
    full = torch.full((b,), slots, device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, full), q, codes, scales, full, 1.0)
    tail = ops.mla_cache_read(codes, scales, dtype=torch.bfloat16)[:, slots - 70:]
    assert torch.equal(tail.double(), qc * qs[..., None])


def test_other_stream_and_graph(cuda):
    from kimi_k3_b200 import ops
    b, h, width, slots = 4, 10, 640, 500
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, 1, h, width, torch.bfloat16, cuda)
    lens = torch.tensor([500, 17, 0, 256], device=cuda)
    x = torch.randn(b, 1, width, device=cuda).bfloat16()
    want = ops.mla_cache_attention(q, codes, scales, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ops.mla_cache_attention(q, codes, scales, lens) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for o in outs:
        assert torch.equal(o, want)
    # a captured step reads its lengths and cache at replay time
    c2, s2, l2 = codes.view(torch.uint8).clone().view(E4M3), scales.clone(), lens.clone()
    with torch.cuda.stream(side):
        ops.mla_cache_write(x, c2, s2, l2)
        ops.mla_cache_attention(q, c2, s2, l2 + 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.mla_cache_write(x, c2, s2, l2)
        seen = l2 + 1
        out = ops.mla_cache_attention(q, c2, s2, seen)
    for n in ([499, 17, 0, 256], [3, 400, 100, 63]):
        c2.view(torch.uint8).copy_(codes.view(torch.uint8))
        s2.copy_(scales)
        l2.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(out, q, c2, s2, l2 + 1, 1.0)


def test_refusals(cuda):
    from kimi_k3_b200 import ops
    codes, scales = make_cache(2, 8, 64, cuda)
    x = torch.randn(2, 3, 64, device=cuda)
    q = torch.randn(2, 1, 3, 64, device=cuda)
    n = torch.tensor([1, 2], device=cuda)
    bad_write = [
        (x.double(), codes, scales, n), (x[:1], codes, scales, n), (x[..., :32], codes, scales, n), (x[0], codes, scales, n),
        (x.cpu(), codes, scales, n), (x, codes.view(torch.uint8), scales, n), (x, codes, scales.double(), n),
        (x, codes, scales[:, :4], n), (x, codes, scales, n.float()), (x, codes, scales, n[:1]), (x, codes, scales, n.cpu()),
        (x, codes[:1].expand(2, -1, -1), scales, n), (x, codes, scales, n, n.float()), (x, codes, scales, n, n[:1]),
    ]
    for args in bad_write:
        with pytest.raises(RuntimeError):
            ops.mla_cache_write(*args)
    for kw in (dict(dtype=torch.float64), dict(tokens=9), dict(tokens=-1)):
        with pytest.raises(RuntimeError):
            ops.mla_cache_read(codes, scales, n, **kw)
    with pytest.raises(RuntimeError):
        ops.mla_cache_read(codes, scales, n[:1])
    for args in [(q.double(), codes, scales, n), (q[:1], codes, scales, n), (q[..., :32], codes, scales, n),
                 (q[:, 0], codes, scales, n), (q.cpu(), codes, scales, n), (q, codes, scales[:, :4], n),
                 (q, codes, scales, n.float()), (q, codes, scales, n[:1])]:
        with pytest.raises(RuntimeError):
            ops.mla_cache_attention(*args)
    with pytest.raises(RuntimeError):
        ops.mla_cache_attention(q, codes, scales, n, query_start=n.float())
    wide_codes, wide_scales = make_cache(2, 4, 2064, cuda)
    with pytest.raises(RuntimeError, match="2048"):
        ops.mla_cache_attention(torch.randn(2, 1, 3, 2064, device=cuda), wide_codes, wide_scales, n)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.mla_cache_attention(q.requires_grad_(), codes, scales, n)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.mla_cache_write(x.requires_grad_(), codes, scales, n)
    # nothing to do is not an error
    empty = ops.mla_cache_attention(q.detach()[:, :0], codes, scales, n)
    assert empty.shape == (2, 0, 3, 64)
    ops.mla_cache_write(x.detach()[:, :0], codes, scales, n)
    assert not ops.mla_cache_attention(q.detach(), codes[:, :0], scales[:, :0], n).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [(1, 3), (2, 8), (3, 8), (4, 8), (1, 24), (4, 12), (5, 10), (6, 12)],
                         ids=lambda r: "x".join(map(str, r)))
@pytest.mark.parametrize("width", [128, 640, 768, 1536])
def test_attention_runs_of_tiles(cuda, width, rows, dtype):
    """Batches large enough that a CTA walks several tiles and crosses from one sequence into the next, at every
    number of query rows; lengths of every residue, empty sequences among them."""
    from kimi_k3_b200 import ops
    tq, h = rows
    b, slots = 24, 1500
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([(i * 397) % (slots + 1) if i % 5 else (0, 1, 64, 65, slots)[i // 5] for i in range(b)], device=cuda)
    out = ops.mla_cache_attention(q, codes, scales, lens, scale=0.6)
    check_attention(out, q, codes, scales, lens, 0.6)
    assert torch.equal(out, ops.mla_cache_attention(q, codes, scales, lens, scale=0.6))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [(32, 1, 12, 768, 128), (64, 1, 16, 1024, 256), (100, 1, 10, 640, 400),
                                  (320, 1, 3, 512, 250), (40, 5, 10, 640, 190)], ids=lambda c: "x".join(map(str, c)))
def test_attention_many_short_sequences(cuda, case, dtype):
    """Batches that fill the GPU with one sequence each, in one wave or several; empty sequences among them."""
    from kimi_k3_b200 import ops
    b, tq, h, width, slots = case
    codes, scales = make_cache(b, slots, width, cuda)
    q = queries(b, tq, h, width, dtype, cuda)
    lens = torch.tensor([(i * 89) % (slots + 1) if i % 4 else (0, 1, 64, 65, slots)[i // 4 % 5] for i in range(b)], device=cuda)
    check_attention(ops.mla_cache_attention(q, codes, scales, lens, scale=0.6), q, codes, scales, lens, 0.6)


# ------------------------------------------------------------------------------------------ through the model
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 4, 16, 21])
def test_layer_against_its_plain_form(cuda, tokens, dtype, monkeypatch):
    """A gated-MLA layer on a quantised cache: kernels against the PyTorch form of the same layer.  Both round to
    the layer's type at the same places but for the order of sums; a few roundings of the output's size apart."""
    from kimi_k3_b200.models.mla import GatedMLA, GatedMLAConfig, QuantizedMLACache
    torch.manual_seed(7)
    layer = GatedMLA(GatedMLAConfig(d_model=640, num_heads=10, q_head_dim=64, v_head_dim=64, kv_latent_dim=640)).to(cuda).eval()
    b, prompt, slots = 3, 70, 120
    x0 = torch.randn(b, prompt, 640, device=cuda)
    mask0 = torch.arange(prompt, device=cuda)[None, :] < torch.tensor([70, 33, 1], device=cuda)[:, None]
    x = torch.randn(b, tokens, 640, device=cuda)
    mask = torch.arange(tokens, device=cuda)[None, :] < torch.tensor([tokens, max(1, tokens // 2), 1], device=cuda)[:, None]
    outs = []
    for kernels in ("1", "0"):
        monkeypatch.setenv("KIMI_K3_KERNELS", kernels)
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
            pre = layer(x0, mask0, use_cache=True).cache
            if kernels == "1":
                first = QuantizedMLACache.from_cache(pre, slots)
                cache = first.clone()
            else:
                cache = first.clone()
            out = layer(x, None if tokens == 1 else mask, cache=cache, use_cache=True)
        outs.append(out.hidden_states.float())
        offsets = cache.sequence_offset.tolist()
    assert offsets == ([71, 34, 2] if tokens == 1 else [70 + tokens, 33 + max(1, tokens // 2), 2])
    err = (outs[0] - outs[1]).abs().max().item() / outs[1].abs().max().item()
    assert err <= (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -11), err


@pytest.mark.parametrize("limit", [0, 64])
def test_layer_attends_or_rebuilds(cuda, limit, monkeypatch):
    """The layer's two forms on a quantised cache, in the latent space and over rebuilt keys and values, at one length:
    each within a few roundings of the PyTorch form of the same layer in fp32."""
    from kimi_k3_b200.models import mla
    torch.manual_seed(8)
    layer = mla.GatedMLA(mla.GatedMLAConfig(d_model=640, num_heads=10, q_head_dim=64, v_head_dim=64,
                                            kv_latent_dim=640)).to(cuda).eval()
    b, prompt, tokens = 2, 90, 30
    x0, x = torch.randn(b, prompt, 640, device=cuda), torch.randn(b, tokens, 640, device=cuda)
    mask0 = torch.arange(prompt, device=cuda)[None, :] < torch.tensor([90, 41], device=cuda)[:, None]
    mask = torch.arange(tokens, device=cuda)[None, :] < torch.tensor([30, 11], device=cuda)[:, None]
    outs = []
    with torch.no_grad():
        first = mla.QuantizedMLACache.from_cache(layer(x0, mask0, use_cache=True).cache, 130)
        for kernels, n in (("1", limit), ("0", 0)):
            monkeypatch.setenv("KIMI_K3_KERNELS", kernels)
            monkeypatch.setattr(mla, "ABSORBED_QUERY_LIMIT", n)
            outs.append(layer(x, mask, cache=first.clone(), use_cache=True).hidden_states)
    err = (outs[0] - outs[1]).abs().max().item() / outs[1].abs().max().item()
    assert err <= 2.0 ** -11, err


def test_graph_decoder_on_a_quantised_cache(cuda):
    from kimi_k3_b200.infer import GenerationConfig, GraphDecoder
    from kimi_k3_b200.models.mla import QuantizedMLACache
    from test_decode_gpu import _small_model
    model = _small_model(cuda)
    ids = torch.randint(5, 1000, (4, 37), device=cuda)
    mask = torch.ones_like(ids, dtype=torch.bool)
    mask[2, 20:] = False
    for cfg in (GenerationConfig(max_new_tokens=12),
                GenerationConfig(max_new_tokens=12, do_sample=True, top_k=40, top_p=0.9, temperature=0.8,
                                 repetition_penalty=1.2, seed=11)):
        kw = dict(max_length=64, generation_config=cfg, cache_dtype=E4M3)
        dec = GraphDecoder(model, **kw)
        graph = dec.generate(ids, mask)
        eager = GraphDecoder(model, use_graph=False, **kw).generate(ids, mask)
        assert torch.equal(graph.generated_ids, eager.generated_ids)
        assert any(isinstance(lc.state, QuantizedMLACache) for lc in graph.cache.layer_caches)
        # a second prompt of the same shape refills the same buffers
        ids2 = torch.randint(5, 1000, (4, 37), device=cuda)
        captured = dec.graph
        again = dec.generate(ids2)
        assert dec.graph is captured
        assert torch.equal(again.generated_ids, GraphDecoder(model, **kw).generate(ids2).generated_ids)
