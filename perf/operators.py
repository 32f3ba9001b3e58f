"""Cases of the 8-bit MLA latent cache: writing it, reading it back and attending over it.

The cache of one gated-MLA layer holds, per sequence, up to ``slots`` latent rows as e4m3 codes with one
power-of-two scale per token (value = code * scale).  Three operators work on it: ``write`` quantises new
latents into their slots, ``read`` gives rows back in a 16- or 32-bit type, ``attend`` is the
weight-absorbed attention of one or a few query tokens per sequence over it.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
TOP = 448.0  # largest e4m3 value
LATENTS = (640, 768, 1024, 1536)  # latent widths of the model configurations, with 10, 12, 16 and 24 heads


def listed():
    return [
        # one decode step's append, gpu_80gb serving batch: latency
        {"name": "write step 64", "op": "write", "batch": 64, "tokens": 1, "slots": 4608, "latent": 1536,
         "dtype": "bf16", "ragged": False},
        # ragged prompts of the small model entering their slots behind earlier turns
        {"name": "write ragged prompts", "op": "write", "batch": 16, "tokens": 1024, "slots": 1537, "latent": 640,
         "dtype": "bf16", "ragged": True},
        # a whole serving batch's prompts
        {"name": "write long prompts", "op": "write", "batch": 64, "tokens": 4096, "slots": 4608, "latent": 1536,
         "dtype": "bf16", "ragged": False},
        # the conversation so far, ragged, for a prompt that continues it
        {"name": "read turns", "op": "read", "batch": 4, "tokens": 2048, "slots": 2048, "latent": 768,
         "dtype": "f16", "ragged": True},
        # a whole serving batch's cache
        {"name": "read full cache", "op": "read", "batch": 64, "tokens": 4608, "slots": 4608, "latent": 1536,
         "dtype": "bf16", "ragged": False},
        # one short chat, one token: latency
        {"name": "attend one short", "op": "attend", "batch": 1, "tokens": 257, "slots": 512, "latent": 640,
         "heads": 10, "queries": 1, "dtype": "bf16", "ragged": False},
        # the small model's decode benchmark batch, all types' plain-precision form
        {"name": "attend f32", "op": "attend", "batch": 4, "tokens": 1000, "slots": 1024, "latent": 640,
         "heads": 10, "queries": 1, "dtype": "f32", "ragged": True},
        # drafted tokens checked in one pass, ragged lengths
        {"name": "attend drafts", "op": "attend", "batch": 8, "tokens": 2048, "slots": 2304, "latent": 768,
         "heads": 12, "queries": 4, "dtype": "bf16", "ragged": True},
        # one long document: the long axis has to be split
        {"name": "attend one long", "op": "attend", "batch": 1, "tokens": 131072, "slots": 131072, "latent": 1024,
         "heads": 16, "queries": 1, "dtype": "f16", "ragged": False},
        # gpu_80gb serving step with the heads split over eight ranks
        {"name": "attend 3 heads", "op": "attend", "batch": 64, "tokens": 4608, "slots": 4608, "latent": 1536,
         "heads": 3, "queries": 1, "dtype": "bf16", "ragged": False},
        # the same step, ragged, half the heads
        {"name": "attend 12 heads ragged", "op": "attend", "batch": 64, "tokens": 4608, "slots": 4608,
         "latent": 1536, "heads": 12, "queries": 1, "dtype": "bf16", "ragged": True},
        # the same step with every head on one GPU
        {"name": "attend 24 heads", "op": "attend", "batch": 64, "tokens": 4608, "slots": 4608, "latent": 1536,
         "heads": 24, "queries": 1, "dtype": "bf16", "ragged": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "attend"))
    latent = rng.choice(LATENTS) if rng.random() < 0.75 else 16 * rng.randint(4, 96)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    batch = _log_int(rng, 1, 64)
    most = 64 * 4608 * 1536 // (batch * latent)
    if op == "write" and rng.random() < 0.4:
        tokens, slots = 1, _log_int(rng, 64, max(65, min(131072, most)))
    else:
        tokens = _log_int(rng, 16, max(17, min(131072 if batch == 1 else 8192, most)))
        slots = tokens + rng.randint(0, tokens // 8 + 1)
    if op != "attend" and dtype == "f32":
        tokens = max(1, tokens // 2)
    case = {"op": op, "batch": batch, "tokens": tokens, "slots": slots, "latent": latent, "dtype": dtype,
            "ragged": rng.random() < 0.6}
    if op == "attend":
        case["heads"] = rng.choice((3, 6, 10, 12, 16, 24)) if rng.random() < 0.75 else rng.randint(1, 24)
        case["queries"] = 1 if rng.random() < 0.6 else rng.randint(2, 8)
        # no dearer than the largest listed case
        cost = 64 * 4608 * 1536 * 24 // (1 if dtype != "f32" else 64)
        per_token = batch * latent * case["heads"] * case["queries"]
        case["tokens"] = max(1, min(tokens, cost // per_token))
        case["slots"] = case["tokens"] + slots - tokens
    return case


def _counts(case):
    """Valid tokens of each sequence: a fixed spread over 0 .. tokens (the first has them all, and with more
    than four sequences the last has none)."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * b
    counts = [max(1, int(t * ((i * 0.6180339887498949 + 0.999999) % 1.0))) for i in range(b)]
    counts[0] = t
    if b > 4:
        counts[-1] = 0
    return counts


def _latents(shape, gen):
    """Latents of a trained compression: channels and tokens of different size."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device="cuda"))
    x *= torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return x


def _quantise(x):
    """codes, scales of f32 rows: the least power of two under which the row fits e4m3."""
    top = x.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(top)
    k = exponent - torch.where(mantissa <= 0.875, 9, 8)
    k = torch.where(top == 0, -126, k).clamp(min=-126)
    scales = torch.ldexp(torch.ones_like(top), k)
    bad = ~torch.isfinite(top)
    codes = torch.where(bad[..., None], 0.0, x / scales[..., None]).to(torch.float8_e4m3fn)
    return codes, torch.where(bad, math.nan, scales)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, t, slots, width, dtype = case["batch"], case["tokens"], case["slots"], case["latent"], DTYPES[case["dtype"]]
    counts = torch.tensor(_counts(case), dtype=torch.long, device="cuda")
    state = dict(case, counts=counts)
    if case["op"] == "write":
        state["x"] = _latents((b, t, width), gen).to(dtype)
        state["codes"] = torch.zeros(b, slots, width, dtype=torch.float8_e4m3fn, device="cuda")
        state["scales"] = torch.zeros(b, slots, device="cuda")
        room = slots - t
        state["offsets"] = (torch.rand(b, generator=gen, device="cuda") * (room + 1)).long().clamp(max=room)
        return state
    # the rows past a sequence's length hold what an earlier sequence left there
    state["codes"], state["scales"] = _quantise(_latents((b, slots, width), gen))
    if case["op"] == "attend":
        # queries absorbed into the latent space; scores of a softmax with some contrast
        q = torch.randn(b, case["queries"], case["heads"], width, generator=gen, device="cuda")
        state["q"] = (q * (10.0 / math.sqrt(width))).to(dtype)
        state["scale"] = 0.125  # head width 64
    return state


def run(state):
    op, codes, scales, counts = state["op"], state["codes"], state["scales"], state["counts"]
    if own:
        from kimi_k3_b200 import ops
        if op == "write":
            ops.mla_cache_write(state["x"], codes, scales, state["offsets"], counts)
            return {"codes": codes, "scales": scales}
        if op == "read":
            return ops.mla_cache_read(codes, scales, counts, dtype=DTYPES[state["dtype"]], tokens=state["tokens"])
        return ops.mla_cache_attention(state["q"], codes, scales, counts, scale=state["scale"])
    device = codes.device
    if op == "write":
        x = state["x"]
        new_codes, new_scales = _quantise(x.float())
        step = torch.arange(x.shape[1], device=device)
        slot = state["offsets"][:, None] + step
        keep = (step < counts[:, None]) & (slot < codes.shape[1])
        row, col = keep.nonzero(as_tuple=True)
        codes.view(torch.uint8)[row, slot[row, col]] = new_codes.view(torch.uint8)[row, col]
        scales[row, slot[row, col]] = new_scales[row, col]
        return {"codes": codes, "scales": scales}
    if op == "read":
        t = state["tokens"]
        valid = torch.arange(t, device=device) < counts[:, None]
        values = codes[:, :t].float() * scales[:, :t, None]
        return torch.where(valid[..., None], values, 0.0).to(DTYPES[state["dtype"]])
    q = state["q"].float()
    b, nq, heads, width = q.shape
    slots = codes.shape[1]
    key = torch.arange(slots, device=device)
    valid = key < counts[:, None]
    values = torch.where(valid[..., None], codes.float() * scales[..., None], 0.0)
    scores = torch.bmm(q.reshape(b, nq * heads, width), values.transpose(1, 2)) * state["scale"]
    last = counts[:, None] - nq + torch.arange(nq, device=device)  # the last key a query token sees
    seen = (valid[:, None, :] & (key <= last[..., None])).repeat_interleave(heads, dim=1)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    return torch.bmm(p, values).reshape(b, nq, heads, width).to(DTYPES[state["dtype"]])


def work(case):
    counts, width, size = _counts(case), case["latent"], BYTES[case["dtype"]]
    total = sum(counts)
    if case["op"] == "write":
        return {"bytes": total * (width * size + width + 4), "flops": 2 * total * width}
    if case["op"] == "read":
        return {"bytes": total * (width + 4) + case["batch"] * case["tokens"] * width * size, "flops": total * width}
    rows = case["queries"] * case["heads"]
    pairs = sum(max(0, c - case["queries"] + 1 + i) for c in counts for i in range(case["queries"]))
    return {"bytes": total * (width + 4) + 2 * case["batch"] * rows * width * size,
            "flops": 4 * case["heads"] * width * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    codes, scales, counts = state["codes"], state["scales"], state["counts"].tolist()
    if case["op"] == "write":
        codes, scales = codes.double(), scales.double()
        for i, n in enumerate(counts):
            n = min(n, case["slots"] - int(state["offsets"][i]))
            if n <= 0:
                continue
            x = state["x"][i, :n].double()
            # ceil(log2(top / 448)), settled by comparison so that a rounded logarithm does not matter
            top = x.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -200)
            k = torch.ceil(torch.log2(top / TOP))
            k = torch.where(torch.exp2(k - 1) * TOP >= top, k - 1, k)
            k = torch.where(torch.exp2(k) * TOP < top, k + 1, k).clamp(min=-126)
            v = x * torch.exp2(-k)
            # e4m3: three bits after the leading one down to 2^-6, steps of 2^-9 below
            e = torch.frexp(v)[1].double() - 1
            ulp = torch.exp2(e.clamp(min=-6) - 3)
            at = int(state["offsets"][i])
            codes[i, at:at + n] = torch.round(v / ulp) * ulp
            scales[i, at:at + n] = torch.exp2(k[:, 0])
        return {"codes": codes, "scales": scales}
    if case["op"] == "read":
        out = codes[:, :case["tokens"]].double() * scales[:, :case["tokens"], None].double()
        for i, n in enumerate(counts):
            out[i, n:] = 0
        return out
    nq = case["queries"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(counts):
        values = codes[i, :n].double() * scales[i, :n, None].double()
        for j in range(nq):
            m = n - nq + 1 + j  # keys that query token j sees
            if m > 0:
                p = torch.softmax(state["q"][i, j].double() @ values[:m].T * state["scale"], dim=-1)
                out[i, j] = p @ values[:m]
    return out
