"""The serving and training operators around the attention kernels, as they are measured.

Four operators: rotary positions (forward and backward), appending keys and values to a paged cache
(16-bit or 4-bit, with the rotation applied on the way), reading the cache back into contiguous keys
and values, and attention of a few new tokens over the cache.  `run` computes each in elementary torch
operations in 32 bits, or, where `own` is true, through flash_attn_volta_b200.

The cache.  A page holds `page` consecutive tokens of one sequence; page_table[b, i] is the page of
tokens i*page .. (i+1)*page - 1 of sequence b.  16-bit pages are two tensors (pages, kv heads, page,
head_dim).  4-bit pages are one uint8 tensor (pages, kv heads, page/16, block bytes); a block holds 16
tokens of one head:
  K codes   16 tokens x D/2 bytes, a token's bytes ordered (t 4, group D/32, hi 2, j 2): byte holds the
            codes of dims 32*group + 8*t + 4*j + hi (low nibble) and the same + 2 (high nibble)
  K params  16 tokens x D/32 groups x (scale, minimum) in fp16
  V codes   ordered (tp 2, g 8, t 4, group D/32, hi 2, bb 2): byte holds the codes of token
            8*tp + 2*t + hi, dims 32*group + 4*g + 2*bb (low nibble) and the same + 1 (high nibble)
  V params  (scale, minimum) x D/32 groups x (t 4, tp 2, hi 2) tokens in fp16
A group is 32 consecutive dims of one token and head: minimum = fp16 below the smallest value, scale =
fp16 above (largest - minimum) / 15, code = round((x - minimum) / scale), value = minimum + scale * code.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ------------------------------------------------------------------ cases
def _rotary(name, dtype, B, S, H, Hkv, D, R, interleaved, factor, first, train):
    return {"name": name, "op": "rotary", "dtype": dtype, "B": B, "S": S, "H": H, "Hkv": Hkv, "D": D,
            "R": R, "interleaved": interleaved, "factor": factor, "first": first, "train": train}


def _append(name, bits, dtype, B, S, H, Hkv, D, R, interleaved, page, lo, hi, read):
    return {"name": name, "op": "append", "bits": bits, "dtype": dtype, "B": B, "S": S, "H": H,
            "Hkv": Hkv, "D": D, "R": R, "interleaved": interleaved, "page": page, "lo": lo, "hi": hi,
            "read": read}


def _read(name, bits, dtype, B, Hkv, D, page, lo, hi):
    return {"name": name, "op": "read", "bits": bits, "dtype": dtype, "B": B, "Hkv": Hkv, "D": D,
            "page": page, "lo": lo, "hi": hi}


def _decode(name, bits, dtype, B, S, H, Hkv, D, page, lo, hi):
    return {"name": name, "op": "decode", "bits": bits, "dtype": dtype, "B": B, "S": S, "H": H,
            "Hkv": Hkv, "D": D, "page": page, "lo": lo, "hi": hi}


def listed():
    return [
        # one token of each of 48 sequences, at scattered far positions: the smallest rotation
        _rotary("rotary-step", "bf16", 48, 1, 32, 8, 128, 128, False, 1.0, 30000, False),
        # the attention layer of a training step, forward and backward (8 x 2048, 16 heads of 128)
        _rotary("rotary-train", "fp16", 8, 2048, 16, 16, 128, 128, False, 1.0, 0, True),
        # one long odd sequence, half of each head in interleaved pairs, positions interpolated
        _rotary("rotary-long-part", "bf16", 1, 40009, 24, 8, 64, 32, True, 8.0, 0, True),
        # a serving step's new tokens, 16-bit cache
        _append("append16-step", 16, "bf16", 64, 1, 32, 8, 128, 128, False, 64, 1, 8191, False),
        # prompts of different lengths written into a fresh 16-bit cache
        _append("append16-prompt", 16, "fp16", 6, 4096, 16, 16, 64, 64, False, 32, 0, 0, False),
        # a chunk of prompt appended to a 4-bit cache, then the whole context read back for the
        # chunk's attention
        _append("append4-chunk-read", 4, "bf16", 4, 1024, 32, 8, 128, 128, False, 64, 2000, 7000, True),
        # contexts of a 4-bit cache read back, ragged
        _read("read4-ragged", 4, "fp16", 12, 8, 64, 16, 33, 6001),
        # one sequence's single token, short context: latency counts
        _decode("decode16-one", 16, "fp16", 1, 1, 16, 16, 64, 64, 777, 777),
        # a batch of single tokens over ragged contexts, grouped heads, 16-bit
        _decode("decode16-batch", 16, "bf16", 64, 1, 32, 8, 128, 64, 5, 8192),
        # the same kind of batch over a 4-bit cache
        _decode("decode4-batch", 4, "bf16", 96, 1, 32, 8, 128, 64, 5, 8192),
        # two very long contexts, 4-bit: the work is split over the context
        _decode("decode4-long", 4, "fp16", 2, 1, 32, 8, 128, 128, 100003, 131072),
        # five drafted tokens per sequence checked at once, causal among themselves, odd lengths
        _decode("decode4-draft", 4, "bf16", 24, 5, 32, 8, 64, 32, 301, 4099),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _draw(rng):
    op = rng.choice(["rotary", "append", "read", "decode", "decode"])
    dtype = rng.choice(["fp16", "bf16"])
    D = rng.choice([32, 64, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    H = Hkv * rng.choice([1, 2, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    bits = rng.choice([4, 16])
    R = rng.choice([D, D, D // 2, D // 4])
    inter = rng.choice([False, True])
    if op == "rotary":
        train = rng.choice([False, True])
        D = rng.choice([16, 32, 64, 80, 96, 128])
        R = rng.choice([D, D, D // 2, D // 4])
        B = _log(rng, 1, 32)
        S = _log(rng, 1, 16384)
        c = _rotary("", dtype, B, S, H, Hkv, D, R, inter, rng.choice([1.0, 4.0, 32.0]),
                    _log(rng, 1, 500000), train)
    elif op == "append":
        lo, more = rng.choice([(0, 0), (_log(rng, 1, 2000), _log(rng, 1, 4000))])
        c = _append("", bits, dtype, _log(rng, 1, 64), _log(rng, 1, 4096), H, Hkv, D, R, inter, page,
                    lo, lo + more, rng.choice([False, True]) or bits == 4)
    elif op == "read":
        lo = _log(rng, 1, 2000) - 1
        c = _read("", bits, dtype, _log(rng, 1, 64), Hkv, D, page, lo, lo + _log(rng, 1, 8000))
    else:
        lo = _log(rng, 1, 30000) - 1
        c = _decode("", bits, dtype, _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 4, 7]), H, Hkv, D, page,
                    lo, lo + _log(rng, 1, 30000))
    del c["name"]
    return c


def _cost(c):
    """Values that the plain form of a case touches (drawn cases stay below the largest listed one)."""
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if c["op"] == "rotary":
        return 4 * B * c["S"] * (c["H"] + Hkv) * D
    if c["op"] == "append":
        return 2 * B * (c["S"] * c["H"] + (c["hi"] + c["S"]) * Hkv * 2) * D
    if c["op"] == "read":
        return 2 * B * c["hi"] * Hkv * D
    return B * c["hi"] * (Hkv * D * 2 + c["H"] * c["S"])


def _spread(c, n):
    """n whole numbers from lo to hi, evenly spaced: the lengths of a case's sequences."""
    lo, hi = c["lo"], c["hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _counts(c):
    """New tokens of each sequence in an append: all of them have S, but for prompts into an empty cache,
    which are of different lengths."""
    S, B = c["S"], c["B"]
    return [S if c["hi"] > 0 else max(1, S - (S // (B + 1)) * i) for i in range(B)]


def work(case):
    c = case
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    token = 2 * D * 2 if c.get("bits", 16) == 16 else D + 8 * (D // 32)  # bytes of a cached token and head
    if c["op"] == "rotary":
        n = B * c["S"] * (c["H"] + Hkv)
        passes = 2 if c["train"] else 1
        return {"bytes": passes * n * D * 2 * 2, "flops": passes * n * c["R"] * 3}
    if c["op"] == "append":
        new = sum(_counts(c))
        n = {"bytes": new * (c["H"] * D * 2 * 2 + Hkv * (2 * D * 2 + token)),
             "flops": new * ((c["H"] + Hkv) * c["R"] * 3 + (0 if c["bits"] == 16 else Hkv * D * 2 * 5))}
        if c["read"]:
            total = sum(_spread(c, B)) + new
            n["bytes"] += total * Hkv * token + B * (c["hi"] + c["S"]) * Hkv * 2 * D * 2
            n["flops"] += total * Hkv * 2 * D * 2
        return n
    if c["op"] == "read":
        total = sum(_spread(c, B))
        return {"bytes": total * Hkv * token + B * c["hi"] * Hkv * 2 * D * 2, "flops": total * Hkv * 2 * D * 2}
    total = sum(_spread(c, B))
    return {"bytes": total * Hkv * token + 2 * B * c["S"] * c["H"] * D * 2,
            "flops": 4 * total * c["S"] * c["H"] * D}


# ------------------------------------------------------------------ inputs
def _pages(c, total, gen):
    """A page table (B, pages of the longest sequence) over a shuffled pool with a few pages to spare."""
    per = [(n + c["page"] - 1) // c["page"] for n in total]
    pool = sum(per) + 3
    order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32)
    width = max(per)
    table = torch.zeros((c["B"], width), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _keys(shape, gen):
    """Keys and values as a model has them: some channels of a head are shifted and larger than others."""
    D = shape[-1]
    shift = torch.randn(D, generator=gen, device=DEVICE)
    size = 0.5 + torch.rand(D, generator=gen, device=DEVICE)
    return torch.randn(shape, generator=gen, device=DEVICE).mul_(size).add_(shift)


def _frequencies(R, factor):
    i = torch.arange(R // 2, dtype=torch.float64, device=DEVICE)
    return 10000.0 ** (-2.0 * i / R) / factor


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    t = TYPES[c["dtype"]]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    s = {"case": c, "scale": 1.0 / math.sqrt(D)}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    if c["op"] == "rotary":
        s["q"] = torch.randn((B, c["S"], c["H"], D), generator=gen, device=DEVICE).to(t)
        s["k"] = _keys((B, c["S"], Hkv, D), gen).to(t)
        start = torch.randint(0, c["first"] + 1, (B, 1), generator=gen, device=DEVICE)
        s["positions"] = (start + torch.arange(c["S"], device=DEVICE)).to(torch.int32)
        s["inv_freq"] = _frequencies(c["R"], c["factor"])
        if c["train"]:
            s["dq"] = torch.randn((B, c["S"], c["H"], D), generator=gen, device=DEVICE).to(t)
            s["dk"] = torch.randn((B, c["S"], Hkv, D), generator=gen, device=DEVICE).to(t)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    mix = torch.randperm(B, generator=gen, device=DEVICE).tolist()
    if c["op"] == "append":
        starts = [_spread(c, B)[i] for i in mix]
        counts = [_counts(c)[i] for i in mix]
        total = [a + n for a, n in zip(starts, counts)]
        s["starts"], s["counts"] = ints(starts), ints(counts)
        s["q"] = torch.randn((B, c["S"], c["H"], D), generator=gen, device=DEVICE).to(t)
        s["k"] = _keys((B, c["S"], Hkv, D), gen).to(t)
        s["v"] = _keys((B, c["S"], Hkv, D), gen).to(t)
        s["inv_freq"] = _frequencies(c["R"], 1.0)
        s["max_len"] = c["hi"] + c["S"]
    else:
        total = [_spread(c, B)[i] for i in mix]
        s["max_len"] = c["hi"]
    s["lengths"] = ints(total)
    s["table"], pool = _pages(c, total, gen)
    shape = (pool, Hkv, c["page"], D)
    if c["bits"] == 16:
        s["k_pages"], s["v_pages"] = _keys(shape, gen).to(t), _keys(shape, gen).to(t)
    else:
        s["blocks"] = _blocks_of(_keys(shape, gen), _keys(shape, gen))
    if c["op"] == "decode":
        s["q"] = 1.5 * torch.randn((B, c["S"], c["H"], D), generator=gen, device=DEVICE)
        s["q"] = s["q"].to(t)
    return s


# ------------------------------------------------------------------ plain forms
def _cos_sin(positions, inv_freq):
    angle = positions.double()[..., None] * inv_freq  # 64 bits: a far position's angle is large
    return torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]


def _rotate(x, cos, sin, interleaved):
    """x (B, S, heads, D) in fp32, cos and sin (B, S, 1, R/2): pairs (i, i + R/2), or (2i, 2i + 1)."""
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([rot, rest], dim=-1)


def _half_toward(x, up):
    """fp32 -> fp16, rounded down, or up."""
    h = x.half()
    wrong = h.float() < x if up else h.float() > x
    bits = h.view(torch.int16).int()
    away = bits >= 0 if up else bits < 0  # the next value away from zero has the next bit pattern
    zero = (bits & 0x7FFF) == 0
    step = torch.where(away, bits + 1, bits - 1)
    step = torch.where(zero, torch.full_like(bits, 1 if up else -32767), step)
    return torch.where(wrong, step, bits).to(torch.int16).view(torch.float16)


def _quantise(x):
    """(..., D) fp32 -> codes (..., D/32, 32) int32, scale and minimum (..., D/32) fp16."""
    g = x.clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    low = _half_toward(g.amin(-1), up=False)
    scale = _half_toward((g.amax(-1) - low.float()) / g.new_full((), 15.0), up=True)  # by a tensor: divides
    code = torch.round((g - low.float()[..., None]) / scale.float()[..., None])
    code = torch.nan_to_num(code, nan=0.0).clamp(0, 15).to(torch.int32)
    return code, scale, low


def _k_bytes(code):
    """(..., groups, 32) codes of a token -> (..., t, group, hi, j) bytes."""
    c = code.unflatten(-1, (4, 2, 2, 2))  # t, j, nibble, hi
    n = c.dim()
    c = c.permute(*range(n - 5), n - 4, n - 5, n - 1, n - 3, n - 2)
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)


def _v_bytes(code):
    """(..., groups, 32) codes of a token -> (..., g, group, bb) bytes."""
    c = code.unflatten(-1, (8, 2, 2)).transpose(-4, -3)  # group, g, bb, nibble -> g, group, bb, nibble
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)


def _parts(blocks, D):
    """Views of a 4-bit cache's K codes, K params, V codes and V params."""
    NG = D // 32
    cut = [0, 8 * D, 8 * D + 64 * NG, 16 * D + 64 * NG, 16 * D + 128 * NG]
    kc, kp, vc, vp = (blocks[..., a:b] for a, b in zip(cut[:-1], cut[1:]))
    kc = kc.unflatten(-1, (16, 4, NG, 2, 2))  # token, t, group, hi, j
    kp = kp.view(torch.float16).unflatten(-1, (16, NG, 2))  # token, group, (scale, minimum)
    vc = vc.unflatten(-1, (2, 8, 4, NG, 2, 2))  # tp, g, t, group, hi, bb
    vp = vp.view(torch.float16).unflatten(-1, (2, NG, 4, 2, 2))  # (scale, minimum), group, t, tp, hi
    return kc, kp, vc, vp


def _put(blocks, D, page, heads, token, k, v):
    """Writes tokens (n, D) k and v to (page, heads, token) of a 4-bit cache."""
    kc, kp, vc, vp = _parts(blocks, D)
    blk, r = token // 16, token % 16
    tp, t, hi = r // 8, r % 8 // 2, r % 2
    code, scale, low = _quantise(k)
    kc[page, heads, blk, r] = _k_bytes(code)
    kp[page, heads, blk, r] = torch.stack([scale, low], dim=-1)
    code, scale, low = _quantise(v)
    vc[page, heads, blk, tp, :, t, :, hi] = _v_bytes(code)
    vp[page, heads, blk, :, :, t, tp, hi] = torch.stack([scale, low], dim=-2)


def _blocks_of(k, v):
    """A 4-bit cache that holds (pages, heads, page, D) k and v."""
    P, Hkv, page, D = k.shape
    blocks = torch.empty((P, Hkv, page // 16, 16 * D + 4 * D), dtype=torch.uint8, device=k.device)
    kc, kp, vc, vp = _parts(blocks, D)
    code, scale, low = _quantise(k)
    kc.copy_(_k_bytes(code).unflatten(2, (-1, 16)))
    kp.copy_(torch.stack([scale, low], dim=-1).unflatten(2, (-1, 16)))
    code, scale, low = _quantise(v)
    b = _v_bytes(code).unflatten(2, (-1, 2, 4, 2))  # P, Hkv, blk, tp, t, hi, g, group, bb
    vc.copy_(b.permute(0, 1, 2, 3, 6, 4, 7, 5, 8))
    p = torch.stack([scale, low], dim=-2).unflatten(2, (-1, 2, 4, 2))  # P, Hkv, blk, tp, t, hi, 2, group
    vp.copy_(p.permute(0, 1, 2, 6, 7, 4, 3, 5))
    return blocks


def _values_of(blocks, D):
    """(..., Hkv, page/16, bytes) -> K and V (..., Hkv, page, D) in fp32: the values the codes stand for."""
    kc, kp, vc, vp = _parts(blocks, D)
    n = kc.dim()
    c = torch.stack([kc & 15, kc >> 4], dim=-1)  # token, t, group, hi, j, nibble
    c = c.permute(*range(n - 5), n - 5, n - 3, n - 4, n - 1, n, n - 2).flatten(-4)  # token, group, 32
    p = kp.float()
    k = p[..., 1:] + p[..., :1] * c.float()
    n = vc.dim()
    c = torch.stack([vc & 15, vc >> 4], dim=-1)  # tp, g, t, group, hi, bb, nibble
    c = c.permute(*range(n - 6), n - 6, n - 4, n - 2, n - 3, n - 5, n - 1, n).flatten(-3)
    c = c.flatten(-5, -3)  # (tp, t, hi), group, 32
    n = vp.dim()
    p = vp.float().permute(*range(n - 5), n - 2, n - 3, n - 1, n - 4, n - 5).flatten(-5, -3)
    v = p[..., 1:] + p[..., :1] * c.float()
    return k.flatten(-2).flatten(-3, -2), v.flatten(-2).flatten(-3, -2)


def _context(s):
    """K and V (B, Hkv, tokens, D) in fp32 of the sequences' pages, up to max_len, zero behind each length."""
    c = s["case"]
    table = s["table"].long()
    if c["bits"] == 16:
        k, v = s["k_pages"][table].float(), s["v_pages"][table].float()
    else:
        k, v = _values_of(s["blocks"][table], c["D"])
    k, v = (x.transpose(1, 2).flatten(2, 3)[:, :, :s["max_len"]] for x in (k, v))
    there = torch.arange(k.shape[2], device=k.device) < s["lengths"][:, None]
    there = there[:, None, :, None]
    return torch.where(there, k, 0.0), torch.where(there, v, 0.0)


def _plain_rotary(s, x, inverse):
    cos, sin = _cos_sin(s["positions"], s["inv_freq"])
    return _rotate(x.detach().float(), cos, -sin if inverse else sin, s["case"]["interleaved"]).to(x.dtype)


def _plain_append(s):
    c = s["case"]
    t = TYPES[c["dtype"]]
    B, S, D = c["B"], c["S"], c["D"]
    at = s["starts"][:, None] + torch.arange(S, device=DEVICE)
    cos, sin = _cos_sin(at, s["inv_freq"])
    q = _rotate(s["q"].float(), cos, sin, c["interleaved"]).to(t)
    k = _rotate(s["k"].float(), cos, sin, c["interleaved"])
    new = torch.arange(S, device=DEVICE) < s["counts"][:, None]
    b = torch.arange(B, device=DEVICE)[:, None].expand(B, S)[new]
    pos = at[new].long()
    page = s["table"][b, pos // c["page"]].long()[:, None]
    token = (pos % c["page"])[:, None]
    heads = torch.arange(c["Hkv"], device=DEVICE)[None]
    if c["bits"] == 16:
        s["k_pages"][page, heads, token] = k[new].to(t)
        s["v_pages"][page, heads, token] = s["v"][new]
    else:
        _put(s["blocks"], D, page, heads, token, k[new], s["v"][new].float())
    return q


def _plain_read(s):
    t = TYPES[s["case"]["dtype"]]
    k, v = _context(s)
    return k.transpose(1, 2).to(t, memory_format=torch.contiguous_format), \
        v.transpose(1, 2).to(t, memory_format=torch.contiguous_format)


def _plain_decode(s):
    c = s["case"]
    B, S, H, Hkv, D = c["B"], c["S"], c["H"], c["Hkv"], c["D"]
    k, v = _context(s)
    q = s["q"].float().unflatten(2, (Hkv, H // Hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    score = (q @ k.transpose(-1, -2)) * s["scale"]  # (B, Hkv, S * group, tokens)
    seen = s["lengths"][:, None] - S + 1 + torch.arange(S, device=DEVICE)  # (B, S): keys that a query sees
    seen = seen[:, None, :, None].expand(B, 1, S, H // Hkv).flatten(2, 3)
    hidden = torch.arange(k.shape[2], device=DEVICE) >= seen[..., None]
    score = score.masked_fill(hidden, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    return o.unflatten(2, (S, H // Hkv)).permute(0, 2, 1, 3, 4).reshape(B, S, H, D).to(s["q"].dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    return (_run_own if own else _run_plain)(s)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        out = [_plain_rotary(s, s["q"], False), _plain_rotary(s, s["k"], False)]
        if c["train"]:
            out += [_plain_rotary(s, s["dq"], True), _plain_rotary(s, s["dk"], True)]
        return out
    if c["op"] == "append":
        q = _plain_append(s)
        if c["read"]:
            return [q, *_plain_read(s)]
        return [q, s["k_pages"], s["v_pages"]]
    if c["op"] == "read":
        return _plain_read(s)
    return _plain_decode(s)


def _run_own(s):
    from flash_attn_volta_b200.kv_cache import PagedKVCache, flash_attn_decode, kv_cache_append, kv_cache_read
    from flash_attn_volta_b200.rotary import Rotary, rotary_embed_qk

    c = s["case"]
    if c["op"] == "rotary":
        q, k = rotary_embed_qk(s["q"], s["k"], Rotary(s["inv_freq"], c["interleaved"]), s["positions"])
        if c["train"]:
            return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
        return [q, k]
    if c["bits"] == 16:
        cache = PagedKVCache(s["k_pages"], s["v_pages"])
    else:
        cache = PagedKVCache.of_blocks(s["blocks"], c["D"], TYPES[c["dtype"]])
    if c["op"] == "append":
        q = kv_cache_append(cache, s["k"], s["v"], s["table"], s["starts"], s["counts"], q=s["q"],
                            rotary=Rotary(s["inv_freq"], c["interleaved"]))
        if c["read"]:
            return [q, *kv_cache_read(cache, s["table"], s["lengths"], s["max_len"])]
        return [q, s["k_pages"], s["v_pages"]]
    if c["op"] == "read":
        return kv_cache_read(cache, s["table"], s["lengths"], s["max_len"])
    return flash_attn_decode(s["q"], cache, s["table"], s["lengths"])


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _turned(x, positions, inv_freq, interleaved, sign=1.0):
    """x (B, S, heads, D) as complex pairs, each times exp(i * sign * position * frequency)."""
    x = x.detach().double()
    R = 2 * inv_freq.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       sign * positions.double()[:, :, None, None] * inv_freq)
    y = x.clone()
    first = slice(0, R, 2) if interleaved else slice(0, R // 2)
    second = slice(1, R, 2) if interleaved else slice(R // 2, R)
    z = torch.complex(x[..., first], x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _four_bits(x):
    """The values that 4-bit groups stand for, with the fp16 minimum and scale on the outer side."""
    y = torch.empty_like(x)
    for d in range(0, x.shape[-1], 32):
        g = x[..., d:d + 32]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        m = low.half()
        m = torch.where(m.double() > low, torch.nextafter(m.cpu(), torch.tensor(-math.inf).half()).to(m.device), m).double()
        step = (high - m) / g.new_full((), 15.0)  # a plain 15 would be multiplied by its inverse
        s = step.half()
        s = torch.where(s.double() < step, torch.nextafter(s.cpu(), torch.tensor(math.inf).half()).to(s.device), s).double()
        y[..., d:d + 32] = m + s * torch.where(s > 0, torch.round((g - m) / s), 0.0)
    return y


def _cached(s, b, n):
    """K and V (n, Hkv, D) in 64 bits of the first n cached tokens of sequence b, token by page and place."""
    c = s["case"]
    page, D, NG = c["page"], c["D"], c["D"] // 32
    j = torch.arange(n, device=DEVICE)
    pages, place = s["table"][b].long()[j // page], j % page
    if c["bits"] == 16:
        return s["k_pages"][pages, :, place].double(), s["v_pages"][pages, :, place].double()
    raw = s["blocks"][pages, :, place // 16]  # (n, Hkv, bytes): the token's block
    r = (place % 16)[:, None]
    d = torch.arange(D, device=DEVICE)
    grp, e = d // 32, d % 32
    at = (((r * 4 + e // 8) * NG + grp) * 2 + e % 2) * 2 + e % 8 // 4  # the K byte of dim d
    k = raw.gather(2, at[:, None].expand(-1, c["Hkv"], -1)).long() >> (e % 4 // 2 * 4) & 15
    halves = raw.view(torch.float16).double()
    base = 4 * D
    at = (base + (r * NG + grp) * 2)[:, None].expand(-1, c["Hkv"], -1)
    k = halves.gather(2, at + 1) + halves.gather(2, at) * k
    tp, t, hi = r // 8, r % 8 // 2, r % 2
    at = 8 * D + 64 * NG + ((((tp * 8 + e // 4) * 4 + t) * NG + grp) * 2 + hi) * 2 + e % 4 // 2
    v = raw.gather(2, at[:, None].expand(-1, c["Hkv"], -1)).long() >> (e % 2 * 4) & 15
    base = 8 * D + 32 * NG
    at = (base + ((grp * 4 + t) * 2 + tp) * 2 + hi)[:, None].expand(-1, c["Hkv"], -1)
    v = halves.gather(2, at + 16 * NG) + halves.gather(2, at) * v
    return k, v


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, D = c["B"], c["D"]
    if c["op"] == "rotary":
        a = (s["positions"], s["inv_freq"], c["interleaved"])
        out = [_turned(s["q"], *a), _turned(s["k"], *a)]
        if c["train"]:
            out += [_turned(s["dq"], *a, -1.0), _turned(s["dk"], *a, -1.0)]
        return out
    if c["op"] == "append":
        at = s["starts"].long()[:, None] + torch.arange(c["S"], device=DEVICE)
        q = _turned(s["q"], at, s["inv_freq"], c["interleaved"])
        k, v = _turned(s["k"], at, s["inv_freq"], c["interleaved"]), s["v"].double()
        if c["bits"] == 4:
            k, v = _four_bits(k), _four_bits(v)
        if not c["read"]:
            kp, vp = s["k_pages"].double(), s["v_pages"].double()
            for b in range(B):
                j = at[b, :s["counts"][b]]
                pages = s["table"][b].long()[j // c["page"]]
                kp[pages, :, j % c["page"]] = k[b, :len(j)]
                vp[pages, :, j % c["page"]] = v[b, :len(j)]
            return [q, kp, vp]
        ks, vs = (torch.zeros((B, s["max_len"], c["Hkv"], D), dtype=torch.float64, device=DEVICE) for _ in range(2))
        for b in range(B):
            n, m = int(s["starts"][b]), int(s["counts"][b])
            ks[b, :n], vs[b, :n] = _cached(s, b, n)
            ks[b, n:n + m], vs[b, n:n + m] = k[b, :m], v[b, :m]
        return [q, ks, vs]
    if c["op"] == "read":
        ks, vs = (torch.zeros((B, s["max_len"], c["Hkv"], D), dtype=torch.float64, device=DEVICE) for _ in range(2))
        for b in range(B):
            n = int(s["lengths"][b])
            ks[b, :n], vs[b, :n] = _cached(s, b, n)
        return [ks, vs]
    out = torch.zeros((B, c["S"], c["H"], D), dtype=torch.float64, device=DEVICE)
    for b in range(B):
        n = int(s["lengths"][b])
        k, v = _cached(s, b, n)
        k, v = (x.repeat_interleave(c["H"] // c["Hkv"], dim=1) for x in (k, v))
        for i in range(c["S"]):
            m = n - c["S"] + 1 + i
            if m > 0:
                score = torch.einsum("hd,nhd->hn", s["q"][b, i].double(), k[:m]) * s["scale"]
                out[b, i] = torch.einsum("hn,nhd->hd", torch.softmax(score, dim=-1), v[:m])
    return out
