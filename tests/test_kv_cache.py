"""The paged key/value cache (flash_attn_volta_b200.kv_cache): append, read and
attention against the float64 oracle.

Tolerances.  Append and read: 16-bit values are copied exactly; rotated keys
as in test_rotary (half a step of the type, and 2^-21 (|x1| + |x2|) for the fp32
arithmetic); a 4-bit value without rotation is the definition's (its minimum,
scale and code are exact in fp32), rounded to the type (half a step, of a value
that fp32 holds to 2^-24); with rotation it is within half a scale of the
rotated value, plus that value's own error and the same rounding, plus one
fp16 step of minimum and scale each (a key that moves by 2^-21 may move them).

Attention.  out = sum p v / sum p.  Its rounding: u |out|.  Each p is rounded to
the operand type once (u' relative), at 4 bits p times the scale once more
(fp16), with at most 2^-25 lost per token where fp16 is subnormal, and its
exponent's error: a score is a sum of D products, which the tensor core sums
with at least 22 bits, so it is off by at most (D + 8) 2^-22 scale sum |q||k|
=: e; exp's own error is below 2^-21.  All relative errors act on sum p |v|:
tolerance u |out| + (k u' + 2^-20 + 2 e) sum p |v| + 15 n 2^-25 (1 + s), with
k = 1 at 16 bits, 2 at 4 bits, |v| at 4 bits being |m| + s c; lse within 2^-20
(1 + |lse|) + e.
"""
import ctypes
import math

import pytest
import torch

from flash_attn_volta_b200 import _lib, check_status, flash_attn, ops
from flash_attn_volta_b200.kv_cache import (PagedKVCache, flash_attn_decode, kv_cache_append,
                                            kv_cache_read)
from flash_attn_volta_b200.rotary import Rotary
from oracle import serving_oracle as so

DEV = torch.device("cuda", 0)
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Pool:
    """A cache whose pages are handed out in shuffled order; every byte that no
    token was written to is 0xFF (a NaN in fp16 and bf16)."""

    def __init__(self, lengths, page, Hkv, D, dtype, bits, seed=0, width=None):
        per = [(n + page - 1) // page for n in lengths]
        self.cache = PagedKVCache.allocate(sum(per) + 2, page, Hkv, D, dtype, bits, DEV)
        for t in (self.cache.k_pages, self.cache.v_pages):
            if t is not None:
                t.view(torch.uint8).fill_(255)
        order = torch.randperm(sum(per) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lengths), width or max(1, max(per))), -7, dtype=torch.int32)
        for b, n in enumerate(per):
            for i in range(n):
                self.table[b, i] = order.pop()
        self.table_dev = self.table.to(DEV)
        self.lengths = _ints(lengths)


def _kv(B, S, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    shift = torch.randn(D, generator=g)
    return [(torch.randn((B, S, Hkv, D), generator=g) + shift).to(dtype) for _ in range(2)]


def _filled(lengths, page, Hkv, D, dtype, bits, seed=0, width=None):
    """A pool holding k, v (B, S, Hkv, D) of those lengths, and what it stands for in
    float64: k, v and |v|'s bound."""
    pool = Pool(lengths, page, Hkv, D, dtype, bits, seed, width)
    B, S = len(lengths), max(1, max(lengths))
    k, v = _kv(B, S, Hkv, D, dtype, seed + 1)
    kv_cache_append(pool.cache, k.to(DEV), v.to(DEV), pool.table_dev, _ints([0] * B), pool.lengths)
    if bits == 16:
        return pool, k.double(), v.double(), v.double().abs()
    kc, km, ks = so.four_bit(k)
    vc, vm, vs = so.four_bit(v)
    return pool, so.values(kc, km, ks), so.values(vc, vm, vs), so.values(vc, vm.abs(), vs)


# ---------------------------------------------------------------- CPU
def test_block_layout_of_the_oracle_holds_each_byte_of_a_token_once():
    """Codes of one token change only that token's bytes."""
    z = torch.zeros(16, 64)
    p = torch.zeros(16, 2, dtype=torch.float64)
    base = so.block_bytes(z, p, p, z, p, p)
    assert base.shape == (20 * 64,)
    owner = torch.full((base.size,), -1)
    for r in range(16):
        c, one = z.clone(), p.clone()
        c[r], one[r] = 15, 1.0
        changed = torch.from_numpy(so.block_bytes(c, one, one, c, one, one) != base)
        assert bool((owner[changed] == -1).all())
        owner[changed] = r


def test_cache_refusals():
    z = lambda *s, t=F16: torch.zeros(s, dtype=t)  # noqa: E731
    blocks = z(2, 1, 4, 20 * 64, t=torch.uint8)
    for bad in (lambda: PagedKVCache(z(2, 1, 64, 64), z(2, 1, 64, 32)),
                lambda: PagedKVCache(z(2, 1, 64, 64), z(2, 1, 64, 64, t=BF16)),
                lambda: PagedKVCache(z(2, 1, 64, 64, t=torch.float32), z(2, 1, 64, 64, t=torch.float32)),
                lambda: PagedKVCache(z(2, 1, 64, 48), z(2, 1, 64, 48)),
                lambda: PagedKVCache(z(2, 1, 24, 64), z(2, 1, 24, 64)),
                lambda: PagedKVCache(z(2, 1, 8, 64), z(2, 1, 8, 64)),
                lambda: PagedKVCache(z(2, 1, 2048, 64), z(2, 1, 2048, 64)),
                lambda: PagedKVCache(z(0, 1, 64, 64), z(0, 1, 64, 64)),
                lambda: PagedKVCache(z(2, 64, 1, 64).transpose(1, 2), z(2, 64, 1, 64).transpose(1, 2)
                                     .expand(2, 1, 64, 64)[:, :, :32]),
                lambda: PagedKVCache.of_blocks(blocks, 128), lambda: PagedKVCache.of_blocks(blocks, 16),
                lambda: PagedKVCache.of_blocks(blocks.short(), 64),
                lambda: PagedKVCache.of_blocks(blocks, 64, torch.float32),
                lambda: PagedKVCache.of_blocks(z(2, 1, 3, 20 * 64, t=torch.uint8), 64),
                lambda: PagedKVCache.allocate(2, 64, 1, 64, bits=8, device="cpu")):
        with pytest.raises(AssertionError):
            bad()
    c = PagedKVCache.of_blocks(blocks, 64)
    assert (c.page_size, c.head_dim, c.bits, c.num_pages, c.n_heads) == (64, 64, 4, 2, 1)


def test_call_refusals():
    """Each wrong argument is refused before anything reaches the device."""
    c = PagedKVCache(torch.zeros(2, 2, 64, 64, dtype=F16), torch.zeros(2, 2, 64, 64, dtype=F16))
    k, q = torch.zeros(1, 3, 2, 64, dtype=F16), torch.zeros(1, 3, 4, 64, dtype=F16)
    table, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for bad in (lambda: kv_cache_append(c, k, k, table, one),  # on the CPU
                lambda: kv_cache_append(c, k[:, :, :1], k[:, :, :1], table, one),
                lambda: kv_cache_append(c, k, k[:, :2], table, one),
                lambda: kv_cache_append(c, k.bfloat16(), k.bfloat16(), table, one),
                lambda: kv_cache_read(c, table, one), lambda: kv_cache_read(c, table, one, -1),
                lambda: flash_attn_decode(q, c, table, one),
                lambda: flash_attn_decode(q[:, :, :3], c, table, one),
                lambda: flash_attn_decode(q[..., :32], c, table, one),
                lambda: flash_attn_decode(q.bfloat16(), c, table, one)):
        with pytest.raises(AssertionError):
            bad()


def test_c_abi_refusals():
    lib = _lib.load()
    base = dict(k_pages=4096, v_pages=4096, num_pages=2, page_size=64, nheads_kv=2, head_dim=64,
                dtype=0, bits=16)
    h = lambda heads=2, inp=256, out=256: _lib.Heads(inp, out, 0, 0, 0, heads)  # noqa: E731

    def calls(cache, H=4, B=1, S=1, width=1, table=256, ints=256, io=256):
        c = ctypes.byref(_lib.KvCache(**cache))
        k, q = ctypes.byref(h(cache["nheads_kv"])), ctypes.byref(h(H, io, io))
        return (lib.fa_sm100_kv_append(c, k, k, q, table, width, ints, None, None, 0, 0, 1.0, B, S,
                                       None, None),
                lib.fa_sm100_kv_read(c, table, width, ints, io, io, B, S, None, None),
                lib.fa_sm100_decode(c, io, io, None, table, width, ints, None, 256, 0, B, S, H, 1.0, 1,
                                    None, None))

    bad = [dict(k_pages=None), dict(k_pages=4104), dict(v_pages=None), dict(num_pages=0),
           dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(nheads_kv=0),
           dict(head_dim=48), dict(head_dim=256), dict(dtype=3), dict(bits=8),
           dict(bits=4, head_dim=16), dict(num_pages=1 << 27)]
    for b in bad:
        assert calls({**base, **b}) == (_lib.FA_ERR_ARG,) * 3, b
    for kw in (dict(B=0), dict(S=0), dict(width=0), dict(table=None), dict(table=258), dict(ints=None),
               dict(io=None), dict(io=264)):
        assert calls(base, **kw) == (_lib.FA_ERR_ARG,) * 3, kw
    assert calls(base, H=3)[2] == _lib.FA_ERR_ARG
    c = ctypes.byref(_lib.KvCache(**base))
    assert lib.fa_sm100_decode_workspace_bytes(c, 1, 1, 1, 3) == 0
    assert lib.fa_sm100_decode_workspace_bytes(c, 4, 1, 1, 4) > 0
    k, k1 = ctypes.byref(h()), ctypes.byref(h(1))
    args = (c, k, k, None, 256, 1, 256, None)
    assert lib.fa_sm100_kv_append(c, k1, k, None, 256, 1, 256, None, None, 0, 0, 1.0, 1, 1, None, None) == 1
    for R in (0, 7, 66):
        assert lib.fa_sm100_kv_append(*args, 256, R, 0, 1.0, 1, 1, None, None) == _lib.FA_ERR_ARG
    assert lib.fa_sm100_kv_append(*args, 260, 64, 0, 1.0, 1, 1, None, None) == _lib.FA_ERR_ARG
    assert lib.fa_sm100_kv_read(c, 256, 1, 256, 256, 256, 65536, 1, None, None) == _lib.FA_ERR_ARG


def test_fake_shapes():
    ops.load()
    m = lambda *s, t=F16: torch.empty(s, dtype=t, device="meta")  # noqa: E731
    q, kp, table, n = m(2, 3, 4, 64), m(9, 2, 32, 64), m(2, 5, t=torch.int32), m(2, t=torch.int32)
    out, lse = torch.ops.fav.decode_lse(q, kp, kp, table, n, None, True, 0.1)
    assert out.shape == q.shape and lse.shape == (2, 4, 3)
    blocks = m(9, 2, 2, 20 * 64, t=torch.uint8)
    k, v = torch.ops.fav.kv_read(blocks, None, BF16, table, n, 77)
    assert k.shape == v.shape == (2, 77, 2, 64) and k.dtype == BF16
    new = m(2, 3, 2, 64)
    assert torch.ops.fav.kv_append(kp, kp, new, new, q, table, n, None, None, False, 1.0).shape == q.shape
    for bad in (lambda: torch.ops.fav.decode(m(2, 3, 3, 64), kp, kp, table, n, None, True, 0.1),
                lambda: torch.ops.fav.decode(q, m(9, 2, 32, 32), m(9, 2, 32, 32), table, n, None, True, 0.1),
                lambda: torch.ops.fav.kv_append(kp, kp, m(2, 3, 1, 64), new, None, table, n, None, None, False, 1.0),
                lambda: torch.ops.fav.kv_read(kp, m(9, 2, 16, 64), F16, table, n, 4)):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------- GPU: append and read
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page,Hkv,D", [(16, 1, 32), (32, 3, 64), (64, 2, 128)])
def test_append4_writes_the_defined_bytes(page, Hkv, D, dtype):
    """Blocks byte for byte, tokens in two calls that end inside a block; bytes
    of tokens that were not appended stay."""
    pool = Pool([37], page, Hkv, D, dtype, 4)
    k, v = _kv(1, 37, Hkv, D, dtype, 3)
    for a, b in ((0, 21), (21, 37)):
        kv_cache_append(pool.cache, k[:, a:b].to(DEV), v[:, a:b].to(DEV), pool.table_dev, _ints([a]))
    check_status(DEV)
    kc, km, ks = so.four_bit(k)
    vc, vm, vs = so.four_bit(v)
    got = pool.cache.k_pages.cpu()
    want = torch.full_like(got, 255)
    for h in range(Hkv):
        for blk in range(3):
            n = min(16, 37 - 16 * blk)
            pick = lambda t, w: torch.cat([t[0, 16 * blk:16 * blk + n, h], t.new_zeros(16 - n, w)])  # noqa: E731
            raw = torch.from_numpy(so.block_bytes(pick(kc, D), pick(km, D // 32), pick(ks, D // 32),
                                                  pick(vc, D), pick(vm, D // 32), pick(vs, D // 32)))
            mark = torch.zeros(16, D)
            mark[:n], one = 15, torch.zeros(16, D // 32, dtype=torch.float64)
            one[:n] = 1.0
            zero = torch.zeros(16, D // 32, dtype=torch.float64)
            mine = torch.from_numpy(so.block_bytes(mark, one - 3 * one, one, mark, one - 3 * one, one) !=
                                    so.block_bytes(mark * 0, zero, zero, mark * 0, zero, zero))
            # every byte of an appended token: codes, and both bytes of its parameters
            for a, b in ((8 * D, 10 * D), (18 * D, 20 * D)):
                half = mine[a:b].view(-1, 2).any(1)
                mine[a:b] = half[:, None].expand(-1, 2).reshape(-1)
            page_id = int(pool.table[0, blk * 16 // page])
            dst = want[page_id, h, blk * 16 % page // 16]
            dst[mine] = raw[mine]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,D", [(16, 16), (16, 64), (16, 128), (4, 32), (4, 64), (4, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_ragged_and_read(bits, D, dtype):
    lengths = [0, 1, 16, 33, 70]
    pool, k, v, _ = _filled(lengths, 16 if D == 32 else 32, 2, D, dtype, bits, seed=D)
    for max_len in (None, 70, 45, 1):
        ko, vo = kv_cache_read(pool.cache, pool.table_dev, pool.lengths, max_len)
        n = ko.shape[1]
        assert ko.is_contiguous() and vo.dtype == dtype
        for b, length in enumerate(lengths):
            m = min(length, n)
            assert not ko[b, m:].any() and not vo[b, m:].any()
            for got, ref in ((ko[b, :m], k[b, :m]), (vo[b, :m], v[b, :m])):
                got = got.cpu().double()
                if bits == 16:
                    assert torch.equal(got, ref)
                else:
                    assert bool(((got - ref).abs() <= HALF[dtype] * (1 + 2.0 ** -10) * ref.abs() + 2.0 ** -25).all())
    check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("R,inter", [(64, False), (64, True), (32, False), (24, True), (8, False)])
def test_append_rotates_on_the_way(bits, R, inter):
    """q and k rotated at the tokens' positions, k stored; rows behind a
    sequence's count are not stored, but its q is rotated."""
    dtype, D, B, S, starts, counts = BF16, 64, 3, 5, [0, 30, 63], [5, 3, 0]
    pool = Pool([70] * 3, 32, 2, D, dtype, bits)
    k, v = _kv(B, S, 2, D, dtype, 5)
    q = _kv(B, S, 6, D, dtype, 6)[0]
    freq = 10000.0 ** (-2.0 * torch.arange(R // 2, dtype=torch.float64) / R)
    qo = kv_cache_append(pool.cache, k.to(DEV), v.to(DEV), pool.table_dev, _ints(starts), _ints(counts),
                         q=q.to(DEV), rotary=Rotary(freq.to(DEV), inter, 1.5))
    check_status(DEV)
    pos = torch.tensor(starts)[:, None] + torch.arange(S)
    ref = so.rotate(q, pos, freq, inter, 1.5)
    slack = lambda x: 2.0 ** -21 * 1.5 * 2 * x.double().abs().amax(-1, True)  # noqa: E731
    assert bool(((qo.cpu().double() - ref).abs() <= HALF[dtype] * ref.abs() + slack(q)).all())
    ko, vo = kv_cache_read(pool.cache, pool.table_dev, pool.lengths)
    kr = so.rotate(k, pos, freq, inter, 1.5)
    _, km, ks = so.four_bit(kr)
    vc, vm, vs = so.four_bit(v)
    for b in range(B):
        for s in range(counts[b]):
            got_k, got_v = ko[b, starts[b] + s].cpu().double(), vo[b, starts[b] + s].cpu().double()
            tol = HALF[dtype] * kr[b, s].abs() + slack(k)[b, s]
            if bits == 4:
                half = (ks[b, s] / 2 + 2.0 ** -10 * km[b, s].abs() + 15 * 2.0 ** -10 * ks[b, s])
                tol = tol + half.repeat_interleave(32, -1) * (1 + HALF[dtype])
                refv = so.values(vc, vm, vs)[b, s]
                assert bool(((got_v - refv).abs() <= HALF[dtype] * (1 + 2.0 ** -10) * refv.abs()).all())
            else:
                assert torch.equal(got_v, v[b, s].double())
            assert bool(((got_k - kr[b, s]).abs() <= tol).all())
    # nothing else was written
    written = torch.zeros(3, 96, dtype=torch.bool)
    for b in range(B):
        written[b, starts[b]:starts[b] + counts[b]] = True
    full = _ints([96] * 3)
    ka, va = kv_cache_read(pool.cache, pool.table_dev, full)
    assert bool(ka.isnan().flatten(2).all(-1).cpu()[~written].all())
    assert bool(va.isnan().flatten(2).all(-1).cpu()[~written].all())
    assert not bool(ka.isnan().flatten(2).any(-1).cpu()[written].any())


@pytest.mark.gpu
@pytest.mark.parametrize("bits,B,S,H,Hkv,D,R,inter,dtype", [
    (16, 1, 4001, 8, 2, 128, 128, False, BF16), (4, 1, 4001, 8, 2, 128, 128, False, BF16),
    (16, 2, 3001, 12, 3, 64, 32, True, F16), (4, 2, 3001, 12, 3, 64, 32, True, F16),
    (16, 3, 2003, 5, 5, 16, 16, False, F16), (4, 3, 2003, 5, 5, 32, 0, False, F16)])
def test_long_prompts_match_short_calls(bits, B, S, H, Hkv, D, R, inter, dtype):
    """Prompts long enough for each thread to stream several rounds: the cache and
    q are bit for bit what appends of a few tokens leave, ragged counts."""
    counts = [S, S - 700, 13][:B]
    g = torch.Generator(device=DEV).manual_seed(S)
    mk = lambda h: torch.randn((B, S, h, D), generator=g, device=DEV).to(dtype)  # noqa: E731
    q, k, v = mk(H), mk(Hkv), mk(Hkv)
    rot = Rotary.build(R, interleaved=inter, device=DEV) if R else None
    long, short = (Pool([S + 9] * B, 32, Hkv, D, dtype, bits) for _ in range(2))
    qo = kv_cache_append(long.cache, k, v, long.table_dev, _ints([9] * B), _ints(counts), q=q, rotary=rot)
    qs = torch.cat([kv_cache_append(short.cache, k[:, a:a + 50], v[:, a:a + 50], short.table_dev,
                                    _ints([9 + a] * B), _ints([max(0, min(50, n - a)) for n in counts]),
                                    q=q[:, a:a + 50], rotary=rot) for a in range(0, S, 50)], 1)
    check_status(DEV)
    assert torch.equal(qo, qs)
    for a, b in ((long.cache.k_pages, short.cache.k_pages), (long.cache.v_pages, short.cache.v_pages)):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_append_strides_and_copy_of_q():
    """k, v and q as slices of one projection, at an odd offset too; without
    rotary q comes back as it is."""
    for off in (0, 1):
        flat = torch.randn(2 * 3 * 8 * 64 + off, generator=torch.Generator().manual_seed(2)).half().to(DEV)
        qkv = flat[off:].view(2, 3, 8, 64)
        q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
        pool = Pool([3, 3], 16, 2, 64, F16, 16)
        qo = kv_cache_append(pool.cache, k, v, pool.table_dev, _ints([0, 0]), q=q)
        ko, vo = kv_cache_read(pool.cache, pool.table_dev, pool.lengths, 3)
        assert torch.equal(qo, q) and torch.equal(ko, k) and torch.equal(vo, v)


@pytest.mark.gpu
def test_four_bit_edge_values():
    """Equal values, tiny ones, ones beyond fp16 and a NaN."""
    D = 64
    x = torch.zeros(1, 6, 1, D)
    x[0, 0] = 3.14159
    x[0, 1] = torch.linspace(0, 3e-7, D)
    x[0, 2] = 3e38 * torch.linspace(-1, 1, D)  # (linspace of +-3e38 itself overflows to NaN)
    x[0, 3] = torch.linspace(-1, 1, D)
    x[0, 3, 0, 5] = math.nan
    x[0, 4] = math.inf
    x[0, 4, 0, :32] = -math.inf
    x[0, 5] = -0.0
    x = x.bfloat16()
    pool = Pool([6], 16, 1, D, BF16, 4)
    kv_cache_append(pool.cache, x.to(DEV), x.to(DEV), pool.table_dev, _ints([0]))
    for got in kv_cache_read(pool.cache, pool.table_dev, pool.lengths, 6):
        got = got.cpu().double()[0, :, 0]
        assert bool(((got[0] - x[0, 0, 0].double()).abs() <= 2.0 ** -8 * 3.2 + 2.0 ** -10).all())
        assert bool(((got[1] - x[0, 1, 0].double()).abs() <= 2.0 ** -24).all())
        want = x[0, 2, 0].double().clamp(-65504, 65504)
        assert bool(((got[2] - want).abs() <= 65504 / 15 + 65504 * 2.0 ** -8).all())
        assert bool(got[3, :32].isnan().all()) and not bool(got[3, 32:].isnan().any())
        assert bool((got[4, :32] == -65536).all() and (got[4, 32:] == 65536).all())  # -+65504 in bf16
        assert bool((got[5] == 0).all())


# ---------------------------------------------------------------- GPU: attention
def _check_decode(q, out, lse, k, v, size, lengths, starts, causal, bits, scale=None):
    B, S, H, D = q.shape
    G = H // k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    u, up = HALF[q.dtype], HALF[q.dtype] if bits == 16 else HALF[F16]
    for b in range(B):
        n = lengths[b]
        for h in range(H):
            first = n - S if starts is None else starts[b]
            limits = [min(n, first + i + 1) if causal else n for i in range(S)]
            ref, rl, mass, reach = so.decode(q[b, :, h].double(), k[b, :n, h // G], v[b, :n, h // G],
                                             size[b, :n, h // G], limits, scale)
            e = ((D + 8) * 2.0 ** -22 * reach)[:, None]
            tol = u * ref.abs() + ((1 if bits == 16 else 2) * up + 2.0 ** -20 + 2 * e) * mass + 2.0 ** -25
            if bits == 4:
                s = 2 * size[b, :n, h // G].max() / 15 if n else 0.0
                tol = tol + 15 * n * 2.0 ** -25 * (1 + s)
            got = out[b, :, h].cpu().double()
            bad = (got - ref).abs() > tol
            assert not bad.any(), (b, h, float(((got - ref).abs() / tol).max()))
            if lse is not None:
                gl = lse[b, h].cpu().double()
                assert torch.equal(gl == math.inf, rl == math.inf)
                there = rl < math.inf
                assert bool(((gl - rl)[there].abs() <= 2.0 ** -20 * (1 + rl[there].abs()) + e[there, 0]).all())


DECODE = [  # bits, B lengths, S, H, Hkv, D, page
    (16, [1], 1, 1, 1, 64, 16), (4, [1], 1, 1, 1, 64, 16),
    (16, [0, 17, 300], 1, 4, 2, 16, 16), (16, [0, 17, 300], 1, 6, 2, 32, 32),
    (16, [5, 64, 65, 129], 1, 8, 1, 64, 64), (16, [5, 1000, 33], 1, 8, 2, 128, 128),
    (4, [0, 17, 300], 1, 6, 2, 32, 32), (4, [5, 128, 129, 257], 1, 8, 1, 64, 64),
    (4, [5, 1000, 33], 1, 8, 2, 128, 128), (4, [31, 47, 16], 1, 5, 5, 128, 16),
    (16, [9, 40, 3, 200], 5, 6, 2, 64, 32), (4, [9, 40, 3, 200], 5, 6, 2, 64, 32),
    (16, [70, 19], 17, 3, 1, 128, 16), (4, [70, 19], 17, 3, 1, 128, 16),
    (4, [2500, 1], 2, 16, 2, 128, 256), (16, [2500, 1], 2, 16, 2, 64, 1024),
    (4, [600], 3, 32, 4, 32, 64), (16, [600], 3, 32, 4, 16, 64),
    (4, [500, 77], 7, 12, 3, 64, 32), (16, [500, 77], 7, 12, 3, 64, 32),
    (4, [290, 3], 9, 8, 2, 32, 16), (16, [290, 3], 9, 8, 2, 32, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits,lengths,S,H,Hkv,D,page", DECODE)
def test_decode_matches_oracle(bits, lengths, S, H, Hkv, D, page, causal, dtype):
    if S == 1 and not causal:
        pytest.skip("one query token sees every cached one either way")
    pool, k, v, size = _filled(lengths, page, Hkv, D, dtype, bits, seed=sum(lengths))
    q = (2 * torch.randn((len(lengths), S, H, D), generator=torch.Generator().manual_seed(9))).to(dtype)
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, causal,
                                 return_softmax_lse=True)
    check_status(DEV)
    assert out.dtype == dtype and out.shape == q.shape and lse.shape == (len(lengths), H, S)
    _check_decode(q, out, lse, k, v, size, lengths, None, causal, bits)
    alone = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, causal)
    assert torch.equal(alone, out)  # and bit for bit the same twice


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_decode_starts(bits):
    """A padded batch: each sequence's first query position is given; rows that
    stand before every token see none."""
    lengths, starts, S = [40, 3, 90], [37, -2, 80], 5
    pool, k, v, size = _filled(lengths, 16, 2, 64, F16, bits, seed=4)
    q = torch.randn((3, S, 4, 64), generator=torch.Generator().manual_seed(8)).half()
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, starts=_ints(starts),
                                 sm_scale=0.3, return_softmax_lse=True)
    _check_decode(q, out, lse, k, v, size, lengths, starts, True, bits, 0.3)
    assert not out[1, :2].any() and bool((lse[1, :, :2] == math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_decode_ignores_what_a_row_does_not_see(bits, bad):
    """NaN and infinity in tokens behind a row's limit, and in what the pages
    hold behind the sequence (0xFF, a NaN), leave the row's output alone."""
    n, S = 45, 4
    pool, k, v, size = _filled([n], 16, 1, 64, BF16, bits, seed=12)
    q = torch.randn((1, S, 2, 64), generator=torch.Generator().manual_seed(8)).bfloat16()
    ref = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths)
    _check_decode(q, ref, None, k, v, size, [n], None, True, bits)
    poison = torch.full((1, 2, 1, 64), bad, dtype=BF16, device=DEV)
    kv_cache_append(pool.cache, poison, poison, pool.table_dev, _ints([n - 2]))
    out = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths)
    assert torch.equal(out[:, :2], ref[:, :2])
    if math.isnan(bad):
        assert bool(out[:, 2:].isnan().all())
    check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_bad_pages_and_lengths_are_reported_and_skipped(bits):
    """A page id outside the cache takes its tokens out; a length beyond the
    table is cut to it; a negative one is none.  Each sets status bit 2."""
    pool, k, v, size = _filled([40, 40, 40], 16, 1, 64, F16, bits, seed=6)
    q = torch.randn((3, 1, 2, 64), generator=torch.Generator().manual_seed(8)).half()
    check_status(DEV)
    for wrong in (-1, pool.cache.num_pages, 2 ** 31 - 1, -2 ** 31):
        table = pool.table.clone()
        table[1, 1] = wrong
        out = flash_attn_decode(q.to(DEV), pool.cache, table.to(DEV), pool.lengths)
        with pytest.raises(RuntimeError, match="status 4"):
            check_status(DEV)
        keep = torch.cat([torch.arange(16), torch.arange(32, 40)])
        ks, vs, ss = (t.clone() for t in (k, v, size))
        for t, src in ((ks, k), (vs, v), (ss, size)):
            t[1, :24] = src[1, keep]
        _check_decode(q, out, None, ks, vs, ss, [40, 24, 40], [39, 39, 39], True, bits)
        ko, vo = kv_cache_read(pool.cache, table.to(DEV), pool.lengths, 40)
        assert not ko[1, 16:32].any() and bool(ko[1, 32:40].any()) and not vo[1, 16:32].any()
        with pytest.raises(RuntimeError, match="status 4"):
            check_status(DEV)
        before = [t.clone() for t in (pool.cache.k_pages, pool.cache.v_pages) if t is not None]
        new = torch.zeros(3, 1, 1, 64, dtype=F16, device=DEV)
        kv_cache_append(pool.cache, new, new, table.to(DEV), _ints([1000, 16, -1]))
        with pytest.raises(RuntimeError, match="status 4"):
            check_status(DEV)
        for t, was in zip((pool.cache.k_pages, pool.cache.v_pages), before):
            assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))
    out = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev[:, :2].contiguous(), _ints([32, 40, -3]))
    with pytest.raises(RuntimeError, match="status 4"):
        check_status(DEV)
    _check_decode(q, out, None, k, v, size, [32, 32, 0], None, True, bits)


@pytest.mark.gpu
def test_empty_calls():
    pool, *_ = _filled([5], 16, 2, 64, F16, 16)
    none = torch.empty((0, 1, 2, 64), dtype=F16, device=DEV)
    table, ints = torch.empty((0, 1), dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV)
    assert flash_attn_decode(none, pool.cache, table, ints).shape == none.shape
    assert kv_cache_append(pool.cache, none, none, table, ints) is None
    assert kv_cache_read(pool.cache, table, ints)[0].shape == (0, 16, 2, 64)
    assert kv_cache_read(pool.cache, pool.table_dev, pool.lengths, 0)[0].shape == (1, 0, 2, 64)
    q = torch.empty((1, 0, 4, 64), dtype=F16, device=DEV)
    assert flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_refusals_on_the_gpu(bits):
    """Arguments that do not fit are refused before a launch; the cache stays."""
    pool, *_ = _filled([20, 5], 16, 2, 64, F16, bits)
    c, table, n = pool.cache, pool.table_dev, pool.lengths
    q, k = torch.zeros((2, 3, 4, 64), dtype=F16, device=DEV), torch.zeros((2, 3, 2, 64), dtype=F16, device=DEV)
    rot, cpu = Rotary.build(64, device=DEV), torch.zeros(2, dtype=torch.int32)
    before = c.k_pages.clone()
    for bad in (lambda: flash_attn_decode(q[:, :, :3], c, table, n), lambda: flash_attn_decode(q[0], c, table, n),
                lambda: flash_attn_decode(q[..., :32], c, table, n), lambda: flash_attn_decode(q.cpu(), c, table, n),
                lambda: flash_attn_decode(q.bfloat16(), c, table, n), lambda: flash_attn_decode(q[:1], c, table, n),
                lambda: flash_attn_decode(q, c, table.long(), n), lambda: flash_attn_decode(q, c, table[0], n),
                lambda: flash_attn_decode(q, c, table[:, :0], n), lambda: flash_attn_decode(q, c, table, n.long()),
                lambda: flash_attn_decode(q, c, table, cpu), lambda: flash_attn_decode(q, c, table, n, starts=n[:1]),
                lambda: kv_cache_append(c, k[:, :, :1], k[:, :, :1], table, n),
                lambda: kv_cache_append(c, k, k[:, :2], table, n), lambda: kv_cache_append(c, k, k.float(), table, n),
                lambda: kv_cache_append(c, k.bfloat16(), k.bfloat16(), table, n),
                lambda: kv_cache_append(c, k, k, table, n, n[:1]), lambda: kv_cache_append(c, k, k, table[:1], n),
                lambda: kv_cache_append(c, k, k, table, n, q=q[:, :2]), lambda: kv_cache_append(c, k, k.cpu(), table, n),
                lambda: kv_cache_append(c, k, k, table, n, rotary=Rotary.build(66, device=DEV)),
                lambda: kv_cache_append(c, k, k, table, n, rotary=Rotary.build(64, device="cpu")),
                lambda: kv_cache_read(c, table, n.long()), lambda: kv_cache_read(c, table[:1], n),
                lambda: kv_cache_read(c, table, cpu)):
        with pytest.raises(AssertionError):
            bad()
    torch.cuda.synchronize(DEV)
    check_status(DEV)
    assert torch.equal(c.k_pages.view(torch.uint8), before.view(torch.uint8))
    assert flash_attn_decode(q, c, table, n).shape == q.shape  # and the right call works
    assert kv_cache_append(c, k, k, table, _ints([0, 0]), q=q, rotary=rot).shape == q.shape


@pytest.mark.gpu
def test_gradients_are_refused():
    pool, *_ = _filled([5], 16, 2, 64, F16, 16)
    q = torch.zeros((1, 1, 2, 64), dtype=F16, device=DEV, requires_grad=True)
    with pytest.raises(AssertionError, match="inference"):
        flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths)
    with torch.no_grad():
        flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_serving_run(bits):
    """A prompt through flash_attn while it is appended, a second chunk of it over
    the prefix read back, then tokens one at a time: each result is the
    attention over everything so far."""
    B, H, Hkv, D, page, chunk = 2, 4, 2, 64, 16, 40
    total = 2 * chunk + 6
    g = torch.Generator().manual_seed(21)
    mk = lambda h: torch.randn((B, total, h, D), generator=g).half()  # noqa: E731
    q, k, v = mk(H), mk(Hkv), mk(Hkv)
    rot = Rotary.build(D, device=DEV)
    freq = rot.inv_freq.cpu()
    pool = Pool([total] * B, page, Hkv, D, F16, bits)
    kr = so.rotate(k, torch.arange(total), freq)
    qr = so.rotate(q, torch.arange(total), freq)
    got = []
    for a in (0, chunk):
        part = slice(a, a + chunk)
        qc = kv_cache_append(pool.cache, k[:, part].to(DEV), v[:, part].to(DEV), pool.table_dev,
                             _ints([a] * B), q=q[:, part].to(DEV), rotary=rot)
        ka, va = kv_cache_read(pool.cache, pool.table_dev, _ints([a + chunk] * B), a + chunk)
        got.append(flash_attn(qc, ka, va, causal=True))
    for n in range(2 * chunk, total):
        one = slice(n, n + 1)
        qc = kv_cache_append(pool.cache, k[:, one].to(DEV), v[:, one].to(DEV), pool.table_dev,
                             _ints([n] * B), q=q[:, one].to(DEV), rotary=rot)
        got.append(flash_attn_decode(qc, pool.cache, pool.table_dev, _ints([n + 1] * B)))
    check_status(DEV)
    out = torch.cat(got, 1).cpu().double()
    ko, vo = (t.cpu().double() for t in kv_cache_read(pool.cache, pool.table_dev, pool.lengths, total))
    half = 0.0 if bits == 16 else 0.5
    _, km, ks = so.four_bit(kr)
    step = (half * ks + 2.0 ** -9 * (km.abs() + 15 * ks)).repeat_interleave(32, -1)
    assert bool(((ko - kr).abs() <= step + 2.0 ** -10 * kr.abs() + 2.0 ** -18).all())
    for b in range(B):
        for h in range(H):
            ref, _, mass, reach = so.decode(qr[b, :, h], ko[b, :, h // 2], vo[b, :, h // 2],
                                            vo[b, :, h // 2].abs(), range(1, total + 1), D ** -0.5)
            # q rounded to fp16 once (2^-11 of the score's reach), p and out once
            # more, 4-bit values read back rounded (2^-11): 2^-8 of the sums
            tol = 2.0 ** -11 * ref.abs() + (2.0 ** -9 + 2 * 2.0 ** -10 * reach[:, None]) * mass + 2.0 ** -12
            assert bool(((out[b, :, h] - ref).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_captured_step_replays_with_other_lengths(bits):
    """Two captured steps (append, then attention) that share the cache, replayed
    in turn with other tokens, starts and lengths, give what eager calls give;
    an eager call in between does not disturb them."""
    lengths = [30, 200]
    pool, *_ = _filled(lengths, 16, 2, 64, BF16, bits, seed=2, width=16)
    used = set(pool.table.flatten().tolist())
    pool.table[0, 2] = next(i for i in range(pool.cache.num_pages) if i not in used)
    table = pool.table.to(DEV)  # sequence 0 grows into a third page
    rot = Rotary.build(64, device=DEV)
    g = torch.Generator().manual_seed(3)
    new = [torch.randn((2, 1, 2, 64), generator=g).bfloat16().to(DEV) for _ in range(6)]
    qs = [torch.randn((2, 1, 8, 64), generator=g).bfloat16().to(DEV) for _ in range(3)]

    def step(k, v, q, starts, lens):
        qr = kv_cache_append(pool.cache, k, v, table, starts, q=q, rotary=rot)
        return flash_attn_decode(qr, pool.cache, table, lens)

    want = []
    saved = pool.cache.k_pages.clone(), None if bits == 4 else pool.cache.v_pages.clone()
    for i in range(3):
        want.append(step(new[2 * i], new[2 * i + 1], qs[i], _ints([30 + i, 200 + i]), _ints([31 + i, 201 + i])))

    def restore():
        pool.cache.k_pages.copy_(saved[0])
        if bits == 16:
            pool.cache.v_pages.copy_(saved[1])

    static = [new[0].clone(), new[1].clone(), qs[0].clone(), _ints([30, 200]), _ints([31, 201])]
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*static))
        graphs.append(graph)
    restore()
    for i in range(3):
        for dst, src in zip(static, (new[2 * i], new[2 * i + 1], qs[i], _ints([30 + i, 200 + i]),
                                     _ints([31 + i, 201 + i]))):
            dst.copy_(src)
        graphs[i % 2].replay()
        flash_attn_decode(qs[0], pool.cache, table, _ints([1, 100]))
        assert torch.equal(outs[i % 2], want[i])
    check_status(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_side_stream_and_two_calls_at_once(bits):
    pool, k, v, size = _filled([700, 90], 32, 2, 128, F16, bits, seed=31)
    q = torch.randn((2, 1, 8, 128), generator=torch.Generator().manual_seed(8)).half().to(DEV)
    want = flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream(DEV))
            with torch.cuda.stream(s):
                got.append(flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths))
    torch.cuda.synchronize(DEV)
    assert all(torch.equal(o, want) for o in got)


@pytest.mark.gpu
def test_shared_pages():
    """Two sequences whose tables name the same pages (a shared prefix)."""
    pool, k, v, size = _filled([64], 16, 2, 64, F16, 4, seed=3)
    q = torch.randn((2, 1, 4, 64), generator=torch.Generator().manual_seed(8)).half()
    out = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev.expand(2, -1), _ints([64, 20]))
    _check_decode(q, out, None, k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1),
                  size.expand(2, -1, -1, -1), [64, 20], None, True, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,pages", [(16, 40000), (4, 60000)])
def test_offsets_beyond_32_bits(bits, pages):
    """Pages at the end of a cache whose byte offsets (and elements) pass 2^32."""
    cache = PagedKVCache.allocate(pages, 64, 8, 128, BF16, bits, DEV)
    assert cache.k_pages.numel() * cache.k_pages.element_size() > 2 ** 32
    k, v = _kv(1, 100, 8, 128, BF16, 3)
    table = _ints([[pages - 1, pages - 2]])
    kv_cache_append(cache, k.to(DEV), v.to(DEV), table, _ints([0]))
    ko, vo = kv_cache_read(cache, table, _ints([100]), 100)
    q = torch.randn((1, 1, 16, 128), generator=torch.Generator().manual_seed(8)).bfloat16()
    out = flash_attn_decode(q.to(DEV), cache, table, _ints([100]))
    check_status(DEV)
    if bits == 16:
        assert torch.equal(ko.cpu(), k) and torch.equal(vo.cpu(), v)
        _check_decode(q, out, None, k.double(), v.double(), v.double().abs(), [100], None, True, 16)
    else:
        kc, km, ks = so.four_bit(k)
        vc, vm, vs = so.four_bit(v)
        _check_decode(q, out, None, so.values(kc, km, ks), so.values(vc, vm, vs),
                      so.values(vc, vm.abs(), vs), [100], None, True, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,S,H,Hkv,D", [(4, 1, 64, 1, 128), (16, 1, 64, 1, 64), (4, 1, 71, 1, 64),
                                            (16, 150, 4, 4, 32), (4, 40, 6, 3, 128)])
def test_many_query_rows(bits, S, H, Hkv, D):
    """More rows than one pass holds: row blocks, the last one short."""
    lengths = [200, 170]
    pool, k, v, size = _filled(lengths, 64, Hkv, D, F16, bits, seed=5)
    q = torch.randn((2, S, H, D), generator=torch.Generator().manual_seed(8)).half()
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths,
                                 return_softmax_lse=True)
    _check_decode(q, out, lse, k, v, size, lengths, None, True, bits)


@pytest.mark.gpu
def test_strided_queries_and_negative_scale():
    pool, k, v, size = _filled([90], 16, 2, 64, BF16, 4, seed=5)
    wide = torch.randn((1, 2, 12, 64), generator=torch.Generator().manual_seed(8)).bfloat16()
    for scale in (-0.2, 0.0):
        out = flash_attn_decode(wide.to(DEV)[:, :, 1:9], pool.cache, pool.table_dev, pool.lengths, sm_scale=scale)
        _check_decode(wide[:, :, 1:9], out, None, k, v, size, [90], None, True, 4, scale)


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than threads of a CTA (each CTA sums the lengths itself)."""
    lengths = [(37 * i) % 50 for i in range(301)]
    pool, k, v, size = _filled(lengths, 16, 1, 32, F16, 16, seed=3)
    q = torch.randn((301, 1, 2, 32), generator=torch.Generator().manual_seed(8)).half()
    out = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths)
    _check_decode(q, out, None, k, v, size, lengths, None, True, 16)


@pytest.mark.gpu
def test_opcheck():
    pool, *_ = _filled([20, 5], 16, 2, 64, F16, 16)
    c = pool.cache
    q = torch.zeros((2, 1, 4, 64), dtype=F16, device=DEV)
    new = torch.zeros((2, 1, 2, 64), dtype=F16, device=DEV)
    tests = ("test_schema", "test_faketensor")
    for op in (torch.ops.fav.decode, torch.ops.fav.decode_lse):
        torch.library.opcheck(op, (q, c.k_pages, c.v_pages, pool.table_dev, pool.lengths, None, True,
                                   0.1), test_utils=tests)
    torch.library.opcheck(torch.ops.fav.kv_read, (c.k_pages, c.v_pages, F16, pool.table_dev, pool.lengths,
                                                  20), test_utils=tests)
    torch.library.opcheck(torch.ops.fav.kv_append, (c.k_pages, c.v_pages, new, new, q, pool.table_dev,
                                                    _ints([3, 4]), None, None, False, 1.0),
                          test_utils=tests)
