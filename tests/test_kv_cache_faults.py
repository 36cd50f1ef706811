"""The paged key/value cache where it can go wrong: waits that run out, infinities
that a row sees, values far below or above one, bad page ids, derivatives."""
import math

import pytest
import torch

from flash_attn_volta_b200 import _lib, check_status, flash_attn
from flash_attn_volta_b200.kv_cache import flash_attn_decode, kv_cache_append, kv_cache_read
from flash_attn_volta_b200.rotary import Rotary
from oracle import serving_oracle as so
from tests.test_kv_cache import BF16, DEV, F16, Pool, _check_decode, _filled, _ints


# ---------------------------------------------------------------- GPU: waits
@pytest.mark.gpu
@pytest.mark.parametrize("bits,length", [(16, 90), (16, 3000), (4, 90), (4, 6000)])
def test_a_wait_that_runs_out_is_reported(bits, length):
    """A test hook leaves one block's copy out: the wait for it ends at its limit, the
    status word says so, the call returns and the next one is right.  Short contexts
    and ones whose tiles outnumber a warp's ring."""
    pool, k, v, size = _filled([length, 40], 16, 1, 64, F16, bits, seed=7)
    q = torch.randn((2, 1, 4, 64), generator=torch.Generator().manual_seed(8)).half()
    call = lambda: flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths)  # noqa: E731
    lib = _lib.load()
    check_status(DEV)
    lib.fa_sm100_set_wait_timeout_ns(50_000_000)
    lib.fa_sm100_set_debug_flags(2)
    try:
        call()
        torch.cuda.synchronize(DEV)
        with pytest.raises(RuntimeError, match="timed out"):
            check_status(DEV)
    finally:
        lib.fa_sm100_set_debug_flags(0)
        lib.fa_sm100_set_wait_timeout_ns(4_000_000_000)
    out = call()
    check_status(DEV)
    _check_decode(q, out, None, k, v, size, [length, 40], None, True, bits)


# ---------------------------------------------------------------- GPU: infinities that a row sees
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("n", [512, 500])
def test_scores_of_minus_infinity_weigh_nothing(n, D, dtype):
    """Keys that hold -inf where q is positive give scores of -inf: the row is the
    attention over its other tokens, whether or not the length fills the tiles; a
    row whose scores are all -inf gets what one without tokens gets."""
    pool, k, v, size = _filled([n, n], 64, 1, D, dtype, 16, seed=3)
    hidden = torch.zeros(2, n, dtype=torch.bool)
    hidden[0, :300], hidden[0, 400:411], hidden[1] = True, True, True
    table = pool.table.long()
    for b in range(2):
        j = hidden[b].nonzero()[:, 0]
        pool.cache.k_pages[table[b, j // 64].to(DEV), 0, (j % 64).to(DEV), 3] = -math.inf
    q = torch.randn((2, 1, 2, D), generator=torch.Generator().manual_seed(8)).to(dtype)
    q[..., 3] = 0.5
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, return_softmax_lse=True)
    check_status(DEV)
    seen = ~hidden[0]
    _check_decode(q[:1], out[:1], lse[:1], k[:1, seen], v[:1, seen], size[:1, seen], [int(seen.sum())], None,
                  True, 16)
    assert not out[1].any() and bool((lse[1] == math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("low", [-2.0 ** 20, -2.0 ** 28, -2.0 ** 33, -1e30])
@pytest.mark.parametrize("D,n", [(16, 512), (64, 500), (128, 512)])
def test_scores_far_below_the_others_weigh_nothing(D, n, low):
    """Keys that were masked by a large negative value, before and between ordinary ones."""
    pool, k, v, size = _filled([n], 64, 1, D, BF16, 16, seed=3)
    hidden = torch.zeros(n, dtype=torch.bool)
    hidden[:300], hidden[400:411] = True, True
    j = hidden.nonzero()[:, 0]
    pool.cache.k_pages[pool.table.long()[0, j // 64].to(DEV), 0, (j % 64).to(DEV), 3] = low
    q = torch.randn((1, 1, 2, D), generator=torch.Generator().manual_seed(8)).bfloat16()
    q[..., 3] = 0.5
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, return_softmax_lse=True)
    check_status(DEV)
    seen = ~hidden
    _check_decode(q, out, lse, k[:, seen], v[:, seen], size[:, seen], [int(seen.sum())], None, True, 16)


# ---------------------------------------------------------------- GPU: weights far below the largest
def _far(n, D, gap, bits, low, high, seed, order="even"):
    """One sequence of n tokens, one head: the scores of tokens 0, 16, 32 and 48 (each warp has one)
    are `gap` above the others' mean, which spread by about 1; values from `low` to `high`, those
    four tokens' all `low`.  `order`: 'even', or values that grow or shrink 1000-fold along the
    context."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((1, 1, 1, D), generator=g).half()
    k = torch.randn((1, n, 1, D), generator=g)
    k[0, :64:16, 0] = q[0, 0, 0].float() * (gap * math.sqrt(D) / float(q.double().square().sum()))
    v = low + (high - low) * torch.rand((1, n, 1, D), generator=g)
    v[0, :64:16] = low
    if order != "even":
        size = torch.logspace(-3, 0, n) if order == "growing" else torch.logspace(0, -3, n)
        v[0] = v[0] * size[:, None, None]
        v[0, :64:16] = low
    k, v = k.half(), v.half()
    pool = Pool([n], 64, 1, D, F16, bits)
    kv_cache_append(pool.cache, k.to(DEV), v.to(DEV), pool.table_dev, _ints([0]))
    if bits == 16:
        return pool, q, k.double(), v.double(), v.double().abs()
    kc, km, ks = so.four_bit(k)
    vc, vm, vs = so.four_bit(v)
    return pool, q, so.values(kc, km, ks), so.values(vc, vm, vs), so.values(vc, vm.abs(), vs)


def _check_far(pool, q, k, v, size, bits):
    """As many sequences of the same pages as CTAs run at once, so that each is one CTA's work.
    Held to relative errors alone.  A probability p, relative to a running maximum that is at
    most 2 (in log2) too low, is brought to 2^12 p and rounded to fp16: half a step of 2^-11, or
    2^-25 where it is subnormal, 2^-37 of p.  At 4 bits its product with the token's scale, taken
    relative to the power of two below the largest scale s, is rounded once more in the same way.
    With n tokens and a sum of at least 1 the subnormal part is below 3 n 2^-37 of the largest
    value (15 s, or |v|).  The rest as in the other tests of the attention."""
    n, D = k.shape[1], q.shape[3]
    B = 2 * torch.cuda.get_device_properties(DEV).multi_processor_count
    out, lse = flash_attn_decode(q.to(DEV).expand(B, -1, -1, -1), pool.cache, pool.table_dev.expand(B, -1),
                                 pool.lengths.expand(B), return_softmax_lse=True)
    check_status(DEV)
    ref, rl, mass, reach = so.decode(q[0, :, 0].double(), k[0, :, 0], v[0, :, 0], size[0, :, 0], [n], 1 / math.sqrt(D))
    e = (D + 8) * 2.0 ** -22 * reach[:, None]
    tol = 2.0 ** -11 * ref.abs() + ((1 if bits == 16 else 2) * 2.0 ** -11 + 2.0 ** -20 + 2 * e) * mass
    tol = tol + 3 * n * 2.0 ** -37 * size.max() + 2.0 ** -25  # (the output's own subnormals)
    off = (out[:, 0, 0].cpu().double() - ref).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), float((off[0].norm() / ref.norm())))
    assert bool(((lse[:, 0, 0].cpu().double() - rl).abs() <= 2.0 ** -20 * (1 + rl.abs()) + e[:, 0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,gap", [(64, 0.0), (9000, 12.0), (70000, 12.0), (70000, 18.0)])
@pytest.mark.parametrize("high", [1.0, 1000.0])
def test_many_small_weights_16_bit(n, gap, high):
    """One token far above the others, whose many small probabilities hold the output."""
    _check_far(*_far(n, 64, gap, 16, 0.0, high, 5), 16)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["even", "growing", "shrinking"])
@pytest.mark.parametrize("n,gap", [(64, 0.0), (9000, 12.0), (70000, 12.0), (70000, 18.0)])
@pytest.mark.parametrize("D,high", [(64, 1.0), (128, 0.003), (32, 3e-4), (64, 6e4)])
def test_many_small_weights_4_bit(D, high, n, gap, order):
    """The same over 4-bit values from 3e-4 to 6e4, whose scales meet those weights."""
    _check_far(*_far(n, D, gap, 4, 0.0, high, 5, order), 4)


@pytest.mark.gpu
def test_scales_that_are_not_seen_or_not_numbers():
    """Tokens behind the length with the largest scales, and a group of NaN before small values:
    the other groups of the row are what they are without them."""
    n, D = 300, 64
    pool, q, k, v, size = _far(n, D, 6.0, 4, 0.0, 0.003, 9)
    B = 3
    call = lambda m: flash_attn_decode(q.to(DEV).expand(B, -1, -1, -1), pool.cache, pool.table_dev.expand(B, -1),  # noqa: E731
                                       _ints([m] * B))
    want = call(250)
    big = torch.zeros((1, 50, 1, D), dtype=F16, device=DEV)
    big[..., ::2] = 6e4
    kv_cache_append(pool.cache, big, big, pool.table_dev, _ints([250]))
    assert torch.equal(call(250), want)
    bad = v[:, :1].half().to(DEV)
    bad[..., 3] = math.nan
    kv_cache_append(pool.cache, k[:, :1].half().to(DEV), bad, pool.table_dev, _ints([0]))
    kv_cache_append(pool.cache, k[:, :1].half().to(DEV), torch.where(bad.isnan(), 0.0, bad), pool.table_dev, _ints([1]))
    out = call(250)
    check_status(DEV)
    assert bool(out[..., :32].isnan().all()) and bool(out[..., 32:].isfinite().all())


# ---------------------------------------------------------------- GPU: page ids
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("wrong", [-2, -3])
def test_every_bad_page_id_is_reported(bits, wrong):
    """(-2 was the kernel's own mark of 'no block here'.)"""
    pool, k, v, size = _filled([40, 40], 16, 1, 64, F16, bits, seed=6)
    q = torch.randn((2, 1, 2, 64), generator=torch.Generator().manual_seed(8)).half()
    table = pool.table.clone()
    table[1, 1] = wrong
    check_status(DEV)
    out = flash_attn_decode(q.to(DEV), pool.cache, table.to(DEV), pool.lengths)
    with pytest.raises(RuntimeError, match="status 4"):
        check_status(DEV)
    keep = torch.cat([torch.arange(16), torch.arange(32, 40)])
    ks, vs, ss = (t.clone() for t in (k, v, size))
    for t, src in ((ks, k), (vs, v), (ss, size)):
        t[1, :24] = src[1, keep]
    _check_decode(q, out, None, ks, vs, ss, [40, 24], [39, 39], True, bits)


# ---------------------------------------------------------------- GPU: the largest 4-bit values
@pytest.mark.gpu
@pytest.mark.parametrize("top", [65504.0, 65472.0, math.inf])
@pytest.mark.parametrize("bottom", [0.0, -65504.0, 60000.0, -math.inf])
def test_the_largest_values_stay_finite_in_fp16(top, bottom):
    """The scale is rounded up, so minimum + 15 scale passes 65504 (0 + 15 x 4368, -65504 + 15 x
    8736): what is read back, and the attention's output, is 65504 at most, not infinite."""
    x = torch.linspace(0.0, 1.0, 64).half().view(1, 1, 1, 64).repeat(1, 2, 1, 1)
    x[..., 7], x[..., 9] = top, bottom
    x[0, 1, 0, 40] = math.nan
    pool = Pool([2], 16, 1, 64, F16, 4)
    kv_cache_append(pool.cache, torch.zeros_like(x).to(DEV), x.to(DEV), pool.table_dev, _ints([0]))
    _, got = kv_cache_read(pool.cache, pool.table_dev, pool.lengths, 2)
    q = torch.ones((1, 1, 1, 64), dtype=F16, device=DEV)
    out = flash_attn_decode(q, pool.cache, pool.table_dev, _ints([1]))
    check_status(DEV)
    want = x[0, 0, 0].double().clamp(-65504, 65504)
    step = (want[:32].max() - want[:32].min()) / 15
    for t in (got[0, 0, 0], out[0, 0, 0]):
        t = t.cpu().double()
        assert bool(t.isfinite().all())
        # half a step, the step's own rounding up (2^-10), 15 times, and the result's rounding
        assert bool(((t[:32] - want[:32]).abs() <= step * (0.5 + 16 * 2.0 ** -10) + 2.0 ** -11 * 65504).all())
        assert t[7] == 65504 or top < 65504
    assert bool(got[0, 1, 0, 32:].isnan().all()) and bool(got[0, 1, 0, :32].isfinite().all())


# ---------------------------------------------------------------- scales and sizes of q
@pytest.mark.gpu
def test_scales_that_are_not_finite_are_refused():
    pool, *_ = _filled([5], 16, 1, 64, F16, 16)
    q = torch.zeros((1, 1, 2, 64), dtype=F16, device=DEV)
    for scale in (math.nan, math.inf, -math.inf):
        with pytest.raises(AssertionError, match="finite"):
            flash_attn_decode(q, pool.cache, pool.table_dev, pool.lengths, sm_scale=scale)


def test_c_abi_refuses_scales_that_are_not_finite():
    import ctypes
    lib = _lib.load()
    c = ctypes.byref(_lib.KvCache(4096, 4096, 2, 64, 2, 64, 0, 16))
    for scale in (math.nan, math.inf, -math.inf):
        assert lib.fa_sm100_decode(c, 256, 256, None, 256, 1, 256, None, 256, 0, 1, 1, 4, scale, 1, None,
                                   None) == _lib.FA_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("power", [-100, 60, 100, 112, 116, 122])
def test_large_queries_and_small_scales(bits, power):
    """q times 2^power with sm_scale times 2^-power is the same attention, bit for bit: bf16 q may be
    as large as 2^127, and a scale as small as 2^-125."""
    pool, k, v, size = _filled([300, 77], 32, 1, 64, BF16, bits, seed=15)
    q = torch.randn((2, 3, 4, 64), generator=torch.Generator().manual_seed(8)).bfloat16().to(DEV)
    call = lambda x, scale: flash_attn_decode(x, pool.cache, pool.table_dev, pool.lengths, sm_scale=scale,  # noqa: E731
                                              return_softmax_lse=True)
    want = call(q, 0.125)
    out = call(q * 2.0 ** power, 0.125 * 2.0 ** -power)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("power", [16, 22, 24, 27, 31, 40, 80, 118])
@pytest.mark.parametrize("n", [300, 3000])
def test_scores_beyond_the_rest_pick_their_token(bits, power, n):
    """q of 2^power at the usual scale: the largest score takes all the weight, next to a row of
    ordinary scores.  (The gap to the second one is over 20 after any halving of the scores, and
    over what the sums of products are off.)"""
    pool, k, v, size = _filled([n], 32, 1, 64, BF16, bits, seed=16)
    q = torch.randn((1, 1, 2, 64), generator=torch.Generator().manual_seed(8)).bfloat16()
    q[:, :, 1] *= 2.0 ** power
    out, lse = flash_attn_decode(q.to(DEV), pool.cache, pool.table_dev, pool.lengths, return_softmax_lse=True)
    score = (k[0, :, 0] @ q[0, 0, 1].double()) / 8
    two, best = score.topk(2)
    reach = float((k[0, :, 0].abs() @ q[0, 0, 1].double().abs()).max()) / 8
    assert float(two[0] - two[1]) > max(40.0, 40 * 2.0 ** -23 * float(two[0]), 4 * 72 * 2.0 ** -22 * reach)
    ref, most = v[0, int(best[0]), 0], size[0, int(best[0]), 0]
    assert bool(((out[0, 0, 1].cpu().double() - ref).abs() <= 2 * 2.0 ** -8 * most + 2.0 ** -25).all())
    assert abs(float(lse[0, 1, 0]) - float(two[0])) <= 2.0 ** -20 * abs(float(two[0])) + 72 * 2.0 ** -22 * reach
    _check_decode(q[:, :, :1], out[:, :, :1], lse[:, :1], k, v, size, [n], None, True, bits)


# ---------------------------------------------------------------- chunks, tracing, threads
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("how", ["decode", "one at a time"])
def test_ragged_chunks(bits, how):
    """Prompts of different lengths in two chunks of different counts: every row that is not padding
    is the attention over its own sequence up to its own position."""
    B, S, H, Hkv, D = 4, 40, 6, 2, 64
    counts = [[40, 17, 1, 33], [30, 40, 5, 0]]
    total = [sum(c) for c in zip(*counts)]
    g = torch.Generator().manual_seed(17)
    mk = lambda h: torch.randn((B, 2 * S, h, D), generator=g).half()  # noqa: E731
    q, k, v = mk(H), mk(Hkv), mk(Hkv)
    pool = Pool(total, 16, Hkv, D, F16, bits)
    starts, got = [0] * B, {}
    for chunk in range(2):
        n = counts[chunk]
        take = lambda x: torch.stack([torch.cat([x[b, starts[b]:starts[b] + n[b]], 9 * torch.ones_like(x[b, n[b]:S])])  # noqa: E731
                                      for b in range(B)]).to(DEV)
        qc = kv_cache_append(pool.cache, take(k), take(v), pool.table_dev, _ints(starts), _ints(n), q=take(q))
        ends = [a + m for a, m in zip(starts, n)]
        if how == "decode":
            out = flash_attn_decode(qc, pool.cache, pool.table_dev, _ints(ends), starts=_ints(starts))
        for b in range(B):
            if how != "decode":
                ka, va = kv_cache_read(pool.cache, pool.table_dev[b:b + 1], _ints(ends[b:b + 1]), ends[b])
                out = {b: flash_attn(qc[b:b + 1, :n[b]], ka, va, causal=True)[0]}
            for i in range(n[b]):
                got[b, starts[b] + i] = out[b][i].cpu()
        starts = ends
    check_status(DEV)
    if bits == 4:
        kc, km, ks = so.four_bit(k)
        vc, vm, vs = so.four_bit(v)
        k, v, size = so.values(kc, km, ks), so.values(vc, vm, vs), so.values(vc, vm.abs(), vs)
    else:
        k, v, size = k.double(), v.double(), v.double().abs()
    if how == "decode":
        rows = torch.stack([torch.stack([got.get((b, i), torch.zeros(H, D).half()) for i in range(2 * S)])
                            for b in range(B)])
        for b in range(B):
            m = slice(b, b + 1), slice(0, total[b])
            _check_decode(q[m], rows[m], None, k[b:b + 1], v[b:b + 1], size[b:b + 1], [total[b]], None, True, bits)
        return
    for (b, i), row in got.items():
        for h in range(H):
            ref, _, mass, reach = so.decode(q[b, i, h][None].double(), k[b, :, h // 3], v[b, :, h // 3],
                                            size[b, :, h // 3], [i + 1], 1 / 8)
            # as in test_serving_run without the rounding of a rotated q: p and out once, k and v read
            # back in fp16 once (2^-11 of a score's reach, and of the values)
            tol = 2.0 ** -11 * ref.abs() + (2.0 ** -9 + 2.0 ** -10 * reach[:, None]) * mass + 2.0 ** -12
            assert bool(((row[h].double() - ref[0]).abs() <= tol[0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
def test_a_traced_step(bits):
    """torch.compile takes append, attention and read as one graph."""
    pool, *_ = _filled([20, 33], 16, 2, 64, F16, bits, seed=2, width=4)
    c, table = pool.cache, pool.table_dev.clamp(min=0)
    rot = Rotary.build(64, device=DEV)
    g = torch.Generator().manual_seed(3)
    mk = lambda h: torch.randn((2, 1, h, 64), generator=g).half().to(DEV)  # noqa: E731
    q, k, v, n = mk(8), mk(2), mk(2), _ints([19, 32])

    def step(q, k, v, n):
        qr = kv_cache_append(c, k, v, table, n, q=q, rotary=rot)
        out, lse = flash_attn_decode(qr, c, table, n + 1, return_softmax_lse=True)
        return (out * 2, lse, *kv_cache_read(c, table, n + 1, 40))

    before = [t.clone() for t in (c.k_pages, c.v_pages) if t is not None]
    want = step(q, k, v, n)
    after = [t.clone() for t in (c.k_pages, c.v_pages) if t is not None]
    for t, was in zip((c.k_pages, c.v_pages), before):
        t.copy_(was)
    torch._dynamo.reset()
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, n)
    check_status(DEV)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for t, is_now in zip((c.k_pages, c.v_pages), after):
        assert torch.equal(t.view(torch.uint8), is_now.view(torch.uint8))


@pytest.mark.gpu
def test_calls_from_two_threads():
    """Two host threads, each with a stream and a cache of its own."""
    import threading
    pools = [_filled([700, 90], 32, 2, 64, F16, bits, seed=31)[0] for bits in (16, 4)]
    q = torch.randn((2, 1, 8, 64), generator=torch.Generator().manual_seed(8)).half().to(DEV)
    call = lambda p: flash_attn_decode(q, p.cache, p.table_dev, p.lengths)  # noqa: E731
    want = [call(p) for p in pools]
    torch.cuda.synchronize(DEV)
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            got = [call(pools[i]) for _ in range(50)]
            torch.cuda.current_stream(DEV).synchronize()
            wrong.extend(i for o in got if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    check_status(DEV)
