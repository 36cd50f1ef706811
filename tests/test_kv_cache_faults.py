"""The paged key/value cache where it can go wrong: waits that run out, infinities
that a row sees, values far below or above one, bad page ids, derivatives."""
import math

import pytest
import torch

from flash_attn_volta_b200 import _lib, check_status
from flash_attn_volta_b200.kv_cache import flash_attn_decode
from tests.test_kv_cache import BF16, DEV, F16, _check_decode, _filled


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
