"""ring_flash_attn(rotary=): each rank rotates its zigzag shard at the positions
its rows have in the whole sequence.  CPU ranks (gloo) with the oracle in place
of the kernels; on one GPU the ring of one rank is the whole sequence."""
import math

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from flash_attn_volta_b200 import flash_attn, ring
from flash_attn_volta_b200.rotary import Rotary, rotary_embed_qk
from oracle.attention_oracle import attention_fwd
from oracle.serving_oracle import rotate
from tests.helpers import make_inputs
from tests.test_ring_cpu import _free_port, _oracle_block_bwd, _oracle_block_fwd

FREQ = 10000.0 ** (-2.0 * torch.arange(8, dtype=torch.float64) / 16)


def test_positions_are_the_shards_rows():
    for world in (1, 2, 3):
        at = torch.arange(24)[None]
        for rank in range(world):
            assert torch.equal(ring.zigzag_positions(rank, world, 24 // world),
                               ring.zigzag_shard(at, rank, world)[0])


def _oracle_rotate(q, k, rotary, positions):
    f = rotary.inv_freq
    return rotate(q, positions, f).float(), rotate(k, positions, f).float()


def _worker(rank, world, port, out):
    import os
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        ring.block_fwd, ring.block_bwd, ring.rotate = _oracle_block_fwd, _oracle_block_bwd, _oracle_rotate
        q, k, v = [t.float() for t in make_inputs(1, 32, 2, 16, seed=5, n=3)]
        q, k, v = (ring.zigzag_shard(t, rank, world).requires_grad_() for t in (q, k, v))
        o = ring.ring_flash_attn(q, k, v, causal=True, rotary=Rotary(FREQ))
        o.square().sum().backward()
        out.put((rank, o.detach(), q.grad, k.grad))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_two_ranks_match_the_whole_sequence():
    ctx = mp.get_context("spawn")
    out, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, out)) for r in range(2)]
    for p in procs:
        p.start()
    got = {}
    for _ in procs:
        rank, *ts = out.get(timeout=120)
        got[rank] = [t.clone() for t in ts]
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    q, k, v = [t.double().requires_grad_() for t in make_inputs(1, 32, 2, 16, seed=5, n=3)]
    o, _ = attention_fwd(rotate(q, torch.arange(32), FREQ), rotate(k, torch.arange(32), FREQ), v, True,
                         1 / math.sqrt(16), dtype=torch.float64)
    o.square().sum().backward()
    for i, ref in enumerate((o.detach(), q.grad, k.grad)):
        whole = ring.zigzag_unshard([got[0][i], got[1][i]])
        # fp32 sums of at most 32 keys and 16 dims, values below 10
        assert float((whole.double() - ref).abs().max()) <= 64 * 2.0 ** -24 * 100


@pytest.mark.gpu
def test_one_rank_is_flash_attn_of_rotated_tensors():
    dev = torch.device("cuda", 0)
    q, k, v = (t.to(dev).requires_grad_() for t in make_inputs(1, 256, 2, 64, seed=6, n=3))
    rot = Rotary.build(64, device=dev)
    o = ring.ring_flash_attn(q, k, v, causal=True, rotary=rot)
    ref = ring.ring_flash_attn(*rotary_embed_qk(q, k, rot), v, causal=True)
    assert torch.equal(o, ref)
    whole = flash_attn(q, k, v, causal=True, rotary=rot)
    # the ring rounds two partial results to fp16 and merges them: 2 half steps of values below 4
    assert float((o - whole).abs().max().detach()) <= 2 * 4 * 2.0 ** -10
    (g,) = torch.autograd.grad(o.float().square().sum(), q)
    assert bool(g.isfinite().all()) and bool(g.any())
