"""Rotary positions (flash_attn_volta_b200.rotary) against the float64 oracle.

Tolerance of a rotated value y = M (x1 c - x2 s): its rounding to the element
type (half a step: eps/2 of |y|, or 2^-25 where fp16 is subnormal), and the fp32
arithmetic before it.  cos and sin are within 2^-22 of the angle's (2 ulp of
sincospif below 1, and the added first-order term), the two products and the
sum each within 2^-24 of their size: 2^-21 (|x1| + |x2|) M covers them.
"""
import math

import pytest
import torch

from flash_attn_volta_b200 import flash_attn, ops
from flash_attn_volta_b200.rotary import Rotary, rotary_embed, rotary_embed_qk
from oracle.serving_oracle import rotate

DEV = torch.device("cuda", 0)
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _freq(R, base=10000.0):
    return base ** (-2.0 * torch.arange(R // 2, dtype=torch.float64) / R)


def _check(y, x, pos, freq, inter, mag=1.0, inverse=False):
    ref = rotate(x.cpu(), pos, freq, inter, mag, inverse)
    R = 2 * len(freq)
    size = x.cpu().double().abs()
    both = size.clone()
    lo = slice(0, R, 2) if inter else slice(0, R // 2)
    hi = slice(1, R, 2) if inter else slice(R // 2, R)
    both[..., lo] = both[..., hi] = size[..., lo] + size[..., hi]
    tol = HALF[x.dtype] * ref.abs() + 2.0 ** -25 + 2.0 ** -21 * mag * both
    assert y.dtype == x.dtype and y.shape == x.shape
    bad = (y.cpu().double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off"
    assert torch.equal(y.cpu()[..., R:], x.cpu()[..., R:])


# ---------------------------------------------------------------- CPU
def test_scalings():
    r = Rotary.build(64, device="cpu")
    assert r.dim == 64 and r.magnitude == 1.0 and torch.equal(r.inv_freq, _freq(64))
    assert torch.allclose(Rotary.build(64, scaling="linear", factor=8.0, device="cpu").inv_freq,
                          _freq(64) / 8.0)
    ntk = Rotary.build(64, scaling="ntk", factor=8.0, device="cpu").inv_freq
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1] * 8.0), float(_freq(64)[-1]), rel_tol=1e-12)
    y = Rotary.build(64, scaling="yarn", factor=8.0, trained_length=4096, device="cpu")
    turns = 4096 * _freq(64) / (2 * math.pi)
    assert torch.equal(y.inv_freq[turns >= 32], _freq(64)[turns >= 32])
    assert torch.equal(y.inv_freq[turns <= 1], _freq(64)[turns <= 1] / 8.0)
    assert bool((y.inv_freq[1:] < y.inv_freq[:-1]).all())
    assert y.magnitude == 0.1 * math.log(8.0) + 1.0


def test_refusals():
    f = torch.ones(4, dtype=torch.float64)
    x = torch.zeros(1, 2, 1, 16, dtype=torch.float16)
    for bad in (lambda: Rotary(torch.ones(4, dtype=torch.int64)), lambda: Rotary(torch.ones(0)),
                lambda: Rotary(torch.ones(2, 2)), lambda: Rotary.build(7),
                lambda: Rotary.build(64, scaling="cubic"), lambda: Rotary.build(64, factor=0.5),
                lambda: Rotary.build(64, scaling="yarn", factor=4.0, device="cpu"),
                lambda: rotary_embed(x, Rotary(f)),  # not on CUDA
                lambda: rotary_embed_qk(x, x, Rotary(f)),
                lambda: flash_attn(x, x, x, positions=torch.arange(2))):
        with pytest.raises(AssertionError):
            bad()


def test_c_abi_refusals():
    import ctypes

    from flash_attn_volta_b200 import _lib
    lib = _lib.load()
    h = _lib.Heads(256, 256, 16, 16, 16, 1)
    ok = dict(q=ctypes.byref(h), k=None, f=256, R=16, inter=0, B=1, S=1, D=16, dt=0)

    def call(**kw):
        a = {**ok, **kw}
        return lib.fa_sm100_rotary(a["q"], a["k"], a["f"], a["R"], a["inter"], 1.0, 0, None, 0, 0, 0,
                                   a["B"], a["S"], a["D"], a["dt"], None)

    odd = _lib.Heads(258, 256, 16, 16, 16, 1)  # a pair that is not 4-byte aligned
    for kw in (dict(q=None), dict(f=None), dict(f=260), dict(R=0), dict(R=15), dict(R=18),
               dict(B=0), dict(S=0), dict(D=15, R=14), dict(dt=5),
               dict(q=ctypes.byref(_lib.Heads(None, 256, 0, 0, 0, 1))),
               dict(q=ctypes.byref(_lib.Heads(256, 256, 0, 0, 0, 0))),
               dict(k=ctypes.byref(_lib.Heads(256, None, 0, 0, 0, 1))),
               dict(q=ctypes.byref(odd), inter=1)):
        assert call(**kw) == _lib.FA_ERR_ARG, kw


def test_fake_shapes():
    ops.load()
    q = torch.empty((2, 5, 4, 64), dtype=torch.float16, device="meta")
    k = torch.empty((2, 5, 2, 64), dtype=torch.float16, device="meta")
    f = torch.empty(32, dtype=torch.float64, device="meta")
    a, b = torch.ops.fav.rotary_qk(q, k, f, None, 0, False, 1.0, False)
    assert a.shape == q.shape and b.shape == k.shape
    with pytest.raises(RuntimeError):
        torch.ops.fav.rotary(q, torch.empty(33, dtype=torch.float64, device="meta"), None, 0, False,
                             1.0, False)
    with pytest.raises(RuntimeError):
        torch.ops.fav.rotary(q, f, torch.empty(4, dtype=torch.int64, device="meta"), 0, False, 1.0,
                             False)


# ---------------------------------------------------------------- GPU
CASES = [  # B, S, H, D, R, interleaved
    (1, 1, 1, 2, 2, False), (1, 1, 1, 2, 2, True), (2, 7, 3, 16, 16, False), (2, 7, 3, 16, 8, True),
    (3, 5, 5, 80, 20, False), (3, 5, 5, 80, 40, True), (1, 33, 4, 64, 64, False),
    (1, 33, 4, 64, 32, True), (2, 17, 32, 128, 128, False), (2, 17, 32, 128, 128, True),
    (1, 3, 2, 256, 96, False), (1, 3, 200, 128, 64, False), (5, 129, 1, 10, 6, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,D,R,inter", CASES)
def test_matches_oracle(B, S, H, D, R, inter, dtype):
    g = torch.Generator().manual_seed(B * 1000 + S)
    q = torch.randn((B, S, H, D), generator=g).to(dtype)
    k = torch.randn((B, S, max(1, H // 2), D), generator=g).to(dtype)
    pos = torch.randint(0, 5000, (B, S), generator=g)
    rot = Rotary(_freq(R).to(DEV), inter, 1.25)
    qo, ko = rotary_embed_qk(q.to(DEV), k.to(DEV), rot, pos.to(DEV))
    _check(qo, q, pos, _freq(R), inter, 1.25)
    _check(ko, k, pos, _freq(R), inter, 1.25)
    # one tensor, default and shared positions, 32-bit positions
    _check(rotary_embed(q.to(DEV), rot), q, torch.arange(S), _freq(R), inter, 1.25)
    _check(rotary_embed(q.to(DEV), rot, first=-3), q, torch.arange(S) - 3, _freq(R), inter, 1.25)
    _check(rotary_embed(q.to(DEV), rot, pos[0].int().to(DEV)), q, pos[0], _freq(R), inter, 1.25)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,Hkv,D,R,inter,dtype", [
    (1, 9001, 24, 8, 64, 64, False, torch.float16), (2, 5003, 32, 1, 80, 40, True, torch.bfloat16),
    (3, 3001, 20, 4, 128, 32, False, torch.bfloat16), (700, 21, 9, 3, 64, 64, True, torch.float16),
    (1, 2500, 50, 7, 96, 12, True, torch.float16), (1, 4001, 33, 3, 40, 20, False, torch.float16)])
def test_many_tokens(B, S, H, Hkv, D, R, inter, dtype):
    """Enough tokens for each thread to stream several rounds; odd counts, and rows
    that are no multiple of the threads."""
    g = torch.Generator(device=DEV).manual_seed(S)
    q = torch.randn((B, S, H, D), generator=g, device=DEV).to(dtype)
    k = torch.randn((B, S, Hkv, D), generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, 30000, (B, 1), generator=g, device=DEV) + torch.arange(S, device=DEV)
    qo, ko = rotary_embed_qk(q, k, Rotary(_freq(R).to(DEV), inter), pos)
    part = slice(0, None, max(1, B // 3)), slice(0, None, 7)
    _check(qo[part], q[part], pos[part].cpu(), _freq(R), inter)
    _check(ko[part], k[part], pos[part].cpu(), _freq(R), inter)
    # every other row is what a call with fewer tokens gives
    for b in (0, B - 1):
        at = slice(S // 2, S // 2 + 5)
        few = rotary_embed_qk(q[b:b + 1, at], k[b:b + 1, at], Rotary(_freq(R).to(DEV), inter), pos[b:b + 1, at])
        assert torch.equal(few[0], qo[b:b + 1, at]) and torch.equal(few[1], ko[b:b + 1, at])


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
def test_more_than_2_31_elements(inter):
    S = 540_000  # x 32 heads of 128: 2.2e9 elements
    x = torch.zeros((1, S, 32, 128), dtype=torch.bfloat16, device=DEV)
    at = [0, 1, 262_143, 262_144, 524_287, 524_288, S - 1]
    x[:, at] = torch.randn((1, len(at), 32, 128), generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    y = rotary_embed(x, Rotary(_freq(128).to(DEV), inter))
    _check(y[:, at], x[:, at], torch.tensor(at), _freq(128), inter)
    # the same rows, every other head of a tensor whose strides pass 31 bits within a call
    z = rotary_embed(x.transpose(0, 1)[at, :, ::2].transpose(0, 1), Rotary(_freq(128).to(DEV), inter),
                     torch.tensor(at, device=DEV))
    assert torch.equal(z, y[:, at][:, :, ::2])


@pytest.mark.gpu
def test_far_positions():
    """Angles of 10^6 and 2^40 rad: an fp32 product would be off by 0.1 rad and more."""
    x = torch.randn((1, 4, 2, 64), generator=torch.Generator().manual_seed(3)).half()
    pos = torch.tensor([0, 1_000_003, 16_777_217, 2 ** 40 + 1])
    _check(rotary_embed(x.to(DEV), Rotary(_freq(64).to(DEV)), pos.to(DEV))[:, :3], x[:, :3], pos[:3],
           _freq(64), False)
    y = rotary_embed(x.to(DEV), Rotary(_freq(64).to(DEV)), pos.to(DEV))
    ref = rotate(x, pos, _freq(64))
    # 2^40 rad in 64 bits is itself rounded to 2^-13 rad
    assert float((y.cpu().double() - ref).abs().max()) <= 2.0 ** -11 * 6 + 2.0 ** -12 * 8


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("how", ["fused_qkv", "transposed", "odd_offset", "odd_rows", "expanded",
                                 "last_dim"])
def test_strides(how, inter):
    g = torch.Generator().manual_seed(7)
    B, S, H, D = 2, 9, 4, 64
    if how == "fused_qkv":
        x = torch.randn((B, S, 3 * H, D), generator=g).half().to(DEV)[:, :, H:2 * H]
    elif how == "transposed":
        x = torch.randn((B, H, S, D), generator=g).half().to(DEV).transpose(1, 2)
    elif how == "odd_offset":
        x = torch.randn(B * S * H * D + 1, generator=g).half().to(DEV)[1:].view(B, S, H, D)
    elif how == "odd_rows":
        x = torch.randn((B, S, H, D + 1), generator=g).half().to(DEV)[..., :D]
    elif how == "expanded":
        x = torch.randn((B, S, 1, D), generator=g).half().to(DEV).expand(B, S, H, D)
    else:
        x = torch.randn((B, S, D, H), generator=g).half().to(DEV).transpose(2, 3)
    y = rotary_embed(x, Rotary(_freq(D).to(DEV), inter))
    assert y.is_contiguous()
    _check(y, x, torch.arange(S), _freq(D), inter)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, f = torch.zeros((2, 3, 4, 64), dtype=torch.float16, device=DEV), _freq(64).to(DEV)
    r, pos = Rotary(f), torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    for bad in (lambda: rotary_embed(x.float(), r), lambda: rotary_embed(x[0], r),
                lambda: rotary_embed(x[..., :32], r), lambda: rotary_embed(x[..., :63], r),
                lambda: rotary_embed(x, Rotary(f.cpu())), lambda: rotary_embed(x.cpu(), r),
                lambda: rotary_embed(x, r, pos.float()), lambda: rotary_embed(x, r, pos[:, :2]),
                lambda: rotary_embed(x, r, pos.cpu()), lambda: rotary_embed_qk(x, x[:, :2], r),
                lambda: rotary_embed_qk(x, x.bfloat16(), r), lambda: rotary_embed_qk(x, x.cpu(), r)):
        with pytest.raises(AssertionError):
            bad()
    torch.cuda.synchronize(DEV)


@pytest.mark.gpu
def test_empty():
    rot = Rotary(_freq(64).to(DEV))
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64), (2, 3, 0, 64)):
        x = torch.empty(shape, dtype=torch.float16, device=DEV)
        assert rotary_embed(x, rot).shape == x.shape
    q, k = rotary_embed_qk(torch.empty((1, 2, 0, 64), dtype=torch.float16, device=DEV),
                           torch.ones((1, 2, 1, 64), dtype=torch.float16, device=DEV), rot)
    _check(k, torch.ones((1, 2, 1, 64), dtype=torch.float16), torch.arange(2), _freq(64), False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,inter", [(64, False), (32, True)])
def test_gradients(R, inter, dtype):
    """dx is dy rotated by -a: against the formula, and <dy, R(x)> against
    differences (the map is linear, so they are exact up to rounding)."""
    g = torch.Generator().manual_seed(11)
    mk = lambda h: torch.randn((2, 21, h, 64), generator=g).to(dtype)  # noqa: E731
    q, k, dq, dk, step = mk(6), mk(3), mk(6), mk(3), mk(6)
    pos = torch.randint(0, 9000, (2, 21), generator=g)
    rot = Rotary(_freq(R).to(DEV), inter, 1.1)
    ql, kl = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    qo, ko = rotary_embed_qk(ql, kl, rot, pos.to(DEV))
    gq, gk = torch.autograd.grad([qo, ko], [ql, kl], [dq.to(DEV), dk.to(DEV)])
    _check(gq, dq, pos, _freq(R), inter, 1.1, inverse=True)
    _check(gk, dk, pos, _freq(R), inter, 1.1, inverse=True)
    # only one of the two, and a strided gradient
    qo, ko = rotary_embed_qk(ql, kl, rot, pos.to(DEV))
    (gk2,) = torch.autograd.grad([ko], [kl], [dk.to(DEV)])
    assert torch.equal(gk2, gk)
    y = rotary_embed(ql, rot, pos.to(DEV))
    wide = torch.zeros((2, 21, 6, 128), dtype=dtype, device=DEV)
    wide[..., :64] = dq.to(DEV)
    (gq2,) = torch.autograd.grad([y], [ql], [wide[..., :64]])
    assert torch.equal(gq2, gq)
    # difference quotient along `step`
    diff = (rotate(q.double() + 0.5 * step.double(), pos, _freq(R), inter, 1.1) -
            rotate(q.double() - 0.5 * step.double(), pos, _freq(R), inter, 1.1))
    lhs = float((diff * dq.double()).sum())
    rhs = float((gq.cpu().double() * step.double()).sum())
    bound = float((gq.cpu().double().abs() * step.double().abs()).sum()) * 2 * HALF[dtype]
    assert abs(lhs - rhs) <= bound


@pytest.mark.gpu
def test_double_backward_and_no_grad():
    x = torch.randn((1, 4, 2, 32), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    rot = Rotary(_freq(32).to(DEV))
    xl = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(rotary_embed(xl, rot).float().square().sum(), xl, create_graph=True)
    assert gx.requires_grad  # the gradient goes through the same operator
    with torch.no_grad():
        assert not rotary_embed(xl, rot).requires_grad
    assert not rotary_embed_qk(x, x, rot)[0].requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("Nk,inter", [(96, False), (160, True)])
def test_flash_attn_with_rotary(Nk, inter):
    """flash_attn(rotary=) is the attention of the rotated q and k, with their
    gradients, bit for bit."""
    g = torch.Generator().manual_seed(5)
    mk = lambda n, h: torch.randn((2, n, h, 64), generator=g).half().to(DEV).requires_grad_()  # noqa: E731
    q, k, v = mk(96, 4), mk(Nk, 2), mk(Nk, 2)
    do = torch.randn((2, 96, 4, 64), generator=g).half().to(DEV)
    rot = Rotary(_freq(64).to(DEV), inter)
    for pos in (None, torch.arange(Nk, device=DEV) * 3):
        if pos is None:
            qr, kr = rotary_embed(q, rot, first=Nk - 96), rotary_embed(k, rot)
        else:
            qr, kr = rotary_embed(q, rot, pos[Nk - 96:]), rotary_embed(k, rot, pos)
        ref = flash_attn(qr, kr, v, causal=True, deterministic=True)
        out = flash_attn(q, k, v, causal=True, deterministic=True, rotary=rot, positions=pos)
        assert torch.equal(out, ref)
        for a, b in zip(torch.autograd.grad(out, [q, k, v], do),
                        torch.autograd.grad(ref, [q, k, v], do)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_graph_stream_and_compile():
    x = [torch.randn((2, 50, 4, 64), generator=torch.Generator().manual_seed(i)).half().to(DEV)
         for i in range(2)]
    rot = Rotary(_freq(64).to(DEV))
    want = [rotary_embed(t, rot) for t in x]
    static = x[0].clone()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        got = rotary_embed(static, rot)
    torch.cuda.current_stream(DEV).wait_stream(side)
    assert torch.equal(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_embed(static, rot)
    for t, w in zip(x[::-1], want[::-1]):
        static.copy_(t)
        graph.replay()
        assert torch.equal(out, w)
    torch._dynamo.reset()
    f = torch.compile(lambda a: rotary_embed(a, rot) * 2, fullgraph=True, backend="aot_eager")
    a, b = x[0].clone().requires_grad_(), x[0].clone().requires_grad_()
    (f(a).float().sum()).backward()
    ((rotary_embed(b, rot) * 2).float().sum()).backward()
    assert torch.equal(f(x[0]), want[0] * 2) and torch.equal(a.grad, b.grad)


@pytest.mark.gpu
def test_opcheck():
    ops.load()
    g = torch.Generator().manual_seed(0)
    q = torch.randn((1, 6, 4, 32), generator=g).half().to(DEV).requires_grad_()
    k = torch.randn((1, 6, 2, 32), generator=g).half().to(DEV).requires_grad_()
    f = _freq(32).to(DEV)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.fav.rotary, (q, f, None, 0, False, 1.0, False), test_utils=tests)
    torch.library.opcheck(torch.ops.fav.rotary_qk, (q, k, f, None, 0, True, 1.0, False),
                          test_utils=tests)
