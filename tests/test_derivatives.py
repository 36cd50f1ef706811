"""Derivatives that the rotary and cache operators do not compute are refused, never
dropped: forward-mode tangents, gradients of frequencies and of cache pages.  On meta
tensors (the checks stand above every device), and on the GPU through the module."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from flash_attn_volta_b200 import flash_attn, ops
from flash_attn_volta_b200.kv_cache import PagedKVCache, flash_attn_decode, kv_cache_append
from flash_attn_volta_b200.rotary import Rotary, rotary_embed, rotary_embed_qk

F16 = torch.float16


def _operators(dev, grad=None):
    """name -> (call, its floating tensors); `grad`: the tensor that requires a gradient."""
    ops.load()
    z = lambda *s, t=F16: torch.zeros(s, dtype=t, device=dev)  # noqa: E731
    ints, table = torch.ones(2, dtype=torch.int32, device=dev), torch.zeros((2, 1), dtype=torch.int32, device=dev)
    table[1:] = 1
    x = {"q": z(2, 1, 4, 64), "k": z(2, 1, 2, 64), "v": z(2, 1, 2, 64), "f": z(32, t=torch.float64),
         "kp": z(9, 2, 32, 64), "vp": z(9, 2, 32, 64)}
    fav = torch.ops.fav
    return x, {
        "rotary": (lambda: fav.rotary(x["q"], x["f"], None, 0, False, 1.0, False), "qf"),
        "rotary_qk": (lambda: fav.rotary_qk(x["q"], x["k"], x["f"], None, 0, False, 1.0, False), "qkf"),
        "kv_append": (lambda: fav.kv_append(x["kp"], x["vp"], x["k"], x["v"], x["q"], table, ints, None, x["f"],
                                            False, 1.0), ("kp", "vp", "k", "v", "q", "f")),
        "kv_read": (lambda: fav.kv_read(x["kp"], x["vp"], F16, table, ints, 4), ("kp", "vp")),
        "decode": (lambda: fav.decode(x["q"], x["kp"], x["vp"], table, ints, None, True, 0.1), ("q", "kp", "vp")),
        "decode_lse": (lambda: fav.decode_lse(x["q"], x["kp"], x["vp"], table, ints, None, True, 0.1),
                       ("q", "kp", "vp")),
    }


NAMES = ["rotary", "rotary_qk", "kv_append", "kv_read", "decode", "decode_lse"]


def _refusals(dev, name):
    x, calls = _operators(dev)
    call, takes = calls[name]
    call()
    for t in takes:
        was = x[t]
        with fwd.dual_level():
            x[t] = fwd.make_dual(was, torch.ones_like(was))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        x[t] = was.clone().requires_grad_()
        if not (name.startswith("rotary") and t in "qk"):  # those have gradients
            with pytest.raises(RuntimeError, match="gradient"):
                call()
            with torch.no_grad():
                call()
        x[t] = was
    call()


@pytest.mark.parametrize("name", NAMES)
def test_operators_refuse_what_they_do_not_differentiate(name):
    _refusals("meta", name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_operators_refuse_what_they_do_not_differentiate_on_the_gpu(name):
    _refusals("cuda", name)


def test_functional_jvp_is_refused():
    x, calls = _operators("meta")
    def f(q):
        x["q"] = q
        return calls["rotary"][0]()
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (x["q"],), (x["q"],))


@pytest.mark.gpu
def test_module_calls_refuse_them():
    dev = torch.device("cuda", 0)
    q = torch.randn((1, 40, 2, 64), device=dev).half()
    f = Rotary.build(64, device=dev).inv_freq
    learned = Rotary(f.clone().requires_grad_())
    for bad in (lambda: rotary_embed(q, learned), lambda: rotary_embed_qk(q, q, learned),
                lambda: rotary_embed(q, Rotary(f.float().requires_grad_())),
                lambda: flash_attn(q, q, q, rotary=learned)):
        with pytest.raises(AssertionError, match="gradient"):
            bad()
    with torch.no_grad():
        assert torch.equal(rotary_embed(q, learned), rotary_embed(q, Rotary(f)))
    cache = PagedKVCache.allocate(4, 16, 2, 64, F16, device=dev)
    table, zero = torch.arange(4, dtype=torch.int32, device=dev)[None], torch.zeros(1, dtype=torch.int32, device=dev)
    with pytest.raises(AssertionError, match="gradient"):
        kv_cache_append(cache, q, q, table, zero, rotary=learned)
    kv_cache_append(cache, q, q, table, zero, rotary=Rotary(f))
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for bad in (lambda: rotary_embed(dual, Rotary(f)), lambda: rotary_embed_qk(q, dual, Rotary(f)),
                    lambda: flash_attn(dual, q, q, rotary=Rotary(f)),
                    lambda: flash_attn_decode(dual[:, :1], cache, table, zero + 40),
                    lambda: kv_cache_append(cache, dual, q, table, zero)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                bad()
