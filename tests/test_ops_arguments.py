"""Arguments of the operators around attention that are no plain numbers or carry derivatives: refused before anything reaches a
GPU, or taken at their value in every call."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import tattn


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def window(**kw):
    a = dict(q=half(2, 4, 8, 32), k=half(2, 2, 8, 32), v=half(2, 2, 8, 32), window=4)
    a.update(kw)
    return tattn.window_attention(**a)


def norm_rope(**kw):
    a = dict(q=torch.zeros(2, 4, 8, 32), k=torch.zeros(2, 2, 8, 32), q_weight=torch.ones(32), k_weight=torch.ones(32),
             cos=torch.ones(8, 16), sin=torch.ones(8, 16))
    a.update(kw)
    return tattn.qk_norm_rope(**a)


def cache():
    return tattn.Cache4.empty(3, 16, 2, 64, dtype=torch.float16, device="cpu")


def attend(**kw):
    a = dict(q=half(2, 4, 64), tables=torch.zeros(2, 3, dtype=torch.int32), lens=i32(0, 0))
    a.update(kw)
    return tattn.cache4_attention(**a, **({} if "cache" in kw else {"cache": cache()}))


def tables(**kw):
    a = dict(lens=i32(3, 0), new_tokens=i32(1, 5), tables=torch.zeros(2, 4, dtype=torch.int32), free_pages=i32(5, 6, 7),
             page_size=16, tokens=8)
    a.update(kw)
    return tattn.page_tables(**a)


# ---- sizes ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("call,bad", [
    (window, dict(window=2.5)), (window, dict(sinks=1.5)), (window, dict(window="4")), (window, dict(sinks=None)),
    (window, dict(window=torch.tensor(2.5))), (window, dict(window=torch.tensor([1, 2]))), (window, dict(window=float("nan"))),
    (attend, dict(window=2.5)), (attend, dict(sinks=0.5)), (tables, dict(page_size=16.5)), (tables, dict(tokens=8.5)),
])
def test_sizes_are_whole_numbers(call, bad):
    with pytest.raises(ValueError, match="must be a whole number"):
        call(**bad)


@pytest.mark.parametrize("call,good", [
    (window, dict(window=4.0)), (window, dict(sinks=True)), (window, dict(window=torch.tensor(4))), (attend, dict(window=3.0)),
    (tables, dict(page_size=16.0, tokens=torch.tensor(8))),
])
def test_whole_numbers_of_other_types_pass_the_checks(call, good):
    with pytest.raises(RuntimeError, match="gfx950"):
        call(**good)


@pytest.mark.gpu
def test_sizes_in_tensors_are_read_in_every_call():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 2, 40, 32, generator=g).to("cuda", torch.float16) for _ in range(3))
    size, first = torch.tensor(4), torch.tensor(0)
    for w, s in ((4, 0), (9, 0), (9, 3)):
        size.fill_(w)
        first.fill_(s)
        assert torch.equal(tattn.window_attention(q, k, v, size, first), tattn.window_attention(q, k, v, w, s))
    cos, sin = (torch.rand(40, 16, generator=g).cuda() for _ in range(2))
    ones, turn = torch.ones(32, dtype=torch.float16, device="cuda"), torch.tensor(False)
    for il in (False, True):
        turn.fill_(il)
        got = tattn.qk_norm_rope(q, k, ones, ones, cos, sin, interleaved=turn)
        assert torch.equal(got[0], tattn.qk_norm_rope(q, k, ones, ones, cos, sin, interleaved=il)[0])


# ---- forward-mode derivatives ----------------------------------------------------------------------

def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("call,arg,t", [
    (window, "q", half(2, 4, 8, 32)), (window, "k", half(2, 2, 8, 32)), (window, "v", half(2, 2, 8, 32)),
    (norm_rope, "q", torch.zeros(2, 4, 8, 32)), (norm_rope, "k", torch.zeros(2, 2, 8, 32)),
    (norm_rope, "q_weight", torch.ones(32)), (norm_rope, "k_weight", torch.ones(32)),
    (norm_rope, "cos", torch.ones(8, 16)), (norm_rope, "sin", torch.ones(8, 16)), (attend, "q", half(2, 4, 64)),
])
def test_tangents_are_refused_not_lost(call, arg, t):
    made = {"cache": cache()} if call is attend else {}
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(**{arg: dual(t)}, **made)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            call(**{arg: dual(t)}, **made)
        with pytest.raises(RuntimeError, match="gfx950"):  # none of its arguments has one
            call()
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda x: call(**{arg: x}, **made), (t,), (t,))


def test_tangents_of_what_a_cache_is_given_are_refused():
    k = half(5, 2, 64)
    with forward_ad.dual_level():
        for a in ((dual(k), k), (k, dual(k))):
            with pytest.raises(ValueError, match="forward-mode"):
                tattn.cache4_write(cache(), *a, torch.zeros(5, dtype=torch.int64))


# ---- a cache without heads -------------------------------------------------------------------------

def test_a_cache_has_a_head():
    with pytest.raises(ValueError, match="at least one kv head"):
        tattn.Cache4.empty(3, 16, 0, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="at least one kv head"):
        tattn.Cache4(torch.zeros(3, 0, 2, 16, 32, dtype=torch.uint8), torch.zeros(3, 0, 2, 16, 2, dtype=torch.uint8), torch.float16)
