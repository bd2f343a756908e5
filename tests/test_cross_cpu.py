"""Refusals of cross_attention, prefix_attention and qk_rope_axes, checked before anything reaches a GPU: the Python wrappers'
messages and the C entry points' codes."""

import ctypes

import pytest
import torch

import tattn
from tattn import _lib


def t(*shape, dtype=torch.float16, device="cpu"):
    return torch.zeros(*shape, dtype=dtype, device=device)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def _cross(**kw):
    a = dict(q=t(2, 4, 3, 64), k=t(2, 2, 5, 64), v=t(2, 2, 5, 64))
    a.update(kw)
    return tattn.cross_attention(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=t(4, 3, 64)), "expected q"),
    (dict(v=t(2, 2, 6, 64)), "equal shape"),
    (dict(q=t(2, 4, 3, 32)), "expected q"),
    (dict(q=t(3, 4, 3, 64)), "share their batch"),
    (dict(q=t(2, 3, 3, 64)), "multiple of kv heads"),
    (dict(q=t(2, 0, 3, 64)), "multiple of kv heads"),
    (dict(q=t(2, 4, 3, 48), k=t(2, 2, 5, 48), v=t(2, 2, 5, 48)), "head dim"),
    (dict(q=t(2, 4, 3, 64, dtype=torch.bfloat16)), "share dtype"),
    (dict(q=t(2, 4, 3, 64, dtype=torch.float64), k=t(2, 2, 5, 64, dtype=torch.float64), v=t(2, 2, 5, 64, dtype=torch.float64)), "share dtype"),
    (dict(v=t(2, 2, 5, 64, device="meta")), "v must be on cpu"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens must be int32"),
    (dict(lens=i32(1, 2, 3)), "lens must be int32 of shape"),
    (dict(lens=torch.zeros(2, dtype=torch.int32, device="meta")), "lens must be on cpu"),
])
def test_cross_attention_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _cross(**bad)


def _prefix(**kw):
    a = dict(q=t(6, 4, 1, 64), prefix_k=t(2, 2, 7, 64), prefix_v=t(2, 2, 7, 64), k=t(6, 2, 5, 64), v=t(6, 2, 5, 64), lens=i32(*range(6)))
    a.update(kw)
    return tattn.prefix_attention(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=t(6, 4, 64)), "expected q"),
    (dict(prefix_v=t(2, 2, 8, 64)), "prefix_k, prefix_v of equal shape"),
    (dict(k=t(6, 2, 4, 64)), "equal shape"),
    (dict(prefix_k=t(2, 1, 7, 64), prefix_v=t(2, 1, 7, 64)), "kv heads"),
    (dict(prefix_k=t(4, 2, 7, 64), prefix_v=t(4, 2, 7, 64)), "multiple of the prefixes"),
    (dict(prefix_k=t(0, 2, 7, 64), prefix_v=t(0, 2, 7, 64)), "multiple of the prefixes"),
    (dict(k=t(5, 2, 5, 64), v=t(5, 2, 5, 64)), "q's batch"),
    (dict(k=t(6, 2, 5, 64, dtype=torch.bfloat16)), "share dtype"),
    ({x: y.float() for x, y in dict(q=t(6, 4, 1, 64), prefix_k=t(2, 2, 7, 64), prefix_v=t(2, 2, 7, 64), k=t(6, 2, 5, 64),
                                    v=t(6, 2, 5, 64)).items()}, "float16 or bfloat16"),
    (dict(lens=i32(1)), "lens must be int32 of shape"),
    (dict(lens=torch.zeros(6)), "lens must be int32"),
    (dict(prefix_lens=i32(1, 2, 3)), "prefix_lens must be int32 of shape"),
    (dict(prefix_lens=torch.zeros(2, dtype=torch.int32, device="meta")), "prefix_lens must be on cpu"),
    (dict(v=t(6, 2, 5, 64).requires_grad_()), "no gradients"),
])
def test_prefix_attention_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _prefix(**bad)


def _rope(**kw):
    a = dict(q=t(2, 4, 3, 32), k=t(2, 2, 3, 32), cos=torch.ones(9, 16), sin=torch.ones(9, 16),
             positions=torch.zeros(3, 2, 3, dtype=torch.int32), axes=(0,) * 4 + (1,) * 6 + (2,) * 6)
    a.update(kw)
    return tattn.qk_rope_axes(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=t(4, 3, 32)), "expected q"),
    (dict(k=t(2, 2, 4, 32)), "expected q"),
    (dict(q=t(2, 4, 3, 48), k=t(2, 2, 3, 48)), "head dim"),
    (dict(k=t(2, 2, 3, 32, dtype=torch.bfloat16)), "share dtype"),
    (dict(cos=torch.ones(9, 8)), "cos must be float32"),
    (dict(sin=torch.ones(8, 16)), "sin must be float32 of shape"),
    (dict(cos=torch.ones(0, 16), sin=torch.ones(0, 16)), "no rows"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions must be int32"),
    (dict(positions=torch.zeros(9, 3, dtype=torch.int32)), "1 to 8 axes"),
    (dict(positions=torch.zeros(3, 3)), "positions must be int32 of shape"),
    (dict(positions=torch.zeros(3, 3, 3, dtype=torch.int32)), "positions must be int32 of shape"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int32, device="meta")), "positions must be on cpu"),
    (dict(axes=(0,) * 15), "axes must hold 16"),
    (dict(axes=(3,) * 16), "axes must hold 16 numbers from -1 to 2"),
    (dict(axes=(-2,) * 16), "axes must hold"),
    (dict(axes=(0.5,) * 16), "whole number"),
    (dict(q_weight=t(32)), "both q_weight and k_weight"),
    (dict(q_weight=t(16), k_weight=t(16)), "q_weight must have shape"),
    (dict(q_weight=t(32), k_weight=t(32, dtype=torch.float32)), "both weights alike"),
])
def test_qk_rope_axes_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _rope(**bad)


@pytest.mark.parametrize("call", [_cross, _prefix, _rope])
def test_there_is_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="gfx950"):
        call()


@pytest.mark.parametrize("call,name", [(_cross, "q"), (_prefix, "k"), (_rope, "q")])
def test_forward_mode_derivatives_are_refused(call, name):
    x = dict(q=t(2, 4, 3, 64), k=t(6, 2, 5, 64))[name] if call is not _rope else t(2, 4, 3, 32)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(**{name: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))})


# ---- C entry points --------------------------------------------------------------------------------

def code(name, *args):
    return getattr(_lib.load(), name)(*args), _lib.last_error()


def s4(*x):
    return (ctypes.c_int64 * 4)(*x)


@pytest.mark.parametrize("bad,msg", [
    (dict(D=48), "head dim"), (dict(Z=0), "positive"), (dict(S=0), "positive"), (dict(N=-1), "length out of range"),
    (dict(H=5), "do not share"), (dict(dtype=9), "unknown dtype"), (dict(N=1 << 30, H=4), "too many rows"),
    (dict(k=None), "k is a null pointer"), (dict(v=8), "v must be 16-byte aligned"), (dict(sk=s4(640, 320, 63, 1)), "multiple of 8"),
    (dict(sk=s4(640, 320, 32, 1)), "rows overlap"), (dict(sq=s4(768, 192, 64, 2)), "d stride must be 1"),
    (dict(sv=s4(640, 320, 1 << 25, 1)), "spans 2 GiB"), (dict(so=None), "o strides are null"), (dict(lens=2), "lens must be 4-byte"),
    (dict(N=1, S=9000, Z=1, work=None), "workspace is a null pointer"),
])
def test_cross_forward_entry_point_refuses(bad, msg):
    a = dict(q=16, k=16, v=16, o=16, m=None, lens=None, work=16, sq=s4(768, 192, 64, 1), sk=s4(640, 320, 64, 1),
             sv=s4(640, 320, 64, 1), so=s4(768, 192, 64, 1), Z=2, H=4, Hk=2, N=3, S=5, D=64, dtype=0, scale=1.0, stream=None)
    a.update(bad)
    rc, text = code("tattn_cross_fwd", *a.values())
    assert rc == 1 and msg in text


@pytest.mark.parametrize("bad,msg", [
    (dict(m=None), "m is a null pointer"), (dict(work=None), "workspace is a null pointer"), (dict(dv=8), "dv must be 16-byte"),
    (dict(sq=s4(768, 192, 32, 1)), "q rows overlap"), (dict(sdo=s4(768, 192, 0, 1)), "do rows overlap"), (dict(Hk=3), "do not share"),
])
def test_cross_backward_entry_point_refuses(bad, msg):
    q, k = s4(768, 192, 64, 1), s4(640, 320, 64, 1)
    a = dict(q=16, k=16, v=16, o=16, dout=16, dq=16, dk=16, dv=16, m=16, lens=None, work=16, sq=q, sk=k, sv=k, so=q, sdo=q, sdq=q,
             sdk=k, sdv=k, Z=2, H=4, Hk=2, N=3, S=5, D=64, dtype=0, scale=1.0, stream=None)
    a.update(bad)
    rc, text = code("tattn_cross_bwd", *a.values())
    assert rc == 1 and msg in text


@pytest.mark.parametrize("bad,msg", [
    (dict(groups=0), "positive"), (dict(P=-1), "key length out of range"), (dict(dtype=1), "TATTN_F16 or TATTN_BF16"),
    (dict(lens=None), "lens is a null pointer"), (dict(pk=None), "prefix_k is a null pointer"), (dict(v=8), "v must be 16-byte"),
    (dict(work=None), "workspace is a null pointer"), (dict(members=1 << 29, N=8), "too many rows"),
])
def test_prefix_entry_point_refuses(bad, msg):
    q, k = s4(256, 64, 64, 1), s4(640, 320, 64, 1)
    a = dict(q=16, pk=16, pv=16, k=16, v=16, o=16, plens=None, lens=16, work=16, sq=q, spk=k, spv=k, sk=k, sv=k, so=q, groups=2,
             members=3, H=4, Hk=2, N=1, P=5, S=5, D=64, dtype=0, scale=1.0, stream=None)
    a.update(bad)
    rc, text = code("tattn_prefix_attention", *a.values())
    assert rc == 1 and msg in text


@pytest.mark.parametrize("bad,msg", [
    (dict(num=0), "1 to 8 axes"), (dict(num=9), "1 to 8 axes"), (dict(axes=None), "axes is a null pointer"),
    (dict(axes=(ctypes.c_int32 * 16)(*[3] * 16)), "axis of pair 0 must be -1 to 2"), (dict(positions=None), "positions is a null pointer"),
    (dict(qw=16), "both weights or neither"), (dict(D=48), "head dim"), (dict(R=0), "no rows"), (dict(qo=None), "q_out is a null pointer"),
])
def test_rope_axes_entry_point_refuses(bad, msg):
    q = s4(384, 96, 32, 1)
    a = dict(q=16, k=16, qw=None, kw=None, cos=16, sin=16, positions=16, axes=(ctypes.c_int32 * 16)(*[0, 1, 2, -1] * 4), qo=16, ko=16,
             sq=q, sk=q, sqo=q, sko=q, num=3, axis_stride=6, pos_stride=3, Z=2, H=4, Hk=4, N=3, D=32, R=9, dtype=0, w_dtype=0,
             interleaved=0, eps=1e-6, stream=None)
    a.update(bad)
    rc, text = code("tattn_rope_axes_fwd", *a.values())
    assert rc == 1 and msg in text


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces_are_finite_and_grow_with_the_work(backward, dtype):
    out = ctypes.c_int64()
    for z, h, hk, n, s, d in ((1, 1, 1, 1, 1, 16), (1, 8, 1, 1, 1 << 20, 128), (64, 32, 8, 4096, 77, 64), (1, 2, 2, 1 << 20, 3, 32)):
        assert _lib.load().tattn_cross_workspace(backward, z, h, hk, n, s, d, dtype, ctypes.byref(out)) == 0
        # delta and the norms, and as many float32 sums as 512 workgroups of the largest block hold
        assert 0 <= out.value <= 2 * z * h * n + 64 + 2 * 513 * 2 * 256 * 130
