"""Refusals of the operators around attention, checked before anything reaches a GPU: the Python
wrappers' messages and the C entry points' codes."""

import ctypes

import pytest
import torch

import tattn
from tattn import _lib


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


# ---- page_tables ---------------------------------------------------------------------------------

def _tables(**kw):
    a = dict(lens=i32(3, 0), new_tokens=i32(1, 5), tables=torch.zeros(2, 4, dtype=torch.int32), free_pages=i32(5, 6, 7),
             page_size=16, tokens=8)
    a.update(kw)
    return tattn.page_tables(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens must be int32"),
    (dict(lens=torch.zeros(2, 1, dtype=torch.int32)), "lens must be int32"),
    (dict(new_tokens=i32(1)), "new_tokens must be int32 of shape"),
    (dict(tables=torch.zeros(3, 4, dtype=torch.int32)), "tables must be int32 of shape"),
    (dict(tables=torch.zeros(4, dtype=torch.int32)), "tables must be int32"),
    (dict(tables=torch.zeros(4, 2, dtype=torch.int32).t()), "updated in place"),
    (dict(tables=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), "updated in place"),
    (dict(free_pages=torch.zeros(3)), "free_pages must be int32"),
    (dict(page_size=24), "page size"),
    (dict(page_size=8), "page size"),
    (dict(page_size=2048), "page size"),
    (dict(tokens=-1), "tokens out of range"),
    (dict(tokens=1 << 31), "tokens out of range"),
    (dict(new_tokens=torch.zeros(2, dtype=torch.int32, device="meta")), "must be on cpu"),
])
def test_page_tables_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _tables(**bad)


def test_page_tables_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="gfx950"):
        _tables()


@pytest.mark.parametrize("bad,msg", [
    (dict(page=20), "page size"), (dict(page=0), "page size"), (dict(T=-1), "tokens out of range"),
    (dict(R=1 << 31), "requests out of range"), (dict(lens=None), "lens is a null pointer"),
    (dict(slots=12), "slots must be 8-byte aligned"), (dict(taken=None), "taken is a null pointer"),
    (dict(stride=3), "rows overlap"),
])
def test_page_tables_entry_point_refuses(bad, msg):
    a = dict(lens=16, add=16, tables=16, free=16, slots=16, pos=16, starts=16, taken=16, R=2, P=4, stride=4, F=3, T=8,
             page=16, stream=None)
    a.update(bad)
    assert _lib.load().tattn_page_tables(*a.values()) == 1
    assert msg in _lib.last_error()


# ---- the cache in 4 bits ------------------------------------------------------------------------

def _cache(dtype=torch.float16, page=16, d=64):
    return tattn.Cache4.empty(3, page, 2, d, dtype=dtype, device="cpu")


def test_cache4_describes_itself():
    c = _cache()
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim, c.dtype) == (3, 16, 2, 64, torch.float16)
    assert c.codes.shape == (3, 2, 2, 16, 32) and c.scales.shape == (3, 2, 2, 16, 2)


@pytest.mark.parametrize("kw,msg", [
    (dict(d=16), "head dim"), (dict(d=256), "head dim"), (dict(page=20), "page size"), (dict(page=8), "page size"),
    (dict(dtype=torch.float32), "dtype"),
])
def test_cache4_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        _cache(**kw)


def test_cache4_refuses_buffers_that_do_not_belong_together():
    c = _cache()
    with pytest.raises(ValueError, match="codes must be uint8"):
        tattn.Cache4(c.codes[0], c.scales, c.dtype)
    with pytest.raises(ValueError, match="scales must be uint8"):
        tattn.Cache4(c.codes, c.scales[..., :1], c.dtype)
    with pytest.raises(ValueError, match="contiguous"):
        tattn.Cache4(c.codes[:, :, :, ::1].transpose(0, 1).contiguous().transpose(0, 1), c.scales, c.dtype)
    with pytest.raises(ValueError, match="scales must be on"):
        tattn.Cache4(c.codes, c.scales.to("meta"), c.dtype)


@pytest.mark.parametrize("bad,msg", [
    (dict(k=torch.zeros(5, 2, 32, dtype=torch.float16)), "expected k, v"),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.float16)), "expected k, v"),
    (dict(v=torch.zeros(5, 2, 64, dtype=torch.bfloat16)), "dtype"),
    (dict(slots=torch.zeros(5, dtype=torch.int32)), "slots must be int64"),
    (dict(slots=torch.zeros(4, dtype=torch.int64)), "slots must be int64"),
    (dict(slots=torch.zeros(5, dtype=torch.int64, device="meta")), "slots must be on"),
])
def test_cache4_write_refuses(bad, msg):
    a = dict(k=torch.zeros(5, 2, 64, dtype=torch.float16), v=torch.zeros(5, 2, 64, dtype=torch.float16),
             slots=torch.zeros(5, dtype=torch.int64))
    a.update(bad)
    with pytest.raises(ValueError, match=msg):
        tattn.cache4_write(_cache(), **a)


def test_cache4_read_refuses():
    for bad in (torch.zeros(5, dtype=torch.int32), torch.zeros(5, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="slots must be int64"):
            tattn.cache4_read(_cache(), bad)
    with pytest.raises(RuntimeError, match="gfx950"):
        tattn.cache4_read(_cache(), torch.zeros(5, dtype=torch.int64))


@pytest.mark.parametrize("bad,msg", [
    (dict(D=16), "head dim"), (dict(dtype=_lib.F32), "dtype"), (dict(page=48), "page size"), (dict(pages=-1), "pages out of range"),
    (dict(codes=None), "codes is a null pointer"), (dict(codes=24), "codes must be 16-byte aligned"),
    (dict(k=8), "k must be 16-byte aligned"), (dict(ks=(ctypes.c_int64 * 2)(128, 60)), "k stride"),
    (dict(vs=None), "v strides are null"), (dict(T=1 << 31), "tokens out of range"),
])
def test_cache4_write_entry_point_refuses(bad, msg):
    st = (ctypes.c_int64 * 2)(128, 64)
    a = dict(codes=16, scales=16, k=16, v=16, slots=16, ks=st, vs=st, T=4, H=2, D=64, pages=3, page=16, dtype=_lib.F16,
             stream=None)
    a.update(bad)
    assert _lib.load().tattn_cache4_write(*a.values()) == 1
    assert msg in _lib.last_error()


# ---- qk_norm_rope --------------------------------------------------------------------------------

def _norm_rope(**kw):
    a = dict(q=torch.zeros(2, 4, 8, 32), k=torch.zeros(2, 2, 8, 32), q_weight=torch.ones(32), k_weight=torch.ones(32),
             cos=torch.ones(8, 16), sin=torch.ones(8, 16))
    a.update(kw)
    return tattn.qk_norm_rope(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=torch.zeros(4, 8, 32)), "expected q"),
    (dict(k=torch.zeros(2, 2, 9, 32)), "expected q"),
    (dict(k=torch.zeros(2, 0, 8, 32)), "at least one head"),
    (dict(q=torch.zeros(2, 4, 8, 48), k=torch.zeros(2, 2, 8, 48)), "head dim"),
    (dict(q=torch.zeros(2, 4, 8, 32).half()), "dtype"),
    (dict(q_weight=torch.ones(16)), "q_weight must have shape"),
    (dict(k_weight=torch.ones(32).half()), "k_weight must have shape"),
    (dict(cos=torch.ones(8, 32)), "cos must be float32"),
    (dict(sin=torch.ones(8, 16).half()), "sin must be float32"),
    (dict(sin=torch.ones(7, 16)), "sin must be float32"),
    (dict(cos=torch.ones(7, 16), sin=torch.ones(7, 16)), "7 rows for 8 positions"),
    (dict(cos=torch.ones(0, 16), sin=torch.ones(0, 16), positions=torch.zeros(8, dtype=torch.int32)), "no rows"),
    (dict(positions=torch.zeros(8, dtype=torch.int64)), "positions must be int32"),
    (dict(positions=torch.zeros(1, 8, dtype=torch.int32)), "positions must be int32"),
    (dict(cos=torch.ones(8, 16, device="meta")), "cos must be on"),
])
def test_qk_norm_rope_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _norm_rope(**bad)


def test_qk_norm_rope_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="gfx950"):
        _norm_rope()


@pytest.mark.parametrize("bad,msg", [
    (dict(D=48), "head dim"), (dict(dtype=9), "unknown dtype"), (dict(wd=_lib.BF16), "weights must be"), (dict(Hk=0), "heads must be positive"),
    (dict(q=8), "q must be 16-byte aligned"), (dict(cos=None), "cos is a null pointer"), (dict(P=0), "no rows"),
    (dict(ks=(ctypes.c_int64 * 4)(64, 60, 32, 1)), "k stride"), (dict(ko=None), "k_out is a null pointer"),
    (dict(qos=(ctypes.c_int64 * 4)(1024, 256, 32, 2)), "q_out d stride must be 1"),
    (dict(Z=1 << 20, N=1 << 20), "too many tokens"),
])
def test_norm_rope_entry_point_refuses(bad, msg):
    st = (ctypes.c_int64 * 4)(1024, 256, 32, 1)
    a = dict(q=16, k=16, qw=16, kw=16, cos=16, sin=16, pos=None, qo=16, ko=16, qs=st, ks=st, qos=st, kos=st, ps=0, Z=2, H=4,
             Hk=2, N=8, D=32, P=8, dtype=_lib.F16, wd=_lib.F16, il=0, eps=1e-6, stream=None)
    a.update(bad)
    assert _lib.load().tattn_norm_rope_fwd(*a.values()) == 1
    assert msg in _lib.last_error()


def test_norm_rope_workspace_rows_match_the_header():
    from test_abi import HEADER

    assert f"#define TATTN_NORM_ROPE_ROWS {_lib.NORM_ROPE_ROWS}" in HEADER.read_text()


# ---- window_attention ----------------------------------------------------------------------------

def _window(**kw):
    a = dict(q=torch.zeros(2, 4, 8, 32).half(), k=torch.zeros(2, 2, 8, 32).half(), v=torch.zeros(2, 2, 8, 32).half(), window=4)
    a.update(kw)
    return tattn.window_attention(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=torch.zeros(4, 8, 32).half()), "expected q"),
    (dict(v=torch.zeros(2, 2, 9, 32).half()), "expected q"),
    (dict(q=torch.zeros(1, 4, 8, 32).half()), "expected q"),
    (dict(q=torch.zeros(2, 3, 8, 32).half()), "multiple of kv heads"),
    (dict(q=torch.zeros(2, 4, 9, 32).half()), "9 queries for 8 keys"),
    (dict(q=torch.zeros(2, 4, 8, 48).half(), k=torch.zeros(2, 2, 8, 48).half(), v=torch.zeros(2, 2, 8, 48).half()), "head dim"),
    (dict(q=torch.zeros(2, 4, 8, 32)), "dtype"),
    (dict(q=torch.zeros(2, 4, 8, 32).double(), k=torch.zeros(2, 2, 8, 32).double(), v=torch.zeros(2, 2, 8, 32).double()), "dtype"),
    (dict(window=0), "window must be positive"),
    (dict(sinks=-1), "sinks not negative"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens must be int32"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "lens must be int32"),
    (dict(lens=torch.zeros(2, dtype=torch.int32, device="meta")), "lens must be on"),
    (dict(lens=torch.zeros(2, dtype=torch.int32), q=torch.zeros(2, 4, 8, 32).half().requires_grad_()), "no gradients with lens"),
])
def test_window_attention_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _window(**bad)


def test_window_attention_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="gfx950"):
        _window()


@pytest.mark.parametrize("bad,msg", [
    (dict(D=48), "head dim"), (dict(dtype=5), "dtype"), (dict(Hk=3), "evenly"), (dict(S=7), "8 queries for 7 keys"),
    (dict(window=0), "window must be positive"), (dict(sinks=-1), "sinks must not be negative"), (dict(N=0), "positive"),
    (dict(k=None), "k is a null pointer"), (dict(v=8), "v must be 16-byte aligned"),
    (dict(ks=(ctypes.c_int64 * 4)(512, 256, 16, 1)), "k rows overlap"), (dict(ks=(ctypes.c_int64 * 4)(512, 256, 36, 1)), "multiple of"),
    (dict(ks=(ctypes.c_int64 * 4)(512, 256, 1 << 25, 1)), "2 GiB"), (dict(vs=(ctypes.c_int64 * 4)(512, 256, 32, 0)), "v d stride must be 1"), (dict(os=None), "o strides are null"),
    (dict(Z=1 << 20, H=1 << 20, Hk=1), "too many rows"),
])
def test_window_entry_point_refuses(bad, msg):
    st = (ctypes.c_int64 * 4)(1024, 256, 32, 1)
    a = dict(q=16, k=16, v=16, o=16, m=None, lens=None, work=None, qs=st, ks=st, vs=st, os=st, Z=2, H=4, Hk=2, N=8, S=8, D=32,
             window=4, sinks=0, dtype=_lib.F16, scale=0.1, stream=None)
    a.update(bad)
    assert _lib.load().tattn_window_fwd(*a.values()) == 1
    assert msg in _lib.last_error()


def test_window_workspace_is_asked_for_where_keys_are_split():
    lib, n = _lib.load(), ctypes.c_int64(-1)
    assert lib.tattn_window_workspace(0, 64, 32, 8, 4096, 4096, 64, 1024, 4, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tattn_window_workspace(0, 1, 8, 2, 1, 8192, 64, 8192, 0, ctypes.byref(n)) == 0 and n.value > 0
    st = (ctypes.c_int64 * 4)(1 << 20, 1 << 19, 64, 1)
    assert lib.tattn_window_fwd(16, 16, 16, 16, None, None, None, st, st, st, st, 1, 8, 2, 1, 8192, 64, 8192, 0, _lib.F16, 0.1, None) == 1
    assert "workspace is a null pointer" in _lib.last_error()
    assert lib.tattn_window_workspace(1, 1, 8, 2, 16384, 16384, 64, 128, 4, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.tattn_window_workspace(1, 8, 8, 2, 16384, 16384, 64, 128, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tattn_window_workspace(1, 1, 8, 1, 8192, 8192, 128, 1024, 0, ctypes.byref(n)) == 0 and n.value > 0  # few key blocks
    assert lib.tattn_window_workspace(1, 1, 8, 2, 16384, 100, 64, 128, 0, ctypes.byref(n)) == 1


@pytest.mark.parametrize("z,h,hk", [(1, 1, 1), (1, 8, 2), (64, 8, 8)])
@pytest.mark.parametrize("n,window,sinks", [(16384, 128, 16384), (16384, 1, 4), (4096, 64, 64), (65536, 1024, 128)])
def test_window_backward_workspace_stays_small(z, h, hk, n, window, sinks):
    """Parts of the first keys' sums: about a thousand of 64 or 128 keys, whatever the sizes."""
    for d in (16, 32, 64, 128):
        out = ctypes.c_int64(-1)
        assert _lib.load().tattn_window_workspace(1, z, h, hk, n, n, d, window, sinks, ctypes.byref(out)) == 0
        assert out.value <= (z * hk * ((min(n, sinks) + 63) // 64) + 2048) * 2 * 128 * d


# ---- cache4_attention ----------------------------------------------------------------------------

def _attend(**kw):
    a = dict(q=torch.zeros(2, 4, 64).half(), cache=_cache(), tables=torch.zeros(2, 3, dtype=torch.int32),
             lens=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return tattn.cache4_attention(**a)


@pytest.mark.parametrize("bad,msg", [
    (dict(q=torch.zeros(2, 4, 1, 64).half()), "expected q"),
    (dict(q=torch.zeros(2, 4, 32).half()), "expected q"),
    (dict(q=torch.zeros(2, 3, 64).half()), "multiple of 2 heads"),
    (dict(q=torch.zeros(2, 0, 64).half()), "expected q"),
    (dict(q=torch.zeros(2, 4, 64).bfloat16()), "cache's dtype"),
    (dict(tables=torch.zeros(2, 3)), "tables must be int32"),
    (dict(tables=torch.zeros(3, 3, dtype=torch.int32)), "tables must be int32"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens must be int32"),
    (dict(window=0), "window must be positive"),
    (dict(sinks=-1), "sinks not negative"),
    (dict(lens=torch.zeros(2, dtype=torch.int32, device="meta")), "lens must be on"),
    (dict(q=torch.zeros(2, 4, 64).half().requires_grad_()), "no gradients"),
])
def test_cache4_attention_refuses(bad, msg):
    with pytest.raises(ValueError, match=msg):
        _attend(**bad)


def test_cache4_attention_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="gfx950"):
        _attend()


@pytest.mark.parametrize("bad,msg", [
    (dict(D=16), "head dim"), (dict(H=3), "evenly"), (dict(dtype=_lib.F32), "dtype"), (dict(page=40), "page size"),
    (dict(pages=0), "no pages"), (dict(width=1 << 28), "2^31 tokens"), (dict(window=-1), "must not be negative"),
    (dict(lens=None), "lens is a null pointer"), (dict(codes=8), "codes must be 16-byte aligned"),
    (dict(qs=(ctypes.c_int64 * 2)(256, 63)), "q stride"), (dict(width=1 << 12), "workspace is a null pointer"),
])
def test_cache4_attention_entry_point_refuses(bad, msg):
    st = (ctypes.c_int64 * 2)(256, 64)
    a = dict(q=16, o=16, codes=16, scales=16, tables=16, lens=16, work=None, qs=st, os=st, ts=3, R=2, H=4, Hk=2, D=64, width=3,
             pages=3, page=16, window=0, sinks=0, dtype=_lib.F16, scale=0.1, stream=None)
    a.update(bad)
    assert _lib.load().tattn_cache4_attention(*a.values()) == 1
    assert msg in _lib.last_error()
