"""The backward of cross_attention reads its saved tensors by the layouts that they come back with: hooks on saved tensors (offload,
compression) may return them in others than the forward saw. On the CPU, with a library that only takes note of its arguments."""

import contextlib
import ctypes

import pytest
import torch

from tattn import _lib, cross


class Library:
    """Takes note of the addresses and strides of the backward's tensors."""

    def __init__(self):
        self.calls = []

    def tattn_cross_workspace(self, *args):
        args[-1]._obj.value = 4
        return 0

    def tattn_cross_fwd(self, *args):
        return 0

    def tattn_cross_bwd(self, *args):
        def strides(at):
            return tuple((ctypes.c_int64 * 4).from_address(at))

        self.calls.append((args[:8], [strides(at) for at in args[11:19]]))
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(cross, "_plans", {})
    monkeypatch.setattr(cross, "_require_gpu", lambda q: None)
    monkeypatch.setattr(cross, "_on_device", lambda q: contextlib.nullcontext())
    monkeypatch.setattr(cross, "_stream", lambda q: None)
    return lib


def dense(t):
    return t.contiguous().clone(memory_format=torch.contiguous_format)


def kept(t):
    return t


def turned(t):
    """Rows of another order: the head's dimension outermost but for the batch."""
    return t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t


def step(library, back):
    """One step with k and v as slices of one projection, saved tensors as `back` returns them."""
    kv = torch.zeros(2, 300, 2, 4, 64, dtype=torch.float16)
    q = torch.zeros(2, 8, 40, 64, dtype=torch.float16, requires_grad=True)
    k, v = (kv[:, :, i].transpose(1, 2).requires_grad_() for i in range(2))
    seen = {}

    def unpack(t):
        t = back(t)
        seen[t.data_ptr()] = t
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        o = cross.cross_attention(q, k, v)
        grads = torch.autograd.grad(o, (q, k, v), torch.zeros_like(o))
    pointers, strides = library.calls[-1]
    for at, name in enumerate(("q", "k", "v", "o")):
        t = seen[pointers[at]]
        assert strides[at] == t.stride(), f"{name} of {tuple(t.stride())} read as of {strides[at]}"
    for g, st in zip(grads, strides[5:]):
        assert g.stride() == st
    return strides


@pytest.mark.parametrize("order", [(kept, dense), (dense, kept), (turned, dense, kept), (dense, turned, dense, kept, turned)])
def test_strides_are_those_of_the_tensors_that_come_back(library, order):
    first = [step(library, back) for back in order]
    assert [step(library, back) for back in order] == first


# ---- qk_rope_axes ----------------------------------------------------------------------------------

class RopeLibrary:
    """Takes a copy of the tables, weights and positions that the backward is given."""

    def tattn_rope_axes_fwd(self, *args):
        return 0

    def tattn_rope_axes_bwd(self, *args):
        self.args = args

        def copy(at, kind, count):
            return list((kind * count).from_address(at))

        self.got = [copy(at, ctypes.c_float, n) for at, n in zip(args[2:6], (32, 32, 9 * 16, 9 * 16))]
        self.got.append(copy(args[6], ctypes.c_int32, 2 * 3 * 5))
        return 0


def columns(t):
    """The same values with the last dimension outermost in memory."""
    return t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.repeat_interleave(2)[::2]


def test_tables_weights_and_positions_are_read_in_the_layout_that_they_come_back_with(monkeypatch):
    from tattn import rope_axes

    lib = RopeLibrary()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(rope_axes, "_plans", {})
    monkeypatch.setattr(rope_axes, "_require_gpu", lambda q: None)
    monkeypatch.setattr(rope_axes, "_on_device", lambda q: contextlib.nullcontext())
    monkeypatch.setattr(rope_axes, "_stream", lambda q: None)
    gen = torch.Generator().manual_seed(1)
    q, k = torch.zeros(3, 4, 5, 32, requires_grad=True), torch.zeros(3, 2, 5, 32, requires_grad=True)
    weights = [torch.randn(32, generator=gen).requires_grad_() for _ in range(2)]
    cos, sin = (torch.randn(9, 16, generator=gen) for _ in range(2))
    positions = torch.randint(0, 9, (2, 3, 5), generator=gen).int()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, columns):
        qo, ko = rope_axes.qk_rope_axes(q, k, cos, sin, positions, (0, 1) * 8, q_weight=weights[0], k_weight=weights[1])
        torch.autograd.grad((qo.sum() + ko.sum()), (q, k, *weights))
    for got, want in zip(lib.got, (*weights, cos, sin, positions)):
        assert got == want.detach().flatten().tolist()
