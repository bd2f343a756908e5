"""Gradients on the GPU where hooks on saved tensors return them in other layouts than the forward saw."""

import pytest
import torch
from test_gpu_cross import BF16, DEV, F16, F32, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from tattn import hip_available

    assert hip_available(DEV), "libtattn_hip.so did not load or the device is not a gfx950"


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def kept(t):
    return t


def turned(t):
    """The other order of heads and rows."""
    return t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t


@pytest.mark.parametrize("order", [(kept, dense), (dense, kept), (turned, dense, kept), (kept, "cpu", kept)])
@pytest.mark.parametrize("dtype,n,s", [(F16, 40, 300), (BF16, 40, 60), (F32, 40, 100)])
def test_gradients_of_slices_of_one_projection(dtype, n, s, order):
    from tattn import cross_attention

    gen = torch.Generator().manual_seed(n + s)
    kv = torch.randn(2, s, 2, 4, 64, generator=gen).to(DEV, dtype)
    q, do = (torch.randn(2, 8, n, 64, generator=gen).to(DEV, dtype) for _ in range(2))
    k, v = (kv[:, :, i].transpose(1, 2) for i in range(2))
    lens = i32(s, s - 7)

    def grads(q, k, v, back):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        hooks = (torch.autograd.graph.save_on_cpu() if back == "cpu" else
                 torch.autograd.graph.saved_tensors_hooks(lambda t: t, back))
        with hooks:
            o = cross_attention(*leaves, lens)
            return torch.autograd.grad(o, leaves, do)

    want = grads(q, dense(k), dense(v), kept)
    for back in order:
        print(dtype, back, flush=True)
        for a, b in zip(grads(q, k, v, back), want):
            assert torch.equal(a, b)
