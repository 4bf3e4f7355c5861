"""GPU tests of lightning_attn_func(save_8bit=True) on heads wider than the kernels take in one piece: q, k and v are each kept once."""
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import checkpoint64  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("d,e", [(64, 512), (512, 64), (512, 512), (128, 1024), (64, 64)])
def test_what_is_kept(cuda_lib, d, e):
    """Between the passes: a byte and a 32nd for each value of q, k and v, and the slopes; 1 % for the allocator's rounding."""
    b, h, n = 2, 4, 1024
    q0, k0, v0 = (torch.randn(b, h, n, w, device=DEV, dtype=torch.bfloat16, requires_grad=True) for w in (d, d, e))
    s = la._build_slope_tensor(h).to(DEV)
    q, k, v = q0 * 1.0, k0 * 2.0, v0 * 3.0
    values = q.numel() + k.numel() + v.numel()
    before = torch.cuda.memory_allocated() - 2 * values
    o = la.lightning_attn_func(q, k, v, s, save_8bit=True)
    del q, k, v
    held = torch.cuda.memory_allocated() - before - 2 * o.numel()
    assert values <= held <= 1.01 * (values + values // 32) + 4096
    del o


@pytest.mark.parametrize("d,e", [(64, 512), (64, 768), (512, 64), (272, 528), (72, 520), (256, 257), (640, 600)])
@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_are_those_at_the_kept_values(cuda_lib, d, e, decay, dtype):
    """Bit for bit those of the call without checkpoints on what the checkpoints stand for: the same kernels on the same slices, summed
    in the same order (n is short of the length from which on that call keeps its forward pass's chunk states)."""
    b, h, n = 1, 2, 140
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, do = ((0.3 * torch.randn(b, h, n, w, generator=g, device=DEV)).to(dtype) for w in (d, d, e, e))
    s = la._build_slope_tensor(h).to(DEV) if decay else None
    q8, k8, v8 = (checkpoint64(t).to(dtype).requires_grad_() for t in (q, k, v))
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o = la.lightning_attn_func(q, k, v, s, save_8bit=True)
    assert o.shape == v.shape and torch.equal(o, la.lightning_attn_func(q, k, v, s))
    want = torch.autograd.grad(la.lightning_attn_func(q8, k8, v8, s), (q8, k8, v8), do)
    for got, ref in zip(torch.autograd.grad(o, (q, k, v), do), want):
        assert got.shape == ref.shape and torch.equal(got, ref)


def test_strided_and_partly_frozen(cuda_lib):
    """(b, n, h, dim) projections of wide heads, and leaves of which some want no gradient."""
    b, h, n, d, e = 2, 2, 77, 64, 320
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, do = ((0.3 * torch.randn(b, n, h, w, generator=g, device=DEV)).bfloat16().transpose(1, 2) for w in (d, d, e, e))
    s = la._build_slope_tensor(h).to(DEV)
    leaves = [t.contiguous().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(la.lightning_attn_func(*leaves, s, save_8bit=True), leaves, do)
    strided = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(la.lightning_attn_func(*strided, s, save_8bit=True), strided, do)
    assert all(torch.equal(u, w) for u, w in zip(got, want))
    o = la.lightning_attn_func(q.detach(), leaves[1], v.detach(), s, save_8bit=True)
    assert torch.equal(torch.autograd.grad(o, leaves[1], do)[0], want[1])
    with torch.no_grad():
        assert not la.lightning_attn_func(*leaves, s, save_8bit=True).requires_grad


def test_hooks_that_change_shapes_are_refused(cuda_lib):
    q, k, v = (torch.randn(1, 2, 64, w, device=DEV).bfloat16().requires_grad_() for w in (64, 64, 512))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t[..., :16]):
        o = la.lightning_attn_func(q, k, v, None, save_8bit=True)
    with pytest.raises(RuntimeError, match="hooks returned another shape"):
        torch.autograd.grad(o, q, torch.ones_like(o))
