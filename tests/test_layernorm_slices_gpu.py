"""GPU tests of slices of wider tensors of three and more dimensions: read where they are, on the native path and through the class."""
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la
from lightning_attention_b200 import _lib

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import assert_within, reference  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["native", "class"])
def path(request, monkeypatch):
    if request.param == "class":
        monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    return request.param


def wide(shape, parts, dtype, seed):
    """The last of `parts` equal slices of a tensor whose last dimension is that many times as wide."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.randn(*shape[:-1], parts * shape[-1], generator=g, device=DEV).to(dtype)
    return t[..., (parts - 1) * shape[-1]:]


# one row stride over all leading dimensions, sizes of one among them; a slice of one tensor of rows; rows that are contiguous as they are
SHAPES = [(2, 3, 64), (4, 33, 1040), (3, 1, 5, 200), (1, 7, 1, 4096), (2, 1, 1, 3, 48), (1, 1, 264), (5, 1, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_same_results_as_contiguous(cuda_lib, path, shape, dtype):
    n = shape[-1]
    w, b = (1 + 0.3 * torch.randn(n, device=DEV)).requires_grad_(), torch.randn(n, device=DEV).requires_grad_()
    for parts in (2, 3):
        x, gate, dy = (wide(shape, parts, dtype, seed) for seed in (1, 2, 3))
        for save_8bit in (False, True):
            for gated in (False, True):
                got = []
                for form in (lambda t: t, lambda t: t.contiguous()):
                    xv, gv = form(x).detach().requires_grad_(), form(gate).detach().requires_grad_()
                    y = la.layer_norm_sigmoid_gate(xv, gv, w, b, save_8bit=save_8bit) if gated else la.layer_norm(xv, w, b, save_8bit=save_8bit)
                    got.append([y.detach(), *torch.autograd.grad(y, (xv, w, b) + ((gv,) if gated else ()), form(dy))])
                assert all(torch.equal(u, v) and u.shape == v.shape for u, v in zip(*got))
            ref = reference(x, gate, w, b, 1e-5, dy, save_8bit)
            for name, t in zip(("y", "dx", "dw", "db", "dgate"), got[0]):
                assert_within(t, ref[name], name)
        assert all(torch.equal(u, v) for u, v in zip(la.pack_8bit(x), la.pack_8bit(x.contiguous())))


def test_leading_dimensions_without_one_stride(cuda_lib, path):
    """Rows that no single stride covers (a slice of tokens too, swapped dimensions, broadcast ones) are copied and give the same."""
    base = torch.randn(4, 10, 6, 128, device=DEV).bfloat16()
    for x in (base[:, :7, :, :64], base.transpose(0, 2)[..., 64:], base[:, :, :1, :64].expand(4, 10, 6, 64), base[::2], base[1:, :, ::3, 64:]):
        want = x.contiguous().requires_grad_()
        y0 = la.layer_norm(want)
        xv = x.detach().requires_grad_()
        y = la.layer_norm(xv)
        dy = torch.randn_like(y0)
        assert torch.equal(y, y0) and torch.equal(torch.autograd.grad(y, xv, dy)[0], torch.autograd.grad(y0, want, dy)[0])
        assert all(torch.equal(u, v) for u, v in zip(la.pack_8bit(x), la.pack_8bit(want)))


def peak(f):
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    return torch.cuda.max_memory_allocated() - before, out


@pytest.mark.parametrize("shape", [(1024, 1024), (4, 256, 1024), (2, 2, 256, 1024), (4, 1, 256, 1024)], ids=["2d", "3d", "4d", "4d with a one"])
@pytest.mark.parametrize("save_8bit", [False, True])
def test_a_slice_is_not_copied(cuda_lib, path, shape, save_8bit):
    """What a call allocates: its outputs, the row statistics and checkpoints, and 512 bytes of rounding for each tensor; one copy
    of x, gate or dy would be 2 MB more."""
    m, n = 1024, 1024
    x, gate, dy = (wide(shape, 2, torch.bfloat16, seed) for seed in (1, 2, 3))
    x.requires_grad_(), gate.requires_grad_()
    kept = 8 * m + (2 * (m * n + m * n // 32) if save_8bit else 0)
    used, y = peak(lambda: la.layer_norm_sigmoid_gate(x, gate, save_8bit=save_8bit))
    assert used <= 2 * m * n + kept + 8 * 512
    used, grads = peak(lambda: torch.autograd.grad(y, (x, gate), dy))
    assert used <= 2 * (2 * m * n) + 8 * 512
    del y, grads
    used, y = peak(lambda: la.layer_norm(x.detach()))
    assert used <= 2 * m * n + 8 * 512
    del y
    used, _ = peak(lambda: la.pack_8bit(x.detach()))
    assert used <= m * n + m * n // 32 + 8 * 512


def test_slices_take_the_native_path(cuda_lib):
    x = wide((4, 33, 1024), 2, torch.bfloat16, 1).requires_grad_()
    assert type(la.layer_norm(x).grad_fn).__name__ == "CppFunction"
    assert _lib.host().pack8(x.detach()) is not None
