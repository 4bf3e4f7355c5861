"""GPU tests of row lengths on both sides of those up to which the layer norms keep a row in registers."""
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import assert_within, reference  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"

# rows that packs do not divide: gated backward, then the others; a multiple of the packs beside each
SIZES = [(torch.bfloat16, n) for n in (4087, 4089, 4090, 4095, 4097, 8183, 8185, 8186, 8191)] + [(torch.float16, n) for n in (4089, 4090, 8185, 8186)] + \
        [(torch.float32, n) for n in (4091, 4093, 4094, 4095, 4097, 8189, 8190, 8191)] + [(torch.bfloat16, 16384), (torch.bfloat16, 16392), (torch.float32, 8196)]


@pytest.mark.parametrize("dtype,n", SIZES, ids=lambda v: str(v).removeprefix("torch."))
@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
def test_both_sides(cuda_lib, dtype, n, gated):
    m = 21  # more rows than a period of shifts, fewer than there are SMs
    g = torch.Generator(device=DEV).manual_seed(n)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)
    x, dy = ((r(m, n) * torch.exp(0.5 * r(n)) + 0.3).to(dtype).requires_grad_(), r(m, n).to(dtype))
    gate = (2 * r(m, n)).to(dtype).requires_grad_() if gated else None
    w, b = (1 + 0.3 * r(n)).requires_grad_(), (0.3 * r(n)).requires_grad_()
    for save_8bit in (False, True):
        y = la.layer_norm_sigmoid_gate(x, gate, w, b, save_8bit=save_8bit) if gated else la.layer_norm(x, w, b, save_8bit=save_8bit)
        leaves = {"dx": x, "dw": w, "db": b, **({"dgate": gate} if gated else {})}
        ref = reference(x, gate, w, b, 1e-5, dy, save_8bit)
        for name, t in {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}.items():
            assert_within(t, ref[name], f"8bit={save_8bit} {name}")
