"""GPU tests of rows whose parts differ: a warp that holds few values far from the row's mean joins the others' statistics without losing any."""
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import assert_within, reference  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def outlier_rows(m, n, dtype, last, seed=0):
    """Rows of unit spread whose last `last` columns lie about 50 spreads away, on one side."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)
    x = r(m, n)
    x[:, n - last:] += 50.0
    gate = 2 * r(m, n)
    w, b, dy = 1 + 0.3 * r(n), 0.3 * r(n), r(m, n)
    return x.to(dtype).requires_grad_(), gate.to(dtype).requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy.to(dtype)


# fp32: one pack a thread where rows are few, so that the last warp has 4 values (516, 1028, 1924) or 8 (1032); more rows and the widths of
# four packs a thread (5000); odd widths, where a row shares its packs with its neighbours (1027, 4099)
@pytest.mark.parametrize("m,n,last", [(3, 516, 4), (3, 1028, 4), (5, 1032, 8), (3, 1924, 4), (1, 1924, 4), (300, 1924, 4), (700, 5000, 4), (40, 1027, 3), (7, 4099, 2)])
@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
def test_outliers_in_a_short_part(cuda_lib, m, n, last, gated):
    x, gate, w, b, dy = outlier_rows(m, n, torch.float32, last)
    for save_8bit in (False, True):
        y = la.layer_norm_sigmoid_gate(x, gate, w, b, save_8bit=save_8bit) if gated else la.layer_norm(x, w, b, save_8bit=save_8bit)
        leaves = {"dx": x, "dw": w, "db": b, **({"dgate": gate} if gated else {})}
        got = {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}
        ref = reference(x, gate if gated else None, w, b, 1e-5, dy, save_8bit)
        for name, t in got.items():
            assert_within(t, ref[name], f"8bit={save_8bit} {name}")
