"""CPU tests of the layer norms and 8-bit checkpoints: refusals, sizes, and the plain implementations the GPU tests compare with."""
import ctypes
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la
from lightning_attention_b200 import _lib

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import checkpoint64, reference  # noqa: E402


def _p():
    buf = (ctypes.c_char * 4096)()
    _p.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255


def test_public_names():
    for name in ("layer_norm", "layer_norm_sigmoid_gate", "LayerNorm", "pack_8bit", "unpack_8bit"):
        assert hasattr(la, name) and name in la.ops.__all__
    m = la.LayerNorm(8)
    assert [n for n, _ in m.named_parameters()] == ["weight", "bias"] and torch.equal(m.weight, torch.ones(8)) and torch.equal(m.bias, torch.zeros(8))
    m.load_state_dict(torch.nn.LayerNorm(8).state_dict())
    assert [n for n, _ in la.LayerNorm(8, bias=False).named_parameters()] == ["weight"]
    assert list(la.LayerNorm(8, elementwise_affine=False).parameters()) == []


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    for call in (lambda: la.layer_norm(x), lambda: la.layer_norm_sigmoid_gate(x, x), lambda: la.pack_8bit(x),
                 lambda: la.unpack_8bit(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8)), lambda: la.LayerNorm(64)(x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    q = torch.zeros(1, 2, 16, 16, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        la.lightning_attn_func(q, q, q, torch.zeros(2), save_8bit=True)


@pytest.mark.parametrize("n", [(1 << 30) + 1, (1 << 32) + 64])
def test_rows_past_what_the_kernels_count_are_refused(n):
    """Lengths that a 32-bit count would cut short, of views that hold one value."""
    x, codes = torch.zeros(1).expand(2, n), torch.zeros(1, dtype=torch.int8).expand(2, n)
    scales = torch.zeros(1, dtype=torch.uint8).expand(2, -(-n // 32))
    for call in (lambda: la.layer_norm(x), lambda: la.layer_norm_sigmoid_gate(x, x), lambda: la.pack_8bit(x), lambda: la.unpack_8bit(codes, scales)):
        with pytest.raises(RuntimeError, match="at most 2\\^30"):
            call()


def test_layernorm_fwd_argument_validation():
    L, p = _lib.lib(), _p()

    def fwd(x=p, ldx=64, gate=None, ldg=64, w=p, b=p, wdt=_lib.BF16, y=p, stats=p, xc=None, xs=None, gc=None, gs=None, M=4, N=64, eps=1e-5, dt=_lib.BF16):
        return L.lab200_layernorm_fwd(x, ldx, gate, ldg, w, b, wdt, y, stats, xc, xs, gc, gs, M, N, eps, dt, None)

    assert fwd(M=0) == 0 and fwd(M=0, x=None, y=None) == 0
    assert fwd(M=-1) == 1 and fwd(N=0) == 1 and fwd(N=(1 << 30) + 1, ldx=1 << 31) == 1 and fwd(M=1 << 40, N=1 << 30, ldx=1 << 30) == 1
    assert fwd(ldx=63) == 1 and fwd(gate=p, ldg=63) == 1 and fwd(x=None) == 1 and fwd(y=None) == 1
    assert fwd(dt=3) == 2 and fwd(wdt=_lib.F16) == 2 and fwd(dt=_lib.F32, wdt=_lib.BF16) == 2
    assert fwd(eps=-1.0) == 1 and fwd(eps=float("nan")) == 1 and fwd(eps=float("inf")) == 1
    assert fwd(xc=p) == 1 and fwd(xs=p) == 1 and fwd(gc=p, gs=p) == 1  # half a checkpoint, a gate's without a gate
    assert fwd(gate=p, xc=p, xs=p) == 1 and fwd(gate=p, gc=p, gs=p) == 1  # both or none
    assert fwd(stats=p + 4) == 6 and fwd(x=p + 1) == 6 and fwd(y=p + 1) == 6 and fwd(gate=p + 1) == 6
    assert fwd(w=p + 1) == 6 and fwd(b=p + 2, w=None, wdt=_lib.F32) == 6


def test_layernorm_bwd_argument_validation():
    L, p = _lib.lib(), _p()

    def bwd(x=p, ldx=64, gate=None, ldg=64, xc=None, xs=None, gc=None, gs=None, stats=p, dy=p, lddy=64, w=p, b=p, wdt=_lib.BF16, dx=p, dg=None, dw=p,
            db=p, ws=p, nbytes=1 << 20, M=4, N=64, dt=_lib.BF16):
        return L.lab200_layernorm_bwd(x, ldx, gate, ldg, xc, xs, gc, gs, stats, dy, lddy, w, b, wdt, dx, dg, dw, db, ws, nbytes, M, N, dt, None)

    assert bwd(M=-1) == 1 and bwd(N=0) == 1 and bwd(ldx=63) == 1 and bwd(lddy=63) == 1 and bwd(gate=p, ldg=63) == 1
    assert bwd(x=None) == 1 and bwd(xc=p, xs=p) == 1 and bwd(x=None, xc=p) == 1  # neither, both, half
    assert bwd(gate=p, gc=p, gs=p) == 1 and bwd(x=None, xc=p, xs=p, gate=p) == 1 and bwd(gc=p, gs=p) == 1
    assert bwd(stats=None) == 1 and bwd(dy=None) == 1 and bwd(dg=p) == 1
    assert bwd(dt=3) == 2 and bwd(wdt=_lib.F16) == 2
    assert bwd(x=p + 1) == 6 and bwd(dy=p + 1) == 6 and bwd(dx=p + 1) == 6 and bwd(w=p + 1) == 6 and bwd(dw=p + 2, wdt=_lib.F32) == 6 and bwd(db=p + 1) == 6
    assert bwd(ws=None) == 3 and bwd(nbytes=8) == 3 and bwd(ws=p + 8) == 6 and bwd(stats=p + 4) == 6
    assert L.lab200_layernorm_bwd_workspace_bytes(0, 64) == 0
    sizes = [L.lab200_layernorm_bwd_workspace_bytes(m, 4096) for m in (1, 100, 4096, 1 << 20, 1 << 40)]
    assert sizes == sorted(sizes) and sizes[0] > 0 and sizes[-1] <= 512 * 2 * 4096 * 4


def test_pack8_argument_validation():
    L, p = _lib.lib(), _p()
    assert L.lab200_pack8(p, 64, p, p, 0, 64, _lib.BF16, None) == 0 and L.lab200_unpack8(p, p, p, 0, 64, _lib.BF16, None) == 0
    assert L.lab200_pack8(p, 63, p, p, 2, 64, _lib.BF16, None) == 1 and L.lab200_pack8(p, 64, p, p, 2, 0, _lib.BF16, None) == 1
    assert L.lab200_pack8(None, 64, p, p, 2, 64, _lib.BF16, None) == 1 and L.lab200_pack8(p, 64, None, p, 2, 64, _lib.BF16, None) == 1
    assert L.lab200_pack8(p, 64, p, None, 2, 64, _lib.BF16, None) == 1 and L.lab200_pack8(p, 64, p, p, 2, 64, 3, None) == 2
    assert L.lab200_unpack8(p, p, p, -1, 64, _lib.BF16, None) == 1 and L.lab200_unpack8(p, p, p, 2, 64, 5, None) == 2
    assert L.lab200_pack8(p + 1, 64, p, p, 2, 64, _lib.BF16, None) == 6 and L.lab200_unpack8(p, p, p + 2, 2, 64, _lib.F32, None) == 6
    assert L.lab200_unpack8(None, p, p, 2, 64, _lib.BF16, None) == 1 and L.lab200_unpack8(p, p, None, 2, 64, _lib.BF16, None) == 1


@pytest.mark.parametrize("gated", [False, True])
def test_reference_gradients_against_differences(gated):
    """The 64-bit formulas of _ln_refs.py against autograd of the definition, and that against differences."""
    torch.manual_seed(0)
    x, g, dy = (torch.randn(5, 33, dtype=torch.float64) for _ in range(3))
    w, b = torch.randn(33, dtype=torch.float64), torch.randn(33, dtype=torch.float64)

    def definition(x, g, w, b):
        y = torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5)
        return y * torch.sigmoid(g) if gated else y

    leaves = [t.clone().requires_grad_() for t in (x, g, w, b)]
    assert torch.autograd.gradcheck(definition, leaves)
    y = definition(*leaves)
    want = dict(zip(("dx", "dgate", "dw", "db"), torch.autograd.grad(y, leaves, dy, allow_unused=True)))
    got = reference(x, g if gated else None, w, b, 1e-5, dy)
    assert set(got) == {"y", "dx", "dw", "db"} | ({"dgate"} if gated else set())
    torch.testing.assert_close(got["y"][0], y.detach(), rtol=1e-12, atol=1e-13)
    for name in got:
        if name != "y":
            torch.testing.assert_close(got[name][0], want[name], rtol=1e-10, atol=1e-12)


def test_reference_checkpoint():
    """Half a step of at most 2^-6 of the group's largest value; powers of two, largest values and empty groups by hand."""
    torch.manual_seed(0)
    x = torch.randn(64, 100, dtype=torch.float64).float()
    c = checkpoint64(x)
    for lo in range(0, 100, 32):
        top = x[:, lo:lo + 32].abs().amax(1, keepdim=True).double()
        assert bool(((c[:, lo:lo + 32] - x[:, lo:lo + 32].double()).abs() <= top / 127 * 1.0001).all())
    hand = torch.tensor([[127.0, 63.5, 0.5, 1.5, -2.5], [127.5, 1.0, -3.0, 0, 0], [128.0, 1.0, -1.0, 0, 0], [0.0, 0, 0, 0, 0]])
    want = [[127.0, 64.0, 0.0, 2.0, -2.0], [128.0, 0.0, -4.0, 0, 0], [128.0, 0.0, 0.0, 0, 0], [0.0, 0, 0, 0, 0]]
    want[2] = [128.0, 0.0, 0.0, 0, 0]  # step 2: 1.0 is half a step, to even
    assert checkpoint64(hand).tolist() == want
    assert torch.isnan(checkpoint64(torch.tensor([[1.0, float("inf")]]))).all()
