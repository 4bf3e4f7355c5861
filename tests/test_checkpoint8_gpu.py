"""GPU tests of the 8-bit checkpoints: every value against the format's definition in 64 bits, and attention's use of them."""
import os
import sys

import pytest
import torch

import lightning_attention_b200 as la

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import checkpoint64  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TOP = {torch.float16: 65504.0, torch.float32: 3.4e38, torch.bfloat16: 3.38e38}


def round_trip(x):
    codes, scales = la.pack_8bit(x)
    assert codes.shape == x.shape and codes.dtype == torch.int8 and scales.dtype == torch.uint8
    assert scales.shape == (*x.shape[:-1], (x.shape[-1] + 31) // 32)
    return codes, scales, la.unpack_8bit(codes, scales, x.dtype)


def want(x):
    """The checkpoint's values in x's type: exact but in fp16, where they are rounded once and kept within its range."""
    v = checkpoint64(x)
    return (v.clamp(-65504, 65504) if x.dtype == torch.float16 else v).to(x.dtype)


@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (3, 32), (3, 33), (1, 7), (5, 64), (300, 192), (7, 80), (129, 100), (33, 1000), (65, 1001), (2, 3, 5, 128), (17, 4096),
                                   (2, 65536), (1, 1000003), (4, 8, 64, 64), (1024,), (70000, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_round_trip(cuda_lib, shape, dtype):
    torch.manual_seed(0)
    x = (torch.randn(shape, device=DEV) * torch.exp(3 * torch.randn(shape, device=DEV))).to(dtype)
    _, _, y = round_trip(x)
    torch.testing.assert_close(y, want(x), rtol=0, atol=0, equal_nan=True)  # a few fp16 inputs are infinite


@pytest.mark.parametrize("m,n", [(70001, 1), (5003, 17), (2, 51), (3001, 51), (1001, 67), (800, 99), (257, 225), (257, 257), (90, 290), (300, 562), (61, 1010)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_rows(cuda_lib, m, n, dtype):
    """Rows that packs do not divide, of 1 to 32 groups: counted over all rows, or by row; contiguous and not; nothing behind the ends."""
    torch.manual_seed(0)
    wide = (torch.randn(m, n + 3, device=DEV) * torch.exp(3 * torch.randn(m, n + 3, device=DEV))).to(dtype)
    for x in (wide[:, :n].contiguous(), wide[:, 1:n + 1]):
        _, _, y = round_trip(x)
        torch.testing.assert_close(y, want(x), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_border(cuda_lib, dtype):
    """Ties, groups whose largest value rounds up to 128 steps, powers of two, zeros, the largest and the smallest values of the type."""
    tiny = torch.finfo(dtype).smallest_normal
    rows = [[127.0, 63.5, 0.5, 1.5, -2.5], [127.5, 1.0, -3.0, 1.0, -1.0], [127.4, 127.0, 126.5, 0.5, 0.25], [128.0, 1.0, -1.0, 3.0, 63.0], [0.0, -0.0, 0, 0, 0],
            [TOP[dtype], -TOP[dtype], 1, 2, 3], [tiny, -tiny, tiny / 2, 0, tiny * 3], [2.0 ** -14, 2.0 ** -15, 2.0 ** -20, -2.0 ** -21, 2.0 ** -24]]
    for scale in (1.0, 2.0 ** -9, 2.0 ** 8):
        x = (torch.tensor(rows, device=DEV, dtype=torch.float64) * scale).clamp(-TOP[dtype], TOP[dtype]).to(dtype)
        wide = torch.zeros(len(rows), 70, device=DEV, dtype=dtype)
        wide[:, :5], wide[:, 32:37], wide[:, 65:70] = x, x, x
        _, _, y = round_trip(wide)
        assert torch.equal(y, want(wide)) and torch.isfinite(y).all()


def test_fp32_extremes(cuda_lib):
    big, small = torch.finfo(torch.float32).max, 2.0 ** -149
    x = torch.zeros(4, 64, device=DEV)
    x[0, 0], x[0, 40], x[1, 0], x[1, 33], x[2, 5], x[3, :] = big, -big, small, 2.0 ** -127, 2.0 ** -120, 2.0 ** -126
    _, scales, y = round_trip(x)
    assert torch.equal(y, want(x))
    assert float(y[0, 0]) == 127 * 2.0 ** 121 and int(scales[0, 0]) == 254 and int(scales[2, 1]) == 7


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_bad_value_spoils_its_group_alone(cuda_lib, dtype, bad):
    x = torch.randn(5, 100, device=DEV).to(dtype)
    x[1, 3] = x[2, 31] = x[3, 99] = x[4, 32] = bad
    codes, scales, y = round_trip(x)
    torch.testing.assert_close(y, want(x), rtol=0, atol=0, equal_nan=True)
    assert torch.isnan(y[1, :32]).all() and torch.isnan(y[3, 96:]).all() and int(torch.isnan(y).sum()) == 32 + 32 + 4 + 32
    assert int(scales[1, 0]) == 255 and not codes[1, :32].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_and_exponent_unpacks(cuda_lib, dtype):
    """All pairs that pack_8bit can write, and the ones that it cannot (code -128, exponent bytes below 7)."""
    codes = torch.arange(-128, 128, device=DEV).to(torch.int8).expand(256, 256)
    e = torch.arange(256, device=DEV)
    scales = e.to(torch.uint8).unsqueeze(1).expand(256, 8)
    rows = (e >= 7) & (e < 255)
    y = la.unpack_8bit(codes, scales, dtype)
    v = codes.double() * torch.exp2(e.double() - 133).unsqueeze(1)
    if dtype == torch.float16:
        v = v.clamp(-65504, 65504)
    elif dtype == torch.float32:
        v = v.float()  # -128 at the highest exponent is past the type
    assert torch.equal(y[rows], v.to(dtype)[rows])
    assert torch.isnan(y[255]).all()


@pytest.mark.parametrize("n", [64, 100, 33, 4096])
def test_strides(cuda_lib, n):
    torch.manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16):
        base = torch.randn(6, n, device=DEV).to(dtype)
        wide = torch.zeros(6, 2 * n + 3, device=DEV, dtype=dtype)
        wide[:, 3:n + 3] = base
        ref = la.pack_8bit(base)
        for x in (wide[:, 3:n + 3], base.t().contiguous().t(), torch.cat([base[:1], base]).reshape(-1)[n:].view(6, n)):
            got = la.pack_8bit(x)
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        one = la.pack_8bit(base[:1].expand(6, n))
        assert torch.equal(one[0], ref[0][:1].expand(6, n))
        wide8 = torch.zeros(6, 2 * n + 3, device=DEV, dtype=torch.int8)
        wide8[:, 3:n + 3] = ref[0]
        assert torch.equal(la.unpack_8bit(wide8[:, 3:n + 3], ref[1].t().contiguous().t(), dtype), la.unpack_8bit(*ref, dtype))


def test_empty_and_refused(cuda_lib):
    codes, scales = la.pack_8bit(torch.zeros(0, 100, device=DEV))
    assert codes.shape == (0, 100) and scales.shape == (0, 4) and la.unpack_8bit(codes, scales).shape == (0, 100)
    x = torch.zeros(4, 64, device=DEV)
    codes, scales = la.pack_8bit(x)
    for bad in ((x.sum(),), (x[:, :0],)):
        with pytest.raises(RuntimeError, match="at least one value"):
            la.pack_8bit(*bad)
    with pytest.raises(TypeError, match="unsupported dtype"):
        la.pack_8bit(x.double())
    with pytest.raises(TypeError, match="unsupported dtype"):
        la.unpack_8bit(codes, scales, torch.float64)
    for c, s in ((codes.int(), scales), (codes, scales.int()), (codes, scales[:, :1]), (codes, scales[:2]), (codes[0, 0], scales[0, 0])):
        with pytest.raises(RuntimeError, match="expected int8 codes"):
            la.unpack_8bit(c, s)


def test_captured(cuda_lib):
    x = torch.randn(300, 100, device=DEV).bfloat16()
    round_trip(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, _, y = round_trip(x)
    x.copy_(torch.randn(300, 100, device=DEV))
    graph.replay()
    assert torch.equal(y, want(x))


def test_more_than_two_to_the_31_elements(cuda_lib):
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    for shape in ((135000, 16384), (22_000_000, 100)):
        x = torch.ones(shape, device=DEV, dtype=torch.bfloat16)
        x[-8:] = torch.randn(8, shape[1], device=DEV).bfloat16()
        codes, scales, y = round_trip(x)
        assert torch.equal(y[-8:], want(x[-8:])) and bool((y[:-8] == 1).all())
        del x, codes, scales, y


@pytest.mark.parametrize("b,h,n,d,e", [(1, 2, 1, 16, 16), (2, 4, 300, 64, 64), (1, 4, 2048, 128, 128), (2, 3, 129, 80, 48), (1, 2, 200, 192, 192), (1, 2, 100, 20, 36), (1, 1, 140, 272, 64)])
@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_gradients_at_the_checkpoints_values(cuda_lib, b, h, n, d, e, decay, dtype):
    """Forward as without; gradients those of the operator at what the checkpoints of q, k, v stand for."""
    torch.manual_seed(0)
    q, k, v, do = ((0.3 * torch.randn(b, h, n, w, device=DEV)).to(dtype).requires_grad_() for w in (d, d, e, e))
    s = la._build_slope_tensor(h).to(DEV) if decay else None
    o = la.lightning_attn_func(q, k, v, s, save_8bit=True)
    assert torch.equal(o, la.lightning_attn_func(q, k, v, s))
    got = torch.autograd.grad(o, (q, k, v), do.detach())
    if d > 256:  # kept in slices of 256, with groups that begin anew in each
        parts = lambda t: torch.cat([want(t[..., lo:lo + 256]) for lo in range(0, d, 256)], -1)
    else:
        parts = want
    q8, k8, v8 = (f(t).requires_grad_() for f, t in ((parts, q), (parts, k), (want, v)))
    ref = torch.autograd.grad(la.lightning_attn_func(q8, k8, v8, s), (q8, k8, v8), do.detach())
    for a, r in zip(got, ref):
        # the same kernels on the same values; where the other call kept its forward pass's chunk states, they are summed in another order
        assert float((a.double() - r.double()).norm()) <= 1e-2 * float(r.double().norm())
    assert all(torch.equal(a, r) for a, r in zip(got, ref)) or n >= 1024


def test_attention_keeps_8_bits(cuda_lib):
    q = torch.randn(2, 4, 4096, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    s = la._build_slope_tensor(4).to(DEV)
    held = {}
    for save_8bit in (False, True):
        a, k, v = q * 1.0, q * 2.0, q * 3.0
        before = torch.cuda.memory_allocated()
        o = la.lightning_attn_func(a, k, v, s, save_8bit=save_8bit)
        del a, k, v
        held[save_8bit] = torch.cuda.memory_allocated() - before
        del o
    assert held[True] - held[False] <= -3 * q.numel() * 2 + 3 * (q.numel() + q.numel() // 32) + 65536
    with torch.no_grad():
        assert not la.lightning_attn_func(q, q, q, s, save_8bit=True).requires_grad
