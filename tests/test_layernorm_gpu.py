"""GPU tests of layer_norm and layer_norm_sigmoid_gate against their definition in 64 bits (tests/_ln_refs.py has the bounds)."""
import gc
import os
import sys
import threading

import pytest
import torch

import lightning_attention_b200 as la

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import assert_within, checkpoint64, reference  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-5


def inputs(m, n, dtype, wdtype=None, gated=False, seed=0, shift=0.3, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)
    x = (r(m, n) * scale * torch.exp(0.5 * r(n)) + shift).to(dtype).requires_grad_()
    gate = (2 * r(m, n)).to(dtype).requires_grad_() if gated else None
    w, b = ((1 + 0.3 * r(n)).to(wdtype or dtype).requires_grad_(), (0.3 * r(n)).to(wdtype or dtype).requires_grad_())
    return x, gate, w, b, r(m, n).to(dtype)


def call(x, gate, w, b, save_8bit=False, eps=EPS):
    if gate is None:
        return la.layer_norm(x, w, b, eps, save_8bit)
    return la.layer_norm_sigmoid_gate(x, gate, w, b, eps, save_8bit)


def fwd_bwd(x, gate, w, b, dy, save_8bit=False, eps=EPS):
    y = call(x, gate, w, b, save_8bit, eps)
    named = {k: t for k, t in (("dx", x), ("dgate", gate), ("dw", w), ("db", b)) if t is not None and t.requires_grad}
    return {"y": y.detach(), **dict(zip(named, torch.autograd.grad(y, list(named.values()), dy)))}


def check(x, gate, w, b, dy, save_8bit=False, eps=EPS, what=""):
    got = fwd_bwd(x, gate, w, b, dy, save_8bit, eps)
    ref = reference(x, gate, w, b, eps, dy, save_8bit)
    for name, t in got.items():
        assert t.dtype == (x.dtype if name in ("y", "dx", "dgate") else w.dtype if name == "dw" else b.dtype)
        assert_within(t, ref[name], f"{what}{name}")
    return got


SHAPES = [(1, 1), (3, 1), (1, 2), (5, 7), (2, 31), (2, 33), (4, 32), (9, 48), (257, 64), (300, 128), (33, 192), (65, 240), (17, 256), (21, 264), (40, 320),
          (130, 512), (17, 768), (9, 1000), (5, 1001), (2, 1023), (3, 1024), (19, 1040), (70, 2048), (5, 2056), (7, 4096), (6, 4104), (5, 5120), (3, 8192),
          (4, 8200), (2, 10000), (2, 16384), (3, 16400), (2, 20001), (2, 40000), (1000, 96), (5000, 17), (2500, 200), (4099, 33)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["fp32", "fp16", "bf16"])
def test_sizes(cuda_lib, m, n, gated, dtype):
    for save_8bit in (False, True):
        for wdtype in {dtype, torch.float32}:
            check(*inputs(m, n, dtype, wdtype, gated), save_8bit=save_8bit, what=f"8bit={save_8bit} {wdtype} ")


@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
@pytest.mark.parametrize("m,n,dtype", [(8192, 1024, torch.bfloat16), (20000, 128, torch.float16), (3001, 4096, torch.bfloat16), (4100, 768, torch.float32)])
def test_many_rows(cuda_lib, m, n, dtype, gated):
    check(*inputs(m, n, dtype, torch.float32, gated))
    check(*inputs(m, n, dtype, torch.float32, gated, seed=1), save_8bit=True)


@pytest.mark.parametrize("m", [149, 445, 741])
@pytest.mark.parametrize("n", [4104, 5120, 6144, 6152, 8192])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_wide_rows(cuda_lib, m, n, dtype):
    """Rows of which an SM has one or two teams, with a last turn that some teams have no row for."""
    for gated in (False, True):
        for save_8bit in (False, True):
            check(*inputs(m, n, dtype, torch.float32, gated), save_8bit=save_8bit, what=f"gate={gated} 8bit={save_8bit} ")


@pytest.mark.parametrize("n", [7776, 7784, 8192, 11872, 11880, 12000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_rows_that_fill_shared_memory(cuda_lib, n, dtype):
    """Lengths on both sides of those at which the gated forward kernel has room for its copies."""
    for save_8bit in (False, True):
        check(*inputs(299, n, dtype, torch.float32, True), save_8bit=save_8bit, what=f"8bit={save_8bit} ")


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("n", [100, 1024, 1001])
def test_without_weight_or_bias(cuda_lib, n, has_w, has_b):
    for gated in (False, True):
        x, gate, w, b, dy = inputs(9, n, torch.bfloat16, torch.float32, gated)
        check(x, gate, w if has_w else None, b if has_b else None, dy)


def test_module_matches_function_and_torch(cuda_lib):
    torch.manual_seed(0)
    m, t = la.LayerNorm(768, device=DEV), torch.nn.LayerNorm(768, device=DEV)
    x = torch.randn(4, 33, 768, device=DEV, requires_grad=True)
    y = m(x)
    assert torch.equal(y, la.layer_norm(x, m.weight, m.bias))
    torch.testing.assert_close(y, t(x), rtol=1e-5, atol=1e-5)
    gate = torch.randn_like(x)
    assert torch.equal(m(x, gate), la.layer_norm_sigmoid_gate(x, gate, m.weight, m.bias))
    assert la.LayerNorm(768, device=DEV, dtype=torch.bfloat16)(x.bfloat16()).dtype == torch.bfloat16


def _views(m, n, dtype, seed):
    """The same values in other strides: a column slice (aligned or not), every second row, a transposed tensor, an odd offset, a broadcast row."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    base = torch.randn(m, n, generator=g, device=DEV).to(dtype)
    wide = torch.zeros(m, 3 * n, device=DEV, dtype=dtype)
    wide[:, n:2 * n] = base
    odd = torch.zeros(m, 2 * n + 1, device=DEV, dtype=dtype)
    odd[:, 1:n + 1] = base
    every = torch.zeros(2 * m, n, device=DEV, dtype=dtype)
    every[::2] = base
    flat = torch.zeros(m * n + 1, device=DEV, dtype=dtype)
    flat[1:] = base.reshape(-1)
    return {"slice": wide[:, n:2 * n], "odd slice": odd[:, 1:n + 1], "every second": every[::2], "transposed": base.t().contiguous().t(),
            "offset": flat[1:].view(m, n)}, base


@pytest.mark.parametrize("m,n", [(6, 64), (5, 100), (3, 1024), (4, 2048), (2, 4100), (3, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strides(cuda_lib, m, n, dtype):
    xs, x = _views(m, n, dtype, 1)
    gs, gate = _views(m, n, dtype, 2)
    dys, dy = _views(m, n, dtype, 3)
    _, _, w, b, _ = inputs(m, n, dtype)
    for save_8bit in (False, True):
        for kind in xs:
            check(xs[kind].requires_grad_(), None, w, b, dys[kind], save_8bit, what=f"{kind} ")
            check(xs[kind].requires_grad_(), gs[kind].requires_grad_(), w, b, dys[kind], save_8bit, what=f"{kind} gated ")
    row = x[:1].expand(m, n).requires_grad_()
    check(row, gate[:1].expand(m, n).requires_grad_(), w, b, dy, what="broadcast ")
    check(x.requires_grad_(), None, w, b, torch.ones((), device=DEV, dtype=dtype).expand(m, n), what="broadcast dy ")
    x3 = x.detach().reshape(1, m, 1, n).requires_grad_()
    y = la.layer_norm(x3, w, b)
    assert y.shape == x3.shape and torch.autograd.grad(y, x3, dy.view_as(y))[0].shape == x3.shape


@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
@pytest.mark.parametrize("m,n", [(5, 100), (3, 33), (4, 2052), (2, 12000), (40, 9)])
def test_c_entry_reads_any_stride_and_alignment(cuda_lib, m, n, gated):
    """lab200_layernorm_fwd / _bwd on rows that no pack of 16 bytes divides, which the Python operators copy."""
    from lightning_attention_b200 import _lib

    L = cuda_lib
    x, gate, w, b, dy = inputs(m, n, torch.bfloat16, torch.float32, gated)
    ref = reference(x, gate, w, b, EPS, dy)
    ld = n + 3
    wide = torch.full((3, m * ld + 1), float("nan"), device=DEV, dtype=torch.bfloat16)

    def odd(k, t):
        v = wide[k][1:].view(m, ld)[:, :n]
        return v.copy_(t.detach())

    xv, dyv = odd(0, x), odd(1, dy)
    gv = odd(2, gate) if gated else None
    y, dx, dg = (torch.full((m * n + 64,), 7.0, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    stats = torch.empty(m, 2, device=DEV)
    dw, db = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    s = torch.cuda.current_stream().cuda_stream
    p = _lib.ptr
    wd, bd = w.detach(), b.detach()
    assert L.lab200_layernorm_fwd(p(xv), ld, p(gv), ld, p(wd), p(bd), _lib.F32, p(y), p(stats), None, None, None, None, m, n, EPS, _lib.BF16, s) == 0
    nbytes = L.lab200_layernorm_bwd_workspace_bytes(m, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    assert L.lab200_layernorm_bwd(p(xv), ld, p(gv), ld, None, None, None, None, p(stats), p(dyv), ld, p(wd), p(bd), _lib.F32, p(dx), p(dg) if gated else None, p(dw),
                                  p(db), p(ws), nbytes, m, n, _lib.BF16, s) == 0
    for name, t in (("y", y), ("dx", dx), *((("dgate", dg),) if gated else ())):
        assert_within(t[:m * n].view(m, n), ref[name], name)
        assert bool((t[m * n:] == 7).all()), f"{name}: written behind the last row"
    assert_within(dw, ref["dw"], "dw")
    assert_within(db, ref["db"], "db")


@pytest.mark.parametrize("n", [33, 64, 100, 1001, 2048, 5120])
@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
def test_nothing_is_written_outside_the_outputs(cuda_lib, n, gated):
    """Guards around every output of the C entries, in both directions, with and without checkpoints."""
    from lightning_attention_b200 import _lib

    L, m = cuda_lib, 37
    p = _lib.ptr
    x, gate, w, b, dy = (None if t is None else t.detach() for t in inputs(m, n, torch.bfloat16, torch.float32, gated))
    ng = (n + 31) // 32
    s = torch.cuda.current_stream().cuda_stream

    def guarded(count, dtype):
        t = torch.full((count + 256,), 77, device=DEV, dtype=dtype)
        return t, t[128:128 + count]

    outs = {k: guarded(m * n, torch.bfloat16) for k in ("y", "dx", "dg")}
    outs |= {"stats": guarded(2 * m, torch.float32), "dw": guarded(n, torch.float32), "db": guarded(n, torch.float32)}
    outs |= {k: guarded(m * n, torch.int8) for k in ("xc", "gc")} | {k: guarded(m * ng, torch.uint8) for k in ("xs", "gs")}
    o = {k: v[1].data_ptr() for k, v in outs.items()}
    gcs = (o["gc"], o["gs"]) if gated else (None, None)
    assert L.lab200_layernorm_fwd(p(x), n, p(gate), n, p(w), p(b), _lib.F32, o["y"], o["stats"], o["xc"], o["xs"], *gcs, m, n, EPS, _lib.BF16, s) == 0
    nbytes = L.lab200_layernorm_bwd_workspace_bytes(m, n)
    ws_all, ws = guarded(nbytes, torch.uint8)
    for saved in (False, True):
        src = (None, n, None, n, o["xc"], o["xs"], *gcs) if saved else (p(x), n, p(gate), n, None, None, None, None)
        assert L.lab200_layernorm_bwd(*src, o["stats"], p(dy), n, p(w), p(b), _lib.F32, o["dx"], o["dg"] if gated else None, o["dw"], o["db"], ws.data_ptr(), nbytes,
                                      m, n, _lib.BF16, s) == 0
        ref = reference(x, gate, w, b, EPS, dy, saved)
        assert_within(outs["dx"][1].view(m, n), ref["dx"], "dx")
        assert_within(outs["dw"][1], ref["dw"], "dw")
    for k, (whole, part) in list(outs.items()) + [("ws", (ws_all, ws))]:
        assert bool((whole[:128] == 77).all()) and bool((whole[128 + part.numel():] == 77).all()), f"written outside {k}"


def test_every_subset_of_gradients(cuda_lib):
    x, gate, w, b, dy = inputs(40, 192, torch.bfloat16, torch.float32, True)
    full = fwd_bwd(x, gate, w, b, dy)
    for mask in range(1, 16):
        ts = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, gate, w, b))]
        part = fwd_bwd(*ts, dy)
        assert len(part) == 1 + bin(mask).count("1")
        for k, v in part.items():
            assert torch.equal(v, full[k]), (mask, k)
    with torch.no_grad():
        y = la.layer_norm_sigmoid_gate(x, gate, w, b, save_8bit=True)
    assert not y.requires_grad and torch.equal(y, full["y"])


def test_no_rows(cuda_lib):
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w, b = torch.ones(64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True)
    for save_8bit in (False, True):
        y = la.layer_norm(x, w, b, save_8bit=save_8bit)
        assert y.shape == (0, 64)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_values_at_the_border(cuda_lib):
    """Constant rows, rows far from zero, rows of the largest and smallest magnitudes, gates where exp overflows."""
    n = 512
    x, gate, w, b, dy = inputs(8, n, torch.float32, gated=True)
    with torch.no_grad():
        x[0] = 3.0
        x[1] = 0.0
        x[2] += 5000.0
        x[3] *= 1e-12
        x[4] *= 1e15
        gate[5, 0::2], gate[5, 1::2] = 200.0, -200.0
        gate[6, 0], gate[6, 1], gate[6, 2], gate[6, 3] = 88.5, -88.5, 1e30, -1e30
        gate[7, 0], gate[7, 1] = float("inf"), -float("inf")
    got = check(x, gate, w, b, dy)
    assert torch.equal(fwd_bwd(x, None, w, b, dy)["y"][0], b.detach())
    assert all(torch.isfinite(t).all() for t in got.values())


@pytest.mark.parametrize("save_8bit", [False, True])
@pytest.mark.parametrize("n", [100, 1024, 1001, 5120])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_value_stays_in_its_row(cuda_lib, n, bad, save_8bit):
    x, gate, w, b, dy = inputs(7, n, torch.bfloat16, gated=True)
    clean = fwd_bwd(x, gate, w, b, dy, save_8bit)
    with torch.no_grad():
        x[3, n // 2] = bad
    got = fwd_bwd(x, gate, w, b, dy, save_8bit)
    others = [i for i in range(7) if i != 3]
    assert torch.isnan(got["y"][3]).all() and torch.isnan(got["dx"][3]).all() and torch.isnan(got["dw"]).all()
    for k in ("y", "dx", "dgate"):
        assert torch.equal(got[k][others], clean[k][others]), k
    assert torch.equal(got["db"], clean["db"])


def test_same_results_every_time(cuda_lib):
    for m, n in ((3000, 1024), (5000, 100), (333, 8192)):
        args = inputs(m, n, torch.bfloat16, torch.float32, True)
        first = fwd_bwd(*args)
        for _ in range(3):
            again = fwd_bwd(*args)
            assert all(torch.equal(first[k], again[k]) for k in first)


def test_gradient_against_differences(cuda_lib):
    """The kernel's forward pass along a direction: the central difference may be off by the roundings of y over 2 h and by its third
    derivative, which the 64-bit definition's own difference shows."""
    x, gate, w, b, dy = inputs(6, 96, torch.float32, gated=True)
    got = fwd_bwd(x, gate, w, b, dy)
    h = 2.0 ** -7
    g = torch.Generator(device=DEV).manual_seed(5)
    for i, (t, name) in enumerate(((x, "dx"), (gate, "dgate"), (w, "dw"), (b, "db"))):
        v = torch.randn(t.shape, generator=g, device=DEV)

        def moved(sign, i=i, v=v):
            ts = [u.detach().clone() for u in (x, gate, w, b)]
            ts[i] += sign * h * v
            return ts

        up, down = moved(1), moved(-1)
        along = ((up[i].double() - down[i].double()) / (2 * h))  # the direction as rounded
        diff = lambda f: float(((f(up) - f(down)) * dy.double()).sum()) / (2 * h)
        mine = diff(lambda ts: call(*ts).double())
        exact = diff(lambda ts: reference(*ts, EPS)["y"][0])
        slope = float((reference(x, gate, w, b, EPS, dy)[name][0] * along).sum())
        ref = [reference(*ts, EPS)["y"] for ts in (up, down)]
        rounding = sum(float(((off + 2.0 ** -24 * y.abs()) * dy.double().abs()).sum()) for y, off in ref) / (2 * h)
        got_slope = float((got[name].double() * along).sum())
        assert abs(mine - got_slope) <= rounding + abs(exact - slope) + 1e-5 * abs(slope) + 1e-5, name


def test_differentiable_once(cuda_lib):
    x, _, w, b, dy = inputs(4, 64, torch.float32)
    for save_8bit in (False, True):
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(la.layer_norm(x, w, b, save_8bit=save_8bit), x, dy, create_graph=True)


def test_changed_input_is_noticed_and_a_checkpoint_does_not_mind(cuda_lib):
    x, _, w, b, dy = inputs(4, 64, torch.float32)
    z = x * 1.0
    y = la.layer_norm(z, w, b)
    z += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    want = fwd_bwd(x, None, w, b, dy, True)["dx"]
    z = x * 1.0
    y = la.layer_norm(z, w, b, save_8bit=True)
    z += 1
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def test_a_checkpoint_is_what_is_kept(cuda_lib):
    """The memory between the passes: 8.25 bits a value and the row statistics in place of the tensors."""
    m, n = 4096, 1024
    base = torch.randn(m, n, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    held = {}
    for save_8bit in (False, True):
        x, gate = base * 1.0, base * 2.0
        before = torch.cuda.memory_allocated()
        y = la.layer_norm_sigmoid_gate(x, gate, save_8bit=save_8bit)
        del x, gate
        held[save_8bit] = torch.cuda.memory_allocated() - before - m * n * 2  # without y
        del y
    assert held[False] <= m * 8 + 4096 and held[True] <= -2 * m * n * 2 + 2 * (m * n + m * n // 32) + m * 8 + 8192


def test_saved_tensor_hooks_may_change_strides(cuda_lib):
    for save_8bit in (False, True):
        x, gate, w, b, dy = inputs(20, 96, torch.bfloat16, gated=True)
        want = fwd_bwd(x, gate, w, b, dy, save_8bit)
        twist = lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu(), lambda t: twist(t.to(DEV))):
            got = fwd_bwd(x, gate, w, b, dy, save_8bit)
        assert all(torch.equal(got[k], want[k]) for k in want)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t[:1]):
            with pytest.raises(RuntimeError, match="hooks returned another shape"):
                fwd_bwd(x, gate, w, b, dy, save_8bit)


def test_refusals(cuda_lib):
    x = torch.zeros(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    for args, match in (((x, w[:32]), "weight must have shape"), ((x, w, w[:1]), "bias must have shape"), ((x.bfloat16(), w.half()), "x's dtype or float32"),
                        ((x, w.bfloat16()), "x's dtype or float32"), ((x.bfloat16(), w.bfloat16(), w), "share one dtype"), ((x, w, w, -1.0), "eps"),
                        ((x, w, w, float("nan")), "eps"), ((x, w.cpu()), "CUDA tensors only"), ((x[:, :0],), "at least one value"), ((x.sum(),), "at least one value")):
        with pytest.raises(RuntimeError, match=match):
            la.layer_norm(*args)
    for gate in (x[:2], x.bfloat16(), x[:, :32]):
        with pytest.raises(RuntimeError, match="gate must match"):
            la.layer_norm_sigmoid_gate(x, gate)
    with pytest.raises(RuntimeError, match="needs a gate"):
        la.layer_norm_sigmoid_gate(x, None)
    with pytest.raises(TypeError, match="unsupported dtype"):
        la.layer_norm(x.double())


def test_rows_past_what_the_kernels_count_are_refused(cuda_lib):
    x = torch.zeros(1, device=DEV).expand(2, (1 << 32) + 64)
    for call in (lambda: la.layer_norm(x), lambda: la.layer_norm_sigmoid_gate(x, x), lambda: la.pack_8bit(x)):
        with pytest.raises(RuntimeError, match="at most 2\\^30"):
            call()


@pytest.mark.parametrize("m,n", [(300, 1024), (9, 1001), (40, 5120)])
def test_one_tensor_in_two_places(cuda_lib, m, n):
    """x as its own gate, and the weight as the bias: gradients add up; a gradient that is the input itself."""
    for save_8bit in (False, True):
        x, _, w, _, _ = inputs(m, n, torch.float32)
        both = fwd_bwd(x, x.detach().clone().requires_grad_(), w, w.detach().clone().requires_grad_(), x.detach(), save_8bit)
        y = call(x, x, w, w, save_8bit)
        dx, dw = torch.autograd.grad(y, (x, w), x.detach())
        assert torch.equal(y.detach(), both["y"]) and torch.equal(dx, both["dx"] + both["dgate"]) and torch.equal(dw, both["dw"] + both["db"])


def test_side_stream_and_two_threads(cuda_lib):
    args = inputs(700, 1024, torch.bfloat16, torch.float32, True)
    want = fwd_bwd(*args)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = fwd_bwd(*args)
                if not all(torch.equal(got[k], want[k]) for k in want):
                    bad.append(1)
        s.synchronize()

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.parametrize("save_8bit", [False, True])
def test_captured_and_replayed(cuda_lib, save_8bit):
    """Forward and backward in one graph, replayed on new values, two graphs in turn; no eager graph of the leaves lives meanwhile."""
    gc.collect()
    made = []
    for m, n in ((300, 1024), (77, 1000)):
        x, gate, w, b, dy = inputs(m, n, torch.bfloat16, torch.float32, True)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fwd_bwd(x, gate, w, b, dy, save_8bit)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fwd_bwd(x, gate, w, b, dy, save_8bit)
        made.append((graph, out, (x, gate, w, b, dy)))
    for seed in (3, 4):
        for graph, out, args in made:
            with torch.no_grad():
                for t, new in zip(args, inputs(*args[0].shape, torch.bfloat16, torch.float32, True, seed=seed)):
                    t.copy_(new)
        for graph, _, _ in made + made[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, args in made:
            want = fwd_bwd(*args, save_8bit)
            assert all(torch.equal(out[k], want[k]) for k in want)


def test_more_than_two_to_the_31_elements(cuda_lib):
    """Offsets past 32 bits: the last rows of a tensor of 2.2e9 values, against the same rows alone."""
    m, n = 135000, 16384
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
    tail = torch.randn(64, n, device=DEV).bfloat16()
    x[:-64] = 1.0
    x[-64:] = tail
    x.requires_grad_()
    y = la.layer_norm(x, save_8bit=True)
    dy = x.detach()
    (dx,) = torch.autograd.grad(y, x, dy)
    small = tail.clone().requires_grad_()
    ys = la.layer_norm(small, save_8bit=True)
    (dxs,) = torch.autograd.grad(ys, small, tail)
    assert torch.equal(y[-64:], ys) and torch.equal(dx[-64:], dxs)
    assert not y[:-64].any()


def test_norm_gate_and_attention_together(cuda_lib):
    """An attention block's middle, everything kept in 8 bits: the gradients against the same chain with each operator's input replaced
    by what its checkpoint stands for, computed by the framework's unsaved operators on those values."""
    b, n, h, d = 2, 300, 4, 64
    torch.manual_seed(0)
    q, k, v = ((torch.randn(b, n, h, d, device=DEV) * 0.3).bfloat16().requires_grad_() for _ in range(3))
    gate = torch.randn(b, n, h * d, device=DEV).bfloat16().requires_grad_()
    norm = la.LayerNorm(h * d, save_8bit=True, device=DEV)
    s = la._build_slope_tensor(h).to(DEV)
    dy = torch.randn(b, n, h * d, device=DEV).bfloat16()
    o = la.lightning_attn_func(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), s, save_8bit=True)
    mid = o.transpose(1, 2).reshape(b, n, h * d)
    y = norm(mid, gate)
    dq, dk, dv, dg, dw = torch.autograd.grad(y, (q, k, v, gate, norm.weight), dy)
    ref = reference(mid, gate, norm.weight, norm.bias, norm.eps, dy, True)
    assert_within(y, ref["y"], "y")
    assert_within(dg, ref["dgate"], "dgate")
    assert_within(dw, ref["dw"], "dw")
    go = torch.autograd.grad(norm(m2 := mid.detach().requires_grad_(), gate), m2, dy)[0]
    q8, k8, v8 = (checkpoint64(t).bfloat16().transpose(1, 2).requires_grad_() for t in (q, k, v))
    o8 = la.lightning_attn_func(q8, k8, v8, s)
    want = torch.autograd.grad(o8, (q8, k8, v8), go.view(b, n, h, d).transpose(1, 2))
    for got, ref in zip((dq, dk, dv), want):
        assert torch.equal(got, ref.transpose(1, 2))


@pytest.mark.parametrize("gated", [False, True], ids=["norm", "gate"])
@pytest.mark.parametrize("save_8bit", [False, True])
@pytest.mark.parametrize("has_w,has_b", [(True, True), (True, False), (False, True), (False, False)])
def test_native_and_python_paths_agree(cuda_lib, monkeypatch, gated, save_8bit, has_w, has_b):
    """csrc/host_ops.cpp and the autograd class: the same results, the same tensors kept, the same refusals."""
    from lightning_attention_b200 import _lib

    x, gate, w, b, dy = inputs(33, 192, torch.bfloat16, torch.float32, gated)
    w, b = w if has_w else None, b if has_b else None

    def everything():
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append((tuple(t.shape), t.dtype)) or t, lambda t: t):
            y = call(x, gate, w, b, save_8bit)
        assert torch.equal(call(x[::2], None if gate is None else gate[::2], w, b, save_8bit), y[::2])
        leaves = [t for t in (x, gate, w, b) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)], kept

    native, kept = everything()
    assert type(call(x, gate, w, b, save_8bit).grad_fn).__name__ == "CppFunction"
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    python, kept_python = everything()
    assert all(torch.equal(u, v) for u, v in zip(native, python)) and kept == kept_python
    codes, scales = la.pack_8bit(x)
    y = la.unpack_8bit(codes, scales)
    monkeypatch.undo()
    assert all(torch.equal(u, v) for u, v in zip(la.pack_8bit(x), (codes, scales))) and torch.equal(la.unpack_8bit(codes, scales), y)


def test_no_graph_without_gradients(cuda_lib):
    x, gate, w, b, _ = inputs(5, 64, torch.bfloat16, gated=True)
    with torch.no_grad():
        assert la.layer_norm(x, w, b).grad_fn is None
    with torch.inference_mode():
        y = la.layer_norm_sigmoid_gate(x.detach().clone(), gate.detach().clone(), w.detach().clone(), b.detach().clone())
    assert not y.requires_grad
    plain = [t.detach() for t in (x, w, b)]
    assert la.layer_norm(*plain).grad_fn is None
