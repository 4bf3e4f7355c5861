"""Plain 64-bit implementations of the layer norms and the 8-bit checkpoints, and what the fp32 kernels may be off by.

Bounds count roundings, u = 2^-24 each, plus half a step of the output's type. K = 64 + N / 32 roundings cover one row's arithmetic:
a thread adds at most N / 32 of its row's values one after the other (fewer where more threads share a row), then ten partial sums are
joined and about fifty operations of one rounding each follow, two of them approximate to 2^-22 (exponential, division).
The exponential adds its argument's rounding; past a gate of 100 the sigmoid is within 2^-100 of its limits, which is added as such."""
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def checkpoint64(x, group=32):
    """The values that the 8-bit checkpoint of x stands for (before any rounding to x's type), from the format's definition."""
    x = x.detach().double()
    shape, n = x.shape, x.shape[-1]
    pad = -n % group
    x = torch.nn.functional.pad(x.reshape(-1, n), (0, pad)).view(-1, (n + pad) // group, group)
    top = x.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(top)
    e = torch.frexp(torch.where(finite & (top > 0), top, 1.0)).exponent.double() - 7  # largest value in [64, 128) steps
    e = torch.where(torch.round(top / torch.exp2(e)) > 127, e + 1, e)
    e = torch.where(top == 0, -126.0, e).clamp(-126, 121)
    step = torch.exp2(e)
    out = torch.where(finite, torch.round(x / step).clamp(-127, 127) * step, float("nan"))
    return out.reshape(-1, n + pad)[:, :n].reshape(shape)


def reference(x, gate, w, b, eps, dy=None, save_8bit=False):
    """{name: (value, bound)} in 64 bits: y, and with dy the gradients dx, dgate, dw, db. `bound` is without the output's rounding."""
    n = x.shape[-1]
    k = (64 + n / 32) * U
    rows = lambda t: None if t is None else t.detach().double().reshape(-1, n)
    x64, g64 = rows(x), rows(gate)
    w64 = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b64 = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    mean = x64.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x64 - mean).square().mean(1, keepdim=True) + eps)
    top = x64.abs().amax(1, keepdim=True)
    sig = lambda t: 1 / (1 + torch.exp(-t))
    z = (x64 - mean) * rstd
    y = z * w64 + b64
    off = k * (z.abs() * w64.abs() + b64.abs()) + 4 * U * top * rstd * w64.abs()
    if gate is not None:
        s = sig(g64)
        y, off = y * s, (off + (k + 4 * U * g64.abs().clamp(max=100)) * y.abs()) * s + 2.0 ** -100
    out = {"y": (y.reshape(x.shape), off.reshape(x.shape))}
    if dy is None:
        return out
    m = x64.shape[0]
    t = rows(dy)
    xs = rows(checkpoint64(x)) if save_8bit else x64
    z = (xs - mean) * rstd
    # the mean is kept in fp32: half a step of it, and what its sum was off by
    zoff = k * z.abs() + 4 * U * (xs.abs().amax(1, keepdim=True) + mean.abs()) * rstd
    toff = torch.zeros_like(t)
    if gate is not None:
        gs = rows(checkpoint64(gate)) if save_8bit else g64
        s, rest = sig(gs), sig(-gs)
        nv = z * w64 + b64
        dg = t * nv * s * rest
        dgoff = t.abs() * s * rest * ((zoff + k * z.abs()) * w64.abs() + k * b64.abs()) + (k + 8 * U * gs.abs().clamp(max=100)) * dg.abs() + 2.0 ** -100
        out["dgate"] = (dg.reshape(x.shape), dgoff.reshape(x.shape))
        t = t * s
        toff = (k + 4 * U * gs.abs().clamp(max=100)) * t.abs() + 2.0 ** -100
    # sums over rows: one rounding of a partial sum for each row added; partial sums of values of either sign stay within four
    # times the root of the sum of squares (or, for few rows, within the sum of magnitudes)
    def over_rows(v, voff):
        partial = torch.minimum(4 * v.square().sum(0).sqrt(), v.abs().sum(0)) + v.sum(0).abs()
        return v.sum(0), voff.sum(0) + (m + 64) * U * partial
    out["db"] = over_rows(t, toff)
    out["dw"] = over_rows(t * z, toff * z.abs() + t.abs() * zoff + U * (t * z).abs())
    u, uoff = t * w64, toff * w64.abs() + U * (t * w64).abs()
    c1, c2 = u.mean(1, keepdim=True), (u * z).mean(1, keepdim=True)
    c1off = uoff.mean(1, keepdim=True) + k * u.abs().mean(1, keepdim=True)
    c2off = (uoff * z.abs() + u.abs() * zoff).mean(1, keepdim=True) + k * (u * z).abs().mean(1, keepdim=True)
    dx = (u - c1 - z * c2) * rstd
    dxoff = rstd * (uoff + c1off + zoff * c2.abs() + z.abs() * c2off + 4 * U * (u.abs() + c1.abs() + (z * c2).abs())) + k * dx.abs()
    out["dx"] = (dx.reshape(x.shape), dxoff.reshape(x.shape))
    return out


def assert_within(got, ref, name):
    """got within bound + half a step of its type (and the smallest step of its type) of the 64-bit value; NaN where that is."""
    value, off = ref
    assert got.shape == value.shape, f"{name}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    g = got.detach().double()
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(g), nan), f"{name}: NaN in other places than in the definition"
    far = (g - value).abs() - (off + HALF_STEP[got.dtype] * (value.abs() + off) + SMALLEST[got.dtype])
    far = torch.where(nan, torch.full_like(far, -1.0), far)
    if far.numel():
        worst = int(far.argmax())
        assert float(far.reshape(-1)[worst]) <= 0, (f"{name}[{worst}]: {float(g.reshape(-1)[worst])!r}, expected {float(value.reshape(-1)[worst])!r} "
                                                    f"+- {float(off.reshape(-1)[worst]):.3g} and half a step")
