"""What the layer norms and the 8-bit activation checkpoints are measured on: a list of cases, a generator of more of the same
ranges, each operator's plain form and its definition in 64 bits.

Kinds of case, each one pass through public entry points:

  serve  layer_norm of the tokens of one decoding step, no gradients
  train  layer_norm forward and backward, with the gradients of weight and bias
  gate   layer_norm_sigmoid_gate forward and backward: what an attention block does between its attention and its output projection
  pack   pack_8bit of a tensor and unpack_8bit of what that gave

In train and gate, `save8` says that the backward pass works from 8-bit checkpoints of x (and of the gate).
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
GROUP = 32  # values that share one exponent in a checkpoint
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST = 1 << 27  # elements of the largest listed case


def _case(name, kind, rows, dim, dtype="bf16", wdtype=None, save8=False, sliced=False):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype, "wdtype": wdtype or dtype, "save8": save8, "sliced": sliced}


def listed():
    return [
        # serving: one token of one sequence, bound by latency
        _case("serve_1x2048", "serve", 1, 2048),
        # the smallest training call: one short fp32 sequence of the norm tests' list
        _case("train_fp32_257x768", "train", 257, 768, dtype="fp32"),
        # the hidden states of an ordinary training batch, parameters kept in fp32
        _case("train_8192x2048", "train", 8192, 2048, wdtype="fp32"),
        # a width that no vector divides, fp16
        _case("train_fp16_4099x1001", "train", 4099, 1001, dtype="fp16"),
        # the hidden states of a long-context training batch
        _case("train_32768x4096", "train", 32768, 4096),
        # a wide model whose norm inputs are checkpointed in 8 bits
        _case("train_save8_16384x5120", "train", 16384, 5120, wdtype="fp32", save8=True),
        # norm and gate of every head's output by itself: many short rows
        _case("gate_heads_131072x128", "gate", 131072, 128),
        # norm and gate of an attention block; the gate is one part of a wider projection
        _case("gate_sliced_8192x2048", "gate", 8192, 2048, wdtype="fp32", sliced=True),
        # the same for a long context, x and gate checkpointed in 8 bits
        _case("gate_save8_32768x4096", "gate", 32768, 4096, save8=True),
        # checkpoint of a small tensor of 192-wide heads: launches and host work
        _case("pack_300x192", "pack", 300, 192),
        # checkpoint of a width whose last group is short
        _case("pack_fp16_20000x1000", "pack", 20000, 1000, dtype="fp16"),
        # checkpoint of one attention operand of the benchmark's workload at n = 8192
        _case("pack_1048576x128", "pack", 4 * 32 * 8192, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["serve", "train", "train", "train", "gate", "gate", "gate", "pack", "pack"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    # head widths, model widths, and now and then any width at all
    dim = rng.choice([16 * rng.randint(2, 16), 256 * rng.randint(2, 32), 8 * rng.randint(16, 640), _log_int(rng, 33, 5000)])
    rows = _log_int(rng, 1, 512) if kind == "serve" else _log_int(rng, 16, MOST // (4 * dim))
    plain = kind in ("serve", "pack")
    wdtype = "fp32" if kind != "pack" and rng.random() < 0.4 else dtype
    c = _case("", kind, rows, dim, dtype, wdtype, save8=not plain and rng.random() < 0.4, sliced=kind == "gate" and rng.random() < 0.3)
    del c["name"]
    return c


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    kind, m, n, dt, wdt = case["kind"], case["rows"], case["dim"], DTYPES[case["dtype"]], DTYPES[case["wdtype"]]

    def rnd(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    grad = kind in ("train", "gate")
    # hidden states: every channel has a spread of its own, a few are much wider, and rows are not centred
    spread = torch.exp(0.5 * rnd(n)) * torch.where(rnd(n) > 2.5, 8.0, 1.0)
    st = {"kind": kind, "save8": case["save8"], "x": (rnd(m, n) * spread + 0.2 * rnd(m, 1)).to(dt).requires_grad_(grad)}
    if kind != "pack":
        st["w"] = (1.0 + 0.2 * rnd(n)).to(wdt).requires_grad_(grad)
        st["b"] = (0.1 * rnd(n)).to(wdt).requires_grad_(grad)
    if kind == "gate":
        wide = (1.5 * rnd(m, 2 * n if case["sliced"] else n)).to(dt)
        st["gate"] = wide[:, wide.shape[1] - n:].requires_grad_(True)
    if grad:
        st["dy"] = rnd(m, n).to(dt)
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def _through_8bit(x):
    """The values that the 8-bit checkpoint of x stands for, in fp32: a group of 32 shares the step 2^(E - 133), where E is the
    exponent field of the group's largest magnitude, one more where that would round to 128 steps."""
    m, n = x.shape
    pad = -n % GROUP
    f = torch.nn.functional.pad(x.detach().float(), (0, pad)).view(m, -1, GROUP)
    field = ((f.abs().amax(-1).view(torch.int32) + 0x10000) >> 23).clamp(7, 254)
    step = torch.pow(2.0, (field - 133).double()).float().unsqueeze(-1)
    return (torch.round(f / step).clamp(-127, 127) * step).view(m, -1)[:, :n]


def _stats(x):
    mean = x.mean(-1, keepdim=True)
    return mean, 1.0 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + EPS)


def _plain(st):
    kind, x = st["kind"], st["x"]
    if kind == "pack":
        return {"x8": _through_8bit(x).to(x.dtype)}
    f, w, b = x.detach().float(), st["w"].detach().float(), st["b"].detach().float()
    mean, rstd = _stats(f)
    y = (f - mean) * rstd * w + b
    if kind == "gate":
        gate = st["gate"].detach().float()
        y = y / (1.0 + torch.exp(-gate))
    out = {"y": y.to(x.dtype)}
    if kind == "serve":
        return out
    del y
    if st["save8"]:
        f = _through_8bit(x)
    dy = st["dy"].float()
    xh = (f - mean) * rstd
    del f
    if kind == "gate":
        if st["save8"]:
            gate = _through_8bit(st["gate"])
        sg = 1.0 / (1.0 + torch.exp(-gate))
        out["dgate"] = (dy * (xh * w + b) * sg * (1.0 / (1.0 + torch.exp(gate)))).to(x.dtype)
        dy = dy * sg
        del sg, gate
    out["db"] = dy.sum(0).to(st["b"].dtype)
    out["dw"] = (dy * xh).sum(0).to(st["w"].dtype)
    g = dy * w
    out["dx"] = ((g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rstd).to(x.dtype)
    return out


def _own(st):
    import lightning_attention_b200 as la

    kind, x = st["kind"], st["x"]
    if kind == "pack":
        codes, scales = la.pack_8bit(x)
        return {"x8": la.unpack_8bit(codes, scales, x.dtype)}
    if kind == "serve":
        return {"y": la.layer_norm(x, st["w"], st["b"], EPS)}
    if kind == "train":
        y = la.layer_norm(x, st["w"], st["b"], EPS, save_8bit=st["save8"])
        dx, dw, db = torch.autograd.grad(y, (x, st["w"], st["b"]), st["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    y = la.layer_norm_sigmoid_gate(x, st["gate"], st["w"], st["b"], EPS, save_8bit=st["save8"])
    dx, dg, dw, db = torch.autograd.grad(y, (x, st["gate"], st["w"], st["b"]), st["dy"])
    return {"y": y, "dx": dx, "dgate": dg, "dw": dw, "db": db}


def run(st):
    return _own(st) if own else _plain(st)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def _checkpoint64(x):
    """Each group's step is the smallest power of two in which no value of it rounds to more than 127 steps."""
    n = x.shape[1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for lo in range(0, n, GROUP):
        part = x.detach()[:, lo:lo + GROUP].double()
        top = part.abs().amax(1, keepdim=True)
        step = torch.exp2(torch.clamp(torch.frexp(top).exponent.double() - 8, min=-126.0))
        while True:
            more = torch.round(top / step) > 127
            if not bool(more.any()):
                break
            step = torch.where(more, 2.0 * step, step)
        out[:, lo:lo + GROUP] = torch.round(part / step) * step
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind, n = case["kind"], case["dim"]
    if kind == "pack":
        return {"x8": _checkpoint64(st["x"])}
    x, w, b = (st[k].detach().double() for k in ("x", "w", "b"))
    mean = x.sum(1, keepdim=True) / n
    sigma = torch.sqrt(torch.var(x, 1, unbiased=False, keepdim=True) + EPS)
    normed = torch.addcmul(b, (x - mean) / sigma, w)
    out = {"y": normed * torch.sigmoid(st["gate"].detach().double()) if kind == "gate" else normed}
    if kind == "serve":
        return out
    del normed
    z = ((_checkpoint64(st["x"]) if case["save8"] else x) - mean) / sigma
    del x
    t = st["dy"].double()
    if kind == "gate":
        gate = _checkpoint64(st["gate"]) if case["save8"] else st["gate"].detach().double()
        sig = torch.sigmoid(gate)
        out["dgate"] = t * torch.addcmul(b, z, w) * sig * torch.sigmoid(-gate)
        t = t * sig
        del sig, gate
    out["db"], out["dw"] = t.sum(0), torch.einsum("mn,mn->n", t, z)
    t = t * w
    along = torch.einsum("mn,mn->m", t, z).unsqueeze(1) / n
    out["dx"] = (t - t.sum(1, keepdim=True) / n - z * along) / sigma
    return out


def work(case):
    """Bytes: every input read once, every output written once. Flops: the arithmetic of the formulas, a few per element."""
    kind, el = case["kind"], case["rows"] * case["dim"]
    size, wsize = (4 if case[k] == "fp32" else 2 for k in ("dtype", "wdtype"))
    if kind == "pack":
        # x in, codes and exponents out and in again, x out
        return {"bytes": 2 * el * size + 2 * (el + case["rows"] * -(-case["dim"] // GROUP)), "flops": 4 * el}
    tensors = {"serve": 2, "train": 4, "gate": 6}[kind]  # x, y; dy, dx; gate, dgate
    params = {"serve": 2, "train": 4, "gate": 4}[kind]  # weight, bias; their gradients
    return {"bytes": tensors * el * size + params * case["dim"] * wsize, "flops": {"serve": 8, "train": 24, "gate": 40}[kind] * el}
