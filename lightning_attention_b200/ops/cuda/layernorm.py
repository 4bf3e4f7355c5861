"""Layer norm with weight and bias, and the same followed by a sigmoid gate, as torch.autograd.Functions backed by liblightning_b200.so.

The norm of the reference's example caller is nn.LayerNorm, its output times a sigmoid gate (examples/module/tnl_attn.py:66-69).
With `save_8bit` the backward pass keeps x (and the gate) as 8-bit checkpoints, which the forward kernel writes beside y and the row statistics.
"""
import torch

from ... import _lib
from .checkpoint8 import check_row, checkpoint_fits, differentiable_once, empty_checkpoint, packed_rows


def _check(x, gate, weight, bias, eps):
    check_row(x, "layer norm takes rows")
    _lib.require_cuda(x, gate, weight, bias)
    _lib.dtype_code(x.dtype)
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype or gate.device != x.device):
        raise RuntimeError(f"gate must match x in shape, dtype and device; got {tuple(gate.shape)} {gate.dtype} {gate.device} vs "
                           f"{tuple(x.shape)} {x.dtype} {x.device}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (tuple(p.shape) != (x.shape[-1],) or p.dtype not in (x.dtype, torch.float32) or p.device != x.device):
            raise RuntimeError(f"{name} must have shape ({x.shape[-1]},), x's dtype or float32, and x's device; got {tuple(p.shape)} {p.dtype} "
                               f"{p.device} with x {x.dtype} {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"weight and bias must share one dtype, got {weight.dtype} and {bias.dtype}")
    if not 0 <= eps < float("inf"):
        raise RuntimeError(f"eps must be a number of at least zero, got {eps}")


def _contiguous(p):
    return None if p is None else p.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weight, bias, eps, save_8bit, wanted):
        _check(x, gate, weight, bias, eps)
        shape, N = x.shape, x.shape[-1]
        x2, ldx = packed_rows(x, N)
        g2, ldg = packed_rows(gate, N) if gate is not None else (None, N)
        weight, bias = _contiguous(weight), _contiguous(bias)
        M = x2.shape[0]
        y = torch.empty(shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((M, 2), dtype=torch.float32, device=x.device) if wanted else None
        xc = xs = gc = gs = None
        if wanted and save_8bit:
            xc, xs = empty_checkpoint((M, N), x.device)
            if gate is not None:
                gc, gs = empty_checkpoint((M, N), x.device)
        wdt = next((p.dtype for p in (weight, bias) if p is not None), torch.float32)
        with torch.cuda.device(x.device):
            rc = _lib.lib().lab200_layernorm_fwd(
                x2.data_ptr(), ldx, _lib.ptr(g2), ldg, _lib.ptr(weight), _lib.ptr(bias), _lib.dtype_code(wdt), y.data_ptr(), _lib.ptr(stats),
                _lib.ptr(xc), _lib.ptr(xs), _lib.ptr(gc), _lib.ptr(gs), M, N, float(eps), _lib.dtype_code(x.dtype), _lib.stream_ptr(x.device))
        _lib.check(rc, "lab200_layernorm_fwd")
        if wanted:
            # the tensors themselves, not copies of other strides: a change to them is noticed
            ctx.save_for_backward(*((xc, xs, gc, gs) if save_8bit else (x, None, gate, None)), stats, weight, bias if gate is not None else None)
            ctx.info = (M, N, x.dtype, x.device, gate is not None, wdt, bool(save_8bit))
        return y

    @staticmethod
    def backward(ctx, dy):
        differentiable_once("layer norm")
        M, N, dtype, device, gated, wdt, save_8bit = ctx.info
        need_x, need_g, need_w, need_b = ctx.needs_input_grad[:4]
        first, xs, second, gs, stats, weight, bias = ctx.saved_tensors
        bad = tuple(stats.shape) != (M, 2) or stats.dtype != torch.float32 or stats.device != device
        for p in (weight, bias):
            bad = bad or (p is not None and (p.numel() != N or p.dtype != wdt or p.device != device))
        x2 = g2 = xc = gc = None
        ldx = ldg = N
        if save_8bit:
            bad = bad or not checkpoint_fits(first, xs, (M, N), device) or (gated and not checkpoint_fits(second, gs, (M, N), device))
            xc, xs, gc, gs = (_contiguous(t) for t in (first, xs, second, gs))
        else:
            bad = bad or any(t.numel() != M * N or t.shape[-1] != N or t.dtype != dtype or t.device != device for t in ((first, second) if gated else (first,)))
            if not bad:
                x2, ldx = packed_rows(first, N)
                g2, ldg = packed_rows(second, N) if gated else (None, N)
        if bad:
            raise RuntimeError("layer norm backward: saved-tensor hooks returned another shape, dtype or device")
        if dy.numel() != M * N:
            raise RuntimeError("gradient and input sizes differ")
        shape = dy.shape
        dy2, lddy = packed_rows(dy.to(dtype), N)
        stats, weight, bias = stats.contiguous(), _contiguous(weight), _contiguous(bias)
        new = lambda on, shape, dt: torch.empty(shape, dtype=dt, device=device) if on else None
        dx, dg, dw, db = new(need_x, shape, dtype), new(need_g, shape, dtype), new(need_w, (N,), wdt), new(need_b, (N,), wdt)
        L = _lib.lib()
        with torch.cuda.device(device):
            nbytes = L.lab200_layernorm_bwd_workspace_bytes(M, N) if need_w or need_b else 0
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            rc = L.lab200_layernorm_bwd(
                _lib.ptr(x2), ldx, _lib.ptr(g2), ldg, _lib.ptr(xc), _lib.ptr(xs), _lib.ptr(gc), _lib.ptr(gs), stats.data_ptr(), dy2.data_ptr(), lddy,
                _lib.ptr(weight), _lib.ptr(bias), _lib.dtype_code(wdt), _lib.ptr(dx), _lib.ptr(dg), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), nbytes,
                M, N, _lib.dtype_code(dtype), _lib.stream_ptr(device))
        _lib.check(rc, "lab200_layernorm_bwd")
        return dx, dg, dw, db, None, None, None


def _apply(x, gate, weight, bias, eps, save_8bit):
    """_LayerNorm through the native call path (csrc/host_ops.cpp) where the call has the common form, else through the class."""
    if not torch.compiler.is_compiling():
        y = _lib.host().layer_norm(x, gate, weight, bias, eps, save_8bit)
        if y is not None:
            return y
    # whether a backward pass can follow, which the class cannot see: inside it gradients are off
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, weight, bias))
    return _LayerNorm.apply(x, gate, weight, bias, eps, save_8bit, wanted)


def layer_norm(x, weight=None, bias=None, eps=1e-5, save_8bit=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension; weight and bias default to ones and zeros.

    x: bf16, fp16 or fp32, any strides; weight, bias: (N,) of x's dtype or fp32, one dtype for both. Statistics and all sums are
    fp32. Differentiable once, in x, weight and bias; gradients are the same every time. save_8bit: the backward pass keeps x as an
    8-bit checkpoint (`pack_8bit`) in place of the tensor, and each row's mean and 1 / sqrt(var + eps) as they were in the forward pass:
    it takes x from the checkpoint in the gradients' formulas and the statistics of x itself, not those of the checkpoint."""
    return _apply(x, None, weight, bias, eps, save_8bit)


def layer_norm_sigmoid_gate(x, gate, weight=None, bias=None, eps=1e-5, save_8bit=False):
    """layer_norm(x, weight, bias, eps) * sigmoid(gate) in one kernel each way; gate has x's shape and dtype. save_8bit: x and gate
    are both kept as 8-bit checkpoints, and the row statistics of x itself."""
    if gate is None:
        raise RuntimeError("layer_norm_sigmoid_gate needs a gate; layer_norm has none")
    return _apply(x, gate, weight, bias, eps, save_8bit)


class LayerNorm(torch.nn.Module):
    """layer_norm as a module, with the parameters of torch.nn.LayerNorm over one dimension."""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True, save_8bit=False, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps, self.save_8bit = dim, eps, save_8bit
        new = lambda fill, on: torch.nn.Parameter(torch.full((dim,), fill, device=device, dtype=dtype)) if on else None
        self.register_parameter("weight", new(1.0, elementwise_affine))
        self.register_parameter("bias", new(0.0, elementwise_affine and bias))

    def forward(self, x, gate=None):
        if gate is None:
            return layer_norm(x, self.weight, self.bias, self.eps, self.save_8bit)
        return layer_norm_sigmoid_gate(x, gate, self.weight, self.bias, self.eps, self.save_8bit)

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}, save_8bit={self.save_8bit}"
