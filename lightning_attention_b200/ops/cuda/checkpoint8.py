"""8-bit activation checkpoints: pack_8bit and unpack_8bit, and what the operators with `save_8bit` use of them.

32 consecutive values of the last dimension share one exponent byte and keep a signed byte each (csrc/pack8.cuh): 8.25 bits per value,
off by at most 1 / 127.5 of the largest of the 32 (of those below 2^-120, where steps end, by up to 2^-127). The step is a power of two, so
that what a checkpoint stands for depends on its input alone, and is exact in fp32 and bf16.
"""
import torch

from ... import _lib

GROUP = 32
MAX_ROW = 1 << 30  # values of a row: the kernels count within one in 32 bits


def check_row(t, what):
    if t.dim() < 1 or not 1 <= t.shape[-1] <= MAX_ROW:
        raise RuntimeError(f"{what} of at least one value and at most 2^30, got shape {tuple(t.shape)}")


def rows(t, N):
    """`t` as rows of N adjacent elements and the elements from one row to the next: a view where its strides allow one, else a copy."""
    t = t.reshape(-1, N)
    M = t.shape[0]
    if (N > 1 and t.stride(1) != 1) or (M > 1 and t.stride(0) < N):
        t = t.contiguous()
    return t, (t.stride(0) if M > 1 else N)


def packed_rows(t, N):
    """The same for the layer norms, whose fast kernels read the rows of a contiguous tensor that begins on 16 bytes, or whole packs of
    16 bytes: other rows are copied, which costs less than reading them value by value."""
    t, ld = rows(t, N)
    size = t.element_size()
    if t.data_ptr() % 16 or (ld != N and (N * size % 16 or ld * size % 16)):
        t, ld = t.clone(memory_format=torch.contiguous_format), N
    return t, ld


def scales_shape(shape):
    return (*shape[:-1], -(-shape[-1] // GROUP))


def empty_checkpoint(shape, device):
    """Uninitialised codes and scales for a tensor of `shape`."""
    return torch.empty(shape, dtype=torch.int8, device=device), torch.empty(scales_shape(shape), dtype=torch.uint8, device=device)


def checkpoint_fits(codes, scales, shape, device):
    return (codes.dtype == torch.int8 and scales.dtype == torch.uint8 and codes.device == device and scales.device == device and
            tuple(codes.shape) == tuple(shape) and tuple(scales.shape) == scales_shape(shape))


def differentiable_once(what):
    """Refuses a backward pass that is to be differentiated again: autograd would take its kernels' results for constants."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} can be differentiated once only: its backward pass does not run with create_graph=True")


def pack_8bit(x):
    """The 8-bit checkpoint of a bf16, fp16 or fp32 tensor: (codes, scales), int8 of x's shape and uint8 with one byte for each 32
    values of the last dimension (its last group may be shorter). A group that holds an infinity or a NaN comes back as NaN. No autograd."""
    if not torch.compiler.is_compiling():
        r = _lib.host().pack8(x)
        if r is not None:
            return r
    check_row(x, "pack_8bit takes a tensor with a last dimension")
    _lib.require_cuda(x)
    dt = _lib.dtype_code(x.dtype)
    N = x.shape[-1]
    codes, scales = empty_checkpoint(x.shape, x.device)
    x, ld = rows(x.detach(), N)
    with torch.cuda.device(x.device):
        rc = _lib.lib().lab200_pack8(x.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), x.shape[0], N, dt, _lib.stream_ptr(x.device))
    _lib.check(rc, "lab200_pack8")
    return codes, scales


def unpack_8bit(codes, scales, dtype=torch.bfloat16):
    """The values that a checkpoint stands for, in codes' shape. Exact in bf16 and fp32; in fp16 rounded, and kept within +-65504."""
    dt = _lib.dtype_code(dtype)
    if not torch.compiler.is_compiling():
        y = _lib.host().unpack8(codes, scales, dt)
        if y is not None:
            return y
    if codes.dim() > 0 and codes.shape[-1] > MAX_ROW:
        raise RuntimeError(f"unpack_8bit takes codes with a last dimension of at most 2^30, got shape {tuple(codes.shape)}")
    _lib.require_cuda(codes, scales)
    if codes.dim() < 1 or codes.shape[-1] < 1 or not checkpoint_fits(codes, scales, codes.shape, codes.device):
        raise RuntimeError("expected int8 codes and uint8 scales with one byte for each 32 codes of the last dimension, on one device; got "
                           f"{codes.dtype} {tuple(codes.shape)} on {codes.device} and {scales.dtype} {tuple(scales.shape)} on {scales.device}")
    codes, scales = codes.contiguous(), scales.contiguous()
    N = codes.shape[-1]
    y = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        rc = _lib.lib().lab200_unpack8(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), codes.numel() // N, N, dt, _lib.stream_ptr(codes.device))
    _lib.check(rc, "lab200_unpack8")
    return y
