"""How far an 8-bit checkpoint's values may be from the tensor's: by the format's definition on the CPU, and by the kernels on the GPU."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from _ln_refs import checkpoint64  # noqa: E402


def groups():
    """fp32 groups of 32: the largest value of each in every position between two powers of two, where the exponent is raised
    (127.5 to 128 steps) more closely, and the rest of the group spread over what that leaves."""
    top = torch.cat([1 + torch.arange(256) / 256, 127.5 / 64 + torch.arange(64) * 2.0 ** -13, torch.tensor([127.5 / 64 - 2.0 ** -23, 2 - 2.0 ** -23])])
    rest = torch.linspace(-1, 1, 31, dtype=torch.float64)
    return torch.cat([top.double().unsqueeze(1), top.double().unsqueeze(1) * rest], 1).float()


def check_bounds(x, values):
    """Half a step, and that is at most 1 / 127.5 of the group's largest value."""
    off = (values.double() - x.double()).abs()
    top = x.double().abs().amax(1, keepdim=True)
    assert bool((off <= top / 127.5).all())
    assert bool((off > top * 2.0 ** -7).any())  # it is no 2^-7


def check_ends(x, values):
    """Steps end at 2^-126 (values up to half of one come back as zero) and at 2^121 (the largest code stands for all from 127.5 steps on)."""
    small, big = values[:2].double(), values[2:].double()
    assert small[0].tolist() == [0.0, 0.0, 2.0 ** -126, 2.0 ** -125] and not small[1].any()
    assert bool((big == 127 * 2.0 ** 121).all())
    assert bool(((x[2:].double() - big).abs() < 2.0 ** 121).all()) and bool(((x[2:].double() - big).abs() > 2.0 ** 120).any())


def ends():
    top = torch.finfo(torch.float32).max
    return torch.tensor([[2.0 ** -128, 2.0 ** -127, 1.01 * 2.0 ** -127, 2.0 ** -125], [2.0 ** -149, 2.0 ** -127, -(2.0 ** -130), 0.0],
                         [top, top, top, top], [127.5 * 2.0 ** 121, 127.75 * 2.0 ** 121, top, 127.25 * 2.0 ** 121]])


def test_definition():
    check_bounds(groups(), checkpoint64(groups()))
    check_ends(ends(), checkpoint64(ends()))


@pytest.mark.gpu
def test_kernels(cuda_lib):
    import lightning_attention_b200 as la

    for scale in (1.0, 2.0 ** -60, 2.0 ** 100):
        x = groups().cuda() * scale
        check_bounds(x, la.unpack_8bit(*la.pack_8bit(x), torch.float32))
    x = ends().cuda()
    check_ends(x, la.unpack_8bit(*la.pack_8bit(x), torch.float32))
