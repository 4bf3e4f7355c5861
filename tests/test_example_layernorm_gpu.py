"""The example attention block (examples/tnl_attention.py) with the layer norm, and with 8-bit checkpoints."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))

pytestmark = pytest.mark.gpu


def run(blk, x, dy):
    blk.zero_grad(set_to_none=True)
    x.grad = None
    y = blk(x)
    y.backward(dy)
    return {"y": y.detach().float(), "dx": x.grad.float(), **{n: p.grad.float() for n, p in blk.named_parameters()}}


def rel(a, b):
    return float((a - b).norm() / (b.norm() + 1e-20))


@pytest.mark.parametrize("embed,heads,n", [(1024, 8, 1024), (768, 12, 300)])
def test_layer_norm_block(cuda_lib, embed, heads, n):
    """Fused against unfused (as test_example_module_gpu.py holds the other norm), then with checkpoints: every gradient is there, y is the
    same, and gradients move by what the values kept do: half a step of a group's values is 2^-8 to 2^-7 of its largest, about
    1 % of values spread like normal ones, and each of the three products of a chain takes one or two such factors."""
    from tnl_attention import TnlAttentionB200

    torch.manual_seed(5)
    blk = TnlAttentionB200(embed, heads, layer_idx=3, norm="layer").cuda().bfloat16()
    x = (torch.randn(2, n, embed, device="cuda") * 0.5).bfloat16().requires_grad_()
    dy = torch.randn(2, n, embed, device="cuda").bfloat16()
    fused = run(blk, x, dy)
    assert set(fused) > {"norm.weight", "norm.bias", "q_proj.weight"} and all(torch.isfinite(t).all() for t in fused.values())
    blk.fused = False
    for name, t in run(blk, x, dy).items():
        assert rel(fused[name], t) < 2e-2, name
    blk.fused, blk.save_8bit, blk.norm.save_8bit = True, True, True
    kept = run(blk, x, dy)
    assert torch.equal(kept["y"], fused["y"])
    for name, t in kept.items():
        assert rel(t, fused[name]) < 5e-2, name


def test_unknown_norm_is_refused():
    from tnl_attention import TnlAttentionB200

    with pytest.raises(ValueError, match="unknown norm"):
        TnlAttentionB200(64, 1, norm="batch")


@pytest.mark.parametrize("use_reentrant", [False, True])
def test_with_activation_checkpointing(cuda_lib, use_reentrant):
    """torch.utils.checkpoint around the block: the same gradients, as everything is computed again from the same inputs."""
    from torch.utils.checkpoint import checkpoint
    from tnl_attention import TnlAttentionB200

    torch.manual_seed(5)
    blk = TnlAttentionB200(256, 4, norm="layer", save_8bit=True).cuda().bfloat16()
    x = (torch.randn(2, 200, 256, device="cuda") * 0.5).bfloat16().requires_grad_()
    dy = torch.randn(2, 200, 256, device="cuda").bfloat16()
    want = run(blk, x, dy)

    class Outer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.blk = blk

        def forward(self, x):
            return checkpoint(self.blk, x, use_reentrant=use_reentrant)

    got = run(Outer(), x, dy)
    for name, t in got.items():
        assert torch.equal(t, want[name.removeprefix("blk.")]), name


def test_backward_twice(cuda_lib):
    import lightning_attention_b200 as la

    torch.manual_seed(0)
    x, g = (torch.randn(50, 1001, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w = torch.randn(1001, device="cuda", requires_grad=True)
    dy = torch.randn(50, 1001, device="cuda").bfloat16()
    for save_8bit in (False, True):
        y = la.layer_norm_sigmoid_gate(x, g, w, save_8bit=save_8bit)
        first = torch.autograd.grad(y, (x, g, w), dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, (x, g, w), dy)))


def test_saved_attention_in_a_graph_and_on_a_stream(cuda_lib):
    """lightning_attn_func(save_8bit=True), forward and backward captured and replayed on new values."""
    import lightning_attention_b200 as la

    q, k, v, do = (torch.empty(1, 4, 300, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    s = la._build_slope_tensor(4).cuda()

    def fill(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            for t in (q, k, v, do):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 0.3)

    def step():
        o = la.lightning_attn_func(q, k, v, s, save_8bit=True)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    fill(0)
    [t.requires_grad_() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
