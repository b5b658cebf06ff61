"""More of what the operators around the attention call have to get right on the GPU: inputs that hold their values in an
unusual way, sums over many rows that come out exactly, products off 16-byte boundaries that fill the chip."""
import pytest
import torch

import flash_window_attention_v2_amd as fwa2
from block_ops_ref import inside, linear_ref, rounded

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def test_lazily_negated_inputs():
    # tensors whose memory holds the negated values give what the same values give anywhere else
    g = _gen(1)
    x, w, b, r = (_rand(g, *s, dtype=BF16) for s in ((70, 64), (40, 64), (40,), (70, 40)))
    v, c, gate = _rand(g, 64, dtype=BF16), _rand(g, 64, dtype=BF16), _rand(g, 7, dtype=BF16)
    neg = [torch._neg_view(-t) for t in (x, w, b, r, v, c, gate)]
    assert all(t.is_neg() for t in neg)
    nx, nw, nb, nr, nv, nc, ngate = neg
    dy = _rand(g, 70, 40, dtype=BF16)

    def grads(call, leaves, d):
        leaves = [t.detach().requires_grad_() for t in leaves]
        out = call(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, d)]

    def both(call, plain, negated, d):
        for a, n in zip(grads(call, plain, d), grads(call, negated, torch._neg_view(-d))):
            assert torch.equal(a, n)

    both(lambda *t: fwa2.fused_linear_func(*t[:3], "gelu", t[3]), (x, w, b, r), (nx, nw, nb, nr), dy)
    dx = _rand(g, 70, 64, dtype=BF16)
    both(lambda *t: fwa2.residual_norm_func(*t, gate=gate), (x, x, v, c), (nx, nx, nv, nc), dx)
    both(lambda *t: fwa2.residual_norm_func(*t, gate=ngate), (x, x, v, c), (nx, nx, nv, nc), dx)
    for a, n in zip(fwa2.quantize_rows_func(x), fwa2.quantize_rows_func(nx)):
        assert torch.equal(a.float(), n.float())
