"""More of what the operators around the attention call have to get right on the GPU: inputs that hold their values in an
unusual way, sums over many rows that come out exactly, products off 16-byte boundaries that fill the chip."""
import ctypes

import pytest
import torch

import flash_window_attention_v2_amd as fwa2
from flash_window_attention_v2_amd import _abi
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


@pytest.mark.parametrize("m,k,n", [(4, 64, 40), (300, 64, 264), (5000, 96, 384), (4096, 512, 2048), (300, 64, 33), (300, 63, 40),
                                   (70000, 192, 512)])
@pytest.mark.parametrize("act", [_abi.ACT_NONE, _abi.ACT_GELU, _abi.ACT_SILU])
@pytest.mark.parametrize("with_residual", [False, True])
def test_z_is_written_whenever_it_is_asked_for(m, k, n, act, with_residual):
    """Through the C entry point: few rows, tiles of several sizes, results and operands off 16 bytes, streamed results."""
    g = _gen(m + n)
    x, w, b = _rand(g, m, k, dtype=BF16), _rand(g, n, k, dtype=BF16, scale=k ** -0.5), _rand(g, n, dtype=BF16)
    r = _rand(g, m, n, dtype=BF16) if with_residual else None
    y, z = (torch.full((m, n), float("nan"), device="cuda", dtype=BF16) for _ in range(2))
    p = _abi.new_linear()
    p.dtype = p.x_dtype = _abi.BF16
    p.activation, p.rows, p.in_features, p.out_features = act, m, k, n
    p.x, p.x_stride, p.weight, p.weight_stride, p.bias = x.data_ptr(), k, w.data_ptr(), k, b.data_ptr()
    if with_residual:
        p.residual, p.residual_stride = r.data_ptr(), n
    p.y, p.z = y.data_ptr(), z.data_ptr()
    p.stream = torch.cuda.current_stream().cuda_stream
    lib = _abi.load()
    assert lib.fwa2_linear_workspace_bytes(ctypes.byref(p), 0) == 0
    assert lib.fwa2_linear_forward(ctypes.byref(p)) == _abi.OK
    name = {_abi.ACT_NONE: None, _abi.ACT_GELU: "gelu", _abi.ACT_SILU: "silu"}[act]
    rows = torch.cat([torch.arange(0, m, max(1, m // 100)), torch.arange(max(0, m - 70), m)]).to(x.device)
    for got, how, res in ((z, None, None), (y, name, r)):
        value, off = linear_ref(x[rows], w, b, how, None if res is None else res[rows])["y"]
        inside(got[rows], value, rounded(value, off, BF16), "z" if got is z else "y")
    assert z.isfinite().all() and y.isfinite().all()
