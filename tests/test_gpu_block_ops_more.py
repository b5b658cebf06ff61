"""More of what the operators around the attention call have to get right on the GPU: inputs that hold their values in an
unusual way, sums over many rows that come out exactly, products off 16-byte boundaries that fill the chip."""
import ctypes

import pytest
import torch

import flash_window_attention_v2_amd as fwa2
from flash_window_attention_v2_amd import _abi
from block_ops_exact import constant_rows, constant_rows_bound, layer, layer_sums, whole
from block_ops_ref import inside, linear8_ref, linear_ref, rounded, slope64

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


# ---- sums over many rows, exactly ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,k,n", [(70000, 8, 8), (16500, 64, 136), (5000, 96, 96), (20000, 96, 40), (9999, 136, 200), (4097, 33, 17),
                                   (16384, 192, 384), (16384, 384, 192), (8192, 2048, 512), (700, 2985, 2987), (129, 72, 40)])
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_of_whole_numbers_are_exact(m, k, n, act, dtype):
    """Every split of a weight gradient and every stretch of a bias gradient arrives once: equality, no tolerance."""
    x, w, b, dy = layer(m, k, n, dtype, "cuda", m + k)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(fwa2.fused_linear_func(*leaves, act), leaves, dy)
    want = layer_sums(x, w, b, dy, act)
    for t, name in zip(got, ("dx", "dw", "db")):
        assert torch.equal(t, want[name].to(dtype)), name


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [512, 513])
def test_bias_gradients_come_from_unrounded_ones(act, dtype, n):
    m = 300
    z, dy = constant_rows(act, n, dtype, "cuda", 3)
    leaves = [torch.zeros(m, 16, device="cuda", dtype=dtype).requires_grad_(), torch.ones(n, 16, device="cuda", dtype=dtype).requires_grad_(),
              z.requires_grad_()]
    got = torch.autograd.grad(fwa2.fused_linear_func(*leaves, act), leaves, dy.expand(m, n))[2]
    want = m * dy.double() * slope64(z.double(), act)
    inside(got, want, constant_rows_bound(want, m, dtype), "db")


@pytest.mark.parametrize("rows,dim", [(40000, 96), (262144, 40), (20001, 520), (5000, 1100), (9000, 1538), (3000, 5000), (1500, 10000), (3, 96)])
@pytest.mark.parametrize("placement", ["post", "pre"])
@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32)], ids=["bf16", "fp32 stream", "f16"])
def test_norm_parameter_gradients_of_whole_numbers_are_exact(rows, dim, placement, types):
    """Through the C entry point, with statistics (0, 1) for every row, so that the normalised rows are the whole numbers."""
    xt, st, wt = types
    g = _gen(rows + dim)
    pre = placement == "pre"
    x, dy = whole(g, rows, dim, dtype=xt, device="cuda"), whole(g, rows, dim, dtype=xt if pre else st, device="cuda")
    s = whole(g, rows, dim, dtype=st, device="cuda") if pre else None
    h = (x.to(st) + s) if pre else None
    w = torch.ones(dim, device="cuda", dtype=wt)
    stats = torch.tensor([0.0, 1.0], device="cuda").expand(rows, 2).contiguous()
    dw, db = (torch.full((dim,), float("nan"), device="cuda", dtype=wt) for _ in range(2))
    code = {BF16: _abi.BF16, F16: _abi.F16, F32: _abi.F32}
    p = _abi.new_norm()
    p.dtype, p.stream_dtype, p.param_dtype = code[xt], code[st], code[wt]
    p.kind, p.placement, p.eps = _abi.NORM_RMS, _abi.NORM_PRE if pre else _abi.NORM_POST, 1e-5
    p.rows, p.dim = rows, dim
    p.x, p.x_stride, p.weight, p.stats = x.data_ptr(), dim, w.data_ptr(), stats.data_ptr()
    p.dy, p.dy_stride, p.dweight, p.dbias = dy.data_ptr(), dim, dw.data_ptr(), db.data_ptr()
    if pre:
        p.shortcut, p.shortcut_stride, p.h = s.data_ptr(), dim, h.data_ptr()
    lib = _abi.load()
    need = lib.fwa2_norm_workspace_bytes(ctypes.byref(p))
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    p.workspace, p.workspace_bytes, p.stream = ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream
    assert lib.fwa2_norm_backward(ctypes.byref(p)) == _abi.OK, lib.fwa2_last_error()
    v = h if pre else x
    assert torch.equal(dw, (dy.double() * v.double()).sum(0).to(wt)) and torch.equal(db, dy.double().sum(0).to(wt))


# ---- products off 16-byte boundaries that fill the chip, and results that are streamed ----------------------------------------
def _sample(m):
    return torch.cat([torch.arange(0, m, max(1, m // 40)), torch.arange(max(0, m - 140), m)]).cuda()


def _layer(m, k, n, dtype, seed):
    g = _gen(seed)
    return (_rand(g, m, k, dtype=dtype), _rand(g, n, k, dtype=dtype, scale=k ** -0.5), _rand(g, n, dtype=dtype, scale=0.3),
            _rand(g, m, n, dtype=dtype), _rand(g, m, n, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_unaligned_products_of_many_tiles(dtype, act):
    """At least two 128 x 128 tiles to a CU, rows and columns that end inside a tile: forward, dx and dW."""
    m, k, n = 14003, 585, 1161
    x, w, b, r, dy = _layer(m, k, n, dtype, 1)
    rows = _sample(m)
    leaf = x.clone().requires_grad_()
    y = fwa2.fused_linear_func(leaf, w, b, act, r)
    dx, = torch.autograd.grad(y, [leaf], dy)
    ref = linear_ref(x[rows], w, b, act, r[rows], dy[rows])
    for got, name in ((y.detach(), "y"), (dx, "dx")):
        inside(got[rows], ref[name][0], rounded(*ref[name], dtype), name)
    m, k, n = 333, 2985, 2987
    x, w, b, r, dy = _layer(m, k, n, dtype, 2)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(fwa2.fused_linear_func(*leaves, act), leaves, dy)
    ref = linear_ref(x, w, b, act, None, dy)
    for t, name in zip(got, ("dx", "dw", "db")):
        inside(t, ref[name][0], rounded(*ref[name], dtype), name)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_unaligned_8bit_products_of_many_tiles(dtype):
    m, k, n = 8200, 601, 1161
    x, w, b, r, _ = _layer(m, k, n, dtype, 3)
    x8, sx = fwa2.quantize_rows_func(x)
    w8, sw = fwa2.quantize_rows_func(w)
    rows = _sample(m)
    for act, bias, res in ((None, None, None), ("gelu", b, r), ("silu", b, None)):
        y = fwa2.fused_linear_fp8_func(x8, sx, w8, sw, bias, act, res, out_dtype=dtype)
        value, off = linear8_ref(x8[rows], sx[rows], w8, sw, bias, act, None if res is None else res[rows])
        inside(y[rows], value, rounded(value, off, dtype), f"{act}")


@pytest.mark.parametrize("m,k,n", [(70000, 96, 512), (70000, 192, 512), (90000, 400, 384), (40000, 512, 1024), (35001, 264, 1000)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_streamed_results(m, k, n, dtype):
    """Results of 64 MB and more, on tiles of every size that has them: with and without a residual, an activation, z."""
    x, w, b, r, dy = _layer(m, k, n, dtype, m)
    rows = _sample(m)
    for act in (None, "gelu", "silu"):
        for res in (None, r):
            ref = linear_ref(x[rows], w, b, act, None if res is None else res[rows], dy[rows])
            with torch.no_grad():
                y = fwa2.fused_linear_func(x, w, b, act, res)
            inside(y[rows], ref["y"][0], rounded(*ref["y"], dtype), f"{act} y")
            leaf = x.clone().requires_grad_()
            again = fwa2.fused_linear_func(leaf, w, b, act, res)
            assert torch.equal(again.detach(), y)
            dx, = torch.autograd.grad(again, [leaf], dy)
            inside(dx[rows], ref["dx"][0], rounded(*ref["dx"], dtype), f"{act} dx")
    # a streamed dx: the contraction is the short side
    wt = w.t().contiguous()
    leaf = dy.clone().requires_grad_()
    dx, = torch.autograd.grad(fwa2.fused_linear_func(leaf, wt), [leaf], x)
    ref = linear_ref(dy[rows], wt, None, None, None, x[rows])["dx"]
    inside(dx[rows], ref[0], rounded(*ref, dtype), "dx")
    x8, sx = fwa2.quantize_rows_func(x)
    w8, sw = fwa2.quantize_rows_func(w)
    for act, res in ((None, None), ("gelu", r), ("silu", None)):
        y = fwa2.fused_linear_fp8_func(x8, sx, w8, sw, b, act, res, out_dtype=dtype)
        value, off = linear8_ref(x8[rows], sx[rows], w8, sw, b, act, None if res is None else res[rows])
        inside(y[rows], value, rounded(value, off, dtype), f"{act} 8 bits")
