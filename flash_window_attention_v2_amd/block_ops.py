"""The operators around the attention call of a transformer block: normalisation with the residual's addition, matrix
products with an epilogue, and the 8-bit forms of both.

The reference composes them from framework calls (`x + drop_path(norm(x))`, nn.Linear, nn.GELU:
flash_win_attn_v2/swin_transformer_v2.py:66-85, 443-445).  Here each is one HIP kernel forward and two or three backward,
described to libfwa2.so by raw pointers and strides; outputs and workspaces are torch tensors allocated on this side.
As for the attention there is no CPU path and no fallback.

Tensors of any strides are taken; what the kernels cannot address (an inner stride other than 1, rows that overlap or lie
2^22 elements apart or more) is copied first.  Leading dimensions are flattened to rows.  Every call works on the current
stream of the tensors' device and can be captured into a graph; gradients are bit-reproducible and cannot be
differentiated a second time (that raises).
"""
import torch
from torch.autograd.function import once_differentiable

from . import _abi
from .kernels import _DTYPES, _on_device

_ACTIVATIONS = {None: _abi.ACT_NONE, "none": _abi.ACT_NONE, "gelu": _abi.ACT_GELU, "gelu_tanh": _abi.ACT_GELU_TANH,
                "silu": _abi.ACT_SILU, "relu": _abi.ACT_RELU}
_KINDS = {"layer": _abi.NORM_LAYER, "rms": _abi.NORM_RMS}
_PLACES = {"post": _abi.NORM_POST, "pre": _abi.NORM_PRE}
_HALF = (torch.float16, torch.bfloat16)
_F8 = torch.float8_e4m3fn
_MAX_STRIDE = 1 << 22


def _rows(t):
    """(`t` as [rows, last] with unit inner stride, row stride): a view where the kernels can address it, a copy
    otherwise."""
    last = t.shape[-1]
    t = t.reshape(-1, last)
    if t.shape[0] <= 1:
        if last > 1 and t.stride(1) != 1:
            t = t.contiguous()
        return t, last
    if (last > 1 and t.stride(1) != 1) or t.stride(0) < last or t.stride(0) >= _MAX_STRIDE:
        t = t.contiguous()
    return t, t.stride(0)


def _count(t):
    n = 1
    for s in t.shape[:-1]:
        n *= s
    return n


def _ptr(t):
    return None if t is None else t.data_ptr()


def _same_device(x, *others):
    assert x.is_cuda, "tensors must be on the GPU"
    for t in others:
        assert t is None or t.device == x.device, "all tensors must be on the same device"


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- normalisation with the residual's addition ----------------------------------------------------------------------
def _check_norm(x, shortcut, weight, bias, eps, kind, placement, gate):
    assert kind in _KINDS, f"kind must be one of {sorted(_KINDS)}"
    assert placement in _PLACES, f"placement must be one of {sorted(_PLACES)}"
    assert x.dim() >= 1 and x.shape[-1] > 0, "x must have at least one value per row"
    dim = x.shape[-1]
    _same_device(x, shortcut, weight, bias, gate)
    assert x.dtype in _DTYPES, "Only support fp16, bf16 and fp32"
    assert placement == "post" or shortcut is not None, "the pre-norm form needs a shortcut"
    if shortcut is not None:
        assert shortcut.shape == x.shape, "shortcut must have the shape of x"
        assert shortcut.dtype in (x.dtype, torch.float32), "shortcut must be of the dtype of x or fp32"
    assert weight is not None and weight.shape == (dim,), "weight must hold one value per column"
    assert weight.dtype in (x.dtype, torch.float32), "weight must be of the dtype of x or fp32"
    if bias is not None:
        assert bias.shape == (dim,) and bias.dtype == weight.dtype, "bias must have the shape and dtype of weight"
    if gate is not None:
        assert gate.dtype in (x.dtype, torch.float32), "gate must be of the dtype of x or fp32"
        assert gate.numel() > 0 and _count(x) % gate.numel() == 0, \
            "gate must hold one factor per sample: the rows of x must be a multiple of its size"
        assert not (torch.is_grad_enabled() and gate.requires_grad), "gate gets no gradient"
    if dim > _abi.NORM_MAX_DIM:
        raise NotImplementedError(f"rows of {dim} values: at most {_abi.NORM_MAX_DIM} are supported")
    assert 0.0 < eps < float("inf"), "eps must be positive"


def _describe_norm(x, weight, bias, eps, kind, placement, gate, stream_dtype):
    p = _abi.new_norm()
    p.dtype, p.stream_dtype, p.param_dtype = _DTYPES[x.dtype], _DTYPES[stream_dtype], _DTYPES[weight.dtype]
    p.kind, p.placement, p.eps = _KINDS[kind], _PLACES[placement], eps
    p.rows, p.dim = _count(x), x.shape[-1]
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    p.weight, p.bias = weight.data_ptr(), _ptr(bias)
    if gate is not None:
        gate = gate.contiguous()
        p.gate, p.gate_dtype, p.rows_per_gate = gate.data_ptr(), _DTYPES[gate.dtype], p.rows // gate.numel()
    p._keep = (weight, bias, gate)      # what the description points at lives as long as it does
    return p


def _norm_forward(x, shortcut, weight, bias, eps, kind, placement, gate, want_stats, want_y8):
    """(y, h, y8, scale, stats); h only in the pre-norm form, y not there with an 8-bit output."""
    pre = placement == "pre"
    stream_dtype = shortcut.dtype if shortcut is not None else x.dtype
    rows = _count(x)

    def new(dtype):
        return torch.empty(x.shape, device=x.device, dtype=dtype)

    h = new(stream_dtype) if pre else None
    y = None if pre and want_y8 else new(x.dtype if pre else stream_dtype)
    y8 = new(_F8) if want_y8 else None
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32) if want_y8 else None
    stats = torch.empty((rows, 2), device=x.device, dtype=torch.float32) if want_stats else None
    if rows == 0:
        return y, h, y8, scale, stats
    p = _describe_norm(x, weight, bias, eps, kind, placement, gate, stream_dtype)
    xr, p.x_stride = _rows(x)
    p.x = xr.data_ptr()
    if shortcut is not None:
        sr, p.shortcut_stride = _rows(shortcut)
        p.shortcut = sr.data_ptr()
    p.y, p.h, p.y8, p.y8_scale, p.stats = _ptr(y), _ptr(h), _ptr(y8), _ptr(scale), _ptr(stats)
    with _on_device(x.device) as stream:
        p.stream = stream
        _abi.check(_abi.load().fwa2_norm_forward(p), "fwa2_norm_forward")
    return y, h, y8, scale, stats


class ResidualNorm(torch.autograd.Function):
    """`residual_norm_func` under autograd: keeps x (post) or the h it returned (pre) and two numbers per row."""

    @staticmethod
    def forward(ctx, x, shortcut, weight, bias, eps, kind, placement, gate):
        y, h, _, _, stats = _norm_forward(x, shortcut, weight, bias, eps, kind, placement, gate, True, False)
        pre = placement == "pre"
        ctx.save_for_backward(h if pre else x, weight, bias, gate, stats)
        ctx.how = (eps, kind, placement, x.dtype, shortcut.dtype if shortcut is not None else x.dtype)
        ctx.set_materialize_grads(False)
        return (h, y) if pre else y

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        v, weight, bias, gate, stats = ctx.saved_tensors
        eps, kind, placement, x_dtype, stream_dtype = ctx.how
        need_x, need_s, need_w, need_b = ctx.needs_input_grad[:4]
        none = (None,) * 8
        pre = placement == "pre"
        dh, dy = grads if pre else (None, grads[0])
        if dy is None and dh is None:
            return none
        need_w = need_w and dy is not None
        need_b = need_b and dy is not None

        def new(dtype):
            return torch.empty(v.shape, device=v.device, dtype=dtype)

        # without a gate and with one type, the two gradients of the pre-norm form are the same numbers
        shared = pre and gate is None and x_dtype == stream_dtype
        ds = new(stream_dtype) if pre and (need_s or (shared and need_x)) else None
        dx = new(x_dtype) if need_x and not shared else None
        dw = torch.empty(weight.shape, device=v.device, dtype=weight.dtype) if need_w else None
        db = torch.empty(bias.shape, device=v.device, dtype=bias.dtype) if need_b else None
        if _count(v) == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif any(t is not None for t in (dx, ds, dw, db)):
            p = _describe_norm(v, weight, bias, eps, kind, placement, gate, stream_dtype)
            p.dtype = _DTYPES[x_dtype]
            if pre:
                p.h = v.data_ptr()      # an output of the forward call: contiguous
                if dh is not None:
                    dhr, p.dh_stride = _rows(dh)
                    p.dh = dhr.data_ptr()
            else:
                vr, p.x_stride = _rows(v)
                p.x = vr.data_ptr()
            if dy is not None:
                dyr, p.dy_stride = _rows(dy)
                p.dy = dyr.data_ptr()
            p.stats = stats.data_ptr()
            p.dx, p.dshortcut, p.dweight, p.dbias = _ptr(dx), _ptr(ds), _ptr(dw), _ptr(db)
            lib = _abi.load()
            with _on_device(v.device) as stream:
                need = lib.fwa2_norm_workspace_bytes(p)
                ws = torch.empty(need, dtype=torch.uint8, device=v.device) if need else None
                p.workspace, p.workspace_bytes, p.stream = _ptr(ws), need, stream
                _abi.check(lib.fwa2_norm_backward(p), "fwa2_norm_backward")
        if shared:
            dx = ds if need_x else None
        if not pre:
            ds = dy
        return dx, (ds if need_s else None), dw, db, None, None, None, None


def residual_norm_func(x, shortcut, weight, bias=None, eps=1e-5, kind="layer", placement="post", gate=None):
    """Normalisation of the rows of x together with the residual's addition.

      placement="post":  shortcut + gate * norm(x)                 -> y (dtype of shortcut; shortcut may be None)
      placement="pre":   h = shortcut + gate * x, y = norm(h)      -> (h, y) (h: dtype of shortcut, y: dtype of x)

    norm is layer normalisation (kind="layer") or root-mean-square normalisation (kind="rms") over the last dimension, times
    `weight`, plus `bias` if given; sums and statistics in fp32, each output rounded once.
    x, shortcut: [..., dim] with dim <= 16384, fp16 / bf16 / fp32, shortcut of the dtype of x or fp32; weight, bias: [dim],
    of the dtype of x or fp32; gate: one factor per sample (x's rows are split evenly over gate.numel() samples, as
    stochastic depth needs), of the dtype of x or fp32, without a gradient.
    Gradients for x, shortcut, weight and bias."""
    _check_norm(x, shortcut, weight, bias, eps, kind, placement, gate)
    if _wants_grad(x, shortcut, weight, bias):
        return ResidualNorm.apply(x, shortcut, weight, bias, eps, kind, placement, gate)
    y, h, _, _, _ = _norm_forward(x, shortcut, weight, bias, eps, kind, placement, gate, False, False)
    return y if h is None else (h, y)


def residual_norm_fp8_func(x, shortcut, weight, bias=None, eps=1e-5, kind="layer", placement="post", gate=None):
    """`residual_norm_func` for inference whose y also leaves in 8 bits: -> (stream, y8, scale).

    stream is y (post) or h (pre); y8 [..., dim] (float8_e4m3fn) holds y / scale with one fp32 scale per row, taken from the
    unrounded y (scale = max |y| / 448; in the pre-norm form y itself is not written).  No gradient: raises where one
    would be recorded."""
    _check_norm(x, shortcut, weight, bias, eps, kind, placement, gate)
    assert not _wants_grad(x, shortcut, weight, bias), "the 8-bit form has no gradient: call it under torch.no_grad()"
    y, h, y8, scale, _ = _norm_forward(x, shortcut, weight, bias, eps, kind, placement, gate, False, True)
    return (y if h is None else h), y8, scale


def quantize_rows_func(x):
    """(x8, scale): the rows of x [..., dim] (fp16 / bf16 / fp32, dim <= 16384) in 8 bits (float8_e4m3fn), each divided by
    its own fp32 scale max |x| / 448.  A row with an infinity or a NaN gets a scale that is not finite.  No gradient."""
    assert x.dim() >= 1 and x.shape[-1] > 0, "x must have at least one value per row"
    assert x.dtype in _DTYPES, "Only support fp16, bf16 and fp32"
    _same_device(x)
    assert not _wants_grad(x), "the 8-bit form has no gradient: call it under torch.no_grad()"
    if x.shape[-1] > _abi.NORM_MAX_DIM:
        raise NotImplementedError(f"rows of {x.shape[-1]} values: at most {_abi.NORM_MAX_DIM} are supported")
    x8 = torch.empty(x.shape, device=x.device, dtype=_F8)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    if _count(x) == 0:
        return x8, scale
    xr, stride = _rows(x)
    with _on_device(x.device) as stream:
        _abi.check(_abi.load().fwa2_quantize_rows(xr.data_ptr(), _DTYPES[x.dtype], xr.shape[0], xr.shape[1], stride,
                                                  x8.data_ptr(), scale.data_ptr(), stream), "fwa2_quantize_rows")
    return x8, scale


# ---- matrix products with an epilogue ----------------------------------------------------------------------------------
def _check_linear(x, weight, bias, activation, residual, dtype):
    assert activation in _ACTIVATIONS, f"activation must be one of {[a for a in _ACTIVATIONS if a]} or None"
    assert x.dim() >= 1 and weight.dim() == 2, "x must be [..., in_features] and weight [out_features, in_features]"
    n, k = weight.shape
    assert x.shape[-1] == k and k > 0 and n > 0, "x and weight do not match"
    _same_device(x, weight, bias, residual)
    assert dtype in _HALF, "Only support fp16 and bf16"
    if bias is not None:
        assert bias.shape == (n,) and bias.dtype == dtype, "bias must be [out_features] of the output's dtype"
    if residual is not None:
        assert residual.shape == (*x.shape[:-1], n) and residual.dtype == dtype, \
            "residual must have the shape and dtype of the output"


def _describe_linear(x, weight, activation, dtype):
    p = _abi.new_linear()
    p.dtype, p.x_dtype = _DTYPES[dtype], _abi.E4M3 if x.dtype == _F8 else _DTYPES[dtype]
    p.activation = _ACTIVATIONS[activation]
    p.rows, p.in_features, p.out_features = _count(x), x.shape[-1], weight.shape[0]
    xr, p.x_stride = _rows(x)
    wr, p.weight_stride = _rows(weight)
    p.x, p.weight = xr.data_ptr(), wr.data_ptr()
    p._keep = (xr, wr)
    return p


def _launch_linear(p, device, backward):
    lib = _abi.load()
    with _on_device(device) as stream:
        need = lib.fwa2_linear_workspace_bytes(p, backward)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        p.workspace, p.workspace_bytes, p.stream = _ptr(ws), need, stream
        if backward:
            _abi.check(lib.fwa2_linear_backward(p), "fwa2_linear_backward")
        else:
            _abi.check(lib.fwa2_linear_forward(p), "fwa2_linear_forward")


def _linear_forward(x, weight, bias, activation, residual, dtype, want_z=False, x_scale=None, weight_scale=None):
    shape = (*x.shape[:-1], weight.shape[0])
    y = torch.empty(shape, device=x.device, dtype=dtype)
    z = torch.empty(shape, device=x.device, dtype=dtype) if want_z else None
    if _count(x) == 0:
        return y, z
    p = _describe_linear(x, weight, activation, dtype)
    if bias is not None:
        bias = bias.contiguous()
        p.bias = bias.data_ptr()
    if residual is not None:
        rr, p.residual_stride = _rows(residual)
        p.residual = rr.data_ptr()
    if x_scale is not None:
        x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
        p.x_scale, p.weight_scale = x_scale.data_ptr(), weight_scale.data_ptr()
    p.y, p.z = y.data_ptr(), _ptr(z)
    _launch_linear(p, x.device, 0)
    return y, z


class FusedLinear(torch.autograd.Function):
    """`fused_linear_func` under autograd: keeps x, weight and, behind an activation, the sums before it."""

    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        want_z = _ACTIVATIONS[activation] != _abi.ACT_NONE and any(ctx.needs_input_grad[:3])
        y, z = _linear_forward(x, weight, bias, activation, residual, x.dtype, want_z)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_x else None
        # dbias is summed on the way to dweight
        dw = torch.empty(weight.shape, device=x.device, dtype=x.dtype) if need_w or need_b else None
        db = torch.empty(weight.shape[:1], device=x.device, dtype=x.dtype) if need_b else None
        if _count(x) == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif dx is not None or dw is not None:
            p = _describe_linear(x, weight, ctx.activation, x.dtype)
            dyr, p.dy_stride = _rows(dy)
            p.dy, p.z = dyr.data_ptr(), _ptr(z)
            p.dx, p.dweight, p.dbias = _ptr(dx), _ptr(dw), _ptr(db)
            _launch_linear(p, x.device, 1)
        return dx, (dw if need_w else None), db, None, (dy if need_r else None)


def fused_linear_func(x, weight, bias=None, activation=None, residual=None):
    """act(x @ weight.T + bias) + residual in one kernel, with its gradients.

    x: [..., in_features], weight: [out_features, in_features], bias: [out_features] or None, residual: the shape of the
    output or None, all of one dtype (fp16 or bf16); activation: None, "gelu", "gelu_tanh", "silu" or "relu".  Products are
    accumulated in fp32 and the output is rounded once.  Gradients for x, weight, bias and residual; behind an activation
    the sums before it are kept in the dtype of x for the backward pass."""
    _check_linear(x, weight, bias, activation, residual, x.dtype)
    assert weight.dtype == x.dtype, "x and weight must have the same dtype"
    if _wants_grad(x, weight, bias, residual):
        return FusedLinear.apply(x, weight, bias, activation, residual)
    return _linear_forward(x, weight, bias, activation, residual, x.dtype)[0]


def fused_linear_fp8_func(x8, x_scale, weight8, weight_scale, bias=None, activation=None, residual=None,
                          out_dtype=torch.bfloat16):
    """`fused_linear_func` for inference over 8-bit rows: act((x8 * x_scale) @ (weight8 * weight_scale).T + bias) + residual.

    x8: [..., in_features] and weight8: [out_features, in_features], float8_e4m3fn; x_scale: [...] and weight_scale:
    [out_features], fp32, as `quantize_rows_func` and `residual_norm_fp8_func` return them; bias, residual and the result
    are of `out_dtype` (fp16 or bf16).  No gradient: raises where one would be recorded."""
    _check_linear(x8, weight8, bias, activation, residual, out_dtype)
    assert x8.dtype == _F8 and weight8.dtype == _F8, "x8 and weight8 must be float8_e4m3fn"
    assert x_scale.dtype == torch.float32 and x_scale.shape == x8.shape[:-1], "x_scale must hold one fp32 value per row"
    assert weight_scale.dtype == torch.float32 and weight_scale.shape == weight8.shape[:1], \
        "weight_scale must hold one fp32 value per row of weight8"
    _same_device(x8, x_scale, weight_scale)
    assert not _wants_grad(bias, residual, x_scale, weight_scale), \
        "the 8-bit form has no gradient: call it under torch.no_grad()"
    return _linear_forward(x8, weight8, bias, activation, residual, out_dtype, False, x_scale, weight_scale)[0]
