"""The operators around the attention call of a transformer block: normalisation with the residual's addition, matrix
products with an epilogue, and the 8-bit forms of both.

The reference composes them from framework calls (`x + drop_path(norm(x))`, nn.Linear, nn.GELU:
flash_win_attn_v2/swin_transformer_v2.py:66-85, 443-445).  Here each is one HIP kernel forward and two to four backward.
The functions of this file check their arguments; what they call (csrc/fwa2_torch.cpp) allocates outputs and workspaces
as torch tensors, records the gradient and hands raw pointers and strides to libfwa2.so.  As for the attention there is no
CPU path and no fallback.

Tensors of any strides are taken; what the kernels cannot address (an inner stride other than 1, rows that overlap or lie
2^22 elements apart or more) is copied first.  Leading dimensions are flattened to rows.  Every call works on the current
stream of the tensors' device and can be captured into a graph (a backward pass, as with any autograd operator: while no
eager graph of the same leaves is alive, whose nodes belong to another stream); gradients are bit-reproducible and
cannot be differentiated a second time (that raises).  Inputs that carry a forward-mode derivative, the transforms of
torch.func and tracers are refused (NotImplementedError or RuntimeError): they would not see what happens in here.
"""
import torch

from . import _abi

_ACTIVATIONS = {None: _abi.ACT_NONE, "none": _abi.ACT_NONE, "gelu": _abi.ACT_GELU, "gelu_tanh": _abi.ACT_GELU_TANH,
                "silu": _abi.ACT_SILU, "relu": _abi.ACT_RELU}
_KINDS = {"layer": _abi.NORM_LAYER, "rms": _abi.NORM_RMS}
_PLACES = {"post": _abi.NORM_POST, "pre": _abi.NORM_PRE}
_HALF = (torch.float16, torch.bfloat16)
_F8 = torch.float8_e4m3fn
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _count(t):
    n = 1
    for s in t.shape[:-1]:
        n *= s
    return n


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
    assert x.dtype in _FLOATS, "Only support fp16, bf16 and fp32"
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
        assert _count(x) == 0 or (gate.numel() > 0 and _count(x) % gate.numel() == 0), \
            "gate must hold one factor per sample: the rows of x must be a multiple of its size"
        assert not (torch.is_grad_enabled() and gate.requires_grad), "gate gets no gradient"
    if dim > _abi.NORM_MAX_DIM:
        raise NotImplementedError(f"rows of {dim} values: at most {_abi.NORM_MAX_DIM} are supported")
    assert 0.0 < eps < float("inf"), "eps must be positive"


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
    got = _abi.load_ext().norm(x, shortcut, weight, bias, eps, _KINDS[kind], _PLACES[placement], gate)
    return got[0] if placement == "post" else tuple(got)


def residual_norm_fp8_func(x, shortcut, weight, bias=None, eps=1e-5, kind="layer", placement="post", gate=None):
    """`residual_norm_func` for inference whose y also leaves in 8 bits: -> (stream, y8, scale).

    stream is y (post) or h (pre); y8 [..., dim] (float8_e4m3fn) holds y / scale with one fp32 scale per row, taken from the
    unrounded y (scale = max |y| / 448; in the pre-norm form y itself is not written).  No gradient: raises where one
    would be recorded."""
    _check_norm(x, shortcut, weight, bias, eps, kind, placement, gate)
    assert not _wants_grad(x, shortcut, weight, bias), "the 8-bit form has no gradient: call it under torch.no_grad()"
    return tuple(_abi.load_ext().norm_fp8(x, shortcut, weight, bias, eps, _KINDS[kind], _PLACES[placement], gate))


def quantize_rows_func(x):
    """(x8, scale): the rows of x [..., dim] (fp16 / bf16 / fp32, dim <= 16384) in 8 bits (float8_e4m3fn), each divided by
    its own fp32 scale max |x| / 448.  A row with an infinity or a NaN gets a scale that is not finite.  No gradient."""
    assert x.dim() >= 1 and x.shape[-1] > 0, "x must have at least one value per row"
    assert x.dtype in _FLOATS, "Only support fp16, bf16 and fp32"
    _same_device(x)
    assert not _wants_grad(x), "the 8-bit form has no gradient: call it under torch.no_grad()"
    if x.shape[-1] > _abi.NORM_MAX_DIM:
        raise NotImplementedError(f"rows of {x.shape[-1]} values: at most {_abi.NORM_MAX_DIM} are supported")
    return _abi.load_ext().quantize_rows(x)


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


def fused_linear_func(x, weight, bias=None, activation=None, residual=None):
    """act(x @ weight.T + bias) + residual in one kernel, with its gradients.

    x: [..., in_features], weight: [out_features, in_features], bias: [out_features] or None, residual: the shape of the
    output or None, all of one dtype (fp16 or bf16); activation: None, "gelu", "gelu_tanh", "silu" or "relu".  Products are
    accumulated in fp32 and the output is rounded once.  Gradients for x, weight, bias and residual; behind an activation
    the sums before it are kept in the dtype of x for the backward pass."""
    _check_linear(x, weight, bias, activation, residual, x.dtype)
    assert weight.dtype == x.dtype, "x and weight must have the same dtype"
    return _abi.load_ext().linear(x, weight, bias, _ACTIVATIONS[activation], residual)


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
    return _abi.load_ext().linear_fp8(x8, x_scale, weight8, weight_scale, bias, _ACTIVATIONS[activation], residual,
                                      out_dtype == torch.bfloat16)
