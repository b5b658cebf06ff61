"""Refusals and host-side decisions of the operators around the attention call, without a GPU: what the C entry points reject
before they touch a device, and what the Python layer asserts."""
import ctypes
import os

import pytest
import torch

import flash_window_attention_v2_amd as fwa2
from flash_window_attention_v2_amd import _abi
from block_ops_exact import constant_rows, constant_rows_bound, layer, layer_sums
from block_ops_ref import slope64

FAKE = 0x100000     # never dereferenced by a validation


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_abi.lib_path()):
        import __graft_entry__

        __graft_entry__.build()
    return _abi.load()


def _norm(backward=False, pre=False):
    p = _abi.new_norm()
    p.dtype = p.stream_dtype = p.param_dtype = _abi.BF16
    p.kind, p.placement, p.eps = _abi.NORM_LAYER, _abi.NORM_PRE if pre else _abi.NORM_POST, 1e-5
    p.rows, p.dim = 64, 96
    p.x, p.x_stride, p.shortcut, p.shortcut_stride = FAKE, 96, FAKE, 96
    p.weight, p.bias, p.y = FAKE, FAKE, FAKE
    if pre:
        p.h = FAKE
    if backward:
        p.stats, p.dy, p.dy_stride, p.dx, p.dweight, p.dbias = FAKE, FAKE, 96, FAKE, FAKE, FAKE
        p.workspace, p.workspace_bytes = FAKE, 1 << 30
    return p


def _refuse(lib, check, p, backward, code, text):
    assert check(ctypes.byref(p), backward) == code
    assert text in lib.fwa2_last_error().decode(), lib.fwa2_last_error()


def test_norm_validate(lib):
    check = lib.fwa2_norm_validate
    for pre in (False, True):
        assert check(_norm(pre=pre), 0) == _abi.OK
        assert check(_norm(True, pre), 1) == _abi.OK
    bad = _abi.ERR_INVALID_ARGUMENT

    def refuse(text, code=bad, backward=0, pre=False, **fields):
        p = _norm(backward, pre)
        for k, v in fields.items():
            setattr(p, k, v)
        _refuse(lib, check, p, backward, code, text)

    assert check(None, 0) == bad
    refuse("layout mismatch", struct_bytes=8)
    refuse("layout mismatch", abi_version=3)
    refuse("fp16, bf16 or fp32", dtype=7)
    refuse("dtype or fp32", stream_dtype=_abi.F16)
    refuse("dtype or fp32", param_dtype=_abi.E4M3)
    refuse("kind", kind=2)
    refuse("placement", placement=5)
    for eps in (0.0, -1.0, 1e-40, float("nan"), float("inf")):
        refuse("eps", eps=eps)
    refuse("rows", rows=0)
    refuse("rows", rows=1 << 31)
    refuse("dim", dim=0)
    refuse("at most", code=_abi.ERR_UNSUPPORTED, dim=_abi.NORM_MAX_DIM + 1)
    refuse("x: null", x=0)
    refuse("x: row stride", x_stride=95)
    refuse("x: pointer", x=FAKE + 1)
    refuse("weight", weight=0)
    refuse("y: null", y=0)
    refuse("shortcut", pre=True, shortcut=0)
    refuse("h: null", pre=True, h=0)
    refuse("y8_scale", y8=FAKE)
    refuse("gate must be", gate=FAKE, gate_dtype=_abi.F16, rows_per_gate=64)
    for per in (0, -1, 7, 65):
        refuse("rows_per_gate", gate=FAKE, gate_dtype=_abi.BF16, rows_per_gate=per)
    refuse("dy: null", backward=1, dy=0)
    refuse("dy: row stride", backward=1, dy_stride=5)
    refuse("stats", backward=1, stats=0)
    refuse("dshortcut", backward=1, dshortcut=FAKE)
    refuse("workspace", backward=1, workspace=0)
    refuse("need", backward=1, workspace_bytes=8)
    refuse("aligned", backward=1, workspace=FAKE + 8)
    refuse("h: null", backward=1, pre=True, h=0, stream_dtype=_abi.F32)
    refuse("x: null", backward=1, pre=True, x=0)
    refuse("shortcut: null", backward=1, pre=True, shortcut=0)
    p = _norm(True, True)       # both incoming gradients may be absent on their own
    p.dy = 0
    assert check(p, 1) == _abi.OK
    # the 8-bit form of the pre-norm does without y
    p = _norm(pre=True)
    p.y, p.y8, p.y8_scale = 0, FAKE, FAKE
    assert check(p, 0) == _abi.OK


def test_norm_workspace(lib):
    p = _norm(True)
    need = lib.fwa2_norm_workspace_bytes(p)
    assert need > 0 and need % (2 * 96 * 4) == 0
    p.dweight = p.dbias = 0
    assert lib.fwa2_norm_workspace_bytes(p) == 0
    for rows, dim in ((0, 96), (1 << 40, 96), (4, 0), (4, 1 << 30)):
        p = _norm(True)
        p.rows, p.dim = rows, dim
        assert lib.fwa2_norm_workspace_bytes(p) == 0


def test_quantize_refuses(lib):
    bad = _abi.ERR_INVALID_ARGUMENT
    q = lib.fwa2_quantize_rows
    assert q(FAKE, 9, 4, 8, 8, FAKE, FAKE, None) == bad
    assert q(FAKE, _abi.F16, 0, 8, 8, FAKE, FAKE, None) == bad
    assert q(FAKE, _abi.F16, 4, 0, 8, FAKE, FAKE, None) == bad
    assert q(FAKE, _abi.F16, 4, 8, 7, FAKE, FAKE, None) == bad
    assert q(None, _abi.F16, 4, 8, 8, FAKE, FAKE, None) == bad
    assert q(FAKE, _abi.F16, 4, 8, 8, None, FAKE, None) == bad
    assert q(FAKE, _abi.F16, 4, 8, 8, FAKE, None, None) == bad
    assert q(FAKE, _abi.F16, 4, _abi.NORM_MAX_DIM + 1, 1 << 20, FAKE, FAKE, None) == _abi.ERR_UNSUPPORTED


def _linear(backward=False, f8=False):
    p = _abi.new_linear()
    p.dtype, p.x_dtype, p.activation = _abi.BF16, _abi.E4M3 if f8 else _abi.BF16, _abi.ACT_GELU
    p.rows, p.in_features, p.out_features = 100, 96, 384
    p.x, p.x_stride, p.weight, p.weight_stride = FAKE, 96, FAKE, 96
    p.bias, p.residual, p.residual_stride, p.y, p.z = FAKE, FAKE, 384, FAKE, FAKE
    if f8:
        p.x_scale = p.weight_scale = FAKE
    if backward:
        p.dy, p.dy_stride, p.dx, p.dweight, p.dbias = FAKE, 384, FAKE, FAKE, FAKE
    p.workspace, p.workspace_bytes = FAKE, 1 << 30
    return p


def test_linear_validate(lib):
    check = lib.fwa2_linear_validate
    assert check(_linear(), 0) == check(_linear(True), 1) == check(_linear(f8=True), 0) == _abi.OK
    bad, no = _abi.ERR_INVALID_ARGUMENT, _abi.ERR_UNSUPPORTED

    def refuse(text, code=bad, backward=0, f8=False, **fields):
        p = _linear(backward, f8)
        for k, v in fields.items():
            setattr(p, k, v)
        _refuse(lib, check, p, backward, code, text)

    assert check(None, 0) == bad
    refuse("layout mismatch", struct_bytes=8)
    refuse("fp16 and bf16", dtype=_abi.F32)
    refuse("e4m3", x_dtype=_abi.F16)
    refuse("activation", activation=5)
    refuse("activation", activation=-1)
    for field in ("rows", "in_features", "out_features"):
        refuse("positive", **{field: 0})
        refuse("positive", **{field: -3})
    refuse("positive", rows=1 << 31)
    refuse("too large", no, in_features=1 << 22, x_stride=1 << 22, weight_stride=1 << 22)
    refuse("too large", no, out_features=1 << 22, residual_stride=1 << 22)
    refuse("too large", no, rows=(1 << 31) - 1, out_features=1 << 20)
    refuse("x: null", x=0)
    refuse("weight: null", weight=0)
    refuse("x: row stride", x_stride=95)
    refuse("2^22", no, x_stride=1 << 22)
    refuse("2^22", no, weight_stride=1 << 22)
    refuse("2^22", no, residual_stride=1 << 23)
    refuse("residual: row stride", residual_stride=383)
    refuse("y: null", y=0)
    refuse("x_scale", f8=True, x_scale=0)
    refuse("weight_scale", f8=True, weight_scale=0)
    refuse("no backward", no, backward=1, f8=True)
    refuse("dy: null", backward=1, dy=0)
    refuse("z: null", backward=1, z=0)
    refuse("without dweight", backward=1, dweight=0)
    refuse("need", backward=1, workspace_bytes=8)
    refuse("aligned", backward=1, workspace=FAKE + 16)
    p = _linear(True)
    p.activation, p.z = _abi.ACT_NONE, 0        # nothing is kept without an activation
    assert check(p, 1) == _abi.OK
    p = _linear(True)
    p.x, p.dweight, p.dbias = 0, 0, 0           # x is read for dweight alone
    assert check(p, 1) == _abi.OK


def test_linear_workspace(lib):
    need = lib.fwa2_linear_workspace_bytes
    p = _linear(True)
    assert need(p, 1) >= 100 * 384 * 2                          # dz
    p.rows = 0
    assert need(p, 1) == 0 and need(None, 1) == 0
    p = _linear(True)
    p.activation = _abi.ACT_NONE
    p.rows = 1 << 18
    with_dw = need(p, 1)
    assert with_dw % 4 == 0 and 0 < with_dw < 1 << 28           # partial weight gradients of a split contraction
    p.dweight = p.dbias = 0
    assert need(p, 1) == 0


def test_python_refusals_without_a_gpu():
    x, w, b = torch.zeros(4, 8), torch.zeros(8), torch.zeros(8)
    with pytest.raises(AssertionError, match="GPU"):
        fwa2.residual_norm_func(x, x, w, b)
    with pytest.raises(AssertionError, match="GPU"):
        fwa2.residual_norm_fp8_func(x, x, w, b)
    with pytest.raises(AssertionError, match="GPU"):
        fwa2.quantize_rows_func(x)
    with pytest.raises(AssertionError, match="GPU"):
        fwa2.fused_linear_func(x.half(), torch.zeros(3, 8).half())
    with pytest.raises(AssertionError, match="kind"):
        fwa2.residual_norm_func(x, x, w, b, kind="batch")
    with pytest.raises(AssertionError, match="placement"):
        fwa2.residual_norm_func(x, x, w, b, placement="middle")
    with pytest.raises(AssertionError, match="activation"):
        fwa2.fused_linear_func(x.half(), torch.zeros(3, 8).half(), activation="mish")
    with pytest.raises(AssertionError, match="do not match"):
        fwa2.fused_linear_func(x.half(), torch.zeros(3, 7).half())
    with pytest.raises(AssertionError, match="at least one value"):
        fwa2.quantize_rows_func(torch.zeros(4, 0))


def test_rows_are_views_where_they_can_be(lib):
    as_rows = _abi.load_ext().rows
    a = torch.zeros(4, 6, 40)
    for t, stride, view in [(a, 40, True), (a[..., 3:20], 40, True), (a[:, :, ::2], 20, False), (a[0], 40, True),
                            (a[:, 0], 240, True), (a[:, :3], 40, False), (a[:1, :1], 40, True), (a[0, 0], 40, True),
                            (a[:, :1].expand(4, 6, 40), 40, False), (a.transpose(1, 2), 6, False)]:
        rows, got = as_rows(t)
        assert rows.dim() == 2 and rows.shape == (t.numel() // t.shape[-1], t.shape[-1]) and got == stride
        assert (rows.untyped_storage().data_ptr() == a.untyped_storage().data_ptr()) == view
        assert torch.equal(rows.reshape(t.shape), t)
    far = torch.zeros(8).as_strided((1, 8), (1 << 30, 1))
    assert as_rows(far)[1] == 8         # the stride of a single row means nothing


def test_struct_sizes_match_the_header(lib):
    # the library reports the size it was compiled with when it is given another one
    for new, check in ((_abi.new_norm, lib.fwa2_norm_validate), (_abi.new_linear, lib.fwa2_linear_validate)):
        p = new()
        size = ctypes.sizeof(p)
        p.struct_bytes = 1
        check(ctypes.byref(p), 0)
        assert f"library {size} bytes" in lib.fwa2_last_error().decode()


def test_rows_of_lazily_negated_views_are_negated(lib):
    # the imaginary part of a conjugate: a real tensor whose memory holds the negated values
    z = torch.randn(3, 8, dtype=torch.complex64)
    neg = z.conj().imag
    assert neg.is_neg()
    rows, stride = _abi.load_ext().rows(neg)
    assert not rows.is_neg() and torch.equal(rows, -z.imag) and stride == 8
    dense = torch._neg_view(torch.randn(3, 8))
    rows, stride = _abi.load_ext().rows(dense)
    assert not rows.is_neg() and torch.equal(rows, dense) and stride == 8


@pytest.mark.parametrize("placement", ["post", "pre"])
def test_no_rows_and_no_gates(lib, monkeypatch, placement):
    # a batch of no samples under stochastic depth: no factors either, and empty results (no kernel runs: the CPU will do)
    from flash_window_attention_v2_amd import block_ops

    monkeypatch.setattr(block_ops, "_same_device", lambda *a: None)
    x, w = torch.empty(0, 5, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    gate = torch.empty(0, 1, 1)
    out = fwa2.residual_norm_func(x, x, w, w, placement=placement, gate=gate)
    for t in out if placement == "pre" else (out,):
        assert t.shape == x.shape
    (out[1] if placement == "pre" else out).sum().backward()
    assert x.grad.shape == x.shape and (w.grad == 0).all()
    with torch.no_grad():
        assert fwa2.residual_norm_fp8_func(x, x, w, w, placement=placement, gate=gate)[1].shape == x.shape
    with pytest.raises(AssertionError, match="one factor per sample"):
        fwa2.residual_norm_func(torch.ones(4, 8), None, w, gate=torch.empty(0))
    with pytest.raises(AssertionError, match="one factor per sample"):
        fwa2.residual_norm_func(torch.ones(4, 8), None, w, gate=torch.ones(3))


# ---- the inputs of the exact sums, with mistakes planted in the oracle ---------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,stretch", [(70000, 8, 8, 320), (16500, 64, 136, 320), (16500, 64, 136, 65), (5000, 96, 96, 20)])
def test_exact_sums_show_a_lost_or_doubled_partial(m, k, n, stretch, dtype):
    x, w, b, dy = layer(m, k, n, dtype, "cpu", m)
    for act in (None, "relu"):
        sums = layer_sums(x, w, b, dy, act)
        want = {name: t.to(dtype) for name, t in sums.items()}
        for lo in range(0, m, stretch):
            part = layer_sums(x[lo:lo + stretch], w, b, dy[lo:lo + stretch], act)
            for name in ("dw", "db"):
                for sign in (-1, 1):
                    assert not torch.equal((sums[name] + sign * part[name]).to(dtype), want[name]), (act, name, lo)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_constant_rows_show_rounded_gradients(act, dtype):
    # the bound that dbias is held to refuses sums of dz rounded to dtype, and takes sums in fp32
    m, n = 300, 512
    z, dy = constant_rows(act, n, dtype, "cpu", 3)
    dz = dy.double() * slope64(z.double(), act)
    bound = constant_rows_bound(m * dz, m, dtype)
    good = dz.float().expand(m, n).sum(0).to(dtype).double()
    assert ((good - m * dz).abs() <= bound).all()
    rounded_first = dz.to(dtype).float().expand(m, n).sum(0).to(dtype).double()
    assert int(((rounded_first - m * dz).abs() > bound).sum()) > n // 10
