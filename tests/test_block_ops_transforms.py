"""What follows a computation from the outside (forward-mode derivatives, tracers, torch.func) does not see into the operators
around the attention call: they refuse where it would lose something.  Empty rows: no kernel runs, so this needs no GPU."""
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

from flash_window_attention_v2_amd import _abi


@pytest.fixture(scope="module")
def ext():
    if not os.path.exists(_abi.lib_path()):
        import __graft_entry__

        __graft_entry__.build()
    return _abi.load_ext()


F16 = torch.float16
X, W, B, R = torch.empty(0, 8, dtype=F16), torch.ones(16, 8, dtype=F16), torch.ones(16, dtype=F16), torch.empty(0, 16, dtype=F16)
V, G = torch.ones(8, dtype=F16), torch.ones(1, dtype=F16)
X8, W8, S, SW = X.to(torch.float8_e4m3fn), W.to(torch.float8_e4m3fn), torch.empty(0), torch.ones(16)

# every call with the arguments that may carry a derivative
CALLS = {
    "linear": (lambda e: lambda x, w, b, r: e.linear(x, w, b, _abi.ACT_GELU, r), (X, W, B, R)),
    "linear_fp8": (lambda e: lambda s, sw, b, r: e.linear_fp8(X8, s, W8, sw, b, 0, r, False), (S, SW, B, R)),
    "norm": (lambda e: lambda x, s, w, b, g: e.norm(x, s, w, b, 1e-5, 0, 1, g), (X, X, V, V, G)),
    "norm_fp8": (lambda e: lambda x, s, w, b, g: e.norm_fp8(x, s, w, b, 1e-5, 0, 0, g), (X, X, V, V, G)),
    "quantize_rows": (lambda e: lambda x: e.quantize_rows(x), (X,)),
}


@pytest.mark.parametrize("name", CALLS)
def test_inputs_with_a_forward_derivative_are_refused(ext, name):
    make, args = CALLS[name]
    call = make(ext)
    call(*args)
    for i in range(len(args)):
        with fwAD.dual_level():
            dual = [fwAD.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)
        with fwAD.dual_level():         # a level alone is no reason
            call(*args)


def test_a_recorded_call_refuses_a_forward_derivative_too(ext):
    call = CALLS["linear"][0](ext)
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwAD.make_dual(X, torch.ones_like(X)), W.clone().requires_grad_(), B, R)


@pytest.mark.parametrize("placement", [0, 1])
def test_a_backward_pass_refuses_a_forward_derivative(ext, placement):
    # the derivative of a gradient along a direction: forward mode over the recorded backward pass
    leaves = [t.clone().requires_grad_() for t in (X, W, B, R)]
    y = ext.linear(*leaves[:3], _abi.ACT_GELU, leaves[3])
    out = ext.norm(leaves[0], leaves[0], V.clone().requires_grad_(), None, 1e-5, 0, placement, None)
    with fwAD.dual_level():
        dy = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode"):
            torch.autograd.grad(y, leaves, dy)
        for o in out:
            d = fwAD.make_dual(torch.ones_like(o), torch.ones_like(o))
            with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode"):
                torch.autograd.grad(o, leaves[0], d, retain_graph=True)


@pytest.mark.parametrize("name", CALLS)
def test_transforms_of_torch_func_are_refused(ext, name):
    make, args = CALLS[name]
    call = make(ext)

    def first(*a):
        out = call(*a)
        return out if isinstance(out, torch.Tensor) else out[0]

    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(first, args, tuple(torch.ones_like(a) for a in args))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda *a: first(*a).float().sum())(*args)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.vmap(lambda a: first(a, *args[1:]))(torch.stack([args[0], args[0]]))


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("recorded", [False, True])
def test_tracers_are_refused(ext, name, recorded):
    """A trace would hold the output's allocation and not what fills it."""
    make, args = CALLS[name]
    call = make(ext)
    if recorded:
        if name in ("linear_fp8", "norm_fp8", "quantize_rows"):
            return
        args = tuple(a.clone().requires_grad_(i < 2) for i, a in enumerate(args))

    def first(*a):
        out = call(*a)
        return out if isinstance(out, torch.Tensor) else out[0]

    with pytest.raises((NotImplementedError, RuntimeError), match="trace"):
        torch.jit.trace(first, args, check_trace=False)
    with pytest.raises((NotImplementedError, RuntimeError), match="trace"):
        make_fx(first)(*(a.detach() for a in args))
    assert first(*args).shape[0] == 0           # afterwards as before
