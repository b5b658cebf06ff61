"""The Swin block's second half on the library's kernels: the model with `is_fused` against the same model without, and where
the fused path steps aside."""
import copy

import pytest
import torch
import torch.nn as nn

from flash_window_attention_v2_amd import SwinTransformerV2
from flash_window_attention_v2_amd import swin_transformer_v2 as swin

KW = dict(img_size=32, patch_size=2, embed_dim=32, depths=[2, 2], num_heads=[1, 2], window_size=8, num_classes=10,
          drop_path_rate=0.0)


def _pair(**kw):
    torch.manual_seed(0)
    plain = SwinTransformerV2(**{**KW, **kw})
    fused = SwinTransformerV2(**{**KW, **kw}, is_fused=True)
    fused.load_state_dict(plain.state_dict())
    for m in (plain, fused):        # post-norms start at zero: give them something to do, the same in both
        g = torch.Generator().manual_seed(1)
        for blk in m.modules():
            if isinstance(blk, swin.SwinTransformerBlock):
                for n in (blk.norm1, blk.norm2):
                    nn.init.normal_(n.weight, 0.5, 0.1, generator=g)
                    nn.init.normal_(n.bias, 0.0, 0.1, generator=g)
    return plain, fused


def test_on_the_cpu_nothing_changes():
    plain, fused = _pair(is_flash=False)
    x = torch.randn(2, 3, 32, 32)
    assert set(plain.state_dict()) == set(fused.state_dict())
    assert torch.equal(plain(x), fused(x))
    assert not any(m.is_fused for m in plain.modules() if isinstance(m, swin.Mlp))
    assert all(m.is_fused and not m.fp8 for m in fused.modules() if isinstance(m, swin.Mlp))
    fp8 = SwinTransformerV2(**KW, is_flash=False, is_fused=True, fp8_mlp=True)
    assert all(m.fp8 for m in fp8.modules() if isinstance(m, swin.Mlp))
    assert not any(m.fp8 for m in SwinTransformerV2(**KW, is_flash=False, fp8_mlp=True).modules() if isinstance(m, swin.Mlp))


def test_gate_is_drawn_as_drop_path_draws_it():
    blk = swin.SwinTransformerBlock(16, (8, 8), 1, window_size=4, drop_path=0.4, is_flash=False, is_fused=True).train()
    x = torch.randn(64, 64, 16)
    torch.manual_seed(3)
    want = swin.drop_path(x, 0.4, True)
    torch.manual_seed(3)
    assert torch.allclose(want, blk._gate(x) * x)
    assert blk.eval()._gate(x) is None


def _grads(m, x, dy):
    m.zero_grad()
    y = m(x)
    y.backward(dy)
    return y.detach(), {k: p.grad.detach().clone() for k, p in m.named_parameters() if p.grad is not None}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("flash", [True, False])
def test_fused_model_against_the_plain_one_in_fp32(dtype, flash):
    plain, fused = _pair(is_flash=flash)
    exact = SwinTransformerV2(**KW, is_flash=False)
    exact.load_state_dict(plain.state_dict())
    exact, plain, fused = exact.cuda().double(), plain.cuda().to(dtype), fused.cuda().to(dtype)
    exact.load_state_dict({k: v.double() if v.is_floating_point() else v for k, v in plain.state_dict().items()})
    torch.manual_seed(5)
    x, dy = torch.randn(4, 3, 32, 32, device="cuda").to(dtype), torch.randn(4, 10, device="cuda").to(dtype)
    want, wg = _grads(exact, x.double(), dy.double())
    (py, pg), (fy, fg) = _grads(plain, x, dy), _grads(fused, x, dy)
    assert set(pg) == set(fg) == set(wg)

    def rel(a, b):
        return float((a.double() - b).norm() / b.norm())

    # the fused form leaves out roundings of the plain one; what both share (the attention) sets the level
    half = torch.finfo(dtype).eps / 2
    assert rel(fy, want) <= 1.5 * rel(py, want) + 2 * half
    # gradients of the block's own second half, which the fused calls compute
    for k in wg:
        if "blocks" in k and (".norm" in k or ".mlp." in k):
            assert rel(fg[k], wg[k]) <= 1.5 * rel(pg[k], wg[k]) + 4 * half, k


@pytest.mark.gpu
def test_fused_calls_are_made(monkeypatch):
    _, fused = _pair()
    fused = fused.cuda().to(torch.bfloat16)
    x = torch.randn(2, 3, 32, 32, device="cuda", dtype=torch.bfloat16)
    calls = []
    for name in ("fused_linear_func", "residual_norm_func", "residual_norm_fp8_func", "fused_linear_fp8_func", "quantize_rows_func"):
        real = getattr(swin, name)
        monkeypatch.setattr(swin, name, lambda *a, _n=name, _f=real, **k: (calls.append(_n), _f(*a, **k))[1])
    fused(x)
    assert calls.count("fused_linear_func") == 8 and calls.count("residual_norm_func") == 8 and len(calls) == 16
    calls.clear()
    # a hook on a part of the MLP, an unknown activation, active dropout: the parts are called one by one
    blk = fused.layers[0].blocks[0]
    h = blk.mlp.act.register_forward_hook(lambda *a: None)
    fused(x)
    assert calls.count("fused_linear_func") == 6 and calls.count("residual_norm_func") == 8
    h.remove()
    calls.clear()
    blk.mlp.act = nn.Tanh()
    fused(x)
    assert calls.count("fused_linear_func") == 6
    blk.mlp.act = nn.GELU(approximate="tanh")
    blk.mlp.drop.p = 0.5
    calls.clear()
    fused.train()(x)
    assert calls.count("fused_linear_func") == 6
    calls.clear()
    fused.eval()(x)
    assert calls.count("fused_linear_func") == 8


@pytest.mark.gpu
def test_fp8_mlp(monkeypatch):
    plain, _ = _pair()
    fp8 = SwinTransformerV2(**KW, is_fused=True, fp8_mlp=True)
    fp8.load_state_dict(plain.state_dict())
    fp8, plain = fp8.cuda().to(torch.bfloat16).eval(), plain.cuda().to(torch.bfloat16).eval()
    x = torch.randn(4, 3, 32, 32, device="cuda", dtype=torch.bfloat16)
    calls = []
    real = swin.fused_linear_fp8_func
    monkeypatch.setattr(swin, "fused_linear_fp8_func", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    with torch.no_grad():
        y, want = fp8(x), plain(x)
    assert len(calls) == 8
    # operands of 2^-4 half steps in the MLPs of four blocks whose outputs are normalised and added to a stream
    assert float((y.float() - want.float()).norm() / want.float().norm()) <= 2.0 ** -3
    mlp = fp8.layers[0].blocks[0].mlp
    with torch.no_grad():
        first = fp8(x)
        fp8.hold_weights8()                 # the same weights, quantised once
        held = mlp.weights8()
        assert mlp.weights8() is held and torch.equal(fp8(x), first)
        mlp.fc1.weight.mul_(2)              # an edit that is recorded: no longer those
        assert mlp.weights8() is not held and torch.equal(mlp.weights8()[0][1], held[0][1] * 2)
        assert not torch.equal(fp8(x), first)
        fp8.hold_weights8(False)
        second = fp8(x)
        mlp.fc1.weight.data.mul_(0.5)       # one that is not: nothing is kept between calls
        assert torch.equal(fp8(x), first) and not torch.equal(second, first)
    calls.clear()
    fp8(x).sum().backward()                                  # with gradients the products stay in 16 bits
    assert not calls and fp8.layers[0].blocks[0].mlp.fc1.weight.grad is not None
    with torch.inference_mode():
        assert fp8(x).isfinite().all() and len(calls) == 8


@pytest.mark.gpu
def test_fused_under_autocast_and_checkpointing():
    plain, fused = _pair(use_checkpoint=True)
    fused = fused.cuda()
    plain = plain.cuda()
    x = torch.randn(2, 3, 32, 32, device="cuda")
    outs = []
    for m in (plain, fused):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
        y.float().square().sum().backward()
        outs.append((y.detach(), m.layers[0].blocks[0].mlp.fc1.weight.grad, m.layers[0].blocks[1].norm2.weight.grad))
    assert outs[0][0].dtype == outs[1][0].dtype
    for a, b in zip(*outs):
        assert a.dtype == b.dtype
        # two bf16 evaluations of one model: a few tens of roundings of 2^-8 apart
        assert float((a.float() - b.float()).norm() / a.float().norm()) <= 2.0 ** -4


@pytest.mark.gpu
def test_fused_training_with_stochastic_depth():
    torch.manual_seed(0)
    m = SwinTransformerV2(**{**KW, "drop_path_rate": 0.5}, is_fused=True).cuda().to(torch.bfloat16).train()
    ref = copy.deepcopy(m)
    for mod in ref.modules():
        if hasattr(mod, "is_fused"):
            mod.is_fused = False
    x = torch.randn(8, 3, 32, 32, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        for blk in [b for mm in (m, ref) for b in mm.modules() if isinstance(b, swin.SwinTransformerBlock)]:
            blk.norm1.weight.fill_(0.5), blk.norm2.weight.fill_(0.5)
    torch.manual_seed(9)
    a = m(x)
    torch.manual_seed(9)
    b = ref(x)
    assert float(((a.float() - b.float()).norm() / b.float().norm()).detach()) <= 2.0 ** -4     # the same samples were dropped
