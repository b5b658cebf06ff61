"""Where the block's second half leaves its modules to themselves: what a user may have put into a block, or hung on its parts,
has to happen with `is_fused` as without it."""
import copy

import pytest
import torch
import torch.nn as nn

from flash_window_attention_v2_amd import swin_transformer_v2 as swin


def _block(**kw):
    torch.manual_seed(0)
    blk = swin.SwinTransformerBlock(**{**dict(dim=16, input_resolution=(8, 8), num_heads=1, window_size=4, is_flash=False), **kw})
    for n in (blk.norm1, blk.norm2):
        nn.init.normal_(n.weight, 1.0, 0.1)
    return blk


@pytest.mark.parametrize("is_fused", [False, True])
@pytest.mark.parametrize("grad", [torch.no_grad, torch.inference_mode, torch.enable_grad])
def test_a_block_takes_any_module_as_its_mlp(is_fused, grad):
    blk = _block(is_fused=is_fused, fp8_mlp=is_fused).eval()
    x = torch.randn(2, 64, 16)
    for mlp in (nn.Sequential(nn.Linear(16, 16), nn.GELU()), nn.Identity()):
        blk.mlp = mlp
        with grad():
            s = x + blk.norm1(_attention(blk, x))
            assert torch.allclose(blk(x), s + blk.norm2(mlp(s)), atol=1e-6)


def _attention(blk, x):
    """The block's first half, by its modules."""
    windows = swin.window_partition(x.view(-1, 8, 8, 16), 4).view(-1, 16, 16)
    return swin.window_reverse(blk.attn(windows).view(-1, 4, 4, 16), 4, 8, 8).reshape(x.shape)


def test_an_mlp_of_another_class_is_called(monkeypatch):
    # the 8-bit path goes around the Mlp's forward: only where that is the one it stands for
    class Other(swin.Mlp):
        def forward(self, x):
            called.append(1)
            return x

    called = []
    blk = _block(is_fused=True, fp8_mlp=True).eval()
    blk.mlp = Other(16, 64)
    monkeypatch.setattr(swin.Mlp, "fp8_ready", lambda self, x: True)
    monkeypatch.setattr(swin.Mlp, "fused_dtype", lambda self, x: torch.float16)
    monkeypatch.setattr(swin.Mlp, "forward_fp8", lambda self, x8, scale, dtype: x8)
    monkeypatch.setattr(blk, "_norm_fused", lambda *a: True)
    monkeypatch.setattr(swin, "residual_norm_func", lambda x, s, *a, **k: s + x)
    monkeypatch.setattr(swin, "residual_norm_fp8_func", lambda x, s, *a, **k: (s + x, s + x, None))
    with torch.no_grad():
        blk._second_half(torch.randn(2, 64, 16), torch.randn(2, 64, 16))
    assert called


def test_a_block_saved_without_is_fused_still_runs():
    # a block pickled whole before it had the attribute
    blk = _block()
    blk.__dict__.pop("is_fused", None)
    x = torch.randn(2, 64, 16)
    want = _block()(x)
    assert torch.equal(blk(x), want)
    with torch.no_grad():
        assert torch.equal(blk(x), want)


class OnGpu:
    """What the decisions look at of an input."""
    is_cuda, dtype, requires_grad, shape = True, torch.bfloat16, False, (2, 64, 16)


def _mlp(**kw):
    mlp = swin.Mlp(16, 64, **kw).to(torch.bfloat16)
    mlp.is_fused = True
    return mlp


def test_dropout_is_judged_by_its_own_mode():
    mlp = _mlp(drop=0.5)
    assert mlp.fused_dtype(OnGpu) is None                    # training: active
    assert mlp.eval().fused_dtype(OnGpu) is torch.bfloat16
    mlp.drop.train()                                         # Monte-Carlo dropout: a module in evaluation drops all the same
    assert mlp.fused_dtype(OnGpu) is None
    mlp.train()
    mlp.drop.eval()
    assert mlp.fused_dtype(OnGpu) is torch.bfloat16
    mlp.drop.train()
    mlp.drop.p = 0.0
    assert mlp.fused_dtype(OnGpu) is torch.bfloat16
    mlp.drop = nn.Identity()                                 # a model without its dropout modules
    assert mlp.fused_dtype(OnGpu) is torch.bfloat16
    mlp.drop = nn.AlphaDropout(0.5).eval()
    assert mlp.fused_dtype(OnGpu) is None


@pytest.mark.parametrize("block_mode", [False, True])
@pytest.mark.parametrize("path_mode", [False, True])
def test_stochastic_depth_is_judged_by_its_own_mode(block_mode, path_mode):
    blk = _block(drop_path=0.4, is_fused=True).train(block_mode)
    blk.drop_path.train(path_mode)
    x = torch.randn(64, 64, 16)
    torch.manual_seed(3)
    want = blk.drop_path(x)
    torch.manual_seed(3)
    gate = blk._gate(x)
    assert (gate is None) == (not path_mode)
    assert torch.allclose(want, x if gate is None else gate * x)


def _fits(blk):
    """Whether the block's two norms and its Mlp would run fused, by what they look at before a call."""
    x = OnGpu()
    x.shape = (2, 64, 16)
    return blk._norm_fused(blk.norm1, x, x), blk.mlp.fused_dtype(x) is not None, blk._norm_fused(blk.norm2, x, x)


def _fused_block(**kw):
    return _block(is_fused=True, **kw).to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre"])
def test_hooks_of_all_modules_are_seen(kind):
    assert _fits(_fused_block()) == (True, True, True)
    hook = getattr(torch.nn.modules.module, f"register_module_{kind}_hook")(lambda *a: None)
    try:
        assert _fits(_fused_block()) == (False, False, False)
    finally:
        hook.remove()
    assert _fits(_fused_block()) == (True, True, True)


def test_a_forward_replaced_on_the_instance_is_seen():
    def replaced(m):
        forward = m.forward
        m.forward = lambda *a: forward(*a)

    for part, want in (("norm1", (False, True, True)), ("norm2", (True, True, False)), ("drop_path", (False, True, False)),
                       ("mlp.fc1", (True, False, True)), ("mlp.act", (True, False, True)), ("mlp.fc2", (True, False, True)),
                       ("mlp.drop", (True, False, True))):
        blk = _fused_block(drop_path=0.1, drop=0.1).eval()
        assert _fits(blk) == (True, True, True)
        replaced(blk.get_submodule(part))
        assert _fits(blk) == want, part


def test_a_forward_replaced_on_the_mlp_is_called(monkeypatch):
    blk = _block(is_fused=True, fp8_mlp=True).eval()
    called = []
    blk.mlp.forward = lambda x: (called.append(1), x)[1]
    monkeypatch.setattr(swin.Mlp, "fp8_ready", lambda self, x: True)
    monkeypatch.setattr(swin.Mlp, "fused_dtype", lambda self, x: torch.float16)
    monkeypatch.setattr(swin.Mlp, "forward_fp8", lambda self, x8, scale, dtype: x8)
    monkeypatch.setattr(blk, "_norm_fused", lambda *a: True)
    monkeypatch.setattr(swin, "residual_norm_func", lambda x, s, *a, **k: s + x)
    monkeypatch.setattr(swin, "residual_norm_fp8_func", lambda x, s, *a, **k: (s + x, s + x, None))
    with torch.no_grad():
        blk._second_half(torch.randn(2, 64, 16), torch.randn(2, 64, 16))
    assert called


def test_an_eps_that_the_kernels_refuse_steps_aside():
    for eps in (0.0, 1e-40, 1e39):
        blk = _fused_block()
        blk.norm1.eps = eps
        assert _fits(blk) == (False, True, True)
    for eps in (2.0 ** -126, 1e-12, 3e38):
        blk = _fused_block()
        blk.norm2.eps = eps
        assert _fits(blk) == (True, True, True)


def test_tracers_and_transforms_get_the_modules():
    """The functions refuse these; the block's modules know how to go along."""
    import torch.autograd.forward_ad as fwAD
    from torch.fx.experimental.proxy_tensor import make_fx

    seen, blk = [], _fused_block()

    def look(x):
        seen.append(_fits(blk))
        return x * 2

    x = torch.ones(3)
    torch.jit.trace(look, x, check_trace=False)
    make_fx(look)(x)
    with fwAD.dual_level():
        look(x)
    torch.func.jvp(look, (x,), (x,))
    torch.func.vmap(look)(x)
    assert seen and set(seen) == {(False, False, False)}
    seen.clear()
    look(x)
    assert seen == [(True, True, True)]


def test_double_precision_under_autocast_keeps_the_modules(monkeypatch):
    # autocast leaves fp64 alone
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda: True)
    x = OnGpu()
    x.dtype = torch.float32
    mlp = _mlp().float()
    assert mlp.fused_dtype(x) is torch.get_autocast_dtype("cuda")
    assert mlp.double().fused_dtype(x) is None
    x.dtype = torch.float64
    assert mlp.fused_dtype(x) is None and mlp.float().fused_dtype(x) is None


class Wrapped(torch.Tensor):
    """A weight that holds its values in a way of its own, as sharded and quantised ones do."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        return super().__torch_function__(func, types, args, kwargs or {})


def test_parameters_of_other_classes_keep_the_modules():
    for part, want in (("mlp.fc1", (True, False, True)), ("mlp.fc2", (True, False, True)), ("norm1", (False, True, True)),
                       ("norm2", (True, True, False))):
        for name in ("weight", "bias"):
            blk = _fused_block()
            m = blk.get_submodule(part)
            wrapped = nn.Parameter(getattr(m, name).detach().as_subclass(Wrapped))
            del m._parameters[name]
            m._parameters[name] = wrapped
            assert type(getattr(m, name)) is Wrapped and _fits(blk) == want, (part, name)


# ---- held 8-bit weights ------------------------------------------------------------------------------------------------
@pytest.fixture
def holding(monkeypatch):
    """An Mlp whose 8-bit rows are made on the CPU, by copies that can be told from the weights they were made of."""
    monkeypatch.setattr(swin, "quantize_rows_func", lambda w: (w.detach().clone(), w.detach().abs().amax(-1)))
    mlp = swin.Mlp(16, 64)
    mlp.is_fused = mlp.fp8 = True
    mlp.hold_weights8()
    assert mlp.weights8() is mlp.weights8()
    return mlp


def _current(mlp):
    return all(torch.equal(q, m.weight) for (q, _), m in zip(mlp.weights8(), (mlp.fc1, mlp.fc2)))


def test_held_weights_belong_to_their_parameters(holding, monkeypatch):
    # another parameter of the same size may get the address, and the version counter, of the one that was freed
    monkeypatch.setattr(swin.Mlp, "_weights_key", lambda self: "the same for both", raising=False)
    holding.hold_weights8()
    held = holding.weights8()
    with torch.no_grad():
        holding.fc1.weight = nn.Parameter(torch.randn(64, 16))
    assert holding.weights8() is not held and _current(holding)


def test_held_weights_after_replacements(holding):
    for _ in range(3):
        holding.hold_weights8()
        holding.load_state_dict({k: torch.randn_like(v) for k, v in holding.state_dict().items()}, assign=True)
        assert _current(holding)
        with torch.no_grad():
            holding.fc2.weight = nn.Parameter(torch.randn(16, 64))
        assert _current(holding)


def test_the_storage_of_held_weights_is_not_given_away(holding):
    # .data of one parameter replaced twice: a storage that had been freed in between could come back under its address
    old = holding.fc1.weight.data_ptr()
    holding.fc1.weight.data = torch.zeros(64, 16)
    for _ in range(8):
        holding.fc1.weight.data = torch.randn(64, 16)
        assert holding.fc1.weight.data_ptr() != old and _current(holding)


def test_conversions_let_held_weights_go(holding):
    held = holding.weights8()
    holding.to("cpu")                       # nothing moves
    assert holding.weights8() is held
    holding.double()
    assert holding._weights8 is None and _current(holding)


def test_modules_with_held_weights_are_copied_and_saved(holding, tmp_path):
    twin = copy.deepcopy(holding)
    assert _current(twin)
    with torch.no_grad():
        twin.fc1.weight.mul_(3)
    assert _current(twin) and _current(holding)
    torch.save(holding, tmp_path / "mlp.pt")
    assert _current(torch.load(tmp_path / "mlp.pt", weights_only=False))


@pytest.mark.gpu
def test_held_weights_on_the_gpu_after_replacements():
    mlp = swin.Mlp(64, 256).cuda().to(torch.bfloat16)
    mlp.is_fused = mlp.fp8 = True
    x = torch.randn(5, 64, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        for _ in range(3):
            mlp.hold_weights8()
            held = mlp(x)
            mlp.hold_weights8(False)
            assert torch.equal(mlp(x), held)
            mlp.hold_weights8()
            state = {k: torch.randn_like(v) for k, v in mlp.state_dict().items()}
            mlp.load_state_dict(state, assign=True)
            got = mlp(x)
            mlp.hold_weights8(False)
            assert torch.equal(mlp(x), got) and not torch.equal(got, held)


@pytest.mark.gpu
@pytest.mark.parametrize("is_fused", [False, True])
def test_a_compiled_block_runs(is_fused):
    """A graph compiler breaks its graph at the library's calls and gives the same numbers."""
    blk = _block(is_fused=is_fused, fp8_mlp=is_fused).cuda().to(torch.bfloat16).eval()
    x = torch.randn(2, 64, 16, device="cuda", dtype=torch.bfloat16)
    compiled = torch.compile(blk, backend="eager")
    with torch.no_grad():
        assert torch.equal(compiled(x), blk(x))
    leaf, twin = x.clone().requires_grad_(), x.clone().requires_grad_()
    compiled(leaf).sum().backward()
    blk(twin).sum().backward()
    assert torch.equal(leaf.grad, twin.grad)
