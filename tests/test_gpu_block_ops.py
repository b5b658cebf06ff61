"""The operators around the attention call against their 64-bit definitions, on the GPU: sizes, types and strides at which a
kernel can go wrong, gradients, and what a caller may do with them (graphs, other streams, odd views)."""
import pytest
import torch

import flash_window_attention_v2_amd as fwa2
from block_ops_ref import check_e4m3, inside, linear8_ref, linear_ref, norm_ref, rounded

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
F8 = torch.float8_e4m3fn


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


# ---- normalisation -------------------------------------------------------------------------------------------------
NORM_TYPES = [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F16), (F16, F32, F16), (F32, F32, F32), (F16, F16, F32)]
# one lane group of every kind, its last size and the first of the next, odd widths among them
NORM_DIMS = [1, 7, 8, 64, 65, 96, 128, 200, 256, 385, 512, 768, 1024, 1100, 1536, 1538, 2048, 2056, 4096, 4099, 8192, 8200,
             16384]


def _norm_case(rows, dim, types, kind, placement, gates, seed, with_bias=True, with_shortcut=True):
    g = _gen(seed)
    xt, st, wt = types
    x = _rand(g, rows, dim, dtype=xt, shift=0.5)
    s = _rand(g, rows, dim, dtype=st) if with_shortcut else None
    w = _rand(g, dim, dtype=wt, scale=0.3, shift=1.0)
    b = _rand(g, dim, dtype=wt, scale=0.2) if with_bias else None
    gate = None
    if gates:
        gate = (torch.arange(gates, device="cuda") % 3 != 1).to(xt) * 1.25
    dy = _rand(g, rows, dim, dtype=xt if placement == "pre" else (st if with_shortcut else xt))
    dh = _rand(g, rows, dim, dtype=st) if placement == "pre" else None
    return x, s, w, b, gate, dy, dh


def _check_norm(rows, dim, types, kind, placement, gates, seed, with_bias=True, with_shortcut=True, eps=1e-5):
    x, s, w, b, gate, dy, dh = _norm_case(rows, dim, types, kind, placement, gates, seed, with_bias, with_shortcut)
    ref = norm_ref(x, s, w, b, eps, kind, placement, gate, dy, dh)
    leaves = {"dx": x, "ds": s, "dw": w, "db": b}
    leaves = {k: v.requires_grad_() for k, v in leaves.items() if v is not None}
    how = dict(eps=eps, kind=kind, placement=placement, gate=gate)
    got = fwa2.residual_norm_func(x, s, w, b, **how)
    if placement == "pre":
        grads = torch.autograd.grad(got, list(leaves.values()), (dh, dy))
        outs = {"h": got[0], "y": got[1]}
    else:
        grads = torch.autograd.grad(got, list(leaves.values()), dy)
        outs = {"y": got}
    outs.update(zip(leaves, grads))
    want_types = {"h": types[1], "y": types[0] if placement == "pre" else (types[1] if with_shortcut else types[0]),
                  "dx": types[0], "ds": types[1], "dw": types[2], "db": types[2]}
    for name, t in outs.items():
        assert t.dtype == want_types[name], name
        value, off = ref[name]
        inside(t.detach(), value, rounded(value, off, t.dtype), name)
    with torch.no_grad():       # without a gradient: the same numbers, and the 8-bit form of the same call
        plain = fwa2.residual_norm_func(x, s, w, b, **how)
        for a, c in zip(plain if placement == "pre" else (plain,), got if placement == "pre" else (got,)):
            assert torch.equal(a, c)
        stream, q, scale = fwa2.residual_norm_fp8_func(x, s, w, b, **how)
        assert torch.equal(stream, got[0] if placement == "pre" else got)
        assert q.dtype == F8 and q.shape == x.shape and scale.shape == x.shape[:-1]
        check_e4m3(q, scale, *ref["y"], "y8")


@pytest.mark.parametrize("dim", NORM_DIMS)
def test_norm_widths(dim):
    for i, (types, kind, placement, gates) in enumerate([
            (NORM_TYPES[0], "layer", "post", 3), (NORM_TYPES[1], "rms", "pre", 0), (NORM_TYPES[2], "layer", "pre", 3),
            (NORM_TYPES[3], "rms", "post", 0)]):
        _check_norm(51, dim, types, kind, placement, gates, 100 * dim + i)


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: "-".join(str(x).split(".")[1] for x in t))
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("placement", ["post", "pre"])
def test_norm_types(types, kind, placement):
    for rows, dim, gates in [(1, 96, 0), (1, 9, 1), (130, 96, 2), (77, 768, 7), (2100, 100, 0), (3, 5000, 3)]:
        _check_norm(rows, dim, types, kind, placement, gates, rows + dim)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_without_bias_or_shortcut(kind):
    _check_norm(65, 192, NORM_TYPES[0], kind, "post", 0, 1, with_bias=False)
    _check_norm(65, 192, NORM_TYPES[2], kind, "post", 5, 2, with_shortcut=False)
    _check_norm(65, 193, NORM_TYPES[1], kind, "pre", 0, 3, with_bias=False)


def test_norm_many_rows():
    # more rows than resident workgroups take in one round, so that every lane sums many of them
    _check_norm(40000, 96, NORM_TYPES[0], "layer", "post", 8, 7)
    _check_norm(20001, 520, NORM_TYPES[1], "layer", "pre", 0, 8)


def test_norm_large_mean():
    # rows far from zero: the squared deviations are summed around the mean
    g = _gen(3)
    x = _rand(g, 33, 768, dtype=F32, scale=0.5, shift=1000.0)
    w, b = torch.ones(768, device="cuda"), torch.zeros(768, device="cuda")
    ref = norm_ref(x, None, w, b, 1e-5, "layer", "post", None)
    value, off = ref["y"]
    inside(fwa2.residual_norm_func(x, None, w, b), value, rounded(value, off, F32), "y")


def test_norm_rows_of_zeros_nan_and_infinity():
    g = _gen(4)
    x = _rand(g, 6, 96, dtype=BF16)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 95] = float("inf")
    s = _rand(g, 6, 96, dtype=BF16)
    w, b = _rand(g, 96, dtype=BF16, shift=1.0), _rand(g, 96, dtype=BF16)
    for kind in ("layer", "rms"):
        y = fwa2.residual_norm_func(x, s, w, b, kind=kind)
        ok = torch.tensor([0, 1, 4, 5], device="cuda")
        value, off = norm_ref(x[ok], s[ok], w, b, 1e-5, kind, "post", None)["y"]
        inside(y[ok], value, rounded(value, off, BF16), "clean rows")
        assert y[2].isnan().all()
        assert y[3].isnan().any()
    # 8 bits: a row of zeros is zeros under a positive scale; a row that is not finite stays so
    q, scale = fwa2.quantize_rows_func(x)
    assert (q[1].float() == 0).all() and scale[1] > 0
    back = q.float() * scale[:, None]
    assert back[2].isnan().any() and back[3].isnan().any()
    check_e4m3(q[[0, 1, 4, 5]], scale[[0, 1, 4, 5]], x[[0, 1, 4, 5]].double(), torch.zeros_like(x[[0, 1, 4, 5]]).double(), "x8")


def test_norm_views_and_leading_dimensions():
    g = _gen(5)
    wide = _rand(g, 4, 9, 300, dtype=F16)
    w, b = _rand(g, 96, dtype=F16, shift=1.0), _rand(g, 192, dtype=F16)[::2]
    base = _rand(g, 4, 1, 96, dtype=F16)
    for x in (wide[..., 3:99], wide[..., 8:104], wide[:, ::2][..., 96:192].expand(4, 5, 96)):
        s = base.expand(x.shape)                                # a broadcast shortcut: its gradient is summed by autograd
        leaf_x, leaf_s = x.detach().clone().requires_grad_(), base.clone().requires_grad_()
        y = fwa2.residual_norm_func(x, s, w, b)
        again = fwa2.residual_norm_func(leaf_x, leaf_s.expand(x.shape), w, b)
        assert torch.equal(y, again)
        value, off = norm_ref(x.reshape(-1, 96), s.reshape(-1, 96), w, b, 1e-5, "layer", "post", None)["y"]
        inside(y.reshape(-1, 96), value, rounded(value, off, F16), "y")
        again.sum().backward()                                   # an expanded gradient
        assert torch.equal(leaf_s.grad, torch.full_like(base, x.shape[1]))
    t = _rand(g, 96, 40, dtype=F16).t()                          # inner stride 40
    assert torch.equal(fwa2.residual_norm_func(t, None, w, b), fwa2.residual_norm_func(t.contiguous(), None, w, b))
    one = _rand(g, 96, dtype=F16)                                # a single row without leading dimensions
    assert fwa2.residual_norm_func(one, one, w, b).shape == (96,)
    assert fwa2.quantize_rows_func(one)[1].shape == ()


def test_norm_only_some_gradients():
    x, s, w, b, gate, dy, dh = _norm_case(37, 192, NORM_TYPES[0], "layer", "pre", 0, 11)
    full = [t.clone().requires_grad_() for t in (x, s, w, b)]
    want = torch.autograd.grad(fwa2.residual_norm_func(*full, placement="pre"), full, (dh, dy))
    for keep in range(4):
        part = [t.clone().requires_grad_(i == keep) for i, t in enumerate((x, s, w, b))]
        got, = torch.autograd.grad(fwa2.residual_norm_func(*part, placement="pre"), [part[keep]], (dh, dy))
        assert torch.equal(got, want[keep]), keep
    # only one of the two outputs is used
    h, y = fwa2.residual_norm_func(*full, placement="pre")
    got = torch.autograd.grad(h, full, dh, retain_graph=True, allow_unused=True)
    assert torch.equal(got[0], dh) and torch.equal(got[1], dh) and got[2] is None and got[3] is None
    got = torch.autograd.grad(y, full, dy)
    ref = norm_ref(x, s, w, b, 1e-5, "layer", "pre", None, dy, None)
    for name, t in zip(("dx", "ds", "dw", "db"), got):
        value, off = ref[name]
        inside(t, value, rounded(value, off, BF16), name)


def test_norm_empty_and_far_rows():
    w = torch.ones(96, device="cuda", dtype=BF16).requires_grad_()
    x = torch.empty(0, 96, device="cuda", dtype=BF16, requires_grad=True)
    y = fwa2.residual_norm_func(x, None, w)
    y.sum().backward()
    assert y.shape == (0, 96) and (w.grad == 0).all() and x.grad.shape == (0, 96)
    assert fwa2.quantize_rows_func(x.detach())[0].shape == (0, 96)
    # rows more than 2^32 bytes and 2^31 elements from the first
    big = torch.zeros(40000, 65536, device="cuda", dtype=BF16)
    g = _gen(12)
    view = big[:, 1000:1096]
    view[::39] = _rand(g, view[::39].shape[0], 96, dtype=BF16)
    value, off = norm_ref(view, None, w.detach(), None, 1e-5, "rms", "post", None)["y"]
    inside(fwa2.residual_norm_func(view, None, w.detach(), kind="rms"), value, rounded(value, off, BF16), "far rows")


# ---- 8-bit rows ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,dim", [(1, 1), (5, 7), (33, 96), (64, 1536), (3, 4100), (2, 16384), (1000, 100)])
def test_quantize_rows(dtype, rows, dim):
    g = _gen(rows * dim)
    x = (_rand(g, rows, dim) * torch.exp(2 * _rand(g, rows, 1))).to(dtype)
    q, scale = fwa2.quantize_rows_func(x)
    check_e4m3(q, scale, x.double(), torch.zeros(rows, dim, dtype=torch.float64, device="cuda"), "x8")
    assert torch.equal(scale, x.float().abs().amax(-1) * torch.tensor(1 / 448, dtype=F32, device="cuda"))
    # quotients are rounded as a division's: exact ties go to even, as the conversion of a quotient does
    assert torch.equal(q.view(torch.uint8), (x.float() / scale[:, None]).to(F8).view(torch.uint8))
    # every representable value of one scale comes back as itself
    table = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).view(F8).float()
    table = table[table.isfinite()][None]
    q, scale = fwa2.quantize_rows_func(table)
    assert float(scale[0]) == 1.0 and torch.equal(q.float(), table)


def test_quantize_more_rows_than_workgroups():
    g = _gen(77)
    x = _rand(g, 70001, 2056, dtype=BF16)       # one workgroup a row, 65536 at most
    q, scale = fwa2.quantize_rows_func(x)
    for rows in (slice(0, 50), slice(65500, 65600), slice(69950, 70001)):
        check_e4m3(q[rows], scale[rows], x[rows].double(), torch.zeros_like(x[rows]).double(), "x8")


# ---- matrix product with an epilogue ---------------------------------------------------------------------------------
LINEAR_SIZES = [(1, 1, 1), (1, 768, 1000), (3, 17, 5), (2, 8, 8), (64, 64, 64), (65, 72, 136), (130, 96, 384), (127, 588, 333),
                (300, 8, 520), (1000, 100, 64), (33, 1030, 40), (257, 136, 1000), (16, 4096, 24), (5000, 96, 96)]


def _linear_case(m, k, n, dtype, with_bias, with_residual, seed):
    g = _gen(seed)
    x = _rand(g, m, k, dtype=dtype)
    w = _rand(g, n, k, dtype=dtype, scale=k ** -0.5)
    b = _rand(g, n, dtype=dtype, scale=0.3) if with_bias else None
    r = _rand(g, m, n, dtype=dtype) if with_residual else None
    return x, w, b, r, _rand(g, m, n, dtype=dtype)


def _check_linear(x, w, b, act, r, dy, what=""):
    ref = linear_ref(x, w, b, act, r, dy)
    leaves = {"dx": x, "dw": w, "db": b, "dr": r}
    leaves = {name: t.detach().requires_grad_() for name, t in leaves.items() if t is not None}
    y = fwa2.fused_linear_func(leaves["dx"], leaves["dw"], leaves.get("db"), act, leaves.get("dr"))
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        assert torch.equal(y, fwa2.fused_linear_func(x, w, b, act, r))
    for name, t in {"y": y.detach(), **grads}.items():
        assert t.dtype == x.dtype
        if name == "dr":
            assert torch.equal(t, dy)
            continue
        value, off = ref[name]
        inside(t, value, rounded(value, off, t.dtype), what + name)


@pytest.mark.parametrize("m,k,n", LINEAR_SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_sizes(m, k, n, dtype):
    for i, (act, bias, res) in enumerate([(None, False, False), ("gelu", True, False), (None, True, True)]):
        _check_linear(*_linear_case(m, k, n, dtype, bias, res, m + k + n + i)[:3], act,
                      *_linear_case(m, k, n, dtype, bias, res, m + k + n + i)[3:], f"{act} ")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "relu", None])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_activations(act, dtype):
    x, w, b, r, dy = _linear_case(200, 64, 136, dtype, True, True, 5)
    _check_linear(x * 3, w, b, act, r, dy)
    # z over the whole range of the activation, large ones included: a row of W picks the value out of x
    x = torch.zeros(64, 8, device="cuda", dtype=dtype)
    x[:, 0] = torch.linspace(-40, 40, 64, device="cuda").to(dtype)
    w = torch.zeros(16, 8, device="cuda", dtype=dtype)
    w[:, 0] = torch.linspace(0.05, 2.0, 16, device="cuda").to(dtype)
    _check_linear(x, w, None, act, None, torch.ones(64, 16, device="cuda", dtype=dtype))


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "relu"])
def test_linear_overflowing_sums(act):
    # sums beyond the range of fp16: finite slopes (0 or 1) all the same
    x = torch.tensor([[300.0] * 8, [-300.0] * 8], device="cuda", dtype=F16)
    w = torch.full((8, 8), 40.0, device="cuda", dtype=F16).requires_grad_()
    leaf = x.clone().requires_grad_()
    y = fwa2.fused_linear_func(leaf, w, None, act)
    y.backward(torch.full_like(y, 0.5))
    assert (y[0] == float("inf")).all() and (y[1] == 0).all()
    assert torch.equal(leaf.grad[0], torch.full_like(leaf.grad[0], 160.0)) and (leaf.grad[1] == 0).all()
    assert w.grad.isfinite().all()


def test_linear_nan_stays_in_its_row():
    x, w, b, r, _ = _linear_case(70, 100, 72, BF16, True, True, 8)
    clean = fwa2.fused_linear_func(x, w, b, "gelu", r)
    x = x.clone()
    x[69, 99] = float("nan")
    x[3, 0] = float("inf")
    y = fwa2.fused_linear_func(x, w, b, "gelu", r)
    assert y[69].isnan().all()
    assert not y[3].isfinite().all()
    rest = [i for i in range(70) if i not in (3, 69)]
    assert torch.equal(y[rest], clean[rest])


def test_linear_views():
    g = _gen(6)
    big = _rand(g, 3, 50, 400, dtype=BF16)
    weights = _rand(g, 400, 400, dtype=BF16, scale=0.1)
    bias = _rand(g, 400, dtype=BF16)
    for lo, k, n in [(0, 96, 64), (8, 96, 72), (3, 96, 64), (0, 100, 33), (1, 17, 9)]:
        x, w, b = big[:, ::2, lo:lo + k], weights[5:5 + n, lo:lo + k], bias[1:2 * n + 1:2]
        r = big[:, :25, 7:7 + n]
        y = fwa2.fused_linear_func(x, w, b, "silu", r)
        assert y.shape == (3, 25, n)
        value, off = linear_ref(x.reshape(-1, k), w, b, "silu", r.reshape(-1, n))["y"]
        inside(y.reshape(-1, n), value, rounded(value, off, BF16), f"{lo} {k} {n}")
    x, wt = big[0, :, :64], weights[:64, :96]
    dy = _rand(g, 50, 96, dtype=BF16)
    _check_linear(x, wt.t(), None, None, None, dy, "transposed weight ")
    _check_linear(x, wt.t(), bias[:96], "gelu", None, dy[:, :1].expand(50, 96), "expanded gradient ")
    _check_linear(big[0, :, 1:65], weights[:97, 1:65], bias[:97], "gelu", None, _rand(g, 50, 200, dtype=BF16)[:, 3:100], "odd ")
    res = _rand(g, 1, 96, dtype=BF16).requires_grad_()           # a broadcast residual
    fwa2.fused_linear_func(x, wt.t().contiguous(), None, None, res.expand(50, 96)).sum().backward()
    assert torch.equal(res.grad, torch.full_like(res, 50.0))
    sq = _rand(g, 64, 64, dtype=BF16)                            # one tensor in several places
    leaf = sq.clone().requires_grad_()
    fwa2.fused_linear_func(leaf, leaf, None, None, leaf).backward(sq)
    parts = [sq.clone().requires_grad_() for _ in range(3)]
    fwa2.fused_linear_func(parts[0], parts[1], None, None, parts[2]).backward(sq)
    want = sum(p.grad.double() for p in parts)
    inside(leaf.grad, want, 3 * sum(p.grad.double().abs() for p in parts) * 2.0 ** -8, "shared")


def test_linear_single_row_without_leading_dimensions():
    x, w, b, r, dy = _linear_case(1, 72, 40, BF16, True, True, 19)
    y = fwa2.fused_linear_func(x[0], w, b, "gelu", r[0])
    assert y.shape == (40,) and torch.equal(y, fwa2.fused_linear_func(x, w, b, "gelu", r)[0])
    leaf = x[0].clone().requires_grad_()
    fwa2.fused_linear_func(leaf, w, b, "gelu").backward(dy[0])
    value, off = linear_ref(x, w, b, "gelu", None, dy)["dx"]
    inside(leaf.grad[None], value, rounded(value, off, BF16), "dx")
    x8, sx = fwa2.quantize_rows_func(x[0])
    w8, sw = fwa2.quantize_rows_func(w)
    assert fwa2.fused_linear_fp8_func(x8, sx, w8, sw).shape == (40,)


@pytest.mark.parametrize("m", [1, 15, 16, 17, 33, 48, 49, 64, 65])
def test_linear_few_rows_agree_with_their_definition(m):
    # the kernel for few rows and its border to the tiles, with contractions that end inside a product
    for k, n in [(8, 24), (40, 16), (520, 200), (4104, 72)]:
        x, w, b, r, dy = _linear_case(m, k, n, F16, True, True, m + k)
        for act, res in ((None, r), ("gelu", None), ("gelu_tanh", r)):
            value, off = linear_ref(x, w, b, act, res)["y"]
            inside(fwa2.fused_linear_func(x, w, b, act, res), value, rounded(value, off, F16), f"{k} {n} {act}")


def test_linear_only_some_gradients():
    x, w, b, r, dy = _linear_case(100, 72, 40, BF16, True, True, 9)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(fwa2.fused_linear_func(*full[:3], "gelu", full[3]), full, dy)
    for keep in range(4):
        part = [t.clone().requires_grad_(i == keep) for i, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(fwa2.fused_linear_func(*part[:3], "gelu", part[3]), [part[keep]], dy)
        assert torch.equal(got, want[keep]), keep


def test_linear_long_contraction_and_many_rows():
    # the weight gradient's contraction over the rows is split and added up afterwards: whole and ragged splits
    for m, k, n in [(20000, 96, 40), (9999, 136, 200), (4097, 33, 17), (70000, 8, 8)]:
        x, w, b, r, dy = _linear_case(m, k, n, BF16, True, False, m)
        _check_linear(x, w, b, None, r, dy, f"{m} ")


@pytest.mark.parametrize("m,k,n", [(22000, 128, 1000), (66000, 192, 248), (65541, 104, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_wide_tiles_of_short_contractions(m, k, n, dtype):
    """256 columns to a tile, tiles that end inside, forward and (contraction n) backward; sampled rows."""
    x, w, b, r, dy = _linear_case(m, k, n, dtype, True, True, m)
    y = fwa2.fused_linear_func(x, w, b, "gelu", r)
    rows = torch.cat([torch.arange(0, m, 997), torch.arange(m - 140, m)]).to(x.device)
    value, off = linear_ref(x[rows], w, b, "gelu", r[rows])["y"]
    inside(y[rows], value, rounded(value, off, dtype), "y")
    leaf = dy.clone().requires_grad_()          # dy W, whose contraction is n: through the product of W transposed
    wt = w.t().contiguous()
    out = fwa2.fused_linear_func(leaf, wt)
    back, = torch.autograd.grad(out, [leaf], x)
    value, off = linear_ref(dy[rows], wt, None, None, None, x[rows])["dx"]
    inside(back[rows], value, rounded(value, off, dtype), "dx")


@pytest.mark.parametrize("m,k,n", [(31, 4096, 1000), (97, 520, 96), (255, 1536, 384), (300, 264, 40), (1, 1024, 16384), (16, 72, 8200)])
def test_linear_few_workgroups_agree_with_their_definition(m, k, n):
    """Groups of 16 and of 32 rows and 4 wavefronts to a workgroup, with products that end inside each."""
    x, w, b, r, dy = _linear_case(m, k, n, BF16, True, True, m + k)
    value, off = linear_ref(x, w, b, "gelu", r)["y"]
    inside(fwa2.fused_linear_func(x, w, b, "gelu", r), value, rounded(value, off, BF16), "y")


@pytest.mark.parametrize("m,k,n", [(16500, 64, 136), (16384, 192, 384), (5000, 512, 192), (8200, 520, 392), (4099, 768, 264),
                                   (8192, 512, 2048), (4100, 1032, 4104), (100, 2048, 2000), (3000, 384, 1160)])
def test_linear_tiles_of_every_size(m, k, n):
    # sizes that the host sends to the 128-, 192- and 256-wide tiles forward and backward, whole and with ragged edges
    x, w, b, r, dy = _linear_case(m, k, n, BF16, True, True, m + k + n)
    _check_linear(x, w, b, "gelu", None, dy)
    _check_linear(x, w, b, None, r, dy)
    x8, sx = fwa2.quantize_rows_func(x)
    w8, sw = fwa2.quantize_rows_func(w)
    rows = torch.arange(0, m, max(1, m // 60), device="cuda")
    y = fwa2.fused_linear_fp8_func(x8, sx, w8, sw, b, "gelu", r)
    value, off = linear8_ref(x8[rows], sx[rows], w8, sw, b, "gelu", r[rows])
    inside(y[rows], value, rounded(value, off, BF16), "8 bits")


def test_linear_empty_and_far_rows():
    w = torch.ones(16, 8, device="cuda", dtype=BF16).requires_grad_()
    x = torch.empty(0, 3, 8, device="cuda", dtype=BF16, requires_grad=True)
    y = fwa2.fused_linear_func(x, w, None, "gelu")
    y.sum().backward()
    assert y.shape == (0, 3, 16) and (w.grad == 0).all() and x.grad.shape == x.shape
    big = torch.zeros(40000, 65536, device="cuda", dtype=BF16)      # 2^31 elements and more apart
    g = _gen(13)
    view = big[:, 30000:30064]
    view[:] = _rand(g, 40000, 64, dtype=BF16)
    w, dy = _rand(g, 72, 64, dtype=BF16, scale=0.1), _rand(g, 40000, 72, dtype=BF16)
    _check_linear(view, w, None, None, None, dy, "far rows ")


def test_linear_gradients_against_differences():
    x, w, b, r, dy = (t.double() for t in _linear_case(6, 5, 4, F16, True, True, 21))
    leaves = [t.to(F16).requires_grad_() for t in (x, w, b)]
    y = fwa2.fused_linear_func(*leaves, "gelu")
    got = torch.autograd.grad(y, leaves, dy.to(F16))

    def loss(x, w, b):
        return (torch.nn.functional.gelu(x @ w.t() + b) * dy.to(F16).double()).sum()

    at = [t.detach().double() for t in leaves]
    for which, grad in enumerate(got):
        flat = at[which].flatten()
        for i in range(0, flat.numel(), 3):
            h = 1e-5
            up, down = [t.clone() for t in at], [t.clone() for t in at]
            up[which].view(-1)[i] += h
            down[which].view(-1)[i] -= h
            diff = float((loss(*up) - loss(*down)) / (2 * h))
            # z and dz are kept in fp16 (2^-11 each) and the gradient is rounded once more
            assert abs(float(grad.flatten()[i]) - diff) <= 2.0 ** -8 * (1 + abs(diff)), (which, i)


# ---- 8-bit product ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,k,n", [(1, 16, 8), (4, 1536, 768), (65, 128, 136), (130, 400, 96), (64, 100, 33), (3, 1, 5),
                                   (200, 1040, 264), (1000, 144, 64), (129, 4096, 24)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear8(m, k, n, dtype):
    g = _gen(m + k + n)
    x, w = _rand(g, m, k, dtype=dtype), _rand(g, n, k, dtype=dtype, scale=k ** -0.5)
    b, r = _rand(g, n, dtype=dtype), _rand(g, m, n, dtype=dtype)
    x8, sx = fwa2.quantize_rows_func(x)
    w8, sw = fwa2.quantize_rows_func(w)
    for act, bias, res in [(None, None, None), ("gelu", b, None), ("silu", b, r)]:
        y = fwa2.fused_linear_fp8_func(x8, sx, w8, sw, bias, act, res, out_dtype=dtype)
        assert y.dtype == dtype
        value, off = linear8_ref(x8, sx, w8, sw, bias, act, res)
        inside(y, value, rounded(value, off, dtype), f"{act}")


def test_linear8_views_and_empty():
    g = _gen(2)
    x8, sx = fwa2.quantize_rows_func(_rand(g, 2, 30, 256))
    w8, sw = fwa2.quantize_rows_func(_rand(g, 80, 256))
    for lo, k in [(0, 64), (16, 96), (5, 40)]:
        xs, ws = x8[:, ::3, lo:lo + k], w8[::2, lo:lo + k]
        y = fwa2.fused_linear_fp8_func(xs, sx[:, ::3], ws, sw[::2])
        value, off = linear8_ref(xs.reshape(-1, k), sx[:, ::3].reshape(-1), ws, sw[::2], None, None, None)
        inside(y.reshape(-1, 40), value, rounded(value, off, BF16), f"{lo} {k}")
    assert fwa2.fused_linear_fp8_func(x8[:0], sx[:0], w8, sw).shape == (0, 30, 80)


# ---- together, and under what a program does with them -----------------------------------------------------------------
def _mlp_block(x, p):
    """x + norm(W2 gelu(W1 x + b1) + b2): the second half of a residual-post-norm block."""
    h = fwa2.fused_linear_func(x, p["w1"], p["b1"], "gelu")
    o = fwa2.fused_linear_func(h, p["w2"], p["b2"])
    return fwa2.residual_norm_func(o, x, p["w"], p["b"], gate=p["gate"])


def _mlp_params(g, dim, dtype):
    return {"w1": _rand(g, 4 * dim, dim, dtype=dtype, scale=dim ** -0.5), "b1": _rand(g, 4 * dim, dtype=dtype, scale=0.1),
            "w2": _rand(g, dim, 4 * dim, dtype=dtype, scale=(4 * dim) ** -0.5), "b2": _rand(g, dim, dtype=dtype, scale=0.1),
            "w": _rand(g, dim, dtype=dtype, shift=1.0, scale=0.1), "b": _rand(g, dim, dtype=dtype, scale=0.1),
            "gate": torch.tensor([1.25, 0.0], device="cuda", dtype=dtype)}


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_block_together(dtype):
    g = _gen(31)
    x, p = _rand(g, 2, 150, 96, dtype=dtype), _mlp_params(g, 96, dtype)
    dy = _rand(g, 2, 150, 96, dtype=dtype)
    names = ["w1", "b1", "w2", "b2", "w", "b"]
    leaves = [x.clone().requires_grad_()] + [p[k].clone().requires_grad_() for k in names]
    y = _mlp_block(leaves[0], {**dict(zip(names, leaves[1:])), "gate": p["gate"]})
    got = torch.autograd.grad(y, leaves, dy)
    F = torch.nn.functional
    d = [t.detach().double().requires_grad_() for t in leaves]
    q = dict(zip(names, d[1:]))
    o = F.linear(F.gelu(F.linear(d[0], q["w1"], q["b1"])), q["w2"], q["b2"])
    z = d[0] + p["gate"].double().view(2, 1, 1) * F.layer_norm(o, (96,), q["w"], q["b"], 1e-5)
    want = torch.autograd.grad(z, d, dy.double())
    # a chain of about ten roundings, each half a step of independent sign: held as a whole (2-norm), 6 half steps
    half = torch.finfo(dtype).eps / 2
    for name, a, b in zip(["y", "dx"] + names, (y.detach(), *got), (z.detach(), *want)):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 6 * half, (name, rel)
    with torch.no_grad():
        # the 8-bit chain: rows leave the norm in 8 bits and go through two 8-bit products
        s, x8, sx = fwa2.residual_norm_fp8_func(o.to(dtype), x, p["w"], p["b"])
        w18, s1 = fwa2.quantize_rows_func(p["w1"])
        w28, s2 = fwa2.quantize_rows_func(p["w2"])
        h = fwa2.fused_linear_fp8_func(x8, sx, w18, s1, p["b1"], "gelu", out_dtype=dtype)
        h8, sh = fwa2.quantize_rows_func(h)
        y8 = fwa2.fused_linear_fp8_func(h8, sh, w28, s2, p["b2"], None, s, out_dtype=dtype)
        ref = s.double() + F.linear(F.gelu(F.linear(s.double(), q["w1"], q["b1"])), q["w2"], q["b2"])
        # four sets of operands with 2^-4 half steps at most, about 2^-5.4 rms over a binade each
        assert float((y8.double() - ref).norm() / ref.norm()) <= 2.0 ** -4


@pytest.mark.parametrize("dtype", [BF16])
def test_block_capture_and_replay(dtype):
    g = _gen(41)
    names = ["w1", "b1", "w2", "b2", "w", "b"]
    p = _mlp_params(g, 96, dtype)
    x, dy = _rand(g, 2, 1030, 96, dtype=dtype), _rand(g, 2, 1030, 96, dtype=dtype)
    leaves = [x.requires_grad_()] + [p[k].requires_grad_() for k in names]

    def step():
        y = _mlp_block(x, p)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2, 3):
        h = _gen(seed)
        with torch.no_grad():
            x.copy_(_rand(h, *x.shape, dtype=dtype))
            dy.copy_(_rand(h, *dy.shape, dtype=dtype))
            p["w1"].copy_(_rand(h, *p["w1"].shape, dtype=dtype, scale=0.1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_two_streams_and_repeated_calls_agree():
    g = _gen(51)
    p = _mlp_params(g, 192, BF16)
    xs = [_rand(g, 2, 700, 192, dtype=BF16) for _ in range(2)]
    names = ["w1", "b1", "w2", "b2", "w", "b"]
    for k in names:
        p[k].requires_grad_()

    def step(x):
        leaf = x.detach().requires_grad_()
        y = _mlp_block(leaf, p)
        return [y.detach(), *torch.autograd.grad(y, [leaf] + [p[k] for k in names], torch.ones_like(y))]

    want = [step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i] = step(x)
        torch.cuda.synchronize()
        for a, b in zip(got[0] + got[1], want[0] + want[1]):
            assert torch.equal(a, b)


def test_second_derivative_raises():
    x, w, b, r, dy = _linear_case(8, 8, 8, BF16, True, False, 1)
    x.requires_grad_()
    gx, = torch.autograd.grad(fused := fwa2.fused_linear_func(x, w, b, "gelu"), x, dy.requires_grad_(), create_graph=True)
    assert fused.requires_grad
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)
