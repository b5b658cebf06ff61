"""Inputs whose sums over many rows come out exactly, so that a partial sum that is lost, doubled or put in the wrong place shows
whatever the tolerance of rounded sums would be: small whole numbers, whose products and sums stay far below 2^24.  The sums
are centred on zero, so that the last rounding (8 or 11 significant bits) hides little of them."""
import torch


def whole(g, *shape, dtype, device, most=2):
    """Whole numbers from -most to most."""
    return torch.randint(-most, most + 1, shape, generator=g, device=device).to(dtype)


def layer(m, k, n, dtype, device, seed):
    """x, weight, bias, dy of a product whose z is never 0 (the bias is one half off the whole numbers), so that relu's slope
    is 0 or 1 beyond doubt and z, dz and every sum are exact."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    x, w = whole(g, m, k, dtype=dtype, device=device), whole(g, n, k, dtype=dtype, device=device, most=1)
    b = whole(g, n, dtype=dtype, device=device) + 0.5
    return x, w, b, whole(g, m, n, dtype=dtype, device=device)


def layer_sums(x, w, b, dy, act):
    """{dx, dw, db} in 64 bits, each exact."""
    X, W, DY = x.double(), w.double(), dy.double()
    if act == "relu":
        DY = DY * (X @ W.t() + b.double() > 0)
    assert float(X.abs().max() * DY.abs().max()) * x.shape[0] < 2 ** 24 and float(DY.abs().max()) * w.shape[0] < 2 ** 24
    return {"dx": DY @ W, "dw": DY.t() @ X, "db": DY.sum(0)}


def constant_rows(act, n, dtype, device, seed):
    """bias and one row of dy for rows of x that are all zero: z is the bias in every row, dz = dy act'(z) too, and what separates
    the sum of m unrounded dz from the sum of m rounded ones is their rounding, the same m times over."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    z = (torch.rand(n, generator=g, device=device) * 2.5 + 0.25).to(dtype)
    return z, (1 + torch.rand(n, generator=g, device=device)).to(dtype)


def half_ulp(value, dtype):
    """Half the distance between the neighbours of `value` in dtype."""
    return torch.exp2(torch.floor(torch.log2(value.abs()))) * torch.finfo(dtype).eps / 2


def constant_rows_bound(db, m, dtype):
    """How far a sum of m unrounded dz may be from m dz: its own rounding; m fp32 additions; the slope's 32 x 2^-24 relative to
    1 + |z| <= 4 against a slope of at least one half, so 256 x 2^-24."""
    slack = db.abs() * (m + 256) * 2.0 ** -24
    return (half_ulp(db.abs() + slack, dtype) + slack)
