"""Cases, 64-bit references and elementwise error bounds for ops.group_norm_act and ops.embedding (shared by the CPU and GPU tests).

w: half a step of fp32 (2^-24), u: of the element type.  With N values in a group:
  mean       off by at most em = w (N + 4) mean|x|       (a sum of N values in any order; in the kernels it is much less)
  variance   from deviations: off by ev = w (N + 8) var + 2 em mean|x - m| + em^2, so 1 / deviation is off by er = ev / (2 (var + eps)) + 3 w, relative
  xh         off by |xh| (er + 2 w) + (em + w |x| ) rstd
  z          off by (bound of xh) |g| + 2 w (|xh g| + |bias|), y by that times max|act'| <= 1.1, and 8 w |z| for the activation, rounded once
The gradient is sums of such values: a sum of n products adds w (n + 4) of the sum of magnitudes."""
import math

import torch

# name, B, C, H, W, groups, act, affine (None, "channel", "sample"), mean, gain_offset
NORM_CASES = [
    ("one_group_small", 2, 16, 4, 4, 1, "none", None, 0.0, 0.0),
    ("first_block", 3, 1536, 4, 4, 16, "silu", "sample", 0.2, 1.0),
    ("odd_size", 2, 48, 7, 5, 16, "relu", "channel", 0.5, 0.0),
    ("scalar_columns", 2, 15, 9, 11, 3, "silu", "channel", -0.3, 0.0),
    ("one_channel_a_group", 2, 12, 13, 6, 12, "silu", "sample", 1.0, 1.0),
    ("groups_inside_a_vector", 2, 40, 6, 6, 20, "none", "channel", 0.0, 0.0),
    ("three_channels_a_group", 1, 96, 33, 31, 32, "silu", "sample", 0.0, 1.0),
    ("large_slab", 2, 64, 40, 48, 4, "relu", "sample", 0.3, 1.0),
    ("three_passes", 2, 96, 96, 80, 16, "silu", "channel", 0.3, 0.0),
    ("three_passes_scalar", 1, 33, 101, 97, 3, "relu", "sample", 0.3, 1.0),
    ("three_passes_wide", 1, 1280, 32, 33, 32, "silu", "channel", 0.0, 0.0),
    ("far_mean", 2, 32, 64, 64, 4, "none", "channel", 300.0, 0.0),
    ("one_pixel", 4, 64, 1, 1, 4, "silu", "channel", 0.0, 0.0),
    ("one_row_of_pixels", 2, 24, 1, 500, 3, "none", "sample", 0.0, 1.0),
]
NORM_IDS = [c[0] for c in NORM_CASES]


def make_norm(case, dtype, device, seed=0):
    _, B, C, H, W, G, act, affine, mean, g0 = case
    g = torch.Generator().manual_seed(seed + 7)
    last = dict(memory_format=torch.channels_last)
    x = (torch.randn(B, C, H, W, generator=g) + mean).to(dtype).to(device).contiguous(**last)
    dy = torch.randn(B, C, H, W, generator=g).to(dtype).to(device).contiguous(**last)
    gain = bias = None
    if affine:
        shape = (B, C) if affine == "sample" else (C,)
        gain = (torch.randn(shape, generator=g) * 0.3 + (1.0 - g0)).to(device).requires_grad_()
        bias = (torch.randn(shape, generator=g) * 0.3).to(device).requires_grad_()
    return x.requires_grad_(), dy, gain, bias


def norm_reference(case, dtype, x, dy, gain, bias, eps=1e-5):
    """-> {name: (value, bound)} in float64, and where z is within its own error of a ReLU's border"""
    _, B, C, H, W, G, act, affine, _, g0 = case
    w, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    X, dY = (t.detach().double().cpu().reshape(B, G, C // G, H * W) for t in (x, dy))
    each = lambda t, one: torch.full((1, G, C // G, 1), one, dtype=torch.float64) if t is None else t.detach().double().cpu().reshape(-1, G, C // G, 1)
    g, b = each(gain, 1.0) + (g0 if gain is not None else 0.0), each(bias, 0.0)
    N = C // G * H * W
    m = X.mean((2, 3), keepdim=True)
    var = (X - m).square().mean((2, 3), keepdim=True)
    r = (var + eps).rsqrt()
    xh = (X - m) * r
    z = xh * g + b
    em = w * (N + 4) * X.abs().mean((2, 3), keepdim=True)
    ev = w * (N + 8) * var + 2 * em * (X - m).abs().mean((2, 3), keepdim=True) + em.square()
    er = ev / (2 * (var + eps)) + 3 * w
    exh = xh.abs() * (er + 2 * w) + (em + w * X.abs()) * r
    ez = exh * g.abs() + 2 * w * ((xh * g).abs() + b.abs())
    s = torch.sigmoid(z)
    y = z * s if act == "silu" else z.clamp_min(0) if act == "relu" else z
    da = s * (1 + z * (1 - s)) if act == "silu" else (z > 0).double() if act == "relu" else torch.ones_like(z)
    eda = ez * 0.5 + 8 * w if act == "silu" else ((z.abs() <= ez).double() if act == "relu" else torch.zeros_like(z))     # |silu''| <= 0.5
    dz, edz = dY * da, dY.abs() * eda + w * (dY * da).abs()
    over = (2, 3)
    dn, edn = dz * g, edz * g.abs() + w * (dz * g).abs()
    mean = lambda t: t.mean(over, keepdim=True)
    c1, c2 = mean(dn), mean(dn * xh)
    e1 = mean(edn) + w * (N + 4) * mean(dn.abs())
    e2 = mean(edn * xh.abs() + dn.abs() * exh) + w * (N + 4) * mean((dn * xh).abs())
    inner = dn - c1 - xh * c2
    dx = inner * r
    edx = (edn + e1 + exh * c2.abs() + xh.abs() * e2 + 3 * w * (dn.abs() + c1.abs() + (xh * c2).abs())) * r + dx.abs() * (er + 2 * w)
    back = lambda t: t.reshape(B, C, H, W)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    out = {"y": (back(y), back(ez * 1.1 + 8 * w * z.abs() + u * y.abs()) + tiny), "dx": (back(dx), back(edx + u * dx.abs()) + tiny)}
    if affine:
        P = H * W
        per = {"dgain": ((dz * xh).sum(3), (edz * xh.abs() + dz.abs() * exh).sum(3) + w * (P + 4) * (dz * xh).abs().sum(3)),
               "dbias": (dz.sum(3), edz.sum(3) + w * (P + 4) * dz.abs().sum(3))}
        for name, (v, e) in per.items():
            v, e = v.reshape(B, C), e.reshape(B, C)
            if affine == "channel":
                e, v = e.sum(0) + w * (B + 1) * v.abs().sum(0), v.sum(0)
            out[name] = (v, e)
    return out


# name, V, D, idx shape, kind of tokens, scale, padding_idx
EMBEDDING_CASES = [
    ("one_token", 1, 1, (1,), "uniform", 1.0, None),
    ("classes", 1000, 128, (64,), "uniform", 1.0, None),
    ("same_token", 10, 24, (100,), "same", 0.5, None),
    ("odd_columns", 37, 33, (5, 7), "uniform", 3.0, 5),
    ("few_limit", 300, 40, (1024,), "skewed", 1.0, None),
    ("sorted", 301, 40, (1025,), "skewed", 1.0, None),
    ("sorted_same", 50, 17, (3000,), "same", 2.0, None),
    ("sorted_padded", 700, 264, (40, 60), "skewed", 11.25, 3),
    ("sorted_one_row", 1, 8, (2000,), "same", 1.0, None),
    ("many_tokens", 5000, 72, (16384,), "skewed", 1.0, None),
    ("many_rows", 600000, 8, (1500,), "uniform", 1.0, None),
    ("outside", 20, 16, (90,), "outside", 1.0, None),
    ("outside_sorted", 20, 16, (1300,), "outside", 1.0, 0),
    ("none", 5, 8, (0,), "uniform", 1.0, None),
]
EMBEDDING_IDS = [c[0] for c in EMBEDDING_CASES]


def make_embedding(case, dtype, device, index=torch.int64):
    _, V, D, shape, kind, _, _ = case
    g = torch.Generator().manual_seed(11)
    n = math.prod(shape)
    if kind == "same":
        idx = torch.full((n,), V // 2)
        idx[:: 7] = 0
    elif kind == "skewed":
        idx = (V ** torch.rand(n, generator=g, dtype=torch.float64)).long().clamp_(0, V - 1)
    elif kind == "outside":
        idx = torch.randint(-10, V + 10, (n,), generator=g)
    else:
        idx = torch.randint(0, V, (n,), generator=g)
    weight = torch.randn(V, D, generator=g).to(dtype).to(device).requires_grad_()
    return idx.view(shape).to(index).to(device), weight, torch.randn(*shape, D, generator=g).to(dtype).to(device)


def embedding_reference(case, dtype, idx, weight, dout):
    _, V, D, shape, _, scale, pad = case
    w, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    t, W, dO = idx.cpu().long().reshape(-1), weight.detach().double().cpu(), dout.double().cpu().reshape(-1, D)
    inside = (t >= 0) & (t < V)
    out = (W[t.clamp(0, V - 1)] * scale).masked_fill(~inside.view(-1, 1), float("nan")).view(*shape, D)
    live = inside & (t != (-1 if pad is None else pad))
    total = lambda x: torch.zeros(V, D, dtype=torch.float64).index_add_(0, t[live], x[live])
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, t[live], torch.ones(int(live.sum()), dtype=torch.float64)).view(-1, 1)
    dw = total(dO) * scale
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return {"out": (out, (u + w) * out.abs() + tiny), "dw": (dw, w * (n + 1) * total(dO.abs()) * abs(scale) + u * dw.abs() + (n > 0) * tiny)}


def check(got, want, name):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(got), nan), name
    bad = ((got - value).abs() > bound) & ~nan
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d values out of bounds, first at %s: %r, want %r +- %.3g" % (
            name, int(bad.sum()), bad.numel(), at, float(got[at]), float(value[at]), float(bound[at])))
