"""Cases, a 64-bit reference and elementwise error bounds for ops.attention (shared by the CPU and GPU tests).

The bounds follow the kernels' roundings.  u: half a step of the element type.  With S_ij = scale sum_c |q_ic| |k_jc| and 32-bit arithmetic (half a
step w = 2^-24):
  scores and exponents      |dp_ij| <= p_ij e,  e = w (4 (d + 4) max S + 4 max |l| + Lk + Lq H / Hk + 32): a sum of n products is off by at most n w
                            times the sum of their magnitudes; the exponent's argument by a few w times its magnitude
  p, ds as operands         rounded to the element type (u relative; fp16 also 2^-25 absolute in its own scale), not at all in fp32
  D_i = do_i . o_i          from the rounded o: off by |do_i| . (bound of o_i)
  underflow                 2^x ends at fp32's smallest normal number, f = 2^-126 (what is below becomes 0), and so do operands and sums of the
                            matrix products: p is off by up to f beside its relative error, ds by f (1 + |dp| + |D|), a sum of n products by n f
  outputs                   one rounding to the element type"""
import math

import torch

# name, B, Lq, Lk, H, Hk, d, dv, causal, k_lens, q_start, layout
CASES = [
    ("one_pair", 1, 1, 1, 1, 1, 8, 8, False, None, None, "plain"),
    ("one_key_many_queries", 2, 70, 1, 2, 1, 16, 16, False, None, None, "plain"),
    ("token_short", 2, 1, 333, 8, 8, 64, 64, False, [37, 333], None, "plain"),
    ("token_grouped_split", 3, 1, 1700, 8, 2, 128, 128, False, [0, 1, 1700], None, "plain"),
    ("token_odd_head", 2, 1, 300, 3, 1, 33, 35, False, [299, 300], None, "odd"),
    ("few_queries_causal", 2, 5, 77, 6, 2, 24, 96, True, None, None, "packed_kv"),
    ("few_queries_wide_values", 1, 7, 130, 2, 1, 64, 256, False, None, None, "plain"),
    ("few_queries_many_heads", 1, 3, 90, 40, 1, 48, 192, True, [80], [60], "plain"),
    ("odd_lengths", 2, 130, 131, 3, 1, 40, 40, False, None, None, "plain"),
    ("odd_everything", 1, 129, 257, 2, 2, 33, 35, False, [250], None, "odd"),
    ("causal_square_packed", 2, 192, 192, 4, 2, 64, 64, True, None, None, "packed"),
    ("causal_more_queries_than_keys", 2, 200, 150, 2, 1, 32, 128, True, None, None, "plain"),
    ("image_block", 2, 256, 64, 1, 1, 48, 192, False, None, None, "plain"),
    ("image_block_narrow", 2, 256, 64, 1, 1, 24, 96, False, None, None, "plain"),
    ("wide_values", 1, 160, 96, 2, 1, 64, 256, False, None, None, "plain"),
    ("head_80", 1, 96, 200, 2, 2, 80, 72, False, None, None, "heads_first"),
    ("causal_padded_shifted", 3, 150, 300, 4, 4, 128, 128, True, [300, 0, 170], [150, 3, 100], "plain"),
    ("padded_none_seen", 2, 40, 50, 2, 2, 16, 16, True, [50, 50], [-100, -20], "plain"),
    ("long_keys_split", 1, 40, 3000, 1, 1, 16, 16, False, None, None, "plain"),
    ("expanded_keys", 2, 64, 100, 4, 4, 32, 32, False, None, None, "expanded"),
]
IDS = [c[0] for c in CASES]


def make(case, dtype, device, seed=0, spread=1.0):
    """-> q, k, v, do (leaves of the case's layout), k_lens, q_start; what lies behind a sequence's last key is NaN"""
    _, B, Lq, Lk, H, Hk, d, dv, causal, lens, start, layout = case
    g = torch.Generator().manual_seed(seed + 1)
    n = lambda *s: torch.randn(*s, generator=g).mul_(spread).to(dtype)
    q, k, v, do = n(B, Lq, H, d), n(B, Lk, Hk, d), n(B, Lk, Hk, dv), n(B, Lq, H, dv)
    if lens is not None:
        for b, m in enumerate(lens):
            k[b, m:], v[b, m:] = float("nan"), float("nan")
    if layout == "packed":                       # views of one buffer, as a fused projection leaves them
        buf = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(device)
        q, k, v = buf.split([H * d, Hk * d, Hk * dv], -1)
        q, k, v = q.unflatten(-1, (H, d)), k.unflatten(-1, (Hk, d)), v.unflatten(-1, (Hk, dv))
    elif layout == "packed_kv":
        buf = torch.cat([k, v], -1).to(device)
        k, v = buf.split([d, dv], -1)
    elif layout == "heads_first":                # [B, H, L, e] memory
        q, k, v, do = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (q, k, v, do))
    elif layout == "odd":                        # rows that start anywhere
        def odd(t):
            w = torch.full(t.shape[:-1] + (t.shape[-1] + 3,), float("nan"), dtype=dtype, device=device)
            w[..., 1:1 + t.shape[-1]] = t.to(device)
            return w[..., 1:1 + t.shape[-1]]
        q, k, v, do = odd(q), odd(k), odd(v), odd(do)
    elif layout == "expanded":                   # one key head, one gradient row, seen as many
        k, v = k[:, :, :1].to(device).expand(-1, -1, Hk, -1), v[:, :, :1].to(device).expand(-1, -1, Hk, -1)
        do = do[:, :1].to(device).expand(-1, Lq, -1, -1)
    ints = lambda t: None if t is None else torch.tensor(t, dtype=torch.int32, device=device)
    q, k, v, do = (t.to(device).detach() for t in (q, k, v, do))
    return q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), do, ints(lens), ints(start)


def seen(case):
    """[B, Lq, Lk]"""
    _, B, Lq, Lk, H, Hk, d, dv, causal, lens, start, _ = case
    j, i = torch.arange(Lk).view(1, 1, -1), torch.arange(Lq).view(1, -1, 1)
    m = j < (torch.full((B,), Lk) if lens is None else torch.tensor(lens)).view(-1, 1, 1)
    if causal:
        m = m & (j <= (torch.full((B,), Lk - Lq) if start is None else torch.tensor(start)).view(-1, 1, 1) + i)
    return m.expand(B, Lq, Lk)


def reference(case, dtype, q, k, v, do, scale=None):
    """-> {name: (value, bound)}, float64 on the CPU, for o, lse, dq, dk, dv"""
    _, B, Lq, Lk, H, Hk, d, dv, causal, lens, start, _ = case
    G = H // Hk
    scale = d ** -0.5 if scale is None else scale
    m = seen(case).unsqueeze(1)                                          # [B, 1, Lq, Lk]
    Q, K, V, dO = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v, do))        # [B, heads, L, e]
    if lens is not None:                                                 # nothing behind the last key counts, whatever it holds
        gone = (torch.arange(Lk).view(1, -1) >= torch.tensor(lens).view(-1, 1)).view(B, 1, Lk, 1)
        K, V = K.masked_fill(gone, 0.0), V.masked_fill(gone, 0.0)
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = (Q @ K.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.unsqueeze(-1).nan_to_num(neginf=0.0)).masked_fill(~m, 0.0)
    o = p @ V
    D = (dO * o).sum(-1, keepdim=True)
    dp = dO @ V.transpose(-1, -2)
    ds = p * (dp - D)
    shared = lambda t: t.view(B, Hk, G, Lk, -1).sum(2)
    dq, dk, dv_ = ds @ K * scale, shared(ds.transpose(-1, -2) @ Q * scale), shared(p.transpose(-1, -2) @ dO)

    w, u, f = 2.0 ** -24, torch.finfo(dtype).eps / 2, 2.0 ** -126
    up = 0.0 if dtype == torch.float32 else u                            # p and ds as operands
    S = (Q.abs() @ K.abs().transpose(-1, -2) * scale).masked_fill(~m, 0.0)
    biggest = lambda t: float(t.masked_fill(~torch.isfinite(t), 0.0).abs().max()) if t.numel() else 0.0
    e = w * (4 * (d + 4) * biggest(S) + 4 * biggest(lse) + Lk + Lq * G + 32)
    f16 = dtype == torch.float16
    A = p @ V.abs()
    seen_v = m.double() @ V.abs()
    b_o = (up + 2 * e) * A + ((2.0 ** -25 if f16 else 0.0) + f) * seen_v + Lk * f + u * o.abs()
    b_lse = torch.full_like(lse, e) + w * 4 * lse.abs().nan_to_num(posinf=0.0)
    aO, aQ, aK = dO.abs(), Q.abs(), K.abs()
    pT = p.transpose(-1, -2)
    mT = m.double().transpose(-1, -2)
    b_dv = (up + e) * (pT @ aO) + ((2.0 ** -31 if f16 else 0.0) + f) * (mT @ aO) + Lq * G * f
    e_dp = w * (dv + 2) * (aO @ V.abs().transpose(-1, -2))
    e_D = (aO * b_o).sum(-1, keepdim=True) + w * (dv + 2) * (aO * o.abs()).sum(-1, keepdim=True)
    E = p * (e_dp + e_D) + (up + e) * ds.abs() + e * p * (dp.abs() + D.abs()) + f * m.double() * (1 + dp.abs() + D.abs())
    if f16:                                                              # ds is held 2^6 / (2^k, the largest |do| of what is summed) times as large
        E = E + 2.0 ** -30 * dO.norm(dim=-1).amax() * m.double()
    b_dq = E @ aK * scale + w * (Lk + 4) * (ds.abs() @ aK) * scale + Lk * f
    b_dk = E.transpose(-1, -2) @ aQ * scale + w * (Lq * G + 4) * (ds.abs().transpose(-1, -2) @ aQ) * scale + Lq * G * f
    back = lambda t: t.transpose(1, 2)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2          # outputs that are subnormal in the type
    out = {"o": (back(o), back(b_o) + tiny), "lse": (lse, b_lse), "dq": (back(dq), back(b_dq + u * dq.abs()) + tiny)}
    for name, value, b in (("dk", dk, shared(b_dk)), ("dv", dv_, shared(b_dv))):
        out[name] = (back(value), back(b + u * value.abs()) + tiny)
    return out


def check(got, want, name):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    inf = torch.isinf(value)
    assert torch.equal(got[inf], value[inf]), name
    bad = ~((got - value).abs() <= bound) & ~inf
    if bool(bad.any()):
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d values out of bounds, first at %s: %r, want %r +- %.3g; worst %.3g bounds" % (
            name, int(bad.sum()), bad.numel(), at, float(got[at]), float(value[at]), float(bound[at]),
            float(((got - value).abs() / bound.clamp_min(1e-300)).nan_to_num(nan=math.inf)[~inf].max())))
