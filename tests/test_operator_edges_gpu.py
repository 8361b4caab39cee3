"""ops.attention, ops.group_norm_act and ops.embedding at the ends of what they accept: values up to the end of fp16, non-finite values, keys that
no query sees, tables and activations whose addresses pass 32 bits."""
import pytest
import torch

from tests import attention_cases as A, norm_embedding_cases as C

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DTYPE_IDS = ["f32", "f16", "bf16"]


# ---- fp16 gradients of large values ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("Lq", [1, 40, 200])
@pytest.mark.parametrize("v,do", [(1.0, 1.0), (200.0, 1.0), (200.0, 0.01), (1000.0, 0.01), (20000.0, 0.01), (65504.0, 2.0 ** -10), (2.0 ** -14, 2.0 ** -14)])
def test_fp16_gradient_of_two_opposite_values(v, do, Lq):
    """two keys with equal scores and values +v, -v: o = 0 exactly and ds = +-dv v do / 2.  ds and dq are rounded once each (u), the exponent log2 2
    and 2^x in 32 bits (8 w together), and a subnormal dq by half of 2^-24."""
    from ic_gan_amd import ops
    d, dv = 32, 128
    q = torch.zeros(1, Lq, 1, d, device="cuda", dtype=torch.float16, requires_grad=True)
    k = torch.zeros(1, 2, 1, d, device="cuda", dtype=torch.float16)
    ds = 0.5 * dv * float(torch.tensor(v).half()) * float(torch.tensor(do).half())
    key = 2.0 ** round(8 - torch.tensor(ds).log2().item()) if ds > 256 else 1.0          # (brings dq into the type's range)
    k[0, 0, 0, 3], k[0, 1, 0, 5] = key, -key
    k.requires_grad_()
    vals = torch.full((1, 2, 1, dv), v, device="cuda", dtype=torch.float16)
    vals[0, 1] *= -1
    o = ops.attention(q, k, vals, scale=1.0)
    assert not o.any()
    dq, dk = torch.autograd.grad(o, (q, k), torch.full_like(o, do))
    want = torch.zeros(1, Lq, 1, d, dtype=torch.float64)
    want[..., 3], want[..., 5] = ds * key, ds * key
    u = 2.0 ** -11
    assert bool(((dq.double().cpu() - want).abs() <= (2 * u * (1 + u) + 8 * 2.0 ** -24) * want.abs() + 2.0 ** -25).all()), (dq[0, 0, 0, 3], ds * key)
    assert not dk.any()                                          # (q is zero)


# (name of the case in attention_cases, factor on v, whether one value alone is that large)
@pytest.mark.parametrize("lone", [False, True], ids=["all_large", "one_large"])
@pytest.mark.parametrize("up", [1e2, 1e3, 1e4])
@pytest.mark.parametrize("name", ["odd_lengths", "causal_square_packed", "head_80", "causal_padded_shifted", "wide_values", "expanded_keys"])
def test_fp16_gradients_of_large_values(name, up, lone):
    """The bounds of attention_cases (each rounding of the kernels), and the step of ds where it is subnormal: ds is held s times as large, s a
    power of two with s max|do| max|v| in [512, 1024) 64, so half a step of 2^-24 is at most 2^-40 max|do| max|v|."""
    from ic_gan_amd import ops
    case = A.CASES[A.IDS.index(name)]
    q, k, v, do, lens, start = A.make(case, torch.float16, "cuda", 5)
    with torch.no_grad():
        if lone:                                                 # (the first key: every query that sees anything sees it)
            v = v.clone()
            v[:, :1] *= up
        else:
            v = (v.float() * up).half()
    v = v.detach().clamp(-65504, 65504).requires_grad_()
    do = (do.float() / up).half()
    o = ops.attention(q, k, v, causal=case[8], k_lens=lens, q_start=start)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    want = A.reference(case, torch.float16, q, k, v, do)
    B, Lq, Lk, H, Hk = case[1:6]
    V = v.detach().double().cpu().transpose(1, 2)
    if lens is not None:
        V = V.masked_fill((torch.arange(Lk).view(1, -1) >= torch.tensor(case[9]).view(-1, 1)).view(B, 1, Lk, 1), 0.0)
    least = 2.0 ** -40 * float(do.double().cpu().norm(dim=-1).max()) * float(V.norm(dim=-1).max())
    m = A.seen(case).unsqueeze(1).double()
    K, Q = (t.detach().double().cpu().transpose(1, 2) for t in (k, q))
    K = K.masked_fill(~torch.isfinite(K), 0.0)
    scale = case[6] ** -0.5
    more_q = (m @ K.abs().repeat_interleave(H // Hk, 1)) * least * scale
    more_k = (m.transpose(-1, -2) @ Q.abs()).view(B, Hk, H // Hk, Lk, -1).sum(2) * least * scale
    for n, got, more in (("o", o, None), ("dq", dq, more_q), ("dk", dk, more_k), ("dv", dv, None)):
        value, bound = want[n]
        A.check(got, (value, bound if more is None else bound + more.transpose(1, 2)), n)
