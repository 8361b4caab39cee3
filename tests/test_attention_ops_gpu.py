"""ops.attention on the GPU against 64 bits, with elementwise bounds (tests/attention_cases.py)."""
import pytest
import torch

from tests import attention_cases as C

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("case", C.CASES, ids=C.IDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "f16", "bf16"])
def test_values_and_gradients(case, dtype):
    from ic_gan_amd import ops
    print("attention", case, dtype, flush=True)
    q, k, v, do, lens, start = C.make(case, dtype, "cuda")
    o, lse = ops.attention(q, k, v, causal=case[8], k_lens=lens, q_start=start, return_lse=True)
    assert o.dtype == dtype and lse.dtype == torch.float32 and not lse.requires_grad
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    want = C.reference(case, dtype, q, k, v, do)
    for name, got in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        C.check(got, want[name], name)
    again = ops.attention(q, k, v, causal=case[8], k_lens=lens, q_start=start)
    assert torch.equal(o, again)
    for a, b in zip((dq, dk, dv), torch.autograd.grad(again, (q, k, v), do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=["f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk", [(3, 3), (40, 7), (130, 700), (2, 5000)])
def test_row_sums_of_the_unrounded_output(Lq, Lk, dtype):
    """q = 0: every p is 1 / Lk and a power of two before the division, so o is a mean in 32 bits.  Values far from zero make do . v - do . o
    cancel, and a row sum of the rounded o would be off by u |do| . |o|.  Left are: the rest of o, rounded (u^2 |o|, or half of 2^-24 where it is
    subnormal in fp16), sums in 32 bits (w times their terms, of which there are dv, Lk and a few), ds and dq rounded (u)."""
    from ic_gan_amd import ops
    g = torch.Generator().manual_seed(Lk)
    B, H, d, dv = 2, 2, 32, 64
    q = torch.zeros(B, Lq, H, d, device="cuda", dtype=dtype, requires_grad=True)
    k = torch.randn(B, Lk, H, d, generator=g).to("cuda", dtype).requires_grad_()
    v = (16.0 + torch.randn(B, Lk, H, dv, generator=g)).to("cuda", dtype).requires_grad_()
    do = torch.randn(B, Lq, H, dv, generator=g).to("cuda", dtype)
    dq, = torch.autograd.grad(ops.attention(q, k, v), (q,), do)
    K, V, dO = (t.detach().double().cpu().transpose(1, 2) for t in (k, v, do))
    o, dp, scale = V.mean(2, keepdim=True), dO @ V.transpose(-1, -2), d ** -0.5
    ds = (dp - (dO * o).sum(-1, keepdim=True)) / Lk
    want = ds @ K * scale
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    terms = dO.abs() @ V.abs().transpose(-1, -2)                         # >= what |do| . |o| has on average over the keys
    off = (w * (dv + Lk + 16) + u * u) * (terms + terms.mean(-1, keepdim=True)) + (2.0 ** -25 * dO.abs().sum(-1, keepdim=True) if dtype == torch.float16 else 0.0)
    bound = (off / Lk + (u + w * (Lk + 16)) * ds.abs() + (2.0 ** -30 * dO.norm(dim=-1).amax() if dtype == torch.float16 else 0.0)) @ K.abs() * scale
    bound = bound * (1 + 2 * u) + u * want.abs() + torch.finfo(dtype).tiny * u
    C.check(dq, (want.transpose(1, 2), bound.transpose(1, 2)), "dq")
