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
