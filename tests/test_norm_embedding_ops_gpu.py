"""ops.group_norm_act and ops.embedding on the GPU against 64 bits, with elementwise bounds (tests/norm_embedding_cases.py)."""
import pytest
import torch

from tests import norm_embedding_cases as C

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DTYPE_IDS = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("case", C.NORM_CASES, ids=C.NORM_IDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_norm(case, dtype):
    from ic_gan_amd import ops
    print("norm", case, dtype, flush=True)
    x, dy, gain, bias = C.make_norm(case, dtype, "cuda")
    y = ops.group_norm_act(x, case[5], gain, bias, act=case[6], gain_offset=case[9])
    assert y.dtype == dtype and y.is_contiguous(memory_format=torch.channels_last)
    leaves = [t for t in (x, gain, bias) if t is not None]
    got = dict(zip(("dx", "dgain", "dbias"), torch.autograd.grad(y, leaves, dy)), y=y)
    for name, want in C.norm_reference(case, dtype, x, dy, gain, bias).items():
        C.check(got[name], want, name)


@pytest.mark.parametrize("case", C.EMBEDDING_CASES, ids=C.EMBEDDING_IDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
def test_embedding(case, dtype):
    from ic_gan_amd import ops
    print("embedding", case, dtype, flush=True)
    for index in (torch.int64, torch.int32):
        idx, weight, dout = C.make_embedding(case, dtype, "cuda", index)
        out = ops.embedding(idx, weight, scale=case[5], padding_idx=case[6])
        (dw,) = torch.autograd.grad(out, (weight,), dout)
        want = C.embedding_reference(case, dtype, idx, weight, dout)
        C.check(out, want["out"], "out")
        C.check(dw, want["dw"], "dw")
