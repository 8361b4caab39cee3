"""ops.attention without a GPU: what it refuses, and its autograd wiring with the kernels emulated (oracle/kernel_ref.py)."""
import pytest
import torch

from oracle import kernel_ref
from tests import attention_cases as C


@pytest.mark.parametrize("case", C.CASES, ids=C.IDS)
def test_wiring(case, monkeypatch):
    kernel_ref.install(monkeypatch)
    from ic_gan_amd import ops
    q, k, v, do, lens, start = C.make(case, torch.float32, "cpu")
    o, lse = ops.attention(q, k, v, causal=case[8], k_lens=lens, q_start=start, return_lse=True)
    got = torch.autograd.grad(o, (q, k, v), do)
    want = C.reference(case, torch.float32, q, k, v, do)
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + got):
        C.check(t, want[name], name)


def test_gradient_against_differences(monkeypatch):
    """the formula of the backward pass, in 64 bits, against central differences of the forward's"""
    case = ("differences", 1, 4, 6, 2, 1, 3, 5, True, [5], [1], "plain")
    q, k, v, do, lens, start = (t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for t in C.make(case, torch.float64, "cpu"))
    k, v = k.detach().nan_to_num(0.0), v.detach().nan_to_num(0.0)
    q = q.detach()
    want = C.reference(case, torch.float64, q, k, v, do)
    f = lambda: float((C.reference(case, torch.float64, q, k, v, do)["o"][0] * do).sum())
    step = 1e-5                                  # error of a central difference: step^2 times third derivatives of order 1, plus 1e-16 / step
    for t, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        flat, grad = t.view(-1), want[name][0].reshape(-1)
        for i in range(flat.numel()):
            x = float(flat[i])
            flat[i] = x + step
            up = f()
            flat[i] = x - step
            down = f()
            flat[i] = x
            assert abs((up - down) / (2 * step) - float(grad[i])) < 1e-8


def _qkv(**change):
    a = dict(B=2, Lq=3, Lk=4, H=4, Hk=2, d=8, dv=8, dtype=torch.float32)
    a.update(change)
    return (torch.zeros(a["B"], a["Lq"], a["H"], a["d"], dtype=a["dtype"]), torch.zeros(a["B"], a["Lk"], a["Hk"], a["d"], dtype=a["dtype"]),
            torch.zeros(a["B"], a["Lk"], a["Hk"], a["dv"], dtype=a["dtype"]))


def test_refusals():
    from ic_gan_amd import ops
    q, k, v = _qkv()
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        ops.attention(q, k, v)
    for bad, match in [
        ((q[0], k, v), "4-D"), ((q, k.half(), v), "one type"), (_qkv(dtype=torch.float64), "fp32, fp16 or bf16"),
        ((q, k[:1], v), "shapes do not fit"), ((q, k, v[:, :3]), "shapes do not fit"), ((q, k[..., :7], v), "shapes do not fit"),
        ((q, k, v[:, :, :1]), "shapes do not fit"), (_qkv(H=5), "query heads"), (_qkv(Hk=0), "query heads"), (_qkv(d=0), "no elements"),
        (_qkv(dv=0), "no elements"), (_qkv(d=136), "not served"), (_qkv(d=72, dv=136), "not served"), (_qkv(d=64, dv=260), "not served"),
    ]:
        with pytest.raises(ValueError, match=match):
            ops.attention(*bad)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            ops.attention(q, k, v, scale=scale)
    for name in ("k_lens", "q_start"):
        for t in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(2, 1, dtype=torch.int32), [1, 2]):
            with pytest.raises(ValueError, match=name):
                ops.attention(q, k, v, **{name: t})


def test_entry_points_refuse_before_a_launch():
    """the C entry points check sizes, pointers and workspaces on the host"""
    import ctypes
    from ic_gan_amd import _lib
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) & ~15
    def fwd(q=p, o=p, o_low=None, B=1, Lq=1, Lk=2048, H=2, Hk=1, d=8, dv=8, scale=1.0, dtype=0, ws=p, nb=0):
        return lib.icg_attention_fwd(q, p, p, None, None, o, o_low, p, B, Lq, Lk, H, Hk, d, dv, *[8] * 9, scale, 0, dtype, ws, nb, None)
    assert fwd(q=None) == -1 and fwd(o=p + 4) == -1 and fwd(o_low=p + 8) == -1 and fwd(Hk=3) == -1 and fwd(d=200) == -1 and fwd(d=128, dv=256) == -1
    assert fwd(scale=0.0) == -1 and fwd(scale=float("nan")) == -1 and fwd(dtype=3) == -1 and fwd(Lq=0) == -1 and fwd(B=1 << 20, H=1 << 12) == -1
    assert lib.icg_attention_fwd_workspace_bytes(1, 1, 2048, 2, 1, 8, 8, 0) > 0 and fwd(nb=0) == -3
    def bwd(dq=p, nb=1 << 20, Lq=1, ws=p):
        return lib.icg_attention_bwd(p, p, p, p, None, p, p, None, None, dq, p, p, 1, Lq, 16, 2, 1, 8, 8, *[8] * 12, 1.0, 0, 0, ws, nb, None)
    assert bwd(dq=None) == -1 and bwd(dq=p + 8) == -1 and bwd(nb=0) == -3 and bwd(ws=None) == -1 and bwd(Lq=-1) == -1
