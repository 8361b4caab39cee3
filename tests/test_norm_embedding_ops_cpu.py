"""ops.group_norm_act and ops.embedding without a GPU: refusals, and their autograd wiring with the kernels emulated (oracle/kernel_ref.py)."""
import pytest
import torch

from oracle import kernel_ref
from tests import norm_embedding_cases as C


@pytest.mark.parametrize("case", C.NORM_CASES, ids=C.NORM_IDS)
def test_norm_wiring(case, monkeypatch):
    kernel_ref.install(monkeypatch)
    from ic_gan_amd import ops
    x, dy, gain, bias = C.make_norm(case, torch.float32, "cpu")
    y = ops.group_norm_act(x, case[5], gain, bias, act=case[6], gain_offset=case[9])
    leaves = [t for t in (x, gain, bias) if t is not None]
    got = dict(zip(("dx", "dgain", "dbias"), torch.autograd.grad(y, leaves, dy)), y=y)
    for name, want in C.norm_reference(case, torch.float32, x, dy, gain, bias).items():
        C.check(got[name], want, name)


@pytest.mark.parametrize("affine", ["channel", "sample"])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_norm_gradient_against_autograd(act, affine):
    """the reference's formula in 64 bits against autograd of the definition"""
    case = ("formula", 2, 12, 3, 5, 3, act, affine, 0.4, 1.0)
    x, dy, gain, bias = C.make_norm(case, torch.float64, "cpu")
    want = C.norm_reference(case, torch.float64, x, dy, gain, bias)
    g64, b64 = gain.detach().double().requires_grad_(), bias.detach().double().requires_grad_()
    rows = lambda t: t.view(-1, 12, 1, 1)
    y = torch.nn.functional.group_norm(x, 3, eps=1e-5) * (1 + rows(g64)) + rows(b64)
    y = torch.nn.functional.silu(y) if act == "silu" else y
    for name, got in zip(("dx", "dgain", "dbias"), torch.autograd.grad(y, (x, g64, b64), dy)):
        assert float((got - want[name][0]).abs().max()) < 1e-12, name


@pytest.mark.parametrize("case", C.EMBEDDING_CASES, ids=C.EMBEDDING_IDS)
def test_embedding_wiring(case, monkeypatch):
    kernel_ref.install(monkeypatch)
    from ic_gan_amd import ops
    idx, weight, dout = C.make_embedding(case, torch.float32, "cpu", torch.int32)
    out = ops.embedding(idx, weight, scale=case[5], padding_idx=case[6])
    (dw,) = torch.autograd.grad(out, (weight,), dout)
    want = C.embedding_reference(case, torch.float32, idx, weight, dout)
    C.check(out, want["out"], "out")
    C.check(dw, want["dw"], "dw")


def test_refusals():
    from ic_gan_amd import ops
    x = torch.zeros(2, 8, 3, 3)
    for args, kw, match in [
        ((x[0], 2), {}, "4-D"), ((x.double(), 2), {}, "fp32, fp16 or bf16"), ((x, 3), {}, "groups over"), ((x, 0), {}, "groups over"),
        ((x, 2.0), {}, "groups over"), ((x, 2), dict(act="gelu"), "act must be"), ((x, 2), dict(eps=-1.0), "eps"), ((x, 2), dict(eps=float("nan")), "eps"),
        ((x, 2, torch.zeros(7)), {}, "gain must be"), ((x, 2, torch.zeros(1, 8)), {}, "gain must be"), ((x, 2, None, torch.zeros(8, dtype=torch.int64)), {}, "bias must be"),
        ((x, 2, torch.zeros(8), torch.zeros(2, 8)), {}, "differ in shape"),
    ]:
        with pytest.raises(ValueError, match=match):
            ops.group_norm_act(*args, **kw)
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        ops.group_norm_act(x, 2)
    w, i = torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
    for args, kw, match in [
        ((i, w[0]), {}, "weight must be"), ((i, w.double()), {}, "weight must be"), ((i.float(), w), {}, "idx must be"), ((i, w[:0]), {}, "not served"),
        ((i, w[:, :0]), {}, "not served"), ((i, w), dict(scale=float("inf")), "scale"), ((i, w), dict(scale=float("nan")), "scale"),
        ((i, w), dict(padding_idx=5), "padding_idx"), ((i, w), dict(padding_idx=-1), "padding_idx"),
    ]:
        with pytest.raises(ValueError, match=match):
            ops.embedding(*args, **kw)
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        ops.embedding(i, w)


def test_entry_points_refuse_before_a_launch():
    import ctypes
    from ic_gan_amd import _lib
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) & ~15
    def fwd(x=p, B=1, HW=1 << 20, C=64, G=4, eps=1e-5, act=0, dtype=0, ws=p, nb=0):
        return lib.icg_groupnorm_act_fwd(x, None, None, p, p, p, B, HW, C, G, 0, 0.0, eps, act, dtype, ws, nb, None)
    assert fwd() == -3 and fwd(x=None) == -1 and fwd(G=5) == -1 and fwd(eps=-1.0) == -1 and fwd(act=3) == -1 and fwd(dtype=4) == -1 and fwd(HW=0) == -1
    assert fwd(ws=None, nb=1 << 30) == -1
    def bwd(dgain=p, dbias=p, nb=1 << 30, C=64):
        return lib.icg_groupnorm_act_bwd(p, p, None, None, p, p, p, dgain, dbias, 1, 16, C, 4, 0, 0.0, 1e-5, 0, 0, p, nb, None)
    assert bwd(nb=0) == -3 and bwd(dgain=None) == -1 and bwd(C=66) == -1
    assert lib.icg_embedding_fwd(p, p, p, 0, 5, 5, 1.0, 1, 0, None) == -1 and lib.icg_embedding_fwd(None, p, p, 5, 5, 5, 1.0, 1, 0, None) == -1
    assert lib.icg_embedding_bwd(p, p, p, 5000, 5, 5, 1.0, -1, 1, 0, p, 16, None) == -3
    assert lib.icg_embedding_bwd(p, p, p, 5000, 5, 5, 1.0, -1, 1, 0, None, 1 << 30, None) == -1
