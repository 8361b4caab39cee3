"""What ops.attention, ops.group_norm_act and ops.embedding refuse at the ends of their ranges, forward-mode derivatives, and the device that a
kernel is launched on (no GPU: kernels emulated or entry points that check on the host)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from oracle import kernel_ref


def _calls(ops):
    q, k, v = (torch.randn(2, n, 2, 8) for n in (3, 5, 5))
    x, gain, bias = torch.randn(2, 8, 3, 3), torch.randn(8), torch.randn(8)
    w, idx = torch.randn(7, 4), torch.tensor([1, 5, 1])
    return {"attention": (lambda q, k, v: ops.attention(q, k, v), (q, k, v)),
            "attention_lse": (lambda q, k, v: ops.attention(q, k, v, return_lse=True)[0], (q, k, v)),
            "group_norm_act": (lambda x, gain, bias: ops.group_norm_act(x, 2, gain, bias, act="silu"), (x, gain, bias)),
            "embedding": (lambda w: ops.embedding(idx, w), (w,))}


@pytest.mark.parametrize("graph", [False, True], ids=["no_gradient", "gradient"])
@pytest.mark.parametrize("name", ["attention", "attention_lse", "group_norm_act", "embedding"])
def test_a_tangent_is_refused_and_not_lost(name, graph, monkeypatch):
    kernel_ref.install(monkeypatch)
    from ic_gan_amd import ops
    f, ins = _calls(ops)[name]
    want = f(*ins)
    with forward_ad.dual_level():
        assert torch.equal(f(*ins), want)                        # (no tangent: an ordinary call)
        for i in range(len(ins)):
            dual = [forward_ad.make_dual(t.clone().requires_grad_(graph), torch.ones_like(t)) if j == i else t for j, t in enumerate(ins)]
            with pytest.raises(NotImplementedError):
                f(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                f(*dual)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(f, ins, tuple(torch.ones_like(t) for t in ins))


@pytest.mark.parametrize("name", ["attention", "group_norm_act", "embedding"])
def test_a_gradient_with_a_tangent_is_refused(name, monkeypatch):
    kernel_ref.install(monkeypatch)
    from ic_gan_amd import ops
    f, ins = _calls(ops)[name]
    ins = [t.clone().requires_grad_() for t in ins]
    y = f(*ins)
    want = torch.autograd.grad(y, ins, torch.ones_like(y), retain_graph=True)
    with forward_ad.dual_level():
        for a, b in zip(torch.autograd.grad(y, ins, torch.ones_like(y), retain_graph=True), want):
            assert torch.equal(a, b)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y, ins, forward_ad.make_dual(torch.ones_like(y), torch.randn_like(y)))


def test_norm_sizes_are_refused_with_the_arguments():
    """a ValueError like every other refusal, before anything is launched"""
    from ic_gan_amd import ops
    for shape, groups in (((65536, 4, 1, 1), 2), ((1, 4, 1 << 15, 1 << 15), 2), ((1, 1 << 20, 1, 1), 1), ((60000, 1024, 1024, 1024), 1024)):
        with pytest.raises(ValueError, match="not served"):
            ops.group_norm_act(torch.empty(shape, device="meta"), groups)
    for shape in ((0, 8, 4, 4), (65535, 1024, 1, 1)):
        with pytest.raises(RuntimeError, match="AMD GPU only"):
            ops.group_norm_act(torch.empty(shape, device="meta"), 2)


def test_a_64_bit_gain_is_refused():
    from ic_gan_amd import ops
    x, one = torch.zeros(2, 8, 3, 3), torch.ones(8)
    for gain, bias, match in ((one.double(), one, "gain must be"), (one, one.double(), "bias must be"), (None, one.double(), "bias must be")):
        with pytest.raises(ValueError, match=match):
            ops.group_norm_act(x, 2, gain, bias)


def test_norm_entry_points_refuse_grids_beyond_the_launch_limit():
    import ctypes
    from ic_gan_amd import _lib
    lib = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) & ~15
    fwd = lambda B, HW, C, G: lib.icg_groupnorm_act_fwd(p, None, None, p, p, p, B, HW, C, G, 0, 0.0, 1e-5, 0, 0, p, 1 << 60, None)
    bwd = lambda B, HW, C, G: lib.icg_groupnorm_act_bwd(p, p, None, None, p, p, p, None, None, B, HW, C, G, 0, 0.0, 1e-5, 0, 0, p, 1 << 60, None)
    for B, HW, C, G in ((65536, 1, 4, 2), (1, 1 << 30, 4, 2), (60000, 1 << 20, 1024, 1024), (1, (1 << 30) - 1, 4097, 1)):
        assert lib.icg_groupnorm_applies(B, HW, C, G, 0) == 0 and fwd(B, HW, C, G) == -1 and bwd(B, HW, C, G) == -1
    assert lib.icg_groupnorm_applies(64, 65536, 96, 16, 0) == 1 and lib.icg_groupnorm_applies(1, 1, 1, 1, 2) == 1
    assert lib.icg_groupnorm_applies(2, 4, 8, 3, 0) == 0 and lib.icg_groupnorm_applies(2, 4, 8, 2, 3) == 0


class _On(torch.Tensor):
    """a host tensor that says it is on a device"""
    device_index = 0

    def get_device(self):
        return self.device_index


@pytest.mark.parametrize("current,tensor", [(0, 0), (0, 3), (2, 1)])
def test_a_kernel_goes_to_the_device_and_stream_of_its_tensors(current, tensor, monkeypatch):
    from ic_gan_amd import _lib
    state, seen = {"device": current}, []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index

        def __exit__(self, *a):
            state["device"] = self.before
    t = torch.zeros(4).as_subclass(_On)
    t.device_index = tensor
    monkeypatch.setattr(_lib, "_raw_stream", lambda d: 1000 + d)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["device"], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setitem(_lib._bound, "icg_pretended", lambda *a: seen.append((state["device"],) + a) or 0)
    _lib.call("icg_pretended", None, 7, t, 2.5)
    assert seen == [(tensor, None, 7, t.data_ptr(), 2.5, 1000 + tensor)] and state["device"] == current
    monkeypatch.setitem(_lib._bound, "icg_pretended", lambda *a: -1)
    with pytest.raises(RuntimeError, match="icg_pretended failed"):
        _lib.call("icg_pretended", t)
    assert state["device"] == current
