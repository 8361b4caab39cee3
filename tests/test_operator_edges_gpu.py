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


@pytest.mark.parametrize("Lq", [1, 50])
def test_fp16_output_stays_within_the_values(Lq):
    """An output is a mean of values, so finite values give finite outputs.  128 keys of score 0, then 3968 of score 1.2 u: their p = 1 + 1.2 u is
    rounded to 1 + 2 u for the product and not in the sum, which brings the quotient to (1 + 0.77 u) times the values' 65504 -- past 65520,
    where a conversion gives inf.  (512 heads: enough that a head's keys are not split, and its running maximum stays at the first keys')"""
    from ic_gan_amd import ops
    u, Lk, B, H = 2.0 ** -11, 4096, 2, 256
    q = torch.zeros(B, Lq, H, 8, device="cuda", dtype=torch.float16)
    q[..., 0] = 1
    k = torch.zeros(1, Lk, 1, 8, device="cuda", dtype=torch.float16)
    k[:, 128:, :, 0] = 1
    for sign in (1.0, -1.0):
        v = torch.full((1, Lk, 1, 16), 65504.0 * sign, device="cuda", dtype=torch.float16)
        kk, vv = (t.expand(B, -1, H, -1) for t in (k, v))
        for grad in (False, True):
            o = ops.attention(q.detach().requires_grad_(grad), kk, vv, scale=1.2 * u).detach()
            assert bool((o.double() * sign >= 65504 * (1 - 3 * u)).all()) and bool((o.double().abs() <= 65504).all()), o
        v[0, 200, 0, 3] = float("inf")                           # (an infinity among the values stays one)
        o = ops.attention(q, kk, vv, scale=1.2 * u)
        assert not torch.isfinite(o[..., 3]).any() and torch.isfinite(o[..., :3]).all()


# ---- keys that no query sees -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("Lq,d,dv", [(1, 64, 64), (5, 24, 96), (33, 128, 128), (130, 40, 40), (150, 64, 256)])
def test_what_lies_behind_the_last_query(Lq, d, dv, dtype, bad):
    """causal with q_start into a longer buffer, as a chunk of a prompt meets a cache: keys behind the last query's own are seen by none, whatever
    they hold, and their gradient is zero"""
    from ic_gan_amd import ops
    B, Lk, H, Hk = 2, 300, 4, 2
    start = [0, 17]
    q, k, v, do = (torch.randn(B, n, h, e, device="cuda").to(dtype) for n, h, e in ((Lq, H, d), (Lk, Hk, d), (Lk, Hk, dv), (Lq, H, dv)))
    runs = []
    for fill in (0.0, bad):
        kk, vv = k.clone(), v.clone()
        for b, s in enumerate(start):
            kk[b, s + Lq:], vv[b, s + Lq:] = fill, fill
        leaves = [t.clone().requires_grad_() for t in (q, kk, vv)]
        o = ops.attention(*leaves, causal=True, q_start=torch.tensor(start, device="cuda", dtype=torch.int32))
        runs.append((o.detach(),) + torch.autograd.grad(o, leaves, do))
    for name, a, b in zip(("o", "dq", "dk", "dv"), *runs):
        assert torch.isfinite(a).all() and torch.equal(a, b), name
    for b, s in enumerate(start):
        assert not runs[1][2][b, s + Lq:].any() and not runs[1][3][b, s + Lq:].any()


# ---- group norm of non-finite values ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=DTYPE_IDS)
@pytest.mark.parametrize("shape,groups", [((2, 48, 7, 5), 16), ((2, 64, 40, 48), 4), ((2, 96, 96, 80), 16), ((1, 33, 101, 97), 3)],
                         ids=["one_pass", "one_pass_wide", "three_passes", "three_passes_scalar"])
def test_norm_shows_what_is_not_finite(shape, groups, dtype, act, bad):
    """one NaN or infinity makes its group's mean and deviation NaN, and so every value and gradient of that group and sample, whatever the
    activation; no other group, and no other sample, changes"""
    from ic_gan_amd import ops
    g = torch.Generator().manual_seed(3)
    B, C, H, W = shape
    x, dy = (torch.randn(*shape, generator=g).to(dtype).cuda().contiguous(memory_format=torch.channels_last) for _ in range(2))
    gain, bias = (torch.randn(B, C, generator=g).cuda() for _ in range(2))
    runs = []
    for value in (None, bad):
        leaves = [x.clone(), gain.clone(), bias.clone()]
        if value is not None:
            leaves[0][B - 1, C // 2, H // 2, W // 3] = value
        for t in leaves:
            t.requires_grad_()
        y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act)
        runs.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
    at = slice(C // 2 // (C // groups) * (C // groups), (C // 2 // (C // groups) + 1) * (C // groups))
    for name, a, b in zip(("y", "dx", "dgain", "dbias"), *runs):
        assert torch.isfinite(a).all()
        if name != "dbias" or act != "none":                     # (without an activation dbias is the sum of dy, whatever x is)
            assert torch.isnan(b[B - 1, at]).all(), name
            b = b.clone()
            b[B - 1, at] = a[B - 1, at]
        assert torch.equal(a, b), name


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", [((3, 32, 4, 4), 8), ((2, 96, 96, 80), 16)], ids=["one_pass", "three_passes"])
def test_norm_shows_a_gain_that_is_not_finite(shape, groups, act):
    from ic_gan_amd import ops
    x = torch.randn(*shape, device="cuda").contiguous(memory_format=torch.channels_last)
    gain, bias = torch.randn(shape[1], device="cuda"), torch.randn(shape[1], device="cuda")
    good = ops.group_norm_act(x, groups, gain, bias, act=act)
    gain[3] = float("nan")
    y = ops.group_norm_act(x, groups, gain, bias, act=act)
    assert torch.isnan(y[:, 3]).all()
    y[:, 3] = good[:, 3]
    assert torch.equal(y, good)


# ---- addresses and grids beyond 32 bits ------------------------------------------------------------------------------------------------
def test_norm_beyond_two_to_the_31_elements():
    """65 samples of 33.5 million elements: the last one begins at element 2^31.  Values and gradients are those of the sample alone, but for
    the chunks that its sums are formed in (equal up to fp32 rounding, so outputs are within one step of bf16)."""
    from ic_gan_amd import ops
    shape = (65, 64, 512, 1024)
    assert (shape[0] - 1) * 64 * 512 * 1024 >= 2 ** 31
    x, dy = (torch.empty(shape, dtype=torch.bfloat16, device="cuda", memory_format=torch.channels_last).normal_() for _ in range(2))
    x.requires_grad_()
    y = ops.group_norm_act(x, 8, act="silu")
    (dx,) = torch.autograd.grad(y, x, dy)
    last = x.detach()[-1:].clone().requires_grad_()
    z = ops.group_norm_act(last, 8, act="silu")
    (dz,) = torch.autograd.grad(z, last, dy[-1:])
    for a, b in ((y[-1:], z), (dx[-1:], dz)):
        a, b = a.detach().float(), b.detach().float()
        assert float(b.abs().max()) > 1 and float(((a - b).abs() / (b.abs() + 1e-2)).max()) <= 2 ** -7


@pytest.mark.parametrize("n", [20, 1500], ids=["few", "sorted"])
def test_embedding_table_beyond_two_to_the_31_elements(n):
    from ic_gan_amd import ops
    V, D = (1 << 22) + 3, 520
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    idx = torch.cat([torch.arange(V - n // 2, V), torch.arange(n - n // 2)]).cuda()
    assert V * D > 2 ** 31 and (V - n // 2) * D > 2 ** 31
    rows = torch.randn(n, D, device="cuda").bfloat16()
    w[idx] = rows
    w.requires_grad_()
    out = ops.embedding(idx, w)
    assert torch.equal(out, rows)
    (dw,) = torch.autograd.grad(out, w, rows.flip(0))
    assert torch.equal(dw[idx], rows.flip(0))                    # (each token once: copies)
    dw[idx] = 0
    assert not any(bool(part.any()) for part in dw.split(1 << 20))


def test_embedding_output_beyond_two_to_the_31_elements():
    from ic_gan_amd import ops
    V, D, n = 11, 520, (1 << 22) + 5
    assert n * D > 2 ** 31
    w = torch.randn(V, D, device="cuda").bfloat16().requires_grad_()
    idx = torch.randint(0, V, (n,), device="cuda")
    out = ops.embedding(idx, w)
    assert torch.equal(out[-1000:], w.detach()[idx[-1000:]]) and torch.equal(out[:1000], w.detach()[idx[:1000]])
    dout = torch.zeros_like(out)
    dout[-100:] = torch.randint(-8, 9, (100, D), device="cuda").bfloat16()
    (dw,) = torch.autograd.grad(out, w, dout)
    want = torch.zeros(V, D, device="cuda").index_add_(0, idx[-100:], dout[-100:].float())       # (whole numbers below 2^11: exact)
    assert torch.equal(dw.float(), want.bfloat16().float())


@pytest.mark.parametrize("n", [9, 1030], ids=["few", "sorted"])
def test_embedding_gradient_of_more_rows_than_a_grid_of_waves(n):
    """2^26 rows and some: a wave for each would be more threads than one dimension of a grid holds (2^32)"""
    from ic_gan_amd import ops
    V, D = (1 << 26) + 7, 3
    w = torch.zeros(V, D, device="cuda", requires_grad=True)
    idx = torch.cat([torch.arange(V - n + 3, V), torch.tensor([0, 5, 5])]).cuda()
    (dw,) = torch.autograd.grad(ops.embedding(idx, w), w, torch.ones(n, D, device="cuda"))
    assert bool((dw[V - n + 3:] == 1).all()) and bool((dw[0] == 1).all()) and bool((dw[5] == 2).all())
    assert float(dw.sum(dtype=torch.float64)) == n * D


@pytest.mark.parametrize("Lq", [1, 17])
def test_attention_of_more_tiles_than_a_grid_of_workgroups(Lq):
    """2^24 sequences and some: a workgroup of 256 for each would be more threads than one dimension of a grid holds (2^32).  One key each, so
    o is the value and its gradient the sum of do (few whole numbers: exact)."""
    from ic_gan_amd import ops
    B = (1 << 24) + 3
    q, k, v = (torch.ones(B, n, 1, 8, device="cuda", dtype=torch.bfloat16) for n in (Lq, 1, 1))
    v[:, 0, 0, 1] = torch.arange(B, device="cuda").remainder(200).bfloat16()
    v.requires_grad_()
    o = ops.attention(q, k, v)
    assert all(torch.equal(a, b.expand_as(a)) for a, b in zip(o.split(1 << 22), v.detach().split(1 << 22)))
    do = (torch.arange(B, device="cuda").remainder(3) + 1).bfloat16().view(B, 1, 1, 1).expand(B, Lq, 1, 8)
    (dv,) = torch.autograd.grad(o, v, do)
    assert torch.equal(dv, (do[:, :1] * Lq))


# ---- the spectral-norm embedding's gradient, its correction term included --------------------------------------------------------------
def test_gradient_of_a_large_spectral_norm_table():
    """layers.SNEmbedding with more labels than the one-hot product takes.  With the vectors of its own power-iteration step, u, v and
    sigma = v W^T u^T, the gradient is (raw - <raw, W> / sigma u^T v) / sigma.  dout is the output itself, so that the correction is a third of
    the raw gradient's norm.  The sums of 640 000 products in 32 bits are off by about sqrt(n) w = 5e-5 of their terms: 2e-4 of the norm."""
    from ic_gan_amd import layers
    torch.manual_seed(0)
    m = layers.SNEmbedding(40000, 16).cuda().train()
    y = torch.randint(0, 300, (2000,), device="cuda")
    u0, w = m.u0.detach().double().clone(), m.weight.detach().double()
    out = m(y)
    d = out.detach().clone()
    out.backward(d)
    v = torch.nn.functional.normalize(u0 @ w, dim=1)
    u = torch.nn.functional.normalize(v @ w.t(), dim=1)
    sigma = float(v @ w.t() @ u.t())
    assert float((m.u0.double() - u).norm()) < 1e-5
    raw = torch.zeros(40000, 16, dtype=torch.float64, device="cuda").index_add_(0, y, d.double())
    correction = float((raw * w).sum()) / sigma * (u.t() @ v)
    want = (raw - correction) / sigma
    assert float(correction.norm()) > 0.2 * float(raw.norm())
    assert float((m.weight.grad.double() - want).norm()) <= 2e-4 * float(want.norm())


@pytest.mark.parametrize("V,D,n,kind", [(70000, 128, 1024, "same"), (10, 4095, 1024, "uniform"), (5, 4096, 1024, "same")])
def test_gradient_of_few_tokens_that_repeat(V, D, n, kind):
    """up to 1024 tokens are not sorted: no cliff to 1025, which are (0.3, 2.2 and 4.5 ms when one wave took a whole row, an entry at a time; 0.01 to
    0.09 now, 0.02 sorted)"""
    from ic_gan_amd import ops

    def best(count):
        idx = torch.full((count,), 3, device="cuda") if kind == "same" else torch.randint(0, V, (count,), device="cuda")
        d = torch.randint(-4, 5, (count, D), device="cuda").float()
        want = torch.zeros(V, D, device="cuda").index_add_(0, idx, d)
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            got = ops.embedding_backward(idx, d, V)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        assert torch.equal(got, want)                            # (whole numbers: exact)
        return min(times)
    assert best(n) <= 2 * best(n + 1) + 0.5                      # (ms)
