"""Norm of queries and keys with the multi-axis rotation (ops.qk_norm_rope, train_ops.qk_norm_rope_bwd) against 64-bit formulas."""
import ctypes
import math

import pytest
import torch

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def plain64(x, w, pos, sections, eps, base=10000.0):
    """The definition in 64 bits (differentiable): x [T, H, D]."""
    half = x.shape[-1] // 2
    angle = torch.zeros(pos.shape[0], half, dtype=torch.float64, device=x.device)
    p = 0
    for a, n in enumerate(sections):
        for j in range(n):
            angle[:, p] = pos[:, a].double() * base ** (-j / n)
            p += 1
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    n = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    a, b = n[..., :half], n[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def inputs(dev, T, hq, hk, D, axes, dtype, seed=0, spread=200):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k = (3 * r(T, hq, D)).to(dtype).to(dev), (0.2 * r(T, hk, D)).to(dtype).to(dev)
    wq, wk = (1 + 0.3 * r(D)).to(dev), (1 + 0.3 * r(D)).to(dev)
    pos = torch.randint(-spread, spread + 1, (T, axes), generator=g, dtype=torch.int32).to(dev)
    return q, k, wq, wk, pos


def close(got, want, terms=1.0):
    """Element by element.  The store's rounding (half a step of the type, or of its subnormals) and some fp32 roundings on the way:
    `terms` times 32 half-steps of fp32 on the row's largest value (a rotated value is the difference of two that large)."""
    dt = got.dtype
    top = want.abs().amax(-1, keepdim=True)
    tol = want.abs() * torch.finfo(dt).eps / 2 * 1.01 + terms * 32 * torch.finfo(torch.float32).eps / 2 * top + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    worst = float(((got.double() - want).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, worst


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_refusals_without_a_gpu():
    from hsi_dmgasr_amd import _lib, ops
    L = _lib.lib()
    D = 64
    axes = ops.RotaryAxes((8, 12, 12), D, device="cpu")
    assert axes.freq.dtype == torch.float64 and abs(float(axes.freq[9]) * 2 * math.pi - 10000.0 ** (-1 / 12)) < 1e-15
    q, k, w, pos = torch.zeros(4, 2, D), torch.zeros(4, 1, D), torch.ones(D), torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.qk_norm_rope(q, k, w, w, pos, axes)
    for bad in (dict(q=q[:3]), dict(k=k[..., :32]), dict(wq=w.double()), dict(wk=w[:32]), dict(pos=pos.long()), dict(pos=pos[:, :2]), dict(eps=-1.0),
                dict(eps=math.nan), dict(q=q[0])):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(**{**dict(q=q, k=k, wq=w, wk=w, pos=pos, axes=axes), **bad})
    for bad in (dict(k=k.half()), dict(q=q.double(), k=k.double())):
        with pytest.raises(TypeError):
            ops.qk_norm_rope(**{**dict(q=q, k=k, wq=w, wk=w, pos=pos, axes=axes), **bad})
    for bad in (((40,), 64), ((8,), 24), ((8,), 272), ((-1, 4), 64), ((), 64), ((1,) * 5, 64)):
        with pytest.raises(ValueError):
            ops.RotaryAxes(*bad, device="cpu")
    with pytest.raises(ValueError, match="base"):
        ops.RotaryAxes((8,), 64, base=1.0, device="cpu")

    def desc(**kw):
        d = _lib.RopeDesc()
        vals = dict(q=64, k=64, wq=64, wk=64, pos=64, freq=64, q_ts=128, q_hs=64, k_ts=64, k_hs=64, T=4, Hq=2, Hk=1, D=64, axes=1, prec=_lib.F16, eps=1e-6)
        for n, v in {**vals, **kw}.items():
            setattr(d, n, v)
        d.sections[0] = kw.get("s0", 8)
        return ctypes.byref(d)

    one = ctypes.c_void_p(64)
    assert L.hsidm_qk_norm_rope(None, one, one, None) == -1
    for bad in (dict(T=0), dict(D=24), dict(D=512), dict(Hq=0), dict(axes=5), dict(axes=0), dict(s0=33), dict(s0=-1), dict(prec=7), dict(q=72), dict(q_hs=63),
                dict(eps=-1.0), dict(freq=None), dict(wq=68)):
        assert L.hsidm_qk_norm_rope(desc(**bad), one, one, None) == -1, bad
        assert L.hsidm_qk_norm_rope_bwd_workspace_bytes(desc(**bad)) == -1, bad
    assert L.hsidm_qk_norm_rope(desc(), None, one, None) == -1
    need = L.hsidm_qk_norm_rope_bwd_workspace_bytes(desc())
    assert need > 0 and need % (2 * 64 * 4) == 0
    assert L.hsidm_qk_norm_rope_bwd(desc(), one, one, one, 128, 64, one, 64, 64, one, one, one, need - 1, None) == -1
    assert L.hsidm_qk_norm_rope_bwd(desc(), one, one, one, 128, 63, one, 64, 64, one, one, one, need, None) == -1


# ------------------------------------------------------------------------------------------------------------------- GPU
CASES = [  # T, hq, hk, D, sections
    (1, 1, 1, 64, (32,)), (64, 4, 4, 64, (16, 16)), (1000, 8, 2, 64, (8, 12, 12)), (37, 3, 1, 80, (7, 13)), (515, 2, 2, 256, (20, 40, 60)),
    (5, 40, 8, 128, (64,)), (260, 1, 1, 16, (3,)), (9, 2, 1, 32, (0, 16)), (130, 16, 4, 96, (1, 2, 3, 4)), (40001, 1, 1, 32, (8, 8)), (33, 1, 1, 64, (0,)),
]


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(dev, case, dtype):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    T, hq, hk, D, sections = case
    q, k, wq, wk, pos = inputs(dev, T, hq, hk, D, len(sections), dtype)
    axes = ops.RotaryAxes(sections, D, device=dev)
    oq, ok = ops.qk_norm_rope(q, k, wq, wk, pos, axes)
    g = torch.Generator().manual_seed(5)
    dq_, dk_ = torch.randn(T, hq, D, generator=g).to(dtype).to(dev), torch.randn(T, hk, D, generator=g).to(dtype).to(dev)
    grads = Tr.qk_norm_rope_bwd(dq_, dk_, q, k, wq, wk, pos, axes)
    again = Tr.qk_norm_rope_bwd(dq_, dk_, q, k, wq, wk, pos, axes)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for x, w, o, do, dx, dw in ((q, wq, oq, dq_, grads[0], grads[2]), (k, wk, ok, dk_, grads[1], grads[3])):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y = plain64(x64, w64, pos, sections, 1e-6)
        close(o, y.detach())
        y.backward(do.double())
        close(dx, x64.grad, terms=4)
        # sums of T * heads products in fp32 along a lane, then in order over the workgroups: the worst of a serial sum, n half-steps of
        # the sum of magnitudes, holds with room; random signs leave far less
        mag = (plain64(x.double().abs(), w.double().abs() * 0 + 1, pos * 0, sections, 1e-6)).abs().mul(do.double().abs().amax()).sum((0, 1))
        assert bool(((dw.double() - w64.grad).abs() <= 64 * 2.0 ** -24 * mag + 1e-30).all())


@GPU
@pytest.mark.parametrize("T, D", [(1, 16), (5, 64), (67, 48), (3, 256)])
def test_no_eps(dev, T, D):
    """eps = 0 is allowed where no row is zero: the lanes behind the last token, which hold zeros, must not reach the weights' gradients."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    q, k, wq, wk, pos = inputs(dev, T, 2, 1, D, 1, torch.float32, seed=4)
    axes = ops.RotaryAxes((D // 4,), D, device=dev)
    outs = ops.qk_norm_rope(q, k, wq, wk, pos, axes, eps=0.0)
    g = torch.Generator().manual_seed(9)
    do = torch.randn(T, 2, D, generator=g).to(dev), torch.randn(T, 1, D, generator=g).to(dev)
    grads = Tr.qk_norm_rope_bwd(*do, q, k, wq, wk, pos, axes, eps=0.0)
    for x, w, o, d, dx, dw in ((q, wq, outs[0], do[0], grads[0], grads[2]), (k, wk, outs[1], do[1], grads[1], grads[3])):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y = plain64(x64, w64, pos, (D // 4,), 0.0)
        close(o, y.detach())
        y.backward(d.double())
        close(dx, x64.grad, terms=4)
        mag = plain64(x.double().abs(), torch.ones_like(w64), pos * 0, (D // 4,), 0.0).mul(d.double().abs().amax()).sum((0, 1))
        assert bool(((dw.double() - w64.grad).abs() <= 64 * 2.0 ** -24 * mag + 1e-30).all())        # (the bound of test_forward_and_backward)


@GPU
def test_gradient_against_differences(dev):
    """d loss / d x along random directions, by central differences of the forward kernel in fp32 (loss = sum of out * do)."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    T, hq, hk, D, sections = 50, 2, 1, 64, (16, 16)
    q, k, wq, wk, pos = inputs(dev, T, hq, hk, D, 2, torch.float32, seed=3)
    axes = ops.RotaryAxes(sections, D, device=dev)
    g = torch.Generator().manual_seed(8)
    dq_, dk_ = torch.randn(T, hq, D, generator=g).to(dev), torch.randn(T, hk, D, generator=g).to(dev)
    dq, dk, dwq, dwk = Tr.qk_norm_rope_bwd(dq_, dk_, q, k, wq, wk, pos, axes)

    def loss(q, k, wq, wk):
        oq, ok = ops.qk_norm_rope(q, k, wq, wk, pos, axes)
        return float((oq.double() * dq_).sum() + (ok.double() * dk_).sum())

    for args in ((q, dq, 0), (k, dk, 1), (wq, dwq, 2), (wk, dwk, 3)):
        x, gx, i = args
        u = torch.randn(x.shape, generator=g).to(dev)
        h = 1e-2 * float(x.abs().mean())
        full = [q, k, wq, wk]
        lo, hi = list(full), list(full)
        lo[i], hi[i] = x - h * u, x + h * u
        want = float((gx.double() * u).sum())
        scale = float((gx.double() * u).abs().sum())
        assert abs((loss(*hi) - loss(*lo)) / (2 * h) - want) < 2e-3 * scale      # the difference's own error is h^2 = 1e-4 of the curvature


@GPU
@pytest.mark.parametrize("spread", [70_000, 2 ** 31 - 1])
def test_far_positions_keep_their_angle(dev, spread):
    from hsi_dmgasr_amd import ops
    q, k, wq, wk, pos = inputs(dev, 300, 2, 1, 64, 2, torch.float32, spread=min(spread, 2 ** 31 - 2))
    axes = ops.RotaryAxes((16, 16), 64, device=dev)
    oq, _ = ops.qk_norm_rope(q, k, wq, wk, pos, axes)
    want = plain64(q.double(), wq.double(), pos, (16, 16), 1e-6)
    # angles up to 2^31 radians: the 64-bit products of either side are off by 2^31 * 2^-52 = 5e-7
    assert float((oq.double() - want).abs().max()) <= (5e-6 if spread > 1e6 else 4e-6) * float(want.abs().max())


@GPU
@pytest.mark.parametrize("layout", ["slices", "odd offset", "transposed", "expanded"])
def test_layouts(dev, layout):
    """Views of one projection's output are read in place; rows off the 16-byte boundary and broadcast heads through a copy."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    T, D, dtype = 77, 64, torch.bfloat16
    x = torch.randn(T * 8 * D + 3, device=dev).to(dtype)
    both = x[:T * 8 * D].view(T, 8, D)
    q, k = {"slices": (both[:, :4], both[:, 4:6]), "odd offset": (x[3:].view(T, 8, D)[:, :4], x[1:1 + T * 2 * D].view(T, 2, D)),
            "transposed": (both.transpose(1, 2).contiguous().transpose(1, 2)[:, :4], x[:2 * T * D].view(2, T, D).transpose(0, 1)),
            "expanded": (both[:, :1].expand(T, 4, D), both[:1, :2].expand(T, 2, D))}[layout]
    w = torch.rand(D + 1, device=dev)[1:]
    pos = torch.arange(2 * T, device=dev, dtype=torch.int32).view(2, T).t()
    axes = ops.RotaryAxes((16, 16), D, device=dev)
    got = ops.qk_norm_rope(q, k, w, w, pos, axes)
    want = ops.qk_norm_rope(q.clone(memory_format=torch.contiguous_format), k.clone(memory_format=torch.contiguous_format), w.clone(), w.clone(), pos.contiguous(), axes)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    room = torch.full((T, 3 * 8, D), 7.0, device=dev, dtype=dtype)
    out = (room[:, 1:5], room[:, 9:11])
    d = (torch.randn(T, 4, 2 * D, device=dev).to(dtype)[..., ::2], torch.randn(T, 2, D, device=dev).to(dtype))
    a = Tr.qk_norm_rope_bwd(*d, q, k, w, w, pos, axes, out=out)
    b = Tr.qk_norm_rope_bwd(*d, q, k, w, w, pos, axes)
    assert all(torch.equal(u, v) for u, v in zip(a, b)) and a[0].data_ptr() == out[0].data_ptr()
    assert bool((room[:, 0] == 7).all()) and bool((room[:, 5:9] == 7).all()) and bool((room[:, 11:] == 7).all())
    with pytest.raises(ValueError, match="out"):
        Tr.qk_norm_rope_bwd(*d, q, k, w, w, pos, axes, out=(torch.empty(T, 4, 2 * D, device=dev, dtype=dtype)[..., ::2], out[1]))
    with pytest.raises(ValueError, match="gradient"):
        Tr.qk_norm_rope_bwd(d[0].float(), d[1], q, k, w, w, pos, axes)


@GPU
def test_no_tokens_and_special_values(dev):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    axes = ops.RotaryAxes((16, 16), 64, device=dev)
    w = torch.ones(64, device=dev)
    e = torch.empty(0, 2, 64, device=dev)
    oq, ok = ops.qk_norm_rope(e, e, w, w, torch.empty(0, 2, device=dev, dtype=torch.int32), axes)
    assert oq.shape == e.shape and ok.shape == e.shape
    g = Tr.qk_norm_rope_bwd(e, e, e, e, w, w, torch.empty(0, 2, device=dev, dtype=torch.int32), axes)
    assert g[0].shape == e.shape and bool((g[2] == 0).all()) and bool((g[3] == 0).all())
    q = torch.randn(3, 2, 64, device=dev)
    q[0, 0] = 0.0                                                   # a zero row stays zero (eps keeps the root finite)
    q[1, 1, 5] = math.nan                                           # and a NaN stays in its own row
    oq, _ = ops.qk_norm_rope(q, q, w, w, torch.ones(3, 2, device=dev, dtype=torch.int32), axes)
    assert bool((oq[0, 0] == 0).all()) and bool(torch.isnan(oq[1, 1]).all())
    assert not bool(torch.isnan(oq[1, 0]).any()) and not bool(torch.isnan(oq[[0, 2]]).any())


@GPU
def test_captured_and_on_another_stream(dev):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    q, k, wq, wk, pos = inputs(dev, 333, 4, 2, 64, 2, torch.float16)
    axes = ops.RotaryAxes((16, 16), 64, device=dev)
    step = lambda: ops.qk_norm_rope(q, k, wq, wk, pos, axes) + Tr.qk_norm_rope_bwd(q, k, q, k, wq, wk, pos, axes)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        q.add_(0.25); pos.add_(3)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


@GPU
def test_offsets_beyond_32_bits(dev):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    T, H, D = 33000, 512, 128
    q = torch.randn(T, H, D, device=dev, dtype=torch.bfloat16)
    k = q[:, 7:9]
    w = torch.rand(D, device=dev) + 0.5
    pos = torch.randint(0, 500, (T, 2), device=dev, dtype=torch.int32)
    axes = ops.RotaryAxes((32, 32), D, device=dev)
    oq, ok = ops.qk_norm_rope(q, k, w, w, pos, axes)
    lq, lk = ops.qk_norm_rope(q[-5:].clone(), k[-5:].clone(), w, w, pos[-5:].contiguous(), axes)
    assert torch.equal(oq[-5:], lq) and torch.equal(ok[-5:], lk)
    g = Tr.qk_norm_rope_bwd(oq, ok, q, k, w, w, pos, axes)
    g1 = Tr.qk_norm_rope_bwd(lq, lk, q[-5:].clone(), k[-5:].clone(), w, w, pos[-5:].contiguous(), axes)
    assert torch.equal(g[0][-5:], g1[0]) and torch.equal(g[1][-5:], g1[1])
