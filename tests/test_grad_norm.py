"""Global gradient norm and clipping (hsidm_grad_norm / hsidm_scale_tensors / hsidm_adam_step_clipped, train_ops.grad_norm /
clip_coef / clip_grad_norm_, Trainer(max_grad_norm=...)) against 64-bit formulas; refusals and the step's orchestration on the CPU."""
import ctypes
import math

import pytest
import torch

import cpu_double

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_refusals_without_a_gpu():
    from hsi_dmgasr_amd import _lib
    from hsi_dmgasr_amd import train_ops as T
    L = _lib.lib()
    item = (_lib.TensorItem * 1)()
    out = ctypes.c_void_p(64)                                       # never read: every call below is refused on the host
    assert L.hsidm_grad_norm_workspace_bytes(-1) == -1
    assert L.hsidm_grad_norm(item, -1, 1.0, 1.0, out, out, None) == -1
    assert L.hsidm_grad_norm(None, 1, 1.0, 1.0, out, out, None) == -1
    assert L.hsidm_grad_norm(item, 0, 1.0, 1.0, None, out, None) == -1
    assert L.hsidm_grad_norm(item, 0, 1.0, 0.0, out, out, None) == -1
    assert L.hsidm_grad_norm(item, 0, 1.0, float("nan"), out, out, None) == -1
    item[0].ptr, item[0].n, item[0].type = 64, 4, 9                 # unknown type
    assert L.hsidm_grad_norm(item, 1, 1.0, 1.0, out, out, None) == -1
    item[0].type, item[0].ptr = _lib.F32X3, 66                      # fp32 at an odd address
    assert L.hsidm_grad_norm(item, 1, 1.0, 1.0, out, out, None) == -1
    item[0].ptr, item[0].n = 64, -1
    assert L.hsidm_scale_tensors(item, 1, out, None) == -1
    assert L.hsidm_scale_tensors(item, 0, None, None) == -1
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.grad_norm([torch.zeros(3)])
    with pytest.raises(TypeError):
        T.TensorList([3.0])


def test_dense_layouts():
    from hsi_dmgasr_amd.train_ops import _is_dense
    x = torch.zeros(4, 6, 3, 3)
    assert _is_dense(x) and _is_dense(x.permute(2, 0, 3, 1)) and _is_dense(x.contiguous(memory_format=torch.channels_last))
    assert _is_dense(torch.zeros(())) and _is_dense(torch.zeros(5)[2:]) and _is_dense(x[1:2])
    assert not _is_dense(x[:, ::2]) and not _is_dense(x[:, :, :, :2]) and not _is_dense(torch.zeros(3, 1).expand(3, 4))


def test_trainer_clips_ahead_of_adam(monkeypatch):
    """Trainer(max_grad_norm): three steps against torch.optim.Adam behind torch.nn.utils.clip_grad_norm_ on the same gradients."""
    from hsi_dmgasr_amd import train_ops
    from test_train_orchestration import build, synth_tensor
    cpu_double.install(monkeypatch)

    def clip_coef(t, max_norm, grad_scale=1.0):
        n = t.double().norm() * grad_scale
        return torch.stack([n, (max_norm / (n + 1e-6)).clamp(max=1.0)]).float()

    def adam_step(p, g, m, v, *a, clip=None, **kw):
        return cpu_double.adam_step(p, g if clip is None else g * clip[1], m, v, *a, **kw)

    monkeypatch.setattr(train_ops, "clip_coef", clip_coef)
    monkeypatch.setattr(train_ops, "adam_step", adam_step)
    cfg, sd, gd, tr = build("tiny", "l1", False)
    data = {k: torch.from_numpy(synth_tensor("clip.%s" % k, (2, 3, 16, 16))) for k in ("HR", "SR")}
    noise, gamma = torch.from_numpy(synth_tensor("clip.noise", (2, 3, 16, 16))), torch.tensor([0.6, 0.2])
    tr.loss_and_grads(data, noise=noise, gamma=gamma)
    bound = 0.3 * float(tr.grad.norm())                             # every step below clips
    tr.max_grad_norm = bound
    ref = [torch.nn.Parameter(p.detach().clone()) for p in tr.net.parameters()]
    opt = torch.optim.Adam(ref, lr=1e-3)
    for _ in range(3):
        tr.loss_and_grads(data, noise=noise, gamma=gamma)
        for r, p in zip(ref, tr.net.parameters()):
            r.grad = tr.G(p).detach().clone()
        want = torch.nn.utils.clip_grad_norm_(ref, bound)
        opt.step()
        tr.optimizer_step()
        assert abs(float(tr.last_grad_norm) - float(want)) < 1e-5 * float(want) and float(want) > bound
        for r, p in zip(ref, tr.net.parameters()):
            assert float((r - p).detach().abs().max()) < 2e-5      # Adam moves by lr = 1e-3 at most
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_grad_norm"):
            tr.max_grad_norm = bad


# ------------------------------------------------------------------------------------------------------------------- GPU
def tensors_of(dev, seed=0):
    """Sizes from none to several runs of a workgroup, views at odd offsets, a channels-last and a transposed one, all three types."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate([1, 0, 3, 7, 4096, 4097, 65535, 300001, 2 ** 20 + 5]):
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            buf = torch.randn(n + 9, generator=g).to(dt).to(dev)
            out.append(buf[i % 5:i % 5 + n])
    out.append(torch.randn(8, 5, 3, 3, generator=g).to(dev).contiguous(memory_format=torch.channels_last))
    out.append(torch.randn(33, 65, generator=g).to(dev).t())
    return out


@GPU
@pytest.mark.parametrize("which", ["mixed", "many", "one", "empty"])
def test_norm(dev, which):
    from hsi_dmgasr_amd import train_ops as T
    ts = {"mixed": lambda: tensors_of(dev), "many": lambda: [torch.randn(1 + 37 * (i % 50), device=dev) for i in range(300)],
          "one": lambda: torch.randn(5_000_011, device=dev), "empty": lambda: [torch.zeros(0, device=dev), None]}[which]()
    want = norm64([ts] if torch.is_tensor(ts) else [t for t in ts if t is not None])
    got = T.grad_norm(ts)
    assert got.shape == () and got.dtype == torch.float32
    # 64-bit squares and sums: the one rounding is the result's, half a step of fp32 (and a 64-bit sum's 1e-12)
    assert abs(float(got) - want) <= (half_step(torch.float32) + 1e-12) * want
    assert torch.equal(got, T.grad_norm(ts))
    assert abs(float(T.grad_norm(ts, grad_scale=0.125)) - want / 8) <= (half_step(torch.float32) + 1e-12) * want


@GPU
@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1e-44])
def test_norm_neither_overflows_nor_underflows(dev, value):
    from hsi_dmgasr_amd import train_ops as T
    t = torch.full((777,), value, device=dev)
    want = float(t[0]) * math.sqrt(777)
    got = float(T.grad_norm([t]))
    if want > torch.finfo(torch.float32).max:
        assert got == math.inf
    else:
        assert abs(got - want) <= half_step(torch.float32) * want + 2.0 ** -150


@GPU
@pytest.mark.parametrize("bound", [0.37, 1e9])
def test_clip_in_place(dev, bound):
    from hsi_dmgasr_amd import train_ops as T
    ts = tensors_of(dev, 1)
    before = [t.clone() for t in ts]
    whole = [t.untyped_storage() for t in ts]
    around = [torch.empty(0, dtype=torch.uint8, device=dev).set_(s).clone() for s in whole]
    versions = [t._version for t in ts]
    norm = T.clip_grad_norm_(ts, bound)
    want = norm64(before)
    assert abs(float(norm) - want) <= (half_step(torch.float32) + 1e-12) * want
    c = min(1.0, bound / (want + 1e-6))
    for t, b, s, a, ver in zip(ts, before, whole, around, versions):
        if c == 1.0:
            assert torch.equal(t, b)
        # the coefficient's and the product's rounding in fp32, the store's in the tensor's type (fp16 / fp32: half a subnormal step)
        tol = b.double().abs() * c * (2 * half_step(torch.float32) + half_step(t.dtype)) * 1.01 + torch.finfo(t.dtype).smallest_normal * half_step(t.dtype) * 2
        assert bool(((t.double() - b.double() * c).abs() <= tol).all())
        assert t._version > ver
        after = torch.empty(0, dtype=torch.uint8, device=dev).set_(s).clone()      # bytes beside the view keep their values
        off, n = t.storage_offset() * t.element_size(), t.numel() * t.element_size()
        assert torch.equal(after[:off], a[:off]) and torch.equal(after[off + n:], a[off + n:])


@GPU
def test_clip_with_infinite_and_nan_gradients(dev):
    from hsi_dmgasr_amd import train_ops as T
    a, b = torch.ones(1000, device=dev), torch.ones(5, device=dev)
    b[2] = math.inf
    assert T.clip_coef([a, b], 1.0).tolist() == [math.inf, 0.0]
    T.clip_grad_norm_([a, b], 1.0)                                  # as torch: 0 * inf is NaN, everything else 0
    assert bool((a == 0).all()) and bool(torch.isnan(b[2])) and float(b[0]) == 0
    b[2] = math.nan
    assert all(math.isnan(v) for v in T.clip_coef([a, b], 1.0).tolist())
    assert math.isnan(float(T.grad_norm([b])))


@GPU
def test_clip_refusals(dev):
    from hsi_dmgasr_amd import train_ops as T
    x = torch.zeros(64, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        T.clip_grad_norm_([x, x], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        T.clip_grad_norm_([x[:33], x[32:]], 1.0)
    T.clip_grad_norm_([x[:32], x[32:]], 1.0)
    w = torch.nn.Parameter(torch.ones(5, device=dev))
    with pytest.raises(ValueError, match="p.grad"):
        T.clip_grad_norm_([w], 1.0)
    assert bool((w == 1).all())
    with pytest.raises(ValueError, match="dense"):
        T.grad_norm([x.view(8, 8)[:, :4]])
    with pytest.raises(TypeError):
        T.grad_norm([x.long()])
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.grad_norm([x, torch.zeros(3)])
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="positive"):
            T.clip_coef([x], bad)
    with pytest.raises(ValueError, match="clip"):
        T.adam_step(x, x.clone(), x.clone(), x.clone(), 1e-3, 0.9, 0.99, 1e-8, 1, clip=x)


@GPU
def test_list_follows_new_storage(dev):
    from hsi_dmgasr_amd import train_ops as T
    x = torch.ones(100, device=dev)
    tl = T.TensorList([x])
    assert float(T.grad_norm(tl)) == 10.0
    x.data = torch.full((400,), 2.0, device=dev)
    assert float(T.grad_norm(tl)) == 40.0
    x.data = torch.ones(7)
    with pytest.raises(RuntimeError, match="ROCm device"):
        T.grad_norm(tl)


@GPU
@pytest.mark.parametrize("n", [1, 5, 4099, 1_000_003])
def test_clipped_adam_step(dev, n):
    """adam_step(clip=clip_coef(g)) = the Adam formula in 64 bits on the clipped gradient."""
    from hsi_dmgasr_amd import train_ops as T
    g = torch.Generator().manual_seed(n)
    p, gr, m, v = (torch.randn(n, generator=g).to(dev) for _ in range(4))
    v = v.square() + 1e-3
    p0, m0, v0 = p.double(), m.double(), v.double()
    bound = 0.25 * norm64([gr])
    clip = T.clip_coef(gr, bound)
    T.adam_step(p, gr, m, v, 1e-2, 0.9, 0.99, 1e-8, 3, clip=clip)
    gd = gr.double() * min(1.0, bound / (norm64([gr]) + 1e-6))
    m1, v1 = 0.9 * m0 + 0.1 * gd, 0.99 * v0 + 0.01 * gd * gd
    p1 = p0 - 1e-2 * (m1 / (1 - 0.9 ** 3)) / ((v1 / (1 - 0.99 ** 3)).sqrt() + 1e-8)
    # a handful of fp32 roundings per value; 1 - beta in fp32 is off by up to 2^-24 / (1 - beta) = 6e-6 relative at 0.99
    tol = 16 * half_step(torch.float32)
    assert bool(((m.double() - m1).abs() <= tol * (m0.abs() + gd.abs())).all())
    assert bool(((v.double() - v1).abs() <= (tol + 1e-5) * v1).all())
    assert bool(((p.double() - p1).abs() <= tol * p0.abs() + 1e-2 * 2e-5 * (1 + (m1 / v1.sqrt()).abs())).all())
    # without clipping: the same bits as the plain step
    a, b = [x.clone() for x in (p, m, v)], [x.clone() for x in (p, m, v)]
    T.adam_step(a[0], gr, a[1], a[2], 1e-2, 0.9, 0.99, 1e-8, 4)
    T.adam_step(b[0], gr, b[1], b[2], 1e-2, 0.9, 0.99, 1e-8, 4, clip=T.clip_coef(gr, 1e9))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@GPU
def test_captured_clip_and_another_stream(dev):
    """One graph of norm + scaling, replayed with new gradients and eager work in between; an eager call on a second stream."""
    from hsi_dmgasr_amd import train_ops as T
    src = [torch.randn(n, device=dev) for n in (5, 70001, 1024)]
    ts = [torch.empty_like(s) for s in src]
    tl = T.TensorList(ts)
    T.clip_grad_norm_(tl, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = T.clip_grad_norm_(tl, 1.0)
    for k in range(4):
        for t, s in zip(ts, src):
            t.copy_(s * (k + 1))
        want_n = T.grad_norm(ts).clone()
        want = [t * T.clip_coef(ts, 1.0)[1] for t in ts]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want_n)
        assert all(torch.equal(t, w) for t, w in zip(ts, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = T.grad_norm(src)
    side.synchronize()
    assert torch.equal(other, T.grad_norm(src))


@GPU
def test_trainer_with_clipping_on_the_device(dev):
    """Eager and captured training steps with max_grad_norm: the reported norm is the gradient's, and the update is the clipped one."""
    from gpu_util import fill_synth
    from hsi_dmgasr_amd import train_ops as T
    from hsi_dmgasr_amd.sr3_modules import diffusion, unet
    from helpers import synth_tensor
    u = unet.UNet(in_channel=6, out_channel=3, inner_channel=32, channel_mults=[1, 2], attn_res=[8], res_blocks=1, image_size=16,
                  precision="fp32").to(dev).train()
    fill_synth(u, "clip.")
    gd = diffusion.GaussianDiffusion(u, image_size=16, channels=3, conditional=True)
    gd.set_loss(dev)
    gd.set_new_noise_schedule(dict(schedule="cosine", n_timestep=20, linear_start=1e-6, linear_end=1e-2), dev)
    tr = gd.trainer(lr=1e-3, max_grad_norm=0.05)
    data = {k: torch.from_numpy(synth_tensor("clip.%s" % k, (2, 3, 16, 16))).to(dev) for k in ("HR", "SR")}
    for i in range(5):                                              # step 0 eager, step 1 captures, then replays
        if i == 4:
            tr.max_grad_norm = 1e6                                  # captures again, does not clip any more
        p, m, v = tr.flat.clone(), tr.m.clone(), tr.v.clone()
        tr.optimize_parameters(data)
        want = norm64([tr.grad])
        assert abs(float(tr.last_grad_norm) - want) <= 1e-6 * want
        T.adam_step(p, tr.grad, m, v, tr.lr, *tr.betas, tr.eps, tr.step_count, clip=T.clip_coef(tr.grad, tr.max_grad_norm))
        # (a captured step reads its bias corrections as two fp32 words: one rounding more)
        assert float((p - tr.flat).abs().max()) <= 1e-3 * 1e-5 + 2.0 ** -23 * float(p.abs().max())
        assert torch.equal(m, tr.m) and torch.equal(v, tr.v)


@GPU
def test_more_than_32_bits_of_elements(dev):
    """One tensor of 2^31 + 5 elements among small ones, to the last element (its value and half of it are powers of two)."""
    from hsi_dmgasr_amd import train_ops as T
    n = 2 ** 31 + 5
    big = torch.full((n,), 2.0 ** -15, device=dev, dtype=torch.bfloat16)
    small = torch.zeros(3, device=dev)
    want = 2.0 ** -15 * math.sqrt(n)
    assert abs(float(T.grad_norm([small, big])) - want) <= (half_step(torch.float32) + 1e-12) * want
    T.clip_grad_norm_([small, big], want / 2 + 1e-6)                # (the coefficient is within 1e-5 of a half; bf16 keeps eight bits)
    assert float(big[-1]) == 2.0 ** -16 and float(big[0]) == 2.0 ** -16 and float(big[2 ** 30]) == 2.0 ** -16


@GPU
def test_clip_of_inference_tensors(dev):
    from hsi_dmgasr_amd import train_ops as T
    with torch.inference_mode():
        x = torch.full((4,), 3.0, device=dev)
        assert float(T.clip_grad_norm_([x], 3.0)) == 6.0
        assert abs(float(x[0]) - 1.5) < 1e-6
