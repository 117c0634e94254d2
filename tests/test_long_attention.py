"""The operators together, as a network uses them: self-attention over maps of more than 1024 tokens, with and without the norm and rotation
of queries and keys, in inference and in the training step with gradient clipping - against the oracle (autograd over torch formulas)."""
import math

import pytest
import torch
import torch.nn.functional as F

import cpu_double
from gpu_util import check, fill_synth
from helpers import synth_tensor

GPU = pytest.mark.gpu
# 48 x 48 = 2304 tokens at the first level (heads of 32 channels), 24 x 24 at the second
CFG = dict(in_channel=6, out_channel=3, inner_channel=32, norm_groups=32, channel_mults=[1, 2], attn_res=[48], res_blocks=1, image_size=48)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def rotate(x, heads, rows, cols):
    """The rotation by (row, column) as a formula: x [B, heads, N, D], half of the pairs with either axis."""
    D = x.shape[-1]
    q = D // 4
    f = 10000.0 ** (-torch.arange(q, dtype=torch.float64) / q)
    n = torch.arange(rows * cols)
    angle = torch.cat([(n // cols).double()[:, None] * f, (n % cols).double()[:, None] * f], 1)
    c, s = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def oracle_attention(n_head=1, fp=torch.float32):
    """sr3_unet.self_attention with heads and, where the state dict has the norms' weights, norm and rotation."""
    def attention(sd, prefix, x, groups):
        b, c, hh, ww = x.shape
        n = F.group_norm(x, groups, sd[prefix + "norm.weight"], sd[prefix + "norm.bias"], eps=1e-5)
        qkv = F.conv2d(n, sd[prefix + "qkv.weight"])
        q, k, v = qkv.reshape(b, n_head, 3, c // n_head, hh * ww).permute(2, 0, 1, 4, 3).unbind(0)        # [b, head, N, D]
        if prefix + "q_norm" in sd:
            norm = lambda t, w: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w  # noqa: E731
            q, k = (rotate(norm(t, sd[prefix + w]), n_head, hh, ww) for t, w in ((q, "q_norm"), (k, "k_norm")))
        p = torch.softmax(q @ k.transpose(2, 3).contiguous() / math.sqrt(c), dim=-1)
        o = (p @ v.contiguous()).permute(0, 1, 3, 2).reshape(b, c, hh, ww)
        return F.conv2d(o, sd[prefix + "out.weight"], sd[prefix + "out.bias"]) + x
    return attention


def packed_doubles(monkeypatch):
    """CPU stand-ins of the packed operators beside cpu_double's (the formulas through autograd)."""
    from hsi_dmgasr_amd import ops, train_ops

    def rope(q, k, wq, wk, pos, axes, eps=1e-6):
        def one(x, w):
            x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
            p, half = axes.freq.numel(), x.shape[-1] // 2
            ax = torch.repeat_interleave(torch.arange(len(axes.sections)), torch.tensor(axes.sections))
            a = (pos.double()[:, ax] * axes.freq * 2 * math.pi)[:, None].to(x.dtype)
            u, v = x[..., :p], x[..., half:half + p]
            return torch.cat([u * a.cos() - v * a.sin(), x[..., p:half], u * a.sin() + v * a.cos(), x[..., half + p:]], -1)
        return one(q, wq), one(k, wk)

    def attn(q, k, v, seqs, causal=False, scale=None, want_lse=False):
        assert not causal
        o = torch.cat([(torch.softmax(scale * a.transpose(0, 1) @ b.permute(1, 2, 0), -1) @ c.transpose(0, 1)).transpose(0, 1)
                       for a, b, c in zip(*(t.split(list(seqs.lengths)) for t in (q, k, v)))])
        return (o, ops.AttentionSaved(None, None)) if want_lse else o

    def attn_bwd(do, q, k, v, out, saved, seqs, causal=False, scale=None, grads=None):
        with torch.enable_grad():
            x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
            attn(*x, seqs, scale=scale).backward(do)
        for g, t in zip(grads, x):
            g.copy_(t.grad)

    def rope_bwd(doq, dok, q, k, wq, wk, pos, axes, eps=1e-6, out=None):
        with torch.enable_grad():
            x = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
            oq, ok = rope(*x, pos, axes)
            ((oq * doq).sum() + (ok * dok).sum()).backward()
        out[0].copy_(x[0].grad)
        out[1].copy_(x[1].grad)
        return out[0], out[1], x[2].grad, x[3].grad

    monkeypatch.setattr(ops, "qk_norm_rope", rope)
    monkeypatch.setattr(ops, "attention_packed", attn)
    monkeypatch.setattr(train_ops, "attention_packed_bwd", attn_bwd)
    monkeypatch.setattr(train_ops, "qk_norm_rope_bwd", rope_bwd)


def network(rope, precision, dev="cpu", train=True):
    from hsi_dmgasr_amd.sr3_modules import diffusion, unet
    u = unet.UNet(precision=precision, attn_qk_norm_rope=rope, **CFG)
    sd = fill_synth(u, "long.")
    for m in u.modules():                                           # (a norm's weight around one, not around zero)
        if isinstance(m, unet.SelfAttention) and rope:
            with torch.no_grad():
                m.q_norm.add_(1.0)
                m.k_norm.add_(1.0)
    sd = {k: v.detach().clone() for k, v in u.state_dict().items()}
    u.to(dev).train(train)
    gd = diffusion.GaussianDiffusion(u, image_size=48, channels=3, loss_type="l2", conditional=True)
    gd.set_loss(dev)
    gd.set_new_noise_schedule(dict(schedule="cosine", n_timestep=20, linear_start=1e-6, linear_end=1e-2), dev)
    return u, sd, gd


def batch():
    hr, sr, noise = (torch.from_numpy(synth_tensor("long.%s" % n, (2, 3, 48, 48))) for n in ("hr", "sr", "noise"))
    return hr, sr, noise, torch.tensor([0.8, 0.3])


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_module_arguments():
    from hsi_dmgasr_amd.sr3_modules import unet
    a = unet.SelfAttention(64, n_head=2, qk_norm_rope=True)
    assert a.q_norm.shape == (32,) and set(dict(a.named_parameters())) == {"norm.weight", "norm.bias", "qkv.weight", "out.weight", "out.bias", "q_norm", "k_norm"}
    assert set(dict(unet.SelfAttention(64).named_parameters())) == {"norm.weight", "norm.bias", "qkv.weight", "out.weight", "out.bias"}
    assert a.packed(16) and not unet.SelfAttention(64).packed(1024) and unet.SelfAttention(64).packed(1025)
    for c, n in ((512, 1), (64, 8)):
        with pytest.raises(ValueError, match="qk_norm_rope"):
            unet.SelfAttention(c, n_head=n, qk_norm_rope=True)
    plan = a.map_plan(2, 3, 5, torch.device("cpu"))
    assert plan[0].lengths == (15, 15) and plan[1].shape == (30, 2) and plan[1][22].tolist() == [1, 2]
    q, k, v = a.heads(torch.arange(2 * 3 * 5 * 192).view(2, 3, 5, 192))
    assert q.shape == (30, 2, 32) and int(q[1, 1, 0]) == 192 + 96 and int(k[1, 1, 0]) == 192 + 96 + 32 and int(v[1, 0, 3]) == 192 + 64 + 3


@pytest.mark.parametrize("rope", [False, True])
def test_training_step_orchestration(monkeypatch, rope):
    """The gradient routing of the packed attention layers (with everything by torch doubles) against the oracle's autograd."""
    from hsi_dmgasr_amd import training
    from oracle import sr3_unet
    from oracle import train as otrain
    from test_train_orchestration import compare
    cpu_double.install(monkeypatch)
    packed_doubles(monkeypatch)
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention())

    class CpuTrainer(training.Trainer):
        def _check_device(self):
            pass

    u, sd, gd = network(rope, "fp32")
    tr = CpuTrainer(gd, lr=1e-3)
    hr, sr, noise, gamma = batch()
    loss = tr.loss_and_grads({"HR": hr, "SR": sr}, noise=noise, gamma=gamma)
    want, grads = otrain.loss_and_grads(sd, CFG, hr, sr, noise, gamma, "l2", 0.0, otrain.drop_key(0, 0))
    assert abs(float(loss) - want) < 1e-4 * abs(want)
    compare(tr, grads)
    assert sum(n.endswith(("q_norm", "k_norm")) for n in grads) == (8 if rope else 0)      # three layers at 48 x 48 (one down, two up) and mid


# ------------------------------------------------------------------------------------------------------------------- GPU
@GPU
@pytest.mark.parametrize("n_head", [1, 2])
@pytest.mark.parametrize("rope", [False, True], ids=["plain", "qk_norm_rope"])
@pytest.mark.parametrize("shape", [(2, 64, 40, 36), (1, 64, 33, 35), (3, 64, 8, 8)], ids=str)
def test_self_attention_module(dev, shape, rope, n_head):
    """The layer on maps beyond and below 1024 tokens, in the fp32 and the fp16 kernel sets."""
    from hsi_dmgasr_amd.sr3_modules import unet
    m = unet.SelfAttention(shape[1], n_head=n_head, qk_norm_rope=rope)
    fill_synth(m, "la%d." % n_head)
    sd = {k: v.detach().clone() for k, v in m.state_dict().items()}
    x = torch.from_numpy(synth_tensor("la.x", shape))
    want = oracle_attention(n_head)(sd, "", x, 32)
    m.to(dev).eval()
    for prec, tol in (("fp32", 1e-4), ("fp16x1", 1.5e-3)):          # the bounds of the same layer on small maps
        m.precision = prec
        from hsi_dmgasr_amd import ops
        with torch.no_grad():
            p = "fp32" if prec == "fp32" else "fp16x1"
            got = ops.to_nchw(m._run(ops.to_nhwc(x.to(dev), p), p), p)
        check("self_attention_packed%s" % (shape,), prec, got, want, tol=tol)


@GPU
@pytest.mark.parametrize("rope", [False, True], ids=["plain", "qk_norm_rope"])
def test_network_and_training_step(dev, rope, monkeypatch):
    """A UNet with attention over 2304 tokens: the forward pass, every gradient, and five optimiser steps with clipping (eager, then
    captured and replayed) whose reported norm is the gradient's."""
    from hsi_dmgasr_amd import train_ops
    from oracle import sr3_unet
    from oracle import train as otrain
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention())
    u, sd, gd = network(rope, "fp32", dev, train=False)
    hr, sr, noise, gamma = batch()
    x = torch.cat([sr, hr], 1)
    with torch.no_grad():
        got = u(x.to(dev), gamma.to(dev)[:, None])
        want = sr3_unet.unet_forward(sd, CFG, x, gamma[:, None])
    check("unet_long_attention", "fp32", got, want)
    u.train()
    tr = gd.trainer(lr=1e-4, max_grad_norm=0.02)
    data = {"HR": hr.to(dev), "SR": sr.to(dev)}
    loss = tr.loss_and_grads(data, noise=noise.to(dev), gamma=gamma)
    want, grads = otrain.loss_and_grads(sd, CFG, hr, sr, noise, gamma, "l2", 0.0, otrain.drop_key(0, 0))
    assert abs(float(loss) - want) < 1e-4 * abs(want)
    scale = max(float(g.norm()) for g in grads.values())
    for name, p in u.named_parameters():
        err = float((tr.G(p).cpu() - grads[name]).norm()) / (float(grads[name].norm()) + 1e-4 * scale)
        assert err < 1e-3, (name, err)
    total = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    assert abs(float(train_ops.grad_norm([tr.G(p) for p in u.parameters()])) - total) < 1e-3 * total
    for i in range(5):
        before = tr.flat.clone()
        tr.optimize_parameters(data)
        now = math.sqrt(float(tr.grad.double().square().sum()))
        assert abs(float(tr.last_grad_norm) - now) < 1e-6 * now
        assert bool(torch.isfinite(tr.flat).all()) and not torch.equal(before, tr.flat)


@GPU
def test_bf16_training_step(dev, monkeypatch):
    """The bf16 training mode on the same network: gradients within the mode's rounding of the oracle's."""
    from oracle import sr3_unet
    from oracle import train as otrain
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention())
    u, sd, gd = network(True, "bf16", dev)
    hr, sr, noise, gamma = batch()
    tr = gd.trainer(lr=1e-4, precision="bf16")
    tr.loss_and_grads({"HR": hr.to(dev), "SR": sr.to(dev)}, noise=noise.to(dev), gamma=gamma)
    _, grads = otrain.loss_and_grads(sd, CFG, hr, sr, noise, gamma, "l2", 0.0, otrain.drop_key(0, 0))
    num = math.sqrt(sum(float((tr.G(p).cpu() - grads[n]).norm()) ** 2 for n, p in u.named_parameters()))
    den = math.sqrt(sum(float(g.norm()) ** 2 for g in grads.values()))
    assert num / den < 4e-2, num / den                              # (TOL["bf16"] of the suite)


@GPU
def test_sampler_over_long_maps(dev):
    """A short reverse chain (captured steps) of the network: finite, and the same latents when the chain is run again."""
    u, _, gd = network(True, "fp32", dev, train=False)
    u.eval()
    gd.noise, gd.seed = "philox", 3
    cond = torch.from_numpy(synth_tensor("long.cond", (2, 3, 48, 48))).to(dev)
    a = gd.p_sample_loop_batched(cond)
    b = gd.p_sample_loop_batched(cond)
    assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@GPU
def test_copies_of_a_used_module(dev):
    """copy.deepcopy and a pickle round trip of a layer that has run (an averaged copy of the network is a common one)."""
    import copy
    import io
    from hsi_dmgasr_amd.sr3_modules import unet
    m = unet.SelfAttention(64, n_head=2, qk_norm_rope=True).to(dev).eval()
    m.precision = "fp32"
    x = torch.from_numpy(synth_tensor("la.x", (1, 64, 36, 34))).to(dev)
    with torch.no_grad():
        want = m(x)
        twin = copy.deepcopy(m)
        buf = io.BytesIO()
        torch.save(m, buf)
        buf.seek(0)
        loaded = torch.load(buf, weights_only=False)                # (written two lines above)
        del m
        torch.cuda.empty_cache()
        assert torch.equal(twin(x), want) and torch.equal(loaded(x), want)
