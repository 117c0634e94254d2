"""Several attention heads in the network: the shipped configuration (512-channel attention layers) with the norm and rotation of queries
and keys, in inference and in the training step, against the oracle."""
import pytest
import torch

import cpu_double
from gpu_util import check, fill_synth
from helpers import synth_tensor
from test_long_attention import CFG, batch, oracle_attention, packed_doubles

GPU = pytest.mark.gpu
FULL = dict(in_channel=6, out_channel=3, inner_channel=64, norm_groups=32, channel_mults=[1, 2, 4, 8, 8], attn_res=[16], res_blocks=2, image_size=128)


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def layers(u):
    from hsi_dmgasr_amd.sr3_modules import unet
    return [m for m in u.modules() if isinstance(m, unet.SelfAttention)]


def network(cfg, n_head, rope, precision, dev="cpu"):
    from hsi_dmgasr_amd.sr3_modules import diffusion, unet
    u = unet.UNet(precision=precision, attn_qk_norm_rope=rope, attn_n_head=n_head, **cfg)
    fill_synth(u, "heads.")
    for m in layers(u):
        if rope:
            with torch.no_grad():
                m.q_norm.add_(1.0)
                m.k_norm.add_(1.0)
    sd = {k: v.detach().clone() for k, v in u.state_dict().items()}
    u.to(dev)
    gd = diffusion.GaussianDiffusion(u, image_size=cfg["image_size"], channels=3, loss_type="l2", conditional=True)
    gd.set_loss(dev)
    gd.set_new_noise_schedule(dict(schedule="cosine", n_timestep=20, linear_start=1e-6, linear_end=1e-2), dev)
    return u, sd, gd


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_the_shipped_configuration_takes_the_option():
    from hsi_dmgasr_amd.sr3_modules import unet
    with pytest.raises(ValueError, match="attn_n_head"):
        unet.UNet(attn_qk_norm_rope=True, **FULL)
    u = unet.UNet(attn_qk_norm_rope=True, attn_n_head=2, **FULL)
    at = layers(u)
    assert len(at) == 6 and all(m.n_head == 2 and m.q_norm.shape == (256,) and m.packed(1) for m in at)
    plain = unet.UNet(**FULL)
    extra = set(u.state_dict()) - set(plain.state_dict())
    assert len(extra) == 12 and all(k.endswith(("q_norm", "k_norm")) for k in extra)
    assert all(m.n_head == 1 for m in layers(plain)) and set(unet.UNet(attn_n_head=2, **FULL).state_dict()) == set(plain.state_dict())


class CpuTrainer:
    """(built on first use: the package's Trainer without its device check)"""
    def __new__(cls, *a, **k):
        from hsi_dmgasr_amd import training

        class Cpu(training.Trainer):
            def _check_device(self):
                pass
        return Cpu(*a, **k)


def test_training_step_orchestration(monkeypatch):
    """The gradient routing of two heads with norm and rotation (everything by torch doubles) against the oracle's autograd."""
    from oracle import sr3_unet
    from oracle import train as otrain
    from test_train_orchestration import compare
    cpu_double.install(monkeypatch)
    packed_doubles(monkeypatch)
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention(2))
    u, sd, gd = network(CFG, 2, True, "fp32")
    tr = CpuTrainer(gd, lr=1e-3)
    hr, sr, noise, gamma = batch()
    loss = tr.loss_and_grads({"HR": hr, "SR": sr}, noise=noise, gamma=gamma)
    want, grads = otrain.loss_and_grads(sd, CFG, hr, sr, noise, gamma, "l2", 0.0, otrain.drop_key(0, 0))
    assert abs(float(loss) - want) < 1e-4 * abs(want)
    compare(tr, grads)


def test_trainer_refuses_heads_without_the_packed_kernels(monkeypatch):
    cpu_double.install(monkeypatch)
    with pytest.raises(NotImplementedError, match="n_head"):
        CpuTrainer(network(CFG, 2, False, "fp32")[2])


# ------------------------------------------------------------------------------------------------------------------- GPU
@GPU
@pytest.mark.parametrize("rope", [False, True], ids=["plain", "qk_norm_rope"])
def test_shipped_network_with_two_heads(dev, rope, monkeypatch):
    """The forward pass at 128 x 128 (attention over 16 x 16 and 8 x 8 maps, heads of 256 channels), bounds of the suite per mode."""
    from oracle import sr3_unet
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention(2))
    u, sd, _ = network(FULL, 2, rope, "fp32", dev)
    u.eval()
    x = torch.from_numpy(synth_tensor("heads.x", (1, 6, 128, 128)))
    gamma = torch.tensor([[0.7]])
    with torch.no_grad():
        want = sr3_unet.unet_forward(sd, FULL, x, gamma)
        for prec in ("fp32", "bf16"):
            u.precision = prec
            check("unet_two_heads_%s" % ("rope" if rope else "plain"), prec, u(x.to(dev), gamma.to(dev)), want)


@GPU
def test_shipped_network_beyond_1024_tokens(dev, monkeypatch):
    """The shipped channels on a 512 x 512 image reach 64 x 64 attention maps; here its attention layer alone, 36 x 34 and two heads of 256
    channels - one head of 512 is refused."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd.sr3_modules import unet
    x = torch.from_numpy(synth_tensor("heads.map", (1, 512, 36, 34)))
    for n_head in (2, 1):
        m = unet.SelfAttention(512, n_head=n_head)
        fill_synth(m, "heads512.")
        sd = {k: v.detach().clone() for k, v in m.state_dict().items()}
        m.to(dev).eval()
        with torch.no_grad():
            run = lambda: ops.to_nchw(m._run(ops.to_nhwc(x.to(dev), "fp32"), "fp32"), "fp32")  # noqa: E731
            if n_head == 1:
                with pytest.raises(ValueError, match="at most 256"):
                    run()
            else:
                check("self_attention_512", "fp32", run(), oracle_attention(2)(sd, "", x, 32), tol=1e-4)


@GPU
def test_training_step_with_two_heads(dev, monkeypatch):
    """Every gradient against the oracle's autograd, then eager and captured optimiser steps."""
    from oracle import sr3_unet
    from oracle import train as otrain
    monkeypatch.setattr(sr3_unet, "self_attention", oracle_attention(2))
    u, sd, gd = network(CFG, 2, True, "fp32", dev)
    u.train()
    hr, sr, noise, gamma = batch()
    tr = gd.trainer(lr=1e-4)
    data = {"HR": hr.to(dev), "SR": sr.to(dev)}
    loss = tr.loss_and_grads(data, noise=noise.to(dev), gamma=gamma)
    want, grads = otrain.loss_and_grads(sd, CFG, hr, sr, noise, gamma, "l2", 0.0, otrain.drop_key(0, 0))
    assert abs(float(loss) - want) < 1e-4 * abs(want)
    scale = max(float(g.norm()) for g in grads.values())
    for name, p in u.named_parameters():
        err = float((tr.G(p).cpu() - grads[name]).norm()) / (float(grads[name].norm()) + 1e-4 * scale)
        assert err < 1e-3, (name, err)
    for _ in range(4):
        before = tr.flat.clone()
        tr.optimize_parameters(data)
        assert bool(torch.isfinite(tr.flat).all()) and not torch.equal(before, tr.flat)
