"""Trainer.last_grad_norm once clipping is switched off: no norm of an earlier step stays behind."""
import torch

import cpu_double


def test_no_norm_without_clipping(monkeypatch):
    from hsi_dmgasr_amd import train_ops
    from test_train_orchestration import build, synth_tensor
    cpu_double.install(monkeypatch)
    monkeypatch.setattr(train_ops, "clip_coef", lambda t, bound, scale=1.0: torch.stack([t.norm() * scale, torch.tensor(1.0)]))
    plain = train_ops.adam_step
    monkeypatch.setattr(train_ops, "adam_step", lambda *a, clip=None, **kw: plain(*a, **kw))
    _, _, _, tr = build("tiny", "l1", False)
    data = {k: torch.from_numpy(synth_tensor("clip.%s" % k, (2, 3, 16, 16))) for k in ("HR", "SR")}
    assert tr.last_grad_norm is None
    tr.max_grad_norm = 1.0
    tr.optimize_parameters(data)
    assert float(tr.last_grad_norm) > 0
    tr.max_grad_norm = 2.0                                           # another bound: the last step's norm is still that
    assert float(tr.last_grad_norm) > 0
    tr.max_grad_norm = None
    assert tr.last_grad_norm is None
    tr.optimize_parameters(data)
    assert tr.last_grad_norm is None
