"""Outputs that a caller hands to the gradients of the token operators: views whose own rows overlap are refused, not raced over."""
import pytest
import torch

GPU = pytest.mark.gpu


def test_rows_apart():
    from hsi_dmgasr_amd import ops
    x = torch.zeros(4096)
    ok = [((5, 3, 16), (48, 16, 1)), ((5, 3, 16), (16, 80, 1)), ((5, 3, 16), (100, 20, 1)), ((1, 3, 16), (1, 16, 1)), ((5, 1, 16), (16, 3, 1)),
          ((1, 1, 16), (2, 2, 1)), ((0, 3, 16), (0, 0, 1))]
    bad = [((5, 3, 16), (16, 16, 1)), ((5, 3, 16), (32, 16, 1)), ((5, 3, 16), (48, 8, 1)), ((5, 1, 16), (8, 16, 1)), ((1, 3, 16), (64, 12, 1)),
           ((5, 3, 16), (47, 16, 1)), ((5, 3, 16), (16, 79, 1))]
    for shape, strides in ok:
        assert ops.rows_apart(x.as_strided(shape, strides)), (shape, strides)
    for shape, strides in bad:
        assert not ops.rows_apart(x.as_strided(shape, strides)), (shape, strides)
        t = x.as_strided(shape, strides)                             # (what "apart" means: as many addresses as elements)
        at = (torch.arange(shape[0])[:, None, None] * strides[0] + torch.arange(shape[1])[:, None] * strides[1] + torch.arange(shape[2]))
        assert at.unique().numel() < t.numel()


def test_overlapping_outputs_are_refused(monkeypatch):
    """(on the CPU: refused ahead of the launch, with every tensor taken for a device tensor)"""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(ops._lib, "on_device", lambda device: (_ for _ in ()).throw(AssertionError("reached the launch")))
    q, k = torch.zeros(6, 2, 64), torch.zeros(6, 2, 64)
    over = torch.zeros(4096).as_strided((6, 2, 64), (64, 64, 1))
    axes, w, pos = ops.RotaryAxes((16,), 64, device="cpu"), torch.ones(64), torch.zeros(6, 1, dtype=torch.int32)
    for out in ((over, k), (q, over)):
        with pytest.raises(ValueError, match="out must be"):
            Tr.qk_norm_rope_bwd(q, k, q, k, w, w, pos, axes, out=out)
    seqs = ops.PackedSequences([6], device="cpu")
    monkeypatch.setattr(ops, "attn_desc", lambda *a: (None, 0, 0, a[:3]))
    saved = ops.AttentionSaved(torch.zeros(2, 6), None)
    for i in range(3):
        grads = [torch.zeros(6, 2, 64) for _ in range(3)]
        grads[i] = over
        with pytest.raises(ValueError, match="grads must be"):
            Tr.attention_packed_bwd(q, q, k, k, q, saved, seqs, grads=grads)
