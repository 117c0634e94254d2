"""Packed attention over more tiles than one launch has workgroups for."""
import pytest
import torch

GPU = pytest.mark.gpu


@GPU
def test_a_million_sequences_of_one_token():
    """2^20 + 1 sequences of one token under 16 heads are 2^24 + 16 workgroups of 256 threads.  A token's output is its own v; the
    gradient of v is the sum over the heads that share it, those of q and k are zero."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    dev = torch.device("cuda:0")
    n, H, D = 2 ** 20 + 1, 16, 8
    g = torch.Generator(device=dev).manual_seed(1)
    q, do = (torch.randn(n, H, D, generator=g, device=dev).bfloat16() for _ in range(2))
    k, v = (torch.randn(n, 1, D, generator=g, device=dev).bfloat16() for _ in range(2))
    seqs = ops.PackedSequences([1] * n, device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, want_lse=True)
    assert torch.equal(o, v.expand(n, H, D))
    s = (q.float() * k.float()).sum(-1) * D ** -0.5
    assert float((saved.lse.t() - s).abs().max()) <= 1e-5            # scores up to about 10, eight fp32 products
    dq, dk, dv = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs)
    # P is one up to lse's rounding (1e-5); the sum of 16 heads is rounded once
    want, mag = do.double().sum(1, keepdim=True), do.double().abs().sum(1, keepdim=True)
    assert bool(((dv.double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * (2.0 ** -8 + 2e-5)).all())
    # dS = P (dP - delta): either sum of eight products is off by eight half-steps of fp32 of |do| |v|, and out + residual is v times an
    # exponential of a rounded exponent, |s| half-steps and a few
    top = float((do.float().norm(dim=-1) * v.float().norm(dim=-1)).max()) * D ** -0.5 * (20 + float(s.abs().max())) * 2.0 ** -24
    assert float(dq.float().abs().max()) <= top * float(k.float().abs().max()) and float(dk.float().abs().max()) <= 16 * top * float(q.float().abs().max())
