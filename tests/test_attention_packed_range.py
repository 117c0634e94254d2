"""Packed attention where fp16's five exponent bits matter: gradients next to a sequence that holds infinities."""
import math

import pytest
import torch

from test_attention_packed import close, make, plain64

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@GPU
@pytest.mark.parametrize("where", ["do", "v", "both"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=str)
def test_gradients_beside_a_sequence_with_infinities(dev, where, bad):
    """fp16: the scale that P and dS share over a call comes from the finite rows.  Gradients of size 300 (a scaled loss): with a scale of
    one, dS would pass 65504."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths = [50, 30, 70]
    q, k, v, do = make(dev, lengths, 2, 1, 64, torch.float16, seed=4)
    do = (do.float() * 300).half()
    want, _ = plain64(q, k, v, lengths, True, 0.125, do)
    seqs = ops.PackedSequences(lengths, device=dev)
    for x in (do,) if where == "do" else (v,) if where == "v" else (do, v):
        x[60, :, 3] = bad
    o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
    got = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=True)
    keep = torch.cat([torch.arange(50), torch.arange(80, 150)]).to(dev)
    for name, g in zip(("dq", "dk", "dv"), got):
        assert bool(torch.isfinite(g[keep]).all()), name
        close(g[keep], want[name][keep], want["m" + name][keep], 4, name)
    close(o[keep], want["o"][keep], want["mo"][keep], 2, "out")
