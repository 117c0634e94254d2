"""Packed attention where fp16's eleven bits and five exponent bits matter: probabilities far below a row's largest one, and gradients next
to a sequence that holds infinities."""
import math

import pytest
import torch

from test_attention_packed import SCORES, close, make, plain64

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@GPU
@pytest.mark.parametrize("dominant", ["first", "last"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32], ids=str)
def test_many_keys_far_below_the_largest(dev, kind, dominant):
    """One key with a score of 18 among 65536 at zero, the same for every query: each of them has e^-18 = 2^-26 of its probability, together
    they are 2^-10 of the row, and they are all there is of the output's first half (the dominant key's values are zero there)."""
    from hsi_dmgasr_amd import ops
    n, D = 65537, 64
    at = 0 if dominant == "first" else n - 1
    q, k = torch.zeros(n, 1, D), torch.zeros(n, 1, D)
    q[:, :, 0], k[at, :, 0] = 1.0, 18.0
    v = torch.rand(n, 1, D, generator=torch.Generator().manual_seed(11)) + 0.5
    v[at, :, :32] = 0.0
    q, k, v = (t.to(kind).to(dev) for t in (q, k, v))
    seqs = ops.PackedSequences([n], device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, scale=1.0, want_lse=True)
    p = torch.exp(k[:, 0, 0].double() - 18.0)
    p = p / p.sum()
    want = p @ v[:, 0].double()                                     # (no negative value: a sum of magnitudes too)
    # the store's half step; a probability's half step, where the type has it as a normal number; below that half a subnormal step - the
    # scale is such that a row's largest probability is between 2^11 and 2^15, so 2^-25 is 2^-36 of it; and fp32 scores, exponentials, sums
    u = torch.finfo(kind).eps / 2
    tol = want * u + want * (0 if kind == torch.float32 else u) + want * SCORES * 2.0 ** -24
    if kind == torch.float16:
        tol = tol + 2.0 ** -36 * v[:, 0].double().sum(0)
    assert bool(((o.double() - want).abs() <= tol).all()), float(((o.double() - want).abs() / tol).max())
    assert float((saved.lse.double() - (18.0 + math.log1p((n - 1) * math.exp(-18.0)))).abs().max()) <= SCORES * 2.0 ** -24 * 2


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


@GPU
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("below", [0, 10, 14, 18])
def test_gradients_far_smaller_than_another_sequences(dev, below, causal):
    """fp16 gradients of a scaled loss: one short sequence at 8192, a long one 2^below times smaller (a mean over its own length, say) -
    all of them normal numbers.  The scale that dS is held at is the sequence's own."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths = [64, 2100, 33]
    q, k, v, do = make(dev, lengths, 4, 2, 64, torch.float16, seed=2, gain=0.5)
    do = do.float() * 8192.0
    do[64:2164] *= 2.0 ** -below
    do[2164:] *= 2.0 ** -below / 4
    do = do.clamp(-6e4, 6e4).half()
    seqs = ops.PackedSequences(lengths, device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, causal=causal, want_lse=True)
    got = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=causal)
    want, _ = plain64(q, k, v, lengths, causal, 0.125, do)
    first = 0
    for n in lengths:
        to = slice(first, first + n)
        first += n
        for name, g in zip(("dq", "dk", "dv"), got):
            # per sequence, as a whole: within 4 half-steps of the type (the bound of test_long_rows_and_gradient_sizes), and half a subnormal
            # step a value for those that the type cannot hold as normal numbers
            w = want[name][to]
            floor = torch.finfo(torch.float16).smallest_normal * torch.finfo(torch.float16).eps * w.numel() ** 0.5
            err = float((g[to].double() - w).norm())
            assert err <= 4 * 2.0 ** -11 * float(w.norm()) + floor, (name, n, err / float(w.norm()) * 2 ** 11)


@GPU
def test_gradients_of_rows_far_smaller_than_others_of_their_sequence(dev):
    """One sequence, causal: the first rows' gradients are 2^16 times the last ones'.  Each row's dQ is held at its own scale."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    n = 700
    q, k, v, do = make(dev, [n], 2, 1, 64, torch.float16, seed=3, gain=0.5)
    do = do.float() * 4096.0
    do[300:] *= 2.0 ** -16
    do = do.half()
    seqs = ops.PackedSequences([n], device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
    got = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=True)
    want, _ = plain64(q, k, v, [n], True, 0.125, do)
    for name, g, to in (("dq", got[0], slice(300, n)), ("dq", got[0], slice(0, 300)), ("dk", got[1], slice(384, n)), ("dv", got[2], slice(300, n))):
        w = want[name][to]               # (dk of keys behind row 384, a tile's edge: every query that sees them is a small one)
        floor = torch.finfo(torch.float16).smallest_normal * torch.finfo(torch.float16).eps * w.numel() ** 0.5
        err = float((g[to].double() - w).norm())
        assert err <= 4 * 2.0 ** -11 * float(w.norm()) + floor, (name, to, err / float(w.norm()) * 2 ** 11)


@GPU
@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e4], ids=str)
def test_other_sequences_gradients_never_matter(dev, bad):
    """Whatever one sequence's tensors hold, the others' fp16 gradients are the same to the last bit."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths = [50, 30, 70, 200]
    q, k, v, do = make(dev, lengths, 4, 2, 64, torch.float16, seed=4)
    seqs = ops.PackedSequences(lengths, device=dev)
    for causal in (False, True):
        o, saved = ops.attention_packed(q, k, v, seqs, causal=causal, want_lse=True)
        want = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=causal)
        qb, kb, vb, db = (x.clone() for x in (q, k, v, do))
        for x in (qb, kb, vb, db):
            x[60, :, 3] = bad
        ob, sb = ops.attention_packed(qb, kb, vb, seqs, causal=causal, want_lse=True)
        got = Tr.attention_packed_bwd(db, qb, kb, vb, ob, sb, seqs, causal=causal)
        keep = torch.cat([torch.arange(50), torch.arange(80, 350)]).to(dev)
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want))
