"""Attention over packed sequences (ops.attention_packed, train_ops.attention_packed_bwd) against 64-bit formulas."""
import ctypes
import math

import pytest
import torch

GPU = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def plain64(q, k, v, lengths, causal, scale, do=None):
    """(out, lse, dq, dk, dv) in 64 bits, sequence by sequence and head by head; with the sums of magnitudes that bound the roundings:
    a row's sum_j P |v| for out, and the like for the gradients."""
    T, Hq, D = q.shape
    g = Hq // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    r = {n: torch.zeros_like(x) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("mo", q), ("mdq", q), ("mdk", k), ("mdv", v))}
    lse = torch.zeros(Hq, T, dtype=torch.float64, device=q.device)
    first = 0
    for n in lengths:
        to = slice(first, first + n)
        first += n
        for h in range(Hq if n else 0):
            qq, kk, vv = q[to, h], k[to, h // g], v[to, h // g]
            s = scale * (qq @ kk.t())
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
            lse[h, to] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[h, to][:, None])
            o = r["o"][to, h] = p @ vv
            r["mo"][to, h] = p @ vv.abs()
            if do is not None:
                d = do[to, h].double()
                dp, delta = d @ vv.t(), (d * o).sum(1, keepdim=True)
                ds = scale * p * (dp - delta)
                mds = scale * p * (d.abs() @ vv.abs().t() + (d.abs() * o.abs()).sum(1, keepdim=True))
                r["dq"][to, h] = ds @ kk
                r["mdq"][to, h] = mds @ kk.abs()
                r["dk"][to, h // g] += ds.t() @ qq
                r["mdk"][to, h // g] += mds.t() @ qq.abs()
                r["dv"][to, h // g] += p.t() @ d
                r["mdv"][to, h // g] += p.t() @ d.abs()
    return r, lse


def close(got, want, mag, factor, what):
    """|got - want| <= half a step of the type on the value, plus `factor` half-steps of the type on the sum of magnitudes that the value is
    made of (every term carries that many roundings of the type: probabilities, dS, the output that delta is formed from), plus the same
    in fp32 for scores, exponentials and sums (64 half-steps of fp32 per unit of score, scores here reach about 40: see SCORES)."""
    dt = got.dtype
    u, u32 = torch.finfo(dt).eps / 2, torch.finfo(torch.float32).eps / 2
    own = 0.0 if dt == torch.float32 else factor * u
    tol = want.abs() * u + mag * (own + SCORES * u32) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    worst = float(((got.double() - want).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, (what, worst)


# fp32 work on a score s: a sum of D <= 256 products is off by at most D half-steps of sum |q k| scale (typically its root), and that is an
# absolute error of the exponent, i.e. a relative one of P; |q||k| scale reaches 60 at D = 256 with the inputs below, and lse carries the
# same: 2 * 256 * 60 would be the strict bound, 4096 covers sqrt(D) growth with a factor of two in hand.
SCORES = 4096.0


def make(dev, lengths, hq, hk, D, dtype, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths)
    r = lambda h: torch.randn(T, h, D, generator=g)  # noqa: E731
    return [(x * gain).to(dtype).to(dev) for x in (r(hq), r(hk))] + [x.to(dtype).to(dev) for x in (r(hk), r(hq))]


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_sequences_and_their_tiles():
    from hsi_dmgasr_amd import ops
    s = ops.PackedSequences([0, 1, 64, 65, 0, 300], device="cpu")
    assert (s.total, s.longest, s.n64, s.n128) == (430, 300, 1 + 1 + 2 + 5, 1 + 1 + 1 + 3)
    t = s._tables.numpy()
    for rows in (64, 128):
        n = getattr(s, "n%d" % rows)
        for kind in ("full", "causal q", "causal k"):
            at = s._at[kind, rows]
            got = t[at:at + n]
            want = {(f, ln, r) for f, ln in ((0, 1), (1, 64), (65, 65), (130, 300)) for r in range(0, ln, rows)}
            assert {tuple(map(int, x[:3])) for x in got} == want and len(want) == n
            work = {"full": got[:, 1], "causal q": [min(x[1], x[2] + rows) for x in got], "causal k": got[:, 1] - got[:, 2]}[kind]
            assert all(a >= b for a, b in zip(work, work[1:]))
    assert ops.PackedSequences([], device="cpu").total == 0 and ops.PackedSequences([0], device="cpu").n64 == 0
    for bad in ([-1], [2 ** 31], [2 ** 30, 2 ** 30], [2 ** 31 - 255]):
        with pytest.raises(ValueError):
            ops.PackedSequences(bad, device="cpu")


def test_refusals_without_a_gpu():
    from hsi_dmgasr_amd import _lib, ops
    from hsi_dmgasr_amd import train_ops as T
    q, k = torch.zeros(10, 4, 64), torch.zeros(10, 2, 64)
    s = ops.PackedSequences([4, 6], device="cpu")
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.attention_packed(q, k, k, s)
    good = dict(q=q, k=k, v=k, seqs=s)
    for bad in (dict(q=q[:9]), dict(v=k[:, :1]), dict(k=torch.zeros(10, 3, 64), v=torch.zeros(10, 3, 64)), dict(seqs=ops.PackedSequences([4, 5], device="cpu")),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=q[0]), dict(q=q[..., :32]),
                dict(q=torch.zeros(10, 4, 260), k=torch.zeros(10, 2, 260), v=torch.zeros(10, 2, 260)),
                dict(q=torch.zeros(10, 4, 36).half(), k=torch.zeros(10, 2, 36).half(), v=torch.zeros(10, 2, 36).half())):
        with pytest.raises(ValueError):
            ops.attention_packed(**{**good, **bad})
    for bad in (dict(k=k.half()), dict(q=q.double(), k=k.double(), v=k.double())):
        with pytest.raises(TypeError):
            ops.attention_packed(**{**good, **bad})
    L = _lib.lib()

    def desc(**kw):
        d = _lib.AttnDesc()
        vals = dict(q=64, k=64, v=64, q_ts=256, q_hs=64, k_ts=128, k_hs=64, v_ts=128, v_hs=64, T=10, qtiles64=64, qtiles128=64, ktiles64=64, ktiles128=64,
                    n64=2, n128=2, longest=6, pairs=31.0, Hq=4, Hk=2, D=64, prec=_lib.BF16, causal=1, scale=0.125)
        for n, v in {**vals, **kw}.items():
            setattr(d, n, v)
        return ctypes.byref(d)

    one = ctypes.c_void_p(64)
    need = L.hsidm_attention_packed_bwd_workspace_bytes(desc())
    assert need > 10 * 4 * 4
    for bad in (dict(T=0), dict(Hk=3), dict(Hk=0), dict(D=0), dict(D=260), dict(D=36), dict(prec=5), dict(scale=0.0), dict(scale=math.nan), dict(q=72),
                dict(k_hs=4), dict(v_ts=-64), dict(n64=0), dict(longest=0), dict(pairs=0.0), dict(pairs=math.nan), dict(qtiles64=None), dict(ktiles128=None)):
        assert L.hsidm_attention_packed_workspace_bytes(desc(**bad)) == -1, bad
        assert L.hsidm_attention_packed(desc(**bad), one, None, one, one, 1 << 30, None) == -1, bad
        assert L.hsidm_attention_packed_bwd(desc(**bad), one, None, one, *[one, 256, 64] * 4, one, 1 << 30, None) == -1, bad
    assert L.hsidm_attention_packed(None, one, None, one, one, 0, None) == -1
    assert L.hsidm_attention_packed(desc(), None, None, one, one, 1 << 30, None) == -1
    assert L.hsidm_attention_packed(desc(longest=100000), one, None, one, one, 0, None) == -1          # the split form without its workspace
    assert L.hsidm_attention_packed_bwd(desc(), one, None, one, *[one, 256, 64] * 4, one, need - 1, None) == -1
    assert L.hsidm_attention_packed_bwd(desc(), one, None, None, *[one, 256, 64] * 4, one, need, None) == -1
    assert L.hsidm_attention_packed_bwd(desc(), one, None, one, *[one, 256, 63] * 4, one, need, None) == -1


def test_structs_match_the_header(tmp_path):
    """Sizes and offsets of the descriptors that the ctypes binding restates, as the C compiler lays them out."""
    import os
    import subprocess
    from hsi_dmgasr_amd import _lib
    structs = {"hsidm_attn_desc": _lib.AttnDesc, "hsidm_rope_desc": _lib.RopeDesc, "hsidm_tensor_item": _lib.TensorItem}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "hsidm.h"', 'int main(void) {', 'printf("%zu\\n", sizeof(hsidm_attn_tile));']
    for name, s in structs.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f, _ in s._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "probe")])
    got = list(map(int, subprocess.check_output([str(tmp_path / "probe")]).split()))
    want = [16]
    for s in structs.values():
        want += [ctypes.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]
    assert got == want


def test_loaded_to_another_device():
    """The sequences say where their tables ARE: the descriptor would otherwise pass addresses of another memory."""
    import io
    from hsi_dmgasr_amd import ops
    s = ops.PackedSequences([3, 70], device="cpu")
    s._plans["x"] = 1
    buf = io.BytesIO()
    torch.save(s, buf)
    buf.seek(0)
    loaded = torch.load(buf, map_location="meta", weights_only=False)          # (written three lines above)
    assert s.device.type == "cpu" and loaded.device.type == "meta" and loaded.lengths == s.lengths and not loaded._plans


# ------------------------------------------------------------------------------------------------------------------- GPU
CASES = [  # lengths, hq, hk, D, causal
    ([1], 1, 1, 64, True), ([1, 1, 1], 2, 1, 32, False), ([31, 1, 64, 7, 103], 8, 2, 64, True), ([33, 0, 65, 129], 4, 4, 128, True),
    ([200, 3, 0], 2, 2, 40, False), ([257, 255], 3, 1, 96, True), ([128, 127, 64], 6, 2, 256, False), ([300, 70], 2, 1, 200, True),
    ([1025], 1, 1, 64, False), ([700, 5], 1, 1, 128, True), ([2049], 8, 1, 8, True), ([500, 400, 300, 200, 100], 16, 8, 16, False),
    ([40] * 150, 8, 4, 64, True), ([1300], 2, 2, 256, True), ([70, 3], 2, 1, 24, False), ([129], 5, 5, 56, True), ([64], 3, 3, 72, False),
]


@GPU
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") if not isinstance(x, list) or len(x) < 9 else "many" for x in c))
def test_forward_and_backward(dev, case, kind):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths, hq, hk, D, causal = case
    dtype = TYPES[kind]
    q, k, v, do = make(dev, lengths, hq, hk, D, dtype)
    seqs = ops.PackedSequences(lengths, device=dev)
    scale = D ** -0.5
    o, saved = ops.attention_packed(q, k, v, seqs, causal=causal, want_lse=True)
    assert torch.equal(o, ops.attention_packed(q, k, v, seqs, causal=causal))
    want, want_lse = plain64(q, k, v, lengths, causal, scale, do)
    close(o, want["o"], want["mo"], 2, "out")
    assert float((saved.lse.double() - want_lse).abs().max()) <= SCORES * 2.0 ** -24 * 2
    # (the residual is what the fp32 output lost in the store: together they are within a step of the residual's own rounding, fp32's errors
    # and the probabilities' rounding)
    assert (saved.residual is None) == (kind == "fp32")
    if saved.residual is not None:
        u = torch.finfo(dtype).eps / 2
        both = o.double() + saved.residual.double()
        tol = want["o"].abs() * u * u * 4 + want["mo"] * (2 * u + SCORES * 2.0 ** -24) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((both - want["o"]).abs() <= tol).all())
        assert bool((saved.residual.double().abs() <= o.double().abs() * 2 * u + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())
    grads = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=causal)
    bare = Tr.attention_packed_bwd(do, q, k, v, o, (saved.lse, None), seqs, causal=causal)
    for name, g in zip(("dq", "dk", "dv"), bare):
        close(g, want[name], want["m" + name], 4, name + " without the residual")
    again = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=causal)
    for name, g, a in zip(("dq", "dk", "dv"), grads, again):
        assert torch.equal(g, a), name
        close(g, want[name], want["m" + name], 4, name)


@GPU
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("do_gain", [1e-4, 1.0, 300.0])
def test_long_rows_and_gradient_sizes(dev, kind, do_gain):
    """4100 keys: probabilities of 2^-12, with gradients small and large - neither underflows nor overflows the type's exponents.  As a
    whole (the 2-norm): within 4 half-steps of the type, which random roundings of every term leave far below."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    dtype = TYPES[kind]
    lengths = [4100]
    q, k, v, do = make(dev, lengths, 2, 1, 64, dtype, seed=2, gain=0.5)
    do = (do.float() * do_gain).to(dtype)
    seqs = ops.PackedSequences(lengths, device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, want_lse=True)
    got = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs)
    want, _ = plain64(q, k, v, lengths, False, 0.125, do)
    u = torch.finfo(dtype).eps / 2
    for name, g in zip(("o", "dq", "dk", "dv"), (o,) + got):
        w = want[name]
        # (fp16 stores of values near its smallest normal keep half a subnormal step)
        floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * w.numel() ** 0.5
        err = float((g.double() - w).norm())
        assert err <= (4 * u + (64 * 2.0 ** -24 if kind == "fp32" else 0)) * float(w.norm()) + floor, (name, err / float(w.norm()))


@GPU
def test_large_scores_and_lazy_maximum(dev):
    """Scores that grow along the keys by far more than the lazy rescaling's threshold, and by less; rows dominated by one key."""
    from hsi_dmgasr_amd import ops
    T, D = 600, 64
    g = torch.Generator().manual_seed(3)
    k = torch.randn(T, 1, D, generator=g)
    q = torch.randn(T, 1, D, generator=g)
    ramp = torch.linspace(0, 1, T)[:, None, None]
    v = torch.randn(T, 1, D, generator=g).to(dev)
    for gain in (0.5, 20.0, 400.0):
        kk = (k * 0.1 + gain * ramp * torch.ones(1, 1, D) / D).to(dev)
        qq = (q * 0.1 + torch.ones(1, 1, D)).to(dev)
        seqs = ops.PackedSequences([T], device=dev)
        for causal in (False, True):
            o, saved = ops.attention_packed(qq, kk, v, seqs, causal=causal, scale=1.0, want_lse=True)
            want, want_lse = plain64(qq, kk, v, [T], causal, 1.0)
            # scores up to 400: an fp32 score is off by 400 * 2^-24 * sqrt(D)
            tol = 2.0 ** -24 * (gain + 8) * 16
            assert float((o.double() - want["o"]).abs().max()) <= tol * 8
            assert float((saved.lse.double() - want_lse).abs().max()) <= tol * 8


@GPU
def test_values_of_other_sequences_never_matter(dev):
    """A NaN or infinity in one sequence stays there, whatever tile it shares; an earlier token's rows do not change with later tokens."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths = [50, 30, 70]
    for dtype in TYPES.values():
        q, k, v, do = make(dev, lengths, 2, 1, 64, dtype, seed=4)
        seqs = ops.PackedSequences(lengths, device=dev)
        o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
        g = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=True)
        for bad in (math.nan, math.inf):
            qb, kb, vb, db = q.clone(), k.clone(), v.clone(), do.clone()
            for x in (qb, kb, vb, db):
                x[60, :, 3] = bad
            ob, lb = ops.attention_packed(qb, kb, vb, seqs, causal=True, want_lse=True)
            keep = torch.cat([torch.arange(50), torch.arange(80, 150)]).to(dev)
            assert torch.equal(ob[keep], o[keep])
            if dtype != torch.float16:                    # fp16 gradients share one scale over the whole call, which a NaN takes away
                gb = Tr.attention_packed_bwd(db, qb, kb, vb, ob, lb, seqs, causal=True)
                assert all(torch.equal(a[keep], b[keep]) for a, b in zip(g, gb))
        k2, v2 = k.clone(), v.clone()
        k2[149], v2[149] = 7.0, -7.0
        o2 = ops.attention_packed(q, k2, v2, seqs, causal=True)
        assert torch.equal(o2[:149], o[:149]) and not torch.equal(o2[149], o[149])


@GPU
@pytest.mark.parametrize("layout", ["thirds", "heads of (q|k|v)", "odd offset", "transposed", "expanded"])
def test_layouts(dev, layout):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths, H, D, dtype = [90, 45], 2, 64, torch.bfloat16
    T = sum(lengths)
    x = torch.randn(T * 3 * H * D + 5, device=dev).to(dtype)
    qkv = x[:T * 3 * H * D]
    grads = torch.full((T, 3 * H + 1, D), 9.0, device=dev, dtype=dtype)
    q, k, v = {"thirds": lambda: qkv.view(T, 3, H, D).unbind(1), "heads of (q|k|v)": lambda: qkv.view(T, H, 3, D).unbind(2),
               "odd offset": lambda: x[5:].view(T, 3, H, D).unbind(1), "transposed": lambda: qkv.view(3, H, T, D).transpose(1, 2).unbind(0),
               "expanded": lambda: [t[:, :1].expand(T, H, D) for t in qkv.view(T, 3, H, D).unbind(1)]}[layout]()
    seqs = ops.PackedSequences(lengths, device=dev)
    dense = [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v)]
    o, saved = ops.attention_packed(q, k, v, seqs, want_lse=True)
    o2, lse2 = ops.attention_packed(*dense, seqs, want_lse=True)
    assert torch.equal(o, o2) and torch.equal(saved.lse, lse2.lse) and torch.equal(saved.residual, lse2.residual)
    do = torch.randn(T, H, 2 * D, device=dev).to(dtype)[..., ::2]
    views = (grads[:, 0:H], grads[:, H:2 * H], grads[:, 2 * H:3 * H])
    got = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, grads=views)
    want = Tr.attention_packed_bwd(do.contiguous(), *dense, o2, lse2, seqs)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((grads[:, 3 * H] == 9).all())
    with pytest.raises(ValueError, match="grads"):
        Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, grads=(views[0], views[1], views[2].float()))
    with pytest.raises(ValueError, match="lse"):
        Tr.attention_packed_bwd(do, q, k, v, o, (saved.lse[:, :-1], None), seqs)
    with pytest.raises(ValueError, match="like q"):
        Tr.attention_packed_bwd(do[:-1], q, k, v, o, saved, seqs)


@GPU
def test_scalar_arguments_are_read_on_every_call(dev):
    """scale and eps given as tensors that the caller rewrites in place."""
    from hsi_dmgasr_amd import ops
    q, k, v = torch.randn(3, 40, 2, 32, generator=torch.Generator().manual_seed(3)).to(dev)
    seqs, s = ops.PackedSequences([40], device=dev), torch.tensor(0.5)
    a = ops.attention_packed(q, k, v, seqs, scale=s)
    s.fill_(2.0)
    b = ops.attention_packed(q, k, v, seqs, scale=s)
    assert torch.equal(a, ops.attention_packed(q, k, v, seqs, scale=0.5)) and torch.equal(b, ops.attention_packed(q, k, v, seqs, scale=2.0))
    assert not torch.equal(a, b)
    axes, w, pos, eps = ops.RotaryAxes((4,), 32, device=dev), torch.ones(32, device=dev), torch.zeros(40, 1, dtype=torch.int32, device=dev), torch.tensor(0.5)
    a = ops.qk_norm_rope(q, k, w, w, pos, axes, eps=eps)[0]
    eps.fill_(2.0)
    b = ops.qk_norm_rope(q, k, w, w, pos, axes, eps=eps)[0]
    assert torch.equal(b, ops.qk_norm_rope(q, k, w, w, pos, axes, eps=2.0)[0]) and not torch.equal(a, b)


@GPU
def test_no_tokens(dev):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    for lengths in ([], [0, 0]):
        seqs = ops.PackedSequences(lengths, device=dev)
        e = torch.empty(0, 2, 64, device=dev)
        o, saved = ops.attention_packed(e, e, e, seqs, want_lse=True)
        assert o.shape == e.shape and saved.lse.shape == (2, 0)
        assert all(g.shape == e.shape for g in Tr.attention_packed_bwd(e, e, e, e, o, saved, seqs))


@GPU
def test_gradient_against_differences(dev):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    lengths = [37, 70]
    q, k, v, do = make(dev, lengths, 4, 2, 32, torch.float32, seed=6)
    seqs = ops.PackedSequences(lengths, device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
    grads = Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=True)
    g = torch.Generator().manual_seed(1)
    for i, gx in enumerate(grads):
        x = [q, k, v]
        u = torch.randn(x[i].shape, generator=g).to(dev)
        h = 5e-3
        f = lambda s: float((ops.attention_packed(*[t + s * u if j == i else t for j, t in enumerate(x)], seqs, causal=True).double() * do).sum())  # noqa: E731
        want, scale = float((gx.double() * u).sum()), float((gx.double() * u).abs().sum())
        assert abs((f(h) - f(-h)) / (2 * h) - want) < 2e-3 * scale       # the difference is off by h^2 of the third derivative and fp32's noise / h


@GPU
@pytest.mark.parametrize("lengths", [[333, 20], [2500]], ids=["whole", "split"])
def test_captured_and_on_another_stream(dev, lengths):
    """A captured forward + backward replayed with new values, eager work in between; two graphs of it; a second stream."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    q, k, v, do = make(dev, lengths, 2, 1, 64, torch.float16, seed=7)
    seqs = ops.PackedSequences(lengths, device=dev)

    def step():
        o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
        return (o, saved.lse, saved.residual) + Tr.attention_packed_bwd(do, q, k, v, o, saved, seqs, causal=True)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for i in range(3):
        q.mul_(0.9); do.add_(0.1)
        want = [t.clone() for t in step()]
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


@GPU
def test_offsets_beyond_32_bits(dev):
    """More than 2^31 elements of queries, keys in rows 128 KB apart and 18 MB apart (through a copy): the last sequence is what it is alone."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    n, H, D = 8, 512, 128
    T = 33000
    lengths = [n] * (T // n)
    q = torch.randn(T, H, D, device=dev, dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31
    k, v = q[:, 5:6], q[:, 300:301]
    seqs, one = ops.PackedSequences(lengths, device=dev), ops.PackedSequences([n], device=dev)
    o, saved = ops.attention_packed(q, k, v, seqs, causal=True, want_lse=True)
    last = [t[-n:].clone() for t in (q, k, v)]
    o1, saved1 = ops.attention_packed(*last, one, causal=True, want_lse=True)
    assert torch.equal(o[-n:], o1) and torch.equal(saved.lse[:, -n:], saved1.lse)
    g = Tr.attention_packed_bwd(q, q, k, v, o, saved, seqs, causal=True)
    g1 = Tr.attention_packed_bwd(last[0], *last, o1, saved1, one, causal=True)
    assert torch.equal(g[0][-n:], g1[0])
    # dk and dv add 512 heads in fp32, split between workgroups or not: sums of the same terms in another order, then one rounding
    for a, b in zip(g[1:], g1[1:]):
        assert float((a[-n:].double() - b.double()).abs().max()) <= 2 * 2.0 ** -8 * float(b.double().abs().max())
    del o, saved, g
    far = torch.randn(100 * 70000, 128, device=dev, dtype=torch.bfloat16).view(100, 70000, 128)      # 17.9 MB from token to token
    qf = far[:, 1:3]
    s100 = ops.PackedSequences([100], device=dev)
    assert not ops.rows_strided(qf)
    assert torch.equal(ops.attention_packed(qf, qf, qf, s100), ops.attention_packed(qf.clone(), qf.clone(), qf.clone(), s100))
