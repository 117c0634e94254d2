"""RotaryAxes whose table or sections are replaced between calls, and gradients written to outputs with a token or head axis of length one."""
import math

import pytest
import torch

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def test_the_descriptor_points_at_the_table_that_is_there(monkeypatch):
    """(on the CPU: the descriptor alone, with every tensor taken for a device tensor)"""
    from hsi_dmgasr_amd import ops
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    axes = ops.RotaryAxes((8, 8), 64, device="cpu")
    q, w, pos = torch.zeros(4, 1, 64), torch.ones(64), torch.zeros(4, 2, dtype=torch.int32)
    call = lambda: ops.rope_desc(q, q, w, w, pos, axes, 1e-6)  # noqa: E731
    assert call()[0].freq == axes.freq.data_ptr()
    old = axes.freq
    axes.freq = old * 0.5
    d, _, keep = call()
    assert d.freq == axes.freq.data_ptr() != old.data_ptr() and any(t is axes.freq for t in keep)
    axes.sections = (4, 12)
    d = call()[0]
    assert list(d.sections)[:2] == [4, 12] and d.axes == 2
    good = axes.freq
    for bad in (good.float(), good[:15], torch.zeros(2, 16, dtype=torch.float64)[:, :8], torch.zeros(32, dtype=torch.float64)[::2]):
        axes.freq = bad
        with pytest.raises(ValueError, match="freq"):
            call()
    axes.freq = good
    for bad in ((20, 20), (-1, 4), ()):
        axes.sections = bad
        with pytest.raises(ValueError):
            call()
    axes.sections, axes.head_dim = (8, 8), 32
    with pytest.raises(ValueError, match="heads have 64"):
        call()


@GPU
def test_rescaled_frequencies(dev):
    """The usual reason: positions of a longer sequence pressed into the trained range by frequencies of a half."""
    from hsi_dmgasr_amd import ops
    g = torch.Generator().manual_seed(1)
    q = torch.randn(50, 2, 64, generator=g).to(dev)
    w = torch.ones(64, device=dev)
    pos = torch.arange(50, dtype=torch.int32, device=dev)[:, None]
    axes, twin = ops.RotaryAxes((32,), 64, device=dev), ops.RotaryAxes((32,), 64, device=dev)
    a = ops.qk_norm_rope(q, q, w, w, 2 * pos, axes)[0]
    axes.freq = axes.freq * 0.5
    b = ops.qk_norm_rope(q, q, w, w, 2 * pos, axes)[0]
    assert torch.equal(b, ops.qk_norm_rope(q, q, w, w, pos, twin)[0]) and not torch.equal(a, b)
    # (half an fp64 frequency at twice a position is the same 64-bit angle)
    assert abs(float(axes.freq[0]) * 2 * math.pi - 0.5) < 1e-15


@GPU
@pytest.mark.parametrize("T, H", [(1, 2), (3, 1), (1, 1)])
def test_outputs_with_an_axis_of_length_one(dev, T, H):
    """The stride of an axis of length one is any number (torch leaves it to the view): it is no reason to refuse an output."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as Tr
    g = torch.Generator().manual_seed(2)
    q, dq, k, dk = (torch.randn(T, H, 64, generator=g).to(dev) for _ in range(4))
    w, pos = torch.ones(64, device=dev), torch.arange(T, dtype=torch.int32, device=dev)[:, None]
    axes = ops.RotaryAxes((16,), 64, device=dev)
    want = Tr.qk_norm_rope_bwd(dq, dk, q, k, w, w, pos, axes)
    strides = (13 if T == 1 else 64 * H, 7 if H == 1 else 64, 1)
    out = tuple(torch.zeros(T * H * 64, device=dev).as_strided((T, H, 64), strides) for _ in range(2))
    assert all(ops.rows_aligned(o) for o in out)
    got = Tr.qk_norm_rope_bwd(dq, dk, q, k, w, w, pos, axes, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is out[0] and got[1] is out[1]
