"""The attention layers' plans per map shape: bounded, held by whoever captured a step that goes by them."""
import gc

import pytest
import torch

from helpers import synth_tensor
from test_long_attention import batch, network

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def layers(u):
    from hsi_dmgasr_amd.sr3_modules import unet
    return [m for m in u.modules() if isinstance(m, unet.SelfAttention)]


def test_plans_of_many_shapes_do_not_pile_up():
    from hsi_dmgasr_amd.sr3_modules import unet
    a, cpu = unet.SelfAttention(64, qk_norm_rope=True), torch.device("cpu")
    first = a.map_plan(1, 2, 2, cpu)
    assert a.map_plan(1, 2, 2, cpu) is first
    for n in range(3, 100):
        a.map_plan(1, 2, n, cpu)
    gc.collect()
    assert len(a._recent) == a.MAPS_KEPT and len(a._maps) <= a.MAPS_KEPT + 1 and not a._pinned
    assert a.map_plan(1, 2, 2, cpu) is first                         # (alive as long as somebody has it)
    del first
    latest = a.map_plan(1, 2, 99, cpu)
    for n in range(100, 100 + a.MAPS_KEPT - 1):
        a.map_plan(1, 2, n, cpu)
    assert a.map_plan(1, 2, 99, cpu) is latest                       # least recently USED goes first
    seqs, pos, axes = latest
    assert latest[0] is seqs and seqs.lengths == (198,) and pos.shape == (198, 2) and axes.head_dim == 64


def test_a_held_plan_stays():
    from hsi_dmgasr_amd.sr3_modules import unet
    a, cpu, mine = unet.SelfAttention(64), torch.device("cpu"), {}
    with unet.holding(mine):
        at = a.map_plan(1, 40, 40, cpu)[0]._tables.data_ptr()
        with unet.holding({}):
            a.map_plan(1, 1, 1, cpu)
        a.map_plan(1, 41, 40, cpu)
    for n in range(200):
        a.map_plan(1, 50, 50 + n, cpu)
    gc.collect()
    assert len(mine) == 2 and a.map_plan(1, 40, 40, cpu)[0]._tables.data_ptr() == at
    assert len(a._maps) <= a.MAPS_KEPT + 2
    mine.clear()
    for n in range(200):
        a.map_plan(1, 50, 50 + n, cpu)
    gc.collect()
    assert len(a._maps) <= a.MAPS_KEPT


@GPU
def test_captured_steps_keep_their_tables(dev, monkeypatch):
    """A reverse chain and a training step captured, other map shapes in between until every plan of the layers' own is another: the
    replays still give what a fresh network gives."""
    from hsi_dmgasr_amd.sr3_modules import unet
    monkeypatch.setattr(unet.SelfAttention, "MAPS_KEPT", 2)
    u, sd, gd = network(True, "fp32", dev, train=False)
    u.eval()
    gd.noise, gd.seed = "philox", 3
    cond = torch.from_numpy(synth_tensor("long.cond", (2, 3, 48, 48))).to(dev)

    def others():
        with torch.no_grad():
            for m in layers(u):
                c = m.qkv.in_channels
                for n in range(6):
                    m(torch.ones(1, c, 4, 5 + n, device=dev))
                assert not any(k[:3] == (2, 48, 48) for k in m._recent)
        junk = [torch.full((1 << 16,), 7, dtype=torch.int32, device=dev) for _ in range(40)]      # (freed tables would be written over)
        del junk
    a = gd.p_sample_loop_batched(cond)
    others()
    b = gd.p_sample_loop_batched(cond)
    assert torch.equal(a, b) and not any(m._pinned for m in layers(u))
    hr, sr, noise, gamma = batch()
    data = {"HR": hr.to(dev), "SR": sr.to(dev)}
    u.train()
    tr = gd.trainer(lr=0.0)                                          # (the weights stay: every step has the drawn noise's gradient)
    for k in range(4):                                               # eager, captured, replayed
        torch.manual_seed(5)
        import numpy as np
        np.random.seed(5)
        loss = float(tr.optimize_parameters(data))
        if k == 0:
            want = loss
        assert abs(loss - want) <= 1e-4 * abs(want), (k, loss, want)
        u.eval()
        others()
        u.train()


@GPU
def test_a_callers_own_capture(dev):
    """A layer captured by a caller: its plan stays with the layer, whatever other shapes come."""
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd.sr3_modules import unet
    m = unet.SelfAttention(64, qk_norm_rope=True).to(dev).eval()
    x = ops.to_nhwc(torch.from_numpy(synth_tensor("la.x", (1, 64, 36, 34))).to(dev), "fp32")
    with torch.no_grad():
        want = m._run(x, "fp32").clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = m._run(x, "fp32")
        for n in range(2 * m.MAPS_KEPT):
            m._run(ops.to_nhwc(torch.ones(1, 64, 4, 4 + n, device=dev), "fp32"), "fp32")
        assert len(m._pinned) == 1 and len(m._recent) == m.MAPS_KEPT
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_a_layer_pickled_before_it_had_plans():
    """A whole-module checkpoint of an earlier build: no plans, no option."""
    from hsi_dmgasr_amd.sr3_modules import unet
    a = unet.SelfAttention(64)
    old = {k: v for k, v in a.__dict__.items() if k not in ("_maps", "_recent", "_pinned", "qk_norm_rope")}
    b = unet.SelfAttention.__new__(unet.SelfAttention)
    b.__setstate__(old)
    assert not b.packed(1024) and b.packed(1025) and b.map_plan(1, 33, 32, torch.device("cpu"))[0].lengths == (1056,)
    # the build before this one kept a dict of tuples there
    c = unet.SelfAttention.__new__(unet.SelfAttention)
    c.__setstate__({**old, "qk_norm_rope": False, "_maps": {}})
    assert c.map_plan(1, 33, 32, torch.device("cpu")) is c.map_plan(1, 33, 32, torch.device("cpu"))
