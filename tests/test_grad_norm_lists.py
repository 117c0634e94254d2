"""TensorList where a tensor keeps its address, its element count and its type, but not its layout."""
import pytest
import torch

GPU = pytest.mark.gpu


def views(big):
    """Views of big [8, 8] that begin where it does and have 32 elements, none of them consecutive in memory."""
    return {"columns": big[:, :4], "every second row": big[::2], "expanded": big[:1, :4].expand(8, 4), "transposed columns": big[:, :4].t(),
            "every second element": big.view(-1)[::2]}


@pytest.mark.parametrize("start", ["contiguous", "transposed"])
@pytest.mark.parametrize("view", ["columns", "every second row", "expanded", "transposed columns", "every second element"])
def test_layouts_are_checked_on_every_call(monkeypatch, view, start):
    """(on the CPU: the list's own checks, with every tensor taken for a device tensor)"""
    from hsi_dmgasr_amd import train_ops as T
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    big = torch.arange(64.0).view(8, 8)
    x = torch.zeros(0)
    x.data = big[:4] if start == "contiguous" else big[:4].t()
    tl = T.TensorList([x])
    items = tl.items()
    assert items[0].n == 32 and items[0].ptr == big.data_ptr() and tl.items() is items
    x.data = views(big)[view]
    assert x.data_ptr() == big.data_ptr() and x.numel() == 32
    with pytest.raises(ValueError, match="dense"):
        tl.items()
    with pytest.raises(ValueError, match="dense"):                   # (and again: a refused state is not kept)
        tl.disjoint()
    x.data = big[:4].t()                                             # a dense layout: followed
    assert tl.items()[0].n == 32
    x.data = big[:4]
    assert tl.items()[0].n == 32


@GPU
def test_nothing_beside_a_repointed_tensor_is_scaled():
    from hsi_dmgasr_amd import train_ops as T
    dev = torch.device("cuda:0")
    big = torch.ones(8, 8, device=dev)
    x = torch.ones(0, device=dev)
    x.data = big[:4]
    tl = T.TensorList([x])
    assert abs(float(T.clip_grad_norm_(tl, 1e9)) - 32 ** 0.5) < 1e-5
    for v in views(big).values():
        x.data = v
        for call in (T.grad_norm, lambda t: T.clip_grad_norm_(t, 0.5)):
            with pytest.raises(ValueError, match="dense"):
                call(tl)
    assert bool((big == 1).all())
