"""The token operators under autograd: a call whose gradient would be lost is refused, one without a gradient to lose is not."""
import pytest
import torch

GPU = pytest.mark.gpu


def calls(dev):
    from hsi_dmgasr_amd import ops
    axes, pos = ops.RotaryAxes((16,), 64, device=dev), torch.zeros(6, 1, dtype=torch.int32, device=dev)
    seqs = ops.PackedSequences([4, 2], device=dev)
    one = lambda *s: torch.full(s, 0.5, device=dev)  # noqa: E731
    return {"rope": (lambda q, k, wq, wk: ops.qk_norm_rope(q, k, wq, wk, pos, axes), [one(6, 2, 64), one(6, 1, 64), one(64), one(64)]),
            "attention": (lambda q, k, v: ops.attention_packed(q, k, v, seqs), [one(6, 2, 64), one(6, 1, 64), one(6, 1, 64)])}


@pytest.mark.parametrize("op", ["rope", "attention"])
def test_a_gradient_is_not_lost_silently(op):
    """(refused before anything looks at the device)"""
    call, args = calls("cpu")[op]
    for i in range(len(args)):
        given = [a.clone().requires_grad_(j == i) for j, a in enumerate(args)]
        with pytest.raises(RuntimeError, match="autograd"):
            call(*given)
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm device"):
            call(*given)
        with pytest.raises(RuntimeError, match="ROCm device"):
            call(*[a.detach() for a in given])


@GPU
@pytest.mark.parametrize("op", ["rope", "attention"])
def test_without_gradients(op):
    dev = torch.device("cuda:0")
    call, args = calls(dev)[op]
    want = call(*args)
    for a in args:
        a.requires_grad_()
    with torch.no_grad():
        got = call(*args)
    with torch.inference_mode():
        also = call(*args)
    pairs = [(want, got), (want, also)] if torch.is_tensor(want) else [*zip(want, got), *zip(want, also)]
    assert all(torch.equal(a, b) for a, b in pairs)
    with pytest.raises(RuntimeError, match="autograd"):
        call(*args)
