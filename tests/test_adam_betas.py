"""Adam with the shipped betas (0.9, 0.999): 1 - beta as the 64-bit formula has it, clipped or not (1 - 0.999 from an fp32 0.999 is 1.3e-5
off, and every step would add its squared gradient that much too small)."""
import pytest
import torch

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


@GPU
@pytest.mark.parametrize("clipped", [False, True], ids=["plain", "clipped"])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.95, 0.9999), (0.0, 0.5)], ids=str)
def test_moments_against_64_bits(dev, betas, clipped):
    from hsi_dmgasr_amd import train_ops as T
    b1, b2 = betas
    n = 100_003
    g = torch.Generator().manual_seed(2)
    p, gr = (torch.randn(n, generator=g).to(dev) for _ in range(2))
    m, v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)     # a first step: the moments ARE the increments
    clip, scale = None, 1.0
    if clipped:
        clip = T.clip_coef(gr, 10.0)
        scale = float(clip[1])
        assert scale < 0.1
    p0, g64 = p.double(), gr.double() * scale
    T.adam_step(p, gr, m, v, 1e-2, b1, b2, 1e-8, 1, clip=clip)
    m1, v1 = (1 - b1) * g64, (1 - b2) * g64 * g64
    # m: 1 - beta1 rounded to fp32, the gradient times the coefficient, their product (3 half-steps); v: 1 - beta2, two products of a
    # scaled gradient (2 * 1 + 3) - six and eight leave room for a fused or an unfused add of zero
    u = 2.0 ** -24
    assert bool(((m.double() - m1).abs() <= 6 * u * m1.abs() + 2.0 ** -149).all())
    assert bool(((v.double() - v1).abs() <= 8 * u * v1 + 2.0 ** -149).all())
    want = p0 - 1e-2 * (m1 / (1 - b1)) / ((v1 / (1 - b2)).sqrt() + 1e-8)
    # the increment is at most lr in size: 64 half-steps of it (both moments' errors above, half of v's in the root; corrections, root,
    # product, sum with eps, quotient, rate: one each) and the parameter's own rounding
    assert bool(((p.double() - want).abs() <= 1e-2 * 64 * u + 2 * u * p0.abs()).all())


@GPU
def test_steps_with_the_shipped_betas_against_torch(dev):
    """Twenty steps against torch.optim.Adam in 64 bits."""
    from hsi_dmgasr_amd import train_ops as T
    n = 4099
    g = torch.Generator().manual_seed(3)
    p = torch.randn(n, generator=g).to(dev)
    m, v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    ref = torch.nn.Parameter(p.double())
    opt = torch.optim.Adam([ref], lr=1e-3, betas=(0.9, 0.999), eps=1e-8)
    for step in range(1, 21):
        gr = torch.randn(n, generator=g).to(dev)
        T.adam_step(p, gr, m, v, 1e-3, 0.9, 0.999, 1e-8, step)
        ref.grad = gr.double()
        opt.step()
    s = opt.state[ref]
    # 20 steps of at most eight roundings each, on sums of positive terms
    assert bool(((v.double() - s["exp_avg_sq"]).abs() <= 160 * 2.0 ** -24 * s["exp_avg_sq"]).all())


@GPU
@pytest.mark.parametrize("clipped", [False, True], ids=["plain", "clipped"])
def test_more_than_32_bits_of_parameters(dev, clipped):
    """2^32 + 7 parameters: every one is stepped once, at the launch's first and last elements and around 2^32."""
    from hsi_dmgasr_amd import train_ops as T
    n = 2 ** 32 + 7
    p, m, v = (torch.zeros(n, device=dev) for _ in range(3))
    g = torch.ones(n, device=dev)
    clip = torch.tensor([1.0, 0.5], device=dev) if clipped else None
    T.adam_step(p, g, m, v, 0.25, 0.5, 0.75, 1e-30, 1, clip=clip)     # m and v hold (1 - beta) g^k, exactly; the increment is lr
    x = 0.5 if clipped else 1.0
    for t, want in ((m, 0.5 * x), (v, 0.25 * x * x)):
        assert float(t[0]) == want and float(t[-1]) == want and torch.equal(t[-1:].expand(n), t)
    assert float(p[0]) == -0.25 and torch.equal(p[:1].expand(n), p)
