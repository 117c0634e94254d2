"""What is measured of the attention / training operators: attention over packed sequences (forward; forward + backward), the RMS norm of
queries and keys with the multi-axis rotation in the same pass (forward; forward + backward), and the global gradient norm with the
clipping inside the Adam step.

``run`` computes them from elementary torch operations in 32 bits (angles in 64) where ``own`` is false, and through
hsi_dmgasr_amd's entry points where it is true; ``exact`` restates the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6                                   # RMS norm of queries and keys
ADAM = dict(lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8, step=10)


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the gradient list of a small network (two levels, 32 channels): where the number of launches counts
        dict(name="norm 61 small tensors fp32", op="norm", type="fp32", tensors=61, elements=700001),
        # mixed-precision gradients of the shipped UNet, one tensor per parameter
        dict(name="norm 419 tensors bf16", op="norm", type="bf16", tensors=419, elements=97807491),
        # the training step's optimiser over the shipped UNet's flat buffers: norm, clipping and Adam
        dict(name="clip + adam, flat 97.8M", op="adam", type="fp32", tensors=1, elements=97807491),
        # one 8x8 map: a bottleneck level of one image
        dict(name="qk norm rope 8x8 fp32", op="rope", type="fp32", images=1, height=8, width=8, hq=1, hk=1, dim=64, sections="16+16", train=False),
        # five spectral groups of a 128x128 image at the first level, band index as the third axis
        dict(name="qk norm rope 128x128 bf16", op="rope", type="bf16", images=5, height=128, width=128, hq=8, hk=2, dim=64, sections="8+12+12", train=False),
        # training at the 64x64 level, odd map sides
        dict(name="qk norm rope train 63x61 fp16", op="rope", type="fp16", images=5, height=63, width=61, hq=4, hk=4, dim=128, sections="32+32", train=True),
        # spectra and token runs of a few lengths in one batch, one token among them: latency
        dict(name="attn short ragged bf16", op="attn", type="bf16", lengths="1+31+64+7+103", hq=8, hk=2, dim=64, causal=True, train=False),
        # full attention over 128x128 maps, one head: what one image and its augmentation bring
        dict(name="attn 2x16384 fp16", op="attn", type="fp16", lengths="16384+16384", hq=1, hk=1, dim=64, causal=False, train=False),
        # long causal sequences of different lengths with grouped heads
        dict(name="attn ragged 8192 bf16 gqa", op="attn", type="bf16", lengths="8192+4097+777+2048+1+5000", hq=16, hk=4, dim=128, causal=True, train=False),
        # a training batch of small 16x16 maps
        dict(name="attn train 4x256 fp16", op="attn", type="fp16", lengths="256+256+256+256", hq=8, hk=8, dim=64, causal=False, train=True),
        # a training batch, causal, grouped heads, ragged
        dict(name="attn train ragged bf16 gqa", op="attn", type="bf16", lengths="4096+1531+2048+63+3001", hq=8, hk=2, dim=128, causal=True, train=True),
        # training at the 64x64 level in the fp32 mode, batch of two, one head
        dict(name="attn train 2x4096 fp32", op="attn", type="fp32", lengths="4096+4096", hq=1, hk=1, dim=128, causal=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "adam", "rope", "rope", "attn", "attn", "attn", "attn"])
    if op == "norm":
        n = _log_int(rng, 1, 900)
        return dict(op=op, type=rng.choice(["fp32", "bf16", "fp16"]), tensors=n, elements=max(n, _log_int(rng, 1000, 90_000_000)))
    if op == "adam":
        return dict(op=op, type="fp32", tensors=1, elements=_log_int(rng, 1000, 90_000_000))
    kind = rng.choice(["bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    hk = rng.choice([1, 2, 4])
    hq = hk * rng.choice([1, 1, 2, 4])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 128, 256])
        axes = rng.choice([1, 2, 3])
        cuts = sorted(rng.randint(1, dim // 2) for _ in range(axes))
        sections = [c - b for b, c in zip([0] + cuts, cuts)]
        rows = 40_000_000 // (dim * (hq + hk))
        h = _log_int(rng, 1, 128)
        w = _log_int(rng, 1, 128)
        return dict(op=op, type=kind, images=max(1, min(rng.randint(1, 8), rows // (h * w))), height=h, width=w, hq=hq, hk=hk, dim=dim,
                    sections="+".join(str(s) for s in sections), train=train)
    dim = rng.choice([32, 40, 64, 96, 128, 256])
    longest = _log_int(rng, 40, 4500 if kind == "fp32" else 9000)
    lengths = [longest] + [_log_int(rng, 1, longest) for _ in range(rng.randint(0, 6))]
    if rng.random() < 0.3:
        lengths.append(0)
    rng.shuffle(lengths)
    case = dict(op=op, type=kind, hq=hq, hk=hk, dim=dim, causal=rng.random() < 0.5, train=train)
    while True:                                          # no more work than the largest listed case of its kind
        case["lengths"] = "+".join(str(n) for n in lengths)
        if work(case)["flops"] <= (6e10 if kind == "fp32" else 3e11):
            return case
        lengths = [(4 * n + 4) // 5 for n in lengths]


def _ints(text):
    return [int(t) for t in text.split("+")]


def _sizes(case):
    """Element counts of a parameter list: three decades of sizes, as weights beside biases, `elements` in all."""
    n, total = case["tensors"], case["elements"]
    w = [math.exp(-7.0 * ((i * 0.6180339887) % 1.0)) for i in range(n)]
    got = [max(1, int((total - n) * x / sum(w))) for x in w]
    got[0] += max(0, total - sum(got))
    return got


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["type"]]
    if case["op"] == "norm":
        n = sum(_sizes(case))
        return {"bytes": n * size + 4, "flops": 2 * n}
    if case["op"] == "adam":
        n = case["elements"]
        return {"bytes": 7 * n * 4, "flops": 14 * n}
    if case["op"] == "rope":
        t = case["images"] * case["height"] * case["width"]
        n = t * (case["hq"] + case["hk"]) * case["dim"]
        side = 4 * t * len(_ints(case["sections"])) + 8 * case["dim"]
        return {"bytes": n * size * (5 if case["train"] else 2) + side, "flops": n * (22 if case["train"] else 8)}
    lens = _ints(case["lengths"])
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
    t, d = sum(lens), case["dim"]
    rows = t * d * size * (2 * case["hq"] + 2 * case["hk"])                    # q, o and k, v
    return {"bytes": rows * (2 if case["train"] else 1), "flops": 2 * d * pairs * case["hq"] * (7 if case["train"] else 2)}


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _freq(sections, base=10000.0):
    """(frequency of every rotated pair in 64 bits, its axis): pair j of an axis with n pairs turns by base^(-j/n) per position."""
    f = np.concatenate([base ** (-np.arange(n) / max(n, 1)) for n in sections])
    a = np.concatenate([np.full(n, i) for i, n in enumerate(sections)])
    return f, a.astype(np.int64)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt = TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    s = dict(case)
    if own:
        from hsi_dmgasr_amd import ops, train_ops
    if case["op"] in ("norm", "adam"):
        s["grads"] = [(rand(n) * 1e-3).to(dt) for n in _sizes(case)] if case["op"] == "norm" else [rand(case["elements"]) * 1e-3]
        s["max_norm"] = 1.0 if case["elements"] > 2_000_000 else 0.01
        if case["op"] == "adam":
            n = case["elements"]
            s["p"], s["m"], s["v"] = rand(n) * 0.05, rand(n) * 1e-3, rand(n).square() * 1e-6
        if own:
            s["list"] = train_ops.TensorList(s["grads"])
        return s
    if case["op"] == "rope":
        b, h, w, hq, hk, d = (case[k] for k in ("images", "height", "width", "hq", "hk", "dim"))
        sections = _ints(case["sections"])
        t = b * h * w
        grid = torch.meshgrid(*[torch.arange(n, device=dev, dtype=torch.int32) for n in (b, h, w)], indexing="ij")
        flat = torch.stack([g.reshape(-1) for g in grid], dim=1)
        # one axis: the running token index; two: (row, column); three: (band group, row, column)
        s["pos"] = {1: torch.arange(t, device=dev, dtype=torch.int32)[:, None], 2: flat[:, 1:], 3: flat}[len(sections)].contiguous()
        # q | k side by side in one projection's output, as the qkv convolution leaves them
        both = rand(t, hq + hk, d).mul_(2.0).to(dt)
        s["q"], s["k"] = both[:, :hq], both[:, hq:]
        s["wq"], s["wk"] = 1.0 + 0.1 * rand(d), 1.0 + 0.1 * rand(d)
        if case["train"]:
            s["dq"], s["dk"] = rand(t, hq, d).to(dt), rand(t, hk, d).to(dt)
        f, a = _freq(sections)
        s["freq"], s["axis"] = torch.from_numpy(f).to(dev), torch.from_numpy(a).to(dev)
        if own:
            s["axes"] = ops.RotaryAxes(sections, d, base=10000.0, device=dev)
        return s
    lens = _ints(case["lengths"])
    t, hq, hk, d = sum(lens), case["hq"], case["hk"], case["dim"]
    s["q"], s["k"], s["v"] = rand(t, hq, d).to(dt), rand(t, hk, d).to(dt), rand(t, hk, d).to(dt)
    if case["train"]:
        s["do"] = rand(t, hq, d).to(dt)
    s["scale"], s["longest"] = d ** -0.5, max(lens)
    s["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
    if own:
        s["seqs"] = ops.PackedSequences(lens, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "adam": _plain_adam, "rope": _plain_rope, "attn": _plain_attn}[s["op"]](s)


def _run_own(s):
    from hsi_dmgasr_amd import ops
    from hsi_dmgasr_amd import train_ops as T
    if s["op"] == "norm":
        return T.grad_norm(s["list"])
    if s["op"] == "adam":
        clip = T.clip_coef(s["list"], s["max_norm"])
        T.adam_step(s["p"], s["grads"][0], s["m"], s["v"], ADAM["lr"], ADAM["beta1"], ADAM["beta2"], ADAM["eps"], ADAM["step"], clip=clip)
        return {"norm": clip[0], "p": s["p"], "m": s["m"], "v": s["v"]}
    if s["op"] == "rope":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["axes"], eps=EPS)
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = T.qk_norm_rope_bwd(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["axes"], eps=EPS)
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if not s["train"]:
        return {"o": ops.attention_packed(s["q"], s["k"], s["v"], s["seqs"], causal=s["causal"], scale=s["scale"])}
    o, lse = ops.attention_packed(s["q"], s["k"], s["v"], s["seqs"], causal=s["causal"], scale=s["scale"], want_lse=True)
    dq, dk, dv = T.attention_packed_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, s["seqs"], causal=s["causal"], scale=s["scale"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _plain_norm(s):
    return torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()


def _plain_adam(s):
    p, g, m, v = s["p"], s["grads"][0], s["m"], s["v"]
    norm = g.square().sum().sqrt()
    g = g * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    b1, b2 = ADAM["beta1"], ADAM["beta2"]
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).add_(g.square(), alpha=1 - b2)
    rate, inv = ADAM["lr"] / (1 - b1 ** ADAM["step"]), (1 - b2 ** ADAM["step"]) ** -0.5
    p.sub_(rate * m / (v.sqrt() * inv + ADAM["eps"]))
    return {"norm": norm, "p": p, "m": m, "v": v}


def _plain_rope(s):
    angle = s["pos"].double()[:, s["axis"]] * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half, pairs = s["dim"] // 2, s["freq"].numel()

    def turn(x, sin):
        a, b = x[..., :pairs], x[..., half:half + pairs]
        return torch.cat([a * cos - b * sin, x[..., pairs:half], a * sin + b * cos, x[..., half + pairs:]], dim=-1)

    def forward(x, w):
        x = x.float()
        return turn(x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w, sin).to(s["q"].dtype)

    def backward(dy, x, w):
        x = x.float()
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        dn, xhat = turn(dy.float(), -sin), x * r
        g = dn * w
        return (r * (g - xhat * (g * xhat).mean(-1, keepdim=True))).to(s["q"].dtype), (dn * xhat).sum((0, 1))

    out = {"q": forward(s["q"], s["wq"]), "k": forward(s["k"], s["wk"])}
    if s["train"]:
        out["dq"], out["dwq"] = backward(s["dq"], s["q"], s["wq"])
        out["dk"], out["dwk"] = backward(s["dk"], s["k"], s["wk"])
    return out


def _plain_attn(s):
    """Sequences padded to the longest one; the heads of a group folded into the rows of their shared key head."""
    cu, longest, hk, dt = s["cu"], s["longest"], s["hk"], s["q"].dtype
    t, hq, d = s["q"].shape
    n, g = cu.numel() - 1, hq // hk
    at = torch.arange(longest, device=cu.device)
    rows = cu[:-1, None] + at
    valid = rows < cu[1:, None]
    rows = rows.clamp(max=t - 1)
    token = torch.arange(t, device=cu.device)
    seq = torch.bucketize(token, cu[1:], right=True)
    place = seq * longest + token - cu[seq]

    def pad(x, heads):                                  # [T, heads, d] -> [n, hk, (heads / hk) * longest, d]
        x = x.float()[rows] * valid[:, :, None, None]
        return x.reshape(n, longest, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)

    def pack(x, heads):                                 # and back
        x = x.reshape(n, hk, heads // hk, longest, d).permute(0, 3, 1, 2, 4).reshape(n * longest, heads, d)
        return x[place].to(dt)

    q, k, v = pad(s["q"], hq), pad(s["k"], hk), pad(s["v"], hk)
    mask = valid[:, None, :].expand(n, longest, longest)
    if s["causal"]:
        mask = mask & (at[None, :] <= at[:, None])
    mask = mask[:, None, None]
    p = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(n, hk, g, longest, longest).masked_fill_(~mask, torch.finfo(torch.float32).min)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(n, hk, g * longest, longest)
    o = p @ v
    out = {"o": pack(o, hq)}
    if s["train"]:
        do = pad(s["do"], hq)
        ds = do @ v.transpose(2, 3)
        ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
        out["dq"], out["dk"], out["dv"] = pack(ds @ k, hq), pack(ds.transpose(2, 3) @ q, hk), pack(p.transpose(2, 3) @ do, hk)
    return out


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "adam"):
        total = sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"])
        norm = math.sqrt(total)
        if case["op"] == "norm":
            return torch.tensor(norm, dtype=torch.float64)
        b1, b2, t = ADAM["beta1"], ADAM["beta2"], ADAM["step"]
        g = s["grads"][0].double() * min(1.0, s["max_norm"] / (norm + 1e-6))
        m = b1 * s["m"].double() + (1 - b1) * g
        v = b2 * s["v"].double() + (1 - b2) * g * g
        p = s["p"].double() - ADAM["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + ADAM["eps"])
        return {"norm": torch.tensor(norm, dtype=torch.float64), "p": p, "m": m, "v": v}
    return _exact_rope(case, s) if case["op"] == "rope" else _exact_attn(case, s)


def _exact_rope(case, s):
    half = case["dim"] // 2
    f, axis = _freq(_ints(case["sections"]))
    turn = torch.zeros(s["pos"].shape[0], half, dtype=torch.float64, device=s["pos"].device)
    for j, (fj, aj) in enumerate(zip(f, axis)):
        turn[:, j] = s["pos"][:, int(aj)].double() * float(fj)
    z = torch.polar(torch.ones_like(turn), turn)[:, None]                   # a rotation of pair (a, b) is a + ib times this
    out = {}
    for name in ("q", "k"):
        x, w = s[name].double(), s["w" + name].double()
        r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
        y = x * r * w
        c = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * z
        out[name] = torch.cat([c.real, c.imag], -1)
        if case["train"]:
            dy = s["d" + name].double()
            c = torch.complex(dy[..., :half].contiguous(), dy[..., half:].contiguous()) * z.conj()
            dn = torch.cat([c.real, c.imag], -1)
            out["dw" + name] = (dn * x * r).sum((0, 1))
            dn = dn * w
            out["d" + name] = r * dn - x * r ** 3 * ((dn * x).sum(-1, keepdim=True) / case["dim"])
    return out


def _exact_attn(case, s):
    lens, group, scale = _ints(case["lengths"]), case["hq"] // case["hk"], s["scale"]
    pairs = sum(n * n for n in lens) * case["hq"]
    if pairs * case["dim"] * (14 if case["train"] else 4) > 3e13:
        return None
    names = ["q", "k", "v"] + (["do"] if case["train"] else [])
    out = {"o": torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)}
    if case["train"]:
        for n in ("q", "k", "v"):
            out["d" + n] = torch.zeros(s[n].shape, dtype=torch.float64, device=s["q"].device)
    first = 0
    for n in lens:
        to = slice(first, first + n)
        first += n
        for h in range(case["hq"] if n else 0):
            x = {name: s[name][to, h if name in ("q", "do") else h // group].double() for name in names}
            w = torch.mm(x["q"], x["k"].t().contiguous()) * scale
            if case["causal"]:
                w = w.masked_fill(torch.ones(n, n, dtype=torch.bool, device=w.device).triu(1), -math.inf)
            w = torch.exp(w - torch.logsumexp(w, dim=1, keepdim=True))
            o = torch.mm(w, x["v"])
            out["o"][to, h] = o
            if case["train"]:
                dw = torch.mm(x["do"], x["v"].t().contiguous())
                out["dv"][to, h // group] += torch.mm(w.t().contiguous(), x["do"])
                dw = scale * w * (dw - (w * dw).sum(1, keepdim=True))
                out["dq"][to, h] = torch.mm(dw, x["k"])
                out["dk"][to, h // group] += torch.mm(dw.t().contiguous(), x["q"])
    return out
