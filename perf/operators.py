"""Cases of the optimizer-state operators: what they compute, in plain torch, and the calls of this package.

adamw8    one (R)AdamW step of many tensors whose two moments are held in 8 bits (blocks of 128, one scale each)
adamw32   one (R)AdamW step of many 16-bit tensors with fp32 moments and an fp32 master copy of each tensor
momentum8 Nesterov momentum of matrices held in 8 bits, and the normalised 16-bit input of Newton-Schulz
apply32   the orthogonalised update applied to fp32 master weights, and their 16-bit copy

A case's tensors are views of one flat buffer per kind (parameters, gradients, codes, scales), each starting at a
multiple of 128 elements, as a training program that flattens its parameters keeps them.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
M32, M64 = (1 << 32) - 1, (1 << 64) - 1
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BETAS, STEP0 = (0.9, 0.95), 11


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the norm weights of a 32-layer decoder: little work, one launch's latency
        {"name": "adamw8 65 norms", "op": "adamw8", "shapes": "65*4096", "dtype": "bf16", "eps": 0.0, "wd": 0.0,
         "master": False},
        # biases, small convolutions and heads of odd sizes in fp32, with the eps form
        {"name": "adamw8 ragged f32", "op": "adamw8",
         "shapes": "9*64x32x3,9*128,3*2x129,5*257x511,1*1000003,1*8191x129", "dtype": "f32", "eps": 1e-8, "wd": 0.1,
         "master": False},
        # the tied embedding of a small decoder with its fp32 master copy
        {"name": "adamw8 embedding master", "op": "adamw8", "shapes": "1*151936x1024,41*1024", "dtype": "bf16",
         "eps": 1e-8, "wd": 0.1, "master": True},
        # embedding and head of an 8B decoder: the longest pass
        {"name": "adamw8 embedding and head", "op": "adamw8", "shapes": "2*128256x4096,65*4096", "dtype": "bf16",
         "eps": 0.0, "wd": 0.1, "master": False},
        # the norm weights of a 20-layer decoder, fp16, master weights
        {"name": "adamw32 82 norms", "op": "adamw32", "shapes": "42*1024,40*128", "dtype": "f16", "eps": 0.0, "wd": 0.0,
         "master": True},
        # one GPU's even share of odd-sized tensors
        {"name": "adamw32 ragged", "op": "adamw32", "shapes": "7*4099x257,3*1021,2*3000001", "dtype": "bf16",
         "eps": 1e-8, "wd": 0.1, "master": True},
        # a tied embedding with fp32 states and master copy
        {"name": "adamw32 embedding", "op": "adamw32", "shapes": "1*151936x1024", "dtype": "bf16", "eps": 0.0,
         "wd": 0.1, "master": True},
        # many tiny matrices: convolution kernels as batches of matrices and a few heads, fp32
        {"name": "momentum8 small conv", "op": "momentum8",
         "shapes": "6*64x32x3,6*64x64x3,6*128x64x5,6*128x128x3,4*128x128,2*2x128", "dtype": "f32", "x": "f16"},
        # the attention matrices of one layer of a small decoder
        {"name": "momentum8 attention", "op": "momentum8", "shapes": "1*2048x1024,2*1024x1024,1*1024x2048",
         "dtype": "bf16", "x": "f16"},
        # one layer of an 8B decoder
        {"name": "momentum8 decoder layer", "op": "momentum8",
         "shapes": "2*4096x4096,2*1024x4096,2*14336x4096,1*4096x14336", "dtype": "bf16", "x": "f16"},
        # one small matrix with its master copy
        {"name": "apply32 1024x1024", "op": "apply32", "shapes": "1*1024x1024", "dtype": "bf16", "x": "f16", "wd": 0.1},
        # one layer of an 8B decoder with master copies
        {"name": "apply32 decoder layer", "op": "apply32",
         "shapes": "2*4096x4096,2*1024x4096,2*14336x4096,1*4096x14336", "dtype": "bf16", "x": "f16", "wd": 0.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw8", "adamw8", "adamw32", "momentum8", "momentum8", "apply32"])
    matrices = op in ("momentum8", "apply32")
    room = {"adamw8": 500_000_000, "adamw32": 120_000_000, "momentum8": 150_000_000, "apply32": 150_000_000}[op]
    parts, kinds = [], rng.randint(1, 4)
    for _ in range(kinds):
        if matrices or rng.random() < 0.5:
            r, c = _log(rng, 2, 12000), _log(rng, 2, 12000)
            if rng.random() < 0.5:
                r, c = -(-r // 8) * 8, -(-c // 8) * 8
            b = _log(rng, 1, 64) if rng.random() < 0.25 else 1
            numel, text = b * r * c, ("%dx%dx%d" % (b, r, c) if b > 1 else "%dx%d" % (r, c))
        else:
            numel = _log(rng, 1, 200_000_000)
            text = str(numel)
        count = _log(rng, 1, 12 if matrices else 60)
        count = min(count, room // (kinds * numel))
        if count >= 1:
            parts.append("%d*%s" % (count, text))
    if not parts:
        parts = ["1*%dx%d" % (_log(rng, 2, 2000), _log(rng, 2, 2000))]
    case = {"op": op, "shapes": ",".join(parts), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "adamw8":
        master = rng.random() < 0.4
        case.update(eps=rng.choice([0.0, 1e-8]), wd=rng.choice([0.0, 0.1]), master=master)
        if master and case["dtype"] == "f32":
            case["dtype"] = "bf16"
    elif op == "adamw32":
        case.update(eps=rng.choice([0.0, 1e-8]), wd=rng.choice([0.0, 0.1]), master=True,
                    dtype=rng.choice(["bf16", "f16"]))
    elif op == "momentum8":
        case["x"] = rng.choice(["f16", "f16", "bf16"])
    else:
        case.update(dtype=rng.choice(["bf16", "f16"]), x=rng.choice(["f16", "bf16"]), wd=rng.choice([0.0, 0.1]))
    return case


def _shapes(case):
    got = []
    for part in case["shapes"].split(","):
        count, shape = part.split("*")
        got += [tuple(int(n) for n in shape.split("x"))] * int(count)
    return got


def _rows(case, shape):
    """How a tensor's blocks lie: (number of runs, length of a run). A run starts a new block."""
    n = math.prod(shape)
    if case["op"] != "momentum8":
        return 1, n
    return n // (shape[-2] * shape[-1]), shape[-2] * shape[-1]


def work(case):
    el = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    n = sum(math.prod(s) for s in _shapes(case))
    scales = sum(b * -(-k // BLOCK) for b, k in (_rows(case, s) for s in _shapes(case)))
    op = case["op"]
    weights = 8 + el if case.get("master") else 2 * el  # a master copy is read and written, its 16-bit copy written
    if op == "adamw8":
        return {"bytes": n * (el + weights + 4) + 4 * scales, "flops": 30 * n}
    if op == "adamw32":
        return {"bytes": n * (el + weights + 16), "flops": 25 * n}
    if op == "momentum8":
        return {"bytes": n * (el + 2 + 2) + 2 * scales, "flops": 12 * n}
    return {"bytes": n * (2 + 8 + el), "flops": 5 * n}


# ----------------------------------------------------------------------------------------- inputs
def _flat(shapes, dtype, align=BLOCK):
    """One zeroed buffer and a view of it for each shape."""
    starts, total = [], 0
    for s in shapes:
        starts.append(total)
        total += -(-math.prod(s) // align) * align
    buf = torch.zeros(total, dtype=torch.uint8 if "float8" in str(dtype) else dtype, device="cuda")
    buf = buf.view(dtype)
    return buf, [buf[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)]


def _nearest_codes(x, codes, scales):
    """Fills codes [runs, n] and scales [runs, blocks] with x [runs, n] to the nearest value of 8 bits."""
    runs, n = x.shape
    nb = scales.shape[-1]
    pad = torch.zeros((runs, nb * BLOCK), device=x.device)
    pad[:, :n] = x
    blocks = pad.view(runs, nb, BLOCK)
    e = torch.ceil(torch.log2(blocks.abs().amax(-1).clamp_min(1e-30) / E4M3_MAX)) + 127
    e = torch.where(blocks.abs().amax(-1) > 0, e.clamp(0, 254), torch.zeros_like(e))
    scales.view(torch.uint8).copy_(e.to(torch.uint8))
    q = (blocks * torch.exp2(127 - e)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    codes.view(torch.uint8).copy_(q.view(torch.uint8).reshape(runs, nb * BLOCK)[:, :n])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes, dt, op = _shapes(case), DTYPES[case["dtype"]], case["op"]

    def normal(shape):
        return torch.randn(shape, generator=gen, device="cuda")

    st = {"op": op, "wd": case.get("wd", 0.0), "eps": case.get("eps", 0.0), "step": STEP0, "lr": 1e-3,
          "seeds": [(seed * 1000003 + 7919 * i) & M64 for i in range(len(shapes))],
          "x": DTYPES[case.get("x", "f16")], "case": case}
    if op != "apply32":
        st["G"], st["g"] = _flat(shapes, dt)
        for g in st["g"]:
            rows = g.view(g.shape[0], -1) if g.ndim > 1 else g.view(1, -1)
            scale = 1e-4 * torch.exp(0.7 * normal((rows.shape[0], 1)))
            if op != "momentum8" and g.ndim > 1:  # rows of an embedding that no token of the batch touched
                scale = scale * (torch.rand((rows.shape[0], 1), generator=gen, device="cuda") > 0.3)
            rows.copy_(normal(rows.shape).mul_(scale))
    if op != "momentum8":
        st["P"], st["p"] = _flat(shapes, dt)
        if case.get("master") or op == "apply32":
            st["W"], st["w"] = _flat(shapes, torch.float32)
        for i, p in enumerate(st["p"]):
            w = normal(p.shape).mul_(0.02)
            p.copy_(w)
            if "w" in st:
                st["w"][i].copy_(w)
    if op == "apply32":
        st["U"], st["u"] = _flat(shapes, st["x"])
        for u in st["u"]:
            u.copy_(normal(u.shape).mul_(min(u.shape[-2:]) ** 0.5 / (u.shape[-2] * u.shape[-1]) ** 0.5))
        return st
    if op == "adamw32":
        for k in "mv":
            st[k.upper()], st[k] = _flat(shapes, torch.float32)
        for m, v, g in zip(st["m"], st["v"], st["g"]):
            m.copy_(normal(m.shape).mul_(0.3e-4).add_(g, alpha=0.1))
            v.copy_((normal(v.shape).square_().add_(0.1)).mul_(1e-8))
        return st
    runs = [_rows(case, s) for s in shapes]
    for k in "mv" if op == "adamw8" else "m":
        st[k.upper()], st[k] = _flat(shapes, torch.float8_e4m3fn)
        st[k.upper() + "S"], st[k + "s"] = _flat([(b, -(-n // BLOCK)) for b, n in runs], torch.float8_e8m0fnu, 16)
        if op == "adamw8":
            st[k + "s"] = [s.view(-1) for s in st[k + "s"]]
    for i, (b, n) in enumerate(runs):
        m = normal((b, n)).mul_(0.3e-4).add_(st["g"][i].reshape(b, n), alpha=0.1)
        _nearest_codes(m, st["m"][i].view(b, n), st["ms"][i].view(b, -1))
        if op == "adamw8":
            v = (normal((b, n)).square_().add_(0.1)).mul_(1e-8)
            _nearest_codes(v, st["v"][i].view(b, n), st["vs"][i].view(b, -1))
    return st


# ------------------------------------------------------------------------- the plain form's pieces
def _mix64(z):
    z = (z + 0x9E3779B97F4A7C15) & M64
    z = ((z ^ (z >> 32)) * 0x6A09E667F3BCC909) & M64
    z = ((z ^ (z >> 29)) * 0xBB67AE8584CAA73B) & M64
    return z ^ (z >> 32)


def _fold(a, b):
    t = a * b  # the low 64 bits of the product, as a signed number
    return ((t >> 32) & M32) ^ (t & M32)


def _reverse16(v):
    for k, mask in ((8, 0x00FF), (4, 0x0F0F), (2, 0x3333), (1, 0x5555)):
        v = ((v >> k) & mask) | ((v & mask) << k)
    return v


def _fractions(runs, n, seed, dev):
    """The rounding fractions in [0, 1) of each element, [runs, n]: four elements share one 32-bit number."""
    key = _mix64(seed)
    q = torch.arange(-(-n // 4), device=dev)
    hi = (q >> 32)[None] + torch.arange(runs, device=dev)[:, None]
    a = ((q & M32) * 0x9E3779B9 + (key & M32)) & M32
    r = _fold(a[None], a[None] ^ (((key >> 32) ^ hi) & M32))
    r = _fold(r, r ^ 0xBB67AE85)
    lo, up = (r & 0xFFFF).int(), (r >> 16).int()
    four = torch.stack([lo, _reverse16(lo), up, _reverse16(up)], -1).float().div_(65536)
    return four.reshape(runs, -1)[:, :n]


def _power(e):
    """2^(e - 127) for whole numbers 1 <= e <= 254, and 2^-127 for 0; NaN for 255."""
    p = torch.where(e == 0, torch.full_like(e, 0x400000), e.int() << 23).view(torch.float32)
    return torch.where(e == 255, torch.full_like(p, math.nan), p)


def _read8(codes, scales, runs, n):
    s = scales.view(torch.uint8).reshape(runs, -1).int()
    return codes.reshape(runs, n).float() * _power(s).repeat_interleave(BLOCK, 1)[:, :n]


def _write8(x, fractions, codes, scales, positive):
    """Rounds x [runs, n] to 8 bits: up with the probability of its distance; writes codes and scales."""
    runs, n = x.shape
    nb = -(-n // BLOCK)
    a = torch.nn.functional.pad(x.abs(), (0, nb * BLOCK - n)).view(runs, nb, BLOCK)
    top = a.amax(-1)
    f, e = torch.frexp(top)  # top = f 2^e, 1/2 <= f < 1: the smallest power of two with top <= 448 2^k
    e = (torch.where(f > 0.875, e - 8, e - 9) + 127).clamp_min(0).int()
    e = torch.where(top > 0, e, torch.zeros_like(e))
    e = torch.where(torch.isfinite(top), e, torch.full_like(e, 255))
    scales.view(torch.uint8).copy_(e.to(torch.uint8).reshape(scales.shape))
    y = a * _power((254 - e).clamp_min(1))[..., None]
    if positive:  # a second moment stays above zero in a block that is not all zero
        y = torch.where((top > 0)[..., None], y.clamp_min(2.0 ** -9), y)
    y = y.reshape(runs, -1)[:, :n]
    lsb = torch.exp2(torch.frexp(y)[1].sub(1).clamp_min(-6).sub(3).float())
    q = (torch.floor((y / lsb).double() + fractions) * lsb).float()
    q = torch.copysign(q, x).to(torch.float8_e4m3fn)
    codes.view(torch.uint8).copy_(q.view(torch.uint8).reshape(codes.shape))


def _update(m, v, g, step, eps):
    b1, b2 = BETAS
    m = m + (g - m) * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    num, den = m * (1 / (1 - b1 ** step)), torch.sqrt(v * (1 / (1 - b2 ** step)))
    return m, v, (torch.atan2(num, den) if eps == 0 else num / (den + eps))


def _decayed(p, u, lr, wd):
    """p - lr (u + wd p where u and p have one sign)."""
    if wd > 0:
        u = torch.where(u * p >= 0, u + wd * p, u)
    return p - lr * u


def _plain(st):
    x = []
    for i, seed in enumerate(st["seeds"]):
        shape = (st["g"] if "g" in st else st["u"])[i].shape
        runs, n = _rows(st["case"], shape)
        if st["op"] == "apply32":
            w = _decayed(st["w"][i], st["u"][i].float(), st["lr"], st["wd"])
            st["w"][i].copy_(w)
            st["p"][i].copy_(w)
            continue
        g = st["g"][i].reshape(runs, n).float()
        if st["op"] == "adamw32":
            m, v, u = _update(st["m"][i].view(runs, n), st["v"][i].view(runs, n), g, st["step"], st["eps"])
            st["m"][i].copy_(m.view(shape))
            st["v"][i].copy_(v.view(shape))
        else:
            fractions = _fractions(runs, n, seed, g.device)
            m = _read8(st["m"][i], st["ms"][i], runs, n)
            if st["op"] == "momentum8":
                _write8(m * BETAS[1] + g, fractions, st["m"][i], st["ms"][i], False)
                u = g + BETAS[1] * _read8(st["m"][i], st["ms"][i], runs, n)
                norm = torch.sqrt((u * u).sum(-1, keepdim=True, dtype=torch.float64)).float()
                x.append((u / (norm + 1e-8)).to(st["x"]).view(shape))
                continue
            m, v, u = _update(m, _read8(st["v"][i], st["vs"][i], runs, n), g, st["step"], st["eps"])
            _write8(m, fractions, st["m"][i], st["ms"][i], False)
            _write8(v, fractions, st["v"][i], st["vs"][i], True)
            del m, v, fractions
        p = (st["w"] if "w" in st else st["p"])[i]
        p.copy_(_decayed(p.reshape(runs, n).float(), u, st["lr"], st["wd"]).view(shape))
        if "w" in st:
            st["p"][i].copy_(p)
    return x


def _own(st):
    import thorn_b200 as T

    if st["op"] == "momentum8":
        return T.momentum_(st["g"], st["m"], st["ms"], beta=BETAS[1], seeds=st["seeds"], dtype=st["x"])
    if st["op"] == "apply32":
        T.apply_update_(st["p"], st["u"], masters=st["w"], lr=st["lr"], weight_decay=st["wd"])
        return []
    T.adamw_(st["p"], st["g"], st["m"], st["v"], step=st["step"], lr=st["lr"], betas=BETAS, eps=st["eps"],
             weight_decay=st["wd"], moment_scales=st.get("ms"), variance_scales=st.get("vs"), masters=st.get("w"),
             seeds=st["seeds"] if st["op"] == "adamw8" else None)
    return []


def run(st):
    if own:
        x = _own(st)
    else:
        x = _plain(st)
    st["step"] += 1
    st["seeds"] = [(s + 0x9E3779B97F4A7C15) & M64 for s in st["seeds"]]  # fresh numbers for every step
    out = {k: st[k] for k in ("P", "W", "M", "MS", "V", "VS") if k in st}
    if st["op"] == "momentum8":
        out["x"] = list(x)
    return out


# ------------------------------------------------------------------------ the definition, in 64 bits
def _limbs(a, b):
    """High and low 32 bits of a product of two 32-bit numbers, from 16-bit halves."""
    a0, a1, b0, b1 = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    mid = a1 * b0 + (a0 * b0 >> 16)
    mid2 = a0 * b1 + (mid & 0xFFFF)
    return a1 * b1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (a0 * b0 & 0xFFFF)


def _exact_thresholds(runs, n, seed, dev):
    """What the distance to the lower of two neighbouring values must reach for the upper one, [runs, n]."""
    key = _mix64(seed)
    i = torch.arange(4 * -(-n // 4), device=dev)
    run = torch.arange(runs, device=dev)[:, None]
    q = i[::4] >> 2
    a = (_limbs(q & M32, torch.tensor(0x9E3779B9, device=dev))[1] + (key & M32)) & M32
    b = a[None] ^ (((run + (q >> 32)[None]) ^ (key >> 32)) & M32)
    h, l = _limbs(a[None].expand_as(b), b)
    c = h ^ l
    h, l = _limbs(c, c ^ 0xBB67AE85)
    r = h ^ l
    weights = torch.tensor([2.0 ** -(16 - k) for k in range(16)], dtype=torch.float64, device=dev)
    out = torch.empty((runs, q.numel(), 4), dtype=torch.float64, device=dev)
    for lane in range(4):
        part = (r >> (16 * (lane // 2))) & 0xFFFF
        s = torch.zeros(part.shape, dtype=torch.float64, device=dev)
        for k in range(16):
            s += ((part >> k) & 1) * weights[15 - k if lane % 2 else k]
        out[..., lane] = 1 - s
    return out.view(runs, -1)[:, :n]


def _exact_value(scales, runs, n):
    s = scales.view(torch.uint8).reshape(runs, -1).double()
    return torch.exp2(s - 127).repeat_interleave(BLOCK, 1)[:, :n]


def _exact_grid(dev):
    return torch.arange(127, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).double()


def _exact_round(x, thresholds, positive):
    """(values of the codes, values of the scales) of x [runs, n]."""
    runs, n = x.shape
    nb = -(-n // BLOCK)
    grid = _exact_grid(x.device)
    pad = torch.zeros((runs, nb * BLOCK), dtype=torch.float64, device=x.device)
    pad[:, :n] = x.abs()
    top = pad.view(runs, nb, BLOCK).amax(-1)
    k = torch.ceil(torch.log2(top / E4M3_MAX)).clamp(-127, 127)
    k = torch.where(top > E4M3_MAX * torch.exp2(k), k + 1, k)
    k = torch.where((top <= E4M3_MAX * torch.exp2(k - 1)) & (k > -127), k - 1, k)
    k = torch.where(top > 0, k, torch.full_like(k, -127.0))
    size = torch.exp2(k).repeat_interleave(BLOCK, 1)[:, :n]
    y = x.abs() / size
    if positive:
        y = torch.where((top > 0).repeat_interleave(BLOCK, 1)[:, :n], y.clamp_min(2.0 ** -9), y)
    i = (torch.searchsorted(grid, y.contiguous(), right=True) - 1).clamp(0, 125)
    lo = grid[i]
    gap = grid[i + 1] - lo
    q = torch.where((y - lo) / gap >= thresholds, lo + gap, lo)
    return torch.sign(x) * q, torch.exp2(k)


def exact(case, seed):
    st = prepare(case, seed)
    shapes = _shapes(case)
    out = {k: torch.zeros(st[k].shape, dtype=torch.float64, device="cuda")
           for k in ("P", "W", "M", "V") if k in st}
    for k in ("MS", "VS"):
        if k in st:
            out[k] = torch.full(st[k].shape, 2.0 ** -127, dtype=torch.float64, device="cuda")
    (b1, b2), t = BETAS, STEP0
    at, bt, xs = 0, 0, []
    for i, shape in enumerate(shapes):
        n = math.prod(shape)
        runs, length = _rows(case, shape)
        put, nsc = slice(at, at + n), runs * -(-length // BLOCK)
        sput = slice(bt, bt + nsc)
        at += -(-n // BLOCK) * BLOCK
        bt += -(-nsc // 16) * 16
        if st["op"] == "apply32":
            m = v = None
            u = st["u"][i].reshape(-1).double()
        else:
            g = st["g"][i].reshape(runs, length).double()
            if "ms" in st:
                thresholds = _exact_thresholds(runs, length, st["seeds"][i], g.device)
            m = st["m"][i].reshape(runs, length).double()
            m = m * _exact_value(st["ms"][i], runs, length) if "ms" in st else m
            if st["op"] == "momentum8":
                q, s = _exact_round(b2 * m + g, thresholds, False)
                out["M"][put], out["MS"][sput] = q.reshape(-1), s.reshape(-1)
                u = g + b2 * q * s.repeat_interleave(BLOCK, 1)[:, :length]
                xs.append((u / (torch.linalg.vector_norm(u, dim=-1, keepdim=True) + 1e-8)).view(shape))
                continue
            v = st["v"][i].reshape(runs, length).double()
            v = v * _exact_value(st["vs"][i], runs, length) if "vs" in st else v
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.square()
            root = (v / (1 - b2 ** t)).sqrt()
            u = m / (1 - b1 ** t)
            u = (torch.atan2(u, root) if st["eps"] == 0 else u / (root + st["eps"])).reshape(-1)
            if "ms" in st:
                for k, val in (("M", m), ("V", v)):
                    q, s = _exact_round(val, thresholds, k == "V")
                    out[k][put], out[k + "S"][sput] = q.reshape(-1), s.reshape(-1)
                del thresholds, q, s
            else:
                out["M"][put], out["V"][put] = m.reshape(-1), v.reshape(-1)
            del m, v, root, g
        p = (st["w"] if "w" in st else st["p"])[i].reshape(-1).double()
        p = p - st["lr"] * (u + st["wd"] * p * (u * p >= 0))
        out["P"][put] = p
        if "W" in out:
            out["W"][put] = p
    if st["op"] == "momentum8":
        out["x"] = xs
    return out
