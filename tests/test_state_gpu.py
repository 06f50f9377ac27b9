"""Optimizer state in 8 bits and in 32 on the GPU: the operators against float64 restatements
(state_reference.py), and THORN groups that use them.

Error bounds.  fp32 arithmetic: each operation is off by at most 2^-24 of its result.
* m' = m + (g - m) w1: three operations and the constant's rounding on magnitudes up to
  |m| + |g|, so at most 5 * 2^-24 (|m| + |g|); v' likewise at most 5 * 2^-24 v' (all terms positive).
* the update u: numerator and denominator carry at most 8 such errors, division and square root
  (or arc tangent) at most 8 more: 16 * 2^-24 |u|, plus the numerator's absolute error over the
  denominator.  p - lr u adds one operation on |p| and one on |lr u|, then one rounding to the
  parameter's dtype (finfo.eps / 2 of the value).
"""
import math

import numpy as np
import pytest
import torch

import cases as C
import state_reference as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# lengths around the vector (8), the block (128), an iteration (2048) and a chunk (8192)
LENGTHS = [1, 7, 8, 127, 128, 129, 2047, 2049, 8191, 8193, 20011]


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def u8(t):
    return t.view(torch.uint8).cpu().numpy().reshape(-1)


def offset_like(t, shift):
    """A copy of t that starts `shift` elements after an aligned address."""
    buf = torch.zeros(t.numel() + shift, dtype=t.dtype if "float8" not in str(t.dtype) else torch.uint8, device=t.device)
    v = buf.view(t.dtype)[shift:].view(t.shape)
    (v if "float8" not in str(t.dtype) else v.view(torch.uint8)).copy_(
        t if "float8" not in str(t.dtype) else t.view(torch.uint8))
    return v


def make_adam(shapes, dtype, eight, master, shift=0, seed=0):
    from thorn_b200 import multi as M

    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    a = dict(params=[], grads=[], moments=[], variances=[])
    if master:
        a["masters"] = []
    if eight:
        a.update(moment_scales=[], variance_scales=[], seeds=[17 * i + seed for i in range(len(shapes))])
    for s in shapes:
        w, g = rnd(s) * 0.02, (rnd(s) * 1e-3).to(dtype)
        m, v = rnd(s) * 3e-4 + 0.1 * g.float(), (rnd(s).square() + 0.01) * 1e-6
        a["params"].append(offset_like(w.to(dtype), shift))
        a["grads"].append(offset_like(g, shift))
        if master:
            a["masters"].append(offset_like(w, shift))
        for k, x, pos in (("moment", m, False), ("variance", v, True)):
            if eight:
                c, sc = M.state8_write(x, positive=pos)
                a[k + "s"].append(offset_like(c, shift))
                a[k + "_scales"].append(offset_like(sc, shift))
            else:
                a[k + "s"].append(offset_like(x, shift))
    return a


def state_of(a, k, i):
    """float64 values of a moment or variance."""
    if "seeds" in a:
        return R.read(u8(a[k + "s"][i]), u8(a[k + "_scales"][i]))
    return f64(a[k + "s"][i])


def snapshot(a):
    n = len(a["params"])
    w = a.get("masters", a["params"])
    return [(f64(w[i]), f64(a["grads"][i]), state_of(a, "moment", i), state_of(a, "variance", i)) for i in range(n)]


def check_adam(a, before, *, lr, step, betas=(0.9, 0.95), eps=0.0, wd=0.1, degenerate=False):
    for i, (w, g, m, v) in enumerate(before):
        if not w.size:
            continue
        t, rate = (step[i] if isinstance(step, list) else step), (lr[i] if isinstance(lr, list) else lr)
        w2, m2, v2, u = R.adamw(w, g, m, v, lr=rate, step=t, betas=betas, eps=eps, wd=wd, degenerate=degenerate)
        em, ev = 5 * E * (np.abs(m) + np.abs(g)), 5 * E * v2
        if "seeds" in a:
            frac = R.fractions(w.size, a["seeds"][i])
            got_m = R.check_state(m2, em, u8(a["moments"][i]), u8(a["moment_scales"][i]), frac, False, (i, "m"))
            R.check_state(v2, ev, u8(a["variances"][i]), u8(a["variance_scales"][i]), frac, True, (i, "v"))
            assert np.isfinite(got_m).all()
        else:
            assert np.all(np.abs(f64(a["moments"][i]) - m2) <= em + 1e-45)
            assert np.all(np.abs(f64(a["variances"][i]) - v2) <= ev + 1e-45)
        bc1, bc2 = 1 / (1 - betas[0] ** t), 1 / (1 - betas[1] ** t)
        num_err = em * (1 if degenerate else bc1)
        den = 1.0 if degenerate else np.maximum(np.sqrt(v2 * bc2) + eps, np.abs(m2) * bc1 if eps == 0 else 0)
        eu = 16 * E * np.abs(u) + num_err / np.maximum(den, 1e-30)
        ew = rate * eu + 2 * E * (np.abs(w) + rate * np.abs(u))
        # an update whose sign the fp32 error may turn takes or leaves its decay
        ew = ew + np.where(np.abs(u) <= 2 * eu + wd * np.abs(w), rate * wd * np.abs(w), 0) * (np.abs(m2) <= 2 * em)
        if "masters" in a:
            assert np.all(np.abs(f64(a["masters"][i]) - w2) <= ew)
            assert torch.equal(a["params"][i], a["masters"][i].to(a["params"][i].dtype))
        else:
            h = HALF_STEP[a["params"][i].dtype]
            assert np.all(np.abs(f64(a["params"][i]) - w2) <= ew + h * (np.abs(w2) + ew) + 2.0 ** -25)


COMBOS = [(dt, True, False) for dt in DTYPES] + [(dt, True, True) for dt in DTYPES[:2]] + \
    [(dt, False, True) for dt in DTYPES[:2]]


@pytest.mark.parametrize("dtype,eight,master", COMBOS)
@pytest.mark.parametrize("eps,wd", [(0.0, 0.1), (1e-8, 0.0)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_matches_float64(dtype, eight, master, eps, wd, shift):
    """All lengths in one call, an empty tensor among them; aligned and not; two steps."""
    import thorn_b200 as T

    shapes = [(n,) for n in LENGTHS] + [(0,), (3, 5, 77), (64, 131)]
    a = make_adam(shapes, dtype, eight, master, shift)
    for step in (1, 2):
        before = snapshot(a)
        T.adamw_(**a, step=step, lr=1e-2, eps=eps, weight_decay=wd)
        torch.cuda.synchronize()
        check_adam(a, before, lr=1e-2, step=step, eps=eps, wd=wd)
        if eight:
            a["seeds"] = [s + 1000 for s in a["seeds"]]


@pytest.mark.parametrize("eight,master", [(True, False), (False, True)])
def test_adamw_per_tensor_scalars_and_many_tensors(eight, master):
    """More tensors than one launch's table holds, each with its own step and learning rate."""
    import thorn_b200 as T

    n = 701
    a = make_adam([(1 + 3 * (i % 50),) for i in range(n)], torch.bfloat16, eight, master)
    steps, lrs = [1 + i % 7 for i in range(n)], [1e-3 * (1 + i % 5) for i in range(n)]
    before = snapshot(a)
    T.adamw_(**a, step=steps, lr=lrs, betas=(0.8, 0.999))
    torch.cuda.synchronize()
    check_adam(a, before, lr=lrs, step=steps, betas=(0.8, 0.999))


@pytest.mark.parametrize("eight,master", [(True, False), (True, True), (False, True)])
def test_adamw_rectified_first_steps_use_the_moment(eight, master):
    import thorn_b200 as T

    a = make_adam([(300,), (129,)], torch.bfloat16, eight, master)
    before = snapshot(a)
    T.adamw_(**a, step=1, lr=1e-2, rectify=True)  # rect is 0: u = m, and its factor 0 leaves p
    torch.cuda.synchronize()
    check_adam(a, before, lr=0.0, step=1, degenerate=True)


def test_adamw_16_and_32_bit_state_without_masters():
    """State without scales or masters is the step of the framework's own AdamW group, bit for bit."""
    import thorn_b200 as T

    for sdt in (torch.float32, torch.bfloat16):
        torch.manual_seed(4)
        p = [torch.nn.Parameter(torch.randn(n, device="cuda", dtype=torch.bfloat16)) for n in (5, 1000)]
        q = [t.detach().clone() for t in p]
        g = [torch.randn_like(t) for t in q]
        opt = T.THORN([{"orthogonalize": False, "params": p, "lr": 1e-2, "state_dtype": sdt}])
        for t, x in zip(p, g):
            t.grad = x.clone()
        opt.step()
        m, v = [torch.zeros_like(t, dtype=sdt) for t in q], [torch.zeros_like(t, dtype=sdt) for t in q]
        T.adamw_(q, g, m, v, step=1, lr=1e-2)
        for t, x, y in zip(p, q, m):
            assert torch.equal(t.detach(), x) and torch.equal(opt.state[t]["moment"], y)


def test_zero_gradients_and_states():
    """Zero state and gradients stay zero and leave the parameters; a block with one touched
    element keeps the others' first moments at zero and their second above it."""
    import thorn_b200 as T

    p = [torch.ones(300, device="cuda", dtype=torch.bfloat16)]
    g = [torch.zeros_like(p[0])]
    (mc, ms), (vc, vs) = T.state8_zeros(p[0]), T.state8_zeros(p[0])
    kw = dict(lr=1e-2, weight_decay=0.0, moment_scales=[ms], variance_scales=[vs])
    for eps in (0.0, 1e-8):
        T.adamw_(p, g, [mc], [vc], step=1, eps=eps, seeds=[3], **kw)
        assert bool((p[0] == 1).all()) and not u8(mc).any() and not u8(vc).any() and not u8(ms).any()
    g[0][5] = 1e-2
    T.adamw_(p, g, [mc], [vc], step=1, seeds=[4], **kw)
    m, v = T.state8_read(mc, ms), T.state8_read(vc, vs)
    assert float(p[0][5]) < 1 and bool((torch.cat([p[0][:5], p[0][6:]]) == 1).all())
    assert bool((m[128:] == 0).all()) and bool((v[128:] == 0).all()) and bool((v[:128] > 0).all())
    assert int((m[:128] != 0).sum()) == 1


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite(bad):
    """One such gradient makes its own parameter NaN or moves it like any large one, and its
    block's state NaN; nothing else changes."""
    import thorn_b200 as T

    a = make_adam([(1000,)], torch.bfloat16, True, False)
    ref = make_adam([(1000,)], torch.bfloat16, True, False)
    a["grads"][0][200] = bad
    T.adamw_(**a, step=3, lr=1e-2)
    T.adamw_(**ref, step=3, lr=1e-2)
    m, v = (T.state8_read(a[k + "s"][0], a[k + "_scales"][0]) for k in ("moment", "variance"))
    for x in (m, v):
        assert bool(x[128:256].isnan().all()) and not bool(x[:128].isnan().any()) and not bool(x[256:].isnan().any())
    same = torch.ones(1000, dtype=torch.bool)
    same[200] = False
    assert torch.equal(a["params"][0].cpu()[same], ref["params"][0].cpu()[same])
    keep = torch.cat([torch.arange(128), torch.arange(256, 1000)])
    assert torch.equal(m.cpu()[keep], T.state8_read(ref["moments"][0], ref["moment_scales"][0]).cpu()[keep])
    g = [torch.full((40, 40), bad, device="cuda")]
    c, s = T.state8_zeros(g[0], per_matrix=True)
    x = T.momentum_(g, [c], [s], beta=0.9, seeds=[1])[0]
    assert bool(x.isnan().all()) and bool(T.state8_read(c, s).isnan().all())


def test_extreme_magnitudes():
    """Moments near the ends of the range keep finite scales and values."""
    import thorn_b200 as T

    for mag in (1e-25, 1e-18, 1e15):
        p = [torch.zeros(256, device="cuda")]
        g = [torch.randn(256, device="cuda") * mag]
        (mc, ms), (vc, vs) = T.state8_zeros(p[0]), T.state8_zeros(p[0])
        T.adamw_(p, g, [mc], [vc], step=1, lr=1.0, weight_decay=0.0, moment_scales=[ms], variance_scales=[vs], seeds=[9])
        m2, v2 = 0.1 * f64(g[0]), 0.05 * f64(g[0]) ** 2
        frac = R.fractions(256, 9)
        R.check_state(m2, 5 * E * np.abs(f64(g[0])), u8(mc), u8(ms), frac, False, (mag, "m"))
        if mag > 1e-20:  # below, g^2 is under the smallest fp32 number
            R.check_state(v2, 5 * E * v2 + 2.0 ** -149, u8(vc), u8(vs), frac, True, (mag, "v"))
        assert bool(p[0].isfinite().all()) and float(p[0].abs().max()) <= math.pi / 2 + 1e-6


def test_rounding_is_unbiased_and_seeded():
    """The mean of a second moment over many seeds is its value (a decay of 0.1 % per step, far
    under half a code's step, is kept), within 5 standard deviations; equal seeds, equal bits."""
    import thorn_b200 as T

    n, reps = 4096, 64
    p = torch.zeros(n, device="cuda")
    v0 = (torch.rand(n, device="cuda") + 0.5) * 1e-6
    c0, s0 = T.state8_write(v0, positive=True)
    before = T.state8_read(c0, s0).double()
    z, zs = T.state8_zeros(p)
    total = torch.zeros(n, dtype=torch.float64, device="cuda")
    last = None
    for r in list(range(reps)) + [reps - 1]:
        c, s = c0.clone(), s0.clone()
        T.adamw_([p], [torch.zeros_like(p)], [z], [c], step=1, lr=0.0, betas=(0.9, 0.999), moment_scales=[zs],
                 variance_scales=[s], seeds=[r])
        now = u8(c).copy()
        if r == reps - 1 and last is not None:
            assert np.array_equal(now, last)
            break
        last = now if r == reps - 1 else None
        total += T.state8_read(c, s).double()
    # a code's step is at most 2^-3 of its value, hit with probability p <= 0.001 * 2^4 = 0.016
    sd = (before * 2.0 ** -3).square().mean().sqrt() * math.sqrt(0.016 / (n * reps))
    assert abs(float((total / reps - 0.999 * before).mean())) <= 5 * float(sd)


def make_matrices(shapes, dtype, seed=0):
    from thorn_b200 import multi as M

    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = [(torch.randn(s, generator=gen, device="cuda") * 1e-3).to(dtype) for s in shapes]
    m = [torch.randn(s, generator=gen, device="cuda") * 5e-3 for s in shapes]
    st = [M.state8_write(t, per_matrix=True) for t in m]
    return g, [c for c, _ in st], [s for _, s in st]


def check_momentum(g, before, codes, scales, x, beta, seed, xdt):
    B, rc = int(np.prod(g.shape[:-2])), g.shape[-2] * g.shape[-1]
    gv, mv = f64(g).reshape(B, rc), before.reshape(B, rc)
    cs, ss, xs = u8(codes).reshape(B, rc), u8(scales).reshape(B, -1), f64(x).reshape(B, rc)
    for b in range(B):
        want = beta * mv[b] + gv[b]
        err = 3 * E * (np.abs(mv[b]) + np.abs(gv[b]))
        new = R.check_state(want, err, cs[b], ss[b], R.fractions(rc, seed, run=b), False, (tuple(g.shape), b))
        u = gv[b] + beta * new
        norm = np.linalg.norm(u)
        # u: three roundings; the norm's sum of rc squares in trees of fp32 partials: under 2^6 * 2^-24
        tol = (HALF_STEP[xdt] + 2.0 ** 6 * E) * np.abs(u) / norm + 3 * E * (np.abs(gv[b]) + np.abs(new)) / norm
        tiny = 2.0 ** -25 if xdt == torch.float16 else 0.0  # half of fp16's smallest step
        assert np.all(np.abs(xs[b] - u / (norm + 1e-8)) <= tol + tiny), (tuple(g.shape), b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("xdt", [torch.float16, torch.bfloat16])
def test_momentum_matches_float64(dtype, xdt):
    """Matrices and stacks whose sizes do and do not divide by the vector and the block, one
    longer than a chunk, an empty one; two steps."""
    import thorn_b200 as T

    shapes = [(1, 1), (2, 3), (8, 16), (5, 7, 9), (4, 6, 8), (2, 3, 5, 13), (129, 127), (65, 128), (3, 65, 200),
              (0, 4), (130, 513)]
    g, m, s = make_matrices(shapes, dtype)
    for step in range(2):
        before = [np.concatenate([R.read(c, b) for c, b in zip(u8(t).reshape(int(np.prod(t.shape[:-2])), -1),
                                                               u8(r).reshape(r.shape[0], -1))])
                  if t.numel() else None for t, r in zip(m, s)]
        seeds = [100 * step + i for i in range(len(shapes))]
        x = T.momentum_(g, m, s, beta=0.95, seeds=seeds, dtype=xdt)
        torch.cuda.synchronize()
        for i in range(len(shapes)):
            assert x[i].shape == g[i].shape and x[i].dtype is xdt
            if g[i].numel():
                check_momentum(g[i], before[i], m[i], s[i], x[i], 0.95, seeds[i], xdt)


def test_momentum_large_and_reproducible():
    """A matrix of many chunks (its norm is summed by a launch of its own): unit Frobenius norm,
    the same bits twice; and a stack of one-element matrices."""
    import thorn_b200 as T

    runs = []
    for _ in range(2):
        g, m, s = make_matrices([(1500, 2049), (5000, 1, 1)], torch.bfloat16, seed=5)
        x = T.momentum_(g, m, s, beta=0.95, seeds=[1, 2])
        runs.append((x, m, s))
        # rounding to fp16 adds an independent relative error of at most 2^-11 per element
        assert abs(float(x[0].double().norm()) - 1) <= 2.0 ** -11
        # one-element matrices: u / (|u| + 1e-8)
        u = g[1].double() + 0.95 * T.state8_read(m[1], s[1]).double()
        assert torch.allclose(x[1].double(), u / (u.abs() + 1e-8), rtol=2.0 ** -10, atol=2.0 ** -24)
    for a, b in zip(runs[0], runs[1]):
        for p, q in zip(a, b):
            assert np.array_equal(u8(p), u8(q))


@pytest.mark.parametrize("xdt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pdt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_apply_matches_float64(xdt, pdt, wd):
    import thorn_b200 as T

    torch.manual_seed(6)
    shapes = [(1, 1), (3, 5, 7), (64, 130), (0, 3), (100, 205)]
    w = [torch.randn(s, device="cuda") * 0.02 for s in shapes]
    p = [t.to(pdt) for t in w]
    u = [(torch.randn(s, device="cuda") * 0.05).to(xdt) for s in shapes]
    lrs = [0.1 * (i + 1) for i in range(len(shapes))]
    before = [f64(t) for t in w]
    T.apply_update_(p, u, masters=w, lr=lrs, weight_decay=wd)
    for i in range(len(shapes)):
        uv = f64(u[i])
        uv = np.where(uv * before[i] >= 0, uv + wd * before[i], uv) if wd else uv
        tol = 4 * E * (np.abs(before[i]) + lrs[i] * np.abs(uv))
        assert np.all(np.abs(f64(w[i]) - (before[i] - lrs[i] * uv)) <= tol)
        assert torch.equal(p[i], w[i].to(pdt))


@pytest.mark.parametrize("shape", [(3, 7, 5), (2, 33, 16), (1, 129, 40)])
@pytest.mark.parametrize("fold", [False, True])
def test_apply_with_row_factors(shape, fold):
    """The per-neuron factors of the C entry: row_scale alone, or with the matrix statistics."""
    from thorn_b200 import _native as N
    from thorn_b200 import multi as M

    torch.manual_seed(7)
    B, Rr, Cc = shape
    U = torch.randn(shape, device="cuda").half()
    w = torch.randn(shape, device="cuda") * 0.02
    p = w.bfloat16()
    rs = torch.rand(B * Rr, device="cuda") + 0.5
    st = torch.rand(B, 2, device="cuda") + 0.5
    w0 = w.double()
    M.launch_apply([(U.data_ptr(), p.data_ptr(), w.data_ptr(), rs.data_ptr(), 0 if fold else st.data_ptr(), B, Rr, Cc,
                     0.1)], torch.float16, torch.bfloat16, 0.1, N.stream_of(U.device))
    f = rs.double().view(B, Rr, 1)
    if not fold:
        f = f * (st[:, 0].double().sqrt() / st[:, 1].double().sqrt()).view(B, 1, 1)
    u = U.double() * f
    u = torch.where(u * w0 >= 0, u + 0.1 * w0, u)
    want = w0 - 0.1 * u
    # the factor: five operations; the product, decay and update four more
    assert bool(((w.double() - want).abs() <= 10 * E * (w0.abs() + 0.1 * u.abs())).all())
    assert torch.equal(p, w.bfloat16())


def test_other_stream_and_neighbours_untouched():
    """Work queued on the current stream, not the default one; memory around the tensors stays."""
    import thorn_b200 as T

    n = 1003
    buf = torch.full((n + 64,), 7.0, device="cuda", dtype=torch.bfloat16)
    p, g = buf[32:32 + n], torch.full((n,), 1e-3, device="cuda", dtype=torch.bfloat16)
    codes = torch.full((n + 64,), 0x55, dtype=torch.uint8, device="cuda")
    c = [codes.view(torch.float8_e4m3fn)[32:32 + n], torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)]
    codes[32:32 + n] = 0
    sc = [torch.zeros(8, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(20_000_000)  # the step must wait for this stream's earlier work
        g.mul_(2.0)
        T.adamw_([p], [g], [c[0]], [c[1]], step=1, lr=1e-2, weight_decay=0.0, moment_scales=[sc[0]],
                 variance_scales=[sc[1]], seeds=[1])
    st.synchronize()
    m = T.state8_read(c[0], sc[0])
    # 0.1 * 2e-3 rounded to one of its two neighbouring codes: at most a step of 2^-3
    assert bool(((m - 2e-4 * 1.0).abs() <= 2e-4 * (2.0 ** -3 + 2.0 ** -8)).all())
    assert bool((buf[:32] == 7).all()) and bool((buf[32 + n:] == 7).all())
    assert bool((codes[:32] == 0x55).all()) and bool((codes[32 + n:] == 0x55).all())


def test_capture_is_refused():
    import thorn_b200 as T

    a = make_adam([(64,)], torch.bfloat16, True, False)
    g, m, s = make_matrices([(8, 8)], torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="capture"):
            T.adamw_(**a, step=1, lr=1e-3)
        with pytest.raises(RuntimeError, match="capture"):
            T.momentum_(g, m, s, beta=0.9, seeds=[1])
    graph.replay()
    torch.cuda.synchronize()
