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
# lengths around the vector (8), the block (128), a warp's segment (1024) and a chunk (4096)
LENGTHS = [1, 7, 8, 127, 128, 129, 1023, 1025, 2047, 4095, 4097, 8191, 8193, 20011]


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
    for eps in (0.0, 1e-8, 1e-40):
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

    shapes = [(1, 1), (2, 3), (8, 16), (5, 7, 9), (70, 6, 8), (2, 3, 5, 13), (9, 15, 17), (9, 30, 30), (3, 40, 40),
              (2, 64, 64), (129, 127), (65, 128), (3, 65, 200), (0, 4), (130, 513)]
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


@pytest.mark.parametrize("shape", [(20, 7, 9), (9, 13, 20), (5, 30, 30), (3, 50, 70), (2, 130, 130), (1, 700, 1101)])
def test_momentum_with_padded_rows(shape):
    """Rows of a longer leading dimension (the Newton-Schulz operand's) hold what the plain
    layout holds, and the padding stays as it was."""
    import thorn_b200 as T
    from thorn_b200 import _native as N
    from thorn_b200 import multi as M

    B, R_, C_ = shape
    g, m, s = make_matrices([shape], torch.bfloat16, seed=3)
    m2, s2 = [t.clone() for t in m], [t.clone() for t in s]
    x, = T.momentum_(g, m, s, beta=0.9, seeds=[4])
    ld = int(N.load().thorn_ns_ld(C_)) + 8
    X = torch.full((B, R_, ld), 9.0, dtype=torch.float16, device="cuda")
    M.launch_momentum8([(g[0].data_ptr(), m2[0].data_ptr(), s2[0].data_ptr(), X.data_ptr(), B, R_, C_, ld, 4)],
                       torch.bfloat16, torch.float16, 0.9, X.device, N.stream_of(X.device))
    assert torch.equal(X[:, :, :C_], x) and bool((X[:, :, C_:] == 9).all())
    assert np.array_equal(u8(m[0]), u8(m2[0])) and np.array_equal(u8(s[0]), u8(s2[0]))
    # the momentum alone writes the same state
    g3, m3, s3 = make_matrices([shape], torch.bfloat16, seed=3)
    M.launch_momentum8([(g3[0].data_ptr(), m3[0].data_ptr(), s3[0].data_ptr(), 0, B, R_, C_, C_, 4)],
                       torch.bfloat16, torch.float16, 0.9, X.device, N.stream_of(X.device))
    assert np.array_equal(u8(m[0]), u8(m3[0])) and np.array_equal(u8(s[0]), u8(s3[0]))


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


def test_offsets_beyond_32_bits():
    """2^32 + 5000 elements: the tail is updated with the random numbers of its own place, and what
    lies before it stays zero.  The tail starts inside a block."""
    import thorn_b200 as T

    n, tail = (1 << 32) + 5000, 4936
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 30 GB")
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    torch.manual_seed(12)
    g[n - tail:] = (torch.randn(tail, device="cuda") * 1e-3).bfloat16()
    (mc, ms), (vc, vs) = T.state8_zeros(p), T.state8_zeros(p)
    T.adamw_([p], [g], [mc], [vc], step=1, lr=1e-2, weight_decay=0.0, moment_scales=[ms], variance_scales=[vs], seeds=[6])
    at = (n - tail) // 128 * 128  # the block that the tail starts in
    x = f64(g[at:])
    frac = R.fractions(n - at, 6, start=at)
    m2, v2 = 0.1 * x, 0.05 * x * x
    R.check_state(m2, 5 * E * np.abs(x), u8(mc[at:]), u8(ms[at // 128:]), frac, False, "m")
    R.check_state(v2, 5 * E * v2, u8(vc[at:]), u8(vs[at // 128:]), frac, True, "v")
    assert bool((p[n - tail:][g[n - tail:] != 0] != 0).all())
    assert int(torch.count_nonzero(mc[:at].view(torch.int64))) == 0 and int(torch.count_nonzero(p[:at].view(torch.int64))) == 0


def test_two_streams_at_once():
    """Calls on two streams, each with its own tensors and scratch, give what they give alone."""
    import thorn_b200 as T

    shapes = [(300, 400), (6, 90, 70), (40, 30)]
    want, got = [], []
    for together in (False, True):
        sets = [make_matrices(shapes, torch.bfloat16, seed=20 + k) for k in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        out = [None, None]
        for step in range(3):
            for k in range(2):
                g, m, s = sets[k]
                with torch.cuda.stream(streams[k]):
                    out[k] = T.momentum_(g, m, s, beta=0.9, seeds=[step, step + 10, step + 20])
                if not together:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        (got if together else want).extend([u8(t).copy() for k in range(2) for t in out[k] + sets[k][1] + sets[k][2]])
    for a, b in zip(want, got):
        assert np.array_equal(a, b)


def test_mixed_parameter_types_in_one_group():
    """fp32, bf16 and fp16 parameters of one group with 8-bit state, a scalar and an empty one
    among the AdamW ones."""
    import thorn_b200 as T

    for ortho, shapes in ((True, [(20, 30), (20, 30), (20, 30)]), (False, [(50,), (), (0,), (7, 9)])):
        dts = [torch.float32, torch.bfloat16, torch.float16, torch.bfloat16][:len(shapes)]
        p = [torch.nn.Parameter((torch.randn(s, device="cuda") * 0.02).to(d)) for s, d in zip(shapes, dts)]
        before = [t.detach().clone() for t in p]
        opt = T.THORN([{"orthogonalize": ortho, "params": p, "lr": 1e-2, "state_dtype": F8, "master_weights": True}])
        for t in p:
            t.grad = torch.ones_like(t) * 1e-3 + torch.arange(t.numel(), device="cuda").reshape(t.shape).to(t.dtype) * 1e-5
        opt.step()
        for t, b, d in zip(p, before, dts):
            assert ("master" in opt.state[t]) == (d is not torch.float32)
            assert bool(t.isfinite().all()) and (t.numel() == 0 or not torch.equal(t.detach(), b))


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


# ---------------------------------------------------------------------------------- THORN groups
F8 = torch.float8_e4m3fn


def _params(shapes, dtype, seed):
    torch.manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, device="cuda") * 0.02).to(dtype)) for s in shapes]


def _grads(params, seed):
    torch.manual_seed(seed)
    return [(torch.randn(p.shape, device="cuda") * 1e-3).to(p.dtype) for p in params]


@pytest.mark.parametrize("opts", [dict(state_dtype=F8), dict(state_dtype=F8, master_weights=True),
                                  dict(master_weights=True), dict(state_dtype=F8, rectify=True, eps=1e-8)])
def test_adam_group_steps_like_the_function(opts):
    """Four steps of a (R)AdamW group are four calls of adamw_, bit for bit."""
    import thorn_b200 as T

    shapes = [(1000,), (33, 130), (5,)]
    p = _params(shapes, torch.bfloat16, 1)
    q = [t.detach().clone() for t in p]
    opt = T.THORN([{"orthogonalize": False, "params": p, "lr": 1e-2, **opts}])
    kw = {k: opts[k] for k in ("rectify", "eps") if k in opts}
    if "master_weights" in opts:
        kw["masters"] = [t.float() for t in q]
    if "state_dtype" in opts:
        st = [T.state8_zeros(t) for t in q + q]
        m, v = [c for c, _ in st[:3]], [c for c, _ in st[3:]]
        kw.update(moment_scales=[s for _, s in st[:3]], variance_scales=[s for _, s in st[3:]])
    else:
        m, v = [torch.zeros(s, device="cuda") for s in shapes], [torch.zeros(s, device="cuda") for s in shapes]
    for step in range(1, 5):
        g = _grads(p, 10 + step)
        for t, x in zip(p, g):
            t.grad = x.clone()
        opt.step()
        seeds = [(i << 32) + step for i in range(3)] if "state_dtype" in opts else None
        T.adamw_(q, g, m, v, step=step, lr=1e-2, seeds=seeds, **kw)
        for i, t in enumerate(p):
            assert torch.equal(t.detach(), q[i]), (step, i)
            assert np.array_equal(u8(opt.state[t]["moment"]), u8(m[i]))
            assert np.array_equal(u8(opt.state[t]["variance"]), u8(v[i]))
            if "masters" in kw:
                assert torch.equal(opt.state[t]["master"], kw["masters"][i])


def _newton_schulz(x, conf):
    """The library's Newton-Schulz result for the inputs x (matrices or stacks), in x's dtype."""
    import ctypes

    from thorn_b200 import _native as N

    lib = N.load()
    R_, C_ = x.shape[-2:]
    B = x.numel() // (R_ * C_)
    ld = int(lib.thorn_ns_ld(C_))
    X = torch.zeros((B, R_, ld), dtype=x.dtype, device="cuda")
    X[:, :, :C_] = x.reshape(B, R_, C_)
    out = torch.empty((B, R_, C_), dtype=x.dtype, device="cuda")
    wsb = int(lib.thorn_ns_workspace_bytes(B, R_, C_))
    ws = torch.empty(max(256, wsb), dtype=torch.uint8, device="cuda")
    co = (ctypes.c_double * (3 * conf.iters))(*[v for abc in conf.coeffs[:conf.iters] for v in abc])
    rs = (ctypes.c_int32 * max(1, len(conf.restarts)))(*conf.restarts)
    N.check(lib.thorn_ns_batched(X.data_ptr(), out.data_ptr(), ws.data_ptr(), wsb, B, R_, C_, N.dtype_code(x.dtype), co,
                                 conf.iters, rs, len(conf.restarts), None, N.stream_of(X.device)), "ns_batched")
    return out.reshape(x.shape)


@pytest.mark.parametrize("ns_dtype", [torch.float16, torch.bfloat16])
def test_ortho_group_with_8_bit_momentum_and_masters(ns_dtype):
    """Two steps: the momentum is momentum_'s bit for bit, and the masters move by the library's
    Newton-Schulz result for momentum_'s input, up to the fp32 roundings of the apply (one
    matrix has rows that need padding, one stack has 3 dimensions); the parameter is the
    rounded master."""
    import thorn_b200 as T
    from thorn_b200.optimizer import GroupConfig

    shapes = [(64, 96), (40, 37), (3, 16, 24), (128, 256)]
    p = _params(shapes, torch.bfloat16, 2)
    opt = T.THORN([{"orthogonalize": True, "params": p, "lr": 1e-2, "weight_decay": 0.0, "betas": (0.9, 0.0),
                    "state_dtype": F8, "master_weights": True}])
    opt.ns_dtype = ns_dtype
    conf = GroupConfig.from_kwargs(**opt.param_groups[0])
    st = [T.state8_zeros(t, per_matrix=True) for t in p]
    for step in range(1, 3):
        g = _grads(p, 20 + step)
        before = [opt.state[t]["master"].clone() if step > 1 else t.detach().float() for t in p]
        for t, x in zip(p, g):
            t.grad = x.clone()
        opt.step()
        x = T.momentum_(g, [c for c, _ in st], [s for _, s in st], beta=0.9, dtype=ns_dtype,
                        seeds=[(i << 32) + step for i in range(4)])
        for i, t in enumerate(p):
            s = opt.state[t]
            assert np.array_equal(u8(s["moment"]), u8(st[i][0])) and np.array_equal(u8(s["moment_scale"]), u8(st[i][1]))
            lr = 1e-2 * conf.lr_scale(*t.shape[-2:])
            want = before[i].double() - lr * _newton_schulz(x[i], conf).double()
            # the rate rounded to fp32, one fma
            assert bool(((s["master"] - want).abs() <= 2 * E * (before[i].abs() + (want - before[i]).abs())).all()), (step, i)
            assert torch.equal(t.detach(), s["master"].bfloat16())
    assert not opt.device_error()


def test_masters_follow_fp32_parameters():
    """bf16 parameters with masters against fp32 parameters of the same values and gradients:
    both groups' masters are the fp32 run's parameters up to fp32 rounding (tall matrices with
    their per-neuron norm among them)."""
    import thorn_b200 as T

    ortho, adam = [(96, 64), (64, 64), (257, 40)], [(500,), (10, 30)]
    a = _params(ortho + adam, torch.bfloat16, 3)
    b = [torch.nn.Parameter(t.detach().float()) for t in a]

    def make(ps, **kw):
        return T.THORN([{"orthogonalize": True, "params": ps[:3], "lr": 1e-2, **kw},
                        {"orthogonalize": False, "params": ps[3:], "lr": 1e-2, **kw}])

    oa, ob = make(a, master_weights=True), make(b)
    start = [t.detach().clone() for t in b]
    for step in range(3):
        for t, u, x in zip(a, b, _grads(a, 30 + step)):
            t.grad, u.grad = x.clone(), x.float()
        oa.step()
        ob.step()
    for i, (t, u) in enumerate(zip(a, b)):
        m = oa.state[t]["master"]
        assert oa.state[t]["moment"].dtype is torch.float32
        moved = (u.detach() - start[i]).abs()
        # AdamW: the update's arithmetic differs by at most 16 roundings per step; the apply of the
        # orthogonalised group is the same arithmetic
        assert bool(((m - u.detach()).abs() <= 3 * 16 * E * (u.detach().abs() + moved + 1e-2)).all()), i
        assert torch.equal(t.detach(), m.bfloat16())


def test_8_bit_state_survives_saving():
    """Four steps against two, a save, a load into a new optimizer and two: the same bits."""
    import thorn_b200 as T

    shapes = [(48, 64), (200,)]

    def make():
        p = _params(shapes, torch.bfloat16, 4)
        return p, T.THORN([{"orthogonalize": True, "params": p[:1], "lr": 1e-2, "state_dtype": F8, "master_weights": True},
                           {"orthogonalize": False, "params": p[1:], "lr": 1e-2, "state_dtype": F8}])

    def run(p, opt, steps):
        for k in steps:
            for t, x in zip(p, _grads(p, 40 + k)):
                t.grad = x
            opt.step()

    p, opt = make()
    run(p, opt, range(4))
    q, opt2 = make()
    run(q, opt2, range(2))
    saved = opt2.state_dict()
    r, opt3 = make()
    for t, u in zip(r, q):
        t.data.copy_(u.data)
    opt3.load_state_dict(saved)
    run(r, opt3, range(2, 4))
    for t, u in zip(p, r):
        assert torch.equal(t.detach(), u.detach())
        for k, v in opt.state[t].items():
            if isinstance(v, torch.Tensor):
                assert np.array_equal(u8(v), u8(opt3.state[u][k])), k


@pytest.mark.parametrize("ortho", [True, False])
def test_update_rate_advances_the_state_only(ortho):
    import thorn_b200 as T

    p = _params([(64, 200)], torch.bfloat16, 5)
    opt = T.THORN([{"orthogonalize": ortho, "params": p, "lr": 1e-2, "state_dtype": F8, "master_weights": True}])
    opt._update_rate = 2
    moved, codes = [], []
    for k in range(4):
        before = p[0].detach().clone()
        p[0].grad = _grads(p, 50 + k)[0]
        opt.step()
        moved.append(not torch.equal(before, p[0].detach()))
        codes.append(u8(opt.state[p[0]]["moment"]).copy())
    assert moved == [True, False, True, False]  # applied where (step + 1) is a multiple of the rate
    assert all(not np.array_equal(a, b) for a, b in zip(codes, codes[1:]))


@pytest.mark.parametrize("ortho", [True, False])
def test_decoupled_magnitudes_and_magma_with_8_bit_state(ortho):
    """decouple_md and momentum_align with 8-bit state.  From zero state and unit gains the
    first momentum is (1 - beta1 for AdamW, 1 for the orthogonalised group) times the gradient to
    within a code's step (2^-3 of the value), and the steps stay finite and move the parameters."""
    import thorn_b200 as T

    torch.manual_seed(9)
    p = _params([(64, 48), (40, 56)], torch.float32, 6)
    g = _grads(p, 60)
    opt = T.THORN([{"orthogonalize": ortho, "params": p, "lr": 1e-2, "decouple_md": True, "momentum_align": True,
                    "state_dtype": F8, "betas": (0.9, 0.95)}])
    before = [t.detach().clone() for t in p]
    for k in range(3):
        for t, x in zip(p, g):
            t.grad = x.clone()
        opt.step()
        if k == 0:
            for t, x in zip(p, g):
                m = T.state8_read(opt.state[t]["moment"], opt.state[t]["moment_scale"])
                want = x if ortho else 0.1 * x
                size = opt.state[t]["moment_scale"].float().max()
                # a gain of softplus(0.5413) = 1 to a rounding
                assert bool(((m - want).abs() <= want.abs() * (2.0 ** -3 + 2.0 ** -10) + size * 2.0 ** -9).all())
    assert all(bool(t.isfinite().all()) for t in p)
    assert any(not torch.equal(t.detach(), b) for t, b in zip(p, before))


def test_functions_chained_as_one_step():
    """momentum_ -> polar_decomp -> apply_update_ beside adamw_: two steps of a small model by the
    functions alone land where THORN's groups do (2e-2 of the movement in the Frobenius norm for
    the matrix, as the other Newton-Schulz tests: the operator normalises its input once more)."""
    import thorn_b200 as T
    from thorn_b200.optimizer import GroupConfig

    p = _params([(64, 96), (96,)], torch.bfloat16, 8)
    w0 = p[0].detach().float()
    opts = dict(lr=1e-2, state_dtype=F8, master_weights=True)
    opt = T.THORN([{"orthogonalize": True, "params": p[:1], **opts}, {"orthogonalize": False, "params": p[1:], **opts}])
    conf = GroupConfig.from_kwargs(**opt.param_groups[0])
    flat = [float(x) for abc in conf.coeffs[:conf.iters] for x in abc]
    a, b = [t.detach().clone() for t in p]
    wa, wb = a.float(), b.float()
    (mc, ms), (nc, ns), (vc, vs) = T.state8_zeros(a, per_matrix=True), T.state8_zeros(b), T.state8_zeros(b)
    for step in range(1, 3):
        ga, gb = _grads(p, 80 + step)
        p[0].grad, p[1].grad = ga.clone(), gb.clone()
        opt.step()
        x, = T.momentum_([ga], [mc], [ms], beta=0.9, seeds=[step])
        u = torch.ops.thorn_b200.polar_decomp(x, flat, list(conf.restarts))
        T.apply_update_([a], [u], masters=[wa], lr=1e-2 * conf.lr_scale(64, 96), weight_decay=0.1)
        T.adamw_([b], [gb], [nc], [vc], step=step, lr=1e-2, moment_scales=[ns], variance_scales=[vs], masters=[wb],
                 seeds=[(1 << 32) + step])
    assert torch.equal(b, p[1].detach()) and torch.equal(wb, opt.state[p[1]]["master"])
    moved = opt.state[p[0]]["master"] - w0
    assert C.rel_fro((wa - w0).cpu().numpy(), moved.cpu().numpy()) <= 2e-2


def _separately_rounded(kind, m, v, g, beta, w):
    """The new state in torch's fp32, one rounding per operation (the products with powers of
    two are exact)."""
    if kind == "momentum":
        return m * beta + g, None
    return m + (g - m) * w[0], v * beta + g * g * w[1]


def test_state_codes_are_those_of_separate_fp32_operations():
    """2^22 elements: the new scales are those of the fp32 state formed operation by operation,
    and every code is one of its two neighbours: the upper one exactly where the fraction asks."""
    import thorn_b200 as T

    n = 1 << 22
    torch.manual_seed(11)
    g = (torch.randn(n, device="cuda") * 1e-3).bfloat16()
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    mc, ms = T.state8_write(torch.randn(n, device="cuda") * 3e-4 + 0.1 * g.float())
    vc, vs = T.state8_write(torch.randn(n, device="cuda").square() * 1e-6, positive=True)
    mat = [t.view(2048, 2048) for t in (g, mc.clone())] + [ms.clone().view(1, -1)]
    m0, v0 = T.state8_read(mc, ms), T.state8_read(vc, vs)
    m1, v1 = _separately_rounded("adam", m0, v0, g.float(), 0.95, (1 - 0.9, 1 - 0.95))
    k1, _ = _separately_rounded("momentum", m0, None, g.float(), 0.95, None)
    T.adamw_([p], [g], [mc], [vc], step=2, lr=1e-3, moment_scales=[ms], variance_scales=[vs], seeds=[5])
    T.momentum_([mat[0]], [mat[1]], [mat[2]], beta=0.95, seeds=[5])
    frac = R.fractions(n, 5)
    for x, c, s, pos in ((m1, mc, ms, False), (v1, vc, vs, True), (k1, mat[1], mat[2], False)):
        R.check_state(f64(x), np.zeros(n), u8(c), u8(s), frac, pos, "bits")
