"""Edges of the optimizer-state kernels on the GPU, against the definitions in float64 (state_reference.py).
Error bounds as in test_state_gpu.py: an fp32 operation is off by at most 2^-24 of its result or,
below the normal numbers, by 2^-150."""
import math

import numpy as np
import pytest
import torch

import state_reference as R
import test_state_gpu as S

pytestmark = pytest.mark.gpu

E, TINY = 2.0 ** -24, 2.0 ** -150
F8 = torch.float8_e4m3fn
FORMS = ["8 bits", "8 bits and masters", "32 bits and masters"]


def zero_state(n, form):
    """Arguments of adamw_ for one tensor of n zeros with zero state; what it moves is in ["w"]."""
    import thorn_b200 as T

    p = [torch.zeros(n, device="cuda", dtype=torch.float32 if form == FORMS[0] else torch.bfloat16)]
    a = dict(params=p, w=p[0])
    if form != FORMS[0]:
        a["masters"] = [torch.zeros(n, device="cuda")]
        a["w"] = a["masters"][0]
    if form == FORMS[2]:
        a.update(moments=[torch.zeros(n, device="cuda")], variances=[torch.zeros(n, device="cuda")])
    else:
        (mc, ms), (vc, vs) = T.state8_zeros(p[0]), T.state8_zeros(p[0])
        a.update(moments=[mc], variances=[vc], moment_scales=[ms], variance_scales=[vs], seeds=[3])
    return a


def step(a, g, **kw):
    import thorn_b200 as T

    args = {k: v for k, v in a.items() if k != "w"}
    T.adamw_(**args, grads=[g.to(a["params"][0].dtype)], step=1, lr=1.0, **{"weight_decay": 0.0, **kw})
    torch.cuda.synchronize()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("exponent", [-5, -12, -14, -15, -16, -17, -18, -19, -20, -22, -25, -32, -38])
@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_small_gradients_keep_the_angle(form, exponent, spread):
    """The first step from zero state is the angle of (g, |g|), pi / 4, at every magnitude whose
    square fp32 holds, and towards pi / 2 as the square is lost: what float64 gives for the second
    moment that fp32 holds.  ``spread``: neighbours over two more powers of ten."""
    n = 1000
    torch.manual_seed(1)
    g = (torch.rand(n, device="cuda") + 0.5) * 10.0 ** exponent * 10.0 ** (2 * spread * (torch.rand(n, device="cuda") - 0.5))
    g = g * (torch.randint(0, 2, (n,), device="cuda") * 2 - 1)
    g[::50] = 0
    a = zero_state(n, form)
    g = g.to(a["params"][0].dtype)
    step(a, g)
    x, u = S.f64(g), -S.f64(a["w"])
    # m: three operations on |g|; v: two products of numbers that may be below the normal ones
    em = 5 * E * np.abs(x) + 3 * TINY
    v, ev = 0.05 * x * x, 5 * E * 0.05 * x * x + 3 * TINY
    bc1, bc2 = 1 / (1 - 0.9), 1 / (1 - 0.95)
    hi = np.arctan2((0.1 * np.abs(x) + em) * bc1, np.sqrt(np.maximum(v - ev, 0) * bc2))
    lo = np.arctan2(np.maximum(0.1 * np.abs(x) - em, 0) * bc1, np.sqrt((v + ev) * bc2))
    some = x != 0
    assert np.all(u[~some] == 0)
    assert np.all(np.sign(u[some]) == np.sign(x[some]))
    assert np.all(np.abs(u[some]) <= hi[some] * (1 + 16 * E)), np.abs(u[some]).max()
    assert np.all(np.abs(u[some]) >= lo[some] * (1 - 16 * E)), np.abs(u[some]).min()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, 1e30])
@pytest.mark.parametrize("eps", [0.0, 1e-8])
def test_infinite_gradients_move_like_the_definition(form, bad, eps):
    """An infinite gradient has the angle of (inf, inf), pi / 4, as in the AdamW step on 16- and
    32-bit state; over an eps it is inf / inf.  A finite one whose square is infinite moves nothing."""
    a = zero_state(300, form)
    g = torch.zeros(300, device="cuda")
    g[130], g[7] = bad, 1e-3
    step(a, g, eps=eps)
    u = -S.f64(a["w"])
    if math.isnan(bad) or (math.isinf(bad) and eps):
        assert math.isnan(u[130])
    else:
        want = math.copysign(math.pi / 4, bad) if math.isinf(bad) else 0.0
        assert abs(u[130] - want) <= 16 * E * abs(want)
    rest = np.delete(u, [7, 130])
    assert np.all(rest == 0) and np.isfinite(u[7]) and u[7] > 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("eps", [1e-8, 1e-18, 1e-20, 1e-30, 1e-44, 1e-50])
@pytest.mark.parametrize("exponent", [-10, -16, -19, -20, -25])
def test_small_eps_beside_small_gradients(form, eps, exponent):
    """g / (|g| + eps) in its float64 value for the moments that fp32 holds, also where the second
    moment is below the normal numbers; an eps below them stays an eps."""
    n = 400
    torch.manual_seed(2)
    g = (torch.rand(n, device="cuda") + 0.5) * 10.0 ** exponent
    a = zero_state(n, form)
    g = g.to(a["params"][0].dtype)
    g[3] = 0
    step(a, g, eps=eps)
    x, u = S.f64(g), -S.f64(a["w"])
    em = 5 * E * np.abs(x) + 3 * TINY
    v, ev = 0.05 * x * x, 5 * E * 0.05 * x * x + 3 * TINY
    low = max(eps, 2.0 ** -126)  # over a smaller one a zero second moment gives numbers near fp32's end
    hi = (0.1 * x + em) * 10 / (np.sqrt(np.maximum(v - ev, 0) * 20) + min(eps, low))
    lo = (0.1 * x - em) * 10 / (np.sqrt((v + ev) * 20) + low)
    some = x != 0
    assert np.all(u[~some] == 0)
    assert np.all((u[some] <= hi[some] * (1 + 16 * E)) & (u[some] >= lo[some] * (1 - 16 * E)))


@pytest.mark.parametrize("form", FORMS[1:])
def test_infinite_weights_without_decay_of_theirs(form):
    """Where update and weight differ in sign nothing is decayed, whatever the weight is: an infinite
    one stays infinite, as in the AdamW step on 16- and 32-bit state."""
    import thorn_b200 as T

    a = zero_state(40, form)
    a["masters"][0][::2], a["masters"][0][1::2] = math.inf, -math.inf
    a["params"][0].copy_(a["masters"][0])
    g = torch.full((40,), -1e-3, device="cuda", dtype=torch.bfloat16)
    g[1::2] *= -1
    p, m, v = [a["params"][0].clone()], [torch.zeros(40, device="cuda")], [torch.zeros(40, device="cuda")]
    T.adamw_(p, [g], m, v, step=1, lr=1.0, weight_decay=0.1)
    step(a, g, weight_decay=0.1)
    assert not bool(p[0].isnan().any())
    assert torch.equal(a["params"][0], p[0]) and torch.equal(a["masters"][0], p[0].float())


@pytest.mark.parametrize("dtype", S.DTYPES)
@pytest.mark.parametrize("per_matrix", [True, False])
@pytest.mark.parametrize("gain", [None, "scalar", "split"])
def test_magma_sums_of_8_bit_moments(dtype, per_matrix, gain):
    """The three sums beside codes and scales are bit for bit those beside their fp32 values: whole
    and ragged rows, blocks that end inside a row's eight, stacks, an unaligned copy, a NaN block."""
    import types

    import thorn_b200 as T
    from thorn_b200.optimizer import GroupConfig

    shapes = [(64, 256), (70, 300), (3, 5, 77), (2, 3, 9, 13), (1, 1), (200, 8), (4, 130, 131), (9, 40, 24)]
    gen = torch.Generator(device="cuda").manual_seed(4)
    opt = T.THORN([{"orthogonalize": True, "params": [torch.nn.Parameter(torch.zeros(2, 2, device="cuda"))], "lr": 1e-3,
                    "decouple_md": gain is not None}])
    cfg = GroupConfig.from_kwargs(**opt.param_groups[0])
    plain, eight = [], []
    for i, s in enumerate(shapes):
        g = (torch.randn(s, generator=gen, device="cuda") * 1e-3).to(dtype)
        x = torch.randn(s, generator=gen, device="cuda") * 10.0 ** torch.randint(-6, 3, s[:-1] + (1,), generator=gen, device="cuda")
        if i == 1:
            x.view(-1)[500] = math.nan
        codes, scales = T.state8_write(x, per_matrix=per_matrix)
        if i % 2:
            codes = S.offset_like(codes, 3)
        gains = {}
        if gain == "scalar":
            gains = dict(gain=torch.rand((), generator=gen, device="cuda").to(dtype))
        elif gain == "split":
            gains = dict(row_gain=torch.rand(s[:-1] + (1,), generator=gen, device="cuda").to(dtype),
                         col_gain=torch.rand(s[:-2] + (1, s[-1]), generator=gen, device="cuda").to(dtype))
        for out, st in ((plain, dict(moment=T.state8_read(codes, scales))), (eight, dict(moment=codes, moment_scale=scales))):
            out.append(types.SimpleNamespace(g=g, state={**st, **gains}, split=gain == "split"))
    a, b = [opt._magma_stats(its, cfg, True).cpu() for its in (plain, eight)]
    assert torch.equal(a.isnan(), b.isnan()) and bool(a[1].isnan().any()) and not bool(a[0].isnan().any())
    assert torch.equal(a.nan_to_num(), b.nan_to_num())


def test_magma_keeps_8_bit_moments_in_8_bits():
    """Magma beside 8-bit state takes no copy of the moments: 64 Mi elements, well under a byte each."""
    import thorn_b200 as T

    p = torch.nn.Parameter(torch.zeros(8192, 8192, device="cuda", dtype=torch.bfloat16))
    opt = T.THORN([{"orthogonalize": False, "params": [p], "lr": 1e-3, "momentum_align": True, "state_dtype": F8}])
    p.grad = torch.full_like(p, 1e-3)
    opt.step()
    g = torch.full_like(p, 1e-3)
    p.grad = g
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    opt.step()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < p.numel() // 8
