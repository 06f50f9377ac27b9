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


def decoded(codes, scales):
    """float64 values of per-matrix state, [matrices, elements]."""
    B = scales.shape[0]
    return np.stack([R.read(c, s) for c, s in zip(S.u8(codes).reshape(B, -1), S.u8(scales).reshape(B, -1))])


def test_more_matrices_than_a_launch_takes():
    """70 short and long matrices and stacks: every pass of the momentum fills its table more than once."""
    import thorn_b200 as T

    kinds = [(3, 5), (40, 40), (65, 130), (2, 70, 90), (8, 16), (90, 100), (5, 64, 65)]
    shapes = [kinds[i % 7] for i in range(70)]
    g, m, s = S.make_matrices(shapes, torch.bfloat16, seed=7)
    before = [decoded(c, r).reshape(-1) for c, r in zip(m, s)]
    seeds = [11 * i for i in range(70)]
    x = T.momentum_(g, m, s, beta=0.95, seeds=seeds)
    torch.cuda.synchronize()
    for i in range(70):
        S.check_momentum(g[i], before[i], m[i], s[i], x[i], 0.95, seeds[i], torch.float16)


def test_more_updates_than_a_launch_takes():
    import thorn_b200 as T

    torch.manual_seed(8)
    shapes = [[(3, 5), (70, 130), (5000,)][i % 3] for i in range(70)]
    w = [torch.randn(s, device="cuda") * 0.02 for s in shapes]
    p = [t.bfloat16() for t in w]
    u = [(torch.randn(s, device="cuda") * 0.05).half() for s in shapes]
    lrs = [1e-2 * (1 + i % 5) for i in range(70)]
    before = [S.f64(t) for t in w]
    T.apply_update_(p, u, masters=w, lr=lrs, weight_decay=0.1)
    for i in range(70):
        uv = S.f64(u[i])
        uv = np.where(uv * before[i] >= 0, uv + 0.1 * before[i], uv)
        assert np.all(np.abs(S.f64(w[i]) - (before[i] - lrs[i] * uv)) <= 4 * E * (np.abs(before[i]) + lrs[i] * np.abs(uv)))
        assert torch.equal(p[i], w[i].bfloat16())


def test_stack_of_matrices_whose_norms_take_a_launch():
    """Three matrices of 550 chunks each and of different magnitudes: each has its own norm."""
    import thorn_b200 as T

    g, m, s = S.make_matrices([(3, 1500, 1500)], torch.bfloat16, seed=9)
    size = torch.tensor([1.0, 1e-3, 1e3], device="cuda").view(3, 1, 1)
    g = [(g[0] * size).bfloat16()]
    m, s = [[t] for t in T.state8_write(T.state8_read(m[0], s[0]) * size, per_matrix=True)]
    before = decoded(m[0], s[0]).reshape(-1)
    x = T.momentum_(g, m, s, beta=0.95, seeds=[12])
    torch.cuda.synchronize()
    S.check_momentum(g[0], before, m[0], s[0], x[0], 0.95, 12, torch.float16)


def _big():
    if torch.cuda.get_device_properties(0).total_memory < 120 << 30:
        pytest.skip("needs 80 GB")


@pytest.mark.parametrize("shape", [(65537, 65536), (3, 37901, 37901)])
def test_momentum_offsets_beyond_32_bits(shape):
    """More than 2^32 elements in one matrix and in a stack: the last 70000 elements, which start
    inside a block, get the random numbers of their place; what lies before them stays zero."""
    import thorn_b200 as T

    _big()
    tail = 70000
    g = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    n, run = g.numel(), shape[-2] * shape[-1]
    assert n > 1 << 32
    torch.manual_seed(13)
    g.view(-1)[n - tail:] = (torch.randn(tail, device="cuda") * 1e-3).bfloat16()
    m, s = T.state8_zeros(g, per_matrix=True)
    x, = T.momentum_([g], [m], [s], beta=0.95, seeds=[6])
    last = run - tail
    at = last // 128 * 128  # the block that the tail starts in, in its matrix
    gv = S.f64(g.view(-1)[n - run + at:])
    frac = R.fractions(run - at, 6, run=len(m.view(-1)) // run - 1, start=at)
    new = R.check_state(gv, np.zeros(gv.size), S.u8(m.view(-1)[n - run + at:]), S.u8(s[-1, at // 128:]), frac, False, "m")
    u = gv + 0.95 * new
    norm = np.linalg.norm(u)
    tol = (2.0 ** -11 + 2.0 ** 6 * E) * np.abs(u) / norm + 3 * E * (np.abs(gv) + np.abs(new)) / norm + 2.0 ** -25
    assert np.all(np.abs(S.f64(x.view(-1)[n - run + at:]) - u / (norm + 1e-8)) <= tol)
    head = (n - run + at) // 8 * 8
    for t in (m.view(torch.uint8), x):
        assert int(torch.count_nonzero(t.view(-1)[:head].view(torch.int64))) == 0


def test_master_offsets_beyond_32_bits():
    """AdamW and the apply onto fp32 masters of 2^32 + 5000 elements: the tail is updated, nothing before it."""
    import thorn_b200 as T

    _big()
    n, tail = (1 << 32) + 5000, 4936
    torch.manual_seed(14)
    p, w = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, device="cuda")
    g = torch.zeros(n, dtype=torch.float16, device="cuda")
    g[n - tail:] = torch.randn(tail, device="cuda").half()
    T.apply_update_([p], [g], masters=[w], lr=0.5, weight_decay=0.1)
    assert torch.equal(w[n - tail:], -0.5 * g[n - tail:].float()) and torch.equal(p[n - tail:], w[n - tail:].bfloat16())
    for t in (p, w):
        assert int(torch.count_nonzero(t[:n - tail].view(torch.int64))) == 0
    w[n - tail:] = 0
    p[n - tail:] = 0
    g = g.bfloat16()
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    T.adamw_([p], [g], [m], [v], step=1, lr=1.0, weight_decay=0.0, masters=[w])
    x = S.f64(g[n - tail:])
    assert np.all(np.abs(S.f64(m[n - tail:]) - 0.1 * x) <= 5 * E * np.abs(x))
    assert np.all(np.abs(S.f64(v[n - tail:]) - 0.05 * x * x) <= 5 * E * 0.05 * x * x)
    want = -np.sign(x) * math.pi / 4
    # pi / 4 is known to the errors of m and of the root of v: under 64 roundings
    assert np.all(np.abs(S.f64(w[n - tail:]) - want) <= 64 * E)
    for t in (p, w, m, v):
        assert int(torch.count_nonzero(t[:n - tail].view(torch.int64))) == 0


@pytest.mark.parametrize("ortho", [True, False])
def test_decoupled_magnitudes_and_magma_beside_32_bit_state(ortho):
    """Three steps of decouple_md and momentum_align, each beside one of fp32 state that holds the
    same values: the same scores, masks and gains, moments that are the roundings of its, and for
    AdamW, whose update uses the moments before they are rounded, the same parameters.  There the two
    updates differ by at most 512 roundings of lr (32 of an angle up to pi / 2; 10 of |m| + |g| times
    bc1 = 10 over a root of at least 0.9 |g|) and the passes behind them by 32 of the parameter."""
    import thorn_b200 as T

    shapes = [(64, 48), (40, 56), (3, 20, 30)]
    p, q = [S._params(shapes, torch.float32, 6) for _ in range(2)]
    opts = dict(orthogonalize=ortho, lr=1e-2, decouple_md=True, momentum_align=True, betas=(0.9, 0.95), none_grad=False)
    a, b = T.THORN([{"params": p, "state_dtype": F8, **opts}]), T.THORN([{"params": q, **opts}])
    grads = S._grads(p, 60)
    moved = 0
    for k in range(3):
        if k:
            for t, u in zip(p, q):
                u.data.copy_(t.data)
                for key, val in a.state[t].items():
                    if key in ("moment", "variance"):
                        b.state[u][key] = T.state8_read(val, a.state[t][key + "_scale"])
                    elif "scale" not in key and key != "rounding_seed":
                        b.state[u][key] = val.clone() if isinstance(val, torch.Tensor) else val
        old = [{key: S.f64(b.state[u][key]) if k else np.zeros(u.numel()) for key in ("moment", "variance")} if
               k == 0 or not ortho else {"moment": S.f64(b.state[u]["moment"])} for u in q]
        at = [t.detach().clone() for t in p]
        for opt, ps in ((a, p), (b, q)):
            torch.manual_seed(70)
            for t, x in zip(ps, grads):
                t.grad = x.clone()
            opt.step()
        for i, (t, u) in enumerate(zip(p, q)):
            s, w = a.state[t], b.state[u]
            for key in w:
                if key not in ("moment", "variance"):
                    same = torch.equal(s[key], w[key]) if isinstance(w[key], torch.Tensor) else s[key] == w[key]
                    assert same, (k, i, key)
            B = int(np.prod(t.shape[:-2]))
            g = S.f64(u.grad)  # the recovered gradient
            assert torch.equal(t.grad, u.grad)
            for key in ("moment", "variance") if not ortho else ("moment",):
                err = 5 * E * (np.abs(old[i][key]) + np.abs(g)) if key == "moment" else 5 * E * S.f64(w[key])
                runs = B if ortho else 1
                cut = lambda z: z.reshape(runs, -1)  # noqa: E731
                seed = (i << 32) + k + 1
                for r in range(runs):
                    R.check_state(cut(S.f64(w[key]))[r], cut(err)[r], cut(S.u8(s[key]))[r], cut(S.u8(s[key + "_scale"]))[r],
                                  R.fractions(t.numel() // runs, seed, run=r), key == "variance", (k, i, key))
            if not ortho:
                assert bool(((t - u).abs() <= 512 * E * 1e-2 + 32 * E * u.abs()).all()), (k, i)
            assert bool(t.isfinite().all())
            moved += not torch.equal(t.detach(), at[i])
    assert moved


@pytest.mark.parametrize("ortho", [True, False])
def test_a_refused_capture_leaves_the_steps_that_follow(ortho):
    """A first step that was refused inside a capture, then two eager ones: what two steps give alone."""
    import thorn_b200 as T

    runs = []
    for refused in (False, True):
        p = S._params([(40, 48)], torch.bfloat16, 1)
        opt = T.THORN([{"orthogonalize": ortho, "params": p, "lr": 1e-2, "state_dtype": F8, "master_weights": True}])
        if refused:
            p[0].grad = S._grads(p, 90)[0]
            graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
            with torch.cuda.graph(graph):
                x.add_(1)
                with pytest.raises(RuntimeError, match="capture"):
                    opt.step()
            graph.replay()
            torch.cuda.synchronize()
            assert "step" not in opt.state[p[0]]
        for k in range(2):
            p[0].grad = S._grads(p, 90 + k)[0]
            opt.step()
        runs.append((p[0].detach(), opt.state[p[0]]["moment"].view(torch.uint8), opt.state[p[0]]["master"]))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def _one_rank(port, q):
    import datetime
    import traceback

    import torch.distributed as dist

    try:
        torch.cuda.set_device(0)
        dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1,
                                timeout=datetime.timedelta(seconds=60), device_id=torch.device("cuda", 0))
        from torch.distributed.device_mesh import init_device_mesh
        from torch.distributed.tensor import Shard, distribute_tensor

        import thorn_b200 as T

        mesh = init_device_mesh("cuda", (1,))
        plain = S._params([(50, 30), (7,)], torch.bfloat16, 1)
        ps = [torch.nn.Parameter(distribute_tensor(t.detach().clone(), mesh, [Shard(0)])) for t in plain]
        opts = dict(orthogonalize=False, lr=1e-2, master_weights=True, momentum_align=True)
        a, b = T.THORN([{"params": plain, **opts}]), T.THORN([{"params": ps, **opts}])
        for k in range(4):
            for opt, group in ((a, plain), (b, ps)):
                torch.manual_seed(30)
                for t, x in zip(group, S._grads(plain, 10 + k)):
                    t.grad = distribute_tensor(x, mesh, [Shard(0)]) if opt is b else x
                opt.step()
        for t, u in zip(plain, ps):
            for x, y in ((t.detach(), u.data), *((a.state[t][k], b.state[u][k]) for k in ("master", "moment", "variance"))):
                assert torch.equal(x, y.to_local())
        torch.cuda.synchronize()
        dist.destroy_process_group()
        q.put(None)
    except Exception:
        q.put(traceback.format_exc())


def test_masters_of_a_sharded_parameter_on_one_rank():
    """A Shard(0) AdamW parameter of one rank steps like a plain one, Magma's sums over the shard group included."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_one_rank, args=(port, q))
    p.start()
    err = q.get(timeout=180)
    p.join(60)
    assert err is None, err


def test_inputs_written_over_their_gradients():
    """``out`` may be ``grads``: every length class, aligned and not, the same bits as apart."""
    import thorn_b200 as T

    shapes = [(5, 7, 9), (2, 64, 64), (9, 30, 30), (129, 127), (3, 65, 200), (1500, 1501)]
    runs = []
    for over in (False, True):
        g, m, s = S.make_matrices(shapes, torch.float16, seed=15)
        x = T.momentum_(g, m, s, beta=0.95, seeds=list(range(len(shapes))), out=g if over else None)
        torch.cuda.synchronize()
        runs.append([S.u8(t) for t in [*x, *m, *s]])
    for a, b in zip(*runs):
        assert np.array_equal(a, b)
