"""Optimizer state in 8 bits and in 32, on the CPU: layouts, refusals, the rounding's definition
and the conversions.  The kernels are tested in test_state_gpu.py."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import state_reference as R
from thorn_b200 import _native as N
from thorn_b200 import build as B
from thorn_b200 import multi as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def lib():
    B.build()
    return N.load()


STRUCTS = {
    "thorn_adamw_state_tensor": (N.AdamStateTensor, M._ADAM),
    "thorn_momentum8_tensor": (N.Momentum8Tensor, M._MOMENTUM),
    "thorn_apply_master_tensor": (N.ApplyMasterTensor, M._APPLY),
}


def test_struct_layouts_match_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "thorn_b200.h"', "int main(void) {"]
    for cname, (st, _) in STRUCTS.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        for f, _ in st._fields_:
            lines.append(f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));')
    lines.append("  return 0; }")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    c = {tuple(line.split()[:2]): int(line.split()[2]) for line in out if line}
    for cname, (st, packed) in STRUCTS.items():
        assert ctypes.sizeof(st) == c[(cname, "size")] == packed.size, cname
        for f, _ in st._fields_:
            assert getattr(st, f).offset == c[(cname, f)], (cname, f)
    # the packed records put every field where the structure has it
    a = M._records(N.AdamStateTensor, [M.adam_record(1, 2, 3, 4, 5, 6, 7, 8, -1, 0.5, 0.25, 2.0, 1)])[0]
    assert [a.p, a.g, a.w, a.m, a.v, a.m_scale, a.v_scale, a.numel] == [1, 2, 3, 4, 5, 6, 7, 8]
    assert (a.seed, a.lr, a.bc1, a.bc2, a.degenerate) == (R.M64, 0.5, 0.25, 2.0, 1)
    a = M._records(N.Momentum8Tensor, [M._MOMENTUM.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10)])[0]
    assert [getattr(a, f) for f, _ in a._fields_] == list(range(1, 11))
    a = M._records(N.ApplyMasterTensor, [M._APPLY.pack(1, 2, 3, 4, 5, 6, 7, 8, 0.5)])[0]
    assert [getattr(a, f) for f, _ in a._fields_] == [1, 2, 3, 4, 5, 6, 7, 8, 0.5]


def test_prototypes_match_header():
    """Parameter counts and scalar types of the bound functions, as the header declares them."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "thorn_b200.h")).read(), flags=re.S)
    scalars = {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "double": ctypes.c_double, "float": ctypes.c_float}
    assert not set(N._STATE_PROTOS) & set(N._PROTOS)
    for name, (res, argtypes) in N._STATE_PROTOS.items():
        m = re.search(r"THORN_API\s+(\w+)\s+" + name + r"\s*\(([^)]*)\)\s*;", text)
        assert scalars[m.group(1)] is res, name
        params = [a.strip().rsplit(None, 1)[0].replace("const", "").strip() for a in m.group(2).split(",")]
        params = [p.rstrip("* ") + "*" if "*" in a else p for p, a in zip(params, m.group(2).split(","))]
        assert len(params) == len(argtypes), name
        for decl, got in zip(params, argtypes):
            t = decl.rstrip("* ")
            if t in STRUCTS:
                assert got is ctypes.POINTER(STRUCTS[t][0]), (name, decl)
            elif decl.endswith("*"):
                assert got is ctypes.c_void_p, (name, decl)
            else:
                assert got is scalars[decl], (name, decl, got)


def test_scratch_bytes(lib):
    # for matrices longer than 4096 elements: an fp32 sum per 4096 elements and one per matrix,
    # padded to 16 bytes
    assert lib.thorn_momentum8_scratch_bytes(7, 32, 128) == 0
    assert lib.thorn_momentum8_scratch_bytes(3, 65, 128) == 48
    assert lib.thorn_momentum8_scratch_bytes(5, 128, 128) == 112
    assert lib.thorn_momentum8_scratch_bytes(0, 8, 8) == 0
    assert lib.thorn_momentum8_scratch_bytes(1, 1 << 40, 1 << 40) == 0  # over the size limit


def test_argument_validation_without_gpu(lib):
    """Bad arguments are rejected before anything touches the device."""
    P = 1 << 20  # a pointer that is never followed

    def adam(fn, n=1, dt=N.BF16, **kw):
        t = N.AdamStateTensor(P, P, P, P, P, P, P, 16, 0, 1e-3, 1.0, 1.0, 0)
        for k, v in kw.items():
            setattr(t, k, v)
        return fn(N.array(N.AdamStateTensor, [t]), n, dt, 0.9, 0.95, 0.0, 0.0, None)

    for fn in (lib.thorn_adamw8_multi, lib.thorn_adamw_master_multi):
        assert adam(fn, n=0) == 0
        assert adam(fn, numel=0) == 0  # an empty tensor needs nothing
        assert adam(fn, n=-1) == 1 and adam(fn, dt=7) == 1
        assert adam(fn, numel=-1) == 1 and adam(fn, numel=1 << 60) == 1
        for k in ("g", "m", "v"):
            assert adam(fn, **{k: None}) == 1, k
        assert fn(None, 1, N.BF16, 0.9, 0.95, 0.0, 0.0, None) == 1
    assert adam(lib.thorn_adamw8_multi, m_scale=None) == 1 and adam(lib.thorn_adamw8_multi, v_scale=None) == 1
    assert adam(lib.thorn_adamw8_multi, dt=N.F32) == 1  # master weights of fp32 parameters
    assert adam(lib.thorn_adamw_master_multi, w=None) == 1 and adam(lib.thorn_adamw_master_multi, dt=N.F32) == 1

    def mom(n=1, dt=N.BF16, xdt=N.F16, **kw):
        t = N.Momentum8Tensor(P, P, P, P, 1, 4096, 4, 4, 0, P)  # a matrix that needs scratch
        for k, v in kw.items():
            setattr(t, k, v)
        return lib.thorn_momentum8_multi(N.array(N.Momentum8Tensor, [t]), n, dt, xdt, 0.9, None)

    assert mom(n=0) == 0 and mom(rows=0) == 0
    assert mom(n=-1) == 1 and mom(dt=9) == 1 and mom(xdt=N.F32) == 1
    for k in ("g", "m", "m_scale", "scratch"):
        assert mom(**{k: None}) == 1, k
    assert mom(ldx=3) == 1 and mom(batch=-1) == 1 and mom(scratch=P + 4) == 1
    assert mom(rows=1 << 40, cols=1 << 40) == 1 and mom(batch=1 << 31) == 1

    def app(n=1, udt=N.F16, dt=N.BF16, **kw):
        t = N.ApplyMasterTensor(P, P, P, None, None, 1, 4, 4, 0.1)
        for k, v in kw.items():
            setattr(t, k, v)
        return lib.thorn_apply_master_multi(N.array(N.ApplyMasterTensor, [t]), n, udt, dt, 0.0, None)

    assert app(n=0) == 0 and app(cols=0) == 0
    assert app(n=-1) == 1 and app(udt=N.F32) == 1 and app(dt=N.F32) == 1 and app(rows=-2) == 1
    for k in ("U", "p", "w"):
        assert app(**{k: None}) == 1, k
    assert app(mat_stats=P) == 1  # matrix factors without row factors


# ------------------------------------------------------------------------------- Python refusals
@pytest.fixture
def on_cpu(monkeypatch):
    """Lets the argument checks run on CPU tensors; a launch would fail the test."""
    monkeypatch.setattr(M, "_device", lambda t: t.device)

    def no_launch(*a, **k):
        raise AssertionError("reached the launch")

    for name in ("launch_adam", "_momentum_call", "launch_apply"):
        monkeypatch.setattr(M, name, no_launch)


def _adam_args(n=2, shape=(3, 50), dtype=torch.bfloat16, eight=True, master=False):
    p = [torch.zeros(shape, dtype=dtype) for _ in range(n)]
    a = dict(params=p, grads=[torch.zeros_like(t) for t in p])
    if eight:
        st = [M.state8_zeros(t) for t in p + p]
        a.update(moments=[c for c, _ in st[:n]], variances=[c for c, _ in st[n:]],
                 moment_scales=[s for _, s in st[:n]], variance_scales=[s for _, s in st[n:]], seeds=list(range(n)))
    else:
        a.update(moments=[torch.zeros(shape) for _ in p], variances=[torch.zeros(shape) for _ in p])
    if master:
        a.update(masters=[t.float() for t in p])
    return dict(a, step=1, lr=1e-3)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        M.adamw_(**_adam_args())
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        M.apply_update_([torch.zeros(2, 2, dtype=torch.bfloat16)], [torch.zeros(2, 2, dtype=torch.float16)],
                        masters=[torch.zeros(2, 2)], lr=1.0)


@pytest.mark.parametrize("change,error", [
    (dict(step=0), ValueError), (dict(step=[1]), ValueError), (dict(lr=[1.0]), ValueError),
    (dict(eps=-1e-8), ValueError), (dict(betas=(0.9, 1.0)), ValueError), (dict(betas=(-0.1, 0.9)), ValueError),
    (dict(seeds=None), ValueError), (dict(seeds=[1]), ValueError), (dict(moment_scales=None), ValueError),
    (dict(grads=[]), ValueError),
    (dict(grads=[torch.zeros(3, 50), torch.zeros(3, 50)]), TypeError),
    (dict(grads=[torch.zeros(3, 51, dtype=torch.bfloat16)] * 2), ValueError),
    (dict(grads=[torch.zeros(50, 3, dtype=torch.bfloat16).T] * 2), ValueError),
    (dict(variances=[torch.zeros(3, 50)] * 2), TypeError),
    (dict(moment_scales=[torch.zeros(1, dtype=torch.uint8).view(torch.float8_e8m0fnu)] * 2), ValueError),
    (dict(variance_scales=[torch.zeros(2)] * 2), TypeError),
    (dict(masters=[torch.zeros(3, 50, dtype=torch.float64)] * 2), TypeError),
])
def test_adamw_refusals(on_cpu, change, error):
    with pytest.raises(error):
        M.adamw_(**{**_adam_args(), **change})


def test_adamw_more_refusals(on_cpu):
    a = _adam_args()
    with pytest.raises(ValueError, match="twice"):
        M.adamw_(**{**a, "params": [a["params"][0]] * 2})
    with pytest.raises(ValueError, match="twice"):
        M.adamw_(**{**a, "moments": [a["moments"][0]] * 2})
    with pytest.raises(ValueError, match="twice"):
        M.adamw_(**{**a, "variance_scales": [a["variance_scales"][0]] * 2})
    with pytest.raises(TypeError, match="16-bit"):
        M.adamw_(**_adam_args(dtype=torch.float32, master=True))
    with pytest.raises(TypeError):  # float64 parameters
        M.adamw_(**_adam_args(dtype=torch.float64, eight=False))
    b = _adam_args(eight=False, master=True)
    with pytest.raises(TypeError, match="fp32 or 8-bit"):
        M.adamw_(**{**b, "moments": [m.half() for m in b["moments"]], "variances": [m.half() for m in b["variances"]]})
    with pytest.raises(ValueError, match="scales"):
        M.adamw_(**{**b, "moment_scales": a["moment_scales"]})
    M.adamw_([], [], [], [], step=1, lr=1e-3)  # nothing to do


def test_momentum_and_apply_refusals(on_cpu):
    g = [torch.zeros(4, 6, 8), torch.zeros(5, 7)]
    st = [M.state8_zeros(t, per_matrix=True) for t in g]
    a = dict(grads=g, moments=[c for c, _ in st], scales=[s for _, s in st], beta=0.9, seeds=[1, 2])
    assert st[0][1].shape == (4, 1) and st[1][1].shape == (1, 1)
    for change, error in [(dict(beta=1.0), ValueError), (dict(seeds=[1]), ValueError),
                          (dict(dtype=torch.float32), TypeError),
                          (dict(grads=[torch.zeros(4, 6, 8), torch.zeros(35)]), ValueError),
                          (dict(moments=[torch.zeros(4, 6, 8), torch.zeros(5, 7)]), TypeError),
                          (dict(scales=[st[0][1][:3], st[1][1]]), ValueError),
                          (dict(out=[torch.zeros(4, 6, 8), torch.zeros(5, 7)]), TypeError),
                          (dict(moments=[st[0][0]]), ValueError)]:
        with pytest.raises(error):
            M.momentum_(**{**a, **change})
    assert M.momentum_([], [], [], beta=0.9, seeds=[]) == []
    p = [torch.zeros(4, 4, dtype=torch.bfloat16)]
    u, w = [torch.zeros(4, 4, dtype=torch.float16)], [torch.zeros(4, 4)]
    for kw, error in [(dict(params=[p[0].float()]), TypeError), (dict(updates=[u[0].float()]), TypeError),
                      (dict(masters=[w[0].half()]), TypeError), (dict(masters=w * 2), ValueError),
                      (dict(masters=[torch.zeros(4, 5)]), ValueError), (dict(lr=[1.0, 2.0]), ValueError)]:
        with pytest.raises(error):
            M.apply_update_(**{**dict(params=p, updates=u, masters=w, lr=1e-3), **kw})


# ----------------------------------------------------------------------------- the 8-bit numbers
def test_codes_are_e4m3():
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, R.GRID)


@pytest.mark.parametrize("shape", [(1,), (127,), (128,), (129,), (3, 5, 77), (4, 128), (0,)])
@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1.0, 1e30])
def test_state_round_trip(shape, scale):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=gen) * scale
    for per_matrix in (False, True) if len(shape) >= 2 else (False,):
        codes, scales = M.state8_write(x, per_matrix)
        assert codes.shape == x.shape and codes.dtype is torch.float8_e4m3fn
        y = M.state8_read(codes, scales)
        runs = x.reshape(shape[0], -1) if per_matrix and len(shape) > 2 else x.reshape(1, -1)
        want = np.concatenate([R.scale_bytes(r.double().numpy()) for r in runs])
        assert np.array_equal(scales.view(torch.uint8).numpy().reshape(-1), want)
        # half a step of 2^-3 at most: 2^-4 of the value, or 2^-10 of the scale below its normal codes
        size = scales.float().reshape(runs.shape[0], -1).repeat_interleave(128, 1)[:, :runs.shape[1]].reshape(shape)
        assert bool(((y - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, size * 2.0 ** -10)).all())


def test_state_special_values():
    x = torch.zeros(3 * 128 + 5)
    x[130] = float("nan")
    x[300] = -448.0 * 2.0 ** -20
    x[301] = 2.0 ** -30
    x[385] = float("inf")
    codes, scales = M.state8_write(x)
    b = scales.view(torch.uint8).tolist()
    assert b == [0, 255, 127 - 20, 255]
    y = M.state8_read(codes, scales)
    assert bool((y[:128] == 0).all()) and bool(y[128:256].isnan().all()) and bool(y[384:].isnan().all())
    assert y[300] == x[300]
    codes, scales = M.state8_write(x[256:384].abs(), positive=True)
    y = M.state8_read(codes, scales)
    assert float(y.min()) == 2.0 ** -9 * 2.0 ** -20  # no second moment at zero beside one that is not
    assert bool((M.state8_read(*M.state8_write(torch.zeros(5), positive=True)) == 0).all())
    z, s = M.state8_zeros(torch.empty(2, 3, 50), per_matrix=True)
    assert s.shape == (2, 2) and bool((M.state8_read(z, s) == 0).all())
    with pytest.raises(ValueError):
        M.state8_zeros(torch.empty(5), per_matrix=True)


def test_rounding_fractions_are_uniform():
    """The generator's fractions: mean 1/2 and flat over 64 cells within 5 standard deviations,
    for neighbouring elements, seeds and runs alike, and neighbours are uncorrelated."""
    n = 1 << 16
    base = R.fractions(n, 12345)
    for f in (base, R.fractions(n, 12346), R.fractions(n, 12345, run=1)):
        assert abs(f.mean() - 0.5) < 5 / np.sqrt(12 * n)
        h = np.histogram(f, bins=64, range=(0, 1))[0]
        assert np.all(np.abs(h - n / 64) < 5 * np.sqrt(n / 64))
        if f is not base:
            assert abs(np.corrcoef(f, base)[0, 1]) < 5 / np.sqrt(n)
    for lag in (4, 8, 128):
        assert abs(np.corrcoef(base[:-lag], base[lag:])[0, 1]) < 5 / np.sqrt(n)


# ---------------------------------------------------------------------------------- THORN groups
def _step(opt, *params, grad=None):
    for p in params:
        p.grad = torch.zeros_like(p) if grad is None else grad
    opt.step()


def test_group_options_are_checked_before_any_state():
    from thorn_b200 import THORN

    w = torch.nn.Parameter(torch.zeros(8, 8, dtype=torch.bfloat16))
    f8 = torch.float8_e4m3fn
    cases = [(dict(orthogonalize=False, master_weights=True, state_dtype=torch.bfloat16), ValueError),
             (dict(orthogonalize=True, master_weights=True, state_dtype=torch.float16), ValueError),
             (dict(orthogonalize=True, master_weights=True, decouple_md=True), NotImplementedError),
             (dict(orthogonalize=False, master_weights=True, decouple_md=True), NotImplementedError)]
    for opts, error in cases:
        opt = THORN([{"params": [w], "lr": 1e-3, **opts}])
        with pytest.raises(error):
            _step(opt, w)
        assert "step" not in opt.state[w]
    sparse = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 8, dtype=torch.bfloat16), (8, 8))
    for opts in (dict(state_dtype=f8), dict(master_weights=True)):
        opt = THORN([{"params": [w], "lr": 1e-3, "orthogonalize": False, **opts}])
        with pytest.raises(NotImplementedError, match="sparse"):
            _step(opt, w, grad=sparse)
    t = torch.nn.Parameter(torch.zeros(8, 6, dtype=torch.bfloat16).T)
    opt = THORN([{"params": [t], "lr": 1e-3, "orthogonalize": True, "state_dtype": f8}])
    with pytest.raises(ValueError, match="contiguous"):
        _step(opt, t)


def test_state_layout_and_state_dict_round_trip():
    """Keys, types and shapes of the state; a saved state comes back as it was (the base class
    casts floating state to the parameter's dtype)."""
    from thorn_b200 import THORN

    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu

    def make():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(3, 10, 30).bfloat16()), torch.nn.Parameter(torch.randn(300).bfloat16())]
        return ps, THORN([{"params": ps[:1], "lr": 1e-3, "orthogonalize": True, "state_dtype": f8, "master_weights": True},
                          {"params": ps[1:], "lr": 1e-3, "orthogonalize": False, "state_dtype": f8}])

    ps, opt = make()
    for p in ps:
        p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        opt.step()
    a, b = opt.state[ps[0]], opt.state[ps[1]] if "step" in opt.state[ps[1]] else None
    if b is None:
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            opt.step(param=ps[1])
        b = opt.state[ps[1]]
    assert set(a) == {"step", "moment", "moment_scale", "rounding_seed", "master"}
    assert set(b) == {"step", "moment", "moment_scale", "variance", "variance_scale", "rounding_seed"}
    assert a["moment"].dtype is f8 and a["moment"].shape == (3, 10, 30) and a["moment_scale"].shape == (3, 3)
    assert a["moment_scale"].dtype is e8 and a["master"].dtype is torch.float32
    assert torch.equal(a["master"], ps[0].detach().float())
    assert b["variance_scale"].shape == (3,) and (a["rounding_seed"], b["rounding_seed"]) == (0, 1 << 32)
    gen = torch.Generator().manual_seed(1)
    for st in (a, b):
        for k in ("moment", "variance"):
            if k in st:
                st[k].view(torch.uint8).copy_(torch.randint(0, 127, st[k].shape, generator=gen, dtype=torch.uint8))
                s = st[k + "_scale"]
                s.view(torch.uint8).copy_(torch.randint(90, 120, s.shape, generator=gen, dtype=torch.uint8))
    a["master"] += 1e-6
    ps2, opt2 = make()
    opt2.load_state_dict(opt.state_dict())
    for p, q in zip(ps, ps2):
        for k, v in opt.state[p].items():
            w = opt2.state[q][k]
            if isinstance(v, torch.Tensor):
                assert w.dtype is v.dtype and torch.equal(w.view(torch.uint8), v.view(torch.uint8)), k
            else:
                assert w == v


# --------------------------------------------------------------------------- the host extension
def test_host_extension_refuses_bad_arguments(lib):
    h = N.host()
    ts = [torch.zeros(3), torch.zeros(4, 5)]
    f32 = torch.float32

    def ptr(buf=None, offset=0, stride=16, t=ts, dtype=f32, device=-1, like=None, mode=0, distinct=True):
        return h.pointers(bytearray(64) if buf is None else buf, offset, stride, t, dtype, device, like, mode, distinct)

    buf = bytearray(64)
    assert ptr(buf=buf, offset=8) is True
    assert [int.from_bytes(buf[16 * i + 8:16 * i + 16], "little") for i in (0, 1)] == [t.data_ptr() for t in ts]
    assert buf[:8] == bytes(8) and buf[32:] == bytes(32)
    assert ptr(dtype=torch.float64) is False and ptr(device=0) is False
    assert ptr(t=[ts[1].T]) is False and ptr(t=[ts[0], ts[0]]) is False and ptr(t=[ts[0], ts[0]], distinct=False) is True
    assert ptr(t=[torch.zeros(0), torch.zeros(0)]) is True  # empty tensors may share an address
    assert ptr(t=[ts[0].to_sparse()]) is False and ptr(t=[torch.zeros(3, device="meta")]) is False
    assert ptr(like=ts, mode=1) is True and ptr(like=ts[::-1], mode=1) is False
    a, b = torch.zeros(300), torch.zeros(2, 10, 30)
    assert ptr(t=[torch.zeros(3), torch.zeros(5)], like=[a, b], mode=2) is True
    assert ptr(t=[torch.zeros(2, 3)], like=[b], mode=3) is True and ptr(t=[torch.zeros(3)], like=[a], mode=3) is False
    for bad, error in [(dict(t=tuple(ts)), TypeError), (dict(t=[1]), TypeError), (dict(dtype="float32"), TypeError),
                       (dict(like=ts[:1], mode=1), ValueError), (dict(buf=bytearray(31)), ValueError),
                       (dict(offset=-8), ValueError), (dict(offset=12), ValueError), (dict(buf=b"x" * 64), BufferError)]:
        with pytest.raises(error):
            ptr(**bad)
    with pytest.raises(ValueError):
        h.values(bytearray(16), 0, 8, 2, "f", [1.0])
    with pytest.raises(ValueError):
        h.values(bytearray(15), 0, 8, 2, "f", 1.0)
    with pytest.raises(TypeError):
        h.values(bytearray(16), 0, 8, 2, "f", ["x", "y"])
    fn = M._scratch_fn()
    with pytest.raises(ValueError, match="matrices"):
        h.matrices(bytearray(64), 0, 64, [torch.zeros(3)], fn)
    rec = bytearray(2 * 40)
    assert h.matrices(rec, 0, 40, [torch.zeros(3, 65, 128), torch.zeros(5, 7)], fn) == (3 * 65 * 128 + 40, 48)
    h.scratch(rec, 0, 32, 40, 2, fn, 4096)
    assert [int.from_bytes(rec[40 * i + 32:40 * i + 40], "little") for i in (0, 1)] == [4096, 4096 + 48]
    assert list(memoryview(rec)[:32].cast("q")) == [3, 65, 128, 128]
    flat = torch.arange(80, dtype=torch.float16)
    v = h.views(flat, [torch.zeros(3, 7), torch.zeros(2, 0, 4), torch.zeros(5, 9)], bytearray(48), 0, 16)
    assert [tuple(x.shape) for x in v] == [(3, 7), (2, 0, 4), (5, 9)] and all(x.is_contiguous() for x in v)
    assert v[2].data_ptr() == flat.data_ptr() + 2 * 24 and float(v[2][4, 8]) == 24 + 44
    with pytest.raises(ValueError, match="short"):
        h.views(flat, [torch.zeros(9, 9)], bytearray(16), 0, 16)
