"""Edges of the optimizer state on the CPU: saving and loading, refusals and host code.  The
kernels' edges are in test_state_edges_gpu.py."""
import pytest
import torch

from thorn_b200 import THORN
from thorn_b200 import build as B
from thorn_b200 import multi as M

F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def built():
    B.build()


def _with_state(groups):
    """A THORN whose parameters' states are made and filled with numbers (the step itself needs a GPU)."""
    opt = THORN(groups)
    gen = torch.Generator().manual_seed(1)
    for group in opt.param_groups:
        for p in group["params"]:
            p.grad = torch.zeros_like(p)
            with pytest.raises(RuntimeError, match="CUDA devices only"):
                opt.step(param=p)
            for k, v in opt.state[p].items():
                if isinstance(v, torch.Tensor) and v.dtype in (torch.float32, torch.bfloat16, torch.float16):
                    v.copy_(torch.randn(v.shape, generator=gen) * 1e-3)
    return opt


def _same_state(a, b):
    for group, other in zip(a.param_groups, b.param_groups):
        for p, q in zip(group["params"], other["params"]):
            assert set(a.state[p]) == set(b.state[q])
            for k, v in a.state[p].items():
                w = b.state[q][k]
                if isinstance(v, torch.Tensor):
                    assert w.dtype is v.dtype, k
                    assert torch.equal(w.reshape(-1).view(torch.uint8), v.reshape(-1).view(torch.uint8)), k
                else:
                    assert w == v, k


def _groups(**opts):
    torch.manual_seed(0)
    ps = [torch.nn.Parameter((torch.randn(s) * 0.02).bfloat16()) for s in ((6, 10), (40,))]
    return [{"params": ps[:1], "lr": 1e-3, "orthogonalize": True, **opts},
            {"params": ps[1:], "lr": 1e-3, "orthogonalize": False, **opts}]


@pytest.mark.parametrize("opts", [dict(state_dtype=torch.float32), dict(state_dtype=torch.float32, decouple_md=True),
                                  dict(state_dtype=torch.float16), dict(master_weights=True), dict(state_dtype=F8),
                                  dict()])
def test_saved_state_comes_back_in_its_types(opts):
    """The base class casts floating state to the parameter's type; state that a group holds in
    another one comes back as it was, bit for bit."""
    opt = _with_state(_groups(**opts))
    other = THORN(_groups(**opts))
    other.load_state_dict(opt.state_dict())
    _same_state(opt, other)


def test_load_hooks_decide_what_is_loaded():
    """A hook that replaces the state dict before it is loaded is followed, and one that runs after
    the load sees the state as it will be."""
    opt = _with_state(_groups(state_dtype=F8, master_weights=True))
    other = THORN(_groups(state_dtype=F8, master_weights=True))
    seen = []

    def zero_masters(optimizer, state_dict):
        state = {k: {**v, "master": torch.zeros_like(v["master"])} for k, v in state_dict["state"].items()}
        return {**state_dict, "state": state}

    def after(optimizer):
        for group in optimizer.param_groups:
            for p in group["params"]:
                st = optimizer.state[p]
                seen.append((st["moment"].dtype, float(st["master"].abs().max())))
                st["master"].fill_(2.0)

    other.register_load_state_dict_pre_hook(zero_masters)
    other.register_load_state_dict_post_hook(after)
    other.load_state_dict(opt.state_dict())
    assert seen == [(F8, 0.0)] * 2
    for p, q in zip(*[[p for g in o.param_groups for p in g["params"]] for o in (opt, other)]):
        assert bool((other.state[q]["master"] == 2).all()) and not bool((opt.state[p]["master"] == 2).any())
        assert torch.equal(opt.state[p]["moment"].view(torch.uint8), other.state[q]["moment"].view(torch.uint8))
    # nothing of the load stays behind: a second one runs the same two hooks
    other.load_state_dict(opt.state_dict())
    assert len(seen) == 4 and len(other._optimizer_load_state_dict_pre_hooks) == 1
    assert len(other._optimizer_load_state_dict_post_hooks) == 1


def test_a_checkpoint_without_masters_says_so():
    """torch takes a group's keys from the checkpoint: one that was saved without master weights
    turns them off, and the load warns."""
    import warnings

    plain = _with_state(_groups())
    other = THORN(_groups(master_weights=True))
    with pytest.warns(UserWarning, match="without master weights"):
        other.load_state_dict(plain.state_dict())
    for opts in (dict(master_weights=True), dict()):  # nothing to say
        opt, other = _with_state(_groups(**opts)), THORN(_groups(**opts))
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            other.load_state_dict(opt.state_dict())
    fp32 = [torch.nn.Parameter(torch.zeros(4))]  # its own master
    groups = [{"params": fp32, "lr": 1e-3, "orthogonalize": False}]
    opt, other = THORN(groups), THORN([{**groups[0], "master_weights": True}])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        other.load_state_dict(opt.state_dict())


class _Cuda:
    """torch.cuda's current device and capture state, for two devices of which the second captures."""

    def __init__(self, monkeypatch):
        self.now = 0
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.now == 1)
        outer = self

        class device:
            def __init__(self, dev):
                self.dev = torch.device(dev)

            def __enter__(self):
                self.old, outer.now = outer.now, self.dev.index

            def __exit__(self, *exc):
                outer.now = self.old

        monkeypatch.setattr(torch.cuda, "device", device)


def test_capture_is_looked_for_on_the_tensors_device(monkeypatch):
    class T:
        def __init__(self, dev):
            self.device = torch.device(dev)

    cuda = _Cuda(monkeypatch)
    assert M._device(T("cuda:0")) == torch.device("cuda:0")
    with pytest.raises(RuntimeError, match="captured"):
        M._device(T("cuda:1"))
    cuda.now = 1  # a capture on another device than the tensors'
    assert M._device(T("cuda:0")) == torch.device("cuda:0")
    with pytest.raises(RuntimeError, match="captured"):
        M._device(T("cuda:1"))
    assert cuda.now == 1


@pytest.mark.parametrize("opts", [dict(state_dtype=F8), dict(master_weights=True)])
@pytest.mark.parametrize("ortho", [True, False])
def test_a_refused_capture_leaves_no_state(monkeypatch, opts, ortho):
    """State that is made during a capture would be filled by the graph's replays only."""
    def capturing(dev):
        raise RuntimeError("captured")

    p = torch.nn.Parameter(torch.ones(8, 8, dtype=torch.bfloat16))
    opt = THORN([{"params": [p], "lr": 1e-3, "orthogonalize": ortho, **opts}])
    p.grad = torch.ones_like(p)
    with monkeypatch.context() as m:
        m.setattr(M, "refuse_capture", capturing)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
        assert "step" not in opt.state[p]
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        opt.step()
    with monkeypatch.context() as m:  # state that is there: refused as well
        m.setattr(M, "refuse_capture", capturing)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()


def test_sparse_gradients_are_refused_by_the_state_that_is_there():
    """A row update beside a master copy would be lost at the next dense step: the state decides,
    also where the group's keys were changed after it was made; fp32 parameters of a group with
    masters have none, and take sparse gradients as ever."""
    def sparse(p):
        return torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 8, dtype=p.dtype), (8, 8),
                                       check_invariants=True)

    for opts in (dict(state_dtype=F8), dict(master_weights=True)):
        p = torch.nn.Parameter(torch.ones(8, 8, dtype=torch.bfloat16))
        opt = _with_state([{"params": [p], "lr": 1e-3, "orthogonalize": False, **opts}])
        opt.param_groups[0].update(state_dtype=None, master_weights=False)
        p.grad = sparse(p)
        with pytest.raises(NotImplementedError, match="sparse"):
            opt.step()
    p = torch.nn.Parameter(torch.ones(8, 8))
    opt = THORN([{"params": [p], "lr": 1e-3, "orthogonalize": False, "master_weights": True}])
    p.grad = sparse(p)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        opt.step()


def _adam_args(ps):
    return dict(params=ps, grads=[torch.zeros_like(p) for p in ps], moments=[torch.zeros_like(p) for p in ps],
                variances=[torch.zeros_like(p) for p in ps], step=1, lr=1e-3)


class _Launched(Exception):
    pass


@pytest.fixture
def host_only(monkeypatch):
    """The functions on CPU tensors up to the launch, which raises."""
    def launch(*a, **k):
        raise _Launched

    monkeypatch.setattr(M, "_device", lambda t: t.device)
    monkeypatch.setattr(M, "_on", lambda dev: M._here)
    monkeypatch.setattr(M, "_stream", lambda dev: 0)
    for name in ("launch_adam", "_momentum_call", "launch_apply"):
        monkeypatch.setattr(M, name, launch)


@pytest.mark.parametrize("order", [1, -1])
def test_tensors_of_a_list_that_overlap_are_refused(host_only, order):
    """Two entries of one list that share some of their memory would be written by two blocks at once."""
    buf = torch.zeros(300, dtype=torch.bfloat16)
    w = torch.zeros(300)
    cuts = [((0, 100), (99, 200)), ((0, 300), (120, 130)), ((5, 6), (0, 300))]
    touching = [((0, 100), (100, 200)), ((7, 9), (9, 10)), ((0, 0), (0, 300)), ((100, 100), (0, 300))]
    for pairs, error in ((cuts, ValueError), (touching, _Launched)):
        for pair in pairs:
            ps, ws = [[t[a:b] for a, b in pair[::order]] for t in (buf, w)]
            us = [p.half() for p in ps]
            apart = [torch.zeros_like(p) for p in ps]
            with pytest.raises(error):
                M.apply_update_(ps, us, masters=[t.float() for t in apart], lr=1e-3)
            with pytest.raises(error):
                M.apply_update_(apart, us, masters=ws, lr=1e-3)
            # what is only read may overlap
            with pytest.raises(_Launched):
                M.apply_update_(apart, ps, masters=[t.float() for t in apart], lr=1e-3)


def test_writes_are_visible_to_autograd(host_only, monkeypatch):
    """What a call writes counts as modified in place, as after torch's own operations: a graph that
    saved it refuses to run backward.  What is only read, 8-bit state, which no operation saves, and
    refused calls count nothing."""
    for name in ("launch_adam", "_momentum_call", "launch_apply"):
        monkeypatch.setattr(M, name, lambda *a, **k: None)
    p = [torch.nn.Parameter(torch.ones(3, 50).bfloat16()) for _ in range(2)]
    st = [M.state8_zeros(t) for t in p + p]
    a = dict(params=p, grads=[torch.zeros_like(t) for t in p], moments=[c for c, _ in st[:2]],
             variances=[c for c, _ in st[2:]], moment_scales=[s for _, s in st[:2]],
             variance_scales=[s for _, s in st[2:]], masters=[t.detach().float() for t in p])
    lists = [a["params"], a["masters"]]
    loss = (p[0] * p[0]).sum()
    was = [[t._version for t in x] for x in lists]
    with pytest.raises(ValueError):
        M.adamw_(**a, seeds=[1], step=1, lr=1e-3)
    assert was == [[t._version for t in x] for x in lists]
    M.adamw_(**a, seeds=[1, 2], step=1, lr=1e-3)
    assert [[v + 1 for v in x] for x in was] == [[t._version for t in x] for x in lists]
    assert all(g._version == 0 for g in a["grads"])
    b = dict(a, moments=[torch.zeros(3, 50) for _ in p], variances=[torch.zeros(3, 50) for _ in p])
    b = {k: v for k, v in b.items() if "scales" not in k}
    M.adamw_(**b, step=1, lr=1e-3)
    assert all(t._version == 1 for k in ("moments", "variances") for t in b[k])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    g, codes, scales = [torch.zeros(5, 7)], *[[t] for t in M.state8_zeros(torch.zeros(5, 7), per_matrix=True)]
    out = [torch.zeros(5, 7, dtype=torch.float16)]
    M.momentum_(g, codes, scales, beta=0.9, seeds=[1], out=out)
    assert (out[0]._version, g[0]._version) == (1, 0)
    q, w, u = [torch.zeros(4).bfloat16()], [torch.zeros(4)], [torch.zeros(4).half()]
    M.apply_update_(q, u, masters=w, lr=1e-3)
    assert (q[0]._version, w[0]._version, u[0]._version) == (1, 1, 0)
    with torch.inference_mode():  # tensors without a version
        M.apply_update_([torch.zeros(4).bfloat16()], [torch.zeros(4).half()], masters=[torch.zeros(4)], lr=1e-3)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_written_blocks_that_are_not_finite_hold_nan_codes(bad):
    """As the kernels write them: they read a block's values as code times scale, and 255 is not a
    scale that makes NaN of every code."""
    x = torch.linspace(-1, 1, 300)
    x[130] = bad
    for positive in (False, True):
        codes, scales = M.state8_write(x.abs() if positive else x, positive=positive)
        c = codes.view(torch.uint8) & 127
        assert bool((c[128:256] == 127).all()) and not bool((c[:128] == 127).any()) and not bool((c[256:] == 127).any())
        assert scales.view(torch.uint8).tolist()[1] == 255


def test_magma8_record_and_refusals():
    """Layout of the record, and bad arguments, which are refused before anything touches the device."""
    import ctypes
    import os
    import subprocess
    import tempfile

    from thorn_b200 import _native as N

    names = [f for f, _ in N.Magma8Tensor._fields_]
    with tempfile.TemporaryDirectory() as d:
        src = "".join(f'printf("%zu\\n", offsetof(thorn_magma8_tensor, {f}));' for f in names)
        open(f"{d}/a.c", "w").write('#include <stdio.h>\n#include <stddef.h>\n#include "thorn_b200.h"\nint main(void) {'
                                    + src + 'printf("%zu\\n", sizeof(thorn_magma8_tensor)); return 0; }')
        subprocess.run(["gcc", "-I", B.INCLUDE, f"{d}/a.c", "-o", f"{d}/a"], check=True)
        want = [int(x) for x in subprocess.run([f"{d}/a"], capture_output=True, text=True, check=True).stdout.split()]
    assert want == [getattr(N.Magma8Tensor, f).offset for f in names] + [ctypes.sizeof(N.Magma8Tensor)]
    lib, P = N.load(), 1 << 20

    def call(n=1, dt=N.BF16, **kw):
        t = N.Magma8Tensor(P, P, P, None, None, 60, 2, 6, 10, P, P, 0)
        for k, v in kw.items():
            setattr(t, k, v)
        return lib.thorn_magma_stats8_multi(N.array(N.Magma8Tensor, [t]), n, dt, None)

    assert call(n=0) == 0 and call(rows=0, run=0) == 0
    assert call(n=-1) == 1 and call(dt=9) == 1 and call(batch=-1) == 1
    for k in ("g", "m", "m_scale", "out", "scratch"):
        assert call(**{k: None}) == 1, k
    assert call(run=61) == 1 and call(run=0) == 1
    assert call(row_gain=P) == 1  # split gains without the columns'


# ------------------------------------------------------------------ masters of sharded parameters
def _sharded_masters(rank, world, port, q):
    import datetime
    import traceback

    import torch.distributed as dist

    try:
        dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world,
                                timeout=datetime.timedelta(seconds=60))
        from torch.distributed.device_mesh import init_device_mesh
        from torch.distributed.tensor import DTensor, Shard, distribute_tensor

        from thorn_b200 import _native as N
        from thorn_b200.optimizer import GroupConfig

        seen = []

        class Lib:
            def thorn_adamw_master_multi(self, recs, n, *scalars):
                seen.extend((t.p, t.g, t.w, t.m, t.v, t.numel) for t in list(recs)[:n])
                return 0

        N.load = lambda build_if_missing=False: Lib()
        N.stream_of = lambda dev: 0
        mesh = init_device_mesh("cpu", (world,))
        torch.manual_seed(0)
        full = [torch.randn(s).bfloat16() for s in ((5, 3), (1,), (7,))]  # shards of different lengths, and an empty one

        def make():
            ps = [torch.nn.Parameter(distribute_tensor(t, mesh, [Shard(0)])) for t in full]
            return ps, THORN([{"params": ps, "lr": 1e-3, "orthogonalize": False, "master_weights": True}])

        ps, opt = make()
        for p in ps:
            p.grad = torch.zeros_like(p)
            opt._init_state(p, opt.state[p], GroupConfig.from_kwargs(**opt.param_groups[0]), opt.param_groups[0])
            st = opt.state[p]
            for k in ("master", "moment", "variance"):
                assert isinstance(st[k], DTensor) and st[k].placements == p.placements
                assert st[k].dtype is torch.float32 and st[k].to_local().shape == p.to_local().shape
            assert torch.equal(st["master"].to_local(), p.to_local().float())
        grads = [p.grad for p in ps]
        opt._adam_local(ps, GroupConfig.from_kwargs(**opt.param_groups[0]))
        loc = [[t.to_local() for t in (p.data, g, *[opt.state[p][k] for k in ("master", "moment", "variance")])]
               for p, g in zip(ps, grads)]
        assert [(*[x or 0 for x in r[:5]], r[5]) for r in seen] == \
            [(*[t.data_ptr() for t in ts], ts[0].numel()) for ts in loc], (rank, seen)
        opt.state[ps[0]]["master"].to_local().add_(1e-6)
        qs, other = make()
        other.load_state_dict(opt.state_dict())
        for p, r in zip(ps, qs):
            for k in ("master", "moment", "variance"):
                a, b = opt.state[p][k], other.state[r][k]
                assert b.dtype is a.dtype and b.placements == a.placements and torch.equal(a.to_local(), b.to_local())
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, None))
    except Exception:
        q.put((rank, traceback.format_exc()))


def test_masters_of_sharded_adamw_parameters():
    """A Shard(0) parameter's master and moments are sharded alike, the step is given each rank's own
    shards, and a load keeps them."""
    import socket

    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_sharded_masters, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(60)
    assert [err for _, err in got] == [None, None], got


# ------------------------------------------------------------------------------------- the build
def test_host_extension_is_of_this_torch_and_python(tmp_path, monkeypatch):
    """Its file is named by what it is compiled against, so one of another torch or Python that
    travelled with the tree is left alone."""
    import sysconfig

    from thorn_b200 import _native as N

    assert torch.__version__ in B.HOST_LIB and sysconfig.get_config_var("SOABI") in B.HOST_LIB
    assert N.host().__spec__.origin == B.HOST_LIB
    monkeypatch.setattr(B, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    other = B.host_lib()
    assert other != B.HOST_LIB and other.startswith(str(tmp_path))
    (tmp_path / "given.so").write_bytes(open(B.HOST_LIB, "rb").read())
    monkeypatch.setenv("THORN_B200_HOST_EXTENSION", str(tmp_path / "given.so"))
    monkeypatch.setattr(N, "_host", None)
    assert N.host().__spec__.origin == str(tmp_path / "given.so")
    monkeypatch.setenv("THORN_B200_HOST_EXTENSION", str(tmp_path / "missing.so"))
    monkeypatch.setattr(N, "_host", None)
    with pytest.raises(RuntimeError, match="host extension not found"):
        N.host()


def test_the_library_is_built_without_the_host_extension(monkeypatch):
    """A machine without a C++ compiler or torch's headers still gets the CUDA library, then the error."""
    import subprocess

    ran = []

    def no_compiler(cmd, **kw):
        ran.append(cmd[0])
        raise FileNotFoundError(cmd[0])

    monkeypatch.setattr(subprocess, "run", no_compiler)
    monkeypatch.setattr(B, "_stale", lambda: False)
    monkeypatch.setattr(B, "HOST_SRC", __file__)  # newer than the extension
    monkeypatch.setattr(B.os.path, "getmtime", lambda p: float(p == __file__))
    assert B.build_library() == B.LIB and not ran
    with pytest.raises(FileNotFoundError):
        B.build()
    monkeypatch.setattr(B, "_stale", lambda: True)
    monkeypatch.setattr(B, "_nvcc", lambda: "nvcc")
    ran.clear()
    with pytest.raises(FileNotFoundError):
        B.build()
    assert ran == ["nvcc"]  # the library comes first
