"""Gradient norm and clipping without a GPU: refusals before any launch, and the sharded norm
over two gloo ranks with the kernels' place taken by their formulas."""
import ctypes
import math
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from muon_sr_b200 import TritonAdamW, _lib, clip_grad_norm_, get_total_norm
from muon_sr_b200 import kernels as K
from muon_sr_b200.sharding import Sharder


def _param(dtype=torch.bfloat16):
    p = torch.nn.Parameter(torch.zeros(4, 4, dtype=dtype))
    p.grad = torch.ones(4, 4, dtype=dtype)
    return p


def test_refusals():
    p = _param()
    for bad in (3.0, 0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            get_total_norm([p.grad], bad)
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([p], 1.0, bad)
    for bad in (-0.5, math.nan, -math.inf):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="grad_scale"):
            clip_grad_norm_([p], 1.0, grad_scale=bad)
    with pytest.raises(ValueError, match="no CPU path"):
        get_total_norm([p.grad])
    with pytest.raises(ValueError, match="no CPU path"):
        clip_grad_norm_(p, 1.0)
    opt = TritonAdamW([p])
    with pytest.raises(ValueError, match="no CPU path"):
        opt.step(max_norm=1.0)
    assert not opt.state                     # refused before the step counted
    with pytest.raises(ValueError, match="grad_scale needs max_norm"):
        opt.step(grad_scale=0.5)


def test_binding_serves_cuda_tensors_only():
    p = _param()
    for args in ([p.grad], [], [None], (p.grad,)):
        assert K.plain_grad_norm(args, 2.0, 1.0, 1.0) is None
    for args in ([p], [], [None], [torch.nn.Parameter(torch.zeros(3))], (p,)):
        assert K.plain_grad_clip_(args, 2.0, 1.0, 1.0) is None
    with pytest.raises(TypeError):
        _lib.native().grad_clip()


def test_nothing_to_clip():
    assert float(get_total_norm([])) == 0.0
    total, each = get_total_norm([], per_tensor=True)
    assert float(total) == 0.0 and each.shape == (0,)
    p = _param()
    p.grad = None
    assert float(clip_grad_norm_([p], 1.0)) == 0.0


def test_dense_means_one_stretch_of_memory():
    x = torch.zeros(6, 8)
    assert K.is_dense(x) and K.is_dense(x.t()) and K.is_dense(x[2:4]) and K.is_dense(x[:1, :1])
    assert K.is_dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))
    assert not K.is_dense(x[:, :4]) and not K.is_dense(x[::2]) and not K.is_dense(x[0].expand(3, 8))
    assert not K.is_dense(torch.zeros(9).as_strided((3, 3), (1, 1)))


def test_c_argument_errors():
    lib = _lib.load()
    at = ctypes.create_string_buffer(64)
    ptr = (ctypes.addressof(at) + 15) // 16 * 16      # never dereferenced: every call is refused
    need = lib.msr_grad_norm_workspace_bytes(1)
    assert need > 0 and lib.msr_grad_norm_workspace_bytes(-1) == 0

    def norm(words=(ptr, 4, 0), count=1, kind=2, scale=1.0, bound=1.0, state=ptr, ws=ptr, size=need):
        arr = (ctypes.c_int64 * 3)(*words)
        st = lib.msr_grad_norm(arr, count, kind, scale, bound, state, None, ws, size, None)
        assert lib.msr_grad_clip(arr, count, kind, scale, bound, state, ws, size, None) == st
        return st
    for kw in (dict(count=-1), dict(kind=3), dict(kind=-1), dict(scale=0.0), dict(scale=math.inf),
               dict(scale=math.nan), dict(bound=-1.0), dict(bound=math.nan), dict(state=None), dict(state=ptr + 4),
               dict(ws=None), dict(ws=ptr + 4), dict(words=(0, 4, 0)), dict(words=(ptr, -1, 0)),
               dict(words=(ptr, 4, 3)), dict(words=(ptr + 1, 4, 0)), dict(words=(ptr + 2, 4, 2))):
        assert norm(**kw) == 1, kw
        assert lib.msr_last_error().startswith(b"msr_grad_clip")
    assert norm(size=need - 1) == 4
    assert lib.msr_grad_norm(None, 1, 2, 1.0, 1.0, ptr, None, ptr, need, None) == 1
    assert lib.msr_grad_factor(None, 2, 1.0, 1.0, None) == 1
    assert lib.msr_grad_factor(ptr, 7, 1.0, 1.0, None) == 1
    two = (ctypes.c_int64 * 6)(ptr, 8, 0, ptr + 14, 8, 0)
    assert lib.msr_grad_scale(two, 2, ptr, None) == 1 and b"overlap" in lib.msr_last_error()
    assert lib.msr_grad_scale(two, 2, None, None) == 1
    assert lib.msr_grad_scale(None, 0, ptr, None) == 0
    assert lib.msr_muon_prepare_scaled(None, 0, 0.9, 0.1, 1, None, None) == 1
    assert lib.msr_adamw_sr_scaled(None, 0, None, None, None) == 1
    assert lib.msr_muon_prepare_rec_scaled(None, 0, ptr, None, None) == 1
    assert lib.msr_muon_prepare_rec_scaled(None, 0, ptr + 4, ptr, None) == 1
    assert lib.msr_adamw_sr_rec_scaled(None, 0, ptr, None, None) == 1
    assert lib.msr_adamw8bit_scaled(None, 0, None, None, None, None, None) == 1


def test_state_layout():
    assert ctypes.sizeof(_lib.ClipState) == 24
    assert (_lib.ClipState.norm.offset, _lib.ClipState.factor.offset, _lib.ClipState.active.offset) == (8, 12, 16)
    n = K.GradNorm("cpu")
    n.state.zero_()
    n.power(2.0).fill_(2.5)
    assert _lib.ClipState.from_buffer_copy(n.state.numpy().tobytes()).power == 2.5
    bits = n.power(math.inf)
    assert bits.dtype == torch.int64 and bits.view(torch.float64).item() == 2.5
    n.norm.fill_(3.0)
    n.factor.fill_(4.0)
    st = _lib.ClipState.from_buffer_copy(n.state.numpy().tobytes())
    assert (st.norm, st.factor) == (3.0, 4.0)


def _fake_kernels():
    """The kernels' formulas on CPU tensors, in place of the launches."""
    class Table:
        def __init__(self, grads, device=None):
            self.grads = self.dense = grads

    def put(out, kind, scale, bound, power):
        norm = (math.sqrt(power) if kind == 2.0 else power) * scale
        out.norm.fill_(norm)
        out.factor.fill_(scale * min(1.0, bound / (norm + 1e-6)) if bound != math.inf else scale)

    def grad_norm(table, kind, scale, bound):
        grads, out = table.grads, K.GradNorm("cpu")
        each = [float(g.double().abs().max()) if kind == math.inf else float((g.double().abs() ** kind).sum())
                for g in grads]
        power = max(each, default=0.0) if kind == math.inf else sum(each)
        out.state[:2].view(torch.float64).fill_(power)
        put(out, kind, scale, bound, power)
        return out

    def factor(out, kind, scale, bound):
        put(out, kind, scale, bound, out.state[:2].view(torch.float64).item())

    def scale(table, out):
        for g in table.grads:
            g.mul_(out.factor.to(g.dtype))
    K.GradTable, K.grad_norm, K.grad_factor, K.grad_scale_ = Table, grad_norm, factor, scale


def _shard_worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.cuda.current_device = lambda: 0
        _fake_kernels()
        # one large and several small tensors, one of them without a gradient
        params = [torch.nn.Parameter(torch.zeros(s)) for s in ((40, 50), (3,), (5,), (2, 2), (7,))]
        opt = torch.optim.SGD(params, lr=0.1)
        sh = Sharder()
        refused = 0
        params[0].grad = torch.ones(40, 50)
        try:
            clip_grad_norm_(params, 1.0, shard=sh)
        except RuntimeError as e:
            refused = int("reduce_grads" in str(e))
        res = []
        for kind in (2.0, 1.0, math.inf):
            for i, p in enumerate(params):
                p.grad = None if i == 3 else torch.full(p.shape, float(1 + i + 2 * rank))
            sh.reduce_grads(opt)      # the mean over the ranks, 2 + i, at its owner
            mine = sh.owned([p for p in params if p.grad is not None])
            kept = {i: p.grad.clone() for i, p in enumerate(params) if p.grad is not None}
            norm = clip_grad_norm_(params, 1.5, kind, grad_scale=0.5, shard=sh)
            full = [2.0 + i for i in range(5) if i != 3 for _ in range(params[i].numel())]
            want = 0.5 * (max(full) if kind == math.inf else sum(x ** kind for x in full) ** (1 / kind))
            f = 0.5 * min(1.0, 1.5 / (want + 1e-6))
            ok = abs(float(norm) - want) < 1e-5 * want
            for i, g in kept.items():
                own = any(params[i] is p for p in mine)
                ok &= bool(torch.allclose(params[i].grad, g * f if own else g, rtol=1e-5))
            # a rank whose share holds a NaN makes every rank's norm NaN
            if mine and rank == 0:
                mine[0].grad.view(-1)[0] = math.nan
            if kind != math.inf:  # (a sum carries it; the maximum goes by the bits, below)
                ok &= math.isnan(float(clip_grad_norm_(params, 1.5, kind, shard=sh)))
            res.append(bool(ok))
        power = torch.tensor([math.nan if rank == 1 else math.inf], dtype=torch.float64).abs().view(torch.int64)
        sh.combine_power(power)
        res.append(math.isnan(power.view(torch.float64).item()))
        # every gradient on one rank: the other has nothing of its own but joins the sum
        for p in params[1:]:
            p.grad = None
        params[0].grad = torch.full((40, 50), 2.0)
        sh.reduce_grads(opt)
        norm = clip_grad_norm_(params, math.inf, shard=sh)
        res.append(abs(float(norm) - 2.0 * math.sqrt(2000)) < 1e-3)
        out.put((rank, refused, res))
    finally:
        dist.destroy_process_group()


def test_sharded_norm_two_ranks_gloo():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29800 + os.getpid() % 1000
    procs = [ctx.Process(target=_shard_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(q.get(timeout=60) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for rank, refused, res in got:
        assert refused == 1 and all(res), (rank, refused, res)
