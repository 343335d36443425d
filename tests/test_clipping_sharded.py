"""Clipped optimizer steps over two gloo ranks, the kernels' place taken by their formulas on the
CPU: powers joined over the ranks, the factor derived again on each, and the updates of every
rank reading it -- against one process."""
import math
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from muon_sr_b200 import TritonMuonSRWithAuxAdam
from muon_sr_b200 import kernels as K
from muon_sr_b200.sharding import Sharder

MUON = [(8, 12)] * 5 + [(12, 8)] * 2
ADAM = [(9, 4), (7,), (1,)]


def fake_kernels(placed):
    """The formulas, without stochastic rounding, in fp32; `placed` notes where a rank without
    gradients puts its state."""
    class Table:
        def __init__(self, grads, device=None):
            self.grads = self.dense = grads
            if not grads:
                placed.append(device)

    def put(out, scale, bound, power):
        norm = math.sqrt(power) * scale
        out.norm.fill_(norm)
        out.factor.fill_(scale * (1.0 if bound == math.inf else min(1.0, bound / (norm + 1e-6))))

    def grad_norm(table, kind, scale, bound):
        out = K.GradNorm("cpu")
        power = sum(float(g.double().square().sum()) for g in table.grads)
        out.power(2.0).fill_(power)
        put(out, scale, bound, power)
        return out

    def grad_factor(out, kind, scale, bound):
        put(out, scale, bound, out.power(2.0).item())

    def read(g):
        return g.float() * (1.0 if K._factor() is None else K._factor())

    def prepare(items, beta, nesterov):
        for g, buf, upd, ctr, seed in items:
            buf.copy_(buf.float().lerp(read(g), 1 - beta))
            upd.copy_(read(g).lerp(buf.float(), beta))

    def apply(items, lr, weight_decay):
        for p, upd, scale, seed in items:
            p.data.copy_(p.float() * (1 - lr * weight_decay) - lr * scale * upd.float())

    def adamw(items, lr, beta1, beta2, eps, weight_decay):
        for p, g, m, v, step, seed in items:
            m.copy_(m.float().lerp(read(g), 1 - beta1))
            v.copy_(v.float().lerp(read(g).square(), 1 - beta2))
            p.data.copy_(p.float() - lr * m.float() / (v.float().sqrt() + eps))
    for name, fn in dict(GradTable=Table, grad_norm=grad_norm, grad_factor=grad_factor, muon_prepare=prepare,
                         muon_apply=apply, adamw_sr=adamw, newton_schulz=lambda x, steps, **kw: x.clone(),
                         plain_grad_norm=lambda *a, **k: None).items():
        setattr(K, name, fn)


def steps(shard, rank, clip, only=None):
    """Parameters, moments and norms after three clipped steps. With a sharder each rank starts from
    its share of the gradients, g plus or minus d, whose mean is g."""
    gen = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.02).bfloat16()) for s in MUON + ADAM]
    sh = shard() if shard else None
    opt = TritonMuonSRWithAuxAdam([dict(params=params[:len(MUON)], use_muon=True, lr=0.02),
                                   dict(params=params[len(MUON):], use_muon=False, lr=1e-3)], batch_ns=True, shard=sh)
    norms = []
    for step in range(3):
        for i, p in enumerate(params):
            # small integers: their means over two ranks are exact in bf16
            g = torch.randint(-40, 41, p.shape, generator=gen).bfloat16()
            d = torch.randint(-20, 21, p.shape, generator=gen).bfloat16()
            p.grad = None if only is not None and i not in only else g if sh is None else g + d * (1 - 2 * rank)
        if sh is not None:
            sh.reduce_grads(opt)
        opt.step(**clip)
        norms.append(opt.grad_norm.clone())
    if sh is not None:
        sh.gather_state(opt)
    moments = [t for _, st in sorted(opt.state_dict()["state"].items())
               for _, t in sorted(st.items()) if torch.is_tensor(t)]
    return [t.detach().float().numpy() for t in params + moments], [float(n) for n in norms]


CASES = {
    # a power of two that clips nothing: the same factor, so the same bits
    "scaled": dict(clip=dict(max_norm=math.inf, grad_scale=0.125)),
    # clipping: a sum in another order may move the factor by an fp32 step
    "clipped": dict(clip=dict(max_norm=0.5, grad_scale=0.5)),
    # one parameter alone: a rank that owns no gradient joins the sum
    "one gradient": dict(clip=dict(max_norm=0.5), only=[0]),
}


def worker(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        placed = []
        fake_kernels(placed)
        got = {name: steps(Sharder, rank, **case) for name, case in CASES.items()}
        out.put((rank, got, placed))
        dist.barrier()
    except BaseException as e:  # the parent reports it
        out.put((rank, repr(e), None))
        raise
    finally:
        dist.destroy_process_group()


@pytest.fixture
def kernels(monkeypatch):
    for name in ("GradTable", "grad_norm", "grad_factor", "muon_prepare", "muon_apply", "adamw_sr", "newton_schulz",
                 "plain_grad_norm"):
        monkeypatch.setattr(K, name, getattr(K, name))
    fake_kernels([])


def test_clipped_steps_two_ranks_gloo(kernels):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29600 + os.getpid() % 100
    procs = [ctx.Process(target=worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted((q.get(timeout=90) for _ in procs), key=lambda g: g[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0, got
    # in "one gradient" one of the ranks owned none, in each of three steps
    assert sorted(len(placed) for _, _, placed in got) == [0, 3]
    for name, case in CASES.items():
        want, norms = steps(None, 0, **case)
        for rank, by_case, _ in got:
            tensors, norms2 = by_case[name]
            assert all(abs(a - b) <= 2.0 ** -23 * a for a, b in zip(norms, norms2)), (name, rank)
            assert len(tensors) == len(want)
            for i, (a, b) in enumerate(zip(want, tensors)):
                if name == "scaled":
                    assert np.array_equal(a, b), (name, rank, i)
                else:
                    # an fp32 step of the factor may move a value across a border between two bf16
                    # values, at most once per step of the optimizer
                    assert np.all(np.abs(a - b) <= 3 * 2.0 ** -7 * np.maximum(np.abs(a), np.abs(b))), (name, rank, i)
        if name != "scaled":
            assert all(n > 1.0 for n in norms)              # the bound was active
