"""Clipping on the GPU where its callers' data goes wrong: non-finite norms, gradients that
share memory, bounds of infinity, and the borders of the chunks."""
import math

import pytest
import torch

from muon_sr_b200 import (MuonSRWithAuxAdam, StepGraph, TritonAdamW, TritonAdamW8bit, TritonMuonSR,
                          TritonMuonSRWithAuxAdam, clip_grad_norm_, get_total_norm, set_sr_noise)
from muon_sr_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def raw(t):
    return t.detach().contiguous().view(-1).view(torch.uint8)


def same_bits(a, b):
    return torch.equal(raw(a), raw(b))


# ---- the 8-bit step under a non-finite norm ---------------------------------------------
SIZES = [5000, 300, 8192, 4097]  # block tails, and one below min_8bit_size (bf16 moments)


def eight_bit(block_size):
    gen = torch.Generator().manual_seed(3)
    params = [torch.nn.Parameter((torch.randn(n, generator=gen) * 0.02).to(torch.bfloat16).to(DEV)) for n in SIZES]
    return params, TritonAdamW8bit(params, lr=1e-3, weight_decay=0.01, min_8bit_size=512, block_size=block_size)


def fill(params, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=gen) * 1e-2).to(torch.bfloat16).to(DEV)


def tensors_of(params, opt):
    return [t for p in params for t in (p, *(v for _, v in sorted(opt.state[p].items()) if torch.is_tensor(v)))]


@pytest.mark.parametrize("lookup", [True, False])
@pytest.mark.parametrize("block_size", [64, 256, 4096])
def test_8bit_step_by_a_nan_norm_leaves_everything(block_size, lookup, monkeypatch):
    """One NaN makes the norm and the factor NaN: no parameter's moments may be lost to it."""
    if not lookup:
        monkeypatch.setattr(K, "quant_tables", lambda *a: None)
    params, opt = eight_bit(block_size)
    for step in range(2):
        fill(params, step)
        opt.step(max_norm=1.0)
    before = [t.detach().clone() for t in tensors_of(params, opt)]
    weights = [p.detach().clone() for p in params]
    fill(params, 2)
    params[0].grad[77] = math.nan
    opt.step(max_norm=1.0)
    assert math.isnan(float(opt.grad_norm))
    for i, (a, b) in enumerate(zip(tensors_of(params, opt), before)):
        assert same_bits(a, b), i
    fill(params, 3)                                           # and training goes on
    opt.step(max_norm=1.0)
    assert math.isfinite(float(opt.grad_norm))
    assert not any(same_bits(p, w) for p, w in zip(params, weights))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_8bit_step_with_a_finite_factor_keeps_the_rule_of_each_element(bad):
    """max_norm = inf clips nothing, so the factor stays 1 whatever the norm, and a non-finite
    gradient touches its own element alone, as in a step without clipping."""
    (pa, oa), (pb, ob) = eight_bit(256), eight_bit(256)
    for step in range(2):
        for ps in (pa, pb):
            fill(ps, step)
            ps[2].grad[4000] = bad
        oa.step()
        ob.step(max_norm=math.inf)
        assert not math.isfinite(float(ob.grad_norm))
        assert all(same_bits(a, b) for a, b in zip(tensors_of(pa, oa), tensors_of(pb, ob)))


def test_8bit_step_by_an_infinite_norm_is_that_of_scaled_gradients():
    """Infinity gives a factor of 0: gradients of 0 and, where they were infinite, NaN."""
    (pa, oa), (pb, ob) = eight_bit(256), eight_bit(256)
    for ps, o in ((pa, oa), (pb, ob)):
        fill(ps, 0)
        o.step()
        fill(ps, 1)
        ps[3].grad[5] = -math.inf
    for p in pa:
        p.grad.mul_(0.0)
    oa.step()
    ob.step(max_norm=1.0)
    assert float(ob.grad_norm) == math.inf
    assert all(same_bits(a, b) for a, b in zip(tensors_of(pa, oa), tensors_of(pb, ob)))

# ---- gradients that share memory ---------------------------------------------------------
def clip(grads, max_norm=0.5):
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=DEV))
        p.grad = g
        params.append(p)
    return clip_grad_norm_(params, max_norm)


@pytest.mark.parametrize("views", [
    lambda x: [x[:, 2:30], x[:, 2:30]],                      # one non-dense view twice
    lambda x: [x[:, 2:30], x[:, 29:40]],                     # a column in common
    lambda x: [x[::2], x[4:9]],                              # rows in common, one view dense
    lambda x: [x, x[:, 5]],
    lambda x: [x[:, ::3], x[:, ::2].t()],
    lambda x: [x[:10, :7], x[20:, 9:], x[9:21, 6:10]],       # the third meets both
])
def test_strided_gradients_that_share_memory_are_refused(views):
    x = torch.randn(40, 64, device=DEV).to(torch.bfloat16)
    before = x.clone()
    with pytest.raises(RuntimeError, match="overlap in memory"):
        clip(views(x))
    assert same_bits(x, before)


@pytest.mark.parametrize("views", [
    lambda x: [x[:, 0::2], x[:, 1::2]],                      # interleaved, nothing in common
    lambda x: [x[:, :30], x[:, 30:].t()],
    lambda x: [x[::2], x[1::2, 3:], x[1::2, :3]],
    lambda x: [x[:, i] for i in range(64)],
    lambda x: [x[:, 5][:0], x[:, 5], x[:, 5][:0]],           # empty views share nothing
])
def test_strided_gradients_side_by_side_are_clipped(views):
    x = torch.randn(40, 64, device=DEV).to(torch.bfloat16)
    before = x.clone()
    grads = views(x)
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    # norm: 33 roundings of fp32 at most on the power, halved by the root, and one more
    assert abs(float(clip(grads, want / 4)) - want) <= 34 * 2.0 ** -24 * want
    factor = (want / 4) / (want + 1e-6)
    inside = torch.zeros_like(x, dtype=torch.bool)
    for g in views(inside):
        g.fill_(True)
    scaled = before.double() * factor
    # half a bf16 step, the factor's error and a product's (34 + 1 + 1 roundings of fp32)
    tol = scaled.abs() * (2.0 ** -8 + 37 * 2.0 ** -24) + 2.0 ** -134
    assert bool(((x.double() - scaled).abs() <= tol)[inside].all())
    assert torch.equal(x[~inside], before[~inside])


# ---- a bound of infinity -----------------------------------------------------------------
@pytest.mark.parametrize("sizes", [[40, 9], [9000, 600000]])  # one cluster, two kernels
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_bound_of_infinity_clips_nothing_whatever_the_norm(sizes, bad):
    grads = [torch.randn(n, device=DEV).to(torch.bfloat16) for n in sizes]
    grads[1][3] = bad
    before = [g.clone() for g in grads]
    norm = float(clip(grads, math.inf))
    assert norm == math.inf if bad == math.inf else math.isnan(norm)
    assert all(same_bits(g, b) for g, b in zip(grads, before))
    params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    clip_grad_norm_(params, math.inf, grad_scale=0.5)                      # (exact: a power of two)
    assert all(torch.equal(g.nan_to_num(7), (b * 0.5).nan_to_num(7)) for g, b in zip(grads, before))


# ---- the norm at the borders of its chunks ------------------------------------------------
# A power is a double sum of fp32 sums of at most 32 values, in two halves that are added: a term
# passes 16 roundings (a square and its addition are one) and that of the halves, 17 * 2^-24 of a
# sum of non-negative terms. The root halves it; the result is rounded to fp32 once more, 2^-24.
# One more covers the products of these errors.
TOL = {1.0: 19 * 2.0 ** -24, 2.0: (17 / 2 + 2) * 2.0 ** -24}


@pytest.mark.parametrize("p", [1.0, 2.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_at_chunk_borders(p, dtype, offset):
    """Chunks are of 2048 vectors of 16 bytes (1024 in the one-cluster kernel): 16384 and 8192
    elements of 16 and 32 bits; together these sets take the two kernels, one by one the cluster."""
    sizes = [4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 16391, 32767, 32768, 32769, 262143, 262144, 262145]
    gen = torch.Generator(device=DEV).manual_seed(offset)
    grads = [(torch.randn(offset + n, device=DEV, generator=gen) * 1e-2).to(dtype)[offset:] for n in sizes]
    power = [float((g.double().abs() ** p).sum()) for g in grads]
    total, each = get_total_norm(grads, p, per_tensor=True)
    assert abs(float(total) - sum(power) ** (1 / p)) <= TOL[p] * sum(power) ** (1 / p)
    for n, g, got, x in zip(sizes, grads, each.tolist(), power):
        want = x ** (1 / p)
        assert abs(got - want) <= TOL[p] * want, n
        assert abs(float(get_total_norm([g], p)) - want) <= TOL[p] * want, n


def test_norm_with_and_without_each():
    """The same partial sums joined in another order: in double, so at most one fp32 step apart."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    grads = [torch.randn(n, device=DEV, generator=gen).to(torch.bfloat16) for n in (1000003, 5, 70001, 64, 4096 * 9)]
    for p in (1.0, 2.0, math.inf):
        for some in (grads, grads[1:2] + grads[3:]):
            a, b = float(get_total_norm(some, p)), float(get_total_norm(some, p, per_tensor=True)[0])
            assert a == b if p == math.inf else abs(a - b) <= 2.0 ** -23 * a


# ---- steps by a NaN norm, every optimizer -------------------------------------------------
MUON = [(24, 40)] * 3 + [(40, 24)] * 2 + [(16, 16)]
ADAM = [(30, 16), (16,), (4099,), (1,)]


def hybrid(cls, params, **kw):
    return cls([dict(params=params[:len(MUON)], use_muon=True, lr=0.02, weight_decay=0.01),
                dict(params=params[len(MUON):], use_muon=False, lr=3e-4, eps=1e-10)], **kw)


OPTIMIZERS = {
    "adamw": lambda ps: TritonAdamW(ps, lr=1e-3, weight_decay=0.01),
    "adamw centralized": lambda ps: TritonAdamW(ps, lr=1e-3, centralization=0.5),
    "muon": lambda ps: TritonMuonSR(ps[:len(MUON)], lr=0.02, weight_decay=0.01),
    "muon batched": lambda ps: TritonMuonSR(ps[:len(MUON)], lr=0.02, weight_decay=0.01, batch_ns=True),
    "hybrid": lambda ps: hybrid(TritonMuonSRWithAuxAdam, ps, batch_ns=True),
    "hybrid random": lambda ps: hybrid(MuonSRWithAuxAdam, ps, batch_ns=True),
}


def parameters(seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.02).to(torch.bfloat16).to(DEV)) for s in MUON + ADAM]


def refill(params, seed):
    """New values in the gradients' memory."""
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        if p.grad is None:
            p.grad = torch.empty_like(p)
        p.grad.copy_((torch.randn(p.shape, generator=gen) * 1e-2).to(torch.bfloat16))


@pytest.fixture(params=["reference", "fast", "none"])
def noise(request):
    set_sr_noise(request.param)
    try:
        yield request.param
    finally:
        set_sr_noise("reference")


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("name", OPTIMIZERS)
def test_step_by_a_nan_norm_leaves_everything(name, offset, noise):
    """Without that, stochastic rounding, which adds to the bits, would turn every weight and moment
    into -0: a NaN's bits are 0x7FFFFFFF."""
    params = parameters()
    if offset:  # weights at odd addresses
        for p in params:
            p.data = torch.cat([p.data.new_zeros(offset), p.data.flatten()])[offset:].view(p.shape)
    opt = OPTIMIZERS[name](params)
    for step in range(2):
        refill(params, step)
        opt.step(max_norm=0.5)
    before = [t.detach().clone() for t in tensors_of(params, opt)]
    refill(params, 2)
    params[4].grad[3, 5] = math.nan
    for _ in range(2):
        opt.step(max_norm=0.5)
        assert math.isnan(float(opt.grad_norm))
        for i, (a, b) in enumerate(zip(tensors_of(params, opt), before)):
            assert same_bits(a, b), i
    refill(params, 3)
    opt.step(max_norm=0.5)
    assert math.isfinite(float(opt.grad_norm))
    assert all(bool(t.isfinite().all()) for t in tensors_of(params, opt))
    assert not same_bits(params[0], before[0])


@pytest.mark.parametrize("name", ["adamw", "muon batched", "hybrid"])
def test_graph_of_steps_by_a_nan_norm(name):
    params = parameters()
    opt = OPTIMIZERS[name](params)
    refill(params, 0)
    opt.step(max_norm=0.5)
    graph = StepGraph(opt, max_norm=0.5)
    refill(params, 1)
    graph.step()
    before = [t.detach().clone() for t in tensors_of(params, opt)]
    params[2].grad[0, 0] = math.nan
    for _ in range(3):
        graph.step()
    assert math.isnan(float(opt.grad_norm))
    assert all(same_bits(a, b) for a, b in zip(tensors_of(params, opt), before))
    refill(params, 2)
    graph.step()
    assert math.isfinite(float(opt.grad_norm)) and not same_bits(params[0], before[0])


def test_step_by_an_infinite_norm_is_that_of_scaled_gradients(noise):
    """Infinity gives a factor of 0, and the damage stays where a step without clipping has it."""
    sets = []
    for scaled in (True, False):
        params = parameters()
        opt = OPTIMIZERS["hybrid"](params)
        refill(params, 0)
        opt.step()
        refill(params, 1)
        params[-2].grad[7] = math.inf
        if scaled:
            for p in params:
                p.grad.mul_(0.0)
            opt.step()
        else:
            opt.step(max_norm=1.0)
            assert float(opt.grad_norm) == math.inf
        sets.append(tensors_of(params, opt))
    assert all(same_bits(a, b) for a, b in zip(*sets))
