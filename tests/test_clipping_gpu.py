"""Global gradient norm and clipping on the GPU, against the definitions in 64 bits.

Tolerances, relative unless said otherwise. A power is a double sum of fp32 sums of at most 64
values, each added with one rounding of 2^-24 (a square and its addition are one fused
operation): at most 64 * 2^-24 on the power, terms being non-negative. The root of a sum of
squares halves that and the result is rounded to fp32 once more: NORM_TOL = 65 * 2^-24 covers
p = 1 and p = 2; the infinity norm is exact. The factor inherits the norm's error and one rounding: FACTOR_TOL =
66 * 2^-24. A scaled gradient adds one fp32 product and the rounding to its own type,
half a step: finfo.eps / 2 of the value, or half the smallest subnormal near zero.
"""
import math

import numpy as np
import pytest
import torch

from muon_sr_b200 import (HostStaging, MuonSRWithAuxAdam, StepGraph, TritonAdamW, TritonAdamW8bit, TritonMuonSR,
                          TritonMuonSRWithAuxAdam, clip_grad_norm_, get_total_norm, set_sr_noise)
from muon_sr_b200 import kernels as K
from oracle import elementwise as ew
from oracle.philox import triton_key
from oracle.sr import bf16_to_f32, rne_bf16
from tests._golden import assert_bits_equal, bits_of, to_bf16

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NORM_TOL = 65 * 2.0 ** -24
FACTOR_TOL = 66 * 2.0 ** -24
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
# around a vector of 16 bytes, a chunk of 1024 vectors (4096 or 8192 elements), several chunks
SIZES = [1, 2, 3, 7, 8, 9, 17, 255, 4095, 4096, 4097, 8191, 8192, 8193, 8200, 16385, 100003, 262147]


def raw(t):
    return t.detach().contiguous().view(-1).view(torch.uint8)


def same_bits(a, b):
    return torch.equal(raw(a), raw(b))


def norm64(tensors, p):
    """The definition in 64 bits: (total, of each)."""
    flat = [t.detach().cpu().double().numpy().ravel() for t in tensors]
    power = [float(np.sum(np.abs(x) ** p)) if p != math.inf else float(np.max(np.abs(x), initial=0.0)) for x in flat]
    if p == math.inf:
        return max(power, default=0.0), power
    return sum(power) ** (1 / p), [x ** (1 / p) for x in power]


def params_of(grads):
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        params.append(p)
    return params


def make(sizes, dtype, seed=0, offset=0, std=1e-2):
    """Views `offset` elements into their buffers, with 8 guard elements at the end."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    bufs = [(torch.randn(offset + n + 8, device=DEV, generator=gen) * std).to(dtype) for n in sizes]
    return bufs, [b[offset:offset + n] for b, n in zip(bufs, sizes)]


def assert_norm(got, want, p):
    got = float(got)
    if want == 0 or not math.isfinite(want):
        assert got == want or (math.isnan(got) and math.isnan(want)), (got, want)
    else:
        assert abs(got - want) <= (2.0 ** -24 if p == math.inf else NORM_TOL) * want, (got, want)


def assert_scaled(got, before, factor, what="", products=1):
    """`products`: fp32 roundings between the gradient and the stored value."""
    want = before.double() * factor
    step, fp32 = torch.finfo(got.dtype).eps / 2, FACTOR_TOL + products * 2.0 ** -24
    tol = want.abs() * (step + fp32 + step * fp32) + SMALLEST[got.dtype] / 2
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()))


# ---- the norm -------------------------------------------------------------------------
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_norm_sizes_and_offsets(p, dtype, offset):
    _, grads = make(SIZES, dtype, seed=offset, offset=offset)
    total, each = get_total_norm(grads, p, per_tensor=True)
    want, want_each = norm64(grads, p)
    assert total.dtype == torch.float32 and total.dim() == 0 and each.shape == (len(grads),)
    assert_norm(total, want, p)
    for i, (a, b) in enumerate(zip(each.tolist(), want_each)):
        assert_norm(a, b, p)
    assert_norm(get_total_norm(grads, p), want, p)          # without the tensors' own norms
    for g, b in zip(grads[:8], want_each):                  # each size by itself
        assert_norm(get_total_norm([g], p), b, p)


def test_norm_mixed_types_and_empty_tensors():
    grads = []
    for k, dtype in enumerate(DTYPES * 3):
        grads += make([5 + 1000 * k], dtype, seed=k, offset=k % 2)[1] + [torch.empty(0, dtype=dtype, device=DEV)]
    for p in (2.0, 1.0, math.inf):
        total, each = get_total_norm(iter(grads), p, per_tensor=True)
        want, want_each = norm64(grads, p)
        assert_norm(total, want, p)
        for a, b in zip(each.tolist(), want_each):
            assert_norm(a, b, p)
    assert float(get_total_norm([])) == 0.0
    total, each = get_total_norm([torch.empty(0, device=DEV)], per_tensor=True)
    assert total.is_cuda and float(total) == 0.0 and each.tolist() == [0.0]
    one = torch.tensor(-3.0, device=DEV)
    assert float(get_total_norm(one)) == 3.0                # a 0-dim tensor, not in a list


@pytest.mark.parametrize("count", [511, 512, 513, 1300])
def test_norm_many_tensors(count):
    """More tensors than one launch takes."""
    _, grads = make([1 + (i * 37) % 301 for i in range(count)], torch.bfloat16, seed=count)
    for p in (2.0, math.inf):
        total, each = get_total_norm(grads, p, per_tensor=True)
        want, want_each = norm64(grads, p)
        assert_norm(total, want, p)
        for a, b in zip(each.tolist(), want_each):
            assert_norm(a, b, p)
        assert_norm(get_total_norm(grads, p), want, p)


@pytest.mark.parametrize("dtype,values", [
    (torch.bfloat16, [1e30, 1e-30, 1e38]), (torch.bfloat16, [1e-30]), (torch.bfloat16, [1e-39, 2e-38]),
    (torch.bfloat16, [1e25, 0.0]), (torch.float32, [3e38, 1e-45]), (torch.float32, [1e-45]), (torch.float32, [1e-30, 0.0]),
    (torch.float32, [1e30]), (torch.float16, [65504.0, 6e-8]), (torch.float16, [6e-8]),
])
def test_norm_values_whose_squares_leave_fp32(dtype, values):
    n = 20011
    g = torch.tensor(values, dtype=torch.float64).repeat(n // len(values) + 1)[:n].to(dtype).to(DEV)
    for p in (2.0, 1.0, math.inf):
        _, each = get_total_norm([g, g[:5]], p, per_tensor=True)
        for got, x in zip(each.tolist(), (g, g[:5])):
            want = norm64([x], p)[0]
            if want > 3.4028235e38:
                assert got == math.inf   # the result itself is beyond fp32
            else:
                # a subnormal result is rounded to a multiple of 2^-149
                assert abs(got - want) <= NORM_TOL * want + 2.0 ** -150, (p, got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", [0, 1, 5000, 40000, 100002])
def test_norm_non_finite_values(dtype, at):
    _, (a, b) = make([100003, 300], dtype, offset=1)
    for p in (2.0, 1.0, math.inf):
        for bad in (math.inf, -math.inf, math.nan):
            x = a.clone()
            x[at] = bad
            total, each = get_total_norm([x, b], p, per_tensor=True)
            want = math.nan if math.isnan(bad) else math.inf
            assert_norm(total, want, p)
            assert_norm(each[0], want, p)
            assert math.isfinite(float(each[1]))
            x[(at + 7) % 100003] = math.nan                # NaN beside infinity is NaN
            assert math.isnan(float(get_total_norm([x, b], p)))
    x = a.clone()
    x[at] = math.nan
    with pytest.raises(RuntimeError, match="non-finite"):
        get_total_norm([x], error_if_nonfinite=True)


def test_norm_zeros_and_signed_zeros():
    g = torch.zeros(50000, dtype=torch.bfloat16, device=DEV)
    for p in (2.0, 1.0, math.inf):
        assert float(get_total_norm([g, -g], p)) == 0.0


def test_norm_strides():
    x = torch.randn(64, 96, device=DEV).to(torch.bfloat16)
    conv = torch.randn(4, 6, 5, 7, device=DEV).to(memory_format=torch.channels_last)
    views = [x.t(), x[:, 3:50], x[::3], x[5].expand(9, 96), conv, conv[:, 1:3]]
    for p in (2.0, 1.0, math.inf):
        total, each = get_total_norm(views, p, per_tensor=True)
        want, want_each = norm64(views, p)
        assert_norm(total, want, p)
        for a, b in zip(each.tolist(), want_each):
            assert_norm(a, b, p)


def test_norm_is_deterministic_and_same_with_and_without_each():
    _, grads = make([1000003, 5, 70001, 64, 4096 * 9], torch.bfloat16)
    first = get_total_norm(grads)
    for _ in range(3):
        assert same_bits(get_total_norm(grads), first)
    total, each = get_total_norm(grads, per_tensor=True)
    again, each2 = get_total_norm(grads, per_tensor=True)
    assert same_bits(total, again) and same_bits(each, each2)


def test_norm_and_clip_past_32_bit_offsets():
    """More than 2^32 elements in one tensor, an odd number of them, the last ones unlike."""
    n = (1 << 32) + 9
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 30 GB")
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    p.grad[-5:] = 1024.0
    want = math.sqrt(n - 5 + 5 * 1024.0 ** 2)
    assert_norm(get_total_norm([p.grad]), want, 2.0)
    norm = clip_grad_norm_(p, want / 4)
    assert_norm(norm, want, 2.0)
    assert_scaled(p.grad[-5:], torch.full((5,), 1024.0, device=DEV), 0.25)
    assert bool((p.grad[:-5] == p.grad[0]).all())
    assert_scaled(p.grad[:1], torch.ones(1, device=DEV), 0.25)


# ---- clipping in place ----------------------------------------------------------------
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_clip_scales_every_element_and_nothing_else(p, dtype, offset):
    bufs, grads = make(SIZES, dtype, seed=11 + offset, offset=offset)
    before = [b.clone() for b in bufs]
    want, _ = norm64(grads, p)
    norm = clip_grad_norm_(params_of(grads), want / 3, p)
    assert_norm(norm, want, p)
    for n, buf, old in zip(SIZES, bufs, before):
        assert_scaled(buf[offset:offset + n], old[offset:offset + n], (want / 3) / (want + 1e-6), n)
        assert same_bits(buf[:offset], old[:offset]) and same_bits(buf[offset + n:], old[offset + n:]), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_within_the_bound_writes_nothing(dtype):
    _, grads = make([8193, 7], dtype)
    before = [g.clone() for g in grads]
    want, _ = norm64(grads, 2.0)
    for bound in (want * 1.01, math.inf):
        assert_norm(clip_grad_norm_(params_of(grads), bound), want, 2.0)
        assert all(same_bits(g, b) for g, b in zip(grads, before))


@pytest.mark.parametrize("sizes", [
    [8192] * 32, [8192] * 32 + [1], [8192] * 31 + [8193], [1] * 32, [1] * 33, [262144], [262145], [40, 8193, 100000],
    [1 + (i * 37) % 301 for i in range(1300)],
])
@pytest.mark.parametrize("offset", [0, 5])
def test_clip_and_norms_where_the_launches_change(sizes, offset):
    """One cluster for up to 32 pieces of 16 KB, two launches up to 512 tensors, more beyond."""
    bufs, grads = make(sizes, torch.bfloat16, seed=len(sizes), offset=offset)
    before = [b.clone() for b in bufs]
    for p in (2.0, 1.0, math.inf):
        for b, old in zip(bufs, before):
            b.copy_(old)
        want, want_each = norm64(grads, p)
        total, each = get_total_norm(grads, p, per_tensor=True)
        assert_norm(total, want, p)
        for a, b in zip(each.tolist(), want_each):
            assert_norm(a, b, p)
        assert_norm(clip_grad_norm_(params_of(grads), want / 2, p), want, p)
        f = (want / 2) / (want + 1e-6)
        assert_scaled(torch.cat(grads), torch.cat([b[offset:offset + n] for b, n in zip(before, sizes)]), f)
        for buf, old, n in zip(bufs, before, sizes):
            assert torch.equal(buf[:offset], old[:offset]) and torch.equal(buf[offset + n:], old[offset + n:])


def test_clip_of_a_set_much_larger_than_the_cache():
    sizes = [300000007, 10000001, 5, 7000000]
    _, grads = make(sizes, torch.bfloat16, offset=3)
    before = [g.clone() for g in grads]
    want = math.sqrt(sum(float(torch.sum(g.double() ** 2)) for g in grads))
    assert_norm(clip_grad_norm_(params_of(grads), want / 3), want, 2.0)
    for g, b in zip(grads, before):
        assert_scaled(g, b, (want / 3) / (want + 1e-6))


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_from_the_powers_of_two_ranks(p):
    """What a sharded norm computes: each rank's power, their sum (or maximum), norm and factor
    from it."""
    _, grads = make([5001, 70001, 33, 9000], torch.bfloat16)
    want, _ = norm64(grads, p)
    parts = [K.grad_norm(K.GradTable(g), p, 0.5, want / 8) for g in (grads[:2], grads[2:])]
    powers = [n.power(p).clone() for n in parts]
    both = torch.maximum(*powers) if p == math.inf else powers[0] + powers[1]
    old = [g.clone() for g in grads]
    for n, g in zip(parts, (grads[:2], grads[2:])):
        n.power(p).copy_(both)
        K.grad_factor(n, p, 0.5, want / 8)
        assert_norm(n.norm, want / 2, p)
        K.grad_scale_(K.GradTable(g), n)
    for g, b in zip(grads, old):
        assert_scaled(g, b, 0.5 * (want / 8) / (want / 2 + 1e-6))
    none = K.grad_norm(K.GradTable([], 0), p)               # a rank that owns no gradient
    assert float(none.norm) == 0.0


def _one_rank(rank, port, out):
    import os

    import torch.distributed as dist

    from muon_sr_b200 import Sharder
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        pa, pb = _twins()
        oa = _hybrid(TritonMuonSRWithAuxAdam, pa)
        sh = Sharder(transport="nccl")
        ob = TritonMuonSRWithAuxAdam([dict(params=pb[:len(MUON)], use_muon=True, lr=0.02, weight_decay=0.01),
                                      dict(params=pb[len(MUON):], use_muon=False, lr=3e-4, eps=1e-10)],
                                     batch_ns=True, shard=sh)
        for step in range(2):
            _fill((pa, pb), 40 + step)
            oa.step(max_norm=0.25)
            sh.reduce_grads(ob)
            ob.step(max_norm=0.25)
            assert same_bits(oa.grad_norm, ob.grad_norm)
            _assert_same(pa, pb, oa, ob, ("sharded", step))
        na, nb = clip_grad_norm_(pa, 0.1), clip_grad_norm_(pb, 0.1, shard=sh)
        assert float(na) == float(nb) or abs(float(na) - float(nb)) <= NORM_TOL * float(na)
        for a, b in zip(pa, pb):
            assert_scaled(b.grad, a.grad, 1.0)
        out.put("ok")
    except BaseException as e:  # the parent reports it
        out.put(repr(e))
        raise
    finally:
        dist.destroy_process_group()


def test_sharded_clipping_on_one_rank():
    import os

    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    proc = ctx.Process(target=_one_rank, args=(0, 29900 + os.getpid() % 1000, q))
    proc.start()
    got = q.get(timeout=120)
    proc.join(timeout=60)
    assert got == "ok" and proc.exitcode == 0, got


def test_clip_mixed_types():
    grads = sum((make([70001, 9, 300], dtype, seed=k, offset=k)[1] for k, dtype in enumerate(DTYPES)), [])
    for some in (grads, grads[1::3]):                       # two launches, one launch
        before = [g.clone() for g in some]
        want, _ = norm64(some, 2.0)
        assert_norm(clip_grad_norm_(params_of(some), want / 2), want, 2.0)
        for g, b in zip(some, before):
            assert_scaled(g, b, (want / 2) / (want + 1e-6))


@pytest.mark.parametrize("std", [1e-12, 1e-16, 1e-18, 1e-22])
def test_norm_of_tiny_gradients(std):
    """Squares around the bottom of fp32's range, on both sides of where sums go to double."""
    _, grads = make([40000, 77], torch.bfloat16, std=std)
    for p in (2.0, 1.0):
        assert_norm(get_total_norm(grads, p), norm64(grads, p)[0], p)


def test_clip_scale_and_bounds():
    _, grads = make([5000, 33], torch.float32)
    before = [g.clone() for g in grads]
    want, _ = norm64(grads, 2.0)
    norm = clip_grad_norm_(params_of(grads), math.inf, grad_scale=0.25)   # a power of two: exact
    assert_norm(norm, want / 4, 2.0)
    assert all(torch.equal(g, b * 0.25) for g, b in zip(grads, before))
    norm = clip_grad_norm_(params_of(grads), 0.5, grad_scale=8.0)
    assert_norm(norm, want * 2, 2.0)
    for g, b in zip(grads, before):
        assert_scaled(g, b * 0.25, 8.0 * 0.5 / (want * 2 + 1e-6))
    clip_grad_norm_(params_of(grads), 0.0)
    assert all(float(g.abs().max()) == 0.0 for g in grads)
    assert float(clip_grad_norm_(params_of(grads), 1.0)) == 0.0           # all zero: nothing to do
    assert all(float(g.abs().max()) == 0.0 for g in grads)


def test_clip_non_finite():
    _, (a, b) = make([9000, 40], torch.bfloat16)
    keep = b.clone()
    a[17] = math.nan
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(params_of([a, b]), 1.0, error_if_nonfinite=True)
    assert same_bits(b, keep)                                             # untouched
    assert math.isnan(float(clip_grad_norm_(params_of([a, b]), 1.0)))
    assert bool(a.isnan().all()) and bool(b.isnan().all())
    _, (a, b) = make([9000, 40], torch.bfloat16)
    a[17] = -math.inf
    assert float(clip_grad_norm_(params_of([a, b]), 1.0)) == math.inf
    assert math.isnan(float(a[17])) and float(b.abs().max()) == 0.0 and float(a[18:].abs().max()) == 0.0


def test_clip_strided_gradients():
    base = torch.randn(40, 64, device=DEV).to(torch.bfloat16)
    before = base.clone()
    conv = torch.randn(4, 6, 5, 7, device=DEV).to(memory_format=torch.channels_last)
    conv_before = conv.clone()
    grads = [base[:, 2:30], base[:, 40:64].t(), conv]
    want, _ = norm64(grads, 2.0)
    params = [torch.nn.Parameter(torch.empty(g.shape, dtype=g.dtype, device=DEV)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    assert_norm(clip_grad_norm_(params, want / 2), want, 2.0)
    f = (want / 2) / (want + 1e-6)
    assert_scaled(base[:, 2:30], before[:, 2:30], f)
    assert_scaled(base[:, 40:], before[:, 40:], f)
    assert_scaled(conv, conv_before, f)
    assert same_bits(base[:, :2], before[:, :2]) and same_bits(base[:, 30:40], before[:, 30:40])


def test_clip_lists_and_refusals():
    _, (a, b) = make([300, 20], torch.bfloat16)
    old = a.clone()
    p, q = params_of([a, b])
    none = torch.nn.Parameter(torch.zeros(3, device=DEV))
    want, _ = norm64([a, b], 2.0)
    # a parameter without a gradient is passed over, one listed twice counts once
    assert_norm(clip_grad_norm_([p, none, q, p], want / 2), want, 2.0)
    assert_scaled(a, old, (want / 2) / (want + 1e-6))
    assert none.grad is None
    assert float(clip_grad_norm_([none], 1.0)) == 0.0
    other = torch.nn.Parameter(torch.empty(200, dtype=torch.bfloat16, device=DEV))
    other.grad = a[100:]
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_([p, other], 1e-9)
    e = torch.nn.Parameter(torch.empty(4, 5, device=DEV))
    e.grad = torch.ones(5, device=DEV).expand(4, 5)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_([e], 1.0)
    d = torch.nn.Parameter(torch.empty(4, dtype=torch.float64, device=DEV))
    d.grad = torch.ones(4, dtype=torch.float64, device=DEV)
    with pytest.raises(ValueError, match="float64"):
        clip_grad_norm_([p, d], 1.0)
    with pytest.raises(ValueError, match="one device|CUDA tensors"):
        get_total_norm([a, torch.ones(3, dtype=torch.bfloat16)])
    s = torch.nn.Parameter(torch.zeros(5, 3, device=DEV))
    s.grad = torch.sparse_coo_tensor([[1]], torch.ones(1, 3), (5, 3), device=DEV)
    with pytest.raises(RuntimeError, match="sparse"):
        clip_grad_norm_([s], 1.0)


def test_binding_and_tables_agree(monkeypatch):
    """Plain gradients go through the native binding, anything else through tables built in
    Python: the same bits, and the binding serves what it says and nothing else."""
    _, grads = make([70001, 9, 300, 8192], torch.bfloat16)
    params = params_of(grads)
    assert K.plain_grad_norm(grads, 2.0, 1.0, 1.0) is not None
    assert K.plain_grad_norm(grads + grads[:1], 2.0, 1.0, 1.0) is not None      # a repetition counts twice
    total2 = get_total_norm(grads + grads)
    assert_norm(total2, norm64(grads + grads, 2.0)[0], 2.0)
    other = torch.nn.Parameter(torch.empty_like(grads[0]))
    other.grad = grads[0].view(-1)[:]
    nongrad = torch.nn.Parameter(torch.zeros(2, device=DEV))
    strided = torch.zeros(6, 8, device=DEV)[:, :4]
    for refused in ([], [nongrad], params + params[:1], [params[0], other], [strided.requires_grad_() * 2], [3], [None]):
        assert K.plain_grad_clip_(refused, 2.0, 1.0, 1.0) is None
    for refused in ([], (grads[0],), [strided], [grads[0], torch.zeros(3)], [grads[0].double()], [None]):
        assert K.plain_grad_norm(refused, 2.0, 1.0, 1.0) is None
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(K, "plain_grad_norm", lambda *a, **k: None)
            monkeypatch.setattr(K, "plain_grad_clip_", lambda *a, **k: None)
        ps = params_of([g.clone() for g in grads])
        total, each = get_total_norm([p.grad for p in ps], per_tensor=True)
        opt = TritonAdamW(ps)
        opt.step(max_norm=0.5, grad_scale=2.0)
        norm = clip_grad_norm_(ps, 0.5, grad_scale=2.0)
        results.append([total, each, opt.grad_norm, norm] + [p.grad for p in ps] + [opt.state[p]["ema"] for p in ps])
    assert all(same_bits(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("native", [True, False])
def test_clip_counts_as_an_in_place_write(native, monkeypatch):
    """A graph that saved a gradient (double backward) notices that it was clipped."""
    if not native:
        monkeypatch.setattr(K, "plain_grad_clip_", lambda *a, **k: None)
    p = torch.nn.Parameter(torch.ones(40, device=DEV))
    (p ** 3).sum().backward()
    p.grad.requires_grad_()
    loss = (p.grad ** 2).sum()                               # saves p.grad
    clip_grad_norm_(p, 1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        q = torch.nn.Parameter(torch.ones(40, device=DEV))
        q.grad = torch.ones(40, device=DEV)
        assert_norm(clip_grad_norm_(q, 1.0), math.sqrt(40), 2.0)
    assert_scaled(q.grad, torch.ones(40, device=DEV), 1 / (math.sqrt(40) + 1e-6))


def test_two_calls_on_two_streams():
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [make([3000001 + k, 70], torch.bfloat16, seed=k)[1] for k in range(2)]
    before = [[g.clone() for g in s] for s in sets]
    wants = [norm64(s, 2.0)[0] for s in sets]
    torch.cuda.synchronize()
    norms = []
    for s, grads, want in zip(streams, sets, wants):
        with torch.cuda.stream(s):
            norms.append(clip_grad_norm_(params_of(grads), want / 2))
    torch.cuda.synchronize()
    for norm, want, grads, old in zip(norms, wants, sets, before):
        assert_norm(norm, want, 2.0)
        for g, b in zip(grads, old):
            assert_scaled(g, b, (want / 2) / (want + 1e-6))


def test_clip_captured_in_two_graphs():
    """Two graphs captured on one stream replay on two others at once, over new gradients."""
    sets = [make([2000003, 70], torch.bfloat16, seed=k)[1] for k in range(2)]
    clip_grad_norm_(params_of(sets[0]), math.inf)
    graphs, norms, totals = [], [], []
    for grads in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            totals.append(get_total_norm(grads, per_tensor=True))
            norms.append(clip_grad_norm_(params_of(grads), 0.5))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(3):
        wants, before = [], []
        for k, grads in enumerate(sets):
            for g, new in zip(grads, make([2000003, 70], torch.bfloat16, seed=10 + 2 * rep + k)[1]):
                g.copy_(new)
            wants.append(norm64(grads, 2.0)[0])
            before.append([g.clone() for g in grads])
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (total, each), norm, want, grads, old in zip(totals, norms, wants, sets, before):
            assert_norm(total, want, 2.0)
            for e, b in zip(each.tolist(), norm64(old, 2.0)[1]):
                assert_norm(e, b, 2.0)
            assert_norm(norm, want, 2.0)
            for g, b in zip(grads, old):
                assert_scaled(g, b, 0.5 / (want + 1e-6))


# ---- the updates that read their gradients times a factor ------------------------------
def _bf16(rng, n, std):
    return rne_bf16((rng.standard_normal(n) * std).astype(np.float32))


@pytest.fixture(params=["reference", "fast", "none"])
def noise(request):
    set_sr_noise(request.param)
    try:
        yield request.param
    finally:
        set_sr_noise("reference")


@pytest.mark.parametrize("offset", [0, 1])
def test_scaled_kernels_match_the_formulas(noise, offset):
    """Prepare and AdamW with a factor, bit for bit against the fp32 formulas on g * factor."""
    rng = np.random.default_rng(5)
    f32 = np.float32
    factor = torch.tensor([0.3712], device=DEV)
    f = f32(factor.item())

    def put(bits):
        buf = torch.zeros(offset + bits.size, dtype=torch.bfloat16, device=DEV)
        buf[offset:] = to_bf16(bits, DEV)
        return buf[offset:]
    for n in (1, 13, 4099, 2048 * 5 + 3):
        g, b, p = _bf16(rng, n, 1e-2), _bf16(rng, n, 1e-3), _bf16(rng, n, 0.02)
        v = rne_bf16(np.abs(rng.standard_normal(n) * 1e-6).astype(f32))
        gs = (bf16_to_f32(g) * f).astype(f32)
        buf, upd = put(b), put(b)
        with K.gradient_factor(factor):
            K.muon_prepare([(put(g), buf, upd, 3 * n, 4242)], 0.95, True)
        bf = bf16_to_f32(b)
        nb = (bf + f32(1.0 - 0.95) * (gs - bf)).astype(f32)
        up = (gs + f32(0.95) * (nb - gs)).astype(f32)
        assert_bits_equal(bits_of(buf), ew.sr_round(nb, triton_key(4242), 3 * n, noise), f"momentum {n}")
        assert_bits_equal(bits_of(upd), rne_bf16(up), f"update {n}")
        tp, tm, tv = put(p), put(b), put(v)
        with K.gradient_factor(factor):
            K.adamw_sr([(tp, put(g), tm, tv, 3, 77)], 3e-4, 0.9, 0.95, 1e-8, 0.01)
        b1, o1, b2, o2, ss, bc, eps, decay = ew.adamw_coefficients(3e-4, 0.9, 0.95, 1e-8, 0.01, 3)
        m1 = (b1 * bf + o1 * gs).astype(f32)
        v1 = (b2 * bf16_to_f32(v) + o2 * gs * gs).astype(f32)
        p1 = (bf16_to_f32(p) * decay).astype(f32)
        p1 = (p1 - ss * m1 / (np.sqrt(v1) / bc + eps).astype(f32)).astype(f32)
        for t, x, add in ((tm, m1, 0), (tv, v1, 1), (tp, p1, 2)):
            assert_bits_equal(bits_of(t), ew.sr_round(x, triton_key(77, add), 0, noise), f"adamw {n} {add}")


MUON = [(24, 40)] * 5 + [(40, 24)] * 3 + [(16, 16)] * 2
ADAM = [(30, 16), (16,), (4099,), (1,)]
OPTIMIZERS = {
    "adamw": lambda ps: TritonAdamW(ps, lr=1e-3, weight_decay=0.01),
    "adamw centralized": lambda ps: TritonAdamW(ps, lr=1e-3, weight_decay=0.01, centralization=0.5),
    "8-bit": lambda ps: TritonAdamW8bit(ps, lr=1e-3, weight_decay=0.01, min_8bit_size=512),
    "8-bit large block": lambda ps: TritonAdamW8bit(ps, lr=1e-3, min_8bit_size=0, block_size=4096),
    "muon": lambda ps: TritonMuonSR(ps[:len(MUON)], lr=0.02, weight_decay=0.01),
    "muon batched": lambda ps: TritonMuonSR(ps[:len(MUON)], lr=0.02, weight_decay=0.01, batch_ns=True),
    "hybrid": lambda ps: _hybrid(TritonMuonSRWithAuxAdam, ps),
    "hybrid random": lambda ps: _hybrid(MuonSRWithAuxAdam, ps),
}


def _hybrid(cls, ps):
    return cls([dict(params=ps[:len(MUON)], use_muon=True, lr=0.02, weight_decay=0.01),
                dict(params=ps[len(MUON):], use_muon=False, lr=3e-4, eps=1e-10)], batch_ns=True)


def _twins(seed=0):
    gen = torch.Generator().manual_seed(seed)
    init = [(torch.randn(s, generator=gen) * 0.02).to(torch.bfloat16) for s in MUON + ADAM]
    return [[torch.nn.Parameter(t.to(DEV)) for t in init] for _ in range(2)]


def _fill(sets, seed):
    gen = torch.Generator().manual_seed(seed)
    for ps in zip(*sets):
        g = (torch.randn(ps[0].shape, generator=gen) * 1e-2).to(torch.bfloat16).to(DEV)
        for p in ps:
            if p.grad is None:
                p.grad = torch.empty_like(p)
            p.grad.copy_(g)


def _assert_same(pa, pb, oa, ob, what):
    for i, (a, b) in enumerate(zip(pa, pb)):
        assert same_bits(a, b), (what, i)
        sa, sb = oa.state.get(a, {}), ob.state.get(b, {})
        assert sa.keys() == sb.keys(), (what, i)
        for k in sa:
            assert same_bits(sa[k], sb[k]) if torch.is_tensor(sa[k]) else sa[k] == sb[k], (what, i, k)


@pytest.mark.parametrize("name", OPTIMIZERS)
def test_step_with_an_exact_factor_equals_scaled_gradients(name, noise):
    """A factor that is a power of two scales bf16 gradients without rounding, so the step that
    scales as it reads has the bits of the step on gradients scaled before; .grad stays."""
    pa, pb = _twins()
    oa, ob = OPTIMIZERS[name](pa), OPTIMIZERS[name](pb)
    for step in range(3):
        _fill((pa, pb), 50 + step)
        keep = [p.grad.clone() for p in pb]
        for p in pa:
            p.grad.mul_(0.125)
        torch.manual_seed(step)
        oa.step()
        torch.manual_seed(step)
        ob.step(max_norm=math.inf, grad_scale=0.125)
        used = [p.grad for g in oa.param_groups for p in g["params"]]
        assert_norm(ob.grad_norm, norm64(used, 2.0)[0], 2.0)
        _assert_same(pa, pb, oa, ob, (name, step))
        assert all(same_bits(p.grad, k) for p, k in zip(pb, keep))
    ob.step()
    assert ob.grad_norm is None


def test_step_clips_by_the_norm_of_all_groups():
    """AdamW's first moment after one step from zero is (1 - beta1) * g * factor, the factor of
    the norm over every group, rounded to nearest (no noise) once."""
    set_sr_noise("none")
    try:
        pa, _ = _twins()
        _fill((pa,), 3)
        opt = TritonAdamW([dict(params=pa[:4]), dict(params=pa[4:])], lr=1e-3)
        want = norm64([p.grad for p in pa], 2.0)[0]
        opt.step(max_norm=want / 5)
        assert_norm(opt.grad_norm, want, 2.0)
        for p in pa:
            # the product by the factor, 1 - beta1 itself and the product by it
            assert_scaled(opt.state[p]["ema"], p.grad, (1 - 0.9) * (want / 5) / (want + 1e-6), products=3)
    finally:
        set_sr_noise("reference")


def test_step_clips_the_gradients_of_its_closure():
    p = torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16, device=DEV))
    opt = TritonAdamW([p])

    def closure():
        opt.zero_grad()
        loss = (p.float() * 0.25).sum()
        loss.backward()
        return loss
    assert float(opt.step(closure, max_norm=1.0)) == 75.0
    assert_norm(opt.grad_norm, 0.25 * math.sqrt(300), 2.0)


def test_step_missing_gradients_and_refusals():
    pa, pb = _twins()
    _fill((pa, pb), 1)
    for ps in (pa, pb):
        ps[3].grad = None
    oa, ob = OPTIMIZERS["hybrid"](pa), OPTIMIZERS["hybrid"](pb)
    for p in pa:
        if p.grad is not None:
            p.grad.mul_(0.5)
    oa.step()
    ob.step(max_norm=math.inf, grad_scale=0.5)
    _assert_same(pa, pb, oa, ob, "missing gradient")
    with pytest.raises(ValueError, match="grad_scale needs max_norm"):
        ob.step(grad_scale=0.5)
    for bad in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, grad_scale=0.0),
                dict(max_norm=1.0, grad_scale=math.inf)):
        with pytest.raises(ValueError):
            ob.step(**bad)
    opt = TritonAdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16, device=DEV))])
    opt.step(max_norm=1.0)                                   # no gradient at all
    assert opt.grad_norm is None


@pytest.mark.parametrize("name", ["adamw", "adamw centralized", "muon batched", "hybrid", "hybrid random"])
def test_graph_of_clipped_steps_matches_eager(name):
    pa, pb = _twins()
    oa, ob = OPTIMIZERS[name](pa), OPTIMIZERS[name](pb)
    clip = dict(max_norm=0.25, grad_scale=0.5)
    _fill((pa, pb), 30)
    for o in (oa, ob):
        torch.manual_seed(9)
        o.step(**clip)
    eager = ob.grad_norm
    graph = StepGraph(ob, **clip)
    assert ob.grad_norm is eager                             # capturing does not step
    for step in range(4):
        _fill((pa, pb), 60 + step)
        for o in (oa, ob):                                   # a new learning rate is picked up
            for g in o.param_groups:
                g["lr"] *= 0.9
        torch.manual_seed(step)
        oa.step(**clip)
        torch.manual_seed(step)
        graph.step()
        assert same_bits(oa.grad_norm, ob.grad_norm)
        _assert_same(pa, pb, oa, ob, (name, step))


@pytest.mark.parametrize("name", ["adamw", "8-bit", "hybrid"])
def test_staged_clipped_steps_match_eager(name):
    pa, pb = _twins()
    oa, ob = OPTIMIZERS[name](pa), OPTIMIZERS[name](pb)
    _fill((pa,), 0)
    host = [torch.empty(p.shape, dtype=torch.bfloat16).pin_memory() for p in pb]
    out = [torch.empty(p.shape, dtype=torch.bfloat16).pin_memory() for p in pb]
    staged = HostStaging(ob, pb, host, out)
    for step in range(3):
        _fill((pa,), 70 + step)
        torch.cuda.synchronize()
        for h, p in zip(host, pa):
            h.copy_(p.grad)
        oa.step(max_norm=0.25)
        staged.step(max_norm=0.25)
        staged.synchronize()
        assert same_bits(oa.grad_norm, ob.grad_norm)
        _assert_same(pa, pb, oa, ob, (name, step))
        assert all(same_bits(p.cpu(), h) for p, h in zip(pb, out))


def test_norm_clip_and_step_in_a_row():
    """Micro-batches accumulated with SR, clipped in place, stepped -- against the step that
    clips as it reads, in round-to-nearest: the two differ by the in-place clip's rounding of each
    gradient to bf16, so the first moments (linear in it, from zero) differ by at most that
    (half a bf16 step, 2^-8 of the value) and one such rounding of each moment."""
    set_sr_noise("none")
    try:
        pa, pb = _twins()
        oa, ob = OPTIMIZERS["adamw"](pa), OPTIMIZERS["adamw"](pb)
        acc = [[torch.empty_like(p) for p in ps] for ps in (pa, pb)]
        for micro in range(2):
            _fill((pa, pb), 90 + micro)
            for ps, bufs in zip((pa, pb), acc):
                for p, b in zip(ps, bufs):
                    K.grad_accum_(b, p.grad, 5, first=micro == 0)
        for ps, bufs in zip((pa, pb), acc):
            for p, b in zip(ps, bufs):
                p.grad = b
        before = get_total_norm([p.grad for p in pa])
        bound = float(before) / 3
        norm = clip_grad_norm_(pa, bound, grad_scale=0.5)
        oa.step()
        ob.step(max_norm=bound, grad_scale=0.5)
        assert same_bits(norm, ob.grad_norm)
        assert_norm(norm, float(before) / 2, 2.0)
        after = float(get_total_norm([p.grad for p in pa]))
        assert abs(after - bound) <= 2.0 ** -8 * bound
        for a, b in zip(pa, pb):
            ma, mb = oa.state[a]["ema"].double(), ob.state[b]["ema"].double()
            assert bool(((ma - mb).abs() <= 3 * 2.0 ** -8 * mb.abs() * (1 + 2.0 ** -7) + 2.0 ** -132).all())
    finally:
        set_sr_noise("reference")
