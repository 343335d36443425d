"""Global gradient norm and clipping on the B200 engine, between the backward pass and the step.

* ``get_total_norm(tensors)`` -- the norm of many gradients taken as one vector.
* ``clip_grad_norm_(parameters, max_norm)`` -- scales ``.grad`` in place so that this norm is at
  most ``max_norm``.
* ``optimizer.step(max_norm=...)``, for every optimizer of this package -- the same clipping
  without the pass that rewrites the gradients: the update kernels multiply each gradient as
  they read it. The product is used in fp32, so the result has one bf16 rounding fewer than
  ``clip_grad_norm_`` followed by ``step()``; ``.grad`` keeps the unclipped values, and
  ``optimizer.grad_norm`` holds the norm.

The first two take the arguments of their namesakes in ``torch.nn.utils``. Sums are kept in
double and norms returned in fp32, whatever the gradients' type, on the device: nothing here
waits for the GPU unless ``error_if_nonfinite`` asks for it. A step by a NaN norm -- one NaN in
any gradient -- leaves weights, momenta and moments as they were and only advances the step
counters; by an infinite norm it does what gradients scaled by 0 would (NaN where they were
infinite). ``grad_norm`` tells.
"""
import contextlib
import math
import operator

import numpy as np
import torch

from . import kernels as K
from . import staging


_FP32 = torch.finfo(torch.float32)


def _norm_type(value):
    value = float(value)
    if value not in K.NORM_TYPES:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {value}")
    return value


def _bounds(max_norm, grad_scale):
    max_norm, grad_scale = float(max_norm), float(grad_scale)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if not _FP32.tiny <= grad_scale <= _FP32.max:
        raise ValueError(f"grad_scale must be positive and within the range of fp32, got {grad_scale}")
    return max_norm, grad_scale


def _refuse_nonfinite(norm, norm_type):
    if not math.isfinite(float(norm)):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients is non-finite, so it cannot be "
                           "clipped. Pass error_if_nonfinite=False to clip with the non-finite norm anyway.")


def get_total_norm(tensors, norm_type=2.0, error_if_nonfinite=False, foreach=None, *, per_tensor=False):
    """The norm of ``tensors`` (bf16, fp16 or fp32 CUDA tensors on one device, mixed at will) as
    one vector: a 0-dim fp32 tensor on their device, 0 for an empty list.

    ``norm_type`` is 1, 2 or inf. With ``per_tensor`` the result is ``(total, norms)``, the
    second the fp32 norm of every tensor, from the same pass. ``error_if_nonfinite`` waits for
    the result and raises ``RuntimeError`` where it is infinite or NaN. ``foreach`` is torch's, whose
    implementations it chooses between: there is one here."""
    norm_type = _norm_type(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        total = torch.zeros(())
        return (total, torch.zeros(0)) if per_tensor else total
    plain = K.plain_grad_norm(tensors, norm_type, 1.0, math.inf, per_tensor)
    if plain is not None:
        _, total, each = plain
    else:
        norm = K.grad_norm(K.GradTable(tensors), norm_type, per_tensor=per_tensor)
        total, each = norm.norm, norm.each
    if error_if_nonfinite:
        _refuse_nonfinite(total, norm_type)
    return (total, each) if per_tensor else total


def _norm_over_ranks(table, norm_type, grad_scale, max_norm, shard):
    """The ``GradNorm`` of a table's gradients -- with a sharder, of every rank's together."""
    norm = K.grad_norm(table, norm_type, grad_scale, max_norm)
    if shard is not None and shard.world > 1:
        shard.combine_power(norm.power(norm_type))
        K.grad_factor(norm, norm_type, grad_scale, max_norm)
    return norm


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None, *, grad_scale=1.0,
                    shard=None):
    """Multiply the gradients of ``parameters`` in place by
    ``grad_scale * min(1, max_norm / (norm + 1e-6))``, ``norm`` being the norm of all of them
    together times ``grad_scale``; returns ``norm`` (0-dim fp32, on their device).

    Arguments:
        parameters: a parameter or an iterable of them; those without a gradient are passed
            over, one that is listed twice counts once
        max_norm (float): the bound; ``math.inf`` clips nothing, whatever the norm (torch's
            function makes every gradient NaN where the norm is not finite)
        norm_type (float): 1, 2 or inf
        error_if_nonfinite (bool): wait for the norm and raise ``RuntimeError``, the gradients
            untouched, where it is infinite or NaN. Otherwise, ``max_norm`` being finite, a NaN
            norm makes every gradient NaN and an infinite gradient makes them 0 (NaN where they
            were infinite). Stochastic rounding carries a NaN over to -0, so a step on such
            gradients leaves no NaN in the weights to notice it by
        foreach: torch's choice of its implementation; there is one here
        grad_scale (float): multiplies every gradient in any case, e.g. 1 / micro-batches
        shard: the ``Sharder`` whose ``reduce_grads`` has brought each gradient to its owner.
            Collective: the norm is over all ranks' gradients, each rank scales those it owns

    Gradients whose norm is within the bound are not written (``grad_scale`` 1). Two parameters
    whose gradients share memory are refused. The factor is an fp32 number: it loses bits below
    2^-126, where ``max_norm`` is that far below the norm."""
    norm_type = _norm_type(norm_type)
    max_norm, grad_scale = _bounds(max_norm, grad_scale)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    whole = shard is None and not error_if_nonfinite
    if whole and not staging.active() and \
            (norm := K.plain_grad_clip_(parameters, norm_type, grad_scale, max_norm)) is not None:
        return norm
    table = _gradients(parameters, shard)
    if table is None:
        return torch.zeros(())
    if table.dense is not table.grads:
        _refuse_shared(table)
    if whole:
        return K.grad_clip_(table, norm_type, grad_scale, max_norm).norm
    norm = _norm_over_ranks(table, norm_type, grad_scale, max_norm, shard)
    if error_if_nonfinite:
        _refuse_nonfinite(norm.norm, norm_type)
    K.grad_scale_(table, norm)
    return norm.norm


class _Place:
    """The elements of a CUDA tensor as an array interface: numpy solves for common elements from
    address, shape and strides alone."""

    def __init__(self, t):
        size = t.element_size()
        self.__array_interface__ = dict(version=3, typestr=f"|V{size}", shape=tuple(t.shape),
                                        strides=tuple(st * size for st in t.stride()), data=(t.data_ptr(), True))


_SHARES_WORK = 1_000_000  # steps of numpy's search, far above what views of matrices take


def _refuse_shared(table):
    """Raise where a gradient that goes through a copy is expanded or shares elements with
    another: the copies lie apart, so the check of the scaling itself would not see it."""
    if any(st == 0 and n > 1 for g in table.grads for st, n in zip(g.stride(), g.shape)):
        raise ValueError("gradients must not be expanded tensors: their elements share memory")
    spans = []
    for g, d in zip(table.grads, table.dense):
        if g.numel():
            last = sum(st * (n - 1) for st, n in zip(g.stride(), g.shape))
            spans.append((g.data_ptr(), g.data_ptr() + (last + 1) * g.element_size(), g is d, np.asarray(_Place(g))))
    spans.sort(key=operator.itemgetter(0))
    reach = []  # those before that end behind the present one's start
    for span in spans:
        reach = [s for s in reach if s[1] > span[0]]
        for other in reach:
            if not (span[2] and other[2]):  # (two dense ones are checked with their launch)
                try:
                    shared = np.shares_memory(span[3], other[3], max_work=_SHARES_WORK)
                except np.exceptions.TooHardError:
                    shared = True
                if shared:
                    raise RuntimeError("two gradients overlap in memory")
        reach.append(span)


def _gradients(parameters, shard):
    """The ``GradTable`` of the parameters that have a gradient, each once (with a sharder: those
    of them that this rank owns), or None where there is nothing to launch."""
    grads = [g for p in parameters if (g := p.grad) is not None]
    if shard is not None or staging.active() or len(set(map(id, grads))) < len(grads):
        params = list({id(p): p for p in parameters if p.grad is not None}.values())
        if shard is not None:
            params = shard.owned(params)
        staging.need(params)
        grads = [p.grad for p in params]
    if not grads and shard is None:
        return None
    return K.GradTable(grads, None if grads else _device_of(parameters))


def _device_of(parameters):
    """The device on which a rank that owns none of the gradients joins the others' sum."""
    first = min(parameters, key=lambda p: p.grad is None, default=None)
    return torch.cuda.current_device() if first is None else first.get_device()


def clipped_step(optimizer, max_norm, grad_scale):
    """The context in which an optimizer's ``step`` issues its launches: with ``max_norm``, the
    norm of all its gradients is launched here and the step's kernels read every gradient times
    the factor; ``optimizer.grad_norm`` is that norm, or None without ``max_norm``."""
    optimizer.grad_norm = None
    if max_norm is None:
        if grad_scale != 1.0:
            raise ValueError("grad_scale needs max_norm (math.inf clips nothing)")
        return contextlib.nullcontext()
    max_norm, grad_scale = _bounds(max_norm, grad_scale)
    shard = getattr(optimizer, "_shard", None)
    if shard is not None:
        shard._ensure(optimizer)
    params = [p for g in optimizer.param_groups for p in g["params"]]
    plain = None
    if shard is None and not staging.active():
        plain = K.plain_grad_norm(params, 2.0, grad_scale, max_norm, of_grads=True)
    if plain is not None:
        norm = K.GradNorm(None, state=plain[0])
    else:
        table = _gradients(params, shard)
        if table is None:
            return contextlib.nullcontext()
        norm = _norm_over_ranks(table, 2.0, grad_scale, max_norm, shard)
    optimizer.grad_norm = norm.norm
    return K.gradient_factor(norm.factor)
