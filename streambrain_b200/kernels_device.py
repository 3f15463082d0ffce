"""Operators on unit codes, on CUDA tensors.

A *code* is the position of one active unit: unit ``i`` of hypercolumn ``h`` of a layer is ``h * minicolumns + i``.  A
sample of a few codes stands for an input row with ones there and zeros elsewhere -- a hidden layer made binary by
:func:`sample_minicolumns`, a complementary-coded binary image, a sequence of tokens.  :func:`lookup` is what
``update_state`` of :mod:`streambrain_b200.kernels_b200` computes from such a row (without the bias),
:func:`lookup_gradient` its gradient, :func:`distill_loss` and :func:`distill_gradient` train a student's hypercolumns on
the kept units of a teacher's.

Tensors live on one CUDA device and the work is queued on torch's current stream there; the calls return without
synchronising, can be captured into a graph and give the same bits for the same inputs.  Supports, weights and gradients
are float32, float64, float16 or bfloat16 (sums are held in 32 bits, for float64 in 64, and rounded once), codes int32 or
int64.  Inputs that are not contiguous are copied.  A wrong dtype, shape or device raises ``TypeError`` or ``ValueError``.
Nothing here records for autograd: the gradients are calls of their own.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from ._lib import Sampling, check, lib

__all__ = ["lookup", "lookup_gradient", "sample_minicolumns", "distill_loss", "distill_gradient"]

_DTYPES = {torch.float32: _lib.F32, torch.float64: _lib.F64, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _dense(t, name, dim, dtypes, device=None):
    """``t`` as a contiguous CUDA tensor of one of ``dtypes``, on ``device`` (a number)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype not in dtypes:
        raise TypeError("%s has dtype %s, expected %s" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    if t.dim() != dim:
        raise ValueError("%s must have %d dimensions, got shape %s" % (name, dim, tuple(t.shape)))
    if device is not None and t.get_device() != device:
        raise ValueError("%s is on cuda:%d, not on cuda:%d" % (name, t.get_device(), device))
    return t if t.is_contiguous() else t.contiguous()


def _call(entry, device, *arguments):
    """``entry(*arguments, stream)`` on torch's current stream of ``device``, with that device current."""
    if _raw_stream is None or _current_device is None:
        with torch.cuda.device(device):
            rc = entry(*arguments, torch.cuda.current_stream(device).cuda_stream)
    elif _current_device() == device:
        rc = entry(*arguments, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = entry(*arguments, _raw_stream(device))
    if rc:
        check(rc)


def _wide(dtype):
    return torch.float64 if dtype is torch.float64 else torch.float32


def lookup(weights, codes, scale=1.0):
    """``out[r] = scale * sum_l weights[codes[r, l]]``: ``weights`` [N, M], ``codes`` [rows, L], result [rows, M] of the
    weights' dtype.  With L = 1 an embedding lookup.  Codes outside ``0 .. N - 1`` (-1 by convention) name nothing; a row
    of such codes, or with L = 0, gives zeros."""
    weights = _dense(weights, "weights", 2, _DTYPES)
    device = weights.get_device()
    codes = _dense(codes, "codes", 2, _INDEX_BYTES, device)
    rows, length = codes.shape
    n, m = weights.shape
    out = weights.new_empty((rows, m))
    _call(lib.sbb_lookup, device, _DTYPES[weights.dtype], weights.data_ptr(), codes.data_ptr(), _INDEX_BYTES[codes.dtype], rows,
          length, n, m, scale, out.data_ptr())
    return out


@lru_cache(maxsize=256)
def _gradient_workspace(code, rows, length, n, m):
    return lib.sbb_lookup_gradient_workspace(code, rows, length, n, m)


def lookup_gradient(grad, codes, in_features, scale=1.0, out=None, accumulate=False):
    """The gradient of :func:`lookup` with respect to its weights: ``out[i] = scale *`` the sum of ``grad[r]`` over the
    ``(r, l)`` with ``codes[r, l] == i``; ``grad`` [rows, M], result [in_features, M] of its dtype, rows that no code names
    zero.  ``out`` (contiguous) receives it; with ``accumulate=True`` the sums are added to what it holds, and rows that no
    code names are left alone."""
    grad = _dense(grad, "grad", 2, _DTYPES)
    device = grad.get_device()
    codes = _dense(codes, "codes", 2, _INDEX_BYTES, device)
    rows, length = codes.shape
    n, m = int(in_features), grad.shape[1]
    if grad.shape[0] != rows:
        raise ValueError("grad has %d rows, codes %d" % (grad.shape[0], rows))
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs the tensor to add to as out")
        if n <= 0:
            raise ValueError("in_features must be above 0")
        out = grad.new_empty((n, m))
    else:
        if _dense(out, "out", 2, (grad.dtype,), device) is not out:
            raise ValueError("out must be contiguous")
        if out.shape != (n, m):
            raise ValueError("out must have shape %s, got %s" % ((n, m), tuple(out.shape)))
    code = _DTYPES[grad.dtype]
    size = _gradient_workspace(code, rows, length, n, m)
    work = grad.new_empty(size, dtype=torch.uint8) if size else None
    _call(lib.sbb_lookup_gradient, device, code, grad.data_ptr(), codes.data_ptr(), _INDEX_BYTES[codes.dtype], rows, length, n, m,
          scale, 1 if accumulate else 0, out.data_ptr(), None if work is None else work.data_ptr(), size)
    return out


def _setting(value, name, rows, dtype, device):
    """A sampling setting: (number, tensor of a value per row or None)."""
    if isinstance(value, torch.Tensor):
        t = _dense(value, name, 1, (dtype,), device)
        if t.shape[0] != rows:
            raise ValueError("%s must be a number or have %d values, got %d" % (name, rows, t.shape[0]))
        return None, t
    return value, None


def sample_minicolumns(support, hypercolumns, minicolumns, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draws one unit of every hypercolumn from the softmax of its support and returns the codes [rows, hypercolumns]
    (int64): ``h * minicolumns + unit``, or -1 where every unit of the hypercolumn is at -infinity.

    ``support`` [rows, hypercolumns * minicolumns]; ``random`` float32 [rows, hypercolumns] in [0, 1).  With
    ``w_i = exp((x_i - max) / temperature)`` and units in order of falling ``w`` (equal ones by index), the first ``top_k``
    are kept (all with 0), of these the shortest beginning whose sum reaches ``top_p`` times their sum (at least one), of
    these the ones with ``w_i >= min_p`` (at least the largest); the unit drawn is the first in index order at which the
    running sum of the kept ``w`` passes ``random`` times their sum (with ``random`` 0 the first kept unit whose ``w`` is above 0
    in 64 bits, however small).  ``temperature`` 0 takes the largest, the first of
    equal ones.  NaN counts as -infinity.  Each setting is a number (rounded to float32) or a CUDA tensor with a value per row
    (``top_k`` int32, the others float32; values out of range act as the nearest in range)."""
    support = _dense(support, "support", 2, _DTYPES)
    device = support.get_device()
    h, mc = int(hypercolumns), int(minicolumns)
    rows, columns = support.shape
    if columns != h * mc:
        raise ValueError("support has %d columns, expected %d hypercolumns of %d units" % (columns, h, mc))
    random = _dense(random, "random", 2, (torch.float32,), device)
    if random.shape != (rows, h):
        raise ValueError("random must have shape %s, got %s" % ((rows, h), tuple(random.shape)))
    t, t_rows = _setting(temperature, "temperature", rows, torch.float32, device)
    k, k_rows = _setting(top_k, "top_k", rows, torch.int32, device)
    p, p_rows = _setting(top_p, "top_p", rows, torch.float32, device)
    low, low_rows = _setting(min_p, "min_p", rows, torch.float32, device)
    how = Sampling(1.0 if t is None else t, 1.0 if p is None else p, 0.0 if low is None else low, 0 if k is None else int(k),
                   *[None if a is None else a.data_ptr() for a in (t_rows, p_rows, low_rows, k_rows)])
    codes = support.new_empty((rows, h), dtype=torch.int64)
    _call(lib.sbb_sample_minicolumns, device, _DTYPES[support.dtype], support.data_ptr(), random.data_ptr(), rows, h, mc,
          ctypes.byref(how), codes.data_ptr())
    return codes


def _distill(support, hypercolumns, minicolumns, teacher_units, teacher_support, temperature, weight, want_gradient):
    support = _dense(support, "support", 2, _DTYPES)
    device = support.get_device()
    h, mc = int(hypercolumns), int(minicolumns)
    rows, columns = support.shape
    if columns != h * mc:
        raise ValueError("support has %d columns, expected %d hypercolumns of %d units" % (columns, h, mc))
    units = _dense(teacher_units, "teacher_units", 3, _INDEX_BYTES, device)
    teacher = _dense(teacher_support, "teacher_support", 3, (support.dtype,), device)
    if units.shape != teacher.shape or units.shape[:2] != (rows, h):
        raise ValueError("teacher_units and teacher_support must both be [%d, %d, k], got %s and %s" % (
            rows, h, tuple(units.shape), tuple(teacher.shape)))
    wide = _wide(support.dtype)
    if weight is not None:
        weight = _dense(weight, "weight", 1, (wide,), device)
        if weight.shape[0] != rows:
            raise ValueError("weight has %d values for %d rows" % (weight.shape[0], rows))
    loss = support.new_empty((rows, h), dtype=wide)
    gradient = support.new_empty((rows, columns)) if want_gradient else None
    _call(lib.sbb_distill, device, _DTYPES[support.dtype], support.data_ptr(), units.data_ptr(), _INDEX_BYTES[units.dtype],
          teacher.data_ptr(), None if weight is None else weight.data_ptr(), rows, h, mc, units.shape[2], temperature,
          loss.data_ptr(), None if gradient is None else gradient.data_ptr())
    return loss, gradient


def distill_loss(support, hypercolumns, minicolumns, teacher_units, teacher_support, temperature=1.0, weight=None):
    """How far a student's hypercolumns are from a teacher's of which the best units are kept; [rows, hypercolumns] in
    float32 (float64 for float64).

    ``support`` [rows, hypercolumns * minicolumns] is the student's; ``teacher_units`` [rows, hypercolumns, k] the units the
    teacher keeps, counted within the hypercolumn (entries out of range are absent, a unit named twice has both parts), and
    ``teacher_support`` their support, of the student's dtype.  With ``p`` the softmax of the kept units and ``q`` that of all
    of the student's, both at ``temperature``: ``loss = weight * temperature**2 * sum_k p_k (log p_k - log q_{unit_k})``.
    ``weight`` [rows] (float32, float64 for float64; default 1).  ``temperature`` is from 1e-15 to 1e15.  In 32 bits an exponential
    ``e**-x`` is off by ``2**-22 + 3 * x * 2**-24`` of itself.  The loss is exactly 0 where the weight is, where nothing is
    kept, and where a hypercolumn of the student or of the teacher is at -infinity throughout; elsewhere NaN where the hypercolumn of
    either holds a NaN or +infinity."""
    return _distill(support, hypercolumns, minicolumns, teacher_units, teacher_support, temperature, weight, False)[0]


def distill_gradient(support, hypercolumns, minicolumns, teacher_units, teacher_support, temperature=1.0, weight=None):
    """:func:`distill_loss` and its gradient with respect to ``support``, of the support's shape and dtype:
    ``weight * temperature * (q_i - sum over the k with unit_k == i of p_k)``, exactly 0 where the loss is for one of the
    reasons named there.  Returns ``(loss, gradient)``; the student's support is read once."""
    return _distill(support, hypercolumns, minicolumns, teacher_units, teacher_support, temperature, weight, True)
