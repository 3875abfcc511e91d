"""Classification losses with a fused forward+backward GPU kernel (``csrc/train_kernels.cu``).

``sigmoid_xent`` sums the binary cross-entropy over classes, ``softmax_xent`` is the softmax
cross-entropy with soft labels; both return one value per example (reference:
``vmoe/train/trainer.py:441-477``).

Distillation (``csrc/distill_kernels.cu``): ``top_logits`` reduces a teacher's logits to its ``k``
largest and one number for all the others, ``distill_xent`` is the divergence of a student from
such a teacher. The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from vmoe_b200.ops import _lib
from vmoe_b200.ops import functional

_vp = ctypes.c_void_p
_LABEL_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.uint8: 2, torch.bool: 2}


class _XentFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, labels, kind):
    n = logits.shape[-1]
    lg = logits.reshape(-1, n)
    lb = labels.reshape(-1, n)
    assert lg.stride(-1) == 1 and lb.stride(-1) == 1
    rows, ld = lg.shape[0], lg.stride(0)
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    need = ctx.needs_input_grad[0]
    # The gradient keeps the (possibly padded) row stride of the logits; padding gets zeros.
    dfull = torch.empty(rows, ld, dtype=torch.bfloat16, device=logits.device) if need else None
    rc = _lib.lib().vmoe_xent(
        ctypes.c_int32(kind), _vp(lg.data_ptr()), _vp(lb.data_ptr()),
        ctypes.c_int32(_LABEL_CODES[lb.dtype]), _vp(loss.data_ptr()), _vp(_lib.ptr(dfull)),
        ctypes.c_int64(rows), ctypes.c_int64(n), ctypes.c_int64(ld),
        ctypes.c_int64(lb.stride(0)), ctypes.c_float(1.0), _vp(_lib.stream_ptr()))
    _lib.check(rc, "vmoe_xent")
    _lib.count_launch()
    ctx.save_for_backward(dfull)
    ctx.shape = logits.shape
    return loss.reshape(logits.shape[:-1])

  @staticmethod
  def backward(ctx, dloss):
    (dfull,) = ctx.saved_tensors
    n = ctx.shape[-1]
    g = dfull * dloss.reshape(-1, 1).to(dfull.dtype)
    return g[:, :n], None, None


def _fast(logits, labels) -> bool:
  return (functional.cuda_kernels_enabled() and logits.is_cuda and
          logits.dtype == torch.bfloat16 and labels.dtype in _LABEL_CODES and
          logits.dim() == 2 and logits.stride(-1) == 1 and labels.shape == logits.shape)


def sigmoid_xent(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
  if _fast(logits, labels):
    return _XentFn.apply(logits, labels.contiguous(), 0)
  x = logits.float()
  return F.binary_cross_entropy_with_logits(x, labels.float(), reduction="none").sum(-1)


def softmax_xent(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
  if _fast(logits, labels):
    return _XentFn.apply(logits, labels.contiguous(), 1)
  return -(labels.float() * F.log_softmax(logits.float(), dim=-1)).sum(-1)


# ------------------------------------------------------------------------------- distillation
_FLOAT_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
TOP_LOGITS_MAX = 256


class TopLogits(NamedTuple):
  """A teacher's answer: its largest logits and their classes, largest first, and the
  log-sum-exp of ``logits / temperature`` over all the other classes."""
  values: torch.Tensor   # (rows, k), the logits' type
  indices: torch.Tensor  # (rows, k) int32
  rest: torch.Tensor     # (rows,) fp32


def _check_logits(logits, temperature, what: str) -> float:
  if logits.dim() != 2:
    raise ValueError(f"{what}: logits must be (rows, classes), got shape {tuple(logits.shape)}")
  if not logits.is_floating_point():
    raise TypeError(f"{what}: logits must be floating point, got {logits.dtype}")
  if logits.shape[1] < 1:
    raise ValueError(f"{what}: there must be at least one class")
  temperature = float(temperature)
  if not 1e-3 <= temperature <= 1e3:
    raise ValueError(f"{what}: temperature must be in [1e-3, 1e3], got {temperature}")
  return temperature


_MAX_CLASSES: dict = {}


def _on_kernels(logits, what: str) -> bool:
  """Whether the kernels take these logits (type, device, classes that fit shared memory)."""
  if not (functional.cuda_kernels_enabled() and logits.is_cuda):
    return False
  code = _FLOAT_CODES.get(logits.dtype)
  if code is None:
    return False
  most = _MAX_CLASSES.get((what, code))
  if most is None:
    most = getattr(_lib.lib(), f"vmoe_{what}_max_classes")(code)
    _MAX_CLASSES[what, code] = most
  return logits.shape[1] <= most


def _rows(t: torch.Tensor) -> torch.Tensor:
  """``t`` with contiguous rows (any distance between them)."""
  return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _ld(t: torch.Tensor) -> int:
  return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def top_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0) -> TopLogits:
  """The ``k`` largest of every row of ``logits (rows, classes)``, ``1 <= k <= min(classes, 256)``.

  Sorted in descending order; equal logits go to the lower class first, NaN counts as larger than
  +inf. ``rest`` is ``logsumexp(logits / temperature)`` over the classes that are not among them,
  ``-inf`` when there are none. No gradient: this is the frozen side of ``distill_xent``.
  """
  temperature = _check_logits(logits, temperature, "top_logits")
  rows, n = logits.shape
  if not 1 <= k <= min(n, TOP_LOGITS_MAX):
    raise ValueError(f"top_logits: k must be in 1 .. {min(n, TOP_LOGITS_MAX)}, got {k}")
  if _on_kernels(logits, "top_logits"):
    with _lib.on_device(logits):
      x = _rows(logits)
      dev = x.device
      values = torch.empty((rows, k), dtype=x.dtype, device=dev)
      indices = torch.empty((rows, k), dtype=torch.int32, device=dev)
      rest = torch.empty(rows, dtype=torch.float32, device=dev)
      rc = _lib.lib().vmoe_top_logits(
          x.data_ptr(), _FLOAT_CODES[x.dtype], rows, n, _ld(x), k, temperature, values.data_ptr(),
          indices.data_ptr(), rest.data_ptr(), _lib.stream_ptr())
      _lib.check(rc, "vmoe_top_logits")
      _lib.count_launch()
    return TopLogits(values, indices, rest)
  logits = logits.detach()
  x = logits.float()
  order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
  others = (x / temperature).scatter(1, order, -math.inf)
  return TopLogits(logits.gather(1, order), order.to(torch.int32), torch.logsumexp(others, dim=1))


class _DistillFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, values, indices, rest, temperature):
    with _lib.on_device(logits):
      rows, n = logits.shape
      x = _rows(logits)
      k = values.shape[1]
      dev = x.device
      loss = torch.empty(rows, dtype=torch.float32, device=dev)
      lib, code = _lib.lib(), _FLOAT_CODES[x.dtype]
      kept = torch.empty(lib.vmoe_distill_kept_floats(rows, n, k, code), dtype=torch.float32,
                         device=dev)
      a = _lib.DistillArgs(x.data_ptr(), values.data_ptr(), indices.data_ptr(), _lib.ptr(rest),
                           loss.data_ptr(), kept.data_ptr(), rows, n, k, _ld(x), _ld(values),
                           _ld(indices), temperature, code, _FLOAT_CODES[values.dtype],
                           indices.dtype == torch.int64)
      _lib.check(lib.vmoe_distill_fwd(ctypes.byref(a), _lib.stream_ptr()), "vmoe_distill_fwd")
      _lib.count_launch(2)
    ctx.save_for_backward(x, indices, kept)
    ctx.args = a
    return loss

  @staticmethod
  @functional.first_order
  def backward(ctx, dloss):
    x, _, _ = ctx.saved_tensors
    a = ctx.args
    rows, n, dtype = a.rows, a.n, x.dtype
    with _lib.on_device(x):
      # Gradient rows keep the logits' place within 16 bytes, so that both sides move in the same
      # vectors; the padding of padded rows (a classification head whose width is not a multiple
      # of 8) is zeroed.
      size = 4 if dtype == torch.float32 else 2
      ld = n + (a.ld - n) % (16 // size)
      phase = a.logits % 16 // size if rows else 0
      if phase:
        grad = torch.empty(phase + rows * ld, dtype=dtype, device=x.device)[phase:].view(rows, ld)
      else:
        grad = torch.empty((rows, ld), dtype=dtype, device=x.device)
      if dloss.dtype != torch.float32:
        dloss = dloss.float()
      rc = _lib.lib().vmoe_distill_bwd(ctypes.byref(a), dloss.data_ptr(), dloss.stride(0),
                                       grad.data_ptr(), ld, ld, _lib.stream_ptr())
      _lib.check(rc, "vmoe_distill_bwd")
      _lib.count_launch()
    return grad if ld == n else grad[:, :n], None, None, None, None


def _distill_reference(logits, values, indices, rest, temperature):
  """The same loss in PyTorch ops (differentiable in the logits), in 64 bits: its first-order
  parts cancel where student and teacher agree."""
  rows, n = logits.shape
  at = indices.long()
  valid = (at >= 0) & (at < n)
  at = torch.where(valid, at, torch.zeros_like(at))
  # Of a class that is listed twice the first entry counts.
  same = (at[:, :, None] == at[:, None, :]) & valid[:, None, :]
  valid = valid & ~same.tril(-1).any(-1)
  log_q = torch.log_softmax(logits.double() / temperature, dim=1)
  kept = torch.zeros(rows, n, dtype=torch.int32, device=logits.device)
  kept = kept.scatter_add(1, at, valid.int()) > 0
  t = (values.double() / temperature).masked_fill(~valid, -math.inf)
  log_q_kept = log_q.gather(1, at)
  if rest is not None:
    t = torch.cat([t, rest.double()[:, None]], dim=1)
    q_rest = torch.logsumexp(log_q.masked_fill(kept, -math.inf), dim=1, keepdim=True)
    log_q_kept = torch.cat([log_q_kept, q_rest], dim=1)
  silent = (t == -math.inf).all(dim=1, keepdim=True)  # a teacher without any mass
  log_p = torch.log_softmax(t.masked_fill(silent, 0.0), dim=1)
  p = log_p.exp().masked_fill(silent, 0.0)
  terms = p * (torch.where(p > 0, log_p, torch.zeros_like(p)) -
               torch.where(p > 0, log_q_kept, torch.zeros_like(p)))
  return (temperature ** 2 * terms.sum(1)).float()


def distill_xent(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor,
                 rest: Optional[torch.Tensor] = None, *, temperature: float = 1.0) -> torch.Tensor:
  """``temperature^2 * KL(teacher || student)`` per example, from a teacher's top logits.

  ``logits (rows, classes)`` are the student's; ``values``, ``indices`` (``(rows, k)``) and ``rest``
  (``(rows,)``) are what ``top_logits`` returned for the teacher at the same temperature. With
  ``rest`` all classes that the teacher did not keep are one more outcome ("any other class") on
  both sides; without it the kept classes, renormalised, are the teacher's whole distribution.

  Entries with an index outside ``0 .. classes - 1`` (padding: -1) are left out, of a class listed
  twice the first entry counts; an example with no entry and no ``rest`` has loss and gradient 0.
  An example whose incoming gradient is 0 gets a zero gradient whatever its logits hold. A student whose
  logits are all -inf has no distribution: its loss is not finite. Gradients flow to ``logits`` only
  (first derivatives, on the kernels).
  """
  temperature = _check_logits(logits, temperature, "distill_xent")
  rows, n = logits.shape
  if values.dim() != 2 or values.shape[0] != rows or values.shape[1] < 1:
    raise ValueError(f"distill_xent: values must be ({rows}, k >= 1), got {tuple(values.shape)}")
  if indices.shape != values.shape:
    raise ValueError("distill_xent: indices must have the shape of values, got "
                     f"{tuple(indices.shape)} and {tuple(values.shape)}")
  if indices.dtype not in (torch.int32, torch.int64):
    raise TypeError(f"distill_xent: indices must be int32 or int64, got {indices.dtype}")
  if not values.is_floating_point():
    raise TypeError(f"distill_xent: values must be floating point, got {values.dtype}")
  if rest is not None and rest.shape != (rows,):
    raise ValueError(f"distill_xent: rest must be ({rows},), got {tuple(rest.shape)}")
  dev = logits.device
  if values.device != dev or indices.device != dev or (rest is not None and rest.device != dev):
    raise ValueError(f"distill_xent: values, indices and rest must be on {dev} like logits")
  if _on_kernels(logits, "distill") and values.shape[1] <= 1 << 20:
    if values.dtype not in _FLOAT_CODES:
      values = values.float()
    if rest is not None and (rest.dtype != torch.float32 or not rest.is_contiguous()):
      rest = rest.to(torch.float32).contiguous()
    return _DistillFn.apply(logits, _rows(values), _rows(indices), rest, temperature)
  values, rest = values.detach(), None if rest is None else rest.detach()
  return _distill_reference(logits, values, indices, rest, temperature)
