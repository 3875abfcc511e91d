"""Gated MLP on the GPU (``csrc/gated_tcgen05.cu``, ``csrc/gated_rows.cuh``), differentiable.

``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo (+ residual)`` per expert. One kernel runs both
projections, the activation and the product (a tcgen05 tile kernel, or a weight-streaming one for up
to 16 or 32 rows); the output projection runs on the same tiles, on the library's GEMM or on the streaming
kernel. Backward (first derivatives only): one kernel for the gradients of both projections and their
column sums, then products for ``dx``, ``dw_in`` and ``dw_out``. Each direction is one call into the
library. The reference has no gated MLP.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
import torch.nn.functional as F

from vmoe_b200.ops import _lib, functional

ACTIVATIONS = {"gelu": 0, "silu": 1}
_GRAD_BF16, _GRAD_F32, _GRAD_ADD = 0, 1, 2  # VMOE_GRAD_*


def _contiguous(t: torch.Tensor) -> torch.Tensor:
  return t if t.is_contiguous() else t.contiguous()


def _bias(b):
  if b is None:
    return None
  return _contiguous(b if b.dtype in (torch.bfloat16, torch.float32) else b.float())


def _weights(w: torch.Tensor) -> torch.Tensor:
  return _contiguous(w if w.dtype == torch.bfloat16 else functional.bf16_shadow(w))


def _forward(x, w_in, b_in, w_out, b_out, residual, act: int, save: bool):
  """``(y, x, hidden, saved)`` with ``x`` as the kernels read it; the last two are inputs of the
  backward pass (``saved`` is None without ``save``). Called where autograd records nothing."""
  x = _contiguous(x)
  w_in, w_out, b_in, b_out = _weights(w_in), _weights(w_out), _bias(b_in), _bias(b_out)
  e, r, h = x.shape
  _, o, m = w_out.shape
  bf16, dev = torch.bfloat16, x.device
  y = torch.empty((e, r, o), dtype=bf16, device=dev)
  hid = torch.empty((e, r, m), dtype=bf16, device=dev)
  saved = torch.empty((e, r, 2, m), dtype=bf16, device=dev) if save else None
  res_batch_stride, ld_res = residual.stride()[:2] if residual is not None else (0, 0)
  b_out_bf16 = b_out is not None and b_out.dtype == bf16
  ptr = _lib.ptr
  g = _lib.GatedArgs(x.data_ptr(), w_in.data_ptr(), ptr(b_in), w_out.data_ptr(), ptr(b_out),
                     ptr(residual), y.data_ptr(), hid.data_ptr(), ptr(saved), None, None, None, None,
                     None, None, None, None, e, r, h, m, o, ld_res, res_batch_stride, act,
                     b_in is not None and b_in.dtype == bf16, b_out_bf16)
  lib = _lib.lib()
  if b_out_bf16:
    size = lib.vmoe_gated_scratch_bytes(ctypes.byref(g), 0)
    if size:
      scratch = torch.empty(size // 4, dtype=torch.float32, device=dev)
      g.scratch = scratch.data_ptr()
  _lib.check(lib.vmoe_gated_fwd(ctypes.byref(g), _lib.stream_ptr()), "vmoe_gated_fwd")
  _lib.count_launch(2)
  return y, x, hid, saved


def _gradient_of(p: torch.Tensor):
  """``(buffer, mode, value for autograd)`` of a parameter's gradient: its bound fp32 buffer, which is
  added to (nothing for autograd), or a new tensor in the parameter's type."""
  tgt = functional._grad_target(p)
  if tgt is not None:
    return tgt, _GRAD_ADD, None
  if p.dtype == torch.bfloat16:
    new = torch.empty(p.shape, dtype=torch.bfloat16, device=p.device)
    return new, _GRAD_BF16, new
  new = torch.empty(p.shape, dtype=torch.float32, device=p.device)
  return new, _GRAD_F32, new


class _GatedMlpFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, w_in, b_in, w_out, b_out, residual, act):
    save = any(ctx.needs_input_grad[:4])
    with _lib.on_device(x):
      y, x, hid, saved = _forward(x, w_in, b_in, w_out, b_out, residual, act, save)
    ctx.save_for_backward(x, w_in, w_out, saved, hid if save else None)
    ctx.biases = (b_in, b_out)
    return y

  @staticmethod
  @functional.first_order
  def backward(ctx, dy):
    x, w_in, w_out, saved, hid = ctx.saved_tensors
    b_in, b_out = ctx.biases
    need_x, need_w_in, need_b_in, need_w_out, need_b_out, need_res, _ = ctx.needs_input_grad
    e, r, h = x.shape
    _, o, m = w_out.shape
    dx = dw_in = db_in = dw_out = db_out = None
    with _lib.on_device(x):
      dy = _contiguous(dy)
      if dy.data_ptr() % 16:
        dy = dy.clone()
      dev = dy.device
      g = _lib.GatedArgs()
      g.x, g.dy = x.data_ptr(), dy.data_ptr()
      g.e, g.rows, g.h, g.m, g.o = e, r, h, m, o
      keep = []  # buffers that must live until the launches are enqueued
      if need_x or need_w_in or need_b_in:
        w16 = _weights(w_out)
        dgu = torch.empty((e, r, 2, m), dtype=torch.bfloat16, device=dev)
        g.saved, g.w_out, g.dgu = saved.data_ptr(), w16.data_ptr(), dgu.data_ptr()
        keep += [w16, dgu]
        launches = 1
      else:
        launches = 0
      if need_x:
        w16 = _weights(w_in)
        dx = torch.empty((e, r, h), dtype=torch.bfloat16, device=dev)
        g.w_in, g.dx = w16.data_ptr(), dx.data_ptr()
        keep.append(w16)
      if need_w_in:
        buf, g.dw_in_mode, dw_in = _gradient_of(w_in)
        g.dw_in = buf.data_ptr()
        keep.append(buf)
      if need_w_out:
        buf, g.dw_out_mode, dw_out = _gradient_of(w_out)
        g.dw_out, g.hid = buf.data_ptr(), hid.data_ptr()
        keep.append(buf)
      if need_b_in:
        buf, g.db_in_mode, db_in = _gradient_of(b_in)
        g.db_in = buf.data_ptr()
        keep.append(buf)
      if need_b_out:
        buf, g.db_out_mode, db_out = _gradient_of(b_out)
        g.db_out = buf.data_ptr()
        keep.append(buf)
      lib = _lib.lib()
      size = lib.vmoe_gated_scratch_bytes(ctypes.byref(g), 1)
      if size:
        keep.append(torch.empty(size // 4, dtype=torch.float32, device=dev))
        g.scratch = keep[-1].data_ptr()
      if launches or need_w_out or need_b_out:
        _lib.check(lib.vmoe_gated_bwd(ctypes.byref(g), _lib.stream_ptr()), "vmoe_gated_bwd")
        _lib.count_launch(launches + int(need_x) + int(need_w_in) + int(need_w_out) +
                          int(need_b_out) + int(need_b_in or need_b_out))
    return dx, dw_in, db_in, dw_out, db_out, dy if need_res else None, None


def gated_reference(x, w_in, b_in, w_out, b_out, act: str, residual=None):
  """The same in PyTorch ops, in the type of ``x``."""
  dt = x.dtype

  def project(i):
    w = w_in[:, i].to(dt).transpose(1, 2)
    return torch.bmm(x, w) if b_in is None else torch.baddbmm(b_in[:, i].to(dt).unsqueeze(1), x, w)

  g = project(0)
  g = F.silu(g) if act == "silu" else F.gelu(g, approximate="tanh")
  hid, w = g * project(1), w_out.to(dt).transpose(1, 2)
  y = torch.bmm(hid, w) if b_out is None else torch.baddbmm(b_out.to(dt).unsqueeze(1), hid, w)
  return y if residual is None else y + residual


def check_args(x, w_in, b_in, w_out, b_out, act, residual) -> None:
  if act not in ACTIVATIONS:
    raise ValueError(f"expert_gated_mlp: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
  xs, ws, wos = x.shape, w_in.shape, w_out.shape
  if len(xs) != 3 or len(ws) != 4 or len(wos) != 3:
    raise ValueError("expert_gated_mlp: x must be (E, R, H), w_in (E, 2, M, H), w_out (E, O, M); got "
                     f"{tuple(xs)}, {tuple(ws)}, {tuple(wos)}")
  e, r, h = xs
  _, o, m = wos
  if ws != (e, 2, m, h) or wos[0] != e or min(h, m, o) < 1:
    raise ValueError("expert_gated_mlp: x (E, R, H), w_in (E, 2, M, H) and w_out (E, O, M) do not fit "
                     f"together: {tuple(xs)}, {tuple(ws)}, {tuple(wos)}")
  if residual is not None and residual.dtype != x.dtype:
    raise TypeError(f"expert_gated_mlp: residual must be {x.dtype} like x, got {residual.dtype}")
  dev = x.device
  for name, t, shape in (("w_in", w_in, None), ("b_in", b_in, (e, 2, m)), ("w_out", w_out, None),
                         ("b_out", b_out, (e, o)), ("residual", residual, (e, r, o))):
    if t is None:
      continue
    if shape is not None and t.shape != shape:
      raise ValueError(f"expert_gated_mlp: {name} must be {shape}, got {tuple(t.shape)}")
    if t.device != dev:
      raise ValueError(f"expert_gated_mlp: {name} is on {t.device}, x on {dev}")
    if not t.is_floating_point():
      raise TypeError(f"expert_gated_mlp: {name} must be floating point, got {t.dtype}")


def gated_mlp(x, w_in, b_in, w_out, b_out, act: str, residual=None) -> torch.Tensor:
  """The kernel path; operands as checked by ``check_args``, ``x`` bf16 on a GPU."""
  h, m, o = x.shape[2], w_in.shape[2], w_out.shape[1]
  hp, mp, op = -h % 8, -m % 8, -o % 8
  if hp or mp or op:
    # TMA rows are multiples of 16 bytes: zero-pad the odd widths (autograd cuts the gradients).
    # Zero hidden units and inputs add nothing, the padded outputs are cut off.
    x = F.pad(x, (0, hp))
    w_in, w_out = F.pad(w_in, (0, hp, 0, mp)), F.pad(w_out, (0, mp, 0, op))
    b_in = None if b_in is None else F.pad(b_in, (0, mp))
    b_out = None if b_out is None else F.pad(b_out, (0, op))
    residual = None if residual is None else F.pad(residual, (0, op))
  if residual is not None:
    batch, row, unit = residual.stride()
    if unit != 1 or row % 8 or batch % 8 or residual.data_ptr() % 16:
      residual = residual.contiguous()
  if x.data_ptr() % 16:  # a view that starts inside 16 bytes
    x = x.clone()
  args = (x, w_in, b_in, w_out, b_out, residual)
  if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in args]):
    y = _GatedMlpFn.apply(*args, ACTIVATIONS[act])
  else:
    with _lib.on_device(x):
      y = _forward(*args, ACTIVATIONS[act], False)[0]
  return y[..., :o] if op else y


def expert_gated_mlp(x: torch.Tensor, w_in: torch.Tensor, b_in: Optional[torch.Tensor],
                     w_out: torch.Tensor, b_out: Optional[torch.Tensor], *, act: str = "gelu",
                     residual: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Per-expert gated MLP ``(act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo (+ residual)``.

  ``x (E_local, rows, H)``; ``w_in (E, 2, M, H)`` holds the gate's projection in ``[:, 0]`` and the
  other one in ``[:, 1]``, ``b_in (E, 2, M)`` their biases; ``w_out (E, O, M)``, ``b_out (E, O)``;
  ``residual (E, rows, O)``. Biases may be None. ``act``: 'gelu' (tanh form) or 'silu'. Any number
  of rows, also none; widths that are not multiples of 8 are zero-padded inside the call.
  """
  check_args(x, w_in, b_in, w_out, b_out, act, residual)
  if functional._fast(x):
    return gated_mlp(x, w_in, b_in, w_out, b_out, act, residual)
  return gated_reference(x, w_in, b_in, w_out, b_out, act, residual)
