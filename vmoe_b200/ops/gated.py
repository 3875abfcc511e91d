"""Gated MLP on the tcgen05 kernels (``csrc/gated_tcgen05.cu``), differentiable.

``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo (+ residual)`` per expert. One kernel runs both
projections, the activation and the product, the output projection is the library's GEMM. Backward:
one kernel for the gradients of both projections (and their column sums), then three GEMMs for
``dx``, ``dw_in`` and ``dw_out``. The reference has no gated MLP.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
import torch.nn.functional as F

from vmoe_b200.ops import _lib, functional
from vmoe_b200.ops.gemm import gemm

_vp = ctypes.c_void_p
ACTIVATIONS = {"gelu": 0, "silu": 1}


def _args(a, w, k, m, act=0) -> "_lib.GatedArgs":
  e, rows = a.shape[:2]
  g = _lib.GatedArgs()
  g.a, g.w = a.data_ptr(), w.data_ptr()
  g.e, g.rows, g.k, g.m = e, rows, k, m
  g.lda, g.a_batch_stride = a.stride(1), a.stride(0)
  g.act = act
  return g


def _forward(x, w_in, b_in, act: int, save: bool):
  """``(hidden (E, R, M), saved (E, R, 2, M) or None)`` of contiguous bf16 operands."""
  e, r, h = x.shape
  m = w_in.shape[2]
  hid = torch.empty(e, r, m, dtype=torch.bfloat16, device=x.device)
  saved = torch.empty(e, r, 2, m, dtype=torch.bfloat16, device=x.device) if save else None
  g = _args(x, w_in, h, m, act)
  g.bias, g.hid, g.saved = _lib.ptr(b_in), hid.data_ptr(), _lib.ptr(saved)
  _lib.check(_lib.lib().vmoe_gated_fwd(ctypes.byref(g), _vp(_lib.stream_ptr())), "vmoe_gated_fwd")
  _lib.count_launch()
  return hid, saved


def _backward(dy, w_out, saved, db: Optional[torch.Tensor], accumulate: bool):
  """Gradients of both projections ``(E, R, 2, M)``; their column sums go to ``db (E, 2, M)``."""
  e, r, o = dy.shape
  m = saved.shape[3]
  grad = torch.empty_like(saved)
  g = _args(dy, w_out, o, m)
  g.saved, g.grad = saved.data_ptr(), grad.data_ptr()
  lib = _lib.lib()
  sums = None
  if db is not None:
    size = lib.vmoe_gated_bwd_sums_bytes(ctypes.c_int64(e), ctypes.c_int64(r), ctypes.c_int64(m))
    sums = torch.empty(size // 4, dtype=torch.float32, device=dy.device)
  rc = lib.vmoe_gated_bwd(ctypes.byref(g), _vp(_lib.ptr(sums)), _vp(_lib.ptr(db)),
                          ctypes.c_int32(int(accumulate)), _vp(_lib.stream_ptr()))
  _lib.check(rc, "vmoe_gated_bwd")
  _lib.count_launch(1 if db is None else 2)
  return grad


def _weight_grad(dy, x, weight, shape):
  """``dy^T x`` for ``weight`` (viewed as ``shape``): None if added to its bound fp32 gradient, else
  in the weight's type."""
  e, n, k = shape
  split = functional._wgrad_split(n, k, dy.shape[1]) if e == 1 else 1
  tgt = functional._grad_target(weight)
  if tgt is not None:
    gemm(dy, x, a_mn_major=True, b_mn_major=True, out=tgt.view(shape), accumulate=True, split_k=split)
    return None
  if dy.shape[1] == 0:
    return torch.zeros_like(weight)
  if weight.dtype == torch.bfloat16 and split == 1:
    return gemm(dy, x, a_mn_major=True, b_mn_major=True).view(weight.shape)
  dw = torch.zeros(shape, dtype=torch.float32, device=dy.device)
  gemm(dy, x, a_mn_major=True, b_mn_major=True, out=dw, accumulate=True, split_k=split)
  return dw.view(weight.shape).to(weight.dtype)


class _GatedMlpFn(torch.autograd.Function):

  @staticmethod
  def forward(ctx, x, w_in, b_in, w_out, b_out, residual, act):
    with _lib.on_device(x):
      x = x.contiguous()
      w_in16, w_out16 = functional.bf16_shadow(w_in), functional.bf16_shadow(w_out)
      b_in32 = None if b_in is None else b_in.detach().float().contiguous()
      b_out32 = None if b_out is None else b_out.detach().float().contiguous()
      hid, saved = _forward(x, w_in16.contiguous(), b_in32, act, any(ctx.needs_input_grad[:4]))
      y = gemm(hid, w_out16.contiguous(), bias=b_out32, residual=residual)
    ctx.save_for_backward(x, w_in, w_out, saved, hid if saved is not None else None)
    ctx.biases = (b_in, b_out)
    return y

  @staticmethod
  def backward(ctx, dy):
    x, w_in, w_out, saved, hid = ctx.saved_tensors
    b_in, b_out = ctx.biases
    need = ctx.needs_input_grad
    e, r, h = x.shape
    m, o = w_in.shape[2], w_out.shape[1]
    dx = dw_in = db_in = dw_out = db_out = None
    with _lib.on_device(x):
      dy = dy.contiguous()
      if need[3]:
        dw_out = _weight_grad(dy, hid, w_out, (e, o, m))
      if b_out is not None and need[4]:
        db_out = functional.bias_grad(dy, b_out)
        db_out = None if db_out is None else db_out.to(b_out.dtype)
      if need[0] or need[1] or need[2]:
        tgt = None
        if b_in is not None and need[2]:
          tgt = functional._grad_target(b_in)
          db_in = tgt if tgt is not None else \
              torch.zeros(e, 2, m, dtype=torch.float32, device=dy.device)
        dgu = _backward(dy, functional.bf16_shadow(w_out).contiguous(), saved, db_in,
                        tgt is not None).view(e, r, 2 * m)
        if db_in is not None:
          db_in = None if tgt is not None else db_in.to(b_in.dtype)
        if need[0]:
          w_in16 = functional.bf16_shadow(w_in).contiguous()
          dx = gemm(dgu, w_in16.view(e, 2 * m, h), b_mn_major=True)
        if need[1]:
          dw_in = _weight_grad(dgu, x, w_in, (e, 2 * m, h))
    return dx, dw_in, db_in, dw_out, db_out, dy if need[5] else None, None


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
  if x.dim() != 3 or w_in.dim() != 4 or w_out.dim() != 3:
    raise ValueError("expert_gated_mlp: x must be (E, R, H), w_in (E, 2, M, H), w_out (E, O, M); got "
                     f"{tuple(x.shape)}, {tuple(w_in.shape)}, {tuple(w_out.shape)}")
  e, r, h = x.shape
  m, o = w_in.shape[2], w_out.shape[1]
  if tuple(w_in.shape) != (e, 2, m, h) or tuple(w_out.shape) != (e, o, m) or min(h, m, o) < 1:
    raise ValueError("expert_gated_mlp: x (E, R, H), w_in (E, 2, M, H) and w_out (E, O, M) do not fit "
                     f"together: {tuple(x.shape)}, {tuple(w_in.shape)}, {tuple(w_out.shape)}")
  for name, t, shape in (("b_in", b_in, (e, 2, m)), ("b_out", b_out, (e, o)),
                         ("residual", residual, (e, r, o))):
    if t is not None and tuple(t.shape) != shape:
      raise ValueError(f"expert_gated_mlp: {name} must be {shape}, got {tuple(t.shape)}")
  if residual is not None and residual.dtype != x.dtype:
    raise TypeError(f"expert_gated_mlp: residual must be {x.dtype} like x, got {residual.dtype}")
  for name, t in (("w_in", w_in), ("b_in", b_in), ("w_out", w_out), ("b_out", b_out),
                  ("residual", residual)):
    if t is not None and t.device != x.device:
      raise ValueError(f"expert_gated_mlp: {name} is on {t.device}, x on {x.device}")
    if t is not None and not t.dtype.is_floating_point:
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
  if residual is not None and (residual.stride(-1) != 1 or residual.stride(-2) % 8):
    residual = residual.contiguous()
  y = _GatedMlpFn.apply(x, w_in, b_in, w_out, b_out, residual, ACTIVATIONS[act])
  return y[..., :o] if op else y
