"""Products of consecutive row groups with a matrix each: a mixture of experts.

    out[i] = lhs[i] . rhs[e(i)]         lhs [M, K], rhs [G, K, N], group_sizes [G]

e(i) is the group row i falls into when the groups, `group_sizes[e]` rows each,
lie one after the other. The reference swaps lax.ragged_dot into its quantized
dot_general for this, forward only (aqt/jax/v2/aqt_ragged_dot.py:23-86); here
the gradients exist too:

    dlhs[i] = g[i] . rhs[e(i)]^T        drhs[e] = sum_{i in e} lhs[i]^T g[i]

    y = ragged_dot(x, w, sizes)                                  # bf16
    y = ragged_dot(x, w, sizes, cfg=block_scaled.dot_general_make())   # fp8
    y = ragged_dot(x, block_quantize(w, 1, square=True), sizes, cfg=...)  # serving

group_sizes (int32 or int64) lives on the device and is never read by the host.
Rows behind the last group give zeros and take no part in drhs; an empty group
has a zero drhs. Sizes are made safe on the device: a negative one counts as
zero, and the running sum is cut at M.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from aqt_b200 import block_engine as be
from aqt_b200.v2 import aqt_tensor
from aqt_b200.v2 import block_scaled


def ragged_dot(lhs, rhs, group_sizes, cfg=None, preferred_element_type=None):
  """lhs [M, K] times rhs [G, K, N], rows grouped by group_sizes [G].

  cfg None: bfloat16 operands, f32 sums. cfg a BlockScaledDotGeneral: float32 or
  bfloat16 operands in block-scaled fp8; rhs may then be a QTensor of 128 x 128
  blocks contracted over axis 1 (serving, without gradient). The result has
  lhs's dtype, or preferred_element_type (float32, bfloat16); without cfg a
  float32 cotangent is rounded to bfloat16, the type of the products.
  """
  out_dtype = _check(lhs, rhs, group_sizes, cfg, preferred_element_type)
  if isinstance(rhs, aqt_tensor.QTensor):
    if torch.is_grad_enabled() and lhs.requires_grad:
      raise NotImplementedError(
          'a product with frozen weights has no gradient; pass float weights')
  elif torch.is_grad_enabled() and (lhs.requires_grad or rhs.requires_grad):
    return _RaggedDot.apply(lhs, rhs, group_sizes, cfg, out_dtype)
  return _forward(lhs, rhs, group_sizes, cfg, out_dtype, (False, False))[0]


def ragged_dot_vjp(lhs, rhs, group_sizes, cfg=None, preferred_element_type=None):
  """(out, backprop) of ragged_dot with backprop(g) -> (dlhs, drhs).

  backprop may read group_sizes and, without cfg, the operands again: they have to
  hold what they held at the call.
  """
  if isinstance(rhs, aqt_tensor.QTensor):
    raise NotImplementedError(
        'a product with frozen weights has no gradient; pass float weights')
  out_dtype = _check(lhs, rhs, group_sizes, cfg, preferred_element_type)
  out, step = _forward(lhs.detach(), rhs.detach(), group_sizes, cfg, out_dtype,
                       (True, True))
  return out, lambda g: _backward(step, step.operands, group_sizes, g,
                                  (True, True))


def _check(lhs, rhs, group_sizes, cfg, preferred):
  q = isinstance(rhs, aqt_tensor.QTensor)
  if cfg is not None and not isinstance(cfg, block_scaled.BlockScaledDotGeneral):
    raise NotImplementedError(
        'cfg is None (bfloat16) or block_scaled.dot_general_make(...)')
  if q and cfg is None:
    raise ValueError('a frozen rhs needs cfg=block_scaled.dot_general_make(...)')
  floats = be._FLOATS if cfg is not None else (torch.bfloat16,)  # pylint: disable=protected-access
  be.check_operand(lhs, 'lhs', floats)
  w = rhs.qvalue if q else rhs
  be.check_operand(w, 'rhs', be._FP8 if q else floats)  # pylint: disable=protected-access
  if not q and lhs.dtype != rhs.dtype:
    raise TypeError(f'Unmatched lhs and rhs dtype: {lhs.dtype} vs {rhs.dtype}')
  if lhs.ndim != 2 or w.ndim != 3:
    raise ValueError('ragged_dot takes lhs [M, K] and rhs [G, K, N] (got '
                     f'{tuple(lhs.shape)}, {tuple(w.shape)})')
  if lhs.shape[1] != w.shape[1]:
    raise ValueError(f'contracted extents differ: lhs {tuple(lhs.shape)}, rhs '
                     f'{tuple(w.shape)}')
  be.check_group_sizes(group_sizes, w.shape[0])
  if not lhs.device == w.device == group_sizes.device:
    be.check_same_device(lhs, w, group_sizes)
  return block_scaled._out_dtype(preferred, lhs)  # pylint: disable=protected-access


class _Step:
  __slots__ = ('cfg', 'operands', 'copied', 'device', 'lhs_dtype', 'rhs_dtype',
               'shape')


def _forward(lhs, rhs, sizes, cfg, out_dtype, grads):
  need_l, need_r = grads
  step = None
  with be.on_device_of(lhs):
    if need_l or need_r:
      step = _Step()
      step.cfg, step.device = cfg, lhs.device
      step.lhs_dtype, step.rhs_dtype = lhs.dtype, rhs.dtype
      step.shape = (*lhs.shape, rhs.shape[2])
    if cfg is None:
      l, w = be.rows_for_tma(lhs), be.matrices_for_tma(rhs, sizes)
      out = be.bf16_rows(l, w, 1, sizes, out_dtype)
      if step is not None:
        # a copy, where one had to be made, serves the backward pass too
        step.operands = be.Residuals(l if need_r else None,
                                     w if need_l else None)
        step.copied = l is not lhs, w is not rhs
      return out, step
    if isinstance(rhs, aqt_tensor.QTensor):
      w, w_n = block_scaled._frozen_operand(rhs, -2), None  # pylint: disable=protected-access
    else:
      w_n, w = be.quantize(rhs, cfg.fwd_dtype, need_l, True, True, cfg.po2_scale)
    l, l_t = be.quantize(lhs, cfg.fwd_dtype, True, need_r, False, cfg.po2_scale,
                         sizes if need_r else None)
    out = be.fp8_rows(l, w, lhs.shape[1], out_dtype, lhs.device, sizes,
                      cfg.po2_scale and not isinstance(rhs, aqt_tensor.QTensor))
    if step is not None:
      step.operands = be.Residuals(l_t, w_n if need_l else None)
  return out, step


def _backward(step, operands, sizes, g, grads):
  need_l, need_r = grads
  cfg = step.cfg
  m, k, n = step.shape
  be.check_operand(g, 'the cotangent')
  g = g.detach()
  if g.device != step.device:
    raise ValueError(
        f'operands on different devices: {step.device}, {g.device}')
  if tuple(g.shape) != (m, n):
    raise ValueError(f'the cotangent has shape {tuple(g.shape)}, the result '
                     f'{(m, n)}')
  dlhs = drhs = None
  if cfg is None:
    with be.on_device_of(g):
      operands.about_to_use()
      g = be.rows_for_tma(be.as_bf16(g))
      if need_l:
        dlhs = be.bf16_rows(g, operands.rhs, 2, sizes, step.lhs_dtype)
      if need_r:
        drhs = be.bf16_contract_rows(operands.lhs, g, sizes, step.rhs_dtype)
    return dlhs, drhs
  with be.on_device_of(g):
    operands.about_to_use()
    q, q_t = be.quantize(g, cfg.bwd_dtype, need_l, need_r, False, cfg.po2_scale,
                         sizes if need_r else None)
    if need_l:
      dlhs = be.fp8_rows(q, operands.rhs, n, step.lhs_dtype, g.device, sizes,
                         cfg.po2_scale)
    if need_r:
      # positions along the groups' padded rows, as both operands were laid out
      drhs = be.fp8_contract_rows(operands.lhs, q_t, operands.lhs.ld, m,
                                  step.rhs_dtype, g.device, sizes, cfg.po2_scale)
  return dlhs, drhs


class _RaggedDot(torch.autograd.Function):

  @staticmethod
  def forward(ctx, lhs, rhs, sizes, cfg, out_dtype):
    out, step = _forward(lhs.detach(), rhs.detach(), sizes, cfg, out_dtype,
                         ctx.needs_input_grad[:2])
    l, w = step.operands.release()
    if cfg is None:
      # operands themselves: saved the way torch watches for writes into them
      l = lhs if l is not None and not step.copied[0] else l
      w = rhs if w is not None and not step.copied[1] else w
    ctx.save_for_backward(sizes, l, w)
    ctx.step = step
    return out

  @staticmethod
  @once_differentiable
  def backward(ctx, g):
    step = ctx.step
    sizes, lhs, rhs = ctx.saved_tensors
    # hooks on saved tensors may give them back in other strides
    sizes = sizes.contiguous()
    if step.cfg is None:
      with be.on_device_of(sizes):
        lhs = None if lhs is None else be.rows_for_tma(lhs.detach())
        rhs = None if rhs is None else be.matrices_for_tma(rhs.detach(), sizes)
    dlhs, drhs = _backward(step, step.operands.regain(lhs, rhs), sizes, g,
                           ctx.needs_input_grad[:2])
    return dlhs, drhs, None, None, None
