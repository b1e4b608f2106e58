"""Block-scaled fp8: one f32 scale for each block of 128 elements.

The reference calls this sub-channel quantization and reaches it by reshaping
the contraction axis of a dot_general into tiles with a scale each
(aqt/jax/v2/tiled_dot_general.py:85-568); here the blocks are 128 long, the
width one tensor-core accumulation covers, and the kernels take them directly:

    qt = block_quantize(w, contract_axis=0, square=True)       # frozen weights
    dg = dot_general_make(fwd_bits='e4m3', bwd_bits='e5m2')
    y = dg(x, qt, dims)                                         # serving
    y = dg(x, w, dims)                                          # training

Activations and cotangents have blocks of 1 x 128 along the contraction of the
product they enter, weights blocks of 128 x 128, so that one quantization of the
weights serves the forward product and dlhs:

    out  = lhs . rhs        lhs 1 x 128 along k, rhs 128 x 128
    dlhs = g . rhs^T        g   1 x 128 along n, the same rhs
    drhs = lhs^T . g        both 128 x 1 along the rows

A block: a = max|x|, s = max((a or 1) / bound, 2^-126) in f32 [, up to a power of
two], q = fp8(x * (1 / s)); products of 128 are summed on the tensor core, scaled
and added in f32, and the result is rounded once to the output's dtype -- for any
scales, also where the product of two is no f32 number and the result is one. With
po2_scale and a bfloat16 result the tensor core scales and sums large products by
itself, 1.3 times as fast; its sums drop what does not fit 24 bits (up to 2^-23 of
the running sum for each 32 products). A NaN or an infinity in a block makes that
block's scale, and what is computed from it, NaN or infinite, as absmax calibration
does (calibration.py:117-157).
"""

from __future__ import annotations

import dataclasses
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from aqt_b200 import _lib
from aqt_b200 import block_engine as be
from aqt_b200.v2 import aqt_tensor
from aqt_b200.v2 import utils

BLOCK = be.BLOCK


@dataclasses.dataclass(frozen=True)
class BlockTiling:
  """How a QTensor's scale divides its last two axes (the reference keeps a
  TilingState there, tiled_dot_general.py:182-330)."""
  contract_axis: int  # -1 or -2
  square: bool


_TILINGS = {(a, s): BlockTiling(a, s) for a in (-1, -2) for s in (False, True)}


def _axis(contract_axis, ndim):
  if contract_axis in (-1, ndim - 1):
    return -1
  if contract_axis in (-2, ndim - 2):
    return -2
  raise NotImplementedError(
      'blocks lie along one of the last two axes '
      f'(contract_axis {contract_axis} of {ndim})')


def block_quantize(x, contract_axis: int = -1, square: bool = False,
                   bits='e4m3', po2_scale: bool = False) -> aqt_tensor.QTensor:
  """Quantizes x [R, C] or [G, R, C] (float32, bfloat16) to fp8 in blocks of 128.

  contract_axis: axis the blocks lie along (one of the last two); `qvalue` has
  that axis contiguous in memory. square: blocks of 128 x 128. bits: 'e4m3' or
  'e5m2'. po2_scale: scales rounded up to powers of two.

  Returns a QTensor with x's shape: `qvalue` fp8, `scale[0]` f32 with every
  blocked axis divided by 128 (rounded up), `tiling_state` a BlockTiling.
  """
  be.check_operand(x, 'x')
  if x.ndim not in (2, 3):
    raise NotImplementedError(
        f'block_quantize takes [R, C] or [G, R, C] (got {tuple(x.shape)})')
  axis = _axis(contract_axis, x.ndim)
  dtype = be.fp8_dtype(bits)
  with be.on_device_of(x):
    q, s = be.quantize_tensors(x, dtype, axis, square, po2_scale)
  return aqt_tensor.QTensor(
      qvalue=q, scale=[s], scale_t=None, dequant_dtype=utils.as_dtype(x.dtype),
      tiling_state=_TILINGS[axis, bool(square)])


def frozen(qvalue, scale, contract_axis: int = -2) -> aqt_tensor.QTensor:
  """A QTensor of weights quantized in 128 x 128 blocks, from a checkpoint's
  values [K, N] or [G, K, N] and scales [.., ceil(K/128), ceil(N/128)].

  The product needs the contraction axis contiguous in memory; values that lie
  otherwise are copied once, here (by a traced step: on every replay).
  """
  be.check_operand(qvalue, 'qvalue', be._FP8)  # pylint: disable=protected-access
  be.check_operand(scale, 'scale', (torch.float32,))
  be.check_same_device(qvalue, scale)
  if qvalue.ndim not in (2, 3):
    raise NotImplementedError('frozen weights are [K, N] or [G, K, N]')
  axis = _axis(contract_axis, qvalue.ndim)
  want = (*qvalue.shape[:-2], -(-qvalue.shape[-2] // BLOCK),
          -(-qvalue.shape[-1] // BLOCK))
  if tuple(scale.shape) != want:
    raise ValueError(f'scale has shape {tuple(scale.shape)}; 128 x 128 blocks '
                     f'of {tuple(qvalue.shape)} need {want}')
  if not _contract_contiguous(qvalue, axis):
    with be.on_device_of(qvalue):
      v = qvalue if axis == -1 else qvalue.transpose(-1, -2)
      v = be.padded_rows(v)
      qvalue = v if axis == -1 else v.transpose(-1, -2)
  return aqt_tensor.QTensor(
      qvalue=qvalue, scale=[scale], scale_t=None, dequant_dtype=None,
      tiling_state=BlockTiling(axis, True))


def _contract_contiguous(q, axis):
  """Contraction contiguous, other strides and the address multiples of 16."""
  other = -3 - axis
  if q.numel() == 0:
    return True
  if (q.stride(axis) != 1 and q.shape[axis] > 1) or q.data_ptr() % 16:
    return False
  if q.shape[other] > 1 and (q.stride(other) % 16 or q.stride(other) <= 0):
    return False
  return q.ndim == 2 or q.shape[0] == 1 or (q.stride(0) % 16 == 0 and
                                            q.stride(0) > 0)


def _frozen_operand(qt, contract_axis):
  """Frozen weights as the Side of a product that contracts `contract_axis`."""
  ts = qt.tiling_state
  if not isinstance(ts, BlockTiling) or not ts.square:
    raise NotImplementedError(
        'a frozen operand is quantized in 128 x 128 blocks: '
        'block_quantize(w, contract_axis=..., square=True) or frozen(...)')
  if not qt.is_full() or not qt.scale:
    raise ValueError('a frozen operand needs its values and its scale')
  if ts.contract_axis != contract_axis:
    raise NotImplementedError(
        f'frozen with axis {ts.contract_axis} contiguous, but the product '
        f'contracts axis {contract_axis}: quantize it for that axis')
  q, s = qt.qvalue, qt.scale[0]
  if not _contract_contiguous(q, contract_axis):
    raise ValueError('frozen values must keep the layout block_quantize or '
                     'frozen gave them (contraction contiguous, 16-byte rows)')
  want = (*q.shape[:-2], -(-q.shape[-2] // BLOCK), -(-q.shape[-1] // BLOCK))
  if tuple(s.shape) != want or s.dtype != torch.float32 or s.device != q.device:
    raise ValueError(
        f'frozen values {tuple(q.shape)} need float32 scales {want} on their '
        f'device (got {s.dtype} {tuple(s.shape)} on {s.device})')
  kept_axis = -3 - contract_axis
  # an axis of one entry may have any stride; the kernel wants a valid one
  ld = (q.stride(kept_axis) if q.shape[kept_axis] > 1 else
        (q.shape[contract_axis] + 15) & -16)
  batched = q.ndim == 3
  return be.Side(q.data_ptr(), ld, q.stride(0) if batched else 0,
                 _CODES[q.dtype], s.data_ptr(), s.stride(0) if batched else 0,
                 s.stride(contract_axis), s.stride(kept_axis),
                 q.shape[kept_axis], (q, s))


_CODES = {torch.float8_e4m3fn: _lib.E4M3, torch.float8_e5m2: _lib.E5M2}


class _Step:
  """One forward product's operands, as its backward pass needs them."""

  __slots__ = ('operands', 'device', 'rows', 'k', 'n', 'lhs_shape', 'lhs_axis',
               'rhs_axis', 'lhs_dtype', 'rhs_dtype')


@dataclasses.dataclass(frozen=True)
class BlockScaledDotGeneral:
  """A block-scaled dot_general with its two gradient products.

  Called like lax.dot_general: lhs [..., K] with any leading axes (or a matrix
  [K, M]), rhs a matrix, one contracted axis each, no batch axes. rhs may be a
  QTensor of 128 x 128 blocks (serving; then without gradient).
  """
  fwd_dtype: Any
  bwd_dtype: Any
  po2_scale: bool = False

  def __call__(self, lhs, rhs, dimension_numbers, precision=None,
               preferred_element_type=None):
    assert precision is None, (
        f'Precision {precision} requested together with quantization.')
    dims = _dims(lhs, rhs, dimension_numbers)
    out_dtype = _out_dtype(preferred_element_type, lhs)
    if isinstance(rhs, aqt_tensor.QTensor):
      if lhs.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(
            'a product with frozen weights has no gradient; pass float weights')
      return self._forward(lhs, rhs, dims, out_dtype, None)[0]
    if (lhs.requires_grad or rhs.requires_grad) and torch.is_grad_enabled():
      return _BlockDot.apply(lhs, rhs, self, dims, out_dtype)
    return self._forward(lhs, rhs, dims, out_dtype, (False, False))[0]

  def vjp(self, lhs, rhs, dimension_numbers, preferred_element_type=None):
    """(out, backprop) with backprop(g) -> (dlhs, drhs)."""
    if isinstance(rhs, aqt_tensor.QTensor):
      raise NotImplementedError(
          'a product with frozen weights has no gradient; pass float weights')
    dims = _dims(lhs, rhs, dimension_numbers)
    out_dtype = _out_dtype(preferred_element_type, lhs)
    out, step = self._forward(lhs.detach(), rhs.detach(), dims, out_dtype,
                              (True, True))
    return out, lambda g: self._backward(step, step.operands, g, (True, True))

  def _forward(self, lhs, rhs, dims, out_dtype, grads):
    lhs_axis, rhs_axis = dims
    x = _as_matrix(lhs, lhs_axis)
    device = lhs.device
    with be.on_device_of(lhs):
      if grads is None:
        need_l = need_r = False
        w, w_t = _frozen_operand(rhs, rhs_axis), None
      else:
        need_l, need_r = grads
        contracts_last = rhs_axis == -1
        sides = be.quantize(rhs, self.fwd_dtype, contracts_last or need_l,
                            not contracts_last or need_l, True, self.po2_scale)
        w, w_t = sides if contracts_last else (sides[1], sides[0])
      l, l_t = be.quantize(x, self.fwd_dtype, True, need_r, False,
                           self.po2_scale)
      m, k = x.shape
      out = be.fp8_rows(l, w, k, out_dtype, device,
                        po2=self.po2_scale and grads is not None)
      step = None
      if need_l or need_r:
        step = _Step()
        step.operands = be.Residuals(l_t, w_t if need_l else None)
        step.device = device
        step.rows, step.k, step.n = m, k, w.kept
        step.lhs_shape, step.lhs_axis, step.rhs_axis = lhs.shape, lhs_axis, rhs_axis
        step.lhs_dtype, step.rhs_dtype = lhs.dtype, rhs.dtype
    if lhs.ndim != 2:
      out = out.view(*lhs.shape[:-1], w.kept)
    return out, step

  def _backward(self, step, operands, g, grads):
    need_l, need_r = grads
    m, k, n = step.rows, step.k, step.n
    be.check_operand(g, 'the cotangent')
    g = g.detach()
    if g.device != step.device:
      raise ValueError(
          f'operands on different devices: {step.device}, {g.device}')
    want = ((*step.lhs_shape[:-1], n) if step.lhs_axis == -1 else (m, n))
    if tuple(g.shape) != want:
      raise ValueError(f'the cotangent has shape {tuple(g.shape)}, the result '
                       f'{want}')
    device = g.device
    gm = _as_matrix(g, -1)
    dlhs = drhs = None
    with be.on_device_of(g):
      operands.about_to_use()
      q, q_t = be.quantize(gm, self.bwd_dtype, need_l, need_r, False,
                           self.po2_scale)
      if need_l:
        dlhs = be.fp8_rows(q, operands.rhs, n, step.lhs_dtype, device,
                           po2=self.po2_scale)
      if need_r:
        # [K, N] as rhs lies: its last axis is the output's contiguous one
        b, a = ((operands.lhs, q_t) if step.rhs_axis == -2 else
                (q_t, operands.lhs))
        drhs = be.fp8_contract_rows(b, a, m, m, step.rhs_dtype, device,
                                    po2=self.po2_scale)
    if need_l:
      if step.lhs_axis == -2:
        dlhs = dlhs.transpose(0, 1)
      elif len(step.lhs_shape) != 2:
        dlhs = dlhs.view(step.lhs_shape)
    return dlhs, drhs


class _BlockDot(torch.autograd.Function):
  """The custom VJP (aqt_dot_general.py:993-997) on torch's tape."""

  @staticmethod
  def forward(ctx, lhs, rhs, cfg, dims, out_dtype):
    ctx.cfg = cfg
    out, ctx.step = cfg._forward(  # pylint: disable=protected-access
        lhs.detach(), rhs.detach(), dims, out_dtype, ctx.needs_input_grad[:2])
    ctx.save_for_backward(*ctx.step.operands.release())
    return out

  @staticmethod
  @once_differentiable
  def backward(ctx, g):
    dlhs, drhs = ctx.cfg._backward(  # pylint: disable=protected-access
        ctx.step, ctx.step.operands.regain(*ctx.saved_tensors), g,
        ctx.needs_input_grad[:2])
    return dlhs, drhs, None, None, None


def dot_general_make(fwd_bits='e4m3', bwd_bits='e5m2',
                     po2_scale: bool = False) -> BlockScaledDotGeneral:
  """Block-scaled products: lhs and rhs in `fwd_bits`, cotangents in `bwd_bits`
  ('e4m3' or 'e5m2'), scales rounded up to powers of two with `po2_scale`."""
  return BlockScaledDotGeneral(be.fp8_dtype(fwd_bits), be.fp8_dtype(bwd_bits),
                               bool(po2_scale))


def _out_dtype(preferred, lhs):
  if preferred is None:
    return lhs.dtype
  d = utils.as_dtype(preferred)
  for t in (torch.float32, torch.bfloat16):
    if utils.as_dtype(t) == d:
      return t
  raise NotImplementedError(
      f'results are float32 or bfloat16 (preferred_element_type {preferred})')


def _dims(lhs, rhs, dimension_numbers):
  """Checks the operands; returns the contracted axes as negative numbers."""
  (lca, rca), (lba, rba) = dimension_numbers
  if lba or rba or len(lca) != 1 or len(rca) != 1:
    raise NotImplementedError(
        'block-scaled products contract one axis of each operand and have no '
        f'batch axes (got {dimension_numbers})')
  be.check_operand(lhs, 'lhs')
  if isinstance(rhs, aqt_tensor.QTensor):
    w = rhs.qvalue
    be.check_operand(w, 'rhs', be._FP8)  # pylint: disable=protected-access
  else:
    w = rhs
    be.check_operand(w, 'rhs')
    if lhs.dtype != w.dtype:
      raise TypeError(f'Unmatched lhs and rhs dtype: {lhs.dtype} vs {w.dtype}')
  if lhs.device != w.device:
    be.check_same_device(lhs, w)
  if w.ndim != 2:
    raise NotImplementedError(f'rhs is a matrix (got {tuple(w.shape)})')
  la, ra = lca[0], rca[0]
  nd = lhs.ndim
  if not -nd <= la < nd or not -2 <= ra < 2:
    raise ValueError(f'contracted axes out of range: {dimension_numbers}')
  la, ra = la % nd - nd, ra % 2 - 2
  if la != -1 and nd != 2:
    raise NotImplementedError(
        'lhs is contracted over its last axis (or is a matrix)')
  if lhs.shape[la] != w.shape[ra]:
    raise ValueError(f'contracted extents differ: {tuple(lhs.shape)} axis {la}, '
                     f'{tuple(w.shape)} axis {ra}')
  return la, ra


def _as_matrix(x, axis):
  """x as [rows, contraction], without a copy where its strides allow it."""
  if axis == -2:
    return x.transpose(0, 1)
  if x.ndim == 2:
    return x
  if x.ndim == 1:
    return x.view(1, -1)
  rows = 1
  for n in x.shape[:-1]:
    rows *= n
  y = x.reshape(rows, x.shape[-1])
  if y.numel() and y.data_ptr() != x.data_ptr() and be.tracing():
    raise _lib.AqtB200Error(
        'a traced step cannot copy an operand into another layout; make it '
        'contiguous first')
  return y
