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
and added in f32, and the result is rounded once to the output's dtype. A NaN or
an infinity in a block makes that block's scale, and what is computed from it,
NaN or infinite, as absmax calibration does (calibration.py:117-157).
"""

from __future__ import annotations

import dataclasses
from typing import Any

import torch

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
    b = be.quantize(x, dtype, row=axis == -1, col=axis == -2, square=square,
                    po2=po2_scale)
  if axis == -1:
    q = b.row[..., :x.shape[-1]].view(dtype)
    s = b.row_scale if square else b.row_scale.transpose(-1, -2)
  else:
    q = b.col[..., :x.shape[-2]].view(dtype).transpose(-1, -2)
    s = b.col_scale
  return aqt_tensor.QTensor(
      qvalue=q, scale=[s], scale_t=None, dequant_dtype=utils.as_dtype(x.dtype),
      tiling_state=BlockTiling(axis, square))


def frozen(qvalue, scale, contract_axis: int = -2) -> aqt_tensor.QTensor:
  """A QTensor of weights quantized in 128 x 128 blocks, from a checkpoint's
  values [K, N] or [G, K, N] and scales [.., ceil(K/128), ceil(N/128)].

  The product needs the contraction axis contiguous in memory; values that lie
  otherwise are copied once, here.
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
      ld = -(-v.shape[-1] // 16) * 16
      buf = torch.zeros(*v.shape[:-1], ld, dtype=torch.uint8, device=v.device)
      buf[..., :v.shape[-1]] = v.view(torch.uint8)
      v = buf[..., :v.shape[-1]].view(qvalue.dtype)
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
  """(values [.., R][ld] bytes, scale [.., R/128, K/128] view, dtype) of frozen
  weights for a product that contracts `contract_axis`."""
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
  if contract_axis == -2:
    q, s = q.transpose(-1, -2), s.transpose(-1, -2)
  return q, s, q.dtype


class _Step:
  """One forward product's operands, as its backward pass needs them."""

  __slots__ = ('lhs', 'rhs', 'keep', 'out_dtype', 'lhs_shape', 'rhs_axis')


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
    out_dtype = _out_dtype(preferred_element_type, lhs)
    dims = _dims(lhs, rhs, dimension_numbers)
    if isinstance(rhs, aqt_tensor.QTensor):
      if torch.is_grad_enabled() and lhs.requires_grad:
        raise NotImplementedError(
            'a product with frozen weights has no gradient; pass float weights')
      return self._forward(lhs, rhs, dims, out_dtype, None)[0]
    if torch.is_grad_enabled() and (lhs.requires_grad or rhs.requires_grad):
      return _BlockDot.apply(lhs, rhs, self, dims, out_dtype)
    return self._forward(lhs, rhs, dims, out_dtype, (False, False))[0]

  def vjp(self, lhs, rhs, dimension_numbers, preferred_element_type=None):
    """(out, backprop) with backprop(g) -> (dlhs, drhs)."""
    if isinstance(rhs, aqt_tensor.QTensor):
      raise NotImplementedError(
          'a product with frozen weights has no gradient; pass float weights')
    out_dtype = _out_dtype(preferred_element_type, lhs)
    dims = _dims(lhs, rhs, dimension_numbers)
    out, step = self._forward(lhs.detach(), rhs.detach(), dims, out_dtype,
                              (True, True))
    return out, lambda g: self._backward(step, g, (True, True))

  def _forward(self, lhs, rhs, dims, out_dtype, grads):
    lhs_axis, rhs_axis = dims
    x = _as_matrix(lhs, lhs_axis)
    m, k = x.shape
    with be.on_device_of(lhs):
      if grads is None:
        a, a_scale, a_dtype = _frozen_operand(rhs, rhs_axis)
        need_l = need_r = False
      else:
        need_l, need_r = grads
        w = be.quantize(rhs, self.fwd_dtype, row=rhs_axis == -1 or need_l,
                        col=rhs_axis == -2 or need_l, square=True,
                        po2=self.po2_scale)
        a, a_scale, a_dtype = _kept_major(w, rhs_axis)
      n = a.shape[-2]
      l = be.quantize(x, self.fwd_dtype, row=True, col=need_r,
                      po2=self.po2_scale)
      out = be.fp8_rows(l.row, l.row_scale, m, a, a_dtype, a_scale, n, k,
                        self.fwd_dtype, out_dtype)
    step = None
    if need_l or need_r:
      step = _Step()
      step.lhs = l if need_r else None
      step.rhs = w if need_l else None
      step.keep = be.Residuals(
          ([l.col, l.col_scale] if need_r else []) +
          (w.tensors() if need_l else []), lhs)
      step.lhs_shape, step.rhs_axis = (lhs.shape, lhs_axis, lhs.dtype), rhs_axis
      step.out_dtype = rhs.dtype
      if need_r:
        l.row = l.row_scale = None
    shape = lhs.shape[:-1] if lhs_axis == -1 else lhs.shape[-1:]
    return out.view(*shape, n), step

  def _backward(self, step, g, grads):
    need_l, need_r = grads
    n = g.shape[-1]
    lhs_shape, lhs_axis, lhs_dtype = step.lhs_shape
    be.check_operand(g, 'the cotangent')
    gm = _as_matrix(g, -1)
    m = gm.shape[0]
    step.keep.about_to_use()
    with be.on_device_of(g):
      q = be.quantize(gm, self.bwd_dtype, row=need_l, col=need_r,
                      po2=self.po2_scale)
      dlhs = drhs = None
      if need_l:
        # contracts the axis the forward pass kept
        keep_axis = -3 - step.rhs_axis
        a, a_scale, a_dtype = _kept_major(step.rhs, keep_axis)
        k = a.shape[-2]
        dlhs = be.fp8_rows(q.row, q.row_scale, m, a, a_dtype, a_scale, k, n,
                           self.bwd_dtype, lhs_dtype)
        dlhs = (dlhs.view(lhs_shape) if lhs_axis == -1 else
                dlhs.transpose(0, 1))
      if need_r:
        l = step.lhs
        k = l.cols
        if step.rhs_axis == -2:  # drhs [K, N]
          drhs = be.fp8_contract_rows(
              l.col, l.col_scale, k, q.col, q.col_scale, n, m, m,
              self.bwd_dtype, self.fwd_dtype, step.out_dtype)
        else:                    # drhs [N, K]
          drhs = be.fp8_contract_rows(
              q.col, q.col_scale, n, l.col, l.col_scale, k, m, m,
              self.fwd_dtype, self.bwd_dtype, step.out_dtype)
    return dlhs, drhs


def _kept_major(blocks, contract_axis):
  """Values [.., kept][contraction], square scale as [.., kept, contraction]."""
  if contract_axis == -1:
    return blocks.row[..., :blocks.cols], blocks.row_scale, blocks.dtype
  return (blocks.col[..., :blocks.rows], blocks.col_scale.transpose(-1, -2),
          blocks.dtype)


class _BlockDot(torch.autograd.Function):
  """The custom VJP (aqt_dot_general.py:993-997) on torch's tape."""

  @staticmethod
  def forward(ctx, lhs, rhs, cfg, dims, out_dtype):
    ctx.cfg = cfg
    out, ctx.step = cfg._forward(  # pylint: disable=protected-access
        lhs.detach(), rhs.detach(), dims, out_dtype, ctx.needs_input_grad[:2])
    return out

  @staticmethod
  def backward(ctx, g):
    dlhs, drhs = ctx.cfg._backward(  # pylint: disable=protected-access
        ctx.step, g, ctx.needs_input_grad[:2])
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
  if tuple(lba) or tuple(rba) or len(tuple(lca)) != 1 or len(tuple(rca)) != 1:
    raise NotImplementedError(
        'block-scaled products contract one axis of each operand and have no '
        f'batch axes (got {dimension_numbers})')
  be.check_operand(lhs, 'lhs')
  q = isinstance(rhs, aqt_tensor.QTensor)
  w = rhs.qvalue if q else rhs
  be.check_operand(w, 'rhs', be._FP8 if q else be._FLOATS)  # pylint: disable=protected-access
  be.check_same_device(lhs, w)
  if not q and lhs.dtype != rhs.dtype:
    raise TypeError(f'Unmatched lhs and rhs dtype: {lhs.dtype} vs {rhs.dtype}')
  if w.ndim != 2:
    raise NotImplementedError(f'rhs is a matrix (got {tuple(w.shape)})')
  la = int(tuple(lca)[0]) % max(lhs.ndim, 1) - lhs.ndim
  ra = int(tuple(rca)[0]) % 2 - 2
  if lhs.ndim < 1 or (la != -1 and lhs.ndim != 2):
    raise NotImplementedError(
        'lhs is contracted over its last axis (or is a matrix)')
  if lhs.shape[la] != w.shape[ra]:
    raise ValueError(f'contracted extents differ: {tuple(lhs.shape)} axis {la}, '
                     f'{tuple(w.shape)} axis {ra}')
  return la, ra


def _as_matrix(x, axis):
  """x as [rows, contraction] without a copy where its strides allow it."""
  if axis == -2:
    return x.transpose(0, 1)
  if x.ndim == 2:
    return x
  if x.ndim == 1:
    return x.view(1, -1)
  y = x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.new_empty(
      (x.numel() if x.ndim == 0 else _prod(x.shape[:-1]), 0))
  from aqt_b200 import engine
  if y.numel() and y.data_ptr() != x.data_ptr() and engine._tape is not None:  # pylint: disable=protected-access
    raise _lib.AqtB200Error(
        'a traced step cannot copy an operand into another layout; make it '
        'contiguous first')
  return y


def _prod(shape):
  n = 1
  for s in shape:
    n *= s
  return n
