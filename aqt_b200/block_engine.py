"""Host side of the block-scaled and grouped products: checks, layouts, buffers.

Turns torch CUDA tensors into calls of aqtb200_block_quantize and
aqtb200_grouped_gemm (include/aqt_b200.h). Everything here only enqueues on the
current stream of the operands' device; group sizes stay on the device and are
never read by the host. The user-facing objects are in
aqt_b200/v2/block_scaled.py and aqt_b200/v2/aqt_ragged_dot.py.

Layouts (contraction index contiguous, rows padded to 16 bytes, as for every
quantized operand of this library; scales with the kept index contiguous):

  Blocks(x [R, C])  row   q [R][ld], scale [C/128][R]     blocks along C
                    col   q [C][ld], scale [R/128][C]     blocks along R
                    square: both orders of q, ONE scale [R/128][C/128]
"""

from __future__ import annotations

import contextlib
import ctypes as C
import dataclasses
from typing import Any

import torch

from aqt_b200 import _lib
from aqt_b200 import engine
from aqt_b200.v2 import utils

BLOCK = 128
_FLOATS = (torch.float32, torch.bfloat16)
_FP8 = (torch.float8_e4m3fn, torch.float8_e5m2)
_NULL_CONTEXT = contextlib.nullcontext()


def fp8_dtype(bits) -> torch.dtype:
  """'e4m3' / 'e5m2' (or the dtype itself) -> torch dtype."""
  table = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}
  if bits in table:
    return table[bits]
  if isinstance(bits, torch.dtype) and bits in _FP8:
    return bits
  raise NotImplementedError(
      f'block-scaled operands are e4m3 or e5m2 (got {bits!r})')


def on_device_of(x):
  """Makes x's device the current one for the calls inside."""
  if not x.is_cuda or x.device.index == torch.cuda.current_device():
    return _NULL_CONTEXT
  return torch.cuda.device(x.device)


def check_operand(x, name, dtypes=_FLOATS):
  if not isinstance(x, torch.Tensor):
    raise TypeError(f'{name} must be a torch tensor (got {type(x).__name__})')
  if not engine._on_device(x):  # pylint: disable=protected-access
    raise _lib.AqtB200Error(f'{name} must be a CUDA tensor (no CPU path)')
  if x.dtype == torch.float16 and x.dtype not in dtypes:
    engine._code(x.dtype)  # raises with the reason  pylint: disable=protected-access
  if x.dtype not in dtypes:
    raise NotImplementedError(
        f'{name} has dtype {x.dtype}; handled here: '
        + ', '.join(str(d) for d in dtypes))


def check_same_device(*tensors):
  first = tensors[0].device
  for t in tensors[1:]:
    if t.device != first:
      raise ValueError(f'operands on different devices: {first}, {t.device}')


def check_group_sizes(group_sizes, groups):
  check_operand(group_sizes, 'group_sizes', (torch.int32, torch.int64))
  if group_sizes.ndim != 1 or group_sizes.shape[0] != groups:
    raise ValueError(
        f'group_sizes has shape {tuple(group_sizes.shape)}; one size for each '
        f'of the {groups} matrices of rhs is wanted')
  if not group_sizes.is_contiguous():
    raise ValueError('group_sizes must be contiguous')
  if not 1 <= groups <= _lib.MAX_GROUPS:
    raise NotImplementedError(
        f'between 1 and {_lib.MAX_GROUPS} groups (got {groups})')


def _up(v, m):
  return (v + m - 1) // m * m


def _cdiv(a, b):
  return -(-a // b)


@dataclasses.dataclass(slots=True)
class Blocks:
  """One operand quantized in blocks (see the module docstring)."""
  rows: int
  cols: int
  dtype: torch.dtype
  square: bool = False
  row: Any = None
  row_scale: Any = None
  col: Any = None
  col_scale: Any = None
  groups: int = 0  # matrices [groups][...]; 0: a single one

  def tensors(self):
    return [t for t in (self.row, self.row_scale, self.col, self.col_scale)
            if t is not None]


def quantize(x, dtype, *, row=True, col=False, square=False, po2=False,
             group_sizes=None) -> Blocks:
  """Quantizes a matrix [R, C] or matrices [G, R, C] in blocks of 128."""
  dev = x.device
  batch = x.shape[0] if x.ndim == 3 else 1
  r, c = x.shape[-2:]
  bs = x.stride(0) if x.ndim == 3 else 0
  rs, cs = x.stride(-2), x.stride(-1)
  # A transposed view is read the way it lies in memory: its rows are then the
  # columns of the call, and the two outputs change places.
  swap = cs != 1 and rs == 1 and group_sizes is None
  if swap:
    r, c, rs, cs, row, col = c, r, cs, rs, col, row
  lead = (batch,) if x.ndim == 3 else ()
  nr, nc = _cdiv(r, BLOCK), _cdiv(c, BLOCK)
  out = Blocks(x.shape[-2], x.shape[-1], dtype, square,
               groups=batch if x.ndim == 3 else 0)
  empty = engine._empty  # pylint: disable=protected-access
  q_row = q_col = s_row = s_col = None
  ld_row, ld_col = _up(c, 16), _up(r, 16)
  row_blocks = nr
  if group_sizes is not None:
    # every group may end in a partial block
    row_blocks = r // BLOCK + min(group_sizes.shape[0], r)
    ld_col = row_blocks * BLOCK
  if row:
    q_row = empty((*lead, r, ld_row), torch.uint8, dev)
    if not square:
      s_row = empty((*lead, nc, r), torch.float32, dev)
  if col:
    q_col = empty((*lead, c, ld_col), torch.uint8, dev)
    if not square:
      s_col = empty((*lead, row_blocks, c), torch.float32, dev)
  if square:
    s_row = empty((*lead, nr, nc), torch.float32, dev)
  ptr = lambda t: None if t is None else t.data_ptr()
  desc = _lib.BlockQuantDesc(
      _lib.View(x.data_ptr(), engine._TORCH_CODE[x.dtype], 0, batch, 1, r, c,  # pylint: disable=protected-access
                bs, 0, rs, cs),
      engine._TORCH_CODE[dtype], int(po2), int(square),  # pylint: disable=protected-access
      int(group_sizes is not None and group_sizes.dtype == torch.int64),
      ptr(q_row), ld_row, ptr(s_row), ptr(q_col), ld_col, ptr(s_col),
      ptr(group_sizes), 0 if group_sizes is None else group_sizes.shape[0])
  _lib.check(engine._call(  # pylint: disable=protected-access
      _lib.load().aqtb200_block_quantize, C.byref(desc), engine._stream()),  # pylint: disable=protected-access
             'block_quantize')
  if swap:
    q_row, q_col = q_col, q_row
    if square:
      s_row = s_row.transpose(-1, -2)
    else:
      s_row, s_col = s_col, s_row
  out.row, out.row_scale, out.col, out.col_scale = q_row, s_row, q_col, s_col
  if square:
    out.col_scale = s_row
  return out


def _gemm(desc, device, what):
  lib = _lib.load()
  nbytes = lib.aqtb200_grouped_gemm_workspace_bytes(C.byref(desc))
  if nbytes:
    ws = engine._empty((nbytes,), torch.uint8, device)  # pylint: disable=protected-access
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), nbytes
  _lib.check(engine._call(  # pylint: disable=protected-access
      lib.aqtb200_grouped_gemm, C.byref(desc),
      engine._status_buf(device).data_ptr(), engine._stream()), what)  # pylint: disable=protected-access


def _sizes(desc, group_sizes):
  if group_sizes is not None:
    desc.group_sizes = group_sizes.data_ptr()
    desc.groups = group_sizes.shape[0]
    desc.sizes_int64 = int(group_sizes.dtype == torch.int64)


def _empty_out(shape, dtype, device):
  return engine._empty(shape, dtype, device)  # pylint: disable=protected-access


def fp8_rows(tokens, tokens_scale, t, a, a_dtype, a_scale, r, k, b_dtype,
             out_dtype, group_sizes=None):
  """out[t][r] = sum_k b[t][k] a[g(t)][r][k], both block-scaled.

  tokens: q [T][ld] with scale [k/128][T]; a: q [.., R][ld] with the square
  scale given as a [.., R/128, k/128]-shaped view.
  """
  dev = tokens.device
  out = _empty_out((t, r), out_dtype, dev)
  code = engine._TORCH_CODE  # pylint: disable=protected-access
  d = _lib.GroupedGemmDesc(
      0, code[a_dtype], code[b_dtype], code[out_dtype], r, t, k, t,
      a.data_ptr(), a.stride(-2), a.stride(0) if a.ndim == 3 else 0,
      tokens.data_ptr(), tokens.stride(0), 0, 0, 1, 0,
      a_scale.data_ptr(), a_scale.stride(0) if a_scale.ndim == 3 else 0,
      a_scale.stride(-1), a_scale.stride(-2),
      tokens_scale.data_ptr(), tokens_scale.stride(0), None, 0,
      out.data_ptr(), r, 0, None, 0)
  _sizes(d, group_sizes)
  _gemm(d, dev, 'block-scaled product')
  return out


def fp8_contract_rows(b, b_scale, t, a, a_scale, r, k, rows, a_dtype, b_dtype,
                      out_dtype, group_sizes=None):
  """out[g][t][r] = sum over the rows of group g: both operands are the
  transposed ("col") copies, blocks along the rows."""
  dev = b.device
  lead = () if group_sizes is None else (group_sizes.shape[0],)
  out = _empty_out((*lead, t, r), out_dtype, dev)
  code = engine._TORCH_CODE  # pylint: disable=protected-access
  d = _lib.GroupedGemmDesc(
      1, code[a_dtype], code[b_dtype], code[out_dtype], r, t, k, rows,
      a.data_ptr(), a.stride(0), 0, b.data_ptr(), b.stride(0), 0, 0, 0, 0,
      a_scale.data_ptr(), 0, a_scale.stride(0), 1,
      b_scale.data_ptr(), b_scale.stride(0), None, 0,
      out.data_ptr(), r, t * r, None, 0)
  _sizes(d, group_sizes)
  _gemm(d, dev, 'block-scaled product')
  return out


def _fits(x, contiguous_axis, other_axis):
  """Whether a tensor map can describe x with that axis contiguous."""
  if x.numel() == 0:
    return False
  if x.stride(contiguous_axis) != 1 and x.shape[contiguous_axis] > 1:
    return False
  if x.data_ptr() % 16:
    return False
  strides = [x.stride(other_axis)] if x.shape[other_axis] > 1 else []
  if x.ndim == 3 and x.shape[0] > 1:
    strides.append(x.stride(0))
  return all(s > 0 and s % 8 == 0 for s in strides)


def pack(x):
  """A copy of bf16 [.., R, C] with C contiguous and rows padded to 16 bytes."""
  ld = _up(max(x.shape[-1], 1), 8)
  batch = x.shape[0] if x.ndim == 3 else 1
  buf = _empty_out((*x.shape[:-1], ld), torch.bfloat16, x.device)
  v = _lib.View(x.data_ptr(), _lib.BF16, 0, batch, 1, x.shape[-2], x.shape[-1],
                x.stride(0) if x.ndim == 3 else 0, 0, x.stride(-2), x.stride(-1))
  _lib.check(engine._call(  # pylint: disable=protected-access
      _lib.load().aqtb200_pack_bf16, C.byref(v), buf.data_ptr(), ld,
      engine._stream()), 'pack_bf16')  # pylint: disable=protected-access
  return buf[..., :x.shape[-1]]


def rows_for_tma(x):
  """x [.., R, C] bf16 itself, or a packed copy, with C contiguous."""
  return x if _fits(x, -1, -2) else pack(x)


def _ld(x, axis):
  """Stride of `axis`, made a valid one where the axis has a single entry."""
  return x.stride(axis) if x.shape[axis] > 1 else _up(max(x.shape[-1], x.shape[-2]), 8)


def bf16_rows(tokens, a, contract_axis, group_sizes, out_dtype):
  """out[t] = tokens[t] . a[g(t)], contracting a's `contract_axis` (1 or 2)."""
  t, k = tokens.shape
  keep = 3 - contract_axis
  r = a.shape[keep]
  dev = tokens.device
  out = _empty_out((t, r), out_dtype, dev)
  tokens = rows_for_tma(tokens)
  if _fits(a, contract_axis, keep):
    mn, ld = 0, _ld(a, keep)
  elif _fits(a, keep, contract_axis):
    mn, ld = 1, _ld(a, contract_axis)
  else:
    a = pack(a)  # its last axis is contiguous
    mn, ld = int(contract_axis == 1), a.stride(1)
  d = _lib.GroupedGemmDesc(
      0, _lib.BF16, _lib.BF16, engine._TORCH_CODE[out_dtype], r, t, k, t,  # pylint: disable=protected-access
      a.data_ptr(), ld, a.stride(0), tokens.data_ptr(), _ld(tokens, 0), mn, 0,
      0, 0, None, 0, 0, 0, None, 0, None, 0, out.data_ptr(), r, 0, None, 0)
  _sizes(d, group_sizes)
  _gemm(d, dev, 'grouped product')
  return out


def bf16_contract_rows(lhs, g, group_sizes, out_dtype):
  """out[e] = lhs_e^T . g_e for the rows of every group e."""
  rows, t = lhs.shape
  r = g.shape[1]
  dev = lhs.device
  out = _empty_out((group_sizes.shape[0], t, r), out_dtype, dev)
  lhs, g = rows_for_tma(lhs), rows_for_tma(g)
  d = _lib.GroupedGemmDesc(
      1, _lib.BF16, _lib.BF16, engine._TORCH_CODE[out_dtype], r, t, rows, rows,  # pylint: disable=protected-access
      g.data_ptr(), _ld(g, 0), 0, lhs.data_ptr(), _ld(lhs, 0), 1, 1, 0, 0,
      None, 0, 0, 0, None, 0, None, 0, out.data_ptr(), r, t * r, None, 0)
  _sizes(d, group_sizes)
  _gemm(d, dev, 'grouped product')
  return out


class Residuals:
  """Buffers a backward pass reads. They are torch allocations of the forward
  pass's stream; used on another one, the allocator is told before they can be
  handed out again."""

  __slots__ = ('stream', 'tensors')

  def __init__(self, tensors, like):
    self.tensors = [t for t in tensors if t is not None]
    self.stream = torch.cuda.current_stream(like.device) if like.is_cuda else None

  def about_to_use(self):
    if self.stream is None:
      return
    now = torch.cuda.current_stream(self.stream.device)
    if now != self.stream:
      for t in self.tensors:
        t.record_stream(now)


def float_name(dtype):
  return utils.as_dtype(dtype).name
