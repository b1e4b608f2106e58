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

Row and col scales come with notes on their range (aqtb200_block_quantize's note_row,
note_col), by which the products find those that f32 has to be careful with.

The calls here are short next to their kernels' launches, so what a product
needs between its kernels is one torch allocation, addressed by offsets, and
operands travel as (address, stride) numbers rather than as tensor views.
"""

from __future__ import annotations

import contextlib
import ctypes as C

import torch
from torch.autograd import forward_ad

from aqt_b200 import _lib
from aqt_b200 import engine

BLOCK = 128
_FLOATS = (torch.float32, torch.bfloat16)
_FP8 = (torch.float8_e4m3fn, torch.float8_e5m2)
_NULL_CONTEXT = contextlib.nullcontext()
_NO_NOTES = ()
_AD_LEVEL = hasattr(forward_ad, '_current_level')


def fp8_dtype(bits) -> torch.dtype:
  """'e4m3' / 'e5m2' (or the dtype itself) -> torch dtype."""
  table = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}
  if bits in table:
    return table[bits]
  if isinstance(bits, torch.dtype) and bits in _FP8:
    return bits
  raise NotImplementedError(
      f'block-scaled operands are e4m3 or e5m2 (got {bits!r})')


def tracing():
  """Whether an engine.TracedStep is recording."""
  return engine._tape is not None  # pylint: disable=protected-access


def on_device_of(x):
  """Makes x's device the current one for the calls inside."""
  if not x.is_cuda or x.device.index == torch.cuda.current_device():
    return _NULL_CONTEXT
  return torch.cuda.device(x.device)


def check_operand(x, name, dtypes=_FLOATS):
  if not isinstance(x, torch.Tensor):
    raise TypeError(f'{name} must be a torch tensor (got {type(x).__name__})')
  if not (x.is_cuda or engine._on_device(x)):  # pylint: disable=protected-access
    raise _lib.AqtB200Error(f'{name} must be a CUDA tensor (no CPU path)')
  if x.dtype == torch.float16 and x.dtype not in dtypes:
    engine._code(x.dtype)  # raises with the reason  pylint: disable=protected-access
  if x.dtype not in dtypes:
    raise NotImplementedError(
        f'{name} has dtype {x.dtype}; handled here: '
        + ', '.join(str(d) for d in dtypes))
  # (torch's note of the open level first: unpacking takes longer than these checks)
  if ((not _AD_LEVEL or forward_ad._current_level >= 0) and  # pylint: disable=protected-access
      forward_ad.unpack_dual(x).tangent is not None):
    raise NotImplementedError(
        f'{name} carries a forward-mode tangent; these products have gradients '
        '(backward) only')


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


class Side:
  """One operand of a product: values with the contraction contiguous and their
  scales, as addresses and strides. `keep` holds the memory."""
  __slots__ = ('ptr', 'ld', 'group', 'code', 'scale', 'scale_group', 'scale_k',
               'scale_r', 'kept', 'keep', 'note')

  def __init__(self, ptr, ld, group, code, scale, scale_group, scale_k, scale_r,
               kept, keep, note=_NO_NOTES):
    self.ptr, self.ld, self.group, self.code = ptr, ld, group, code
    self.scale, self.scale_group = scale, scale_group
    self.scale_k, self.scale_r = scale_k, scale_r
    self.kept, self.keep = kept, keep
    self.note = note  # address, strides of a block of k and of 128 kept, padded

  def at(self, base, memory):
    """This operand with its memory, once at `base`, in `memory` (or in none)."""
    shift = 0 if memory is None else memory.data_ptr() - base
    return Side(self.ptr + shift, self.ld, self.group, self.code,
                self.scale + shift, self.scale_group, self.scale_k, self.scale_r,
                self.kept, memory, self.note and (self.note[0] + shift, *self.note[1:]))




def _scratch(nbytes, device):
  t = torch.empty(nbytes, dtype=torch.uint8, device=device)
  if engine._tape is not None:  # pylint: disable=protected-access
    engine._tape.keep.append(t)  # pylint: disable=protected-access
  return t


def quantize(x, dtype, row=True, col=False, square=False, po2=False,
             group_sizes=None):
  """Quantizes a matrix [R, C] or matrices [G, R, C] in blocks of 128.

  Returns (row, col) Sides: the first contracts C, the second contracts R; None
  where not asked for.
  """
  code = engine._TORCH_CODE  # pylint: disable=protected-access
  shape, strides = x.shape, x.stride()
  if x.ndim == 3:
    batch, r, c = shape
    bs, rs, cs = strides
  else:
    r, c = shape
    rs, cs = strides
    batch, bs = 1, 0
  # A transposed view is read the way it lies in memory: its rows are then the
  # columns of the call, and the two outputs change places.
  swap = cs != 1 and rs == 1 and group_sizes is None
  if swap:
    r, c, rs, cs, row, col = c, r, cs, rs, col, row
  nr, nc = -(-r // BLOCK), -(-c // BLOCK)
  ld_row = ld_col = groups = int64 = sizes_ptr = 0
  row_blocks = nr
  if group_sizes is not None:
    # every group may end in a partial block
    groups = group_sizes.shape[0]
    row_blocks = r // BLOCK + min(groups, r)
    int64 = int(group_sizes.dtype == torch.int64)
    sizes_ptr = group_sizes.data_ptr()
  at_q_row = at_s_row = at_q_col = at_s_col = at_n_row = at_n_col = end = 0
  if row:
    ld_row = (c + 15) & -16
    end = (batch * r * ld_row + 255) & -256
  if square:
    at_s_row = end
    end += (batch * nr * nc * 4 + 255) & -256
  elif row:
    at_s_row = end
    end += (batch * nc * r * 4 + 255) & -256
  if col:
    at_q_col = end
    ld_col = (r + 15) & -16 if group_sizes is None else row_blocks * BLOCK
    end += (batch * c * ld_col + 255) & -256
    if not square:
      at_s_col = end
      end += (batch * row_blocks * c * 4 + 255) & -256
  notes = not square and batch == 1
  if notes:
    nbytes = (row_blocks * nc * 16 + 255) & -256
    if row:
      at_n_row = end
      end += nbytes
    if col:
      at_n_col = end
      end += nbytes
  ws = _scratch(end, x.device)
  base = ws.data_ptr()
  desc = _lib.BlockQuantDesc(
      _lib.View(x.data_ptr(), code[x.dtype], 0, batch, 1, r, c, bs, 0, rs, cs),
      code[dtype], po2, square, int64,
      base + at_q_row if row else None, ld_row,
      base + at_s_row if row or square else None,
      base + at_q_col if col else None, ld_col,
      base + at_s_col if col and not square else None, sizes_ptr, groups,
      base + at_n_row if notes and row else None,
      base + at_n_col if notes and col else None)
  _run('block_quantize', _lib.load().aqtb200_block_quantize, C.byref(desc),
       engine._stream())  # pylint: disable=protected-access
  q = code[dtype]
  a = b = None
  if row:
    s = ((base + at_s_row, nr * nc, 1, nc) if square else
         (base + at_s_row, nc * r, r, 1))
    a = Side(base + at_q_row, ld_row, r * ld_row, q, *s, r, ws,
             (base + at_n_row, 1, nc, sizes_ptr != 0) if notes else _NO_NOTES)
  if col:
    s = ((base + at_s_row, nr * nc, nc, 1) if square else
         (base + at_s_col, row_blocks * c, c, 1))
    b = Side(base + at_q_col, ld_col, c * ld_col, q, *s, c, ws,
             (base + at_n_col, nc, 1, 0) if notes else _NO_NOTES)
  return (b, a) if swap else (a, b)


def quantize_tensors(x, dtype, axis, square, po2):
  """Quantizes x for one contraction axis (-1 or -2) into tensors of their own:
  (values of x's shape, scales as the QTensor's user sees them)."""
  code = engine._TORCH_CODE  # pylint: disable=protected-access
  empty = engine._empty  # pylint: disable=protected-access
  lead, (r, c) = tuple(x.shape[:-2]), x.shape[-2:]
  batch, bs = (lead[0], x.stride(0)) if lead else (1, 0)
  rs, cs = x.stride(-2), x.stride(-1)
  row = axis == -1
  swap = cs != 1 and rs == 1
  if swap:
    r, c, rs, cs, row = c, r, cs, rs, not row
  nr, nc = -(-r // BLOCK), -(-c // BLOCK)
  kept, contracted = (r, c) if row else (c, r)
  ld = (contracted + 15) & -16
  if ld == contracted:
    q = view = empty((*lead, kept, ld), dtype, x.device)
  else:
    q = empty((*lead, kept, ld), torch.uint8, x.device)
    view = q[..., :contracted].view(dtype)
  if square:
    s = empty((*lead, nr, nc), torch.float32, x.device)
  else:
    s = empty((*lead, nc, r) if row else (*lead, nr, c), torch.float32, x.device)
  qp, sp = q.data_ptr(), s.data_ptr()
  desc = _lib.BlockQuantDesc(
      _lib.View(x.data_ptr(), code[x.dtype], 0, batch, 1, r, c, bs, 0, rs, cs),
      code[dtype], po2, square, 0, qp if row else None, ld,
      sp if row or square else None, None if row else qp, ld,
      None if row or square else sp, None, 0)
  _run('block_quantize', _lib.load().aqtb200_block_quantize, C.byref(desc),
       engine._stream())  # pylint: disable=protected-access
  # back to x's axes: values lie [kept][contracted], row scales [block][kept]
  if axis == -2:
    view = view.transpose(-1, -2)
  if square:
    s = s.transpose(-1, -2) if swap else s
  elif row != swap:
    s = s.transpose(-1, -2) if axis == -1 else s
  else:
    s = s if axis == -2 else s.transpose(-1, -2)
  return view, s


def _run(what, fn, *args):
  """engine._call and the check of its answer, in one frame."""
  rc = fn(*args)
  if engine._tape is not None:  # pylint: disable=protected-access
    engine._tape.ops.append((fn, args))  # pylint: disable=protected-access
  if rc:
    _lib.check(rc, what)


def _gemm(desc, device, what):
  # a product of an earlier call that gave up is reported by the next one
  words = engine._words.get(device) or engine.status_words(device)  # pylint: disable=protected-access
  if words[0]:
    engine.poll_words(words)
  _run(what, _lib.load().aqtb200_grouped_gemm, C.byref(desc), words.address,
       engine._stream())  # pylint: disable=protected-access


def _sizes(group_sizes):
  """(address, number, whether int64) for a descriptor."""
  if group_sizes is None:
    return None, 0, 0
  return (group_sizes.data_ptr(), group_sizes.shape[0],
          int(group_sizes.dtype == torch.int64))


def _empty_out(shape, dtype, device):
  return engine._empty(shape, dtype, device)  # pylint: disable=protected-access


def fp8_rows(tokens, a, k, out_dtype, device, group_sizes=None, po2=False):
  """out[t][r] = sum_k tokens[t][k] a[g(t)][r][k]; a has 128 x 128 blocks. The
  call before this one has to be the one that quantized the tokens. po2: all
  scales are powers of two."""
  t, r = tokens.kept, a.kept
  out = _empty_out((t, r), out_dtype, device)
  sizes, groups, int64 = _sizes(group_sizes)
  _gemm(_lib.GroupedGemmDesc(
      0, a.code, tokens.code, engine._TORCH_CODE[out_dtype], r, t, k, t,  # pylint: disable=protected-access
      a.ptr, a.ld, a.group, tokens.ptr, tokens.ld, 0, 0, 1, int64, po2, 1,
      a.scale, a.scale_group, a.scale_k, a.scale_r,
      tokens.scale, tokens.scale_k, sizes, groups,
      out.data_ptr(), r, 0, None, 0, *tokens.note), device, 'block-scaled product')
  return out


def fp8_contract_rows(b, a, k, rows, out_dtype, device, group_sizes=None,
                      po2=False):
  """out[g][t][r] = sum over the rows of group g: both operands are the
  transposed ("col") copies, blocks along the rows."""
  t, r = b.kept, a.kept
  lead = () if group_sizes is None else (group_sizes.shape[0],)
  out = _empty_out((*lead, t, r), out_dtype, device)
  sizes, groups, int64 = _sizes(group_sizes)
  _gemm(_lib.GroupedGemmDesc(
      1, a.code, b.code, engine._TORCH_CODE[out_dtype], r, t, k, rows,  # pylint: disable=protected-access
      a.ptr, a.ld, 0, b.ptr, b.ld, 0, 0, 0, int64, po2, 0,
      a.scale, 0, a.scale_k, 1, b.scale, b.scale_k, sizes, groups,
      out.data_ptr(), r, t * r, None, 0, *a.note), device, 'block-scaled product')
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


def pack(x, group_sizes=None):
  """A copy of bf16 [.., R, C] with C contiguous and rows padded to 16 bytes;
  given the sizes of x's groups, of those matrices only whose group has rows."""
  ld = (max(x.shape[-1], 1) + 7) & -8
  batch = x.shape[0] if x.ndim == 3 else 1
  buf = _empty_out((*x.shape[:-1], ld), torch.bfloat16, x.device)
  v = _lib.View(x.data_ptr(), _lib.BF16, 0, batch, 1, x.shape[-2], x.shape[-1],
                x.stride(0) if x.ndim == 3 else 0, 0, x.stride(-2), x.stride(-1))
  sizes, _, int64 = _sizes(group_sizes)
  _run('pack_bf16', _lib.load().aqtb200_pack_bf16_groups, C.byref(v), sizes, int64,
       buf.data_ptr(), ld, engine._stream())  # pylint: disable=protected-access
  return buf[..., :x.shape[-1]]


def as_bf16(x):
  """x itself, or rounded to bfloat16: torch's work, which a traced step has to
  be told of, into memory it holds."""
  if x.dtype == torch.bfloat16:
    return x
  out = _empty_out(x.shape, torch.bfloat16, x.device)
  engine.tape_op(lambda: out.copy_(x))
  return out


def padded_rows(q):
  """A copy of fp8 [.., R, C] with C contiguous and rows of whole 16 bytes."""
  n = q.shape[-1]
  buf = _empty_out((*q.shape[:-1], (n + 15) & -16), torch.uint8, q.device)
  q8, rows = q.view(torch.uint8), buf[..., :n]
  engine.tape_op(lambda: (buf.zero_(), rows.copy_(q8)))
  return rows.view(q.dtype)


def rows_for_tma(x):
  """x [.., R, C] bf16 itself, or a packed copy, with C contiguous."""
  return x if _fits(x, -1, -2) else pack(x)


def matrices_for_tma(x, group_sizes):
  """x [G, R, C] bf16 itself, if a tensor map can describe it with either of the
  last axes contiguous, or a packed copy."""
  return x if _fits(x, -1, -2) or _fits(x, -2, -1) else pack(x, group_sizes)


def _ld(x, axis):
  """Stride of `axis`, made a valid one where the axis has a single entry."""
  return x.stride(axis) if x.shape[axis] > 1 else (max(x.shape[-1], x.shape[-2]) + 7) & -8


def bf16_rows(tokens, a, contract_axis, group_sizes, out_dtype):
  """out[t] = tokens[t] . a[g(t)], contracting a's `contract_axis` (1 or 2);
  tokens from rows_for_tma, a from matrices_for_tma."""
  t, k = tokens.shape
  keep = 3 - contract_axis
  r = a.shape[keep]
  dev = tokens.device
  out = _empty_out((t, r), out_dtype, dev)
  if _fits(a, contract_axis, keep):
    mn, ld = 0, _ld(a, keep)
  else:
    mn, ld = 1, _ld(a, contract_axis)
  sizes, groups, int64 = _sizes(group_sizes)
  _gemm(_lib.GroupedGemmDesc(
      0, _lib.BF16, _lib.BF16, engine._TORCH_CODE[out_dtype], r, t, k, t,  # pylint: disable=protected-access
      a.data_ptr(), ld, a.stride(0), tokens.data_ptr(), _ld(tokens, 0), mn, 0,
      0, int64, 0, 0, None, 0, 0, 0, None, 0, sizes, groups, out.data_ptr(), r, 0,
      None, 0), dev, 'grouped product')
  return out


def bf16_contract_rows(lhs, g, group_sizes, out_dtype):
  """out[e] = lhs_e^T . g_e for the rows of every group e; both from
  rows_for_tma."""
  rows, t = lhs.shape
  r = g.shape[1]
  dev = lhs.device
  out = _empty_out((group_sizes.shape[0], t, r), out_dtype, dev)
  sizes, groups, int64 = _sizes(group_sizes)
  d = _lib.GroupedGemmDesc(
      1, _lib.BF16, _lib.BF16, engine._TORCH_CODE[out_dtype], r, t, rows, rows,  # pylint: disable=protected-access
      g.data_ptr(), _ld(g, 0), 0, lhs.data_ptr(), _ld(lhs, 0), 1, 1, 0, int64, 0, 0,
      None, 0, 0, 0, None, 0, sizes, groups, out.data_ptr(), r, t * r, None, 0)
  # room for the groups' last, partial slabs
  nbytes = _lib.load().aqtb200_grouped_gemm_workspace_bytes(C.byref(d))
  if nbytes:
    ws = _scratch(nbytes, dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), nbytes
  _gemm(d, dev, 'grouped product')
  return out


class Residuals:
  """The operands a backward pass reads: Sides, tensors or None.

  Their memory is torch allocations of the forward pass's stream; used on
  another one, the allocator is told before it can be handed out again. On
  torch's tape the graph keeps it, not this object: release() hands it out for
  save_for_backward, and regain() takes what the graph gives back, which hooks may
  have moved.
  """

  __slots__ = ('lhs', 'rhs', 'stream', 'memory', 'base')

  def __init__(self, lhs, rhs):
    self.lhs, self.rhs = lhs, rhs
    self.stream = engine._stream()  # pylint: disable=protected-access
    self.memory = (lhs.keep if isinstance(lhs, Side) else lhs,
                   rhs.keep if isinstance(rhs, Side) else rhs)

  def about_to_use(self):
    """Called with the operands' device current."""
    if engine._stream() != self.stream:  # pylint: disable=protected-access
      for t in self.memory:
        if t is not None and t.is_cuda:
          t.record_stream(torch.cuda.current_stream())

  def release(self):
    memory, self.memory = self.memory, None
    self.base = tuple([t if t is None else t.data_ptr() for t in memory])
    if isinstance(self.lhs, Side):
      self.lhs.keep = None
    else:
      self.lhs = None
    if isinstance(self.rhs, Side):
      self.rhs.keep = None
    else:
      self.rhs = None
    return memory

  def regain(self, lhs, rhs):
    r = object.__new__(Residuals)
    r.stream, r.memory = self.stream, (lhs, rhs)
    r.lhs = _regain(self.lhs, self.base[0], lhs)
    r.rhs = _regain(self.rhs, self.base[1], rhs)
    return r


def _regain(side, base, t):
  if side is None or t is None:
    return t
  if t.data_ptr() == base:
    return side
  if t.data_ptr() % 256 or not t.is_contiguous():
    t = t.clone(memory_format=torch.contiguous_format)  # aligned as at first
  return side.at(base, t)
