"""tests/fake_lib.py with the block-scaled and grouped entry points: numpy on host
memory, from the semantics written in include/aqt_b200.h, in 64 bits.

TEST INFRASTRUCTURE, as its base is: it lets the CPU suite run what lies above
the C ABI (layouts, swapped operands, gradients, group handling).
"""

import ctypes as C

import numpy as np

from aqt_b200 import _lib
from tests import block_ref
from tests import fake_lib

_BITS = {_lib.E4M3: 'e4m3', _lib.E5M2: 'e5m2'}
_strided = fake_lib._strided  # pylint: disable=protected-access


def _sizes(ptr, groups, int64, rows):
  if not ptr:
    return None
  raw = (C.c_char * (groups * (8 if int64 else 4))).from_address(ptr)
  n = np.frombuffer(raw, np.int64 if int64 else np.int32)
  return block_ref.spans(n.tolist(), rows)



class FakeBlockLib(fake_lib.FakeLib):

  def aqtb200_block_quantize(self, desc, stream):
    del stream
    d = desc._obj
    v = d.x
    if not (v.b0 * v.b1 and v.rows and v.cols):
      return 0
    if v.dtype not in (_lib.F32, _lib.BF16) or d.qdtype not in _BITS:
      return self._fail(-2, 'dtype')
    x = fake_lib._view_array(v).reshape(v.b0 * v.b1, v.rows, v.cols).astype(  # pylint: disable=protected-access
        np.float32)
    bits = _BITS[d.qdtype]
    nr, nc = -(-v.rows // 128), -(-v.cols // 128)
    spans = _sizes(d.group_sizes, d.groups, d.sizes_int64, v.rows)
    for b in range(v.b0 * v.b1):
      if d.q_row:
        q, s = block_ref.quantize(x[b], 128 if d.square else 1, 128, bits,
                                  d.po2_scale)
        self._put(d.q_row + b * v.rows * d.ld_row, d.qdtype, q, d.ld_row, v.cols)
        if d.square:
          self._put32(d.scale_row + 4 * b * nr * nc, s)
        else:
          self._put32(d.scale_row + 4 * b * nc * v.rows, s.T)
      if d.q_col and spans is None:
        q, s = block_ref.quantize(x[b], 128, 128 if d.square else 1, bits,
                                  d.po2_scale)
        self._put(d.q_col + b * v.cols * d.ld_col, d.qdtype, q.T, d.ld_col, v.rows)
        if d.square:
          for p in (d.scale_row, d.scale_col):
            if p:
              self._put32(p + 4 * b * nr * nc, s)
        else:
          self._put32(d.scale_col + 4 * b * nr * v.cols, s)
      elif d.q_col:
        at = 0
        for begin, end in spans:
          blocks = -(-(end - begin) // 128)
          if not blocks:
            continue
          p = np.zeros((blocks * 128, v.cols), np.float32)
          p[:end - begin] = x[b, begin:end]
          q, s = block_ref.quantize(p, 128, 1, bits, d.po2_scale)
          self._put(d.q_col + at * 128, d.qdtype, q.T, d.ld_col, blocks * 128)
          self._put32(d.scale_col + 4 * at * v.cols, s)
          at += blocks
    return 0

  def _put(self, ptr, code, q, ld, width):
    _strided(ptr, code, [q.shape[0], width], [ld, 1], True)[...] = q

  def _put32(self, ptr, s):
    _strided(ptr, _lib.F32, [s.size], [1], True)[...] = s.reshape(-1)

  def aqtb200_grouped_gemm_workspace_bytes(self, desc):
    del desc
    return 0

  def aqtb200_grouped_gemm(self, desc, status, stream):
    del status, stream
    d = desc._obj
    if not (d.r and d.t):
      return 0
    rows = d.t if d.contract_groups == 0 else d.rows
    spans = _sizes(d.group_sizes, d.groups, d.sizes_int64, rows)
    fp8 = d.a_dtype in _BITS
    groups = d.groups if spans else 1

    def operand(ptr, code, kept, ld, mn, k, offset=0):
      es = 1 if fp8 else 2
      st = [1, ld] if mn else [ld, 1]
      return _strided(ptr + offset * es, code, [kept, k], st).astype(np.float64)

    def scales(ptr, kept, sk, sr, k, square, offset=0):
      nb = -(-k // 128)
      n = -(-kept // 128) if square else kept
      s = _strided(ptr + 4 * offset, _lib.F32, [n, nb], [sr, sk]).astype(np.float64)
      if square:
        s = np.repeat(s, 128, 0)[:kept]
      return np.repeat(s, 128, 1)[:, :k]

    def put(t0, value, group=0):
      es = 4 if d.out_dtype == _lib.F32 else 2
      out = _strided(d.out + es * (group * d.out_group_stride + t0 * d.out_ld),
                     d.out_dtype, value.shape, [d.out_ld, 1], True)
      out[...] = value.astype(np.float32).astype(out.dtype)

    b = operand(d.b, d.b_dtype, d.t, d.b_ld, d.b_mn_major, d.k)
    if fp8 and d.k:
      with np.errstate(invalid='ignore'):
        b = b * scales(d.b_scale, d.t, d.b_scale_k_stride, 1, d.k, False)
    if d.contract_groups == 0:
      at = 0
      for g, (begin, end) in enumerate(spans or [(0, d.t)]):
        a = operand(d.a, d.a_dtype, d.r, d.a_ld, d.a_mn_major, d.k,
                    g * d.a_group_stride)
        if fp8 and d.k:
          a = a * scales(d.a_scale, d.r, d.a_scale_k_stride, d.a_scale_r_stride,
                         d.k, d.a_scale_square, g * d.a_scale_group_stride)
        if end > begin:
          put(begin, b[begin:end] @ a.T)
        at = end
      if at < d.t:
        put(at, np.zeros((d.t - at, d.r)))
      return 0
    a = operand(d.a, d.a_dtype, d.r, d.a_ld, d.a_mn_major, d.k)
    if fp8 and d.k:
      with np.errstate(invalid='ignore'):  # positions no group fills
        a = a * scales(d.a_scale, d.r, d.a_scale_k_stride, d.a_scale_r_stride,
                       d.k, False)
    at = 0
    for g, (begin, end) in enumerate(spans or [(0, d.k)]):
      if spans and fp8:  # padded positions
        begin, end = at, at + -(-(end - begin) // 128) * 128
        at = end
      put(0, b[:, begin:end] @ a[:, begin:end].T, g)
    assert groups
    return 0

  def aqtb200_pack_bf16(self, view, out, ld, stream):
    return self.aqtb200_pack_bf16_groups(view, None, 0, out, ld, stream)

  def aqtb200_pack_bf16_groups(self, view, sizes, int64, out, ld, stream):
    del stream
    v = view._obj
    n = v.b0 * v.b1 * v.rows
    if not n:
      return 0
    to = _strided(out, _lib.BF16, [n, ld], [ld, 1], True)
    x = fake_lib._view_array(v).reshape(n, v.cols)  # pylint: disable=protected-access
    for b in range(v.b0 * v.b1):
      rows = slice(b * v.rows, (b + 1) * v.rows)
      span = _sizes(sizes, v.b0 * v.b1, int64, 1 << 40)
      if span is not None and span[b][0] == span[b][1]:
        continue
      to[rows] = 0
      if v.cols:
        to[rows, :v.cols] = x[rows]
    return 0


def install(monkeypatch):
  from aqt_b200 import engine
  fake = FakeBlockLib()
  monkeypatch.setattr(_lib, 'load', lambda: fake)
  monkeypatch.setattr(engine, '_stream', lambda: 0)
  monkeypatch.setattr(engine, '_on_device', lambda *t: True)
  return fake
