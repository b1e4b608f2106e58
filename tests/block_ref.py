"""Block-scaled and grouped products in 64 bits, from their definitions.

A block's scale, its reciprocal and the scaled value that is rounded to 8 bits
are 32-bit numbers by definition; everything after that is exact here.
"""

import ml_dtypes
import numpy as np

BLOCK = 128
BOUND = {'e4m3': 448.0, 'e5m2': 57344.0}
FP8 = {'e4m3': ml_dtypes.float8_e4m3fn, 'e5m2': ml_dtypes.float8_e5m2}


def quantize(x, br, bc, bits, po2=False):
  """x [R, C] -> (q [R, C] in fp8, s [R/br, C/bc] float32)."""
  x = np.asarray(x, np.float32)
  r, c = x.shape
  nr, nc = -(-r // br), -(-c // bc)
  p = np.zeros((nr * br, nc * bc), np.float32)
  p[:r, :c] = x
  p = p.reshape(nr, br, nc, bc)
  with np.errstate(all='ignore'):
    a = np.abs(p).max(axis=(1, 3))
    s = np.where(a == 0, np.float32(1), a) / np.float32(BOUND[bits])
    s = np.maximum(s, np.float32(2.0 ** -126))  # keeps a NaN
    if po2:
      m, e = np.frexp(s)
      s = np.ldexp(np.float32(1), np.where(m == 0.5, e - 1, e)).astype(np.float32)
    y = p * (np.float32(1) / s)[:, None, :, None]
    y = np.clip(y, -BOUND[bits], BOUND[bits]).astype(np.float32)
    q = y.astype(FP8[bits]).reshape(nr * br, nc * bc)[:r, :c]
  return q, s


def widen(q, s, br, bc):
  r, c = q.shape
  s = np.repeat(np.repeat(s.astype(np.float64), br, 0), bc, 1)[:r, :c]
  return q.astype(np.float64) * s


def fake(x, br, bc, bits, po2=False):
  return widen(*quantize(x, br, bc, bits, po2), br, bc)


def spans(sizes, rows):
  """(first, end) of every group after the device's rules."""
  out, at = [], 0
  for n in sizes:
    end = min(at + max(int(n), 0), rows)
    out.append((at, end))
    at = end
  return out


def ragged(lhs, rhs, sizes):
  """(out, bound): the product and sum |a||b|, which error bounds go by."""
  out = np.zeros((lhs.shape[0], rhs.shape[2]))
  mag = np.zeros_like(out)
  for e, (a, b) in enumerate(spans(sizes, lhs.shape[0])):
    out[a:b] = lhs[a:b] @ rhs[e]
    mag[a:b] = np.abs(lhs[a:b]) @ np.abs(rhs[e])
  return out, mag


def ragged_drhs(lhs, g, sizes, groups):
  """Per-group lhs^T g; lhs and g may be functions of a group's rows."""
  out, mag = [], []
  for a, b in spans(sizes, lhs.shape[0]):
    out.append(lhs[a:b].T @ g[a:b])
    mag.append(np.abs(lhs[a:b]).T @ np.abs(g[a:b]))
  assert len(out) == groups
  return np.stack(out), np.stack(mag)


def assert_close(got, want, mag, k, half_step, what=''):
  """|got - want| within what the arithmetic allows.

  A sum of k exact products in f32, in any order and with truncation, is off by
  at most k 2^-23 sum|ab| (each of its additions by one unit in the last place
  of a partial sum, which is at most sum|ab|); block scales add three roundings
  of 2^-24 per 128. The result is rounded once: half_step, relative, plus half
  the smallest subnormal.
  """
  acc = (k + 3 * (k // BLOCK + 1)) * 2.0 ** -23 * mag
  tol = acc + half_step * (np.abs(want) + acc) + 2.0 ** -134
  bad = ~(np.abs(got - want) <= tol)
  assert not bad.any(), (
      f'{what}: {bad.sum()} of {bad.size} outside the bound, worst '
      f'{np.nanmax(np.abs(got - want) / tol):.3g} times it at '
      f'{np.argwhere(bad)[:3].tolist()}')
