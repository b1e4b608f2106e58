"""Block-scaled products whose scales are powers of two: wide tiles (results of some
1500 x 1500 and more) with a bfloat16 result let the tensor core scale and sum.
Against the definition in 64 bits, with blocks of very different sizes, so that a
scale in the wrong place shows."""

import numpy as np
import pytest
import torch

from aqt_b200 import engine
from aqt_b200.v2 import aqt_ragged_dot as rd
from aqt_b200.v2 import block_scaled as bs
from tests import block_ref as ref

pytestmark = pytest.mark.gpu
DIMS = (((1,), (0,)), ((), ()))
BF = torch.bfloat16
HALF = 2.0 ** -8


def _data(shape, seed, spread=3):
  """Normal values times powers of two that change with the 128-block of each of
  the last two axes and with the row."""
  rng = np.random.default_rng(seed)
  x = rng.standard_normal(shape)
  r, c = shape[-2:]
  e = rng.integers(-spread, spread + 1, (*shape[:-2], r, -(-c // 128)))
  f = rng.integers(-spread, spread + 1, (*shape[:-2], -(-r // 128), c))
  x = x * 2.0 ** np.repeat(e, 128, -1)[..., :c] * 2.0 ** np.repeat(
      f, 128, -2)[..., :r, :]
  return torch.from_numpy(x.astype(np.float32)).to(BF).cuda()


def _f32(t):
  return t.detach().float().cpu().numpy()


def _done():
  torch.cuda.synchronize()
  engine.check_status()


def _close(got, a, b, k, what=''):
  ref.assert_close(_f32(got).astype(np.float64), a @ b, np.abs(a) @ np.abs(b), k,
                   HALF, what)


def _check_step(x, w, g, got, fwd='e4m3', bwd='e5m2'):
  f = lambda v, br, bc, bits: ref.fake(_f32(v), br, bc, bits, True)
  wq = f(w, 128, 128, fwd)
  out, dl, dr = got
  _close(out, f(x, 1, 128, fwd), wq, x.shape[1], 'out')
  _close(dl, f(g, 1, 128, bwd), wq.T, g.shape[1], 'dlhs')
  _close(dr, f(x, 128, 1, fwd).T, f(g, 128, 1, bwd), x.shape[0], 'drhs')


@pytest.mark.parametrize('m,k,n', [
    (129, 129, 129), (160, 64, 300), (224, 512, 225), (256, 1, 257),
    (300, 640, 520), (449, 1300, 16), (700, 384, 1000), (2047, 257, 130), (512, 1100, 512),
    # forward, or all three products, in wide tiles: one accumulator, two
    (2048, 300, 2000), (1700, 1650, 1750), (3000, 200, 2000), (1999, 129, 2561)])
@pytest.mark.parametrize('fwd,bwd', [('e4m3', 'e5m2'), ('e5m2', 'e4m3')])
def test_step(m, k, n, fwd, bwd):
  x, w, g = _data((m, k), 1), _data((k, n), 2), _data((m, n), 3)
  out, bp = bs.dot_general_make(fwd, bwd, po2_scale=True).vjp(x, w, DIMS)
  got = (out, *bp(g))
  _done()
  assert all(t.dtype == BF for t in got)
  _check_step(x, w, g, got, fwd, bwd)


def test_step_over_either_axis_of_rhs():
  x, w, g = _data((200, 300), 4), _data((300, 260), 5), _data((200, 260), 6)
  out, bp = bs.dot_general_make(po2_scale=True).vjp(
      x, w.t().contiguous(), (((1,), (1,)), ((), ())))
  dl, dr = bp(g)
  _done()
  _check_step(x, w, g, (out, dl, dr.t()))


@pytest.mark.parametrize('m,k,n,sizes', [
    (700, 200, 136, [0, 700, 0]),
    (900, 384, 264, [1, 0, 127, 300, 65, 400]),     # seven rows left over
    (600, 129, 450, [128, 129, 300, 43]),
    (513, 130, 256, [-5, 300, -1, 600]),            # cut at the end
    (400, 64, 200, [0, 0, 0]),
    (3000, 1400, 1300, [0, 700, 1, 1500, 130, 600])])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_ragged_step(m, k, n, sizes, index):
  x, w, g = _data((m, k), 7), _data((len(sizes), k, n), 8), _data((m, n), 9)
  cfg = bs.dot_general_make(po2_scale=True)
  out, bp = rd.ragged_dot_vjp(
      x, w, torch.tensor(sizes, dtype=index, device='cuda'), cfg=cfg)
  dl, dr = bp(g)
  _done()
  spans = ref.spans(sizes, m)
  for e, (a, b) in enumerate(spans):
    if a == b:
      assert not dr[e].any()
    else:
      _check_step(x[a:b], w[e], g[a:b], (out[a:b], dl[a:b], dr[e]))
  left = spans[-1][1]
  assert not out[left:].any() and not dl[left:].any()


def test_many_tiles_a_cluster():
  """More tiles than the device holds at once: scales and operands are fetched
  ahead across tiles, a different number of blocks in each."""
  sizes = [0, 3, 250, 1, 0, 777, 130, 2000, 64, 900]
  m = sum(sizes)
  x, w, g = _data((m, 136), 10), _data((len(sizes), 136, 1800), 11), _data(
      (m, 1800), 12)
  s = torch.tensor(sizes, dtype=torch.int32, device='cuda')
  cfg = bs.dot_general_make(po2_scale=True)
  out, bp = rd.ragged_dot_vjp(x, w, s, cfg=cfg)
  dl, dr = bp(g)
  again = rd.ragged_dot(x, w, s, cfg=cfg)
  _done()
  assert torch.equal(out, again)
  for e, (a, b) in enumerate(ref.spans(sizes, m)):
    if a < b:
      _check_step(x[a:b], w[e], g[a:b], (out[a:b], dl[a:b], dr[e]))


def test_one_accumulator_and_a_second_tile():
  """Few tiles expected, so that one wide accumulator is chosen, and more come."""
  sizes = [193] * 31 + [1] * 19
  m = sum(sizes)
  x, w = _data((m, 136), 30), _data((50, 136, 256), 31)
  out = rd.ragged_dot(x, w, torch.tensor(sizes, dtype=torch.int32, device='cuda'),
                      cfg=bs.dot_general_make(po2_scale=True))
  _done()
  for e, (a, b) in enumerate(ref.spans(sizes, m)):
    _close(out[a:b], ref.fake(_f32(x[a:b]), 1, 128, 'e4m3', True),
           ref.fake(_f32(w[e]), 128, 128, 'e4m3', True), 136)


def test_zero_blocks_and_extreme_scales():
  """Blocks of zeros, and scales at both ends of what a product can hold."""
  x, w = _data((2048, 512), 13), _data((512, 1400), 14)
  x[:, 128:256] = 0
  x[5] = 0
  w[256:384, :128] = 0
  x[7] *= 2.0 ** 60
  x[8] *= 2.0 ** -60
  w[:, 130:] *= 2.0 ** -40
  out = bs.dot_general_make(po2_scale=True)(x, w, DIMS)
  _done()
  _close(out, ref.fake(_f32(x), 1, 128, 'e4m3', True),
         ref.fake(_f32(w), 128, 128, 'e4m3', True), 512)
  assert not out[5].any()


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_nan_and_inf_stay_in_their_rows(bad):
  x, w, g = (_data((1700, 1650), 15), _data((1650, 1750), 16),
             _data((1700, 1750), 17))
  cfg = bs.dot_general_make(po2_scale=True)

  def step():
    out, bp = cfg.vjp(x, w, DIMS)
    return (out, *bp(g))

  clean = step()
  x[7, 3] = bad
  g[200, 1749] = bad
  out, dl, dr = step()
  _done()
  rows = lambda t, *skip: t[[i for i in range(t.shape[0]) if i not in skip]]
  assert torch.equal(rows(out, 7), rows(clean[0], 7))
  assert torch.isnan(out[7]).all()
  assert torch.equal(rows(dl, 200), rows(clean[1], 200))
  assert torch.isnan(dl[200]).all()
  # x[7, 3] reaches row 3 of drhs, g[200, 1749] its last column
  assert torch.isnan(dr[3]).all() and torch.isnan(dr[:, 1749]).all()
  assert torch.equal(rows(dr, 3)[:, :1749], rows(clean[2], 3)[:, :1749])


def test_groups_do_not_mix():
  sizes = [1000, 0, 850, 645]
  m, k, n = 2600, 1400, 1700
  x, w, g = _data((m, k), 18), _data((4, k, n), 19), _data((m, n), 20)
  s = torch.tensor(sizes, dtype=torch.int32, device='cuda')
  cfg = bs.dot_general_make(po2_scale=True)

  def step():
    out, bp = rd.ragged_dot_vjp(x, w, s, cfg=cfg)
    return (out, *bp(g))

  out, dl, dr = step()
  x[2495:] = float('nan')
  g[2495:] = float('nan')
  x[1000, 5] = float('nan')   # first row of the third group
  g[1849, 7] = float('inf')   # its last row
  out2, dl2, dr2 = step()
  _done()
  keep = [i for i in range(m) if not 1000 <= i < 1850]
  assert torch.equal(out[keep], out2[keep]) and torch.equal(dl[keep], dl2[keep])
  for e in (0, 1, 3):
    assert torch.equal(dr[e], dr2[e]), e
  assert torch.isnan(out2[1000]).all() and torch.isnan(dr2[2, 5]).all()


@pytest.mark.parametrize('k', [14336, 262144, 262400])
def test_long_positive_sums(k):
  """All products positive: what the tensor core's sums drop adds up, up to
  2^-23 of the result for each 32 products as long as it is left to sum (262144
  products), and stays below a bfloat16 step. Equal values make the result exact:
  every block is its maximum, one code, and the sum k times one product."""
  x = torch.full((), 1.25, dtype=BF, device='cuda').expand(2048, k)
  w = torch.full((), 0.75, dtype=BF, device='cuda').expand(k, 1300)
  out = bs.dot_general_make(po2_scale=True)(x, w, DIMS)
  _done()
  # 1.25 and 0.75 are codes of e4m3 under any power of two
  want = 1.25 * 0.75 * k
  drop = k / 32 * 2.0 ** -23 * want
  assert ((out.double() - want).abs() <= drop + HALF * (want + drop)).all()


def test_float32_results_keep_their_bits():
  """float32 results are summed in registers: the same bits whichever scales are
  known to be powers of two, frozen weights included."""
  x, w = _data((300, 640), 21), _data((640, 260), 22)
  cfg = bs.dot_general_make(po2_scale=True)
  a = cfg(x, w, DIMS, preferred_element_type=torch.float32)
  qt = bs.block_quantize(w, 0, square=True, po2_scale=True)
  b = cfg(x, qt, DIMS, preferred_element_type=torch.float32)
  _done()
  assert torch.equal(a, b)


def test_frozen_scales_need_not_be_powers_of_two():
  x, w = _data((300, 640), 23), _data((640, 260), 24)
  qt = bs.block_quantize(w, 0, square=True)
  out = bs.dot_general_make(po2_scale=True)(x, qt, DIMS)
  _done()
  _close(out, ref.fake(_f32(x), 1, 128, 'e4m3', True),
         ref.fake(_f32(w), 128, 128, 'e4m3', False), 640)


def test_captured_and_replayed():
  x, w, g = _data((1700, 260), 25), _data((260, 1750), 26), _data((1700, 1750), 27)
  cfg = bs.dot_general_make(po2_scale=True)

  def step():
    out, bp = cfg.vjp(x, w, DIMS)
    return (out, *bp(g))

  step()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=side):
    got = step()
  for seed in (28, 29):
    x.copy_(_data((1700, 260), seed))
    graph.replay()
    _done()
    _check_step(x, w, g, got)


@pytest.mark.parametrize('a,b', [(-60, -62), (-70, -66), (100, -60), (-60, 100),
                                 (-108, 90), (110, -100), (-45, -97), (60, 40)])
@pytest.mark.parametrize('m,k,n', [(2048, 384, 2560), (200, 300, 129)])
def test_far_exponents(m, k, n, a, b):
  """Scales whose product f32 does not hold, results that it does."""
  rng = np.random.default_rng(76)

  def values(shape, e):
    v = rng.integers(-15, 16, shape).astype(np.float64)
    return torch.from_numpy(np.ldexp(v + (v == 0), e).astype(np.float32)).to(
        torch.bfloat16).cuda()

  x, w, g = values((m, k), a), values((k, n), b), values((m, n), -a // 2)
  out, bp = bs.dot_general_make('e4m3', 'e4m3', po2_scale=True).vjp(x, w, DIMS)
  got = (out, *bp(g))
  _done()
  f = lambda t, br, bc: ref.fake(t.float().cpu().numpy(), br, bc, 'e4m3', True)
  w_ = f(w, 128, 128)
  for name, t, (p, q) in zip(('out', 'dlhs', 'drhs'), got, (
      (f(x, 1, 128), w_), (f(g, 1, 128), w_.T), (f(x, 128, 1).T, f(g, 128, 1)))):
    want, mag = p @ q, np.abs(p) @ np.abs(q)
    held = mag < 2.0 ** 127  # the others pass f32's range, in sum or on the way
    t = t.float().cpu().numpy().astype(np.float64)
    ref.assert_close(t[held], want[held], mag[held], p.shape[1], 2.0 ** -8, name)
