"""Block-scaled fp8 on the GPU against the definition in 64 bits: quantized
values and scales bit for bit, products within the bound of their arithmetic."""

import numpy as np
import pytest
import torch

from aqt_b200 import engine
from aqt_b200.v2 import aqt_dot_general
from aqt_b200.v2 import block_scaled as bs
from tests import block_ref as ref
from tests import util

pytestmark = pytest.mark.gpu

DIMS = (((1,), (0,)), ((), ()))
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _data(shape, dtype, seed, spread=2.0):
  rng = np.random.default_rng(seed)
  x = rng.standard_normal(shape) * np.exp(
      spread * rng.standard_normal((*shape[:-1], 1)))
  return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def _f32(t):
  return t.float().cpu().numpy()


def _done():
  torch.cuda.synchronize()
  engine.check_status()


def _check_quantized(x, qt, axis, square, bits, po2=False):
  br = ref.BLOCK if square or axis == -2 else 1
  bc = ref.BLOCK if square or axis == -1 else 1
  q, s = ref.quantize(_f32(x), br, bc, bits, po2)
  got = util.to_numpy(qt.qvalue)
  assert got.dtype == q.dtype and got.shape == q.shape
  np.testing.assert_array_equal(qt.scale[0].cpu().numpy(), s)
  # bytes, but for the sign of a NaN: that of infinity times zero is not defined
  nan = np.isnan(q.astype(np.float32))
  np.testing.assert_array_equal(np.isnan(got.astype(np.float32)), nan)
  np.testing.assert_array_equal(got.view(np.uint8)[~nan], q.view(np.uint8)[~nan])


@pytest.mark.parametrize('shape', [(1, 1), (1, 128), (7, 129), (128, 128),
                                   (130, 1), (255, 384), (300, 515)])
@pytest.mark.parametrize('axis', [-1, -2])
@pytest.mark.parametrize('square', [False, True])
@pytest.mark.parametrize('bits', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_quantize_bit_exact(shape, axis, square, bits, dtype):
  x = _data(shape, dtype, 1)
  qt = bs.block_quantize(x, contract_axis=axis, square=square, bits=bits)
  _done()
  _check_quantized(x, qt, axis, square, bits)
  assert qt.qvalue.stride(axis) == 1 or x.shape[axis] == 1


@pytest.mark.parametrize('axis', [-1, -2])
@pytest.mark.parametrize('square', [False, True])
def test_quantize_powers_of_two(axis, square):
  x = _data((200, 300), torch.float32, 2)
  x[0, :128] = 0
  x[0, 0] = 448 * 0.25  # a scale that is a power of two already stays
  qt = bs.block_quantize(x, axis, square, po2_scale=True)
  _done()
  _check_quantized(x, qt, axis, square, 'e4m3', po2=True)
  m, _ = np.frexp(qt.scale[0].cpu().numpy())
  assert (m == 0.5).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_quantize_zeros_tiny_and_huge(dtype):
  x = torch.zeros(6, 256, dtype=dtype, device='cuda')
  x[1, 3] = 1e-39                              # below the smallest normal scale
  x[2, 3] = torch.finfo(dtype).max
  x[3, :] = -torch.finfo(dtype).max
  x[4, 130] = torch.finfo(dtype).tiny
  qt = bs.block_quantize(x)
  _done()
  _check_quantized(x, qt, -1, False, 'e4m3')
  assert float(qt.scale[0][0, 0]) == float(np.float32(1) / np.float32(448))


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_quantize_nan_and_inf_stay_in_their_block(bad):
  x = _data((256, 256), torch.bfloat16, 3)
  x[5, 17] = bad
  for axis in (-1, -2):
    for square in (False, True):
      qt = bs.block_quantize(x, axis, square)
      _done()
      _check_quantized(x, qt, axis, square, 'e4m3')


def _layouts(shape, dtype, seed):
  """The same values lying in memory in ways a caller may have them."""
  x = _data(shape, dtype, seed)
  wide = torch.zeros(shape[0], shape[1] + 24, dtype=dtype, device='cuda')
  wide[:, 3:3 + shape[1]] = x  # rows off the 16-byte boundary
  yield 'offset columns', x, wide[:, 3:3 + shape[1]]
  yield 'transposed', x, x.t().contiguous().t()
  every = torch.zeros(shape[0] * 2, shape[1] * 3, dtype=dtype, device='cuda')
  every[::2, ::3] = x
  yield 'both strides', x, every[::2, ::3]
  yield 'expanded rows', x[:1].expand(shape[0], -1).clone(), x[:1].expand(
      shape[0], -1)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('axis', [-1, -2])
@pytest.mark.parametrize('square', [False, True])
def test_quantize_any_strides(dtype, axis, square):
  for name, x, view in _layouts((140, 264), dtype, 4):
    qt = bs.block_quantize(view, axis, square)
    _done()
    np.testing.assert_array_equal(_f32(x), _f32(view), err_msg=name)
    _check_quantized(x, qt, axis, square, 'e4m3')


def test_quantize_matrices():
  x = _data((3, 140, 200), torch.bfloat16, 5)
  for axis in (-1, -2):
    for square in (False, True):
      qt = bs.block_quantize(x, axis, square)
      qs = bs.block_quantize(x.transpose(1, 2).contiguous().transpose(1, 2),
                             axis, square)
      _done()
      for g in range(3):
        for t in (qt, qs):
          one = t.replace(qvalue=t.qvalue[g], scale=[t.scale[0][g]])
          _check_quantized(x[g], one, axis, square, 'e4m3')


def test_quantize_empty():
  for shape in ((0, 5), (5, 0), (0, 128, 128)):
    qt = bs.block_quantize(torch.zeros(shape, device='cuda'))
    assert tuple(qt.qvalue.shape) == shape


def _want(x, w, g, po2=False, fwd='e4m3', bwd='e5m2'):
  """(out, dlhs, drhs) with their magnitudes."""
  f = lambda v, br, bc, b: ref.fake(v, br, bc, b, po2)
  w_ = f(w, 128, 128, fwd)
  pairs = [(f(x, 1, 128, fwd), w_)]
  if g is not None:
    pairs += [(f(g, 1, 128, bwd), w_.T),
              (f(x, 128, 1, fwd).T, f(g, 128, 1, bwd))]
  return [(a @ b, np.abs(a) @ np.abs(b), a.shape[1]) for a, b in pairs]


SIZES = [(1, 64, 64), (1, 128, 300), (3, 1, 17), (33, 300, 129), (64, 640, 256),
         (129, 257, 511), (300, 1000, 777), (520, 384, 1040)]


@pytest.mark.parametrize('m,k,n', SIZES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('po2', [False, True])
def test_step_matches_definition(m, k, n, dtype, po2):
  x, w, g = (_data((m, k), dtype, 6, 1.0), _data((k, n), dtype, 7, 0.3),
             _data((m, n), dtype, 8, 1.0))
  out, bp = bs.dot_general_make(po2_scale=po2).vjp(x, w, DIMS)
  dl, dr = bp(g)
  _done()
  for name, got, (want, mag, kk) in zip(('out', 'dlhs', 'drhs'), (out, dl, dr),
                                        _want(_f32(x), _f32(w), _f32(g), po2)):
    assert got.dtype == dtype
    ref.assert_close(_f32(got).astype(np.float64), want, mag, kk, HALF[dtype],
                     name)


@pytest.mark.parametrize('fwd,bwd', [('e4m3', 'e4m3'), ('e5m2', 'e4m3'),
                                     ('e5m2', 'e5m2')])
def test_step_formats(fwd, bwd):
  x, w, g = (_data((70, 200), torch.bfloat16, 6, 1.0),
             _data((200, 300), torch.bfloat16, 7, 0.3),
             _data((70, 300), torch.bfloat16, 8, 1.0))
  out, bp = bs.dot_general_make(fwd, bwd).vjp(x, w, DIMS)
  got = (out, *bp(g))
  _done()
  for a, (want, mag, kk) in zip(got, _want(_f32(x), _f32(w), _f32(g), False, fwd,
                                           bwd)):
    ref.assert_close(_f32(a).astype(np.float64), want, mag, kk, 2.0 ** -8)


@pytest.mark.parametrize('m,k,n', SIZES + [(16, 2048, 512), (5, 4096, 256),
                                           (257, 1280, 640)])
def test_frozen_weights(m, k, n):
  x, w = _data((m, k), torch.bfloat16, 9, 1.0), _data((k, n), torch.bfloat16, 10)
  cfg = bs.dot_general_make()
  qt = bs.block_quantize(w, contract_axis=0, square=True)
  (want, mag, kk), = _want(_f32(x), _f32(w), None)
  # as quantized, and through a checkpoint's plain layout
  again = bs.frozen(qt.qvalue.contiguous(), qt.scale[0].clone())
  for q in (qt, again):
    for dt in (torch.bfloat16, torch.float32):
      out = cfg(x, q, DIMS, preferred_element_type=dt)
      _done()
      assert out.dtype == dt
      ref.assert_close(_f32(out).astype(np.float64), want, mag, kk, HALF[dt])


def test_dimension_numbers():
  """rhs contracted over either axis, lhs with leading axes or transposed."""
  x, w = _data((6, 10, 200), torch.bfloat16, 11, 1.0), _data(
      (200, 96), torch.bfloat16, 12)
  cfg = bs.dot_general_make()
  plain = cfg(x.view(60, 200), w, DIMS)
  a = cfg(x, w, (((2,), (0,)), ((), ())))
  b = cfg(x, w.t().contiguous(), (((2,), (1,)), ((), ())))
  c = cfg(x.view(60, 200).t().contiguous(), w, (((0,), (0,)), ((), ())))
  d = aqt_dot_general.einsum('abk,kn->abn', x, w, dg=cfg)
  e = cfg(x[:, ::2], w, (((2,), (0,)), ((), ())))  # rows no single stride spans
  f = cfg(x[0, 0], w, (((0,), (0,)), ((), ())))
  _done()
  assert torch.equal(a.view(60, 96), plain) and torch.equal(d, a)
  assert torch.equal(b.view(60, 96), plain) and torch.equal(c, plain)
  assert torch.equal(e, a[:, ::2])
  assert torch.equal(f, a[0, 0])


@pytest.mark.parametrize('rhs_axis', [0, 1])
@pytest.mark.parametrize('lhs_t', [False, True])
def test_gradients_follow_their_operands(rhs_axis, lhs_t):
  x, w, g = (_data((40, 200), torch.bfloat16, 13, 1.0),
             _data((200, 96), torch.bfloat16, 14, 0.3),
             _data((40, 96), torch.bfloat16, 15, 1.0))
  cfg = bs.dot_general_make()
  out, bp = cfg.vjp(x, w, DIMS)
  dl, dr = bp(g)
  a = x.t().contiguous() if lhs_t else x
  b = w.t().contiguous() if rhs_axis else w
  out2, bp2 = cfg.vjp(a, b, (((0 if lhs_t else 1,), (rhs_axis,)), ((), ())))
  dl2, dr2 = bp2(g)
  _done()
  assert torch.equal(out, out2)
  assert dl2.shape == a.shape and dr2.shape == b.shape
  assert torch.equal(dl2.t() if lhs_t else dl2, dl)
  assert torch.equal(dr2.t() if rhs_axis else dr2, dr)


def test_autograd_matches_vjp_and_skips_what_is_not_asked():
  x, w, g = (_data((40, 200), torch.bfloat16, 16, 1.0),
             _data((200, 96), torch.bfloat16, 17, 0.3),
             _data((40, 96), torch.bfloat16, 18, 1.0))
  cfg = bs.dot_general_make()
  out, bp = cfg.vjp(x, w, DIMS)
  dl, dr = bp(g)
  for need_l, need_r in ((True, True), (True, False), (False, True)):
    a, b = x.clone().requires_grad_(need_l), w.clone().requires_grad_(need_r)
    y = cfg(a, b, DIMS)
    y.backward(g)
    assert torch.equal(y, out)
    assert torch.equal(a.grad, dl) if need_l else a.grad is None
    assert torch.equal(b.grad, dr) if need_r else b.grad is None
  # a broadcast cotangent (strides 0)
  a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
  cfg(a, b, DIMS).sum().backward()
  _, bp = cfg.vjp(x, w, DIMS)
  ones = torch.ones_like(g)
  dl, dr = bp(ones)
  _done()
  assert torch.equal(a.grad, dl) and torch.equal(b.grad, dr)


def test_gradients_against_differences():
  """With values that 8 bits hold exactly the product is linear, so differences
  of the forward product are its gradients."""
  rng = np.random.default_rng(19)
  ints = lambda *s: torch.from_numpy(
      rng.integers(-3, 4, s).astype(np.float32)).cuda()
  x, w, g = ints(6, 130), ints(130, 9), ints(6, 9)
  for t in (x, w, g):
    t.view(-1)[::7] = 0
  # every block's maximum is 7, so each scale is the same power of two
  x[:, 0] = x[:, 129] = 7
  w[0, :] = w[128, :] = 7
  g[:, 0] = 7
  cfg = bs.dot_general_make('e4m3', 'e4m3', po2_scale=True)
  out, bp = cfg.vjp(x, w, DIMS)
  dl, dr = bp(g)
  _done()
  x64, w64, g64 = (_f32(t).astype(np.float64) for t in (x, w, g))
  np.testing.assert_array_equal(_f32(out), x64 @ w64)
  loss = lambda a, b: float(((a @ b) * g64).sum())
  for i, j in ((0, 1), (3, 128), (5, 50)):
    d = np.zeros_like(x64)
    d[i, j] = 1
    assert float(dl[i, j]) == (loss(x64 + d, w64) - loss(x64 - d, w64)) / 2
  for i, j in ((1, 0), (129, 8), (64, 3)):
    d = np.zeros_like(w64)
    d[i, j] = 1
    assert float(dr[i, j]) == (loss(x64, w64 + d) - loss(x64, w64 - d)) / 2


def test_nan_and_inf_stay_in_their_rows():
  x, w = _data((40, 256), torch.bfloat16, 20, 1.0), _data(
      (256, 300), torch.bfloat16, 21)
  cfg = bs.dot_general_make()
  clean = cfg(x, w, DIMS)
  x[7, 3] = float('nan')
  x[9, 200] = float('inf')
  out = cfg(x, w, DIMS)
  _done()
  rest = [i for i in range(40) if i not in (7, 9)]
  assert torch.equal(out[rest], clean[rest])
  assert torch.isnan(out[7]).all() and torch.isnan(out[9]).all()


def test_empty_extents():
  cfg = bs.dot_general_make()
  for m, k, n in ((0, 64, 32), (4, 0, 32), (4, 64, 0)):
    x = torch.ones(m, k, device='cuda', dtype=torch.bfloat16)
    w = torch.ones(k, n, device='cuda', dtype=torch.bfloat16)
    out, bp = cfg.vjp(x, w, DIMS)
    dl, dr = bp(torch.ones(m, n, device='cuda', dtype=torch.bfloat16))
    _done()
    assert tuple(out.shape) == (m, n) and not out.any()
    assert dl.shape == x.shape and not dl.any()
    assert dr.shape == w.shape and not dr.any()


def test_captured_replayed_and_on_another_stream():
  x, w, g = (_data((100, 384), torch.bfloat16, 22, 1.0),
             _data((384, 200), torch.bfloat16, 23, 0.3),
             _data((100, 200), torch.bfloat16, 24, 1.0))
  cfg = bs.dot_general_make()

  def step():
    out, bp = cfg.vjp(x, w, DIMS)
    return (out, *bp(g))

  want = [t.clone() for t in step()]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    out, bp = cfg.vjp(x, w, DIMS)
  torch.cuda.current_stream().wait_stream(side)
  got = (out, *bp(g))  # backward on another stream than the forward pass
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = step()
  new = _data((100, 384), torch.bfloat16, 25, 1.0)
  x.copy_(new)
  graph.replay()
  again = step()
  _done()
  assert all(torch.equal(a, b) for a, b in zip(outs, again))


def test_traced_step():
  x, w = _data((30, 256), torch.bfloat16, 26), _data((256, 64), torch.bfloat16, 27)
  qt = bs.block_quantize(w, 0, square=True)
  cfg = bs.dot_general_make()
  step = engine.TracedStep(lambda a: cfg(a, qt, DIMS), x)
  x.copy_(_data((30, 256), torch.bfloat16, 28))
  got = step(x).clone()
  want = cfg(x, qt, DIMS)
  _done()
  assert torch.equal(got, want)


def test_projection_stack_runs_on_block_scaled_products():
  """The decoder stack's projections, one layer, a training micro-step: runs, and
  the weight gradients agree with the int8 stack's to what 8 bits leave."""
  from aqt_b200 import layer_stack
  x = _data((128, layer_stack.D_MODEL), torch.bfloat16, 29, 0.0)
  grads = []
  for cfg in (bs.dot_general_make('e4m3', 'e4m3'), None):
    stack = layer_stack.ProjectionStack('cuda', layers=1, cfg=cfg)
    loss = stack.micro_step(x)
    _done()
    assert torch.isfinite(loss)
    grads.append(stack.grad[0])
  for name in grads[0]:
    a, b = grads[0][name].double(), grads[1][name].double()
    # two operands a product, each off by at most 2^-4 (e4m3); the longest chain
    # to a weight gradient is five products deep
    assert float((a - b).norm() / b.norm()) < 2 * 2.0 ** -4 * 5, name


@pytest.mark.parametrize('m,k,n', [(1700, 1650, 1750), (3000, 200, 2001),
                                   (2048, 129, 2560)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_step_in_wide_tiles(m, k, n, dtype):
  """Results that take more tiles of 128 columns than the device holds at once."""
  x, w, g = (_data((m, k), dtype, 40, 1.0), _data((k, n), dtype, 41, 0.3),
             _data((m, n), dtype, 42, 1.0))
  out, bp = bs.dot_general_make().vjp(x, w, DIMS)
  got = (out, *bp(g))
  _done()
  for name, a, (want, mag, kk) in zip(('out', 'dlhs', 'drhs'), got,
                                      _want(_f32(x), _f32(w), _f32(g))):
    ref.assert_close(_f32(a).astype(np.float64), want, mag, kk, HALF[dtype], name)


@pytest.mark.parametrize('m,k,n', [(1, 4096, 512), (16, 8192, 1024),
                                   (700, 2048, 256), (3000, 1024, 2048)])
@pytest.mark.parametrize('po2', [False, True])
def test_products_back_to_back(m, k, n, po2):
  """A product starts while its operand is still being quantized: queued without
  a pause, on changing values and memory that is used over and over, each gives
  what it gives alone. Weights are written anew just before, too."""
  cfg = bs.dot_general_make(po2_scale=po2)
  xs = [_data((m, k), torch.bfloat16, 50 + i, 1.0) for i in range(4)]
  ws = [_data((k, n), torch.bfloat16, 60 + i, 0.3) for i in range(2)]
  alone = {}
  for i, x in enumerate(xs):
    for j, w in enumerate(ws):
      alone[i, j] = cfg(x, bs.block_quantize(w, 0, square=True), DIMS)
      _done()
  x = torch.empty_like(xs[0])
  got = []
  for turn in range(40):
    i, j = turn % 4, turn % 2
    x.copy_(xs[i])
    qt = bs.block_quantize(ws[j], 0, square=True)
    got.append((i, j, cfg(x, qt, DIMS)))
    x.zero_()  # queued behind the product
    del qt
  _done()
  for i, j, out in got:
    assert torch.equal(out, alone[i, j]), (i, j)


# Exponents of the operands' magnitudes: the block scales' product (about 2^17.6
# less) lies below f32's normal numbers, at zero or above its range, or one scale
# alone takes a block's sum out of it, where the results do not.
EXPONENTS = [(-60, -62), (-70, -66), (-100, 20), (100, -60), (-60, 100), (-108, 90),
             (110, -100), (-45, -97)]


def _far(shape, dtype, seed, exponent):
  """Values whose blocks' maxima are all the same size, times 2^exponent; the
  rounding to 8 bits is then the same for every exponent but for the scale."""
  rng = np.random.default_rng(seed)
  x = rng.integers(-15, 16, shape).astype(np.float64)
  x = np.ldexp(x + (x == 0), exponent)
  return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


@pytest.mark.parametrize('m,k,n', [(3, 640, 70), (200, 300, 129),
                                   (2048, 384, 2560)])
@pytest.mark.parametrize('a,b', EXPONENTS)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('rhs_axis', [0, 1])
def test_scales_whose_product_leaves_the_range(m, k, n, a, b, dtype, rhs_axis):
  x, w, g = (_far((m, k), dtype, 70, a), _far((k, n), dtype, 71, b),
             _far((m, n), dtype, 72, -a // 2))
  v = w.t().contiguous() if rhs_axis else w
  out, bp = bs.dot_general_make('e4m3', 'e4m3').vjp(x, v, (((1,), (rhs_axis,)),
                                                           ((), ())))
  dl, dr = bp(g)
  _done()
  dr = dr.t() if rhs_axis else dr
  for name, got, (want, mag, kk) in zip(
      ('out', 'dlhs', 'drhs'), (out, dl, dr),
      _want(_f32(x), _f32(w), _f32(g), False, 'e4m3', 'e4m3')):
    _check_in_range(got, want, mag, kk, HALF[dtype], name)


def _check_in_range(got, want, mag, k, half, name):
  """What f32 holds on the way is right; what it cannot hold is not finite. (Sums
  between the two may overflow in one order and not in another, and two partial
  sums of either sign past the range add up to a NaN.)"""
  got = _f32(got).astype(np.float64)
  held = mag < 2.0 ** 127
  ref.assert_close(got[held], want[held], mag[held], k, half, name)
  past = np.abs(want) - (k + 3) * 2.0 ** -22 * mag >= 2.0 ** 128
  assert not np.isfinite(got[past]).any(), name


@pytest.mark.parametrize('m,n', [(3, 70), (2048, 2560)])
@pytest.mark.parametrize('e', [60, 72, 100])
def test_large_scales_on_operands_that_hardly_meet(m, n, e):
  """Each operand's large values meet the other's zeros, its small ones each
  other: the scales' product is past f32's range, the results are not."""
  k = 256
  x = torch.zeros(m, k, device='cuda')
  w = torch.zeros(k, n, device='cuda')
  x[:, 0::8], w[1::8, :] = 2.0 ** e, 2.0 ** e      # scales near 2^(e - 8.8)
  x[:, 2::16] = 2.0 ** (e - 15)                    # 2^-6 in units of a scale
  w[2::16, ::3] = 2.0 ** (e - 15)
  qt = bs.block_quantize(w, 0, square=True)
  (want, mag, kk), = _want(_f32(x), _f32(w), None)
  cfg = bs.dot_general_make()
  for q in (w, qt):
    out = cfg(x, q, DIMS)
    _done()
    got = _f32(out)
    assert not got[:, 1::3].any() and not got[:, 2::3].any()
    _check_in_range(out, want, mag, kk, 2.0 ** -24, '')


def test_far_scales_leave_other_rows_alone():
  """Rows that need the careful products change no bit of the others."""
  x, w = _data((300, 384), torch.bfloat16, 73, 1.0), _data((384, 200),
                                                         torch.bfloat16, 74, 0.3)
  cfg = bs.dot_general_make()
  w[:128] *= 2.0 ** -60
  out, bp = cfg.vjp(x, w, DIMS)
  g = _data((300, 200), torch.bfloat16, 75, 1.0)
  dl, dr = bp(g)
  x2, g2 = x.clone(), g.clone()
  x2[7] *= 2.0 ** -75
  g2[9] *= 2.0 ** -90
  g2[:, 5] *= 2.0 ** -110
  x2[:, 3] *= 2.0 ** 60
  rest = [i for i in range(300) if i not in (7, 9)]
  out2 = cfg.vjp(x2, w, DIMS)[0]
  x3 = x.clone()
  x3[7] *= 2.0 ** -75
  assert torch.equal(cfg.vjp(x3, w, DIMS)[0][rest], out[rest])
  assert torch.isfinite(out2.float()).all()
  dr3 = cfg.vjp(x, w, DIMS)[1](g)[1]
  g3 = g.clone()
  g3[:, 5] *= 2.0 ** -110
  dr4 = cfg.vjp(x, w, DIMS)[1](g3)[1]
  _done()
  cols = [i for i in range(200) if i != 5]
  assert torch.equal(dr3, dr) and torch.equal(dr4[:, cols], dr[:, cols])


def test_projection_stack_product_by_product():
  """Each projection of a micro-step gets its own product's gradient, and those of
  the keys and values are the definition's for the operands they got."""
  from aqt_b200 import layer_stack
  cfg, seen = bs.dot_general_make(), []

  class Watched:

    def vjp(self, x, w, dims):
      out, bp = cfg.vjp(x, w, dims)
      at = {'x': x.clone(), 'w': w, 'out': out.clone()}
      seen.append(at)

      def back(g):
        at['g'] = g.clone()
        at['dl'], at['dr'] = bp(g)
        return at['dl'], at['dr'].clone()

      return out, back

  stack = layer_stack.ProjectionStack('cuda', layers=1, cfg=Watched())
  stack.micro_step(_data((130, layer_stack.D_MODEL), torch.bfloat16, 29, 0.0))
  _done()
  names = [n for n, _, _ in layer_stack.PROJ]
  assert len(seen) == len(names)
  for name, at in zip(names, seen):
    assert torch.equal(stack.grad[0][name], at['dr']), name
    if name in ('wk', 'wv'):
      for what, (want, mag, kk) in zip(('out', 'dl', 'dr'), _want(
          _f32(at['x']), _f32(at['w']), _f32(at['g']))):
        ref.assert_close(_f32(at[what]).astype(np.float64), want, mag, kk,
                         2.0 ** -8, f'{name} {what}')


@pytest.mark.parametrize('m,n', [(1500, 5120), (2047, 7168), (3300, 3500), (700, 12000),
                                 (130, 200)])
@pytest.mark.parametrize('rows', [128, 1])
def test_far_rows_wherever_they_lie(m, n, rows):
  """Tiles of any width: rows that need care lie in any one of the blocks of 128 that
  a tile covers, its middle one too."""
  k = 256
  x, w = _data((m, k), torch.float32, 76, 1.0), _data((k, n), torch.float32, 77, 0.3)
  w *= 2.0 ** -50  # scales that alone are no reason for care
  cfg = bs.dot_general_make()
  qt = bs.block_quantize(w, 0, square=True)
  assert float(qt.scale[0].min()) > 2.0 ** -63
  base = cfg(x, qt, DIMS)
  mag = cfg(x.abs(), bs.frozen(qt.qvalue.float().abs().to(torch.float8_e4m3fn),
                               qt.scale[0]), DIMS).double()
  for first in range(0, m, 128):
    at = slice(first + (17 if rows == 1 and first + 17 < m else 0), None)
    at = slice(at.start, min(at.start + rows, m))
    far = x.clone()
    far[at] *= 2.0 ** -75
    out = cfg(far, qt, DIMS)
    # two sums of the same products, each off by k 2^-23 of their magnitudes
    off = (out[at].double() * 2.0 ** 75 - base[at].double()).abs()
    assert (off <= 2 * (k + 9) * 2.0 ** -23 * mag[at]).all(), first
    same = torch.ones(m, dtype=torch.bool, device='cuda')
    same[at] = False
    assert torch.equal(out[same], base[same]), first
  _done()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_far_scales_of_transposed_operands(dtype):
  """Operands read the way they lie: their marks change places with their values."""
  x, w, g = (_data((300, 384), dtype, 78, 1.0), _data((384, 200), dtype, 79, 0.3),
             _data((300, 200), dtype, 80, 1.0))
  x[:130] *= 2.0 ** -70
  x[130:, :128] *= 2.0 ** 30
  w[:, :128] *= 2.0 ** -66
  g[:, 150:] *= 2.0 ** -90
  cfg = bs.dot_general_make()
  out, bp = cfg.vjp(x, w, DIMS)
  want = (out, *bp(g))
  flip = lambda t: t.t().contiguous().t()
  out, bp = cfg.vjp(flip(x), flip(w), DIMS)
  got = (out, *bp(flip(g)))
  _done()
  for a, b, (value, mag, kk) in zip(got, want, _want(_f32(x), _f32(w), _f32(g))):
    assert torch.equal(a, b)
    ref.assert_close(_f32(a).astype(np.float64), value, mag, kk, HALF[dtype])


@pytest.mark.parametrize('g_exponent', [-90, -100, -112])
def test_small_cotangents(g_exponent):
  """Scales below what a sum could stand, and sums that are large enough: the
  products' own results are right and stay, those of columns that cancel are made
  anew."""
  m, k, n = 1500, 300, 1750
  x, w, g = (_data((m, k), torch.float32, 81, 1.0), _data((k, n), torch.float32, 82, 0.3),
             _data((m, n), torch.float32, 83, 1.0) * 2.0 ** g_exponent)
  x[::2, 7] = 0   # meets next to nothing of a column's cotangents
  g[1::2, 11] = 0
  g[1::2, 11][::9] = 2.0 ** (g_exponent - 13)
  out, bp = bs.dot_general_make().vjp(x, w, DIMS)
  dl, dr = bp(g)
  _done()
  for got, (want, mag, kk) in zip((out, dl, dr), _want(_f32(x), _f32(w), _f32(g))):
    ref.assert_close(_f32(got).astype(np.float64), want, mag, kk, 2.0 ** -24)
