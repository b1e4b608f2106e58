"""Host logic of the block-scaled and grouped products on the CPU: layouts,
operand orders, gradients and groups against the definition in 64 bits, with the
library replaced by tests/fake_block_lib.py."""

import numpy as np
import pytest
import torch

from aqt_b200 import engine
from aqt_b200.v2 import aqt_dot_general
from aqt_b200.v2 import aqt_ragged_dot as rd
from aqt_b200.v2 import block_scaled as bs
from tests import block_ref as ref
from tests import fake_block_lib
from tests import util

DIMS = (((1,), (0,)), ((), ()))
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def fake(monkeypatch):
  return fake_block_lib.install(monkeypatch)


def _data(shape, dtype, seed, scale=1.0):
  rng = np.random.default_rng(seed)
  return torch.from_numpy((rng.standard_normal(shape) * scale).astype(
      np.float32)).to(dtype)


def _np(t):
  return t.detach().float().numpy()


def _off(t):
  wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype)
  wide[..., 2:2 + t.shape[-1]] = t
  return wide[..., 2:2 + t.shape[-1]]


def _flip(t):
  return t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize('shape', [(1, 1), (5, 130), (129, 16), (3, 40, 150)])
@pytest.mark.parametrize('axis', [-1, -2])
@pytest.mark.parametrize('square', [False, True])
@pytest.mark.parametrize('layout', [lambda t: t, _off, _flip])
def test_quantize(shape, axis, square, layout):
  x = _data(shape, torch.bfloat16, 1)
  qt = bs.block_quantize(layout(x), axis, square, 'e5m2', po2_scale=True)
  br = 128 if square or axis == -2 else 1
  bc = 128 if square or axis == -1 else 1
  for g in range(shape[0] if len(shape) == 3 else 1):
    pick = (lambda t: t[g]) if len(shape) == 3 else (lambda t: t)
    q, s = ref.quantize(_np(pick(x)), br, bc, 'e5m2', True)
    np.testing.assert_array_equal(pick(qt.scale[0]).numpy(), s)
    np.testing.assert_array_equal(util.to_numpy(pick(qt.qvalue)).view(np.uint8),
                                  q.view(np.uint8))


def _dot_want(x, w, g):
  f = ref.fake
  wq = f(w, 128, 128, 'e4m3')
  return (f(x, 1, 128, 'e4m3') @ wq, f(g, 1, 128, 'e5m2') @ wq.T,
          f(x, 128, 1, 'e4m3').T @ f(g, 128, 1, 'e5m2'))


def _same(got, want, half):
  got = _np(got).astype(np.float64)
  assert got.shape == want.shape
  # computed in 64 bits and rounded through f32: half a step each
  tol = (half + 2.0 ** -24) * np.abs(want) + 2.0 ** -120
  assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize('m,k,n', [(1, 5, 3), (40, 200, 136), (130, 129, 257)])
@pytest.mark.parametrize('rhs_axis', [0, 1])
@pytest.mark.parametrize('lhs_t', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_dot_step(m, k, n, rhs_axis, lhs_t, dtype):
  x, w, g = (_data((m, k), dtype, 2), _data((k, n), dtype, 3, 0.3), _data(
      (m, n), dtype, 4))
  a = x.t().contiguous() if lhs_t else _off(x)
  b = w.t().contiguous() if rhs_axis else w
  dims = (((0 if lhs_t else 1,), (rhs_axis,)), ((), ()))
  out, bp = bs.dot_general_make().vjp(a, b, dims)
  dl, dr = bp(_off(g))
  want = _dot_want(_np(x), _np(w), _np(g))
  _same(out, want[0], HALF[dtype])
  _same(dl, want[1].T if lhs_t else want[1], HALF[dtype])
  _same(dr, want[2].T if rhs_axis else want[2], HALF[dtype])


def test_dot_shapes_and_frozen():
  x, w = _data((2, 3, 200), torch.bfloat16, 5), _data((200, 24), torch.bfloat16, 6)
  cfg = bs.dot_general_make()
  plain = cfg(x.reshape(6, 200), w, DIMS)
  assert torch.equal(cfg(x, w, (((2,), (0,)), ((), ()))), plain.view(2, 3, 24))
  assert torch.equal(cfg(x, w, (((-1,), (-2,)), ((), ()))), plain.view(2, 3, 24))
  assert torch.equal(aqt_dot_general.einsum('abk,kn->abn', x, w, dg=cfg),
                     plain.view(2, 3, 24))
  assert torch.equal(cfg(x[1, 2], w, (((0,), (0,)), ((), ()))), plain[5])
  qt = bs.block_quantize(w, 0, square=True)
  assert torch.equal(cfg(x.reshape(6, 200), qt, DIMS), plain)
  again = bs.frozen(qt.qvalue.contiguous(), qt.scale[0])
  assert torch.equal(cfg(x.reshape(6, 200), again, DIMS), plain)
  qt = bs.block_quantize(w.t().contiguous(), 1, square=True)
  assert torch.equal(cfg(x.reshape(6, 200), qt, (((1,), (1,)), ((), ()))), plain)


def test_dot_autograd():
  x, w, g = (_data((9, 40), torch.float32, 7), _data((40, 24), torch.float32, 8),
             _data((9, 24), torch.float32, 9))
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
  # no second derivative: refused, not silently zero
  a, h = x.clone().requires_grad_(), g.clone().requires_grad_()
  first, = torch.autograd.grad(cfg(a, w, DIMS), a, h, create_graph=True)
  with pytest.raises(RuntimeError, match='once_differentiable'):
    first.sum().backward()
  with pytest.raises(ValueError, match='cotangent'):
    bp(g[:4])


RAGGED = [(1, 8, 8, [1]), (7, 200, 24, [3, 0, 2]), (300, 40, 72, [130, 0, 129]),
          (20, 16, 8, [-3, 15, 9]), (6, 8, 16, [0, 0])]


@pytest.mark.parametrize('m,k,n,sizes', RAGGED)
@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('layout', [lambda t: t, _off, _flip])
def test_ragged_step(m, k, n, sizes, q, index, layout):
  x, w, g = (_data((m, k), torch.bfloat16, 10), _data(
      (len(sizes), k, n), torch.bfloat16, 11, 0.2), _data((m, n), torch.bfloat16, 12))
  out, bp = rd.ragged_dot_vjp(layout(x), layout(w), torch.tensor(sizes, dtype=index),
                              cfg=bs.dot_general_make() if q else None)
  dl, dr = bp(layout(g))
  xs, ws, gs = _np(x), _np(w), _np(g)
  want = [np.zeros((m, n)), np.zeros((m, k)), np.zeros((len(sizes), k, n))]
  for e, (a, b) in enumerate(ref.spans(sizes, m)):
    if b > a:
      part = (_dot_want(xs[a:b], ws[e], gs[a:b]) if q else
              tuple(v.astype(np.float64) for v in (
                  xs[a:b].astype(np.float64) @ ws[e],
                  gs[a:b].astype(np.float64) @ ws[e].T,
                  xs[a:b].T.astype(np.float64) @ gs[a:b])))
      want[0][a:b], want[1][a:b], want[2][e] = part
  for got, value in zip((out, dl, dr), want):
    _same(got, value, 2.0 ** -8)


def test_ragged_frozen_and_autograd():
  m, k, n, sizes = 12, 40, 24, [5, 0, 6]
  x, w, g = (_data((m, k), torch.bfloat16, 13), _data(
      (3, k, n), torch.bfloat16, 14), _data((m, n), torch.bfloat16, 15))
  s = torch.tensor(sizes)
  for cfg in (None, bs.dot_general_make()):
    out, bp = rd.ragged_dot_vjp(x, w, s, cfg=cfg)
    dl, dr = bp(g)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = rd.ragged_dot(a, b, s, cfg=cfg)
    y.backward(g)
    assert torch.equal(y, out) and torch.equal(a.grad, dl)
    assert torch.equal(b.grad, dr)
    # sizes written over before the backward pass are noticed
    y = rd.ragged_dot(a, b, s, cfg=cfg)
    s.add_(0)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
      y.backward(g)
    if cfg is not None:
      qt = bs.block_quantize(w, 1, square=True)
      assert torch.equal(rd.ragged_dot(x, qt, s, cfg=cfg), out)


def test_scales_named_powers_of_two_are(monkeypatch):
  """The product is told so exactly where every scale it gets is one."""
  import ctypes as C
  from aqt_b200 import _lib
  lib = _lib.load()
  told = []
  gemm = lib.aqtb200_grouped_gemm

  def spy(desc, *args):
    d = desc._obj
    told.append(d.scales_po2)
    if d.scales_po2:
      nb = -(-d.k // 128)
      b = np.frombuffer((C.c_char * (4 * nb * d.t)).from_address(d.b_scale),
                        np.float32)
      if not d.group_sizes or d.contract_groups == 0:
        assert (np.frexp(b)[0] == 0.5).all()
    return gemm(desc, *args)

  monkeypatch.setattr(lib, 'aqtb200_grouped_gemm', spy, raising=False)
  x, w, g = (_data((140, 200), torch.bfloat16, 60), _data(
      (200, 30), torch.bfloat16, 61), _data((140, 30), torch.bfloat16, 62))
  s = torch.tensor([100, 40], dtype=torch.int32)
  wg = _data((2, 200, 30), torch.bfloat16, 63)
  for po2 in (False, True):
    cfg = bs.dot_general_make(po2_scale=po2)
    for run in (lambda: cfg.vjp(x, w, DIMS),
                lambda: rd.ragged_dot_vjp(x, wg, s, cfg=cfg)):
      told.clear()
      run()[1](g)
      assert told == [int(po2)] * 3
    told.clear()
    cfg(x, bs.block_quantize(w, 0, square=True), DIMS)
    rd.ragged_dot(x, bs.block_quantize(wg, 1, square=True), s, cfg=cfg)
    rd.ragged_dot(x, wg, s)
    assert told == [0, 0, 0]


@pytest.mark.parametrize('lhs_copy,rhs_copy', [(True, False), (False, True),
                                               (True, True)])
def test_ragged_copies_are_made_once(monkeypatch, lhs_copy, rhs_copy):
  """Operands no tensor map describes are copied once a step; the backward pass
  reads the copies."""
  from aqt_b200 import _lib
  m, k, n, sizes = 20, 24 + 5 * lhs_copy, 16, [8, 0, 9]
  x = _data((m, k), torch.bfloat16, 70)
  w = _data((3, k, n), torch.bfloat16, 71)
  if rhs_copy:
    w = _off(w)
  g, s = _data((m, n), torch.bfloat16, 72), torch.tensor(sizes)
  lib = _lib.load()
  calls = []
  pack = lib.aqtb200_pack_bf16_groups
  monkeypatch.setattr(
      lib, 'aqtb200_pack_bf16_groups',
      lambda *a: calls.append(a[1]) or pack(*a), raising=False)
  a = x.clone().requires_grad_()
  b = (_off(w) if rhs_copy else w.clone()).requires_grad_()
  y = rd.ragged_dot(a, b, s)
  y.backward(g)
  # lhs, rhs (with the sizes: empty groups are skipped); g needs none
  assert sorted(bool(c) for c in calls) == [False] * lhs_copy + [True] * rhs_copy
  x64, w64, g64 = (_np(t).astype(np.float64) for t in (x, w, g))
  _same(y, ref.ragged(x64, w64, sizes)[0], 2.0 ** -8)
  _same(a.grad, ref.ragged(g64, w64.transpose(0, 2, 1), sizes)[0], 2.0 ** -8)
  _same(b.grad, ref.ragged_drhs(x64, g64, sizes, 3)[0], 2.0 ** -8)
  # twice through the same graph
  a.grad = b.grad = None
  y = rd.ragged_dot(a, b, s)
  y.backward(g, retain_graph=True)
  once = a.grad.clone(), b.grad.clone()
  a.grad = b.grad = None
  y.backward(g)
  assert torch.equal(a.grad, once[0]) and torch.equal(b.grad, once[1])
  out, bp = rd.ragged_dot_vjp(x, w, s)
  p, q = bp(g)
  p2, q2 = bp(g)
  assert torch.equal(p, p2) and torch.equal(q, q2)


def test_products_that_follow_their_quantizer(monkeypatch):
  """A product is launched early exactly where the call before it is the one that
  wrote its tokens and their scales, and nothing else of it."""
  from aqt_b200 import _lib
  lib = _lib.load()
  seen = []
  quantize, gemm = lib.aqtb200_block_quantize, lib.aqtb200_grouped_gemm

  def q(desc, *args):
    d = desc._obj
    seen.append([d.q_row, d.q_col, d.scale_row, d.scale_col])
    return quantize(desc, *args)

  def mm(desc, *args):
    d = desc._obj
    if d.follows_quantize:
      wrote = [p for p in seen[-1] if p]
      assert d.contract_groups == 0 and d.b in wrote and d.b_scale in wrote
      assert d.a not in wrote and d.a_scale not in wrote
    seen.append(d.follows_quantize)
    return gemm(desc, *args)

  monkeypatch.setattr(lib, 'aqtb200_block_quantize', q, raising=False)
  monkeypatch.setattr(lib, 'aqtb200_grouped_gemm', mm, raising=False)
  x, w, g = (_data((140, 200), torch.bfloat16, 80), _data(
      (200, 30), torch.bfloat16, 81), _data((140, 30), torch.bfloat16, 82))
  s = torch.tensor([100, 40], dtype=torch.int32)
  wg = _data((2, 200, 30), torch.bfloat16, 83)
  cfg = bs.dot_general_make()
  flags = lambda: [v for v in seen if not isinstance(v, list)]
  for run in (lambda: cfg.vjp(x, w, DIMS)[1](g),
              lambda: cfg.vjp(x, w.t().contiguous(), (((1,), (1,)), ((), ())))[1](g),
              lambda: rd.ragged_dot_vjp(x, wg, s, cfg=cfg)[1](g)):
    seen.clear()
    run()
    assert flags() == [1, 1, 0]
  seen.clear()
  cfg(x, bs.block_quantize(w, 0, square=True), DIMS)
  rd.ragged_dot(x, bs.block_quantize(wg, 1, square=True), s, cfg=cfg)
  rd.ragged_dot(x, wg, s)
  assert flags() == [1, 1, 0]


@pytest.fixture
def temporaries(monkeypatch):
  """Conversions torch makes stay allocated, as in the blocks of a caching
  allocator that nobody has been given yet."""
  held = []
  to = torch.Tensor.to

  def hold(t, *args, **kw):
    held.append(to(t, *args, **kw))
    return held[-1]

  monkeypatch.setattr(torch.Tensor, 'to', hold)
  return held


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', [lambda t: t, _off, _flip])
@pytest.mark.parametrize('q', [False, True])
def test_traced_ragged_step_reads_the_new_cotangent(temporaries, dtype, layout, q):
  """A replayed step follows its operands, a float32 cotangent among them, which
  the bfloat16 products need rounded."""
  m, k, n = 12, 40, 24
  x, w, s = (_data((m, k), torch.bfloat16, 90), _data(
      (3, k, n), torch.bfloat16, 91), torch.tensor([5, 0, 6]))
  g = layout(_data((m, n), dtype, 92))
  cfg = bs.dot_general_make() if q else None

  def step(x, w, g):
    out, bp = rd.ragged_dot_vjp(x, w, s, cfg=cfg, preferred_element_type=dtype)
    return (out, *bp(g))

  temporaries.clear()
  traced = engine.TracedStep(step, x, w, g)
  inside = list(temporaries)
  for i in range(2):
    for t, seed in ((x, 93), (w, 94), (g, 95)):
      t.copy_(_data(t.shape, t.dtype, seed + 10 * i))
    for t in inside:
      t.fill_(7)  # handed to somebody else meanwhile
    got = [t.clone() for t in traced(x, w, g)]
    for a, b in zip(got, step(x, w, g)):
      assert torch.equal(a, b)


@pytest.mark.parametrize('k,n', [(200, 24), (256, 130)])
@pytest.mark.parametrize('ragged', [False, True])
def test_traced_step_that_freezes_weights(monkeypatch, k, n, ragged):
  """Values of another layout, brought into the product's inside the step."""
  held = []
  zeros = torch.zeros
  monkeypatch.setattr(torch, 'zeros',
                      lambda *a, **kw: held.append(zeros(*a, **kw)) or held[-1])
  lead = (2,) if ragged else ()
  qt = bs.block_quantize(_data((*lead, k, n), torch.bfloat16, 96), -2, square=True)
  other = bs.block_quantize(_data((*lead, k, n), torch.bfloat16, 97), -2, square=True)
  values, scales = qt.qvalue.contiguous(), qt.scale[0].clone()
  x, s = _data((9, k), torch.bfloat16, 98), torch.tensor([4, 4])
  cfg = bs.dot_general_make()

  def step(x):
    w = bs.frozen(values, scales)
    return rd.ragged_dot(x, w, s, cfg=cfg) if ragged else cfg(x, w, DIMS)

  held.clear()
  traced = engine.TracedStep(step, x)
  for t in held:
    t.fill_(9)  # handed to somebody else meanwhile
  assert torch.equal(traced(x), step(x))
  values.copy_(other.qvalue)
  scales.copy_(other.scale[0])
  assert torch.equal(traced(x), step(x))


@pytest.fixture
def gives_up(monkeypatch):
  """Products that report a wait that ran out, as many as the list says."""
  import ctypes as C
  from aqt_b200 import _lib
  lib = _lib.load()
  gemm, left = lib.aqtb200_grouped_gemm, []

  def failing(desc, status, stream):
    if left:
      (C.c_int32 * 4).from_address(status)[0] = left.pop()
    return gemm(desc, status, stream)

  monkeypatch.setattr(lib, 'aqtb200_grouped_gemm', failing, raising=False)
  yield left
  engine._words.clear()  # pylint: disable=protected-access


@pytest.mark.parametrize('run', ['dot', 'frozen', 'ragged', 'ragged fp8'])
def test_a_product_that_gave_up_is_reported(gives_up, run):
  from aqt_b200 import _lib
  x, w = _data((9, 40), torch.bfloat16, 100), _data((40, 24), torch.bfloat16, 101)
  s, cfg = torch.tensor([9]), bs.dot_general_make()
  call = {'dot': lambda: cfg(x, w, DIMS),
          'frozen': lambda: cfg(x, bs.block_quantize(w, 0, square=True), DIMS),
          'ragged': lambda: rd.ragged_dot(x, w[None], s),
          'ragged fp8': lambda: rd.ragged_dot(x, w[None], s, cfg=cfg)}[run]
  good = call()
  gives_up.append(3)
  call()
  with pytest.raises(_lib.AqtB200Error, match='role 3'):
    call()
  assert torch.equal(call(), good)  # said once
  gives_up.append(1)
  call()
  with pytest.raises(_lib.AqtB200Error, match='role 1'):
    engine.check_status()
  engine.check_status()
  traced = engine.TracedStep(lambda a: call(), x)
  gives_up.append(2)
  traced(x)
  with pytest.raises(_lib.AqtB200Error, match='role 2'):
    traced(x)


def _graphs():
  """name -> (leaves, cotangent, product of the leaves)."""
  m, k, n, s = 12, 41, 24, torch.tensor([5, 0, 6])
  cfg = bs.dot_general_make()
  x, g = _data((m, k), torch.bfloat16, 110), _data((m, n), torch.bfloat16, 111)
  w = _data((3, k, n), torch.bfloat16, 112)
  return {
      'dot': ([x, w[0]], g, lambda a, b: cfg(a, b, DIMS)),
      'ragged': ([x, w], g, lambda a, b: rd.ragged_dot(a, b, s)),
      'ragged own': ([x[:, :40], w[:, :40]], g,
                     lambda a, b: rd.ragged_dot(a, b, s)),
      'ragged fp8': ([x, w], g, lambda a, b: rd.ragged_dot(a, b, s, cfg=cfg)),
  }


GRAPHS = ['dot', 'ragged', 'ragged own', 'ragged fp8']


def _leaves(tensors):
  return [t.clone().contiguous().requires_grad_() for t in tensors]


@pytest.mark.parametrize('name', GRAPHS)
def test_a_graph_is_used_up_by_its_backward_pass(name):
  """As torch's own products: a second pass needs retain_graph, and what was kept
  for the first goes with it although the result lives on."""
  import gc
  import weakref
  from aqt_b200 import block_engine as be
  tensors, g, run = _graphs()[name]
  leaves = _leaves(tensors)
  made = []

  def watch(f):
    def made_one(*args):
      t = f(*args)
      made.append(weakref.ref(t))
      return t
    return made_one

  real = {f: getattr(be, f) for f in ('_scratch', '_empty_out')}
  try:
    for f in real:
      setattr(be, f, watch(real[f]))
    y = run(*leaves)
  finally:
    for f in real:
      setattr(be, f, real[f])
  gc.collect()
  y.backward(g, retain_graph=True)
  once = [t.grad.clone() for t in leaves]
  for t in leaves:
    t.grad = None
  y.backward(g)
  assert all(torch.equal(t.grad, o) for t, o in zip(leaves, once))
  gc.collect()
  left = [r() for r in made if r() is not None and r() is not y]
  assert not left
  with pytest.raises(RuntimeError, match='second time'):
    y.backward(g)


@pytest.mark.parametrize('name', GRAPHS)
@pytest.mark.parametrize('strided', [False, True])
def test_hooks_on_saved_tensors_see_the_residuals(name, strided):
  """Offloading and the like: what the hooks give back is what is read."""
  tensors, g, run = _graphs()[name]
  a = _leaves(tensors)
  run(*a).backward(g)
  b = _leaves(tensors)
  packed = []

  def pack(t):
    packed.append(t)
    return t.detach().clone()

  def unpack(t):
    if not strided:
      return t
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype)
    wide[..., 0] = t
    return wide[..., 0]  # the same values, elements apart

  with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
    y = run(*b)
  own = {leaf.data_ptr() for leaf in b}
  for t in packed:
    if t.data_ptr() not in own and t.dtype in (torch.uint8, torch.bfloat16):
      t.detach().zero_()  # its memory is somebody else's from here on
  y.backward(g)
  assert len(packed) >= 2
  for s, t in zip(a, b):
    assert torch.equal(s.grad, t.grad)
