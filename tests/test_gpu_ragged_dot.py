"""Products grouped by expert on the GPU against the definition in 64 bits."""

import numpy as np
import pytest
import torch

from aqt_b200 import block_engine as be
from aqt_b200 import engine
from aqt_b200.v2 import aqt_ragged_dot as rd
from aqt_b200.v2 import block_scaled as bs
from tests import block_ref as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _data(shape, dtype, seed, scale=1.0):
  rng = np.random.default_rng(seed)
  return torch.from_numpy((rng.standard_normal(shape) * scale).astype(
      np.float32)).to(dtype).cuda()


def _f32(t):
  return t.float().cpu().numpy()


def _done():
  torch.cuda.synchronize()
  engine.check_status()


def _sizes(values, dtype=torch.int32):
  return torch.tensor(values, dtype=dtype, device='cuda')


def _want(x, w, g, sizes, q, po2=False, fwd='e4m3', bwd='e5m2'):
  x, w, g = (np.asarray(v, np.float64) for v in (x, w, g))
  if not q:
    pairs = (x, w, g, x, g)
  else:
    f = lambda v, br, bc, b: ref.fake(v, br, bc, b, po2)
    xt, gt = np.zeros_like(x), np.zeros_like(g)
    for a, b in ref.spans(sizes, len(x)):
      if b > a:  # blocks along the rows start at each group's first row
        xt[a:b], gt[a:b] = f(x[a:b], 128, 1, fwd), f(g[a:b], 128, 1, bwd)
    pairs = (f(x, 1, 128, fwd), np.stack([f(m, 128, 128, fwd) for m in w]),
             f(g, 1, 128, bwd), xt, gt)
  xr, wq, gr, xt, gt = pairs
  k, n = w.shape[1:]
  out = (*ref.ragged(xr, wq, sizes), k)
  dl = (*ref.ragged(gr, wq.transpose(0, 2, 1), sizes), n)
  dr = (*ref.ragged_drhs(xt, gt, sizes, len(w)), len(x))
  return out, dl, dr


def _check(got, want, half, what):
  value, mag, k = want
  ref.assert_close(_f32(got).astype(np.float64), value, mag, k, half, what)


# rows, K, N, group sizes
CASES = [
    (1, 64, 64, [1]),
    (1, 64, 72, [0, 1, 0]),
    (5, 8, 8, [0, 0, 0]),                       # every row behind the last group
    (40, 200, 136, [40]),
    (300, 264, 520, [1, 0, 63, 64, 65, 100]),   # seven rows left over
    (300, 129, 77, [128, 129, 43]),             # odd strides
    (513, 384, 256, [256, 257]),
    (700, 136, 264, [0, 700, 0]),
    (90, 72, 96, [30] * 40),                    # more than there are rows
    (90, 72, 96, [-5, 40, -1, 60]),             # negative sizes, cut at the end
    (70, 64, 64, [2] * 35),
]


@pytest.mark.parametrize('m,k,n,sizes', CASES)
@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_step_matches_definition(m, k, n, sizes, q, index):
  x, w, g = (_data((m, k), torch.bfloat16, 1), _data(
      (len(sizes), k, n), torch.bfloat16, 2, 0.1), _data((m, n), torch.bfloat16, 3))
  cfg = bs.dot_general_make() if q else None
  out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes, index), cfg=cfg)
  dl, dr = bp(g)
  _done()
  want = _want(_f32(x), _f32(w), _f32(g), sizes, q)
  for name, got, wt in zip(('out', 'dlhs', 'drhs'), (out, dl, dr), want):
    assert got.dtype == torch.bfloat16
    _check(got, wt, 2.0 ** -8, name)
  left = max(b for _, b in ref.spans(sizes, m))
  assert not out[left:].any() and not dl[left:].any()


@pytest.mark.parametrize('m,k,n,sizes', CASES)
def test_float32_operands_and_results(m, k, n, sizes):
  x, w, g = (_data((m, k), torch.float32, 4), _data(
      (len(sizes), k, n), torch.float32, 5, 0.1), _data((m, n), torch.float32, 6))
  cfg = bs.dot_general_make('e4m3', 'e4m3', po2_scale=True)
  out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), cfg=cfg)
  dl, dr = bp(g)
  _done()
  for got, wt in zip((out, dl, dr), _want(_f32(x), _f32(w), _f32(g), sizes, True,
                                          True, 'e4m3', 'e4m3')):
    assert got.dtype == torch.float32
    _check(got, wt, 2.0 ** -24, '')
  xb, wb = x.bfloat16(), w.bfloat16()
  out = rd.ragged_dot(xb, wb, _sizes(sizes), preferred_element_type=torch.float32)
  _done()
  assert out.dtype == torch.float32
  _check(out, _want(_f32(xb), _f32(wb), _f32(g), sizes, False)[0], 2.0 ** -24, '')


@pytest.mark.parametrize('m,k,n,sizes', CASES)
def test_frozen_weights(m, k, n, sizes):
  x, w, g = (_data((m, k), torch.bfloat16, 7), _data(
      (len(sizes), k, n), torch.bfloat16, 8, 0.1), np.zeros((m, n)))
  qt = bs.block_quantize(w, contract_axis=1, square=True)
  again = bs.frozen(qt.qvalue.contiguous(), qt.scale[0].clone())
  want = _want(_f32(x), _f32(w), g, sizes, True)[0]
  for t in (qt, again):
    out = rd.ragged_dot(x, t, _sizes(sizes), cfg=bs.dot_general_make())
    _done()
    _check(out, want, 2.0 ** -8, '')


def test_long_decode_shares_the_contraction():
  """One or two rows against long contractions: few tiles, so each one's
  contraction is divided; the result must not depend on it."""
  for m, sizes in ((1, [1]), (2, [1, 1]), (33, [33])):
    for q in (False, True):
      x, w = _data((m, 4104), torch.bfloat16, 9), _data(
          (len(sizes), 4104, 264), torch.bfloat16, 10, 0.05)
      cfg = bs.dot_general_make() if q else None
      a = rd.ragged_dot(x, w, _sizes(sizes), cfg=cfg)
      b = rd.ragged_dot(x, w, _sizes(sizes), cfg=cfg)
      _done()
      assert torch.equal(a, b)
      _check(a, _want(_f32(x), _f32(w), np.zeros((m, 264)), sizes, q)[0],
             2.0 ** -8, '')


def test_many_groups():
  g = 1024
  rng = np.random.default_rng(11)
  sizes = rng.integers(0, 3, g)
  m = int(sizes.sum()) + 4
  x, w = _data((m, 64), torch.bfloat16, 12), _data((g, 64, 32), torch.bfloat16, 13)
  ct = _data((m, 32), torch.bfloat16, 14)
  for q in (False, True):
    out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes),
                                cfg=bs.dot_general_make() if q else None)
    dl, dr = bp(ct)
    _done()
    for got, wt in zip((out, dl, dr), _want(_f32(x), _f32(w), _f32(ct), sizes, q)):
      _check(got, wt, 2.0 ** -8, '')


@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_groups_do_not_mix(q, bad):
  """What lies in other groups' rows, or behind the last group, reaches nothing."""
  m, k, n, sizes = 200, 136, 72, [30, 0, 70, 50]
  x, w, g = (_data((m, k), torch.bfloat16, 15), _data(
      (4, k, n), torch.bfloat16, 16), _data((m, n), torch.bfloat16, 17))
  cfg = bs.dot_general_make() if q else None

  def step():
    out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), cfg=cfg)
    return (out, *bp(g))

  out, dl, dr = step()
  x[150:] = bad
  g[150:] = bad
  x[30, 5] = bad   # first row of the third group
  g[99, 7] = bad   # its last row
  out2, dl2, dr2 = step()
  _done()
  keep = [i for i in range(200) if not 30 <= i < 100]
  assert torch.equal(out[keep], out2[keep]) and torch.equal(dl[keep], dl2[keep])
  assert not out2[150:].any() and not dl2[150:].any()
  for e in (0, 1, 3):
    assert torch.equal(dr[e], dr2[e]), e
  assert not torch.isfinite(out2[30]).any()
  assert not torch.isfinite(dr2[2, 5]).any()


@pytest.mark.parametrize('q', [False, True])
def test_any_strides(q):
  m, k, n, sizes = 150, 72, 88, [50, 60, 30]
  x, w, g = (_data((m, k), torch.bfloat16, 18), _data(
      (3, k, n), torch.bfloat16, 19), _data((m, n), torch.bfloat16, 20))
  cfg = bs.dot_general_make() if q else None

  def step(a, b, c):
    out, bp = rd.ragged_dot_vjp(a, b, _sizes(sizes), cfg=cfg)
    return (out, *bp(c))

  want = step(x, w, g)

  def off(t):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 9, dtype=t.dtype,
                       device=t.device)
    wide[..., 1:1 + t.shape[-1]] = t
    return wide[..., 1:1 + t.shape[-1]]

  flip = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)
  every = torch.zeros(6, k, n, dtype=w.dtype, device='cuda')
  every[::2] = w
  for a, b, c in ((off(x), off(w), off(g)), (flip(x), flip(w), flip(g)),
                  (x, every[::2], g), (x[:, :], w, g)):
    got = step(a, b, c)
    _done()
    for s, t in zip(got, want):
      assert torch.equal(s, t)


def test_broadcast_weights():
  """One matrix for every group (stride 0): gradients come per group."""
  m, k, n, sizes = 60, 64, 48, [20, 10, 30]
  x, one, g = (_data((m, k), torch.bfloat16, 21), _data(
      (k, n), torch.bfloat16, 22), _data((m, n), torch.bfloat16, 23))
  for q in (False, True):
    cfg = bs.dot_general_make() if q else None
    leaf = one.clone().requires_grad_()
    out = rd.ragged_dot(x, leaf.expand(3, k, n), _sizes(sizes), cfg=cfg)
    out.backward(g)
    _, bp = rd.ragged_dot_vjp(x, one.expand(3, k, n).contiguous(), _sizes(sizes),
                              cfg=cfg)
    want = bp(g)[1].sum(0)
    _done()
    assert torch.equal(leaf.grad, want)


def test_autograd_matches_vjp():
  m, k, n, sizes = 100, 72, 64, [40, 0, 55]
  x, w, g = (_data((m, k), torch.bfloat16, 24), _data(
      (3, k, n), torch.bfloat16, 25), _data((m, n), torch.bfloat16, 26))
  for q in (False, True):
    cfg = bs.dot_general_make() if q else None
    out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), cfg=cfg)
    dl, dr = bp(g)
    for need_l, need_r in ((True, True), (True, False), (False, True)):
      a, b = x.clone().requires_grad_(need_l), w.clone().requires_grad_(need_r)
      y = rd.ragged_dot(a, b, _sizes(sizes), cfg=cfg)
      y.backward(g, retain_graph=True)
      assert torch.equal(y, out)
      assert torch.equal(a.grad, dl) if need_l else a.grad is None
      assert torch.equal(b.grad, dr) if need_r else b.grad is None
      y.backward(g)  # a second time, from the same residuals
    _done()


def test_gradients_against_differences():
  rng = np.random.default_rng(27)
  ints = lambda *s: torch.from_numpy(
      rng.integers(-3, 4, s).astype(np.float32)).cuda()
  sizes = [3, 0, 4]
  x, w, g = ints(8, 16), ints(3, 16, 8), ints(8, 8)
  out, bp = rd.ragged_dot_vjp(x.bfloat16(), w.bfloat16(), _sizes(sizes))
  dl, dr = bp(g.bfloat16())
  _done()
  x64, w64, g64 = (_f32(t).astype(np.float64) for t in (x, w, g))
  loss = lambda a, b: float((ref.ragged(a, b, sizes)[0] * g64).sum())
  for i, j in ((0, 1), (6, 15), (7, 3)):
    d = np.zeros_like(x64)
    d[i, j] = 1
    assert float(dl[i, j]) == (loss(x64 + d, w64) - loss(x64 - d, w64)) / 2
  for e, i, j in ((0, 1, 0), (1, 2, 2), (2, 15, 7)):
    d = np.zeros_like(w64)
    d[e, i, j] = 1
    assert float(dr[e, i, j]) == (loss(x64, w64 + d) - loss(x64, w64 - d)) / 2


def test_empty_extents():
  for q in (False, True):
    cfg = bs.dot_general_make() if q else None
    for m, k, n in ((0, 64, 32), (4, 0, 32), (4, 64, 0)):
      x = torch.ones(m, k, device='cuda', dtype=torch.bfloat16)
      w = torch.ones(2, k, n, device='cuda', dtype=torch.bfloat16)
      out, bp = rd.ragged_dot_vjp(x, w, _sizes([m // 2, m // 2]), cfg=cfg)
      dl, dr = bp(torch.ones(m, n, device='cuda', dtype=torch.bfloat16))
      _done()
      assert tuple(out.shape) == (m, n) and not out.any()
      assert dl.shape == x.shape and not dl.any()
      assert dr.shape == w.shape and not dr.any()


@pytest.mark.parametrize('q', [False, True])
def test_captured_with_other_sizes_at_replay(q):
  """The sizes are read by the kernels: a captured step follows new ones."""
  m, k, n = 120, 136, 72
  x, w, g = (_data((m, k), torch.bfloat16, 28), _data(
      (4, k, n), torch.bfloat16, 29), _data((m, n), torch.bfloat16, 30))
  sizes = _sizes([30, 30, 30, 30])
  cfg = bs.dot_general_make() if q else None

  def step():
    out, bp = rd.ragged_dot_vjp(x, w, sizes, cfg=cfg)
    return (out, *bp(g))

  step()
  torch.cuda.synchronize()
  graphs, outs = [], []
  for _ in range(2):  # two graphs alive at once
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      outs.append(step())
    graphs.append(graph)
  for values in ([0, 119, 1, 0], [64, 0, 3, 20], [1, 1, 1, 117]):
    sizes.copy_(_sizes(values))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      graphs[1].replay()
    graphs[0].replay()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    _done()
    for got in outs:
      for s, t in zip(got, want):
        assert torch.equal(s, t)


def test_expert_layer():
  """Router, experts and their gradients together, as a model runs them: rows
  sorted by expert, gate and up products, a gated product, the down product,
  weighted and added back; against the same layer in 64 bits."""
  tokens, d, f, e, top = 96, 128, 192, 6, 2
  x = _data((tokens, d), torch.bfloat16, 31)
  router = _data((d, e), torch.float32, 32, 0.2)
  ws = [_data((e, d, f), torch.bfloat16, 33, 0.1), _data(
      (e, d, f), torch.bfloat16, 34, 0.1), _data((e, f, d), torch.bfloat16, 35, 0.1)]
  p, chosen = torch.softmax(x.float() @ router, -1).topk(top, -1)
  expert = chosen.reshape(-1)
  order = expert.argsort(stable=True)
  sizes = torch.bincount(expert, minlength=e).to(torch.int32)
  row = order // top
  weight = p.reshape(-1)[order]
  ct = _data((tokens, d), torch.float32, 36)

  def layer(x, ws, product, cast):
    rows = x[row]
    gate, up = product(rows, ws[0]), product(rows, ws[1])
    hidden = cast(torch.nn.functional.silu(gate.double()) * up.double())
    down = product(hidden, ws[2]).double() * weight.double()[:, None]
    return torch.zeros(tokens, d, dtype=torch.float64, device='cuda').index_add(
        0, row, down)

  def run(cfg, exact):
    leaves = [t.double().requires_grad_() if exact else
              t.clone().requires_grad_() for t in [x] + ws]
    ends = sizes.cumsum(0).tolist()
    if exact:
      def product(a, w):
        return torch.cat([a[b:c] @ w[i] for i, (b, c) in enumerate(
            zip([0] + ends[:-1], ends))])
      y = layer(leaves[0], leaves[1:], product, lambda t: t)
    else:
      y = layer(leaves[0], leaves[1:],
                lambda a, w: rd.ragged_dot(a, w, sizes, cfg=cfg),
                lambda t: t.bfloat16())
    (y * ct.double()).sum().backward()
    return [y.detach()] + [t.grad.double() for t in leaves]

  want = run(None, True)
  # relative error, in the 2-norm, of a chain of three products: bf16 rounds
  # operands and results by 2^-8 at most, four times along the longest path and
  # its gradient twice that; fp8 operands are off by at most 2^-4 (e4m3) or 2^-3
  # (e5m2) each, two operands a product
  for cfg, tol in ((None, 8 * 2.0 ** -8 * 2), (bs.dot_general_make(
      'e4m3', 'e4m3'), 6 * 2 * 2.0 ** -4)):
    got = run(cfg, False)
    _done()
    for a, b in zip(got, want):
      assert float((a - b).norm() / b.norm()) < tol


@pytest.mark.parametrize('what', ['bf16', 'frozen', 'backward'])
def test_first_call_of_a_thread(what):
  """A thread that has made no CUDA call yet."""
  import threading
  x, w, g = (_data((40, 64), torch.bfloat16, 60), _data(
      (2, 64, 72), torch.bfloat16, 61), _data((40, 72), torch.bfloat16, 62))
  sizes = _sizes([25, 10])
  cfg = bs.dot_general_make()
  if what == 'bf16':
    run = lambda: (rd.ragged_dot(x, w, sizes),)
  elif what == 'frozen':
    qt = bs.block_quantize(w, 1, square=True)
    run = lambda: (rd.ragged_dot(x, qt, sizes, cfg=cfg),)
  else:
    back = rd.ragged_dot_vjp(x, w, sizes)[1]
    run = lambda: back(g)
  want = run()
  _done()
  got = []
  t = threading.Thread(target=lambda: got.extend(run()))
  t.start()
  t.join()
  _done()
  assert len(got) == len(want)
  assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_copies_of_experts_without_rows_are_left_out():
  """Rows no tensor map describes: only the matrices in use are copied, the
  places of the others hold whatever they held."""
  g, k, n = 40, 133, 77
  sizes = [0] * g
  sizes[3], sizes[17], sizes[39] = 5, 1, 2
  x, w, ct = (_data((9, k), torch.bfloat16, 50), _data(
      (g, k, n), torch.bfloat16, 51, 0.1), _data((9, n), torch.bfloat16, 52))
  # memory the allocator hands out next: NaN
  torch.full((4 * g * k * 80,), float('nan'), dtype=torch.bfloat16, device='cuda')
  for index in (torch.int32, torch.int64):
    out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes, index))
    dl, dr = bp(ct)
    _done()
    for got, wt in zip((out, dl, dr), _want(_f32(x), _f32(w), _f32(ct), sizes,
                                            False)):
      _check(got, wt, 2.0 ** -8, '')


@pytest.mark.parametrize('m,k,n,sizes', [
    (3000, 1400, 1304, [0, 700, 1, 1500, 130, 600]),
    (2500, 1401, 1303, [1250, 1249]),
    (5000, 72, 1800, [300, 0, 900, 64, 2000, 1, 257, 1400])])
@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
def test_step_in_wide_tiles(m, k, n, sizes, q, out):
  """More tiles of 128 columns than the device holds at once."""
  x, w, g = (_data((m, k), torch.bfloat16, 53), _data(
      (len(sizes), k, n), torch.bfloat16, 54, 0.1), _data((m, n), out, 55))
  y, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), preferred_element_type=out,
                            cfg=bs.dot_general_make() if q else None)
  dl, dr = bp(g)
  _done()
  assert y.dtype == out
  gf = g if q else g.bfloat16()  # without cfg cotangents are bfloat16
  for name, got, wt in zip(('out', 'dlhs', 'drhs'), (y, dl, dr),
                           _want(_f32(x), _f32(w), _f32(gf), sizes, q)):
    _check(got, wt, HALF[got.dtype], name)
  left = sum(sizes)
  assert not y[left:].any() and not dl[left:].any()


@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_traced_step(q, dtype):
  """Replayed on new operands, after other work has used the memory between."""
  m, k, n = 130, 136, 77
  x, w, g = (_data((m, k), torch.bfloat16, 63), _data(
      (3, k, n), torch.bfloat16, 64, 0.1), _data((m, n), dtype, 65))
  sizes = _sizes([70, 0, 55])
  cfg = bs.dot_general_make() if q else None

  def step(x, w, g):
    out, bp = rd.ragged_dot_vjp(x, w, sizes, cfg=cfg, preferred_element_type=dtype)
    return (out, *bp(g))

  traced = engine.TracedStep(step, x, w, g)
  for turn in range(3):
    for i, t in enumerate((x, w, g)):
      t.copy_(_data(t.shape, t.dtype, 66 + 3 * turn + i, 0.1))
    # blocks of every size a temporary of the step may have had
    junk = [torch.full((1 << b,), float('nan'), dtype=torch.bfloat16, device='cuda')
            for b in range(5, 21) for _ in range(4)]
    del junk
    got = [t.clone() for t in traced(x, w, g)]
    want = step(x, w, g)
    _done()
    for a, b in zip(got, want):
      assert torch.equal(a, b)


@pytest.mark.parametrize('q', [False, True])
@pytest.mark.parametrize('k', [136, 133])
def test_checkpointed_and_offloaded(q, k):
  """Residuals that torch computes anew, or keeps in host memory meanwhile."""
  from torch.utils.checkpoint import checkpoint
  x, w, g = (_data((130, k), torch.bfloat16, 80), _data(
      (3, k, 77), torch.bfloat16, 81, 0.1), _data((130, 77), torch.bfloat16, 82))
  sizes = _sizes([70, 0, 55])
  cfg = bs.dot_general_make() if q else None
  dense = bs.dot_general_make()
  dims = (((1,), (0,)), ((), ()))

  def layer(a, b):
    y = rd.ragged_dot(a, b, sizes, cfg=cfg)
    return dense(y, b[0].t(), dims).mul(0.1) + a

  def step(run):
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = run(a, b)
    filler = [torch.full((1 << i,), float('nan'), device='cuda') for i in range(5, 20)]
    del filler
    y.backward(x)
    return y.detach(), a.grad, b.grad

  def offloaded(a, b):
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
      return layer(a, b)

  want = step(layer)
  for run in (offloaded, lambda a, b: checkpoint(layer, a, b, use_reentrant=False)):
    got = step(run)
    _done()
    for s, t in zip(got, want):
      assert torch.equal(s, t)


@pytest.mark.parametrize('m,k,n,sizes', [
    (60, 640, 72, [10, 0, 7, 20, 3]),
    (700, 300, 264, [257, 130, 1, 0, 300]),
    (5000, 384, 1800, [700, 2000, 0, 129, 2100])])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('frozen', [False, True])
def test_scales_whose_product_leaves_the_range(m, k, n, sizes, out, frozen):
  """Each expert has a magnitude of its own, and so have its rows: some products of
  two block scales are below f32's normal numbers, some above all of them."""
  rng = np.random.default_rng(90)

  def values(shape, exponents):  # one exponent for each of the first axis
    v = rng.integers(-15, 16, shape).astype(np.float64)
    v = np.ldexp(v + (v == 0), np.asarray(exponents).reshape(-1, *[1] * (v.ndim - 1)))
    return torch.from_numpy(v.astype(np.float32)).cuda()

  rows, cots = np.zeros(m, int), np.zeros(m, int)
  of_x, of_w, of_g = (-70, 30, -20, 0, 100), (-64, 5, 60, 0, -95), (-66, 20, -120, 0, 60)
  for e, (a, b) in enumerate(ref.spans(sizes, m)):
    rows[a:b], cots[a:b] = of_x[e], of_g[e]
  rows[::9] += 3
  x, w, g = values((m, k), rows), values((len(sizes), k, n), of_w), values((m, n), cots)
  cfg = bs.dot_general_make('e4m3', 'e4m3')
  want = _want(_f32(x), _f32(w), _f32(g), sizes, True, False, 'e4m3', 'e4m3')
  if frozen:
    y = rd.ragged_dot(x, bs.block_quantize(w, 1, square=True), _sizes(sizes), cfg=cfg,
                      preferred_element_type=out)
    got, want = (y,), want[:1]
  else:
    y, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), cfg=cfg, preferred_element_type=out)
    got = (y, *bp(g))
  _done()
  for name, t, (value, mag, kk) in zip(('out', 'dlhs', 'drhs'), got, want):
    t, half = _f32(t).astype(np.float64), HALF[t.dtype]
    held = mag < 2.0 ** 127  # the others pass f32's range, in sum or on the way
    ref.assert_close(t[held], value[held], mag[held], kk, half, name)
    past = np.abs(value) - (kk + 3) * 2.0 ** -22 * mag >= 2.0 ** 128
    assert not np.isfinite(t[past]).any(), name


@pytest.mark.parametrize('sizes', [[5, 0, 11], [300, 129, 200]])
def test_far_scales_leave_other_groups_alone(sizes):
  """What a far group or row needs changes no bit of the others."""
  m = sum(sizes)
  x, w, g = (_data((m, 384), torch.bfloat16, 91), _data(
      (3, 384, 200), torch.bfloat16, 92, 0.1), _data((m, 200), torch.bfloat16, 93))
  w[0] *= 2.0 ** -60
  cfg = bs.dot_general_make()

  def step(x, g):
    out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes), cfg=cfg)
    return (out, *bp(g))

  out, dl, dr = step(x, g)
  x2, g2 = x.clone(), g.clone()
  x2[2] *= 2.0 ** -75
  g2[3] *= 2.0 ** -90
  out2, dl2, _ = step(x2, g2)
  rest = [i for i in range(m) if i not in (2, 3)]
  assert torch.equal(out[rest], out2[rest]) and torch.equal(dl[rest], dl2[rest])
  assert torch.equal(out[3], out2[3]) and torch.equal(dl[2], dl2[2])
  g3 = g.clone()
  g3[:sizes[0], 7] *= 2.0 ** -110
  _, _, dr3 = step(x, g3)
  _done()
  cols = [i for i in range(200) if i != 7]
  assert torch.equal(dr[0][:, cols], dr3[0][:, cols])
  assert torch.equal(dr[1:], dr3[1:])


def test_first_calls_of_many_threads_at_once():
  """Every kind of product, each from four threads on streams of their own."""
  import threading
  x, w, g = (_data((300, 200), torch.bfloat16, 94), _data(
      (3, 200, 136), torch.bfloat16, 95, 0.1), _data((300, 136), torch.bfloat16, 96))
  sizes = _sizes([150, 20, 100])
  kinds = (None, bs.dot_general_make(), bs.dot_general_make(po2_scale=True))

  def run(cfg):
    out, bp = rd.ragged_dot_vjp(x, w, sizes, cfg=cfg)
    return (out, *bp(g))

  want = [run(cfg) for cfg in kinds]
  _done()
  got, start = {}, threading.Barrier(12)

  def work(i):
    stream = torch.cuda.Stream()
    start.wait()
    with torch.cuda.stream(stream):
      got[i] = run(kinds[i % 3])
    stream.synchronize()

  threads = [threading.Thread(target=work, args=(i,)) for i in range(12)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  _done()
  for i in range(12):
    assert all(torch.equal(a, b) for a, b in zip(got[i], want[i % 3])), i


def test_results_that_torch_fills_first():
  """Deterministic algorithms: torch fills every new tensor with NaN, between the
  quantizer and the product that is launched beside it."""
  x, w = _data((400, 384), torch.bfloat16, 97), _data((4, 384, 200), torch.bfloat16, 98,
                                                      0.1)
  qt = bs.block_quantize(w, 1, square=True)
  cfg = bs.dot_general_make()
  sizes = _sizes([20, 0, 30, 5])  # most rows lie behind the last group
  want = rd.ragged_dot(x, qt, sizes, cfg=cfg)
  _done()
  torch.use_deterministic_algorithms(True)
  try:
    got = [rd.ragged_dot(x, qt, sizes, cfg=cfg) for _ in range(50)]
  finally:
    torch.use_deterministic_algorithms(False)
  _done()
  assert not want[55:].any()
  assert all(torch.equal(t, want) for t in got)


@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_matrices_of_empty_experts_are_not_read(monkeypatch, index):
  """The packed copy's memory holds NaN before it is written, and only the matrices
  of experts with rows are filled in."""
  g, k, n = 40, 133, 77
  sizes = [0] * g
  sizes[3], sizes[17], sizes[39] = 5, 1, 2
  x, w, ct = (_data((9, k), torch.bfloat16, 50), _data(
      (g, k, n), torch.bfloat16, 51, 0.1), _data((9, n), torch.bfloat16, 52))
  copies = []
  empty = be._empty_out  # pylint: disable=protected-access

  def poisoned(shape, dtype, device):
    t = empty(shape, dtype, device)
    if dtype == torch.bfloat16:
      t.fill_(float('nan'))
      if tuple(t.shape) == (g, k, 80):
        copies.append(t)
    return t

  monkeypatch.setattr(be, '_empty_out', poisoned)
  out, bp = rd.ragged_dot_vjp(x, w, _sizes(sizes, index))
  dl, dr = bp(ct)
  _done()
  assert len(copies) == 1
  left = torch.isnan(copies[0].float()).flatten(1).all(1)
  assert left.tolist() == [v == 0 for v in sizes]
  for got, wt in zip((out, dl, dr), _want(_f32(x), _f32(w), _f32(ct), sizes, False)):
    _check(got, wt, 2.0 ** -8, '')


@pytest.mark.parametrize('po2', [False, True])
def test_expert_layer_in_fp8_product_by_product(po2):
  """The layer of test_expert_layer in fp8, each product against the definition on
  the operands and the cotangent that it got."""
  tokens, d, f, e, top = 200, 264, 392, 6, 2
  x = _data((tokens, d), torch.bfloat16, 83)
  router = _data((d, e), torch.float32, 84, 0.2)
  ws = [_data((e, d, f), torch.bfloat16, 85, 0.1), _data(
      (e, d, f), torch.bfloat16, 86, 0.1), _data((e, f, d), torch.bfloat16, 87, 0.1)]
  p, chosen = torch.softmax(x.float() @ router, -1).topk(top, -1)
  order = chosen.reshape(-1).argsort(stable=True)
  sizes = torch.bincount(chosen.reshape(-1), minlength=e).to(torch.int32)
  row, weight = order // top, p.reshape(-1)[order]
  cfg = bs.dot_general_make('e4m3', 'e5m2', po2_scale=po2)
  leaf = x.clone().requires_grad_()
  weights = [w.clone().requires_grad_() for w in ws]
  seen = []

  def product(a, w):
    y = rd.ragged_dot(a, w, sizes, cfg=cfg)
    at = {'a': a.detach().clone(), 'w': w, 'y': y.detach().clone()}
    y.register_hook(lambda g: at.__setitem__('g', g.clone()))
    seen.append(at)
    return y

  rows = leaf[row]
  hidden = (torch.nn.functional.silu(product(rows, weights[0]).float()) *
            product(rows, weights[1]).float()).bfloat16()
  down = product(hidden, weights[2]).float() * weight[:, None]
  y = torch.zeros(tokens, d, device='cuda').index_add(0, row, down)
  (y * _data((tokens, d), torch.float32, 88)).sum().backward()
  _done()
  assert len(seen) == 3
  for at, w in zip(seen, weights):
    out, dl, dr = _want(_f32(at['a']), _f32(w.detach()), _f32(at['g']), sizes.tolist(), True, po2)
    _check(at['y'], out, 2.0 ** -8, 'out')
    _check(w.grad, dr, 2.0 ** -8, 'drhs')
    at['dl'], at['mag'] = dl[0], dl[1]
  # the tokens' gradient: two products' rows, summed over the experts of a token;
  # rounded to bfloat16 by either product, in their sum, and in each of the sums
  want, mag = np.zeros((tokens, d)), np.zeros((tokens, d))
  for at in seen[:2]:
    np.add.at(want, row.cpu().numpy(), at['dl'])
    np.add.at(mag, row.cpu().numpy(), at['mag'])
  tol = (2 + top) * 2.0 ** -8 * mag + f * 2.0 ** -23 * mag
  assert (np.abs(_f32(leaf.grad) - want) <= tol).all()


@pytest.mark.parametrize('m,n,sizes', [(1700, 6000, [100, 900, 0, 655]),
                                       (300, 264, [33, 200, 0, 60])])
def test_far_rows_wherever_they_lie(m, n, sizes):
  """Rows that need care lie in any block of 128 that a tile of a group covers,
  counted from the first row (serving) or from the group's (training)."""
  k = 256
  x, w = _data((m, k), torch.float32, 100), _data((4, k, n), torch.float32, 101,
                                                 0.3 * 2.0 ** -50)
  cfg = bs.dot_general_make()
  s, qt = _sizes(sizes), bs.block_quantize(w, 1, square=True)
  assert float(qt.scale[0].min()) > 2.0 ** -63
  leaf = lambda t: t.clone().requires_grad_()
  runs = (lambda t: rd.ragged_dot(t, qt, s, cfg=cfg),
          lambda t: rd.ragged_dot(leaf(t), leaf(w), s, cfg=cfg).detach())
  base = runs[0](x)
  assert torch.equal(base, runs[1](x))
  mag = rd.ragged_dot(x.abs(), bs.frozen(qt.qvalue.float().abs().to(
      torch.float8_e4m3fn), qt.scale[0]), s, cfg=cfg).double()
  for first in range(0, sum(sizes), 61):
    at = slice(first, min(first + 3, m))
    far = x.clone()
    far[at] *= 2.0 ** -75
    for run in runs:
      out = run(far)
      off = (out[at].double() * 2.0 ** 75 - base[at].double()).abs()
      assert (off <= 2 * (k + 9) * 2.0 ** -23 * mag[at]).all(), first
      same = torch.ones(m, dtype=torch.bool, device='cuda')
      same[at] = False
      assert torch.equal(out[same], base[same]), first
  _done()


@pytest.mark.parametrize('q', [False, True])
def test_captured_training_step_on_torchs_tape(q):
  """Forward and backward through autograd in one graph: residuals are memory of the
  graph, and replays follow new operands and sizes."""
  x, w, g = (_data((130, 136), torch.bfloat16, 102), _data(
      (3, 136, 77), torch.bfloat16, 103, 0.1), _data((130, 77), torch.bfloat16, 104))
  sizes = _sizes([70, 0, 55])
  cfg = bs.dot_general_make() if q else None
  a, b = x.clone().requires_grad_(), w.clone().requires_grad_()

  def step():
    y = rd.ragged_dot(a, b, sizes, cfg=cfg)
    return (y.detach(), *torch.autograd.grad(y, (a, b), g))

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = step()
  for seed, values in ((105, [70, 0, 55]), (106, [1, 100, 29])):
    with torch.no_grad():
      a.copy_(_data(x.shape, x.dtype, seed))
      b.copy_(_data(w.shape, w.dtype, seed + 10, 0.1))
    sizes.copy_(_sizes(values))
    graph.replay()
    out, bp = rd.ragged_dot_vjp(a, b, sizes, cfg=cfg)
    want = (out, *bp(g))
    _done()
    for s, t in zip(got, want):
      assert torch.equal(s, t)
