"""Block-scaled fp8 products and products grouped by expert: cases, plain forms
and the framework's calls.

  quantize   one fp8 value per element, one f32 scale per block of 128 (or 128 x 128)
  dot        lhs [M, K] . rhs [K, N], rhs frozen in 128 x 128 blocks (serving)
  dot_step   the same with float rhs: forward, dlhs, drhs (training)
  ragged     lhs [M, K] . rhs [G, K, N], rows grouped by group_sizes [G]; bf16 or
             frozen block-scaled fp8 weights (serving)
  ragged_step  forward, dlhs, drhs of the grouped product, bf16 or block-scaled fp8
"""

import math

import numpy as np
import torch

own = False

BLOCK = 128
BOUND = {'e4m3': 448.0, 'e5m2': 57344.0}
FP8 = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}
FLOAT = {'bf16': torch.bfloat16, 'f32': torch.float32}
DIMS = (((1,), (0,)), ((), ()))


def listed():
  return [
      # activations of one decode step before a projection
      dict(name='quantize_decode', op='quantize', r=16, c=4096, axis=-1,
           square=False, bits='e4m3', po2=False, dtype='bf16'),
      # a projection's weights at conversion: 128 x 128 blocks, stored with the
      # contraction index contiguous
      dict(name='quantize_weights', op='quantize', r=4096, c=14336, axis=0,
           square=True, bits='e4m3', po2=False, dtype='bf16'),
      # a cotangent for the weight gradient: blocks along the tokens, ragged tail
      dict(name='quantize_tokens', op='quantize', r=8111, c=4096, axis=0,
           square=False, bits='e5m2', po2=True, dtype='f32'),
      # one token through a projection with frozen weights
      dict(name='dot_decode_1', op='dot', m=1, k=4096, n=4096, po2=False,
           dtype='bf16'),
      # a decode batch through the large projection of the serving benchmark
      dict(name='dot_decode_16', op='dot', m=16, k=8192, n=28672, po2=False,
           dtype='bf16'),
      # a prompt through an up projection, odd number of tokens
      dict(name='dot_prompt', op='dot', m=2047, k=4096, n=14336, po2=False,
           dtype='bf16'),
      # training step of the float32 parity configuration's shape
      dict(name='dot_step_f32', op='dot_step', m=1024, k=4096, n=4096,
           po2=False, dtype='f32'),
      # training step of a projection
      dict(name='dot_step', op='dot_step', m=8192, k=4096, n=14336, po2=False,
           dtype='bf16'),
      # decode batch of a mixture of experts: few rows an expert, some none
      dict(name='ragged_decode', op='ragged', m=64, pad=0, k=4096, n=14336, g=8,
           q=False, po2=False, dtype='bf16', spread=0.5),
      # the same with many small experts and frozen fp8 weights
      dict(name='ragged_decode_q', op='ragged', m=257, pad=15, k=2048, n=1408,
           g=64, q=True, po2=False, dtype='bf16', spread=0.7),
      # training step of an expert layer in bf16
      dict(name='ragged_step', op='ragged_step', m=8192, pad=0, k=2048, n=1408,
           g=16, q=False, po2=False, dtype='bf16', spread=0.4),
      # the same in block-scaled fp8, odd sizes, rows behind the last group
      dict(name='ragged_step_q', op='ragged_step', m=16301, pad=83, k=4096,
           n=1832, g=8, q=True, po2=True, dtype='bf16', spread=0.4),
  ]


def _log(rng, lo, hi):
  return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo),
                                                        math.log(hi)))))))


def draw(rng):
  op = rng.choice(['quantize', 'dot', 'dot_step', 'ragged', 'ragged',
                   'ragged_step', 'ragged_step'])
  po2 = rng.random() < 0.3
  dtype = 'f32' if rng.random() < 0.2 else 'bf16'
  if op == 'quantize':
    return dict(op=op, r=_log(rng, 1, 8192), c=_log(rng, 1, 14336),
                axis=rng.choice([-1, 0]), square=rng.random() < 0.4,
                bits=rng.choice(['e4m3', 'e5m2']), po2=po2, dtype=dtype)
  if op == 'dot':
    return dict(op=op, m=_log(rng, 1, 2048), k=_log(rng, 64, 14336),
                n=_log(rng, 64, 14336), po2=po2, dtype=dtype)
  if op == 'dot_step':
    return dict(op=op, m=_log(rng, 1, 8192), k=_log(rng, 64, 8192),
                n=_log(rng, 64, 7168), po2=po2, dtype=dtype)
  g = _log(rng, 1, 64)
  q = rng.random() < 0.5
  if op == 'ragged':
    return dict(op=op, m=_log(rng, 1, 1024), pad=rng.choice([0, 0, 1, 37]),
                k=_log(rng, 64, 4096), n=_log(rng, 64, 4096), g=g, q=q, po2=po2,
                dtype=dtype if q else 'bf16', spread=rng.choice([0.0, 0.5, 1.0]))
  return dict(op=op, m=_log(rng, 64, 16384), pad=rng.choice([0, 0, 5, 130]),
              k=_log(rng, 64, 4096), n=_log(rng, 64, 2048), g=min(g, 32), q=q,
              po2=po2, dtype=dtype if q else 'bf16',
              spread=rng.choice([0.0, 0.4, 0.8]))


# -- inputs -------------------------------------------------------------------


def _group_sizes(case, seed):
  """Rows an expert gets from a router: uneven, an expert without any now and
  then; they add up to m."""
  r = np.random.default_rng(seed)
  p = np.exp(case['spread'] * r.standard_normal(case['g']))
  if case['g'] > 2 and case['spread']:
    p[r.integers(case['g'])] = 0.0
  return r.multinomial(case['m'], p / p.sum())


def _weight_blocks(w, po2):
  """Frozen weights [..., K, N]: fp8 values stored with k contiguous, f32 scales
  [..., ceil(K/128), ceil(N/128)]."""
  q, s = _quantize(w, -2, True, 'e4m3', po2)
  *lead, k, n = q.shape
  ld = -(-k // 16) * 16
  store = torch.zeros(*lead, n, ld, dtype=torch.uint8, device=w.device)
  store[..., :k] = q.view(torch.uint8).transpose(-1, -2)
  return store[..., :k].view(FP8['e4m3']).transpose(-1, -2), s


def prepare(case, seed):
  dev = 'cuda'
  gen = torch.Generator(device=dev)
  gen.manual_seed(seed)
  dt = FLOAT[case['dtype']]

  def acts(rows, cols):
    # activations and cotangents: normal, with rows and columns of larger
    # magnitude, as behind a norm and a residual stream
    x = torch.randn(rows, cols, device=dev, generator=gen)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device=dev, generator=gen))
    x *= torch.exp(0.3 * torch.randn(1, cols, device=dev, generator=gen))
    return x.to(dt)

  def weights(*shape):
    return (torch.randn(*shape, device=dev, generator=gen) *
            shape[-2] ** -0.5).to(dt)

  st = {'case': dict(case)}
  op = case['op']
  if op == 'quantize':
    st['x'] = acts(case['r'], case['c'])
    return st
  rows = case['m'] + case.get('pad', 0)
  st['x'] = acts(rows, case['k'])
  if op in ('dot', 'dot_step'):
    w = weights(case['k'], case['n'])
  else:
    w = weights(case['g'], case['k'], case['n'])
    sizes = _group_sizes(case, seed)
    st['sizes'] = torch.tensor(sizes, dtype=torch.int32, device=dev)
    st['most'] = int(sizes.max())  # the plain form pads its groups to this
  if op == 'dot' or (op == 'ragged' and case['q']):
    st['wq'], st['ws'] = _weight_blocks(w, case['po2'])
  else:
    st['w'] = w
  if op.endswith('_step'):
    st['g'] = acts(rows, case['n'])
  return st


# -- plain forms --------------------------------------------------------------


def _scale(amax, bits, po2):
  # divided by a tensor: by a number torch would multiply by its reciprocal
  s = (torch.where(amax == 0, torch.ones_like(amax), amax) /
       torch.full_like(amax, BOUND[bits]))
  s = s.clamp_min(2.0 ** -126)
  if po2:
    m, e = torch.frexp(s)  # s = m 2^e, m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(s), torch.where(m == 0.5, e - 1, e))
  return s


def _quantize(x, axis, square, bits, po2):
  """(q, s) of the last two axes of x: blocks of 128 along `axis` (or 128 x 128)."""
  *lead, r, c = x.shape
  br = BLOCK if square or axis == -2 else 1
  bc = BLOCK if square or axis == -1 else 1
  nr, nc = -(-r // br), -(-c // bc)
  xp = torch.zeros(*lead, nr * br, nc * bc, dtype=torch.float32, device=x.device)
  xp[..., :r, :c] = x
  xb = xp.view(*lead, nr, br, nc, bc)
  s = _scale(xb.abs().amax(dim=(-3, -1)), bits, po2)
  y = xb * (1.0 / s)[..., :, None, :, None]
  y = y.clamp(-BOUND[bits], BOUND[bits]).to(FP8[bits])
  return y.view(*lead, nr * br, nc * bc)[..., :r, :c], s


def _widen(q, s, axis, square):
  """Values that (q, s) stand for, in f32."""
  if square or axis == -2:
    s = s.repeat_interleave(BLOCK, dim=-2)[..., :q.shape[-2], :]
  if square or axis == -1:
    s = s.repeat_interleave(BLOCK, dim=-1)[..., :q.shape[-1]]
  return q.float() * s


def _fake(x, axis, square, bits, po2):
  q, s = _quantize(x, axis, square, bits, po2)
  return _widen(q, s, axis, square)


def _places(sizes, rows, most):
  """Where each row sits when the groups are padded to `most` rows."""
  ends = sizes.long().cumsum(0)
  at = torch.arange(rows, device=sizes.device)
  group = torch.searchsorted(ends, at, right=True)
  inside = group < sizes.numel()
  group = group.clamp_max(sizes.numel() - 1)
  pos = (at - (ends - sizes)[group]).clamp(0, max(most - 1, 0))
  return group, pos, inside


def _spread(x, place, groups, most):
  """[rows, C] -> [groups, most, C], zero where a group has no such row."""
  group, pos, inside = place
  y = torch.zeros(groups, most, x.shape[1], dtype=torch.float32, device=x.device)
  y[group[inside], pos[inside]] = x[inside].float()
  return y


def _gather(y, place):
  group, pos, inside = place
  out = y[group, pos]
  return torch.where(inside[:, None], out, torch.zeros_like(out))


def run(st):
  case = st['case']
  if own:
    return _run_own(st, case)
  op, po2 = case['op'], case['po2']
  x = st['x']
  if op == 'quantize':
    return _quantize(x, -1 if case['axis'] == -1 else -2, case['square'],
                     case['bits'], po2)
  dt = x.dtype
  if op == 'dot':
    return (_fake(x, -1, False, 'e4m3', po2) @
            _widen(st['wq'], st['ws'], -2, True)).to(dt)
  if op == 'dot_step':
    w = _fake(st['w'], -2, True, 'e4m3', po2)
    g = st['g']
    out = _fake(x, -1, False, 'e4m3', po2) @ w
    dx = _fake(g, -1, False, 'e5m2', po2) @ w.T
    dw = (_fake(x, -2, False, 'e4m3', po2).T @ _fake(g, -2, False, 'e5m2', po2))
    return out.to(dt), dx.to(dt), dw.to(dt)
  groups, most = case['g'], max(st['most'], 1)
  place = _places(st['sizes'], x.shape[0], most)
  if op == 'ragged':
    xv = _fake(x, -1, False, 'e4m3', po2) if case['q'] else x
    w = _widen(st['wq'], st['ws'], -2, True) if case['q'] else st['w'].float()
    return _gather(torch.bmm(_spread(xv, place, groups, most), w), place).to(dt)
  g = st['g']
  if case['q']:
    w = _fake(st['w'], -2, True, 'e4m3', po2)
    xf = _spread(_fake(x, -1, False, 'e4m3', po2), place, groups, most)
    gf = _spread(_fake(g, -1, False, 'e5m2', po2), place, groups, most)
    xt = _fake(_spread(x, place, groups, most), -2, False, 'e4m3', po2)
    gt = _fake(_spread(g, place, groups, most), -2, False, 'e5m2', po2)
  else:
    w = st['w'].float()
    xf = xt = _spread(x, place, groups, most)
    gf = gt = _spread(g, place, groups, most)
  out = _gather(torch.bmm(xf, w), place)
  dx = _gather(torch.bmm(gf, w.transpose(1, 2)), place)
  dw = torch.bmm(xt.transpose(1, 2), gt)
  return out.to(dt), dx.to(dt), dw.to(dt)


# -- the framework's calls ----------------------------------------------------


def _run_own(st, case):
  from aqt_b200.v2 import aqt_ragged_dot
  from aqt_b200.v2 import block_scaled
  op, x = case['op'], st['x']
  if op == 'quantize':
    qt = block_scaled.block_quantize(
        x, contract_axis=case['axis'], square=case['square'], bits=case['bits'],
        po2_scale=case['po2'])
    return qt.qvalue, qt.scale[0]
  cfg = None
  if op.startswith('dot') or case['q']:
    cfg = block_scaled.dot_general_make('e4m3', 'e5m2', po2_scale=case['po2'])
  if 'wq' in st:
    w = block_scaled.frozen(st['wq'], st['ws'])
  else:
    w = st['w']
  if op == 'dot':
    return cfg(x, w, DIMS)
  if op == 'ragged':
    return aqt_ragged_dot.ragged_dot(x, w, st['sizes'], cfg=cfg)
  if op == 'dot_step':
    out, backprop = cfg.vjp(x, w, DIMS)
  else:
    out, backprop = aqt_ragged_dot.ragged_dot_vjp(x, w, st['sizes'], cfg=cfg)
  dx, dw = backprop(st['g'])
  return out, dx, dw


# -- work ---------------------------------------------------------------------


def work(case):
  es = 4 if case['dtype'] == 'f32' else 2
  if case['op'] == 'quantize':
    r, c = case['r'], case['c']
    br = BLOCK if case['square'] or case['axis'] == 0 else 1
    bc = BLOCK if case['square'] or case['axis'] == -1 else 1
    scales = -(-r // br) * -(-c // bc)
    return {'bytes': r * c * (es + 1) + 4 * scales, 'flops': 3 * r * c}
  m, k, n = case['m'], case['k'], case['n']
  rows = m + case.get('pad', 0)
  # weights that some row needs: every expert, or as many as a draw of m rows
  # meets on average
  g = case.get('g', 1)
  met = g * (1.0 - (1.0 - 1.0 / g) ** m) if g > 1 else 1.0
  if case['op'] == 'dot' or (case['op'] == 'ragged' and case['q']):
    return {'bytes': met * (k * n + 4 * (-(-k // BLOCK)) * (-(-n // BLOCK))) +
                     es * (m * k + rows * n), 'flops': 2 * m * n * k}
  if case['op'] == 'ragged':
    return {'bytes': es * (met * k * n + m * k + rows * n),
            'flops': 2 * m * n * k}
  return {'bytes': es * (met * k * n + g * k * n + 2 * rows * (k + n)),
          'flops': 6 * m * n * k}


# -- the definition in 64 bits ------------------------------------------------


def _round_fp8(y, bits):
  """Nearest fp8 value, ties to even, of f32 values within the format's range."""
  mant, least = (3, -6) if bits == 'e4m3' else (2, -14)
  y = y.double()
  _, e = torch.frexp(y)
  step = torch.ldexp(torch.ones_like(y), (e - 1).clamp_min(least) - mant)
  return torch.round(y / step) * step


def _exact_quantize(x, block_r, block_c, bits, po2):
  """(values, scales, values times scales) in 64 bits. The scale is a 32-bit
  number by definition, and so are its reciprocal and the scaled value that is
  rounded to 8 bits: each is computed in 64 bits and rounded to 32."""
  r, c = x.shape
  pad = (0, -c % block_c, 0, -r % block_r)
  t = torch.nn.functional.pad(x.double(), pad)
  t = t.unflatten(1, (-1, block_c)).unflatten(0, (-1, block_r))
  top = t.abs().amax(dim=(1, 3), keepdim=True)
  top[top == 0] = 1.0
  s = torch.clamp((top / BOUND[bits]).float().double(), min=2.0 ** -126)
  if po2:
    s = torch.exp2(torch.ceil(torch.log2(s)))
  y = (t * (1.0 / s).float().double()).float().double()
  q = _round_fp8(y.clamp(-BOUND[bits], BOUND[bits]), bits)
  flat = lambda v: v.flatten(2, 3).flatten(0, 1)[:r, :c]
  return flat(q), s[:, 0, :, 0], flat(q * s)


def exact(case, seed):
  st = prepare(case, seed)
  op, po2 = case['op'], case['po2']
  x = st['x']
  if op == 'quantize':
    br = BLOCK if case['square'] or case['axis'] == 0 else 1
    bc = BLOCK if case['square'] or case['axis'] == -1 else 1
    q, s, _ = _exact_quantize(x, br, bc, case['bits'], po2)
    return q, s
  if 'wq' in st:
    k, n = case['k'], case['n']
    rk = torch.arange(k, device=x.device) // BLOCK
    rn = torch.arange(n, device=x.device) // BLOCK
    w = st['wq'].double() * st['ws'].double()[..., rk, :][..., rn]
  q = case['op'].startswith('dot') or case['q']

  def one(xg, gg, wg):
    """out, dlhs, drhs of one group's rows."""
    if 'wq' not in st:
      wv = _exact_quantize(wg, BLOCK, BLOCK, 'e4m3', po2)[2] if q else wg.double()
    else:
      wv = wg
    xv = _exact_quantize(xg, 1, BLOCK, 'e4m3', po2)[2] if q else xg.double()
    out = xv @ wv
    if gg is None:
      return out, None, None
    gv = _exact_quantize(gg, 1, BLOCK, 'e5m2', po2)[2] if q else gg.double()
    xt = _exact_quantize(xg, BLOCK, 1, 'e4m3', po2)[2] if q else xg.double()
    gt = _exact_quantize(gg, BLOCK, 1, 'e5m2', po2)[2] if q else gg.double()
    return out, gv @ wv.T, xt.T @ gt

  g = st.get('g')
  if 'wq' not in st:
    w = st['w']
  if op.startswith('dot'):
    out, dx, dw = one(x, g, w)
    return out if g is None else (out, dx, dw)
  rows, k, n = x.shape[0], case['k'], case['n']
  out = torch.zeros(rows, n, dtype=torch.float64, device=x.device)
  dx = torch.zeros(rows, k, dtype=torch.float64, device=x.device)
  dw = torch.zeros(case['g'], k, n, dtype=torch.float64, device=x.device)
  at = 0
  for e, size in enumerate(st['sizes'].tolist()):
    if size:
      part = slice(at, at + size)
      o, a, b = one(x[part], None if g is None else g[part], w[e])
      out[part] = o
      if g is not None:
        dx[part], dw[e] = a, b
    at += size
  return out if g is None else (out, dx, dw)
