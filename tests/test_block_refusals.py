"""What the block-scaled and grouped products refuse, and how: no GPU needed."""

import ctypes as C

import pytest
import torch

from aqt_b200 import _lib
from aqt_b200.v2 import aqt_ragged_dot as rd
from aqt_b200.v2 import aqt_tensor
from aqt_b200.v2 import block_scaled as bs
from tests import fake_lib

DIMS = (((1,), (0,)), ((), ()))
BF = torch.bfloat16


def test_cpu_tensors_are_refused():
  x, w = torch.zeros(4, 128), torch.zeros(128, 8)
  cfg = bs.dot_general_make()
  with pytest.raises(_lib.AqtB200Error, match='no CPU path'):
    bs.block_quantize(x)
  with pytest.raises(_lib.AqtB200Error, match='no CPU path'):
    cfg(x, w, DIMS)
  with pytest.raises(_lib.AqtB200Error, match='no CPU path'):
    rd.ragged_dot(x.to(BF), w.to(BF)[None], torch.tensor([4]))


@pytest.fixture
def on_cpu(monkeypatch):
  """Lets CPU tensors through to the checks behind the device check."""
  return fake_lib.install(monkeypatch)


def _frozen(k=128, n=8, axis=-2, g=None):
  lead = () if g is None else (g,)
  q = torch.zeros(*lead, n, k, dtype=torch.float8_e4m3fn).transpose(-1, -2)
  return aqt_tensor.QTensor(
      qvalue=q, scale=[torch.ones(*lead, -(-k // 128), -(-n // 128))],
      scale_t=None, tiling_state=bs.BlockTiling(axis, True))


@pytest.mark.parametrize('call,error', [
    (lambda: bs.block_quantize(torch.zeros(4)), NotImplementedError),
    (lambda: bs.block_quantize(torch.zeros(2, 2, 2, 2)), NotImplementedError),
    (lambda: bs.block_quantize(torch.zeros(2, 4, 4), contract_axis=0),
     NotImplementedError),
    (lambda: bs.block_quantize(torch.zeros(4, 4, dtype=torch.float16)),
     NotImplementedError),
    (lambda: bs.block_quantize(torch.zeros(4, 4, dtype=torch.float64)),
     NotImplementedError),
    (lambda: bs.block_quantize(torch.zeros(4, 4), bits=8), NotImplementedError),
    (lambda: bs.block_quantize([[1.0]]), TypeError),
    (lambda: bs.dot_general_make('int8'), NotImplementedError),
    (lambda: bs.frozen(torch.zeros(4, 4), torch.ones(1, 1)),
     NotImplementedError),
    (lambda: bs.frozen(torch.zeros(4, 4, dtype=torch.float8_e4m3fn),
                       torch.ones(2, 1)), ValueError),
    (lambda: bs.frozen(torch.zeros(4, 4, dtype=torch.float8_e4m3fn),
                       torch.ones(1, 1, dtype=BF)), NotImplementedError),
])
def test_quantize_and_make(on_cpu, call, error):
  with pytest.raises(error):
    call()


@pytest.mark.parametrize('lhs,rhs,dims,error', [
    ((4, 128), (64, 8), DIMS, ValueError),                       # extents
    ((2, 4, 128), (2, 128, 8), (((2,), (1,)), ((0,), (0,))),
     NotImplementedError),                                       # batch axes
    ((4, 128), (128, 8, 2), DIMS, NotImplementedError),
    ((4, 8, 16), (8, 16), (((1, 2), (0, 1)), ((), ())), NotImplementedError),
    ((128, 4, 2), (128, 8), (((0,), (0,)), ((), ())), NotImplementedError),
])
def test_dot_shapes(on_cpu, lhs, rhs, dims, error):
  with pytest.raises(error):
    bs.dot_general_make()(torch.zeros(lhs), torch.zeros(rhs), dims)


def test_dot_types_and_frozen(on_cpu):
  cfg = bs.dot_general_make()
  x = torch.zeros(4, 128)
  with pytest.raises(TypeError):
    cfg(x, torch.zeros(128, 8, dtype=BF), DIMS)
  with pytest.raises(NotImplementedError):
    cfg(x, torch.zeros(128, 8), DIMS, preferred_element_type=torch.float16)
  with pytest.raises(AssertionError):
    cfg(x, torch.zeros(128, 8), DIMS, precision='highest')
  with pytest.raises(NotImplementedError, match='128 x 128'):
    cfg(x, _frozen().replace(tiling_state=None), DIMS)
  with pytest.raises(NotImplementedError, match='128 x 128'):
    cfg(x, _frozen().replace(tiling_state=bs.BlockTiling(-2, False)), DIMS)
  with pytest.raises(NotImplementedError, match='quantize it for that axis'):
    cfg(x, _frozen().replace(tiling_state=bs.BlockTiling(-1, True)), DIMS)
  with pytest.raises(ValueError, match='layout'):
    qt = _frozen()
    cfg(x, qt.replace(qvalue=qt.qvalue.contiguous()), DIMS)
  with pytest.raises(NotImplementedError, match='no gradient'):
    cfg(x.clone().requires_grad_(), _frozen(), DIMS)
  with pytest.raises(NotImplementedError, match='no gradient'):
    cfg.vjp(x, _frozen(), DIMS)


def test_ragged(on_cpu):
  x, w = torch.zeros(4, 128, dtype=BF), torch.zeros(2, 128, 8, dtype=BF)
  s = torch.tensor([2, 2], dtype=torch.int32)
  cfg = bs.dot_general_make()
  bad = [
      (lambda: rd.ragged_dot(x, w[0], s), ValueError),
      (lambda: rd.ragged_dot(x[None], w, s), ValueError),
      (lambda: rd.ragged_dot(x[:, :64], w, s), ValueError),
      (lambda: rd.ragged_dot(x, w, s[:1]), ValueError),
      (lambda: rd.ragged_dot(x, w, s[:, None]), ValueError),
      (lambda: rd.ragged_dot(x, w, torch.zeros(4, dtype=torch.int32)[::2]),
       ValueError),
      (lambda: rd.ragged_dot(x, w, s.float()), NotImplementedError),
      (lambda: rd.ragged_dot(x, w, s.to(torch.int16)), NotImplementedError),
      (lambda: rd.ragged_dot(x, w, [2, 2]), TypeError),
      (lambda: rd.ragged_dot(x.float(), w.float(), s), NotImplementedError),
      (lambda: rd.ragged_dot(x.half(), w.half(), s, cfg=cfg),
       NotImplementedError),
      (lambda: rd.ragged_dot(x, w.float(), s, cfg=cfg), TypeError),
      (lambda: rd.ragged_dot(x, _frozen(g=2), s), ValueError),
      (lambda: rd.ragged_dot(x, w, s, cfg='fp8'), NotImplementedError),
      (lambda: rd.ragged_dot_vjp(x, _frozen(g=2), s, cfg=cfg),
       NotImplementedError),
      (lambda: rd.ragged_dot(x.clone().requires_grad_(), _frozen(g=2), s,
                             cfg=cfg), NotImplementedError),
      (lambda: rd.ragged_dot(
          x, torch.zeros(1, 128, 8, dtype=BF).expand(1025, 128, 8),
          torch.zeros(1025, dtype=torch.int32)), NotImplementedError),
      (lambda: rd.ragged_dot(x, w[:0], s[:0]), NotImplementedError),
  ]
  for i, (call, error) in enumerate(bad):
    with pytest.raises(error):
      call()
      pytest.fail(f'call {i} was not refused')


@pytest.fixture(scope='module')
def lib():
  from aqt_b200 import build
  build.build()
  return _lib.load()


def _quant_desc(**kw):
  d = _lib.BlockQuantDesc()
  d.x = _lib.View(256, _lib.BF16, 0, 1, 1, 4, 128, 0, 0, 128, 1)
  d.qdtype, d.q_row, d.ld_row, d.scale_row = _lib.E4M3, 256, 128, 256
  for k, v in kw.items():
    setattr(d, k, v)
  return d


def test_abi_quantize(lib):
  call = lambda d: lib.aqtb200_block_quantize(C.byref(d), None)
  assert lib.aqtb200_block_quantize(None, None) == -1
  assert call(_quant_desc(qdtype=_lib.S8)) == -2
  assert call(_quant_desc(q_row=None)) == -1
  assert call(_quant_desc(scale_row=None)) == -1
  assert call(_quant_desc(ld_row=120)) == -1
  assert call(_quant_desc(q_row=257)) == -1
  assert call(_quant_desc(q_col=256, ld_col=16)) == -1           # no scales
  assert call(_quant_desc(group_sizes=256, groups=0)) == -1
  assert call(_quant_desc(group_sizes=256, groups=1, square=1)) == -2
  # grouped: q_col holds whole blocks
  assert call(_quant_desc(group_sizes=256, groups=3, q_col=256, ld_col=128,
                          scale_col=256)) == -1
  d = _quant_desc()
  d.x.dtype = _lib.S8
  assert call(d) == -2
  d = _quant_desc()
  d.x.rows = -1
  assert call(d) == -1


def _gemm_desc(**kw):
  d = _lib.GroupedGemmDesc()
  d.a_dtype = d.b_dtype = d.out_dtype = _lib.BF16
  d.r, d.t, d.k, d.rows = 64, 8, 64, 8
  d.a, d.a_ld, d.b, d.b_ld, d.out, d.out_ld = 256, 64, 256, 64, 256, 64
  for k, v in kw.items():
    setattr(d, k, v)
  return d


def test_abi_gemm(lib):
  call = lambda d: lib.aqtb200_grouped_gemm(C.byref(d), None, None)
  assert lib.aqtb200_grouped_gemm(None, None, None) == -1
  assert lib.aqtb200_grouped_gemm_workspace_bytes(None) == 0
  assert call(_gemm_desc(contract_groups=2)) == -1
  assert call(_gemm_desc(a_dtype=_lib.E4M3)) == -2
  assert call(_gemm_desc(a_dtype=_lib.S8, b_dtype=_lib.S8)) == -2
  assert call(_gemm_desc(out_dtype=_lib.S8)) == -1
  assert call(_gemm_desc(t=-1)) == -1
  assert call(_gemm_desc(out=None)) == -1
  assert call(_gemm_desc(a_dtype=_lib.E4M3, b_dtype=_lib.E4M3)) == -1   # scales
  assert call(_gemm_desc(a_dtype=_lib.E4M3, b_dtype=_lib.E5M2,
                         a_mn_major=1)) == -2
  assert call(_gemm_desc(group_sizes=256, groups=1025)) == -2
  assert call(_gemm_desc(group_sizes=256, groups=0)) == -2
  assert call(_gemm_desc(k=1 << 31)) == -2
  d = _gemm_desc(contract_groups=1, group_sizes=256, groups=2, a_mn_major=1,
                 b_mn_major=1)
  assert lib.aqtb200_grouped_gemm_workspace_bytes(C.byref(d)) >= (
      2 * 64 * (64 + 8) * 2)


def test_abi_pack(lib):
  v = _lib.View(256, _lib.F32, 0, 1, 1, 4, 8, 0, 0, 8, 1)
  assert lib.aqtb200_pack_bf16(C.byref(v), 256, 8, None) == -1
  v.dtype = _lib.BF16
  assert lib.aqtb200_pack_bf16(C.byref(v), 256, 4, None) == -1
  assert lib.aqtb200_pack_bf16(C.byref(v), None, 8, None) == -1
  assert lib.aqtb200_pack_bf16(C.byref(v), 264, 8, None) == -1
  assert lib.aqtb200_pack_bf16(C.byref(v), 256, 12, None) == -1
  assert lib.aqtb200_pack_bf16(None, 256, 8, None) == -1


def test_abi_gemm_grouped_positions(lib):
  """The contraction over grouped rows has to hold all of them."""
  call = lambda d: lib.aqtb200_grouped_gemm(C.byref(d), None, None)
  common = dict(contract_groups=1, group_sizes=256, groups=3)
  assert call(_gemm_desc(a_mn_major=1, b_mn_major=1, k=64, rows=65,
                         **common)) == -1
  # fp8: 300 rows in three groups take up to 2 + 3 blocks
  fp8 = dict(a_dtype=_lib.E4M3, b_dtype=_lib.E5M2, a_scale=256, b_scale=256,
             rows=300, **common)
  assert call(_gemm_desc(k=4 * 128, **fp8)) == -1
  assert call(_gemm_desc(k=5 * 128, r=0, **fp8)) == 0
  assert call(_gemm_desc(k=0, rows=0, r=0, **common)) == 0


@pytest.mark.parametrize('q', [False, True])
def test_cotangent_on_another_device(monkeypatch, q):
  """Refused before any address of one device meets a kernel of another."""
  from tests import fake_block_lib
  fake_block_lib.install(monkeypatch)
  cfg = bs.dot_general_make()
  x, w = torch.zeros(4, 128, dtype=BF), torch.zeros(2, 128, 8, dtype=BF)
  s = torch.tensor([2, 2], dtype=torch.int32)
  backs = [rd.ragged_dot_vjp(x, w, s, cfg=cfg if q else None)[1]]
  if q:
    backs.append(cfg.vjp(x, w[0], DIMS)[1])
  for back in backs:
    with pytest.raises(ValueError, match='different devices'):
      back(torch.zeros(4, 8, dtype=BF, device='meta'))


def test_forward_mode_tangents(monkeypatch):
  """Refused, not dropped: with or without a leaf that wants a gradient."""
  from torch.autograd import forward_ad
  from tests import fake_block_lib
  fake_block_lib.install(monkeypatch)
  cfg = bs.dot_general_make()
  x, w = torch.ones(4, 128, dtype=BF), torch.ones(2, 128, 8, dtype=BF)
  s = torch.tensor([2, 2], dtype=torch.int32)
  qt, g = bs.block_quantize(w[0], 0, square=True), torch.ones(4, 8, dtype=BF)
  backs = [cfg.vjp(x, w[0], DIMS)[1], rd.ragged_dot_vjp(x, w, s)[1]]
  dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
  with forward_ad.dual_level():
    calls = [lambda: cfg(dual(x), w[0], DIMS), lambda: cfg(x, dual(w[0]), DIMS),
             lambda: cfg(dual(x), w[0].clone().requires_grad_(), DIMS),
             lambda: cfg(dual(x), qt, DIMS), lambda: cfg.vjp(dual(x), w[0], DIMS),
             lambda: bs.block_quantize(dual(x)),
             lambda: rd.ragged_dot(dual(x), w, s),
             lambda: rd.ragged_dot(x, dual(w), s, cfg=cfg),
             lambda: rd.ragged_dot_vjp(dual(x), w, s, cfg=cfg)]
    calls += [lambda back=back: back(dual(g)) for back in backs]
    for i, call in enumerate(calls):
      with pytest.raises(NotImplementedError, match='tangent'):
        call()
        pytest.fail(f'call {i} was not refused')
    cfg(x, w[0], DIMS)  # a level without tangents of its operands


def test_abi_gemm_columns_of_groups(lib):
  """With b's columns contiguous a group's tiles would start at any column, where
  no tiled copy may: refused before anything is launched."""
  call = lambda d: lib.aqtb200_grouped_gemm(C.byref(d), None, None)
  assert call(_gemm_desc(b_mn_major=1, b_ld=8, group_sizes=256, groups=2,
                         a_group_stride=4096)) == -2


def test_abi_notes_on_scales(lib):
  """Notes are of one matrix with 1 x 128 blocks, sixteen bytes each."""
  call = lambda d: lib.aqtb200_block_quantize(C.byref(d), None)
  assert call(_quant_desc(note_row=264)) == -2
  assert call(_quant_desc(note_row=256, square=1)) == -2
  d = _quant_desc(note_row=256)
  d.x.b0 = 2
  assert call(d) == -2
  d = _gemm_desc(a_dtype=_lib.E4M3, b_dtype=_lib.E4M3, a_scale=256, b_scale=256, note=264)
  assert lib.aqtb200_grouped_gemm(C.byref(d), None, None) == -1
