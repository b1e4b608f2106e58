"""The status words of the block-scaled and grouped products on a device: memory
that its kernels and the host share."""

import ctypes as C

import pytest
import torch

from aqt_b200 import _lib
from aqt_b200 import engine
from aqt_b200.v2 import aqt_ragged_dot as rd
from aqt_b200.v2 import block_scaled as bs

pytestmark = pytest.mark.gpu

DIMS = (((1,), (0,)), ((), ()))


def _data(shape, seed):
  gen = torch.Generator('cuda').manual_seed(seed)
  return torch.randn(shape, device='cuda', generator=gen).bfloat16()


def test_kernels_write_what_the_host_reads():
  words = engine.status_words(torch.device('cuda', 0))
  engine.check_status()
  x = torch.zeros(1, 8, device='cuda', dtype=torch.bfloat16)
  x[0, 0] = 1.0  # the 16 bytes of the words: 0x3f80, zeros
  view = _lib.View(x.data_ptr(), _lib.BF16, 0, 1, 1, 1, 8, 0, 0, 8, 1)
  _lib.check(_lib.load().aqtb200_pack_bf16(C.byref(view), words, 8,
                                           engine._stream()), 'pack')  # pylint: disable=protected-access
  torch.cuda.synchronize()
  assert list(words) == [0x3f80, 0, 0, 0]
  a, w = _data((5, 128), 1), _data((128, 64), 2)
  with pytest.raises(_lib.AqtB200Error, match='gave up'):
    bs.dot_general_make()(a, w, DIMS)
  engine.check_status()
  bs.dot_general_make()(a, w, DIMS)
  engine.check_status()


def test_first_call_under_capture():
  """Its graph can report, and what it reported outlives the graph."""
  x, w = _data((20, 128), 3), _data((2, 128, 64), 4)
  sizes = torch.tensor([12, 8], device='cuda')
  cfg = bs.dot_general_make()
  want = rd.ragged_dot(x, w, sizes), rd.ragged_dot(x, w, sizes, cfg=cfg)
  torch.cuda.synchronize()
  engine._words.clear()  # pylint: disable=protected-access
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = rd.ragged_dot(x, w, sizes), rd.ragged_dot(x, w, sizes, cfg=cfg)
  words = engine._words[x.device]  # pylint: disable=protected-access
  graph.replay()
  engine.check_status()
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  del graph, got
  words[0] = 4  # as a kernel of a replay would
  with pytest.raises(_lib.AqtB200Error, match='role 4'):
    rd.ragged_dot(x, w, sizes)
  engine.check_status()


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'po2', 'decode'])
def test_the_sm_budget_caps_these_products_too(kind):
  """A caller that keeps SMs free for a collective beside the products."""
  m = 16 if kind == 'decode' else 2048
  x, w = _data((m, 2048), 5), _data((2048, 8192), 6)
  if kind == 'bf16':
    sizes = torch.tensor([m], device='cuda')
    run = lambda: rd.ragged_dot(x, w[None], sizes)
  else:
    cfg = bs.dot_general_make(po2_scale=kind == 'po2')
    w = bs.block_quantize(w, 0, square=True) if kind == 'decode' else w
    run = lambda: cfg(x, w, DIMS)

  def products():
    """Results, and microseconds of the product kernels alone."""
    out = run()
    torch.cuda.synchronize()
    with torch.profiler.profile(
        activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
      for _ in range(3):
        run()
      torch.cuda.synchronize()
    return out, min(e.device_time_total for e in prof.events()
                    if 'grouped_gemm' in e.name)

  out, free = products()
  engine.set_gemm_sm_budget(8)
  try:
    capped, slow = products()
  finally:
    engine.set_gemm_sm_budget(0)
  engine.check_status()
  # 8 of 148 SMs: 18 times the work an SM; a decode stops at the memory's rate and
  # loses less
  assert slow > (2 if kind == 'decode' else 4) * free
  assert torch.allclose(out.float(), capped.float(), rtol=2.0 ** -7,
                        atol=float(out.abs().max()) * 2.0 ** -8)
