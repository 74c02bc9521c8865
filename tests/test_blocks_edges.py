"""CPU tests of advoc_amd.blocks at its edges: the oracle with values that are no numbers at dropped places, and refusals of sizes
that no launch can be made for.  Nothing here reaches a device."""
import pytest
import torch

from advoc_amd import _lib, blocks
from oracle import blocks_torch as O


@pytest.fixture(scope='module')
def lib():
  import os
  if not os.path.isfile(_lib.LIB_PATH):
    import __graft_entry__ as g
    g.build()
  return _lib.load()


def test_the_oracle_selects_what_is_kept():
  """An infinity or NaN at a dropped place changes neither r nor a gradient."""
  g = torch.Generator().manual_seed(0)
  h, x, dr, gate, scale = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((6, 40), (6, 40), (6, 40), (6, 40), (40,)))
  mask = O.keep_mask(h.shape, 1, 0, 0.5)
  kw = dict(post='none', pre='none', keep=0.5, mask=mask, scale=scale)
  res = []
  for fill in (0.0, float('nan'), float('inf')):
    hh = torch.where(mask, h, torch.full((), fill, dtype=h.dtype))
    o = O.residual_norm(hh, x, gate, **kw)
    res.append((o['r'], O.residual_norm_backward(None, dr, hh, o['r'], o['stats'], gate, **kw)[0]))
  for r, grads in res[1:]:
    assert torch.equal(r, res[0][0])
    for k, v in grads.items():
      assert torch.equal(v, res[0][1][k]), k


def test_sizes_beyond_a_launch_are_refused(lib):
  """A launch holds 2^32 - 1 work-items: what would need more is refused before it is made, whatever form a product takes."""
  def drop(rows, cols, pad=0):
    return lib.advoc_dropout(64, cols + pad, 64, cols + pad, rows, cols, 1, 0.5, 0, 0, None, None)
  assert drop(2 ** 25, 1024) == -2 and drop(2 ** 25, 1024, 8) == -2 and drop(1, 2 ** 35) == -2

  def mul(m, n, k, dtype):
    return lib.advoc_matmul_nt_f8(64, 64, 0, 64, 64, 0, 64, dtype, 0, m, n, k, None, 0, None)
  for dtype in (0, 1):
    assert mul(1, 2 ** 26, 128, dtype) == -2 and mul(2, 2 ** 31, 128, dtype) == -2      # dot products: 64 work-items a column
    assert mul(3, 2 ** 27, 1024, dtype) == -2                                           # thin: 32 of them
    assert mul(2 ** 31, 1, 128, dtype) == -2 and mul(2 ** 22, 2 ** 18, 128, dtype) == -2      # tiles
