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
