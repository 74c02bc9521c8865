"""One batch sweep of the LWS phase reconstruction against the float64 local sums of oracle/lws_np.py, bin by bin, with windows
that are symmetric (the sweep's weights are real numbers but for turns) and windows that are not.

u = 2^-24.  A bin's sum has 62 terms w x: 62 roundings of their sum, at most 30 more of a term (its value and weight turned, a weight
rounded when the table was, the sum turned back): |dz| <= 128 u S, S = sum |w x|.  The bin becomes a z / |z|: off by a |dz| / |z| and a
few u.  Bins where |dz| / |z| could pass 1 / 16 are left out; there are few."""
import numpy as np
import pytest
import torch

from oracle import lws_np

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def table(awin, swin):
  K = lws_np.projection_kernel(awin, swin, 256, 5)
  q, r = np.arange(-3, 4), np.arange(4)
  return K, (K[:, :, None] * np.exp(-0.5j * np.pi * (q[:, None, None] * r[None, None, :]))).astype(np.complex64)


def windows(kind):
  n = np.arange(1024)
  w = np.sin(np.pi * (n + 0.5) / 1024) / np.sqrt(2)
  if kind == 'symmetric':
    return w, w
  if kind == 'two':                                       # symmetric both, but not the same
    return w, w * (1 + 0.3 * np.cos(2 * np.pi * (n + 0.5) / 1024))
  if kind == 'nearly':                                    # off by more than a table's rounding, and by less than shows
    return w * (1 + 1e-5 * n / 1024), w
  return w * (0.3 + n / 1024), w * (1.2 - n / 1024)


@pytest.mark.parametrize('T', [1, 5, 8, 21])
@pytest.mark.parametrize('kind', ['symmetric', 'two', 'nearly', 'asymmetric'])
def test_a_sweep_is_the_local_sums(hip, kind, T):
  from advoc_amd import _lib
  lib = _lib.load()
  awin, swin = windows(kind)
  K, W = table(awin, swin)
  rng = np.random.default_rng(T)
  clips = 2
  X = (rng.standard_normal((clips, T, 513)) + 1j * rng.standard_normal((clips, T, 513))).astype(np.complex64)
  X[:, :, 0] = X[:, :, 0].real                             # (as a real signal's is; the mirrored bins are its neighbours')
  mag = (np.abs(X) * rng.uniform(0.5, 2.0, X.shape)).astype(np.float32)
  mean = mag.mean(axis=(1, 2)).astype(np.float32)
  d = [torch.from_numpy(t).cuda() for t in (X.view(np.float32), mag, mean, W.view(np.float32))]
  out = torch.full((clips, T, 513, 2), float('nan'), device='cuda')
  _lib.check(lib.advoc_lws_batch_c64(_lib.ptr(d[0]), _lib.ptr(out), _lib.ptr(d[1]), _lib.ptr(d[2]), clips, T, 1024, 256, _lib.ptr(d[3]),
                                     4, 5, 0.7, _lib.stream()))
  got = torch.view_as_complex(out).cpu().numpy()
  left_out = 0
  for c in range(clips):
    above = mag[c] > np.float32(0.7) * mean[c]
    assert 0 < above.sum() < above.size and np.array_equal(got[c][~above], X[c][~above])
    z = lws_np.local_sums(X[c].astype(np.complex128), K, 256, 1024, list(range(-3, 4)))
    size = lws_np.local_sums(np.abs(X[c]).astype(np.complex128), np.abs(K), 256, 1024, [0]).real
    for q in (-3, -2, -1, 1, 2, 3):                       # (of magnitudes: without the turns of other frames)
      size[max(0, -q):T - max(0, q)] += lws_np.local_sums(np.abs(X[c][max(0, q):T + min(0, q)]).astype(np.complex128), np.abs(K[q + 3:q + 4]),
                                                           256, 1024, [0], include_centre=True).real if T > abs(q) else 0
    turn = 128 * U * size / np.abs(z)
    sure = above & (turn < 1 / 16)
    left_out += (above & ~sure).sum()
    want = mag[c] * z / np.abs(z)
    err, tol = np.abs(got[c] - want), mag[c] * (1.1 * turn + 8 * U)
    assert (err[sure] <= tol[sure]).all(), (err[sure] / tol[sure]).max()
    assert np.allclose(np.abs(got[c][above]), mag[c][above], rtol=8 * U)
  assert left_out < 0.01 * clips * T * 513
