"""CPU tests of the residual-block operators: the oracle's own formulas (gradients against autograd and differences, 8-bit rounding
against torch's types), and what the library and the binding refuse before anything reaches a device."""
import ctypes

import numpy as np
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


# ---- the oracle ----
def test_philox_known_answers():
  """The generator's published vectors for a zero and an all-ones counter are not reachable through a 64-bit counter except the
  zero one: counter 0, key 0 -> 6627e8d5 e169c58d bc57ac4c 9b00dbd8."""
  assert [hex(w) for w in O.philox_words(0, 0, 4)] == ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']
  a = O.philox_words(2 ** 40 + 5, 0, 64)
  assert np.array_equal(O.philox_words(2 ** 40 + 5, 13, 20), a[13:33])


def _norm_case(post, pre, gate, act, rows=(2, 3), cols=7, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)      # noqa: E731
  t = dict(h=r(*rows, cols), x=r(*rows, cols), gate=None if gate == 'none' else r(rows[0], rows[1] if gate == 'row' else 1, cols))
  p = dict(w_post=r(cols) if post != 'none' else None, b_post=r(cols) if post != 'none' else None, scale=r(cols),
           w_pre=r(cols) if pre != 'none' else None, b_pre=r(cols) if pre != 'none' else None)
  return t, p, dict(post=post, pre=pre, act=act, alpha=0.7)


@pytest.mark.parametrize('post,pre,gate,act', [('rms', 'layer', 'row', 'sigmoid'), ('layer', 'rms', 'clip', 'none'),
                                               ('none', 'layer', 'none', 'none'), ('layer', 'none', 'clip', 'sigmoid')])
def test_oracle_gradients_are_autograds_and_differences(post, pre, gate, act):
  t, p, kw = _norm_case(post, pre, gate, act)
  keep = 0.6
  mask = O.keep_mask(t['h'].shape, 3, 0, keep)
  leaves = {k: v.requires_grad_() for k, v in {**t, **p}.items() if v is not None}
  g = torch.Generator().manual_seed(9)
  dz, dr = (torch.randn(t['h'].shape, generator=g, dtype=torch.float64) for _ in range(2))

  def loss(**over):
    f = {**t, **p, **over}
    o = O.residual_norm(keep=keep, mask=mask, **f, **kw)
    return (o['r'] * dr).sum() + (0 if o['z'] is None else (o['z'] * dz).sum()), o
  total, o = loss()
  want = dict(zip(leaves, torch.autograd.grad(total, list(leaves.values()))))
  f = {k: None if v is None else v.detach() for k, v in {**t, **p}.items()}
  del f['x'], kw['alpha']
  got, _ = O.residual_norm_backward(None if pre == 'none' else dz, dr, f.pop('h'), o['r'].detach(), o['stats'].detach(), keep=keep,
                                    mask=mask, alpha=0.7, **f, **kw)
  assert sorted(got) == sorted('d' + k for k in want)
  kw['alpha'] = 0.7
  for k, w in want.items():
    torch.testing.assert_close(got['d' + k], w, rtol=1e-11, atol=1e-12)
    v = leaves[k].detach()
    d = torch.randn(v.shape, generator=g, dtype=torch.float64)
    with torch.no_grad():
      diff = (loss(**{k: v + 1e-6 * d})[0] - loss(**{k: v - 1e-6 * d})[0]) / 2e-6
    assert abs(diff - (w * d).sum()) < 1e-7 * (1 + (w * d).abs().sum()), k


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
def test_oracle_rounding_is_the_types(fmt):
  kind = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}[fmt]
  g = torch.Generator().manual_seed(1)
  x = torch.randn(40, 300, generator=g, dtype=torch.float64) * torch.exp(3 * torch.randn(40, 1, generator=g, dtype=torch.float64))
  x = x.to(torch.bfloat16).double()                        # ties happen
  v, e = O.f8_blocks(x, fmt)
  s = torch.exp2(e.double() - 127).repeat_interleave(128, 1)[:, :300]
  assert torch.equal((x / s).float().to(kind).double() * s, v)
  top = O.F8[fmt][2]
  amax = torch.nn.functional.pad(x, (0, 84)).reshape(40, 3, 128).abs().amax(-1)
  assert (amax <= top * torch.exp2(e.double() - 127)).all() and (amax > top * torch.exp2(e.double() - 128)).all()


# ---- refusals: nothing below reaches a device ----
def test_struct_layout_matches_the_header(tmp_path):
  import os
  import subprocess
  fields = [f[0] for f in _lib.ResidualNorm._fields_]
  src = ['#include <stdio.h>', '#include <stddef.h>', '#include "advoc_hip.h"', 'int main(void) {',
         '  printf("sizeof %zu\\n", sizeof(advoc_residual_norm));']
  src += ['  printf("%s %%zu\\n", offsetof(advoc_residual_norm, %s));' % (f, f) for f in fields] + ['  return 0;', '}']
  c, exe = tmp_path / 'layout.c', tmp_path / 'layout'
  c.write_text('\n'.join(src))
  subprocess.run(['gcc', '-std=c99', '-I', os.path.dirname(_lib.HEADER_PATH), str(c), '-o', str(exe)], check=True)
  out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
  assert int(out['sizeof']) == ctypes.sizeof(_lib.ResidualNorm)
  for f in fields:
    assert int(out[f]) == getattr(_lib.ResidualNorm, f).offset, f


def test_packed_descriptor_is_the_struct():
  n = len(blocks._DESCRIPTOR.unpack(bytes(blocks._DESCRIPTOR.size)))
  assert blocks._DESCRIPTOR.size == ctypes.sizeof(_lib.ResidualNorm) == blocks._DESCRIPTOR_HEAD.size + blocks._DESCRIPTOR_TAIL.size
  d = _lib.ResidualNorm.from_buffer_copy(blocks._DESCRIPTOR.pack(*range(1, n + 1)))
  flat = []
  for name, _ in _lib.ResidualNorm._fields_:
    v = getattr(d, name)
    flat += [v.p, v.pitch] if isinstance(v, _lib.Rows) else [v]
  assert flat == list(range(1, n + 1))


def test_dropout_entry_refuses(lib):
  ok = dict(x=16, xp=8, y=16, yp=8, rows=2, cols=8, dtype=0, keep=0.5, seed=0, offset=0, dev=None)

  def call(**kw):
    a = {**ok, **kw}
    return lib.advoc_dropout(*a.values(), None)
  assert call(x=None) == -4 and call(y=None) == -4
  assert call(rows=-1) == -1 and call(cols=-1) == -1 and call(xp=7) == -1 and call(yp=7) == -1
  for keep in (0.0, -0.5, 1.5, float('nan')):
    assert call(keep=keep) == -1
  assert call(dtype=3) == -2 and call(offset=2) == -2
  assert call(rows=2 ** 40, cols=2, xp=2, yp=2) == -2
  assert call(rows=2, cols=2 ** 31, xp=2 ** 31 + 1, yp=2 ** 31) == -2
  assert call(rows=0, x=None) == 0 and call(cols=0, x=None) == 0


def _norm_desc(**kw):
  d = _lib.ResidualNorm()
  d.rows, d.cols, d.gate_group, d.alpha, d.eps, d.keep_prob, d.norm_post, d.norm_pre = 4, 8, 1, 1.0, 1e-5, 1.0, 1, 1
  for name in ('h', 'x', 'r', 'z', 'dz', 'dr', 'dh', 'dx'):
    getattr(d, name).p, getattr(d, name).pitch = 64, 8
  d.stats = 64
  for k, v in kw.items():
    if isinstance(v, tuple):
      getattr(d, k).p, getattr(d, k).pitch = v
    else:
      setattr(d, k, v)
  return ctypes.byref(d)


@pytest.mark.parametrize('bad,code', [
    (dict(rows=-1), -1), (dict(cols=0), -1), (dict(eps=0.0), -1), (dict(eps=float('nan')), -1), (dict(keep_prob=0.0), -1),
    (dict(keep_prob=1.1), -1), (dict(norm_post=3), -2), (dict(norm_pre=-1), -2), (dict(gate_act=2), -2), (dict(dtype=3), -2),
    (dict(dtype=1, res_dtype=2), -2), (dict(cols=8193), -2), (dict(rows=2 ** 31), -2), (dict(offset=1), -2),
    (dict(gate=(64, 8), gate_group=3), -1), (dict(gate=(64, 8), gate_group=0), -1), (dict(gate=(64, 7)), -1), (dict(h=(64, 7)), -1),
    (dict(x=(64, 7)), -1), (dict(z=(64, 7)), -1), (dict(r=(64, 7)), -1), (dict(h=(None, 0)), -1), (dict(stats=68), -2),
    (dict(h=(None, 0), norm_post=0, norm_pre=0), -1)])
def test_norm_entries_refuse(lib, bad, code):
  assert lib.advoc_residual_norm_forward(_norm_desc(**bad), None) == code
  if 'x' not in bad:                                       # the backward pass reads r
    assert lib.advoc_residual_norm_backward(_norm_desc(**bad), None) == code


def test_norm_entries_refuse_missing_tensors(lib):
  none = (None, 0)
  fwd, bwd = lib.advoc_residual_norm_forward, lib.advoc_residual_norm_backward
  assert fwd(None, None) == -4 and bwd(None, None) == -4
  assert fwd(_norm_desc(x=none), None) == -4 and fwd(_norm_desc(r=none), None) == -4 and fwd(_norm_desc(z=none), None) == -4
  assert bwd(_norm_desc(dz=none), None) == -4 and bwd(_norm_desc(r=none), None) == -4 and bwd(_norm_desc(stats=None), None) == -4
  assert bwd(_norm_desc(norm_pre=0, dr=none), None) == -4
  assert bwd(_norm_desc(dw_pre=64), None) == -4            # wants scratch, has none
  assert bwd(_norm_desc(dw_pre=64, workspace=64, workspace_bytes=4), None) == -4
  assert bwd(_norm_desc(dgate=(64, 7), gate=(64, 8)), None) == -1
  assert fwd(_norm_desc(rows=0), None) == 0 and bwd(_norm_desc(rows=0), None) == 0
  assert lib.advoc_residual_norm_workspace_bytes(None) == 0
  assert lib.advoc_residual_norm_workspace_bytes(_norm_desc()) == 0
  one, two = (lib.advoc_residual_norm_workspace_bytes(_norm_desc(**k)) for k in (dict(dw_pre=64), dict(dw_pre=64, dscale=64)))
  assert one > 0 and two == 2 * one


def test_f8_entries_refuse(lib):
  q = dict(x=64, pitch=8, rows=2, cols=8, dtype=0, fmt=0, q=64, s=64, qt=64, st=64)

  def quant(**kw):
    return lib.advoc_f8_quantize(*{**q, **kw}.values(), None)
  assert quant(x=None) == -4 and quant(q=None, qt=None) == -4 and quant(s=None) == -4 and quant(st=None) == -4
  assert quant(rows=-1) == -1 and quant(pitch=7) == -1 and quant(dtype=9) == -2 and quant(fmt=2) == -2 and quant(q=72) == -2
  assert quant(rows=2 ** 31) == -2 and quant(rows=1, cols=2 ** 30) == -2 and quant(rows=0) == 0
  m = dict(a=64, sa=64, fa=0, b=64, sb=64, fb=0, out=64, dtype=0, acc=0, m=4, n=4, k=4, ws=None, wsb=0)

  def mul(**kw):
    return lib.advoc_matmul_nt_f8(*{**m, **kw}.values(), None)
  for k in ('a', 'sa', 'b', 'sb', 'out'):
    assert mul(**{k: None}) == -4
  assert mul(m=-1) == -1 and mul(k=0) == -1 and mul(fa=2) == -2 and mul(fb=-1) == -2 and mul(dtype=5) == -2
  assert mul(acc=1, dtype=1) == -2 and mul(a=72) == -2 and mul(sa=66) == -2 and mul(sb=65) == -2 and mul(k=2 ** 24) == -2 and mul(n=2 ** 32) == -2 and mul(m=2 ** 24, n=2 ** 24) == -2
  assert mul(m=0) == 0 and mul(n=0, out=None) == 0
  assert lib.advoc_matmul_nt_f8_workspace_bytes(0, 4, 4, 0) == 0 and lib.advoc_matmul_nt_f8_workspace_bytes(1, 4, 4, 0) == 0


def test_binding_refuses_what_is_not_on_a_device():
  x = torch.zeros(4, 8)
  for call in (lambda: blocks.dropout(x, 0.5, 1), lambda: blocks.quantize_f8(x), lambda: blocks.quantize_f8_both(x),
               lambda: blocks.ResidualNorm(8).forward(x, x), lambda: blocks.ResidualNorm(8).backward(x, x, x, x, x),
               lambda: blocks.matmul_nt_f8(x, x)):
    with pytest.raises(_lib.AdvocHipError):
      call()


def test_binding_refuses_bad_options():
  for kw in (dict(cols=0), dict(cols=8193), dict(cols=8, post='batch'), dict(cols=8, pre=None), dict(cols=8, gate_act='tanh'),
             dict(cols=8, eps=0.0), dict(cols=8, keep_prob=0.0), dict(cols=8, keep_prob=1.5),
             dict(cols=8, post='none', w_post=torch.zeros(8)), dict(cols=8, pre='none', b_pre=torch.zeros(8))):
    with pytest.raises(_lib.AdvocHipError):
      blocks.ResidualNorm(**kw)
