"""GPU tests of advoc_amd.blocks where a call meets what it should not let through: values that are no numbers at places that are
dropped, empty calls, outputs of other shapes and types, and the ends of the exponent range.  Expected values are exact (the same
bits as a call without the bad value, or whole numbers and powers of two), but for where a tolerance is derived beside it."""
import ctypes

import pytest
import torch

import test_hip_blocks as T
from oracle import blocks_torch as O

pytestmark = pytest.mark.gpu
BAD = [float('inf'), -float('inf'), float('nan')]
COLS = [5, 40, 96, 200, 513, 1000, 2048, 4100]      # every way a row lies on lanes


@pytest.fixture(scope='module')
def blocks():
  from advoc_amd import _lib, blocks
  assert torch.cuda.is_available(), 'gpu-marked test running without a HIP device'
  _lib.load()
  return blocks


def gen(seed):
  return torch.Generator().manual_seed(seed)


# ---- values that are no numbers where an element is dropped ----
@pytest.mark.parametrize('gates', ['none', 'row', 'clip'])
@pytest.mark.parametrize('cols', COLS)
def test_a_dropped_value_that_is_no_number_adds_nothing_to_gradients(blocks, cols, gates):
  """Without a post norm an infinity or NaN of h at a dropped place leaves r and z as they were; every gradient has the bits it
  has with a zero in that place."""
  clips, frames, keep, seed = 3, 7, 0.5, 19
  r = lambda *s: torch.randn(*s, generator=gen(cols + sum(s)))      # noqa: E731
  h, x, dz, dr = (r(clips, frames, cols) + i for i in range(4))
  gate = {'none': None, 'row': r(clips, frames, cols), 'clip': r(clips, 1, cols)}[gates]
  gate = None if gate is None else gate.cuda()
  dropped = ~O.keep_mask(h.shape, seed, 0, keep)
  spots = dropped.flatten().nonzero().flatten()[::5]
  for pre in ('layer', 'none'):
    norm = blocks.ResidualNorm(cols, post='none', pre=pre, gate_act='sigmoid', alpha=0.7, keep_prob=keep, scale=r(cols).cuda(),
                               w_pre=r(cols).cuda() if pre != 'none' else None)
    call = dict(gate=gate, seed=seed)
    res = []
    for fill in (torch.zeros(len(spots)), torch.tensor(BAD).repeat(len(spots))[:len(spots)]):
      hh = h.clone().flatten()
      hh[spots] = fill
      hh = hh.reshape(h.shape).cuda()
      o, z, stats = norm.forward(hh, x.cuda(), save=True, **call)
      g = norm.backward(dz.cuda() if pre != 'none' else None, dr.cuda(), hh, o, stats, **call)
      res.append(dict(r=o, z=z, stats=stats, **g._asdict()))
    for name, want in res[0].items():
      if want is not None:
        assert torch.isfinite(want).all() and torch.equal(res[1][name], want), (pre, name)


@pytest.mark.parametrize('cols', COLS)
def test_a_bad_row_adds_nothing_where_it_is_dropped(blocks, cols):
  """With a post norm a NaN makes its row one: the column sums of elements that are dropped in that row stay what they are without
  it, and so does a gate's gradient there."""
  rows, keep, seed = 9, 0.5, 23
  r = lambda *s: torch.randn(*s, generator=gen(cols + sum(s)))      # noqa: E731
  h, x, dr, gate = (r(rows, cols) + i for i in range(4))
  dropped = ~O.keep_mask(h.shape, seed, 0, keep)
  norm = blocks.ResidualNorm(cols, post='rms', pre='none', keep_prob=keep, w_post=r(cols).cuda(), b_post=r(cols).cuda(), scale=r(cols).cuda())
  res = []
  for bad in (0.0, float('nan')):
    h[4, 2] = bad
    o, _, stats = norm.forward(h.cuda(), x.cuda(), gate=gate.cuda(), seed=seed, save=True)
    res.append(norm.backward(None, dr.cuda(), h.cuda(), o, stats, gate=gate.cuda(), seed=seed))
  at = dropped[4].cuda()
  for name in ('dscale', 'dw_post', 'db_post'):
    assert torch.equal(getattr(res[0], name)[at], getattr(res[1], name)[at]), name
  assert torch.equal(res[0].dgate[4][at], res[1].dgate[4][at]) and torch.equal(res[0].dx, res[1].dx)
  others = [i for i in range(rows) if i != 4]
  assert torch.equal(res[0].dh[others], res[1].dh[others]) and torch.equal(res[0].dgate[others], res[1].dgate[others])


def test_an_infinite_gate_leaves_a_dropped_gradient_zero(blocks):
  """The gradient of what was dropped is 0 whatever its gate holds."""
  cols, keep, seed = 200, 0.5, 3
  x, gate = torch.ones(6, cols), torch.ones(6, cols)
  dropped = ~O.keep_mask(x.shape, seed, 0, keep)
  gate[dropped] = float('inf')
  norm = blocks.ResidualNorm(cols, post='none', pre='none', keep_prob=keep)
  g = norm.backward(None, x.cuda(), x.cuda(), x.cuda(), None, gate=gate.cuda(), seed=seed)
  assert bool((g.dh.cpu()[dropped] == 0).all()) and bool((g.dgate.cpu()[dropped] == 0).all())
  assert bool((g.dh.cpu()[~dropped] == 2).all())


# ---- empty calls, and outputs of other shapes and types ----
@pytest.mark.parametrize('has_h', [True, False])
def test_a_backward_call_without_rows_clears_what_it_overwrites(blocks, has_h):
  """Sums over no rows are 0: written by the C entry, left alone where they are added to or not wanted."""
  from advoc_amd import _lib
  cols = 1030
  arena = torch.full((6, cols), 3.0, device='cuda')
  names = ['dw_post', 'db_post', 'dscale', 'dw_pre', 'db_pre']
  q = _lib.ResidualNorm()
  q.cols, q.gate_group, q.alpha, q.eps, q.keep_prob, q.norm_pre, q.norm_post = cols, 1, 1.0, 1e-5, 1.0, 1, 1 if has_h else 0
  if has_h:
    q.h.p, q.h.pitch = arena.data_ptr(), cols
  for i, name in enumerate(names):
    setattr(q, name, arena[i].data_ptr())
  q.db_pre = None
  lib = _lib.load()
  q.accumulate = 1
  _lib.check(lib.advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  assert bool((arena == 3).all())
  q.accumulate = 0
  _lib.check(lib.advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  cleared = ('dw_post', 'db_post', 'dscale', 'dw_pre') if has_h else ('dscale', 'dw_pre')
  for i, name in enumerate(names):
    assert bool((arena[i] == (0 if name in cleared else 3)).all()), name
  assert bool((arena[5] == 3).all())


def test_a_backward_call_without_rows_through_the_binding(blocks):
  e = torch.zeros(0, 16, device='cuda')
  norm = blocks.ResidualNorm(16, w_pre=torch.ones(16, device='cuda'), scale=torch.ones(16, device='cuda'))
  into = {k: torch.full((16,), 5.0, device='cuda') for k in ('dw_pre', 'dscale')}
  r, z, stats = norm.forward(e, e, save=True)
  g = norm.backward(z, r, e, r, stats, into=into, accumulate=True)
  assert bool((g.dw_pre == 5).all()) and bool((g.dscale == 5).all())
  g = norm.backward(z, r, e, r, stats, into=into)
  assert g.dw_pre is into['dw_pre'] and bool((g.dw_pre == 0).all()) and bool((g.dscale == 0).all())


def test_gradients_have_their_tensors_shapes(blocks):
  """h may lie in another leading shape than x, as a product leaves it: its gradient has h's."""
  x = torch.randn(2, 6, 40, generator=gen(0)).cuda()
  h = torch.randn(12, 40, generator=gen(1)).cuda().bfloat16()
  norm = blocks.ResidualNorm(40, scale=torch.ones(40, device='cuda'))
  r, z, stats = norm.forward(h, x, save=True)
  assert r.shape == z.shape == x.shape
  g = norm.backward(z, r, h, r, stats)
  same = norm.backward(z, r, h.view(2, 6, 40), r, stats)
  assert g.dh.shape == h.shape and g.dh.dtype == h.dtype and g.dx.shape == x.shape
  assert same.dh.shape == x.shape and torch.equal(same.dh.view(12, 40), g.dh)


def test_product_into_a_buffer_of_another_type_than_asked(blocks):
  """out decides the result's type when no type is named; one that is named has to be its."""
  from advoc_amd._lib import AdvocHipError
  x = torch.randn(20, 200, generator=gen(0)).cuda()
  q = blocks.quantize_f8(x)
  out = torch.empty(20, 20, dtype=torch.bfloat16, device='cuda')
  assert blocks.matmul_nt_f8(q, q, out=out) is out and torch.equal(out, blocks.matmul_nt_f8(q, q, out_dtype=torch.bfloat16))
  assert blocks.matmul_nt_f8(q, q, out=out, out_dtype=torch.bfloat16) is out and blocks.matmul_nt_f8(q, q).dtype == torch.float32
  for other in (torch.float32, torch.float16):
    with pytest.raises(AdvocHipError):
      blocks.matmul_nt_f8(q, q, out=out, out_dtype=other)


def test_buffers_that_a_call_would_not_write_are_refused(blocks):
  from advoc_amd._lib import AdvocHipError
  x, buf = torch.randn(4, 40, generator=gen(0)).cuda(), torch.full((4, 40), 7.0, device='cuda')
  with pytest.raises(AdvocHipError):
    blocks.ResidualNorm(40).forward(None, x, r=buf)                      # r is x
  with pytest.raises(AdvocHipError):
    blocks.ResidualNorm(40, pre='none').forward(x, x, z=buf)             # there is no z
  assert bool((buf == 7).all())
  r, z, _ = blocks.ResidualNorm(40).forward(None, x, r=x, z=buf)
  assert r is x and z is buf


def test_tensors_that_autograd_follows_are_refused(blocks):
  """No call records a gradient: a tensor that needs one is taken only where autograd is off."""
  from advoc_amd._lib import AdvocHipError
  x = torch.randn(4, 40, generator=gen(0)).cuda()
  leaf = x.clone().requires_grad_()
  norm = blocks.ResidualNorm(40)
  r, z, stats = norm.forward(x, x, save=True)
  calls = [lambda t: blocks.dropout(t, 0.5, 1), lambda t: blocks.quantize_f8(t), lambda t: blocks.quantize_f8_both(t),
           lambda t: norm.forward(t, x), lambda t: norm.forward(x, t), lambda t: norm.forward(x, x, gate=t),
           lambda t: norm.backward(t, x, x, r, stats), lambda t: norm.backward(z, x, t, r, stats)]
  for i, call in enumerate(calls):
    for t in (leaf, leaf * 2):
      with pytest.raises(AdvocHipError, match='autograd'):
        call(t)
        pytest.fail('case %d was taken' % i)
    with torch.no_grad():
      call(leaf)
    call(leaf.detach())
  # parameters belong to whoever updates them with the gradients that backward returns
  p = torch.nn.Parameter(torch.ones(40, device='cuda'))
  assert blocks.ResidualNorm(40, w_pre=p).forward(x, x)[1].requires_grad is False


# ---- the ends of the exponent range ----
@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('m', [1, 3, 16, 70, 300])
def test_product_at_the_ends_of_the_exponent_range(blocks, fmt, m):
  """fp32 outputs of three rows and more take what a value stands for as a bfloat16: a multiple of 2^-133 below 2^-130, infinite at
  2^128.  16-bit outputs and one or two rows take it as it is.  A term to an output, powers of two on the other side: exact."""
  types = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}
  lead = torch.tensor([100.0, 110, 114, 116, 118, 120, 124, 126])
  tiny = torch.zeros(64, 128)
  tiny[:, 0] = torch.exp2(-lead).repeat(8)                              # the block's largest, times 0
  tiny[:, 1] = tiny[:, 0] * torch.exp2(-torch.arange(64) / 4.0)
  huge = torch.zeros(8, 128)
  huge[:, 1] = torch.tensor([1.5e38, 1.7e38, 3.0e38, 3.1e38, 3.2e38, 3.3e38, 3.39e38, torch.finfo(torch.float32).max])
  for b, up in ((tiny, 2.0 ** 100), (huge, 2.0 ** -120)):
    a = torch.zeros(m, 128)
    a[:, 1] = up
    qa, qb = blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda(), fmt)
    v = qb.data.cpu().view(types[fmt]).float()[:, 1].double() * torch.exp2(qb.scale.cpu()[:, 0].double() - 127)
    assert bool((v == 2.0 ** 128).any()) == (b is huge)
    as_taken = v if m < 3 else v.bfloat16().double()
    assert torch.equal(blocks.matmul_nt_f8(qa, qb).cpu().double(), (as_taken * up).expand(m, -1))
    got = blocks.matmul_nt_f8(qa, qb, out_dtype=torch.bfloat16).cpu()
    assert torch.equal(got, (v * up).bfloat16().expand(m, -1))


def test_a_sigmoid_gate_that_is_nearly_shut(blocks):
  """Within 6 units in the last place down to the smallest normal number; a smaller value is 0 or that near."""
  gate = torch.linspace(-104, -86, 512, device='cuda').reshape(1, 512)
  norm = blocks.ResidualNorm(512, post='none', pre='none', gate_act='sigmoid')
  r = norm.forward(torch.ones(1, 512, device='cuda'), torch.zeros(1, 512, device='cuda'), gate=gate)[0].cpu().double()
  want = torch.sigmoid(gate.cpu().double())
  near = (r - want).abs() <= 12 * 2.0 ** -24 * want
  normal = want >= 2.0 ** -126 * (1 + 2.0 ** -20)
  assert bool(near[normal].all()) and bool((near | (r == 0))[~normal].all()) and 0 < int(normal.sum()) < 100


# ---- rows of a little more than a power of two ----
@pytest.mark.parametrize('kind', [0, 1, 2, 3])
@pytest.mark.parametrize('cols', [2050, 2057, 2303, 2304, 2305, 4097, 4103, 4607, 4608, 4609])
def test_norm_of_nine_columns_a_lane(blocks, cols, kind):
  """Every output against float64 at the edges of these widths (tolerances of tests/test_hip_blocks.py)."""
  T.check_norm(blocks, cols + kind, (3, 5), cols, *T.TYPES[kind], *T.KINDS[kind])


@pytest.mark.parametrize('cols', [2050, 2304, 4100])
def test_norm_of_nine_columns_a_lane_over_its_inputs(blocks, cols):
  """r over x and z over h, dx over dr and dh over h: a workgroup's waves that hold the same columns, clips cut into segments."""
  from advoc_amd import _lib
  norm, d, call, g, (r, z, stats) = T.check_norm(blocks, 2, (200, 3), cols, 'f32', 'f32', 'rms', 'layer', 'clip', 'sigmoid', 0.9)
  h, x = d['h'].clone(), d['x'].clone()
  norm.forward(h, x, r=x, z=h, **call)
  assert torch.equal(x, r) and torch.equal(h, z)
  h, dr = d['h'].clone(), d['dr'].clone()
  q = T.descriptor(norm, r, d['gate'], call)
  for name, t in (('dz', d['dz']), ('dr', dr), ('dx', dr), ('h', h), ('dh', h)):
    getattr(q, name).p, getattr(q, name).pitch = t.data_ptr(), cols
  q.stats = stats.data_ptr()
  assert _lib.load().advoc_residual_norm_workspace_bytes(ctypes.byref(q)) == 0
  _lib.check(_lib.load().advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  assert torch.equal(dr, g.dx) and torch.equal(h, g.dh)


def test_the_modules_example(blocks):
  """The block of the module's text, twice in a row in 16 bits: what one block hands back is what the one before takes."""
  import textwrap
  lines = textwrap.dedent(blocks.__doc__[blocks.__doc__.index('  norm = blocks'):])
  cols, r = 136, lambda *s: torch.randn(*s, generator=gen(sum(s))).cuda()      # noqa: E731
  f = dict(blocks=blocks, cols=cols, w_post=r(cols), scale=r(cols), w_pre=r(cols), w=r(cols, cols) * cols ** -0.5, step=3, x=r(2, 9, cols),
           gate=r(2, 1, cols).bfloat16(), z=r(2, 9, cols).bfloat16(), dz1=r(2, 9, cols).bfloat16(), dr=r(2, 9, cols))
  for _ in range(2):
    exec(lines, f)
    assert f['y'].dtype == f['dz'].dtype == f['z1'].dtype == torch.bfloat16 and f['dw'].dtype == torch.float32
    assert f['dz'].shape == (18, cols) and f['dw'].shape == (cols, cols) and f['g'].dh.shape == f['y'].shape
    assert all(bool(torch.isfinite(f[k]).all()) for k in ('r', 'z1', 'dz', 'dw'))
    f.update(dz1=f['dz'].view(2, 9, cols), dr=f['g'].dx)                       # one block back


@pytest.mark.parametrize('cols', [5, 200, 520, 1000, 2048, 2050, 4096, 4100, 8192])
@pytest.mark.parametrize('dt,res', [('f32', 'f32'), ('bf16', 'f32'), ('f16', 'f16')])
def test_norm_before_the_first_block_at_every_width(blocks, cols, dt, res):
  """z = N_pre(x) alone, with weight and bias, and its gradients."""
  t, p, kw, _ = T.norm_case(cols, (2, 5), cols, dt, res, 'none', 'layer', 'none', 'none', 1.0)
  norm = blocks.ResidualNorm(cols, post='none', pre='layer', w_pre=p['w_pre'].cuda(), b_pre=p['b_pre'].cuda())
  z = torch.empty(2, 5, cols, dtype=T.DT[dt], device='cuda')
  r, z, stats = norm.forward(None, t['x'].cuda(), z=z, save=True)
  w = T.f64({**t, **p})
  want = O.residual_norm(None, w['x'], pre='layer', w_pre=w['w_pre'], b_pre=w['b_pre'])
  m1, s1 = (want['stats'].reshape(2, 5, 4)[..., i:i + 1] for i in (2, 3))
  rb = w['x'].abs().amax(-1, keepdim=True)
  T.off(z, want['z'], ((rb + m1.abs()) * s1 * w['w_pre'].abs() + w['b_pre'].abs()) * (1 + rb * s1), 256, 'z')
  g = norm.backward(t['dz'].cuda(), t['dr'].cuda(), None, r, stats)
  ref, size = O.residual_norm_backward(w['dz'], w['dr'], None, w['x'], stats.cpu().double(), pre='layer', w_pre=w['w_pre'], b_pre=w['b_pre'])
  T.off(g.dx, ref['dx'], size['dx'], 256, 'dx')
  for name in ('dw_pre', 'db_pre'):
    T.off(getattr(g, name), ref[name], size[name], 10 + 416, name)
