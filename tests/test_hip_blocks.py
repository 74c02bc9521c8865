"""GPU tests of advoc_amd.blocks against oracle/blocks_torch.py in float64.

Tolerances, from the arithmetic alone.  u = 2^-24 is half a step of fp32; half a step of an output type is eps / 2 of the value.
  * a row's sum is at most 16 terms in a lane, 6 exchanges and 8 waves: 30 roundings; two sums per norm, two norms, and under 100
    roundings of single operations around them (the sigmoid's exponential counts 4): a row output is within 256 u of the largest
    term of its row, before its own rounding;
  * a column sum adds a worker's rows, the workers of a workgroup (at most 32), a sixteenth of the workgroups (at most 32) and these
    16 in turn, under 160 roundings: within (rows / workers + 160 + 256) u of the sum of the terms' magnitudes -- rows are few here,
    so `rows` itself is taken;
  * an 8-bit product passes at most 128 additions inside an instruction, one per block of 128, and 16 + 64 where waves or splits
    meet: within (208 + k / 128) u of sum |a b|.  For 16-bit outputs the instruction also drops, of each of eight neighbouring
    products, what is below 2^-13 of the largest of them: under 8 2^-13 of that one, so 2^-10 of sum |a b| in all;
  * dropout multiplies once in fp32 and rounds once: the bits of the same two steps on the CPU.
"""
import pytest
import torch

from oracle import blocks_torch as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


@pytest.fixture(scope='module')
def blocks():
  from advoc_amd import _lib, blocks
  assert torch.cuda.is_available(), 'gpu-marked test running without a HIP device'
  _lib.load()
  return blocks


def gen(seed):
  return torch.Generator().manual_seed(seed)


def off(got, want, big, ulps, what=''):
  """|got - want| <= half a step of got's type + ulps u big, everywhere; beyond the type's range (fp16 ends at 65504) the rounded
  value is an infinity, which got has to be then."""
  w = want.double()
  over = torch.isinf(want.to(got.dtype))
  assert torch.equal(got.cpu()[over], want.to(got.dtype)[over]), what
  got, w, big = got.cpu().masked_fill(over, 0), w.masked_fill(over, 0), big.masked_fill(over, 0)
  err = (got.cpu().double() - w).abs()
  tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps      # the step between subnormals
  tol = w.abs() * (torch.finfo(got.dtype).eps / 2) + ulps * U * big.double() * 1.01 + tiny
  assert got.shape == want.shape, (what, got.shape, want.shape)
  assert bool((err <= tol).all()), '%s: %g of the tolerance' % (what, (err / tol).max().item())


# ---- dropout ----
def dropped(x, seed, offset, keep):
  m = O.keep_mask(x.shape, seed, offset, keep)
  scale = torch.tensor(1.0 / float(torch.tensor(keep, dtype=torch.float32)), dtype=torch.float32)
  return torch.where(m, x.float() * scale, torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('rows,cols,pad', [(1, 1, 0), (3, 5, 0), (3, 5, 2), (1, 513, 0), (40, 513, 15), (257, 8, 8), (5, 1030, 1), (2049, 3, 1),
                                           (64, 2048, 0), (7, 9001, 7)])
def test_dropout_values(blocks, dt, rows, cols, pad):
  x = torch.randn(rows, cols + pad, generator=gen(rows + cols)).to(DT[dt])
  seed, offset, keep = 2 ** 63 + 12345, 4 * 1000003, 0.7
  d = x.cuda()[:, :cols]
  want = dropped(x[:, :cols].contiguous(), seed, offset, keep)
  assert torch.equal(blocks.dropout(d, keep, seed, offset).cpu(), want)
  out = torch.full((rows, cols + 3), 7.0, dtype=DT[dt], device='cuda')      # a pitch of its own, and padding that stays
  got = blocks.dropout(d, keep, seed, offset, out=out[:, :cols])
  assert torch.equal(got.cpu(), want) and bool((out[:, cols:] == 7).all())
  full = x.cuda()
  blocks.dropout(full[:, :cols], keep, seed, offset, out=full[:, :cols])      # in place
  assert torch.equal(full[:, :cols].cpu(), want) and torch.equal(full[:, cols:].cpu(), x[:, cols:])


@pytest.mark.parametrize('keep', [1e-6, 0.1, 0.5, 0.9, 1.0 - 2.0 ** -24, 1.0])
def test_dropout_draws_the_stored_masks_stream(blocks, keep):
  """The elements kept are those of advoc_dropout_mask_u8 at the same (seed, offset)."""
  from advoc_amd import _lib
  n, seed, offset = 100003, 77, 2 ** 34
  mask = torch.empty(n, dtype=torch.uint8, device='cuda')
  _lib.check(_lib.load().advoc_dropout_mask_u8(_lib.ptr(mask), n, seed, offset, keep, _lib.stream()))
  got = blocks.dropout(torch.ones(n, device='cuda'), keep, seed, offset)
  assert torch.equal(got != 0, mask != 0)


def test_dropout_of_a_shard_is_the_whole_batchs(blocks):
  x = torch.randn(8, 16, 513, generator=gen(0)).cuda()
  whole = blocks.dropout(x, 0.5, 5)
  half = blocks.dropout(x[4:], 0.5, 5, offset=4 * 16 * 513)
  assert torch.equal(whole[4:], half)


def test_dropped_elements_are_zero_whatever_they_held(blocks):
  for bad in (float('inf'), float('nan'), -float('inf')):
    x = torch.full((4096,), bad, device='cuda')
    m = O.keep_mask((4096,), 3, 0, 0.5).cuda()
    y = blocks.dropout(x, 0.5, 3)
    assert bool((y[~m] == 0).all()) and not bool(torch.isfinite(y[m]).any())


def test_dropout_past_32_bits(blocks):
  n, tail = 2 ** 32 + 4096, 5000
  x = torch.ones(n, dtype=torch.bfloat16, device='cuda')
  blocks.dropout(x, 0.5, 9, out=x)
  want = dropped(torch.ones(tail, dtype=torch.bfloat16), 9, n - tail - (n - tail) % 4, 0.5)
  assert torch.equal(x[n - tail - (n - tail) % 4:][:tail].cpu(), want)


def test_dropout_seed_word_and_empty(blocks):
  x = torch.ones(1000, device='cuda')
  word = torch.tensor([41], dtype=torch.int64, device='cuda')
  assert torch.equal(blocks.dropout(x, 0.5, 1, seed_dev=word), blocks.dropout(x, 0.5, 42))
  assert blocks.dropout(x[:0], 0.5, 1).numel() == 0
  assert blocks.dropout(torch.ones(0, 5, device='cuda'), 0.5, 1).shape == (0, 5)


# ---- residual norm ----
def norm_case(seed, lead, cols, dt, res, post, pre, gate, act, keep):
  g = gen(seed)
  r = lambda *s: torch.randn(*s, generator=g)      # noqa: E731
  t = dict(h=(r(*lead, cols) * torch.exp(0.5 * r(*lead, 1)) + 0.5).to(DT[dt]), x=r(*lead, cols).to(DT[res]), gate=None)
  if gate == 'row':
    t['gate'] = r(*lead, cols).to(DT[dt])
  elif gate == 'clip':
    t['gate'] = r(lead[0], 1, cols).to(DT[dt])
  p = dict(w_post=r(cols) if post != 'none' else None, b_post=r(cols) if post != 'none' else None, scale=r(cols),
           w_pre=r(cols) if pre != 'none' else None, b_pre=r(cols) if pre != 'none' else None)
  kw = dict(post=post, pre=pre, alpha=0.7, eps=1e-5)
  t['dz'] = None if pre == 'none' else r(*lead, cols).to(DT[dt])
  t['dr'] = r(*lead, cols).to(DT[res])
  return t, p, kw, dict(act=act, keep=keep, mask=O.keep_mask(t['h'].shape, 11 + seed, 8, keep) if keep < 1 else None)


def up(d):
  return {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}


def f64(d):
  return {k: v.double() if torch.is_tensor(v) and v.dtype != torch.bool else v for k, v in d.items()}


def check_norm(blocks, seed, lead, cols, dt, res, post, pre, gate, act, keep):
  t, p, kw, dk = norm_case(seed, lead, cols, dt, res, post, pre, gate, act, keep)
  norm = blocks.ResidualNorm(cols, gate_act=act, keep_prob=keep, **up(p), **kw)
  d = up(t)
  call = dict(gate=d['gate'], seed=11 + seed, offset=8)
  r, z, stats = norm.forward(d['h'], d['x'], save=True, **call)
  w = f64({**t, **p})
  want = O.residual_norm(w['h'], w['x'], w['gate'], **{k: w[k] for k in p}, **kw, **dk)
  # sizes: a normed value is a difference from the mean over the spread
  m0, s0, m1, s1 = (want['stats'].reshape(tuple(lead) + (4,))[..., i:i + 1] for i in range(4))
  ub = w['h'].abs() if post == 'none' else (w['h'].abs() + m0.abs()) * s0 * w['w_post'].abs() + w['b_post'].abs()
  gt = 1.0 if w['gate'] is None else O.gate_act(w['gate'], act).abs()
  rb = (w['x'].abs() + 0.7 * w['scale'].abs() * gt * ub / keep).amax(-1, keepdim=True)
  off(r, want['r'], rb.expand_as(want['r']), 256, 'r')
  if pre == 'none':
    assert z is None
  else:
    zb = (rb + m1.abs()) * s1 * w['w_pre'].abs() + w['b_pre'].abs()
    # the spread's own error: relative to the spread, the row's errors relative to it
    off(z, want['z'], zb * (1 + rb * s1), 256, 'z')
  sb = torch.cat([w['h'].abs().amax(-1, keepdim=True), s0 * (1 + s0 * w['h'].abs().amax(-1, keepdim=True)), rb, s1 * (1 + s1 * rb)],
                 -1).reshape(-1, 4)
  off(stats, want['stats'], sb, 256, 'stats')
  # the backward pass is the gradient at the r and statistics it is given
  got = norm.backward(d['dz'], d['dr'], d['h'], r, stats, **call)
  wr, ws = r.cpu().double(), stats.cpu().double()
  g, size = O.residual_norm_backward(w['dz'], w['dr'], w['h'], wr, ws, w['gate'], post, pre, alpha=0.7, **{k: w[k] for k in p}, **dk)
  rows = t['h'].numel() // cols
  for name, val in got._asdict().items():
    if val is None:
      assert name not in g or name[1:] in p and p[name[1:]] is None, name
      continue
    ulps = 256 if name in ('dh', 'dx') else rows + 416
    off(val, g[name], size[name], ulps, name)
  return norm, d, call, got, (r, z, stats)


KINDS = [('rms', 'rms', 'none', 'none', 1.0), ('layer', 'rms', 'clip', 'none', 0.9), ('rms', 'layer', 'row', 'sigmoid', 0.5),
         ('none', 'layer', 'clip', 'sigmoid', 0.9), ('layer', 'none', 'row', 'none', 1.0), ('none', 'none', 'row', 'sigmoid', 0.5)]
TYPES = [('f32', 'f32'), ('bf16', 'bf16'), ('bf16', 'f32'), ('f16', 'f16'), ('f16', 'f32')]


@pytest.mark.parametrize('dt,res', TYPES)
@pytest.mark.parametrize('kind', range(len(KINDS)))
def test_norm_types_and_options(blocks, dt, res, kind):
  check_norm(blocks, kind, (3, 37), 200, dt, res, *KINDS[kind])


@pytest.mark.parametrize('cols', [1, 2, 7, 8, 9, 16, 80, 127, 128, 129, 256, 257, 512, 513, 514, 575, 576, 577, 1000, 1024, 1025, 2048, 2049, 4096, 4099, 8191, 8192])
def test_norm_widths(blocks, cols):
  """Every instance of the kernels, at its edges, whole chunks and ragged ones."""
  check_norm(blocks, cols, (2, 5), cols, 'bf16', 'f32', *KINDS[1 + cols % 2])


@pytest.mark.parametrize('lead', [(1, 1), (1, 2), (1, 700), (700, 1), (129, 3), (5, 257), (2, 2500)])
def test_norm_rows_and_clips(blocks, lead):
  """One row, many rows to a worker, many clips to a worker, workers that share a clip."""
  check_norm(blocks, 1, lead, 72, 'f16', 'f32', *KINDS[1])


@pytest.mark.parametrize('lead,cols', [((13000, 2), 16), ((2500, 2), 1000), ((900, 3), 1100), ((300, 2), 2500), ((300, 2), 4100)])
def test_norm_more_clips_than_workers(blocks, lead, cols):
  """A worker that passes through several gate rows carries the sums of those before, at every width that holds rows its own way."""
  check_norm(blocks, 3, lead, cols, 'bf16', 'bf16', *KINDS[1])


@pytest.mark.parametrize('kind', [1, 3])
@pytest.mark.parametrize('lead,cols', [((3, 64), 7), ((3, 64), 100), ((3, 64), 200), ((3, 64), 300), ((3, 64), 520), ((3, 64), 1000), ((64, 40), 1000),
                                       ((3, 65), 520)])
def test_norm_clips_cut_into_whole_workgroups(blocks, lead, cols, kind):
  """A gate row's gradient that meets in a workgroup before it leaves, and (65 frames) one that cannot."""
  check_norm(blocks, 4, lead, cols, 'bf16', 'f32', *KINDS[kind])


def test_norm_many_rows(blocks):
  check_norm(blocks, 2, (3, 5001), 16, 'bf16', 'bf16', *KINDS[3])


def test_norm_past_32_bits(blocks):
  """Elements past 2^32: the last rows of a call are those of a call of these rows at their offset, both ways."""
  rows, cols, tail = 2 ** 20 + 5, 4200, 3
  h, x = (torch.empty(rows, cols, dtype=torch.bfloat16, device='cuda').normal_() for _ in range(2))
  vec = [torch.rand(cols, generator=gen(i)).cuda() for i in range(3)]
  norm = blocks.ResidualNorm(cols, post='rms', pre='layer', w_post=vec[0], scale=vec[1], w_pre=vec[2], keep_prob=0.9)
  r, z, stats = norm.forward(h, x, seed=3, save=True)
  last = dict(seed=3, offset=(rows - tail) * cols)
  r2, z2, stats2 = norm.forward(h[-tail:], x[-tail:], save=True, **last)
  assert torch.equal(r[-tail:], r2) and torch.equal(z[-tail:], z2) and torch.equal(stats[-tail:], stats2)
  g = norm.backward(z, x, h, r, stats, seed=3)
  g2 = norm.backward(z2, x[-tail:], h[-tail:], r2, stats2, **last)
  assert torch.equal(g.dh[-tail:], g2.dh) and torch.equal(g.dx[-tail:], g2.dx)


def test_norm_repeats_bit_for_bit_and_takes_buffers(blocks):
  norm, d, call, g, (r, z, stats) = check_norm(blocks, 5, (4, 300), 513, 'bf16', 'f32', *KINDS[1])
  again = norm.backward(d['dz'], d['dr'], d['h'], r, stats, **call)
  for a, b in zip(g, again):
    assert torch.equal(a, b)
  # parameter gradients into the slices of an arena, written and then added to
  arena = torch.full((5, 513), float('nan'), device='cuda')
  into = {k: arena[i] for i, k in enumerate(('dw_post', 'db_post', 'dscale', 'dw_pre', 'db_pre'))}
  norm.backward(d['dz'], d['dr'], d['h'], r, stats, into=into, **call)
  for k, v in into.items():
    assert torch.equal(v, getattr(g, k)), k
  norm.backward(d['dz'], d['dr'], d['h'], r, stats, into=into, accumulate=True, **call)
  for k, v in into.items():
    assert torch.equal(v, 2 * getattr(g, k)), k
  # r over x, z into a padded buffer, inputs with a pitch
  wide = torch.full((4, 300, 520), 3.0, dtype=torch.bfloat16, device='cuda')
  hp = torch.zeros(4, 300, 530, dtype=torch.bfloat16, device='cuda')
  hp[..., :513] = d['h']
  x = d['x'].clone()
  r2, z2, _ = norm.forward(hp[..., :513], x, r=x, z=wide[..., :513], **call)
  assert r2 is x and torch.equal(x, r) and torch.equal(z2, z) and bool((wide[..., 513:] == 3).all())


def descriptor(norm, r, gate, call):
  """The C entries' struct for float32 rows, with everything but the tensors that a test binds itself."""
  from advoc_amd import _lib
  rows, ptr = r.numel() // norm.cols, lambda t: None if t is None else t.data_ptr()      # noqa: E731
  q = _lib.ResidualNorm(rows, norm.cols, 0, 0, norm.post, norm.pre, norm.gate_act, 1 if gate is None else rows // (gate.numel() // norm.cols),
                        ptr(norm.w_post), ptr(norm.b_post), ptr(norm.scale), ptr(norm.w_pre), ptr(norm.b_pre), norm.alpha, norm.eps,
                        norm.keep_prob, 0, call['seed'], call['offset'])
  for name, t in (('r', r), ('gate', gate)):
    getattr(q, name).p, getattr(q, name).pitch = ptr(t), norm.cols
  return q


@pytest.mark.parametrize('cols', [40, 513, 2500])
def test_norm_backward_in_place(blocks, cols):
  """dx over dr and dh over h through the C entry, ragged rows included."""
  import ctypes
  from advoc_amd import _lib
  norm, d, call, g, (r, z, stats) = check_norm(blocks, 6, (2, 9), cols, 'f32', 'f32', *KINDS[0])
  q = descriptor(norm, r, None, call)
  h, dr = d['h'].clone(), d['dr'].clone()
  for name, t in (('dz', d['dz']), ('dr', dr), ('dx', dr), ('h', h), ('dh', h)):
    getattr(q, name).p, getattr(q, name).pitch = t.data_ptr(), cols
  q.stats = stats.data_ptr()
  assert _lib.load().advoc_residual_norm_workspace_bytes(ctypes.byref(q)) == 0
  _lib.check(_lib.load().advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  assert torch.equal(dr, g.dx) and torch.equal(h, g.dh)


@pytest.mark.parametrize('lead,cols', [((600, 2), 1032), ((300, 3), 2056), ((9, 40), 1544), ((2200, 1), 700), ((3, 70), 80), ((3, 64), 1000)])
def test_norm_every_output_over_an_input(blocks, lead, cols):
  """dx over dr, dh over h and dgate over a gate per clip: whole clips to a worker and clips cut up, waves that hold the same columns."""
  import ctypes
  from advoc_amd import _lib
  norm, d, call, g, (r, z, stats) = check_norm(blocks, 8, lead, cols, 'f32', 'f32', 'rms', 'layer', 'clip', 'sigmoid', 0.9)
  h, dr, gate = d['h'].clone(), d['dr'].clone(), d['gate'].clone()
  q = descriptor(norm, r, gate, call)
  for name, t in (('dz', d['dz']), ('dr', dr), ('dx', dr), ('h', h), ('dh', h), ('dgate', gate)):
    getattr(q, name).p, getattr(q, name).pitch = t.data_ptr(), cols
  sums = {k: torch.full((cols,), float('nan'), device='cuda') for k in ('dw_post', 'db_post', 'dscale', 'dw_pre', 'db_pre')}
  for k, t in sums.items():
    setattr(q, k, t.data_ptr())
  q.stats = stats.data_ptr()
  n = _lib.load().advoc_residual_norm_workspace_bytes(ctypes.byref(q))
  work = torch.empty(n // 4, device='cuda')
  q.workspace, q.workspace_bytes = work.data_ptr(), n
  _lib.check(_lib.load().advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  assert torch.equal(dr, g.dx) and torch.equal(h, g.dh) and torch.equal(gate, g.dgate)
  for k, t in sums.items():
    assert torch.equal(t, getattr(g, k)), k


def test_norm_before_the_first_block(blocks):
  g = gen(3)
  x, w, dz, dr = (torch.randn(*s, generator=g) for s in ((6, 80), (80,), (6, 80), (6, 80)))
  norm = blocks.ResidualNorm(80, pre='layer', w_pre=w.cuda())
  r, z, stats = norm.forward(None, x.cuda(), save=True)
  want = O.residual_norm(None, x.double(), pre='layer', w_pre=w.double())
  off(z, want['z'], 20 * torch.ones_like(want['z']), 256)
  got = norm.backward(dz.cuda(), None, None, r, stats)
  ref, size = O.residual_norm_backward(dz.double(), None, None, x.double(), stats.cpu().double(), pre='layer', w_pre=w.double())
  off(got.dx, ref['dx'], size['dx'], 256)
  off(got.dw_pre, ref['dw_pre'], size['dw_pre'], 422)
  assert got.dh is None and got.dscale is None and got.dw_post is None


def test_norm_of_zeros_constants_and_bad_rows(blocks):
  """A row of zeros gives the bias, a constant row has no spread, and a NaN or infinity stays in its row."""
  for kind in ('rms', 'layer'):
    norm = blocks.ResidualNorm(96, post=kind, pre=kind, b_pre=torch.full((96,), 2.0, device='cuda'))
    h = torch.zeros(6, 96, device='cuda')
    x = torch.randn(6, 96, generator=gen(1)).cuda()
    clean = norm.forward(h, x, save=True)
    z = norm.forward(h, torch.zeros_like(x))[1]
    assert bool((z == 2).all())
    x2, h2 = x.clone(), h.clone()
    x2[1, 5], h2[3, 90], h2[4, 0] = float('inf'), float('nan'), -float('inf')
    r, z, stats = norm.forward(h2, x2, save=True)
    for i in (0, 2, 5):
      assert torch.equal(z[i], clean[1][i]) and torch.equal(r[i], clean[0][i])
    assert not torch.isfinite(z[1]).all() and torch.isnan(z[3]).all()
    ones = torch.ones_like(x)
    g = norm.backward(ones, ones, h2, r, stats)
    c = norm.backward(ones, ones, h, clean[0], clean[2])
    for i in (0, 2, 5):
      assert torch.equal(g.dx[i], c.dx[i]) and torch.equal(g.dh[i], c.dh[i])
  z = blocks.ResidualNorm(96, pre='layer').forward(None, torch.full((2, 96), 1e4, device='cuda'))[1]
  assert bool((z == 0).all())


def test_norm_of_kind_none_takes_no_weight_or_bias(blocks):
  """What a C caller leaves in a descriptor's w_post, b_post (w_pre, b_pre) is ignored without the norm they belong to."""
  import ctypes
  from advoc_amd import _lib
  norm, d, call, g, (r, z, stats) = check_norm(blocks, 9, (2, 7), 72, 'f32', 'f32', 'none', 'none', 'row', 'none', 0.9)
  q = descriptor(norm, r, d['gate'], call)
  q.x.p, q.x.pitch = d['x'].data_ptr(), 72
  wrong = torch.full((72,), 7.0, device='cuda')
  q.w_post = q.b_post = q.w_pre = q.b_pre = wrong.data_ptr()
  out = {k: torch.empty_like(r) for k in ('r', 'dh', 'dx', 'dgate')}
  for name, t in (('h', d['h']), ('r', out['r']), ('dr', d['dr']), ('dh', out['dh']), ('dx', out['dx']), ('dgate', out['dgate'])):
    getattr(q, name).p, getattr(q, name).pitch = t.data_ptr(), 72
  _lib.check(_lib.load().advoc_residual_norm_forward(ctypes.byref(q), _lib.stream()))
  _lib.check(_lib.load().advoc_residual_norm_backward(ctypes.byref(q), _lib.stream()))
  assert torch.equal(out['r'], r)
  for k in ('dh', 'dx', 'dgate'):
    assert torch.equal(out[k], getattr(g, k)), k


def test_norm_sigmoid_of_extreme_gates(blocks):
  """Shut at minus infinity, open at infinity, a NaN passed on; in between within 6 units in the last place."""
  norm = blocks.ResidualNorm(512, post='none', pre='none', gate_act='sigmoid', scale=torch.ones(512, device='cuda'))
  inf = float('inf')
  edge = torch.tensor([-inf, inf, -1e30, 1e30, -89.0, 89.0, 0.0, -0.0], device='cuda')
  gate = torch.cat([edge, torch.linspace(-87, 87, 504, device='cuda')]).reshape(1, 512)
  h, x = torch.ones(1, 512, device='cuda'), torch.zeros(1, 512, device='cuda')
  r = norm.forward(h, x, gate=gate)[0].cpu().double().flatten()
  assert r[:8].tolist() == [0, 1, 0, 1, 0, 1, 0.5, 0.5]
  want = torch.sigmoid(gate.cpu().double().flatten())[8:]
  assert bool(((r[8:] - want).abs() <= 12 * U * want).all())
  gate[0, 100] = float('nan')
  r = norm.forward(h, x, gate=gate)[0]
  assert bool(torch.isnan(r[0, 100])) and int(torch.isnan(r).sum()) == 1
  st = torch.zeros(1, 4, device='cuda')
  g = norm.backward(None, torch.ones_like(x), h, r, st, gate=gate)
  assert bool((g.dgate[0, :6] == 0).all()) and bool((g.dgate[0, 6:8] == 0.25).all()) and int(torch.isnan(g.dgate).sum()) == 1


def test_norm_empty(blocks):
  norm = blocks.ResidualNorm(16, w_pre=torch.ones(16, device='cuda'))
  e = torch.zeros(0, 16, device='cuda')
  r, z, stats = norm.forward(e, e, save=True)
  g = norm.backward(z, r, e, r, stats)
  assert z.shape == (0, 16) and g.dh.shape == (0, 16) and bool((g.dw_pre == 0).all())


def test_norm_refuses(blocks):
  from advoc_amd._lib import AdvocHipError
  norm = blocks.ResidualNorm(16, w_pre=torch.ones(16, device='cuda'))
  x = torch.zeros(2, 4, 16, device='cuda')
  bad = [lambda: norm.forward(x, x[:1]), lambda: norm.forward(x[..., :8], x), lambda: norm.forward(x.double(), x),
         lambda: norm.forward(x.bfloat16(), x.half()), lambda: norm.forward(x, x.bfloat16()), lambda: norm.forward(x, x, gate=x[0]),
         lambda: norm.forward(x, x, gate=x[:1]), lambda: norm.forward(x, x, gate=x.bfloat16()), lambda: norm.forward(x, x.cpu()),
         lambda: norm.forward(x.transpose(0, 1), x), lambda: norm.forward(x[..., ::2], x[..., :8]), lambda: norm.forward(None, x, gate=x),
         lambda: norm.forward(x, x[:1, :1].expand(2, 4, 16)), lambda: norm.forward(x, x, seed_dev=x), lambda: norm.forward(x, x, offset=2),
         lambda: norm.backward(None, x, x, x, None), lambda: norm.backward(x, x, x, x, None),
         lambda: norm.backward(x, x, x, x, torch.zeros(7, 4, device='cuda')), lambda: norm.backward(x.half(), x, x, x, torch.zeros(8, 4, device='cuda')),
         lambda: norm.backward(x, x, x, x, torch.zeros(8, 4, device='cuda'), into={'dw': x}),
         lambda: norm.backward(x, x, x, x, torch.zeros(8, 4, device='cuda'), into={'dscale': x}),
         lambda: norm.backward(x, x, x, x, torch.zeros(8, 4, device='cuda'), accumulate=True),
         lambda: blocks.ResidualNorm(16, w_pre=torch.ones(16)).forward(x, x),
         lambda: blocks.ResidualNorm(16, w_pre=torch.ones(8, device='cuda')).forward(x, x)]
  for i, call in enumerate(bad):
    with pytest.raises(AdvocHipError):
      call()
      pytest.fail('case %d was taken' % i)


# ---- 8-bit operands ----
F8T = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}


def values(q, fmt):
  """What an F8Matrix stands for, float64 [rows, k], after checking its padding."""
  d, s = q.data.cpu(), q.scale.cpu()
  kb = d.shape[1] // 128
  assert bool((d[:, q.k:] == 0).all()) and bool((s[:, kb:] == 0).all())
  scale = torch.exp2(s[:, :kb].double() - 127).repeat_interleave(128, 1)
  return (d.view(F8T[fmt]).float().double() * scale)[:, :q.k], s[:, :kb]


def same(a, b):
  return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('rows,cols,pad', [(1, 1, 0), (1, 1000, 0), (3, 128, 0), (130, 129, 3), (257, 513, 15), (128, 640, 0), (65, 100, 0)])
def test_quantize_is_exact(blocks, fmt, dt, rows, cols, pad):
  x = (torch.randn(rows, cols + pad, generator=gen(cols)) * torch.exp(3 * torch.randn(rows, 1, generator=gen(rows)))).to(DT[dt])
  x[0, 0] = 0
  d, x = x.cuda()[:, :cols], x[:, :cols].double()
  a, t = blocks.quantize_f8_both(d, fmt)
  for q, ref in ((a, x), (blocks.quantize_f8(d, fmt), x), (t, x.t()), (blocks.quantize_f8_transposed(d, fmt), x.t())):
    want, e = O.f8_blocks(ref, fmt)
    got, s = values(q, fmt)
    assert torch.equal(s, e) and torch.equal(got, want)


def test_quantize_past_32_bits(blocks):
  rows, cols, start = 2 ** 20 + 130, 4220, 2 ** 20
  x = torch.empty(rows, cols, dtype=torch.bfloat16, device='cuda').normal_()
  a, t = blocks.quantize_f8_both(x)
  b, u = blocks.quantize_f8_both(x[start:])
  assert torch.equal(a.data[start:], b.data) and torch.equal(a.scale[start:], b.scale)
  assert torch.equal(t.data[:, start:], u.data) and torch.equal(t.scale[:, start // 128:start // 128 + 2], u.scale[:, :2])
  only = blocks.quantize_f8(x)
  assert torch.equal(only.data[start:], b.data) and torch.equal(only.scale[start:], b.scale)


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
def test_quantize_extremes(blocks, fmt):
  """Blocks of zeros, the smallest and largest numbers, and infinities and NaN, which leave their block's scale alone."""
  x = torch.randn(8, 256, generator=gen(4))
  x[0] = 0
  x[1] *= 1e-42
  x[2] *= 3e37
  x[3, :128] = torch.finfo(torch.float32).max
  x[4, 7], x[4, 200], x[5, 0] = float('inf'), float('nan'), -float('inf')
  x[6] = float('nan')
  x[7] = O.F8[fmt][2]
  want, e = O.f8_blocks(x.double(), fmt)
  for q in (blocks.quantize_f8(x.cuda(), fmt), blocks.quantize_f8_transposed(x.t().contiguous().cuda(), fmt)):
    got, s = values(q, fmt)
    assert torch.equal(s, e) and same(got, want)


def product_ulps(out, k):
  return 208 + k / 128 + (0 if out.dtype == torch.float32 else 2 ** 14)


def ints(rows, k, seed):
  """Small whole numbers, some blocks scaled by powers of two: exact in 8 bits, and their products exact in fp32."""
  g = gen(seed)
  x = torch.randint(-3, 4, (rows, k), generator=g).float()
  return x * torch.exp2(torch.randint(0, 3, (rows, -(-k // 128)), generator=g).float()).repeat_interleave(128, 1)[:, :k]


SHAPES = [(1, 1, 1), (1, 512, 8192), (1, 17, 100), (2, 1, 9000), (2, 513, 1025), (3, 50, 1300), (16, 16, 128), (17, 15, 129), (33, 513, 1000), (64, 10240, 100), (64, 100, 2000),
          (65, 64, 128), (65, 1, 300), (100, 70, 513), (128, 128, 256), (129, 130, 1000), (300, 257, 1100), (1285, 513, 1000), (700, 600, 640),
          (200, 300, 5000), (1100, 1200, 4096), (4100, 4099, 200), (70, 16000, 130), (1000, 1100, 12000)]


@pytest.mark.parametrize('m,n,k', SHAPES)
def test_product_of_whole_numbers_is_exact(blocks, m, n, k):
  """Every kernel form, split and ragged edge: |sum| < 2^24, so the fp32 result has to be the integer one.  Guard values around
  the output stay."""
  a, b = ints(m, k, m), ints(n, k, n + 1)
  want = (a.double().cuda() @ b.double().cuda().t())
  assert want.abs().max() < 2 ** 24
  qa, qb = blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda())
  guard = torch.full((m * n + 2048,), -5.0, device='cuda')
  out = guard[1024:1024 + m * n].view(m, n)
  assert blocks.matmul_nt_f8(qa, qb, out=out) is out
  assert torch.equal(out.double(), want)
  assert bool((guard[:1024] == -5).all()) and bool((guard[1024 + m * n:] == -5).all())
  blocks.matmul_nt_f8(qa, qb, out=out, accumulate=True)
  assert torch.equal(out.double(), 2 * want)
  for dt in (torch.bfloat16, torch.float16):
    assert torch.equal(blocks.matmul_nt_f8(qa, qb, out_dtype=dt), want.float().to(dt))


@pytest.mark.parametrize('fa,fb', [('e4m3', 'e4m3'), ('e5m2', 'e4m3'), ('e4m3', 'e5m2'), ('e5m2', 'e5m2')])
@pytest.mark.parametrize('m,n,k', [(1, 70, 8300), (2, 33, 1000), (3, 50, 1000), (50, 200, 4000), (90, 100, 300), (600, 700, 2000), (300, 200, 9000), (4200, 3900, 512)])
def test_product_values(blocks, fa, fb, m, n, k):
  g = gen(m)
  a = torch.randn(m, k, generator=g) * torch.exp(2 * torch.randn(m, 1, generator=g))
  b = torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
  qa, qb = blocks.quantize_f8(a.cuda(), fa), blocks.quantize_f8(b.cuda(), fb)
  va, vb = values(qa, fa)[0].cuda(), values(qb, fb)[0].cuda()
  want, big = (va @ vb.t()).cpu(), (va.abs() @ vb.abs().t()).cpu()
  for dt in DT.values():
    got = blocks.matmul_nt_f8(qa, qb, out_dtype=dt)
    off(got, want, big, product_ulps(got, k))
    assert torch.equal(got, blocks.matmul_nt_f8(qa, qb, out_dtype=dt))


def test_product_without_workspace_and_with(blocks):
  """A split contraction and, when the caller brings no scratch, the unsplit one: the same whole numbers."""
  from advoc_amd import _lib
  lib = _lib.load()
  m, n, k = 200, 300, 5000
  assert lib.advoc_matmul_nt_f8_workspace_bytes(m, n, k, 0) > 0
  a, b = ints(m, k, 0), ints(n, k, 1)
  qa, qb = blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda())
  out = torch.empty(m, n, device='cuda')
  _lib.check(lib.advoc_matmul_nt_f8(qa.data_ptr, qa.scale_ptr, 0, qb.data_ptr, qb.scale_ptr, 0, _lib.ptr(out), 0, 0, m, n,
                                    k, None, 0, _lib.stream()))
  assert torch.equal(out, blocks.matmul_nt_f8(qa, qb)) and torch.equal(out.cpu().double(), a.double() @ b.double().t())


def test_product_carries_bad_values_in_their_rows(blocks):
  a, b = ints(70, 300, 0), ints(80, 300, 1)
  clean = blocks.matmul_nt_f8(blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda()))
  a[3, 5], b[7, 299] = float('nan'), float('inf')
  got = blocks.matmul_nt_f8(blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda()))
  bad = torch.zeros(70, 80, dtype=torch.bool, device='cuda')
  bad[3], bad[:, 7] = True, True
  assert not torch.isfinite(got[bad]).any() and torch.equal(got[~bad], clean[~bad])


def test_product_output_past_32_bits(blocks):
  m, n, k = 70000, 32768, 128
  a, b = ints(m, k, 0), ints(n, k, 1)
  out = blocks.matmul_nt_f8(blocks.quantize_f8(a.cuda()), blocks.quantize_f8(b.cuda()), out_dtype=torch.bfloat16)
  for rows in (slice(0, 64), slice(m - 64, m)):
    assert torch.equal(out[rows].cpu(), (a[rows].double() @ b.double().t()).float().bfloat16())


def test_f8_refuses(blocks):
  from advoc_amd._lib import AdvocHipError
  x = torch.zeros(4, 8, device='cuda')
  q = blocks.quantize_f8(x)
  bad = [lambda: blocks.quantize_f8(x, 'e3m4'), lambda: blocks.quantize_f8(x.double()), lambda: blocks.quantize_f8(x[:0]),
         lambda: blocks.quantize_f8(x.t()), lambda: blocks.matmul_nt_f8(q, blocks.quantize_f8(x[:, :7])), lambda: blocks.matmul_nt_f8(q, x),
         lambda: blocks.matmul_nt_f8(q, q, out_dtype=torch.float64), lambda: blocks.matmul_nt_f8(q, q, accumulate=True),
         lambda: blocks.matmul_nt_f8(q, q, out=torch.zeros(4, 5, device='cuda')),
         lambda: blocks.matmul_nt_f8(q, q, out=torch.zeros(4, 4, device='cuda', dtype=torch.bfloat16), accumulate=True),
         lambda: blocks.dropout(x, 0.5, 1, offset=2), lambda: blocks.dropout(x, 0.0, 1), lambda: blocks.dropout(x.double(), 0.5, 1),
         lambda: blocks.dropout(x, 0.5, 1, out=x.half()), lambda: blocks.dropout(x.t(), 0.5, 1), lambda: blocks.dropout(x, 0.5, 1, seed_dev=x)]
  for i, call in enumerate(bad):
    with pytest.raises(AdvocHipError):
      call()
      pytest.fail('case %d was taken' % i)


# ---- together ----
class Block(object):
  """z -> y = W z in 8 bits -> r = x + alpha scale gate dropout(N(y)), z' = N(r); and back."""

  def __init__(self, blocks, cols, seed):
    g = gen(seed)
    self.b, r = blocks, lambda *s: torch.randn(*s, generator=g).cuda()
    self.w = r(cols, cols) * cols ** -0.5
    self.w8, self.w8t = blocks.quantize_f8(self.w), blocks.quantize_f8_transposed(self.w)
    self.norm = blocks.ResidualNorm(cols, post='rms', pre='layer', gate_act='sigmoid', alpha=0.5, keep_prob=0.9, w_post=1 + 0.1 * r(cols),
                                    scale=r(cols), w_pre=1 + 0.1 * r(cols), b_pre=0.1 * r(cols))

  def step(self, x, z, gate, dz, dr, word=None):
    b = self.b
    z8, z8t = b.quantize_f8_both(z)
    y = b.matmul_nt_f8(z8, self.w8, out_dtype=z.dtype).view(z.shape)
    r, z1, stats = self.norm.forward(y, x, gate=gate, seed=21, seed_dev=word, save=True)
    g = self.norm.backward(dz, dr, y, r, stats, gate=gate, seed=21, seed_dev=word)
    dy8, dy8t = b.quantize_f8_both(g.dh, 'e5m2')
    dz0 = b.matmul_nt_f8(dy8, self.w8t, out_dtype=z.dtype).view(z.shape)
    dw = b.matmul_nt_f8(dy8t, z8t)
    return dict(y=y, r=r, z1=z1, stats=stats, dz0=dz0, dw=dw, **{k: v for k, v in g._asdict().items() if v is not None})


def block_inputs(clips, frames, cols, seed, dt=torch.bfloat16):
  g = gen(seed)
  r = lambda *s: torch.randn(*s, generator=g).cuda()      # noqa: E731
  return r(clips, frames, cols), r(clips, frames, cols).to(dt), r(clips, 1, cols).to(dt), r(clips, frames, cols).to(dt), r(clips, frames, cols)


@pytest.mark.parametrize('clips,frames,cols', [(1, 1, 512), (3, 100, 256), (2, 129, 513)])
def test_a_block_forward_and_backward(blocks, clips, frames, cols):
  """Each stage against float64 at what the stage before gave it."""
  blk = Block(blocks, cols, 0)
  x, z, gate, dz, dr = block_inputs(clips, frames, cols, 1)
  o = blk.step(x, z, gate, dz, dr)
  rows = clips * frames
  f = lambda t: t.cpu().double()      # noqa: E731
  vz, vw = O.f8_blocks(f(z).reshape(rows, cols), 'e4m3')[0], O.f8_blocks(f(blk.w), 'e4m3')[0]
  off(o['y'].reshape(rows, cols), vz @ vw.t(), vz.abs() @ vw.abs().t(), product_ulps(o['y'], cols), 'y')
  p = {k: f(getattr(blk.norm, k)) for k in ('w_post', 'scale', 'w_pre', 'b_pre')}
  mask = O.keep_mask((clips, frames, cols), 21, 0, 0.9)
  kw = dict(post='rms', pre='layer', act='sigmoid', alpha=0.5, keep=0.9, mask=mask, **p)
  want = O.residual_norm(f(o['y']), f(x), f(gate), **kw)
  for name in ('r', 'z1'):
    w = want[name[0]]
    off(o[name], w, 8 * w.abs().amax(-1, keepdim=True).expand_as(w) + 8, 256, name)
  g, size = O.residual_norm_backward(f(dz), f(dr), f(o['y']), f(o['r']), f(o['stats']), f(gate), **kw)
  for name in g:
    if name in o:
      off(o[name], g[name], size[name], 256 if name in ('dh', 'dx') else rows + 416, name)
  dy = f(o['dh']).reshape(rows, cols)
  vd, vwt = O.f8_blocks(dy, 'e5m2')[0], O.f8_blocks(f(blk.w).t().contiguous(), 'e4m3')[0]
  off(o['dz0'].reshape(rows, cols), vd @ vwt.t(), vd.abs() @ vwt.abs().t(), product_ulps(o['dz0'], cols), 'dz0')
  vdt, vzt = O.f8_blocks(dy.t().contiguous(), 'e5m2')[0], O.f8_blocks(f(z).reshape(rows, cols).t().contiguous(), 'e4m3')[0]
  off(o['dw'], vdt @ vzt.t(), vdt.abs() @ vzt.abs().t(), product_ulps(o['dw'], rows), 'dw')
  # and the gradient through the quantised products is near the one without them: 2^-3 of e5m2, 2^-4 of e4m3 per operand
  true = dy @ f(blk.w)
  assert (f(o['dz0']).reshape(rows, cols) - true).norm() < (2 ** -3 + 2 ** -4) * true.norm() * 1.1


def test_a_block_captured_replayed_and_on_another_stream(blocks):
  """One graph of the whole step, replayed between eager work, gives the eager bits; two graphs do not share scratch; a seed word
  that changes between replays changes the mask."""
  blk = Block(blocks, 256, 0)
  ins = [block_inputs(2, 70, 256, s) for s in (1, 2)]
  word = torch.zeros(1, dtype=torch.int64, device='cuda')
  eager = [blk.step(*i, word=word) for i in ins]
  side = torch.cuda.Stream()
  graphs, outs = [], []
  for i in ins:
    with torch.cuda.stream(side):
      blk.step(*i, word=word)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
      outs.append(blk.step(*i, word=word))
    graphs.append(gr)
  for turn in range(4):
    for gr in graphs:
      gr.replay()
    busy = blk.step(*ins[turn % 2], word=word)
    torch.cuda.synchronize()
    for e, o in zip(eager, outs):
      for k in e:
        assert torch.equal(e[k], o[k]), (turn, k)
    for k in busy:
      assert torch.equal(busy[k], eager[turn % 2][k]), k
  word.fill_(1)
  again = blk.step(*ins[0], word=word)
  graphs[0].replay()
  torch.cuda.synchronize()
  assert torch.equal(outs[0]['r'], again['r']) and not torch.equal(outs[0]['r'], eager[0]['r'])
  s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
  word.fill_(0)
  torch.cuda.synchronize()
  res = []
  for s, i in ((s1, ins[0]), (s2, ins[1])):      # two calls at once
    with torch.cuda.stream(s):
      res.append(blk.step(*i, word=word))
  torch.cuda.synchronize()
  for e, o in zip(eager, res):
    for k in e:
      assert torch.equal(e[k], o[k]), k
