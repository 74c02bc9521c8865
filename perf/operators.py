"""The residual-block operators as measured: counter-based dropout, the residual norm and the 8-bit block-scaled product.

Where `own` is false, run() computes them in their plain form with elementary torch operations in 32 bits; where it is true
it makes the calls a user makes of advoc_amd.blocks.  The shapes are those of spectrogram frames: a clip is 256 frames, a
batch 32 or 64 clips, a frame 513 bins or 512 ... 4096 channels; streaming inference sees one frame at a time.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
F8_TOP = {'e4m3': 9, 'e5m2': 16}          # the largest value of a format is 0.875 * 2^top
F8_TYPE = {'e4m3': torch.float8_e4m3fn, 'e5m2': torch.float8_e5m2}
EPS = 1e-5


def listed():
  return [
      # one frame of 513 bins: dropout that stays on in streaming inference, a launch's latency
      dict(name='dropout_frame', op='dropout', rows=1, cols=513, pad=0, dtype='f32', keep=0.5),
      # the gradient of 32 clips of 513 bins inside wider rows: odd width, padded pitch
      dict(name='dropout_bins', op='dropout', rows=8192, cols=513, pad=15, dtype='f16', keep=0.9),
      # the widest activation of a training step: 256 clips of 256 frames
      dict(name='dropout_clips', op='dropout', rows=65536, cols=1024, pad=0, dtype='bf16', keep=0.9),
      # one frame through the glue between two blocks in streaming inference
      dict(name='norm_frame', op='norm', way='fwd', clips=1, frames=1, cols=512, dtype='bf16', res='f32', post='rms', pre='rms',
           gates='clip', act='none', keep=1.0, save=False),
      # a training step's forward pass: 64 clips, a gate per clip, residual stream in fp32, the rows' statistics kept
      dict(name='norm_clips', op='norm', way='fwd', clips=64, frames=256, cols=1024, dtype='bf16', res='f32', post='layer',
           pre='rms', gates='clip', act='none', keep=0.9, save=True),
      # and its backward pass
      dict(name='norm_clips_grad', op='norm', way='bwd', clips=64, frames=256, cols=1024, dtype='bf16', res='f32', post='layer',
           pre='rms', gates='clip', act='none', keep=0.9),
      # frames of 513 bins in fp32, a gate per element through a sigmoid, odd numbers of clips and frames
      dict(name='norm_bins_grad', op='norm', way='bwd', clips=31, frames=129, cols=513, dtype='f32', res='f32', post='rms',
           pre='layer', gates='row', act='sigmoid', keep=0.5),
      # wide rows without a gate, everything in 16 bits
      dict(name='norm_wide_grad', op='norm', way='bwd', clips=16, frames=256, cols=4096, dtype='f16', res='f16', post='rms',
           pre='rms', gates='none', act='none', keep=1.0),
      # one position of a deep 4 x 4 x 512 -> 512 layer as a product: bound by reading the weights
      dict(name='product_frame', op='product', way='fwd', m=1, k=8192, n=512, dtype='bf16', fmt='e4m3'),
      # nothing a multiple of anything: 5 clips of 257 frames, 1000 channels to 513 bins, fp32 in and out
      dict(name='product_bins', op='product', way='fwd', m=1285, k=1000, n=513, dtype='f32', fmt='e4m3'),
      # 64 clips through a wide layer: bound by the matrix cores
      dict(name='product_clips', op='product', way='fwd', m=16384, k=4096, n=4096, dtype='bf16', fmt='e4m3'),
      # both gradients of 64 clips through a square layer, the output gradient in e5m2
      dict(name='product_clips_grad', op='product', way='bwd', m=16384, k=1024, n=1024, dtype='bf16', fmt='e5m2'),
  ]


def _log(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(['dropout', 'norm', 'norm', 'product', 'product'])
  dtype = rng.choice(['f32', 'bf16', 'f16'])
  if op == 'dropout':
    cols = _log(rng, 1, 4096)
    return dict(op=op, rows=_log(rng, 1, 65536 * 1024 // 2 // cols), cols=cols, pad=rng.choice([0, 0, 1, 8, 15]), dtype=dtype,
                keep=rng.choice([0.5, 0.9, 0.95]))
  if op == 'norm':
    cols = _log(rng, 8, 8192)
    rows = _log(rng, 1, 64 * 256 * 1024 // cols)
    clips = _log(rng, 1, min(64, rows))
    return dict(op=op, way=rng.choice(['fwd', 'bwd']), clips=clips, frames=max(1, rows // clips), cols=cols, dtype=dtype,
                res=rng.choice([dtype, 'f32']), post=rng.choice(['none', 'rms', 'layer']), pre=rng.choice(['none', 'rms', 'layer']),
                gates=rng.choice(['none', 'clip', 'row']), act=rng.choice(['none', 'sigmoid']), keep=rng.choice([0.5, 0.9, 1.0]),
                save=rng.choice([False, True]))
  return dict(op=op, way=rng.choice(['fwd', 'bwd']), m=_log(rng, 1, 16384), k=_log(rng, 16, 4096), n=_log(rng, 16, 4096),
              dtype=dtype, fmt=rng.choice(['e4m3', 'e5m2']))


# ---- inputs ----
def _inputs(case, seed):
  """The tensors of a case, from its seed alone."""
  dev = torch.device('cuda', torch.cuda.current_device())
  g = torch.Generator(device=dev).manual_seed(seed)

  def normal(*shape, std=1.0, mean=0.0, dtype='f32'):
    return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(DTYPES[dtype])

  dt = case['dtype']
  if case['op'] == 'dropout':
    x = normal(case['rows'], case['cols'] + case['pad'], dtype=dt)
    return dict(x=x[:, :case['cols']], seed=seed * 7919 + 1)
  if case['op'] == 'norm':
    b, t, c, res = case['clips'], case['frames'], case['cols'], case['res']
    d = dict(seed=seed * 7919 + 1)
    # channels of a frame differ in size by an order of magnitude, frames by their loudness
    size = torch.exp(normal(c)) * 0.5
    loud = torch.exp(0.5 * normal(b, t, 1))
    d['h'] = (normal(b, t, c) * size * loud + 0.1).to(DTYPES[dt])
    d['gate'] = None
    if case['gates'] != 'none':
      d['gate'] = normal(b, t if case['gates'] == 'row' else 1, c, std=0.5, mean=0.5, dtype=dt)
    d['w_post'], d['b_post'] = (None, None) if case['post'] == 'none' else (normal(c, std=0.1, mean=1.0), normal(c, std=0.1))
    d['w_pre'], d['b_pre'] = (None, None) if case['pre'] == 'none' else (normal(c, std=0.1, mean=1.0), normal(c, std=0.1))
    d['scale'] = normal(c, std=0.05, mean=0.3)
    d['x'] = normal(b, t, c, std=1.5, dtype=res)
    if case['way'] == 'bwd':
      d['dz'] = None if case['pre'] == 'none' else normal(b, t, c, std=1e-2, dtype=dt)
      d['dr'] = normal(b, t, c, std=1e-2, dtype=res)
    return d
  m, k, n = case['m'], case['k'], case['n']
  d = dict(w=normal(n, k, std=k ** -0.5, dtype=dt))
  d['x'] = (normal(m, k) * torch.exp(0.5 * normal(m, 1))).to(DTYPES[dt])
  if case['way'] == 'bwd':
    d['dy'] = normal(m, n, std=1e-3, dtype=dt)
  return d


def prepare(case, seed):
  d = _inputs(case, seed)
  if case['op'] == 'norm':
    if own:
      from advoc_amd import blocks
      d['norm'] = blocks.ResidualNorm(case['cols'], post=case['post'], pre=case['pre'], gate_act=case['act'], alpha=0.5, eps=EPS,
                                      keep_prob=case['keep'], w_post=d['w_post'], b_post=d['b_post'], scale=d['scale'],
                                      w_pre=d['w_pre'], b_pre=d['b_pre'])
    if case['way'] == 'bwd':
      # what the forward pass left behind: the residual stream and each row's statistics
      d['r'] = _norm_fwd(case, d)[0].to(DTYPES[case['res']])
      d['stats'] = torch.stack(_stats(d['h'].float(), case['post']) + _stats(d['r'].float(), case['pre']), dim=-1).reshape(-1, 4)
  if case['op'] == 'product':
    # weights are laid out once; a backward pass finds the inputs as the forward pass left them
    fmt = 'e4m3' if case['way'] == 'bwd' else case['fmt']
    w, x = d.pop('w'), d['x']
    if case['way'] == 'bwd':
      d.pop('x')
    if own:
      from advoc_amd import blocks
      d['w8'] = blocks.quantize_f8(w, fmt) if case['way'] == 'fwd' else blocks.quantize_f8_transposed(w, fmt)
      if case['way'] == 'bwd':
        d['x8'] = blocks.quantize_f8_transposed(x, fmt)
    else:
      d['w8'] = _to_f8(w.float(), fmt) if case['way'] == 'fwd' else _to_f8(w.float().t().contiguous(), fmt)
      if case['way'] == 'bwd':
        d['x8'] = _to_f8(x.float().t().contiguous(), fmt)
  return dict(case, **d)


# ---- the plain forms ----
def _keep_mask(n, seed, keep, device):
  """n keep decisions: word i % 4 of Philox-4x32-10 under key `seed` at counter i // 4, against (1 - keep) 2^32."""
  low = 0xffffffff
  i = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
  c0, c1, c2, c3 = i & low, i >> 32, torch.zeros_like(i), torch.zeros_like(i)
  k0, k1 = seed & low, (seed >> 32) & low
  for _ in range(10):
    p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57        # the low 64 bits, whatever their sign
    c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
    k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
  words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]
  return words >= _threshold(keep)


def _threshold(keep):
  return int(float((torch.tensor(1.0) - torch.tensor(keep)) * 4294967296.0))


def _drop(x, seed, keep):
  if keep == 1.0:
    return x
  m = _keep_mask(x.numel(), seed, keep, x.device).reshape(x.shape)
  return torch.where(m, x / torch.tensor(keep, device=x.device), torch.zeros((), device=x.device))


def _stats(a, kind):
  """[mean, 1 / sqrt(variance + eps)] of each row; the mean an RMS norm leaves in place is 0."""
  zero = torch.zeros_like(a[..., 0])
  if kind == 'none':
    return [zero, zero]
  mean = a.mean(-1) if kind == 'layer' else zero
  d = a - mean[..., None]
  return [mean, 1 / torch.sqrt((d * d).mean(-1) + EPS)]


def _normed(a, kind, w, b):
  if kind == 'none':
    return a
  mean, rstd = _stats(a, kind)
  return (a - mean[..., None]) * rstd[..., None] * w + b


def _gate(case, gate):
  return gate.float().sigmoid() if case['act'] == 'sigmoid' else gate.float()


def _norm_fwd(case, s):
  v = _drop(_normed(s['h'].float(), case['post'], s['w_post'], s['b_post']), s['seed'], case['keep'])
  if s['gate'] is not None:
    v = v * _gate(case, s['gate'])
  r = s['x'].float() + 0.5 * s['scale'] * v
  return r, _normed(r, case['pre'], s['w_pre'], s['b_pre'])


def _norm_back(g, hat, rstd, kind):
  """The gradient of a row given that of its normed values."""
  if kind == 'none':
    return g
  out = g - hat * (g * hat).mean(-1, keepdim=True)
  if kind == 'layer':
    out = out - g.mean(-1, keepdim=True)
  return out * rstd


def _norm_bwd(case, s):
  c, post, pre = case['cols'], case['post'], case['pre']
  h, r, g = s['h'].float(), s['r'].float(), s['dr'].float()
  stats = s['stats'].reshape(h.shape[:-1] + (4,))
  mean0, rstd0, mean1, rstd1 = (stats[..., i:i + 1] for i in range(4))
  out = {}
  if pre != 'none':
    dz, hat = s['dz'].float(), (r - mean1) * rstd1
    out['dw_pre'], out['db_pre'] = (dz * hat).reshape(-1, c).sum(0), dz.reshape(-1, c).sum(0)
    g = g + _norm_back(dz * s['w_pre'], hat, rstd1, pre)
  out['dx'] = g.to(s['r'].dtype)
  hat = h if post == 'none' else (h - mean0) * rstd0
  v = _drop(hat if post == 'none' else hat * s['w_post'] + s['b_post'], s['seed'], case['keep'])
  gate = 1.0 if s['gate'] is None else _gate(case, s['gate'])
  out['dscale'] = (0.5 * g * v * gate).reshape(-1, c).sum(0)
  if s['gate'] is not None:
    dgate = 0.5 * g * s['scale'] * v
    dgate = dgate.sum(1, keepdim=True) if case['gates'] == 'clip' else dgate
    out['dgate'] = (dgate * gate * (1 - gate) if case['act'] == 'sigmoid' else dgate).to(s['gate'].dtype)
  du = _drop(0.5 * g * s['scale'] * gate, s['seed'], case['keep'])
  if post != 'none':
    out['dw_post'], out['db_post'] = (du * hat).reshape(-1, c).sum(0), du.reshape(-1, c).sum(0)
    du = _norm_back(du * s['w_post'], hat, rstd0, post)
  out['dh'] = du.to(s['h'].dtype)
  return out


def _to_f8(x, fmt):
  """Rows of fp32 rounded to 8 bits with a power of two for each block of 128, as the values they stand for."""
  rows, k = x.shape
  x = torch.nn.functional.pad(x, (0, -k % 128)).reshape(rows, -1, 128)
  part, power = torch.frexp(x.abs().amax(-1, keepdim=True))
  power = (power - F8_TOP[fmt] + (part > 0.875).int()).clamp(min=-126)
  q = (x * _two_to(-power)).to(F8_TYPE[fmt]).float()
  return (q * _two_to(power)).reshape(rows, -1)[:, :k]


def _two_to(power):
  """2^power in fp32 from its bits: the library's own power function is not exact on every device."""
  return ((power + 127) << 23).view(torch.float32)


def run(state):
  s = state
  if own:
    return _run_own(s)
  if s['op'] == 'dropout':
    return _drop(s['x'].float(), s['seed'], s['keep']).to(s['x'].dtype)
  if s['op'] == 'norm':
    if s['way'] == 'bwd':
      return _norm_bwd(s, s)
    r, z = _norm_fwd(s, s)
    out = dict(r=r.to(s['x'].dtype))
    if s['pre'] != 'none':
      out['z'] = z.to(s['h'].dtype)
    if s['save']:
      out['stats'] = torch.stack(_stats(s['h'].float(), s['post']) + _stats(r, s['pre']), dim=-1).reshape(-1, 4)
    return out
  if s['way'] == 'fwd':
    return (_to_f8(s['x'].float(), s['fmt']) @ s['w8'].t()).to(s['x'].dtype)
  dy = s['dy'].float()
  dx = _to_f8(dy, s['fmt']) @ s['w8'].t()
  return dict(dx=dx.to(s['dy'].dtype), dw=_to_f8(dy.t().contiguous(), s['fmt']) @ s['x8'].t())


def _run_own(s):
  from advoc_amd import blocks
  if s['op'] == 'dropout':
    return blocks.dropout(s['x'], s['keep'], s['seed'])
  if s['op'] == 'norm':
    if s['way'] == 'fwd':
      r, z, stats = s['norm'].forward(s['h'], s['x'], gate=s['gate'], seed=s['seed'], save=s['save'])
      return {k: v for k, v in dict(r=r, z=z, stats=stats).items() if v is not None}
    g = s['norm'].backward(s['dz'], s['dr'], s['h'], s['r'], s['stats'], gate=s['gate'], seed=s['seed'])
    return {k: v for k, v in g._asdict().items() if v is not None}
  if s['way'] == 'fwd':
    return blocks.matmul_nt_f8(blocks.quantize_f8(s['x'], s['fmt']), s['w8'], out_dtype=s['x'].dtype)
  rows, cols = blocks.quantize_f8_both(s['dy'], s['fmt'])
  return dict(dx=blocks.matmul_nt_f8(rows, s['w8'], out_dtype=s['dy'].dtype), dw=blocks.matmul_nt_f8(cols, s['x8']))


# ---- the definitions in 64 bits ----
def _exact_words(n, seed, device):
  """The first n words of the stream: multiplications in 16-bit halves, so that no product leaves 53 bits."""
  def mul(a, b):
    lo = a * (b & 0xffff)
    hi = a * (b >> 16) + (lo >> 16)
    return hi >> 16, ((hi & 0xffff) << 16) | (lo & 0xffff)
  q = (n + 3) // 4
  x = [torch.arange(q, device=device) % 2 ** 32, torch.arange(q, device=device) // 2 ** 32,
       torch.zeros(q, dtype=torch.int64, device=device), torch.zeros(q, dtype=torch.int64, device=device)]
  for step in range(10):
    key = [(seed + step * 0x9E3779B9) % 2 ** 32, ((seed // 2 ** 32) + step * 0xBB67AE85) % 2 ** 32]
    h0, l0 = mul(x[0], 0xD2511F53)
    h1, l1 = mul(x[2], 0xCD9E8D57)
    x = [h1 ^ x[1] ^ key[0], l1, h0 ^ x[3] ^ key[1], l0]
  return torch.stack(x, -1).flatten()[:n]


def _exact_factor(shape, seed, keep, device):
  """m / keep of every element, keep as the fp32 number that it is."""
  keep = float(torch.tensor(keep, dtype=torch.float32).double())
  if keep == 1.0:
    return torch.ones(shape, dtype=torch.float64, device=device)
  cut = int(float(torch.tensor(1.0 - keep, dtype=torch.float32).double()) * 2.0 ** 32)
  n = math.prod(shape)
  return (_exact_words(n, seed, device) >= cut).double().div(keep).reshape(shape)


def _exact_norm(a, kind, w, b):
  if kind == 'none':
    return a
  if kind == 'layer':
    a = a - a.sum(-1, keepdim=True) / a.shape[-1]
  return a / (a.square().sum(-1, keepdim=True) / a.shape[-1] + EPS).sqrt() * w + b


def _exact_stat(a, kind, which):
  mean = a.sum(-1) / a.shape[-1] * (kind == 'layer')
  if which == 0 or kind == 'none':
    return mean * (which == 0)
  return 1 / ((a - mean[..., None]).square().sum(-1) / a.shape[-1] + EPS).sqrt()


def _exact_round(x, fmt):
  """Nearest value of the 8-bit format under each block's power of two, ties to even."""
  rows, k = x.shape
  bits, low, top = (3, -6, 448.0) if fmt == 'e4m3' else (2, -14, 57344.0)
  full = torch.zeros(rows, (k + 127) // 128 * 128, dtype=torch.float64, device=x.device)
  full[:, :k] = x
  full = full.view(rows, -1, 128)
  big = full.abs().max(-1, keepdim=True).values

  def floor_log2(a):       # of positive normal numbers, from their bits
    return (a.contiguous().view(torch.int64) >> 52) - 1023

  def exp2(p):
    return ((p + 1023) << 52).view(torch.float64)
  ratio = big.clamp(min=2.0 ** -126 * top) / top
  power = floor_log2(ratio)
  power = power + (ratio > exp2(power))
  y = full / exp2(power)
  step = exp2(floor_log2(y.abs().clamp(min=2.0 ** low)) - bits)
  return (torch.round(y / step) * step * exp2(power)).view(rows, -1)[:, :k]


def exact(case, seed):
  d = {k: v.double() if torch.is_tensor(v) else v for k, v in _inputs(case, seed).items()}
  if case['op'] == 'dropout':
    return d['x'] * _exact_factor(d['x'].shape, d['seed'], case['keep'], d['x'].device)
  if case['op'] == 'product':
    fmt = case['fmt']
    if case['way'] == 'fwd':
      return _exact_round(d['x'], fmt).matmul(_exact_round(d['w'], fmt).t())
    x, w = _exact_round(d['x'].t(), 'e4m3'), _exact_round(d['w'].t(), 'e4m3')
    return dict(dx=_exact_round(d['dy'], fmt).matmul(w.t()), dw=_exact_round(d['dy'].t(), fmt).matmul(x.t()))
  back = case['way'] == 'bwd'
  names = ['h', 'x', 'gate', 'w_post', 'b_post', 'scale', 'w_pre', 'b_pre']
  leaves = {k: d[k].requires_grad_(back) for k in names if d[k] is not None}
  factor = _exact_factor(d['h'].shape, d['seed'], case['keep'], d['h'].device)
  v = _exact_norm(d['h'], case['post'], d['w_post'], d['b_post']) * factor * d['scale'] * 0.5
  if d['gate'] is not None:
    v = v * (1 / (1 + torch.exp(-d['gate'])) if case['act'] == 'sigmoid' else d['gate'])
  r = d['x'] + v
  if not back:
    out = dict(r=r)
    if case['pre'] != 'none':
      out['z'] = _exact_norm(r, case['pre'], d['w_pre'], d['b_pre'])
    if case['save']:
      out['stats'] = torch.stack([_exact_stat(a, kind, which) for a, kind in ((d['h'], case['post']), (r, case['pre']))
                                  for which in (0, 1)], -1).view(-1, 4)
    return out
  # the norm before the next block sees the residual stream as it was stored
  total = (r * d['dr']).sum()
  if case['pre'] != 'none':
    with torch.no_grad():
      stored = _norm_fwd(case, {k: t.float() if torch.is_tensor(t) else t for k, t in d.items()})[0]
    stored = stored.to(DTYPES[case['res']]).double()
    total = total + (_exact_norm(r + (stored - r).detach(), case['pre'], d['w_pre'], d['b_pre']) * d['dz']).sum()
  keys = list(leaves)
  grads = dict(zip(keys, torch.autograd.grad(total, [leaves[k] for k in keys])))
  return {'d' + k: g for k, g in grads.items()}


def work(case):
  size = {'f32': 4, 'bf16': 2, 'f16': 2}
  e = size[case['dtype']]
  if case['op'] == 'dropout':
    n = case['rows'] * case['cols']
    return dict(bytes=2 * n * e, flops=n)
  if case['op'] == 'norm':
    rows, c, s = case['clips'] * case['frames'], case['cols'], size[case['res']]
    gate = {'none': 0, 'clip': case['clips'] * c * e, 'row': rows * c * e}[case['gates']]
    z = 0 if case['pre'] == 'none' else rows * c * e
    if case['way'] == 'fwd':
      return dict(bytes=rows * c * (e + 2 * s) + z + gate + 20 * c + 16 * rows * case['save'], flops=16 * rows * c)
    return dict(bytes=rows * c * (2 * e + 3 * s) + z + 2 * gate + 16 * rows + 36 * c, flops=40 * rows * c)
  m, k, n = case['m'], case['k'], case['n']
  blocks = lambda a: a + (a + 127) // 128      # noqa: E731  one byte an element, one a block
  if case['way'] == 'fwd':
    return dict(bytes=m * k * e + n * blocks(k) + m * n * e, flops=2 * m * n * k)
  return dict(bytes=m * n * e + k * blocks(n) + k * blocks(m) + m * k * e + 4 * n * k, flops=4 * m * n * k)
