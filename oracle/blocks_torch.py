"""Float64 restatement of the residual-block operators (advoc_amd/blocks.py) for the tests: the counter-based keep mask, the
residual norm with its gradients written out, and rounding to 8-bit blocks.  Test infrastructure; runs on the CPU."""
import numpy as np
import torch


def philox_words(seed, start, count):
  """Words start ... start + count - 1 of the Philox-4x32-10 stream under a 64-bit key, as numpy uint32."""
  q0, q1 = start // 4, (start + count + 3) // 4
  q = np.arange(q0, q1, dtype=np.uint64)
  low = np.uint64(0xffffffff)
  c = [q & low, q >> np.uint64(32), np.zeros_like(q), np.zeros_like(q)]
  k = [seed & 0xffffffff, (seed >> 32) & 0xffffffff]
  for _ in range(10):
    p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
    c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
    k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
  words = np.stack(c, axis=1).reshape(-1)
  return words[start - 4 * q0:start - 4 * q0 + count].astype(np.uint32)


def keep_mask(shape, seed, offset, keep):
  """Boolean tensor: element i (in logical order) is kept."""
  n = int(np.prod(shape))
  t = (np.float32(1.0) - np.float32(keep)) * np.float32(2.0 ** 32)
  cut = np.uint32(min(int(t), 2 ** 32 - 1))
  return torch.from_numpy(philox_words(seed, offset, n) >= cut).reshape(shape)


def norm_stats(a, kind, eps):
  mean = a.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(a[..., :1])
  if kind == 'none':
    return mean, torch.zeros_like(mean)
  return mean, 1 / torch.sqrt((a - mean).square().mean(-1, keepdim=True) + eps)


def drop(v, mask, keep):
  """What is dropped is 0 whatever it held."""
  return v if mask is None else torch.where(mask, v / float(np.float32(keep)), torch.zeros((), dtype=v.dtype))


def gate_act(gate, act):
  return torch.sigmoid(gate) if act == 'sigmoid' else gate


def residual_norm(h, x, gate=None, post='rms', pre='rms', act='none', alpha=1.0, eps=1e-5, keep=1.0, mask=None, w_post=None,
                  b_post=None, scale=None, w_pre=None, b_pre=None):
  """dict(r, z, stats) in the inputs' precision (float64).  mask: keep_mask of h's shape, or None."""
  one = torch.ones((), dtype=x.dtype)
  r = x
  mean0 = rstd0 = torch.zeros_like(x[..., :1])
  if h is not None:
    mean0, rstd0 = norm_stats(h, post, eps)
    u = h if post == 'none' else (h - mean0) * rstd0 * (one if w_post is None else w_post) + (0 if b_post is None else b_post)
    r = x + alpha * (one if scale is None else scale) * (one if gate is None else gate_act(gate, act)) * drop(u, mask, keep)
  mean1, rstd1 = norm_stats(r, pre, eps)
  z = None if pre == 'none' else (r - mean1) * rstd1 * (one if w_pre is None else w_pre) + (0 if b_pre is None else b_pre)
  return dict(r=r, z=z, stats=torch.cat([mean0, rstd0, mean1, rstd1], -1).reshape(-1, 4))


def residual_norm_backward(dz, dr, h, r, stats, gate=None, post='rms', pre='rms', act='none', alpha=1.0, keep=1.0, mask=None,
                           w_post=None, b_post=None, scale=None, w_pre=None, b_pre=None):
  """The gradients written out, and under 'size' what bounds the fp32 error of each: for row outputs the largest term of the
  row's sums, for column sums the sum of the terms' magnitudes."""
  c = r.shape[-1]
  one = torch.ones((), dtype=r.dtype)
  m0, s0, m1, s1 = (stats.reshape(r.shape[:-1] + (4,))[..., i:i + 1] for i in range(4))
  g = torch.zeros_like(r) if dr is None else dr
  out, size = {}, {}

  def colsum(name, t):
    out[name], size[name] = t.reshape(-1, c).sum(0), t.abs().reshape(-1, c).sum(0)

  def back(t, hat, rstd, kind):
    y = t - hat * (t * hat).mean(-1, keepdim=True)
    if kind == 'layer':
      y = y - t.mean(-1, keepdim=True)
    big = rstd * (t.abs() + t.abs().mean(-1, keepdim=True) + hat.abs() * (t * hat).abs().mean(-1, keepdim=True))
    return y * rstd, big
  big = g.abs()
  if pre != 'none':
    hat = (r - m1) * s1
    colsum('dw_pre', dz * hat)
    colsum('db_pre', dz)
    y, b = back(dz * (one if w_pre is None else w_pre), hat, s1, pre)
    g, big = g + y, big + b
    # r enters through its difference from the mean
    big = big + s1 * (r.abs() + m1.abs()) * s1 * (dz * (one if w_pre is None else w_pre)).abs().amax(-1, keepdim=True)
  out['dx'], size['dx'] = g, big.amax(-1, keepdim=True).expand_as(g)
  if h is None:
    return out, size
  gbig = size['dx']
  hat = h if post == 'none' else (h - m0) * s0
  v = drop(h if post == 'none' else hat * (one if w_post is None else w_post) + (0 if b_post is None else b_post), mask, keep)
  hbig = (h.abs() + (0 if post == 'none' else m0.abs())) * (1 if post == 'none' else s0)
  vbig = drop(hbig * (one if w_post is None else w_post.abs()) + (0 if b_post is None else b_post.abs()), mask, keep)
  gt = one if gate is None else gate_act(gate, act)
  k = alpha * (one if scale is None else scale)
  colsum('dscale', alpha * g * gt * v)
  size['dscale'] = (abs(alpha) * gbig * gt.abs() * vbig).reshape(-1, c).sum(0)
  if gate is not None:
    dact = gt * (1 - gt) if act == 'sigmoid' else one
    dg = g * k * v * dact
    dgb = (gbig * k.abs() * vbig * dact.abs()).expand_as(dg)
    for d in range(dg.dim() - 1):
      if gate.shape[d] == 1 and dg.shape[d] > 1:
        dg, dgb = dg.sum(d, keepdim=True), dgb.sum(d, keepdim=True)
    out['dgate'], size['dgate'] = dg, dgb
  du = drop((k * gt * g).expand_as(h), mask, keep)
  dub = drop(((k * gt).abs() * gbig).expand_as(h), mask, keep)
  if post != 'none':
    colsum('dw_post', du * (hat if mask is None else torch.where(mask, hat, torch.zeros((), dtype=hat.dtype))))
    colsum('db_post', du)
    size['dw_post'] = (dub * hbig).expand_as(du).reshape(-1, c).sum(0)
    size['db_post'] = dub.expand_as(du).reshape(-1, c).sum(0)
    w = one if w_post is None else w_post
    t = du * w
    y, _ = back(t, hat, s0, post)
    tb = (dub * w.abs()).expand_as(du)
    b = s0 * (tb + tb.mean(-1, keepdim=True) + hbig * (tb * hbig).mean(-1, keepdim=True))
    out['dh'], size['dh'] = y, b.amax(-1, keepdim=True).expand_as(y)
  else:
    out['dh'], size['dh'] = du, dub.expand_as(du)
  return out, size


F8 = {'e4m3': (3, -6, 448.0), 'e5m2': (2, -14, 57344.0)}


def f8_blocks(x, fmt):
  """(values, exponent bytes) of the rows of a float64 tensor in 8 bits: blocks of 128, a power of two each; x's infinities and
  NaN stay what the format can hold."""
  rows, k = x.shape
  bits, low, top = F8[fmt]
  kb = -(-k // 128)
  full = np.zeros((rows, kb * 128))
  full[:, :k] = x.numpy()
  full = full.reshape(rows, kb, 128)
  mag = np.abs(full)
  amax = np.where(np.isfinite(mag), mag, 0).max(-1)
  part, power = np.frexp(amax / top)                       # amax / top = part 2^power, part in [0.5, 1)
  e = np.maximum(np.where(part > 0.5, power, power - 1), -126)
  e = np.where(amax == 0, -126, e)
  y = full * np.exp2(-e.astype(np.float64))[..., None]
  _, ye = np.frexp(np.where(np.isfinite(y), y, 0))
  step = np.exp2((np.maximum(ye - 1, low) - bits).astype(np.float64))
  q = np.where(np.isfinite(y), np.round(np.where(np.isfinite(y), y, 0) / step) * step, y if fmt == 'e5m2' else np.nan)
  v = (q * np.exp2(e.astype(np.float64))[..., None]).reshape(rows, -1)[:, :k]
  return torch.from_numpy(v), torch.from_numpy((e + 127).astype(np.uint8))
