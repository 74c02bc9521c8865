"""Operators of residual blocks over the frames of a clip: dropout without a stored mask, the norms around a block with its
gate and residual scale, and products of 8-bit block-scaled matrices, each with its gradients.

Like ``conv.Layer`` this module only checks arguments and calls into libadvoc_hip.so (``include/advoc_hip.h`` holds the
formulas); no arithmetic happens in Python/torch, and there is no CPU path.  Tensors live in HBM; fp32, bf16 and fp16 are
taken, rows may be padded (unit stride inside a row, one distance between rows).  Every call is asynchronous on the current
stream of the tensors' device and can be captured into a graph.  None takes part in torch's autograd: gradients come from the
backward calls below, and a tensor that autograd follows is refused while it is on (parameters of a norm are taken as they are).

  one block:   z = N_pre(x);   y = W z;   r = x + alpha * scale * gate * dropout(N_post(y));   next block's z1 = N_pre(r)

  norm = blocks.ResidualNorm(cols, post='rms', pre='rms', w_post=w_post, scale=scale, w_pre=w_pre, keep_prob=0.9)
  w8, w8t = blocks.quantize_f8(w), blocks.quantize_f8_transposed(w)              # once per update of w [cols, cols]
  z8, z8t = blocks.quantize_f8_both(z)                                           # z8t is for dw
  y = blocks.matmul_nt_f8(z8, w8, out_dtype=z.dtype)
  r, z1, stats = norm.forward(y, x, gate=gate, seed=step, save=True)
  g = norm.backward(dz1, dr, y, r, stats, gate=gate, seed=step)                  # g.dh is dL/dy, g.dx dL/dx
  dy8, dy8t = blocks.quantize_f8_both(g.dh, 'e5m2')
  dz = blocks.matmul_nt_f8(dy8, w8t, out_dtype=z.dtype)                          # the dz1 of the block before
  dw = blocks.matmul_nt_f8(dy8t, z8t)
"""
import collections
import functools
import struct

import torch

from advoc_amd import _lib

NORMS = {'none': 0, 'rms': 1, 'layer': 2}
GATE_ACTS = {'none': 0, 'sigmoid': 1}
FORMATS = {'e4m3': 0, 'e5m2': 1}
MAX_COLS = 8192

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MASK64 = 2 ** 64 - 1


def _choice(table, key, what):
  try:
    return table[key]
  except (KeyError, TypeError):
    raise _lib.AdvocHipError('{} {!r} is none of {}'.format(what, key, sorted(table)))


def _dtype(t, name):
  code = _DTYPES.get(t.dtype)
  if code is None:
    raise _lib.AdvocHipError('{} must be float32, bfloat16 or float16, got {}'.format(name, t.dtype))
  return code


def _rows(t, name, index=None):
  """(address, rows, cols, elements from row to row) of a tensor as rows of its last dimension; index: the device it must be on."""
  if not isinstance(t, torch.Tensor) or not t.is_cuda:
    raise _lib.AdvocHipError('{} must be a torch tensor on a HIP device (no CPU path exists)'.format(name))
  if index is not None and t.get_device() != index:
    raise _lib.AdvocHipError('{} is on {}, the other tensors on device {}'.format(name, t.device, index))
  if t.requires_grad and torch.is_grad_enabled():
    raise _lib.AdvocHipError('{} needs a gradient, which autograd does not get from here: call under torch.no_grad() or on '
                             '{}.detach(), and the backward calls by hand'.format(name, name))
  if not t.dim():
    raise _lib.AdvocHipError('{} must have at least one dimension'.format(name))
  cols = t.shape[-1]
  if t.is_contiguous():
    return t.data_ptr(), t.numel() // cols if cols else 0, cols, cols
  rows, pitch, expect = 1, cols, None
  for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
    if size == 1:
      continue
    if expect is None:
      pitch = stride
    elif stride != expect:
      raise _lib.AdvocHipError('{} (shape {}, strides {}) is not rows at one distance'.format(name, tuple(t.shape), t.stride()))
    rows *= size
    expect = stride * size
  if cols > 1 and t.stride(-1) != 1 or rows > 1 and pitch < cols:
    raise _lib.AdvocHipError('{} (shape {}, strides {}): a row must have unit stride and rows must not overlap'.format(
        name, tuple(t.shape), t.stride()))
  return t.data_ptr(), rows, cols, pitch


def _seed_word(seed_dev, index):
  if seed_dev is None:
    return 0
  if not isinstance(seed_dev, torch.Tensor) or not seed_dev.is_cuda or seed_dev.get_device() != index or (
      seed_dev.numel() != 1) or seed_dev.dtype not in (torch.int64, torch.uint64):
    raise _lib.AdvocHipError('seed_dev must be one int64 or uint64 on device {}'.format(index))
  return seed_dev.data_ptr()


# (torch.cuda.current_stream() and current_device() spend 9 us in Python per call, several times what the smallest kernels take)
_raw_stream = torch._C._cuda_getCurrentRawStream
_devices = None


def _call(fn, what, index, *args):
  """One library call on the current stream of device `index`, with that device current."""
  global _devices
  if _devices is None:
    _devices = torch.cuda.device_count()
  if _devices == 1 or torch.cuda.current_device() == index:
    rc = fn(*args, _raw_stream(index))
  else:
    with torch.cuda.device(index):
      rc = fn(*args, _raw_stream(index))
  if rc:
    _lib.check(rc, what)


def dropout(x, keep_prob, seed, offset=0, seed_dev=None, out=None):
  """x / keep_prob where a counter-based generator keeps an element, 0 elsewhere (``advoc_dropout``): the same elements as the
  mask ``advoc_dropout_mask_u8`` writes for (seed, offset), without the mask.  The gradient is the same call on dy with the
  same numbers.

  Element i (in logical order, whatever the strides) draws at offset + i: shards of a batch that pass their own offset (a
  multiple of 4) drop what the whole batch would.  seed_dev: one int64 on the device, added to the seed by the kernel, for
  graphs whose replays must not repeat a mask.  out: a tensor of x's shape and dtype, or x itself."""
  px, rows, cols, pitch = _rows(x, 'x')
  code = _dtype(x, 'x')
  index = x.get_device()
  if out is None:
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    py, out_pitch = out.data_ptr(), cols
  else:
    py, _, _, out_pitch = _rows(out, 'out', index)
    if out.shape != x.shape or out.dtype != x.dtype:
      raise _lib.AdvocHipError('out must have the shape and dtype of x')
  _call(_lib.load().advoc_dropout, 'advoc_dropout', index, px, pitch, py, out_pitch, rows, cols, code, keep_prob,
        seed & _MASK64, offset & _MASK64, _seed_word(seed_dev, index))
  return out


ResidualNormGrads = collections.namedtuple('ResidualNormGrads',
                                           ['dh', 'dx', 'dgate', 'dw_post', 'db_post', 'dscale', 'dw_pre', 'db_pre'])


_PARAMETER_GRADS = ResidualNormGrads._fields[3:]

# struct advoc_residual_norm packed in one go (a ctypes structure costs 4 us a call to fill): up to the parameter gradients, and the
# workspace behind them
_DESCRIPTOR_HEAD = struct.Struct('@q6iq5P3fi2QP' + 'Pq' * 5 + 'P' + 'Pq' * 5 + '5P')
_DESCRIPTOR_TAIL = struct.Struct('@Pq')
_DESCRIPTOR = struct.Struct(_DESCRIPTOR_HEAD.format + _DESCRIPTOR_TAIL.format[1:])
_ABSENT = (0, 0)
_NO_BACKWARD = (0,) * 17
_NO_WORKSPACE = _DESCRIPTOR_TAIL.pack(0, 0)


class ResidualNorm(object):
  """The glue between two residual blocks (``advoc_residual_norm_forward / _backward``), per row of `cols` channels:

    u = N_post(h) * w_post + b_post                   the norm behind the block that computed h
    r = x + alpha * scale * act(gate) * dropout(u)    its gate, residual scale and dropout, and the residual sum
    z = N_pre(r) * w_pre + b_pre                      the norm before the next block

  post, pre: 'none' | 'rms' | 'layer'; gate_act: 'none' | 'sigmoid'.  The parameters are float32 [cols] tensors, each may be
  None; they are read at every call, so in-place updates are seen.  h, gate and z have one dtype; x and r have that dtype or
  float32."""

  def __init__(self, cols, post='rms', pre='rms', gate_act='none', alpha=1.0, eps=1e-5, keep_prob=1.0, w_post=None,
               b_post=None, scale=None, w_pre=None, b_pre=None):
    if not 1 <= cols <= MAX_COLS:
      raise _lib.AdvocHipError('cols must be 1 ... {}, got {}'.format(MAX_COLS, cols))
    if not eps > 0 or not 0 < keep_prob <= 1:
      raise _lib.AdvocHipError('eps must be positive and keep_prob in (0, 1]')
    self.cols, self._shape = cols, torch.Size((cols,))
    self.post, self.pre = _choice(NORMS, post, 'norm'), _choice(NORMS, pre, 'norm')
    self.gate_act = _choice(GATE_ACTS, gate_act, 'gate activation')
    self.alpha, self.eps, self.keep_prob = alpha, eps, keep_prob
    self.w_post, self.b_post, self.scale, self.w_pre, self.b_pre = w_post, b_post, scale, w_pre, b_pre
    if not self.post and (w_post is not None or b_post is not None) or not self.pre and (w_pre is not None or b_pre is not None):
      raise _lib.AdvocHipError('a norm of kind none takes no weight or bias')

  def _vector(self, t, name, index):
    if t is None:
      return 0
    if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dtype != torch.float32 or t.shape != self._shape or (
        not t.is_contiguous()):
      raise _lib.AdvocHipError('{} must be a contiguous float32 tensor of {} on device {}'.format(name, self.cols, index))
    return t.data_ptr()

  def _tensor(self, name, t, rows, index, dtype=None):
    """(address, pitch) of `rows` rows of self.cols; dtype: the one it has to have."""
    p, n, cols, pitch = _rows(t, name, index)
    if n != rows or cols != self.cols:
      raise _lib.AdvocHipError('{} has shape {}: {} rows of {} wanted'.format(name, tuple(t.shape), rows, self.cols))
    if dtype is not None and t.dtype != dtype:
      raise _lib.AdvocHipError('{} is {}, {} wanted'.format(name, t.dtype, dtype))
    return p, pitch

  def _head(self, x, name, dtype, gate, seed, offset, seed_dev, has_h):
    """What both directions share; x (r in the backward pass) sets rows, device and residual dtype.  -> (device index, rows, x's
    address and pitch, the gate's, the descriptor's fields up to the gate group, those from the weights to keep_prob, seed to
    seed_dev)"""
    px, rows, cols, pitch = _rows(x, name)
    if cols != self.cols:
      raise _lib.AdvocHipError('{} has {} columns, {} wanted'.format(name, cols, self.cols))
    index = x.get_device()
    code, res_code = _DTYPES.get(dtype, -1), _dtype(x, name)
    if code < 0 or res_code not in (code, 0):
      raise _lib.AdvocHipError('{} is {}: it must be float32 or the dtype of the block ({})'.format(name, x.dtype, dtype))
    w_pre, b_pre = self._vector(self.w_pre, 'w_pre', index), self._vector(self.b_pre, 'b_pre', index)
    if not has_h:
      if gate is not None:
        raise _lib.AdvocHipError('a gate needs a block output h')
      return (index, rows, px, pitch, _ABSENT, (rows, cols, code, res_code, 0, self.pre, 0, 1),
              (0, 0, 0, w_pre, b_pre, self.alpha, self.eps, self.keep_prob), (0, 0, 0))
    pg, group = _ABSENT, 1
    if gate is not None:
      p, n, gate_cols, gate_pitch = _rows(gate, 'gate', index)
      if gate_cols != cols or gate.dtype != dtype or (rows % n if n else rows):
        raise _lib.AdvocHipError('gate {} {} does not divide {} rows of {} {}'.format(
            gate.dtype, tuple(gate.shape), rows, cols, dtype))
      self._check_gate_shape(gate, x)
      pg, group = (p, gate_pitch), rows // n if n else 1
    return (index, rows, px, pitch, pg, (rows, cols, code, res_code, self.post, self.pre, self.gate_act, group),
            (self._vector(self.w_post, 'w_post', index), self._vector(self.b_post, 'b_post', index),
             self._vector(self.scale, 'scale', index), w_pre, b_pre, self.alpha, self.eps, self.keep_prob),
            (seed & _MASK64, offset & _MASK64, _seed_word(seed_dev, index)))

  def _check_gate_shape(self, gate, x):
    """A gate has x's shape, with ones for trailing row dimensions that share it: [clips, 1, cols] for [clips, frames, cols]."""
    if gate.shape == x.shape:
      return
    lead, want = gate.shape[:-1], x.shape[:-1]
    if len(lead) == len(want):
      i = 0
      while i < len(lead) and lead[i] == want[i]:
        i += 1
      if all(n == 1 for n in lead[i:]):
        return
    raise _lib.AdvocHipError('gate of shape {} for rows of shape {}'.format(tuple(gate.shape), tuple(x.shape)))

  def forward(self, h, x, gate=None, seed=0, offset=0, seed_dev=None, save=False, r=None, z=None):
    """(r, z, stats).  h None: only z = N_pre(x), the norm before the first block (r is x).  z is None without a pre norm,
    stats [rows, 4] is None unless `save` (a later backward needs it).  r, z: buffers to write into; r may be x."""
    like = h if h is not None else z if z is not None else x
    if not isinstance(like, torch.Tensor):
      raise _lib.AdvocHipError('h and x must be torch tensors')
    dtype = like.dtype
    index, rows, px, pitch, pg, shape, weights, draw = self._head(x, 'x', dtype, gate, seed, offset, seed_dev, h is not None)
    ph = pr = pz = _ABSENT
    if h is None:
      if not self.pre:
        raise _lib.AdvocHipError('neither h nor a pre norm: nothing to compute')
      if r is not None and r is not x:
        raise _lib.AdvocHipError('without h the residual stream stays x: r is not written')
      r = x
    else:
      ph = self._tensor('h', h, rows, index)
      if r is None:
        r = torch.empty_like(x, memory_format=torch.contiguous_format)
        pr = r.data_ptr(), self.cols
      else:
        pr = self._tensor('r', r, rows, index, x.dtype)
    if not self.pre:
      if z is not None:
        raise _lib.AdvocHipError('without a pre norm there is no z')
    elif z is None:
      z = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
      pz = z.data_ptr(), self.cols
    else:
      pz = self._tensor('z', z, rows, index, dtype)
    stats = torch.empty(rows, 4, dtype=torch.float32, device=x.device) if save else None
    d = _DESCRIPTOR.pack(*shape, *weights, 0, *draw, *ph, px, pitch, *pg, *pr, *pz, stats.data_ptr() if save else 0,
                         *_NO_BACKWARD)
    _call(_lib.load().advoc_residual_norm_forward, 'advoc_residual_norm_forward', index, d)
    return r, z, stats

  def backward(self, dz, dr, h, r, stats, gate=None, seed=0, offset=0, seed_dev=None, into=None, accumulate=False):
    """Gradients of forward(h, x, gate, seed, offset) with its r and stats (h None: r is x).  dz: gradient of z (None without a
    pre norm), dr: gradient of r from elsewhere (may be None with a pre norm).  Gradients of what was not given are None, the
    others have the shapes of h, r, the gate and the parameters.
    into: {'dw_post': float32 [cols] buffer, ...} to write parameter gradients into, or with `accumulate` to add to."""
    like = h if h is not None else dz
    if not isinstance(like, torch.Tensor):
      raise _lib.AdvocHipError('h or dz is needed')
    index, rows, p, pitch, pg, shape, weights, draw = self._head(r, 'r', like.dtype, gate, seed, offset, seed_dev, h is not None)
    if (dz is None) != (not self.pre) or (dz is None and dr is None):
      raise _lib.AdvocHipError('dz goes with a pre norm, and dz or dr must be given')
    pdz = _ABSENT if dz is None else self._tensor('dz', dz, rows, index, like.dtype)
    pdr = _ABSENT if dr is None else self._tensor('dr', dr, rows, index, r.dtype)
    ph = _ABSENT if h is None else self._tensor('h', h, rows, index)
    pstats = 0
    if self.pre or h is not None and self.post:
      if not isinstance(stats, torch.Tensor) or stats.get_device() != index or stats.dtype != torch.float32 or (
          stats.shape != (rows, 4) or not stats.is_contiguous()):
        raise _lib.AdvocHipError('stats must be the contiguous float32 [rows, 4] tensor of forward(..., save=True)')
      pstats = stats.data_ptr()
    contiguous, cols = torch.contiguous_format, self.cols
    dx = torch.empty_like(r, memory_format=contiguous)
    dh = dgate = None
    pdh = pdgate = _ABSENT
    if h is not None:
      dh = torch.empty_like(h, memory_format=contiguous)
      pdh = dh.data_ptr(), cols
    if gate is not None:
      dgate = torch.empty_like(gate, memory_format=contiguous)
      pdgate = dgate.data_ptr(), cols
    # dw_post, db_post, dscale, dw_pre, db_pre
    wanted = [w is not None for w in (self.w_post, self.b_post, self.scale, self.w_pre, self.b_pre)]
    if h is None:
      wanted[:3] = (False, False, False)
    g = [None] * 5
    if into:
      unknown = set(into) - {name for name, want in zip(_PARAMETER_GRADS, wanted) if want}
      if unknown:
        raise _lib.AdvocHipError('no such parameter gradients here: {}'.format(sorted(unknown)))
      for i, name in enumerate(_PARAMETER_GRADS):
        g[i] = into.get(name)
        self._vector(g[i], name, index)
    new = [i for i in range(5) if wanted[i] and g[i] is None]
    if new:
      if accumulate:
        raise _lib.AdvocHipError('accumulate needs a buffer for {}'.format([_PARAMETER_GRADS[i] for i in new]))
      for i, t in zip(new, torch.empty(len(new), cols, dtype=torch.float32, device=r.device).unbind()):
        g[i] = t
    pgrads = [0 if t is None else t.data_ptr() for t in g]
    head = _DESCRIPTOR_HEAD.pack(*shape, *weights, 1 if accumulate else 0, *draw, *ph, *_ABSENT, *pg, p, pitch, *_ABSENT, pstats,
                                 *pdz, *pdr, *pdh, dx.data_ptr(), cols, *pdgate, *pgrads)
    lib = _lib.load()
    nbytes = lib.advoc_residual_norm_workspace_bytes(head + _NO_WORKSPACE)
    work = torch.empty(nbytes // 4, dtype=torch.float32, device=r.device) if nbytes else None
    _call(lib.advoc_residual_norm_backward, 'advoc_residual_norm_backward', index,
          head + _DESCRIPTOR_TAIL.pack(work.data_ptr(), nbytes) if nbytes else head + _NO_WORKSPACE)
    return ResidualNormGrads(dh, dx, dgate, *g)


class F8Matrix(object):
  """A matrix held in 8 bits with a power of two for each block of 128 along its rows, made by the quantize_f8 functions:
  `data` [rows, kp] and `scale` [rows, sp] (uint8; layout in include/advoc_hip.h) are two parts of one buffer."""
  __slots__ = ('buffer', 'rows', 'k', 'format', 'data_ptr', 'scale_ptr')

  def __init__(self, rows, k, format, device):
    kp = -(-k // 128) * 128
    self.rows, self.k, self.format = rows, k, format
    self.buffer = torch.empty(rows * (kp + -(-kp // 512) * 4), dtype=torch.uint8, device=device)
    self.data_ptr = self.buffer.data_ptr()
    self.scale_ptr = self.data_ptr + rows * kp

  @property
  def shape(self):
    return (self.rows, self.k)

  @property
  def data(self):
    kp = -(-self.k // 128) * 128
    return self.buffer[:self.rows * kp].view(self.rows, kp)

  @property
  def scale(self):
    return self.buffer[self.rows * (-(-self.k // 128) * 128):].view(self.rows, -1)


def _quantize(x, fmt, want_rows, want_cols):
  code = _choice(FORMATS, fmt, 'format')
  p, rows, cols, pitch = _rows(x, 'x')
  if not rows or not cols:
    raise _lib.AdvocHipError('x of shape {} holds nothing to quantise'.format(tuple(x.shape)))
  a = F8Matrix(rows, cols, code, x.device) if want_rows else None
  t = F8Matrix(cols, rows, code, x.device) if want_cols else None
  _call(_lib.load().advoc_f8_quantize, 'advoc_f8_quantize', x.get_device(), p, pitch, rows, cols, _dtype(x, 'x'), code,
        a and a.data_ptr, a and a.scale_ptr, t and t.data_ptr, t and t.scale_ptr)
  return a, t


def quantize_f8(x, fmt='e4m3'):
  """The rows of x [..., k] in 8 bits ('e4m3' | 'e5m2'), a scale per block of 128 along k: an operand of matmul_nt_f8."""
  return _quantize(x, fmt, True, False)[0]


def quantize_f8_transposed(x, fmt='e4m3'):
  """x^T in 8 bits, blocks of 128 along x's rows: the operand of a product that contracts over the rows of x."""
  return _quantize(x, fmt, False, True)[1]


def quantize_f8_both(x, fmt='e4m3'):
  """(quantize_f8(x), quantize_f8_transposed(x)) with one read of x."""
  return _quantize(x, fmt, True, True)


@functools.lru_cache(maxsize=4096)
def _product_workspace(m, n, k, code):
  return _lib.load().advoc_matmul_nt_f8_workspace_bytes(m, n, k, code)


def matmul_nt_f8(a, b, out_dtype=None, out=None, accumulate=False):
  """a b^T of two F8Matrix operands with the same k -> [a.rows, b.rows] (``advoc_matmul_nt_f8``); a float32 result is
  accumulated in fp32 throughout, a 16-bit one in the 8-bit matrix instruction's sums, at twice the rate and 1.5e-5 off in norm
  (bounds in include/advoc_hip.h).  out_dtype: that of `out`, without one float32.  accumulate: add to `out` (float32), e.g. a
  gradient arena's slice."""
  if not isinstance(a, F8Matrix) or not isinstance(b, F8Matrix) or a.k != b.k or a.buffer.device != b.buffer.device:
    raise _lib.AdvocHipError('two F8Matrix operands with the same k on one device are needed')
  device, m, n = a.buffer.device, a.rows, b.rows
  if out is None:
    if accumulate:
      raise _lib.AdvocHipError('accumulate needs out')
    out = torch.empty(m, n, dtype=out_dtype or torch.float32, device=device)
  elif not isinstance(out, torch.Tensor) or out.device != device or out.shape != (m, n) or not out.is_contiguous():
    raise _lib.AdvocHipError('out must be a contiguous [{}, {}] tensor on {}'.format(m, n, device))
  elif out_dtype is not None and out.dtype != out_dtype:
    raise _lib.AdvocHipError('out is {}, out_dtype {}'.format(out.dtype, out_dtype))
  code = _dtype(out, 'out')
  lib = _lib.load()
  nbytes = _product_workspace(m, n, a.k, code)
  work = torch.empty(nbytes // 4, dtype=torch.float32, device=device) if nbytes else None
  _call(lib.advoc_matmul_nt_f8, 'advoc_matmul_nt_f8', device.index, a.data_ptr, a.scale_ptr, a.format, b.data_ptr, b.scale_ptr,
        b.format, out.data_ptr(), code, int(bool(accumulate)), m, n, a.k,
        work.data_ptr() if nbytes else None, nbytes)
  return out
