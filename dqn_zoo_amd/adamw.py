"""AdamW over a list of tensors (include/dqnzoo_hip.h: dz_adamw_*; csrc/dz_adamw.hip).

The fused learners' optimisers (`learner.AdamConfig`, `learner.RmsPropConfig`) update one network's
flat float32 parameter vector inside the learner step.  `AdamW` is the optimiser for everything
else: any list of float32, bfloat16 or float16 tensors, decoupled weight decay, clipping by the
global norm, master weights, moments in 32 or 8 bits.

    opt = adamw.AdamW([w1, b1, w2, b2], adamw.AdamWConfig(weight_decay=0.1, state_bits=8),
                      decay=[True, False, True, False])
    opt.step([dw1, db1, dw2, db2])       # gradients of this step
    bound = opt.bind([dw1, ...])         # or: buffers that every step's gradients are written to
    opt.step(bound)

Work is enqueued on the current stream of the parameters' device; nothing synchronises.  A step may
be captured into a graph: the step count and the learning rate live on the device.  The parameters
(and bound gradients) have to stay where they are in memory, as for any captured work.
"""

import ctypes
import operator
import typing

import numpy as np
import torch

from dqn_zoo_amd import _lib

_SHAPE, _DTYPE = operator.attrgetter('shape'), operator.attrgetter('dtype')


class AdamWConfig(typing.NamedTuple):
  """p -= learning_rate * (m_hat / (sqrt(v_hat) + eps) + weight_decay * p) behind a clip by the
  global norm (max_global_grad_norm <= 0: none).  state_bits: 32, or 8 (one byte per moment and
  element, one scale per 256 elements, rounded at random; see dz_adamw_args_t)."""
  learning_rate: float = 3e-4
  b1: float = 0.9
  b2: float = 0.999
  eps: float = 1e-8
  weight_decay: float = 0.01
  max_global_grad_norm: float = 0.0
  state_bits: int = 32


class BoundGradients:
  """Gradient buffers whose addresses are on the device (`AdamW.bind`)."""

  def __init__(self, owner, grads, table, dtype):
    self.owner, self.grads, self.table, self.dtype = owner, grads, table, dtype


def _extent(t):
  return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class AdamW:

  def __init__(self, params: typing.Sequence[torch.Tensor], config: AdamWConfig,
               decay: typing.Optional[typing.Sequence[bool]] = None,
               master_weights: typing.Optional[bool] = None, seed: int = 1):
    """`decay[i]` False exempts params[i] from the weight decay (default: none exempt).
    `master_weights` (default: True for 16-bit parameters): keep a float32 copy that the steps
    update and the parameters are rounded from.  `seed`: of the 8-bit moments' rounding."""
    params = list(params)
    if not params:
      raise ValueError('AdamW needs at least one parameter tensor')
    self._index = _lib.gpu_index('params[0]', params[0])
    self.device = torch.device('cuda', self._index)
    dtype = params[0].dtype
    if _lib.dtype_code(dtype) is None:
      raise TypeError('parameters must be float32, bfloat16 or float16, got %s' % dtype)
    for i, p in enumerate(params):
      if _lib.gpu_index('params[%d]' % i, p) != self._index:
        raise ValueError('params[%d] is on another device than params[0]' % i)
      if p.dtype != dtype:
        raise TypeError('params[%d] is %s, params[0] %s' % (i, p.dtype, dtype))
      if not p.is_contiguous() or not p.numel():
        raise ValueError('params[%d] must be contiguous and not empty, got shape %s, strides %s' %
                         (i, tuple(p.shape), p.stride()))
    extents = sorted((_extent(p), i) for i, p in enumerate(params))
    for ((_, end), i), ((start, _), j) in zip(extents, extents[1:]):
      if start < end:
        raise ValueError('params[%d] and params[%d] share memory' % (i, j))
    c = AdamWConfig(*config)
    if c.state_bits not in (8, 32):
      raise ValueError('state_bits must be 8 or 32, got %r' % (c.state_bits,))
    if not (0 <= c.b1 < 1 and 0 <= c.b2 < 1 and c.eps >= 0):
      raise ValueError('need 0 <= b1, b2 < 1 and eps >= 0, got %s' % (c,))
    if decay is None:
      decay = [True] * len(params)
    if len(decay) != len(params):
      raise ValueError('decay has %d entries for %d parameters' % (len(decay), len(params)))
    if master_weights is None:
      master_weights = dtype != torch.float32
    if master_weights and dtype == torch.float32:
      raise ValueError('float32 parameters need no master weights')
    self._lib = _lib.load()
    self.config = c
    self.params = params
    self._extents = extents
    self._dtype = dtype
    self._shapes = [p.shape for p in params]
    self._seed = int(seed) & 0xFFFFFFFFFFFFFFFF

    block, chunk = _lib.ADAMW_STATE_BLOCK, _lib.ADAMW_CHUNK
    sizes = np.array([p.numel() for p in params], np.int64)
    room = -(-sizes // block) * block
    self.offsets = (np.cumsum(room) - room).tolist()
    total = int(room.sum())
    self.state_size = total
    table = (_lib.AdamWTensor * len(params))()
    for i, p in enumerate(params):
      table[i] = _lib.AdamWTensor(p.data_ptr(), p.numel(), self.offsets[i],
                                  c.weight_decay if decay[i] else 0.0, 0)
    pieces = -(-sizes // chunk)
    which = np.repeat(np.arange(len(params)), pieces)
    first = np.cumsum(pieces) - pieces
    chunks = np.stack([which, np.arange(len(which)) - first[which]], 1).astype(np.int32)
    f32 = dict(dtype=torch.float32, device=self.device)
    u8 = dict(dtype=torch.uint8, device=self.device)
    self._tensors = torch.from_numpy(np.frombuffer(table, np.uint8).copy()).to(self.device)
    self._chunks = torch.from_numpy(chunks).to(self.device)
    self._table = torch.zeros(len(params), dtype=torch.int64, device=self.device)
    self.master = None
    if master_weights:
      self.master = torch.zeros(total, **f32)
      for p, o in zip(params, self.offsets):
        self.master[o:o + p.numel()] = p.detach().reshape(-1).float()
    self.m_scale = self.v_scale = None
    if c.state_bits == 8:
      self.m, self.v = torch.zeros(total, **u8), torch.zeros(total, **u8)
      self.m_scale, self.v_scale = torch.zeros(total // block, **f32), torch.zeros(total // block, **f32)
    else:
      self.m, self.v = torch.zeros(total, **f32), torch.zeros(total, **f32)
    self._count = torch.zeros(1, dtype=torch.int32, device=self.device)
    self._lr = torch.full((1,), float(c.learning_rate), **f32)
    self._scalars = torch.zeros(8, **f32)
    clip = c.max_global_grad_norm > 0
    self._partials = torch.zeros(len(chunks), **f32) if clip else None
    self._args = _lib.AdamWArgs(
        _lib.dtype_code(dtype), _lib.dtype_code(dtype), c.state_bits, len(chunks),
        self._tensors.data_ptr(), self._chunks.data_ptr(), None, _lib.ptr(self.master),
        self.m.data_ptr(), self.v.data_ptr(), _lib.ptr(self.m_scale), _lib.ptr(self.v_scale),
        self._count.data_ptr(), self._lr.data_ptr(), self._scalars.data_ptr(),
        _lib.ptr(self._partials), c.b1, c.b2, c.eps, c.max_global_grad_norm, 1.0, 0,
        self._seed)

  # -- gradients ----------------------------------------------------------------
  def _check(self, grads):
    """Shapes, types, devices and layouts of one gradient per parameter; their dtype."""
    if len(grads) != len(self.params):
      raise ValueError('%d gradients for %d parameters' % (len(grads), len(self.params)))
    for i, g in enumerate(grads):
      if not isinstance(g, torch.Tensor):
        raise TypeError('grads[%d] must be a tensor, got %s' % (i, type(g).__name__))
    if list(map(_SHAPE, grads)) != self._shapes:
      bad = [i for i, (g, s) in enumerate(zip(grads, self._shapes)) if g.shape != s]
      raise ValueError('grads[%d] has shape %s, its parameter %s' % (
          bad[0], tuple(grads[bad[0]].shape), tuple(self._shapes[bad[0]])))
    dtypes = set(map(_DTYPE, grads))
    if len(dtypes) > 1 or not dtypes <= {self._dtype, torch.float32}:
      raise TypeError('gradients must be all %s or all float32, got %s' %
                      (self._dtype, sorted(map(str, dtypes))))
    if not all(map(torch.Tensor.is_contiguous, grads)):
      raise ValueError('gradients must be contiguous')
    if set(map(torch.Tensor.get_device, grads)) != {self._index}:
      raise ValueError('gradients must be on the parameters\' device %s' % self.device)
    return dtypes.pop()

  def _upload(self, grads, table):
    pointers = (ctypes.c_void_p * len(grads))(*[g.data_ptr() for g in grads])
    _lib.check(self._lib.dz_adamw_bind(pointers, len(grads), table.data_ptr(),
                                       _lib.stream_ptr(self._index)), 'dz_adamw_bind')

  def bind(self, grads: typing.Sequence[torch.Tensor]) -> BoundGradients:
    """Buffers that later steps' gradients will be in: `step(bound)` then checks and sends
    nothing per tensor."""
    grads = list(grads)
    dtype = self._check(grads)
    ends = sorted([(e, 0) for e, _ in self._extents] + [(_extent(g), 1) for g in grads])
    last = [0, 0]   # the furthest end of a parameter, of a gradient
    for (start, end), kind in ends:
      if start < last[1 - kind]:
        raise ValueError('a gradient shares memory with a parameter')
      last[kind] = max(last[kind], end)
    with _lib.device_guard(self._index):
      table = _lib.new_output(len(grads), torch.int64, self.device)
      self._upload(grads, table)
    return BoundGradients(self, grads, table, dtype)

  # -- the step -----------------------------------------------------------------
  def step(self, grads, grad_scale: float = 1.0) -> None:
    """One update.  `grads`: one tensor per parameter (its type, or float32), or what `bind`
    returned.  `grad_scale` multiplies the gradients first (1 / the loss scale, or 1 / the number
    of accumulated batches); a graph keeps the value it was captured with."""
    with _lib.device_guard(self._index):
      if isinstance(grads, BoundGradients):
        if grads.owner is not self:
          raise ValueError('these gradients were bound by another optimizer')
        dtype, table = grads.dtype, grads.table
      else:
        grads = list(grads)
        dtype, table = self._check(grads), self._table
        self._upload(grads, table)
      a = self._args
      a.grads = table.data_ptr()
      a.grad_dtype = _lib.dtype_code(dtype)
      a.grad_scale = grad_scale
      _lib.check(self._lib.dz_adamw_step(ctypes.byref(a), _lib.stream_ptr(self._index)),
                 'dz_adamw_step')

  @property
  def learning_rate(self) -> float:
    return float(self._lr.item())

  @learning_rate.setter
  def learning_rate(self, value: float) -> None:
    """Takes effect on the device in stream order: a graph of a captured step follows it."""
    with _lib.device_guard(self._index):
      self._lr.fill_(float(value))

  @property
  def grad_norm(self) -> torch.Tensor:
    """The last step's global norm (of the scaled gradients, before the clip), a device scalar;
    0 without clipping."""
    return self._scalars[0]

  @property
  def count(self) -> int:
    return int(self._count.item())

  # -- moments and state ----------------------------------------------------------
  def moments(self, dtype: torch.dtype = torch.float32):
    """(m, v) as numbers, flat in the state's layout: params[i] at offsets[i]."""
    code = _lib.dtype_code(dtype)
    if code is None:
      raise TypeError('moments are float32, bfloat16 or float16, not %s' % dtype)
    if self.config.state_bits == 32:
      return self.m.to(dtype), self.v.to(dtype)
    with _lib.device_guard(self._index):
      m = _lib.new_output(self.state_size, dtype, self.device)
      v = _lib.new_output(self.state_size, dtype, self.device)
      _lib.check(self._lib.dz_adamw_moments(
          self.m.data_ptr(), self.v.data_ptr(), self.m_scale.data_ptr(), self.v_scale.data_ptr(),
          self.state_size, code, m.data_ptr(), v.data_ptr(), _lib.stream_ptr(self._index)),
                 'dz_adamw_moments')
    return m, v

  def _state_tensors(self):
    named = (('m', self.m), ('v', self.v), ('m_scale', self.m_scale), ('v_scale', self.v_scale),
             ('master', self.master))
    return [(k, t) for k, t in named if t is not None]

  def get_state(self) -> dict:
    """Copies on the host, for `set_state` of an optimizer of the same tensors."""
    return {'count': self.count, **{k: t.cpu() for k, t in self._state_tensors()}}

  def set_state(self, state: typing.Mapping[str, typing.Any]) -> None:
    """Restores `get_state`'s dict (tensors on any device).  Without 'master', the master weights
    stay what they are."""
    known = dict(self._state_tensors())
    names = set(state) - {'count'}
    if not set(known) - {'master'} <= names <= set(known) or 'count' not in state:
      raise ValueError('state has %s, this optimizer %s and count' % (sorted(state), sorted(known)))
    for k in sorted(names):
      t, want = state[k], known[k]
      if t.dtype != want.dtype or t.shape != want.shape:
        raise ValueError('state %r must be %s %s, got %s %s' % (
            k, want.dtype, tuple(want.shape), t.dtype, tuple(t.shape)))
    for k in sorted(names):
      known[k].copy_(state[k])
    self._count.fill_(int(state['count']))
