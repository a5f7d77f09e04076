"""A dense layer with bias, activation and residual, and its backward pass
(include/dqnzoo_hip.h: dz_linear, dz_linear_backward; csrc/dz_linear.hip).

The learners' networks (`networks.RainbowNetwork`, `DenseNetwork`, `IqnNetwork`) have their layers
inside their fused float32 steps.  `linear` and `linear_backward` are the layer for everything
else: any sizes from one row on, float32, bfloat16 or float16, strided rows, the weight as (in, out)
-- the networks' layout -- or as the transposed view of (out, in).

    y, z = linear.linear(x, w, b, activation='gelu', save_preact=True)
    dx, dw, db = linear.linear_backward(dy, x, w, activation='gelu', preact=z)

Plain buffers in and out, no autograd.  Work is enqueued on the current stream of the tensors'
device; nothing synchronises.
"""

import ctypes
import typing

import torch

from dqn_zoo_amd import _lib

ACTIVATIONS = {'none': 0, 'relu': 1, 'gelu': 2, 'silu': 3}


def _activation(name):
  code = ACTIVATIONS.get(name)
  if code is None:
    raise ValueError('activation must be one of %s, got %r' % (sorted(ACTIVATIONS), name))
  return code


def _type(name, t, dtype, device):
  if not isinstance(t, torch.Tensor) or t.dtype != dtype:
    raise TypeError('%s must be a %s tensor, got %s' % (
        name, dtype, getattr(t, 'dtype', type(t).__name__)))
  if t.get_device() != device:
    raise ValueError('%s is on another device than x' % name)


def _rows(name, t, shape, dtype, device):
  """Row pitch of a [rows, cols] matrix with adjacent elements in rows that do not overlap."""
  _type(name, t, dtype, device)
  if t.shape != shape:
    raise ValueError('%s must have shape %s, got %s' % (name, tuple(shape), tuple(t.shape)))
  ld, inner = t.stride()
  if (inner != 1 and shape[1] > 1) or (ld < shape[1] and shape[0] > 1):
    raise ValueError('%s must have adjacent elements in rows that do not overlap, got strides %s' %
                     (name, t.stride()))
  return ld if shape[0] > 1 else max(ld, shape[1])


def _weight(name, t, shape, dtype, device):
  """(pitch, transposed) of a [k, n] weight stored in rows of k or of n."""
  _type(name, t, dtype, device)
  if t.shape != shape:
    raise ValueError('%s must have shape %s, got %s' % (name, tuple(shape), tuple(t.shape)))
  (k, n), (sk, sn) = shape, t.stride()
  if (sn == 1 or n == 1) and (sk >= n or k == 1):
    return (sk if k > 1 else max(sk, n)), 0
  if (sk == 1 or k == 1) and (sn >= k or n == 1):
    return (sn if n > 1 else max(sn, k)), 1
  raise ValueError('%s must be stored in rows, as (in, out) or transposed, got strides %s' % (name, t.stride()))


def _vector(name, t, n, dtype, device):
  """Whether the [n] vector is float32 (next to `dtype`)."""
  if not isinstance(t, torch.Tensor) or t.dtype not in (dtype, torch.float32):
    raise TypeError('%s must be a %s or float32 tensor, got %s' % (
        name, dtype, getattr(t, 'dtype', type(t).__name__)))
  if t.shape != (n,) or not t.is_contiguous():
    raise ValueError('%s must be contiguous with shape (%d,), got %s' % (name, n, tuple(t.shape)))
  if t.get_device() != device:
    raise ValueError('%s is on another device than x' % name)
  return int(t.dtype == torch.float32)


def _apart(name, output, taken):
  """Outputs may not lie on what the kernels still read, or on each other; `output` joins `taken`,
  a list of (name, first byte, last byte)."""
  a, b = _lib.span(output)
  for other, c, d in taken:
    if a < d and c < b:
      raise ValueError('%s shares memory with %s' % (name, other))
  taken.append((name, a, b))


def _spans(**tensors):
  return [(n, *_lib.span(t)) for n, t in tensors.items() if t is not None]


def _start(x, w):
  """The argument block with what the two passes share; (args, device, dtype, m, k, n)."""
  device = _lib.gpu_index('x', x)
  dtype = x.dtype
  code = _lib.dtype_code(dtype)
  if code is None:
    raise TypeError('x must be float32, bfloat16 or float16, got %s' % dtype)
  if x.dim() != 2 or not x.numel():
    raise ValueError('x must be [rows, in] and not empty, got %s' % (tuple(x.shape),))
  if not isinstance(w, torch.Tensor) or w.dim() != 2 or not w.numel():
    raise ValueError('w must be [in, out] and not empty')
  (m, k), n = x.shape, w.shape[1]
  a = _lib.LinearArgs()
  a.dtype, a.m, a.k, a.n = code, m, k, n
  a.ldx = _rows('x', x, (m, k), dtype, device)
  a.ldw, a.w_transposed = _weight('w', w, (k, n), dtype, device)
  a.x, a.w = x.data_ptr(), w.data_ptr()
  return a, device, dtype, m, k, n


def _workspace(lib, a, backward, device, workspace):
  need = ctypes.c_int64()
  _lib.check(lib.dz_linear_workspace(ctypes.byref(a), backward, ctypes.byref(need)),
             'dz_linear_workspace')
  if not need.value and workspace is None:
    return None
  ws = _lib.scratch(need.value, device, workspace)
  a.ws, a.ws_bytes = ws.data_ptr(), need.value
  return ws


def workspace_bytes(rows: int, inputs: int, outputs: int, dtype: torch.dtype, *,
                    backward: bool = False, activation: str = 'none',
                    transposed: bool = False) -> int:
  """Bytes of `linear`'s (or `linear_backward`'s) workspace= for these sizes; may be 0.
  `transposed`: the weight is the transposed view of (out, in)."""
  code = _lib.dtype_code(dtype)
  if code is None:
    raise TypeError('dtype must be float32, bfloat16 or float16, got %s' % dtype)
  a = _lib.LinearArgs()
  a.dtype, a.activation, a.m, a.k, a.n = code, _activation(activation), rows, inputs, outputs
  a.w_transposed = int(transposed)
  need = ctypes.c_int64()
  _lib.check(_lib.load().dz_linear_workspace(ctypes.byref(a), int(backward), ctypes.byref(need)),
             'dz_linear_workspace')
  return need.value


def linear(x: torch.Tensor, w: torch.Tensor, b: typing.Optional[torch.Tensor] = None, *,
           activation: str = 'none', residual: typing.Optional[torch.Tensor] = None,
           save_preact: bool = False, out: typing.Optional[torch.Tensor] = None,
           preact: typing.Optional[torch.Tensor] = None,
           workspace: typing.Optional[torch.Tensor] = None):
  """act(x w + b) + residual, and x w + b with it where `save_preact`.

  x [rows, in] in rows of any pitch; w [in, out], stored in rows of either index; b [out] of x's
  type or float32; residual [rows, out].  Activations: none, relu, gelu (erf), silu.  `out`,
  `preact`, `workspace` (uint8, `workspace_bytes`): the caller's buffers, needed inside
  `_lib.capture_graph`; `out` may be `residual` itself.
  """
  a, device, dtype, m, _, n = _start(x, w)
  a.activation = _activation(activation)
  if b is not None:
    a.bias_f32 = _vector('b', b, n, dtype, device)
    a.bias = b.data_ptr()
  if residual is not None:
    a.ldr = _rows('residual', residual, (m, n), dtype, device)
    a.residual = residual.data_ptr()
  if preact is not None and not save_preact:
    raise ValueError('preact= is a buffer for save_preact=True')
  with _lib.device_guard(device):
    given = out is not None or preact is not None
    taken = _spans(x=x, w=w, b=b) if given else None
    if out is None:
      out = _lib.new_like(x, (m, n))
      a.ldy = n
    else:
      a.ldy = _rows('out', out, (m, n), dtype, device)
      same = residual is not None and residual.data_ptr() == out.data_ptr() and a.ldr == a.ldy
      if residual is not None and not same:
        taken += _spans(residual=residual)
      _apart('out', out, taken)
    if save_preact:
      if preact is None:
        preact = _lib.new_like(x, (m, n))
        a.ldz = n
      else:
        a.ldz = _rows('preact', preact, (m, n), dtype, device)
        _apart('preact', preact, taken + _spans(residual=residual))
      a.preact = preact.data_ptr()
    a.y = out.data_ptr()
    lib = _lib.load()
    ws = _workspace(lib, a, 0, x.device, workspace)  # pylint: disable=unused-variable
    _lib.check(lib.dz_linear(ctypes.byref(a), _lib.stream_ptr(device)), 'dz_linear')
  return (out, preact) if save_preact else out


def linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *,
                    activation: str = 'none', preact: typing.Optional[torch.Tensor] = None,
                    need: typing.Sequence[bool] = (True, True, True),
                    dx: typing.Optional[torch.Tensor] = None,
                    dw: typing.Optional[torch.Tensor] = None,
                    db: typing.Optional[torch.Tensor] = None,
                    workspace: typing.Optional[torch.Tensor] = None):
  """(dx, dw, db) of `linear`; the residual's gradient is dy itself.

  `preact`: what `linear` saved (not needed for activation 'none').  `need`: which of the three
  are computed; None stands for the others.  dx, dw, db: the caller's buffers; dw and db may both
  be float32 (sums of gradients, or an optimizer's type) where x is not.  A new dw is stored as w
  is.  `workspace` as for `linear`.
  """
  a, device, dtype, m, k, n = _start(x, w)
  a.activation = _activation(activation)
  a.lddy = _rows('dy', dy, (m, n), dtype, device)
  a.dy = dy.data_ptr()
  if a.activation:
    if preact is None:
      raise ValueError('activation %r needs preact' % activation)
    a.ldz = _rows('preact', preact, (m, n), dtype, device)
    a.preact = preact.data_ptr()
  else:
    preact = None
  if len(need) != 3 or not any(need):
    raise ValueError('need names at least one of dx, dw, db, got %r' % (need,))
  for name, wanted, t in zip(('dx', 'dw', 'db'), need, (dx, dw, db)):
    if t is not None and not wanted:
      raise ValueError('%s= is given but not needed' % name)
  given = dx is not None or dw is not None or db is not None
  taken = _spans(dy=dy, x=x, w=w, preact=preact) if given else None
  with _lib.device_guard(device):
    if need[0]:
      if dx is None:
        dx = _lib.new_like(x, (m, k))
        a.lddx = k
      else:
        a.lddx = _rows('dx', dx, (m, k), dtype, device)
        _apart('dx', dx, taken)
      a.dx = dx.data_ptr()
    grads = [t for t in (dw, db) if t is not None]
    kind = grads[0].dtype if grads else dtype
    if any(g.dtype != kind for g in grads) or kind not in (dtype, torch.float32):
      raise TypeError('dw and db must both be %s or both float32' % dtype)
    a.grads_f32 = int(kind == torch.float32)
    if need[1]:
      if dw is None:
        stored = (n, k) if a.w_transposed else (k, n)
        dw = _lib.new_like(w, stored) if kind == dtype else _lib.new_output(stored, kind, x.device)
        a.lddw = k if a.w_transposed else n
        dw = dw.t() if a.w_transposed else dw
      else:
        a.lddw = _rows('dw, stored as w is,', dw.t() if a.w_transposed else dw,
                       (n, k) if a.w_transposed else (k, n), kind, device)
        _apart('dw', dw, taken)
      a.dw = dw.data_ptr()
    if need[2]:
      if db is None:
        db = _lib.new_like(w, n) if kind == dtype else _lib.new_output((n,), kind, x.device)
      else:
        _vector('db', db, n, dtype, device)
        _apart('db', db, taken)
      a.db = db.data_ptr()
    lib = _lib.load()
    ws = _workspace(lib, a, 1, x.device, workspace)  # pylint: disable=unused-variable
    _lib.check(lib.dz_linear_backward(ctypes.byref(a), _lib.stream_ptr(device)),
               'dz_linear_backward')
  return dx, dw, db
