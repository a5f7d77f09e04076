"""Clipped policy loss with a KL term and an entropy bonus, with its gradient
(include/dqnzoo_hip.h: dz_policy_loss; csrc/dz_policy_loss.hip).

The Q-learners' losses live inside their fused steps (`learner.RainbowLearner`, `DenseLearner`,
`IqnLearner`).  `policy_loss` is the loss of a policy over actions or tokens, on logits of any
number of classes: one call gives the loss, each row's log-probability and entropy, and the
gradient with respect to the logits, which `linear.linear_backward` takes from there.

Work is enqueued on the current stream of the logits' device; nothing synchronises.
"""

import ctypes
import typing

import torch

from dqn_zoo_amd import _lib


class PolicyLossConfig(typing.NamedTuple):
  """-min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(d) - d - 1)
  - entropy_coef H with rho = exp(logp - old_logp), d = ref_logp - logp."""
  clip_low: float = 0.2
  clip_high: float = 0.2
  kl_coef: float = 0.0
  entropy_coef: float = 0.0


class PolicyLossOutputs(typing.NamedTuple):
  loss: torch.Tensor                       # float32 scalar
  logp: torch.Tensor                       # float32 [rows], of the actions taken
  entropy: torch.Tensor                    # float32 [rows]
  dlogits: typing.Optional[torch.Tensor]   # like the logits


def workspace_bytes(rows: int, classes: int, dtype: torch.dtype) -> int:
  """Bytes of `policy_loss`'s workspace= for these sizes; may be 0."""
  code = _lib.dtype_code(dtype)
  if code is None:
    raise TypeError('logits must be float32, bfloat16 or float16, got %s' % dtype)
  return _workspace_bytes(code, rows, classes)


def _workspace_bytes(code, rows, classes):
  n = ctypes.c_int64()
  _lib.check(_lib.load().dz_policy_loss_workspace(code, rows, classes, ctypes.byref(n)),
             'dz_policy_loss_workspace')
  return n.value


def _row_vector(name, t, rows, dtype, device):
  if t is None:
    return None
  if not isinstance(t, torch.Tensor) or t.dtype != dtype:
    raise TypeError('%s must be a %s tensor, got %s' % (name, dtype, getattr(t, 'dtype', type(t).__name__)))
  if t.shape != (rows,) or not t.is_contiguous():
    raise ValueError('%s must be contiguous with shape (%d,), got %s' % (name, rows, tuple(t.shape)))
  if t.get_device() != device:
    raise ValueError('%s is on another device than the logits' % name)
  return t.data_ptr()


def _matrix(name, t, shape, dtype, device):
  if not isinstance(t, torch.Tensor) or t.dtype != dtype:
    raise TypeError('%s must be a %s tensor, got %s' % (name, dtype, getattr(t, 'dtype', type(t).__name__)))
  if t.shape != shape:
    raise ValueError('%s must have shape %s, got %s' % (name, tuple(shape), tuple(t.shape)))
  if t.get_device() != device:
    raise ValueError('%s is on another device than the logits' % name)
  rows, cols = shape
  ld, inner = t.stride()
  if (inner != 1 and cols > 1) or (ld < cols and rows > 1):
    raise ValueError('%s must have adjacent elements in rows that do not overlap, got strides %s' %
                     (name, t.stride()))
  return max(ld, cols)


def _check_apart(out, logits, **inputs):
  """A row's outputs may be written while another workgroup still reads that row's inputs."""
  taken = [(n, *_lib.span(t)) for n, t in inputs.items() if t is not None]
  for name, t in zip(out._fields, out):
    if t is None:
      continue
    a, b = _lib.span(t)
    if not (name == 'dlogits' and logits.data_ptr() == a and logits.stride() == t.stride()):
      c, d = _lib.span(logits)
      if a < d and c < b:
        raise ValueError('out.%s overlaps logits' % name)
    for other, c, d in taken:
      if a < d and c < b:
        raise ValueError('out.%s overlaps %s' % (name, other))
    taken.append((name, a, b))


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, advantages: torch.Tensor,
                old_logp: torch.Tensor, ref_logp: typing.Optional[torch.Tensor] = None,
                weights: typing.Optional[torch.Tensor] = None, *,
                config: PolicyLossConfig = PolicyLossConfig(),
                normalizer: typing.Optional[float] = None, grad_scale: float = 1.0,
                with_gradient: bool = True, out: typing.Optional[PolicyLossOutputs] = None,
                status: typing.Optional[torch.Tensor] = None,
                workspace: typing.Optional[torch.Tensor] = None) -> PolicyLossOutputs:
  """Loss, log-probabilities, entropies and d loss / d logits of `logits` [rows, classes].

  actions int64 [rows]; advantages, old_logp, ref_logp, weights float32 [rows].  `weights`: 0 for
  padding (the row is not read, its gradient is 0), any other number otherwise.  `normalizer`
  divides the sum instead of the weights' sum (e.g. the tokens of all ranks or accumulated
  batches).  `grad_scale` multiplies the gradient only (a loss scale).  ref_logp is needed where
  config.kl_coef is not 0.

  Masked classes have a logit of -inf (or the type's lowest value).  A row with nothing but -inf is
  NaN, as is one whose action is not a class; the latter sets ST_BAD_INDEX in `status` (int32 [1])
  if given.  `out` and `workspace` (uint8, `workspace_bytes`): the caller's buffers, needed inside
  `_lib.capture_graph`; out.dlogits may be `logits` itself.
  """
  device = _lib.gpu_index('logits', logits)
  code = _lib.dtype_code(logits.dtype)
  if code is None:
    raise TypeError('logits must be float32, bfloat16 or float16, got %s' % logits.dtype)
  if logits.dim() != 2 or not logits.numel():
    raise ValueError('logits must be [rows, classes] and not empty, got %s' % (tuple(logits.shape),))
  shape = logits.shape
  rows, classes = shape
  a = _lib.PolicyLossArgs()
  a.dtype, a.rows, a.classes = code, rows, classes
  a.ld = _matrix('logits', logits, shape, logits.dtype, device)
  a.logits = logits.data_ptr()
  f32 = torch.float32
  if actions is None or advantages is None or old_logp is None:
    raise TypeError('actions, advantages and old_logp are needed')
  a.actions = _row_vector('actions', actions, rows, torch.int64, device)
  a.advantages = _row_vector('advantages', advantages, rows, f32, device)
  a.old_logp = _row_vector('old_logp', old_logp, rows, f32, device)
  a.ref_logp = _row_vector('ref_logp', ref_logp, rows, f32, device)
  a.weights = _row_vector('weights', weights, rows, f32, device)
  clip_low, clip_high, kl_coef, entropy_coef = config
  if not (clip_low >= 0 and clip_high >= 0):
    raise ValueError('clip_low and clip_high must not be negative, got %s' % (config,))
  if kl_coef and ref_logp is None:
    raise ValueError('kl_coef %g needs ref_logp' % kl_coef)
  if normalizer is not None and not 0 < normalizer < float('inf'):
    raise ValueError('normalizer must be positive and finite, got %r' % (normalizer,))
  a.clip_low, a.clip_high, a.kl_coef, a.entropy_coef = clip_low, clip_high, kl_coef, entropy_coef
  a.normalizer = normalizer or 0.0
  a.grad_scale = grad_scale
  if status is not None:
    a.status = _row_vector('status', status, 1, torch.int32, device)
  with _lib.device_guard(device):
    if out is None:
      logp, entropy = _lib.new_like(advantages, (2, rows)).unbind()
      out = PolicyLossOutputs(_lib.new_like(advantages, ()), logp, entropy,
                              _lib.new_like(logits, shape) if with_gradient else None)
      a.ldg = classes
    else:
      if _row_vector('out.loss', out.loss.view(1), 1, f32, device) is None or (
          out.dlogits is None) == with_gradient:
        raise ValueError('out.dlogits must be given exactly if with_gradient')
      _row_vector('out.logp', out.logp, rows, f32, device)
      _row_vector('out.entropy', out.entropy, rows, f32, device)
      if with_gradient:
        a.ldg = _matrix('out.dlogits', out.dlogits, shape, logits.dtype, device)
      _check_apart(out, logits=logits, actions=actions, advantages=advantages, old_logp=old_logp,
                   ref_logp=ref_logp, weights=weights, status=status)
    a.loss, a.logp, a.entropy = out.loss.data_ptr(), out.logp.data_ptr(), out.entropy.data_ptr()
    if with_gradient:
      a.dlogits = out.dlogits.data_ptr()
    lib = _lib.load()
    need = _workspace_bytes(code, rows, classes)
    if need or workspace is not None:
      ws = _lib.scratch(need, logits.device, workspace)
      a.ws, a.ws_bytes = ws.data_ptr(), need
    _lib.check(lib.dz_policy_loss(ctypes.byref(a), _lib.stream_ptr(device)), 'dz_policy_loss')
  return out
