"""CPU half of the policy-training operators: the oracle against torch's autograd and types, the C
entries' refusals and workspace sizes (host code), and the refusal to run without a GPU."""

import ctypes

import numpy as np
import pytest
import torch

from dqn_zoo_amd import _lib
from dqn_zoo_amd import build as dz_build
from oracle import policy_oracle as po


@pytest.fixture(scope='module')
def lib():
  dz_build.build()
  return _lib.load()


# ---- the oracle -------------------------------------------------------------
def test_oracle_policy_loss_gradient_is_autograds():
  g = torch.Generator().manual_seed(0)
  rows, classes = 12, 9
  x = (2 * torch.randn(rows, classes, generator=g, dtype=torch.float64)).requires_grad_()
  actions = torch.randint(0, classes, (rows,), generator=g)
  adv, dold, dref = (torch.randn(rows, generator=g, dtype=torch.float64) for _ in range(3))
  lp = torch.log_softmax(x, -1)
  logp = lp.gather(1, actions[:, None])[:, 0]
  old, ref = (logp + 0.5 * dold).detach(), (logp + 0.3 * dref).detach()
  w = torch.rand(rows, generator=g, dtype=torch.float64)
  w[3] = 0
  rho = torch.exp(logp - old)
  d = ref - logp
  value = -torch.minimum(rho * adv, rho.clamp(0.8, 1.3) * adv) + 0.2 * (torch.exp(d) - d - 1) + \
      0.05 * (lp.exp() * lp).sum(-1)
  loss = (w * value).sum() / w.sum()
  loss.backward()
  got = po.policy_loss(x.detach().numpy(), actions.numpy(), adv.numpy(), old.numpy(), ref.numpy(), w.numpy(),
                       clip_low=0.2, clip_high=0.3, kl_coef=0.2, entropy_coef=0.05)
  assert abs(got[0] - float(loss.detach())) < 1e-12
  np.testing.assert_allclose(got[3], x.grad.numpy(), atol=1e-13)


@pytest.mark.parametrize('activation', ['none', 'relu', 'gelu', 'silu'])
def test_oracle_linear_gradients_are_autograds(activation):
  g = torch.Generator().manual_seed(1)
  x, w, b, r, dy = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
                    for s in ((5, 7), (7, 4), (4,), (5, 4), (5, 4)))
  z = x @ w + b
  f = {'none': lambda t: t, 'relu': torch.relu, 'gelu': torch.nn.functional.gelu,
       'silu': torch.nn.functional.silu}[activation]
  y = f(z) + r
  y.backward(dy.detach())
  n = lambda t: t.detach().numpy()
  want_y, want_z = po.linear(n(x), n(w), n(b), activation, n(r))
  np.testing.assert_allclose(want_y, n(y), atol=1e-14)
  dx, dw, db = po.linear_backward(n(dy), n(x), n(w), activation, want_z)
  for got, t in ((dx, x), (dw, w), (db, b)):
    np.testing.assert_allclose(got, t.grad.numpy(), atol=1e-13)


def test_oracle_adamw_is_torchs():
  g = torch.Generator().manual_seed(2)
  p = torch.randn(50, generator=g, dtype=torch.float64).requires_grad_()
  opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
  q, m, v = p.detach().numpy().copy(), np.zeros(50), np.zeros(50)
  for step in range(1, 6):
    p.grad = torch.randn(50, generator=g, dtype=torch.float64)
    opt.step()
    q, m, v = po.adamw(q, p.grad.numpy(), m, v, step, 1e-2, 0.9, 0.99, 1e-8, 0.1)
    np.testing.assert_allclose(q, p.detach().numpy(), atol=1e-14)


def test_eight_bit_formats():
  codes = np.arange(256, dtype=np.uint8)
  e4m3 = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()
  held = (codes & 127) != 127           # (NaN: never stored)
  np.testing.assert_array_equal(po.decode_e4m3(codes)[held], e4m3[held])
  v = po.decode_e5m3(codes)
  assert v[0] == 0 and v[255] == 1.875 and (np.diff(v) > 0).all()
  assert v[1] == 2.0 ** -33 and v[8] == 2.0 ** -30
  # 16-bit draws: each half of the range about as often
  m, n = po.adamw_noise(1, 5, np.arange(100000))
  for draw in (m, n):
    assert draw.min() >= 0 and draw.max() < 65536 and abs((draw < 32768).mean() - 0.5) < 0.01
  assert (po.adamw_noise(1, 6, np.arange(1000))[0] != m[:1000]).mean() > 0.99


# ---- refusals of the C entries: host code, nothing is launched --------------------
def _linear_args(m, k, n, **more):
  a = _lib.LinearArgs()
  a.dtype, a.activation, a.m, a.k, a.n = _lib.BF16, 0, m, k, n
  for key, value in more.items():
    setattr(a, key, value)
  return a


def test_linear_workspace_sizes(lib):
  need = ctypes.c_int64()
  def size(a, backward=0):
    assert lib.dz_linear_workspace(ctypes.byref(a), backward, ctypes.byref(need)) == 0
    return need.value
  aligned = dict(x=4096, ldx=512, w=8192, ldw=768)
  # operands that can be read where they lie take nothing, others their copies
  assert size(_linear_args(4096, 512, 768, **aligned)) == 0
  copies = (4096 * 512 + 512 * 768) * 2
  assert size(_linear_args(4096, 512, 768)) == copies
  for key, value in (('x', 4098), ('ldx', 513), ('ldx', (1 << 23) + 8)):
    assert size(_linear_args(4096, 512, 768, **{**aligned, key: value})) == 4096 * 512 * 2
  for key, value in (('w', 8194), ('ldw', 769)):
    assert size(_linear_args(4096, 512, 768, **{**aligned, key: value})) == 512 * 768 * 2
  # sizes alone cover every call of these sizes
  for m, k, n in ((1, 3136, 512), (300, 264, 520), (8192, 4096, 4096), (7, 9, 11)):
    for act in range(4):
      for t in (0, 1):
        whole = size(_linear_args(m, k, n, activation=act, w_transposed=t), 1)
        at = dict(x=4096, ldx=k, w=8192, ldw=k if t else n, dy=16, lddy=n, preact=32, ldz=n, dx=64, lddx=k,
                  dw=128, lddw=k if t else n, db=256)
        for drop in ((), ('dx',), ('dw',), ('db',), ('dx', 'dw')):
          args = {**at, **{d: None for d in drop}}
          assert size(_linear_args(m, k, n, activation=act, w_transposed=t, **args), 1) <= whole


def test_c_entries_refuse(lib):
  bad = _lib.DZ_ERR_INVALID_ARG
  need = ctypes.c_int64()
  for a in (_linear_args(0, 8, 8), _linear_args(8, 0, 8), _linear_args(8, 8, -1), _linear_args(1 << 31, 8, 8),
            _linear_args(8, (1 << 23) + 1, 8), _linear_args(8, 8, 8, dtype=3), _linear_args(8, 8, 8, activation=4)):
    assert lib.dz_linear_workspace(ctypes.byref(a), 0, ctypes.byref(need)) == bad
    assert lib.dz_linear(ctypes.byref(a), None) == bad
    assert lib.dz_linear_backward(ctypes.byref(a), None) == bad
  ok = dict(x=4096, ldx=8, w=4096, ldw=8, y=4096, ldy=8)
  for change in (dict(x=None), dict(w=None), dict(y=None), dict(ldx=7), dict(ldw=7), dict(ldy=7),
                 dict(residual=4096, ldr=7), dict(preact=4096, ldz=7)):
    assert lib.dz_linear(ctypes.byref(_linear_args(8, 8, 8, **{**ok, **change})), None) == bad, change
  # (above 32 rows an operand that cannot be read where it lies needs a workspace for its copy)
  assert lib.dz_linear(ctypes.byref(_linear_args(64, 8, 8, **{**ok, 'x': 4098})), None) == bad
  back = dict(x=4096, ldx=8, w=4096, ldw=8, dy=4096, lddy=8, dx=4096, lddx=8, dw=4096, lddw=8)
  for change in (dict(dy=None), dict(lddy=7), dict(lddx=7), dict(lddw=7), dict(activation=1), dict(x=None),
                 dict(w=None), dict(dx=None, dw=None)):
    assert lib.dz_linear_backward(ctypes.byref(_linear_args(8, 8, 8, **{**back, **change})), None) == bad, change

  def loss(**change):
    a = _lib.PolicyLossArgs()
    at = dict(dtype=0, rows=4, classes=6, logits=4096, ld=6, actions=4096, advantages=4096, old_logp=4096,
              logp=4096, entropy=4096, loss=4096, dlogits=4096, ldg=6)
    for key, value in {**at, **change}.items():
      setattr(a, key, value)
    return lib.dz_policy_loss(ctypes.byref(a), None)
  for change in (dict(dtype=5), dict(rows=0), dict(classes=0), dict(rows=1 << 31), dict(classes=1 << 30),
                 dict(logits=None), dict(actions=None), dict(advantages=None), dict(old_logp=None), dict(logp=None),
                 dict(entropy=None), dict(loss=None), dict(ld=5), dict(ldg=5), dict(clip_low=-0.1),
                 dict(clip_high=-0.1), dict(normalizer=-1.0), dict(ws=4100),
                 dict(classes=300, ld=300, ldg=300),   # needs a workspace
                 dict(classes=300, ld=300, ldg=300, rows=1 << 26, ws=4096, ws_bytes=1 << 40),   # more threads than
                 dict(classes=5000, ld=5000, ldg=5000, rows=1 << 24, ws=4096, ws_bytes=1 << 40)):   # a launch has
    assert loss(**change) == bad, change

  def adamw(**change):
    a = _lib.AdamWArgs()
    at = dict(param_dtype=1, grad_dtype=1, state_bits=8, num_chunks=1, tensors=16, chunks=16, grads=16, m=16, v=16,
              m_scale=16, v_scale=16, count=16, lr=16, scalars=16, partials=16, b1=0.9, b2=0.99, eps=1e-8)
    for key, value in {**at, **change}.items():
      setattr(a, key, value)
    return lib.dz_adamw_step(ctypes.byref(a), None)
  for change in (dict(param_dtype=9), dict(grad_dtype=2), dict(state_bits=16), dict(num_chunks=0), dict(tensors=None),
                 dict(m_scale=None), dict(param_dtype=0, grad_dtype=0, master=16), dict(max_norm=1.0, partials=None),
                 dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(lr=None)):
    assert adamw(**change) == bad, change
  assert lib.dz_adamw_moments(16, 16, 16, 16, 255, 0, 16, 16, None) == bad
  pointers = (ctypes.c_void_p * 2)(16, None)
  assert lib.dz_adamw_bind(pointers, 2, 16, None) == bad


def test_no_cpu_fallback():
  from dqn_zoo_amd import adamw, linear, policy_loss
  x = torch.zeros(4, 6)
  v = torch.zeros(4)
  with pytest.raises(_lib.HipLibraryError, match='no CPU fallback'):
    linear.linear(x, x.t())
  with pytest.raises(_lib.HipLibraryError, match='no CPU fallback'):
    linear.linear_backward(x, x, x)
  with pytest.raises(_lib.HipLibraryError, match='no CPU fallback'):
    policy_loss.policy_loss(x, v.long(), v, v)
  with pytest.raises(_lib.HipLibraryError, match='no CPU fallback'):
    adamw.AdamW([x], adamw.AdamWConfig())
  with pytest.raises(TypeError, match='dtype must be'):
    linear.workspace_bytes(4, 6, 8, torch.float64)
  with pytest.raises(ValueError, match='activation'):
    linear.workspace_bytes(4, 6, 8, torch.float32, activation='tanh')
  with pytest.raises(TypeError, match='logits must be'):
    policy_loss.workspace_bytes(4, 6, torch.float64)
