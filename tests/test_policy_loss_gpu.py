"""The clipped policy loss and its gradient against the float64 oracle (oracle/policy_oracle.py)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import policy_oracle as po

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}


def _np(t):
  return None if t is None else t.detach().double().cpu().numpy()


def _inputs(rows, classes, dtype, seed, extra=0, masked=0.0, ref=True, padded=0.0):
  g = torch.Generator().manual_seed(seed)
  logits = torch.randn(rows, classes + extra, generator=g) * 2
  actions = torch.randint(0, classes, (rows,), generator=g)
  if masked:
    off = torch.rand(rows, classes + extra, generator=g) < masked
    off[torch.arange(rows), actions] = False
    logits[off] = -float('inf')
  logits = logits.to(dtype)
  x = logits[:, :classes].double()
  logp = torch.log_softmax(x, -1)[torch.arange(rows), actions]
  rnd = lambda s: s * torch.randn(rows, generator=g)
  weights = None
  if padded:
    weights = (torch.rand(rows, generator=g) >= padded).float() * torch.rand(rows, generator=g)
    weights[0] = 0.7
  return dict(logits=logits.cuda()[:, :classes], actions=actions.cuda(), advantages=rnd(1.0).cuda(),
              old_logp=(logp.float() + rnd(0.3)).cuda(),
              ref_logp=(logp.float() + rnd(0.3)).cuda() if ref else None,
              weights=None if weights is None else weights.cuda())


def _oracle(i, cfg, **more):
  return po.policy_loss(_np(i['logits']), i['actions'].cpu().numpy(), _np(i['advantages']),
                        _np(i['old_logp']), _np(i['ref_logp']), _np(i['weights']),
                        clip_low=cfg[0], clip_high=cfg[1], kl_coef=cfg[2], entropy_coef=cfg[3], **more)


# Roundings in units of U32 (half a float32 step):
#  * log p: u carries the rounding of the difference and of the product (|x| <= 12: the logits are
#    of deviation 2), up to 2 * 35 in base 2; S is a sum of positive terms in at most 12 + 6 + 16 +
#    10 levels, each e with u's error; the exponential and logarithm are good to 2 steps:
#    70 + 50 + 8 < 160 absolute, in natural units;
#  * H: the mean of u, twice as much;
#  * rho, exp(d) - 1: log p's error absolute in the exponent + 2 old_logp's scale: 200 relative;
#  * gradient elements: p's relative error 160, k1 u + k0 relative to the terms' sizes: 600 covers it.
LOGP, ENT, GRAD = 160, 320, 600


def _check(i, out, cfg, dtype, **more):
  loss, logp, ent, grad = _oracle(i, cfg, **more)
  w = np.ones(len(logp)) if i['weights'] is None else _np(i['weights'])
  norm = more.get('normalizer') or w.sum()
  s = np.abs(w) / norm
  assert np.abs(_np(out.logp) - logp).max() <= LOGP * U32 + U32 * np.abs(logp).max()
  assert np.abs(_np(out.entropy) - ent).max() <= ENT * U32 + U32 * np.abs(ent).max()
  adv = np.abs(_np(i['advantages']))
  rho = np.exp(logp - _np(i['old_logp']))
  kl = cfg[2] * np.exp(np.abs(_np(i['ref_logp']) - logp)) if i['ref_logp'] is not None else 0.0
  size = rho * adv + kl + cfg[3] * (np.abs(ent) + 30)   # of the terms of a row's value and slope
  assert abs(float(out.loss) - loss) <= GRAD * U32 * (s * size).sum() + U32 * abs(loss)
  if out.dlogits is None:
    return
  x = _np(i['logits'])
  with np.errstate(invalid='ignore'):
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
  p[np.arange(len(p)), i['actions'].cpu().numpy()] = 1.0
  tol = GRAD * U32 * more.get('grad_scale', 1.0) * (s * size)[:, None] * p
  got = _np(out.dlogits)
  bad = np.abs(got - grad) > tol + HALF[dtype] * (np.abs(grad) + tol) + TINY[dtype]
  bad &= (w != 0)[:, None]
  assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5], got[bad][:5], grad[bad][:5])
  assert (got[w == 0] == 0).all()


SIZES = [(1, 1), (1, 2), (5, 4), (32, 18), (1000, 18), (7, 64), (3, 255), (70, 256), (2, 257), (9, 511),
         (6, 513), (5, 1025), (3, 2049), (2, 4097), (130, 8193), (3, 16385), (129, 33000), (2, 70001)]


@pytest.mark.parametrize('rows,classes', SIZES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_formula(rows, classes, dtype):
  from dqn_zoo_amd import policy_loss as pl
  many = rows * classes > 300000
  i = _inputs(rows, classes, dtype, rows + classes, extra=3 if rows % 2 else 0,
              masked=0.3 if classes > 2 and not many else 0.0, padded=0.3 if rows > 4 else 0.0)
  cfg = pl.PolicyLossConfig(0.2, 0.28, 0.1, 0.02)
  _check(i, pl.policy_loss(**i, config=cfg), cfg, dtype)


@pytest.mark.parametrize('rows,classes', [(140, 140000), (1, 140000), (3, 1)])
def test_rows_longer_than_a_workgroup(rows, classes):
  """Against torch's log-softmax in float64 on the device (the oracle's loops would take minutes)."""
  from dqn_zoo_amd import policy_loss as pl
  i = _inputs(rows, classes, torch.bfloat16, 5, padded=0.3 if rows > 4 else 0.0)
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.1, 0.02)
  out = pl.policy_loss(**i, config=cfg)
  lp = torch.log_softmax(i['logits'].double(), -1)
  w = i['weights'].double() if i['weights'] is not None else torch.ones(rows, device='cuda').double()
  live = w != 0
  logp = lp.gather(1, i['actions'][:, None])[:, 0]
  h = -(lp.exp() * lp).sum(-1)
  rho = torch.exp(logp - i['old_logp'].double())
  adv = i['advantages'].double()
  free, kept = rho * adv, rho.clamp(0.8, 1.2) * adv
  d = i['ref_logp'].double() - logp
  value = -torch.minimum(free, kept) + 0.1 * (d.expm1() - d) - 0.02 * h
  slope = torch.where(free <= kept, -free, 0.0) - 0.1 * d.expm1()
  f = (w / w.sum())[:, None]
  grad = (-slope[:, None] * lp.exp() + 0.02 * lp.exp() * (lp + h[:, None]))
  grad.scatter_add_(1, i['actions'][:, None], slope[:, None])
  grad *= f
  assert (out.logp.double() - logp)[live].abs().max() < 400 * U32
  assert (out.entropy.double() - h)[live].abs().max() < 800 * U32
  # (entropies up to 12, |k1 u| up to 0.02 * 30)
  scale = (free.abs() + 0.1 * d.abs().exp() + 0.02 * 40)[:, None] * f
  p = lp.exp().scatter(1, i['actions'][:, None], 1.0)
  tol = 2 * GRAD * U32 * scale * p
  bad = (out.dlogits.double() - grad).abs() > tol + HALF[torch.bfloat16] * (grad.abs() + tol) + 1e-38
  assert not bad[live].any()
  assert (out.dlogits[~live] == 0).all() and (out.logp[~live] == 0).all()
  want = torch.where(live, f[:, 0] * value, 0.0).sum()
  assert abs(float(out.loss) - float(want)) < 2 * GRAD * U32 * float(scale.sum())


@pytest.mark.parametrize('low,high,kl,ent', [(0.0, 0.0, 0.0, 0.0), (0.2, 0.5, 0.0, 0.0), (0.1, 0.1, 0.5, 0.0),
                                             (0.3, 0.3, 0.0, 0.1)])
def test_terms_one_by_one_and_their_borders(low, high, kl, ent):
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(low, high, kl, ent)
  for classes in (6, 700):
    i = _inputs(64, classes, torch.float32, 21, ref=kl > 0)
    _check(i, pl.policy_loss(**i, config=cfg), cfg, torch.float32)
    # ratios far outside the clip on both sides of both signs of the advantage
    i['old_logp'] = i['old_logp'] + torch.linspace(-4, 4, 64, device='cuda')
    i['advantages'] = torch.tensor([1.0, -1.0], device='cuda').repeat(32)
    _check(i, pl.policy_loss(**i, config=cfg), cfg, torch.float32)


@pytest.mark.parametrize('classes', [5, 300, 5000, 140000])
def test_gradient_is_the_difference_quotient(classes):
  """Central differences of the float64 loss at the measured logits: error h^2/6 f''' + 2 eps/h."""
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.3, 0.05)
  i = _inputs(3, classes, torch.float32, 33)
  out = pl.policy_loss(**i, config=cfg)
  x = _np(i['logits'])
  rest = (i['actions'].cpu().numpy(), _np(i['advantages']), _np(i['old_logp']), _np(i['ref_logp']))
  kw = dict(clip_low=0.2, clip_high=0.2, kl_coef=0.3, entropy_coef=0.05)
  for row in range(3):
    for col in {0, classes - 1, classes // 2, int(rest[0][row])}:
      h = 1e-4
      up, down = x.copy(), x.copy()
      up[row, col] += h
      down[row, col] -= h
      want = (po.policy_loss(up, *rest, **kw)[0] - po.policy_loss(down, *rest, **kw)[0]) / (2 * h)
      # third derivatives of the row's loss are at most 20 here; 2e-12 / 2e-4 from the quotient
      assert abs(float(out.dlogits[row, col]) - want) < 20 * h * h / 6 + 1e-8 + GRAD * U32


@pytest.mark.parametrize('classes', [6, 700, 3000, 12000])
def test_masks_padding_and_bad_values(classes):
  from dqn_zoo_amd import _lib
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.0, 0.05)
  inf, nan = float('inf'), float('nan')
  for dtype in (torch.float32, torch.bfloat16, torch.float16):
    i = _inputs(8, classes, dtype, 3, ref=False)
    x = i['logits']
    i['actions'][:] = 1
    low = torch.finfo(dtype).min
    x[0] = -inf                 # one class left
    x[0, 1] = 0.5
    x[1, 2:] = low              # the type's lowest value as a mask
    x[2] = low                  # nothing but it: uniform over the classes
    x[3] = nan                  # padding: not read
    x[4, 0] = -inf
    w = torch.ones(8, device='cuda')
    w[3] = 0
    i['weights'] = w
    i['actions'][3] = -100      # padding's action is not looked at either
    i['advantages'][3] = nan
    i['old_logp'][3] = nan
    status = torch.zeros(1, dtype=torch.int32, device='cuda')
    out = pl.policy_loss(**i, config=cfg, status=status)
    assert torch.isfinite(out.loss) and torch.isfinite(out.dlogits).all() and int(status) == 0
    assert float(out.logp[0]) == 0 and float(out.entropy[0]) == 0 and (out.dlogits[0] == 0).all()
    assert (out.dlogits[1, 2:] == 0).all()
    assert abs(float(out.logp[2]) + np.log(classes)) < 20 * U32 * np.log(classes)
    assert abs(float(out.entropy[2]) - np.log(classes)) < 40 * U32 * np.log(classes)
    assert float(out.logp[3]) == 0 and (out.dlogits[3] == 0).all()
    assert float(out.dlogits[4, 0]) == 0
    # rows that have no softmax are NaN, and no others
    x[5] = -inf
    x[6, 0] = nan
    x[7, 0] = inf
    out = pl.policy_loss(**i, config=cfg)
    assert torch.isnan(out.logp[5:]).all() and torch.isnan(out.loss)
    assert torch.isnan(out.dlogits[5:]).all() and torch.isfinite(out.dlogits[:5]).all()
    assert torch.isfinite(out.logp[:5]).all()
    # no such class
    for bad in (-1, classes, 2 ** 40):
      j = _inputs(8, classes, dtype, 3, ref=False)
      j['actions'][2] = bad
      status.zero_()
      out = pl.policy_loss(**j, config=cfg, status=status)
      assert int(status) == _lib.ST_BAD_INDEX
      assert torch.isnan(out.loss) and torch.isnan(out.logp[2])
      assert torch.isnan(out.logp).sum() == 1 and torch.isfinite(out.dlogits[3:]).all()


@pytest.mark.parametrize('classes', [6, 700, 5000, 70000])
def test_all_padding_gives_zero(classes):
  from dqn_zoo_amd import policy_loss as pl
  i = _inputs(100, classes, torch.bfloat16, 3)
  i['weights'] = torch.zeros(100, device='cuda')
  i['logits'].fill_(float('nan'))
  out = pl.policy_loss(**i, config=pl.PolicyLossConfig(0.2, 0.2, 0.1, 0.1))
  assert float(out.loss) == 0 and (out.dlogits == 0).all() and (out.logp == 0).all()
  assert (out.entropy == 0).all()


@pytest.mark.parametrize('rows,classes', [(40, 18), (3000, 18), (50, 900), (9, 9000), (4, 40000)])
def test_normalizer_scale_in_place_and_values_only(rows, classes):
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.1, 0.02)
  i = _inputs(rows, classes, torch.float32, 8, padded=0.2)
  small = rows * classes < 200000
  a = pl.policy_loss(**i, config=cfg, normalizer=37.5, grad_scale=8.0)
  if small:
    _check(i, a, cfg, torch.float32, normalizer=37.5, grad_scale=8.0)
  b = pl.policy_loss(**i, config=cfg, normalizer=37.5, with_gradient=False)
  assert b.dlogits is None
  for x, y in zip(a[:3], b[:3]):
    assert torch.equal(x, y)
  c = pl.policy_loss(**i, config=cfg, normalizer=37.5, grad_scale=8.0)
  for x, y in zip(a, c):
    assert torch.equal(x, y)        # the same call gives the same bits
  where = pl.PolicyLossOutputs(*(torch.empty_like(t) for t in a[:3]), i['logits'])
  d = pl.policy_loss(**i, config=cfg, normalizer=37.5, grad_scale=8.0, out=where)
  assert d.dlogits.data_ptr() == i['logits'].data_ptr()
  for x, y in zip(a, d):
    assert torch.equal(x, y)


def test_rows_of_one_pitch_into_rows_of_another():
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.0, 0.02)
  for classes in (18, 601, 9001):
    i = _inputs(20, classes, torch.bfloat16, 8, ref=False, extra=7)
    a = pl.policy_loss(**i, config=cfg)
    wide = torch.full((20, classes + 2), 7.0, dtype=torch.bfloat16, device='cuda')
    out = pl.PolicyLossOutputs(*(torch.empty_like(t) for t in a[:3]), wide[:, 1:classes + 1])
    pl.policy_loss(**i, config=cfg, out=out)
    assert torch.equal(out.dlogits, a.dlogits)
    assert (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all()


@pytest.mark.parametrize('rows,classes', [(32, 18), (500, 18), (64, 3000), (2, 50000)])
def test_captured_and_replayed(rows, classes):
  from dqn_zoo_amd import _lib
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.1, 0.02)
  i = _inputs(rows, classes, torch.bfloat16, 8, padded=0.2)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    first = pl.policy_loss(**i, config=cfg)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      got = pl.policy_loss(**i, config=cfg)
    # the library's own capture takes the caller's buffers, and refuses to make any
    with pytest.raises(RuntimeError, match='buffers'):
      _lib.capture_graph(side.cuda_stream, lambda: pl.policy_loss(**i, config=cfg))
    mine = pl.PolicyLossOutputs(*(torch.empty_like(t) for t in first))
    ws = torch.empty(pl.workspace_bytes(rows, classes, torch.bfloat16), dtype=torch.uint8, device='cuda')
    own = _lib.capture_graph(side.cuda_stream, lambda: pl.policy_loss(**i, config=cfg, out=mine, workspace=ws))
  for k in range(4):
    i['logits'].add_(0.25 * k)
    i['advantages'].mul_(-1)
    torch.cuda.synchronize()
    eager = pl.policy_loss(**i, config=cfg)
    graph.replay()
    _lib.check(_lib.load().dz_graph_launch(own, side.cuda_stream), 'dz_graph_launch')
    torch.cuda.synchronize()
    for x, y, z in zip(eager, got, mine):
      assert torch.equal(x, y) and torch.equal(x, z)
  _lib.load().dz_graph_destroy(own)


def test_more_rows_than_workgroups():
  # (2^20 workgroups of 8 rows go round; the halves do not)
  from dqn_zoo_amd import policy_loss as pl
  rows, classes = (1 << 23) + 1003, 130
  g = torch.Generator('cuda').manual_seed(11)
  logits = torch.randn(4099, classes, generator=g, device='cuda').bfloat16().repeat(rows // 4099 + 1, 1)[:rows]
  actions = torch.randint(0, classes, (rows,), generator=g, device='cuda')
  advantages, old = torch.randn(2, rows, generator=g, device='cuda').unbind()
  old = old - 5.0
  run = lambda a, b: pl.policy_loss(logits[a:b], actions[a:b], advantages[a:b], old[a:b], normalizer=float(rows))
  whole, cut = run(0, rows), rows // 2 + 5
  first, last = run(0, cut), run(cut, rows)
  assert torch.equal(whole.dlogits, torch.cat([first.dlogits, last.dlogits]))
  assert torch.equal(whole.logp, torch.cat([first.logp, last.logp]))
  # three roundings to float32 of sums in double
  big = max(abs(first.loss.item()), abs(last.loss.item()), abs(whole.loss.item()))
  assert abs(whole.loss.item() - (first.loss.item() + last.loss.item())) <= 4 * U32 * big


def test_two_streams_at_once():
  from dqn_zoo_amd import policy_loss as pl
  cfg = pl.PolicyLossConfig(0.2, 0.2, 0.1, 0.02)
  cases = [_inputs(400, 3000, torch.bfloat16, 8, padded=0.2), _inputs(4, 90000, torch.float32, 9, padded=0.2)]
  want = [pl.policy_loss(**i, config=cfg) for i in cases]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  outs = [[], []]
  for _ in range(10):
    for k in (0, 1):
      with torch.cuda.stream(streams[k]):
        outs[k].append(pl.policy_loss(**cases[k], config=cfg))
  torch.cuda.synchronize()
  for k in (0, 1):
    for o in outs[k]:
      assert all(torch.equal(x, y) for x, y in zip(o, want[k]))


def test_refusals():
  from dqn_zoo_amd import _lib
  from dqn_zoo_amd import policy_loss as pl
  i = _inputs(4, 6, torch.float32, 1)
  def refused(error, match, **change):
    with pytest.raises(error, match=match):
      pl.policy_loss(**{**i, **change})
  refused(_lib.HipLibraryError, 'no CPU fallback', logits=i['logits'].cpu())
  refused(TypeError, 'must be a tensor', logits=[1])
  refused(TypeError, 'float32, bfloat16 or float16', logits=i['logits'].double())
  refused(ValueError, 'not empty', logits=i['logits'][:0])
  refused(ValueError, 'not empty', logits=i['logits'][0])
  refused(ValueError, 'adjacent', logits=torch.zeros(6, 4, device='cuda').t())
  refused(ValueError, 'adjacent', logits=torch.zeros(1, 6, device='cuda').expand(4, 6))
  refused(TypeError, 'actions', actions=i['actions'].int())
  refused(ValueError, 'actions', actions=i['actions'][:3])
  refused(TypeError, 'needed', advantages=None)
  refused(TypeError, 'advantages', advantages=i['advantages'].double())
  refused(ValueError, 'another device', old_logp=i['old_logp'].cpu())
  refused(ValueError, 'contiguous', weights=torch.ones(8, device='cuda')[::2])
  refused(ValueError, 'negative', config=pl.PolicyLossConfig(-0.1))
  refused(ValueError, 'needs ref_logp', config=pl.PolicyLossConfig(kl_coef=0.1), ref_logp=None)
  refused(ValueError, 'normalizer', normalizer=0.0)
  refused(ValueError, 'normalizer', normalizer=float('nan'))
  refused(TypeError, 'status', status=torch.zeros(1, device='cuda'))
  refused(TypeError, 'workspace', workspace=torch.zeros(4, device='cuda'))
  big = _inputs(4, 9000, torch.float32, 1)
  with pytest.raises(ValueError, match='workspace needs'):
    pl.policy_loss(**big, workspace=torch.zeros(4, dtype=torch.uint8, device='cuda'))
  o = pl.policy_loss(**i)
  refused(ValueError, 'exactly if', out=o, with_gradient=False)
  refused(ValueError, 'exactly if', out=o._replace(dlogits=None))
  buf = torch.zeros(5, 6, device='cuda')
  refused(ValueError, 'overlaps', logits=buf[:4], out=o._replace(dlogits=buf[1:]))
  for name in ('advantages', 'old_logp', 'ref_logp'):   # another workgroup may still read them
    refused(ValueError, 'out.logp overlaps ' + name, out=o._replace(logp=i[name]))
  w = torch.ones(4, device='cuda')
  refused(ValueError, 'out.entropy overlaps weights', weights=w, out=o._replace(entropy=w))
  refused(ValueError, 'out.entropy overlaps logp', out=o._replace(entropy=o.logp))
  # the C entry refuses before it launches anything
  lib = _lib.load()
  n = ctypes.c_int64()
  assert lib.dz_policy_loss_workspace(7, 4, 6, ctypes.byref(n)) == _lib.DZ_ERR_INVALID_ARG
  assert lib.dz_policy_loss_workspace(0, 0, 6, ctypes.byref(n)) == _lib.DZ_ERR_INVALID_ARG
  assert lib.dz_policy_loss(ctypes.byref(_lib.PolicyLossArgs()), None) == _lib.DZ_ERR_INVALID_ARG
