"""A policy's training step out of the operators: two dense layers on the torso's 3136 features,
the clipped loss over the 18 actions, both backward passes, AdamW -- eager, in a graph, and its
gradients against the float64 formulas and against differences."""

import numpy as np
import pytest
import torch

from oracle import policy_oracle as po

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
CFG = dict(clip_low=0.2, clip_high=0.2, kl_coef=0.1, entropy_coef=0.01)


def _np(t):
  return t.detach().double().cpu().numpy()


class Policy:

  def __init__(self, rows, dtype, features=3136, hidden=512, actions=18, seed=0):
    from dqn_zoo_amd import adamw
    g = torch.Generator().manual_seed(seed)
    uni = lambda fan, *s: ((torch.rand(*s, generator=g) * 2 - 1) / fan ** 0.5).to(dtype).cuda()
    self.params = [uni(features, features, hidden), uni(features, hidden),
                   uni(hidden, hidden, actions), uni(hidden, actions)]
    self.x = torch.rand(rows, features, generator=g).to(dtype).cuda()
    self.actions = torch.randint(0, actions, (rows,), generator=g).cuda()
    self.adv = torch.randn(rows, generator=g).cuda()
    self.weights = (torch.rand(rows, generator=g) > 0.2).float().cuda()
    with torch.no_grad():
      lp = torch.log_softmax(self.logits().float(), -1).gather(1, self.actions[:, None])[:, 0]
    self.old = lp + 0.2 * torch.randn(rows, generator=g).cuda()
    self.ref = lp + 0.2 * torch.randn(rows, generator=g).cuda()
    self.grads = [torch.zeros_like(p) for p in self.params]
    self.opt = adamw.AdamW(self.params, adamw.AdamWConfig(1e-3, max_global_grad_norm=1.0, weight_decay=0.01,
                                                          state_bits=8),
                           decay=[True, False, True, False], seed=5)
    self.bound = self.opt.bind(self.grads)

  def logits(self):
    from dqn_zoo_amd import linear
    w1, b1, w2, b2 = self.params
    self.h, self.z = linear.linear(self.x, w1, b1, activation='relu', save_preact=True)
    return linear.linear(self.h, w2, b2)

  def gradients(self):
    from dqn_zoo_amd import linear, policy_loss
    out = policy_loss.policy_loss(self.logits(), self.actions, self.adv, self.old, self.ref, self.weights,
                                  config=policy_loss.PolicyLossConfig(**CFG))
    w1, _, w2, _ = self.params
    d1, e1, d2, e2 = self.grads
    dh, _, _ = linear.linear_backward(out.dlogits, self.h, w2, dw=d2, db=e2)
    linear.linear_backward(dh, self.x, w1, activation='relu', preact=self.z, need=(False, True, True), dw=d1, db=e1)
    return out

  def step(self):
    out = self.gradients()
    self.opt.step(self.bound)
    return out


def _exact(p, params=None):
  w1, b1, w2, b2 = params or [_np(t) for t in p.params]
  x = _np(p.x)
  h, z = po.linear(x, w1, b1, 'relu')
  logits, _ = po.linear(h, w2, b2)
  loss, logp, ent, dl = po.policy_loss(logits, p.actions.cpu().numpy(), _np(p.adv), _np(p.old), _np(p.ref),
                                       _np(p.weights), **CFG)
  dh, dw2, db2 = po.linear_backward(dl, h, w2)
  _, dw1, db1 = po.linear_backward(dh, x, w1, 'relu', z)
  return loss, [dw1, db1, dw2, db2], h, logits


@pytest.mark.parametrize('rows,dtype', [(32, torch.float32), (1, torch.float32), (70, torch.bfloat16),
                                        (1, torch.bfloat16)])
def test_gradients_of_the_chain(rows, dtype):
  """Relative to each gradient's norm.  float32: sums of up to 3136 terms and the chain's few hundred
  roundings, 2 sqrt(3136) + 300 < 500 half steps.  bfloat16: h, z, logits, dlogits, dh, dz and the
  result are rounded to half a step (2^-8) each, and h's rounding moves the logits by at most
  2^-8 |h| |w2| ~ 2^-8 of their size, which the loss' slope (below 4 relative here) carries: 7 + 4
  half steps and as many again for hidden units whose sign turns: 24."""
  p = Policy(rows, dtype)
  if rows == 1:
    p.weights.fill_(1.0)
  out = p.gradients()
  loss, want, _, _ = _exact(p)
  tol = (500 if dtype == torch.float32 else 24) * HALF[dtype]
  assert abs(float(out.loss) - loss) <= tol * max(1.0, abs(loss))
  for got, ref, name in zip(p.grads, want, ('dw1', 'db1', 'dw2', 'db2')):
    assert np.linalg.norm(_np(got) - ref) <= tol * np.linalg.norm(ref), name


def test_gradients_against_differences():
  """Along random directions of all parameters, of the float64 loss: error h^2/6 f''' (the loss is
  piecewise smooth; h = 1e-5 of the parameters' size) and the gradient's own 500 half steps."""
  p = Policy(16, torch.float32, features=96, hidden=40, actions=6)
  p.gradients()
  params = [_np(t) for t in p.params]
  rs = np.random.RandomState(0)
  for _ in range(4):
    d = [rs.standard_normal(t.shape) / np.sqrt(t.size) for t in params]
    h = 1e-5
    up = _exact(p, [t + h * e for t, e in zip(params, d)])[0]
    down = _exact(p, [t - h * e for t, e in zip(params, d)])[0]
    want = (up - down) / (2 * h)
    got = sum(float((_np(g) * e).sum()) for g, e in zip(p.grads, d))
    size = np.sqrt(sum(float((_np(g) ** 2).sum()) for g in p.grads))
    assert abs(got - want) <= 500 * HALF[torch.float32] * size + 1e-8


@pytest.mark.parametrize('rows,dtype', [(32, torch.bfloat16), (300, torch.float32)])
def test_captured_step_replays_as_the_eager_one(rows, dtype):
  a, b = Policy(rows, dtype), Policy(rows, dtype)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    a.step()
    b.step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      captured = a.step()
  for k in range(4):
    for p in (a, b):
      p.adv.mul_(-0.9)
      p.opt.learning_rate = 1e-3 / (k + 1)
    torch.cuda.synchronize()
    graph.replay()
    eager = b.step()
    torch.cuda.synchronize()
    for x, y in zip(captured, eager):
      assert torch.equal(x, y)
    for x, y in zip(a.params + a.grads, b.params + b.grads):
      assert torch.equal(x, y)
    assert torch.equal(a.opt.m, b.opt.m) and torch.equal(a.opt.v, b.opt.v)
    assert torch.equal(a.opt.grad_norm, b.opt.grad_norm) and torch.isfinite(eager.loss)
  assert a.opt.count == b.opt.count == 5


def test_two_captured_steps_share_nothing():
  """Two graphs of two policies, replayed at once on two streams."""
  policies = [Policy(64, torch.bfloat16, seed=s) for s in (1, 2)]
  twins = [Policy(64, torch.bfloat16, seed=s) for s in (1, 2)]
  graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
  for p, s in zip(policies, streams):
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
      p.step()
      s.synchronize()
      graphs.append(torch.cuda.CUDAGraph())
      with torch.cuda.graph(graphs[-1], stream=s):
        p.step()
  torch.cuda.synchronize()
  for _ in range(5):
    for g, s in zip(graphs, streams):
      with torch.cuda.stream(s):
        g.replay()
  torch.cuda.synchronize()
  for t in twins:
    for _ in range(6):
      t.step()
  for p, t in zip(policies, twins):
    for x, y in zip(p.params, t.params):
      assert torch.equal(x, y)
