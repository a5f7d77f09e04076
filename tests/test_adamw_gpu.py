"""AdamW over a list of tensors against the float64 oracle (oracle/policy_oracle.py)."""

import numpy as np
import pytest
import torch

from oracle import policy_oracle as po

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24   # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _np(t):
  return t.detach().double().cpu().numpy()


def _make(sizes, dtype, seed, packed=False, scale=1e-3):
  g = torch.Generator().manual_seed(seed)
  params, grads = [], []
  total = sum(int(np.prod(s)) for s in sizes)
  flats = [torch.empty(total + 64, dtype=dtype, device='cuda') for _ in range(2)] if packed else None
  at = 1   # (packed tensors begin at an odd element)
  for s in sizes:
    n = int(np.prod(s))
    p = (torch.randn(n, generator=g) * 0.1).to(dtype)
    d = (torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g)) * scale).to(dtype)
    if packed:
      for flat, x in zip(flats, (p, d)):
        flat[at:at + n] = x.cuda()
      params.append(flats[0][at:at + n].view(s))
      grads.append(flats[1][at:at + n].view(s))
      at += n
    else:
      params.append(p.cuda().view(s))
      grads.append(d.cuda().view(s))
  return params, grads


def _flat(opt, tensors):
  out = np.zeros(opt.state_size)
  for t, o in zip(tensors, opt.offsets):
    out[o:o + t.numel()] = _np(t).reshape(-1)
  return out


def _close(got, want, tol, what):
  bad = np.abs(got - want) > tol
  assert not bad.any(), '%s: %d off, worst %g of its tolerance' % (
      what, bad.sum(), np.max(np.abs(got - want)[bad] / tol[bad]))


# One update's roundings, each at most U32 relative to what it rounds.
#   g: coef (1 for the product, up to 20 from the norm: 16 squares and 8 additions of positive
#      terms halved by the root, its float32 value, the division) -> 22;
#   m: 3 of its own + g's on the second term;  v: 4 + twice g's;
#   step: m's, half of v's, and 6 of its own (two divisions, the bias corrections' float32 values,
#      root, sum), p: 3 more.
M_ROUND, V_ROUND, S_ROUND = 26, 50, 64


@pytest.mark.parametrize('sizes,dtype,packed,clip', [
    ([(1,)], torch.float32, False, 0.0),
    ([(3,), (255,), (256,), (257,)], torch.float32, True, 1e-3),
    ([(33, 31), (4096,), (4097,), (5, 7, 3), (1,)], torch.float32, True, 1e6),
    ([(1000, 37), (64,)], torch.bfloat16, False, 1e-2),
    ([(100, 37), (64,), (1,)], torch.bfloat16, True, 0.0),
    ([(129, 65), (7,)], torch.float16, True, 1e-2),
    ([(3136, 512), (512,), (512, 18), (18,)], torch.float32, False, 10.0),
])
@pytest.mark.parametrize('master', [None, False])
def test_float32_moments_follow_the_formula(sizes, dtype, packed, clip, master):
  from dqn_zoo_amd import adamw
  params, grads = _make(sizes, dtype, 3, packed)
  decay = [len(s) > 1 for s in sizes]
  cfg = adamw.AdamWConfig(1e-2, 0.9, 0.99, 1e-8, 0.1, clip)
  opt = adamw.AdamW(params, cfg, decay=decay, master_weights=master)
  kept = opt.master is not None
  assert kept == (dtype != torch.float32 and master is None)
  wd = np.zeros(opt.state_size)
  for o, s, d in zip(opt.offsets, sizes, decay):
    wd[o:o + int(np.prod(s))] = 0.1 * d
  guard = [p.clone() for p in grads]
  for step in range(1, 4):
    p0 = _np(opt.master) if kept else _flat(opt, params)
    m0, v0, g = _np(opt.m), _np(opt.v), _flat(opt, grads)
    norm = np.sqrt((g * g).sum())
    coef = min(1.0, clip / norm) if clip > 0 else 1.0
    p, m, v = po.adamw(p0, g, m0, v0, step, 1e-2, 0.9, 0.99, 1e-8, wd, coef)
    opt.step(grads if step < 3 else opt.bind(grads))
    if clip > 0:
      assert abs(float(opt.grad_norm) - norm) <= 16 * U32 * norm
    gm = 0.1 * np.abs(g) * coef
    _close(_np(opt.m), m, U32 * M_ROUND * (0.9 * np.abs(m0) + gm) + 1e-38, 'm')
    _close(_np(opt.v), v, U32 * V_ROUND * v + 1e-38, 'v')
    # (cancellation in m enters the step relative to the terms of m)
    upd = (0.9 * np.abs(m0) + gm) / (1 - 0.9 ** step) / (np.sqrt(v / (1 - 0.99 ** step)) + 1e-8)
    tol = U32 * (3 * np.abs(p0) + S_ROUND * 1e-2 * (upd + wd * np.abs(p0))) + 1e-38
    if kept:
      _close(_np(opt.master), p, tol, 'master')
      want, got = _np(opt.master), _flat(opt, params)   # the parameters: the master, rounded
      _close(got, want, HALF[dtype] * np.abs(want) + 1e-7 * (dtype == torch.float16) + 1e-38, 'params')
    else:
      _close(_flat(opt, params), p, tol + HALF[dtype] * (np.abs(p) + tol) +
             1e-7 * (dtype == torch.float16), 'params')
  assert opt.count == 3
  for a, b in zip(grads, guard):
    assert torch.equal(a, b)


@pytest.mark.parametrize('sizes,dtype,packed', [
    ([(1,), (300,)], torch.float32, True),
    ([(64, 129), (4096,), (5,)], torch.bfloat16, False),
    ([(3136, 40)], torch.float16, False),
])
def test_eight_bit_moments(sizes, dtype, packed):
  """Scales, codes (given the draws) and parameters of each step, from the state before it."""
  from dqn_zoo_amd import adamw
  params, grads = _make(sizes, dtype, 5, packed, scale=1e-3)
  opt = adamw.AdamW(params, adamw.AdamWConfig(1e-3, state_bits=8, weight_decay=0.0), seed=77)
  real = _flat(opt, [torch.ones_like(p) for p in params]) > 0
  pos = np.arange(opt.state_size)
  for step in range(1, 5):
    m0 = po.decode_e4m3(opt.m.cpu().numpy()) * np.repeat(_np(opt.m_scale), 256)
    v0 = po.decode_e5m3(opt.v.cpu().numpy()) * np.repeat(_np(opt.v_scale), 256)
    p0 = _np(opt.master) if opt.master is not None else _flat(opt, params)
    g = _flat(opt, grads)
    p, m, v = po.adamw(p0, g, m0, v0, step, 1e-3, 0.9, 0.999, 1e-8, 0.0)
    opt.step(grads)
    got_p = _np(opt.master) if opt.master is not None else _flat(opt, params)
    upd = (0.9 * np.abs(m0) + 0.1 * np.abs(g)) / (1 - 0.9 ** step) / (
        np.sqrt(v / (1 - 0.999 ** step)) + 1e-8)
    _close(got_p, p, U32 * (3 * np.abs(p0) + S_ROUND * 1e-3 * upd) + 1e-38, 'p')
    noise = po.adamw_noise(77, step, pos)
    for codes, scale, exact, u, top_value, least, name in (
        (opt.m, opt.m_scale, m, noise[0], 448.0, -6, 'm'),
        (opt.v, opt.v_scale, v, noise[1], 1.875, -30, 'v')):
      codes, scale = codes.cpu().numpy(), _np(scale)
      decode = po.decode_e4m3 if name == 'm' else po.decode_e5m3
      top = np.abs(exact).reshape(-1, 256).max(1)
      _close(scale, top / top_value, 60 * U32 * top / top_value + 1e-45, name + ' scale')
      y = np.abs(exact) / np.repeat(np.maximum(top / top_value, 1e-300), 256)
      unit = po.eight_bit_steps(y, least)
      place = y / unit + u / 65536.0
      want = np.minimum(np.floor(place) * unit, top_value)
      if name == 'v':
        want = np.where((y > 0) & (want == 0), 2.0 ** -33, want)
      else:
        want = np.copysign(want, exact)
      have = decode(codes)
      # a draw next to the border may fall on either side: y's own error, V_ROUND U32 of at most 16
      # steps, is far below 2^-12 of one
      border = np.abs(place - np.round(place)) < 2.0 ** -12
      assert (have == want)[~border].all(), name
      assert (np.abs(have - want) <= unit * 1.0001)[border].all(), name
      assert border.mean() < 2.0 ** -9
      assert (have[~real] == 0).all() and (codes[~real] == 0).all()
  mm, vv = opt.moments()
  np.testing.assert_array_equal(_np(mm), (po.decode_e4m3(opt.m.cpu().numpy()).astype(np.float32) *
                                          np.repeat(opt.m_scale.cpu().numpy(), 256)).astype(np.float64))
  np.testing.assert_array_equal(_np(vv), (po.decode_e5m3(opt.v.cpu().numpy()).astype(np.float32) *
                                          np.repeat(opt.v_scale.cpu().numpy(), 256)).astype(np.float64))


def test_eight_bit_average_is_kept():
  """A constant gradient's moments after many steps are its mean and square, as in float32: the
  random rounding has no drift.  v's stationary noise is at most half a step (1/16) times
  sqrt(1 / (2 (1 - b2))) per element and averages over 65536 elements; 2 % is over 10 deviations."""
  from dqn_zoo_amd import adamw
  n = 65536
  p = [torch.zeros(n, device='cuda')]
  g = [torch.full((n,), 1e-3, device='cuda')]
  opt = adamw.AdamW(p, adamw.AdamWConfig(0.0, 0.9, 0.99, state_bits=8))
  opt.step([torch.full((n,), 3e-3, device='cuda')])   # v starts nine times too high and has to decay
  for _ in range(400):
    opt.step(g)
  m, v = opt.moments()
  assert abs(float(m.mean()) / 1e-3 - 1) < 0.02
  assert abs(float(v.mean()) / (1e-6 * (1 - 0.99 ** 400) + 0.08e-6 * 0.99 ** 400) - 1) < 0.02


def test_blocks_of_very_different_and_of_bad_values():
  from dqn_zoo_amd import adamw
  g = torch.zeros(1024, device='cuda')
  g[:256] = torch.logspace(-6, 0, 256)      # six decades in a block
  g[256:512] = 0.0
  g[512:768] = 1e-30                        # squares below the least normal float32
  g[768] = float('nan')
  g[800] = float('inf')
  for bits in (8, 32):
    p = [torch.ones(1024, device='cuda')]
    opt = adamw.AdamW(p, adamw.AdamWConfig(1e-2, weight_decay=0.0, state_bits=bits))
    opt.step([g])
    out = p[0].cpu()
    assert torch.isfinite(out[:768]).all()
    # a first step is lr * g / (|g| + eps')
    assert (out[:256] < 1).all() and (out[:256] >= 0.99 - 1e-6).all()
    assert (out[256:512] == 1).all()
    bad = ~torch.isfinite(out[768:])
    assert bad[0] and bad[32] and int(bad.sum()) == 2
    m, v = opt.moments()
    assert torch.isfinite(m[:768]).all() and torch.isfinite(v[:768]).all()
    assert (v[:256] > 0).all()
    assert torch.isnan(m[768]) and not torch.isfinite(v[800])
    p2 = p[0].clone()
    opt.step([torch.zeros(1024, device='cuda')])
    assert torch.isfinite(p[0][:768]).all() and not torch.isfinite(p[0][768])
    assert (p[0][:256] <= p2[:256]).all()


def test_gradient_scale_and_float32_gradients():
  from dqn_zoo_amd import adamw
  params, grads = _make([(65, 9), (130,)], torch.bfloat16, 9)
  params2 = [p.clone() for p in params]
  cfg = adamw.AdamWConfig(1e-2, max_global_grad_norm=1e-3)
  a, b = adamw.AdamW(params, cfg), adamw.AdamW(params2, cfg)
  a.step(grads)
  b.step([g.float() * 64 for g in grads], grad_scale=1.0 / 64)   # powers of two: exact
  assert torch.equal(a.m, b.m) and torch.equal(a.v, b.v) and torch.equal(a.master, b.master)
  assert all(torch.equal(p, q) for p, q in zip(params, params2))
  assert torch.equal(a.grad_norm, b.grad_norm)


def test_state_round_trip_and_determinism():
  from dqn_zoo_amd import adamw
  for bits in (8, 32):
    params, grads = _make([(65, 9), (130,), (4099,)], torch.bfloat16, 11)
    cfg = adamw.AdamWConfig(1e-2, max_global_grad_norm=1.0, state_bits=bits)
    a = adamw.AdamW(params, cfg, seed=4)
    a.step(grads)
    copies = [p.clone() for p in params]
    b = adamw.AdamW(copies, cfg, seed=4)
    b.set_state(a.get_state())
    for _ in range(3):
      a.step(grads)
      b.step(grads)
    assert a.count == b.count == 4
    for x, y in zip(params, copies):
      assert torch.equal(x, y)
    for k, v in a.get_state().items():
      assert k == 'count' or torch.equal(v, b.get_state()[k]), k


def test_captured_step_follows_count_and_learning_rate():
  from dqn_zoo_amd import adamw
  sizes = [(65, 9), (4099,)]
  params, grads = _make(sizes, torch.float32, 12)
  eager, _ = _make(sizes, torch.float32, 12)
  cfg = adamw.AdamWConfig(1e-2, max_global_grad_norm=1e-2, state_bits=8)
  a, b = adamw.AdamW(params, cfg), adamw.AdamW(eager, cfg)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    a.step(grads)
    b.step(grads)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      a.step(grads)
  torch.cuda.synchronize()
  for i in range(4):
    lr = 1e-2 / (i + 1)
    a.learning_rate = lr
    b.learning_rate = lr
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    b.step(grads)
    torch.cuda.synchronize()
    for x, y in zip(params, eager):
      assert torch.equal(x, y)
  assert a.count == 5


def test_more_tensors_than_one_upload_holds():
  from dqn_zoo_amd import adamw
  sizes = [(3 + i % 5,) for i in range(1000)]
  params, grads = _make(sizes, torch.float32, 13, packed=True)
  before = [p.clone() for p in params]
  opt = adamw.AdamW(params, adamw.AdamWConfig(1e-2, weight_decay=0.0))
  opt.step(grads)
  for p, q, g in zip(params, before, grads):
    want = _np(q) - 1e-2 * _np(g) / (np.abs(_np(g)) + 1e-8)
    _close(_np(p), want, U32 * (3 * np.abs(_np(q)) + S_ROUND * 1e-2), 'p')


def test_refusals():
  from dqn_zoo_amd import _lib, adamw
  mk = lambda *s, **k: torch.zeros(*s, device='cuda', **k)
  cfg = adamw.AdamWConfig()
  with pytest.raises(ValueError, match='at least one'):
    adamw.AdamW([], cfg)
  with pytest.raises(TypeError, match='float32, bfloat16 or float16'):
    adamw.AdamW([mk(4, dtype=torch.float64)], cfg)
  with pytest.raises(TypeError, match=r'params\[1\]'):
    adamw.AdamW([mk(4), mk(4, dtype=torch.bfloat16)], cfg)
  with pytest.raises(ValueError, match='contiguous and not empty'):
    adamw.AdamW([mk(4, 3).t()], cfg)
  with pytest.raises(ValueError, match='contiguous and not empty'):
    adamw.AdamW([mk(0)], cfg)
  with pytest.raises(_lib.HipLibraryError, match='no CPU fallback'):
    adamw.AdamW([mk(4), torch.zeros(4)], cfg)
  x = mk(16)
  with pytest.raises(ValueError, match='share memory'):
    adamw.AdamW([x, x], cfg)
  with pytest.raises(ValueError, match='share memory'):
    adamw.AdamW([x[:9], x[8:]], cfg)
  with pytest.raises(ValueError, match='state_bits'):
    adamw.AdamW([x], cfg._replace(state_bits=16))
  with pytest.raises(ValueError, match='b1'):
    adamw.AdamW([x], cfg._replace(b1=1.0))
  with pytest.raises(ValueError, match='decay has'):
    adamw.AdamW([x], cfg, decay=[True, False])
  with pytest.raises(ValueError, match='master'):
    adamw.AdamW([x], cfg, master_weights=True)
  opt = adamw.AdamW([x, mk(3, 2)], cfg)
  with pytest.raises(ValueError, match='1 gradients for 2'):
    opt.step([mk(16)])
  with pytest.raises(ValueError, match=r'grads\[1\] has shape'):
    opt.step([mk(16), mk(2, 3)])
  with pytest.raises(TypeError, match='gradients must be'):
    opt.step([mk(16), mk(3, 2, dtype=torch.bfloat16)])
  with pytest.raises(ValueError, match='contiguous'):
    opt.step([mk(16), mk(2, 3).t()])
  with pytest.raises(TypeError, match='must be a tensor'):
    opt.step([mk(16), None])
  with pytest.raises(ValueError, match='device'):
    opt.step([mk(16), torch.zeros(3, 2)])
  with pytest.raises(ValueError, match='shares memory'):
    opt.bind([x, mk(3, 2)])
  other = adamw.AdamW([mk(16), mk(3, 2)], cfg)
  with pytest.raises(ValueError, match='another optimizer'):
    opt.step(other.bind([mk(16), mk(3, 2)]))
  with pytest.raises(ValueError, match='state has'):
    opt.set_state({'m': opt.m})
  with pytest.raises(ValueError, match="state 'm'"):
    opt.set_state({'count': 1, 'm': opt.m[:10], 'v': opt.v})
  with pytest.raises(TypeError, match='moments are'):
    opt.moments(torch.int32)
  assert opt.count == 0 and float(x.abs().sum()) == 0
