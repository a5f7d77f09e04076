"""The dense layer with its epilogue, and its backward pass, against the float64 oracle."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import policy_oracle as po

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _np(t):
  return None if t is None else t.detach().double().cpu().numpy()


def _pitched(t, pad):
  """The same values in rows of `pad` more elements, and one element past an aligned address if
  pad is odd."""
  if not pad:
    return t
  shift = pad % 2
  flat = torch.full((t.shape[0] * (t.shape[1] + pad) + shift,), 3.0, dtype=t.dtype, device=t.device)
  wide = flat[shift:].view(t.shape[0], t.shape[1] + pad)
  wide[:, :t.shape[1]] = t
  return wide[:, :t.shape[1]]


def _make(m, k, n, dtype, seed, transposed=False, pad=0):
  g = torch.Generator().manual_seed(seed)
  rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
  x = _pitched(rnd(m, k), pad)
  w = (torch.randn(n, k, generator=g) / k ** 0.5).to(dtype).cuda()
  w = _pitched(w, pad).t() if transposed else _pitched(w.t().contiguous(), pad)
  return x, w, rnd(n), rnd(m, n)


def _sum_tol(depth, terms):
  """Of a float32 sum of `depth` terms whose absolute values add up to `terms`: the roundings, at
  most U32 of a partial sum each, go either way; 2 sqrt(depth) of them is over 6 deviations."""
  return (2 * np.sqrt(depth) + 8) * U32 * terms


def _close(got, want, tol, dtype, what):
  tol = tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype]
  bad = ~(np.abs(got - want) <= tol)
  assert not bad.any(), '%s: %d of %d off, worst %g of its tolerance at %s' % (
      what, bad.sum(), bad.size, np.max(np.abs(got - want)[bad] / tol[bad]), np.argwhere(bad)[:4].tolist())


def _check_forward(x, w, b, r, activation, y, z, dtype):
  xn, wn = _np(x), _np(w)
  bn = 0.0 if b is None else _np(b)
  want_y, want_z = po.linear(xn, wn, None if b is None else bn, activation, _np(r))
  ztol = _sum_tol(xn.shape[1], np.abs(xn) @ np.abs(wn) + np.abs(bn))
  if z is not None:
    _close(_np(z), want_z, ztol, dtype, 'preact')
  # slopes are at most 1.13; the activation's own operations: 8 roundings of terms up to |z|
  ytol = 1.13 * ztol + 8 * U32 * np.abs(want_z) + 2 * U32 * np.abs(want_y)
  _close(_np(y), want_y, ytol, dtype, 'y')


SHAPES = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (16, 64, 64), (17, 72, 40), (64, 128, 64), (65, 130, 129),
          (128, 256, 128), (1, 3136, 512), (32, 3136, 18), (200, 64, 300), (257, 1000, 513)]


@pytest.mark.parametrize('m,k,n', SHAPES)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('transposed', [False, True])
def test_forward(m, k, n, dtype, transposed):
  from dqn_zoo_amd import linear
  for pad, activation in ((0, 'none'), (8, 'gelu'), (1, 'relu'), (0, 'silu')):
    x, w, b, r = _make(m, k, n, dtype, m + k + n, transposed, pad)
    residual = r if activation in ('gelu', 'silu') else None
    bias = None if activation == 'none' else b.float() if activation == 'silu' else b
    y, z = linear.linear(x, w, bias, activation=activation, residual=residual, save_preact=True)
    _check_forward(x, w, bias, residual, activation, y, z, dtype)
    alone = linear.linear(x, w, bias, activation=activation, residual=residual)
    assert torch.equal(alone, y)


@pytest.mark.parametrize('m,k,n', SHAPES)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('transposed', [False, True])
def test_backward(m, k, n, dtype, transposed):
  from dqn_zoo_amd import linear
  for pad, activation in ((0, 'none'), (8, 'gelu'), (1, 'relu'), (0, 'silu')):
    x, w, _, z = _make(m, k, n, dtype, m + k + n + 1, transposed, pad)
    dy = _pitched(torch.randn(m, n, generator=torch.Generator().manual_seed(2)).to(dtype).cuda(), pad)
    preact = None if activation == 'none' else z
    got = linear.linear_backward(dy, x, w, activation=activation, preact=preact)
    _check_backward(dy, x, w, activation, preact, got, dtype)
    assert got[1].stride() == ((1, k) if transposed and n > 1 and k > 1 else got[1].stride())


@pytest.mark.parametrize('m,k,n', [(9, 1951, 2057), (1, 513, 3137), (32, 3001, 1001), (31, 1001, 257), (33, 1001, 257)])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('transposed', [False, True])
def test_few_rows_of_any_alignment(m, k, n, dtype, transposed):
  from dqn_zoo_amd import linear
  for pad in (1, 3, 8):
    x, w, b, r = _make(m, k, n, dtype, m + k + n, transposed, pad)
    y, z = linear.linear(x, w, b, activation='silu', residual=r, save_preact=True)
    _check_forward(x, w, b, r, 'silu', y, z, dtype)
    dy = _pitched(torch.randn(m, n, generator=torch.Generator().manual_seed(3)).to(dtype).cuda(), pad)
    got = linear.linear_backward(dy, x, w, activation='silu', preact=z)
    _check_backward(dy, x, w, 'silu', z, got, dtype)


def _check_backward(dy, x, w, activation, preact, got, dtype, kind=None):
  kind = kind or dtype
  dyn, xn, wn, zn = _np(dy), _np(x), _np(w), _np(preact)
  want = po.linear_backward(dyn, xn, wn, activation, zn)
  dz = dyn if activation == 'none' else dyn * po.act_slope(zn, activation)
  # the slope: 8 roundings of terms up to 1 + |z|; dz is rounded before the products, not in db
  slope = 0.0 if activation in ('none', 'relu') else 10 * U32 * np.abs(dyn) * (1 + np.abs(zn))
  rounded = slope + (0.0 if activation in ('none', 'relu') else HALF[dtype] * np.abs(dz) + TINY[dtype])
  mag = np.abs(dz) + rounded
  dx, dw, db = got
  if dx is not None:
    _close(_np(dx), want[0], _sum_tol(wn.shape[1], mag @ np.abs(wn).T) + (rounded + 0 * dz) @ np.abs(wn).T,
           dtype, 'dx')
  if dw is not None:
    _close(_np(dw), want[1], _sum_tol(xn.shape[0], np.abs(xn).T @ mag) + np.abs(xn).T @ (rounded + 0 * dz),
           kind, 'dw')
  if db is not None:
    _close(_np(db), want[2], _sum_tol(xn.shape[0], mag.sum(0)) + (slope + 0 * dz).sum(0), kind, 'db')


def test_more_rows_than_a_launch_of_small_tiles_has():
  from dqn_zoo_amd import linear
  m = (1 << 30) + 77   # 2^24 tiles of 64 rows and 256 threads
  x = torch.arange(-128, 128, device='cuda').to(BF16).repeat(m // 256 + 1)[:m].view(m, 1)
  w = torch.full((1, 1), -2.0, dtype=BF16, device='cuda')
  y = linear.linear(x, w)
  assert torch.equal(y, x.mul_(-2))   # exact: at most 9 bits


# every tile, whole and ragged, with and without splits along the depth
@pytest.mark.parametrize('m,k,n', [(512, 512, 512), (520, 1096, 776), (1024, 64, 2048), (2048, 2048, 2048),
                                   (8, 8192, 256), (4096, 24, 264), (300, 4104, 136), (16, 40, 20000),
                                   (20000, 40, 16)])
@pytest.mark.parametrize('dtype', [BF16, F32])
@pytest.mark.parametrize('transposed', [False, True])
def test_larger_sizes(m, k, n, dtype, transposed):
  from dqn_zoo_amd import linear
  x, w, b, z = _make(m, k, n, dtype, 7, transposed)
  y = linear.linear(x, w, b, activation='relu')
  _check_forward(x, w, b, None, 'relu', y, None, dtype)
  dy = torch.randn(m, n, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
  got = linear.linear_backward(dy, x, w, activation='relu', preact=z)
  _check_backward(dy, x, w, 'relu', z, got, dtype)


@pytest.mark.parametrize('m,k,n', [(5, 7, 9), (64, 72, 80), (1030, 520, 264)])
def test_float32_gradients_of_16_bit_layers_and_parts(m, k, n):
  from dqn_zoo_amd import linear
  x, w, _, z = _make(m, k, n, BF16, 1)
  dy = torch.randn(m, n, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
  dw = torch.full((k, n), 9.0, device='cuda')
  db = torch.full((n,), 9.0, device='cuda')
  kw = dict(activation='gelu', preact=z)
  full = linear.linear_backward(dy, x, w, dw=dw, db=db, **kw)
  assert full[1] is dw and full[2] is db
  _check_backward(dy, x, w, 'gelu', z, full, BF16, kind=F32)
  for need in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
    part = linear.linear_backward(dy, x, w, need=need, **kw)
    for got, want, wanted in zip(part, full, need):
      assert (got is not None) == wanted
      if wanted:
        assert torch.equal(got, want.to(got.dtype))


def test_gradients_are_the_difference_quotients():
  """Of sum(dy * y) in float64: error h^2/6 f''' (|f'''| < 3 per unit here) + rounding / h."""
  from dqn_zoo_amd import linear
  for activation in ('none', 'gelu', 'silu'):
    x, w, b, _ = _make(4, 6, 5, F32, 3)
    dy = torch.randn(4, 5, generator=torch.Generator().manual_seed(2)).cuda()
    _, z = linear.linear(x, w, b, activation=activation, save_preact=True)
    dx, dw, db = (_np(t) for t in linear.linear_backward(dy, x, w, activation=activation, preact=z))
    args = [_np(x), _np(w), _np(b)]
    loss = lambda a: float((_np(dy) * po.linear(*a, activation)[0]).sum())
    h = 1e-4
    for which, grad in enumerate((dx, dw, db)):
      for at in np.ndindex(grad.shape):
        up, down = [a.copy() for a in args], [a.copy() for a in args]
        up[which][at] += h
        down[which][at] -= h
        want = (loss(up) - loss(down)) / (2 * h)
        # (dz and its sums: 100 roundings of terms up to 40)
        assert abs(grad[at] - want) < 500 * h * h / 6 + 1e-9 + 100 * U32 * 40, (activation, which, at)


@pytest.mark.parametrize('m,k,n', [(1, 512, 512), (70, 520, 136), (300, 64, 300)])
def test_rows_behind_the_outputs_are_left_alone_and_residual_in_place(m, k, n):
  from dqn_zoo_amd import linear
  x, w, b, r = _make(m, k, n, BF16, 4)
  want = linear.linear(x, w, b, activation='gelu', residual=r, save_preact=True)
  wide = torch.full((m + 1, n + 3), 7.0, dtype=BF16, device='cuda')
  wide2 = wide.clone()
  out, pre = wide[:m, 1:n + 1], wide2[:m, 2:n + 2]
  out.copy_(r)
  got = linear.linear(x, w, b, activation='gelu', residual=out, out=out, save_preact=True, preact=pre)
  assert got[0] is out and torch.equal(out, want[0]) and torch.equal(pre, want[1])
  assert (wide[m] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all()
  assert (wide2[m] == 7).all() and (wide2[:, :2] == 7).all() and (wide2[:, n + 2:] == 7).all()
  dy = r
  dxw = torch.full((m + 1, k + 3), 7.0, dtype=BF16, device='cuda')
  dww = torch.full((k + 1, n + 3), 7.0, dtype=BF16, device='cuda')
  a = linear.linear_backward(dy, x, w)
  c = linear.linear_backward(dy, x, w, dx=dxw[:m, 1:k + 1], dw=dww[:k, 1:n + 1])
  for p, q in zip(a, c):
    assert torch.equal(p, q)
  assert (dxw[m] == 7).all() and (dxw[:, 0] == 7).all() and (dxw[:, k + 1:] == 7).all()
  assert (dww[k] == 7).all() and (dww[:, 0] == 7).all() and (dww[:, n + 1:] == 7).all()


def test_what_lies_past_the_edges_does_not_count():
  """NaN behind the rows, and rows after the last, in padded buffers."""
  from dqn_zoo_amd import linear
  for m, k, n in ((5, 72, 40), (130, 136, 264), (3, 33, 65), (70, 8, 8)):
    x, w, b, r = _make(m, k, n, BF16, 4)
    want = linear.linear(x, w, b, residual=r)
    nan = lambda t: torch.full((t.shape[0] + 8, t.shape[1] + 8), float('nan'), dtype=BF16, device='cuda')
    def hide(t):
      big = nan(t)
      big[:t.shape[0], :t.shape[1]] = t
      return big[:t.shape[0], :t.shape[1]]
    got = linear.linear(hide(x), hide(w), b, residual=hide(r))
    assert torch.equal(got, want)
    for p, q in zip(linear.linear_backward(r, x, w), linear.linear_backward(hide(r), hide(x), hide(w))):
      assert torch.equal(p, q)


def test_special_values_stay_in_their_rows_and_columns():
  from dqn_zoo_amd import linear
  x, w, b, _ = _make(70, 136, 72, BF16, 4)
  x[3, 5] = float('nan')
  x[9, 1] = float('inf')
  y = linear.linear(x, w, b, activation='relu')
  bad = ~torch.isfinite(y)
  assert bad[3].all() and not bad[[i for i in range(70) if i not in (3, 9)]].any()
  assert (y[9][torch.isfinite(y[9])] == 0).all()       # relu(-inf)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_activations_far_out(dtype):
  """Infinite and very large pre-activations have the limits' values and slopes, NaN stays NaN."""
  from dqn_zoo_amd import linear
  inf = float('inf')
  far = torch.tensor([inf, -inf, 6e4, -6e4, 40.0, -40.0, 0.0, float('nan')], dtype=dtype, device='cuda')
  x, w = torch.ones(1, 1, dtype=dtype, device='cuda'), torch.zeros(1, 8, dtype=dtype, device='cuda')
  for name in ('relu', 'gelu', 'silu'):
    y, z = linear.linear(x, w, far, activation=name, save_preact=True)
    assert torch.equal(z[0, :7], far[:7]) and torch.isnan(z[0, 7])
    want = torch.tensor([inf, 0, 6e4, 0, 40, 0, 0], dtype=dtype, device='cuda')
    # (silu(-40) is -1.7e-16)
    assert torch.allclose(y[0, :7].float(), want.float(), atol=1e-15, rtol=0) and torch.isnan(y[0, 7]), (name, y)
    dy = torch.ones(1, 8, dtype=dtype, device='cuda')
    _, _, db = linear.linear_backward(dy, x, w, activation=name, preact=z, need=(False, False, True))
    zero = 0.0 if name == 'relu' else 0.5
    want = torch.tensor([1, 0, 1, 0, 1, 0, zero], dtype=dtype, device='cuda')
    assert torch.allclose(db[:7].float(), want.float(), atol=1e-14, rtol=2 * U32) and torch.isnan(db[7]), (name, db)


@pytest.mark.parametrize('m,k,n', [(1, 3136, 512), (300, 264, 520), (8, 4096, 64)])
def test_captured_and_replayed(m, k, n):
  from dqn_zoo_amd import _lib, linear
  x, w, b, r = _make(m, k, n, BF16, 4)
  dy = r.clone()
  calls = lambda **o: linear.linear(x, w, b, activation='gelu', residual=r, save_preact=True, **o)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    first = calls()
    linear.linear_backward(dy, x, w, activation='gelu', preact=first[1])
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
      got = calls()
      grads = linear.linear_backward(dy, x, w, activation='gelu', preact=got[1])
    with pytest.raises(RuntimeError, match='buffers'):
      _lib.capture_graph(side.cuda_stream, calls)
    ws = torch.empty(max(16, linear.workspace_bytes(m, k, n, BF16)), dtype=torch.uint8, device='cuda')
    mine = [torch.empty_like(t) for t in first]
    own = _lib.capture_graph(side.cuda_stream, lambda: calls(out=mine[0], preact=mine[1], workspace=ws))
  for step in range(4):
    x.mul_(-1.5)
    dy.add_(step)
    torch.cuda.synchronize()
    eager = calls()
    eager_grads = linear.linear_backward(dy, x, w, activation='gelu', preact=eager[1])
    graph.replay()
    _lib.check(_lib.load().dz_graph_launch(own, side.cuda_stream), 'dz_graph_launch')
    torch.cuda.synchronize()
    for p, q in zip((*eager, *eager_grads), (*got, *grads)):
      assert torch.equal(p, q)
    for p, q in zip(eager, mine):
      assert torch.equal(p, q)
  _lib.load().dz_graph_destroy(own)


def test_two_streams_at_once():
  from dqn_zoo_amd import linear
  cases = [_make(8, 4096, 256, BF16, 1), _make(600, 512, 700, BF16, 2)]
  want = [linear.linear(x, w, b, residual=r) for x, w, b, r in cases]
  torch.cuda.synchronize()
  streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
  for _ in range(10):
    for i in (0, 1):
      with torch.cuda.stream(streams[i]):
        x, w, b, r = cases[i]
        outs[i].append(linear.linear(x, w, b, residual=r))
  torch.cuda.synchronize()
  assert all(torch.equal(o, want[i]) for i in (0, 1) for o in outs[i])


def test_refusals():
  from dqn_zoo_amd import _lib, linear
  x, w, b, r = _make(4, 6, 8, F32, 1)
  z = torch.zeros
  def refused(error, match, *args, **kw):
    with pytest.raises(error, match=match):
      linear.linear(*args, **kw)
  refused(_lib.HipLibraryError, 'no CPU fallback', x.cpu(), w)
  refused(TypeError, 'must be a tensor', None, w)
  refused(TypeError, 'float32, bfloat16 or float16', x.double(), w)
  refused(TypeError, 'w must be', x, w.half())
  refused(ValueError, 'w must have shape', x, w.t())
  refused(ValueError, 'not empty', x[:0], w)
  refused(ValueError, 'not empty', x, w[:, :0])
  refused(ValueError, 'not empty', x[0], w)
  refused(ValueError, 'adjacent', z(6, 4, device='cuda').t(), w)
  refused(ValueError, 'adjacent', z(1, 6, device='cuda').expand(4, 6), w)
  refused(ValueError, 'stored in rows', x, z(12, 16, device='cuda')[::2, ::2])
  refused(ValueError, 'another device', x, w.cpu())
  refused(ValueError, 'activation', x, w, activation='tanh')
  refused(TypeError, 'b must be', x, w, b.half())
  refused(ValueError, 'b must be contiguous', x, w, b[:7])
  refused(ValueError, 'residual must have', x, w, residual=r[:, :7])
  refused(ValueError, 'preact= is', x, w, preact=r)
  refused(ValueError, 'out must have', x, w, out=z(4, 9, device='cuda'))
  buf = z(5, 8, device='cuda')
  refused(ValueError, 'out shares memory with residual', x, w, residual=buf[:4], out=buf[1:])
  refused(ValueError, 'preact shares memory with out', x, w, out=buf[:4], preact=buf[1:], save_preact=True)
  square = z(6, 6, device='cuda')
  refused(ValueError, 'out shares memory with x', x, square, out=x)
  def back(error, match, *args, **kw):
    with pytest.raises(error, match=match):
      linear.linear_backward(*args, **kw)
  dy = r
  back(ValueError, 'needs preact', dy, x, w, activation='gelu')
  back(ValueError, 'dy must have', dy[:, :7], x, w)
  back(TypeError, 'dy must be', dy.half(), x, w)
  back(ValueError, 'at least one', dy, x, w, need=(False, False, False))
  back(ValueError, 'dx= is given', dy, x, w, dx=x.clone(), need=(False, True, True))
  back(TypeError, 'both', dy.half(), x.half(), w.half(), dw=w.clone(), db=b.half())
  back(ValueError, 'dw, stored', dy, x, w, dw=w.t().contiguous().t())
  back(ValueError, 'dx shares memory with x', dy, x, w, dx=x)
  back(ValueError, 'dw shares memory with w', dy, x, w, dw=w)
  lib = _lib.load()
  n = ctypes.c_int64()
  bad = _lib.LinearArgs()
  assert lib.dz_linear_workspace(ctypes.byref(bad), 0, ctypes.byref(n)) == _lib.DZ_ERR_INVALID_ARG
  assert lib.dz_linear(ctypes.byref(bad), None) == _lib.DZ_ERR_INVALID_ARG
  assert lib.dz_linear_backward(ctypes.byref(bad), None) == _lib.DZ_ERR_INVALID_ARG
