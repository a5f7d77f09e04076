"""NumPy float64 oracle of the policy-training operators (linear, policy loss, AdamW).

Plain restatements of the formulas that include/dqnzoo_hip.h gives for dz_linear_*,
dz_policy_loss and dz_adamw_*; tests compare the HIP kernels with them (checker only).
"""

import numpy as np

MASK64 = (1 << 64) - 1


# ------------------------------------------------------------------ AdamW
def mix64(x):
  x = (np.asarray(x, np.uint64) + np.uint64(0x9E3779B97F4A7C15))
  x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
  x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
  return x ^ (x >> np.uint64(31))


def adamw_noise(seed, step, positions):
  """The two 16-bit draws (for m, for v) of the elements at `positions` of the flat state."""
  with np.errstate(over='ignore'):
    key = mix64(np.uint64(seed) ^ mix64(np.uint64(step)))
    pos = np.asarray(positions, np.uint64)
    h = mix64(key + (pos >> np.uint64(1)))
  shift = np.uint64(32) * (pos & np.uint64(1))
  return ((h >> shift) & np.uint64(0xFFFF)).astype(np.int64), \
      ((h >> (shift + np.uint64(16))) & np.uint64(0xFFFF)).astype(np.int64)


def adamw(p, g, m, v, step, lr, b1, b2, eps, decay, coef=1.0):
  """One float64 update; returns p, m, v."""
  g = g * coef
  m = b1 * m + (1 - b1) * g
  v = b2 * v + (1 - b2) * g * g
  upd = (m / (1 - b1 ** step)) / (np.sqrt(v / (1 - b2 ** step)) + eps)
  return p - lr * (upd + decay * p), m, v


def eight_bit_steps(y, least):
  """Spacing of a format with 3 fraction bits and least normal exponent `least` at y."""
  e = np.floor(np.log2(np.maximum(y, 2.0 ** least)))
  return 2.0 ** (e - 3)


def decode_e4m3(codes):
  c = codes.astype(np.int64)
  mag = c & 127
  val = np.where(mag < 8, mag * 2.0 ** -9, (1 + (mag & 7) / 8) * 2.0 ** ((mag >> 3) - 7.0))
  return np.where(c & 128, -val, val)


def decode_e5m3(codes):
  c = codes.astype(np.int64)
  return np.where(c < 8, c * 2.0 ** -33, (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 31.0))


# ------------------------------------------------------------------ policy loss
def policy_loss(logits, actions, advantages, old_logp, ref_logp=None, weights=None, *, clip_low,
                clip_high, kl_coef, entropy_coef, normalizer=None, grad_scale=1.0):
  """loss, logp, entropy, dlogits in float64; rows of weight 0 are not looked at."""
  x = np.asarray(logits, np.float64)
  n, _ = x.shape
  w = np.ones(n) if weights is None else np.asarray(weights, np.float64)
  norm = w.sum() if normalizer is None else normalizer
  loss, logp, ent, grad = 0.0, np.zeros(n), np.zeros(n), np.zeros_like(x)
  for i in range(n):
    if w[i] == 0:
      continue
    with np.errstate(invalid='ignore', over='ignore'):
      t = x[i] - x[i].max()
      lse = np.log(np.exp(t).sum())
      lp = t - lse
      p = np.exp(lp)
      plp = np.where(p > 0, p * lp, 0 * p)
      a, adv = int(actions[i]), float(advantages[i])
      logp[i], ent[i] = lp[a], -plp.sum()
      rho = np.exp(lp[a] - old_logp[i])
      free, held = rho * adv, np.clip(rho, 1 - clip_low, 1 + clip_high) * adv
      value, slope = -min(free, held) - entropy_coef * ent[i], -free if free <= held else 0.0
      if ref_logp is not None and kl_coef:
        d = ref_logp[i] - lp[a]
        value += kl_coef * (np.expm1(d) - d)
        slope -= kl_coef * np.expm1(d)
      s = w[i] / norm if norm else 0.0
      loss += s * value
      onehot = np.zeros_like(p)
      onehot[a] = 1
      grad[i] = grad_scale * s * (slope * (onehot - p) + entropy_coef * (plp + p * ent[i]))
  return loss, logp, ent, grad


# ------------------------------------------------------------------ linear
def erf(z):
  from scipy import special
  return special.erf(z)


def act(z, name):
  if name == 'none':
    return z
  if name == 'relu':
    return np.where(z < 0, 0.0, z)
  if name == 'gelu':
    return 0.5 * z * (1 + erf(z / np.sqrt(2)))
  return z / (1 + np.exp(-z))


def act_slope(z, name):
  if name == 'none':
    return np.ones_like(z)
  if name == 'relu':
    return (z > 0).astype(np.float64)
  if name == 'gelu':
    return 0.5 * (1 + erf(z / np.sqrt(2))) + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
  s = 1 / (1 + np.exp(-z))
  return s * (1 + z * (1 - s))


def linear(x, w, b=None, activation='none', residual=None):
  """y, z in float64."""
  z = x @ w
  if b is not None:
    z = z + b
  y = act(z, activation)
  return (y if residual is None else y + residual), z


def linear_backward(dy, x, w, activation='none', preact=None):
  """dx, dw, db in float64."""
  dz = dy if activation == 'none' else dy * act_slope(preact, activation)
  return dz @ w.T, x.T @ dz, dz.sum(0)
