// The clipped policy loss with a KL term and an entropy bonus, and its gradient with respect to
// the logits, reading the logits once where a row fits the registers of its workgroup.
//
// Row i with logits x, action a, advantage A, weight w:
//   t_j = x_j - max x,  l = log sum exp t,  log p_j = t_j - l,  H = -sum_j p_j log p_j
//   rho = exp(log p_a - old),  d = ref - log p_a
//   value = -min(rho A, clip(rho, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1) - ent H
//   loss  = sum_i w_i value_i / norm
//   d loss / d x_j = w / norm ( s (1[j = a] - p_j) + ent p_j (log p_j + H) ),
//   s = -rho A [rho A <= clip(rho) A] - kl (exp(d) - 1)
//
// log p_j + H = t_j - mean of t, so that a gradient element is p_j (ent (t_j - mean t) - s), and at
// j = a, s more.  Rows held by a team run in base 2: with c = log2 e, u_j = c x_j - c max x is one
// fused multiply-add, e_j = 2^u_j; c max x is rounded, the same for every element, and what the
// rounding left (one more fused multiply-add a row) is taken out of log sum e.  A gradient element is
//   e_j (k1 u_j + k0),   k1 = ent ln2 / S,  k0 = (-ent mean t - s) / S,
// times the row's factor: one exponential and five other operations an element and pass.  u is held
// above -200 (2^-200 is 0 in float32), so that a masked logit (-inf, or the type's lowest value)
// gives 0 and not 0 * inf.  A row whose maximum is beyond 10^38 (every logit the lowest value)
// takes x - max first: c max overflows there.  A row in which every logit is -inf, or one is NaN or
// +inf, is NaN, as its log-softmax is: its maximum is not finite (the maxima keep NaN); a row of
// weight 0 is not read.
//
// Bound: bytes (the logits in and the gradient out).  Four forms by the size of a row:
//   * few: 1 - 32 lanes to a row, 8 elements a lane (up to 256 logits: actions; the row's own terms,
//     a hundred instructions, are what is to be shared by rows).  One workgroup does
//     a small problem, weights' sum and loss included, in one launch;
//   * team: 64, 256 or 1024 threads hold the row in registers, 1 - 16 16-byte vectors each;
//   * split: rows that are longer than a workgroup's registers, or too few of them to fill the chip:
//     pieces of a row are reduced by one launch and turned into the gradient by the next, for as
//     many rows at a time as the 256 MB Infinity Cache holds, so that the second read stays on it.
// The rows' values are summed in double in a fixed order.
#include <type_traits>

#include "dz_elem.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kWeightBlocks = 64;    // partial sums of the weights: one wave folds them

struct LossArgs {
  const void* logits; int64_t ld;
  void* grad; int64_t ldg;           // NULL: values only
  const int64_t* actions;
  const float* advantages; const float* old_logp; const float* ref_logp; const float* weights;
  float* logp; float* entropy; float* loss;
  uint32_t* status;
  double* values;                    // one partial loss per workgroup (row in the split form)
  const double* weight_sums;         // kWeightBlocks partial sums, or NULL: inv_norm holds
  double inv_norm;
  double low, high, kl, ent_coef;    // of the values, in double: a coefficient's rounding is the same in every row
  float ent, grad_scale;
  int64_t rows; int classes;
};

struct RowSums { float top, s, t; };   // max x, sum e, sum e u  (u relative to top)

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN stays
__device__ __forceinline__ bool huge(float top) { return !(fabsf(top) < 1e38f); }
__device__ __forceinline__ float held(float u) { return fmaxf(u, -200.0f); }
// u of x in a row of maximum `top`: FAR where top is huge
template <bool FAR>
__device__ __forceinline__ float unit(float x, float top) {
  return held(FAR ? (x - top) * kLog2e : __builtin_fmaf(x, kLog2e, -(top * kLog2e)));
}

template <int W>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
  for (int o = W / 2; o; o >>= 1) x = maximum(x, __shfl_xor(x, o));
  return x;
}
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int o = W / 2; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// `part` in units of the whole row's maximum (a part of masked logits alone adds 0: f is held too).
// The rounded products are subtracted, as the elements' u were formed.
__device__ __forceinline__ void rescale(RowSums& part, float top) {
  const float f = held(huge(top) ? (part.top - top) * kLog2e : part.top * kLog2e - top * kLog2e);
  const float g = exp2_fast(f);
  part.t = g * __builtin_fmaf(part.s, f, part.t);
  part.s = g * part.s;
}

// what the rounding of c * top left: u = c (x - top) + residue
__device__ __forceinline__ float residue(float top) {
  return huge(top) ? 0.0f : __builtin_fmaf(top, kLog2e, -(top * kLog2e));
}

// The sum's logarithm, once a row: logf is 5e-8 low on average, which a loss of 10^5 rows whose terms
// cancel shows (8e-6 of it).
__device__ __forceinline__ float log_sum(float s) { return (float)log((double)s); }

struct RowOut { double value; float logp, entropy, slope; };

// `lse`: log sum exp t; `mean`: of t; both of the natural t = x - top
__device__ __forceinline__ RowOut row_values(const LossArgs& a, float top, float lse, float mean, float xa, float adv,
                                             float old, float ref) {
  RowOut o;
  if (!(fabsf(top) < __builtin_inff())) lse = __builtin_nanf("");
  o.logp = (xa - top) - lse;
  o.entropy = lse - mean;
  const double rho = (double)expf(o.logp - old), free = rho * (double)adv;
  const double kept = (rho < a.low ? a.low : rho > a.high ? a.high : rho) * (double)adv;
  o.value = -(free <= kept ? free : kept);
  double slope = free <= kept ? -free : 0.0;
  if (free != free || kept != kept) o.value = slope = __builtin_nan("");
  if (a.ref_logp) {
    const double d = (double)ref - (double)o.logp, e = expm1(d);
    o.value += a.kl * (e - d);
    slope -= a.kl * e;
  }
  o.value -= a.ent_coef * (double)o.entropy;
  o.slope = (float)slope;
  return o;
}
// The slope alone, in float32: what the gradient's threads need.
__device__ __forceinline__ float row_slope(const LossArgs& a, float logp, float adv, float old, float ref) {
  const float rho = expf(logp - old), free = rho * adv;
  const float kept = (rho < (float)a.low ? (float)a.low : rho > (float)a.high ? (float)a.high : rho) * adv;
  float slope = free <= kept ? -free : 0.0f;
  if (free != free || kept != kept) slope = __builtin_nanf("");
  return a.ref_logp ? __builtin_fmaf(-(float)a.kl, expm1f(ref - logp), slope) : slope;
}
// A row in base 2 for its gradient (k1, k0 without the row's factor; the slope) ...
__device__ __forceinline__ float row_gradient(const LossArgs& a, const RowSums& r, float xa, float adv, float old,
                                              float ref, float& k1, float& k0) {
  const float inv_s = 1.0f / r.s, left = residue(r.top) * kLn2;
  const float slope = row_slope(a, (xa - r.top) - (logf(r.s) - left), adv, old, ref);
  const float scale = fabsf(r.top) < __builtin_inff() ? inv_s : __builtin_nanf("");
  k1 = a.ent * kLn2 * scale;
  k0 = __builtin_fmaf(-a.ent, r.t * inv_s * kLn2, -slope) * scale;
  return slope;
}
// ... and for its value (one wave of a team: 200 instructions of double are 20 us of a 370 us launch
// if sixteen waves do them).
__device__ __forceinline__ RowOut row_values(const LossArgs& a, const RowSums& r, float xa, float adv, float old,
                                             float ref) {
  const float left = residue(r.top);
  return row_values(a, r.top, log_sum(r.s) - left * kLn2, (r.t / r.s - left) * kLn2, xa, adv, old, ref);
}

// d loss / d x_j without the action's own term; k1 and k0 have the row's factor
template <bool FAR>
__device__ __forceinline__ float gradient(float x, float top, float k1, float k0) {
  const float u = unit<FAR>(x, top);
  return exp2_fast(u) * __builtin_fmaf(k1, u, k0);
}

__device__ __forceinline__ double inverse_norm(const LossArgs& a) {   // (whole waves)
  if (!a.weight_sums) return a.inv_norm;
  const double s = wave_sum_f64(a.weight_sums[threadIdx.x & 63]);
  return s != 0.0 ? 1.0 / s : 0.0;
}

struct RowIn { float w, adv, old, ref, xa; int64_t action; };

template <typename T>
__device__ __forceinline__ RowIn row_in(const LossArgs& a, int64_t row) {
  RowIn i;
  i.w = a.weights ? a.weights[row] : 1.0f;
  i.adv = a.advantages[row]; i.old = a.old_logp[row];
  i.ref = a.ref_logp ? a.ref_logp[row] : 0.0f;
  i.xa = __builtin_nanf("");
  i.action = a.actions[row];
  if (i.w == 0.0f) return i;
  if (i.action >= 0 && i.action < a.classes) {
    i.xa = (float)((const T*)a.logits)[row * a.ld + i.action];
  } else {                      // no such class: the row, and with it the loss, is NaN
    i.action = -1;
    if (a.status) atomicOr(a.status, DZ_ST_BAD_INDEX);
  }
  return i;
}

__global__ __launch_bounds__(256) void loss_weights_kernel(const float* __restrict__ w, int64_t n,
                                                           double* __restrict__ sums) {
  double s = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) s += (double)w[i];
  __shared__ double red[4];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) sums[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(1024) void loss_total_kernel(LossArgs a, int64_t n) {
  const double inv = inverse_norm(a);
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += a.values[i];
  __shared__ double red[16];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; ++i) s += red[i];
  *a.loss = (float)(s * inv);
}

// ---- few: G lanes to a row --------------------------------------------------
// ALL: the one workgroup takes every row in turn, and the weights' sum and the loss with them.  (In
// natural units and with the library's functions: nothing here is bound by the elements.)
template <typename T, int G, bool ALL>
__global__ __launch_bounds__(256) void loss_few_kernel(LossArgs a) {
  constexpr int E = 8, ROWS = 256 / G;
  const int lane = threadIdx.x % G;
  __shared__ double red[4];
  double inv, total = 0.0;
  if (ALL && a.weights && a.inv_norm == 0.0) {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < a.rows; i += 256) s += (double)a.weights[i];
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    inv = s != 0.0 ? 1.0 / s : 0.0;
  } else {
    inv = inverse_norm(a);
  }
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
    const int64_t row = base + threadIdx.x / G;
    const bool live = row < a.rows;
    RowIn in{};
    if (live) in = row_in<T>(a, row);
    const bool used = live && in.w != 0.0f;
    const T* x = (const T*)a.logits + row * a.ld;
    float v[E];
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = j * G + lane;
      v[j] = used && c < a.classes ? (float)x[c] : -__builtin_inff();
      top = maximum(top, v[j]);
    }
    top = lanes_max<G>(top);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (j * G >= a.classes) break;   // (uniform)
      const float d = fmaxf(v[j] - top, -200.0f), e = expf(d);
      v[j] = d;
      s += e;
      t = __builtin_fmaf(e, d, t);
    }
    s = lanes_sum<G>(s);
    t = lanes_sum<G>(t);
    const float mean = t / s;
    const RowOut o = row_values(a, top, log_sum(s), mean, in.xa, in.adv, in.old, in.ref);
    const float factor = (float)(used ? (double)in.w * inv * (double)a.grad_scale : 0.0);
    if (live && lane == 0) {
      a.logp[row] = used ? o.logp : 0.0f;
      a.entropy[row] = used ? o.entropy : 0.0f;
      if (used) total += (double)in.w * o.value;
    }
    if (a.grad && live) {
      T* g = (T*)a.grad + row * a.ldg;
      const float inv_s = fabsf(top) < __builtin_inff() ? 1.0f / s : __builtin_nanf("");
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = j * G + lane;
        if (c >= a.classes) continue;
        float y = expf(v[j]) * inv_s * (__builtin_fmaf(a.ent, v[j] - mean, -o.slope) * factor);
        if (c == in.action) y += o.slope * factor;
        g[c] = (T)(used ? y : 0.0f);
      }
    }
  }
  total = wave_sum_f64(total);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = (red[0] + red[1]) + (red[2] + red[3]);
    if (ALL) *a.loss = (float)(total * inv);
    else a.values[blockIdx.x] = total;
  }
}

// ---- team: TEAM threads hold a row -------------------------------------------
// A thread's part of a row, as it lies in memory.  `forget` between the passes: the compiler would
// keep the float32 values of the first for the second, twice the registers (8 vectors of bf16 in
// 1024 threads: 111 registers against 56, so one workgroup per CU and not two; 16 vectors spill).
template <typename T, int NV>
struct RowRegs {
  static constexpr int VE = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(4))) uint32_t Words;
  Words w[NV];

  template <int PLACE>   // (another text at each place: equal ones of two branches would be hoisted)
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("; pass %1" : "+v"(w[i]) : "n"(PLACE));
  }
  __device__ __forceinline__ DzPack<T, VE> get(int i) const { return __builtin_bit_cast(DzPack<T, VE>, w[i]); }
  __device__ __forceinline__ float at(int i, int j) const { return (float)get(i).v[j]; }
};

// The 16 bytes from element c of a row of n that end behind it: what is there, and -inf (a rolled
// loop: one thread of a row has such a vector, and eight two-byte loads each would cost registers).
template <typename T>
__device__ __forceinline__ typename RowRegs<T, 1>::Words row_end(const T* x, int c, int n) {
  typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Raw;
  const uint64_t none = __builtin_bit_cast(Raw, (T)-__builtin_inff());
  const uint64_t fill = sizeof(T) == 2 ? none * 0x0001000100010001ull : none * 0x0000000100000001ull;
  uint64_t q[2] = {fill, fill};
#pragma unroll 1
  for (int j = 0; c + j < n; ++j) {
    const int bit = j * 8 * (int)sizeof(T);
    const uint64_t flip = (none ^ (uint64_t)__builtin_bit_cast(Raw, x[c + j])) << (bit & 63);
    q[0] ^= bit < 64 ? flip : 0;
    q[1] ^= bit < 64 ? 0 : flip;
  }
  typename RowRegs<T, 1>::Words w;
  w[0] = (uint32_t)q[0]; w[1] = (uint32_t)(q[0] >> 32); w[2] = (uint32_t)q[1]; w[3] = (uint32_t)(q[1] >> 32);
  return w;
}

// vector i of thread t is vector i * TEAM + t of the row; what is past the row is -inf
template <typename T, int TEAM, int NV>
__device__ __forceinline__ void load_row(const T* x, int n, int tid, RowRegs<T, NV>& r) {
  constexpr int VE = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TEAM + tid) * VE;
    r.w[i] = c + VE <= n ? __builtin_bit_cast(typename RowRegs<T, NV>::Words, dz_load<T, VE>(x + c)) : row_end<T>(x, c, n);
  }
}

template <bool FAR, typename T, int NV>
__device__ __forceinline__ void sum_exponentials(RowRegs<T, NV>& r, RowSums& o) {
  r.template forget<FAR>();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) {
      const float u = unit<FAR>(r.at(i, j), o.top), e = exp2_fast(u);
      o.s += e;
      o.t = __builtin_fmaf(e, u, o.t);
    }
    __builtin_amdgcn_sched_barrier(0);   // (one vector's values at a time: registers)
  }
}

template <typename T, int NV>
__device__ __forceinline__ RowSums sum_row(RowRegs<T, NV>& r) {   // one wave's part
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(T); ++j) m = maximum(m, r.at(i, j));
    __builtin_amdgcn_sched_barrier(0);
  }
  RowSums o{lanes_max<64>(m), 0.f, 0.f};
  if (huge(o.top)) sum_exponentials<true>(r, o);
  else sum_exponentials<false>(r, o);
  o.s = lanes_sum<64>(o.s);
  o.t = lanes_sum<64>(o.t);
  return o;
}

template <bool FAR, typename T, int TEAM, int NV>
__device__ __forceinline__ void store_rows(T* g, int n, int tid, RowRegs<T, NV>& x, float top, float k1, float k0,
                                           float own, int64_t action) {
  constexpr int VE = 16 / sizeof(T);
  x.template forget<2 + FAR>();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TEAM + tid) * VE;
    if (c >= n) break;
    float y[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) y[j] = gradient<FAR>(x.at(i, j), top, k1, k0);
    if (action >= c && action < c + VE) {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (c + j == action) y[j] += own;
    }
    if (c + VE <= n) {
      dz_store<T, VE>(g + c, dz_round<T, VE>(y));
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (c + j < n) g[c + j] = (T)y[j];
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <typename T, int TEAM, int NV>
__device__ __forceinline__ void store_gradient(T* g, int n, int tid, RowRegs<T, NV>& x, const RowSums& r,
                                               float slope, float k1, float k0, float factor, int64_t action,
                                               bool used) {
  constexpr int VE = 16 / sizeof(T);
  if (!used) {
    DzPack<T, VE> zero;
#pragma unroll
    for (int j = 0; j < VE; ++j) zero.v[j] = (T)0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TEAM + tid) * VE;
      if (c + VE <= n) {
        dz_store<T, VE>(g + c, zero);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (c + j < n) g[c + j] = (T)0.0f;
      }
    }
    return;
  }
  k1 *= factor;
  k0 *= factor;
  const float own = slope * factor;
  if (huge(r.top)) store_rows<true, T, TEAM, NV>(g, n, tid, x, r.top, k1, k0, own, action);
  else store_rows<false, T, TEAM, NV>(g, n, tid, x, r.top, k1, k0, own, action);
}

template <typename T, int TEAM, int NV>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM, NV <= 8 ? 8 : 4) void loss_team_kernel(LossArgs a) {
  constexpr int THREADS = TEAM < 256 ? 256 : TEAM, PER = THREADS / TEAM, WAVES = TEAM / 64;
  const int tid = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int64_t row = (int64_t)blockIdx.x * PER + team;
  __shared__ RowSums parts[THREADS / 64];
  __shared__ double vals[PER];
  const double inv = inverse_norm(a);
  const bool live = row < a.rows;
  RowIn in{};
  if (live) in = row_in<T>(a, row);
  const bool used = live && in.w != 0.0f;
  RowRegs<T, NV> x;
  RowSums r{0.f, 1.f, 0.f};
  if (used) {
    load_row<T, TEAM, NV>((const T*)a.logits + row * a.ld, a.classes, tid, x);
    r = sum_row<T, NV>(x);
  }
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = r;
    __syncthreads();
    // lane k of every wave takes part k
    const int k = threadIdx.x & 63;
    RowSums q = k < WAVES ? parts[k] : RowSums{-__builtin_inff(), 0.f, 0.f};
    r.top = __shfl(lanes_max<WAVES>(q.top), 0);
    rescale(q, r.top);
    r.s = __shfl(lanes_sum<WAVES>(q.s), 0);
    r.t = __shfl(lanes_sum<WAVES>(q.t), 0);
  }
  const float factor = (float)(used ? (double)in.w * inv * (double)a.grad_scale : 0.0);
  if (a.grad && live) {
    float k1, k0;
    const float slope = row_gradient(a, r, in.xa, in.adv, in.old, in.ref, k1, k0);
    store_gradient<T, TEAM, NV>((T*)a.grad + row * a.ldg, a.classes, tid, x, r, slope, k1, k0, factor, in.action, used);
  }
  if (tid < 64) {   // (one wave of the team)
    const RowOut o = row_values(a, r, in.xa, in.adv, in.old, in.ref);
    if (tid == 0) {
      if (live) {
        a.logp[row] = used ? o.logp : 0.0f;
        a.entropy[row] = used ? o.entropy : 0.0f;
      }
      vals[team] = used ? (double)in.w * o.value : 0.0;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < PER; ++i) s += vals[i];
    a.values[blockIdx.x] = s;
  }
}

// ---- split: pieces of a row ---------------------------------------------------
constexpr int kSplitVectors = 4;
template <typename T> constexpr int split_piece() { return 256 * kSplitVectors * (16 / (int)sizeof(T)); }

struct SplitWs { RowSums* parts; float* xa; int64_t first; int pieces; };

template <typename T>
__global__ __launch_bounds__(256) void loss_split_sums_kernel(LossArgs a, SplitWs ws) {
  const int64_t local = blockIdx.x / ws.pieces, row = ws.first + local;
  const int piece = blockIdx.x % ws.pieces, c0 = piece * split_piece<T>();
  if (a.weights && a.weights[row] == 0.0f) return;
  if (piece == 0 && threadIdx.x == 0) ws.xa[local] = row_in<T>(a, row).xa;
  RowRegs<T, kSplitVectors> x;
  load_row<T, 256, kSplitVectors>((const T*)a.logits + row * a.ld + c0, min(a.classes - c0, split_piece<T>()),
                                  threadIdx.x, x);
  RowSums q = sum_row<T, kSplitVectors>(x);
  __shared__ RowSums red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = q;
  __syncthreads();
  if (threadIdx.x) return;
  RowSums r{maximum(maximum(red[0].top, red[1].top), maximum(red[2].top, red[3].top)), 0.f, 0.f};
  for (int i = 0; i < 4; ++i) {
    q = red[i];
    rescale(q, r.top);
    r.s += q.s;
    r.t += q.t;
  }
  ws.parts[local * ws.pieces + piece] = r;
}

template <typename T>
__global__ __launch_bounds__(256) void loss_split_gradient_kernel(LossArgs a, SplitWs ws) {
  const int64_t local = blockIdx.x / ws.pieces, row = ws.first + local;
  const int piece = blockIdx.x % ws.pieces, c0 = piece * split_piece<T>();
  const float w = a.weights ? a.weights[row] : 1.0f;
  const bool used = w != 0.0f;
  const double inv = inverse_norm(a);
  RowRegs<T, kSplitVectors> x;
  const int n = min(a.classes - c0, split_piece<T>());
  RowSums r{0.f, 1.f, 0.f};
  float slope = 0.f, k1 = 0.f, k0 = 0.f;
  const float adv = a.advantages[row], old = a.old_logp[row], ref = a.ref_logp ? a.ref_logp[row] : 0.0f;
  int64_t action = a.actions[row];
  if (used) {
    if (a.grad) load_row<T, 256, kSplitVectors>((const T*)a.logits + row * a.ld + c0, n, threadIdx.x, x);
    const RowSums* parts = ws.parts + local * ws.pieces;   // every wave folds the row's parts, in one order
    float top = -__builtin_inff();
    for (int i = threadIdx.x & 63; i < ws.pieces; i += 64) top = maximum(top, parts[i].top);
    r.top = lanes_max<64>(top);
    r.s = r.t = 0.f;
    for (int i = threadIdx.x & 63; i < ws.pieces; i += 64) {
      RowSums q = parts[i];
      rescale(q, r.top);
      r.s += q.s;
      r.t += q.t;
    }
    r.s = lanes_sum<64>(r.s);
    r.t = lanes_sum<64>(r.t);
    slope = row_gradient(a, r, ws.xa[local], adv, old, ref, k1, k0);
  }
  const float factor = (float)(used ? (double)w * inv * (double)a.grad_scale : 0.0);
  if (a.grad)
    store_gradient<T, 256, kSplitVectors>((T*)a.grad + row * a.ldg + c0, n, threadIdx.x, x, r, slope, k1, k0,
                                          factor, action - c0, used);
  if (piece == 0 && threadIdx.x < 64) {
    const RowOut o = row_values(a, r, used ? ws.xa[local] : 0.0f, adv, old, ref);
    if (threadIdx.x) return;
    a.logp[row] = used ? o.logp : 0.0f;
    a.entropy[row] = used ? o.entropy : 0.0f;
    a.values[row] = used ? (double)w * o.value : 0.0;
  }
}

// ---- host ----------------------------------------------------------------------
enum class Form { kOne, kFew, kTeam, kSplit };

struct Plan {
  Form form;
  int lanes;         // few: lanes to a row
  int team, vectors; // team
  int64_t blocks;    // workgroups of the main launch = partial losses
  int pieces; int64_t group;   // split: pieces of a row, rows in one pair of launches
  int64_t ws_bytes;
};

constexpr int64_t kCacheBytes = 128ll << 20;
constexpr int64_t kMostGroups = 1 << 20, kMaxThreads = 1ll << 32;   // a launch has fewer than kMaxThreads threads

Plan make_plan(int dtype, int64_t rows, int classes) {
  Plan p{};
  const int ve = dtype == DZ_F32 ? 4 : 8;
  int64_t bytes = kWeightBlocks * 8;
  if (classes <= 256) {
    p.lanes = 1;
    while (p.lanes * 8 < classes) p.lanes *= 2;
    const int64_t per = 256 / p.lanes;
    p.blocks = (rows + per - 1) / per;
    if (p.blocks > kMostGroups) p.blocks = kMostGroups;   // (which go round)
    p.form = p.blocks <= 2 ? Form::kOne : Form::kFew;
    p.ws_bytes = p.form == Form::kOne ? 0 : bytes + p.blocks * 8;
    return p;
  }
  const int vecs = (classes + ve - 1) / ve;
  p.pieces = (classes + 256 * kSplitVectors * ve - 1) / (256 * kSplitVectors * ve);
  // Few rows leave most of the chip idle in the team form.
  if (vecs > 16 * 1024 || (p.pieces >= 4 && rows < 128)) {
    p.form = Form::kSplit;
    p.group = kCacheBytes / ((int64_t)classes * dz_elem_bytes(dtype));
    if (p.group < 1) p.group = 1;
    if (p.group > rows) p.group = rows;
    if (p.group * p.pieces >= (1ll << 31)) p.group = ((1ll << 31) - 1) / p.pieces;
    p.blocks = rows;
    p.ws_bytes = bytes + rows * 8 + p.group * p.pieces * (int64_t)sizeof(RowSums) + p.group * 4;
    return p;
  }
  p.form = Form::kTeam;
  p.team = vecs <= 64 * 4 ? 64 : vecs <= 256 * 8 ? 256 : 1024;
  p.vectors = 1;
  while (p.vectors * p.team < vecs) p.vectors *= 2;
  const int per = p.team < 256 ? 256 / p.team : 1;
  p.blocks = (rows + per - 1) / per;
  p.ws_bytes = bytes + p.blocks * 8;
  return p;
}

template <typename T, int TEAM, int NV>
void launch_team(const LossArgs& k, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((loss_team_kernel<T, TEAM, NV>), dim3(grid), dim3(TEAM < 256 ? 256 : TEAM), 0, s, k);
}
template <typename T, bool ALL>
void launch_few(const LossArgs& k, int lanes, unsigned grid, hipStream_t s) {
  switch (lanes) {
    case 1: hipLaunchKernelGGL((loss_few_kernel<T, 1, ALL>), dim3(grid), dim3(256), 0, s, k); break;
    case 2: hipLaunchKernelGGL((loss_few_kernel<T, 2, ALL>), dim3(grid), dim3(256), 0, s, k); break;
    case 4: hipLaunchKernelGGL((loss_few_kernel<T, 4, ALL>), dim3(grid), dim3(256), 0, s, k); break;
    case 8: hipLaunchKernelGGL((loss_few_kernel<T, 8, ALL>), dim3(grid), dim3(256), 0, s, k); break;
    case 16: hipLaunchKernelGGL((loss_few_kernel<T, 16, ALL>), dim3(grid), dim3(256), 0, s, k); break;
    default: hipLaunchKernelGGL((loss_few_kernel<T, 32, ALL>), dim3(grid), dim3(256), 0, s, k); break;
  }
}

template <typename T>
int launch_rows(const LossArgs& k, const Plan& p, void* tail, hipStream_t s) {
  const unsigned grid = (unsigned)p.blocks;
  switch (p.form) {
    case Form::kOne: launch_few<T, true>(k, p.lanes, 1, s); break;
    case Form::kFew: launch_few<T, false>(k, p.lanes, grid, s); break;
    case Form::kTeam:
      switch (p.team * 100 + p.vectors) {
        case 6401: launch_team<T, 64, 1>(k, grid, s); break;
        case 6402: launch_team<T, 64, 2>(k, grid, s); break;
        case 6404: launch_team<T, 64, 4>(k, grid, s); break;
        case 25602: launch_team<T, 256, 2>(k, grid, s); break;
        case 25604: launch_team<T, 256, 4>(k, grid, s); break;
        case 25608: launch_team<T, 256, 8>(k, grid, s); break;
        case 102404: launch_team<T, 1024, 4>(k, grid, s); break;
        case 102408: launch_team<T, 1024, 8>(k, grid, s); break;
        case 102416: launch_team<T, 1024, 16>(k, grid, s); break;
        default: return DZ_ERR_UNSUPPORTED;
      }
      break;
    case Form::kSplit: {
      SplitWs ws;
      ws.parts = (RowSums*)tail;
      ws.xa = (float*)(ws.parts + p.group * p.pieces);
      ws.pieces = p.pieces;
      for (ws.first = 0; ws.first < k.rows; ws.first += p.group) {
        const int64_t n = k.rows - ws.first < p.group ? k.rows - ws.first : p.group;
        const dim3 g((unsigned)(n * p.pieces));
        hipLaunchKernelGGL((loss_split_sums_kernel<T>), g, dim3(256), 0, s, k, ws);
        DZ_LAUNCH_CHECK();
        hipLaunchKernelGGL((loss_split_gradient_kernel<T>), g, dim3(256), 0, s, k, ws);
        DZ_LAUNCH_CHECK();
      }
      break;
    }
  }
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

bool sizes_ok(int dtype, int64_t rows, int64_t classes) {
  return dz_is_dtype(dtype) && rows > 0 && rows < (1ll << 31) && classes > 0 && classes < (1ll << 30);
}

}  // namespace

extern "C" int dz_policy_loss_workspace(int dtype, int64_t rows, int64_t classes, int64_t* bytes) {
  DZ_REQUIRE(bytes && sizes_ok(dtype, rows, classes));
  *bytes = make_plan(dtype, rows, (int)classes).ws_bytes;
  return DZ_OK;
}

extern "C" int dz_policy_loss(const dz_policy_loss_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(a && sizes_ok(a->dtype, a->rows, a->classes));
  DZ_REQUIRE(a->logits && a->actions && a->advantages && a->old_logp && a->logp && a->entropy && a->loss);
  DZ_REQUIRE(a->ld >= a->classes && (!a->dlogits || a->ldg >= a->classes));
  DZ_REQUIRE(((uintptr_t)a->ws & 15) == 0);
  DZ_REQUIRE(a->clip_low >= 0.0 && a->clip_high >= 0.0 && a->normalizer >= 0.0 && a->normalizer < __builtin_inf());
  const Plan p = make_plan(a->dtype, a->rows, (int)a->classes);
  DZ_REQUIRE(p.form != Form::kTeam || p.blocks * (p.team < 256 ? 256 : p.team) < kMaxThreads);
  DZ_REQUIRE(p.ws_bytes == 0 || (a->ws && a->ws_bytes >= p.ws_bytes));
  const hipStream_t s = dz_s(stream);
  double* sums = (double*)a->ws;
  const bool summed = a->weights && !(a->normalizer > 0.0);
  LossArgs k{};
  k.logits = a->logits; k.ld = a->ld; k.grad = a->dlogits; k.ldg = a->ldg;
  k.actions = a->actions; k.advantages = a->advantages; k.old_logp = a->old_logp;
  k.ref_logp = a->kl_coef != 0.0 ? a->ref_logp : nullptr;   // (0 * inf)
  k.weights = a->weights;
  k.logp = a->logp; k.entropy = a->entropy; k.loss = a->loss; k.status = a->status;
  k.values = sums + kWeightBlocks;
  k.weight_sums = summed && p.form != Form::kOne ? sums : nullptr;
  // 0 in the one-workgroup form means: sum the weights
  k.inv_norm = summed ? 0.0 : 1.0 / (a->normalizer > 0.0 ? a->normalizer : (double)a->rows);
  k.low = 1.0 - a->clip_low; k.high = 1.0 + a->clip_high;
  k.kl = a->kl_coef; k.ent_coef = a->entropy_coef; k.ent = (float)a->entropy_coef; k.grad_scale = a->grad_scale;
  k.rows = a->rows; k.classes = (int)a->classes;
  if (k.weight_sums) {
    hipLaunchKernelGGL(loss_weights_kernel, dim3(kWeightBlocks), dim3(256), 0, s, a->weights, a->rows, sums);
    DZ_LAUNCH_CHECK();
  }
  int rc = DZ_OK;
  dz_for_dtype(a->dtype, [&](auto t) { rc = launch_rows<decltype(t)>(k, p, k.values + p.blocks, s); });
  if (rc != DZ_OK) return rc;
  if (p.form != Form::kOne) {
    hipLaunchKernelGGL(loss_total_kernel, dim3(1), dim3(1024), 0, s, k, p.blocks);
    DZ_LAUNCH_CHECK();
  }
  return DZ_OK;
}
