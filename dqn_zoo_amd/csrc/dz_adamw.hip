// AdamW over a list of tensors: one launch reads every gradient once, and every parameter and
// moment once and writes them back.
//
//   g = grad * coef                       coef = grad_scale * min(1, max_norm / (grad_scale |grad|))
//   m = b1 m + (1 - b1) g ;  v = b2 v + (1 - b2) g^2
//   p = p - lr ( (m / bc1) / (sqrt(v / bc2) + eps) + decay p )
//
// in float32, in this order (no contraction), on the float32 master copy where there is one.
//
// The moments are held in float32, or in 8 bits per element with one float32 scale per 256
// elements (a block never spans two tensors):
//   m: e4m3 (4 exponent bits, 3 fraction bits) in units of the block's largest |m| / 448;
//   v: unsigned, 5 exponent and 3 fraction bits, in units of the block's largest v / 1.875; the
//      smallest code stands for the largest / 2^34, so that a block may hold gradients whose sizes
//      differ by 10^5, and a v that is not 0 never becomes 0 (m / eps would follow).
// Both are rounded up or down at random with the probabilities that keep the mean.  Rounding to
// the nearest would lose the average itself: v moves by (1 - b2) = 0.1 % a step, half a step of
// the format is 3 - 6 %, so v would never decay.  The 16 random bits of an element come from the
// counter-based generator of the library's other draws (splitmix64), keyed by (seed, step), one
// 64-bit draw per two elements; the result depends on nothing else.
//
// Bound: bytes.  28 bytes per element with everything in float32, 20 with bf16 parameters and
// gradients, master weights and 8-bit moments, against about 60 instructions.
#include "dz_elem.h"

namespace {

constexpr int kBlock = 256;             // elements to a scale = one wave's elements in a round
constexpr int kRounds = 4;              // rounds of a wave
constexpr int kChunk = 4 * kRounds * kBlock;   // elements of one workgroup (4 waves)
static_assert(kChunk == DZ_ADAMW_CHUNK && kBlock == DZ_ADAMW_STATE_BLOCK, "the header's sizes");
constexpr float kTiny = 0x1p-118f;      // a block whose largest is below this is all zero
constexpr int kUpload = 448;            // gradient pointers in one launch's arguments

// what the one-block launch leaves for the update: float words of args.scalars
enum { kNorm = 0, kCoef = 1, kBc1 = 2, kBc2 = 3, kKey = 4 /* two words */ };

__device__ __forceinline__ uint64_t adamw_mix64(uint64_t x) {   // splitmix64
  x += 0x9E3779B97F4A7C15ull;
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

struct UploadArgs { const void* g[kUpload]; };
__global__ void adamw_upload_kernel(UploadArgs a, const void** table, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) table[i] = a.g[i];
}

// `per` pieces per workgroup: four where there are many (136 M elements: 75 -> 72 us, and a quarter of
// the partial sums to fold, 12 -> 5 us), one where that would leave the chip empty (1.7 M: 2.0 us
// against 4.0).  Eight elements at a time whatever the type: the sum's order is the same.
template <typename G>
__global__ __launch_bounds__(256) void adamw_norm_kernel(const dz_adamw_tensor_t* __restrict__ tensors,
                                                         const int32_t* __restrict__ chunks, int num_chunks, int per,
                                                         const void* const* __restrict__ grads,
                                                         float* __restrict__ partials) {
  constexpr int VE = 8, LOADS = kChunk / (256 * VE);
  float s = 0.f;
  for (int q = 0; q < per; ++q) {
    const int at = blockIdx.x * per + q;
    if (at >= num_chunks) break;
    const int t = chunks[2 * at], c = chunks[2 * at + 1];
    const int64_t n = tensors[t].n, first = (int64_t)c * kChunk;
    const G* g = (const G*)grads[t] + first;
    const int left = (int)(n - first < kChunk ? n - first : kChunk);
    DzPack<G, VE> x[LOADS];
#pragma unroll
    for (int r = 0; r < LOADS; ++r) {
      const int i = (r * 256 + threadIdx.x) * VE;
      if (i + VE <= left) {
        x[r] = dz_load<G, VE>(g + i);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) x[r].v[j] = i + j < left ? g[i + j] : (G)0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < LOADS; ++r)
#pragma unroll
      for (int j = 0; j < VE; ++j) { const float y = (float)x[r].v[j]; s = __builtin_fmaf(y, y, s); }
  }
  __shared__ float red[4];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partials[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// The step's scalars: counts the step, folds the norm's partials (in double, always in the same
// order), forms the bias corrections in double and the random key.
__global__ __launch_bounds__(1024) void adamw_scalars_kernel(const float* __restrict__ partials, int n,
                                                             int32_t* __restrict__ count,
                                                             float* __restrict__ scalars, double b1,
                                                             double b2, float max_norm,
                                                             float grad_scale, uint64_t seed) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 8 * 1024) {   // eight loads in flight
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = partials[min(i + e * 1024, n - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e) s += i + e * 1024 < n ? (double)x[e] : 0.0;
  }
  __shared__ double red[16];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; ++i) s += red[i];
  const int step = *count + 1;
  *count = step;
  const float norm = (float)(sqrt(s) * fabs((double)grad_scale));
  scalars[kNorm] = norm;
  scalars[kCoef] = grad_scale * (max_norm > 0.f && !(norm < max_norm) ? max_norm / norm : 1.0f);
  scalars[kBc1] = (float)(1.0 - pow(b1, (double)step));
  scalars[kBc2] = (float)(1.0 - pow(b2, (double)step));
  const uint64_t key = adamw_mix64(seed ^ adamw_mix64((uint64_t)step));
  scalars[kKey] = __uint_as_float((uint32_t)key);
  scalars[kKey + 1] = __uint_as_float((uint32_t)(key >> 32));
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
  return x;
}

// One block's scale and the factor that maps its values onto the format.  The maximum is taken
// over the bits of |x|, which orders infinities and NaN above every finite value: a block that
// holds one gets a NaN scale, and so reads back as NaN.
__device__ __forceinline__ void block_scale(uint32_t top_bits, float largest, float& scale, float& inv) {
  const float top = __uint_as_float(top_bits);
  const bool bad = top_bits >= 0x7f800000u, zero = !bad && top < kTiny;
  scale = bad ? __builtin_nanf("") : zero ? 0.0f : top / largest;
  inv = bad || zero ? 0.0f : largest / top;
}
// y >= 0, already in the format's units and at most its largest value; `noise`: 16 random bits
__device__ __forceinline__ uint32_t to_e4m3(float y, uint32_t noise) {
  const uint32_t small = (uint32_t)floorf(fminf(y, 0x1p-6f) * 512.0f + (float)noise * 0x1p-16f);
  return y < 0x1p-6f ? small : ((__float_as_uint(y) + (noise << 4)) >> 20) - 960u;
}
__device__ __forceinline__ uint32_t to_e5m3(float y, uint32_t noise) {
  const uint32_t small = (uint32_t)floorf(fminf(y, 0x1p-30f) * 0x1p33f + (float)noise * 0x1p-16f);
  const uint32_t c = y < 0x1p-30f ? small : ((__float_as_uint(y) + (noise << 4)) >> 20) - 768u;
  return y > 0.f && c == 0 ? 1u : c;
}
__device__ __forceinline__ float from_e5m3(uint32_t c) {
  return c < 8 ? (float)c * 0x1p-33f : __uint_as_float((c + 768u) << 20);
}
template <int B>
__device__ __forceinline__ float from_e4m3(uint32_t word) { return __builtin_amdgcn_cvt_f32_fp8((int)word, B); }

struct AdamwKernelArgs {
  const dz_adamw_tensor_t* tensors;
  const int32_t* chunks;
  const void* const* grads;
  float* master;
  void* m; void* v;
  float* m_scale; float* v_scale;
  const float* lr; const float* scalars;
  float b1, b2, one_minus_b1, one_minus_b2, eps;
};

// One wave: kRounds rounds of 256 elements, four per lane; the loads of all rounds are issued
// before the first one's arithmetic.
template <typename P, typename G, bool MASTER, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_step_kernel(AdamwKernelArgs a) {
  const int t = a.chunks[2 * blockIdx.x], c = a.chunks[2 * blockIdx.x + 1];
  const dz_adamw_tensor_t ten = a.tensors[t];
  const G* g = (const G*)a.grads[t];
  P* p = (P*)ten.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float coef = a.scalars[kCoef], bc1 = a.scalars[kBc1], bc2 = a.scalars[kBc2], lr = *a.lr;
  const uint64_t key = (uint64_t)__float_as_uint(a.scalars[kKey]) |
                       (uint64_t)__float_as_uint(a.scalars[kKey + 1]) << 32;
  const int64_t first = (int64_t)c * kChunk + wave * (kRounds * kBlock);   // of this wave, in the tensor

  DzPack<G, 4> gx[kRounds];
  DzPack<P, 4> px[kRounds];
  float4 w[kRounds], m32[kRounds], v32[kRounds];
  uint32_t m8[kRounds], v8[kRounds];
  float ms[kRounds], vs[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * kBlock + lane * 4, s = ten.offset + i;
    if (first + r * kBlock >= ten.n) break;   // (wave-uniform; the state is padded to whole blocks)
    if (i + 4 <= ten.n) {
      gx[r] = dz_load<G, 4>(g + i);
      if constexpr (!MASTER) px[r] = dz_load<P, 4>(p + i);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        gx[r].v[j] = i + j < ten.n ? g[i + j] : (G)0.0f;
        if constexpr (!MASTER) px[r].v[j] = i + j < ten.n ? p[i + j] : (P)0.0f;
      }
    }
    if constexpr (MASTER) w[r] = *(const float4*)(a.master + s);
    if constexpr (EIGHT) {
      m8[r] = *(const uint32_t*)((const uint8_t*)a.m + s);
      v8[r] = *(const uint32_t*)((const uint8_t*)a.v + s);
      ms[r] = a.m_scale[s / kBlock];
      vs[r] = a.v_scale[s / kBlock];
    } else {
      m32[r] = *(const float4*)((const float*)a.m + s);
      v32[r] = *(const float4*)((const float*)a.v + s);
    }
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * kBlock + lane * 4, s = ten.offset + i;
    if (first + r * kBlock >= ten.n) break;
    float m[4], v[4], q[4];
    if constexpr (EIGHT) {
      m[0] = from_e4m3<0>(m8[r]) * ms[r]; m[1] = from_e4m3<1>(m8[r]) * ms[r];
      m[2] = from_e4m3<2>(m8[r]) * ms[r]; m[3] = from_e4m3<3>(m8[r]) * ms[r];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = from_e5m3((v8[r] >> (8 * j)) & 255u) * vs[r];
    } else {
      m[0] = m32[r].x; m[1] = m32[r].y; m[2] = m32[r].z; m[3] = m32[r].w;
      v[0] = v32[r].x; v[1] = v32[r].y; v[2] = v32[r].z; v[3] = v32[r].w;
    }
    if constexpr (MASTER) {
      q[0] = w[r].x; q[1] = w[r].y; q[2] = w[r].z; q[3] = w[r].w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = (float)px[r].v[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = (float)gx[r].v[j] * coef;
      m[j] = a.b1 * m[j] + a.one_minus_b1 * gj;
      v[j] = a.b2 * v[j] + a.one_minus_b2 * (gj * gj);
      const float step = (m[j] / bc1) / (sqrtf(v[j] / bc2) + a.eps);
      q[j] = q[j] - lr * (step + ten.decay * q[j]);
    }
    // elements past the tensor's end (only the last block has any): gradient 0, moments kept 0
    if (i + 4 <= ten.n) {
      dz_store<P, 4>(p + i, dz_round<P, 4>(q));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i + j < ten.n) p[i + j] = (P)q[j];
        else m[j] = v[j] = q[j] = 0.f;
      }
    }
    if constexpr (MASTER) *(float4*)(a.master + s) = make_float4(q[0], q[1], q[2], q[3]);
    if constexpr (EIGHT) {
      uint32_t mt = 0, vt = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mt = max(mt, __float_as_uint(m[j]) & 0x7fffffffu);
        vt = max(vt, __float_as_uint(v[j]) & 0x7fffffffu);
      }
      mt = wave_max_u32(mt);
      vt = wave_max_u32(vt);
      float mscale, minv, vscale, vinv;
      block_scale(mt, 448.0f, mscale, minv);
      block_scale(vt, 1.875f, vscale, vinv);
      uint32_t mw = 0, vw = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t u = adamw_mix64(key + (uint64_t)((s >> 1) + h));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int j = 2 * h + k;
          const uint32_t mn = (uint32_t)(u >> (32 * k)) & 0xffffu, vn = (uint32_t)(u >> (32 * k + 16)) & 0xffffu;
          // (a NaN fails the comparison of fminf and becomes the format's largest: the scale is NaN)
          uint32_t mc = to_e4m3(fminf(fabsf(m[j]) * minv, 448.0f), mn);
          const uint32_t vc = to_e5m3(fminf(v[j] * vinv, 1.875f), vn);
          if (m[j] < 0.f) mc |= 128u;
          mw |= mc << (8 * j);
          vw |= vc << (8 * j);
        }
      }
      *(uint32_t*)((uint8_t*)a.m + s) = mw;
      *(uint32_t*)((uint8_t*)a.v + s) = vw;
      if (lane == 0) {
        a.m_scale[s / kBlock] = mscale;
        a.v_scale[s / kBlock] = vscale;
      }
    } else {
      *(float4*)((float*)a.m + s) = make_float4(m[0], m[1], m[2], m[3]);
      *(float4*)((float*)a.v + s) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// The 8-bit moments as numbers: 16 elements per lane.
template <typename T>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t* __restrict__ m,
                                                            const uint8_t* __restrict__ v,
                                                            const float* __restrict__ m_scale,
                                                            const float* __restrict__ v_scale,
                                                            int64_t n, T* __restrict__ m_out,
                                                            T* __restrict__ v_out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= n) return;   // (n is a multiple of 256)
  const uint2 mw = *(const uint2*)(m + i), vw = *(const uint2*)(v + i);
  const float ms = m_scale[i / kBlock], vs = v_scale[i / kBlock];
  float mo[8], vo[8];
  const uint32_t mws[2] = {mw.x, mw.y}, vws[2] = {vw.x, vw.y};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mo[4 * h] = from_e4m3<0>(mws[h]) * ms; mo[4 * h + 1] = from_e4m3<1>(mws[h]) * ms;
    mo[4 * h + 2] = from_e4m3<2>(mws[h]) * ms; mo[4 * h + 3] = from_e4m3<3>(mws[h]) * ms;
#pragma unroll
    for (int j = 0; j < 4; ++j) vo[4 * h + j] = from_e5m3((vws[h] >> (8 * j)) & 255u) * vs;
  }
  dz_store<T, 8>(m_out + i, dz_round<T, 8>(mo));
  dz_store<T, 8>(v_out + i, dz_round<T, 8>(vo));
}

template <typename P, typename G>
void launch_step(const AdamwKernelArgs& k, bool master, bool eight, unsigned grid, hipStream_t s) {
  if (master) {
    if (eight) hipLaunchKernelGGL((adamw_step_kernel<P, G, true, true>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((adamw_step_kernel<P, G, true, false>), dim3(grid), dim3(256), 0, s, k);
  } else {
    if (eight) hipLaunchKernelGGL((adamw_step_kernel<P, G, false, true>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((adamw_step_kernel<P, G, false, false>), dim3(grid), dim3(256), 0, s, k);
  }
}

}  // namespace

extern "C" int dz_adamw_bind(const void* const* grads, int num_tensors, const void** table, dz_stream_t stream) {
  DZ_REQUIRE(grads && table && num_tensors > 0);
  for (int i = 0; i < num_tensors; i += kUpload) {
    UploadArgs a;
    const int n = num_tensors - i < kUpload ? num_tensors - i : kUpload;
    for (int j = 0; j < kUpload; ++j) a.g[j] = j < n ? grads[i + j] : nullptr;
    for (int j = 0; j < n; ++j) DZ_REQUIRE(a.g[j]);
    hipLaunchKernelGGL(adamw_upload_kernel, dim3((n + 255) / 256), dim3(256), 0, dz_s(stream), a, table + i, n);
    DZ_LAUNCH_CHECK();
  }
  return DZ_OK;
}

extern "C" int dz_adamw_step(const dz_adamw_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(a && a->tensors && a->chunks && a->grads && a->m && a->v && a->count && a->lr && a->scalars);
  DZ_REQUIRE(a->num_chunks > 0 && (a->state_bits == 8 || a->state_bits == 32));
  DZ_REQUIRE(dz_is_dtype(a->param_dtype) && (a->grad_dtype == a->param_dtype || a->grad_dtype == DZ_F32));
  DZ_REQUIRE(a->state_bits == 32 || (a->m_scale && a->v_scale));
  DZ_REQUIRE(!(a->master && a->param_dtype == DZ_F32));
  DZ_REQUIRE(!(a->max_norm > 0.f) || a->partials);
  DZ_REQUIRE(a->b1 >= 0.0 && a->b1 < 1.0 && a->b2 >= 0.0 && a->b2 < 1.0 && a->eps >= 0.f);
  const hipStream_t s = dz_s(stream);
  const unsigned grid = (unsigned)a->num_chunks;
  const bool clip = a->max_norm > 0.f;
  const int per = grid >= 8192 ? 4 : 1;
  const unsigned norms = (grid + per - 1) / per;
  if (clip) {
    dz_for_dtype(a->grad_dtype, [&](auto g) {
      hipLaunchKernelGGL((adamw_norm_kernel<decltype(g)>), dim3(norms), dim3(256), 0, s, a->tensors, a->chunks,
                         a->num_chunks, per, a->grads, a->partials);
    });
    DZ_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(1024), 0, s, a->partials, clip ? (int)norms : 0, a->count,
                     a->scalars, a->b1, a->b2, a->max_norm, a->grad_scale, a->seed);
  DZ_LAUNCH_CHECK();
  AdamwKernelArgs k{a->tensors, a->chunks, a->grads, a->master, a->m, a->v, a->m_scale, a->v_scale, a->lr,
                    a->scalars, (float)a->b1, (float)a->b2, (float)(1.0 - a->b1), (float)(1.0 - a->b2), a->eps};
  dz_for_dtype(a->param_dtype, [&](auto p) {
    using P = decltype(p);
    if (a->grad_dtype == DZ_F32) launch_step<P, float>(k, a->master, a->state_bits == 8, grid, s);
    else launch_step<P, P>(k, a->master, a->state_bits == 8, grid, s);
  });
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

extern "C" int dz_adamw_moments(const uint8_t* m, const uint8_t* v, const float* m_scale, const float* v_scale,
                                int64_t count, int dtype, void* m_out, void* v_out, dz_stream_t stream) {
  DZ_REQUIRE(m && v && m_scale && v_scale && m_out && v_out && count > 0 && count % kBlock == 0);
  DZ_REQUIRE(dz_is_dtype(dtype) && count / 2048 < (1ll << 31));
  dz_for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((adamw_moments_kernel<T>), dim3((unsigned)((count + 2047) / 2048)), dim3(256), 0, dz_s(stream),
                       m, v, m_scale, v_scale, count, (T*)m_out, (T*)v_out);
  });
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}
