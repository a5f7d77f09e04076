// The matrix product of the dense-layer operator, for any sizes, strides and alignments:
//
//   D[i][j] = sum_k A(i, k) B(k, j)          float32 accumulation on the matrix pipe
//
// Each operand lies in memory in one of two ways: its depth index k adjacent ("KC": A[i][k], B[j][k])
// or its output index adjacent ("RC": A[k][i], B[k][j]); the three products of a layer and its
// backward pass, with the weight stored either way, are (KC, RC), (KC, KC) and (RC, RC).
//
// Tile: BM x BN by WM x WN waves, a stage is 128 bytes deep (64 16-bit or 32 float32 elements), two
// stages in LDS.  An LDS stage holds a KC operand as rows of eight 16-byte units, unit u of row r in
// place u ^ (r & 7): the 16 rows of a fragment read (ds_read_b128: 8 consecutive k of a 16-bit row, 4
// of a float32 one) then start in different banks.  It holds an RC operand as rows of k; 16-bit
// fragments are read by ds_read_b64_tr_b16, which hands lane i of a 16-lane group column i of a 4 x
// 16 block, float32 ones by ds_read_b32; the 32-byte (64-byte) columns of a row are permuted by k & 7
// ((k >> 2) & 3), which puts the rows of one read in different banks.
//
// Both operands come by 16-byte LDS-DMA: their rows begin at multiples of 16 bytes and hold whole
// 16-byte units (operands that do not are copied into such rows first, linear_pack_kernel, zeros
// behind their ends; with up to 32 rows of A both come through registers instead,
// linear_rows_any_kernel).  What is past an edge along the output index is read from a clamped place
// and not stored; what is past it along k is zeroed in LDS.
//
// MFMA 16 x 16 with the operands exchanged (rows of the instruction are columns of D): a lane ends
// with four adjacent columns of one row, so that bias, residual and outputs are vector accesses.
#pragma once

#include <type_traits>

#include "dz_elem.h"
#include "dz_glds.h"

struct DzGemmShape { int bm, bn, wm, wn, buffers; };

struct DzGemmArgs {
  const void* a; int64_t lda;
  const void* b; int64_t ldb;
  int m, n, k;
  int k_split;             // depth of one split, a multiple of the stage (or >= k)
  int splits;
  // epilogue: y = act(D + bias) + residual; with splits > 1 the products go to `slabs` and
  // linear_finish_kernel takes it from there
  const void* bias; int bias_f32;
  const void* residual; int64_t ldr;
  void* y; int64_t ldy; int y_f32;
  void* preact; int64_t ldz;
  int activation;
  float* slabs; int64_t slab_ld, slab_stride;
  int stream;              // y and preact are stored past the caches
};

struct DzPackArgs {
  struct One { const void* src; int64_t ld; int64_t rows; int cols; void* dst; int64_t ldd; };
  One one, two;
};

// dz = dy act'(z) (or dy) and its column sums over `rows` rows of one workgroup: 64 threads hold 16
// bytes of columns each, 4 rows at a time.
struct DzDactArgs {
  const void* dy; int64_t ldy;
  const void* z; int64_t ldz;
  void* dz; int64_t lddz;        // NULL: sums only
  float* sums;                   // [chunks][n], or NULL
  void* db; int db_f32;          // the sums themselves where one chunk covers all rows
  int m, n, rows, activation;
};

namespace {

constexpr int kMaxSplits = 64;

template <typename T> struct MfmaFrag;   // 16 bytes of one row or column
template <> struct MfmaFrag<dz_bf16> { typedef __attribute__((ext_vector_type(8))) __bf16 V; };
template <> struct MfmaFrag<dz_f16> { typedef __attribute__((ext_vector_type(8))) _Float16 V; };
template <> struct MfmaFrag<float> { typedef __attribute__((ext_vector_type(4))) float V; };
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

__device__ __forceinline__ f32x4 mfma16(MfmaFrag<dz_bf16>::V a, MfmaFrag<dz_bf16>::V b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(MfmaFrag<dz_f16>::V a, MfmaFrag<dz_f16>::V b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// (lane group g holds k = 4 g + q: the same order in both operands)
__device__ __forceinline__ f32x4 mfma16(MfmaFrag<float>::V a, MfmaFrag<float>::V b, f32x4 c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[q], c, 0, 0, 0);
  return c;
}

// Phi(-|z|) of the standard normal, and exp(-z^2 / 2) with it.  16-bit layers take
// erfc(x) = t (a1 + ... + a5 t^4) exp(-x^2), t = 1 / (1 + 0.3275911 x), of Abramowitz and Stegun
// 7.1.26: 1.5e-7 absolute, 2^-13 of a bf16 half step near 1, for one exponential and one reciprocal
// (with erff and expf the GELU kernels were bound by arithmetic: dz of 8192 x 4096 took 62 us, 46 so).
template <typename T>
__device__ __forceinline__ float normal_tail(float z, float& density) {
  if constexpr (sizeof(T) == 4) {
    density = expf(-0.5f * z * z);
    return 0.5f * erfcf(fabsf(z) * 0.70710678118654752f);
  } else {
    density = __builtin_amdgcn_exp2f(-0.72134752044448170f * (z * z));   // log2(e) / 2
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
    float q = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    q = __builtin_fmaf(t, q, 0.5f * 1.421413741f);
    q = __builtin_fmaf(t, q, 0.5f * -0.284496736f);
    q = __builtin_fmaf(t, q, 0.5f * 0.254829592f);
    return q * t * density;
  }
}
template <typename T>
__device__ __forceinline__ float logistic(float z) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-z));
  else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}

// Infinite z have their limits' values (a factor that vanishes is multiplied by a bounded z; a NaN
// comes back through the other factor).
constexpr float kBound = 1e30f;
template <typename T>
__device__ __forceinline__ float linear_act(float z, int act) {
  float density;
  switch (act) {
    case DZ_ACT_RELU: return z < 0.f ? 0.f : z;   // (NaN stays)
    case DZ_ACT_GELU: return fmaxf(z, 0.f) - fminf(fabsf(z), kBound) * normal_tail<T>(z, density);   // z Phi(z)
    case DZ_ACT_SILU: return fmaxf(z, -kBound) * logistic<T>(z);
    default: return z;
  }
}
template <typename T>
__device__ __forceinline__ float linear_act_slope(float z, int act) {
  const float bounded = fminf(fmaxf(z, -kBound), kBound);
  switch (act) {
    case DZ_ACT_RELU: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    case DZ_ACT_GELU: {
      float density;
      const float tail = normal_tail<T>(z, density);
      return __builtin_fmaf(bounded * 0.39894228040143268f, density, z < 0.f ? tail : 1.0f - tail);
    }
    case DZ_ACT_SILU: {
      const float s = logistic<T>(z);
      return s * (1.0f + bounded * (1.0f - s));
    }
    default: return 1.f;
  }
}

// W adjacent columns from column j of a finished row: bias, activation, residual and outputs.  The
// columns' bias is the same for every row of a thread.
// (16 bytes past the caches; other widths as usual)
template <typename T, int W>
__device__ __forceinline__ void store_past(T* p, const DzPack<T, W>& x) {
  if constexpr (sizeof(x) == 16) {
    typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned U;
    U u;
    __builtin_memcpy(&u, &x, 16);
    __builtin_nontemporal_store(u, (U*)p);
  } else {
    dz_store<T, W>(p, x);
  }
}

template <typename T, int W>
struct Epilogue {
  float bias[W];
  int count;   // columns inside the matrix

  __device__ void init(const DzGemmArgs& p, int j) {
    count = min(W, p.n - j);
#pragma unroll
    for (int c = 0; c < W; ++c) {
      bias[c] = 0.f;
      if (p.bias && c < count) bias[c] = p.bias_f32 ? ((const float*)p.bias)[j + c] : (float)((const T*)p.bias)[j + c];
    }
  }
  __device__ void row(const DzGemmArgs& p, int64_t i, int j, const float (&d)[W]) const {
    T* pre = (T*)p.preact + i * p.ldz + j;
    const T* res = (const T*)p.residual + i * p.ldr + j;
    float z[W], y[W];
#pragma unroll
    for (int c = 0; c < W; ++c) z[c] = d[c] + bias[c];
    if (count == W) {
      DzPack<T, W> r;
      if (p.residual) r = dz_load<T, W>(res);
      if (p.preact) {
        if (p.stream) store_past<T, W>(pre, dz_round<T, W>(z));
        else dz_store<T, W>(pre, dz_round<T, W>(z));
      }
#pragma unroll
      for (int c = 0; c < W; ++c) y[c] = linear_act<T>(z[c], p.activation);
      if (p.residual) {
#pragma unroll
        for (int c = 0; c < W; ++c) y[c] += (float)r.v[c];
      }
      if (p.y_f32) dz_store<float, W>((float*)p.y + i * p.ldy + j, dz_round<float, W>(y));
      else if (p.stream) store_past<T, W>((T*)p.y + i * p.ldy + j, dz_round<T, W>(y));
      else dz_store<T, W>((T*)p.y + i * p.ldy + j, dz_round<T, W>(y));
    } else {
#pragma unroll
      for (int c = 0; c < W; ++c) {
        if (c >= count) break;
        if (p.preact) pre[c] = (T)z[c];
        float v = linear_act<T>(z[c], p.activation);
        if (p.residual) v += (float)res[c];
        if (p.y_f32) ((float*)p.y)[i * p.ldy + j + c] = v;
        else ((T*)p.y)[i * p.ldy + j + c] = (T)v;
      }
    }
  }
};

// ---- one operand's stage -------------------------------------------------------
// EXT: rows of the tile along the output index; unit q of the stage is 16 bytes at LDS byte 16 q.
template <typename T, bool KC, int EXT>
struct Operand {
  static constexpr int VE = 16 / sizeof(T), BK = 128 / sizeof(T);
  static constexpr int UNITS = EXT * 8;

  // first output index and depth of unit q
  __device__ static void place(int q, int& i, int& k) {
    if constexpr (KC) {
      i = q >> 3;
      k = ((q & 7) ^ (i & 7)) * VE;
    } else {
      constexpr int UPR = EXT / VE;
      k = q / UPR;
      const int u = q % UPR;
      if constexpr (sizeof(T) == 2) i = (((u >> 1) ^ (k & (EXT / 16 - 1) & 7)) * 2 + (u & 1)) * VE;
      else i = (((u >> 2) ^ ((k >> 2) & (EXT / 16 - 1) & 3)) * 4 + (u & 3)) * VE;
    }
  }
  // 16 consecutive output indices from 16 blk, depth step s of 2
  __device__ static typename MfmaFrag<T>::V fragment(const char* lds, int blk, int s, int lane) {
    const int j = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int r = blk * 16 + j, u = (4 * s + g) ^ (r & 7);
      return *(const typename MfmaFrag<T>::V*)(lds + r * 128 + u * 16);
    } else if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4* Lds;
      union { s16x4 h[2]; typename MfmaFrag<T>::V v; } f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int k = 32 * s + 8 * g + 4 * t + (j >> 2);
        const char* at = lds + k * (EXT * 2) + ((blk ^ (k & (EXT / 16 - 1) & 7)) * 32) + (j & 3) * 8;
        f.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at);
      }
      return f.v;
    } else {
      typename MfmaFrag<T>::V f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = 16 * s + 4 * g + q;
        f[q] = *(const float*)(lds + k * (EXT * 4) + ((blk ^ ((k >> 2) & (EXT / 16 - 1) & 3)) * 64) + j * 4);
      }
      return f;
    }
  }
};

// The stages of one operand by LDS-DMA: a scalar base that moves by a stage, and one constant 32-bit
// offset per unit of this thread (no vector arithmetic in the main loop).
template <typename T, bool KC, int EXT, int THREADS>
struct Stager {
  using O = Operand<T, KC, EXT>;
  static constexpr int PER = O::UNITS / THREADS;
  static_assert(O::UNITS % THREADS == 0, "whole units per thread");
  const char* base;
  int64_t stage_bytes, k_bytes;   // one stage along k; one k
  unsigned off[PER];

  __device__ static int unit(int n, int wave, int lane) { return (wave * PER + n) * 64 + lane; }
  // what lies past the edge along the output index is read from a clamped place: its products are
  // not stored
  __device__ void init(const T* x, int64_t ld, int i0, int ext, int k0, int wave, int lane) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int i, k;
      O::place(unit(n, wave, lane), i, k);
      i = min(i + i0, KC ? ext - 1 : (ext - 1) / O::VE * O::VE) - i0;
      off[n] = (unsigned)((KC ? i * ld + k : k * ld + i) * (int64_t)sizeof(T));
    }
    base = (const char*)(KC ? x + i0 * ld + k0 : x + k0 * ld + i0);
    k_bytes = (KC ? 1 : ld) * (int64_t)sizeof(T);
    stage_bytes = O::BK * k_bytes;
  }
  __device__ void issue(unsigned lds_byte, int wave) {
#pragma unroll
    for (int n = 0; n < PER; ++n)
      dz_glds16_base(base, off[n], lds_byte + (wave * PER + n) * 1024u);
    base += stage_bytes;
  }
  // a stage that is only `rem` deep, `stages` whole ones from here: what lies past it along k is
  // read from its first k, and zeroed in LDS, by the lanes that asked for it, once it is there
  __device__ void issue_tail(unsigned lds_byte, int wave, int lane, int rem, int stages) const {
    const char* tail = base + stages * stage_bytes;
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int i, k;
      O::place(unit(n, wave, lane), i, k);
      const unsigned o = k < rem ? off[n] : off[n] - (unsigned)(k * k_bytes);
      dz_glds16_base(tail, o, lds_byte + (wave * PER + n) * 1024u);
    }
  }
  __device__ static void zero_tail(char* lds, int wave, int lane, int rem) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int i, k;
      O::place(unit(n, wave, lane), i, k);
      if (k >= rem) *(uint4*)(lds + unit(n, wave, lane) * 16) = make_uint4(0, 0, 0, 0);
    }
  }
};

// Workgroups go round the 8 XCDs in turn; each takes a run of neighbouring tiles, in bands of 8 tile
// rows, so that the tiles an XCD works on at one time share rows of A and columns of B in its L2.
__device__ __forceinline__ void tile_of(int id, int tiles, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int xcd = id & 7, chunk = tiles >> 3, rest = tiles & 7;
  id = xcd * chunk + min(xcd, rest) + (id >> 3);
  const int band = id / (8 * tiles_n), first = band * 8, rows = min(8, tiles_m - first);
  const int in = id - band * 8 * tiles_n;
  tm = first + in % rows;
  tn = in / rows;
}

template <typename T, bool A_KC, bool B_KC, int BM, int BN, int WM, int WN, int NBUF>
__global__ __launch_bounds__(64 * WM * WN) void linear_gemm_kernel(DzGemmArgs p) {
  constexpr int THREADS = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, BK = 128 / sizeof(T);
  constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
  using SA = Stager<T, A_KC, BM, THREADS>;
  using SB = Stager<T, B_KC, BN, THREADS>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;
  int tm, tn;
  tile_of(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const int i0 = tm * BM, j0 = tn * BN, split = blockIdx.y;
  const int k0 = split * p.k_split, k_end = min(p.k, k0 + p.k_split);
  const int stages = (k_end - k0 + BK - 1) / BK;
  const T* a = (const T*)p.a;
  const T* b = (const T*)p.b;
  const unsigned lds0 = (unsigned)(uintptr_t)lds;

  const int rem = (k_end - k0) % BK;   // a stage that is not whole is taken first, out of the main loop

  f32x4 acc[FM][FN] = {};
  SA ra;
  SB rb;
  ra.init(a, p.lda, i0, p.m, k0, wave, lane);
  rb.init(b, p.ldb, j0, p.n, k0, wave, lane);
  auto fetch = [&](int buf) {
    ra.issue(lds0 + buf * STAGE, wave);
    rb.issue(lds0 + buf * STAGE + A_BYTES, wave);
  };
  // Stage t is used from buffer t % NBUF while the NBUF - 1 behind it are on their way.
  constexpr int AHEAD = NBUF - 2, OUT = AHEAD * (SA::PER + SB::PER);   // stages, DMAs that may still be out
  if (rem) {
    ra.issue_tail(lds0, wave, lane, rem, stages - 1);
    rb.issue_tail(lds0 + A_BYTES, wave, lane, rem, stages - 1);
  } else {
    fetch(0);
  }
#pragma unroll
  for (int n = 1; n <= AHEAD; ++n)
    if (n < stages) fetch(n);
  auto land = [&](bool all) {   // this wave's DMAs of the next stage (or all) are in LDS
    if (all || AHEAD == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OUT) : "memory");
  };
  land(stages <= AHEAD);
  if (rem) {
    SA::zero_tail(lds, wave, lane, rem);
    SB::zero_tail(lds + A_BYTES, wave, lane, rem);
  }
  __syncthreads();
  auto step = [&](int t, int buf) {
    const bool more = t + NBUF - 1 < stages;
    if (more) fetch((buf + NBUF - 1) % NBUF);
    const char* sa = lds + buf * STAGE;
    const char* sb = sa + A_BYTES;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename MfmaFrag<T>::V fa[FM], fb[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) fb[f] = Operand<T, B_KC, BN>::fragment(sb, wn * FN + f, s, lane);
#pragma unroll
      for (int f = 0; f < FM; ++f) fa[f] = Operand<T, A_KC, BM>::fragment(sa, wm * FM + f, s, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma16(fb[j], fa[i], acc[i][j]);
    }
    land(!more);
    __syncthreads();   // the next stage is there, and nobody reads this one any more
  };
  if constexpr (!A_KC) {
    // One copy of the step: the transposing reads take an address per column block and buffer, and
    // two copies of it spill (256 x 256, 4096 x 4096 x 8192: 228 -> 213 us).
    int buf = 0;
#pragma unroll 1
    for (int t = 0; t < stages; ++t) {
      step(t, buf);
      buf = buf == NBUF - 1 ? 0 : buf + 1;
    }
  } else {
    int t = 0;
    for (; t + NBUF <= stages; t += NBUF) {   // (constant LDS addresses)
#pragma unroll
      for (int n = 0; n < NBUF; ++n) step(t + n, n);
    }
#pragma unroll
    for (int n = 0; n < NBUF - 1; ++n)
      if (t + n < stages) step(t + n, n);
  }

  // Through LDS, so that a lane holds eight adjacent columns of a row and neighbours make whole lines,
  // with one copy of the epilogue's code for each pass of up to 64 rows.  16-byte unit u of row r lies
  // in place u ^ (r & 7 or 15): the writes (16 rows each) start in different banks.
  constexpr int TN = BN / WN, UPR = TN / 4, FIT = NBUF * STAGE / (WM * WN * 16 * TN * 4), W = 8, LPR = TN / W;
  constexpr int PASS = FM <= FIT ? FM : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
  static_assert(FIT >= 1 && FM % PASS == 0, "whole passes that fit the stage buffers");
  float* mine = (float*)lds + wave * (PASS * 16 * TN);
  const int cu = lane % LPR, c = j0 + wn * TN + cu * W;
  Epilogue<T, W> epi;
  epi.init(p, c);
#pragma unroll
  for (int h = 0; h < FM / PASS; ++h) {
#pragma unroll
    for (int i = 0; i < PASS; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int r = i * 16 + (lane & 15), u = (j * 4 + (lane >> 4)) ^ (r & (UPR - 1) & 15);
        *(f32x4*)(mine + r * TN + u * 4) = acc[h * PASS + i][j];
      }
    // (a wave reads what itself has written: no barrier)
    constexpr int ROWS = 64 / LPR;
#pragma unroll 1
    for (int r0 = 0; r0 < PASS * 16; r0 += ROWS) {
      const int r = r0 + lane / LPR, sw = r & (UPR - 1) & 15;
      const f32x4 v0 = *(const f32x4*)(mine + r * TN + ((2 * cu) ^ sw) * 4);
      const f32x4 v1 = *(const f32x4*)(mine + r * TN + ((2 * cu + 1) ^ sw) * 4);
      const int64_t row = i0 + (wm * FM + h * PASS) * 16 + r;
      if (row >= p.m || epi.count <= 0) continue;
      const float d[W] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
      if (p.splits > 1) {   // (rows of the slabs are padded to whole vectors)
        float* slab = p.slabs + split * p.slab_stride + row * p.slab_ld + c;
        *(float4*)slab = make_float4(d[0], d[1], d[2], d[3]);
        *(float4*)(slab + 4) = make_float4(d[4], d[5], d[6], d[7]);
      } else {
        epi.row(p, row, c, d);
      }
    }
  }
}

// Up to 16 or 32 rows (the tokens of a generation step, one observation, a learner's batch of 32): a
// workgroup has 32 columns and
// the whole depth, its eight waves take its stages in turn, each through a ring of its own -- no barrier
// until the waves' sums meet in LDS, no slabs, one launch.  Bound by the weight's bytes: 64 KB of them
// are on their way in each CU.
constexpr int kRowsWaves = 8, kRowsN = 32;
constexpr int rows_buffers(int rows) { return rows == 16 ? 3 : 2; }   // (160 KB of LDS)
// The waves' sums, added in order, and the epilogue.
template <typename T, int ROWS>
__device__ __forceinline__ void rows_finish(const DzGemmArgs& p, const f32x4 (&acc)[ROWS / 16][kRowsN / 16], float* sums,
                                            int j0, int wave, int lane) {
  constexpr int FM = ROWS / 16, FN = kRowsN / 16;
  __syncthreads();   // (the rings have been read)
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int f = 0; f < FN; ++f)
      *(f32x4*)(sums + (wave * ROWS + i * 16 + (lane & 15)) * kRowsN + f * 16 + 4 * (lane >> 4)) = acc[i][f];
  __syncthreads();
  static_assert(kRowsWaves * 64 >= ROWS * kRowsN / 4, "a thread per four columns");
  const int row = threadIdx.x / (kRowsN / 4), c = threadIdx.x % (kRowsN / 4) * 4;
  if (row >= p.m || row >= ROWS || j0 + c >= p.n) return;
  Epilogue<T, 4> epi;
  epi.init(p, j0 + c);
  f32x4 v = *(const f32x4*)(sums + row * kRowsN + c);
#pragma unroll
  for (int w = 1; w < kRowsWaves; ++w) v += *(const f32x4*)(sums + (w * ROWS + row) * kRowsN + c);
  const float d[4] = {v[0], v[1], v[2], v[3]};
  epi.row(p, row, j0 + c, d);
}

template <typename T, bool B_KC, int ROWS>
__global__ __launch_bounds__(64 * kRowsWaves) void linear_rows_kernel(DzGemmArgs p) {
  constexpr int BK = 128 / sizeof(T), FM = ROWS / 16, FN = kRowsN / 16, NBUF = rows_buffers(ROWS);
  constexpr int A_BYTES = ROWS * 128, STAGE = (ROWS + kRowsN) * 128, RING = NBUF * STAGE;
  using SA = Stager<T, true, ROWS, 64>;
  using SB = Stager<T, B_KC, kRowsN, 64>;
  constexpr int OUT = (NBUF - 2) * (SA::PER + SB::PER);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j0 = blockIdx.x * kRowsN;
  const int whole = p.k / BK, rem = p.k % BK;
  // this wave's whole stages: wave, wave + 8, ...; the last wave also has the one that is not whole
  const bool tail = rem && wave == kRowsWaves - 1;
  const int own = (whole - wave + kRowsWaves - 1) / kRowsWaves, stages = own + tail;
  char* ring = lds + wave * RING;
  const unsigned lds0 = (unsigned)(uintptr_t)ring;

  f32x4 acc[FM][FN] = {};
  SA ra;
  SB rb;
  ra.init((const T*)p.a, p.lda, 0, p.m, 0, 0, lane);
  rb.init((const T*)p.b, p.ldb, j0, p.n, 0, 0, lane);
  const char* a0 = ra.base;
  const char* b0 = rb.base;
  int next = wave;
  auto fetch = [&](int n, int buf) {   // stage n of this wave
    const unsigned at = lds0 + buf * STAGE;
    if (tail && n == 0) {
      ra.base = a0; rb.base = b0;
      ra.issue_tail(at, 0, lane, rem, whole);
      rb.issue_tail(at + A_BYTES, 0, lane, rem, whole);
    } else {
      ra.base = a0 + next * ra.stage_bytes;
      rb.base = b0 + next * rb.stage_bytes;
      next += kRowsWaves;
      ra.issue(at, 0);
      rb.issue(at + A_BYTES, 0);
    }
  };
#pragma unroll
  for (int n = 0; n < NBUF - 1; ++n)
    if (n < stages) fetch(n, n);
  auto step = [&](int t, int buf) {
    // the next buffer's reads are done (their products are issued), stage t is here
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + NBUF - 1 < stages) {
      fetch(t + NBUF - 1, (buf + NBUF - 1) % NBUF);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OUT + SA::PER + SB::PER) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    char* sa = ring + buf * STAGE;
    if (tail && t == 0) {
      SA::zero_tail(sa, 0, lane, rem);
      SB::zero_tail(sa + A_BYTES, 0, lane, rem);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename MfmaFrag<T>::V fa[FM];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = Operand<T, true, ROWS>::fragment(sa, i, s, lane);
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        const auto fb = Operand<T, B_KC, kRowsN>::fragment(sa + A_BYTES, f, s, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][f] = mfma16(fb, fa[i], acc[i][f]);
      }
    }
  };
  int t = 0;
  for (; t + NBUF <= stages; t += NBUF) {
#pragma unroll
    for (int n = 0; n < NBUF; ++n) step(t + n, n);
  }
#pragma unroll
  for (int n = 0; n < NBUF - 1; ++n)
    if (t + n < stages) step(t + n, n);

  rows_finish<T, ROWS>(p, acc, (float*)lds, j0, wave, lane);
}

// The same for operands whose rows are not whole 16-byte units: through registers, a stage ahead.
// (9 x 1951 x 7059 float32 from rows of 1959: 14.3 us; copying the weight first, 37.8.)
template <typename T, bool KC, int EXT>
struct RegStager {
  using O = Operand<T, KC, EXT>;
  static constexpr int PER = O::UNITS / 64;
  DzPack<T, O::VE> r[PER];

  // What is past the edge along the output index is not used; what is past k_end is 0.
  __device__ void load(const T* x, int64_t ld, int i0, int ext, int k0, int k_end, int lane) {
    if (k0 + O::BK <= k_end && (KC || i0 + EXT <= ext)) {   // (uniform)
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int i, k;
        O::place(n * 64 + lane, i, k);
        if (KC) r[n] = dz_load<T, O::VE>(x + (int64_t)min(i0 + i, ext - 1) * ld + k0 + k);
        else r[n] = dz_load<T, O::VE>(x + (int64_t)(k0 + k) * ld + i0 + i);
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int i, k;
      O::place(n * 64 + lane, i, k);
      i += i0;
      k += k0;
#pragma unroll
      for (int e = 0; e < O::VE; ++e) {
        const int ie = KC ? i : i + e, ke = KC ? k + e : k;
        r[n].v[e] = ie < ext && ke < k_end ? x[KC ? (int64_t)ie * ld + ke : (int64_t)ke * ld + ie] : (T)0.0f;
      }
    }
  }
  __device__ void write(char* lds, int lane) const {
#pragma unroll
    for (int n = 0; n < PER; ++n)
      *(DzPack<T, O::VE>*)__builtin_assume_aligned(lds + (n * 64 + lane) * 16, 16) = r[n];
  }
};

template <typename T, bool B_KC, int ROWS>
__global__ __launch_bounds__(64 * kRowsWaves) void linear_rows_any_kernel(DzGemmArgs p) {
  constexpr int BK = 128 / sizeof(T), FM = ROWS / 16, FN = kRowsN / 16;
  constexpr int A_BYTES = ROWS * 128, STAGE = (ROWS + kRowsN) * 128;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j0 = blockIdx.x * kRowsN;
  const int stages = ((p.k + BK - 1) / BK - wave + kRowsWaves - 1) / kRowsWaves;   // wave, wave + 8, ...
  char* ring = lds + wave * 2 * STAGE;

  f32x4 acc[FM][FN] = {};
  RegStager<T, true, ROWS> ra;
  RegStager<T, B_KC, kRowsN> rb;
  auto load = [&](int t) {
    const int k0 = (wave + t * kRowsWaves) * BK;
    ra.load((const T*)p.a, p.lda, 0, p.m, k0, p.k, lane);
    rb.load((const T*)p.b, p.ldb, j0, p.n, k0, p.k, lane);
  };
  auto write = [&](int buf) {
    ra.write(ring + buf * STAGE, lane);
    rb.write(ring + buf * STAGE + A_BYTES, lane);
  };
  if (stages > 0) {
    load(0);
    write(0);
  }
#pragma unroll 1
  for (int t = 0; t < stages; ++t) {
    if (t + 1 < stages) load(t + 1);
    const char* sa = ring + (t & 1) * STAGE;   // (a wave's LDS accesses are in order: no barrier)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename MfmaFrag<T>::V fa[FM];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = Operand<T, true, ROWS>::fragment(sa, i, s, lane);
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        const auto fb = Operand<T, B_KC, kRowsN>::fragment(sa + A_BYTES, f, s, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][f] = mfma16(fb, fa[i], acc[i][f]);
      }
    }
    if (t + 1 < stages) write((t + 1) & 1);
  }
  rows_finish<T, ROWS>(p, acc, (float*)lds, j0, wave, lane);
}

// Copies one or two operands into rows of whole 16-byte units, zeros behind their ends: 64 threads
// along a row, four times two rows (4095 x 4095 fp16 alone: one 17.2 us, two 14.9, four 15.0; 1777 x
// 1235 and 1235 x 1001 together 6.7, 7.0, 7.4).
constexpr int kPackRows = 2;
template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(DzPackArgs p) {
  constexpr int VE = 16 / sizeof(T);
  const DzPackArgs::One q = blockIdx.z ? p.two : p.one;
  const int c = (blockIdx.x * 64 + (threadIdx.x & 63)) * VE;
  if (c >= q.cols) return;
  const bool whole = c + VE <= q.cols;
  for (int64_t row = blockIdx.y * (4 * kPackRows) + (threadIdx.x >> 6); row < q.rows; row += gridDim.y * (4 * kPackRows)) {
    DzPack<T, VE> v[kPackRows];
#pragma unroll
    for (int r = 0; r < kPackRows; ++r) {
      const T* x = (const T*)q.src + min(row + 4 * r, q.rows - 1) * q.ld + c;
      if (whole) {
        v[r] = dz_load<T, VE>(x);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[r].v[e] = c + e < q.cols ? x[e] : (T)0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < kPackRows; ++r)
      if (row + 4 * r < q.rows) dz_store<T, VE>((T*)q.dst + (row + 4 * r) * q.ldd + c, v[r]);
  }
}

// The splits' slabs, added in order, and the epilogue: four columns per thread, 64 threads along a
// row.
template <typename T>
__global__ __launch_bounds__(64) void linear_finish_kernel(DzGemmArgs p) {
  const int c = (blockIdx.x * 64 + threadIdx.x) * 4;
  if (c >= p.n) return;
  Epilogue<T, 4> epi;
  epi.init(p, c);
  for (int64_t row = blockIdx.y; row < p.m; row += gridDim.y) {
    const float* at = p.slabs + row * p.slab_ld + c;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.splits; k += 8) {   // eight loads in flight; the sums in order
      float4 x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = *(const float4*)(at + min(k + e, p.splits - 1) * p.slab_stride);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (k + e >= p.splits) break;
        s.x += x[e].x; s.y += x[e].y; s.z += x[e].z; s.w += x[e].w;
      }
    }
    const float d[4] = {s.x, s.y, s.z, s.w};
    epi.row(p, row, c, d);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void linear_dact_kernel(DzDactArgs p) {
  constexpr int VE = 16 / sizeof(T);
  const int c = (blockIdx.x * 64 + (threadIdx.x & 63)) * VE, r = threadIdx.x >> 6;
  const bool inside = (blockIdx.x + 1) * 64 * VE <= p.n;   // (uniform: every unit of these columns is whole)
  const int count = min(VE, p.n - c);
  const int64_t first = (int64_t)blockIdx.y * p.rows, end = min((int64_t)p.m, first + p.rows);
  float s[VE] = {};
  auto row = [&](int64_t i, DzPack<T, VE> d, DzPack<T, VE> z, auto whole) {
    float y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      y[e] = (float)d.v[e];
      if (p.z) y[e] *= linear_act_slope<T>((float)z.v[e], p.activation);
      s[e] += y[e];
    }
    if (!p.dz) return;
    T* o = (T*)p.dz + i * p.lddz + c;
    if (whole || count == VE) {
      dz_store<T, VE>(o, dz_round<T, VE>(y));
    } else {
      // (dz's rows are padded to whole units; what is behind their ends is 0)
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] = e < count ? y[e] : 0.f;
      dz_store<T, VE>(o, dz_round<T, VE>(y));
    }
  };
  const T* dy = (const T*)p.dy + c;
  const T* z = (const T*)p.z + c;
  auto rows = [&](auto load, auto whole) {
    constexpr int FLY = whole ? 4 : 1;   // rows of a thread in flight
    for (int64_t i = first + r; i < end; i += 4 * FLY) {
      DzPack<T, VE> d[FLY], zv[FLY];
#pragma unroll
      for (int f = 0; f < FLY; ++f) {
        const int64_t j = min(i + 4 * f, end - 1);
        d[f] = load(dy + j * p.ldy);
        if (p.z) zv[f] = load(z + j * p.ldz);
      }
#pragma unroll
      for (int f = 0; f < FLY; ++f)
        if (i + 4 * f < end) row(i + 4 * f, d[f], zv[f], whole);
    }
  };
  if (inside) {
    rows([](const T* x) { return dz_load<T, VE>(x); }, std::true_type{});
  } else if (count > 0) {
    // One loop for whole units and the row's last: two would take turns in its wave (2431 x 151 bf16 with
    // SiLU 27 us; 9.0 with this and half the rows a workgroup).  A row at a time: four are 64 registers
    // of single elements, which all workgroups pay (8192 x 4096 bf16, GELU: 54 -> 77 us).  The last
    // element stands for those that are not there.
    rows([&](const T* x) {
      if (count == VE) return dz_load<T, VE>(x);
      DzPack<T, VE> v;
#pragma unroll
      for (int e = 0; e < VE; ++e) v.v[e] = x[min(e, count - 1)];
      return v;
    }, std::false_type{});
  }
  if (!p.sums && !p.db) return;
  __shared__ float red[4][VE][64];
#pragma unroll
  for (int e = 0; e < VE; ++e) red[r][e][threadIdx.x & 63] = s[e];
  __syncthreads();
  if (r || count <= 0) return;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    if (e >= count) break;
    const float o = (red[0][e][threadIdx.x] + red[1][e][threadIdx.x]) + (red[2][e][threadIdx.x] + red[3][e][threadIdx.x]);
    if (p.sums) p.sums[(int64_t)blockIdx.y * p.n + c + e] = o;
    else if (p.db_f32) ((float*)p.db)[c + e] = o;
    else ((T*)p.db)[c + e] = (T)o;
  }
}

// The chunks' sums: 64 columns and four runs of chunks per workgroup, each in order.
template <typename T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* __restrict__ sums, int chunks, int n, void* db,
                                                        int db_f32) {
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6, run = (chunks + 3) / 4;
  const int first = part * run, end = min(chunks, first + run);
  float s = 0.f;
  if (c < n)
    for (int i = first; i < end; i += 8) {   // eight loads in flight
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = sums[(int64_t)min(i + e, end - 1) * n + c];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < end) s += x[e];
    }
  __shared__ float red[4][64];
  red[part][threadIdx.x & 63] = s;
  __syncthreads();
  if (part || c >= n) return;
  s = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
  if (db_f32) ((float*)db)[c] = s;
  else ((T*)db)[c] = (T)s;
}

}  // namespace
