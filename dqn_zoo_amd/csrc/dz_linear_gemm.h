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
// behind their ends).  What is past an edge along the output index is read from a clamped place and
// not stored; what is past it along k is zeroed in LDS.
//
// MFMA 16 x 16 with the operands exchanged (rows of the instruction are columns of D): a lane ends
// with four adjacent columns of one row, so that bias, residual and outputs are vector accesses.
#pragma once

#include "dz_elem.h"
#include "dz_glds.h"

struct DzGemmShape { int bm, bn, wm, wn; };

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

__device__ __forceinline__ float linear_act(float z, int act) {
  switch (act) {
    case DZ_ACT_RELU: return z < 0.f ? 0.f : z;   // (NaN stays)
    case DZ_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case DZ_ACT_SILU: return z / (1.0f + expf(-z));
    default: return z;
  }
}
__device__ __forceinline__ float linear_act_slope(float z, int act) {
  switch (act) {
    case DZ_ACT_RELU: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    case DZ_ACT_GELU:
      return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    case DZ_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.f;
  }
}

// Four adjacent columns of a finished row.
template <typename T>
__device__ __forceinline__ void linear_epilogue(const DzGemmArgs& p, int64_t i, int j, const float (&d)[4]) {
  const int count = min(4, p.n - j);
  float z[4], y[4];
  if (count == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c) z[c] = d[c];
    if (p.bias) {
      if (p.bias_f32) {
        const auto b = dz_load<float, 4>((const float*)p.bias + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] += b.v[c];
      } else {
        const auto b = dz_load<T, 4>((const T*)p.bias + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] += (float)b.v[c];
      }
    }
    if (p.preact) dz_store<T, 4>((T*)p.preact + i * p.ldz + j, dz_round<T, 4>(z));
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = linear_act(z[c], p.activation);
    if (p.residual) {
      const auto r = dz_load<T, 4>((const T*)p.residual + i * p.ldr + j);
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] += (float)r.v[c];
    }
    if (p.y_f32) dz_store<float, 4>((float*)p.y + i * p.ldy + j, dz_round<float, 4>(y));
    else dz_store<T, 4>((T*)p.y + i * p.ldy + j, dz_round<T, 4>(y));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c >= count) break;
      float zc = d[c];
      if (p.bias) zc += p.bias_f32 ? ((const float*)p.bias)[j + c] : (float)((const T*)p.bias)[j + c];
      if (p.preact) ((T*)p.preact)[i * p.ldz + j + c] = (T)zc;
      float yc = linear_act(zc, p.activation);
      if (p.residual) yc += (float)((const T*)p.residual)[i * p.ldr + j + c];
      if (p.y_f32) ((float*)p.y)[i * p.ldy + j + c] = yc;
      else ((T*)p.y)[i * p.ldy + j + c] = (T)yc;
    }
  }
}

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
      else i = (((u >> 2) ^ ((k >> 2) & 3)) * 4 + (u & 3)) * VE;
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
        f[q] = *(const float*)(lds + k * (EXT * 4) + ((blk ^ ((k >> 2) & 3)) * 64) + j * 4);
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
  static constexpr int PIECES = O::UNITS / 64;                            // DMA instructions of a stage
  static constexpr int PER = (PIECES + THREADS / 64 - 1) / (THREADS / 64);  // of a wave
  const char* base;
  int64_t stage_bytes, k_bytes;   // one stage along k; one k
  unsigned off[PER];

  __device__ static int unit(int n, int wave, int lane) { return (wave * PER + n) * 64 + lane; }
  // (a short operand has fewer pieces than there are waves)
  __device__ static bool has(int n, int wave) { return PIECES % (THREADS / 64) == 0 || wave * PER + n < PIECES; }
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
      if (has(n, wave)) dz_glds16_base(base, off[n], lds_byte + (wave * PER + n) * 1024u);
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
      if (has(n, wave)) dz_glds16_base(tail, o, lds_byte + (wave * PER + n) * 1024u);
    }
  }
  __device__ static void zero_tail(char* lds, int wave, int lane, int rem) {
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      int i, k;
      O::place(unit(n, wave, lane), i, k);
      if (has(n, wave) && k >= rem) *(uint4*)(lds + unit(n, wave, lane) * 16) = make_uint4(0, 0, 0, 0);
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

template <typename T, bool A_KC, bool B_KC, int BM, int BN, int WM, int WN>
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
  auto land = [] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };   // this wave's DMAs are in LDS
  if (rem) {
    ra.issue_tail(lds0, wave, lane, rem, stages - 1);
    rb.issue_tail(lds0 + A_BYTES, wave, lane, rem, stages - 1);
    land();
    SA::zero_tail(lds, wave, lane, rem);
    SB::zero_tail(lds + A_BYTES, wave, lane, rem);
  } else {
    fetch(0);
    land();
  }
  __syncthreads();
  auto step = [&](int t, int buf) {
    if (t + 1 < stages) fetch(buf ^ 1);
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
    land();
    __syncthreads();   // the next stage is there, and nobody reads this one any more
  };
  int t = 0;
  for (; t + 2 <= stages; t += 2) {   // (constant LDS addresses)
    step(t, 0);
    step(t + 1, 1);
  }
  if (t < stages) step(t, 0);

  // Through LDS, so that 16 lanes hold 64 adjacent columns of a row: whole lines to memory, and one
  // copy of the epilogue's code for each pass of up to 64 rows.  16-byte unit u of row r lies in
  // place u ^ (r & 15 or 7): the writes (16 rows each) start in different banks.
  constexpr int TN = BN / WN, UPR = TN / 4, FIT = 2 * STAGE / (WM * WN * 16 * TN * 4);
  constexpr int PASS = FM <= FIT ? FM : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
  static_assert(FIT >= 1 && FM % PASS == 0, "whole passes that fit the stage buffers");
  float* mine = (float*)lds + wave * (PASS * 16 * TN);
#pragma unroll
  for (int h = 0; h < FM / PASS; ++h) {
#pragma unroll
    for (int i = 0; i < PASS; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int r = i * 16 + (lane & 15), u = (j * 4 + (lane >> 4)) ^ (r & (UPR - 1));
        *(f32x4*)(mine + r * TN + u * 4) = acc[h * PASS + i][j];
      }
    // (a wave reads what itself has written: no barrier)
    constexpr int ROWS = 64 / UPR;
#pragma unroll 1
    for (int r0 = 0; r0 < PASS * 16; r0 += ROWS) {
      const int r = r0 + lane / UPR, u = lane % UPR;
      const f32x4 v = *(const f32x4*)(mine + r * TN + ((u ^ (r & (UPR - 1))) * 4));
      const int64_t row = i0 + (wm * FM + h * PASS) * 16 + r;
      const int c = j0 + wn * TN + u * 4;
      if (row >= p.m || c >= p.n) continue;
      const float d[4] = {v[0], v[1], v[2], v[3]};
      if (p.splits > 1) {   // (rows of the slabs are padded to whole vectors)
        *(float4*)(p.slabs + split * p.slab_stride + row * p.slab_ld + c) = make_float4(d[0], d[1], d[2], d[3]);
      } else {
        linear_epilogue<T>(p, row, c, d);
      }
    }
  }
}

// Copies one or two operands into rows of whole 16-byte units, zeros behind their ends: a unit per
// thread.
template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(DzPackArgs p) {
  constexpr int VE = 16 / sizeof(T);
  const DzPackArgs::One q = blockIdx.y ? p.two : p.one;
  const int64_t per_row = q.ldd / VE, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= per_row * q.rows) return;
  const int64_t row = id / per_row;
  const int c = (int)(id - row * per_row) * VE;
  const T* x = (const T*)q.src + row * q.ld + c;
  DzPack<T, VE> v;
  if (c + VE <= q.cols) {
    v = dz_load<T, VE>(x);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v.v[e] = c + e < q.cols ? x[e] : (T)0.0f;
  }
  dz_store<T, VE>((T*)q.dst + row * q.ldd + c, v);
}

// The splits' slabs, added in order, and the epilogue: four columns per thread.
template <typename T>
__global__ __launch_bounds__(256) void linear_finish_kernel(DzGemmArgs p) {
  const int64_t per_row = p.slab_ld / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= per_row * p.m) return;
  const int64_t row = id / per_row;
  const int c = (int)(id - row * per_row) * 4;
  if (c >= p.n) return;
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
  linear_epilogue<T>(p, row, c, d);
}

template <typename T>
__global__ __launch_bounds__(256) void linear_dact_kernel(DzDactArgs p) {
  constexpr int VE = 16 / sizeof(T);
  const int c = (blockIdx.x * 64 + (threadIdx.x & 63)) * VE, r = threadIdx.x >> 6;
  const int count = min(VE, p.n - c);
  const int64_t first = (int64_t)blockIdx.y * p.rows, end = min((int64_t)p.m, first + p.rows);
  float s[VE] = {};
  auto row = [&](int64_t i, DzPack<T, VE> d, DzPack<T, VE> z) {
    float y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      y[e] = (float)d.v[e];
      if (p.z) y[e] *= linear_act_slope((float)z.v[e], p.activation);
      s[e] += y[e];
    }
    if (!p.dz) return;
    T* o = (T*)p.dz + i * p.lddz + c;
    if (count == VE) {
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
  if (count == VE) {
    for (int64_t i = first + r; i < end; i += 8) {   // two rows in flight
      const bool two = i + 4 < end;
      const int64_t j = two ? i + 4 : i;
      DzPack<T, VE> z0, z1;
      const auto d0 = dz_load<T, VE>(dy + i * p.ldy), d1 = dz_load<T, VE>(dy + j * p.ldy);
      if (p.z) {
        z0 = dz_load<T, VE>(z + i * p.ldz);
        z1 = dz_load<T, VE>(z + j * p.ldz);
      }
      row(i, d0, z0);
      if (two) row(j, d1, z1);
    }
  } else if (count > 0) {
    for (int64_t i = first + r; i < end; i += 4) {
      DzPack<T, VE> d0, z0;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        d0.v[e] = e < count ? dy[i * p.ldy + e] : (T)0.0f;
        z0.v[e] = p.z && e < count ? z[i * p.ldz + e] : (T)0.0f;
      }
      row(i, d0, z0);
    }
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

// The chunks' sums, in order.
template <typename T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* __restrict__ sums, int chunks, int n, void* db,
                                                        int db_f32) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (int i = 0; i < chunks; i += 8) {   // eight loads in flight; the sums in order
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = sums[(int64_t)min(i + e, chunks - 1) * n + c];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < chunks) s += x[e];
  }
  if (db_f32) ((float*)db)[c] = s;
  else ((T*)db)[c] = (T)s;
}

}  // namespace
