// The launches of the dense-layer operator for one element type; included by one unit per type.
#pragma once

#include "dz_linear.h"

namespace {

template <typename T, bool A_KC, bool B_KC, int TILE>
int launch_gemm_tile(const DzGemmArgs& p, hipStream_t s) {
  constexpr DzGemmShape t = kGemmTiles[TILE];
  // (256 x 256 from two KC operands: 207 us as 4 x 2 waves, 212 as 2 x 4; 897 against 883 and 224
  // against 213 in the other layouts' cases)
  constexpr int wm = A_KC && B_KC && t.wm != t.wn ? t.wn : t.wm, wn = A_KC && B_KC && t.wm != t.wn ? t.wm : t.wn;
  constexpr int kLds = t.buffers * (t.bm + t.bn) * 128;
  const int64_t tiles = (int64_t)((p.m + t.bm - 1) / t.bm) * ((p.n + t.bn - 1) / t.bn);
  if (tiles * 64 * t.wm * t.wn >= (1ll << 32)) return DZ_ERR_UNSUPPORTED;
  auto kernel = linear_gemm_kernel<T, A_KC, B_KC, t.bm, t.bn, wm, wn, t.buffers>;
  if (kLds > 65536)
    DZ_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)p.splits), dim3(64 * t.wm * t.wn), kLds, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T, bool A_KC, bool B_KC>
int launch_gemm_kind(const DzGemmArgs& p, const DzGemmPlan& plan, hipStream_t s) {
  switch (plan.tile) {
    case 0: return launch_gemm_tile<T, A_KC, B_KC, 0>(p, s);
    case 1: return launch_gemm_tile<T, A_KC, B_KC, 1>(p, s);
    case 2: return launch_gemm_tile<T, A_KC, B_KC, 2>(p, s);
    default: return DZ_ERR_UNSUPPORTED;
  }
}

template <typename T, bool B_KC, int ROWS>
int launch_rows_of(const DzGemmArgs& p, bool any, hipStream_t s) {
  const int lds = kRowsWaves * (any ? 2 : rows_buffers(ROWS)) * (ROWS + kRowsN) * 128;
  auto kernel = any ? linear_rows_any_kernel<T, B_KC, ROWS> : linear_rows_kernel<T, B_KC, ROWS>;
  DZ_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL(kernel, dim3((p.n + kRowsN - 1) / kRowsN), dim3(64 * kRowsWaves), lds, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T, bool B_KC>
int launch_rows(const DzGemmArgs& p, bool any, hipStream_t s) {
  return p.m <= 16 ? launch_rows_of<T, B_KC, 16>(p, any, s) : launch_rows_of<T, B_KC, 32>(p, any, s);
}

template <typename T>
int launch_gemm(const DzGemmArgs& p, const DzGemmPlan& plan, bool a_kc, bool b_kc, hipStream_t s) {
  if (plan.tile < 0) {
    if (!a_kc || p.m > kRowsMost || p.splits != 1) return DZ_ERR_UNSUPPORTED;
    const bool any = plan.tile == kRowsAnyTile;
    return b_kc ? launch_rows<T, true>(p, any, s) : launch_rows<T, false>(p, any, s);
  }
  int rc;
  if (a_kc && b_kc) rc = launch_gemm_kind<T, true, true>(p, plan, s);
  else if (a_kc) rc = launch_gemm_kind<T, true, false>(p, plan, s);
  else if (!b_kc) rc = launch_gemm_kind<T, false, false>(p, plan, s);
  else rc = DZ_ERR_UNSUPPORTED;
  if (rc != DZ_OK || p.splits == 1) return rc;
  const dim3 grid((p.n + 255) / 256, p.m < 65535 ? p.m : 65535);
  hipLaunchKernelGGL((linear_finish_kernel<T>), grid, dim3(64), 0, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
int launch_dact(const DzDactArgs& p, int chunks, hipStream_t s) {
  hipLaunchKernelGGL((linear_dact_kernel<T>), dim3((p.n + 64 * (16 / (int)sizeof(T)) - 1) / (64 * (16 / (int)sizeof(T))), chunks), dim3(256), 0, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
int launch_pack(const DzPackArgs& p, hipStream_t s) {
  constexpr int kCols = 64 * (16 / (int)sizeof(T));
  const int cols = p.one.cols > p.two.cols ? p.one.cols : p.two.cols;
  int64_t rows = ((p.one.rows > p.two.rows ? p.one.rows : p.two.rows) + 4 * kPackRows - 1) / (4 * kPackRows);
  if (rows > 65535) rows = 65535;
  const dim3 grid((cols + kCols - 1) / kCols, (unsigned)rows, p.two.src ? 2 : 1);
  hipLaunchKernelGGL((linear_pack_kernel<T>), grid, dim3(256), 0, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
int launch_db(const float* sums, int chunks, int n, void* db, int db_f32, hipStream_t s) {
  hipLaunchKernelGGL((linear_db_kernel<T>), dim3((n + 63) / 64), dim3(256), 0, s, sums, chunks, n, db, db_f32);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
const DzLinearLaunch* linear_launches() {
  static const DzLinearLaunch l = {launch_gemm<T>, launch_dact<T>, launch_pack<T>, launch_db<T>};
  return &l;
}

}  // namespace
