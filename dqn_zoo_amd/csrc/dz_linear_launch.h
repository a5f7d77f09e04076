// The launches of the dense-layer operator for one element type; included by one unit per type.
#pragma once

#include "dz_linear.h"

namespace {

template <typename T, bool A_KC, bool B_KC, int TILE>
int launch_gemm_tile(const DzGemmArgs& p, hipStream_t s) {
  constexpr DzGemmShape t = kGemmTiles[TILE];
  constexpr int kLds = 2 * (t.bm + t.bn) * 128;
  const int64_t tiles = (int64_t)((p.m + t.bm - 1) / t.bm) * ((p.n + t.bn - 1) / t.bn);
  if (tiles >= (1ll << 31)) return DZ_ERR_UNSUPPORTED;
  auto kernel = linear_gemm_kernel<T, A_KC, B_KC, t.bm, t.bn, t.wm, t.wn>;
  if (kLds > 65536)
    DZ_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)p.splits), dim3(64 * t.wm * t.wn), kLds, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T, bool A_KC, bool B_KC>
int launch_gemm_kind(const DzGemmArgs& p, const DzGemmPlan& plan, hipStream_t s) {
  switch (plan.tile) {
    case 0:   // (16 rows: only where the rows of A lie one behind the other)
      if constexpr (A_KC) return launch_gemm_tile<T, A_KC, B_KC, 0>(p, s);
      return DZ_ERR_UNSUPPORTED;
    case 1: return launch_gemm_tile<T, A_KC, B_KC, 1>(p, s);
    case 2: return launch_gemm_tile<T, A_KC, B_KC, 2>(p, s);
    case 3: return launch_gemm_tile<T, A_KC, B_KC, 3>(p, s);
    default: return DZ_ERR_UNSUPPORTED;
  }
}

template <typename T>
int launch_gemm(const DzGemmArgs& p, const DzGemmPlan& plan, bool a_kc, bool b_kc, hipStream_t s) {
  int rc;
  if (a_kc && b_kc) rc = launch_gemm_kind<T, true, true>(p, plan, s);
  else if (a_kc) rc = launch_gemm_kind<T, true, false>(p, plan, s);
  else if (!b_kc) rc = launch_gemm_kind<T, false, false>(p, plan, s);
  else rc = DZ_ERR_UNSUPPORTED;
  if (rc != DZ_OK || p.splits == 1) return rc;
  const int64_t blocks = (p.slab_ld / 4 * p.m + 255) / 256;
  if (blocks >= (1ll << 31)) return DZ_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((linear_finish_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, p);
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
  const int64_t one = p.one.rows * (p.one.ldd / (16 / (int64_t)sizeof(T)));
  const int64_t two = p.two.src ? p.two.rows * (p.two.ldd / (16 / (int64_t)sizeof(T))) : 0;
  const int64_t blocks = ((one > two ? one : two) + 255) / 256;
  if (blocks >= (1ll << 31)) return DZ_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((linear_pack_kernel<T>), dim3((unsigned)blocks, p.two.src ? 2 : 1), dim3(256), 0, s, p);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
int launch_db(const float* sums, int chunks, int n, void* db, int db_f32, hipStream_t s) {
  hipLaunchKernelGGL((linear_db_kernel<T>), dim3((n + 255) / 256), dim3(256), 0, s, sums, chunks, n, db, db_f32);
  DZ_LAUNCH_CHECK();
  return DZ_OK;
}

template <typename T>
const DzLinearLaunch* linear_launches() {
  static const DzLinearLaunch l = {launch_gemm<T>, launch_dact<T>, launch_pack<T>, launch_db<T>};
  return &l;
}

}  // namespace
