// What the dense-layer operator's units share: one product's plan, made on the host
// (dz_linear.hip), and the launches of each element type (dz_linear_{f32,bf16,f16}.hip).
#pragma once

#include "dz_linear_gemm.h"

struct DzGemmPlan {
  int tile;            // index of the tile sizes, or kRows*Tile
  int splits, k_split;
  int64_t slab_bytes;  // 0 without splits
};

// Every launch of one element type.  The functions return DZ_OK or a DZ_ERR_* code.
struct DzLinearLaunch {
  int (*gemm)(const DzGemmArgs&, const DzGemmPlan&, bool a_kc, bool b_kc, hipStream_t);
  int (*dact)(const DzDactArgs&, int chunks, hipStream_t);
  int (*pack)(const DzPackArgs&, hipStream_t);   // two.src may be NULL
  int (*db)(const float* sums, int chunks, int n, void* db, int db_f32, hipStream_t);
};
const DzLinearLaunch* dz_linear_launch_f32();
const DzLinearLaunch* dz_linear_launch_bf16();
const DzLinearLaunch* dz_linear_launch_f16();

constexpr DzGemmShape kGemmTiles[] = {{64, 64, 2, 2, 3}, {128, 128, 2, 2, 2}, {256, 256, 2, 4, 2}};
constexpr int kGemmTileCount = sizeof(kGemmTiles) / sizeof(kGemmTiles[0]);
constexpr int kRowsTile = -1;      // linear_rows_kernel
constexpr int kRowsAnyTile = -2;   // linear_rows_any_kernel: operands of any alignment
constexpr int kRowsMost = 32;      // their rows
