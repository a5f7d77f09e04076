// The dense layer as an operator: y = act(x w + b) + residual, and its gradients
// (include/dqnzoo_hip.h: dz_linear, dz_linear_backward).  Host side: argument checks, the choice of
// tiles and splits, workspaces.  Kernels: dz_linear_gemm.h.
#include "dz_linear.h"

namespace {

constexpr int kCus = 256;

const DzLinearLaunch* launches(int dtype) {
  return dtype == DZ_F32 ? dz_linear_launch_f32() : dtype == DZ_BF16 ? dz_linear_launch_bf16()
       : dtype == DZ_F16 ? dz_linear_launch_f16() : nullptr;
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Rows at multiples of 16 bytes, and whole 16-byte units of the adjacent index.
bool unit_aligned(const void* x, int64_t ld, int64_t adjacent, int64_t elem) {
  const int64_t ve = 16 / elem;
  return ((uintptr_t)x & 15) == 0 && ld % ve == 0 && adjacent % ve == 0;
}

// Tile and number of splits: the least estimated time.  A workgroup's stage costs its matrix
// instructions or its share of the memory system, whichever is more; workgroups run in rounds of
// the chip; splits add the slabs' way out and back.
DzGemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int64_t elem, bool dma) {
  DzGemmPlan best{};
  best.dma = dma;
  double best_us = 1e30;
  const int bk = (int)(128 / elem);
  const int64_t stages = (k + bk - 1) / bk;
  for (int t = 0; t < (dma ? kGemmTileCount : 2); ++t) {   // (256 x 256 staged through registers would spill)
    const DzGemmShape g = kGemmTiles[t];
    const int64_t tiles = ((m + g.bm - 1) / g.bm) * ((n + g.bn - 1) / g.bn);
    const int per_cu = t == 0 ? 4 : t == 1 ? 2 : 1;
    for (int s = 1; s <= kMaxSplits; s *= 2) {
      if (s > 1 && (stages / s < 2 || tiles * s > 4 * kCus)) break;
      const int64_t depth = (stages + s - 1) / s;
      // us of one stage of one workgroup alone on its CU: products at ~60 % of the CU's rate
      const double rate = elem == 2 ? 5.5e6 : 0.5e6;   // flop / us of a CU
      const double busy = 2.0 * g.bm * g.bn * bk / rate;
      const int64_t on_chip = tiles * s < (int64_t)kCus * per_cu ? tiles * s : (int64_t)kCus * per_cu;
      const double rounds = (double)((tiles * s + (int64_t)kCus * per_cu - 1) / ((int64_t)kCus * per_cu));
      const double sharing = on_chip > kCus ? (double)on_chip / kCus : 1.0;
      const double latency = 0.5;                      // us a stage takes at least
      const double stage_us = busy * sharing > latency ? busy * sharing : latency;
      double us = 2.0 + rounds * depth * stage_us;
      if (s > 1) us += 3.0 + 2.0 * s * (double)m * n * 4 / 4e6;
      if (us < best_us) {
        best_us = us;
        best.tile = t;
        best.splits = s;
        best.k_split = (int)(depth * bk);
      }
    }
  }
  best.splits = (int)((stages + best.k_split / bk - 1) / (best.k_split / bk));
  best.slab_bytes = best.splits > 1 ? best.splits * m * round_up(n, 4) * 4 : 0;
  return best;
}

int64_t slab_bytes(int64_t m, int64_t n, int64_t k, int64_t elem) {   // whichever way it will be staged
  const int64_t a = plan_gemm(m, n, k, elem, true).slab_bytes, b = plan_gemm(m, n, k, elem, false).slab_bytes;
  return a > b ? a : b;
}

void use_plan(DzGemmArgs& g, const DzGemmPlan& plan, void* slabs) {
  g.splits = plan.splits;
  g.k_split = plan.k_split;
  g.slabs = (float*)slabs;
  g.slab_ld = round_up(g.n, 4);
  g.slab_stride = g.m * g.slab_ld;
}

// rows of one chunk of the column sums: enough workgroups to fill the chip
int dact_rows(int64_t m, int64_t n) {
  const int64_t cols = (n + 255) / 256;
  int64_t chunks = 4 * kCus / cols;
  if (chunks < 1) chunks = 1;
  int64_t rows = round_up((m + chunks - 1) / chunks, 4);
  return (int)(rows < 32 ? 32 : rows);
}

struct BackwardPlan {
 bool dz;                       // dz is formed in the workspace
  int64_t ld_dz;
  int rows, chunks;
  int64_t dz_at, sums_at, slabs_at, bytes;
};

BackwardPlan plan_backward(const dz_linear_args_t* a) {
  BackwardPlan b{};
  const int64_t elem = dz_elem_bytes(a->dtype);
  b.dz = a->activation != DZ_ACT_NONE;
  b.ld_dz = round_up(a->n, 16 / elem);
  b.rows = dact_rows(a->m, a->n);
  b.chunks = (int)((a->m + b.rows - 1) / b.rows);
  int64_t at = 0;
  b.dz_at = at;
  if (b.dz) at += round_up(a->m * b.ld_dz * elem, 256);
  b.sums_at = at;
  if (b.chunks > 1) at += round_up((int64_t)b.chunks * a->n * 4, 256);
  b.slabs_at = at;
  const int64_t dx = slab_bytes(a->m, a->k, a->n, elem);
  const int64_t dw = a->w_transposed ? slab_bytes(a->n, a->k, a->m, elem) : slab_bytes(a->k, a->n, a->m, elem);
  b.bytes = at + (dx > dw ? dx : dw);
  return b;
}

bool sizes_ok(const dz_linear_args_t* a) {
  const int64_t most = (1ll << 31) - 1024;
  return a && dz_is_dtype(a->dtype) && a->activation >= DZ_ACT_NONE && a->activation <= DZ_ACT_SILU &&
         a->m > 0 && a->k > 0 && a->n > 0 && a->m < most && a->k < most && a->n < most;
}
bool strides_ok(const dz_linear_args_t* a) {
  return a->x && a->w && a->ldx >= a->k && a->ldw >= (a->w_transposed ? a->k : a->n);
}
bool workspace_ok(const dz_linear_args_t* a, int64_t need) {
  return need == 0 || (a->ws && a->ws_bytes >= need && ((uintptr_t)a->ws & 15) == 0);
}

}  // namespace

extern "C" int dz_linear_workspace(const dz_linear_args_t* a, int backward, int64_t* bytes) {
  DZ_REQUIRE(bytes && sizes_ok(a));
  *bytes = backward ? plan_backward(a).bytes : slab_bytes(a->m, a->n, a->k, dz_elem_bytes(a->dtype));
  return DZ_OK;
}

extern "C" int dz_linear(const dz_linear_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(sizes_ok(a) && strides_ok(a) && a->y && a->ldy >= a->n);
  DZ_REQUIRE(!a->residual || a->ldr >= a->n);
  DZ_REQUIRE(!a->preact || a->ldz >= a->n);
  const int64_t elem = dz_elem_bytes(a->dtype);
  const DzGemmPlan plan = plan_gemm(
      a->m, a->n, a->k, elem,
      unit_aligned(a->x, a->ldx, a->k, elem) && unit_aligned(a->w, a->ldw, a->w_transposed ? a->k : a->n, elem));
  DZ_REQUIRE(workspace_ok(a, slab_bytes(a->m, a->n, a->k, elem)));
  DzGemmArgs g{};
  g.a = a->x; g.lda = a->ldx;
  g.b = a->w; g.ldb = a->ldw;
  g.m = (int)a->m; g.n = (int)a->n; g.k = (int)a->k;
  g.bias = a->bias; g.bias_f32 = a->bias_f32;
  g.residual = a->residual; g.ldr = a->ldr;
  g.y = a->y; g.ldy = a->ldy;
  g.preact = a->preact; g.ldz = a->ldz;
  g.activation = a->activation;
  use_plan(g, plan, a->ws);
  return launches(a->dtype)->gemm(g, plan, true, a->w_transposed != 0, dz_s(stream));
}

extern "C" int dz_linear_backward(const dz_linear_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(sizes_ok(a) && a->dy && a->lddy >= a->n && (a->dx || a->dw || a->db));
  DZ_REQUIRE(!a->dx || (a->w && a->ldw >= (a->w_transposed ? a->k : a->n) && a->lddx >= a->k));
  DZ_REQUIRE(!a->dw || (a->x && a->ldx >= a->k && a->lddw >= (a->w_transposed ? a->k : a->n)));
  DZ_REQUIRE(a->activation == DZ_ACT_NONE || (a->preact && a->ldz >= a->n));
  const BackwardPlan b = plan_backward(a);
  DZ_REQUIRE(workspace_ok(a, b.bytes));
  const hipStream_t s = dz_s(stream);
  const int64_t elem = dz_elem_bytes(a->dtype);
  const DzLinearLaunch* l = launches(a->dtype);
  char* ws = (char*)a->ws;
  const void* dz = a->dy;
  int64_t lddz = a->lddy;
  if (b.dz || a->db) {
    DzDactArgs d{};
    d.dy = a->dy; d.ldy = a->lddy;
    if (b.dz) {
      d.z = a->preact; d.ldz = a->ldz;
      if (a->dx || a->dw) {
        d.dz = ws + b.dz_at; d.lddz = b.ld_dz;
        dz = d.dz; lddz = b.ld_dz;
      }
    }
    d.m = (int)a->m; d.n = (int)a->n; d.rows = b.rows; d.activation = a->activation;
    if (a->db) {
      if (b.chunks > 1) d.sums = (float*)(ws + b.sums_at);
      else { d.db = a->db; d.db_f32 = a->grads_f32; }
    }
    int rc = l->dact(d, b.chunks, s);
    if (rc != DZ_OK) return rc;
    if (d.sums) rc = l->db(d.sums, b.chunks, d.n, a->db, a->grads_f32, s);
    if (rc != DZ_OK) return rc;
  }
  if (a->dx) {   // dx[m][k] = dz[m][n] w[k][n]^T
    const DzGemmPlan plan = plan_gemm(
        a->m, a->k, a->n, elem,
        unit_aligned(dz, lddz, a->n, elem) && unit_aligned(a->w, a->ldw, a->w_transposed ? a->k : a->n, elem));
    DzGemmArgs g{};
    g.a = dz; g.lda = lddz;
    g.b = a->w; g.ldb = a->ldw;
    g.m = (int)a->m; g.n = (int)a->k; g.k = (int)a->n;
    g.y = a->dx; g.ldy = a->lddx;
    use_plan(g, plan, ws + b.slabs_at);
    const int rc = l->gemm(g, plan, true, a->w_transposed == 0, s);
    if (rc != DZ_OK) return rc;
  }
  if (a->dw) {   // dw[k][n] = x[m][k]^T dz[m][n], or its transpose in a transposed weight's layout
    const bool t = a->w_transposed != 0;
    const DzGemmPlan plan = plan_gemm(t ? a->n : a->k, t ? a->k : a->n, a->m, elem,
                                      unit_aligned(dz, lddz, a->n, elem) && unit_aligned(a->x, a->ldx, a->k, elem));
    DzGemmArgs g{};
    g.a = t ? dz : a->x; g.lda = t ? lddz : a->ldx;
    g.b = t ? a->x : dz; g.ldb = t ? a->ldx : lddz;
    g.m = (int)(t ? a->n : a->k); g.n = (int)(t ? a->k : a->n); g.k = (int)a->m;
    g.y = a->dw; g.ldy = a->lddw; g.y_f32 = a->grads_f32;
    use_plan(g, plan, ws + b.slabs_at);
    const int rc = l->gemm(g, plan, false, false, s);
    if (rc != DZ_OK) return rc;
  }
  return DZ_OK;
}
