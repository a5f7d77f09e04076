// The dense layer as an operator: y = act(x w + b) + residual, and its gradients
// (include/dqnzoo_hip.h: dz_linear, dz_linear_backward).  Host side: argument checks, the choice of
// tiles and splits, workspaces.  Kernels: dz_linear_gemm.h.
#include "dz_linear.h"

namespace {

constexpr int kCus = 256;
constexpr int64_t kMaxPitchBytes = 1 << 24;   // 256 rows of it in a 32-bit offset
constexpr int64_t kMaxThreads = 1ll << 32;    // of one launch, along one axis of its grid

const DzLinearLaunch* launches(int dtype) {
  return dtype == DZ_F32 ? dz_linear_launch_f32() : dtype == DZ_BF16 ? dz_linear_launch_bf16()
       : dtype == DZ_F16 ? dz_linear_launch_f16() : nullptr;
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// A matrix in memory: `rows` rows of `cols` adjacent elements, `ld` elements apart.
struct Matrix { const void* at; int64_t ld, rows, cols; };

// Whether the main loop can read it where it lies: rows of whole 16-byte units.
bool readable(const Matrix& x, int64_t elem) {
  const int64_t ve = 16 / elem;
  return x.at && ((uintptr_t)x.at & 15) == 0 && x.ld % ve == 0 && x.cols % ve == 0 && x.ld * elem <= kMaxPitchBytes;
}
// Rows of a copy begin at multiples of 128 bytes: a stage's piece of one would lie in two cache lines
// otherwise (1777 x 1235 x 1001 fp16: 18.2 -> 15.9 us).
int64_t packed_ld(const Matrix& x, int64_t elem) { return round_up(x.cols, 128 / elem); }
int64_t packed_bytes(const Matrix& x, int64_t elem) { return round_up(x.rows * packed_ld(x, elem) * elem, 256); }

// Measured on this card (us; sweeps of tiles and splits over 30 shapes): what a stage of a workgroup
// takes when its CU has nothing else (`alone`, of one workgroup on the chip, up to `full` of 256),
// and what each of many costs a busy CU.
struct TileCost { double alone, full, busy; int per_cu; };
constexpr double kAnySlower = 1.5;   // the rows' kernel through registers
constexpr TileCost kCost16[] = {{0.22, 0.25, 0.185, 3}, {0.61, 0.95, 0.53, 2}, {1.10, 1.90, 1.90, 1}};
constexpr TileCost kCost32[] = {{0.58, 0.60, 0.455, 3}, {2.00, 2.00, 1.85, 2}, {7.20, 7.40, 7.40, 1}};

// Tile and number of splits: the least estimated time, with the operands' bytes at 5.3 TB/s as its
// floor.  A split costs its slab's way out and back and a second launch.  Up to 32 rows may take the
// rows' kernel: 1 x 3136 x 512 in 5.2 us against 8.7 (tile 64 x 64, 7 splits), 16 x 8192 x 4096 from
// a transposed weight in 15.0 against 15.7; its 64-byte pieces of an (in, out) weight's rows come at
// 2.4 TB/s (16 x 8192 x 4096: 25.8 against 16.8).
DzGemmPlan plan_gemm(int64_t m, int64_t n, int64_t k, int64_t elem, bool a_kc, bool b_kc, int64_t copied = 0,
                     bool rows = true) {
  DzGemmPlan best{};
  double best_us = 1e30;
  const int bk = (int)(128 / elem);
  const int64_t stages = (k + bk - 1) / bk;
  const double bytes = (double)(m + n) * k * elem;
  const double copy = copied ? 3.0 + 2.0 * copied / 4e6 : 0.0;   // `copied` bytes of operands, a launch of their own
  if (rows && a_kc && m <= kRowsMost) {
    const int64_t rounds = ((n + kRowsN - 1) / kRowsN + kCus - 1) / kCus, depth = (stages + kRowsWaves - 1) / kRowsWaves;
    const double work = rounds * depth * (elem == 2 ? 0.30 : m <= 16 ? 0.56 : 1.0), flow = bytes / (b_kc || elem == 4 ? 5.3e6 : 2.4e6);
    best_us = 3.0 + (work > flow ? work : flow) * (copied ? kAnySlower : 1.0) + 0.9 * (rounds - 1);
    best.tile = copied ? kRowsAnyTile : kRowsTile;
    best.splits = 1;
    best.k_split = (int)(stages * bk);
  }
  for (int t = 0; t < kGemmTileCount; ++t) {
    const DzGemmShape g = kGemmTiles[t];
    const TileCost c = elem == 2 ? kCost16[t] : kCost32[t];
    const int64_t tiles = ((m + g.bm - 1) / g.bm) * ((n + g.bn - 1) / g.bn);
    if (t + 1 < kGemmTileCount && tiles * g.wm * g.wn * 64 >= kMaxThreads) continue;
    for (int s = 1; s <= kMaxSplits; s *= 2) {
      if (s > 1 && (stages / s < 2 || tiles * s > 4 * kCus)) break;
      const int64_t depth = (stages + s - 1) / s, groups = tiles * s;
      const int64_t per_cu = (groups + kCus - 1) / kCus, rounds = (per_cu + c.per_cu - 1) / c.per_cu;
      const double load = groups < kCus ? (double)groups / kCus : 1.0;
      const double one = c.alone + (c.full - c.alone) * load;
      const double stage = rounds * one > per_cu * c.busy ? rounds * one : per_cu * c.busy;
      double us = 3.5 + copy + (depth * stage > bytes / 5.3e6 ? depth * stage : bytes / 5.3e6);
      if (s > 1) us += 2.8 + 0.1 * s + 2.0 * s * (double)m * n * 4 / 3e6;
      if (us < best_us) {
        best_us = us;
        best.tile = t;
        best.splits = s;
        best.k_split = (int)(depth * bk);
      }
    }
  }
  best.splits = (int)((stages + best.k_split / bk - 1) / (best.k_split / bk));
  best.slab_bytes = best.splits > 1 ? best.splits * m * round_up(n, 8) * 4 : 0;
  return best;
}

void use_plan(DzGemmArgs& g, const DzGemmPlan& plan, void* slabs) {
  g.splits = plan.splits;
  g.k_split = plan.k_split;
  g.slabs = (float*)slabs;
  g.slab_ld = round_up(g.n, 8);
  g.slab_stride = g.m * g.slab_ld;
}

Matrix x_of(const dz_linear_args_t* a) { return {a->x, a->ldx, a->m, a->k}; }
Matrix w_of(const dz_linear_args_t* a) {
  return a->w_transposed ? Matrix{a->w, a->ldw, a->n, a->k} : Matrix{a->w, a->ldw, a->k, a->n};
}

// What a call keeps in its workspace, from its start.  (`a` may have no pointers yet: an operand
// without an address is taken to need its copy.)
struct Layout {
  bool pack_x, pack_w, form_dz;
  DzGemmPlan fwd, dx, dw;
  int64_t x_at, w_at, dz_at, sums_at, slabs_at, bytes;
  int rows, chunks;          // of the column sums
};

Layout plan_forward(const dz_linear_args_t* a) {
  Layout l{};
  const int64_t elem = dz_elem_bytes(a->dtype);
  l.pack_x = !readable(x_of(a), elem);
  l.pack_w = !readable(w_of(a), elem);
  const int64_t copied = (l.pack_x ? packed_bytes(x_of(a), elem) : 0) + (l.pack_w ? packed_bytes(w_of(a), elem) : 0);
  // (sizes alone: the copies and the slabs that a call may need, so not the rows' kernel)
  l.fwd = plan_gemm(a->m, a->n, a->k, elem, true, a->w_transposed != 0, copied, a->x && a->w);
  if (l.fwd.tile == kRowsAnyTile) l.pack_x = l.pack_w = false;
  if (l.pack_x) { l.x_at = l.bytes; l.bytes += packed_bytes(x_of(a), elem); }
  if (l.pack_w) { l.w_at = l.bytes; l.bytes += packed_bytes(w_of(a), elem); }
  l.slabs_at = l.bytes;
  l.bytes += l.fwd.slab_bytes;
  return l;
}

Layout plan_backward(const dz_linear_args_t* a) {
  Layout l{};
  const int64_t elem = dz_elem_bytes(a->dtype);
  const bool sizes_only = !a->dy, dx = sizes_only || a->dx, dw = sizes_only || a->dw, db = sizes_only || a->db;
  const Matrix dy{a->dy, a->lddy, a->m, a->n};
  l.form_dz = (dx || dw) && (a->activation != DZ_ACT_NONE || !readable(dy, elem));
  l.pack_x = dw && !readable(x_of(a), elem);
  l.pack_w = dx && !readable(w_of(a), elem);
  if (dx) l.dx = plan_gemm(a->m, a->k, a->n, elem, true, a->w_transposed == 0,
                           l.pack_w ? packed_bytes(w_of(a), elem) : 0, !sizes_only);
  if (l.dx.tile == kRowsAnyTile) l.pack_w = false;
  if (dw) l.dw = a->w_transposed ? plan_gemm(a->n, a->k, a->m, elem, false, false)
                                       : plan_gemm(a->k, a->n, a->m, elem, false, false);
  // rows of one chunk of the column sums: four workgroups per CU, if the rows allow; one chunk for a
  // batch of 32 (no second launch)
  const int64_t cols = (a->n + 64 * (16 / elem) - 1) / (64 * (16 / elem));
  const int64_t wanted = 4 * kCus / cols < 1 ? 1 : 4 * kCus / cols;
  const int64_t rows = round_up((a->m + wanted - 1) / wanted, 8);
  l.rows = (int)(a->m <= 32 ? 32 : rows < 16 ? 16 : rows);
  l.chunks = (int)((a->m + l.rows - 1) / l.rows);
  if (l.pack_x) { l.x_at = l.bytes; l.bytes += packed_bytes(x_of(a), elem); }
  if (l.pack_w) { l.w_at = l.bytes; l.bytes += packed_bytes(w_of(a), elem); }
  if (l.form_dz) { l.dz_at = l.bytes; l.bytes += packed_bytes(dy, elem); }
  if (db && l.chunks > 1) { l.sums_at = l.bytes; l.bytes += round_up((int64_t)l.chunks * a->n * 4, 256); }
  l.slabs_at = l.bytes;
  l.bytes += l.dx.slab_bytes > l.dw.slab_bytes ? l.dx.slab_bytes : l.dw.slab_bytes;
  return l;
}

// x and w as the main loop reads them, copied first where they have to be
int operands(const dz_linear_args_t* a, const Layout& l, Matrix& x, Matrix& w, hipStream_t s) {
  const int64_t elem = dz_elem_bytes(a->dtype);
  char* ws = (char*)a->ws;
  x = x_of(a);
  w = w_of(a);
  DzPackArgs p{};
  auto copy = [&](Matrix& q, int64_t at) {
    DzPackArgs::One& one = p.one.src ? p.two : p.one;
    one = {q.at, q.ld, q.rows, (int)q.cols, ws + at, packed_ld(q, elem)};
    q.at = one.dst;
    q.ld = one.ldd;
  };
  if (l.pack_x) copy(x, l.x_at);
  if (l.pack_w) copy(w, l.w_at);
  return p.one.src ? launches(a->dtype)->pack(p, s) : DZ_OK;
}

bool sizes_ok(const dz_linear_args_t* a) {
  if (!a || !dz_is_dtype(a->dtype) || a->activation < DZ_ACT_NONE || a->activation > DZ_ACT_SILU) return false;
  const int64_t wide = kMaxPitchBytes / dz_elem_bytes(a->dtype);
  return a->m > 0 && a->k > 0 && a->n > 0 && a->m < (1ll << 31) - 1024 && a->k <= wide && a->n <= wide;
}
bool workspace_ok(const dz_linear_args_t* a, int64_t need) {
  return need == 0 || (a->ws && a->ws_bytes >= need && ((uintptr_t)a->ws & 15) == 0);
}

}  // namespace

extern "C" int dz_linear_workspace(const dz_linear_args_t* a, int backward, int64_t* bytes) {
  DZ_REQUIRE(bytes && sizes_ok(a));
  *bytes = backward ? plan_backward(a).bytes : plan_forward(a).bytes;
  return DZ_OK;
}

extern "C" int dz_linear(const dz_linear_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(sizes_ok(a) && a->x && a->w && a->ldx >= a->k && a->ldw >= (a->w_transposed ? a->k : a->n));
  DZ_REQUIRE(a->y && a->ldy >= a->n);
  DZ_REQUIRE(!a->residual || a->ldr >= a->n);
  DZ_REQUIRE(!a->preact || a->ldz >= a->n);
  const Layout l = plan_forward(a);
  DZ_REQUIRE(workspace_ok(a, l.bytes));
  const hipStream_t s = dz_s(stream);
  Matrix x, w;
  const int rc = operands(a, l, x, w, s);
  if (rc != DZ_OK) return rc;
  const int64_t elem = dz_elem_bytes(a->dtype);
  DzGemmArgs g{};
  g.a = x.at; g.lda = x.ld;
  g.b = w.at; g.ldb = w.ld;
  g.m = (int)a->m; g.n = (int)a->n; g.k = (int)a->k;
  g.bias = a->bias; g.bias_f32 = a->bias_f32;
  g.residual = a->residual; g.ldr = a->ldr;
  g.y = a->y; g.ldy = a->ldy;
  g.preact = a->preact; g.ldz = a->ldz;
  g.activation = a->activation;
  // An output that no cache would hold until it is read: 4 - 5 % on 256 MB, nothing on 64.
  g.stream = a->m * a->n * elem * (a->preact ? 2 : 1) >= (128ll << 20);
  use_plan(g, l.fwd, (char*)a->ws + l.slabs_at);
  return launches(a->dtype)->gemm(g, l.fwd, true, a->w_transposed != 0, s);
}

extern "C" int dz_linear_backward(const dz_linear_args_t* a, dz_stream_t stream) {
  DZ_REQUIRE(sizes_ok(a) && a->dy && a->lddy >= a->n && (a->dx || a->dw || a->db));
  DZ_REQUIRE(!a->dx || (a->w && a->ldw >= (a->w_transposed ? a->k : a->n) && a->lddx >= a->k));
  DZ_REQUIRE(!a->dw || (a->x && a->ldx >= a->k && a->lddw >= (a->w_transposed ? a->k : a->n)));
  DZ_REQUIRE(a->activation == DZ_ACT_NONE || (a->preact && a->ldz >= a->n));
  const Layout l = plan_backward(a);
  DZ_REQUIRE(workspace_ok(a, l.bytes));
  const hipStream_t s = dz_s(stream);
  const DzLinearLaunch* launch = launches(a->dtype);
  const int64_t elem = dz_elem_bytes(a->dtype);
  char* ws = (char*)a->ws;
  Matrix dz{a->dy, a->lddy, a->m, a->n}, x, w;
  int rc = DZ_OK;
  if (l.form_dz || a->db) {
    DzDactArgs d{};
    d.dy = a->dy; d.ldy = a->lddy;
    if (a->activation != DZ_ACT_NONE) { d.z = a->preact; d.ldz = a->ldz; }
    if (l.form_dz) {
      d.dz = ws + l.dz_at; d.lddz = packed_ld(dz, elem);
      dz.at = d.dz; dz.ld = d.lddz;
    }
    d.m = (int)a->m; d.n = (int)a->n; d.rows = l.rows; d.activation = a->activation;
    if (a->db) {
      if (l.chunks > 1) d.sums = (float*)(ws + l.sums_at);
      else { d.db = a->db; d.db_f32 = a->grads_f32; }
    }
    rc = launch->dact(d, l.chunks, s);
    if (rc == DZ_OK && d.sums) rc = launch->db(d.sums, l.chunks, d.n, a->db, a->grads_f32, s);
    if (rc != DZ_OK) return rc;
  }
  rc = operands(a, l, x, w, s);
  if (rc != DZ_OK) return rc;
  if (a->dx) {   // dx[m][k] = dz[m][n] w[k][n]^T
    DzGemmArgs g{};
    g.a = dz.at; g.lda = dz.ld;
    g.b = w.at; g.ldb = w.ld;
    g.m = (int)a->m; g.n = (int)a->k; g.k = (int)a->n;
    g.y = a->dx; g.ldy = a->lddx;
    use_plan(g, l.dx, ws + l.slabs_at);
    rc = launch->gemm(g, l.dx, true, a->w_transposed == 0, s);
    if (rc != DZ_OK) return rc;
  }
  if (a->dw) {   // dw[k][n] = x[m][k]^T dz[m][n], or its transpose in a transposed weight's layout
    const bool t = a->w_transposed != 0;
    DzGemmArgs g{};
    g.a = t ? dz.at : x.at; g.lda = t ? dz.ld : x.ld;
    g.b = t ? x.at : dz.at; g.ldb = t ? x.ld : dz.ld;
    g.m = (int)(t ? a->n : a->k); g.n = (int)(t ? a->k : a->n); g.k = (int)a->m;
    g.y = a->dw; g.ldy = a->lddw; g.y_f32 = a->grads_f32;
    use_plan(g, l.dw, ws + l.slabs_at);
    rc = launch->gemm(g, l.dw, false, false, s);
  }
  return rc;
}
