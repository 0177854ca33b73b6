// Dispatch of the dense head's linear layers: which kernel takes a product, how it
// is split, and where its intermediates live in the caller's workspace.
#include "dense.h"

namespace sft {
namespace dense {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

namespace {

constexpr int kStage = 64;         // bytes of k per pipeline stage
constexpr int64_t kCus = 256;
constexpr int64_t kStrideMost = (int64_t)1 << 23;  // bytes: a tile's rows span less than 32 bits count

size_t a256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t type_size(int dtype) { return dtype == SFT_TYPE_F32 ? 4 : 2; }
int64_t padded(int64_t n, int64_t es) { return (n + 16 / es - 1) & ~(16 / es - 1); }

#define SFT_DENSE_CALL(dtype, F, ...)                         \
  (dtype == SFT_TYPE_F32   ? F<float>(__VA_ARGS__)            \
   : dtype == SFT_TYPE_F16 ? F<f16_t>(__VA_ARGS__)            \
                           : F<bf16_t>(__VA_ARGS__))

// How a product is cut into tiles, and its k into parts whose sums one more launch
// adds.  Taken is what a model of the time says is least: a CU works through its share
// of the tiles at a time per stage that was measured with many of them (below, us, at
// 8192^3 and 65536 x 1040 x 4096), each round of workgroups adds its first copies'
// latency and its results' stores, and partials are written and read at 4 TB/s.
// Measured both sides of the rule (bf16, us): 8192^3 forward 1550 in 64 x 128 tiles, 1180 in
// 128 x 128, 816 in 256 x 256; 16384 x 1040 x 1040 input grad 61, 51, 66; 2048^3 weight
// grad 25, 24, 41; 16384 x 1040 x 128 forward 15, 18, 26 (binary32: input grad 41, 44).
// Splitting k: weight grad of 16384 x 1040 x 128 108 -> 24 (binary32 549 -> 45), of
// 65536 x 1040 x 4096 897 -> 520, of 5000 x 1040 x 520 36 -> 22.
struct Cut {
  int tile, tiles_m, tiles_n, splits, split_k;
};
struct TileCost {
  int rows, cols, slots;              // slots: workgroups the card holds at once
  double stage[2], alone[2], round;   // us a stage of 16-bit types and of binary32, with many and one per CU
};
constexpr TileCost kTiles[3] = {{64, 128, 768, {0.22, 0.42}, {0.32, 0.58}, 4.0},
                                {128, 128, 768, {0.29, 0.70}, {0.42, 0.60}, 5.0},
                                {256, 256, 256, {0.84, 0.0}, {0.84, 0.0}, 8.0}};
Cut cut_of(int dtype, int64_t M, int64_t N, int64_t K) {
  const int64_t es = type_size(dtype), stages = ceil_div(K * es, kStage);
  Cut best = {};
  double least = 0.0;
  for (int t = 0; t < (es == 2 ? 3 : 2); ++t) {
    const TileCost &c = kTiles[t];
    const int64_t tm = ceil_div(M, c.rows), tn = ceil_div(N, c.cols), n = tm * tn;
    for (int64_t s = 1; s <= 64 && s * 8 <= stages + 7; ++s) {
      const int64_t per = ceil_div(stages, s), parts = ceil_div(stages, per);
      if (parts != s) continue;
      const int64_t load = ceil_div(n * s, kCus);
      const double stage = load == 1 ? c.alone[es == 4] : (double)load * c.stage[es == 4];
      double cost = (double)per * stage + (double)ceil_div(n * s, c.slots) * c.round;
      if (s > 1) cost += 4.0 + (double)s * (double)M * (double)N * 8.0 / 4e6;
      if (best.splits && cost >= least) continue;
      least = cost;
      best = Cut{t, (int)tm, (int)tn, (int)s, (int)(per * (kStage / es))};
    }
  }
  return best;
}

size_t part_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  const int s = cut_of(dtype, M, N, K).splits;
  return s > 1 ? a256((size_t)s * M * N * 4) : 0;
}

// Whether the row kernel takes a forward.  Each of its workgroups reads the rows (in
// groups of 16, 32 or 64) and 16 outputs' weights itself, which is all it does up to the
// bytes below; from there on tiles with split k win.  us, row kernel / tiles: bf16 K = 1040,
// N = 4096 1 row 2.9 / 6.6, 64 rows 5.3 / 10.1; K = 2048, N = 2048 48 rows 9.5 / 9.8, 64 rows
// 10.9 / 10.2; K = 4096, N = 1040 16 rows 8.9 / 10.9, 32 rows 12.4 / 11.3, 64 rows 19.6 / 12.6;
// binary32 K = 1040, N = 4096 64 rows 10.7 / 15.2, K = 4096, N = 1040 16 rows 16.0 / 12.5.
constexpr int64_t kRowsMost = 64, kRowBytesMost = 360 << 10;
bool few_rows(int64_t M, int64_t K, int64_t es) {
  const int64_t rows = M <= 16 ? 16 : M <= 32 ? 32 : 64;
  return M <= kRowsMost && (rows + 16) * K * es <= kRowBytesMost;
}

// A matrix that a product reads: rows of dense elements.
struct Matrix {
  const void *p;
  int64_t ld, rows, cols;
  // Whole aligned chunks with a stride that tiles can address: read in place.
  bool direct(int64_t es) const {
    return ((uintptr_t)p | (uintptr_t)(ld * es)) % 16 == 0 && cols % (16 / es) == 0 && ld * es <= kStrideMost;
  }
  size_t copy_bytes(int64_t es) const { return a256((size_t)rows * padded(cols, es) * es); }
};

// Takes pieces of the workspace.
struct Scratch {
  char *at;
  void *take(size_t n) {
    char *p = at;
    at += n;
    return p;
  }
};

// Replaces what is not read in place by aligned copies, in one launch.
int align(int dtype, Matrix *a, Matrix *b, Scratch &ws, hipStream_t s) {
  const int64_t es = type_size(dtype);
  Copy c[2] = {};
  int n = 0;
  Matrix *m[2] = {a, b};
  for (Matrix *x : m) {
    if (!x || x->direct(es)) continue;
    const int64_t ld = padded(x->cols, es);
    void *to = ws.take(x->copy_bytes(es));
    c[n++] = Copy{x->p, to, x->ld, ld, x->rows, x->cols};
    *x = Matrix{to, ld, x->rows, ld};
  }
  if (!n) return SFT_OK;
  ProfScope prof(kProfDenseAlign, s);
  return SFT_DENSE_CALL(dtype, launch_align, c[0], c[1], s);
}

// Whether the epilogue may access V elements at once.
bool epilogue_vec(const Epilogue &e, int64_t N, int64_t es, int64_t V) {
  auto ok = [&](const void *p, int64_t ld) { return !p || ((uintptr_t)p | (uintptr_t)(ld * es)) % (V * es) == 0; };
  return N % V == 0 && ok(e.y, e.ldy) && ok(e.bias, 0) && ok(e.residual, e.ldr) && ok(e.deriv, 0);
}

// C [M, N] of operands that are read in place.
int run_gemm(int dtype, int layout, const Matrix &a, const Matrix &b, int64_t M, int64_t N, int64_t K,
             const Epilogue &epi, float *sums, Scratch ws, hipStream_t s) {
  const int64_t es = type_size(dtype);
  const bool ak = layout != kWeightGrad, bk = layout == kForward;
  Gemm g = {};
  g.a = a.p;
  g.b = b.p;
  g.lda = a.ld;
  g.ldb = b.ld;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.ma = (int)(ak ? a.rows : a.cols);
  g.ka = (int)(ak ? a.cols : a.rows);
  g.nb = (int)(bk ? b.rows : b.cols);
  g.kb = (int)(bk ? b.cols : b.rows);
  if (g.K < g.ka) g.K = g.ka;
  if (g.K < g.kb) g.K = g.kb;
  g.epi = epi;
  g.epi.vec = epilogue_vec(epi, N, es, 16 / es);
  // Results past the caches, where a product's arithmetic takes longer than its stores:
  // they leave the operands their room.  65536 x 1040 x 4096 bf16 622 -> 561 us, 16384 x
  // 1040 x 1040 64 -> 59; with 4 stages (65536 x 1040 from 128) 46 -> 61.
  g.epi.stream = g.epi.vec && K * es >= 16 * kStage;
  const Cut c = cut_of(dtype, M, N, K);
  g.tile = c.tile;
  g.tiles_m = c.tiles_m;
  g.tiles_n = c.tiles_n;
  g.splits = c.splits;
  g.split_k = c.split_k;
  g.sums = sums;
  g.part = c.splits > 1 ? static_cast<float *>(ws.take(0)) : nullptr;
  ProfScope prof(kProfDenseProduct, s);
  return SFT_DENSE_CALL(dtype, launch_gemm, g, layout, s);
}

// The bias grad without an activation, from the weight grad's product: where its last tiles
// have a wave past the last column, that wave sums dy instead of idling, and dy is not read
// for it: 65536 x 1040 x 4096 bf16 1.81 -> 1.71 ms a step.  Else, and of binary32, whose products take
// six instructions, dy is read once more.  Returns the number of partials, 0 for else.
int product_sums(int dtype, bool dw, int64_t M, int64_t K, int64_t N, int act) {
  if (!dw || act != SFT_ACT_NONE || dtype == SFT_TYPE_F32) return 0;
  const Cut c = cut_of(dtype, N, K, M);
  return ceil_div(K, kWaveCols) * kWaveCols < (int64_t)c.tiles_n * kTiles[c.tile].cols ? c.splits : 0;
}

// The shape of the activation's backward and bias sums: about 1024 workgroups.
void shape_act_bwd(int dtype, int64_t M, int64_t N, ActBwd &p) {
  const int64_t chunks = ceil_div(N, 16 / type_size(dtype));
  p.M = M;
  p.N = (int)N;
  p.tx = 1;
  while (p.tx < kWave && p.tx < chunks) p.tx *= 2;
  const int64_t ty = kBlock / p.tx, want = ceil_div(1024, ceil_div(chunks, p.tx));
  p.rows = ceil_div(ceil_div(M, want), ty) * ty;
  p.parts = (int)ceil_div(M, p.rows);
}

__global__ __launch_bounds__(kBlock) void zero16_kernel(uint16_t *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) p[i] = 0;
}
void zero16(void *p, int64_t n, hipStream_t s) {
  const int64_t blocks = ceil_div(n, kBlock);
  hipLaunchKernelGGL(zero16_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kBlock), 0, s,
                     static_cast<uint16_t *>(p), n);
}

size_t copy_bytes(const Matrix &m, int64_t es, bool copied) { return copied || !m.direct(es) ? m.copy_bytes(es) : 0; }

}  // namespace

}  // namespace dense

using namespace dense;

// Workspace of the forward of these operands; copied: whatever their alignment.
size_t linear_fwd_workspace(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t M, int64_t K,
                            int64_t N, bool copied) {
  const int64_t es = type_size(dtype);
  if (few_rows(M, K, es)) return 0;
  return copy_bytes(Matrix{x, ldx, M, K}, es, copied) + copy_bytes(Matrix{w, ldw, N, K}, es, copied) +
         part_bytes(dtype, M, N, K);
}

int linear_fwd(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias,
               const void *residual, int64_t ldr, void *y, int64_t ldy, void *deriv, int64_t M, int64_t K, int64_t N,
               int act, void *workspace, hipStream_t s) {
  Epilogue epi{bias, residual, y, act == SFT_ACT_NONE ? nullptr : deriv, ldr, ldy, act, false, false};
  if (few_rows(M, K, type_size(dtype))) {
    Gemm g = {};
    g.a = x;
    g.b = w;
    g.lda = ldx;
    g.ldb = ldw;
    g.M = (int)M;
    g.N = (int)N;
    g.K = (int)K;
    g.epi = epi;
    g.epi.vec = epilogue_vec(epi, N, type_size(dtype), 4);
    ProfScope prof(kProfDenseProduct, s);
    return SFT_DENSE_CALL(dtype, launch_rows, g, s);
  }
  Scratch ws{static_cast<char *>(workspace)};
  Matrix a{x, ldx, M, K}, b{w, ldw, N, K};
  const int rc = align(dtype, &a, &b, ws, s);
  return rc ? rc : run_gemm(dtype, kForward, a, b, M, N, K, epi, nullptr, ws, s);
}

size_t linear_bwd_workspace(int dtype, const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w,
                            int64_t ldw, bool dx, bool dw, bool db, int64_t M, int64_t K, int64_t N, int act,
                            bool copied) {
  if (M == 0) return 0;
  const int64_t es = type_size(dtype);
  ActBwd p = {};
  shape_act_bwd(dtype, M, N, p);
  const Matrix g{dy, lddy, M, N};
  size_t n = act != SFT_ACT_NONE ? g.copy_bytes(es) : dx || dw ? copy_bytes(g, es, copied) : 0;
  const int sums = product_sums(dtype, dw, M, K, N, act);
  // the size for all grads covers calls for some: without dw the bias's partials are p.parts
  if (db) n += a256((size_t)(sums > p.parts ? sums : p.parts) * N * 4);
  if (dx) n += copy_bytes(Matrix{w, ldw, N, K}, es, copied);
  if (dw) n += copy_bytes(Matrix{x, ldx, M, K}, es, copied);
  const size_t in = dx ? part_bytes(dtype, M, K, N) : 0, weight = dw ? part_bytes(dtype, N, K, M) : 0;
  return n + (in > weight ? in : weight);
}

int linear_bwd(int dtype, const void *dy, int64_t lddy, const void *deriv, const void *x, int64_t ldx, const void *w,
               int64_t ldw, void *dx, void *dw, void *db, int64_t M, int64_t K, int64_t N, int act, void *workspace,
               hipStream_t s) {
  const int64_t es = type_size(dtype);
  if (M == 0) {  // no rows: the sums are empty
    if (dw) zero16(dw, K * N * es / 2, s);
    if (db) zero16(db, N * es / 2, s);
    return check_launch("sft_linear_bwd");
  }
  Scratch ws{static_cast<char *>(workspace)};
  Matrix dz{dy, lddy, M, N};
  ActBwd p = {};
  shape_act_bwd(dtype, M, N, p);
  p.dy = dy;
  p.lddy = lddy;
  if (act != SFT_ACT_NONE) {
    p.deriv = deriv;
    p.lddz = padded(N, es);
    p.dz = ws.take(dz.copy_bytes(es));
    dz = Matrix{p.dz, p.lddz, M, p.lddz};
  }
  const int sums = product_sums(dtype, dw, M, K, N, act), parts = sums ? sums : p.parts;
  if (db) p.part = static_cast<float *>(ws.take(a256((size_t)parts * N * 4)));
  int rc = SFT_OK;
  if (act != SFT_ACT_NONE || (db && !sums)) {
    ProfScope prof(kProfDenseActBwd, s);
    rc = SFT_DENSE_CALL(dtype, launch_act_bwd, p, s);
  }
  Matrix in{x, ldx, M, K}, weight{w, ldw, N, K};
  if (!rc && (dx || dw)) rc = align(dtype, &dz, nullptr, ws, s);
  if (!rc) rc = align(dtype, dx ? &weight : nullptr, dw ? &in : nullptr, ws, s);
  if (!rc && dx)
    rc = run_gemm(dtype, kInputGrad, dz, weight, M, K, N,
                  Epilogue{nullptr, nullptr, dx, nullptr, 0, K, SFT_ACT_NONE, false, false}, nullptr, ws, s);
  if (!rc && dw)
    rc = run_gemm(dtype, kWeightGrad, dz, in, N, K, M,
                  Epilogue{nullptr, nullptr, dw, nullptr, 0, K, SFT_ACT_NONE, false, false}, sums ? p.part : nullptr,
                  ws, s);
  if (!rc && db) {
    ProfScope prof(kProfDenseActBwd, s);
    rc = SFT_DENSE_CALL(dtype, launch_bias_join, p.part, parts, (int)N, db, s);
  }
  return rc;
}

}  // namespace sft
