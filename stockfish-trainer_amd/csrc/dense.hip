// Dispatch of the dense head's linear layers: which kernel takes a product, how it
// is split, and where its intermediates live in the caller's workspace.
#include "dense.h"

namespace sft {
namespace dense {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

namespace {

constexpr int kStage = 128;          // bytes of k per pipeline stage
constexpr int kTile = 128;           // rows and columns of a tile
constexpr int64_t kRowsMost = 64;    // rows the row kernel takes
constexpr int64_t kSlots = 2 * 256;  // tile workgroups the card holds at once

size_t a256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t type_size(int dtype) { return dtype == SFT_TYPE_F32 ? 4 : 2; }

// A product with few tiles and a long k is split along k, so that the card is full,
// as long as every part has at least 8 stages.
int splits_of(int dtype, int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ceil_div(M, kTile) * ceil_div(N, kTile);
  const int64_t stages = ceil_div(K * type_size(dtype), kStage);
  int64_t s = kSlots / tiles;
  if (s > stages / 8) s = stages / 8;
  if (s < 1) return 1;
  const int64_t per = ceil_div(stages, s);
  return (int)ceil_div(stages, per);
}

size_t part_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  const int s = splits_of(dtype, M, N, K);
  return s > 1 ? a256((size_t)s * M * N * 4) : 0;
}

bool rows16(const void *p, int64_t ld, int64_t es) { return ((uintptr_t)p | (uintptr_t)(ld * es)) % 16 == 0; }
bool rows4(const void *p, int64_t ld, int64_t es) { return !p || ((uintptr_t)p | (uintptr_t)(ld * es)) % (4 * es) == 0; }

int run_gemm(int dtype, Gemm &g, int layout, hipStream_t s) {
  const int64_t es = type_size(dtype), epc = 16 / es;
  const bool ak = layout != kWeightGrad, bk = layout == kForward;
  // A direct copy moves whole aligned chunks, with 32-bit offsets inside a tile.
  g.direct = rows16(g.a, g.lda, es) && rows16(g.b, g.ldb, es) && (ak ? g.K : g.M) % epc == 0 &&
             (bk ? g.K : g.N) % epc == 0 && g.lda * es < (1 << 22) && g.ldb * es < (1 << 22);
  g.epi.vec = g.N % 4 == 0 && rows4(g.epi.y, g.epi.ldy, es) && rows4(g.epi.bias, 0, es) &&
              rows4(g.epi.residual, g.epi.ldr, es) && rows4(g.epi.deriv, 0, es);
  g.tiles_m = (int)ceil_div(g.M, kTile);
  g.tiles_n = (int)ceil_div(g.N, kTile);
  g.splits = splits_of(dtype, g.M, g.N, g.K);
  const int64_t stages = ceil_div(g.K * es, kStage);
  g.split_k = (int)(ceil_div(stages, g.splits) * (kStage / es));
  if (g.splits == 1) g.part = nullptr;
  ProfScope prof(kProfDenseProduct, s);
  if (dtype == SFT_TYPE_F32) return launch_gemm<float>(g, layout, s);
  if (dtype == SFT_TYPE_F16) return launch_gemm<f16_t>(g, layout, s);
  return launch_gemm<bf16_t>(g, layout, s);
}

__global__ __launch_bounds__(kBlock) void zero16_kernel(uint16_t *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) p[i] = 0;
}
void zero16(void *p, int64_t n, hipStream_t s) {
  const int64_t blocks = ceil_div(n, kBlock);
  hipLaunchKernelGGL(zero16_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kBlock), 0, s,
                     static_cast<uint16_t *>(p), n);
}

// The shape of the activation's backward and bias sums: about 1024 workgroups.
void shape_act_bwd(int dtype, int64_t M, int64_t N, ActBwd &p) {
  const int64_t V = 16 / type_size(dtype);
  p.M = M;
  p.N = (int)N;
  p.vec = N % V == 0;
  const int64_t cols = p.vec ? N / V : N;
  p.tx = 1;
  while (p.tx < kWave && p.tx < cols) p.tx *= 2;
  const int64_t ty = kBlock / p.tx, want = ceil_div(1024, ceil_div(cols, p.tx));
  p.rows = ceil_div(ceil_div(M, want), ty) * ty;
  p.parts = (int)ceil_div(M, p.rows);
}

}  // namespace

}  // namespace dense

using namespace dense;

size_t linear_fwd_workspace(int dtype, int64_t M, int64_t K, int64_t N) {
  return M <= kRowsMost ? 0 : part_bytes(dtype, M, N, K);
}

int linear_fwd(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias,
               const void *residual, int64_t ldr, void *y, int64_t ldy, void *deriv, int64_t M, int64_t K, int64_t N,
               int act, void *ws, hipStream_t s) {
  Gemm g = {};
  g.a = x;
  g.b = w;
  g.lda = ldx;
  g.ldb = ldw;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.part = static_cast<float *>(ws);
  g.epi = Epilogue{bias, residual, y, act == SFT_ACT_NONE ? nullptr : deriv, ldr, ldy, act, false};
  if (M <= kRowsMost) {
    const int64_t es = type_size(dtype);
    g.epi.vec = N % 4 == 0 && rows4(y, ldy, es) && rows4(bias, 0, es) && rows4(residual, ldr, es) &&
                rows4(g.epi.deriv, 0, es);
    ProfScope prof(kProfDenseProduct, s);
    if (dtype == SFT_TYPE_F32) return launch_rows<float>(g, s);
    if (dtype == SFT_TYPE_F16) return launch_rows<f16_t>(g, s);
    return launch_rows<bf16_t>(g, s);
  }
  return run_gemm(dtype, g, kForward, s);
}

size_t linear_bwd_workspace(int dtype, int64_t M, int64_t K, int64_t N, int act) {
  if (M == 0) return 0;
  ActBwd p = {};
  shape_act_bwd(dtype, M, N, p);
  const size_t dz = act == SFT_ACT_NONE ? 0 : a256((size_t)M * N * type_size(dtype));
  const size_t bias = a256((size_t)p.parts * N * 4);
  const size_t in = part_bytes(dtype, M, K, N), weight = part_bytes(dtype, N, K, M);
  return dz + bias + (in > weight ? in : weight);
}

int linear_bwd(int dtype, const void *dy, int64_t lddy, const void *deriv, const void *x, int64_t ldx, const void *w,
               int64_t ldw, void *dx, void *dw, void *db, int64_t M, int64_t K, int64_t N, int act, void *ws,
               hipStream_t s) {
  const int64_t es = type_size(dtype);
  if (M == 0) {  // no rows: the sums are empty
    if (dw) zero16(dw, K * N * es / 2, s);
    if (db) zero16(db, N * es / 2, s);
    return check_launch("sft_linear_bwd");
  }
  char *at = static_cast<char *>(ws);
  ActBwd p = {};
  shape_act_bwd(dtype, M, N, p);
  p.dy = dy;
  p.lddy = lddy;
  const void *dz = dy;
  int64_t lddz = lddy;
  if (act != SFT_ACT_NONE) {
    p.deriv = deriv;
    p.dz = at;
    dz = at;
    lddz = N;
    at += a256((size_t)M * N * es);
  }
  if (db) p.part = reinterpret_cast<float *>(at);
  at += a256((size_t)p.parts * N * 4);
  int rc = SFT_OK;
  if (db || act != SFT_ACT_NONE) {
    ProfScope prof(kProfDenseActBwd, s);
    rc = dtype == SFT_TYPE_F32   ? launch_act_bwd<float>(p, db, s)
         : dtype == SFT_TYPE_F16 ? launch_act_bwd<f16_t>(p, db, s)
                                 : launch_act_bwd<bf16_t>(p, db, s);
    if (rc) return rc;
  }
  Gemm g = {};
  g.epi.act = SFT_ACT_NONE;
  g.part = reinterpret_cast<float *>(at);
  if (dx) {
    Gemm in = g;
    in.a = dz;
    in.lda = lddz;
    in.b = w;
    in.ldb = ldw;
    in.M = (int)M;
    in.N = (int)K;
    in.K = (int)N;
    in.epi.y = dx;
    in.epi.ldy = K;
    rc = run_gemm(dtype, in, kInputGrad, s);
    if (rc) return rc;
  }
  if (dw) {
    Gemm wt = g;
    wt.a = dz;
    wt.lda = lddz;
    wt.b = x;
    wt.ldb = ldx;
    wt.M = (int)N;
    wt.N = (int)K;
    wt.K = (int)M;
    wt.epi.y = dw;
    wt.epi.ldy = K;
    rc = run_gemm(dtype, wt, kWeightGrad, s);
  }
  return rc;
}

}  // namespace sft
