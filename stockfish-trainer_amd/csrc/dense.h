// Host-side descriptions of the dense head's products, shared by the type-specific
// translation units and the dispatch.
#pragma once

#include "common.h"

namespace sft {
namespace dense {

enum Layout { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };
// Tiles of a product: 64 x 128, 128 x 128 and, of 16-bit types, 256 x 256.
enum TileKind { kTile64 = 0, kTile128 = 1, kTile256 = 2 };

constexpr int kWaveCols = 64;  // columns of a tile's waves

// What becomes of a product's sums: y = residual + act(sum + bias), rounded once.
struct Epilogue {
  const void *bias;      // [N] or null
  const void *residual;  // [M, N], rows ldr apart, or null
  void *y;               // [M, N], rows ldy apart
  void *deriv;           // dense [M, N] of act', or null
  int64_t ldr, ldy;
  int act;
  bool vec;     // bias, residual, y and deriv take 16-byte accesses (of few rows: of 4 elements)
  bool stream;  // y goes past the caches
};

// C[M, N] = sum over K of A(m, k) B(n, k).  Operands padded to whole chunks have ma >= M
// rows or nb >= N columns, and ka, kb <= K of the k's each; what lacks is zero.
struct Gemm {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N, K;
  int ma, nb, ka, kb;
  int tile, tiles_m, tiles_n;
  int splits, split_k;  // k per split, whole stages
  float *part;          // [splits][M][N] when splits > 1
  float *sums;          // [splits][M] sums of A over k, or null: of weight grads with a spare wave
  Epilogue epi;
};

struct ActBwd {
  const void *dy, *deriv;  // deriv null: dz is dy, only the sums are made
  void *dz;                // rows lddz apart, whole chunks
  float *part;             // [parts][N] or null
  int64_t lddy, lddz, M, rows;
  int N, parts, tx;
};

struct Copy {
  const void *from;
  void *to;
  int64_t ld, to_ld, rows, cols;  // elements
};

template <typename T>
int launch_gemm(const Gemm &g, int layout, hipStream_t s);
template <typename T>
int launch_rows(const Gemm &g, hipStream_t s);
template <typename T>
int launch_act_bwd(const ActBwd &p, hipStream_t s);
template <typename T>
int launch_bias_join(const float *part, int parts, int N, void *db, hipStream_t s);
template <typename T>
int launch_align(const Copy &a, const Copy &b, hipStream_t s);

}  // namespace dense
}  // namespace sft
