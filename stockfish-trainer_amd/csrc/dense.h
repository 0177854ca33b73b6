// Host-side descriptions of the dense head's products, shared by the type-specific
// translation units and the dispatch.
#pragma once

#include "common.h"

namespace sft {
namespace dense {

enum Layout { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };

// What becomes of a product's sums: y = residual + act(sum + bias), rounded once.
struct Epilogue {
  const void *bias;      // [N] or null
  const void *residual;  // [M, N], rows ldr apart, or null
  void *y;               // [M, N], rows ldy apart
  void *deriv;           // dense [M, N] of act', or null
  int64_t ldr, ldy;
  int act;
  bool vec;  // rows of bias, residual, y and deriv take 4-element accesses
};

// C[M, N] = sum over K of A(m, k) B(n, k).
struct Gemm {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N, K;
  int tiles_m, tiles_n;
  int splits, split_k;  // k per split, whole stages
  float *part;          // [splits][M][N] when splits > 1
  bool direct;          // both operands take aligned 16-byte copies
  Epilogue epi;
};

struct ActBwd {
  const void *dy, *deriv;  // deriv null: dz is dy, only the sums are made
  void *dz;
  float *part;  // [parts][N] or null
  int64_t lddy, M, rows;
  int N, parts, tx;
  bool vec;
};

template <typename T>
int launch_gemm(const Gemm &g, int layout, hipStream_t s);
template <typename T>
int launch_rows(const Gemm &g, hipStream_t s);
template <typename T>
int launch_act_bwd(const ActBwd &p, void *db, hipStream_t s);

}  // namespace dense
}  // namespace sft
