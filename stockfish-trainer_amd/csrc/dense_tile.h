// Matrix products of the dense head on the matrix cores:
//   C[m, n] = sum_k A(m, k) B(n, k),   then the epilogue  y = residual + act(C + bias).
// One template serves the three products of a linear layer y = act(x W^T + b) + r:
//   forward  C = x W^T     A = x  [M, K]   B = W  [N, K]    both with k contiguous
//   input    C = dz W      A = dz [M, N]   B(k', n) = W[n, k']: k (here n) is the row index of W
//   weight   C = dz^T x    A(n, m) = dz[m, n], B(k, m) = x[m, k]: the row index of both
// so an operand is either "k-major" (a row holds consecutive k) or "row-k" (a row
// holds one k of consecutive m or n).  Each type has its translation unit.
#pragma once

#include <type_traits>

#include "common.h"
#include "dense.h"

namespace sft {
namespace dense {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define SFT_LDS __attribute__((address_space(3)))

constexpr float kLog2E = 1.44269504088896341f;
constexpr int kStageBytes = 64;  // bytes of k per tile row and pipeline stage: one fragment's

// ---- activations ----
// z = act(z) and d = act'(z) of V values, in binary32.  The derivatives at the kinks
// are those of torch's clamp: 0 at relu's 0, 1 at both ends of the clipped ones.
template <int V>
__device__ __forceinline__ void activate(float (&z)[V], float (&d)[V], int act) {
  switch (act) {
    case SFT_ACT_RELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = z[i] > 0.f ? 1.f : 0.f;
        z[i] = z[i] < 0.f ? 0.f : z[i];
      }
      break;
    case SFT_ACT_CRELU:
    case SFT_ACT_SCRELU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float c = z[i] < 0.f ? 0.f : (z[i] > 1.f ? 1.f : z[i]);
        const float in = (z[i] >= 0.f && z[i] <= 1.f) ? 1.f : 0.f;
        d[i] = act == SFT_ACT_CRELU ? in : 2.f * c * in;
        z[i] = act == SFT_ACT_CRELU ? c : c * c;
      }
      break;
    // Base-2 exponentials and reciprocals of the hardware, each within a unit in the
    // last place or so.
    case SFT_ACT_SILU:
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2E * z[i]));
        d[i] = s * (1.f + z[i] * (1.f - s));
        z[i] *= s;
      }
      break;
    case SFT_ACT_GELU:
      // erfc by the rational approximation 7.1.26 of Abramowitz and Stegun, within
      // 1.5e-7; its exponential is the derivative's too.
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float a = fabsf(z[i]) * 0.70710678118654752f, e = __builtin_amdgcn_exp2f(-kLog2E * a * a);
        const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * a);
        const float tail =
            0.5f * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f)))) * e;
        const float cdf = z[i] < 0.f ? tail : 1.f - tail;
        d[i] = cdf + z[i] * (0.39894228040143268f * e);
        z[i] *= cdf;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = 1.f;
  }
}

// The derivative as the backward reads it: binary32 for a binary32 layer, otherwise
// a 16-bit fixed-point number with 14 fractional bits.  All derivatives lie in
// [-0.2, 2], so its error is 2^-15 (2^-14 at screlu's 2, which saturates) where a
// bfloat16 of the same size would be off by up to 2^-9 of the value.
template <typename T>
struct Deriv {
  typedef int16_t type;
  static __device__ __forceinline__ int16_t pack(float d) {
    return (int16_t)fminf(fmaxf(rintf(d * 16384.f), -32767.f), 32767.f);
  }
  static __device__ __forceinline__ float unpack(int16_t d) { return (float)d * (1.f / 16384.f); }
};
template <>
struct Deriv<float> {
  typedef float type;
  static __device__ __forceinline__ float pack(float d) { return d; }
  static __device__ __forceinline__ float unpack(float d) { return d; }
};

// V consecutive elements in one access, or the first `cnt` one by one.
template <typename T, int V>
__device__ __forceinline__ void load_v(const T *p, bool vec, int cnt, T (&v)[V]) {
  if (vec) {
    __builtin_memcpy(v, __builtin_assume_aligned(p, sizeof(T) * V), sizeof(T) * V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < cnt ? p[i] : (T)0;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, bool vec, int cnt, const T (&v)[V]) {
  if (vec) {
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T) * V), v, sizeof(T) * V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < cnt) p[i] = v[i];
  }
}

// The bias of V columns (0 without one).
template <typename T, int V>
__device__ __forceinline__ void load_bias(const Epilogue &e, int n, int N, bool vec, float (&b)[V]) {
  T v[V] = {};
  if (e.bias) load_v(static_cast<const T *>(e.bias) + n, vec, N - n, v);
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = (float)v[i];
}

// y[m, n..n+V-1] = residual + act(z + bias), rounded once; the derivative beside it.
// Called only with m < M and n < N.  STREAM: y past the caches, in whole 16 bytes.
template <typename T, bool STREAM, int V>
__device__ __forceinline__ void finish(const Epilogue &e, int64_t m, int n, int N, const float (&bias)[V], float (&z)[V],
                                       bool vec) {
  const int cnt = N - n;
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] += bias[i];
  if (e.act != SFT_ACT_NONE) {
    float d[V];
    activate(z, d, e.act);
    if (e.deriv) {
      typedef typename Deriv<T>::type D;
      D q[V];
#pragma unroll
      for (int i = 0; i < V; ++i) q[i] = Deriv<T>::pack(d[i]);
      store_v(static_cast<D *>(e.deriv) + m * N + n, vec, cnt, q);
    }
  }
  if (e.residual) {
    T r[V];
    load_v(static_cast<const T *>(e.residual) + m * e.ldr + n, vec, cnt, r);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] += (float)r[i];
  }
  T y[V];
#pragma unroll
  for (int i = 0; i < V; ++i) y[i] = (T)z[i];
  T *to = static_cast<T *>(e.y) + m * e.ldy + n;
  if constexpr (STREAM) {
    u32x4 q;
    __builtin_memcpy(&q, y, 16);
    __builtin_nontemporal_store(q, reinterpret_cast<u32x4 *>(to));
    return;
  }
  store_v(to, vec, cnt, y);
}

// ---- tiles in LDS ----
// A stage of an operand is kStageBytes of k for each of its BMN rows (m or n), held
// in 16-byte chunks.  k-major: [BMN][64 bytes]; row-k: [stage k][BMN].  Chunks are
// permuted within a row so that the reads below touch every LDS bank equally; the
// copies from global memory write LDS linearly (the hardware's rule for direct
// copies: lane l writes base + 16 l), so the permutation is applied to the global
// addresses instead.
template <typename T, int BMN, bool KMAJ>
struct TileMap {
  static constexpr int kEs = sizeof(T);
  static constexpr int kEpc = 16 / kEs;                       // elements per chunk
  static constexpr int kStageK = kStageBytes / kEs;           // k per stage
  static constexpr int kRowBytes = KMAJ ? kStageBytes : BMN * kEs;
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kBytes = BMN * kStageBytes;
  // The chunk of its row that the slot holds.
  static __device__ __forceinline__ int chunk_at(int row, int slot) {
    if (KMAJ) return slot ^ ((0 - (row >> 2)) & 3);
    if (kEs == 2) return slot ^ (((((row & 3) | ((row >> 1) & 4)) << 1)) & (kRowChunks - 1));
    return slot ^ ((((row >> 2) & 3) << 2) & (kRowChunks - 1));
  }
};

// Copies a stage's chunks straight to LDS with bounds-checked buffer loads (out of
// range reads give zeros).  Rows are 16-byte aligned and hold whole chunks.  What a
// stage adds to a wave's scalar work delays its products, so ranges are 32-bit (a
// tile's rows span less) and the end of k is cut once, by clip().
template <typename T, int BMN, bool KMAJ, int THREADS>
struct DirectLoader {
  typedef TileMap<T, BMN, KMAJ> Map;
  static constexpr int kLoads = Map::kBytes / 16 / THREADS;
  static_assert(Map::kBytes % (16 * THREADS) == 0, "whole copies");
  static constexpr uint32_t kOut = 0xffffff00u;  // beyond any range below
  const char *base;
  int64_t step;
  uint32_t range;  // k-major: bytes from base to the end of the tile's rows
  uint32_t pitch, width;  // row-k: bytes of a row's stride, and of its part in the tile
  uint32_t off[kLoads];
  int kleft;   // k of the operand from the next stage's first
  int kchunk;  // k-major: first k of this thread's chunk within a stage
  // mn0: first row of the tile; k0: first k; K: end of the operand's k.
  __device__ __forceinline__ void init(const void *p, int64_t ld, int mn0, int MN, int k0, int K) {
    const int tid = threadIdx.x;
    pitch = (uint32_t)(ld * Map::kEs);
    kleft = K - k0;
    if (KMAJ) {
      const int rows = MN - mn0 < BMN ? MN - mn0 : BMN;
      base = static_cast<const char *>(p) + ((int64_t)mn0 * ld + k0) * Map::kEs;
      range = rows > 0 && K > k0 ? (uint32_t)(rows - 1) * pitch + (uint32_t)(K - k0) * Map::kEs : 0u;
      step = kStageBytes;
    } else {
      base = static_cast<const char *>(p) + ((int64_t)k0 * ld + mn0) * Map::kEs;
      width = MN > mn0 ? (uint32_t)(MN - mn0) * Map::kEs : 0u;
      step = (int64_t)Map::kStageK * ld * Map::kEs;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int q = j * THREADS + tid;
      const int row = q / Map::kRowChunks, c = Map::chunk_at(row, q % Map::kRowChunks);
      off[j] = (uint32_t)row * pitch + (uint32_t)c * 16u;
      if (!KMAJ && mn0 + c * Map::kEpc >= MN) off[j] = kOut;
      if (KMAJ) kchunk = c * Map::kEpc;  // the same for every j: THREADS / 4 rows apart
    }
  }
  // Before a stage with fewer than kStageK k left: the chunks past them.
  __device__ __forceinline__ void clip() {
    if (!KMAJ || kleft >= Map::kStageK) return;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) off[j] = kchunk < kleft ? off[j] : kOut;
  }
  // lds: the wave's part of the stage.
  __device__ __forceinline__ void load(SFT_LDS char *lds) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass has no such builtins
    uint32_t n;
    if (KMAJ) {
      n = range;
      range = (uint32_t)uniform((int)(range > kStageBytes ? range - kStageBytes : 0u));
    } else {  // the last row's part ends the range
      const int rows = kleft < Map::kStageK ? kleft : Map::kStageK;
      n = rows > 0 ? (uint32_t)(rows - 1) * pitch + width : 0u;
    }
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, (int)n, 0x00020000);
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (SFT_LDS void *)(lds + j * THREADS * 16), 16, off[j], 0, 0, 0);
#endif
    base += step;
    kleft -= Map::kStageK;
  }
};

// A 16-byte chunk whose first `cnt` elements exist; zeros after them.  The hardware
// takes any element alignment.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T *p, int64_t cnt) {
  constexpr int V = 16 / (int)sizeof(T);
  u32x4 r = {0u, 0u, 0u, 0u};
  if (cnt >= V) {
    __builtin_memcpy(&r, p, 16);
  } else if (cnt > 0) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = i < cnt ? p[i] : (T)0;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

// ---- fragments: 16 rows (m or n) by 64 bytes of k, as the matrix instructions take them ----
template <typename T>
struct Frag;
template <>
struct Frag<bf16_t> {
  u32x4 v;
};
template <>
struct Frag<f16_t> {
  u32x4 v;
};
template <>
struct Frag<float> {
  u32x4 v;  // four k of one row
};
// One step of a fragment's k: all 64 bytes of 16-bit types, a quarter of binary32's.
template <typename T>
struct Mma;
template <>
struct Mma<bf16_t> {
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ f32x4 step(const Frag<bf16_t> &a, const Frag<bf16_t> &b, f32x4 c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v),
                                                   c, 0, 0, 0);
  }
};
template <>
struct Mma<f16_t> {
  static constexpr int kSteps = 1;
  static __device__ __forceinline__ f32x4 step(const Frag<f16_t> &a, const Frag<f16_t> &b, f32x4 c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c,
                                                  0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static constexpr int kSteps = 4;
  static __device__ __forceinline__ f32x4 step(const Frag<float> &a, const Frag<float> &b, f32x4 c, int s) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a.v)[s], __builtin_bit_cast(f32x4, b.v)[s],
                                                c, 0, 0, 0);
  }
};
// acc[i][j] += the product of fragment i of A and j < NJ of B.
template <typename T, int FM, int FN>
__device__ __forceinline__ void mma_all(const Frag<T> (&fa)[FM], const Frag<T> (&fb)[FN], f32x4 (&acc)[FM][FN]) {
#pragma unroll
  for (int s = 0; s < Mma<T>::kSteps; ++s)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::step(fb[j], fa[i], acc[i][j], s);
}

// binary32 products on the bfloat16 matrix instructions, whose rate is 16 times that of
// the binary32 ones: a number is the exact sum of three bfloat16 (8 bits of its 24
// each, cut off, not rounded), and of the nine partial products the six that reach
// 2^-24 of the whole are added, in binary32.  What is left out and the sums' own
// rounding are of the size of a binary32 product's rounding; a row with an infinity
// becomes NaN (inf - inf) where a binary32 product would keep the infinity.
// 65536 x 1040 x 128 forward 98 us, 178 TFLOP/s, where the binary32 instructions' products
// of 8192^3 come to 153.  Bound by the vector work of the splitting, about as long as the
// products beside it.
// One fragment of each part: 8 k of a lane, 4 from each of two stages.
struct Split {
  u32x4 part[3];
  // The 4 numbers of stage `half` of the pair.
  __device__ __forceinline__ void take(const u32x4 &raw, int half) {
#ifdef __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t a = raw[2 * p], b = raw[2 * p + 1];
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        part[t][2 * half + p] = __builtin_amdgcn_perm(b, a, 0x07060302);  // the upper halves of both
        if (t == 2) break;
        const float fa = __builtin_bit_cast(float, a) - __builtin_bit_cast(float, a & 0xffff0000u);
        const float fb = __builtin_bit_cast(float, b) - __builtin_bit_cast(float, b & 0xffff0000u);
        a = __builtin_bit_cast(uint32_t, fa);
        b = __builtin_bit_cast(uint32_t, fb);
      }
    }
#endif
  }
};
// acc[j] += a times b[j], the smallest partial products first.
template <int FN>
__device__ __forceinline__ void mma_split(const Split &a, const Split (&b)[FN], f32x4 (&acc)[FN]) {
  constexpr int kA[6] = {0, 2, 1, 0, 1, 0}, kB[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
  for (int t = 0; t < 6; ++t)
#pragma unroll
    for (int j = 0; j < FN; ++j)
      acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b[j].part[kB[t]]),
                                                       __builtin_bit_cast(bf16x8, a.part[kA[t]]), acc[j], 0, 0, 0);
}

// Reads the fragments of F consecutive 16-row groups of an LDS tile, from row mn0.
// Lane l holds row l % 16 and the 16 bytes number l / 16 of its 64 bytes of k.
template <typename T, int BMN, bool KMAJ, int F>
struct FragReader {
  typedef TileMap<T, BMN, KMAJ> Map;
  int at[KMAJ ? 1 : F];
  __device__ __forceinline__ void init(int mn0) {
    const int i = lane_id() % 16, g = lane_id() / 16;
    if (KMAJ) {
      const int row = mn0 + i;  // 16 f more rows leave the permutation as it is
      at[0] = row * kStageBytes + (Map::chunk_at(row, g) << 4);
    } else if (Map::kEs == 2) {
      // A transposing read gives lane i of 16 the element i of 4 rows: the lane reads
      // 4 elements of row i / 4 and gets one of each row.
      const int row = g * 8 + i / 4;
#pragma unroll
      for (int f = 0; f < F; ++f)
        at[f] = row * Map::kRowBytes + (Map::chunk_at(row, (mn0 / 16 + f) * 2) << 4) + (i % 4) * 8;
    } else {
      const int row = g * 4;
#pragma unroll
      for (int f = 0; f < F; ++f)
        at[f] = row * Map::kRowBytes + (Map::chunk_at(row, (mn0 / 16 + f) * 4 + i / 4) << 4) + (i % 4) * 4;
    }
  }
  __device__ __forceinline__ Frag<T> read(const SFT_LDS char *lds, int f) const {
    Frag<T> r;
    if constexpr (KMAJ) {
      r.v = *(const SFT_LDS u32x4 *)(lds + at[0] + f * 16 * kStageBytes);
    } else if constexpr (Map::kEs == 2) {
      const SFT_LDS char *p = lds + at[f];
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SFT_LDS i16x4 *)p));
      const u32x2 hi = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SFT_LDS i16x4 *)(p + 4 * Map::kRowBytes)));
      r.v = u32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
      const SFT_LDS char *p = lds + at[f];
#pragma unroll
      for (int s = 0; s < 4; ++s) r.v[s] = *(const SFT_LDS uint32_t *)(p + s * Map::kRowBytes);
    }
    return r;
  }
};

// ---- the tiled product ----
// Workgroup number -> tile.  Workgroup i runs on XCD i % 8, so each XCD gets a
// contiguous run of the order below and its L2 serves the tiles' shared operands:
// groups of kGroupM rows of tiles, column by column.
constexpr int kGroupM = 8;
__device__ __forceinline__ void tile_of(const Gemm &g, int &tm, int &tn, int &split) {
  const uint32_t n = gridDim.x, b = blockIdx.x;
  const uint32_t xcd = b % 8u, q = n / 8u, rem = n % 8u;
  uint32_t t = xcd * q + (xcd < rem ? xcd : rem) + b / 8u;
  const uint32_t tiles = (uint32_t)g.tiles_m * (uint32_t)g.tiles_n;
  split = (int)(t / tiles);
  t %= tiles;
  const uint32_t per = kGroupM * (uint32_t)g.tiles_n;
  const uint32_t group = t / per, in = t % per;
  const uint32_t rows = (uint32_t)g.tiles_m - group * kGroupM < kGroupM ? (uint32_t)g.tiles_m - group * kGroupM : kGroupM;
  tm = (int)(group * kGroupM + in % rows);
  tn = (int)(in / rows);
}

// What a workgroup of WM x WN waves does with its BM x BN sums.
template <typename T, int BM, int BN, int WM, int WN>
struct TileWork {
  static constexpr int kThreads = WM * WN * kWave;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int kStageK = kStageBytes / (int)sizeof(T);
  static constexpr int kStage = (BM + BN) * kStageBytes;
  int split, m0, n0, wm, wn, k0, kend;
  __device__ __forceinline__ explicit TileWork(const Gemm &g) {
    int tm, tn;
    tile_of(g, tm, tn, split);
    m0 = tm * BM;
    n0 = tn * BN;
    k0 = split * g.split_k;
    kend = g.K - k0 < g.split_k ? g.K : k0 + g.split_k;
    const int wave = uniform(threadIdx.x / kWave);
    wm = (wave / WN) * (BM / WM);
    wn = (wave % WN) * (BN / WN);
  }
  // The first operand's rows are the result's four registers: lane l holds m = l % 16
  // and n = 4 (l / 16) + 0..3 of each fragment.  A wave turns its sums in LDS, 32 rows
  // at a time, so that its lanes take whole vectors of a row (single elements where
  // rows are not made of them): memory sees full lines, and the epilogue's code is
  // there once per part.
  static constexpr int kWaveN = BN / WN, kPitch = kWaveN + 4;  // floats; 4 spread the rows over the banks
  static constexpr int kParts = FM / 2, kPartRows = 32;
  static constexpr int kTurnBytes = kPartRows * kPitch * 4 * WM * WN;
  template <int V, bool STREAM>
  __device__ __forceinline__ void finish_part(const Gemm &g, int m1, const float *turn) const {
    constexpr int kLanes = kWaveN / V, kRows = kWave / kLanes;
    const int lane = lane_id();
    const int c = lane % kLanes * V, n = n0 + wn + c;
    const int rows = n < g.N ? (g.M - m1 < kPartRows ? g.M - m1 : kPartRows) : 0;
    float bias[V] = {};
    if (rows > 0 && !g.part) load_bias<T>(g.epi, n, g.N, true, bias);
#pragma unroll 2
    for (int r = lane / kLanes; r < rows; r += kRows) {
      float z[V];
      __builtin_memcpy(z, __builtin_assume_aligned(turn + r * kPitch + c, 4 * (V < 4 ? V : 4)), 4 * V);
      if (g.part)
        store_v(g.part + ((int64_t)split * g.M + m1 + r) * g.N + n, true, V, z);
      else
        finish<T, STREAM>(g.epi, m1 + r, n, g.N, bias, z, true);
    }
  }
  __device__ __forceinline__ void finish_all(const Gemm &g, const f32x4 (&acc)[FM][FN], char *lds) const {
    constexpr int V = 16 / (int)sizeof(T);
    const int lane = lane_id();
    float *turn = reinterpret_cast<float *>(lds) + (threadIdx.x / kWave) * (kPartRows * kPitch);
    const bool wide = g.part ? g.N % V == 0 : g.epi.vec;
    __syncthreads();  // every wave has done with the stages
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          *reinterpret_cast<f32x4 *>(turn + (i * 16 + lane % 16) * kPitch + j * 16 + lane / 16 * 4) =
              acc[part * 2 + i][j];
      wave_lds_barrier();
      const int m1 = m0 + wm + part * kPartRows;
      if (!wide)
        finish_part<1, false>(g, m1, turn);
      else if (g.epi.stream && !g.part)
        finish_part<V, true>(g, m1, turn);
      else
        finish_part<V, false>(g, m1, turn);
      wave_lds_barrier();
    }
  }
};

// Three things overlap: the copies of later stages from memory to a ring in LDS, the
// reads of stage s + 1's fragments into registers, and the products of stage s.  The
// waves meet once in MEET stages: then the next MEET stages are in LDS, the slots of
// the past ones are free, and as many copies are made.  The copies carry their own
// bounds checks, so those past the end are made too (they give zeros) and every
// meeting waits for the same number of outstanding ones.
//
// Bound by feeding the matrix cores: with 256 x 256 tiles, which read least from LDS and
// memory a product, 8192^3 bf16 runs at 1.35 to 1.41 PFLOP/s; the cores are busy 65% of the
// cycles, LDS has no bank conflicts, and waves spend 30% of their time at the meetings.
// 65536 x 1040 x 4096, us: forward 573 (0.97 PFLOP/s; its 537 MB of results take 115 at a
// copy's rate), input grad 524, weight grad 520.  Smaller tiles have several workgroups a
// CU, one's copies and results under another's products: 16384 x 1040 x 1040 59, 51, 54.
template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, int RING, int MEET>
__global__ __launch_bounds__(WM *WN *kWave, BM / WM * BN / WN > 128 * 64 ? 1 : 2) void gemm_ring_kernel(const Gemm g) {
  typedef TileWork<T, BM, BN, WM, WN> Work;
  constexpr int FM = Work::FM, FN = Work::FN, kStage = Work::kStage;
  typedef DirectLoader<T, BM, AK, Work::kThreads> LoadA;
  typedef DirectLoader<T, BN, BK, Work::kThreads> LoadB;
  constexpr int kCopies = LoadA::kLoads + LoadB::kLoads;
  __shared__ __attribute__((aligned(1024))) char lds[RING * kStage > Work::kTurnBytes ? RING * kStage
                                                                                   : Work::kTurnBytes];
  const Work w(g);
  LoadA la;
  LoadB lb;
  la.init(g.a, g.lda, w.m0, g.ma, w.k0, w.kend < g.ka ? w.kend : g.ka);
  lb.init(g.b, g.ldb, w.n0, g.nb, w.k0, w.kend < g.kb ? w.kend : g.kb);
  FragReader<T, BM, AK, FM> ra;
  FragReader<T, BN, BK, FN> rb;
  ra.init(w.wm);
  rb.init(w.wn);
  f32x4 acc[FM][FN] = {};
  const int steps = (w.kend - w.k0 + Work::kStageK - 1) / Work::kStageK;
  SFT_LDS char *ring = (SFT_LDS char *)lds;
  SFT_LDS char *ring_to = ring + uniform(threadIdx.x / kWave) * (kWave * 16);  // the wave's part of a copy
  int at = 0;  // slot of the next copy
  auto clip = [&]() {
    la.clip();
    lb.clip();
  };
  auto copy = [&](SFT_LDS char *__restrict__ to) {
    la.load(to);
    lb.load(to + BM * kStageBytes);
  };
  auto read = [&](const SFT_LDS char *__restrict__ from, Frag<T>(&fa)[FM], Frag<T>(&fb)[FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = ra.read(from, i);
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = rb.read(from + BM * kStageBytes, j);
  };
  // The slots differ; without the restricts the compiler would wait for the copies
  // before it reads.
  auto copy_read = [&](SFT_LDS char *__restrict__ to, const SFT_LDS char *__restrict__ from, Frag<T>(&fa)[FM],
                       Frag<T>(&fb)[FN]) {
    la.load(to);
    lb.load(to + BM * kStageBytes);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = ra.read(from, i);
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = rb.read(from + BM * kStageBytes, j);
  };
  // All own copies but those of the last `left` stages are in LDS and own fragment
  // reads are done; then the same holds for every wave.
  auto meet = [&](auto left) {
    constexpr int n = decltype(left)::value * kCopies;
    static_assert(n < 64, "a 6-bit count");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4 << 14) | 0x70);  // vmcnt(n) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // The order of one stage: a product or two after each fragment read, then after each
  // copy, and the rest of the products, in whose time the last reads arrive.
  auto interleave = []() {
    constexpr int kReads = FM * (AK ? 1 : sizeof(T) == 2 ? 2 : 4) + FN * (BK ? 1 : sizeof(T) == 2 ? 2 : 4);
    constexpr int kProducts = FM * FN * Mma<T>::kSteps;
    constexpr int kPer = 2 * kReads > kProducts ? 2 : 1;  // reads a product
#pragma unroll
    for (int i = 0; i < kReads / kPer; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);  // LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // matrix instruction
    }
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // memory read
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
  };
  auto next = [](int slot) { return slot == RING - 1 ? 0 : slot + 1; };
  for (int s = 0; s <= RING - MEET; ++s, at = next(at)) {
    clip();
    copy(ring_to + s * kStage);
  }
  static_assert(BN / WN == kWaveCols, "the rule for spare waves");
  Frag<T> fa[2][FM], fb[2][FN];
  meet(std::integral_constant<int, RING - MEET>{});  // stage 0
  read(ring, fa[0], fb[0]);
  int slot = 1 % RING;  // of the next stage to read
  typedef std::integral_constant<int, RING - 2 * MEET> Under;
  constexpr bool kPairs = sizeof(T) == 4;  // stages in pairs; one past the end holds zeros
  Split sa[kPairs ? FM : 1], sb[kPairs ? FN : 1];
  if (w.m0 + w.wm < g.M && w.n0 + w.wn < g.N) {
    for (int s = 0; s < steps; s += 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (kPairs || s + h < steps) {
          clip();
          if (h % MEET == 0) meet(Under{});
          copy_read(ring_to + at * kStage, ring + slot * kStage, fa[1 - h], fb[1 - h]);
          if constexpr (kPairs) {
#pragma unroll
            for (int j = 0; j < FN; ++j) sb[j].take(fb[h][j].v, h);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
              sa[i].take(fa[h][i].v, h);
              if (h == 1) mma_split(sa[i], sb, acc[i]);
            }
            if (h == 1) {  // the splitting of one fragment beside the products of the one before
#pragma unroll
              for (int i = 0; i < FM * FN * 6; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instruction
                __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);  // vector arithmetic
              }
            }
          } else {
            mma_all<T>(fa[h], fb[h], acc);
            interleave();
          }
          at = next(at);
          slot = next(slot);
        }
      }
    }
  } else if (!AK && !kPairs && g.sums && w.m0 + w.wm < g.M && w.n0 + w.wn - g.N < kWaveCols) {
    // The first wave past the last column: the sums of A over k, as products with ones.
    Frag<T> ones;
    ones.v = u32x4{1u, 1u, 1u, 1u} * (std::is_same<T, bf16_t>::value ? 0x3f803f80u : 0x3c003c00u);
    auto copy_read_a = [&](SFT_LDS char *__restrict__ to, const SFT_LDS char *__restrict__ from, Frag<T>(&f)[FM]) {
      la.load(to);
      lb.load(to + BM * kStageBytes);
#pragma unroll
      for (int i = 0; i < FM; ++i) f[i] = ra.read(from, i);
    };
    for (int s = 0; s < steps; s += 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (s + h < steps) {
          clip();
          if (h % MEET == 0) meet(Under{});
          copy_read_a(ring_to + at * kStage, ring + slot * kStage, fa[1 - h]);
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[i][0] = Mma<T>::step(ones, fa[h][i], acc[i][0], 0);
          at = next(at);
          slot = next(slot);
        }
      }
    }
    if (lane_id() < 16) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = w.m0 + w.wm + i * 16 + lane_id();
        if (m < g.M) g.sums[(int64_t)w.split * g.M + m] = acc[i][0].x;
      }
    }
  } else {  // a wave past the edge: its share of the copies only
    for (int s = 0; s < steps + (kPairs ? steps % 2 : 0); ++s, at = next(at)) {
      clip();
      if (s % MEET == 0) meet(Under{});
      copy(ring_to + at * kStage);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the stages
  w.finish_all(g, acc, lds);
}

// Sums a split product's partials in split order and finishes them; V elements a thread,
// with the loads of 8 splits under way.  Bound by those, from the memory-side cache: 6.5 us
// for the weight grad of 16384 x 1040 x 1040.
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void gemm_join_kernel(const Gemm g) {
  const int64_t vecs = g.N / V;  // N is a multiple of V
  const int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (q >= vecs * g.M) return;
  const int64_t m = q / vecs;
  const int n = (int)(q % vecs) * V;
  float z[V] = {};
  const float *p = g.part + m * g.N + n;
#pragma unroll 8
  for (int s = 0; s < g.splits; ++s, p += (int64_t)g.M * g.N) {
    float v[V];
    load_v(p, true, V, v);
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] += v[i];
  }
  float bias[V];
  load_bias<T>(g.epi, n, g.N, true, bias);
  finish<T, false>(g.epi, m, n, g.N, bias, z, true);
}

// ---- few rows ----
// y for up to 16 FM rows: a workgroup holds 16 outputs of every row; its waves take
// 256-byte pieces of k in turn, straight from global memory (W is read once and
// there is no reuse for LDS to serve), and are summed in wave order.  Bound by the latency
// of W's one read, then by its rate: a row x 1040 x 4096 bf16 2.9 us (2.9 TB/s), 64 rows 5.3.
constexpr int kRowWaves = 8;
template <typename T, int FM>
__global__ __launch_bounds__(kRowWaves *kWave) void gemm_rows_kernel(const Gemm g) {
  constexpr int kEpc = 16 / (int)sizeof(T);
  __shared__ f32x4 red[kRowWaves][FM][kWave];
  const int lane = lane_id(), i = lane % 16, c = lane / 16;
  const int wave = uniform(threadIdx.x / kWave);
  const int n0 = blockIdx.x * 16;
  // rows and columns past the last: its own again, not stored
  const T *w = static_cast<const T *>(g.b) + (int64_t)(n0 + i < g.N ? n0 + i : g.N - 1) * g.ldb;
  const T *x[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) x[f] = static_cast<const T *>(g.a) + (int64_t)(f * 16 + i < g.M ? f * 16 + i : g.M - 1) * g.lda;
  f32x4 acc[FM] = {};
  auto products = [&](const Frag<T> &fw, const Frag<T>(&fx)[FM]) {
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
      for (int t = 0; t < Mma<T>::kSteps; ++t) acc[f] = Mma<T>::step(fw, fx[f], acc[f], t);
  };
  // Whole chunks: loads without branches, so that a piece's are under way together;
  // what lies past them is read as the last one and not used.
  const int whole = g.K / kEpc;
  for (int q0 = wave * 16; q0 < whole; q0 += kRowWaves * 16) {
    Frag<T> fw[4], fx[4][FM];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int q = q0 + u * 4 + c, at = (q < whole ? q : whole - 1) * kEpc;
      __builtin_memcpy(&fw[u].v, w + at, 16);
#pragma unroll
      for (int f = 0; f < FM; ++f) __builtin_memcpy(&fx[u][f].v, x[f] + at, 16);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (q0 + u * 4 + c >= whole) {
        fw[u].v = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int f = 0; f < FM; ++f) fx[u][f].v = u32x4{0u, 0u, 0u, 0u};
      }
      products(fw[u], fx[u]);
    }
  }
  if (wave == kRowWaves - 1 && g.K % kEpc) {  // the last elements
    Frag<T> fw, fx[FM];
    const int at = whole * kEpc, cnt = c == 0 ? g.K - at : 0;
    fw.v = load_chunk(w + at, cnt);
#pragma unroll
    for (int f = 0; f < FM; ++f) fx[f].v = load_chunk(x[f] + at, cnt);
    products(fw, fx);
  }
#pragma unroll
  for (int f = 0; f < FM; ++f) red[wave][f][lane] = acc[f];
  __syncthreads();
  const int f = threadIdx.x / kWave;  // one wave finishes one group of rows
  if (f >= FM) return;
  f32x4 sum = red[0][f][lane];
#pragma unroll
  for (int s = 1; s < kRowWaves; ++s) sum += red[s][f][lane];
  const int m = f * 16 + i, n = n0 + c * 4;
  float z[4] = {sum.x, sum.y, sum.z, sum.w};
  if (m >= g.M || n >= g.N) return;
  float bias[4];
  load_bias<T>(g.epi, n, g.N, g.epi.vec, bias);
  finish<T, false>(g.epi, m, n, g.N, bias, z, g.epi.vec);
}

// ---- gradient of the activation, and the bias grad's partial sums ----
// dz = dy * act'(z), rounded to the layer's type for the products that follow (its
// rows are padded with zeros to whole chunks), and the sums of the unrounded dz over
// `rows` rows per workgroup and column.  A thread holds a chunk of V columns; a
// workgroup is tx chunks by 256 / tx rows.  Reading and writing bound it: 16384 x 1040 bf16
// 20 us, 5.1 TB/s, the sums alone at 65536 x 4096 4.8 TB/s.
template <typename T>
__global__ __launch_bounds__(kBlock) void act_bwd_kernel(const ActBwd p) {
  typedef typename Deriv<T>::type D;
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float red[kBlock * V];
  const int tx = p.tx, ty = kBlock / tx;
  const int cx = threadIdx.x % tx, ry = threadIdx.x / tx;
  const int n = (blockIdx.x * tx + cx) * V, cnt = p.N - n;
  const int64_t first = (int64_t)blockIdx.y * p.rows;
  const int64_t last = first + p.rows < p.M ? first + p.rows : p.M;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  if (cnt > 0) {
    for (int64_t m = first + ry; m < last; m += ty) {
      T dy[V];
      *reinterpret_cast<u32x4 *>(dy) = load_chunk(static_cast<const T *>(p.dy) + m * p.lddy + n, cnt);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (float)dy[i];
      if (p.deriv) {
        D d[V];
        *reinterpret_cast<u32x4 *>(d) = load_chunk(static_cast<const D *>(p.deriv) + m * p.N + n, cnt);
        T dz[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] = i < cnt ? v[i] * Deriv<T>::unpack(d[i]) : 0.f;
          dz[i] = (T)v[i];
        }
        *reinterpret_cast<u32x4 *>(static_cast<T *>(p.dz) + m * p.lddz + n) = *reinterpret_cast<u32x4 *>(dz);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += v[i];
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < V; ++i) red[i * kBlock + threadIdx.x] = sum[i];
  __syncthreads();
  if (ry != 0 || cnt <= 0) return;
  for (int r = 1; r < ty; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += red[i * kBlock + r * tx + cx];
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < cnt) p.part[(int64_t)blockIdx.y * p.N + n + i] = sum[i];
}

// db[n] = the sum of column n's partials: 64 threads take every 64th each, and are
// added in order.  4 us, mostly the launch and one round of loads.
constexpr int kJoinCols = 16, kJoinRows = 64;
template <typename T>
__global__ __launch_bounds__(kJoinCols *kJoinRows) void bias_join_kernel(const float *__restrict__ part, int parts,
                                                                         int N, void *db) {
  __shared__ float red[kJoinRows][kJoinCols];
  const int c = threadIdx.x % kJoinCols, r = threadIdx.x / kJoinCols;
  const int n = blockIdx.x * kJoinCols + c;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int i = r; i < parts; i += kJoinRows) s += part[(int64_t)i * N + n];
  }
  red[r][c] = s;
  __syncthreads();
  if (r != 0 || n >= N) return;
  for (int i = 1; i < kJoinRows; ++i) s += red[i][c];
  static_cast<T *>(db)[n] = (T)s;
}

// ---- copies of operands with whole, aligned rows ----
// Up to two matrices of rows x cols elements, to rows of a whole number of chunks with
// zeros past cols.  One chunk a thread: 5003 x 1037 f16 5.6 us, 3.7 TB/s.  (Operands read in
// place by guarded loads through registers, in the product itself, were slower: every
// tile pays for them again.)
template <typename T>
__global__ __launch_bounds__(kBlock) void align_rows_kernel(const Copy a, const Copy b, int64_t blocks_a) {
  const bool second = (int64_t)blockIdx.x >= blocks_a;
  const Copy c = second ? b : a;
  const int64_t q = ((int64_t)blockIdx.x - (second ? blocks_a : 0)) * kBlock + threadIdx.x;
  const int64_t chunks = c.to_ld / (16 / (int)sizeof(T)), row = q / chunks, at = q % chunks * (16 / (int)sizeof(T));
  if (row >= c.rows) return;
  *reinterpret_cast<u32x4 *>(static_cast<T *>(c.to) + row * c.to_ld + at) =
      load_chunk(static_cast<const T *>(c.from) + row * c.ld + at, c.cols - at);
}

// ---- launchers, instantiated per type ----
template <typename T, bool AK, bool BK>
int launch_gemm_as(const Gemm &g, hipStream_t s) {
  const int64_t grid = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  // Rings as deep as keep three workgroups of the smaller tiles on a CU (48 KB each) and one
  // of the largest (128 of 160 KB; 5 slots: the same 1.24 PFLOP/s of 8192^3 at that time; a
  // meeting in two stages 1.16).
#define SFT_RING(BM, BN, WM, WN, RING, MEET)                                                                  \
  hipLaunchKernelGGL((gemm_ring_kernel<T, AK, BK, BM, BN, WM, WN, RING, MEET>), dim3((unsigned)grid),         \
                     dim3(WM *WN *kWave), 0, s, g)
  if (g.tile == kTile64) {
    SFT_RING(64, 128, 2, 2, 4, 1);
  } else if (g.tile == kTile128) {
    SFT_RING(128, 128, 2, 2, 3, 1);
  } else {
    if constexpr (sizeof(T) == 2) SFT_RING(256, 256, 2, 4, 4, 1);
  }
#undef SFT_RING
  if (g.splits > 1) {
    constexpr int V = 16 / (int)sizeof(T);
    const dim3 block(kBlock);
    const int64_t n = (int64_t)g.N * g.M;
    if (g.epi.vec)
      hipLaunchKernelGGL((gemm_join_kernel<T, V>), dim3((unsigned)ceil_div(n / V, kBlock)), block, 0, s, g);
    else
      hipLaunchKernelGGL((gemm_join_kernel<T, 1>), dim3((unsigned)ceil_div(n, kBlock)), block, 0, s, g);
  }
  return check_launch("dense product");
}

template <typename T>
int launch_gemm(const Gemm &g, int layout, hipStream_t s) {
  if (layout == kForward) return launch_gemm_as<T, true, true>(g, s);
  if (layout == kInputGrad) return launch_gemm_as<T, true, false>(g, s);
  return launch_gemm_as<T, false, false>(g, s);
}

template <typename T>
int launch_rows(const Gemm &g, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(g.N, 16)), block(kRowWaves * kWave);
  if (g.M <= 16)
    hipLaunchKernelGGL((gemm_rows_kernel<T, 1>), grid, block, 0, s, g);
  else if (g.M <= 32)
    hipLaunchKernelGGL((gemm_rows_kernel<T, 2>), grid, block, 0, s, g);
  else
    hipLaunchKernelGGL((gemm_rows_kernel<T, 4>), grid, block, 0, s, g);
  return check_launch("dense product of few rows");
}

template <typename T>
int launch_act_bwd(const ActBwd &p, hipStream_t s) {
  const int64_t chunks = ceil_div(p.N, 16 / (int64_t)sizeof(T));
  hipLaunchKernelGGL((act_bwd_kernel<T>), dim3((unsigned)ceil_div(chunks, p.tx), (unsigned)p.parts), dim3(kBlock), 0, s,
                     p);
  return check_launch("dense activation backward");
}

template <typename T>
int launch_bias_join(const float *part, int parts, int N, void *db, hipStream_t s) {
  hipLaunchKernelGGL((bias_join_kernel<T>), dim3((unsigned)ceil_div(N, kJoinCols)), dim3(kJoinCols * kJoinRows), 0, s,
                     part, parts, N, db);
  return check_launch("dense bias grad");
}

template <typename T>
int launch_align(const Copy &a, const Copy &b, hipStream_t s) {
  const int64_t epc = 16 / (int64_t)sizeof(T);
  const int64_t na = ceil_div(a.rows * (a.to_ld / epc), kBlock), nb = ceil_div(b.rows * (b.to_ld / epc), kBlock);
  hipLaunchKernelGGL((align_rows_kernel<T>), dim3((unsigned)(na + nb)), dim3(kBlock), 0, s, a, b, na);
  return check_launch("dense aligned copy");
}

#define SFT_DENSE_TYPE(T)                                                \
  template int launch_gemm<T>(const Gemm &, int, hipStream_t);           \
  template int launch_rows<T>(const Gemm &, hipStream_t);                \
  template int launch_act_bwd<T>(const ActBwd &, hipStream_t);           \
  template int launch_bias_join<T>(const float *, int, int, void *, hipStream_t); \
  template int launch_align<T>(const Copy &, const Copy &, hipStream_t);

}  // namespace dense
}  // namespace sft
