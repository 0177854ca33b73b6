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

constexpr int kStageBytes = 128;  // bytes of k per tile row and pipeline stage

// ---- activations ----
// act(z) and its derivative, in binary32.  The derivatives at the kinks are those
// of torch's clamp: 0 at relu's 0, 1 at both ends of the clipped ones.
__device__ __forceinline__ float act_value(float z, int act, float &d) {
  switch (act) {
    case SFT_ACT_RELU:
      d = z > 0.f ? 1.f : 0.f;
      return z < 0.f ? 0.f : z;
    case SFT_ACT_CRELU:
      d = (z >= 0.f && z <= 1.f) ? 1.f : 0.f;
      return z < 0.f ? 0.f : (z > 1.f ? 1.f : z);
    case SFT_ACT_SCRELU: {
      const float c = z < 0.f ? 0.f : (z > 1.f ? 1.f : z);
      d = (z >= 0.f && z <= 1.f) ? 2.f * c : 0.f;
      return c * c;
    }
    case SFT_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      d = s * (1.f + z * (1.f - s));
      return z * s;
    }
    case SFT_ACT_GELU: {
      const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      d = cdf + z * (0.39894228040143268f * expf(-0.5f * z * z));
      return z * cdf;
    }
    default:
      d = 1.f;
      return z;
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

// 4 consecutive elements (guarded: the first `cnt` of them).
template <typename T>
struct Quad {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void load4(const T *p, bool vec, int cnt, T (&v)[4]) {
  if (vec) {
    const Quad<T> q = *reinterpret_cast<const Quad<T> *>(__builtin_assume_aligned(p, sizeof(T) * 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < cnt ? p[i] : (T)0;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, bool vec, int cnt, const T (&v)[4]) {
  if (vec) {
    Quad<T> q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = v[i];
    *reinterpret_cast<Quad<T> *>(__builtin_assume_aligned(p, sizeof(T) * 4)) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < cnt) p[i] = v[i];
  }
}

// y[m, n..n+3] = residual + act(acc + bias), rounded once; the derivative beside it.
// Called only with m < M and n < N.
template <typename T>
__device__ __forceinline__ void finish4(const Epilogue &e, int64_t m, int n, int N, f32x4 acc) {
  const int cnt = N - n;
  float z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = acc[i];
  if (e.bias) {
    T b[4];
    load4(static_cast<const T *>(e.bias) + n, e.vec, cnt, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] += (float)b[i];
  }
  if (e.act != SFT_ACT_NONE) {
    float d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = act_value(z[i], e.act, d[i]);
    if (e.deriv) {
      typedef typename Deriv<T>::type D;
      D q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = Deriv<T>::pack(d[i]);
      store4(static_cast<D *>(e.deriv) + m * N + n, e.vec, cnt, q);
    }
  }
  if (e.residual) {
    T r[4];
    load4(static_cast<const T *>(e.residual) + m * e.ldr + n, e.vec, cnt, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] += (float)r[i];
  }
  T y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (T)z[i];
  store4(static_cast<T *>(e.y) + m * e.ldy + n, e.vec, cnt, y);
}

// ---- tiles in LDS ----
// A stage of an operand is kStageBytes of k for each of its BMN rows (m or n), held
// in 16-byte chunks.  k-major: [BMN][128 bytes]; row-k: [stage k][BMN].  Chunks are
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
    if (KMAJ) return slot ^ ((row >> 1) & 7);
    if (kEs == 2) return slot ^ (((((row & 3) | ((row >> 1) & 4)) << 1)) & (kRowChunks - 1));
    return slot ^ ((((row >> 2) & 3) << 2) & (kRowChunks - 1));
  }
};

// Copies a stage's chunks straight to LDS with bounds-checked buffer loads (out of
// range reads give zeros).  Needs 16-byte aligned rows and whole chunks.
template <typename T, int BMN, bool KMAJ, int THREADS>
struct DirectLoader {
  typedef TileMap<T, BMN, KMAJ> Map;
  static constexpr int kLoads = Map::kBytes / 16 / THREADS;
  static_assert(Map::kBytes % (16 * THREADS) == 0, "whole copies");
  static constexpr uint32_t kOut = 0x80000000u;  // beyond any range below
  const char *base;
  int64_t left;  // bytes from base to the end of the operand
  int64_t step;
  uint32_t off[kLoads];
  int kchunk;  // k-major: first k of this thread's chunk within a stage
  // mn0: first row of the tile; k0: first k; K: end of the k range.
  __device__ __forceinline__ void init(const void *p, int64_t ld, int mn0, int MN, int k0, int K) {
    const int tid = threadIdx.x;
    if (KMAJ) {
      base = static_cast<const char *>(p) + ((int64_t)mn0 * ld + k0) * Map::kEs;
      left = ((int64_t)(MN - 1 - mn0) * ld + K - k0) * Map::kEs;
      step = kStageBytes;
    } else {
      base = static_cast<const char *>(p) + ((int64_t)k0 * ld + mn0) * Map::kEs;
      left = ((int64_t)(K - 1 - k0) * ld + MN - mn0) * Map::kEs;
      step = (int64_t)Map::kStageK * ld * Map::kEs;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int q = j * THREADS + tid;
      const int row = q / Map::kRowChunks, c = Map::chunk_at(row, q % Map::kRowChunks);
      off[j] = (uint32_t)row * (uint32_t)(ld * Map::kEs) + (uint32_t)c * 16u;
      if (!KMAJ && mn0 + c * Map::kEpc >= MN) off[j] = kOut;
      if (KMAJ) kchunk = c * Map::kEpc;  // the same for every j: THREADS / 8 rows apart
    }
  }
  // kleft: k from the stage's first to the end of the range.
  __device__ __forceinline__ void load(char *lds, int kleft) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass has no such builtins
    const uint32_t n = (uint32_t)(left < 0x7ffffff0ll ? left : 0x7ffffff0ll);
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, (int)n, 0x00020000);
    const int wave = uniform(threadIdx.x / kWave);
    const bool in = !KMAJ || kchunk < kleft;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (SFT_LDS void *)(lds + (j * THREADS + wave * kWave) * 16), 16,
                                               in ? off[j] : kOut, 0, 0, 0);
#endif
    base += step;
    left -= step;
  }
  __device__ __forceinline__ void store(char *) {}
};

// The same stage through registers, for any alignment and size: a chunk is read
// whole where it lies inside the operand, element by element at its edge.
template <typename T, int BMN, bool KMAJ, int THREADS>
struct GuardedLoader {
  typedef TileMap<T, BMN, KMAJ> Map;
  static constexpr int kLoads = Map::kBytes / 16 / THREADS;
  const T *base;
  int64_t ld;
  int mnleft;  // rows of the operand from the tile's first
  u32x4 v[kLoads];
  __device__ __forceinline__ void init(const void *p, int64_t ld_, int mn0, int MN, int k0, int) {
    ld = ld_;
    mnleft = MN - mn0;
    base = static_cast<const T *>(p) + (KMAJ ? (int64_t)mn0 * ld + k0 : (int64_t)k0 * ld + mn0);
  }
  __device__ __forceinline__ void load(char *, int kleft) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int q = j * THREADS + threadIdx.x;
      const int row = q / Map::kRowChunks, c = Map::chunk_at(row, q % Map::kRowChunks) * Map::kEpc;
      const int rows = KMAJ ? mnleft : kleft, cols = KMAJ ? kleft : mnleft;
      v[j] = load_chunk<T>(base + row * ld + c, row < rows ? cols - c : 0);
    }
    base += KMAJ ? Map::kStageK : Map::kStageK * ld;
  }
  __device__ __forceinline__ void store(char *lds) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4 *>(lds + (j * THREADS + threadIdx.x) * 16) = v[j];
  }
  template <typename U>
  static __device__ __forceinline__ u32x4 load_chunk(const U *p, int cnt) {
    u32x4 r = {0u, 0u, 0u, 0u};
    if (cnt >= 16 / (int)sizeof(U)) {
      __builtin_memcpy(&r, p, 16);  // one 16-byte load: the hardware takes any element alignment
    } else if (cnt > 0) {
      U e[16 / sizeof(U)];
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(U); ++i) e[i] = i < cnt ? p[i] : (U)0;
      __builtin_memcpy(&r, e, 16);
    }
    return r;
  }
};

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
template <typename T>
__device__ __forceinline__ f32x4 mma(const Frag<T> &a, const Frag<T> &b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma(const Frag<bf16_t> &a, const Frag<bf16_t> &b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c,
                                                 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma(const Frag<f16_t> &a, const Frag<f16_t> &b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c, 0,
                                                0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma(const Frag<float> &a, const Frag<float> &b, f32x4 c) {
  const f32x4 fa = __builtin_bit_cast(f32x4, a.v), fb = __builtin_bit_cast(f32x4, b.v);
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[s], fb[s], c, 0, 0, 0);
  return c;
}

// Reads fragments of F consecutive 16-row groups of an LDS tile, from row mn0.
// Lane l holds row l % 16, and of each 64 bytes of k the 16 bytes number l / 16.
template <typename T, int BMN, bool KMAJ, int F>
struct FragReader {
  typedef TileMap<T, BMN, KMAJ> Map;
  int at[KMAJ ? 2 : F];
  __device__ __forceinline__ void init(int mn0) {
    const int i = lane_id() % 16, g = lane_id() / 16;
    if (KMAJ) {
      const int row = mn0 + i;
      // mn0 + 16 f leaves the permutation as it is
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) at[kk] = row * kStageBytes + (Map::chunk_at(row, kk * 4 + g) << 4);
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
  __device__ __forceinline__ Frag<T> read(const char *lds, int f, int kk) const {
    Frag<T> r;
    if constexpr (KMAJ) {
      r.v = *reinterpret_cast<const u32x4 *>(lds + at[kk] + f * 16 * kStageBytes);
    } else if constexpr (Map::kEs == 2) {
      const char *p = lds + at[f] + kk * 32 * Map::kRowBytes;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SFT_LDS i16x4 *)p));
      const u32x2 hi = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((SFT_LDS i16x4 *)(p + 4 * Map::kRowBytes)));
      r.v = u32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
      const char *p = lds + at[f] + kk * 16 * Map::kRowBytes;
#pragma unroll
      for (int s = 0; s < 4; ++s) r.v[s] = *reinterpret_cast<const uint32_t *>(p + s * Map::kRowBytes);
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

// BM x BN outputs per workgroup of WM x WN waves; two LDS stages, the copy of one
// beside the products of the other.
template <typename T, bool AK, bool BK, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(WM *WN *kWave) void gemm_tile_kernel(const Gemm g) {
  constexpr int kThreads = WM * WN * kWave;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int kStageK = kStageBytes / (int)sizeof(T);
  constexpr int kStage = (BM + BN) * kStageBytes;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  int tm, tn, split;
  tile_of(g, tm, tn, split);
  const int m0 = tm * BM, n0 = tn * BN;
  const int k0 = split * g.split_k;
  const int kend = g.K - k0 < g.split_k ? g.K : k0 + g.split_k;
  const int wave = uniform(threadIdx.x / kWave);
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  typedef typename std::conditional<DIRECT, DirectLoader<T, BM, AK, kThreads>,
                                    GuardedLoader<T, BM, AK, kThreads>>::type LoadA;
  typedef typename std::conditional<DIRECT, DirectLoader<T, BN, BK, kThreads>,
                                    GuardedLoader<T, BN, BK, kThreads>>::type LoadB;
  LoadA la;
  LoadB lb;
  la.init(g.a, g.lda, m0, g.M, k0, kend);
  lb.init(g.b, g.ldb, n0, g.N, k0, kend);
  FragReader<T, BM, AK, FM> ra;
  FragReader<T, BN, BK, FN> rb;
  ra.init(wm);
  rb.init(wn);

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int steps = (kend - k0 + kStageK - 1) / kStageK;
  la.load(lds, kend - k0);
  lb.load(lds + BM * kStageBytes, kend - k0);
  la.store(lds);
  lb.store(lds + BM * kStageBytes);
  for (int it = 0; it < steps; ++it) {
    char *cur = lds + (it & 1) * kStage, *nxt = lds + (~it & 1) * kStage;
    // this stage has arrived, and every wave has done with the other one
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool more = it + 1 < steps;
    if (more) {
      const int kleft = kend - k0 - (it + 1) * kStageK;
      la.load(nxt, kleft);
      lb.load(nxt + BM * kStageBytes, kleft);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      Frag<T> fa[FM], fb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = ra.read(cur, i, kk);
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = rb.read(cur + BM * kStageBytes, j, kk);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
    }
    if (more) {
      la.store(nxt);
      lb.store(nxt + BM * kStageBytes);
    }
  }
  // The first operand's rows are the result's four registers: lane l holds
  // m = l % 16 and n = 4 (l / 16) + 0..3 of each fragment.
  const int lane = lane_id();
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = m0 + wm + i * 16 + lane % 16;
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + j * 16 + lane / 16 * 4;
      if (n >= g.N) continue;
      if (g.part) {
        float v[4] = {acc[i][j].x, acc[i][j].y, acc[i][j].z, acc[i][j].w};
        store4(g.part + ((int64_t)split * g.M + m) * g.N + n, g.N % 4 == 0, g.N - n, v);
      } else {
        finish4<T>(g.epi, m, n, g.N, acc[i][j]);
      }
    }
  }
}

// Sums a split product's partials in split order and finishes them.
template <typename T>
__global__ __launch_bounds__(kBlock) void gemm_join_kernel(const Gemm g) {
  const int64_t quads = (g.N + 3) / 4;
  const int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (q >= quads * g.M) return;
  const int64_t m = q / quads;
  const int n = (int)(q % quads) * 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const float *p = g.part + m * g.N + n;
  for (int s = 0; s < g.splits; ++s, p += (int64_t)g.M * g.N) {
    float v[4];
    load4(p, g.N % 4 == 0, g.N - n, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += v[i];
  }
  finish4<T>(g.epi, m, n, g.N, acc);
}

// ---- few rows ----
// y for up to 16 FM rows: a workgroup holds 16 outputs of every row; its waves take
// 256-byte pieces of k in turn, straight from global memory (W is read once and
// there is no reuse for LDS to serve), and are summed in wave order.
constexpr int kRowWaves = 8;
template <typename T, int FM>
__global__ __launch_bounds__(kRowWaves *kWave) void gemm_rows_kernel(const Gemm g) {
  constexpr int kEpc = 16 / (int)sizeof(T), kPiece = 16 * kEpc;
  __shared__ f32x4 red[kRowWaves][FM][kWave];
  const int lane = lane_id(), i = lane % 16, c = lane / 16;
  const int wave = uniform(threadIdx.x / kWave);
  const int n0 = blockIdx.x * 16;
  const bool nin = n0 + i < g.N;
  const T *w = static_cast<const T *>(g.b) + (int64_t)(nin ? n0 + i : 0) * g.ldb;
  const T *x[FM];
  bool in[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) {
    in[f] = f * 16 + i < g.M;
    x[f] = static_cast<const T *>(g.a) + (int64_t)(in[f] ? f * 16 + i : 0) * g.lda;
  }
  f32x4 acc[FM];
#pragma unroll
  for (int f = 0; f < FM; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  typedef GuardedLoader<T, 16, true, kWave> Chunk;
  for (int k0 = wave * kPiece; k0 < g.K; k0 += kRowWaves * kPiece) {
    Frag<T> fw[4], fx[FM][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + (u * 4 + c) * kEpc;
      fw[u].v = Chunk::load_chunk(w + k, nin ? g.K - k : 0);
#pragma unroll
      for (int f = 0; f < FM; ++f) fx[f][u].v = Chunk::load_chunk(x[f] + k, in[f] ? g.K - k : 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int f = 0; f < FM; ++f) acc[f] = mma<T>(fw[u], fx[f][u], acc[f]);
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
  if (m < g.M && n < g.N) finish4<T>(g.epi, m, n, g.N, sum);
}

// ---- gradient of the activation, and the bias grad's partial sums ----
// dz = dy * act'(z), rounded to the layer's type for the products that follow, and
// the sums of the unrounded dz over `rows` rows per workgroup and column.  A thread
// holds V columns; a workgroup is tx column groups by 256 / tx rows.
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void act_bwd_kernel(const ActBwd p) {
  typedef typename Deriv<T>::type D;
  __shared__ float red[kBlock * V];
  const int tx = p.tx, ty = kBlock / tx;
  const int cx = threadIdx.x % tx, ry = threadIdx.x / tx;
  const int n = (blockIdx.x * tx + cx) * V;
  const int64_t first = (int64_t)blockIdx.y * p.rows;
  const int64_t last = first + p.rows < p.M ? first + p.rows : p.M;
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  if (n < p.N) {
    for (int64_t m = first + ry; m < last; m += ty) {
      T dy[V];
      __builtin_memcpy(dy, static_cast<const T *>(p.dy) + m * p.lddy + n, sizeof(T) * V);
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (float)dy[i];
      if (p.deriv) {
        D d[V];
        __builtin_memcpy(d, static_cast<const D *>(p.deriv) + m * p.N + n, sizeof(D) * V);
        T dz[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] *= Deriv<T>::unpack(d[i]);
          dz[i] = (T)v[i];
        }
        __builtin_memcpy(static_cast<T *>(p.dz) + m * p.N + n, dz, sizeof(T) * V);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += v[i];
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = sum[i];
  __syncthreads();
  if (ry != 0 || n >= p.N) return;
  for (int r = 1; r < ty; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += red[(r * tx + cx) * V + i];
#pragma unroll
  for (int i = 0; i < V; ++i) p.part[(int64_t)blockIdx.y * p.N + n + i] = sum[i];
}

// db[n] = the partials of column n in order.  A workgroup holds 64 columns, its four
// waves a quarter of the partials each.
template <typename T>
__global__ __launch_bounds__(kBlock) void bias_join_kernel(const float *__restrict__ part, int parts, int N, void *db) {
  __shared__ float red[kWavesPerBlock][kWave];
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  const int n = blockIdx.x * kWave + lane;
  const int per = (parts + kWavesPerBlock - 1) / kWavesPerBlock;
  float s = 0.f;
  if (n < N)
    for (int r = w * per; r < (w + 1) * per && r < parts; ++r) s += part[(int64_t)r * N + n];
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && n < N) static_cast<T *>(db)[n] = (T)((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
}

// ---- launchers, instantiated per type ----
template <typename T, bool AK, bool BK>
int launch_gemm_as(const Gemm &g, hipStream_t s) {
  const int64_t grid = (int64_t)g.tiles_m * g.tiles_n * g.splits;
#define SFT_TILE(BM, BN, WM, WN, DIRECT)                                                                       \
  hipLaunchKernelGGL((gemm_tile_kernel<T, AK, BK, BM, BN, WM, WN, DIRECT>), dim3((unsigned)grid),              \
                     dim3(WM *WN *kWave), 0, s, g)
  if (g.direct)
    SFT_TILE(128, 128, 2, 2, true);
  else
    SFT_TILE(128, 128, 2, 2, false);
#undef SFT_TILE
  if (g.splits > 1) {
    const int64_t quads = ((int64_t)g.N + 3) / 4 * g.M;
    hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)ceil_div(quads, kBlock)), dim3(kBlock), 0, s, g);
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
int launch_act_bwd(const ActBwd &p, void *db, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int cols = p.vec ? (int)ceil_div(p.N, V) : p.N;
  const dim3 grid((unsigned)ceil_div(cols, p.tx), (unsigned)p.parts);
  if (p.vec)
    hipLaunchKernelGGL((act_bwd_kernel<T, V>), grid, dim3(kBlock), 0, s, p);
  else
    hipLaunchKernelGGL((act_bwd_kernel<T, 1>), grid, dim3(kBlock), 0, s, p);
  if (db)
    hipLaunchKernelGGL((bias_join_kernel<T>), dim3((unsigned)ceil_div(p.N, kWave)), dim3(kBlock), 0, s, p.part,
                       p.parts, p.N, db);
  return check_launch("dense activation backward");
}

#define SFT_DENSE_TYPE(T)                                                \
  template int launch_gemm<T>(const Gemm &, int, hipStream_t);           \
  template int launch_rows<T>(const Gemm &, hipStream_t);                \
  template int launch_act_bwd<T>(const ActBwd &, void *, hipStream_t);

}  // namespace dense
}  // namespace sft
