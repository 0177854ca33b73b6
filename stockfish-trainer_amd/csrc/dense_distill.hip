// Distillation from a teacher's top classes.  For a row with student logits s over V
// classes and teacher logits t_j for k of them (class i_j; an index outside [0, V)
// leaves the slot empty), at temperature tau:
//   p = softmax(s / tau) over all classes, q = softmax(t / tau) over the filled slots
//   loss = tau^2 sum_j q_j (log q_j - log p_{i_j})
//   d loss / d s_v = tau (p_v - sum of q_j over the slots of class v)
// Slots with q = 0 add nothing, whatever the student says there.  A row without a
// filled slot (or whose teacher logits are all -inf), or without a class above -inf,
// has loss 0 and no gradient.
//
// Bound by reading the logits once and writing the gradient once: a row stays in the
// registers of the waves that hold it, as loaded, between the maximum, the sum and
// the gradient.  Rows longer than the registers of a workgroup are read again, from
// L2 or the memory-side cache.
#include "dense.h"

namespace sft {

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Distill {
  const void *s, *t, *idx;
  int64_t lds, rows;
  int V, k, ttype, idx64;
  float tau;
  const float *weight;  // [rows] or null (1): scale of a row's gradient
  float *loss;          // [rows] or null
  void *ds;             // dense [rows, V] or null
};

constexpr int kSlots = SFT_DISTILL_MAX_K / kWave;  // slots per lane

template <int TPR>
struct Team {  // the threads of a row: a wave, or the workgroup
  static constexpr int kWaves = TPR / kWave;
  static __device__ __forceinline__ float max(float x, float *red) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
    if (kWaves == 1) return x;
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) x = fmaxf(x, red[i]);
    return x;
  }
  static __device__ __forceinline__ float sum(float x, float *red) {
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) x += __shfl_xor(x, m);
    if (kWaves == 1) return x;
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) x += red[i];
    return x;
  }
};

__device__ __forceinline__ float load_type(const void *p, int64_t i, int type) {
  if (type == SFT_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == SFT_TYPE_F16) return (float)static_cast<const f16_t *>(p)[i];
  return (float)static_cast<const bf16_t *>(p)[i];
}

// The teacher's side of a row, in one wave: lane l holds the slots l + 64 j.
struct Teacher {
  int idx[kSlots];    // class, or -1
  float q[kSlots];    // probability
  float cross;        // sum_j q_j (log q_j - s_{i_j} / tau)
  bool any;
  template <typename T>
  __device__ __forceinline__ void load(const Distill &d, int64_t row, const T *s) {
    const int lane = lane_id();
    const float c = 1.f / d.tau;
    float t[kSlots], at[kSlots], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      idx[j] = -1;
      t[j] = -INFINITY;
      at[j] = 0.f;
      if (j * kWave >= d.k) continue;  // uniform
      const int slot = lane + j * kWave;
      if (slot < d.k) {
        const int64_t o = row * d.k + slot;
        const int64_t i = d.idx64 ? static_cast<const int64_t *>(d.idx)[o] : static_cast<const int32_t *>(d.idx)[o];
        if (i >= 0 && i < d.V) {
          idx[j] = (int)i;
          t[j] = load_type(d.t, o, d.ttype) * c;
          at[j] = (float)s[i] * c;
        }
      }
      m = t[j] > m || t[j] != t[j] ? t[j] : m;  // a NaN stays
    }
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) {
      const float o = __shfl_xor(m, x);
      m = o > m || o != o ? o : m;
    }
    any = !(m == -INFINITY);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      q[j] = 0.f;
      if (j * kWave >= d.k) continue;
      q[j] = any ? expf(t[j] - m) : 0.f;
      sum += q[j];
    }
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) sum += __shfl_xor(sum, x);
    const float inv = any ? 1.f / sum : 0.f, log_sum = any ? logf(sum) : 0.f;
    cross = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kWave >= d.k) continue;
      q[j] *= inv;
      if (q[j] != 0.f) cross += q[j] * (t[j] - m - log_sum - at[j]);
    }
#pragma unroll
    for (int x = 1; x < kWave; x <<= 1) cross += __shfl_xor(cross, x);
  }
  // q of the class of slot j, over all its slots (classes may be named twice).
  __device__ __forceinline__ void merged(int k, float (&total)[kSlots]) const {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) total[j] = 0.f;
#pragma unroll
    for (int o = 0; o < kSlots; ++o) {
      const int n = k - o * kWave < kWave ? k - o * kWave : kWave;
      for (int l = 0; l < n; ++l) {
        const int i = __builtin_amdgcn_readlane(idx[o], l);
        const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, q[o]), l));
#pragma unroll
        for (int j = 0; j < kSlots; ++j) total[j] += idx[j] == i ? v : 0.f;
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void load_chunk(const T *p, int cnt, u32x4 &v) {
  constexpr int V = 16 / (int)sizeof(T);
  if (cnt >= V) {
    __builtin_memcpy(&v, p, 16);
  } else {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = i < cnt ? p[i] : (T)(-INFINITY);
    __builtin_memcpy(&v, e, 16);
  }
}
template <typename T>
__device__ __forceinline__ void unpack(const u32x4 &v, float (&x)[16 / sizeof(T)]) {
  T e[16 / sizeof(T)];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) x[i] = (float)e[i];
}
template <typename T>
__device__ __forceinline__ void store_chunk(T *p, int cnt, const float (&x)[16 / sizeof(T)]) {
  constexpr int V = 16 / (int)sizeof(T);
  T e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = (T)x[i];
  if (cnt >= V) {
    __builtin_memcpy(p, e, 16);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < cnt) p[i] = e[i];
  }
}

// TPR threads per row (one wave, or the whole workgroup of TPR), C chunks a thread.
// C = 0: the row does not fit, its chunks are read again.
template <typename T, int TPR, int C>
__global__ __launch_bounds__(TPR == kWave ? kBlock : TPR) void distill_kernel(const Distill d) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int kRowsPer = TPR == kWave ? kWavesPerBlock : 1;
  __shared__ float red[2][TPR / kWave];
  const int tid = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRowsPer + uniform(threadIdx.x / TPR);
  if (row >= d.rows) return;  // whole waves, and never part of a team
  const T *s = static_cast<const T *>(d.s) + row * d.lds;
  const int chunks = (d.V + V - 1) / V;
  const bool first = uniform(threadIdx.x / kWave) % (TPR / kWave) == 0;  // the team's first wave

  u32x4 raw[C ? C : 1];
  float m = -INFINITY;
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j) load_chunk<T>(s + (int64_t)(tid + TPR * j) * V, d.V - (tid + TPR * j) * V, raw[j]);
  }
  Teacher te;
  te.load(d, row, s);  // every wave: all need `any`
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float x[V];
      unpack<T>(raw[j], x);
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
    }
  } else {
    for (int c = tid; c < chunks; c += TPR) {
      u32x4 v;
      float x[V];
      load_chunk<T>(s + (int64_t)c * V, d.V - c * V, v);
      unpack<T>(v, x);
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
    }
  }
  m = Team<TPR>::max(m, red[0]);
  const bool live = te.any && m > -INFINITY;
  const float c2 = 1.44269504088896341f / d.tau;  // exp(x / tau) = 2^(x c2)
  float sum = 0.f;
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float x[V];
      unpack<T>(raw[j], x);
#pragma unroll
      for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - m) * c2);
    }
  } else {
    for (int c = tid; c < chunks; c += TPR) {
      u32x4 v;
      float x[V];
      load_chunk<T>(s + (int64_t)c * V, d.V - c * V, v);
      unpack<T>(v, x);
#pragma unroll
      for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - m) * c2);
    }
  }
  sum = Team<TPR>::sum(sum, red[1]);
  if (d.loss && tid == 0) d.loss[row] = live ? d.tau * d.tau * (te.cross + m / d.tau + logf(sum)) : 0.f;
  if (!d.ds) return;

  T *ds = static_cast<T *>(d.ds) + row * (int64_t)d.V;
  const float g = d.tau * (d.weight ? d.weight[row] : 1.f), gp = g / sum;
  auto put = [&](int c, const u32x4 &v) {
    float x[V];
    unpack<T>(v, x);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = live ? gp * __builtin_amdgcn_exp2f((x[i] - m) * c2) : 0.f;
    store_chunk<T>(ds + (int64_t)c * V, d.V - c * V, x);
  };
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if ((tid + TPR * j) * V < d.V) put(tid + TPR * j, raw[j]);
  } else {
    for (int c = tid; c < chunks; c += TPR) {
      u32x4 v;
      load_chunk<T>(s + (int64_t)c * V, d.V - c * V, v);
      put(c, v);
    }
  }
  if (!live) return;  // the same in the whole team
  // The teacher's classes once more, after the stores above have been made.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (TPR > kWave) __syncthreads();
  if (!first) return;
  float total[kSlots];
  te.merged(d.k, total);
#pragma unroll
  for (int j = 0; j < kSlots; ++j)
    if (te.idx[j] >= 0)
      ds[te.idx[j]] = (T)(gp * __builtin_amdgcn_exp2f(((float)s[te.idx[j]] - m) * c2) - g * total[j]);
}

template <typename T>
void launch(const Distill &d, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t chunks = ceil_div(d.V, V);
#define SFT_DISTILL(most, TPR, C)                                                                                  \
  if (chunks <= most) {                                                                                            \
    hipLaunchKernelGGL((distill_kernel<T, TPR, C>),                                                                \
                       dim3((unsigned)ceil_div(d.rows, TPR == kWave ? kWavesPerBlock : 1)),                        \
                       dim3(TPR == kWave ? kBlock : TPR), 0, s, d);                                                \
    return;                                                                                                        \
  }
  SFT_DISTILL(64, 64, 1)
  SFT_DISTILL(128, 64, 2)
  SFT_DISTILL(256, 64, 4)
  SFT_DISTILL(512, 64, 8)
  SFT_DISTILL(1024, 256, 4)
  SFT_DISTILL(2048, 256, 8)
  SFT_DISTILL(4096, 1024, 4)
  SFT_DISTILL(8192, 1024, 8)
  SFT_DISTILL(16384, 1024, 16)
  SFT_DISTILL(INT64_MAX, 1024, 0)
#undef SFT_DISTILL
}

}  // namespace

int distill(int dtype, const void *student, int64_t lds, int ttype, const void *teacher, const void *idx, int idx64,
            int64_t rows, int V, int k, float tau, const float *weight, float *loss, void *ds, hipStream_t s) {
  const Distill d{student, teacher, idx, lds, rows, V, k, ttype, idx64, tau, weight, loss, ds};
  ProfScope prof(kProfDenseDistill, s);
  if (dtype == SFT_TYPE_F32) launch<float>(d, s);
  else if (dtype == SFT_TYPE_F16) launch<f16_t>(d, s);
  else launch<bf16_t>(d, s);
  return check_launch("sft_distill");
}

}  // namespace sft
