// Distillation from a teacher's top classes.  For a row with student logits s over V
// classes and teacher logits t_j for k of them (class i_j; an index outside [0, V)
// leaves the slot empty), at temperature tau:
//   p = softmax(s / tau) over all classes, q = softmax(t / tau) over the filled slots
//   loss = tau^2 sum_j q_j (log q_j - log p_{i_j})
//   d loss / d s_v = tau (p_v - sum of q_j over the slots of class v)
// Slots with q = 0 add nothing, whatever the student says there.  A row without a
// filled slot (or whose teacher logits are all -inf), or with all classes at -inf, has
// loss 0 and no gradient; a NaN anywhere in a taught row makes both NaN.
//
// Bound by reading the logits once and writing the gradient once.  A row is read as it
// comes, with a running maximum and sum per thread, and stays in the registers of the
// waves that hold it, as loaded, until the gradient; rows longer than a workgroup's
// registers are read again, from L2 or the memory-side cache.  Rows start anywhere, so
// they are cut at the logits' 16-byte lines: whole chunks, and the few elements before
// and after them one a thread.  All loads of a row are made without branches, so that
// they are under way together.  Long rows hold a CU with one workgroup whose reading,
// reducing and writing follow each other: 2048 x 100003 bf16 takes 97 us for the loss and
// 218 for the gradient, 4.2 and 3.8 TB/s.
#include "dense.h"
#include "dense_reduce.h"

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

// The running maximum m of some x and the sum of 2^((x - m) c).
struct Running {
  float m = -INFINITY, sum = 0.f;
  template <int V>
  __device__ __forceinline__ void add(const float (&x)[V], float c) {
    float top = m;
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
    const float at = top == -INFINITY ? 0.f : top;  // nothing above -inf yet: all terms are 0
    sum *= __builtin_amdgcn_exp2f((m - at) * c);
#pragma unroll
    for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - at) * c);
    m = top;
  }
  __device__ __forceinline__ float scaled(float top, float c) const {
    return sum * __builtin_amdgcn_exp2f((m - (top == -INFINITY ? 0.f : top)) * c);
  }
  // Over the wave.
  __device__ __forceinline__ void join(float c) {
    const float top = dense::group_max<kWave>(m);
    sum = dense::group_sum<kWave>(scaled(top, c));
    m = top;
  }
};

__device__ __forceinline__ float load_type(const void *p, int64_t i, int type) {
  if (type == SFT_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == SFT_TYPE_F16) return (float)static_cast<const f16_t *>(p)[i];
  return (float)static_cast<const bf16_t *>(p)[i];
}

// The teacher's side of a row, in one wave: lane l holds the slots l + 64 j.
struct Teacher {
  int idx[kSlots];     // class, or -1
  float q[kSlots];     // probability
  float log_q[kSlots];
  float at[kSlots];    // the student's logit there
  bool any;
  template <typename T>
  __device__ __forceinline__ void load(const Distill &d, int64_t row, const T *s) {
    const int lane = lane_id();
    const float c = 1.f / d.tau;
    float t[kSlots], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      idx[j] = -1;
      t[j] = -INFINITY;
      log_q[j] = at[j] = 0.f;
      if (j * kWave >= d.k) continue;  // uniform
      const int slot = lane + j * kWave;
      if (slot < d.k) {
        const int64_t o = row * d.k + slot;
        const int64_t i = d.idx64 ? static_cast<const int64_t *>(d.idx)[o] : static_cast<const int32_t *>(d.idx)[o];
        if (i >= 0 && i < d.V) {
          idx[j] = (int)i;
          t[j] = load_type(d.t, o, d.ttype);
          at[j] = (float)s[i];
        }
      }
      m = t[j] > m || t[j] != t[j] ? t[j] : m;  // a NaN stays
    }
    m = dense::group_reduce<kWave>(m, [](float a, float b) { return b > a || b != b ? b : a; });
    any = !(m == -INFINITY);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      q[j] = 0.f;
      if (j * kWave >= d.k) continue;
      log_q[j] = any ? (t[j] - m) * c : 0.f;
      q[j] = any ? expf(log_q[j]) : 0.f;
      sum += q[j];
    }
    sum = dense::group_sum<kWave>(sum);
    const float inv = any ? 1.f / sum : 0.f, log_sum = any ? logf(sum) : 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kWave >= d.k) continue;
      q[j] *= inv;
      log_q[j] -= log_sum;
    }
  }
  // sum_j q_j (log q_j - log p_{i_j}), of a student's row with maximum m and sum of
  // exponentials: taken slot by slot, since sums of either part would cancel.
  __device__ __forceinline__ float divergence(const Distill &d, float m, float sum) const {
    const float c = 1.f / d.tau, log_sum = logf(sum);
    float all = 0.f;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      if (j * kWave >= d.k) continue;
      if (q[j] != 0.f) all += q[j] * (log_q[j] - ((at[j] - m) * c - log_sum));
    }
    return dense::group_sum<kWave>(all);
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
__device__ __forceinline__ void unpack(const u32x4 &v, float (&x)[16 / sizeof(T)]) {
  T e[16 / sizeof(T)];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) x[i] = (float)e[i];
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&x)[16 / sizeof(T)]) {
  T e[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) e[i] = (T)x[i];
  u32x4 v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

// TPR threads per row (one wave, or the whole workgroup of TPR), C chunks a thread.
// C = 0: the row does not fit, its chunks are read again.
template <typename T, int TPR, int C>
__global__ __launch_bounds__(TPR == kWave ? kBlock : TPR) void distill_kernel(const Distill d) {
  constexpr int V = 16 / (int)sizeof(T), kWaves = TPR / kWave;
  constexpr int kRowsPer = TPR == kWave ? kWavesPerBlock : 1;
  __shared__ float top[kWaves], sums[kWaves];
  __shared__ int shared_any;
  __shared__ int slot_idx[kWaves > 1 ? SFT_DISTILL_MAX_K : 1];  // the teacher's side, until the end
  __shared__ float slot_q[kWaves > 1 ? SFT_DISTILL_MAX_K : 1];
  __shared__ float slot_log_q[kWaves > 1 ? SFT_DISTILL_MAX_K : 1];
  __shared__ float slot_at[kWaves > 1 ? SFT_DISTILL_MAX_K : 1];
  const int tid = threadIdx.x % TPR, wave = uniform(tid / kWave);
  const int64_t row = (int64_t)blockIdx.x * kRowsPer + uniform(threadIdx.x / TPR);
  if (row >= d.rows) return;  // whole waves, and never part of a row's
  const T *s = static_cast<const T *>(d.s) + row * d.lds;
  T *ds = static_cast<T *>(d.ds) + row * (int64_t)d.V;
  // `head` elements, whole chunks, and the rest; thread i < edge has one of the others
  const int shift = (int)((uintptr_t)s / sizeof(T) % V);
  int head = shift ? V - shift : 0;
  head = head < d.V ? head : d.V;
  const int body = (d.V - head) / V, edge = d.V - body * V;
  const int mine = tid < head ? tid : d.V - edge + tid;
  const T *sb = s + head;
  T *dsb = ds + head;
  const float c2 = 1.44269504088896341f / d.tau;  // exp(x / tau) = 2^(x c2)

  T nothing[V];
#pragma unroll
  for (int i = 0; i < V; ++i) nothing[i] = (T)(-INFINITY);
  u32x4 none;
  __builtin_memcpy(&none, nothing, 16);
  u32x4 raw[C ? C : 1];
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = tid + TPR * j;
      if (body > 0) __builtin_memcpy(&raw[j], sb + (int64_t)(c < body ? c : body - 1) * V, 16);
    }
  }
  float x_edge = (float)s[tid < edge ? mine : 0];
  if (tid >= edge) x_edge = -INFINITY;
  Teacher te;
  if (wave == 0) {
    te.load(d, row, s);
    if (kWaves > 1) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        slot_idx[lane_id() + j * kWave] = te.idx[j];
        slot_q[lane_id() + j * kWave] = te.q[j];
        slot_log_q[lane_id() + j * kWave] = te.log_q[j];
        slot_at[lane_id() + j * kWave] = te.at[j];
      }
    }
  }
  Running run;
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (tid + TPR * j >= body) raw[j] = none;
      float x[V];
      unpack<T>(raw[j], x);
      run.add(x, c2);
    }
  } else {
#pragma unroll 4
    for (int c = tid; c < body; c += TPR) {
      u32x4 v;
      float x[V];
      __builtin_memcpy(&v, sb + (int64_t)c * V, 16);
      unpack<T>(v, x);
      run.add(x, c2);
    }
  }
  {
    const float x[1] = {x_edge};
    run.add(x, c2);
  }
  run.join(c2);
  if (kWaves > 1) {
    if (tid % kWave == 0) {
      top[wave] = run.m;
      sums[wave] = run.sum;
    }
    if (tid == 0) shared_any = te.any;
    __syncthreads();
    // every wave joins the waves' results, in the same order
    const int l = lane_id();
    run.m = l < kWaves ? top[l] : -INFINITY;
    run.sum = l < kWaves ? sums[l] : 0.f;
    run.join(c2);
    te.any = shared_any;
  }
  const float m = run.m, sum = run.sum;
  // a row whose numbers are all NaN or -inf has no maximum either, but its sum is NaN
  const bool live = te.any && (m > -INFINITY || sum != 0.f);
  auto put_loss = [&]() {
    if (!d.loss || wave != 0) return;
    if (kWaves > 1) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        te.q[j] = slot_q[lane_id() + j * kWave];
        te.log_q[j] = slot_log_q[lane_id() + j * kWave];
        te.at[j] = slot_at[lane_id() + j * kWave];
      }
    }
    const float kl = te.divergence(d, m, sum);
    if (tid == 0) d.loss[row] = live ? d.tau * d.tau * kl : 0.f;
  };
  // With a gradient to come, a workgroup's loss waits until the row has left the registers:
  // beside it 2048 x 49152 bf16 takes 95 us instead of 84.
  if (kWaves == 1 || !d.ds) put_loss();
  if (!d.ds) return;

  const float g = d.tau * (d.weight ? d.weight[row] : 1.f), gp = g / sum;
  auto grad = [&](float x) { return live ? gp * __builtin_amdgcn_exp2f((x - m) * c2) : 0.f; };
  auto put = [&](int c, const u32x4 &v) {
    float x[V];
    unpack<T>(v, x);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = grad(x[i]);
    const u32x4 e = pack<T>(x);
    __builtin_memcpy(dsb + (int64_t)c * V, &e, 16);
  };
  if (C) {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (tid + TPR * j < body) put(tid + TPR * j, raw[j]);
  } else {
#pragma unroll 4
    for (int c = tid; c < body; c += TPR) {
      u32x4 v;
      __builtin_memcpy(&v, sb + (int64_t)c * V, 16);
      put(c, v);
    }
  }
  if (tid < edge) ds[mine] = (T)grad(x_edge);
  if (kWaves > 1) put_loss();
  if (!live) return;  // the same for the whole row
  // The teacher's classes once more, after the stores above have been made.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (kWaves > 1) __syncthreads();
  if (wave != 0) return;
  if (kWaves > 1) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      te.idx[j] = slot_idx[lane_id() + j * kWave];
      te.q[j] = slot_q[lane_id() + j * kWave];
    }
  }
  float total[kSlots];
  te.merged(d.k, total);
#pragma unroll
  for (int j = 0; j < kSlots; ++j)
    if (te.idx[j] >= 0)
      ds[te.idx[j]] = (T)(gp * __builtin_amdgcn_exp2f(((float)s[te.idx[j]] - m) * c2) - g * total[j]);
}

// A row goes to the fewest waves whose registers hold it: a row of one wave needs no
// meeting, and no chunk slot should be idle.  us of loss and gradient in bf16, k = 32, as
// chosen / with the next larger form of the list: 65536 x 512 104 / 154 and 32768 x 2048
// 81 / 90 (a wave / a workgroup), 16384 x 4096 65 / 82 (8 chunks of a wave / 4 of four waves),
// 8192 x 16384 115 / 149, 2048 x 49152 84 / 98 (6 chunks / 8), 2048 x 104000 187 / 210 (13 / 16).
// Rows beyond 16 chunks of 16 waves are read twice: 1024 x 131000 143 held, 150 read twice.
// At 16384 x 4096 the rows are read and written at 4.3 TB/s, what a copy reaches.
template <typename T>
void launch(const Distill &d, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int64_t chunks = d.V / V;
#define SFT_DISTILL(most, TPR, C)                                                                                  \
  if (chunks <= most) {                                                                                            \
    hipLaunchKernelGGL((distill_kernel<T, TPR, C>),                                                                \
                       dim3((unsigned)ceil_div(d.rows, TPR == kWave ? kWavesPerBlock : 1)),                        \
                       dim3(TPR == kWave ? kBlock : TPR), 0, s, d);                                                \
    return;                                                                                                        \
  }
  SFT_DISTILL(64, 64, 1)  // an edge of up to 14 elements fits any wave
  SFT_DISTILL(128, 64, 2)
  SFT_DISTILL(256, 64, 4)
  SFT_DISTILL(512, 64, 8)
  SFT_DISTILL(1024, 256, 4)
  SFT_DISTILL(2048, 256, 8)
  SFT_DISTILL(4096, 1024, 4)
  SFT_DISTILL(6144, 1024, 6)
  SFT_DISTILL(8192, 1024, 8)
  SFT_DISTILL(10240, 1024, 10)
  SFT_DISTILL(13312, 1024, 13)
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
