// The router's balance loss.  For the kept positions t of n, with p = softmax of a
// position's logits and S_t its top_k experts:
//   counts_e = #{t : e in S_t},  f_e = counts_e / (n top_k),  P_e = mean_t p_te
//   loss     = E sum_e f_e P_e
//   d loss / d logit_tj = E / n p_tj (f_j - sum_e f_e p_te)      (f is piecewise constant)
// A position is kept if its mask byte is set (or there is no mask) and not all its logits
// are -inf; a NaN in a kept one makes the loss NaN.  Experts are chosen by logit, equal ones by the lower number; those at
// -inf are never chosen.
//
// Bound by reading the logits (and, in the backward, writing as much): every row is
// held by a group of G lanes in 16-byte chunks, G the power of two that covers it, so
// softmax, choice and gradient need one read and shuffles inside the group.  The
// sums over positions stay in registers of the lane that owns the expert; workgroups
// write partials that one more launch adds in a fixed order, in binary64.  524288 x 64
// bf16, two experts a position: forward 28 to 30 us (2.3 TB/s; the choice's comparisons
// take as long as the loads), join 5, backward 35 (3.8 TB/s).
#include "dense.h"
#include "dense_reduce.h"

namespace sft {

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

using dense::group_max;
using dense::group_reduce;
using dense::group_sum;

constexpr int kThreads = 1024;   // of the forward: 16 waves, whose sums leave as one partial
// Its workgroups, one per CU: with two, 524288 x 8 bf16 takes 16.0 us instead of 13.7 and
// 65536 x 256 31.1 instead of 25.8 (twice the partials to join), 524288 x 64 33 either way.
constexpr int kMaxParts = 256;

// A row's logits: lane t of the group holds the chunks t + G j of V elements.  Loads
// have no branches, so that the next row's are under way beside this one's work; open()
// turns them into numbers, -inf past E.  WHOLE: E is a multiple of V, and a chunk is one
// load (524288 x 64 bf16 forward 33 us, element by element 47.5).
template <typename T, int G, int C, bool WHOLE>
struct Row {
  static constexpr int V = 16 / (int)sizeof(T);
  T raw[C][V];
  float x[C][V];
  __device__ __forceinline__ void load(const T *row, int E, int t) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int e0 = (t + G * j) * V;
      if (WHOLE) {
        __builtin_memcpy(raw[j], row + (e0 < E ? e0 : 0), 16);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) raw[j][i] = row[e0 + i < E ? e0 + i : 0];
      }
    }
  }
  __device__ __forceinline__ void open(int E, int t) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) x[j][i] = (t + G * j) * V + i < E ? (float)raw[j][i] : -INFINITY;
  }
  __device__ __forceinline__ float max() const {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) m = fmaxf(m, x[j][i]);
    return group_max<G>(m);
  }
  // p = exp(x - m) / sum, and the sum: 0 where all is -inf (p means nothing then), NaN
  // where a NaN is in the row, which max() passes over.
  __device__ __forceinline__ float softmax(float m, float (&p)[C][V]) const {
    if (m == -INFINITY) m = 0.f;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[j][i] = __builtin_amdgcn_exp2f((x[j][i] - m) * 1.44269504088896341f);
        s += p[j][i];
      }
    s = group_sum<G>(s);
    const float r = 1.f / s;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) p[j][i] *= r;
    return s;
  }
};

// One workgroup: counts, the number of kept rows and the loss from the partials.
// Threads (slice, expert): a slice adds every kSlices-th partial, the slices are
// added in order.
__device__ __forceinline__ void join_parts(const float *part_p, const int32_t *part_c, const int32_t *part_n, int parts,
                                           int E, int top_k, float *loss, int64_t *counts, int64_t *kept) {
  __shared__ double red_p[kThreads];
  __shared__ int64_t red_c[kThreads];
  __shared__ double sums[kThreads / kWave];
  const int tid = threadIdx.x;
  int width = 1;
  while (width < E) width <<= 1;  // <= kThreads
  const int slices = kThreads / width, e = tid % width, slice = tid / width;
  // kept rows: wave 0 adds the parts
  int64_t n = 0;
  for (int i = tid; i < parts; i += kThreads) n += part_n[i];
  red_c[tid] = n;
  __syncthreads();
  for (int d = kThreads / 2; d > 0; d >>= 1) {
    if (tid < d) red_c[tid] += red_c[tid + d];
    __syncthreads();
  }
  n = red_c[0];
  __syncthreads();
  double p = 0.0;
  int64_t c = 0;
  if (e < E) {
#pragma unroll 8
    for (int i = slice; i < parts; i += slices) {
      p += (double)part_p[(int64_t)i * E + e];
      c += part_c[(int64_t)i * E + e];
    }
  }
  red_p[tid] = p;
  red_c[tid] = c;
  __syncthreads();
  double term = 0.0;
  if (slice == 0 && e < E) {
    for (int i = 1; i < slices; ++i) {
      p += red_p[i * width + e];
      c += red_c[i * width + e];
    }
    counts[e] = c;
    term = (double)c * p;
  }
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) term += __shfl_xor(term, m);
  if (tid % kWave == 0) sums[tid / kWave] = term;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kThreads / kWave; ++i) term += sums[i];
    *kept = n;
    *loss = n ? (float)(term * E / ((double)n * (double)n * top_k)) : 0.f;
  }
}

// part_p [parts][E] sums of p, part_c [parts][E] counts, part_n [parts] kept rows.
template <typename T, int G, int C, bool WHOLE>
__global__ __launch_bounds__(kThreads) void balance_fwd_kernel(const T *__restrict__ logits, int64_t ld,
                                                               const uint8_t *__restrict__ mask, int64_t rows, int E,
                                                               int top_k, float *part_p, int32_t *part_c, int32_t *part_n,
                                                               float *loss,
                                                               int64_t *counts, int64_t *kept_rows) {
  constexpr int V = Row<T, G, C, WHOLE>::V, kRows = kThreads / G, kWaves = kThreads / kWave;
  __shared__ float red_p[kWaves][G * C * V];
  __shared__ int32_t chosen[G * C * V];  // whole numbers: the order of adding does not matter
  __shared__ int32_t red_n[kWaves];
  const int lane = lane_id(), t = lane % G, wave = uniform(threadIdx.x / kWave);
  const uint64_t group = (G == kWave ? ~0ull : ((1ull << (G % kWave)) - 1)) << (lane / G * G);
  float sum[C][V] = {};
  int32_t kept = 0;
  for (int e = threadIdx.x; e < G * C * V; e += kThreads) chosen[e] = 0;
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  Row<T, G, C, WHOLE> row;
  uint8_t use = 0, use_next = 0;
  auto load = [&](int64_t i, uint8_t &u) {  // of a row past the end: the last one's, not used
    const int64_t at = i < rows ? i : rows - 1;
    u = mask ? mask[at] : 1;
    row.load(logits + at * ld, E, t);
    if (i >= rows) u = 0;
  };
  if (rows > 0) load(r, use);
  // the whole wave goes round while any of its rows is left
  for (int64_t left = rows - (int64_t)blockIdx.x * kRows - wave * (kWave / G); left > 0; left -= step) {
    row.open(E, t);
    load(r + step, use_next);
    const float m = row.max();
    float p[C][V];
    const bool keep = row.softmax(m, p) != 0.f && use;  // the same in all lanes of a group
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[j][i] += keep ? p[j][i] : 0.f;
    kept += keep && t == 0;
    // The choice: the largest value left, its lowest element, top_k times.
    float best = keep ? m : -INFINITY;
    for (int k = 0; k < top_k; ++k) {
      if (k > 0) {
        best = row.max();
        if (!keep) best = -INFINITY;
      }
      bool open = best > -INFINITY;  // still to be found, in order of the elements
#pragma unroll
      for (int j = 0; j < C; ++j) {
        int first = V;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) first = row.x[j][i] == best ? i : first;
        const uint64_t hits = ballot(open && first < V) & group;
        const bool mine = hits && lane == __builtin_ctzll(hits);
        if (mine) atomicAdd(&chosen[(t + G * j) * V + first], 1);
        if (k + 1 < top_k) {
          const int taken = mine ? first : V;
#pragma unroll
          for (int i = 0; i < V; ++i) row.x[j][i] = i == taken ? -INFINITY : row.x[j][i];
        }
        open = open && !hits;
      }
    }
    use = use_next;
    r += step;
  }
  // Sums over the row groups of the wave, then over the waves.
  auto add = [](auto a, auto b) { return a + b; };
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int m = G; m < kWave; m <<= 1) sum[j][i] += __shfl_xor(sum[j][i], m);
      if (lane < G) red_p[wave][(t + G * j) * V + i] = sum[j][i];
    }
  kept = group_reduce<kWave>(kept, add);
  if (lane == 0) red_n[wave] = kept;
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kThreads) {
    float p = red_p[0][e];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) p += red_p[w][e];
    part_p[(int64_t)blockIdx.x * E + e] = p;
    part_c[(int64_t)blockIdx.x * E + e] = chosen[e];
  }
  if (threadIdx.x == 0) {
    int32_t n = 0;
    for (int w = 0; w < kWaves; ++w) n += red_n[w];
    part_n[blockIdx.x] = n;
  }
  if (gridDim.x > 1) return;
  __threadfence_block();
  __syncthreads();
  join_parts(part_p, part_c, part_n, 1, E, top_k, loss, counts, kept_rows);  // the only part: no launch for it (300 x 8 9.4 us, with one 10.7)
}

__global__ __launch_bounds__(kThreads) void balance_join_kernel(const float *__restrict__ part_p,
                                                                const int32_t *__restrict__ part_c,
                                                                const int32_t *__restrict__ part_n, int parts, int E,
                                                                int top_k, float *__restrict__ loss,
                                                                int64_t *__restrict__ counts,
                                                                int64_t *__restrict__ kept) {
  join_parts(part_p, part_c, part_n, parts, E, top_k, loss, counts, kept);
}

template <typename T, int G, int C, bool WHOLE>
__global__ __launch_bounds__(kBlock) void balance_bwd_kernel(const T *__restrict__ logits, int64_t ld,
                                                             const uint8_t *__restrict__ mask, int64_t rows, int E,
                                                             int top_k, const int64_t *__restrict__ counts,
                                                             const int64_t *__restrict__ kept,
                                                             const float *__restrict__ grad, T *__restrict__ out) {
  constexpr int V = Row<T, G, C, WHOLE>::V, kRows = kBlock / G;
  const int t = lane_id() % G;
  const double n = (double)*kept;
  const float share = n > 0 ? (float)(1.0 / (n * top_k)) : 0.f;
  const float scale = n > 0 ? (float)((double)*grad * E / n) : 0.f;
  float f[C][V];
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = (t + G * j) * V + i;
      f[j][i] = e < E ? (float)counts[e] * share : 0.f;
    }
  Row<T, G, C, WHOLE> row;
  uint8_t use = 0;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  auto load = [&](int64_t i) {
    const int64_t at = i < rows ? i : rows - 1;
    use = mask ? mask[at] : 1;
    row.load(logits + at * ld, E, t);
  };
  load(r);
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += step, r += step) {
    row.open(E, t);
    const uint8_t used = use;
    load(r + step);
    const float m = row.max();
    float p[C][V];
    const bool keep = row.softmax(m, p) != 0.f && used;
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) dot += f[j][i] * p[j][i];
    dot = group_sum<G>(dot);
    if (r >= rows) continue;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int e0 = (t + G * j) * V;
      T d[V];
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = (T)(keep ? scale * p[j][i] * (f[j][i] - dot) : 0.f);
      if (e0 + V <= E) {
        __builtin_memcpy(out + r * E + e0, d, 16);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (e0 + i < E) out[r * E + e0 + i] = d[i];
      }
    }
  }
}

struct Call {
  const void *logits;
  int64_t ld;
  const uint8_t *mask;
  int64_t rows;
  int E, top_k;
  float *loss;
  int64_t *counts, *kept;
  void *ws;
  const float *grad;
  void *out;
};

size_t a256(size_t n) { return (n + 255) & ~(size_t)255; }

// Lanes per row and chunks per lane.
void row_shape(int E, int V, int *G, int *C) {
  const int chunks = (E + V - 1) / V;
  *G = 1;
  while (*G < kWave && *G < chunks) *G *= 2;
  *C = 1;
  while (*G * *C < chunks) *C *= 2;
}

template <typename T, int G, int C, bool WHOLE>
void launch(const Call &c, int parts, hipStream_t s) {
  const T *logits = static_cast<const T *>(c.logits);
  if (c.out) {
    const int64_t blocks = ceil_div(c.rows, kBlock / G);
    hipLaunchKernelGGL((balance_bwd_kernel<T, G, C, WHOLE>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kBlock), 0,
                       s, logits, c.ld, c.mask, c.rows, c.E, c.top_k, c.counts, c.kept, c.grad,
                       static_cast<T *>(c.out));
    return;
  }
  float *part_p = static_cast<float *>(c.ws);
  int32_t *part_c = reinterpret_cast<int32_t *>(part_p + (int64_t)parts * c.E);
  int32_t *part_n = part_c + (int64_t)parts * c.E;
  hipLaunchKernelGGL((balance_fwd_kernel<T, G, C, WHOLE>), dim3(parts), dim3(kThreads), 0, s, logits, c.ld, c.mask, c.rows,
                     c.E, c.top_k, part_p, part_c, part_n, c.loss, c.counts, c.kept);
  if (parts > 1)
    hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(kThreads), 0, s, part_p, part_c, part_n, parts, c.E, c.top_k,
                     c.loss, c.counts, c.kept);
}

int parts_of(int64_t rows, int E, int es) {
  int G, C;
  row_shape(E, 16 / es, &G, &C);
  const int64_t blocks = ceil_div(rows, kThreads / G);
  return (int)(blocks < 1 ? 1 : blocks < kMaxParts ? blocks : kMaxParts);
}

template <typename T>
void launch_type(const Call &c, hipStream_t s) {
  const int parts = parts_of(c.rows, c.E, sizeof(T));
  int G, C;
  row_shape(c.E, 16 / (int)sizeof(T), &G, &C);
#define SFT_BALANCE(g, k) \
  if (G == g && C == k) return c.E % (16 / (int)sizeof(T)) ? launch<T, g, k, false>(c, parts, s) : launch<T, g, k, true>(c, parts, s)
  SFT_BALANCE(1, 1);
  SFT_BALANCE(2, 1);
  SFT_BALANCE(4, 1);
  SFT_BALANCE(8, 1);
  SFT_BALANCE(16, 1);
  SFT_BALANCE(32, 1);
  SFT_BALANCE(64, 1);
  SFT_BALANCE(64, 2);
  if constexpr (sizeof(T) == 4) SFT_BALANCE(64, 4);
#undef SFT_BALANCE
}

int run(int dtype, const Call &c, hipStream_t s, const char *who) {
  ProfScope prof(kProfDenseBalance, s);
  if (dtype == SFT_TYPE_F32) launch_type<float>(c, s);
  else if (dtype == SFT_TYPE_F16) launch_type<f16_t>(c, s);
  else launch_type<bf16_t>(c, s);
  return check_launch(who);
}

}  // namespace

size_t balance_fwd_workspace(int dtype, int64_t rows, int E) {
  const size_t parts = parts_of(rows, E, dtype == SFT_TYPE_F32 ? 4 : 2);
  return a256(parts * (size_t)E * 8 + parts * 4);
}

int balance_fwd(int dtype, const void *logits, int64_t ld, const uint8_t *mask, int64_t rows, int E, int top_k,
                float *loss, int64_t *counts, int64_t *kept, void *ws, hipStream_t s) {
  return run(dtype, Call{logits, ld, mask, rows, E, top_k, loss, counts, kept, ws, nullptr, nullptr}, s,
             "sft_balance_fwd");
}

int balance_bwd(int dtype, const void *logits, int64_t ld, const uint8_t *mask, int64_t rows, int E, int top_k,
                const int64_t *counts, const int64_t *kept, const float *grad, void *out, hipStream_t s) {
  return run(dtype,
             Call{logits, ld, mask, rows, E, top_k, nullptr, const_cast<int64_t *>(counts),
                  const_cast<int64_t *>(kept), nullptr, grad, out},
             s, "sft_balance_bwd");
}

}  // namespace sft
