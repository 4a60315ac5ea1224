/* Distillation from a teacher's top logits, forward and backward.
 *
 *   p = softmax over a row's slots of t/T,  q = softmax over the vocabulary of x/T
 *   loss = T^2 sum_k p_k (log p_k - log q[i_k]),  dloss/dx_v = T (q_v - sum_{k: i_k = v} p_k)
 *
 * A slot with a negative index, or with a logit of -inf, has no mass.  A row
 * without mass has loss 0 and gradient 0 whatever its logits hold; an index
 * past the vocabulary makes the row's loss and gradient NaN.
 *
 * Bound by memory: the logits are read once forward with the running maximum
 * and sum of the softmax, and once backward beside the gradient's write.
 */
#include "common.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MOST_SLOTS = 1024;

/* 16-bit logits carry 2^-9 of error themselves: the short exp costs nothing
 * against that and a third of the instructions. */
template <typename T>
__device__ inline float exp_of(float v) {
  if constexpr (sizeof(T) == 4) return expf(v);
  else return __expf(v);
}

/* The running maximum and the sum of exp relative to it. */
struct Run {
  float m, s;
};

template <typename T>
__device__ inline Run join(Run a, Run b) {
  Run r;
  r.m = fmaxf(a.m, b.m);
  if (a.m != a.m || b.m != b.m) r.m = NAN; /* fmaxf drops a NaN */
  r.s = (a.s ? a.s * exp_of<T>(a.m - r.m) : 0.f) + (b.s ? b.s * exp_of<T>(b.m - r.m) : 0.f);
  return r;
}

__device__ inline float any_f(const void *p, int64_t i, int dtype) {
  if (dtype == DT_F32) return ((const float *)p)[i];
  if (dtype == DT_BF16) return to_f<bf16>(((const bf16 *)p)[i]);
  return to_f<fp16>(((const fp16 *)p)[i]);
}

/* One wave: the row's loss from its maximum and sum, and the slots' mass for
 * the backward pass, where a class that is named twice is folded into its
 * first slot so that no two slots write to one place. */
template <typename T>
__device__ void finish(const DistillArgs &p, int64_t row, Run all, float *sp, int *si) {
  int lane = threadIdx.x % 64;
  float inv_t = 1.f / p.temperature;
  const T *x = (const T *)p.x + row * p.ldx;
  /* no finite logit at all: as the formula, NaN */
  float lse = all.m == -INFINITY ? NAN : all.m + logf(all.s);

  float high = -INFINITY;
  bool bad = false, nan = false;
  for (int k = lane; k < p.top; k += 64) {
    int64_t i = p.index_bytes == 8 ? ((const int64_t *)p.index)[row * p.ldi + k]
                                   : ((const int32_t *)p.index)[row * p.ldi + k];
    float t = p.teacher ? any_f(p.teacher, row * p.ldt + k, p.ttype) * inv_t : 0.f;
    bool here = i >= 0 && t != -INFINITY;
    bad |= i >= p.v;
    nan |= here && t != t;
    si[k] = here && i < p.v ? (int)i : -1;
    sp[k] = here ? t : -INFINITY;
    high = fmaxf(high, sp[k]);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) high = fmaxf(high, __shfl_xor(high, o, 64));
  bool some = __any(high != -INFINITY || nan);
  bad = __any(bad);
  if (bad) lse = NAN;
  some |= bad;
  float mass = 0.f;
  for (int k = lane; k < p.top; k += 64) mass += expf(sp[k] - high);
  mass = wave_sum(mass);
  float log_mass = logf(mass), loss = 0.f;
  for (int k = lane; k < p.top; k += 64) {
    float log_p = sp[k] - high - log_mass;
    float q = expf(sp[k] - high) / mass;
    if (some && si[k] >= 0 && q != 0.f)
      loss += q * (log_p - (to_f<T>(x[si[k]]) * inv_t - lse));
    sp[k] = q;
  }
  loss = wave_sum(loss);
  if (bad) loss = NAN;
  if (lane == 0) {
    p.rows_loss[row] = some ? loss * p.temperature * p.temperature : 0.f;
    if (p.lse) p.lse[row] = lse;
  }
  if (!p.slot_p) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); /* other lanes' slots */
  __builtin_amdgcn_wave_barrier();
  for (int k = lane; k < p.top; k += 64) {
    int i = si[k];
    float q = sp[k];
    for (int j = 0; i >= 0 && j < p.top; j++) {
      if (si[j] != i || j == k) continue;
      if (j < k) i = -1; /* folded into slot j */
      else q += sp[j];
    }
    /* a row without mass is told by the first slot, whose mass is -1 */
    p.slot_p[row * p.top + k] = some ? q : -1.f;
    p.slot_i[row * p.top + k] = some ? i : -1;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void distill_forward(DistillArgs p) {
  constexpr int V = Vec<T>::N, U = 4;
  __shared__ Run lds[4];
  __shared__ float sp[MOST_SLOTS];
  __shared__ int si[MOST_SLOTS];
  int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= p.rows) return;
  float inv_t = 1.f / p.temperature;
  const T *x = (const T *)p.x + row * p.ldx;
  int64_t vecs = (p.v + V - 1) / V;
  int64_t from = vecs * blockIdx.x / p.chunks, to = vecs * (blockIdx.x + 1) / p.chunks;
  Run r = {-INFINITY, 0.f};
  for (int64_t i = from + threadIdx.x; i < to; i += 256 * U) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; u++) {
      int64_t at = i + u * 256;
      int n = at < to ? (int)min((int64_t)V, p.v - at * V) : 0;
      load_vec<T>(x + at * V, n, v[u]);
#pragma unroll
      for (int e = 0; e < V; e++) v[u][e] = e < n ? v[u][e] * inv_t : -INFINITY;
    }
    float m = r.m;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        m = fmaxf(m, v[u][e]);
        nan |= v[u][e] != v[u][e];
      }
    if (nan) m = NAN;
    if (m == -INFINITY) continue;
    float s = r.s ? r.s * exp_of<T>(r.m - m) : 0.f;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < V; e++) s += exp_of<T>(v[u][e] - m);
    r.m = m;
    r.s = s;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    Run q;
    q.m = __shfl_xor(r.m, o, 64);
    q.s = __shfl_xor(r.s, o, 64);
    r = join<T>(r, q);
  }
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = r;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  r = join<T>(join<T>(lds[0], lds[1]), join<T>(lds[2], lds[3]));
  if (p.chunks == 1) {
    finish<T>(p, row, r, sp, si);
  } else if (threadIdx.x == 0) {
    p.part[(row * p.chunks + blockIdx.x) * 2] = r.m;
    p.part[(row * p.chunks + blockIdx.x) * 2 + 1] = r.s;
  }
}

/* A wave a row: joins the chunks in their order. */
template <typename T>
__global__ __launch_bounds__(64) void distill_join(DistillArgs p) {
  __shared__ float sp[MOST_SLOTS];
  __shared__ int si[MOST_SLOTS];
  int64_t row = blockIdx.x;
  Run r = {-INFINITY, 0.f};
  for (int c = threadIdx.x; c < p.chunks; c += 64) {
    Run q;
    q.m = p.part[(row * p.chunks + c) * 2];
    q.s = p.part[(row * p.chunks + c) * 2 + 1];
    r = join<T>(r, q);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    Run q;
    q.m = __shfl_xor(r.m, o, 64);
    q.s = __shfl_xor(r.s, o, 64);
    r = join<T>(r, q);
  }
  finish<T>(p, row, r, sp, si);
}

/* The rows' losses to one, and how many rows had a target. */
__global__ __launch_bounds__(1024) void distill_total(DistillArgs p) {
  __shared__ float lds[2][16];
  float s = 0.f, n = 0.f;
  for (int64_t r = threadIdx.x; r < p.rows; r += 1024) {
    s += p.rows_loss[r];
    n += p.slot_p[r * p.top] >= 0.f || p.slot_p[r * p.top] != p.slot_p[r * p.top] ? 1.f : 0.f;
  }
  s = wave_sum(s);
  n = wave_sum(n);
  if (threadIdx.x % 64 == 0) {
    lds[0][threadIdx.x / 64] = s;
    lds[1][threadIdx.x / 64] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; w++) {
    s += lds[0][w];
    n += lds[1][w];
  }
  *p.loss = p.reduction == 2 ? s / fmaxf(n, 1.f) : s;
  *p.count = n;
}

template <typename T>
__global__ __launch_bounds__(256) void distill_backward(DistillArgs p) {
  constexpr int V = Vec<T>::N;
  int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= p.rows) return;
  float inv_t = 1.f / p.temperature;
  const T *x = (const T *)p.x + row * p.ldx;
  T *dx = (T *)p.dx + row * p.lddx;
  const float *slot_p = p.slot_p + row * p.top;
  const int32_t *slot_i = p.slot_i + row * p.top;
  int64_t vecs = (p.v + V - 1) / V;
  int64_t from = vecs * blockIdx.x / p.chunks, to = vecs * (blockIdx.x + 1) / p.chunks;
  bool some = slot_p[0] != -1.f;
  float scale = p.grad[p.reduction ? 0 : row] * p.temperature;
  if (p.reduction == 2) scale /= fmaxf(*p.count, 1.f);
  float lse = p.lse[row];
  for (int64_t i = from + threadIdx.x; i < to; i += 256) {
    int n = (int)min((int64_t)V, p.v - i * V);
    float v[V];
    if (some) load_vec<T>(x + i * V, n, v);
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = some ? scale * exp_of<T>(v[e] * inv_t - lse) : 0.f;
    store_vec<T>(dx + i * V, n, v);
  }
  if (!some) return;
  /* The few classes that the teacher names, from the unrounded q; the
   * barrier orders them behind this workgroup's own stores. */
  __threadfence_block();
  __syncthreads();
  int64_t first = from * V, last = min(to * V, p.v);
  for (int k = threadIdx.x; k < p.top; k += 256) {
    int64_t c = slot_i[k];
    if (c < first || c >= last) continue;
    float q = exp_of<T>(to_f<T>(x[c]) * inv_t - lse);
    dx[c] = from_f<T>(scale * (q - slot_p[k]));
  }
}

dim3 rows_grid(int chunks, int64_t rows) {
  return dim3((unsigned)chunks, (unsigned)std::min<int64_t>(rows, 65535),
              (unsigned)((rows + 65534) / 65535));
}

template <typename T>
int run(const DistillArgs &p, hipStream_t s) {
  if (p.dx) {
    distill_backward<T><<<rows_grid(p.chunks, p.rows), 256, 0, s>>>(p);
    return OPS_LAUNCHED();
  }
  distill_forward<T><<<rows_grid(p.chunks, p.rows), 256, 0, s>>>(p);
  if (p.chunks > 1) distill_join<T><<<(unsigned)p.rows, 64, 0, s>>>(p);
  if (p.reduction) distill_total<<<1, 1024, 0, s>>>(p);
  return OPS_LAUNCHED();
}

}  // namespace

extern "C" {

/* Into how many workgroups a row is cut: one where the rows alone fill the
 * card, else pieces of no less than 4096 classes. */
int32_t vgpu_ops_distill_chunks(int64_t rows, int64_t v, int32_t backward) {
  int64_t want = backward ? std::max<int64_t>((v + 16383) / 16384, 2048 / rows)
                          : (rows >= 1024 ? 1 : 2048 / rows);
  return (int32_t)std::max<int64_t>(1, std::min({want, (v + 4095) / 4096, (int64_t)1024}));
}

int vgpu_ops_distill(const DistillArgs *args, void *stream) {
  const DistillArgs &p = *args;
  if (p.rows <= 0 || p.rows >= (int64_t)1 << 31 || p.v <= 0 || p.v >= (int64_t)1 << 31 ||
      p.top <= 0 || p.top > MOST_SLOTS || p.chunks < 1 || !(p.temperature > 0.f) ||
      (p.index_bytes != 4 && p.index_bytes != 8) || p.reduction < 0 || p.reduction > 2)
    return OPS_BAD_ARG;
  if (p.dx ? !(p.grad && p.lse && p.slot_p && p.slot_i && (p.reduction != 2 || p.count))
           : !p.rows_loss || (p.chunks > 1 && !p.part) ||
                 (p.reduction && !(p.loss && p.count && p.slot_p && p.slot_i)))
    return OPS_BAD_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (p.dtype == DT_F32) return run<float>(p, s);
  if (p.dtype == DT_BF16) return run<bf16>(p, s);
  if (p.dtype == DT_FP16) return run<fp16>(p, s);
  return OPS_BAD_ARG;
}

}  // extern "C"
