/* Distillation from a teacher's top logits, forward and backward.
 *
 *   p = softmax over a row's slots of t/T,  q = softmax over the vocabulary of x/T
 *   loss = T^2 sum_k p_k (log p_k - log q[i_k]),  dloss/dx_v = T (q_v - sum_{k: i_k = v} p_k)
 *
 * A slot with a negative index, or with a logit of -inf, has no mass.  A row
 * without mass has loss 0 and gradient 0 whatever its logits hold; an index
 * past the vocabulary makes the row's loss and gradient NaN.
 *
 * Bound by memory.  Without a gradient the logits are read once, with the
 * running maximum and sum of the softmax.  With one, and a loss that is one
 * number, the workgroup that has read a row keeps it in registers and goes on
 * to write its gradient for an upstream gradient of 1, so that the logits are
 * read once for both.  (A second reading from the last-level cache costs as
 * much as one from memory: the way there is what bounds it.)  The backward
 * pass has then nothing left to do, unless the upstream gradient turns out to
 * be another number, and writes the gradient anew.  4096 x 131072 bf16: 200 us for
 * the loss alone, 5.4 TB/s; 411 us with its gradient, 5.2 TB/s.
 */
#include "common.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MOST_SLOTS = 1024;

/* Logits enter the softmax as x c.  In fp32 c is 1/T and the exponential expf.
 * 16-bit logits carry 2^-9 of error themselves, so theirs is the hardware's
 * power of two, with log2(e) in c: one multiply-add and one instruction. */
template <typename T>
struct Unit {
  static constexpr bool TWO = sizeof(T) == 2;
  static __device__ float c(float temperature) { return (TWO ? 1.44269504089f : 1.f) / temperature; }
  static __device__ float exp(float v) { return TWO ? __builtin_amdgcn_exp2f(v) : expf(v); }
  static __device__ float from_natural(float v) { return TWO ? v * 1.44269504089f : v; }
};

/* exp((x - m) c - log_sum) around a row's greatest logit m.  For 16-bit logits
 * of ordinary size in one multiply-add, x c - offset, whose rounding is then
 * below 2^-14 of the result; logits of any size, as of a row masked with the
 * type's lowest value, and those of fp32 are taken from m first. */
template <typename T>
struct Around {
  float m, c, log_sum, offset;
  bool near;
  __device__ Around(float top, float scale, float log = 0.f)
      : m(top), c(scale), log_sum(log), offset(top * scale + log),
        near(Unit<T>::TWO && fabsf(offset) < 1024.f) {}
  __device__ float operator()(float x) const {
    return Unit<T>::exp(near ? fmaf(x, c, -offset) : fmaf(x - m, c, -log_sum));
  }
};

/* The running maximum of x and the sum of exp relative to it.  It starts at
 * the lowest finite number, so that -inf adds nothing and NaN makes the sum
 * NaN without being asked for. */
struct Run {
  float m, s;
};

template <typename T>
__device__ inline Run join(Run a, Run b, float c) {
  float m = fmaxf(a.m, b.m);
  return {m, a.s * Unit<T>::exp((a.m - m) * c) + b.s * Unit<T>::exp((b.m - m) * c)};
}

__device__ inline Run no_run() { return {-3.402823466e38f, 0.f}; }

__device__ inline Run wave_neighbour(Run r, int o) {
  return {__shfl_xor(r.m, o, 64), __shfl_xor(r.s, o, 64)};
}

__device__ inline int64_t index_at(const DistillArgs &p, int64_t row, int k) {
  return p.index_bytes == 8 ? ((const int64_t *)p.index)[row * p.ldi + k]
                            : ((const int32_t *)p.index)[row * p.ldi + k];
}

__device__ inline float any_f(const void *p, int64_t i, int dtype) {
  if (dtype == DT_F32) return ((const float *)p)[i];
  if (dtype == DT_BF16) return to_f<bf16>(((const bf16 *)p)[i]);
  return to_f<fp16>(((const fp16 *)p)[i]);
}

/* A row's state: no slot with mass, a target, an index past the vocabulary. */
constexpr float NO_TARGET = 0.f, TARGET = 1.f, BAD_INDEX = 2.f;
constexpr int SLOT_ROWS = 16; /* rows a workgroup of distill_slots */

/* What the teacher says of a row, a wave each: the slots' masses, and
 * sum_k p_k (T log p_k - (x[i_k] - o)) with o the greatest of the slots' logits,
 * to which the loss adds T times the log of the softmax's sum, above o; it is that
 * sum times T, and finite where x/T need not be.  Where all of
 * the slots' logits are -inf, o is 0: the sum is then +inf, and not NaN.  A class that is
 * named twice is folded into its first slot, so that no two slots write to one
 * place of the gradient.  4096 rows of 64 slots: 18 us, most of it waiting for
 * the logits that the slots name. */
template <typename T>
__global__ __launch_bounds__(1024) void distill_slots(DistillArgs p) {
  extern __shared__ float slots[]; /* of each wave: top masses, top classes */
  __shared__ int targets[SLOT_ROWS];
  int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
  float *sp = slots + (int64_t)wave * 2 * p.top;
  int *si = (int *)(sp + p.top);
  float inv_t = 1.f / p.temperature;
  int64_t block = flat_block();
  if (block * SLOT_ROWS >= p.rows) return;
  for (int q = wave; q < SLOT_ROWS; q += waves) {
    int64_t row = block * SLOT_ROWS + q;
    if (row >= p.rows) {
      if (lane == 0) targets[q] = 0;
      continue;
    }
    const T *x = (const T *)p.x + row * p.ldx;
    float high = -INFINITY;
    bool bad = false, some = false;
    for (int k = lane; k < p.top; k += 64) {
      int64_t i = index_at(p, row, k);
      float t = p.teacher ? any_f(p.teacher, row * p.ldt + k, p.ttype) : 0.f;
      bool here = i >= 0 && t != -INFINITY;
      bad |= i >= p.v;
      some |= here;
      si[k] = here && i < p.v ? (int)i : -1;
      sp[k] = here ? t : -INFINITY;
      high = fmaxf(high, sp[k]);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) high = fmaxf(high, __shfl_xor(high, o, 64));
    bad = __any(bad);
    some = __any(some);
    float state = bad ? BAD_INDEX : some ? TARGET : NO_TARGET;
    /* divided by T behind the difference: logits of any size stay in range */
    float mass = 0.f;
    for (int k = lane; k < p.top; k += 64) mass += expf((sp[k] - high) * inv_t);
    mass = wave_sum(mass);
    float log_mass = logf(mass), loss = 0.f, origin = -INFINITY;
    for (int k = lane; k < p.top; k += 64)
      if (si[k] >= 0) origin = fmaxf(origin, to_f<T>(x[si[k]]));
#pragma unroll
    for (int o = 32; o; o >>= 1) origin = fmaxf(origin, __shfl_xor(origin, o, 64));
    if (origin == -INFINITY) origin = 0.f;
    for (int k = lane; k < p.top; k += 64) {
      float t = (sp[k] - high) * inv_t, log_p = t - log_mass, m = expf(t) / mass;
      if (some && si[k] >= 0 && m != 0.f)
        loss += m * (p.temperature * log_p - (to_f<T>(x[si[k]]) - origin));
      sp[k] = m;
    }
    loss = wave_sum(loss);
    if (lane == 0) {
      targets[q] = state != NO_TARGET;
      p.rows_loss[row] = loss;
      p.state[row] = state;
      p.origin[row] = origin;
    }
    if (!p.slot_p) continue;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); /* other lanes' slots */
    __builtin_amdgcn_wave_barrier();
    for (int k = lane; k < p.top; k += 64) {
      int i = si[k];
      float m = sp[k];
      for (int j = 0; i >= 0 && j < p.top; j++) {
        if (si[j] != i || j == k) continue;
        if (j < k) i = -1; /* folded into slot j */
        else m += sp[j];
      }
      p.slot_p[row * p.top + k] = m;
      p.slot_i[row * p.top + k] = i;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); /* read before the next row's */
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (threadIdx.x || !p.counts) return;
  int n = 0;
  for (int q = 0; q < SLOT_ROWS; q++) n += targets[q];
  p.counts[block] = (float)n;
}

/* Ends a row, one thread's work: its loss from the teacher's part and the
 * softmax's sum.  Gives the natural log of the sum relative to the maximum; of
 * no finite logit at all that is -inf, and what follows from it NaN. */
template <typename T>
__device__ inline float finish(const DistillArgs &p, int64_t row, Run all) {
  float log_sum = logf(all.s), state = p.state[row];
  if (state == BAD_INDEX) log_sum = NAN;
  float above = (all.m - p.origin[row]) + p.temperature * log_sum;
  p.rows_loss[row] = state == NO_TARGET ? 0.f : (p.rows_loss[row] + above) * p.temperature;
  if (p.most) {
    p.most[row] = all.m;
    p.log_sum[row] = log_sum;
  }
  return log_sum;
}

/* A vector as its bits. */
template <typename T>
struct Bits {
  static __device__ u32x4 load(const T *p) {
    return __builtin_bit_cast(u32x4, *(const typename Loose<T>::type *)p);
  }
  static __device__ float get(u32x4 q, int e) {
    return to_f<T>(__builtin_bit_cast(typename Vec<T>::type, q)[e]);
  }
  static __device__ u32x4 nothing() { /* -inf */
    typename Vec<T>::type v;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; e++) v[e] = (T)-INFINITY;
    return __builtin_bit_cast(u32x4, v);
  }
};

/* N vectors' part of the running maximum and sum. */
template <typename T, int N>
__device__ inline Run scan_vecs(const u32x4 *q, float c, Run r) {
  constexpr int V = Vec<T>::N;
  float top = -INFINITY;
#pragma unroll
  for (int u = 0; u < N; u++)
#pragma unroll
    for (int e = 0; e < V; e++) top = fmaxf(top, Bits<T>::get(q[u], e));
  float m = fmaxf(r.m, top), s = r.s * Unit<T>::exp((r.m - m) * c);
  Around<T> part(m, c);
  if (part.near) {
#pragma unroll
    for (int u = 0; u < N; u++)
#pragma unroll
      for (int e = 0; e < V; e++) s += Unit<T>::exp(fmaf(Bits<T>::get(q[u], e), c, -part.offset));
  } else {
#pragma unroll
    for (int u = 0; u < N; u++)
#pragma unroll
      for (int e = 0; e < V; e++) s += Unit<T>::exp((Bits<T>::get(q[u], e) - m) * c);
  }
  return {m, s};
}

/* N vectors TH apart from i on, as far as whole ones go; -inf for the others. */
template <typename T, int TH, int N>
__device__ inline void load_vecs(const T *x, int64_t i, int64_t whole, u32x4 *q) {
#pragma unroll
  for (int u = 0; u < N; u++)
    q[u] = i + u * TH < whole ? Bits<T>::load(x + (i + u * TH) * Vec<T>::N) : Bits<T>::nothing();
}

/* The classes behind the last whole vector, as one vector. */
template <typename T>
__device__ inline u32x4 load_tail(const T *x, int64_t v) {
  constexpr int V = Vec<T>::N;
  typename Vec<T>::type q;
#pragma unroll
  for (int e = 0; e < V; e++) q[e] = v / V * V + e < v ? x[v / V * V + e] : (T)-INFINITY;
  return __builtin_bit_cast(u32x4, q);
}

/* The running maximum and sum over vectors i, i + TH, ... below `to`, of
 * which all but the row's last are whole. */
template <typename T, int TH>
__device__ inline Run scan(const DistillArgs &p, const T *x, int64_t i, int64_t to, float c, Run r) {
  constexpr int U = 4;
  int64_t whole = min(to, p.v / Vec<T>::N);
  u32x4 q[U];
  for (; i < whole; i += U * TH) {
    load_vecs<T, TH, U>(x, i, whole, q);
    r = scan_vecs<T, U>(q, c, r);
  }
  if (threadIdx.x == 0 && whole < to) {
    q[0] = load_tail<T>(x, p.v);
    r = scan_vecs<T, 1>(q, c, r);
  }
  return r;
}

/* Of all TH threads; the first wave has the result. */
template <typename T, int TH>
__device__ inline Run join_all(Run r, float c) {
  __shared__ Run lds[TH / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) r = join<T>(r, wave_neighbour(r, o), c);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = r;
  __syncthreads();
  if (threadIdx.x < 64) {
    r = lds[0];
#pragma unroll
    for (int w = 1; w < TH / 64; w++) r = join<T>(r, lds[w], c);
  }
  return r;
}

template <typename T>
__device__ inline void write_vec(u32x4 q, T *dx, int n, const Around<T> &part, float scale) {
  constexpr int V = Vec<T>::N;
  float v[V];
  if (part.near) { /* asked once a vector: the same for the whole row */
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = fmaf(Bits<T>::get(q, e), part.c, -part.offset);
  } else {
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = fmaf(Bits<T>::get(q, e) - part.m, part.c, -part.log_sum);
  }
#pragma unroll
  for (int e = 0; e < V; e++) v[e] = scale * Unit<T>::exp(v[e]);
  store_vec<T>(dx, n, v);
}

/* The gradient of the same vectors. */
template <typename T, int TH>
__device__ inline void write(const DistillArgs &p, const T *x, T *dx, int64_t i, int64_t to,
                             const Around<T> &part, float scale) {
  constexpr int U = 4, V = Vec<T>::N;
  int64_t whole = min(to, p.v / V);
  u32x4 q[U];
  for (; i < whole; i += U * TH) {
    load_vecs<T, TH, U>(x, i, whole, q);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + u * TH < whole) write_vec<T>(q[u], dx + (i + u * TH) * V, V, part, scale);
  }
  if (threadIdx.x == 0 && whole < to)
    write_vec<T>(load_tail<T>(x, p.v), dx + whole * V, (int)(p.v - whole * V), part, scale);
}

template <typename T, int TH>
__device__ inline void write_zeros(const DistillArgs &p, T *dx, int64_t i, int64_t to) {
  constexpr int V = Vec<T>::N;
  float zero[V] = {};
  for (; i < to; i += TH) store_vec<T>(dx + i * V, (int)min((int64_t)V, p.v - i * V), zero);
}

/* A class that the teacher names: its place in the row, its logit and mass. */
template <typename T>
struct Named {
  int at;
  float x, mass;
  __device__ Named(const DistillArgs &p, int64_t row, const T *logits, int k) : at(-1), x(0.f), mass(0.f) {
    if (k >= p.top) return;
    at = p.slot_i[row * p.top + k];
    mass = p.slot_p[row * p.top + k];
    if (at >= 0) x = to_f<T>(logits[at]);
  }
  /* from the unrounded q; behind a barrier after the row's other stores */
  __device__ void write(T *dx, int64_t from, int64_t to, const Around<T> &part, float scale) const {
    if (at < 0 || at < from || at >= to) return;
    dx[at] = from_f<T>(scale * (part(x) - mass));
  }
};

/* The number of rows with a target, by one wave; all lanes get it. */
__device__ inline float count_rows(const DistillArgs &p) {
  float n = 0.f;
  for (int64_t i = threadIdx.x % 64; i < (p.rows + SLOT_ROWS - 1) / SLOT_ROWS; i += 64)
    n += p.counts[i];
  return wave_sum(n);
}

template <typename T>
__global__ __launch_bounds__(256) void distill_forward(DistillArgs p) {
  constexpr int V = Vec<T>::N;
  int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= p.rows) return;
  const T *x = (const T *)p.x + row * p.ldx;
  int64_t vecs = (p.v + V - 1) / V;
  int64_t from = vecs * blockIdx.x / p.chunks, to = vecs * (blockIdx.x + 1) / p.chunks;
  float c = Unit<T>::c(p.temperature);
  Run r = join_all<T, 256>(scan<T, 256>(p, x, from + threadIdx.x, to, c, no_run()), c);
  if (threadIdx.x) return;
  if (p.chunks == 1) {
    finish<T>(p, row, r);
  } else {
    p.part[(row * p.chunks + blockIdx.x) * 2] = r.m;
    p.part[(row * p.chunks + blockIdx.x) * 2 + 1] = r.s;
  }
}

/* A row's loss and gradient.  The first 16 vectors of each thread stay in
 * registers in between; what a row has beyond them is read again. */
template <typename T, int TH>
__global__ __launch_bounds__(TH) void distill_both(DistillArgs p) {
  constexpr int V = Vec<T>::N, KEEP = 16, U = 4;
  __shared__ float told[3];
  int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= p.rows) return;
  const T *x = (const T *)p.x + row * p.ldx;
  T *dx = (T *)p.dx + row * p.lddx;
  int64_t whole = p.v / V, vecs = (p.v + V - 1) / V, i = threadIdx.x;
  float c = Unit<T>::c(p.temperature);
  u32x4 kept[KEEP];
  load_vecs<T, TH, KEEP>(x, i, whole, kept);
  Named<T> named(p, row, x, threadIdx.x);
  float state = p.state[row], scale = p.temperature * p.scale;
  if (p.reduction == 2 && threadIdx.x < 64) scale /= fmaxf(count_rows(p), 1.f);
  Run r = no_run();
#pragma unroll
  for (int k = 0; k < KEEP; k += U) {
    __builtin_amdgcn_sched_barrier(0); /* four vectors unpacked at a time */
#pragma unroll
    for (int u = 0; u < U; u++) asm volatile("" : "+v"(kept[k + u]));
    r = scan_vecs<T, U>(kept + k, c, r);
  }
  r = join_all<T, TH>(scan<T, TH>(p, x, i + KEEP * TH, vecs, c, r), c);
  if (threadIdx.x == 0) {
    told[0] = r.m;
    told[1] = Unit<T>::from_natural(finish<T>(p, row, r));
    told[2] = scale;
  }
  __syncthreads();
  Around<T> part(told[0], c, told[1]);
  scale = told[2];
  if (state == NO_TARGET) {
    write_zeros<T, TH>(p, dx, i, vecs);
    return;
  }
#pragma unroll
  for (int k = 0; k < KEEP; k++) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(kept[k])); /* unpacked anew, not kept unpacked */
    if (i + k * TH < whole) write_vec<T>(kept[k], dx + (i + k * TH) * V, V, part, scale);
  }
  write<T, TH>(p, x, dx, i + KEEP * TH, vecs, part, scale);
  __threadfence_block();
  __syncthreads();
  named.write(dx, 0, p.v, part, scale);
  for (int k = threadIdx.x + TH; k < p.top; k += TH)
    Named<T>(p, row, x, k).write(dx, 0, p.v, part, scale);
}

/* A wave a row: joins the chunks in their order. */
template <typename T>
__global__ __launch_bounds__(64) void distill_join(DistillArgs p) {
  int64_t row = blockIdx.x;
  float scale = Unit<T>::c(p.temperature);
  Run r = no_run();
  for (int c = threadIdx.x; c < p.chunks; c += 64) {
    const float *q = p.part + (row * p.chunks + c) * 2;
    r = join<T>(r, Run{q[0], q[1]}, scale);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) r = join<T>(r, wave_neighbour(r, o), scale);
  if (threadIdx.x == 0) finish<T>(p, row, r);
}

/* The rows' losses to one. */
__global__ __launch_bounds__(1024) void distill_total(DistillArgs p) {
  __shared__ float lds[16];
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < p.rows; r += 1024) s += p.rows_loss[r];
  s = wave_sum(s);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float n = p.reduction == 2 ? fmaxf(count_rows(p), 1.f) : 1.f;
  if (threadIdx.x) return;
  for (int w = 1; w < 16; w++) s += lds[w];
  *p.loss = s * p.scale / n;
}

/* Pieces of rows in turn; nothing to do where the forward pass has written
 * the gradient for an upstream gradient of 1 and that is what came. */
template <typename T>
__global__ __launch_bounds__(256) void distill_backward(DistillArgs p) {
  constexpr int V = Vec<T>::N;
  if (p.written && *p.grad == 1.f) return;
  __shared__ float told;
  if (threadIdx.x < 64) {
    float n = p.reduction == 2 ? fmaxf(count_rows(p), 1.f) : 1.f;
    if (threadIdx.x == 0) told = n;
  }
  __syncthreads();
  int64_t vecs = (p.v + V - 1) / V;
  float c = Unit<T>::c(p.temperature);
  for (int64_t q = blockIdx.x; q < p.rows * p.chunks; q += gridDim.x) {
    int64_t row = q / p.chunks, piece = q % p.chunks;
    int64_t from = vecs * piece / p.chunks, to = vecs * (piece + 1) / p.chunks;
    const T *x = (const T *)p.x + row * p.ldx;
    T *dx = (T *)p.dx + row * p.lddx;
    if (p.state[row] == NO_TARGET) {
      write_zeros<T, 256>(p, dx, from + threadIdx.x, to);
      continue;
    }
    float scale = p.grad[p.reduction ? 0 : row] * (p.temperature * p.scale / told);
    Around<T> part(p.most[row], c, Unit<T>::from_natural(p.log_sum[row]));
    Named<T> named(p, row, x, threadIdx.x);
    write<T, 256>(p, x, dx, from + threadIdx.x, to, part, scale);
    __threadfence_block();
    __syncthreads();
    named.write(dx, from * V, min(to * V, p.v), part, scale);
    for (int k = threadIdx.x + 256; k < p.top; k += 256)
      Named<T>(p, row, x, k).write(dx, from * V, min(to * V, p.v), part, scale);
  }
}

dim3 rows_grid(int chunks, int64_t rows) {
  return dim3((unsigned)chunks, (unsigned)std::min<int64_t>(rows, 65535),
              (unsigned)((rows + 65534) / 65535));
}

template <typename T>
int run(const DistillArgs &p, hipStream_t s) {
  if (p.grad) {
    int64_t pieces = p.rows * p.chunks;
    /* few workgroups where most often there is nothing to do; else as many as
     * a launch holds */
    int64_t most = p.written ? 4096 : (1 << 24) - 1;
    distill_backward<T><<<(unsigned)std::min(pieces, most), 256, 0, s>>>(p);
    return OPS_LAUNCHED();
  }
  int waves = std::min(16, 65536 / (p.top * 8)); /* as far as 64 KB of LDS go */
  distill_slots<T><<<flat_grid((p.rows + SLOT_ROWS - 1) / SLOT_ROWS), waves * 64,
                     waves * p.top * 8, s>>>(p);
  /* the fewest threads whose registers hold the row */
  dim3 grid = rows_grid(p.chunks, p.rows);
  int64_t bytes = p.v * sizeof(T);
  if (!p.dx) distill_forward<T><<<grid, 256, 0, s>>>(p);
  else if (bytes <= 256 * 256) distill_both<T, 256><<<grid, 256, 0, s>>>(p);
  else if (bytes <= 512 * 256) distill_both<T, 512><<<grid, 512, 0, s>>>(p);
  else distill_both<T, 1024><<<grid, 1024, 0, s>>>(p);
  if (p.chunks > 1) distill_join<T><<<(unsigned)p.rows, 64, 0, s>>>(p);
  if (p.reduction) distill_total<<<1, 1024, 0, s>>>(p);
  return OPS_LAUNCHED();
}

}  // namespace

extern "C" {

/* The number of the capture that a stream takes part in, 0 for none. */
uint64_t vgpu_ops_capture(void *stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError(); /* not the next launch's */
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}

/* Into how many pieces a row is cut.  Forward: one where the rows alone fill
 * the card, else pieces of no less than 4096 classes.  Backward: pieces that
 * workgroups take in turn. */
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
  if (!p.state || !p.most != !p.log_sum) return OPS_BAD_ARG;
  if (p.grad ? !(p.dx && p.most && p.slot_p && p.slot_i)
             : !(p.rows_loss && p.index && p.origin) || !p.slot_p != !p.slot_i || (p.chunks > 1 && (!p.part || p.dx)) ||
                   (p.reduction && !p.loss) || (p.dx && !(p.slot_p && p.slot_i && p.reduction)))
    return OPS_BAD_ARG;
  if (p.reduction == 2 && !p.counts) return OPS_BAD_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (p.dtype == DT_F32) return run<float>(p, s);
  if (p.dtype == DT_BF16) return run<bf16>(p, s);
  if (p.dtype == DT_FP16) return run<fp16>(p, s);
  return OPS_BAD_ARG;
}

}  // extern "C"
