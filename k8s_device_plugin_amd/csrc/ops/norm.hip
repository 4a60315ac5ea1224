/* Layer norm over groups of d neighbouring values, forward and backward.
 *
 *   y = h w + b,  h = (x - mean) rstd        (per row and group)
 *   dx = rstd (a - mean(a) - h mean(a h)),   a = dy w
 *   dw = sum over rows of dy h,  db = sum over rows of dy
 *
 * Bound by memory: a row is read once and stays in registers between its
 * statistics and its result; the variance is taken around the mean, in fp32.
 * 16384 x 8192 bf16: forward 110 us, 4.9 TB/s; backward 158 us, 5.1 TB/s, and 6
 * to join the weight's partial sums.
 */
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

/* The sum over the TH threads of a row; every one of them gets it.  Waves
 * join through LDS, in their order; TH = 64 is one wave. */
template <int TH, int COUNT>
__device__ inline void row_sum(float (&v)[COUNT], float *lds) {
#pragma unroll
  for (int c = 0; c < COUNT; c++) v[c] = wave_sum(v[c]);
  if constexpr (TH > 64) {
    constexpr int WAVES = TH / 64;
    __syncthreads(); /* the last use of lds is over */
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int c = 0; c < COUNT; c++) lds[c * WAVES + threadIdx.x / 64] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < COUNT; c++) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) s += lds[c * WAVES + w];
      v[c] = s;
    }
  }
}

/* Rows of up to 64 lanes' worth take a wave each, four waves a workgroup. */
template <int TH>
constexpr int rows_at_once() { return TH == 64 ? 4 : 1; }
template <int TH>
constexpr int block_of() { return TH == 64 ? 256 : TH; }

template <typename T, typename W, int TH, int VECS>
__global__ __launch_bounds__(block_of<TH>()) void norm_forward(NormArgs p) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[TH / 64];
  int lane = threadIdx.x % TH;
  int64_t row = flat_block() * rows_at_once<TH>() + threadIdx.x / TH;
  if (row >= p.rows) return; /* a whole wave where TH is 64, else all of them */
  int64_t group = blockIdx.y, d = p.d;
  const T *x = (const T *)p.x + row * p.ldx + group * d;
  float v[VECS][V];
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    int64_t at = (int64_t)(i * TH + lane) * V;
    int n = (int)min((int64_t)V, d - at);
    load_vec<T>(x + at, n, v[i]);
#pragma unroll
    for (int e = 0; e < V; e++) s[0] += v[i][e];
  }
  row_sum<TH>(s, lds);
  float mean = s[0] / d;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    int64_t at = (int64_t)(i * TH + lane) * V;
#pragma unroll
    for (int e = 0; e < V; e++) {
      v[i][e] = at + e < d ? v[i][e] - mean : 0.f;
      s[0] += v[i][e] * v[i][e];
    }
  }
  row_sum<TH>(s, lds);
  float rstd = 1.f / sqrtf(s[0] / d + p.eps);
  if (lane == 0 && p.mean) {
    p.mean[row * p.groups + group] = mean;
    p.rstd[row * p.groups + group] = rstd;
  }
  const W *w = (const W *)p.weight + group * d, *b = (const W *)p.bias + group * d;
  T *y = (T *)p.y + row * p.ldy + group * d;
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    int64_t at = (int64_t)(i * TH + lane) * V;
    int n = (int)min((int64_t)V, d - at);
    if (n <= 0) continue;
    float o[V];
#pragma unroll
    for (int e = 0; e < V; e++) o[e] = v[i][e] * rstd;
    if (p.weight) {
      float t[V];
      constexpr int VW = Vec<W>::N;
#pragma unroll
      for (int h = 0; h < V; h += VW) load_vec<W>(w + at + h, n - h, t + h);
#pragma unroll
      for (int e = 0; e < V; e++) o[e] *= t[e];
    }
    if (p.bias) {
      float t[V];
      constexpr int VW = Vec<W>::N;
#pragma unroll
      for (int h = 0; h < V; h += VW) load_vec<W>(b + at + h, n - h, t + h);
#pragma unroll
      for (int e = 0; e < V; e++) o[e] += t[e];
    }
    store_vec<T>(y + at, n, o);
  }
}

/* Each workgroup takes every parts-th row, or four, keeps its columns' sums of
 * dy h and dy in registers and writes them once, so x and dy are read a single
 * time for all three gradients.  The next row is asked for before this one's
 * sums are taken.  A single workgroup writes the gradients themselves. */
template <typename T, typename W, int TH, int VECS>
__global__ __launch_bounds__(block_of<TH>()) void norm_backward(NormArgs p) {
  constexpr int V = Vec<T>::N, R = rows_at_once<TH>(), WAVES = TH / 64;
  __shared__ float lds[2][2 * WAVES];
  __shared__ float waves[TH == 64 ? R - 1 : 1][TH == 64 ? 64 * VECS * V : 1];
  int lane = threadIdx.x % TH;
  int64_t group = blockIdx.y, d = p.d;
  const W *w = (const W *)p.weight + group * d;
  typedef typename Loose<T>::type raw;
  constexpr int VW = Vec<W>::N;
  raw rx[VECS], rg[VECS];
  typename Loose<W>::type rw[VECS][V / VW];
  /* the weight stays in registers: loads end in their order, so one inside
   * the loop would wait for the next row's */
#pragma unroll
  for (int i = 0; i < VECS; i++)
#pragma unroll
    for (int c = 0; c < V; c += VW) {
      int64_t at = (int64_t)(i * TH + lane) * V + c;
      if (p.weight) rw[i][c / VW] = load_raw<W>(w + at, (int)min((int64_t)VW, d - at));
      else
#pragma unroll
        for (int e = 0; e < VW; e++) rw[i][c / VW][e] = (W)1.f;
    }
  float row_mean = 0.f, row_rstd = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= p.rows) return;
    const T *x = (const T *)p.x + row * p.ldx + group * d;
    const T *dy = (const T *)p.dy + row * p.lddy + group * d;
    row_mean = p.mean[row * p.groups + group];
    row_rstd = p.rstd[row * p.groups + group];
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      int64_t at = (int64_t)(i * TH + lane) * V;
      int n = (int)min((int64_t)V, d - at);
      rx[i] = load_raw<T>(x + at, n);
      rg[i] = load_raw<T>(dy + at, n);
    }
  };
  float dw[VECS][V] = {}, db[VECS][V] = {};
  int64_t step = (int64_t)p.parts * R;
  int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / TH;
  fetch(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    float mean = row_mean, rstd = row_rstd;
    float h[VECS][V], a[VECS][V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VECS; i++)
#pragma unroll
      for (int e = 0; e < V; e++) {
        h[i][e] = to_f<T>(rx[i][e]);
        a[i][e] = to_f<T>(rg[i][e]);
      }
    fetch(row + step);
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      int64_t at = (int64_t)(i * TH + lane) * V;
      int n = (int)min((int64_t)V, d - at);
#pragma unroll
      for (int e = 0; e < V; e++) {
        h[i][e] = e < n ? (h[i][e] - mean) * rstd : 0.f;
        dw[i][e] += a[i][e] * h[i][e];
        db[i][e] += a[i][e];
        a[i][e] *= to_f<W>(rw[i][e / VW][e % VW]);
        s[0] += a[i][e];
        s[1] += a[i][e] * h[i][e];
      }
    }
    if (!p.dx) continue; /* the same for all threads */
    /* the row before used the other half of lds, and every wave has passed
     * the barrier since */
#pragma unroll
    for (int c = 0; c < 2; c++) s[c] = wave_sum(s[c]);
    if constexpr (WAVES > 1) {
      if (threadIdx.x % 64 == 0)
#pragma unroll
        for (int c = 0; c < 2; c++) lds[turn][c * WAVES + threadIdx.x / 64] = s[c];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 2; c++) {
        s[c] = 0.f;
#pragma unroll
        for (int q = 0; q < WAVES; q++) s[c] += lds[turn][c * WAVES + q];
      }
    }
    float ma = s[0] / d, mah = s[1] / d;
    T *dx = (T *)p.dx + row * p.lddx + group * d;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      int64_t at = (int64_t)(i * TH + lane) * V;
      int n = (int)min((int64_t)V, d - at);
      float o[V];
#pragma unroll
      for (int e = 0; e < V; e++) o[e] = rstd * (a[i][e] - ma - h[i][e] * mah);
      store_vec<T>(dx + at, n, o);
    }
  }
  if (!p.dweight && !p.dbias) return;
  if constexpr (TH == 64) { /* the four waves' sums, in their order */
    int wave = threadIdx.x / 64;
    auto add = [&](float(&v)[VECS][V]) {
      __syncthreads();
      if (wave)
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
          for (int e = 0; e < V; e++) waves[wave - 1][(i * V + e) * 64 + lane] = v[i][e];
      __syncthreads();
      if (!wave)
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
          for (int e = 0; e < V; e++)
            for (int q = 0; q < R - 1; q++) v[i][e] += waves[q][(i * V + e) * 64 + lane];
    };
    add(dw);
    add(db);
    if (wave) return;
  }
  auto write = [&](auto *out, float(&v)[VECS][V]) {
    typedef std::remove_pointer_t<decltype(out)> D;
    constexpr int VD = Vec<D>::N;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      int64_t at = (int64_t)(i * TH + lane) * V;
      int n = (int)min((int64_t)V, d - at);
#pragma unroll
      for (int c = 0; c < V; c += VD) store_vec<D>(out + group * d + at + c, n - c, v[i] + c);
    }
  };
  if (p.parts == 1) {
    if (p.dweight) write((W *)p.dweight, dw);
    if (p.dbias) write((W *)p.dbias, db);
  } else {
    int64_t width = p.groups * d;
    write(p.part + blockIdx.x * width, dw);
    write(p.part + (p.parts + blockIdx.x) * width, db);
  }
}

/* blockIdx.y: 0 the weight, 1 the bias. */
template <typename W>
__global__ __launch_bounds__(1024) void norm_join(NormArgs p) {
  int64_t width = p.groups * p.d;
  join_columns<W>(p.part + blockIdx.y * p.parts * width, p.parts, width,
                  (W *)(blockIdx.y ? p.dbias : p.dweight));
}

template <typename T, typename W, int TH, int VALUES>
void launch(const NormArgs &p, hipStream_t s) {
  constexpr int VECS = VALUES / Vec<T>::N;
  constexpr int R = rows_at_once<TH>();
  if (p.dy)
    norm_backward<T, W, TH, VECS>
        <<<dim3(p.parts, (unsigned)p.groups), block_of<TH>(), 0, s>>>(p);
  else
    norm_forward<T, W, TH, VECS>
        <<<flat_grid((p.rows + R - 1) / R, p.groups), block_of<TH>(), 0, s>>>(p);
}

/* The fewest threads whose registers hold the row, with 16 values each or (of
 * one wave's rows, and the widest) 32.  16384 x 8192 bf16 backward: 165 us with
 * 512 threads of 16, 170 with 256 of 32; forward 109 and 114. */
template <typename T, typename W>
void dispatch(const NormArgs &p, hipStream_t s) {
  if (p.d <= 64 * 8) launch<T, W, 64, 8>(p, s);
  else if (p.d <= 64 * 16) launch<T, W, 64, 16>(p, s);
  else if (p.d <= 64 * 32) launch<T, W, 64, 32>(p, s);
  else if (p.d <= 256 * 16) launch<T, W, 256, 16>(p, s);
  else if (p.d <= 512 * 16) launch<T, W, 512, 16>(p, s);
  else if (p.d <= 1024 * 16) launch<T, W, 1024, 16>(p, s);
  else launch<T, W, 1024, 32>(p, s);
  if (p.dy && p.parts > 1 && (p.dweight || p.dbias)) {
    int64_t width = p.groups * p.d;
    norm_join<W><<<dim3((unsigned)((width + 63) / 64), 2), 1024, 0, s>>>(p);
  }
}

template <typename T>
int run(const NormArgs &p, hipStream_t s) {
  if (p.wtype == DT_F32) dispatch<T, float>(p, s);
  else if (p.wtype == p.dtype) dispatch<T, T>(p, s);
  else return OPS_BAD_ARG;
  return OPS_LAUNCHED();
}

}  // namespace

extern "C" {

/* How many workgroups share the rows: one a CU, since each one's partial sums
 * are written and read again (16384 x 8192 bf16: 165 us with 256, 181 with 512,
 * 195 with 1024); four rows in a row's place each, so that up to four (or, of
 * short rows, sixteen) rows need no partial sums. */
int32_t vgpu_ops_norm_parts(int64_t rows, int64_t groups, int64_t d) {
  int64_t at_once = d <= 64 * 32 ? 4 : 1, share = 4 * at_once;
  int64_t most = std::max<int64_t>(1, 256 / groups);
  return (int32_t)std::max<int64_t>(1, std::min((rows + share - 1) / share, most));
}

int vgpu_ops_norm(const NormArgs *args, void *stream) {
  const NormArgs &p = *args;
  if (p.rows <= 0 || p.rows >= (int64_t)1 << 31 || p.groups <= 0 || p.groups > 65535 || p.d <= 0 ||
      p.d > 1024 * 32 ||
      (p.dy ? p.parts < 1 || (p.parts > 1 && (p.dweight || p.dbias) && !p.part) : !p.y))
    return OPS_BAD_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (p.dtype == DT_F32) return run<float>(p, s);
  if (p.dtype == DT_BF16) return run<bf16>(p, s);
  if (p.dtype == DT_FP16) return run<fp16>(p, s);
  return OPS_BAD_ARG;
}

}  // extern "C"
