/* Shared pieces of the head operators (gfx950 only): element types, vector
 * loads, wave reductions, activations and the C interface's structures.
 *
 * Sums, statistics and accumulators are held in fp32; values are rounded to
 * the tensors' type once, when they are stored.
 */
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

typedef __bf16 bf16;
typedef _Float16 fp16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

enum DType { DT_F32 = 0, DT_BF16 = 1, DT_FP16 = 2 };
enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

/* What the entry points return beside HIP's own codes (which are >= 0). */
enum { OPS_BAD_ARG = -1, OPS_TOO_LONG = -2 };

template <typename T>
struct Vec { /* 16 bytes of T */
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N)));
};

template <typename T>
__device__ inline float to_f(T v) { return (float)v; }
template <typename T>
__device__ inline T from_f(float v) { return (T)v; }

/* A finite v as the nearest finite value of T's range: for what is stored to
 * take a slope at, which has a limit there but is NaN at an infinity. */
template <typename T>
__device__ inline float in_range(float v) {
  if constexpr (sizeof(T) == 4) return v;
  constexpr float MOST = std::is_same_v<T, fp16> ? 65504.f : 0x1.fep127f;
  return fabsf(v) < INFINITY ? fminf(fmaxf(v, -MOST), MOST) : v;
}

/* n <= Vec<T>::N values at p, in one access where all N are there.  Global
 * accesses of 16 bytes need no alignment beyond the element's, so rows of an
 * odd width or start take the same path. */
template <typename T>
struct Loose {
  typedef T type __attribute__((ext_vector_type(Vec<T>::N), aligned(sizeof(T))));
};

template <typename T>
struct Loose4 { /* four of them */
  typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

template <typename T>
__device__ inline void load_vec(const T *p, int n, float *out) {
  constexpr int V = Vec<T>::N;
  if (n >= V) {
    typename Loose<T>::type v = *(const typename Loose<T>::type *)p;
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = to_f<T>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = i < n ? to_f<T>(p[i]) : 0.f;
  }
}

/* The same, unconverted. */
template <typename T>
__device__ inline typename Loose<T>::type load_raw(const T *p, int n) {
  typename Loose<T>::type v = {};
  if (n >= Vec<T>::N) return *(const typename Loose<T>::type *)p;
#pragma unroll
  for (int i = 0; i < Vec<T>::N; i++)
    if (i < n) v[i] = p[i];
  return v;
}

template <typename T>
__device__ inline void store_vec(T *p, int n, const float *in) {
  constexpr int V = Vec<T>::N;
  if (n >= V) {
    typename Loose<T>::type v;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = from_f<T>(in[i]);
    *(typename Loose<T>::type *)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i < n) p[i] = from_f<T>(in[i]);
  }
}

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

/* Phi(z), the normal distribution, and e = exp(-z^2/2), which its slope
 * needs too.  In fp32 by erff.  For 16-bit results by Abramowitz and Stegun's
 * 7.1.26, which is off by 1.5e-7 at most: a fifth of erff's instructions,
 * which in a product's epilogue stand against the matrix cores' time. */
template <typename T>
__device__ inline float normal_cdf(float z, float *e) {
  *e = __expf(-0.5f * z * z);
  if constexpr (sizeof(T) == 4) return 0.5f * (1.f + erff(z * 0.70710678118654752f));
  float x = fabsf(z) * 0.70710678118654752f;
  float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
  float q = t * (0.254829592f +
                 t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  q *= 0.5f * *e;
  return z < 0.f ? q : 1.f - q;
}

template <typename T>
__device__ inline float logistic(float z) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}

/* y = act(z); gelu is z Phi(z). */
template <typename T, int ACT>
__device__ inline float activate(float z) {
  float e;
  if (ACT == ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if (ACT == ACT_GELU) return z * normal_cdf<T>(z, &e);
  if (ACT == ACT_SILU) return z * logistic<T>(z);
  return z;
}

/* Of a whole array, so that its elements' chains run beside each other. */
template <typename T, int ACT, int N>
__device__ inline void activate_each(f32x4 (&v)[N]) {
#pragma unroll
  for (int q = 0; q < N; q++)
#pragma unroll
    for (int e = 0; e < 4; e++) v[q][e] = activate<T, ACT>(v[q][e]);
}

template <typename T, int N>
__device__ inline void activate_all(f32x4 (&v)[N], int act) {
  if (act == ACT_RELU) activate_each<T, ACT_RELU>(v);
  else if (act == ACT_GELU) activate_each<T, ACT_GELU>(v);
  else if (act == ACT_SILU) activate_each<T, ACT_SILU>(v);
}

/* g act'(z).  relu drops g where z is not above 0, an infinite one too. */
template <typename T>
__device__ inline float slope(float g, float z, int act) {
  if (act == ACT_RELU) return z <= 0.f ? 0.f : g;
  if (act == ACT_GELU) {
    float e, cdf = normal_cdf<T>(z, &e);
    return g * (cdf + z * 0.39894228040143268f * e);
  }
  if (act == ACT_SILU) {
    float s = logistic<T>(z);
    return g * (s * (1.f + z * (1.f - s)));
  }
  return g;
}

/* The kernels that a product may run on: tiles of 256 x 256, 128 x 128,
 * 64 x 128 or 32 x 128 of y; few rows; a sum of at most OUTER_K terms. */
enum { PLAN_TILES = 4, PLAN_ROWS = 4, PLAN_OUTER = 5 };
constexpr int OUTER_K = 32, OUTER_ROWS = 8;
constexpr int STEP_BYTES = 64; /* of k per row: what one fragment covers */
constexpr int STEPS = 2;       /* a stage: whole lines of 128 bytes */

/* y[m,n] = act(sum_k a[m,k] b[n,k] + bias[n]) + res[m,n].
 * a_kc: a's element (m,k) is at a[m*lda + k]; otherwise at a[k*lda + m].
 * Likewise b.  Extents are the bytes that may be read from a and b on. */
struct GemmArgs {
  const void *a, *b;
  int64_t lda, ldb, a_extent, b_extent;
  int64_t m, n, k;
  const void *bias, *res;
  int64_t ldr;
  void *y;
  int64_t ldy;
  void *z; /* the value before the activation, where backward needs it; finite where
              the sum is */
  int64_t ldz;
  float *work; /* splits x m x n partial sums */
  int32_t dtype, a_kc, b_kc, act;
  int32_t plan, splits;
};

/* dz = dy act'(z) into rows of lddz elements with zeros behind n, and dbias,
 * the sums of dz's columns, by way of sums over runs of rows in part [parts, n]
 * where there is more than one run. */
struct SlopeArgs {
  const void *dy, *z;
  void *dz, *dbias;
  float *part;
  int64_t lddy, ldz, lddz, m, n;
  int32_t dtype, act, parts;
};

int launch_gemm(const GemmArgs &p, hipStream_t s);
int launch_slope(const SlopeArgs &p, hipStream_t s);
int launch_repack(const void *src, int64_t rs, int64_t cs, int64_t rows, int64_t cols, void *dst,
                  int64_t ld, int size, hipStream_t s);

/* y = act(x W^T + bias) + res, x [m,k] and W [n,k] of any strides (in
 * elements), y and z [m,n] contiguous.  With dy, the backward pass instead: z
 * is then what the slope is taken at, and dx [m,k], dw [n,k], db [n] what is
 * written of the gradients, contiguous; x is wanted for dw alone, W for dx. */
struct LinearArgs {
  const void *x, *w, *bias, *res, *dy;
  void *y, *z, *dx, *dw, *db, *work;
  int64_t m, n, k, xs0, xs1, ws0, ws1, ldr, lddy, work_bytes;
  int32_t dtype, act;
};

/* Layer norm of each (row, group): x [rows, groups*d].  mean and rstd hold
 * rows*groups values; with more than one part, part holds 2 x parts x groups*d
 * partial sums of the weight's and bias's gradients. */
struct NormArgs {
  const void *x, *weight, *bias, *dy;
  void *y, *dx, *dweight, *dbias;
  float *mean, *rstd, *part;
  int64_t ldx, ldy, lddy, lddx, rows, groups, d;
  int32_t dtype, wtype;
  int32_t parts;
  float eps;
};

/* Distillation from a teacher's top logits.  rows_loss, state, origin, most
 * and log_sum hold one value a row, slot_p and slot_i `top` values a row, part
 * 2 x chunks a row; counts holds, for each 16 rows, how many of them have a
 * target. */
struct DistillArgs {
  const void *x, *index, *teacher;
  void *dx;
  const float *grad; /* of the loss: one value, or one a row */
  float *rows_loss, *state, *origin, *most, *log_sum, *slot_p, *loss, *counts;
  int32_t *slot_i;
  float *part;
  int64_t ldx, lddx, ldi, ldt, rows, v;
  int32_t dtype, ttype, index_bytes, top;
  int32_t chunks, reduction; /* 0 none, 1 sum, 2 mean */
  int32_t written;           /* dx holds the gradient for an upstream one of 1 */
  float temperature, scale;  /* scale: of the loss that is one number */
};

/* Column sums of part [parts, width] in a fixed order: 16 runs of rows a
 * column, joined through LDS.  1024 threads for 64 columns. */
template <typename W>
__device__ inline void join_columns(const float *part, int64_t parts, int64_t width, W *out) {
  __shared__ float lds[16][64];
  int64_t col = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
  int run = threadIdx.x / 64;
  float s = 0.f;
  if (col < width)
    for (int64_t r = run; r < parts; r += 16) s += part[r * width + col];
  lds[run][threadIdx.x % 64] = s;
  __syncthreads();
  if (run || col >= width) return;
  for (int r = 1; r < 16; r++) s += lds[r][threadIdx.x];
  if (out) out[col] = from_f<W>(s);
}

#define OPS_LAUNCHED() ((int)hipGetLastError())

/* A launch holds fewer than 2^32 threads along an axis: `blocks` of at most
 * 1024 threads in rows of up to 2^20 along x and z, `y` along y.  flat_block() is
 * a workgroup's number, which may pass the last. */
constexpr int64_t GRID_ROW = 1 << 20;
inline dim3 flat_grid(int64_t blocks, int64_t y = 1) {
  return dim3((unsigned)(blocks < GRID_ROW ? blocks : GRID_ROW), (unsigned)y,
              (unsigned)((blocks + GRID_ROW - 1) / GRID_ROW));
}
__device__ inline int64_t flat_block() {
  return (int64_t)blockIdx.z * GRID_ROW + blockIdx.x;
}
