/* The linear layer's entry points: how operands are laid out for the kernels
 * of gemm.hip, which of them runs, and the workspace that this takes.  Host
 * code only. */
#include "common.h"

#include <algorithm>

namespace {

constexpr int64_t LONGEST = 1 << 23; /* bytes of a row: tiles use 32-bit offsets */

int64_t tiles_of(int plan, int64_t m, int64_t n) {
  static const int side[4][2] = {{256, 256}, {128, 128}, {64, 128}, {32, 128}};
  return ((m + side[plan][0] - 1) / side[plan][0]) * ((n + side[plan][1] - 1) / side[plan][1]);
}

/* A launch holds fewer than 2^32 threads along an axis. */
constexpr int64_t MOST_TILES = (1 << 24) - 1;
constexpr int64_t MOST_STRIPS = (1 << 23) - 1; /* of 512 threads */

/* What a product takes in us with tiles of one kind, k in `splits` parts: in
 * turns of as many workgroups as the card holds (256 of the largest tile, 512
 * of the others; a last turn of up to 256 has a CU each), each of so much a
 * stage and so much for itself.  A split writes and reads partial sums and
 * costs a launch.  The numbers are a least-squares fit to 2700 timings (m 40 to
 * 8192, n 1000 to 11000, k 1024 to 14336, all layouts); what it picks takes
 * 3.3% more than the best of them on average in 16 bits, 0.2% in fp32. */
double tile_time(int plan, int64_t splits, int64_t m, int64_t n, int64_t k, int size) {
  struct Cost {
    double stage, own; /* us */
  };
  static const Cost full[2][4] = {{{1.33, 7.9}, {0.86, 5.0}, {0.595, 3.7}, {0.417, 4.2}},
                                  {{7.37, 5.9}, {3.71, 3.3}, {1.975, 2.3}, {1.096, 2.4}}};
  static const Cost half[2][4] = {{{1.33, 7.9}, {0.56, 3.7}, {0.378, 3.1}, {0.321, 2.6}},
                                  {{7.37, 5.9}, {1.99, 3.1}, {1.110, 1.2}, {0.657, 0.0}}};
  int64_t tiles = tiles_of(plan, m, n);
  int64_t stages = (k * size + STEPS * STEP_BYTES - 1) / (STEPS * STEP_BYTES);
  int64_t each = (stages + splits - 1) / splits, slots = plan == 0 ? 256 : 512;
  int64_t turns = tiles * splits / slots, rest = tiles * splits % slots;
  const Cost &f = full[size == 4][plan], &h = half[size == 4][plan];
  double time = turns * (each * f.stage + f.own);
  if (rest > 256) time += each * f.stage + f.own;
  else if (rest) time += each * h.stage + h.own;
  if (splits > 1) time += (size == 4 ? 9. : 5.8) + m * n * splits * 0.9e-6;
  return time;
}

double best_tiles(int64_t m, int64_t n, int64_t k, int size, int32_t *plan, int32_t *splits) {
  static const int parts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
  double best = 1e30;
  for (int q = 0; q < 4; q++)
    for (int s : parts) {
      /* partial sums of no more than 1.5 GB */
      if (s > 1 && ((double)m * n * s * 4 > 1.5e9 || k * size < s * STEPS * STEP_BYTES)) break;
      double time = tile_time(q, s, m, n, k, size);
      if (time < best && (q == 0 || tiles_of(q, m, n) <= MOST_TILES)) {
        best = time;
        *plan = q;
        *splits = s;
      }
    }
  return best;
}

/* Which kernel, over how many parts k is split, and how many of the rows go
 * there: the others, a last band of up to 32, may go to a launch of their own
 * rather than to a row of tiles. */
struct Plan {
  int32_t plan, splits;
  int64_t rows;
};

Plan choose(int64_t m, int64_t n, int64_t k, int size, bool a_kc, bool b_kc, bool bare, bool odd) {
  Plan p = {0, 1, m};
  if (k <= OUTER_K && !a_kc && !b_kc && bare && m <= 65535 * 4 * OUTER_ROWS) {
    p.plan = PLAN_OUTER;
    return p;
  }
  /* Up to 16 rows stream b past the matrix cores while it is small, and beyond
   * that where a row of it is long enough for its workgroup and a's few rows
   * cost nothing beside it; tiles take the others.  us, rows and tiles, weights
   * out of the cache: 1 x 4096 -> 4096 bf16 10.8 and 15.8; 1 x 50000 -> 4096
   * bf16 71 and 81; 16 of them 115 and 85; 1 x 4096 -> 50000 bf16 90 and 82.
   * With k strided in b, 8 rows fp32: 14336 -> 4096 48 and 53, 4096 -> 50000
   * 166 and 158.  16-bit rows that start on 2 bytes only the former reads where
   * they lie; for the tiles they would be laid out anew: 8 x 20001 -> 8001 127 us
   * and 193. */
  bool rows = odd || (b_kc ? n * k * size <= 1 << 26 || (m <= 4 && k * size >= 1 << 14) : n < 1 << 15);
  if (a_kc && m <= 16 && rows) {
    p.plan = PLAN_ROWS;
    int64_t steps = (k * size + STEP_BYTES - 1) / STEP_BYTES;
    int64_t strip = b_kc ? 16 : 256 / size, strips = (n + strip - 1) / strip;
    p.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({256 / strips, steps / 64, 64}));
    return p;
  }
  double time = best_tiles(m, n, k, size, &p.plan, &p.splits);
  int64_t band = m % 256;
  if (m > 256 && band >= 1 && band <= 32) {
    Plan q = p;
    q.rows = m - band;
    /* the band reads b once more, at 4.5 TB/s */
    if (best_tiles(q.rows, n, k, size, &q.plan, &q.splits) + 6. + (double)n * k * size / 4.5e6 < time)
      return q;
  }
  return p;
}

/* choose() takes a microsecond or two; a program asks for few sizes. */
Plan planned(int64_t m, int64_t n, int64_t k, int size, bool a_kc, bool b_kc, bool bare, bool odd) {
  struct Entry {
    int64_t m, n, k;
    int form;
    Plan plan;
  };
  static thread_local Entry known[64];
  int form = 16 | size << 5 | a_kc | b_kc << 1 | bare << 2 | odd << 3;
  Entry &e = known[(uint64_t)(m * 1000003 + n * 10007 + k * 101 + form) % 64];
  if (e.m != m || e.n != n || e.k != k || e.form != form)
    e = {m, n, k, form, choose(m, n, k, size, a_kc, b_kc, bare, odd)};
  return e.plan;
}

struct Matrix { /* [rows, k]; strides in elements */
  const void *p;
  int64_t rows, k, s0, s1;
};

struct Operand { /* as the kernels read it */
  const void *p;
  int64_t ld, extent, k;
  bool kc, odd = false; /* rows start on 2 bytes */
};

/* One call: run for good, or (without a workspace) only to see how much of it
 * the call takes. */
struct Call {
  char *base;
  int size;
  int32_t dtype;
  hipStream_t stream;
  int64_t used = 0;
  int code = 0;

  void *take(int64_t bytes) {
    int64_t at = used;
    used += (bytes + 255) / 256 * 256;
    return (void *)((uintptr_t)base + at);
  }
  template <typename F>
  void launch(F f) {
    if (base && code == 0) code = f();
  }
  int64_t padded(int64_t n) const { return (n * size + 15) / 16 * 16 / size; }

  static int64_t dwords(int64_t bytes) { return (bytes + 3) / 4 * 4; }

  /* Loads take dwords, and are cut off at the extent dword by dword, so rows
   * that do not start on 4 bytes are laid out anew; so is a matrix that is
   * contiguous along neither axis, or not along k where any_axis is false.
   * Where k is too long for a row (a weight's gradient over many tokens), the
   * other axis is taken in any case.  The kernel for few rows reads b's wherever
   * they start, where a launch of it holds them. */
  Operand prepare(Matrix t, bool any_axis, bool anywhere = false) {
    bool fits = padded(t.k) * size <= LONGEST;
    if (!fits) any_axis = true;
    bool aligned = (uintptr_t)t.p % 4 == 0;
    if (t.rows == 1 && t.s1 == 1) t.s0 = fits ? dwords(t.k * size) / size : 1;
    bool odd = !aligned || t.s0 * size % 4;
    if (t.s1 == 1 && (anywhere || !odd) && t.s0 * size <= LONGEST && fits)
      return {t.p, t.s0, dwords(((t.rows - 1) * t.s0 + t.k) * size), t.k, true, odd};
    if (aligned && any_axis && t.s0 == 1 && t.s1 >= t.rows && t.s1 * size % 4 == 0 &&
        t.s1 * size <= LONGEST)
      return {t.p, t.s1, dwords(((t.k - 1) * t.s1 + t.rows) * size), t.k, false};
    bool along = any_axis && (!fits || (t.s0 == 1 && t.s1 != 1)) && padded(t.rows) * size <= LONGEST;
    int64_t rows = along ? t.k : t.rows, cols = along ? t.rows : t.k, ld = padded(cols);
    if (ld * size > LONGEST) code = OPS_TOO_LONG;
    void *to = take(rows * ld * size);
    launch([&] {
      return launch_repack(t.p, along ? t.s1 : t.s0, along ? t.s0 : t.s1, rows, cols, to, ld, size,
                           stream);
    });
    return {to, ld, rows * ld * size, t.k, !along};
  }

  /* out [m,n] = a b^T; `out` says where to and with what epilogue. */
  void product(const Operand &a, const Operand &b, int64_t m, int64_t n, GemmArgs out) {
    int64_t k = a.k;
    bool bare = !out.bias && !out.res && !out.z && out.act == ACT_NONE;
    Plan p = planned(m, n, k, size, a.kc, b.kc, bare, b.odd);
    if (p.plan == 0 && tiles_of(0, p.rows, n) > MOST_TILES) code = OPS_TOO_LONG;
    if (p.rows < m) {
      auto below = [&](const void *q, int64_t ld) {
        return q ? (void *)((uintptr_t)q + p.rows * ld * size) : nullptr;
      };
      GemmArgs rest = out;
      rest.res = below(out.res, out.ldr);
      rest.y = below(out.y, out.ldy);
      rest.z = below(out.z, out.ldz);
      Operand band = a;
      if (a.kc) {
        band.p = below(a.p, a.ld);
        band.extent -= p.rows * a.ld * size;
      } else {
        band = prepare({below(a.p, 1), m - p.rows, a.k, 1, a.ld}, false);
      }
      product(band, b, m - p.rows, n, rest);
    }
    out.a = a.p, out.lda = a.ld, out.a_extent = a.extent, out.a_kc = a.kc;
    out.b = b.p, out.ldb = b.ld, out.b_extent = b.extent, out.b_kc = b.kc;
    out.m = p.rows, out.n = n, out.k = k, out.dtype = dtype;
    out.plan = p.plan, out.splits = p.splits;
    if (p.splits > 1) out.work = (float *)take(p.splits * p.rows * n * 4);
    launch([&] { return launch_gemm(out, stream); });
  }
  void product(const Matrix &a, const Matrix &b, const GemmArgs &out) {
    /* few rows are read with k contiguous, but for short sums */
    Operand p = prepare(a, a.rows > 16 || a.k <= OUTER_K);
    bool anywhere = a.rows <= 16 && p.kc && b.rows <= MOST_STRIPS * 16;
    product(p, prepare(b, true, anywhere), a.rows, b.rows, out);
  }

  void forward(const LinearArgs &p) {
    GemmArgs out = {};
    out.bias = p.bias, out.res = p.res, out.ldr = p.ldr, out.act = p.act;
    out.y = p.y, out.z = p.z, out.ldy = out.ldz = p.n;
    product({p.x, p.m, p.k, p.xs0, p.xs1}, {p.w, p.n, p.k, p.ws0, p.ws1}, out);
  }

  void backward(const LinearArgs &p) {
    Matrix dz = {p.dy, p.m, p.n, p.lddy, 1};
    /* rows of dy that the loads do not allow are copied along with the slope */
    bool copy = (p.dx || p.dw) && (p.act != ACT_NONE || p.lddy * size % 4 || (uintptr_t)p.dy % 4);
    if (p.db || copy) {
      SlopeArgs s = {};
      s.dy = p.dy, s.z = p.z, s.lddy = p.lddy, s.ldz = p.n, s.m = p.m, s.n = p.n;
      s.dtype = dtype, s.act = p.act, s.lddz = padded(p.n), s.dbias = p.db;
      /* runs of rows for the columns' sums: about four workgroups a CU, and at
       * least 8 rows each; up to 16 rows need no second launch */
      int64_t blocks = (s.lddz * size + 1023) / 1024;
      s.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>((p.m + 7) / 8, 1024 / blocks));
      if (p.m <= 16) s.parts = 1;
      if (copy) s.dz = take(p.m * s.lddz * size);
      if (p.db && s.parts > 1) s.part = (float *)take(s.parts * p.n * 4);
      if (copy) dz = {s.dz, p.m, p.n, s.lddz, 1};
      launch([&] { return launch_slope(s, stream); });
    }
    if (p.dx) {
      GemmArgs out = {};
      out.y = p.dx, out.ldy = p.k;
      product(dz, {p.w, p.k, p.n, p.ws1, p.ws0}, out);
    }
    if (p.dw) {
      GemmArgs out = {};
      out.y = p.dw, out.ldy = p.k;
      product({dz.p, p.n, p.m, 1, dz.s0}, {p.x, p.k, p.m, p.xs1, p.xs0}, out);
    }
  }

  void run(const LinearArgs &p) {
    if (p.dy) backward(p);
    else forward(p);
  }
};

bool sound(const LinearArgs &p) {
  return p.m > 0 && p.n > 0 && p.k > 0 && p.dtype >= DT_F32 && p.dtype <= DT_FP16 &&
         p.act >= ACT_NONE && p.act <= ACT_SILU && p.xs0 >= 0 && p.xs1 >= 0 && p.ws0 >= 0 &&
         p.ws1 >= 0 && (p.x || (p.dy && !p.dw)) && (p.w || (p.dy && !p.dx)) &&
         (p.dy ? p.act == ACT_NONE || p.z : p.y != nullptr);
}

}  // namespace

extern "C" {

/* The bytes of workspace that a call takes, or a code below 0. */
int64_t vgpu_ops_linear_work(const LinearArgs *args) {
  if (!sound(*args)) return OPS_BAD_ARG;
  Call call = {nullptr, args->dtype == DT_F32 ? 4 : 2, args->dtype, nullptr};
  call.run(*args);
  return call.code ? call.code : call.used;
}

int vgpu_ops_linear(const LinearArgs *args, void *stream) {
  int64_t bytes = vgpu_ops_linear_work(args);
  if (bytes < 0) return (int)bytes;
  if (bytes > args->work_bytes || (bytes && (!args->work || (uintptr_t)args->work % 256)))
    return OPS_BAD_ARG;
  /* without a workspace any address will do: nothing is taken from it */
  char *base = bytes ? (char *)args->work : (char *)256;
  Call call = {base, args->dtype == DT_F32 ? 4 : 2, args->dtype, (hipStream_t)stream};
  call.run(*args);
  return call.code;
}

}  // extern "C"
