/* Matrix product with bias, activation and residual in its epilogue.
 *
 *   y = act(a b^T + bias) + res,   a [m,k], b [n,k], y [m,n]
 *
 * Either operand may lie with k contiguous or with k strided, so one kernel
 * serves x W^T and both gradients (dz W and dz^T x) without a transposed copy.
 */
#include "common.h"

#include <algorithm>
#include <type_traits>

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr uint32_t OUT_OF_RANGE = 0x80000000u; /* past any num_records below */

/* A fragment is what one lane gives one 64-byte step of k: 16 bytes.  Lane l
 * holds row l%16 and, of the step's k, the (l/16)-th quarter. */
template <typename T>
struct Frag {
  typename Vec<T>::type v;
};

/* The matrix instructions of one pair of fragments: one, or four in fp32,
 * where step j takes element j of every lane: both operands number k alike, so
 * the order in which k is summed is free. */
template <typename T>
constexpr int PARTS = sizeof(T) == 4 ? 4 : 1;

__device__ inline f32x4 mma(const Frag<bf16> &a, const Frag<bf16> &b, f32x4 c, int) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Frag<fp16> &a, const Frag<fp16> &b, f32x4 c, int) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Frag<float> &a, const Frag<float> &b, f32x4 c, int j) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
}

/* The same with the sum held in the accumulation registers for good.  Where
 * all 256 of them are sums the compiler would move some back and forth in
 * every step.  It cannot see what these write: the caller keeps other products
 * between two into the same sum, and waits (settle) before it reads one.  Nor
 * does it put the two wait states between a vector instruction's write of a or b
 * and these: fragments come from LDS reads alone.  A test reads the compiled
 * code for both. */
__device__ inline void mma_pinned(const Frag<bf16> &a, const Frag<bf16> &b, f32x4 &c, int) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a.v), "v"(b.v));
}
__device__ inline void mma_pinned(const Frag<fp16> &a, const Frag<fp16> &b, f32x4 &c, int) {
  asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a.v), "v"(b.v));
}
__device__ inline void mma_pinned(const Frag<float> &a, const Frag<float> &b, f32x4 &c, int j) {
  float x = a.v[j], y = b.v[j];
  asm volatile("v_mfma_f32_16x16x4_f32 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
}
/* Between other writes or reads of pinned sums and the products: 32 wait
 * states, more than the longest of these takes to write its sum.  The empty
 * statements keep the compiler's own moves on their side of it. */
template <int M, int N>
__device__ inline void settle(f32x4 (&c)[M][N]) {
  auto hold = [&] {
#pragma unroll
    for (int i = 0; i < M; i++)
#pragma unroll
      for (int j = 0; j < N; j++) asm volatile("" : "+a"(c[i][j]));
  };
  hold();
  asm volatile("s_nop 15\n\ts_nop 15");
  hold();
}

/* A window on memory of which nothing past `extent` bytes is read: a buffer's
 * descriptor (base, no stride, size in bytes, raw 32-bit data). */
__device__ inline u32x4 window(const void *base, int64_t extent) {
  uintptr_t at = (uintptr_t)base;
  auto same = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
  return u32x4{same((uint32_t)at), same((uint32_t)(at >> 32) & 0xffffu),
               same((uint32_t)min(max(extent, (int64_t)0), (int64_t)0x7ffffff0)), 0x00020000u};
}

__device__ inline u32x4 load16(u32x4 from, uint32_t offset) {
  __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
      (void *)(((uintptr_t)from[1] << 32) | from[0]), 0, (int)from[2], (int)from[3]);
  return __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, 0);
}

/* 16 bytes a lane straight to LDS, at `to` + SKIP + 16 lane.  Written out
 * because the compiler, which cannot tell this buffer from the ones being read,
 * would wait for it before the next read of LDS; land_and_meet() does the
 * waiting.  It has no result.  m0 is reserved, no register that the compiler keeps
 * values in (it warns where a clobber names it): it writes it anew before each
 * instruction of its own that reads it. */
template <int SKIP>
__device__ inline void load16_to_lds(u32x4 from, uint32_t offset, uint32_t to) {
  asm volatile(
      "s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(to), "v"(offset), "s"(from), "n"(SKIP)
      : "memory", "scc");
}

/* One operand's tile of R rows (of m or n) by STEPS steps of k in LDS, filled
 * by loads that go to LDS directly: lane l of a wave writes base + 16 l, so
 * the order of 16-byte chunks is chosen by which chunk a lane asks for.
 *
 * k contiguous: the chunks of a row are spread by xor with higher bits of the
 * row, so that the 16 rows that a fragment reads at once fall on all 64 banks.
 * k strided: rows are k; a 16-bit fragment is read with the transposing read
 * (4 rows of k by 16 columns), so 32-byte pieces of rows that are read
 * together are spread by xor; fp32 reads 64-byte pieces of 4 rows.
 * Counted on 8192^3: no bank conflicts in any layout. */
template <typename T, bool KC, int R, int THREADS>
struct Tile {
  static constexpr int E = Vec<T>::N;
  static constexpr int STAGE = STEPS * STEP_BYTES;
  static constexpr int BYTES = R * STAGE;
  static constexpr int LOADS = BYTES / (THREADS * 16);
  static constexpr int ROW_CHUNKS = KC ? STAGE / 16 : R / E;
  static_assert(LOADS * THREADS * 16 == BYTES, "whole loads");
  static_assert((ROW_CHUNKS & (ROW_CHUNKS - 1)) == 0, "the xor stays in the row");
  static constexpr int ROWS = THREADS / ROW_CHUNKS; /* between a thread's chunks */
  uint32_t off[LOADS];                              /* bytes */
  int kpos; /* k contiguous: first k of the thread's chunks, which the xor,
               repeating every 16 rows, leaves alike */
  static_assert(!KC || ROWS % 16 == 0, "chunks alike");

  static __device__ int spread(int row) {
    int x;
    if (KC) x = row >> 1;
    else if (sizeof(T) == 4) x = ((row >> 2) & 3) << 2;
    else x = ((row & 3) | (((row >> 3) & 1) << 2)) << 1;
    return x & (ROW_CHUNKS - 1);
  }

  __device__ void init(int64_t ld, int tid) {
    int r = tid / ROW_CHUNKS, c = tid % ROW_CHUNKS;
    kpos = (c ^ spread(r)) * E;
#pragma unroll
    for (int i = 0; i < LOADS; i++)
      off[i] = (r + i * ROWS) * (uint32_t)(ld * sizeof(T)) + (c ^ spread(r + i * ROWS)) * 16;
  }

  /* One of a stage's loads.  What lies past the operand's end comes as zeros,
   * dword by dword: with k strided that is all past the end of k, with k
   * contiguous chunks past it are asked for there.  Rows past m or n only feed results that are
   * not stored. */
  template <int I>
  __device__ void load(u32x4 from, int k_left, uint32_t lds) const {
    load16_to_lds<I * THREADS * 16>(from, !KC || kpos < k_left ? off[I] : OUT_OF_RANGE, lds);
  }

  /* Where k, which is contiguous, ends inside a chunk: zeros behind, instead
   * of what follows the row in memory.  `left` of the stage's k are there. */
  static __device__ void trim(char *lds, int left) {
    for (int r = threadIdx.x; r < R; r += THREADS) {
      T *q = (T *)(lds + r * STAGE + (left / E ^ spread(r)) * 16);
#pragma unroll 1
      for (int e = left % E; e < E; e++) q[e] = T(0);
    }
  }

  /* The fragment of rows row0 .. row0+15 at one of the stage's steps. */
  static __device__ Frag<T> frag(const char *lds, int row0, int step, int lane) {
    int i = lane & 15, g = lane >> 4;
    Frag<T> f;
    if constexpr (KC) {
      int c = (step * 4 + g) ^ spread(i); /* row0 is a multiple of 16 */
      f.v = *(const typename Vec<T>::type *)(lds + (row0 + i) * STAGE + c * 16);
    } else if constexpr (sizeof(T) == 4) {
      int c = ((row0 + i) >> 2) ^ spread(4 * g);
      const char *p = lds + (step * 16 + 4 * g) * (R * 4) + c * 16 + (i & 3) * 4;
#pragma unroll
      for (int j = 0; j < 4; j++) f.v[j] = *(const float *)(p + j * (R * 4));
    } else {
      int k = step * 32 + 8 * g + (i >> 2);
      int c = ((row0 >> 3) + ((i & 3) >> 1)) ^ spread(k);
      const char *p = lds + k * (R * 2) + c * 16 + (i & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      union {
        s16x4 s[2];
        typename Vec<T>::type v;
      } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p);
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * (R * 2)));
      f.v = u.v;
    }
    return f;
  }
};

/* Finishes rows of four neighbouring columns: bias, activation, residual,
 * store, or the partial sums of a split.  Accesses of four need no alignment
 * beyond the element's. */
template <typename T>
struct Epilogue {
  template <typename D>
  using Four = typename Loose4<D>::type;
  const GemmArgs &p;
  float *part; /* of this split, or null */

  __device__ Epilogue(const GemmArgs &args, int split = 0)
      : p(args), part(args.splits > 1 ? args.work + (int64_t)split * args.m * args.n : nullptr) {}

  /* COUNT rows, `step` apart, all there and four columns wide: everything is
   * asked for before anything is used. */
  template <int COUNT>
  __device__ void rows(int64_t m, int step, int64_t col, f32x4 (&v)[COUNT]) const {
    if (part) {
#pragma unroll
      for (int q = 0; q < COUNT; q++)
        *(Four<float> *)(part + (m + q * step) * p.n + col) = v[q];
      return;
    }
    Four<T> res[COUNT], bias;
    if (p.res)
#pragma unroll
      for (int q = 0; q < COUNT; q++)
        res[q] = *(const Four<T> *)((const T *)p.res + (m + q * step) * p.ldr + col);
    if (p.bias) bias = *(const Four<T> *)((const T *)p.bias + col);
    if (p.bias)
#pragma unroll
      for (int q = 0; q < COUNT; q++) v[q] += wide(bias);
    if (p.z)
#pragma unroll
      for (int q = 0; q < COUNT; q++)
        *(Four<T> *)((T *)p.z + (m + q * step) * p.ldz + col) = narrow(kept(v[q]));
    activate_all<T>(v, p.act);
    if (p.res)
#pragma unroll
      for (int q = 0; q < COUNT; q++) v[q] += wide(res[q]);
#pragma unroll
    for (int q = 0; q < COUNT; q++)
      *(Four<T> *)((T *)p.y + (m + q * step) * p.ldy + col) = narrow(v[q]);
  }

  /* What there is of one row's four. */
  __device__ void one(int64_t m, int64_t col, f32x4 v) const {
    if (m >= p.m) return;
    if (col + 4 <= p.n) {
      f32x4 row[1] = {v};
      rows(m, 0, col, row);
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (col + e >= p.n) return;
      if (part) {
        part[m * p.n + col + e] = v[e];
        continue;
      }
      f32x4 u[1] = {{v[e], 0.f, 0.f, 0.f}};
      if (p.bias) u[0][0] += to_f<T>(((const T *)p.bias)[col + e]);
      if (p.z) ((T *)p.z)[m * p.ldz + col + e] = from_f<T>(in_range<T>(u[0][0]));
      activate_all<T>(u, p.act);
      if (p.res) u[0][0] += to_f<T>(((const T *)p.res)[m * p.ldr + col + e]);
      ((T *)p.y)[m * p.ldy + col + e] = from_f<T>(u[0][0]);
    }
  }

  static __device__ f32x4 wide(Four<T> t) {
    return f32x4{to_f<T>(t[0]), to_f<T>(t[1]), to_f<T>(t[2]), to_f<T>(t[3])};
  }
  static __device__ f32x4 kept(f32x4 v) {
    return f32x4{in_range<T>(v[0]), in_range<T>(v[1]), in_range<T>(v[2]), in_range<T>(v[3])};
  }
  static __device__ Four<T> narrow(f32x4 v) {
    return Four<T>{from_f<T>(v[0]), from_f<T>(v[1]), from_f<T>(v[2]), from_f<T>(v[3])};
  }
};

/* Workgroups are dealt to the 8 XCDs in turn; give each XCD a run of tiles
 * that share rows of a and b in its own L2, in bands of 8 tiles of m. */
__device__ inline void tile_of(int block, int blocks, int tiles_m, int tiles_n, int *tm, int *tn) {
  int q = blocks / 8, r = blocks % 8, xcd = block % 8;
  int t = xcd * q + min(xcd, r) + block / 8;
  constexpr int BAND = 8;
  int band = t / (BAND * tiles_n), first = band * BAND;
  int height = min(BAND, tiles_m - first);
  int in = t - first * tiles_n;
  *tm = first + in % height;
  *tn = in / height;
}

/* f(0), f(1), ... with constants. */
template <int N, int I = 0, typename F>
__device__ inline void each(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    each<N, I + 1>(f);
  }
}

/* Waits until at most N of the wave's loads to LDS are in flight and its LDS
 * reads are done, then for the other waves.  The compiler moves no memory
 * access across it. */
template <int N>
__device__ inline void land_and_meet() {
  static_assert(N < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

/* A TM x TN tile of y per workgroup of WR x WC waves, and BUFFERS stages of
 * STEPS steps of k in LDS.  The fragments of a step are read while the step
 * before is multiplied, so the matrix cores wait for neither; one barrier a
 * stage says both that the next stage has landed and that this one has been
 * read, and its buffer is filled again at once.
 *
 * Bound by the matrix cores: four waves with a quarter of 256 x 256 each read
 * the fewest bytes of LDS a product, and fill the registers.  Smaller tiles are
 * for sizes that leave CUs idle; they have more stages in flight, since their
 * loads have less time to land.  8192^3 bf16: 1400 TFLOP/s with k contiguous or
 * strided on either side. */
template <typename T, bool AKC, bool BKC, int TM, int TN, int WR, int WC, int BUFFERS>
__global__ __launch_bounds__(WR *WC * 64, TM == 256 ? 1 : 2) void gemm_tile(GemmArgs p) {
  constexpr int THREADS = WR * WC * 64;
  constexpr int BK = STEPS * STEP_BYTES / sizeof(T);
  constexpr int FM = TM / WR / 16, FN = TN / WC / 16;
  using TA = Tile<T, AKC, TM, THREADS>;
  using TB = Tile<T, BKC, TN, THREADS>;
  constexpr int LOADS = TA::LOADS + TB::LOADS, BYTES = TA::BYTES + TB::BYTES;
  constexpr bool PINNED = FM * FN == 64; /* a wave's sums fill 256 registers */
  __shared__ __attribute__((aligned(1024))) char lds[BUFFERS * BYTES];

  int tid = threadIdx.x, lane = tid & 63;
  int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tiles_m = (int)((p.m + TM - 1) / TM), tiles_n = (int)((p.n + TN - 1) / TN);
  int tm, tn;
  tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, &tm, &tn);
  int64_t m0 = (int64_t)tm * TM, n0 = (int64_t)tn * TN;
  int stages_all = (int)((p.k + BK - 1) / BK);
  int s0 = (int)((int64_t)stages_all * blockIdx.y / p.splits);
  int s1 = (int)((int64_t)stages_all * (blockIdx.y + 1) / p.splits);

  TA ta;
  TB tb;
  ta.init(p.lda, tid);
  tb.init(p.ldb, tid);
  /* past this part's last stage the loads bring zeros from empty windows, so
   * that their number stays the same */
  struct Source {
    u32x4 a, b;
    int left;
  };
  auto source = [&](int s) {
    int64_t k = (int64_t)s * BK;
    int64_t oa = (AKC ? m0 * p.lda + k : k * p.lda + m0) * (int64_t)sizeof(T);
    int64_t ob = (BKC ? n0 * p.ldb + k : k * p.ldb + n0) * (int64_t)sizeof(T);
    bool some = s < s1;
    return Source{window((const char *)p.a + oa, some ? p.a_extent - oa : 0),
                  window((const char *)p.b + ob, some ? p.b_extent - ob : 0),
                  (int)min(p.k - k, (int64_t)BK)};
  };
  uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void *)lds;
  auto load = [&](auto i, const Source &q, int buffer) {
    constexpr int I = decltype(i)::value;
    uint32_t at = lds_at + buffer * BYTES + wave * 1024;
    if constexpr (I < TA::LOADS) ta.template load<I>(q.a, q.left, at);
    else tb.template load<I - TA::LOADS>(q.b, q.left, at + TA::BYTES);
  };

  f32x4 acc[FM][FN] = {};
  int wm = wave / WC * (TM / WR), wn = wave % WC * (TN / WC);
  struct Step {
    Frag<T> a[FM], b[FN];
  } even, odd;
  auto read = [&](int f, Step &h, const char *at, int step) {
    if (f < FN) h.b[f] = TB::frag(at + TA::BYTES, wn + f * 16, step, lane);
    else h.a[f - FN] = TA::frag(at, wm + (f - FN) * 16, step, lane);
  };
  /* Product number q of a step, by rows, so that the last fragments are not
   * needed at once; between two into one sum lie FN - 1 others at least. */
  auto multiply = [&](const Step &h, int q) {
    int i = q / (FN * PARTS<T>), part = q / FN % PARTS<T>, j = q % FN;
    if constexpr (PINNED) mma_pinned(h.b[j], h.a[i], acc[i][j], part);
    else acc[i][j] = mma(h.b[j], h.a[i], acc[i][j], part);
  };
  /* A step's products, with the reads of the next one and the loads dealt out
   * between them: in a row they would hold up the matrix cores of all waves. */
  constexpr int FRAGS = FM + FN, PRODUCTS = FM * FN * PARTS<T>;
  constexpr int TURNS = FRAGS > LOADS ? FRAGS : LOADS;
  auto step = [&](const Step &now, Step &then, const char *from, int which, const Source *q,
                  int to) {
    __builtin_amdgcn_sched_barrier(0);
    each<TURNS>([&](auto turn) {
      constexpr int F = decltype(turn)::value, P0 = PRODUCTS * F / TURNS,
                    P1 = PRODUCTS * (F + 1) / TURNS;
      if (F < FRAGS) read(F, then, from, which);
#pragma unroll
      for (int m = P0; m < P1; m++) {
        if constexpr (F < LOADS)
          if (q && m == P0 + (P1 - P0) / 2) load(turn, *q, to);
        multiply(now, m);
      }
      if constexpr (P0 == P1 && F < LOADS)
        if (q) load(turn, *q, to);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  /* the stage in which k ends inside a chunk */
  int ragged = p.k % TA::E ? stages_all - 1 : -1;
  auto trim = [&](int s, char *at) {
    if (s != ragged) return;
    int left = (int)(p.k - (int64_t)s * BK);
    if (AKC) TA::trim(at, left);
    if (BKC) TB::trim(at + TA::BYTES, left);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  int buffer = 0;
  /* the stage whose first step is in `now`; leaves the next one's there */
  auto stage = [&](int s, Step &now, Step &then) {
    int at = buffer;
    buffer = buffer + 1 == BUFFERS ? 0 : buffer + 1;
    Source q = source(s + BUFFERS);
    step(now, then, lds + at * BYTES, 1, nullptr, 0);
    land_and_meet<(BUFFERS - 2) * LOADS>();
    if constexpr (AKC || BKC) trim(s + 1, lds + buffer * BYTES);
    step(then, now, lds + buffer * BYTES, 0, &q, at);
  };

#pragma unroll
  for (int i = 0; i < BUFFERS; i++) {
    Source q = source(s0 + i);
    each<LOADS>([&](auto f) { load(f, q, i); });
  }
  land_and_meet<(BUFFERS - 1) * LOADS>();
  if constexpr (AKC || BKC) trim(s0, lds);
#pragma unroll
  for (int f = 0; f < FRAGS; f++) read(f, even, lds, 0);
  if constexpr (PINNED) settle(acc);
  for (int s = s0; s < s1; s++) stage(s, even, odd);
  land_and_meet<0>();
  if constexpr (PINNED) settle(acc);

  /* b is the first operand of the product, so a lane holds 4 neighbouring
   * columns of row lane%16.  Each wave turns its part through its own piece
   * of LDS, so that rows are stored whole and the epilogue's code is there
   * once; 16-byte pieces are spread by xor over the banks. */
  constexpr int WM = TM / WR, WN = TN / WC, PIECES = WN / 4;
  constexpr int PIECE_LDS = (int)sizeof(lds) / (WR * WC);
  constexpr int FIT = PIECE_LDS / (WN * 4);
  constexpr int ROWS = FIT >= WM ? WM : FIT >= WM / 2 ? WM / 2 : WM / 4;
  static_assert(ROWS % 16 == 0 && ROWS <= FIT, "whole fragments a pass");
  static_assert(64 % PIECES == 0, "a lane keeps its columns");
  constexpr int DOWN = 64 / PIECES, U = ROWS / DOWN < 8 ? ROWS / DOWN : 8;
  float *mine = (float *)(lds + wave * PIECE_LDS);
  Epilogue<T> finish(p, blockIdx.y);
  int row = lane / PIECES, piece = lane % PIECES;
#pragma unroll
  for (int pass = 0; pass < WM / ROWS; pass++) {
#pragma unroll
    for (int i = 0; i < ROWS / 16; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) {
        int r = i * 16 + (lane & 15), c = (j * 4 + (lane >> 4)) ^ (r & (PIECES - 1));
        *(f32x4 *)(mine + r * WN + c * 4) = acc[pass * (ROWS / 16) + i][j];
      }
    auto at = [&](int r) {
      return *(const f32x4 *)(mine + r * WN + (piece ^ (r & (PIECES - 1))) * 4);
    };
    int64_t m = m0 + wm + pass * ROWS, n = n0 + wn + piece * 4;
    if (m + ROWS <= p.m && n0 + wn + WN <= p.n) {
#pragma unroll 1
      for (int r = row; r < ROWS; r += DOWN * U) {
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = at(r + u * DOWN);
        finish.rows(m + r, DOWN, n, v);
      }
    } else {
#pragma unroll 1
      for (int r = row; r < ROWS; r += DOWN) finish.one(m + r, n, at(r));
    }
  }
}

/* Adds the splits' partial sums in their order and finishes the rows. */
template <typename T>
__global__ __launch_bounds__(256) void gemm_join(GemmArgs p) {
  int64_t fours = (p.n + 3) / 4;
  int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.m * fours) return;
  int64_t m = at / fours, n = at % fours * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const float *q = p.work + m * p.n + n;
  if (n + 4 <= p.n && p.n % 4 == 0) {
    for (int s = 0; s < p.splits; s++) v += *(const f32x4 *)(q + (int64_t)s * p.m * p.n);
  } else {
    for (int s = 0; s < p.splits; s++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (n + e < p.n) v[e] += q[(int64_t)s * p.m * p.n + e];
  }
  p.splits = 1;
  Epilogue<T> finish(p);
  finish.one(m, n, v);
}

/* Few rows (m <= 16): b is read once, at the memory's rate, straight into the
 * matrix cores' registers.  A workgroup takes a strip of n; its eight waves
 * share k between them, a step of 64 bytes of a's k at a time, and join in
 * LDS.
 *
 * k contiguous in b: the strip is 16 rows of b, a step 16 rows by 64 bytes.
 * k strided: the strip is 16 lanes by 16 bytes of n, a step 4 V rows of k;
 * lane i holds V neighbouring columns, of which the j-th go to the j-th
 * product, so 16-bit values are only turned inside a lane.
 * LOOSE: rows of 16-bit values that start on 2 bytes, by loads that may.
 *
 * Bound by reading b.  1 x 4096 -> 4096 bf16: 9.3 us; 1 x 25088 -> 4096 fp32: 77
 * us, 5.3 TB/s, and 2 rows of it in a training step 95 us, 4.3 TB/s; with k strided
 * (their gradient) 76 us, 5.4 TB/s. */
template <typename T, bool BKC, bool LOOSE>
__global__ __launch_bounds__(512, BKC ? 4 : 2) void gemm_rows(GemmArgs p) {
  constexpr int V = Vec<T>::N, WAVES = 8;
  constexpr int FN = BKC ? 1 : V;    /* products a step */
  constexpr int STRIP = 16 * FN;     /* columns of y */
  constexpr int LOADS = BKC ? 1 : V; /* of b a step */
  /* Steps a wave has in flight, twice: with k contiguous 6, whose registers
   * leave room for a second workgroup on the CU.  us for 6, and for 8 with one
   * workgroup: 1 x 5155 -> 4311 bf16 33 and 43, 1 x 501 -> 20000 24 and 34, 1 x
   * 4096 -> 4096 10.9 and 10.6. */
  constexpr int C = BKC ? 6 : 8 / LOADS;
  typedef typename Vec<T>::type vec;
  __shared__ f32x4 lds[WAVES][16][STRIP / 4];

  int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t n0 = (int64_t)blockIdx.x * STRIP;
  int64_t all = (p.k + 4 * V - 1) / (4 * V);
  int64_t s0 = all * blockIdx.y / p.splits, s1 = all * (blockIdx.y + 1) / p.splits;
  const char *b = (const char *)p.b + n0 * (BKC ? p.ldb : 1) * (int64_t)sizeof(T);
  int64_t b_left = p.b_extent - (b - (const char *)p.b);
  u32x4 ra = window(p.a, p.a_extent);

  uint32_t a_off = i < p.m ? (uint32_t)(i * p.lda * sizeof(T)) + g * 16 : OUT_OF_RANGE;
  uint32_t b_off[LOADS];
#pragma unroll
  for (int t = 0; t < LOADS; t++) {
    if (BKC) b_off[t] = n0 + i < p.n ? (uint32_t)(i * p.ldb * sizeof(T)) + g * 16 : OUT_OF_RANGE;
    else b_off[t] = n0 + i * V < p.n ? (uint32_t)((g * V + t) * p.ldb * sizeof(T)) + i * 16
                                     : OUT_OF_RANGE;
  }

  struct Step {
    u32x4 a, b[LOADS];
  };
  auto fetch = [&](Step &q, int64_t s) {
    bool in = s < s1 && (s * 4 + g) * V < p.k;
    uint32_t at = (uint32_t)(s * 64);
    q.a = load16(ra, in ? a_off + at : OUT_OF_RANGE);
    if constexpr (LOOSE) {
      int64_t k = (s * 4 + g) * V;
      int n = in && n0 + i < p.n ? (int)min((int64_t)V, p.k - k) : 0;
      q.b[0] = __builtin_bit_cast(u32x4, load_raw<T>((const T *)b + i * p.ldb + k, n));
      return;
    }
    int64_t skip = BKC ? 0 : s * 4 * V * p.ldb * (int64_t)sizeof(T);
    u32x4 rb = window(b + skip, b_left - skip);
#pragma unroll
    for (int t = 0; t < LOADS; t++)
      q.b[t] = load16(rb, (BKC ? in : s < s1) ? b_off[t] + (BKC ? at : 0) : OUT_OF_RANGE);
  };

  f32x4 acc[FN] = {};
  int ragged = (int)(p.k % V); /* values of a chunk in which k ends */
  int64_t last = p.k / V;
  auto multiply = [&](const Step &q, int64_t s) {
    Frag<T> fa, fb[FN];
    fa.v = __builtin_bit_cast(vec, q.a);
    if constexpr (BKC) fb[0].v = __builtin_bit_cast(vec, q.b[0]);
    if (ragged && s == last / 4) { /* zeros behind it, not what follows the row */
      bool here = g == (int)(last % 4);
#pragma unroll
      for (int e = 1; e < V; e++)
        if (here && e >= ragged) {
          fa.v[e] = T(0);
          if (BKC) fb[0].v[e] = T(0);
        }
    }
    if constexpr (!BKC) {
      vec r[V];
#pragma unroll
      for (int t = 0; t < V; t++) r[t] = __builtin_bit_cast(vec, q.b[t]);
#pragma unroll
      for (int j = 0; j < V; j++)
#pragma unroll
        for (int t = 0; t < V; t++) fb[j].v[t] = r[t][j];
    }
#pragma unroll
    for (int e = 0; e < PARTS<T>; e++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[j] = mma(fb[j], fa, acc[j], e);
  };
  Step even[C], odd[C];
  auto take = [&](Step(&now)[C], Step(&then)[C], int64_t s) {
#pragma unroll
    for (int c = 0; c < C; c++) fetch(then[c], s + WAVES * C + c);
    __builtin_amdgcn_sched_barrier(0); /* the loads go out before the products */
#pragma unroll
    for (int c = 0; c < C; c++) multiply(now[c], s + c);
    __builtin_amdgcn_sched_barrier(0);
  };
  int64_t s = s0 + wave * C;
#pragma unroll
  for (int c = 0; c < C; c++) fetch(even[c], s + c);
  for (; s < s1; s += 2 * WAVES * C) { /* steps past s1 are zeros */
    take(even, odd, s);
    take(odd, even, s + WAVES * C);
  }

#pragma unroll
  for (int j = 0; j < FN; j++)
#pragma unroll
    for (int e = 0; e < 4; e++) /* column (4 g + e) FN + j of the strip, row i */
      ((float *)lds[wave][i])[(4 * g + e) * FN + j] = acc[j][e];
  __syncthreads();
  Epilogue<T> finish(p, blockIdx.y);
  for (int q = threadIdx.x; q < 16 * (STRIP / 4); q += 512) {
    int r = q / (STRIP / 4), c = q % (STRIP / 4);
    int64_t n = n0 + c * 4;
    if (r >= p.m || n >= p.n) continue;
    f32x4 v = lds[0][r][c];
#pragma unroll
    for (int w = 1; w < WAVES; w++) v += lds[w][r][c];
    finish.one(r, n, v);
  }
}

/* A short sum (k <= 32) with k strided on both sides, as a weight's gradient
 * from few rows is: bound by writing y.  A wave holds 8 rows by 64 vectors of
 * columns; a's values are the same for the whole wave.  4096 x 25088 fp32 of 2
 * rows: 56 us, 7.4 TB/s. */
template <typename T>
__global__ __launch_bounds__(256) void gemm_outer(GemmArgs p) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[OUTER_K][4 * OUTER_ROWS];
  int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t m0 = (int64_t)blockIdx.y * (4 * OUTER_ROWS);
  const T *a = (const T *)p.a, *b = (const T *)p.b;
  for (int q = threadIdx.x; q < p.k * 4 * OUTER_ROWS; q += 256) {
    int k = q / (4 * OUTER_ROWS), r = q % (4 * OUTER_ROWS);
    lds[k][r] = m0 + r < p.m ? to_f<T>(a[k * p.lda + m0 + r]) : 0.f;
  }
  __syncthreads();
  int64_t n = ((int64_t)blockIdx.x * 64 + lane) * V;
  int count = (int)max((int64_t)0, min((int64_t)V, p.n - n));
  float acc[OUTER_ROWS][V] = {};
  for (int k = 0; k < p.k; k++) {
    float v[V];
    load_vec<T>(b + k * p.ldb + n, count, v);
#pragma unroll
    for (int r = 0; r < OUTER_ROWS; r++) {
      float w = lds[k][wave * OUTER_ROWS + r];
#pragma unroll
      for (int e = 0; e < V; e++) acc[r][e] += w * v[e];
    }
  }
#pragma unroll
  for (int r = 0; r < OUTER_ROWS; r++) {
    int64_t m = m0 + wave * OUTER_ROWS + r;
    if (m < p.m) store_vec<T>((T *)p.y + m * p.ldy + n, count, acc[r]);
  }
}

template <typename T, bool BKC, bool LOOSE>
void launch_rows(const GemmArgs &p, hipStream_t stream) {
  constexpr int STRIP = BKC ? 16 : 16 * Vec<T>::N;
  dim3 grid((unsigned)((p.n + STRIP - 1) / STRIP), (unsigned)p.splits);
  gemm_rows<T, BKC, LOOSE><<<grid, 512, 0, stream>>>(p);
}

template <typename T, bool AKC, bool BKC>
void launch_tile(const GemmArgs &p, hipStream_t stream) {
  auto blocks = [&](int tm, int tn) {
    return dim3((unsigned)(((p.m + tm - 1) / tm) * ((p.n + tn - 1) / tn)), (unsigned)p.splits);
  };
  if (p.plan == 0)
    gemm_tile<T, AKC, BKC, 256, 256, 2, 2, 2><<<blocks(256, 256), 256, 0, stream>>>(p);
  else if (p.plan == 1)
    gemm_tile<T, AKC, BKC, 128, 128, 2, 2, 2><<<blocks(128, 128), 256, 0, stream>>>(p);
  else if (p.plan == 2)
    gemm_tile<T, AKC, BKC, 64, 128, 2, 2, 3><<<blocks(64, 128), 256, 0, stream>>>(p);
  else
    gemm_tile<T, AKC, BKC, 32, 128, 1, 4, 4><<<blocks(32, 128), 256, 0, stream>>>(p);
}

template <typename T>
int join(const GemmArgs &p, hipStream_t stream) {
  if (p.splits > 1) {
    int64_t items = p.m * ((p.n + 3) / 4);
    gemm_join<T><<<(unsigned)((items + 255) / 256), 256, 0, stream>>>(p);
  }
  return OPS_LAUNCHED();
}

template <typename T>
int run(const GemmArgs &p, hipStream_t stream) {
  if (p.plan == PLAN_OUTER) {
    dim3 grid((unsigned)((p.n + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N)),
              (unsigned)((p.m + 4 * OUTER_ROWS - 1) / (4 * OUTER_ROWS)));
    gemm_outer<T><<<grid, 256, 0, stream>>>(p);
    return OPS_LAUNCHED();
  }
  if (p.plan == PLAN_ROWS && p.b_kc) {
    if constexpr (sizeof(T) == 2)
      if ((uintptr_t)p.b % 4 || p.ldb % 2) {
        launch_rows<T, true, true>(p, stream);
        return join<T>(p, stream);
      }
    launch_rows<T, true, false>(p, stream);
  }
  else if (p.plan == PLAN_ROWS) launch_rows<T, false, false>(p, stream);
  else if (p.a_kc && p.b_kc) launch_tile<T, true, true>(p, stream);
  else if (p.a_kc) launch_tile<T, true, false>(p, stream);
  else if (p.b_kc) launch_tile<T, false, true>(p, stream);
  else launch_tile<T, false, false>(p, stream);
  return join<T>(p, stream);
}

/* The bits of [rows, cols] of any strides to rows of `ld` elements, zeros
 * behind. */
template <typename T>
__global__ __launch_bounds__(256) void repack(const T *src, int64_t rs, int64_t cs, int64_t rows,
                                              int64_t cols, T *dst, int64_t ld) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < ld; c += (int64_t)gridDim.x * 256)
      dst[r * ld + c] = c < cols ? src[r * rs + c * cs] : T(0);
}

/* The same of rows that are contiguous, in loads of 16 bytes that start on any
 * element: a thread a chunk, 2^shift chunks of a row beside each other in a
 * workgroup.  Bound by memory: 8001 x 20001 16-bit values 102 us, 6.3 TB/s. */
template <typename T>
__global__ __launch_bounds__(256) void repack_rows(const T *src, int64_t rs, int64_t rows,
                                                   int64_t cols, T *dst, int64_t ld, int shift) {
  constexpr int V = Vec<T>::N;
  int64_t c = (((int64_t)blockIdx.x << shift) + (threadIdx.x & ((1 << shift) - 1))) * V;
  int64_t at_once = 256 >> shift;
  if (c >= ld) return;
  int n = (int)min((int64_t)V, cols - c);
  for (int64_t r = blockIdx.y * at_once + (threadIdx.x >> shift); r < rows; r += gridDim.y * at_once)
    *(typename Vec<T>::type *)(dst + r * ld + c) = load_raw<T>(src + r * rs + c, n);
}

/* dz = dy act'(z) and the columns' sums in one pass over dy and z, which bounds
 * it.  A workgroup's four waves share 64 vectors of columns; wave w takes rows w,
 * w+4, ... of the workgroup's run of rows.  4099 x 10240 fp16, gelu: 58 us, 4.3
 * TB/s. */
template <typename T>
__global__ __launch_bounds__(256) void slope_rows(SlopeArgs p) {
  constexpr int V = Vec<T>::N;
  __shared__ float lds[3][64][V + 1];
  int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int64_t col = ((int64_t)blockIdx.x * 64 + lane) * V;
  int n = (int)max((int64_t)0, min((int64_t)V, p.n - col));
  int64_t from = p.m * blockIdx.y / p.parts, to = p.m * (blockIdx.y + 1) / p.parts;
  const T *dy = (const T *)p.dy, *z = (const T *)p.z;
  T *dz = (T *)p.dz;
  float sum[V] = {};
  for (int64_t r = from + wave; r < to; r += 4) {
    float g[V], u[V];
    load_vec<T>(dy + r * p.lddy + col, n, g);
    if (p.act != ACT_NONE) {
      load_vec<T>(z + r * p.ldz + col, n, u);
#pragma unroll
      for (int e = 0; e < V; e++) g[e] = slope<T>(g[e], u[e], p.act);
    }
#pragma unroll
    for (int e = 0; e < V; e++) sum[e] += g[e];
    if (dz && col < p.lddz) store_vec<T>(dz + r * p.lddz + col, (int)min((int64_t)V, p.lddz - col), g);
  }
  if (!p.dbias) return;
  if (wave)
#pragma unroll
    for (int e = 0; e < V; e++) lds[wave - 1][lane][e] = sum[e];
  __syncthreads();
  if (wave || n <= 0) return;
#pragma unroll
  for (int e = 0; e < V; e++)
    for (int w = 0; w < 3; w++) sum[e] += lds[w][lane][e];
  if (p.parts == 1) {
    store_vec<T>((T *)p.dbias + col, n, sum);
    return;
  }
  float *part = p.part + blockIdx.y * p.n + col;
#pragma unroll
  for (int e = 0; e < V; e++)
    if (e < n) part[e] = sum[e];
}

template <typename T>
__global__ __launch_bounds__(1024) void slope_join(SlopeArgs p) {
  join_columns<T>(p.part, p.parts, p.n, (T *)p.dbias);
}

template <typename T>
int run_slope(const SlopeArgs &p, hipStream_t s) {
  int64_t vecs = (std::max(p.n, p.dz ? p.lddz : p.n) + Vec<T>::N - 1) / Vec<T>::N;
  slope_rows<T><<<dim3((unsigned)((vecs + 63) / 64), (unsigned)p.parts), 256, 0, s>>>(p);
  if (p.dbias && p.parts > 1) slope_join<T><<<(unsigned)((p.n + 63) / 64), 1024, 0, s>>>(p);
  return OPS_LAUNCHED();
}

}  // namespace

int launch_slope(const SlopeArgs &p, hipStream_t s) {
  if (p.dtype == DT_F32) return run_slope<float>(p, s);
  if (p.dtype == DT_BF16) return run_slope<bf16>(p, s);
  return run_slope<fp16>(p, s);
}

int launch_gemm(const GemmArgs &p, hipStream_t s) {
  if (p.dtype == DT_F32) return run<float>(p, s);
  if (p.dtype == DT_BF16) return run<bf16>(p, s);
  return run<fp16>(p, s);
}

int launch_repack(const void *src, int64_t rs, int64_t cs, int64_t rows, int64_t cols, void *dst,
                  int64_t ld, int size, hipStream_t s) {
  if (cs == 1) {
    int64_t chunks = ld * size / 16;
    int shift = 0;
    while (shift < 8 && (int64_t)1 << shift < chunks) shift++;
    int64_t blocks = (rows + (256 >> shift) - 1) / (256 >> shift);
    dim3 grid((unsigned)((chunks + ((int64_t)1 << shift) - 1) >> shift),
              (unsigned)std::min<int64_t>(blocks, 16384));
    if (size == 4)
      repack_rows<<<grid, 256, 0, s>>>((const uint32_t *)src, rs, rows, cols, (uint32_t *)dst, ld, shift);
    else
      repack_rows<<<grid, 256, 0, s>>>((const uint16_t *)src, rs, rows, cols, (uint16_t *)dst, ld, shift);
    return OPS_LAUNCHED();
  }
  dim3 grid((unsigned)std::min<int64_t>((ld + 255) / 256, 1024),
            (unsigned)std::min<int64_t>(rows, 16384));
  if (size == 4)
    repack<<<grid, 256, 0, s>>>((const uint32_t *)src, rs, cs, rows, cols, (uint32_t *)dst, ld);
  else
    repack<<<grid, 256, 0, s>>>((const uint16_t *)src, rs, cs, rows, cols, (uint16_t *)dst, ld);
  return OPS_LAUNCHED();
}
