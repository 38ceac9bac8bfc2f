// CDNA4 (gfx950) orthogonalisation of weight gradients by Newton-Schulz
// products, and the optimiser step around it.
//
//   X_0 = G / max(|G|_F, eps)                     on the shorter side: m <= n
//   A = X X^T        B = b A + c A^2        X' = a X + B X      (`steps` times)
//
// drives every singular value of G towards 1.  The optimiser step is
//
//   M' = mu M + G     U = G + mu M' (look-ahead) or M'     O = orthogonal(U)
//   W' = keep W - step O
//
// Arithmetic.  Small singular values grow by `a` per step (485-fold in five),
// and so does the rounding noise that lies in their directions: iterates held
// in 8 or 11 bits lose gradients of low rank (error 2e-2 to 9e-2 of the
// result).  The iterates are bounded, so they are kept here as sums of two
// fp16 numbers, x 2^s = hi + lo, 22 bits, and a product is three fp16 matrix
// products accumulated in fp32: hi hi + hi lo + lo hi.  By norms that is about
// as exact as fp32 (0.2 to 1.6 times its error after five steps, on full-rank,
// low-rank, rank-1 and graded gradients) at a third of the fp16 matrix rate, 3
// times the fp32 rate.  The last place of lo is 2^-24: x under 2^-17 has fewer
// than 22 bits, to the nearest 2^-39 (rows of 1e-9 of the norm are 1 to 6 % off).
// Results of 16 bits are computed in the same way and rounded at the store: a
// bf16 result is as good as its rounding (4096 x 4096: off by 1.66e-3 of its
// norm; with hi hi alone in A and A^2, and hi (hi + lo) in B X, 1.82e-3, in 1854
// us for 3415).
//
// A and A^2 are symmetric: tiles on or above the diagonal are computed, and
// each is written to both places.
//
// Three ways, by size: matrices whose shorter side is 16 or less are iterated as
// their small square alone, in fp64, in a launch or two for five steps; those that
// fit a CU's LDS are held there, in one launch for all of a table; the rest goes
// through working planes in memory, padded with zeros to whole tiles, which the
// iteration keeps, so that only the first and the last kernel look at ragged edges.
// These share their launches too: 2 + 3 * steps, and one more a step where sums are
// shared out.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <math.h>

#include <algorithm>
#include <stdint.h>
#include <type_traits>

namespace {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2, T_F64 = 3 };

constexpr int kMats = 24;        // matrices to a launch: the table is an argument
constexpr int kNormBlocks = 1024;  // most blocks that sum one matrix' squares
constexpr float kScaleX = 16384.f;  // |x| <= 1.9: within fp16
constexpr float kScaleA = 16384.f;  // |x|^2 <= 3.7

struct Mat {
  f16* ws;         // X^T (two), A, B: two planes each; of a thin one X, in fp64
  double* part;    // sums of squares
  const void* g;   // gradient, rows x cols
  float* mom;      // momentum buffer, or null
  void* w;         // weights, or the result
  int m, n;        // shorter and longer side
  int mp, np;      // padded to whole tiles of B X
  int ma;          // m padded to whole tiles of A as well
  int parts;       // sums of squares, or chunks of a thin matrix
  int chunk;       // its columns to a block
  int rows, cols;  // as the caller has it
  float step;
  int first;       // first block of this matrix in a launch
  int split;       // blocks to a tile of A, each with kpart of K
  int kpart;
  float* sums;     // their sums, tile by tile, if there are several
};

struct Table {
  Mat mat[kMats];
  int count;
  int gtype, wtype;
  float mu, keep, eps;
  int nesterov;
};

// ---- working planes ---------------------------------------------------------

// A plane holds rows of K values in panels of 32: panel after panel, row after
// row, 64 bytes each.  A tile's share of a panel is one piece of memory, so
// copies to LDS and the writes of a 32 x 32 piece run over whole cache lines
// (in plain rows a step takes 64 or 128 bytes here and there, at distances
// that fall on few channels of L2 when K is a power of two).
//
// X is kept as its transpose alone, np rows of ma values (mp of them in use):
// B X sums over these and A over the rows, which LDS turns as it reads.  (With
// X as well, read by A alone, 1000 x 4000 twice took 575 us for 553 in fp32.)
// A and B have ma rows of ma.  Sums over m run to mp, so what lies behind it
// meets nothing.
__host__ __device__ inline int tiles_of(int n, int side) { return (n + side - 1) / side; }

// A's tiles are panels of X', whose distance is not to be a power of two: 5 KB
// more (1024 x 4096 f32: 330 us without, 327 with).
constexpr int kGap = 80;
__host__ __device__ inline int rows_xt(int np) { return np + kGap; }
__host__ __device__ inline size_t plane_xt(const Mat& t) { return (size_t)rows_xt(t.np) * t.ma; }
__host__ __device__ inline size_t plane_a(const Mat& t) { return (size_t)t.ma * t.ma; }
// place of (row, k) in a plane of `rows` rows
__device__ __forceinline__ size_t place(int rows, int row, int k) {
  return ((size_t)(k >> 5) * rows + row) * 32 + (k & 31);
}
__device__ __forceinline__ f16* ws_xt(const Mat& t, int which, int p) {
  return t.ws + (2 * which + p) * plane_xt(t);
}
__device__ __forceinline__ f16* ws_a(const Mat& t, int p) {
  return t.ws + 4 * plane_xt(t) + p * plane_a(t);
}
__device__ __forceinline__ f16* ws_b(const Mat& t, int p) {
  return t.ws + 4 * plane_xt(t) + (2 + p) * plane_a(t);
}

// (Every function that takes the table is inlined: it stays in the arguments'
// memory, and is copied to each lane's stack as soon as one is not.)
__device__ __forceinline__ int find(const Table& tab, int block) {
  int k = 0;
  while (k + 1 < tab.count && block >= tab.mat[k + 1].first) ++k;
  return k;
}

__device__ __forceinline__ float load_as(const void* p, size_t i, int type) {
  if (type == T_F32) return ((const float*)p)[i];
  if (type == T_BF16) return (float)((const __bf16*)p)[i];
  return (float)((const f16*)p)[i];
}

__device__ __forceinline__ void store_as(void* p, size_t i, int type, float v) {
  if (type == T_F32)
    ((float*)p)[i] = v;
  else if (type == T_BF16)
    ((__bf16*)p)[i] = (__bf16)v;
  else
    ((f16*)p)[i] = (f16)v;
}

// 8 values side by side, `left` of them within the matrix.
__device__ __forceinline__ void load8(const void* p, size_t at, int type, int left, float* v) {
  if (left >= 8) {
    if (type == T_F32) {
      typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
      const f32x4 x = *(const f32x4*)((const float*)p + at), y = *(const f32x4*)((const float*)p + at + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = x[k], v[4 + k] = y[k];
    } else if (type == T_BF16) {
      typedef __bf16 b8 __attribute__((ext_vector_type(8), aligned(2)));
      const b8 x = *(const b8*)((const __bf16*)p + at);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (float)x[k];
    } else {
      typedef f16 h8 __attribute__((ext_vector_type(8), aligned(2)));
      const h8 x = *(const h8*)((const f16*)p + at);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = (float)x[k];
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? load_as(p, at + k, type) : 0.f;
  }
}

__device__ __forceinline__ void store8(void* p, size_t at, int type, int left, const float* v) {
  if (left >= 8) {
    if (type == T_F32) {
      typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
      *(f32x4*)((float*)p + at) = f32x4{v[0], v[1], v[2], v[3]};
      *(f32x4*)((float*)p + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else if (type == T_BF16) {
      typedef __bf16 b8 __attribute__((ext_vector_type(8), aligned(2)));
      b8 x;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = (__bf16)v[k];
      *(b8*)((__bf16*)p + at) = x;
    } else {
      typedef f16 h8 __attribute__((ext_vector_type(8), aligned(2)));
      h8 x;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = (f16)v[k];
      *(h8*)((f16*)p + at) = x;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) store_as(p, at + k, type, v[k]);
  }
}

// The empty statement makes v a number of fp32: without it the compiler may
// round the product that v comes from straight to fp16 for one use of hi and by
// way of fp32 for the other, and a tie between them costs lo its meaning.
__device__ __forceinline__ void split(float v, f16& hi, f16& lo) {
  asm volatile("" : "+v"(v));
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

// U, what is orthogonalised, for 8 values: G, or G with its momentum.
__device__ __forceinline__ void load_u(const Table& tab, const Mat& t, size_t at, int left, float* u) {
  load8(t.g, at, tab.gtype, left, u);
  if (t.mom) {
    float m[8];
    load8(t.mom, at, T_F32, left, m);
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = tab.nesterov ? u[k] + tab.mu * m[k] : m[k];
  }
}

// ---- sums of squares, and the momentum ---------------------------------------

// In 64 bits: a long sum, and squares of values near the ends of fp32.  Bound by
// HBM where there is a momentum to move on (1024 x 4096 twice: 100 MB, 19 us).
__global__ __launch_bounds__(256) void flowml_ns_norm(Table tab) {
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int b = blockIdx.x - t.first;
  const size_t total = (size_t)t.rows * t.cols, stride = (size_t)t.parts * 2048;
  double s = 0.0;
  for (size_t at = ((size_t)b * 256 + threadIdx.x) * 8; at < total; at += stride) {
    const int left = total - at < 8 ? (int)(total - at) : 8;
    float u[8];
    if (t.mom) {
      float g[8], m[8];
      load8(t.g, at, tab.gtype, left, g);
      load8(t.mom, at, T_F32, left, m);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = tab.mu * m[k] + g[k];
        u[k] = tab.nesterov ? g[k] + tab.mu * m[k] : m[k];
      }
      store8(t.mom, at, T_F32, left, m);
    } else {
      load8(t.g, at, tab.gtype, left, u);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s += (double)u[k] * (double)u[k];
  }
  __shared__ double red[4];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) t.part[b] = red[0] + red[1] + red[2] + red[3];
}

// ---- the first iterate: 64 x 64 tiles of the caller's matrix -------------------

// Bound by memory: 4096 x 4096 bf16, 33 MB in and 67 MB out, 21 us.

__global__ __launch_bounds__(256) void flowml_ns_first(Table tab) {
  __shared__ double red[4];
  __shared__ uint32_t tile[64][65];
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int b = blockIdx.x - t.first, tid = threadIdx.x;
  const bool turned = t.rows > t.cols;  // the caller's rows run along n
  const int across = (turned ? t.mp : t.np) / 64;
  const int r0 = b / across * 64, c0 = b % across * 64;

  // |G|: every block adds the same partial sums in the same order
  double s = 0.0;
  for (int k = tid; k < t.parts; k += 256) s += t.part[k];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  const double norm = sqrt(red[0] + red[1] + red[2] + red[3]);
  const float scale = norm <= (double)tab.eps ? (float)(kScaleX / (double)tab.eps)
                                              : (float)(kScaleX / norm);  // NaN stays
  f16 *const to_hi = ws_xt(t, 0, 0), *const to_lo = ws_xt(t, 0, 1);
  const int r8 = tid >> 3, c8 = (tid & 7) * 8;
#pragma unroll
  for (int h = 0; h < 64; h += 32) {
    const int r = r0 + r8 + h, c = c0 + c8;
    float u[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < t.rows && c < t.cols) load_u(tab, t, (size_t)r * t.cols + c, t.cols - c, u);
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f16 x, y;
      split(u[k] * scale, x, y);
      hi[k] = x;
      lo[k] = y;
      tile[r8 + h][c8 + k] = (uint32_t)__builtin_bit_cast(uint16_t, x) |
                             ((uint32_t)__builtin_bit_cast(uint16_t, y) << 16);
    }
    if (turned) {
      const size_t at = place(rows_xt(t.np), r, c);
      *(f16x8*)(to_hi + at) = hi;
      *(f16x8*)(to_lo + at) = lo;
    }
  }
  if (turned) return;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 64; h += 32) {
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t v = tile[c8 + k][r8 + h];
      hi[k] = __builtin_bit_cast(f16, (uint16_t)(v & 0xffff));
      lo[k] = __builtin_bit_cast(f16, (uint16_t)(v >> 16));
    }
    const size_t at = place(rows_xt(t.np), c0 + r8 + h, r0 + c8);
    *(f16x8*)(to_hi + at) = hi;
    *(f16x8*)(to_lo + at) = lo;
  }
}

// ---- products -----------------------------------------------------------------

enum { TO_A = 0, TO_B = 1, TO_X = 2, TO_END = 3 };

// A block's tile and the WM x WN waves that share it.
template <int TM_, int TN_, int WM_, int WN_>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WAVES = WM * WN;
  static constexpr int FM = TM / WM / 32, FN = TN / WN / 32;
};

// Where in its 64 bytes of LDS a row keeps a 16-byte chunk: those of 16
// neighbouring rows fall on all 64 banks.
__device__ __forceinline__ int swizzle(int chunk, int row) { return chunk ^ ((row >> 2) & 3); }

typedef __attribute__((address_space(3))) void lds_void;

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// All waves' LDS reads so far are over and their finished copies can be seen.
__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 8 values of a column: a lane gets those of its own column from two times 4
// rows, whose 4 x 16 values the 16 lanes around it address, 4 values each.
__device__ __forceinline__ f16x8 read_turned(const f16* at, int rows4) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef __fp16 h4 __attribute__((vector_size(8)));
  typedef __attribute__((address_space(3))) h4 lds_h4;
  const f16x4 a = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_h4*)at));
  const f16x4 b =
      __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_h4*)(at + rows4)));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
#else
  return f16x8{};
#endif
}

// acc += P Q^T over K: P has TM rows, Q TN rows, each as two planes, hi and lo.
// S stages of operands in LDS: the copies of S - 1 steps are under way while a
// step is multiplied, and a step waits for its own copies alone.
//
// A step is cut into units of some matrix instructions.  Between them a unit
// sends its share of the copies and reads the next unit's fragments, across
// the steps' borders too: a wave issues in order, and a row of reads in front
// of the multiplications keeps the matrix core idle as long as LDS takes to
// accept them (64 x 64 tiles: 1040 cycles a step, 400 of them multiplying).
// The scheduling barriers keep the compiler from gathering them again.
template <class T, int BK, int S, bool TURNED>
__device__ __forceinline__ void product(const f16* const (&P)[2], int rows_p, const f16* const (&Q)[2],
                                        int rows_q, int K, f16* lds, f32x16 (&acc)[T::FM][T::FN]) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass does not know buffer resources
  constexpr int STAGE = 2 * (T::TM + T::TN) * BK;
  constexpr int LA = T::TM * BK / 512 / T::WAVES, LB = T::TN * BK / 512 / T::WAVES;
  constexpr int LOADS = 2 * (LA + LB);  // copies per wave and stage
  constexpr int KG = BK / 16, UNITS = KG * T::FM;
  // units that send copies: with two stages these are waited for at this
  // step's end, and leave early
  constexpr int SPREAD = S == 2 ? (UNITS + 3) / 4 : UNITS;
  static_assert(KG % 2 == 0, "fragments alternate between two sets");
  static_assert(T::TM * 32 % (512 * T::WAVES) == 0 && T::TN * 32 % (512 * T::WAVES) == 0,
                "every wave copies as much of a panel");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave / T::WN) * (T::TM / T::WM), wn = (wave % T::WN) * (T::TN / T::WN);

  // 1 KB, 16 rows of a panel, to a copy.  A lane's 16 bytes land at 16 * lane,
  // so the swizzle is in the place they come from; the rest of it is scalar.
  __amdgpu_buffer_rsrc_t rp[2], rq[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    rp[p] = __builtin_amdgcn_make_buffer_rsrc((void*)P[p], 0, -1, 0x00020000);
    rq[p] = __builtin_amdgcn_make_buffer_rsrc((void*)Q[p], 0, -1, 0x00020000);
  }
  const int from = (lane >> 2) * 64 + swizzle(lane & 3, lane >> 2) * 16;
  auto copy = [&](int k0, f16* s, int which) {
    const bool first = which < 2 * LA;
    const int w = first ? which : which - 2 * LA, l = first ? LA : LB;
    const int p = w / l, i = w % l;
    const auto plane = first ? rp[p] : rq[p];
    f16* to = s + (first ? p * T::TM : 2 * T::TM + p * T::TN) * BK;
    if (TURNED) {
      const int panel = (wave * l + i) / (BK / 16), piece = (wave * l + i) % (BK / 16);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          plane, (lds_void*)(to + (panel * BK + piece * 16) * 32), 16, lane * 16,
          (panel * (first ? rows_p : rows_q) + k0 + piece * 16) * 64, 0, 0);
      return;
    }
    const int panel = i / (l / (BK / 32)), j = i % (l / (BK / 32));
    const int rows = first ? T::TM : T::TN, piece = wave * (l / (BK / 32)) + j;
    const int panels = (k0 >> 5) + panel;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        plane, (lds_void*)(to + panel * rows * 32 + piece * 512), 16, from,
        panels * (first ? rows_p : rows_q) * 64 + piece * 1024, 0, 0);
  };
  const int column = ((lane >> 5) * 8 + ((lane & 15) >> 2)) * 32 + (lane & 16) + (lane & 3) * 4;
  auto read = [&](const f16* plane, int rows, int row, int kk) {
    if (TURNED) return read_turned(plane + ((row >> 5) * BK + kk * 16) * 32 + column, 4 * 32);
    return *(const f16x8*)(plane + (kk >> 1) * rows * 32 + row * 32 +
                           swizzle((kk & 1) * 2 + (lane >> 5), row) * 8);
  };
  f16x8 a[2][2], b[2][2][T::FN];
  // Reads and multiplications of a unit, in the order in which the fragments
  // are needed: lo hi, hi lo, hi hi.
  auto read_one = [&](const f16* s, int u, int which) {
    const int kg = u / T::FM, f = u % T::FM;
    const bool late = which > T::FN && f == 0;  // the planes of the second product
    const int pb = late ? 1 : 0;
    if (which == 0 || which == (f == 0 ? T::FN + 1 : 1)) {
      const int p = which == 0 ? 1 : 0;
      a[u & 1][p] = read(s + p * T::TM * BK, T::TM, wm + f * 32 + (lane & 31), kg);
    } else {
      const int g = late ? which - T::FN - 2 : which - 1;
      b[kg & 1][pb][g] = read(s + (2 * T::TM + pb * T::TN) * BK, T::TN,
                              wn + g * 32 + (lane & 31), kg);
    }
  };
  constexpr int MULS = 3 * T::FN;
  auto multiply_one = [&](int u, int which) {
    const int kg = u / T::FM, f = u % T::FM;
    const int c = which / T::FN, g = which % T::FN;
    const int pa = c == 0 ? 1 : 0, pb = c == 1 ? 1 : 0;
    acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[u & 1][pa], b[kg & 1][pb][g], acc[f][g],
                                                       0, 0, 0);
  };

  // the last unit's copies that go behind the wait after its first instruction
  constexpr int LAST = SPREAD < UNITS ? 0 : LOADS - (UNITS - 1) * LOADS / UNITS;
  constexpr int REST = LAST - LAST / MULS;

  const int steps = K / BK;
#pragma unroll
  for (int i = 0; i < S - 1; ++i)
    if (i < steps) {
#pragma unroll
      for (int c = 0; c < LOADS; ++c) copy(i * BK, lds + i * STAGE, c);
    }
  if (S - 1 <= steps)
    wait_loads<LOADS*(S - 2)>();
  else
    wait_loads<0>();
  block_barrier();
  [&](const f16* __restrict s) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 2 + 2 * T::FN; ++r) read_one(s, 0, r);
  }(lds);
  int cur = 0, free = (S - 1) * STAGE;  // the stage read, and the one to fill
  // (Stages are distinct memory as far as the compiler is told, or it lets every
  // turned read wait for all copies.)
  auto step = [&](auto more, int i, const f16* __restrict now, const f16* __restrict then,
                  f16* __restrict later) __attribute__((always_inline)) {
    constexpr bool MORE = decltype(more)::value;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const bool last = u + 1 == UNITS;
      const int reads = 2 + ((u + 1) % T::FM == 0 ? 2 * T::FN : 0);
      const int c0 = u < SPREAD ? u * LOADS / SPREAD : LOADS;
      const int copies = u < SPREAD ? (u + 1) * LOADS / SPREAD - c0 : 0;
#pragma unroll
      for (int m = 0; m < MULS; ++m) {
        multiply_one(u, m);
        if (MORE) {
#pragma unroll
          for (int c = m * copies / MULS; c < (m + 1) * copies / MULS; ++c)
            copy((i + S - 1) * BK, later, c0 + c);
        }
        if (last && m == 0 && (MORE || i + 1 < steps)) {
          // of this step's own copies, REST are still to be sent
          wait_loads<MORE ? LOADS*(S - 2) - REST : 0>();
          // (naming the stages keeps their reads and copies on their sides)
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::"s"((lds_void*)now),
                       "s"((lds_void*)then), "s"((lds_void*)later)
                       : "memory");
        }
        if (!last || MORE || i + 1 < steps) {
          // two at a time: what LDS delivers during a matrix instruction
          const int r1 = m + 1 == MULS || 2 * m + 2 > reads ? reads : 2 * m + 2;
#pragma unroll
          for (int r = 2 * m; r < r1; ++r) read_one(last ? then : now, (u + 1) % UNITS, r);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto turn_step = [&](auto more, int i) __attribute__((always_inline)) {
    const int next = cur + STAGE == S * STAGE ? 0 : cur + STAGE;
    step(more, i, lds + cur, lds + next, lds + free);
    free = cur;
    cur = next;
  };
  int i = 0;
  for (; i + S - 1 < steps; ++i) turn_step(std::true_type{}, i);
  for (; i < steps; ++i) turn_step(std::false_type{}, i);
#endif
}

// The result, or the weights' update, for 8 values of one row of the caller's.
__device__ __forceinline__ void deliver(const Table& tab, const Mat& t, int row, int col, float* v) {
  if (row >= t.rows || col >= t.cols) return;
  const size_t at = (size_t)row * t.cols + col;
  if (t.mom) {
    float w[8];
    load8(t.w, at, tab.wtype, t.cols - col, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = tab.keep * w[k] - t.step * v[k];
  }
  store8(t.w, at, tab.wtype, t.cols - col, v);
}

constexpr int kPieceLd = 36;                  // floats from row to row of a piece in LDS
constexpr int kPieceHalfs = 32 * kPieceLd * 2;

// A's values at a piece of B, 8 to a lane, twice.
struct Old {
  f16x8 hi[2], lo[2];
};

__device__ __forceinline__ Old load_old(const Mat& t, int i0, int j0) {
  const int lane = threadIdx.x & 63, r4 = lane >> 2, c8 = (lane & 3) * 8;
  Old o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const size_t at = place(t.ma, j0 + h * 16 + r4, i0 + c8);
    o.hi[h] = *(const f16x8*)(ws_a(t, 0) + at);
    o.lo[h] = *(const f16x8*)(ws_a(t, 1) + at);
  }
  return o;
}

// The 32 x 32 piece at (i0, j0) of A, B, X' or the result: kb * (product), for B
// with ka * A and kd on the diagonal besides.  B holds a I + b A + c A^2, for
// then B X is X' and nothing is read here to make it.  (With a X added here
// instead, 1000 x 4000 twice took 546 us for 532.)
// A lane holds 4 neighbouring rows of a column, 4 times; the piece goes through
// the wave's own LDS so that every global access is 16 bytes per lane, side by
// side.  (Written from the registers, 2 and 8 bytes per lane, the tiles' ends
// took 8 us of 31 at 128 x 128 and 100 us of 360 at 256 x 256.)
template <int TO>
__device__ __forceinline__ void finish(const Table& tab, const Mat& t, int turn, float ka, float kb,
                                       float kd, int i0, int j0, bool mirror, const f32x16& acc,
                                       const Old& old, float* lds) {
  const int lane = threadIdx.x & 63;
  const bool turned = t.rows > t.cols;
  f16* ch = TO == TO_A ? ws_a(t, 0) : TO == TO_B ? ws_b(t, 0) : ws_xt(t, turn ^ 1, 0);
  f16* cl = TO == TO_A ? ws_a(t, 1) : TO == TO_B ? ws_b(t, 1) : ws_xt(t, turn ^ 1, 1);
  const int r4 = lane >> 2, c8 = (lane & 3) * 8;
  const int rows_j = TO == TO_A || TO == TO_B ? t.ma : rows_xt(t.np);  // of a plane whose rows are columns j
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *(float4*)(lds + (lane & 31) * kPieceLd + q * 8 + (lane >> 5) * 4) =
        make_float4(kb * acc[q * 4], kb * acc[q * 4 + 1], kb * acc[q * 4 + 2], kb * acc[q * 4 + 3]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = h * 16 + r4;
    float* p = lds + j * kPieceLd + c8;
    const float4 x = *(const float4*)p, y = *(const float4*)(p + 4);
    float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    if (TO == TO_B) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] += ka * ((float)old.hi[h][k] + (float)old.lo[h][k]);
        if (i0 + c8 + k == j0 + j) v[k] += kd;
      }
    }
    if (TO == TO_END) {
      if (turned) {
        deliver(tab, t, j0 + j, i0 + c8, v);
      } else {
        *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      continue;
    }
    f16x8 hi, lo;
    uint32_t both[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f16 a, b;
      split(v[k], a, b);
      hi[k] = a;
      lo[k] = b;
      both[k] = (uint32_t)__builtin_bit_cast(uint16_t, a) |
                ((uint32_t)__builtin_bit_cast(uint16_t, b) << 16);
    }
    const size_t at = place(rows_j, j0 + j, i0 + c8);
    *(f16x8*)(ch + at) = hi;
    *(f16x8*)(cl + at) = lo;
    *(uint4*)p = make_uint4(both[0], both[1], both[2], both[3]);
    *(uint4*)(p + 4) = make_uint4(both[4], both[5], both[6], both[7]);
  }
  if (TO == TO_X || !mirror || (TO == TO_END && turned)) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 16 + r4;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = lds[(c8 + k) * kPieceLd + i];
    if (TO == TO_END) {
      deliver(tab, t, i0 + i, j0 + c8, v);
      continue;
    }
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t u = __float_as_uint(v[k]);
      hi[k] = __builtin_bit_cast(f16, (uint16_t)(u & 0xffff));
      lo[k] = __builtin_bit_cast(f16, (uint16_t)(u >> 16));
    }
    const size_t at = place(t.ma, i0 + i, j0 + c8);
    *(f16x8*)(ch + at) = hi;
    *(f16x8*)(cl + at) = lo;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Blocks go round the 8 XCDs in turn, each with an L2 of its own.  Every XCD
// takes a run of neighbouring tiles of a matrix instead, and a run is about
// square, so that its blocks share operands in their L2.
__device__ __forceinline__ int xcd_order(int block, int blocks) {
  const int x = block & 7, each = blocks >> 3, more = blocks & 7;
  return x * each + (x < more ? x : more) + (block >> 3);
}

__device__ __forceinline__ int run_height(int tiles, int rows) {
  const int g = (int)sqrtf((float)(tiles >> 3));
  return g < 1 ? 1 : g > rows ? rows : g;
}

// Strips of g tile rows, column by column.
__device__ __forceinline__ void tile_of_grid(int b, int rows, int cols, int& ti, int& tj) {
  const int g = run_height(rows * cols, rows), strip = b / (g * cols);
  const int h = rows - strip * g < g ? rows - strip * g : g;  // of this strip
  b -= strip * g * cols;
  ti = strip * g + b % h;
  tj = b / h;
}

// The same on the tiles with ti <= tj: a strip begins with a triangle.
__device__ __forceinline__ void tile_of_triangle(int b, int rows, int& ti, int& tj) {
  const int g = run_height(rows * (rows + 1) / 2, rows);
  int top = 0, h = g;
  for (;; top += g) {
    h = rows - top < g ? rows - top : g;
    const int count = h * (h + 1) / 2 + h * (rows - top - h);
    if (b < count) break;
    b -= count;
  }
  const int corner = h * (h + 1) / 2;
  if (b >= corner) {
    ti = top + (b - corner) % h;
    tj = top + h + (b - corner) / h;
  } else {
    int c = 0;
    while ((c + 1) * (c + 2) / 2 <= b) ++c;
    ti = top + b - c * (c + 1) / 2;
    tj = top + c;
  }
}

constexpr int most(int a, int b) { return a > b ? a : b; }

// One tile of A, B, X' or the result.  Bound by the matrix rate where there are
// tiles enough (4096 x 4096: B X 301 us, 1.37 PFLOP/s; A 180 us, 1.14), by the
// time of a copy into LDS and by the tiles' ends where there are not (1024 x
// 4096: B X 26 us, 0.98 PFLOP/s, A 17 and 7 to join).
template <class T, int BK, int S, int TO>
__global__ __launch_bounds__(T::WAVES * 64) void flowml_ns_product(Table tab, int turn, float ka,
                                                                  float kb, float kd) {
  constexpr bool SYM = TO == TO_A || TO == TO_B;
  constexpr int HALFS = most(2 * (T::TM + T::TN) * BK * S, T::WAVES * kPieceHalfs);
  __shared__ __align__(16) f16 lds[HALFS];
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  int ti, tj, tile, part = 0;
  if (SYM) {
    const int mt = tiles_of(t.mp, T::TM), tiles = mt * (mt + 1) / 2;
    tile = xcd_order(blockIdx.x - t.first, tiles * (TO == TO_A ? t.split : 1));
    if (TO == TO_A) {
      part = tile / tiles;
      tile -= part * tiles;
    }
    tile_of_triangle(tile, mt, ti, tj);
  } else {
    const int mt = t.mp / T::TM, nt = t.np / T::TN;
    tile = xcd_order(blockIdx.x - t.first, mt * nt);
    tile_of_grid(tile, mt, nt, ti, tj);
  }
  const int i0 = ti * T::TM, j0 = tj * T::TN;

  const f16* P[2];
  const f16* Q[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (TO == TO_A) {
      P[p] = ws_xt(t, turn, p) + place(rows_xt(t.np), 0, i0);
      Q[p] = ws_xt(t, turn, p) + place(rows_xt(t.np), 0, j0);
    } else {
      P[p] = (TO == TO_B ? ws_a(t, p) : ws_b(t, p)) + i0 * 32;
      Q[p] = (TO == TO_B ? ws_a(t, p) : ws_xt(t, turn, p)) + j0 * 32;
    }
  }
  int K = TO == TO_A ? t.np : t.mp;
  const int rows_p = TO == TO_A ? rows_xt(t.np) : t.ma, rows_q = TO == TO_B ? t.ma : rows_xt(t.np);
  if (TO == TO_A && t.split > 1) {
    const int k0 = part * t.kpart;
    K = K - k0 < t.kpart ? K - k0 : t.kpart;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      P[p] += (size_t)k0 * 32;
      Q[p] += (size_t)k0 * 32;
    }
  }

  f32x16 acc[T::FM][T::FN];
#pragma unroll
  for (int f = 0; f < T::FM; ++f)
#pragma unroll
    for (int g = 0; g < T::FN; ++g)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[f][g][r] = 0.f;
  product<T, BK, S, TO == TO_A>(P, rows_p, Q, rows_q, K, lds, acc);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool mirror = !SYM || ti != tj;
  // a tile on the diagonal is its own mirror image: one writer for each value,
  // since (i, j) and (j, i) may differ in the last bit
  block_barrier();
  float* piece = (float*)(lds + wave * kPieceHalfs);
  const int wi = i0 + (wave / T::WN) * (T::TM / T::WM), wj = j0 + (wave % T::WN) * (T::TN / T::WN);
  if (TO == TO_A && t.split > 1) {
    const int mt = tiles_of(t.mp, T::TM), tiles = mt * (mt + 1) / 2;
    float* to = t.sums + ((size_t)part * tiles + tile) * (T::TM * T::TN);
#pragma unroll
    for (int f = 0; f < T::FM; ++f)
#pragma unroll
      for (int g = 0; g < T::FN; ++g) {
        const int pi = (wi - i0) / 32 + f, pj = (wj - j0) / 32 + g;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(float4*)(to + (pi * (T::TN / 32) + pj) * 1024 + q * 256 + lane * 4) =
              make_float4(acc[f][g][q * 4], acc[f][g][q * 4 + 1], acc[f][g][q * 4 + 2],
                          acc[f][g][q * 4 + 3]);
      }
    return;
  }
  // a piece's values of A are under way while the piece before it is finished
  Old old = {}, next = {};
  if (TO == TO_B) old = load_old(t, wi, wj);
#pragma unroll
  for (int f = 0; f < T::FM; ++f)
#pragma unroll
    for (int g = 0; g < T::FN; ++g) {
      const int p = f * T::FN + g + 1;
      if (TO == TO_B && p < T::FM * T::FN)
        next = load_old(t, wi + p / T::FN * 32, wj + p % T::FN * 32);
      finish<TO>(tab, t, turn, ka, kb, kd, wi + f * 32, wj + g * 32, mirror, acc[f][g], old, piece);
      old = next;
      __builtin_amdgcn_sched_barrier(0);
    }
}

// A from the sums of its parts of K, one 32 x 32 piece to a wave, parts in order
// (7 us for 72 tiles of 128 in 3 parts, 14 MB; a launch is 3 of them).
__global__ __launch_bounds__(256) void flowml_ns_join(Table tab, int side, float kb) {
  __shared__ __align__(16) f16 lds[4 * kPieceHalfs];
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int mt = tiles_of(t.mp, side), tiles = mt * (mt + 1) / 2;
  const int across = side / 32, pieces = across * across;
  const int at = (blockIdx.x - t.first) * 4 + wave, tile = at / pieces, piece = at - tile * pieces;
  if (tile >= tiles) return;
  int ti, tj;
  tile_of_triangle(tile, mt, ti, tj);
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll 4
  for (int s = 0; s < t.split; ++s) {
    const float* from =
        t.sums + (((size_t)s * tiles + tile) * pieces + piece) * 1024 + lane * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 v = *(const float4*)(from + q * 256);
      acc[q * 4] += v.x;
      acc[q * 4 + 1] += v.y;
      acc[q * 4 + 2] += v.z;
      acc[q * 4 + 3] += v.w;
    }
  }
  const int pi = piece / across, pj = piece - pi * across;
  finish<TO_A>(tab, t, 0, 0.f, kb, 0.f, ti * side + pi * 32, tj * side + pj * 32, ti != tj, acc, Old{},
               (float*)(lds + wave * kPieceHalfs));
}

// ---- matrices that one block holds ----------------------------------------------

// What fits 160 KB of LDS (a small network's layers; 64 x 416, 128 x 160): the
// whole iteration in one launch, with iterates as pairs of fp16.  Latency
// bounds it: three or four barriers a step, chains of matrix instructions
// between them (five steps of 41 x 128: 21 us, 64 x 256: 33 us).
//
// Only the transpose of X is kept.  B X reads its rows; X X^T takes columns,
// through LDS reads that transpose: 16 lanes load 4 rows of 16 values, and
// each gets a column.  Rows lie 16 bytes more than a multiple of 64 apart, so
// that 16 neighbouring rows' chunks fall on all 64 banks.

constexpr int kSmallM = 128, kSmallThreads = 512, kSmallWaves = kSmallThreads / 64;
constexpr size_t kSmallLds = 160 * 1024 - 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// pieces of 16 on the shorter side: 2, 4 or 8
__host__ __device__ inline int small_pieces(int m) { return m <= 32 ? 2 : m <= 64 ? 4 : 8; }

size_t small_lds(int m, int n) {
  const size_t mt = small_pieces(m), mp = mt * 16, np = (n + 31) / 32 * 32;
  return 2 * (np + (mt == 8 ? 1 : 2) * mp) * (mp + 8) * sizeof(f16);
}

bool small_fits(int m, int n) { return m <= kSmallM && n < 4096 && small_lds(m, n) <= kSmallLds; }

// A lane's 8 values of a chunk of 32 in a row of 16 rows' operand, both planes.
struct Halves {
  f16x8 hi, lo;
};

__device__ __forceinline__ Halves small_read(const f16* plane, int low, int at) {
  return {*(const f16x8*)(plane + at), *(const f16x8*)(plane + low + at)};
}

// the same of 32 rows from `k` on, columns i to i + 15
__device__ __forceinline__ f16x8 read_columns(const f16* plane, int ld, int k, int i, int lane) {
  return read_turned(
      plane + (k + (lane >> 4) * 8 + ((lane & 15) >> 2)) * ld + i + (lane & 3) * 4, 4 * ld);
}

__device__ __forceinline__ Halves small_columns(const f16* plane, int low, int ld, int k, int i,
                                                int lane) {
  return {read_columns(plane, ld, k, i, lane), read_columns(plane + low, ld, k, i, lane)};
}

// acc += x y; ALL: the product of the lower halves too, which counts where few
// values are summed (17 columns: 1.5 times fp32's error without, 1.2 with)
template <bool ALL>
__device__ __forceinline__ void small_multiply(const Halves& x, const Halves& y, f32x4& acc) {
  if (ALL) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.lo, y.lo, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.lo, y.hi, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.hi, y.lo, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.hi, y.hi, acc, 0, 0, 0);
}

struct Poly {
  float a, b, c, scale_b;
  int steps;
};

// U for 8 values side by side; `update`: the momentum is moved on, too
__device__ __forceinline__ void small_u(const Table& tab, const Mat& t, bool update, size_t at,
                                        int left, float* u) {
  load8(t.g, at, tab.gtype, left, u);
  if (t.mom) {
    float m[8];
    load8(t.mom, at, T_F32, left, m);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (update) m[k] = tab.mu * m[k] + u[k];
      u[k] = tab.nesterov ? u[k] + tab.mu * m[k] : m[k];
    }
    if (update) store8(t.mom, at, T_F32, left, m);
  }
}

template <int MT>
__device__ __forceinline__ void small_matrix(const Table& tab, const Mat& t, const Poly& poly,
                                             f16* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int mp = MT * 16, ld = mp + 8, KC = MT / 2;  // KC: chunks of 32 in m
  constexpr bool ALL = MT == 2, APART = MT < 8;          // B apart from A
  const int np = (t.n + 31) / 32 * 32;
  const int lo_x = np * ld;
  constexpr int lo_a = mp * ld;
  f16* XT = lds;            // np rows
  f16* A = XT + 2 * lo_x;   // mp rows
  f16* B = APART ? A + 2 * lo_a : A;
  const bool turned = t.rows > t.cols;

  // Pieces of 8 values of the caller's rows.  Neighbouring lanes take
  // neighbouring m: so their 2-byte writes do not meet in a bank.
  const int per_row = (t.cols + 7) / 8, pieces = t.rows * per_row;
  auto piece = [&](int p, int& r, int& c) {
    if (turned) {
      r = p / per_row;
      c = (p - r * per_row) * 8;
    } else {
      c = p / t.rows;
      r = p - c * t.rows;
      c *= 8;
    }
  };
  double sum = 0.0;
  for (int p = tid; p < pieces; p += kSmallThreads) {
    int r, c;
    piece(p, r, c);
    float u[8];
    small_u(tab, t, true, (size_t)r * t.cols + c, t.cols - c, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += (double)u[k] * (double)u[k];
  }
  uint4* clear = (uint4*)XT;
  for (int i = tid; i < lo_x / 4; i += kSmallThreads) clear[i] = make_uint4(0, 0, 0, 0);
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  __shared__ double red[kSmallWaves];
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int k = 0; k < kSmallWaves; ++k) total += red[k];
  const double norm = sqrt(total);
  const float scale = norm <= (double)tab.eps ? (float)(kScaleX / (double)tab.eps)
                                              : (float)(kScaleX / norm);
  for (int p = tid; p < pieces; p += kSmallThreads) {
    int r, c;
    piece(p, r, c);
    float u[8];
    small_u(tab, t, false, (size_t)r * t.cols + c, t.cols - c, u);
    f16x8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f16 x, y;
      split(u[k] * scale, x, y);
      hi[k] = x;
      lo[k] = y;
    }
    if (turned) {  // what load8 puts behind the row's end is 0
      *(f16x8*)(XT + r * ld + c) = hi;
      *(f16x8*)(XT + lo_x + r * ld + c) = lo;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < t.cols) {
          XT[(c + k) * ld + r] = hi[k];
          XT[lo_x + (c + k) * ld + r] = lo[k];
        }
    }
  }
  __syncthreads();

  const float sx = kScaleX, sa = kScaleA, sb = poly.scale_b;
  const float to_a = sa / (sx * sx), b_old = poly.b * sb / sa, b_new = poly.c * sb / (sa * sa);
  const float to_x = 1.f / sb, to_end = 1.f / (sb * sx);
  const int row = (lane >> 4) * 4, col = lane & 15;  // 4 rows of a column to a lane
  const int from = (lane >> 4) * 8;                  // of an operand's chunk of 32
  // A and B, which is a I + b A + c A^2: AW pieces of a row of pieces to a wave
  constexpr int AW = MT * MT / kSmallWaves < 1 ? 1 : MT * MT / kSmallWaves;
  const int ai = wave * AW / MT * 16, aj = wave * AW % MT * 16;
  const bool has_a = wave * AW < MT * MT;
  auto put = [&](f16* plane, int low, int at, const f32x4& v) {
    f16x4 h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f16 x, y;
      split(v[r], x, y);
      h[r] = x;
      l[r] = y;
    }
    *(f16x4*)(plane + at) = h;
    *(f16x4*)(plane + low + at) = l;
  };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < poly.steps; ++s) {
    // A and B are kept as their transposes, one bit apart at most
    f32x4 v[AW];
#pragma unroll
    for (int q = 0; q < AW; ++q) v[q] = zero;
    if (has_a) {
#pragma unroll 2
      for (int k = 0; k < np; k += 32) {
        const Halves x = small_columns(XT, lo_x, ld, k, ai, lane);
#pragma unroll
        for (int q = 0; q < AW; ++q)
          small_multiply<ALL>(x, small_columns(XT, lo_x, ld, k, aj + q * 16, lane), v[q]);
      }
#pragma unroll
      for (int q = 0; q < AW; ++q)
        put(A, lo_a, (aj + q * 16 + col) * ld + ai + row, v[q] * to_a);
    }
    __syncthreads();
    if (has_a) {
      Halves x[KC];
#pragma unroll
      for (int k = 0; k < KC; ++k) x[k] = small_read(A, lo_a, (ai + col) * ld + from + k * 32);
#pragma unroll
      for (int q = 0; q < AW; ++q) {
        const int at = (aj + q * 16 + col) * ld + ai + row;
        const f16x4 h = *(const f16x4*)(A + at), l = *(const f16x4*)(A + lo_a + at);
        f32x4 w = zero;
#pragma unroll
        for (int k = 0; k < KC; ++k)
          small_multiply<ALL>(
              x[k], small_read(A, lo_a, (aj + q * 16 + col) * ld + from + k * 32), w);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[q][r] = b_new * w[r] + b_old * ((float)h[r] + (float)l[r]);
          if (ai + row + r == aj + q * 16 + col) v[q][r] += poly.a * sb;
        }
      }
    }
    if (!APART) __syncthreads();
    if (has_a) {
#pragma unroll
      for (int q = 0; q < AW; ++q)
        put(B, lo_a, (aj + q * 16 + col) * ld + ai + row, v[q]);
    }
    __syncthreads();
    // X' = B X; a wave takes whole rows of X^T, which nobody else reads here
    for (int j = wave * 16; j < np; j += kSmallWaves * 16) {
      Halves y[KC];
#pragma unroll
      for (int k = 0; k < KC; ++k) y[k] = small_read(XT, lo_x, (j + col) * ld + from + k * 32);
      f32x4 x[MT];
#pragma unroll
      for (int p = 0; p < MT; ++p) {
        x[p] = zero;
#pragma unroll
        for (int k = 0; k < KC; ++k)
          small_multiply<ALL>(small_read(B, lo_a, (p * 16 + col) * ld + from + k * 32), y[k], x[p]);
      }
      if (s + 1 < poly.steps) {
#pragma unroll
        for (int p = 0; p < MT; ++p) put(XT, lo_x, (j + col) * ld + p * 16 + row, x[p] * to_x);
      } else {
#pragma unroll
        for (int p = 0; p < MT; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = p * 16 + row + r;
            if (i < t.m && j + col < t.n) {
              const size_t at =
                  turned ? (size_t)(j + col) * t.cols + i : (size_t)i * t.cols + j + col;
              float o = to_end * x[p][r];
              if (t.mom) o = tab.keep * load_as(t.w, at, tab.wtype) - t.step * o;
              store_as(t.w, at, tab.wtype, o);
            }
          }
      }
    }
    __syncthreads();
  }
}

// Shorter sides up to 16, longer ones of any length.  The polynomials of A
// commute, so the iteration needs X only at its ends: with A_0 = U U^T / |U|^2,
//
//   Q = a I + b A + c A^2     P <- Q P     A <- Q A Q      O = P U / |U|
//
// on 16 x 16 matrices.  A squares the condition of U, which 64 bits bear (in
// fp32 this form is 10 to 100 times less exact than the other), but not for any
// number of steps: where U has no part, A is rounding noise, 2^-53 and as often
// below 0 as above, which a step multiplies by a^2 <= 91 and of which, below 0, Q
// makes more without end.  So after a run of 5 steps (2^-53 a^10: 3e-11 for a =
// 3.44) X <- P X is written out, in fp64, and the next run begins with A = X X^T:
// as exact as steps on X itself in fp64.  Longer ones take a block for every 256
// columns or more, 64 blocks at most; the sums of A_0 are then made by a launch
// of their own, and every block adds them and iterates for itself.  (5 x 1024:
// one block 15 us, four 14.)

constexpr int kThinM = 16, kThinLd = 17, kThinRun = 5;
typedef double f64x4 __attribute__((ext_vector_type(4)));

// Place of (i, j) in the caller's matrix, i on its shorter side.
__device__ __forceinline__ size_t thin_place(const Mat& t, int i, int j) {
  return t.rows > t.cols ? (size_t)j * t.cols + i : (size_t)i * t.cols + j;
}

// Where X lies between two runs: columns of m values.
__device__ __forceinline__ double* thin_x(const Mat& t, int i, int j) {
  return (double*)t.ws + (size_t)j * t.m + i;
}

template <typename G>
using Held = std::conditional_t<std::is_same<G, double>::value, double, float>;

// U(i, j), or X(i, j) for G = double.  Places outside are read at the nearest one
// inside and dropped: no branch, so that many loads are under way.
template <typename G>
__device__ __forceinline__ Held<G> thin_u(const Table& tab, const Mat& t, bool update, int i, int j,
                                          int end) {
  const bool in = i < t.m && j < end;
  i = i < t.m ? i : t.m - 1;
  j = j < end ? j : end - 1;
  if constexpr (std::is_same<G, double>::value) {
    const double x = *thin_x(t, i, j);
    return in ? x : 0.0;
  }
  const size_t at = thin_place(t, i, j);
  float u = (float)((const G*)t.g)[at];
  if (t.mom) {
    float m = t.mom[at];
    if (update) {
      m = tab.mu * m + u;
      if (in) t.mom[at] = m;
    }
    u = tab.nesterov ? u + tab.mu * m : m;
  }
  return in ? u : 0.f;
}

// f(a value of the type that is read): the type is asked for once, not at every
// load, where the branches would let one load follow the other.
template <typename F>
__device__ __forceinline__ void by_type(int type, F f) {
  if (type == T_F32)
    f(0.f);
  else if (type == T_BF16)
    f((__bf16)0.f);
  else if (type == T_F16)
    f((f16)0.f);
  else
    f(0.0);
}

// this block's share of U U^T, or of X X^T in a later run, into 256 doubles of LDS
__device__ __forceinline__ void thin_gram(const Table& tab, const Mat& t, int run, int chunk,
                                          double* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int WAVES = kSmallWaves;
  f64x4 acc = {0.0, 0.0, 0.0, 0.0};
  const int end = t.n - chunk * t.chunk < t.chunk ? t.n : (chunk + 1) * t.chunk;
  by_type(run ? T_F64 : tab.gtype, [&](auto like) {
    for (int j = chunk * t.chunk + wave * 16; j < end; j += 4 * WAVES * 16) {
      Held<decltype(like)> u[4][4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          u[h][e] = thin_u<decltype(like)>(tab, t, true, lane & 15,
                                           j + h * WAVES * 16 + (lane >> 4) * 4 + e, end);
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (j + h * WAVES * 16 < end) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)u[h][e], (double)u[h][e], acc, 0, 0, 0);
        }
    }
  });
#pragma unroll
  for (int r = 0; r < 4; ++r) lds[wave * 256 + (r * 4 + (lane >> 4)) * 16 + (lane & 15)] = acc[r];
  __syncthreads();
  double s = 0.0;
  if (tid < 256)
    for (int k = 0; k < WAVES; ++k) s += lds[k * 256 + tid];
  __syncthreads();
  if (tid < 256) lds[tid] = s;
  __syncthreads();
}

__global__ __launch_bounds__(kSmallThreads) void flowml_ns_thin_gram(Table tab, int run) {
  __shared__ double lds[kSmallThreads / 64 * 256];
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int chunk = blockIdx.x - t.first;
  if (t.parts == 1) return;  // one block does it all
  thin_gram(tab, t, run, chunk, lds);
  if (threadIdx.x < 256) t.part[(size_t)chunk * 256 + threadIdx.x] = lds[threadIdx.x];
}

// One run of steps, from A's sums to P applied.
__device__ __forceinline__ void thin_run(const Table& tab, const Mat& t, const Poly& poly, int run,
                                         int chunk, double* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int WAVES = kSmallWaves;
  const int left = poly.steps - run * kThinRun, steps = left < kThinRun ? left : kThinRun;
  const bool last = left <= kThinRun;
  if (t.parts == 1) {
    thin_gram(tab, t, run, 0, lds);
  } else {
    double s = 0.0;
    if (tid < 256) {
      for (int k = 0; k < t.parts; ++k) s += t.part[(size_t)k * 256 + tid];
      lds[tid] = s;
    }
    __syncthreads();
  }
  double inv = 1.0;
  if (run == 0) {
    double total = 0.0;
    for (int k = 0; k < 16; ++k) total += lds[k * 17];
    const double norm = sqrt(total);
    inv = norm <= (double)tab.eps ? 1.0 / (double)tab.eps : 1.0 / norm;
  }

  // Wave 0 iterates.  A lane's operands of a product of symmetric matrices are
  // the values (lane & 15, 4 s + lane / 16); it is given (4 r + lane / 16, lane & 15).
  double* buf = lds + 256;  // 16 rows of kThinLd
  const int c = lane & 15, q = lane >> 4;
  if (wave == 0) {
    f64x4 A, P;  // operands
#pragma unroll
    for (int r = 0; r < 4; ++r) A[r] = lds[c * 16 + 4 * r + q] * inv * inv;
    auto times = [&](const f64x4& x, const f64x4& y) {
      f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(x[r], y[r], acc, 0, 0, 0);
      return acc;
    };
    auto operand = [&](const f64x4& v) {
#pragma unroll
      for (int r = 0; r < 4; ++r) buf[(4 * r + q) * kThinLd + c] = v[r];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      f64x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = buf[c * kThinLd + 4 * r + q];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      return o;
    };
    for (int s = 0; s < steps; ++s) {
      f64x4 Q = operand(times(A, A));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        Q[r] = (double)poly.c * Q[r] + (double)poly.b * A[r] + (c == 4 * r + q ? (double)poly.a : 0.0);
      P = s ? operand(times(Q, P)) : Q;
      if (s + 1 < steps) A = operand(times(operand(times(Q, A)), Q));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) buf[c * kThinLd + 4 * r + q] = P[r] * inv;
  }
  __syncthreads();
  f64x4 P;
#pragma unroll
  for (int r = 0; r < 4; ++r) P[r] = buf[c * kThinLd + 4 * r + q];
  const int end = t.n - chunk * t.chunk < t.chunk ? t.n : (chunk + 1) * t.chunk;
  by_type(run ? T_F64 : tab.gtype, [&](auto like) {
    for (int j0 = chunk * t.chunk + wave * 16; j0 < end; j0 += 4 * WAVES * 16) {
      Held<decltype(like)> u[4][4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          u[h][r] = thin_u<decltype(like)>(tab, t, false, 4 * r + q, j0 + h * WAVES * 16 + c, end);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int j = j0 + h * WAVES * 16 + c;
        if (j - c >= end) break;
        f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc = __builtin_amdgcn_mfma_f64_16x16x4f64(P[r], (double)u[h][r], acc, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * r + q;
          if (i >= t.m || j >= end) continue;
          if (!last) {
            *thin_x(t, i, j) = acc[r];
            continue;
          }
          const size_t at = thin_place(t, i, j);
          float o = (float)acc[r];
          if (t.mom) o = tab.keep * load_as(t.w, at, tab.wtype) - t.step * o;
          store_as(t.w, at, tab.wtype, o);
        }
      }
    }
  });
}

extern __shared__ __align__(16) char flowml_ns_lds[];

// Matrices of one block all runs, others run `run`.
__global__ __launch_bounds__(kSmallThreads) void flowml_ns_small(Table tab, Poly poly, int run) {
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  if (t.parts > 1) {
    thin_run(tab, t, poly, run, blockIdx.x - t.first, (double*)flowml_ns_lds);
    return;
  }
  if (run) return;
  if (t.m <= kThinM)
    for (int r = 0; r * kThinRun < poly.steps; ++r) {
      thin_run(tab, t, poly, r, 0, (double*)flowml_ns_lds);
      __syncthreads();  // X is written, P is read
    }
  else if (small_pieces(t.m) == 2)
    small_matrix<2>(tab, t, poly, (f16*)flowml_ns_lds);
  else if (small_pieces(t.m) == 4)
    small_matrix<4>(tab, t, poly, (f16*)flowml_ns_lds);
  else
    small_matrix<8>(tab, t, poly, (f16*)flowml_ns_lds);
}

// ---- launch plan ----------------------------------------------------------------

constexpr int kPerNormBlock = 8192;

int pad(int v, int t) { return (v + t - 1) / t * t; }

// Tile sides of a call's products, and the parts of K of A.  Large tiles run at
// twice the rate of small ones, but are worth it only if there are enough for
// the 256 CUs.  Measured on normally distributed values, us a product (tiles):
//   A of 1024 x 4096:    64 (136) 28   96 (66) 53    128 (36) 58
//   A of 2048 x 4096:    64 (528) 92   96 (253) 80   128 (136) 83   192 (66) 128
//   its A^2:             64 (528) 47   96 (253) 42   128 (136) 45   192 (66) 70
//   A of 4096 x 4096:    96 (946) 283  128 (528) 259 192 (253) 206  256 (136) 253
//   B X of 1024 x 4096:  64 (1024) 31  128 (256) 26  256 (64) 55
//   two of these:        128 (512) 50  128 x 256 (256) 48
//   B X of 2048 x 4096:  128 (512) 105 128 x 256 (256) 98  256 (128) 118
//   B X of 4096 x 4096:  128 (1024) 378  128 x 256 (512) 353  256 (256) 330
// For A and B a side is taken by the time that follows from such figures.  Where
// A has few tiles and a long K, blocks take parts of K and a launch more joins
// them: two of 1024 x 4096 take 50 us as 272 tiles of 64, and 32 + 6 us
// as 72 of 128 in 3 parts; all steps of 100 x 100000, 2800 and 377 us.
struct Sides {
  int a, b, m, n;  // A, B, and B X along m and n
  int kpart;       // K of A to a block
};
constexpr int kWhole = 1 << 30;  // a kpart that no K passes

int shorter(int r, int c) { return std::min(r, c); }
int longer(int r, int c) { return std::max(r, c); }

struct Sym {
  int side;
  double us;  // for 64 of K, if a tile has a CU
};
constexpr Sym kSym[] = {{64, 0.30}, {96, 0.63}, {128, 0.83}, {192, 1.75}, {256, 2.80}};

// us of a symmetric product of so many blocks, from times measured over matrices
// of 512 to 4096 rows.  A full chip runs slower than one block alone: clocks
// and memory are shared.
double time_of(const Sym& y, long long blocks, int K) {
  const double fill = blocks / 256.0, rounds = (double)((blocks + 255) / 256);
  return y.us * (rounds + 0.5 * fill) * ((K + 63) / 64) + 2.0 + y.side / 32.0;
}

Sides sides_for(int count, const int* rows, const int* cols) {
  auto tiles = [&](int ti, int tj) {
    long long sum = 0;
    for (int k = 0; k < count; ++k)
      sum += (long long)tiles_of(shorter(rows[k], cols[k]), ti) *
             tiles_of(longer(rows[k], cols[k]), tj);
    return sum;
  };
  Sides s;
  // a larger side has to make good the padding of matrices that are low
  const long long t64 = tiles(64, 64), t128 = tiles(128, 128), t256 = tiles(256, 256);
  s.m = t256 >= 200 && 3 * t256 <= t128 ? 256 : t128 >= 128 && 8 * t128 <= 3 * t64 ? 128 : 64;
  s.n = s.m == 128 && tiles(128, 256) >= 200 ? 256 : s.m;

  int km = 0, kn = 0;  // the longest K of B and of A
  for (int k = 0; k < count; ++k) {
    km = std::max(km, pad(shorter(rows[k], cols[k]), s.m));
    kn = std::max(kn, pad(longer(rows[k], cols[k]), s.n));
  }
  // blocks of a symmetric product, and how many of them leave their sums
  auto triangle = [&](int side, int kpart, long long* several) {
    long long sum = 0;
    *several = 0;
    for (int k = 0; k < count; ++k) {
      const long long mt = tiles_of(pad(shorter(rows[k], cols[k]), s.m), side);
      const int split = tiles_of(pad(longer(rows[k], cols[k]), s.n), kpart);
      sum += mt * (mt + 1) / 2 * split;
      if (split > 1) *several += mt * (mt + 1) / 2 * split;
    }
    return sum;
  };
  double best_a = 1e30, best_b = 1e30;
  for (const Sym& y : kSym) {
    long long sums;
    const long long whole = triangle(y.side, kWhole, &sums);
    const double us = time_of(y, whole, km);
    if (us < best_b) {
      best_b = us;
      s.b = y.side;
    }
    for (int parts = 1; parts <= 64; ++parts) {
      const int kpart = parts == 1 ? kWhole : pad(tiles_of(kn, parts), 64);
      const long long blocks = parts == 1 ? whole : triangle(y.side, kpart, &sums);
      // parts that are short or for which there is no CU bring nothing
      if (parts > 1 && (kpart < 256 || blocks > 512)) break;
      const double us = time_of(y, blocks, std::min(kpart, kn)) +
                        (sums ? 4.0 + 0.15 * parts + sums * y.side * y.side * 1.2e-6 : 0.0);
      if (us < best_a) {
        best_a = us;
        s.a = y.side;
        s.kpart = kpart;
      }
    }
  }
  return s;
}

struct Sizes {
  int mp, np, ma, split;
  size_t bytes;  // sums of squares and planes
  size_t sums;   // floats of A's parts
};

Sizes sizes_of(int rows, int cols, Sides s) {
  Sizes z;
  z.mp = pad(shorter(rows, cols), s.m);
  z.np = pad(longer(rows, cols), s.n);
  z.ma = std::max(pad(z.mp, s.a), pad(z.mp, s.b));
  z.split = tiles_of(z.np, s.kpart);
  const size_t nx = rows_xt(z.np), ma = z.ma, mt = tiles_of(z.mp, s.a);
  z.bytes = kNormBlocks * sizeof(double) + (4 * nx * ma + 4 * ma * ma) * sizeof(f16);
  z.sums = z.split > 1 ? mt * (mt + 1) / 2 * s.a * s.a * z.split : 0;
  return z;
}

// one product for all matrices of a table; `first` of each is set here
template <class T, int BK, int S, int TO>
void product_of(Table& tab, int turn, float ka, float kb, float kd, hipStream_t st) {
  int blocks = 0;
  for (int k = 0; k < tab.count; ++k) {
    Mat& t = tab.mat[k];
    t.first = blocks;
    const int mt = tiles_of(t.mp, T::TM);
    blocks += TO == TO_A   ? mt * (mt + 1) / 2 * t.split
              : TO == TO_B ? mt * (mt + 1) / 2
                           : (t.mp / T::TM) * (t.np / T::TN);
  }
  hipLaunchKernelGGL((flowml_ns_product<T, BK, S, TO>), dim3(blocks), dim3(T::WAVES * 64),
                     0, st, tab, turn, ka, kb, kd);
}

void join(Sides s, Table& tab, float kb, hipStream_t st) {
  int blocks = 0;
  for (int k = 0; k < tab.count; ++k) {
    Mat& t = tab.mat[k];
    t.first = blocks;
    const int mt = tiles_of(t.mp, s.a), pieces = mt * (mt + 1) / 2 * (s.a / 32) * (s.a / 32);
    if (t.split > 1) blocks += tiles_of(pieces, 4);
  }
  if (blocks) hipLaunchKernelGGL(flowml_ns_join, dim3(blocks), dim3(256), 0, st, tab, s.a, kb);
}

template <int TO>
void product(Sides s, Table& tab, int turn, float ka, float kb, float kd, hipStream_t st) {
  // tile, waves, and the depth and stages of LDS
  if constexpr (TO == TO_A || TO == TO_B) {
    const int side = TO == TO_A ? s.a : s.b;
    if (side == 256)
      product_of<Tile<256, 256, 2, 4>, 32, 2, TO>(tab, turn, ka, kb, kd, st);
    else if (side == 192)
      product_of<Tile<192, 192, 2, 2>, 32, 3, TO>(tab, turn, ka, kb, kd, st);
    else if (side == 96)
      product_of<Tile<96, 96, 3, 1>, 32, 6, TO>(tab, turn, ka, kb, kd, st);
    else if (side == 128)
      product_of<Tile<128, 128, 2, 2>, 32, 4, TO>(tab, turn, ka, kb, kd, st);
    else
      product_of<Tile<64, 64, 2, 2>, 32, 5, TO>(tab, turn, ka, kb, kd, st);
    if (TO == TO_A && s.kpart < kWhole) join(s, tab, kb, st);
  } else {
    if (s.m == 256)
      product_of<Tile<256, 256, 2, 4>, 32, 2, TO>(tab, turn, ka, kb, kd, st);
    else if (s.n == 256)
      product_of<Tile<128, 256, 2, 4>, 32, 3, TO>(tab, turn, ka, kb, kd, st);
    else if (s.m == 128)
      product_of<Tile<128, 128, 2, 4>, 32, 4, TO>(tab, turn, ka, kb, kd, st);
    else
      product_of<Tile<64, 64, 2, 2>, 32, 5, TO>(tab, turn, ka, kb, kd, st);
  }
}

// The way a matrix goes: one block holds it, or 2 + 3 * steps launches.  A
// short side of 16 or less goes the first way in any company (in 64 bits, where
// few values leave fp16 pairs' roundings nothing to cancel against); other
// small ones do if all are small, for a long launch hides them.
enum { THIN = 0, SMALL = 1, LARGE = 2 };

void ways(int count, const int* rows, const int* cols, int* way) {
  bool large = false;
  for (int k = 0; k < count; ++k) {
    const int m = rows[k] < cols[k] ? rows[k] : cols[k], n = rows[k] < cols[k] ? cols[k] : rows[k];
    way[k] = m <= kThinM ? THIN : small_fits(m, n) ? SMALL : LARGE;
    large |= way[k] == LARGE;
  }
  if (large)
    for (int k = 0; k < count; ++k)
      if (way[k] == SMALL) way[k] = LARGE;
}

// columns of a thin matrix to a block
int thin_chunk(int n) {
  const int c = (n + 63) / 64;
  return c < 256 ? 256 : c;
}

// its blocks' sums, and X if there is more than one run
size_t thin_sums(int rows, int cols) {
  const int n = rows < cols ? cols : rows, c = thin_chunk(n), chunks = (n + c - 1) / c;
  return chunks > 1 ? (size_t)chunks * 256 * sizeof(double) : 0;
}
size_t thin_bytes(int rows, int cols, int steps) {
  const size_t x = steps > kThinRun ? (size_t)rows * cols * sizeof(double) : 0;
  return thin_sums(rows, cols) + (x + 255) / 256 * 256;
}

struct Call {
  int count;
  const int *rows, *cols;
  const void* const* g;
  float* const* mom;
  void* const* w;
  const float* step;
};

// up to kMats matrices of the way `way` (or, for SMALL, both that one block
// holds), from index k0 on; returns the index behind them
int gather(Table& tab, const Call& c, const int* way, bool large, int k0) {
  tab.count = 0;
  int k = k0;
  for (; k < c.count && tab.count < kMats; ++k) {
    if ((way[k] == LARGE) != large) continue;
    Mat& t = tab.mat[tab.count++];
    t.rows = c.rows[k];
    t.cols = c.cols[k];
    t.m = t.rows < t.cols ? t.rows : t.cols;
    t.n = t.rows < t.cols ? t.cols : t.rows;
    t.g = c.g[k];
    t.mom = c.mom ? c.mom[k] : nullptr;
    t.w = c.w[k];
    t.step = c.step ? c.step[k] : 0.f;
  }
  return k;
}

// the large ones' shapes alone, for the tiles' sides
int large_shapes(int count, const int* rows, const int* cols, const int* way, int* r, int* c) {
  int n = 0;
  for (int k = 0; k < count; ++k)
    if (way[k] == LARGE) {
      r[n] = rows[k];
      c[n++] = cols[k];
    }
  return n;
}

}  // namespace

// ---- host entry points ------------------------------------------------------------

// workspace of a call, in bytes, or -1 if a plane's 32-bit places do not reach
// over one of its matrices; `scratch`: 3 * count integers
extern "C" long long muon_workspace(int count, const int* rows, const int* cols, int steps,
                                    int* scratch) {
  int *way = scratch, *r = scratch + count, *c = scratch + 2 * count;
  ways(count, rows, cols, way);
  const int n = large_shapes(count, rows, cols, way, r, c);
  const Sides s = sides_for(n, r, c);
  size_t sum = 0;
  for (int k = 0; k < count; ++k) {
    if (way[k] == LARGE) {
      const Sizes z = sizes_of(rows[k], cols[k], s);
      if ((long long)std::max(rows_xt(z.np), z.ma) * z.ma >= 1LL << 30) return -1;
      sum += z.bytes + z.sums * sizeof(float);
    }
    if (way[k] == THIN) sum += thin_bytes(rows[k], cols[k], steps);
  }
  return (long long)sum;
}

// g: gradients; mom: momentum buffers, or null for the orthogonalisation
// alone; w: weights, or results.  coef: a, b, c; scale_b: a power of two that
// brings B into fp16.  ws: muon_workspace() bytes; scratch: as there.
extern "C" void launch_muon(int count, const int* rows, const int* cols, const void* const* g,
                            float* const* mom, void* const* w, const float* step, int gtype,
                            int wtype, float mu, float keep, float eps, int nesterov, int steps,
                            const float* coef, float scale_b, void* ws, int* scratch, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  int* way = scratch;
  ways(count, rows, cols, way);
  const int n = large_shapes(count, rows, cols, way, scratch + count, scratch + 2 * count);
  const Sides sides = sides_for(n, scratch + count, scratch + 2 * count);
  const Call call = {count, rows, cols, g, mom, w, step};
  const float sa = kScaleA, sx = kScaleX, sb = scale_b;
  Table tab;
  tab.gtype = gtype;
  tab.wtype = wtype;
  tab.mu = mu;
  tab.keep = keep;
  tab.eps = eps;
  tab.nesterov = nesterov;
  char* at = (char*)ws;

  for (int k0 = 0; k0 < count;) {
    k0 = gather(tab, call, way, false, k0);
    if (!tab.count) break;
    int blocks = 0;
    bool chunks = false;
    size_t lds = (256 + 16 * kThinLd + kSmallThreads / 64 * 256) * sizeof(double);
    for (int k = 0; k < tab.count; ++k) {
      Mat& t = tab.mat[k];
      t.part = (double*)at;
      t.first = blocks;
      t.parts = 1;
      if (t.m <= kThinM) {
        t.chunk = thin_chunk(t.n);
        t.parts = (t.n + t.chunk - 1) / t.chunk;
        t.ws = (f16*)(at + thin_sums(t.rows, t.cols));
        at += thin_bytes(t.rows, t.cols, steps);
        chunks |= t.parts > 1;
      } else {
        const size_t b = small_lds(t.m, t.n);
        lds = lds > b ? lds : b;
      }
      blocks += t.parts;
    }
    const Poly poly = {coef[0], coef[1], coef[2], sb, steps};
    for (int run = 0; run == 0 || (chunks && run * kThinRun < steps); ++run) {
      if (chunks)
        hipLaunchKernelGGL(flowml_ns_thin_gram, dim3(blocks), dim3(kSmallThreads), 0, st, tab, run);
      hipLaunchKernelGGL(flowml_ns_small, dim3(blocks), dim3(kSmallThreads), lds, st, tab, poly, run);
    }
  }

  for (int k0 = 0; k0 < count;) {
    k0 = gather(tab, call, way, true, k0);
    if (!tab.count) break;
    // the largest first: what a launch's last blocks do is then little
    std::stable_sort(tab.mat, tab.mat + tab.count, [](const Mat& x, const Mat& y) {
      return (double)x.m * x.n > (double)y.m * y.n;
    });
    int blocks = 0;
    for (int k = 0; k < tab.count; ++k) {
      Mat& t = tab.mat[k];
      const Sizes z = sizes_of(t.rows, t.cols, sides);
      t.mp = z.mp;
      t.np = z.np;
      t.ma = z.ma;
      t.split = z.split;
      t.kpart = sides.kpart;
      t.part = (double*)at;
      t.ws = (f16*)(at + kNormBlocks * sizeof(double));
      t.sums = (float*)(at + z.bytes);
      at += z.bytes + z.sums * sizeof(float);
      const size_t want = ((size_t)t.rows * t.cols + kPerNormBlock - 1) / kPerNormBlock;
      t.parts = (int)(want < kNormBlocks ? want : kNormBlocks);
      t.first = blocks;
      blocks += t.parts;
    }
    hipLaunchKernelGGL(flowml_ns_norm, dim3(blocks), dim3(256), 0, st, tab);
    blocks = 0;
    for (int k = 0; k < tab.count; ++k) {
      tab.mat[k].first = blocks;
      blocks += (tab.mat[k].mp / 64) * (tab.mat[k].np / 64);
    }
    hipLaunchKernelGGL(flowml_ns_first, dim3(blocks), dim3(256), 0, st, tab);
    for (int s = 0; s < steps; ++s) {
      product<TO_A>(sides, tab, s & 1, 0.f, sa / (sx * sx), 0.f, st);
      product<TO_B>(sides, tab, 0, coef[1] * sb / sa, coef[2] * sb / (sa * sa), coef[0] * sb, st);
      if (s + 1 < steps)
        product<TO_X>(sides, tab, s & 1, 0.f, 1.f / sb, 0.f, st);
      else
        product<TO_END>(sides, tab, s & 1, 0.f, 1.f / (sb * sx), 0.f, st);
    }
  }
}
