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
// products accumulated in fp32: hi hi + hi lo + lo hi.  That is as exact as
// fp32 (1.0 to 1.25 times its error on full-rank, low-rank and rank-1
// gradients) at a third of the fp16 matrix rate, 5 times the fp32 rate.
// Where the result is rounded to bf16, A and A^2 take hi hi alone and B X
// takes hi (hi + lo): an error in A or B turns the left singular vectors by
// 2^-12 but leaves the row space of X exact, so no noise grows.
//
// A and A^2 are symmetric: tiles on or above the diagonal are computed, and
// each is written to both places.
//
// All operands are stored with the summed index side by side, so that every
// product is rows times rows: X serves X X^T, its transpose serves B X, and
// the epilogue of B X writes both.  Working matrices are padded with zeros to
// whole tiles, which the iteration keeps, so that only the first and the last
// kernel look at ragged edges.
//
// The matrices of one call share their launches: 2 + 3 * steps, whatever
// their number and shapes.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <math.h>
#include <stdint.h>

namespace {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

constexpr int kMats = 24;        // matrices to a launch: the table is an argument
constexpr int kNormBlocks = 64;  // most blocks that sum one matrix' squares
constexpr float kScaleX = 16384.f;  // |x| <= 1.9: within fp16
constexpr float kScaleA = 16384.f;  // |x|^2 <= 3.7

struct Mat {
  f16* ws;         // X, X^T (two), A, B: two planes each
  double* part;    // sums of squares
  const void* g;   // gradient, rows x cols
  float* mom;      // momentum buffer, or null
  void* w;         // weights, or the result
  int m, n;        // shorter and longer side
  int mp, np;      // padded to whole tiles
  int rows, cols;  // as the caller has it
  int full;        // 1: three products everywhere
  float step;
  int first;       // first block of this matrix in a launch
  int blocks;      // and their number
};

struct Table {
  Mat mat[kMats];
  int count;
  int gtype, wtype;
  float mu, keep, eps;
  int nesterov;
};

// ---- working planes ---------------------------------------------------------

__host__ __device__ inline size_t plane_x(const Mat& t) { return (size_t)t.mp * t.np; }
__host__ __device__ inline size_t plane_a(const Mat& t) { return (size_t)t.mp * t.mp; }
__device__ __forceinline__ f16* ws_x(const Mat& t, int p) { return t.ws + p * plane_x(t); }
__device__ __forceinline__ f16* ws_xt(const Mat& t, int which, int p) {
  return t.ws + (2 + 2 * which + p) * plane_x(t);
}
__device__ __forceinline__ f16* ws_a(const Mat& t, int p) {
  return t.ws + 6 * plane_x(t) + p * plane_a(t);
}
__device__ __forceinline__ f16* ws_b(const Mat& t, int p) {
  return t.ws + 6 * plane_x(t) + (2 + p) * plane_a(t);
}

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

// ---- sums of squares, and the momentum ---------------------------------------

__global__ __launch_bounds__(256) void flowml_ns_norm(Table tab) {
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int b = blockIdx.x - t.first;
  const size_t total = (size_t)t.rows * t.cols;
  double s = 0.0;
  for (size_t i = (size_t)b * 256 + threadIdx.x; i < total; i += (size_t)t.blocks * 256) {
    float u = load_as(t.g, i, tab.gtype);
    if (t.mom) {
      const float v = tab.mu * t.mom[i] + u;
      t.mom[i] = v;
      u = tab.nesterov ? u + tab.mu * v : v;
    }
    s += (double)u * (double)u;
  }
  __shared__ double red[4];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) t.part[b] = red[0] + red[1] + red[2] + red[3];
}

// ---- the first iterate: 64 x 64 tiles of the caller's matrix -------------------

__global__ __launch_bounds__(256) void flowml_ns_first(Table tab, int norm_blocks_of_one) {
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int b = blockIdx.x - t.first;
  const bool turned = t.rows > t.cols;  // the caller's rows run along n
  const int prow = turned ? t.np : t.mp, pcol = turned ? t.mp : t.np;
  const int r0 = (b / (pcol / 64)) * 64, c0 = (b % (pcol / 64)) * 64;

  // |G|: every block adds the same partial sums in the same order
  const size_t total = (size_t)t.rows * t.cols;
  int parts = (int)((total + norm_blocks_of_one - 1) / norm_blocks_of_one);
  if (parts > kNormBlocks) parts = kNormBlocks;
  double s = 0.0;
  for (int k = 0; k < parts; ++k) s += t.part[k];
  const double norm = sqrt(s);
  const float scale = norm <= (double)tab.eps ? (float)(kScaleX / (double)tab.eps)
                                              : (float)(kScaleX / norm);  // NaN stays

  __shared__ uint32_t tile[64][65];
  f16* straight[2];
  f16* turned_p[2];
  for (int p = 0; p < 2; ++p) {
    straight[p] = turned ? ws_xt(t, 0, p) : ws_x(t, p);
    turned_p[p] = turned ? ws_x(t, p) : ws_xt(t, 0, p);
  }
  const int tc = threadIdx.x & 63, tr = threadIdx.x >> 6;
  for (int i = tr; i < 64; i += 4) {
    const int r = r0 + i, c = c0 + tc;
    float u = 0.f;
    if (r < t.rows && c < t.cols) {
      const size_t at = (size_t)r * t.cols + c;
      u = load_as(t.g, at, tab.gtype);
      if (t.mom) u = tab.nesterov ? u + tab.mu * t.mom[at] : t.mom[at];
      u *= scale;
    }
    const f16 hi = (f16)u, lo = (f16)(u - (float)hi);
    straight[0][(size_t)r * pcol + c] = hi;
    straight[1][(size_t)r * pcol + c] = lo;
    tile[i][tc] = (uint32_t)__builtin_bit_cast(uint16_t, hi) |
                  ((uint32_t)__builtin_bit_cast(uint16_t, lo) << 16);
  }
  __syncthreads();
  for (int i = tr; i < 64; i += 4) {
    const uint32_t v = tile[tc][i];
    const size_t at = (size_t)(c0 + i) * prow + r0 + tc;
    turned_p[0][at] = __builtin_bit_cast(f16, (uint16_t)(v & 0xffff));
    turned_p[1][at] = __builtin_bit_cast(f16, (uint16_t)(v >> 16));
  }
}

// ---- products -----------------------------------------------------------------

enum { TO_A = 0, TO_B = 1, TO_X = 2, TO_END = 3 };

template <int BK>
__device__ __forceinline__ int swizzle(int chunk, int row) {
  // eight neighbouring rows' pieces of one chunk fall on all 32 banks
  return BK == 64 ? (chunk ^ (row & 7)) : (chunk ^ ((row >> 1) & 3));
}

// acc += P Q^T over K: P has TM rows, Q TN rows, BK values of K at a time.
// PA, PB: planes of each (2: hi and lo).
template <int TM, int TN, int WM, int WN, int BK, int PA, int PB>
__device__ __forceinline__ void product(const f16* const (&P)[2], int ldp,
                                        const f16* const (&Q)[2], int ldq, int K, f16* lds,
                                        f32x16 (&acc)[TM / WM / 32][TN / WN / 32]) {
  constexpr int NT = WM * WN * 64;
  constexpr int CH = BK / 8;                 // 16-byte chunks in a row
  constexpr int LA = TM * CH / NT, LB = TN * CH / NT;
  constexpr int FM = TM / WM / 32, FN = TN / WN / 32;
  constexpr int STAGE = (PA * TM + PB * TN) * BK;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = (wave / WN) * (TM / WM), wn = (wave % WN) * (TN / WN);

  f16x8 ra[PA][LA], rb[PB][LB];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int p = 0; p < PA; ++p)
#pragma unroll
      for (int i = 0; i < LA; ++i) {
        const int c = tid + i * NT;
        ra[p][i] = *(const f16x8*)(P[p] + (size_t)(c / CH) * ldp + k0 + (c % CH) * 8);
      }
#pragma unroll
    for (int p = 0; p < PB; ++p)
#pragma unroll
      for (int i = 0; i < LB; ++i) {
        const int c = tid + i * NT;
        rb[p][i] = *(const f16x8*)(Q[p] + (size_t)(c / CH) * ldq + k0 + (c % CH) * 8);
      }
  };
  auto keep = [&](f16* s) {
#pragma unroll
    for (int p = 0; p < PA; ++p)
#pragma unroll
      for (int i = 0; i < LA; ++i) {
        const int c = tid + i * NT, r = c / CH;
        *(f16x8*)(s + p * TM * BK + r * BK + swizzle<BK>(c % CH, r) * 8) = ra[p][i];
      }
#pragma unroll
    for (int p = 0; p < PB; ++p)
#pragma unroll
      for (int i = 0; i < LB; ++i) {
        const int c = tid + i * NT, r = c / CH;
        *(f16x8*)(s + (PA * TM + p * TN) * BK + r * BK + swizzle<BK>(c % CH, r) * 8) = rb[p][i];
      }
  };

  fetch(0);
  keep(lds);
  __syncthreads();
  int turn = 0;
  for (int k0 = 0; k0 < K; k0 += BK, turn ^= 1) {
    if (k0 + BK < K) fetch(k0 + BK);
    const f16* s = lds + turn * STAGE;
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      f16x8 a[PA][FM], b[PB][FN];
      const int chunk = kk * 2 + (lane >> 5);
#pragma unroll
      for (int p = 0; p < PA; ++p)
#pragma unroll
        for (int f = 0; f < FM; ++f) {
          const int r = wm + f * 32 + (lane & 31);
          a[p][f] = *(const f16x8*)(s + p * TM * BK + r * BK + swizzle<BK>(chunk, r) * 8);
        }
#pragma unroll
      for (int p = 0; p < PB; ++p)
#pragma unroll
        for (int f = 0; f < FN; ++f) {
          const int r = wn + f * 32 + (lane & 31);
          b[p][f] =
              *(const f16x8*)(s + (PA * TM + p * TN) * BK + r * BK + swizzle<BK>(chunk, r) * 8);
        }
#pragma unroll
      for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int g = 0; g < FN; ++g) {
          if constexpr (PA == 2)
            acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1][f], b[0][g], acc[f][g], 0, 0, 0);
          if constexpr (PB == 2)
            acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][f], b[1][g], acc[f][g], 0, 0, 0);
          acc[f][g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][f], b[0][g], acc[f][g], 0, 0, 0);
        }
    }
    if (k0 + BK < K) keep(lds + (turn ^ 1) * STAGE);
    __syncthreads();
  }
}

__device__ __forceinline__ void split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

// One tile of A, B, X' or the result.  `ka`, `kb`: the tile is
// ka * (old tile) + kb * (product).
template <int T, int WM, int WN, int BK, int TO>
__global__ __launch_bounds__(WM * WN * 64) void flowml_ns_product(Table tab, int turn, float ka,
                                                                  float kb) {
  constexpr int FM = T / WM / 32, FN = T / WN / 32;
  __shared__ __align__(16) f16 lds[2 * 4 * T * BK];
  const Mat& t = tab.mat[find(tab, blockIdx.x)];
  const int b = blockIdx.x - t.first;
  int ti, tj;
  if (TO == TO_A || TO == TO_B) {
    // b = tj (tj + 1) / 2 + ti, ti <= tj
    tj = (int)((sqrtf(8.f * b + 1.f) - 1.f) * 0.5f);
    while ((tj + 1) * (tj + 2) / 2 <= b) ++tj;
    while (tj * (tj + 1) / 2 > b) --tj;
    ti = b - tj * (tj + 1) / 2;
  } else {
    ti = b % (t.mp / T);
    tj = b / (t.mp / T);
  }
  const int i0 = ti * T, j0 = tj * T;

  const f16* P[2];
  const f16* Q[2];
  int ld, K;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if (TO == TO_A) {
      P[p] = ws_x(t, p) + (size_t)i0 * t.np;
      Q[p] = ws_x(t, p) + (size_t)j0 * t.np;
    } else if (TO == TO_B) {
      P[p] = ws_a(t, p) + (size_t)i0 * t.mp;
      Q[p] = ws_a(t, p) + (size_t)j0 * t.mp;
    } else {
      P[p] = ws_b(t, p) + (size_t)i0 * t.mp;
      Q[p] = ws_xt(t, turn, p) + (size_t)j0 * t.mp;
    }
  }
  ld = K = TO == TO_A ? t.np : t.mp;

  f32x16 acc[FM][FN];
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int g = 0; g < FN; ++g)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[f][g][r] = 0.f;
  if (t.full)
    product<T, T, WM, WN, BK, 2, 2>(P, ld, Q, ld, K, lds, acc);
  else if (TO == TO_A || TO == TO_B)
    product<T, T, WM, WN, BK, 1, 1>(P, ld, Q, ld, K, lds, acc);
  else
    product<T, T, WM, WN, BK, 1, 2>(P, ld, Q, ld, K, lds, acc);

  // a lane holds 4 neighbouring rows of a column, 4 times per 32 x 32 piece
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = i0 + (wave / WN) * (T / WM), wj = j0 + (wave % WN) * (T / WN);
#pragma unroll
  for (int f = 0; f < FM; ++f)
#pragma unroll
    for (int g = 0; g < FN; ++g)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = wi + f * 32 + q * 8 + (lane >> 5) * 4;
        const int j = wj + g * 32 + (lane & 31);
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = kb * acc[f][g][q * 4 + r];
        if (TO != TO_A) {
          // the old tile, from the copy in which its rows lie side by side
          const size_t at = (size_t)j * t.mp + i;
          const f16x4 h = *(const f16x4*)((TO == TO_B ? ws_a(t, 0) : ws_xt(t, turn, 0)) + at);
          f16x4 l = {0, 0, 0, 0};
          if (TO != TO_B || t.full)
            l = *(const f16x4*)((TO == TO_B ? ws_a(t, 1) : ws_xt(t, turn, 1)) + at);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += ka * ((float)h[r] + (float)l[r]);
        }
        if (TO == TO_END) {
          const bool turned = t.rows > t.cols;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (i + r < t.m && j < t.n) {
              const size_t at = turned ? (size_t)j * t.cols + i + r : (size_t)(i + r) * t.cols + j;
              float o = v[r];
              if (t.mom) o = tab.keep * load_as(t.w, at, tab.wtype) - t.step * o;
              store_as(t.w, at, tab.wtype, o);
            }
          }
          continue;
        }
        f16x4 h, l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f16 x, y;
          split(v[r], x, y);
          h[r] = x;
          l[r] = y;
        }
        const size_t across = (size_t)j * t.mp + i;  // [j][i..i+3]
        f16* ch = TO == TO_A ? ws_a(t, 0) : TO == TO_B ? ws_b(t, 0) : ws_xt(t, turn ^ 1, 0);
        f16* cl = TO == TO_A ? ws_a(t, 1) : TO == TO_B ? ws_b(t, 1) : ws_xt(t, turn ^ 1, 1);
        const bool low = TO == TO_X || t.full;
        *(f16x4*)(ch + across) = h;
        if (low) *(f16x4*)(cl + across) = l;
        // a tile on the diagonal is its own mirror image: one writer for each
        // value, since (i, j) and (j, i) may differ in the last bit
        if (TO != TO_X && ti == tj) continue;
        f16* sh = TO == TO_X ? ws_x(t, 0) : ch;
        f16* sl = TO == TO_X ? ws_x(t, 1) : cl;
        const int ldc = TO == TO_X ? t.np : t.mp;
        const bool low_s = TO == TO_X ? (bool)t.full : low;  // X X^T takes hi alone
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sh[(size_t)(i + r) * ldc + j] = h[r];
          if (low_s) sl[(size_t)(i + r) * ldc + j] = l[r];
        }
      }
}

// ---- launch plan ----------------------------------------------------------------

constexpr int kPerNormBlock = 16384;

int pad(int v, int t) { return (v + t - 1) / t * t; }

// Tile side for a whole call: 128 where B X then has a tile for every CU.
int tile_for(int count, const int* rows, const int* cols) {
  long long tiles = 0;
  for (int k = 0; k < count; ++k)
    tiles += (long long)((rows[k] + 127) / 128) * ((cols[k] + 127) / 128);
  return tiles >= 256 ? 128 : 64;
}

size_t bytes_of(int rows, int cols, int tile) {
  const size_t mp = pad(rows < cols ? rows : cols, tile), np = pad(rows < cols ? cols : rows, tile);
  return kNormBlocks * sizeof(double) + (6 * mp * np + 4 * mp * mp) * sizeof(f16);
}

template <int T, int WM, int WN, int BK>
void products(Table& tab, int steps, const float* coef, float scale_b, hipStream_t st) {
  const float sa = kScaleA, sx = kScaleX, sb = scale_b;
  int sym = 0, all = 0, first_all[kMats];
  for (int k = 0; k < tab.count; ++k) {
    Mat& t = tab.mat[k];
    const int mt = t.mp / T;
    t.first = sym;
    first_all[k] = all;
    sym += mt * (mt + 1) / 2;
    all += mt * (t.np / T);
  }
  Table tall = tab;
  for (int k = 0; k < tab.count; ++k) tall.mat[k].first = first_all[k];
  const dim3 block(WM * WN * 64);
  for (int s = 0; s < steps; ++s) {
    hipLaunchKernelGGL((flowml_ns_product<T, WM, WN, BK, TO_A>), dim3(sym), block, 0, st, tab, 0,
                       0.f, sa / (sx * sx));
    hipLaunchKernelGGL((flowml_ns_product<T, WM, WN, BK, TO_B>), dim3(sym), block, 0, st, tab, 0,
                       coef[1] * sb / sa, coef[2] * sb / (sa * sa));
    if (s + 1 < steps)
      hipLaunchKernelGGL((flowml_ns_product<T, WM, WN, BK, TO_X>), dim3(all), block, 0, st, tall,
                         s & 1, coef[0], 1.f / sb);
    else
      hipLaunchKernelGGL((flowml_ns_product<T, WM, WN, BK, TO_END>), dim3(all), block, 0, st, tall,
                         s & 1, coef[0] / sx, 1.f / (sb * sx));
  }
}

}  // namespace

// ---- host entry points ------------------------------------------------------------

// workspace of a call, in bytes
extern "C" long long muon_workspace(int count, const int* rows, const int* cols) {
  const int tile = tile_for(count, rows, cols);
  size_t sum = 0;
  for (int k = 0; k < count; ++k) sum += bytes_of(rows[k], cols[k], tile);
  return (long long)sum;
}

// g: gradients; mom: momentum buffers, or null for the orthogonalisation
// alone; w: weights, or results.  coef: a, b, c; scale_b: a power of two that
// brings B into fp16.  full: three products for every matrix, whatever its
// size.
extern "C" void launch_muon(int count, const int* rows, const int* cols, const void* const* g,
                            float* const* mom, void* const* w, const float* step, int gtype,
                            int wtype, float mu, float keep, float eps, int nesterov, int steps,
                            const float* coef, float scale_b, int full, void* ws, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  const int tile = tile_for(count, rows, cols);
  char* at = (char*)ws;
  for (int k0 = 0; k0 < count; k0 += kMats) {
    Table tab;
    tab.count = count - k0 < kMats ? count - k0 : kMats;
    tab.gtype = gtype;
    tab.wtype = wtype;
    tab.mu = mu;
    tab.keep = keep;
    tab.eps = eps;
    tab.nesterov = nesterov;
    int norm_blocks = 0;
    for (int k = 0; k < tab.count; ++k) {
      Mat& t = tab.mat[k];
      t.rows = rows[k0 + k];
      t.cols = cols[k0 + k];
      t.m = t.rows < t.cols ? t.rows : t.cols;
      t.n = t.rows < t.cols ? t.cols : t.rows;
      t.mp = pad(t.m, tile);
      t.np = pad(t.n, tile);
      t.part = (double*)at;
      t.ws = (f16*)(at + kNormBlocks * sizeof(double));
      at += bytes_of(t.rows, t.cols, tile);
      t.g = g[k0 + k];
      t.mom = mom ? mom[k0 + k] : nullptr;
      t.w = w[k0 + k];
      t.step = step ? step[k0 + k] : 0.f;
      t.full = full || t.m < 256;
      const size_t total = (size_t)t.rows * t.cols;
      const size_t want = (total + kPerNormBlock - 1) / kPerNormBlock;
      t.first = norm_blocks;
      t.blocks = (int)(want < kNormBlocks ? want : kNormBlocks);
      norm_blocks += t.blocks;
    }
    hipLaunchKernelGGL(flowml_ns_norm, dim3(norm_blocks), dim3(256), 0, st, tab);
    int tiles = 0;
    for (int k = 0; k < tab.count; ++k) {
      tab.mat[k].first = tiles;
      tiles += (tab.mat[k].mp / 64) * (tab.mat[k].np / 64);
    }
    hipLaunchKernelGGL(flowml_ns_first, dim3(tiles), dim3(256), 0, st, tab, kPerNormBlock);
    if (tile == 128)
      products<128, 2, 2, 32>(tab, steps, coef, scale_b, st);
    else
      products<64, 2, 2, 64>(tab, steps, coef, scale_b, st);
  }
}
