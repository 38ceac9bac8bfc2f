// CDNA4 (gfx950) layer norm with a fused activation, forward and backward.
//
//   mu = sum_j x_j / D          var = sum_j (x_j - mu)^2 / D
//   rstd = 1 / sqrt(var + eps)  xh_j = (x_j - mu) rstd
//   y_j = act(xh_j g_j + b_j)
//
//   dz = dy act'(y)             p = dz g
//   dx = rstd (p - mean(p) - xh mean(p xh))
//   dg = sum_rows dz xh         db = sum_rows dz
//
// Both passes are bound by HBM.  A row of up to 16384 values lives in the
// registers of the lanes that share it, so each input is read once and each
// output is written once, and the variance is the centred sum of a second look
// at registers, not of a second read (no E[x^2] - E[x]^2 cancellation).  Longer
// rows are read three times.  How many lanes take a row, with how many 16-byte
// pieces each, follows from its length (forward_shape, backward_shape): of 128
// bf16, 16 lanes with one piece, so that four rows share a wave and their sums
// are DPP moves without LDS; a row that is more than a wave holds has a block to
// itself, of as many waves as it needs.  All sums and statistics are fp32;
// values are rounded to the tensor's type once, at the store.
//
// Times in the comments are of the kernels alone: beside a kernel over inputs
// that no cache holds, for two ways of one thing in a loop over one input, of
// which the last-level cache keeps a part.
//
// The activation's derivative is taken from the stored output y (relu: y > 0,
// sigmoid: y (1 - y)), as the dgrad kernel of the GEMM stack does: a sign
// recomputed from x could differ from the one the forward pass acted on.
//
// dg and db are summed without atomics: a lane owns its columns over all rows
// of its block, the block's row groups are added in LDS in a fixed order, and
// a second kernel adds the blocks' slabs in a fixed order, so that two runs
// agree bit for bit.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <stdint.h>

#include <algorithm>

namespace {

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

// 16-byte pieces at element alignment: the hardware takes unaligned global
// accesses, so odd row lengths and odd strides use the same wide loads.
template <typename T>
struct Piece {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T raw __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef raw vec __attribute__((aligned(sizeof(T))));
};

// 0 behind the row's end
template <typename T>
__device__ __forceinline__ typename Piece<T>::raw load_raw(const T* p, int left) {
  constexpr int VEC = Piece<T>::VEC;
  if (left >= VEC) return *reinterpret_cast<const typename Piece<T>::vec*>(p);
  typename Piece<T>::raw r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r[k] = k < left ? p[k] : (T)0.f;
  return r;
}

template <typename T>
__device__ __forceinline__ void load_piece(const T* p, int left, float* v) {
  const typename Piece<T>::raw r = load_raw<T>(p, left);
#pragma unroll
  for (int k = 0; k < Piece<T>::VEC; ++k) v[k] = (float)r[k];
}

// stream: past the caches, for results that do not fit them (1M x 128 bf16: 87
// us instead of 102, 200000 x 500 bf16 75 instead of 97; loads past the caches
// lose as much).  The empty statements keep the compiler from making one store
// of the two, which is not past anything.
template <typename T>
__device__ __forceinline__ void store_piece(T* p, int left, const float* v, bool stream) {
  constexpr int VEC = Piece<T>::VEC;
  if (left >= VEC) {
    typename Piece<T>::raw r;
#pragma unroll
    for (int k = 0; k < VEC; ++k) r[k] = (T)v[k];
    if (stream) {
      asm volatile("" ::: "memory");
      __builtin_nontemporal_store(r, reinterpret_cast<typename Piece<T>::vec*>(p));
      asm volatile("" ::: "memory");
    } else {
      *reinterpret_cast<typename Piece<T>::vec*>(p) = r;
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k < left) p[k] = (T)v[k];
  }
}

// VEC weights of neighbouring columns; `none` for a missing vector or column
template <int VEC>
__device__ __forceinline__ void load_columns(const float* p, int c, int D, float none, float* v) {
  if (p && c + VEC <= D) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) load_piece<float>(p + c + k, 4, v + k);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = (p && c + k < D) ? p[c + k] : none;
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Sum over groups of LANES <= 64 neighbouring lanes; every lane gets it, with
// the same bits.  All lanes of the wave take part.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  if (LANES >= 2) v += dpp<0xB1>(v);   // quad_perm 1,0,3,2
  if (LANES >= 4) v += dpp<0x4E>(v);   // quad_perm 2,3,0,1
  if (LANES >= 8) v += dpp<0x141>(v);  // mirror within 8
  if (LANES >= 16) v += dpp<0x140>(v); // mirror within 16
  if (LANES >= 32) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (LANES >= 64) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Rows of up to a wave's lanes share blocks of four waves; a longer row has a
// block to itself, of as many waves as it needs (LANES = 0: blockDim.x).
constexpr int kWaves = 16;  // most waves of a block
constexpr int block_of(int lanes) { return lanes ? 256 : kWaves * 64; }

// `lds` of the sums below: words that no wave still reads (callers alternate),
// 0 where the block has no wave.
__device__ __forceinline__ void clear_sums(float* lds, int n) {
  if ((int)threadIdx.x < n) lds[threadIdx.x] = 0.f;
  __syncthreads();
}

// Sum over the lanes that share a row: part of a wave, or the whole block.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  if constexpr (LANES > 0) {
    return lanes_sum<LANES>(v);
  } else {
    v = lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lanes_sum<kWaves>(lds[threadIdx.x % kWaves]);
  }
}

// Two such sums behind one barrier.
template <int LANES>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* lds) {
  a = lanes_sum<(LANES ? LANES : 64)>(a);
  b = lanes_sum<(LANES ? LANES : 64)>(b);
  if constexpr (LANES == 0) {
    if ((threadIdx.x & 63) == 0) {
      lds[threadIdx.x >> 6] = a;
      lds[kWaves + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = lanes_sum<kWaves>(lds[threadIdx.x % kWaves]);
    b = lanes_sum<kWaves>(lds[kWaves + threadIdx.x % kWaves]);
  }
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == 1) return z < 0.f ? 0.f : z;  // keeps NaN
  if (act == 2) return 1.f / (1.f + expf(-z));
  return z;
}

__device__ __forceinline__ float activate_grad(float dy, float y, int act) {
  if (act == 1) return y > 0.f ? dy : 0.f;
  if (act == 2) return dy * (y * (1.f - y));
  return dy;
}

// ---------------------------------------------------------------------------
// forward: LANES lanes x NV pieces hold a row
// ---------------------------------------------------------------------------

// The next row of a group is under way while this one is worked on: 32 waves
// a CU with 16 bytes a lane are not quite enough to keep HBM busy.  1M x 128
// bf16: 94 us, 5.5 TB/s; 5003 x 4099 f32: 30 us, 5.4 TB/s; 256 x 64 f32: 3 us.
template <typename T, int LANES, int NV>
__global__ __launch_bounds__(block_of(LANES)) void flowml_layer_norm(
    const T* __restrict__ X, long long ldx, const float* __restrict__ gamma,
    const float* __restrict__ beta, T* __restrict__ Y, float* __restrict__ mean,
    float* __restrict__ rstd, long long N, int D, float eps, int act, bool stream) {
  constexpr int VEC = Piece<T>::VEC;
  constexpr int GROUPS = LANES ? 256 / LANES : 1;
  __shared__ float s_red[2][LANES ? 1 : kWaves];
  const int lanes = LANES ? LANES : blockDim.x;
  const int lane = threadIdx.x % lanes;
  const int group = threadIdx.x / lanes;
  const float d = (float)D;
  if (!LANES) clear_sums(s_red[0], 2 * kWaves);

  float g[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_columns<VEC>(gamma, (i * lanes + lane) * VEC, D, 1.f, g[i]);
    load_columns<VEC>(beta, (i * lanes + lane) * VEC, D, 0.f, b[i]);
  }

  const long long stride = (long long)gridDim.x * GROUPS;
  typename Piece<T>::raw raw[NV];
  // lanes without a row of their own repeat the last one: the sums below need
  // every lane of the wave
  auto fetch = [&](long long row) {
    const T* x = X + (row < N ? row : N - 1) * ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * VEC;
      raw[i] = load_raw<T>(x + c, D - c);
    }
  };
  fetch((long long)blockIdx.x * GROUPS + group);
  for (long long row0 = (long long)blockIdx.x * GROUPS; row0 < N; row0 += stride) {
    const long long row = row0 + group;
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[i][k] = (float)raw[i][k];
        s += v[i][k];
      }
    if (row0 + stride < N) fetch(row + stride);
    const float mu = row_sum<LANES>(s, s_red[0]) / d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[i][k] -= mu;
        q += c + k < D ? v[i][k] * v[i][k] : 0.f;
      }
    }
    const float r = 1.f / sqrtf(row_sum<LANES>(q, s_red[1]) / d + eps);
    if (row < N) {
      T* y = Y + row * D;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + lane) * VEC;
        if (c < D) {
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            v[i][k] = activate(v[i][k] * r * g[i][k] + b[i][k], act);
          store_piece<T>(y + c, D - c, v[i], stream);
        }
      }
      if (lane == 0) {
        mean[row] = mu;
        rstd[row] = r;
      }
    }
  }
}

// Rows longer than a block's registers: three looks at the row (8000 x 30000 bf16:
// 285 us, 3.4 TB/s of what has to move).
template <typename T>
__global__ __launch_bounds__(1024) void flowml_layer_norm_long(
    const T* __restrict__ X, long long ldx, const float* __restrict__ gamma,
    const float* __restrict__ beta, T* __restrict__ Y, float* __restrict__ mean,
    float* __restrict__ rstd, long long N, int D, float eps, int act, bool stream) {
  constexpr int VEC = Piece<T>::VEC;
  __shared__ float s_red[2][kWaves];
  const float d = (float)D;
  for (long long row = blockIdx.x; row < N; row += gridDim.x) {
    const T* x = X + row * ldx;
    float v[VEC];
    float s = 0.f;
    for (int c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
      load_piece<T>(x + c, D - c, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += v[k];
    }
    const float mu = row_sum<0>(s, s_red[0]) / d;
    float q = 0.f;
    for (int c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
      load_piece<T>(x + c, D - c, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) q += c + k < D ? (v[k] - mu) * (v[k] - mu) : 0.f;
    }
    const float r = 1.f / sqrtf(row_sum<0>(q, s_red[1]) / d + eps);
    T* y = Y + row * D;
    for (int c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
      float g[VEC], b[VEC];
      load_piece<T>(x + c, D - c, v);
      load_columns<VEC>(gamma, c, D, 1.f, g);
      load_columns<VEC>(beta, c, D, 0.f, b);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = activate((v[k] - mu) * r * g[k] + b[k], act);
      store_piece<T>(y + c, D - c, v, stream);
    }
    if (threadIdx.x == 0) {
      mean[row] = mu;
      rstd[row] = r;
    }
  }
}

// ---------------------------------------------------------------------------
// backward: dx, and one slab (dg, db) per block in part[block][2][D].  1M x 128
// bf16 with relu: 193 us and 5 for the slabs, 5.2 TB/s; 8192 x 8192 f16: 83 us
// and 5, 4.6 TB/s
// ---------------------------------------------------------------------------

template <typename T, int LANES, int NV, bool ACT>
__global__ __launch_bounds__(block_of(LANES)) void flowml_layer_norm_grad(
    const T* __restrict__ dY, long long lddy, const T* __restrict__ X, long long ldx,
    const T* __restrict__ Y, long long ldy, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ gamma,
    T* __restrict__ dX, float* __restrict__ part, long long N, int D, int act, bool stream) {
  constexpr int VEC = Piece<T>::VEC;
  constexpr int GROUPS = LANES ? 256 / LANES : 1;
  constexpr int WIDTH = LANES * NV * VEC;
  __shared__ float s_red[2][LANES ? 1 : 2 * kWaves];
  __shared__ float s_cols[GROUPS > 1 ? 256 * NV * VEC : 1];
  const int lanes = LANES ? LANES : blockDim.x;
  const int lane = threadIdx.x % lanes;
  const int group = threadIdx.x / lanes;
  const float d = (float)D;
  if (!LANES) clear_sums(s_red[0], 4 * kWaves);

  float g[NV][VEC], dg[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_columns<VEC>(gamma, (i * lanes + lane) * VEC, D, 1.f, g[i]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) dg[i][k] = db[i][k] = 0.f;
  }

  const long long stride = (long long)gridDim.x * GROUPS;
  typename Piece<T>::raw rx[NV], rd[NV], ry[ACT ? NV : 1];
  float next_mu, next_r;
  auto fetch = [&](long long row) {
    if (row >= N) row = N - 1;
    next_mu = mean[row];
    next_r = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * VEC;
      rx[i] = load_raw<T>(X + row * ldx + c, D - c);
      rd[i] = load_raw<T>(dY + row * lddy + c, D - c);
      if constexpr (ACT) ry[i] = load_raw<T>(Y + row * ldy + c, D - c);
    }
  };
  // with 16 values of four arrays to a lane, 128 registers do not hold two rows
  constexpr bool AHEAD = LANES || NV * VEC < 16;
  if (AHEAD) fetch((long long)blockIdx.x * GROUPS + group);
  int turn = 0;  // the block-wide sums of two neighbouring rows use other words
  for (long long row0 = (long long)blockIdx.x * GROUPS; row0 < N; row0 += stride, turn ^= 1) {
    const long long row = row0 + group;
    const bool live = row < N;
    if (!AHEAD) fetch(row);
    const float mu = next_mu, r = next_r;
    float xh[NV][VEC], dz[NV][VEC];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        dz[i][k] = (float)rd[i][k];
        if constexpr (ACT) dz[i][k] = activate_grad(dz[i][k], (float)ry[i][k], act);
        xh[i][k] = ((float)rx[i][k] - mu) * r;
        // past the row's end dz is 0, and with it p and both sums
        const float p = dz[i][k] * g[i][k];
        s += p;
        q += c + k < D ? p * xh[i][k] : 0.f;
        if (live) {
          dg[i][k] += dz[i][k] * xh[i][k];
          db[i][k] += dz[i][k];
        }
      }
    }
    if (AHEAD && row0 + stride < N) fetch(row + stride);
    row_sum2<LANES>(s, q, s_red[turn]);
    s /= d;
    q /= d;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + lane) * VEC;
        if (c < D) {
          float o[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            o[k] = r * (dz[i][k] * g[i][k] - s - xh[i][k] * q);
          store_piece<T>(dX + row * D + c, D - c, o, stream);
        }
      }
    }
  }

  float* slab = part + (long long)blockIdx.x * 2 * D;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * lanes + lane) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (c + k < D) {
          slab[c + k] = dg[i][k];
          slab[D + c + k] = db[i][k];
        }
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          s_cols[group * WIDTH + (i * lanes + lane) * VEC + k] = half ? db[i][k] : dg[i][k];
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += 256) {
        float t = 0.f;
        for (int o = 0; o < GROUPS; ++o) t += s_cols[o * WIDTH + c];
        slab[half * D + c] = t;
      }
    }
  }
}

// Long rows: dx alone, two looks at the row (2000 x 30000 bf16, with the columns:
// 210 us, 1.7 TB/s of what has to move) ...
template <typename T>
__global__ __launch_bounds__(1024) void flowml_layer_norm_grad_long(
    const T* __restrict__ dY, long long lddy, const T* __restrict__ X, long long ldx,
    const T* __restrict__ Y, long long ldy, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ gamma,
    T* __restrict__ dX, long long N, int D, int act) {
  constexpr int VEC = Piece<T>::VEC;
  __shared__ float s_red[2][2 * kWaves];
  const float d = (float)D;
  int turn = 0;
  for (long long row = blockIdx.x; row < N; row += gridDim.x, turn ^= 1) {
    const float mu = mean[row], r = rstd[row];
    float s = 0.f, q = 0.f;
    for (int look = 0; look < 2; ++look) {
      for (int c = threadIdx.x * VEC; c < D; c += 1024 * VEC) {
        float x[VEC], dz[VEC], y[VEC], g[VEC];
        load_columns<VEC>(gamma, c, D, 1.f, g);
        load_piece<T>(X + row * ldx + c, D - c, x);
        load_piece<T>(dY + row * lddy + c, D - c, dz);
        if (act) load_piece<T>(Y + row * ldy + c, D - c, y);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const bool in = c + k < D;
          const float p = (act ? activate_grad(dz[k], y[k], act) : dz[k]) * g[k];
          const float xh = (x[k] - mu) * r;
          if (look == 0) {
            s += p;
            q += in ? p * xh : 0.f;
          } else {
            x[k] = r * (p - s - xh * q);
          }
        }
        if (look) store_piece<T>(dX + row * D + c, D - c, x, false);
      }
      if (look == 0) {
        row_sum2<0>(s, q, s_red[turn]);
        s /= d;
        q /= d;
      }
    }
  }
}

// ... and the columns: a block sums 256 columns over a chunk of the rows
template <typename T>
__global__ __launch_bounds__(256) void flowml_layer_norm_grad_cols(
    const T* __restrict__ dY, long long lddy, const T* __restrict__ X, long long ldx,
    const T* __restrict__ Y, long long ldy, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ part, long long N, int D,
    long long chunk, int act) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  const long long lo = blockIdx.y * chunk;
  const long long hi = lo + chunk < N ? lo + chunk : N;
  float dg = 0.f, db = 0.f;
  for (long long row = lo; row < hi; ++row) {
    const float x = (float)X[row * ldx + c];
    float dz = (float)dY[row * lddy + c];
    if (act) dz = activate_grad(dz, (float)Y[row * ldy + c], act);
    dg += dz * ((x - mean[row]) * rstd[row]);
    db += dz;
  }
  float* slab = part + (long long)blockIdx.y * 2 * D;
  slab[c] = dg;
  slab[D + c] = db;
}

// dg[c], db[c]: sums of part[s][0][c] and part[s][1][c] over the slabs, in an
// order that G alone sets: 32 columns x 32 runs of slabs per block.
__global__ __launch_bounds__(1024) void flowml_layer_norm_slabs(
    const float* __restrict__ part, float* __restrict__ dg, float* __restrict__ db, int G, int D) {
  __shared__ float s[32][33];
  const int W = 2 * D;
  const int c = blockIdx.x * 32 + (threadIdx.x & 31);
  const int run = threadIdx.x >> 5;
  float t = 0.f;
  if (c < W) {
    int k = run;
    for (; k + 7 * 32 < G; k += 8 * 32) {  // eight loads under way
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = part[(long long)(k + e * 32) * W + c];
#pragma unroll
      for (int e = 0; e < 8; ++e) t += v[e];
    }
    for (; k < G; k += 32) t += part[(long long)k * W + c];
  }
  s[run][threadIdx.x & 31] = t;
  __syncthreads();
  if (run == 0 && c < W) {
    float u = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) u += s[k][threadIdx.x];
    if (c < D)
      dg[c] = u;
    else
      db[c - D] = u;
  }
}

// ---------------------------------------------------------------------------
// launch plans
// ---------------------------------------------------------------------------

constexpr int kCUs = 256;

// Whether a result is too large for the 256 MB of last-level cache to be found
// there by whoever reads it next.  Short rows with ragged ends go through the
// caches all the same, which make whole lines of them (2M x 41 f32: 156 us, past
// them 165).
bool streams(long long N, int D, size_t size) {
  const long long row = D * (long long)size;
  return N * row >= (128LL << 20) && (row >= 256 || row % 16 == 0);
}

// Lanes and pieces for a row of D values of VEC to the piece.  Up to a wave, a
// power of two with one piece to a lane, unless that leaves a quarter or more of
// the lanes idle and three pieces to fewer lanes do not: rows that share a wave
// are what keeps memory busy.
struct Shape {
  int lanes, nv;
};

// pieces that three to each of `lanes` hold, and one to each of twice as many does not
bool three_fit(int pieces, int lanes) { return pieces > 2 * lanes && pieces <= 3 * lanes; }

// Forward, beyond a wave's lanes: two or three pieces to them (112500 x 800 bf16:
// 68 us, with two waves 79; 150000 x 600 bf16: 32 lanes x 3 71, two waves 99; of
// f32 60 and 67 to 76), then up to 16 values to a lane (as many weights and
// biases).  Lanes without a piece cost their share of the row there, and waves
// that wait for each other 3 % apiece (us, lanes x pieces; 5003 x 2051 f32: 192 x
// 3 14, 256 x 3 16, 320 x 2 16, 576 x 1 18; 8000 x 5000 f16: 320 x 2 34, 640 x 1
// 40).  Three pieces to a part of a wave: 300000 x 300 bf16 97 and 81 us; not of
// f32 (340909 x 132: 74 and 76).
Shape forward_shape(int D, int vec) {
  const int pieces = (D + vec - 1) / vec;
  if (vec == 8 && three_fit(pieces, 16)) return {16, 3};
  for (int l = 1; l <= 64; l *= 2)
    if (pieces <= l) return {l, 1};
  if (three_fit(pieces, 32)) return {32, 3};
  if (pieces <= 128) return {64, 2};
  if (pieces <= 192) return {64, 3};
  Shape best = {0, 0};
  int least = 1 << 30;
  for (int v = 1; v <= 16 / vec; ++v) {
    const int w = std::max(2, (pieces + 64 * v - 1) / (64 * v)), cost = w * v * (100 + 3 * w);
    if (w <= kWaves && cost < least) {
      least = cost;
      best = {w * 64, v};
    }
  }
  return best;
}

// Blocks of the forward pass that a CU holds: by the registers of so many
// values, and a place less on its four SIMDs where a block's waves do not
// divide among them.  More wait for a second round (20000 x 2056 bf16, 320
// lanes: 40 us with 5, 48 with 6).
int forward_blocks(Shape s, int vec) {
  const int w = s.lanes / 64, values = s.nv * vec;
  const int places = 4 * (values <= 8 ? 8 : values <= 12 ? 6 : vec == 8 ? 5 : 4);
  return std::max(1, (w < 4 || w % 4 == 0 ? places : places - 4) / w);
}

// Backward.  Three pieces to fewer lanes serve all but f32 with an activation,
// which has a third array (300000 x 300 bf16 186 and 140 us, 150000 x 600 bf16 181
// and 128, 561600 x 80 f32 131 and 109; 236842 x 190 f32 with relu 163 and 184),
// four pieces to half a wave 16-bit rows without one (90000 x 1000 bf16: 110 us,
// 64 x 2 132; with relu 159 and 151).  Beyond, one piece to a lane as far as a
// block goes, for four arrays and two sums of columns live in registers (20000 x
// 2056 bf16: 61 us with one piece to 320 lanes, 70 with two to 192).
Shape backward_shape(int D, int vec, bool act) {
  const int pieces = (D + vec - 1) / vec;
  const bool three = vec == 8 || !act;
  for (int l = 8; three && l <= 16; l *= 2)
    if (three_fit(pieces, l)) return {l, 3};
  for (int l = 1; l <= 64; l *= 2)
    if (pieces <= l) return {l, 1};
  if (vec == 8 && three_fit(pieces, 32)) return {32, 3};
  if (pieces <= 128) return vec == 8 && !act ? Shape{32, 4} : Shape{64, 2};
  if (three && pieces <= 192) return {64, 3};
  for (int v = 1; v <= 16 / vec; v *= 2) {
    const int w = (pieces + 64 * v - 1) / (64 * v);
    if (w <= kWaves) return {w * 64, v};
  }
  return {0, 0};
}

// Its blocks to a CU: what registers allow, and few, for each leaves sums to add
// (20000 x 2056 bf16, 320 lanes: 67 us with 3, 83 with 4).
int backward_blocks(Shape s, int vec) {
  return s.lanes <= 64 ? 4 : std::max(1, (s.nv * vec == 4 ? 20 : 16) / (s.lanes / 64));
}

int rows_per_block(Shape s) { return s.lanes > 64 ? 1 : 256 / s.lanes; }
int threads_of(Shape s) { return s.lanes > 64 ? s.lanes : 256; }

template <typename T>
void forward(const T* X, long long ldx, const float* g, const float* b, T* Y, float* mean,
             float* rstd, long long N, int D, float eps, int act, hipStream_t st) {
  const Shape s = forward_shape(D, Piece<T>::VEC);
  const bool stream = streams(N, D, sizeof(T));
  if (!s.lanes) {
    const int grid = (int)(N < 2 * kCUs ? N : 2 * kCUs);
    hipLaunchKernelGGL((flowml_layer_norm_long<T>), dim3(grid), dim3(1024), 0, st, X, ldx, g, b, Y,
                       mean, rstd, N, D, eps, act, stream);
    return;
  }
  const int rpb = rows_per_block(s);
  const long long want = (N + rpb - 1) / rpb;
  const long long most = kCUs * (s.lanes > 64 ? forward_blocks(s, Piece<T>::VEC) : 16);
  const int grid = (int)(want < most ? want : most);
#define LN_CASE(L, V)                                                                           \
  if ((s.lanes > 64 ? 0 : s.lanes) == L && s.nv == V)                                           \
    hipLaunchKernelGGL((flowml_layer_norm<T, L, V>), dim3(grid), dim3(threads_of(s)), 0, st, X, \
                       ldx, g, b, Y, mean, rstd, N, D, eps, act, stream)
  LN_CASE(1, 1);
  LN_CASE(2, 1);
  LN_CASE(4, 1);
  LN_CASE(8, 1);
  LN_CASE(16, 1);
  LN_CASE(32, 1);
  LN_CASE(64, 1);
  LN_CASE(32, 3);
  LN_CASE(64, 2);
  LN_CASE(64, 3);
  LN_CASE(0, 1);
  LN_CASE(0, 2);
  if constexpr (Piece<T>::VEC == 4) {
    LN_CASE(0, 3);
    LN_CASE(0, 4);
  } else {
    LN_CASE(16, 3);
  }
#undef LN_CASE
}

// slabs (and blocks) of the backward pass
int grad_slabs(long long N, int D, int vec, bool act) {
  const Shape s = backward_shape(D, vec, act);
  long long want, most;
  if (!s.lanes) {
    // columns kernel: 256 columns to a block, chunks of rows to fill the chip
    want = (N + 15) / 16;
    most = (4 * kCUs * 256LL + D - 1) / D;
    if (most < 1) most = 1;
  } else {
    const int rpb = rows_per_block(s);
    want = (N + rpb - 1) / rpb;
    most = kCUs * backward_blocks(s, vec);
  }
  return (int)(want < most ? want : most);
}

template <typename T>
void backward(const T* dY, long long lddy, const T* X, long long ldx, const T* Y, long long ldy,
              const float* mean, const float* rstd, const float* g, T* dX, float* part,
              float* dg, float* db, long long N, int D, int act, hipStream_t st) {
  const Shape s = backward_shape(D, Piece<T>::VEC, act);
  const bool stream = streams(N, D, sizeof(T));
  const int slabs = N ? grad_slabs(N, D, Piece<T>::VEC, act) : 0;
  if (slabs && !s.lanes) {
    const int grid = (int)(N < 2 * kCUs ? N : 2 * kCUs);
    hipLaunchKernelGGL((flowml_layer_norm_grad_long<T>), dim3(grid), dim3(1024), 0, st, dY, lddy, X,
                       ldx, Y, ldy, mean, rstd, g, dX, N, D, act);
    const long long chunk = (N + slabs - 1) / slabs;
    hipLaunchKernelGGL((flowml_layer_norm_grad_cols<T>), dim3((D + 255) / 256, slabs),
                       dim3(256), 0, st, dY, lddy, X, ldx, Y, ldy, mean, rstd, part, N, D, chunk, act);
  } else if (slabs) {
#define LN_CASE1(L, V, A)                                                                     \
  hipLaunchKernelGGL((flowml_layer_norm_grad<T, L, V, A>), dim3(slabs), dim3(threads_of(s)),  \
                     0, st, dY, lddy, X, ldx, Y, ldy, mean, rstd, g, dX, part, N, D, act, stream)
#define LN_CASE(L, V, A) \
  if ((s.lanes > 64 ? 0 : s.lanes) == L && s.nv == V && (act != 0) == A) LN_CASE1(L, V, A)
#define LN_CASES(L, V)   \
  LN_CASE(L, V, false);  \
  LN_CASE(L, V, true)
    LN_CASES(1, 1);
    LN_CASES(2, 1);
    LN_CASES(4, 1);
    LN_CASES(8, 1);
    LN_CASES(16, 1);
    LN_CASES(32, 1);
    LN_CASES(64, 1);
    LN_CASES(0, 1);
    LN_CASES(0, 2);
    LN_CASE(8, 3, false);
    LN_CASE(16, 3, false);
    LN_CASE(64, 2, true);
    LN_CASE(64, 3, false);
    if constexpr (Piece<T>::VEC == 4) {
      LN_CASE(64, 2, false);
      LN_CASES(0, 4);
    } else {
      LN_CASE(8, 3, true);
      LN_CASE(16, 3, true);
      LN_CASES(32, 3);
      LN_CASE(32, 4, false);
      LN_CASE(64, 3, true);
    }
#undef LN_CASES
#undef LN_CASE
#undef LN_CASE1
  }
  hipLaunchKernelGGL(flowml_layer_norm_slabs, dim3((2 * D + 31) / 32), dim3(1024), 0, st,
                     part, dg, db, slabs, D);
}

}  // namespace

// ---------------------------------------------------------------------------
// host launchers (type: 0 f32, 1 bf16, 2 f16; strides in values)
// ---------------------------------------------------------------------------

extern "C" void launch_layer_norm(int type, const void* X, long long ldx, const float* g,
                                  const float* b, void* Y, float* mean, float* rstd, long long N,
                                  int D, float eps, int act, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (type == T_F32)
    forward((const float*)X, ldx, g, b, (float*)Y, mean, rstd, N, D, eps, act, st);
  else if (type == T_BF16)
    forward((const __bf16*)X, ldx, g, b, (__bf16*)Y, mean, rstd, N, D, eps, act, st);
  else
    forward((const _Float16*)X, ldx, g, b, (_Float16*)Y, mean, rstd, N, D, eps, act, st);
}

// slabs of 2 * D floats that the backward pass wants as a workspace
extern "C" int layer_norm_grad_slabs(int type, long long N, int D, int act) {
  return N ? grad_slabs(N, D, type == T_F32 ? 4 : 8, act) : 0;
}

extern "C" void launch_layer_norm_grad(int type, const void* dY, long long lddy, const void* X,
                                       long long ldx, const void* Y, long long ldy,
                                       const float* mean, const float* rstd, const float* g,
                                       void* dX, float* part, float* dg, float* db, long long N,
                                       int D, int act, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (type == T_F32)
    backward((const float*)dY, lddy, (const float*)X, ldx, (const float*)Y, ldy, mean, rstd, g,
             (float*)dX, part, dg, db, N, D, act, st);
  else if (type == T_BF16)
    backward((const __bf16*)dY, lddy, (const __bf16*)X, ldx, (const __bf16*)Y, ldy, mean, rstd, g,
             (__bf16*)dX, part, dg, db, N, D, act, st);
  else
    backward((const _Float16*)dY, lddy, (const _Float16*)X, ldx, (const _Float16*)Y, ldy, mean,
             rstd, g, (_Float16*)dX, part, dg, db, N, D, act, st);
}
