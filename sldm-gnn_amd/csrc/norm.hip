// Layer norm over the last dimension, forward and backward.
//
//   mean, rstd = 1/sqrt(var + eps) of each row;  xhat = (x - mean) rstd
//   y  = xhat w + b
//   dx = rstd (g - mean_j(g) - xhat mean_j(g xhat)),  g = dy w
//   dw = sum_rows dy xhat,  db = sum_rows dy
//
// Both directions are bound by memory: x in, y out (x and dy in, dx out), each
// once.  A row lives in the registers of the lanes that own it (2^k <= 64 lanes
// of a wave, or a workgroup of 256), 16 bytes a lane and load, so mean and
// variance are two passes over registers in fp32.  A width that 16 bytes do
// not divide costs nothing extra: loads need element alignment only, and the
// last lane of a row steps back to end with it (what it shares with its
// neighbour is masked out of the sums and stored twice, with the same value).
// Workgroups stay and walk rows, so a lane's columns of w and b are read once
// and its part of dw and db is summed in registers; the parts meet in LDS, one
// row of partials a workgroup, and a second kernel adds those in a fixed order.
// The next row's loads are issued over this row's sums.
//
// Measured (MI355X, where copies run at 4.6 to 6.3 TB/s): 1M x 256 bf16
// forward 218 us (4.7 TB/s), backward 307 us (5.0 TB/s) and 5 us for the sums;
// 20011 x 1031 bf16 20, 33 and 4 us; 9600 x 96 fp32 4.6, 7.1 and 3.0 us, where
// the host's 68 us for the three launches and the autograd engine count.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kBlock = 256;

typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4a4 __attribute__((ext_vector_type(4), aligned(4)));

// V elements of a row as they lie in memory, at element alignment (16-byte
// accesses for V = 16 / sizeof(T)).
template <typename T, int V>
struct Raw {
  static constexpr bool kWide = sizeof(T) * V == 16;
  uint4 w;
  T one;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (!kWide) one = *p;
    else if constexpr (sizeof(T) == 2) w = __builtin_bit_cast(uint4, *reinterpret_cast<const u4a2*>(p));
    else w = __builtin_bit_cast(uint4, *reinterpret_cast<const u4a4*>(p));
  }
  __device__ __forceinline__ void get(float (&r)[V]) const {
    if constexpr (!kWide) {
      sldm::Vec<T, 1>::load(&one, r);
    } else if constexpr (sizeof(T) == 2) {
      r[0] = sldm::bf16_lo(w.x); r[1] = sldm::bf16_hi(w.x); r[2] = sldm::bf16_lo(w.y); r[3] = sldm::bf16_hi(w.y);
      r[4] = sldm::bf16_lo(w.z); r[5] = sldm::bf16_hi(w.z); r[6] = sldm::bf16_lo(w.w); r[7] = sldm::bf16_hi(w.w);
    } else {
      r[0] = __uint_as_float(w.x); r[1] = __uint_as_float(w.y);
      r[2] = __uint_as_float(w.z); r[3] = __uint_as_float(w.w);
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&r)[V]) {
  if constexpr (!Raw<T, V>::kWide)
    sldm::Vec<T, V>::store(p, r);
  else if constexpr (sizeof(T) == 2)
    *reinterpret_cast<u4a2*>(p) = u4a2{sldm::pack_bf16x2(r[0], r[1]), sldm::pack_bf16x2(r[2], r[3]),
                                       sldm::pack_bf16x2(r[4], r[5]), sldm::pack_bf16x2(r[6], r[7])};
  else
    *reinterpret_cast<u4a4*>(p) = u4a4{__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]),
                                       __float_as_uint(r[3])};
}

// V columns of weight or bias; `none` where there is none
template <int V>
__device__ __forceinline__ void load_param(const float* p, int f, bool on, float none, float (&r)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) r[k] = none;
  if (!p || !on) return;
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const u4a4 u = *reinterpret_cast<const u4a4*>(p + f + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[k + e] = __uint_as_float(u[e]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = p[f + k];
  }
}

// Sum over the lanes of a row: lpr lanes of a wave, or the workgroup
// (WIDE; `slot` alternates between calls so that one barrier each is enough).
template <bool WIDE>
__device__ __forceinline__ float row_sum(float v, int lpr, float* red, int slot) {
  if constexpr (!WIDE) return sldm::group_sum(v, lpr);
  v = sldm::group_sum(v, 64);
  float* r = red + slot * (kBlock / 64);
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
  __syncthreads();
  return (r[0] + r[1]) + (r[2] + r[3]);
}

// Two such sums, one barrier.
template <bool WIDE>
__device__ __forceinline__ void row_sum2(float& u, float& v, int lpr, float* red, int slot) {
  u = sldm::group_sum(u, WIDE ? 64 : lpr);
  v = sldm::group_sum(v, WIDE ? 64 : lpr);
  if constexpr (WIDE) {
    float* r = red + slot * (2 * kBlock / 64);
    if ((threadIdx.x & 63) == 0) {
      r[threadIdx.x >> 6] = u;
      r[4 + (threadIdx.x >> 6)] = v;
    }
    __syncthreads();
    u = (r[0] + r[1]) + (r[2] + r[3]);
    v = (r[4] + r[5]) + (r[6] + r[7]);
  }
}

struct Lanes {          // which columns a lane holds
  int rows;             // rows a workgroup holds at once
  int row, lane, lpr;
};
__device__ __forceinline__ Lanes lanes(int lpr_log2) {
  const int lpr = 1 << lpr_log2;
  return {kBlock >> lpr_log2, (int)threadIdx.x >> lpr_log2, (int)threadIdx.x & (lpr - 1), lpr};
}

template <typename T, int V, int NCH, bool WIDE>
__global__ __launch_bounds__(kBlock) void norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                          int width, int lpr_log2, const float* __restrict__ w,
                                                          const float* __restrict__ b, float eps,
                                                          T* __restrict__ y, float* __restrict__ mean_out,
                                                          float* __restrict__ rstd_out) {
  __shared__ float red[2 * kBlock / 64];
  const Lanes L = lanes(lpr_log2);
  int f0[NCH], skip[NCH];
  float wv[NCH][V], bv[NCH][V];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int f = (L.lane + c * L.lpr) * V;
    f0[c] = f + V <= width ? f : width - V;
    skip[c] = f < width ? f - f0[c] : V;     // leading elements another lane owns
    load_param<V>(w, f0[c], skip[c] < V, 1.f, wv[c]);
    load_param<V>(b, f0[c], skip[c] < V, 0.f, bv[c]);
  }
  const float n = (float)width;   // a division: a constant row's mean stays exact
  Raw<T, V> next[NCH];
  auto fetch = [&](int64_t row) {
    const T* xr = x + (row < rows ? row : rows - 1) * ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (skip[c] < V) next[c].load(xr + f0[c]);
  };
  const int64_t stride = (int64_t)gridDim.x * L.rows;
  fetch((int64_t)blockIdx.x * L.rows + L.row);
  for (int64_t r0 = (int64_t)blockIdx.x * L.rows; r0 < rows; r0 += stride) {
    const int64_t row = r0 + L.row;
    const bool live = row < rows;
    float v[NCH][V], sum = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      next[c].get(v[c]);
#pragma unroll
      for (int k = 0; k < V; ++k) sum += k >= skip[c] ? v[c][k] : 0.f;
    }
    if (r0 + stride < rows) fetch(row + stride);   // over this row's sums
    const float mean = row_sum<WIDE>(sum, L.lpr, red, 0) / n;
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[c][k] -= mean;
        sq += k >= skip[c] ? v[c][k] * v[c][k] : 0.f;
      }
    const float rstd = 1.f / sqrtf(row_sum<WIDE>(sq, L.lpr, red, 1) / n + eps);
    if (!live) continue;
    if (mean_out && L.lane == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (skip[c] >= V) continue;
      float o[V];
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = __builtin_fmaf(v[c][k] * rstd, wv[c][k], bv[c][k]);
      store_row<T, V>(y + row * (int64_t)width + f0[c], o);
    }
  }
}

template <typename T, int V, int NCH, bool WIDE>
__global__ __launch_bounds__(kBlock) void norm_bwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                          const T* __restrict__ dy, int64_t lddy, int64_t rows,
                                                          int width, int lpr_log2, const float* __restrict__ w,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                          float* __restrict__ part) {
  __shared__ float red[4 * kBlock / 64];
  __shared__ float cols[WIDE ? 1 : kBlock * V];
  const Lanes L = lanes(lpr_log2);
  int f0[NCH], skip[NCH];
  float wv[NCH][V], dw[NCH][V], db[NCH][V];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int f = (L.lane + c * L.lpr) * V;
    f0[c] = f + V <= width ? f : width - V;
    skip[c] = f < width ? f - f0[c] : V;
    load_param<V>(w, f0[c], skip[c] < V, 1.f, wv[c]);
#pragma unroll
    for (int k = 0; k < V; ++k) dw[c][k] = db[c][k] = 0.f;
  }
  const float n = (float)width;
  Raw<T, V> xn[NCH], gn[NCH];
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](int64_t row) {
    const int64_t at = row < rows ? row : rows - 1;
    mean_n = mean_in[at];
    rstd_n = rstd_in[at];
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (skip[c] < V) {
        xn[c].load(x + at * ldx + f0[c]);
        gn[c].load(dy + at * lddy + f0[c]);
      }
  };
  const int64_t stride = (int64_t)gridDim.x * L.rows;
  if (rows > 0) fetch((int64_t)blockIdx.x * L.rows + L.row);
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * L.rows; r0 < rows; r0 += stride) {
    const int64_t row = r0 + L.row;
    const bool live = row < rows;
    Raw<T, V> xr[NCH], gr[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) xr[c] = xn[c], gr[c] = gn[c];
    const float mean = mean_n, rstd = rstd_n;
    if (r0 + stride < rows) fetch(row + stride);   // over this row's work
    float sg = 0.f, sgx = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float xh[V], g[V];
      xr[c].get(xh);
      gr[c].get(g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        xh[k] = (xh[k] - mean) * rstd;
        if (live && k >= skip[c]) {
          dw[c][k] += g[k] * xh[k];
          db[c][k] += g[k];
        }
        g[k] *= wv[c][k];
        if (k >= skip[c]) {
          sg += g[k];
          sgx += g[k] * xh[k];
        }
      }
    }
    if (!dx) continue;
    row_sum2<WIDE>(sg, sgx, L.lpr, red, turn);
    const float mg = sg / n, mgx = sgx / n;
    turn ^= 1;
    if (!live) continue;
    // xhat and g again from the row's 16 bytes a chunk: holding them in fp32 costs
    // 16 registers a chunk, and waves
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (skip[c] >= V) continue;
      float xh[V], g[V], o[V];
      xr[c].get(xh);
      gr[c].get(g);
#pragma unroll
      for (int k = 0; k < V; ++k)
        o[k] = rstd * (g[k] * wv[c][k] - mg - (xh[k] - mean) * rstd * mgx);
      store_row<T, V>(dx + row * (int64_t)width + f0[c], o);
    }
  }
  if (!part) return;
  float* p = part + (int64_t)blockIdx.x * 2 * width;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float(&s)[V] = half ? db[c] : dw[c];
      if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k >= skip[c]) p[half * width + f0[c] + k] = s[k];
      } else {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < V; ++k) cols[(L.row * L.lpr + L.lane) * V + k] = s[k];
        __syncthreads();
        // column f of this chunk: element f - f0 of the lane that owns it
        for (int i = threadIdx.x; i < L.lpr * V; i += kBlock) {
          const int lane = i / V, k = i % V;
          const int f = (lane + c * L.lpr) * V, at = f + V <= width ? f : width - V;
          if (f < width && k >= f - at) {
            float sum = 0.f;
            for (int r = 0; r < L.rows; ++r) sum += cols[r * L.lpr * V + i];
            p[half * width + at + k] = sum;
          }
        }
      }
    }
}

// Any width: a workgroup walks its row in steps, three times (twice from the
// caches).  The columns' sums have a kernel of their own.
template <typename T>
__device__ __forceinline__ float val(const T* p) {
  float r[1];
  sldm::Vec<T, 1>::load(p, r);
  return r[0];
}
template <typename T>
__device__ __forceinline__ void put(T* p, float v) {
  sldm::Vec<T, 1>::store(p, &v);
}
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_fwd_long_kernel(const T* x, int64_t ldx, int64_t width,
                                                               const float* w, const float* b, float eps, T* y,
                                                               float* mean_out, float* rstd_out) {
  __shared__ float red[2 * kBlock / 64];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const float n = (float)width;
  float sum = 0.f, sq = 0.f;
  for (int64_t i = threadIdx.x; i < width; i += kBlock) sum += val(xr + i);
  const float mean = row_sum<true>(sum, 0, red, 0) / n;
  for (int64_t i = threadIdx.x; i < width; i += kBlock) {
    const float d = val(xr + i) - mean;
    sq += d * d;
  }
  const float rstd = 1.f / sqrtf(row_sum<true>(sq, 0, red, 1) / n + eps);
  if (mean_out && threadIdx.x == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
  for (int64_t i = threadIdx.x; i < width; i += kBlock)
    put(y + row * width + i, __builtin_fmaf((val(xr + i) - mean) * rstd, w ? w[i] : 1.f, b ? b[i] : 0.f));
}
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_bwd_long_kernel(const T* x, int64_t ldx, const T* dy, int64_t lddy,
                                                               int64_t width, const float* w, const float* mean_in,
                                                               const float* rstd_in, T* dx) {
  __shared__ float red[2 * kBlock / 64];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * ldx, *dr = dy + row * lddy;
  const float n = (float)width, mean = mean_in[row], rstd = rstd_in[row];
  float sg = 0.f, sgx = 0.f;
  for (int64_t i = threadIdx.x; i < width; i += kBlock) {
    const float g = val(dr + i) * (w ? w[i] : 1.f);
    sg += g;
    sgx += g * (val(xr + i) - mean) * rstd;
  }
  const float mg = row_sum<true>(sg, 0, red, 0) / n, mgx = row_sum<true>(sgx, 0, red, 1) / n;
  for (int64_t i = threadIdx.x; i < width; i += kBlock) {
    const float g = val(dr + i) * (w ? w[i] : 1.f);
    put(dx + row * width + i, rstd * (g - mg - (val(xr + i) - mean) * rstd * mgx));
  }
}
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_cols_long_kernel(const T* x, int64_t ldx, const T* dy, int64_t lddy,
                                                                int64_t rows, int64_t width, const float* mean_in,
                                                                const float* rstd_in, float* part) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = val(dy + r * lddy + i);
    dw += d * (val(x + r * ldx + i) - mean_in[r]) * rstd_in[r];
    db += d;
  }
  float* p = part + (int64_t)blockIdx.y * 2 * width;
  p[i] = dw;
  p[width + i] = db;
}

// out[j] = sum over the partial rows, in order: 16 columns a workgroup, its
// 1024 threads as 64 row groups.
constexpr int kSumCols = 16, kSumRows = 64;
__global__ __launch_bounds__(kSumCols* kSumRows) void norm_sum_kernel(const float* part, int parts, int64_t width,
                                                                      float* dw, float* db) {
  __shared__ float red[kSumRows][kSumCols + 1];
  const int col = threadIdx.x % kSumCols, grp = threadIdx.x / kSumCols;
  const int64_t j = (int64_t)blockIdx.x * kSumCols + col;
  float s = 0.f;
  if (j < 2 * width) {
#pragma unroll 4
    for (int p = grp; p < parts; p += kSumRows) s += part[(int64_t)p * 2 * width + j];
  }
  red[grp][col] = s;
  __syncthreads();
  if (grp == 0 && j < 2 * width) {
    s = 0.f;
    for (int r = 0; r < kSumRows; ++r) s += red[r][col];
    if (j < width) {
      if (dw) dw[j] = s;
    } else if (db) {
      db[j - width] = s;
    }
  }
}

// Lanes and chunks of a row.  Up to 64 lanes x 4 chunks of 16 bytes a wave owns
// it, then a workgroup up to 8192 elements; past that it is re-read.  The bf16
// backward goes over to the workgroup past three chunks: four hold 256 registers a
// lane (20011 x 2040: 64 us by waves, 54 us by workgroups).
struct Shape {
  int v, lpr_log2, nch;
  bool wide, loop;
};
Shape shape_of(int dtype, int64_t width, bool backward) {
  const int full = dtype == SLDM_F32 ? 4 : 8;
  Shape s{width >= full ? full : 1, 0, 1, false, width > 8192};
  const int64_t need = (width + s.v - 1) / s.v;
  if (need > (backward && full == 8 ? 128 : 64 * 4)) {
    s.wide = true;
    s.lpr_log2 = 8;
  } else {
    while (s.lpr_log2 < 6 && (1 << s.lpr_log2) < need) ++s.lpr_log2;
  }
  const int64_t lpr = 1 << s.lpr_log2;
  while ((int64_t)s.nch * lpr < need) s.nch *= 2;
  // bf16: three chunks where powers of two leave much room empty (forward / backward:
  // 400000 x 264 112 -> 85 / 159 -> 133 us, 100000 x 513 51 -> 39 / 82 -> 72 us,
  // 10000 x 4104 38 -> 30 / 87 -> 58 us; the backward at 500000 x 176, 22 of 32 chunks,
  // would lose: 107 -> 114 us, and both at 1M x 96).  fp32 is at the memory's rate.
  const int64_t room = s.nch * lpr, most = backward && room < 256 ? 5 : 6;   // eighths of it
  if (full == 8 && !s.loop && room >= 32 && room != 512 && 8 * need <= most * room) {
    s.nch = 3;
    s.wide = room == 1024;
    s.lpr_log2 = 0;
    while ((int64_t)4 << s.lpr_log2 < room) ++s.lpr_log2;
  }
  return s;
}
int64_t row_groups(const Shape& s, int64_t rows) {
  const int64_t per = kBlock >> s.lpr_log2;
  return (rows + per - 1) / per;
}
// Workgroups of the backward, each with a row of partial sums: enough to fill the
// chip, few enough that wide rows of partials do not outweigh the rows (bf16,
// 512 / 1024 / 2048 of them: 5003 x 8000 76 / 107 / 121 us, 100000 x 513 82 / 93 /
// 83 us).
int parts_of(const Shape& s, int64_t rows, int64_t width) {
  if (s.loop) return (int)std::max<int64_t>(1, std::min<int64_t>(rows, 64));
  const int64_t n = row_groups(s, rows);
  return (int)std::max<int64_t>(1, std::min<int64_t>(width > 512 ? 512 : 1024, std::max<int64_t>(n / 4, std::min<int64_t>(n, 256))));
}

template <typename T>
void fwd(const T* x, int64_t ldx, int64_t rows, int64_t width, const float* w, const float* b, float eps, T* y,
         float* mean, float* rstd, hipStream_t st) {
  const Shape s = shape_of(sizeof(T) == 4 ? SLDM_F32 : SLDM_BF16, width, false);
  if (s.loop) {
    norm_fwd_long_kernel<T><<<(unsigned)rows, kBlock, 0, st>>>(x, ldx, width, w, b, eps, y, mean, rstd);
    return;
  }
  // rows enough a wave that reading w and b once pays (20011 x 2048 bf16, reading
  // them for every two rows: 66 us; for five: 30 us)
  const unsigned grid = (unsigned)std::min<int64_t>(row_groups(s, rows), s.nch == 1 ? 2048 : 1024);
  constexpr int F = 16 / sizeof(T);
#define SLDM_GO(V, N, W) \
  norm_fwd_kernel<T, V, N, W><<<grid, kBlock, 0, st>>>(x, ldx, rows, (int)width, s.lpr_log2, w, b, eps, y, mean, rstd)
  if (s.v == 1) SLDM_GO(1, 1, false);
  else if (s.wide) {
    if (s.nch == 2) SLDM_GO(F, 2, true);
    else if (F == 8 && s.nch == 3) SLDM_GO(F, F == 8 ? 3 : 2, true);
    else if (s.nch == 4) SLDM_GO(F, 4, true);
    else if constexpr (F == 4) SLDM_GO(F, 8, true);
  } else {
    if (s.nch == 1) SLDM_GO(F, 1, false);
    else if (s.nch == 2) SLDM_GO(F, 2, false);
    else if (F == 8 && s.nch == 3) SLDM_GO(F, F == 8 ? 3 : 2, false);
    else SLDM_GO(F, 4, false);
  }
#undef SLDM_GO
}

template <typename T>
void bwd(const T* x, int64_t ldx, const T* dy, int64_t lddy, int64_t rows, int64_t width, const float* w,
         const float* mean, const float* rstd, T* dx, float* dw, float* db, float* part, hipStream_t st) {
  const Shape s = shape_of(sizeof(T) == 4 ? SLDM_F32 : SLDM_BF16, width, true);
  const int parts = parts_of(s, rows, width);
  if (!dw && !db) part = nullptr;
  if (s.loop) {
    if (dx && rows) norm_bwd_long_kernel<T><<<(unsigned)rows, kBlock, 0, st>>>(x, ldx, dy, lddy, width, w, mean, rstd, dx);
    if (part)
      norm_cols_long_kernel<T><<<dim3((unsigned)((width + kBlock - 1) / kBlock), parts), kBlock, 0, st>>>(
          x, ldx, dy, lddy, rows, width, mean, rstd, part);
  } else {
    constexpr int F = 16 / sizeof(T);
#define SLDM_GO(V, N, W)                                                                                        \
  norm_bwd_kernel<T, V, N, W><<<parts, kBlock, 0, st>>>(x, ldx, dy, lddy, rows, (int)width, s.lpr_log2, w, mean, \
                                                        rstd, dx, part)
    if (s.v == 1) SLDM_GO(1, 1, false);
    else if (s.wide) {
      if (F == 8 && s.nch == 1) SLDM_GO(F, F == 8 ? 1 : 2, true);
      else if (s.nch == 2) SLDM_GO(F, 2, true);
      else if (F == 8 && s.nch == 3) SLDM_GO(F, F == 8 ? 3 : 2, true);
      else if (s.nch == 4) SLDM_GO(F, 4, true);
      else if constexpr (F == 4) SLDM_GO(F, 8, true);
    } else {
      if (s.nch == 1) SLDM_GO(F, 1, false);
      else if (s.nch == 2) SLDM_GO(F, 2, false);
      else SLDM_GO(F, F == 8 ? 3 : 4, false);
    }
#undef SLDM_GO
  }
  if (part)
    norm_sum_kernel<<<(unsigned)((2 * width + kSumCols - 1) / kSumCols), kSumCols * kSumRows, 0, st>>>(part, parts,
                                                                                                      width, dw, db);
}

int check_args(int dtype, int64_t rows, int64_t width) {
  SLDM_REQUIRE(dtype == SLDM_F32 || dtype == SLDM_BF16, "layer norm: dtype must be fp32 or bf16");
  SLDM_REQUIRE(rows >= 0 && width >= 1 && width < ((int64_t)1 << 30), "layer norm: bad shape %lld x %lld",
               (long long)rows, (long long)width);
  SLDM_REQUIRE(width <= 8192 || rows < ((int64_t)1 << 24), "layer norm: too many rows (%lld) of width %lld",
               (long long)rows, (long long)width);
  return SLDM_OK;
}

}  // namespace

extern "C" int sldm_layer_norm_fwd(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width,
                                   const float* weight, const float* bias, float eps, void* y, float* mean,
                                   float* rstd, void* stream) {
  if (const int rc = check_args(dtype, rows, width)) return rc;
  if (rows == 0) return SLDM_OK;
  SLDM_REQUIRE(x && y && (mean == nullptr) == (rstd == nullptr), "sldm_layer_norm_fwd: null argument");
  hipStream_t st = sldm::as_stream(stream);
  if (dtype == SLDM_F32)
    fwd<float>((const float*)x, ldx, rows, width, weight, bias, eps, (float*)y, mean, rstd, st);
  else
    fwd<uint16_t>((const uint16_t*)x, ldx, rows, width, weight, bias, eps, (uint16_t*)y, mean, rstd, st);
  SLDM_LAUNCH_CHECK("norm_fwd_kernel");
  return SLDM_OK;
}

extern "C" size_t sldm_layer_norm_bwd_workspace_bytes(int dtype, int64_t rows, int64_t width) {
  if (check_args(dtype, rows, width) != SLDM_OK) return 0;
  return (size_t)parts_of(shape_of(dtype, width, true), rows, width) * 2 * width * 4;
}

extern "C" int sldm_layer_norm_bwd(int dtype, const void* x, int64_t ldx, const void* dy, int64_t lddy,
                                   int64_t rows, int64_t width, const float* weight, const float* mean,
                                   const float* rstd, void* dx, float* dweight, float* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (const int rc = check_args(dtype, rows, width)) return rc;
  SLDM_REQUIRE(!(dweight || dbias) ||
                   (workspace && workspace_bytes >= sldm_layer_norm_bwd_workspace_bytes(dtype, rows, width)),
               "sldm_layer_norm_bwd: workspace too small");
  if (!dx && !dweight && !dbias) return SLDM_OK;
  SLDM_REQUIRE(rows == 0 || (x && dy && mean && rstd), "sldm_layer_norm_bwd: null argument");
  hipStream_t st = sldm::as_stream(stream);
  if (dtype == SLDM_F32)
    bwd<float>((const float*)x, ldx, (const float*)dy, lddy, rows, width, weight, mean, rstd, (float*)dx, dweight,
               dbias, (float*)workspace, st);
  else
    bwd<uint16_t>((const uint16_t*)x, ldx, (const uint16_t*)dy, lddy, rows, width, weight, mean, rstd,
                  (uint16_t*)dx, dweight, dbias, (float*)workspace, st);
  SLDM_LAUNCH_CHECK("norm_bwd_kernel");
  return SLDM_OK;
}
