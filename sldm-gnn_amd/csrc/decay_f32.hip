// Decay attention in fp32 (mathematics: decay.hpp): chunks of 16 tokens on
// v_mfma_f32_16x16x4_f32, operands straight from memory.
//
// A wave owns 16 or 32 value columns of one (batch, head, segment) and nothing
// is shared: no LDS, no barrier.  In fp32 an operand is one value a lane and
// product, so rows come as 16 bytes a lane (q, k: lane = row, four neighbouring
// columns are four products' contraction slots), and the transposed operands of
// P V and K^T V (lane = column) as 4-byte loads whose 16 lanes share a 64-byte
// piece of a row.  The chunk is as short as a tile because the products inside a
// chunk cost C (Dk + Dv) a token against 2 Dk Dv between chunks, and because a
// 16-wide head then wastes no part of a tile.  The next chunk's q and k are
// loaded over this chunk's second half, k^T and v over its first.
#include "decay.hpp"

namespace sldm_decay {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
constexpr int C = 16;

__device__ __forceinline__ f4v mfma(float a, float b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// four columns from `col` of a row of d; zeros past d
__device__ __forceinline__ f4v load4(const float* row, int col, int d, bool vec) {
  if (vec) return col < d ? *reinterpret_cast<const f4v*>(row + col) : f4v{0.f, 0.f, 0.f, 0.f};
  f4v v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = col + e < d ? row[col + e] : 0.f;
  return v;
}

template <int KT, int NV, bool OUT>
__global__ __launch_bounds__(256) void decay_f32_kernel(Args a) {
  const Role& R = a.role[blockIdx.y];
  const int slices = (R.vd + 16 * NV - 1) / (16 * NV);
  const int task = xcd_order() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = task / slices, v0 = task % slices * 16 * NV;
  if (id >= a.groups) return;
  const Span s = span_of(a, R, id);
  const int lane = threadIdx.x & 63, m = lane & 15, h = lane >> 4;
  const int kd = R.kd, vd = R.vd;
  const float ld2 = a.log_decay[s.hd] * 1.44269504088896340736f;
  const int seg = (int)(s.seg0 / a.seg_len);

  // state: lane = value column, registers = state rows 16 t + 4 h + r
  f4v S[KT][NV];
  {
    const float* s0 = R.s0 ? R.s0 + s.bh * R.s0_bh + seg * R.s0_seg : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kr = 16 * t + 4 * h + r, vc = v0 + 16 * v + m;
          S[t][v][r] = s0 && kr < kd && vc < vd ? s0[kr * R.s_k + vc * R.s_v] : 0.f;
        }
  }

  const int pad = (int)((C - s.n % C) % C);
  const int64_t nch = (s.n + pad) / C;
  const int64_t sign = R.reverse ? -1 : 1;
  const bool qvec = R.q.vec && kd % 4 == 0, kvec = R.k.vec && kd % 4 == 0;
  const float* qh = reinterpret_cast<const float*>(R.q.p) + s.b * R.q.sb + (s.hd / R.q.hdiv) * R.q.sh;
  const float* kh = reinterpret_cast<const float*>(R.k.p) + s.b * R.k.sb + (s.hd / R.k.hdiv) * R.k.sh;
  const float* vh = reinterpret_cast<const float*>(R.v.p) + s.b * R.v.sb + (s.hd / R.v.hdiv) * R.v.sh;
  const int64_t q_row = sign * m * R.q.st, k_row = sign * m * R.k.st;

  f4v q[KT], k[KT], kt[KT], vv[NV];
  auto load_rows = [&](int64_t x0, bool first) {     // q, k: lane = row m
    const int64_t tok = s.base + sign * x0;
    const float *qp = qh + tok * R.q.st + q_row, *kp = kh + tok * R.k.st + k_row;
    const bool on = !first || x0 + m >= 0;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      q[t] = k[t] = f4v{0.f, 0.f, 0.f, 0.f};
      if (on && 16 * t < kd) {
        q[t] = load4(qp, 16 * t + 4 * h, kd, qvec);
        k[t] = load4(kp, 16 * t + 4 * h, kd, kvec);
      }
    }
  };
  auto load_cols = [&](int64_t x0, bool first) {     // k^T, v: lane = column, registers = rows 4 h + r
    const int64_t tok = s.base + sign * x0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = 4 * h + r;
      const bool on = !first || x0 + j >= 0;
      const float *kp = kh + tok * R.k.st + sign * j * R.k.st, *vp = vh + tok * R.v.st + sign * j * R.v.st;
#pragma unroll
      for (int t = 0; t < KT; ++t) kt[t][r] = on && 16 * t + m < kd ? kp[16 * t + m] : 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) vv[v][r] = on && v0 + 16 * v + m < vd ? vp[v0 + 16 * v + m] : 0.f;
    }
  };

  float d[4], w[4];                                  // D (lane = i, registers = j), the update's weights
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = 4 * h + r;
    d[r] = m >= j ? powg(ld2, m - j) * R.p_scale : 0.f;
    w[r] = powg(ld2, C - 1 - j + R.delta) * R.upd_scale;
  }
  bool have_state = R.s0 != nullptr;
  if (OUT && nch > 0) load_rows(-pad, true);
  for (int64_t c = 0; c < nch; ++c) {
    const int64_t x0 = c * C - pad;
    const int padc = c == 0 ? pad : 0;
    load_cols(x0, c == 0);
    f4v O[NV];
    f4v P = {0.f, 0.f, 0.f, 0.f};
    if constexpr (OUT) {
#pragma unroll
      for (int v = 0; v < NV; ++v) O[v] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < KT; ++t)
        if (16 * t < kd)
#pragma unroll
          for (int r = 0; r < 4; ++r) P = mfma(k[t][r], q[t][r], P);
      if (have_state) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
          if (16 * t < kd)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int v = 0; v < NV; ++v) O[v] = mfma(S[t][v][r], q[t][r], O[v]);
        const float rd = powg(ld2, m - padc + 1 - R.delta) * R.read_scale;
#pragma unroll
        for (int v = 0; v < NV; ++v) O[v] *= rd;
      }
      if (c + 1 < nch) load_rows(x0 + C, false);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = P[r] * d[r];
#pragma unroll
        for (int v = 0; v < NV; ++v) O[v] = mfma(vv[v][r], p, O[v]);
      }
    }
    const float gn = powg(ld2, C - padc);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v) S[t][v] *= gn;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const float u = vv[v][r] * w[r];
#pragma unroll
        for (int t = 0; t < KT; ++t)
          if (16 * t < kd) S[t][v] = mfma(kt[t][r], u, S[t][v]);
      }
    have_state = true;
    if constexpr (OUT) {
      if (x0 + m >= 0) {
        float* o = reinterpret_cast<float*>(R.o) + s.b * R.o_sb + (s.base + sign * (x0 + m)) * R.o_st + s.hd * R.o_sh;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c0 = v0 + 16 * v + 4 * h;
          if (R.o_vec) {
            if (c0 < vd) *reinterpret_cast<f4v*>(o + c0) = O[v];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c0 + r < vd) o[c0 + r] = O[v][r];
          }
        }
      }
    }
  }
  if (R.s1) {
    float* s1 = R.s1 + s.bh * R.s1_bh + seg * R.s1_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kr = 16 * t + 4 * h + r, vc = v0 + 16 * v + m;
          if (kr < kd && vc < vd) s1[kr * R.s_k + vc * R.s_v] = S[t][v][r];
        }
  }
  if constexpr (OUT) {                               // tokens behind the sequence's end: zeros
    const int64_t t1 = s.seg0 + a.seg_len < a.T ? s.seg0 + a.seg_len : a.T;
    const int cols = vd - v0 < 16 * NV ? vd - v0 : 16 * NV;
    for (int64_t t = s.len > s.seg0 ? s.len : s.seg0; t < t1; ++t)
      if (lane < cols)
        reinterpret_cast<float*>(R.o)[s.b * R.o_sb + t * R.o_st + s.hd * R.o_sh + v0 + lane] = 0.f;
  }
}

template <int KT, bool OUT>
void launch(const Args& a, int roles, hipStream_t st) {
  int vd = 0;
  for (int i = 0; i < roles; ++i) vd = a.role[i].vd > vd ? a.role[i].vd : vd;
  const int nv = vd <= 16 ? 1 : 2;
  int64_t most = 0;
  for (int i = 0; i < roles; ++i) {
    const int64_t w = (int64_t)a.groups * ((a.role[i].vd + 16 * nv - 1) / (16 * nv));
    most = w > most ? w : most;
  }
  const unsigned grid = (unsigned)((most + 31) / 32 * 8);
  if (nv == 1) decay_f32_kernel<KT, 1, OUT><<<dim3(grid, roles), 256, 0, st>>>(a);
  else decay_f32_kernel<KT, 2, OUT><<<dim3(grid, roles), 256, 0, st>>>(a);
}

template <bool OUT>
void by_rows(const Args& a, int roles, hipStream_t st) {
  int kd = 0;
  for (int i = 0; i < roles; ++i) kd = a.role[i].kd > kd ? a.role[i].kd : kd;
  if (kd <= 16) launch<1, OUT>(a, roles, st);
  else if (kd <= 32) launch<2, OUT>(a, roles, st);
  else if (kd <= 64) launch<4, OUT>(a, roles, st);
  else launch<8, OUT>(a, roles, st);
}

}  // namespace

void run_f32(const Args& a, int roles, bool out, hipStream_t st) {
  out ? by_rows<true>(a, roles, st) : by_rows<false>(a, roles, st);
}

}  // namespace sldm_decay
