// Linear attention with a decay for each head: the chunked sequence kernel.
//
//   S_t = g S_{t-1} + k_t v_t^T        S [Dk, Dv] fp32, g = exp(log_decay[h])
//   o_t = scale q_t S_t
//
// over C consecutive tokens at once (i, j count inside the chunk, S is the
// state before it):
//   O   = scale ((Q K^T o D) V + diag(g^{i+1}) Q S),   D_ij = g^{i-j}, i >= j
//   S' <- g^C S + K^T diag(g^{C-1-j}) V
// Every exponent is >= 0, so no decay, however strong, overflows.
//
// The gradients are the same recurrence with other operands
//   dq_t = scale S_t do_t                              q,k,v := do, v, k   (S^T)
//   G_t  = scale q_t do_t^T + g G_{t+1}                time reversed
//   dv_t = k_t G_t                                     q,k,v := k, q, do   (G)
//   dk_t = G_t v_t                                     q,k,v := v, do, q   (G^T)
// so one kernel serves all of them: a Role names the operands, the direction
// of time, where the scale goes and how the state is laid out.  In reversed
// time the state is kept already decayed to the next token (delta = 1): its
// weight on position i is g^i and position j enters with g^{n-j}, so the
// final state's gradient starts it as it is and the initial state's comes out.
//
// Layout: a workgroup owns one (batch, head, segment) and walks its chunks; a
// wave owns 32 value columns and keeps its Dk x 32 slice of S in MFMA
// accumulators for the whole walk.  The accumulator layout (lane = column,
// registers = rows) is at once an A operand (rows = lane, k = register), so S
// feeds diag() Q S from registers, and so does P = Q K^T o D, computed
// transposed: neither goes through LDS.  Q, K and V tiles are staged in LDS
// (16-byte granules XOR-swizzled so that both the row reads and the transposed
// reads spread over the banks) while the next chunk's loads are in flight.
// A sequence is aligned to the END of its chunks: the first chunk is padded
// with zero rows in front, which leaves every decay table a constant.
//
// bf16: v_mfma_f32_32x32x16_bf16, fp32 accumulation.  P is rounded to bf16
// once (its products with V are exact), like the output it feeds; S is read
// as hi + lo (16 significant bits), and the state's update takes V g^{n-1-j}
// as hi + mid + lo (all 24), so the state is an fp32 sum of exact products.
// fp32: v_mfma_f32_32x32x2_f32 throughout.
#pragma once

#include "common.hpp"

namespace sldm_decay {

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct Operand {
  const void* p;
  int64_t sb, st, sh;   // element strides of batch, token, head; columns are contiguous
  int hdiv;             // head h reads head h / hdiv
  int vec;              // every row starts on a 16-byte boundary
};

struct Role {
  Operand q, k, v;      // q, k: kd columns; v: vd columns
  void* o;              // [B, T, H, vd] with strides below; null: the state only
  int64_t o_sb, o_st, o_sh;
  int o_f32, o_vec;
  const float* s0;      // state before each segment (null: zero); element (a, c) at a s_k + c s_v
  float* s1;            // state behind each segment (null: not written), the same layout
  int64_t s0_bh, s0_seg, s1_bh, s1_seg;
  int64_t s_k, s_v;
  float read_scale, p_scale, upd_scale;
  int delta, reverse;
  int kd, vd;
};

struct Args {
  Role role[3];
  int64_t B, H, T, seg_len;
  int nseg, groups;     // groups = B H nseg
  const float* log_decay;
  const void* lengths;  // null: T each
  int lengths64;
};

__device__ __forceinline__ float powg(float ld2, int n) { return n <= 0 ? 1.f : exp2f(ld2 * (float)n); }

__device__ __forceinline__ int64_t seq_len(const Args& a, int64_t b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.lengths64 ? reinterpret_cast<const int64_t*>(a.lengths)[b]
                                : (int64_t)reinterpret_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// Swizzle of row r for rows of RB bytes: the XOR on its 16-byte granules.
// bf16: the four rows of a transposed read (64 bytes each) fall into the four
// quarters of the 64 banks, and eight rows read at one granule into eight
// granules.  fp32: eight rows at one granule.
template <typename T, int RB>
__device__ __forceinline__ int swz(int r) {
  if constexpr (sizeof(T) == 4) return r & 7;
  else if constexpr (RB == 64) return ((r >> 2) & 1) | ((r >> 2) & 2);
  else if constexpr (RB == 128) return ((r & 2) << 1) | ((r >> 2) & 1) | ((r >> 2) & 2);
  else return ((r & 3) << 2) | ((r >> 2) & 1) | ((r >> 2) & 2);
}

template <typename T> struct Elem;
template <> struct Elem<uint16_t> {
  static constexpr int kChunk = 64;
};
template <> struct Elem<float> {
  static constexpr int kChunk = 32;
};

// One 16-byte granule (elements e0 ..) of a row of d elements; zeros past d.
template <typename T>
__device__ __forceinline__ uint4 load_granule(const T* row, int e0, int d, bool vec) {
  constexpr int E = 16 / sizeof(T);
  if (vec && e0 + E <= d) return *reinterpret_cast<const uint4*>(row + e0);
  T tmp[E];
#pragma unroll
  for (int e = 0; e < E; ++e) tmp[e] = e0 + e < d ? row[e0 + e] : T(0);
  uint4 w;
  __builtin_memcpy(&w, tmp, 16);
  return w;
}

// A C x (DT * 32) tile held by the workgroup's registers on its way to LDS.
template <typename T, int DT, int NTH>
struct Stage {
  static constexpr int C = Elem<T>::kChunk;
  static constexpr int RB = DT * 32 * (int)sizeof(T);
  static constexpr int GR = RB / 16;
  static constexpr int N = (C * GR + NTH - 1) / NTH;
  uint4 w[N];
  // rows r of the tile are positions x = x0 + r of the segment (x < 0: zero);
  // position x is token base + x, or base - x in reversed time
  __device__ __forceinline__ void load(const Operand& t, const T* head, int64_t x0, int64_t base,
                                       int reverse, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = (int)threadIdx.x + i * NTH;
      const int r = idx / GR, g = idx % GR;
      const int64_t x = x0 + r;
      w[i] = make_uint4(0, 0, 0, 0);
      if (r < C && x >= 0 && g * (16 / (int)sizeof(T)) < d) {
        const int64_t tok = reverse ? base - x : base + x;
        w[i] = load_granule<T>(head + tok * t.st, g * (16 / (int)sizeof(T)), d, t.vec);
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = (int)threadIdx.x + i * NTH;
      const int r = idx / GR, g = idx % GR;
      if (r < C) *reinterpret_cast<uint4*>(lds + r * RB + ((g ^ swz<T, RB>(r)) << 4)) = w[i];
    }
  }
};

// lane -> column inside a 32-wide tile (bf16): the middle two bits of each
// 16-group swapped, which makes the eight accumulator rows 8s .. 8s+7 of a half
// wave eight consecutive columns (16-byte stores, and 16-byte operand reads).
__device__ __forceinline__ int perm16(int m) {
  return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1);
}

// MFMA operand whose rows are the tile's columns: lane m of tile ct holds
// column 32 ct + perm16(m) of the eight rows t0 + 8h .. + 7.
template <int RB>
__device__ __forceinline__ bf8v tr_frag(const char* lds, int ct, int t0, int lane) {
  const int q = lane >> 4, r16 = lane & 15;
  const int blk = r16 & 3, b = ((blk & 1) << 1) | (blk >> 1);
  const int g = 4 * ct + 2 * (q & 1) + (b >> 1);
  const int r0 = t0 + 8 * (q >> 1) + (r16 >> 2), r1 = r0 + 4;
  const char* p0 = lds + r0 * RB + ((g ^ swz<uint16_t, RB>(r0)) << 4) + ((b & 1) << 3);
  const char* p1 = lds + r1 * RB + ((g ^ swz<uint16_t, RB>(r1)) << 4) + ((b & 1) << 3);
  typedef __attribute__((address_space(3))) s4v* lp;
  const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p0));
  const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p1));
  typedef short s8v __attribute__((ext_vector_type(8)));
  const s8v v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf8v, v);
}

// MFMA operand whose rows are the tile's rows: eight columns 16 step + 8h ..
template <int RB>
__device__ __forceinline__ bf8v row_frag(const char* lds, int row, int step, int h) {
  return *reinterpret_cast<const bf8v*>(lds + row * RB + (((2 * step + h) ^ swz<uint16_t, RB>(row)) << 4));
}

__device__ __forceinline__ bf8v pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = sldm::pack_bf16x2(v[2 * e], v[2 * e + 1]);
  return __builtin_bit_cast(bf8v, make_uint4(w[0], w[1], w[2], w[3]));
}

// ------------------------------------------------------------- bf16 chunk --
template <int KT, int NW, bool OUT>
struct ChunkBf16 {
  static constexpr int C = 64, NT = 2, RBK = KT * 64, RBV = NW * 64;
  // O[it]: lane = token 32 it + (lane & 31), registers 8s + e = value column
  // 16s + 8h + e of the wave's 32.
  static __device__ __forceinline__ void run(const char* lq, const char* lk, const char* lv,
                                             const float* wtab, int wave, int lane, int kd,
                                             bool have_state, const float (&d0)[16],
                                             const float (&d1)[16], const float (&rd)[NT], float gn,
                                             f16v (&S)[KT], f16v (&O)[NT]) {
    const int m = lane & 31, h = lane >> 5, pm = perm16(m);
    bf8v vf[NT][2];
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
#pragma unroll
      for (int s = 0; s < 2; ++s) vf[jt][s] = tr_frag<RBV>(lv, wave, 32 * jt + 16 * s, lane);
    if constexpr (OUT) {
#pragma unroll
      for (int it = 0; it < NT; ++it)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[it][r] = 0.f;
      if (have_state) {
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t) {
          if (16 * t < kd) {
            float a[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = S[t >> 1][8 * (t & 1) + e];
            sldm::bf16x8 hi, lo;
            sldm::split_bf16x8(a, hi, lo);
#pragma unroll
            for (int it = 0; it < NT; ++it) {
              const bf8v qf = row_frag<RBK>(lq, 32 * it + m, t, h);
              O[it] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, lo), qf, O[it], 0, 0, 0);
              O[it] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, hi), qf, O[it], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int it = 0; it < NT; ++it)
#pragma unroll
          for (int r = 0; r < 16; ++r) O[it][r] *= rd[it];
      }
#pragma unroll
      for (int it = 0; it < NT; ++it)
#pragma unroll
        for (int jt = 0; jt <= it; ++jt) {
          f16v P;
#pragma unroll
          for (int r = 0; r < 16; ++r) P[r] = 0.f;
#pragma unroll
          for (int t = 0; t < 2 * KT; ++t)
            if (16 * t < kd)
              P = __builtin_amdgcn_mfma_f32_32x32x16_bf16(row_frag<RBK>(lk, 32 * jt + pm, t, h),
                                                          row_frag<RBK>(lq, 32 * it + m, t, h), P, 0, 0, 0);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            float a[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = P[8 * s + e] * (it == jt ? d0[8 * s + e] : d1[8 * s + e]);
            O[it] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[jt][s], pack8(a), O[it], 0, 0, 0);
          }
        }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] *= gn;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float* w = wtab + 32 * jt + 16 * s + 8 * h;
        const uint4 u = __builtin_bit_cast(uint4, vf[jt][s]);
        float a[8] = {sldm::bf16_lo(u.x) * w[0], sldm::bf16_hi(u.x) * w[1], sldm::bf16_lo(u.y) * w[2],
                      sldm::bf16_hi(u.y) * w[3], sldm::bf16_lo(u.z) * w[4], sldm::bf16_hi(u.z) * w[5],
                      sldm::bf16_lo(u.w) * w[6], sldm::bf16_hi(u.w) * w[7]};
        sldm::bf16x8 hi, mid, lo;
        sldm::split3_bf16x8(a, hi, mid, lo);
#pragma unroll
        for (int t = 0; t < KT; ++t)
          if (32 * t < kd) {
            const bf8v kf = tr_frag<RBK>(lk, t, 32 * jt + 16 * s, lane);
            S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, __builtin_bit_cast(bf8v, lo), S[t], 0, 0, 0);
            S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, __builtin_bit_cast(bf8v, mid), S[t], 0, 0, 0);
            S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, __builtin_bit_cast(bf8v, hi), S[t], 0, 0, 0);
          }
      }
  }
};

// ------------------------------------------------------------- fp32 chunk --
template <int KT, int NW, bool OUT>
struct ChunkF32 {
  static constexpr int C = 32, NT = 1, RBK = KT * 128, RBV = NW * 128;
  static __device__ __forceinline__ float elem(const char* lds, int rb, int row, int col) {
    return *reinterpret_cast<const float*>(lds + row * rb + (((col >> 2) ^ (row & 7)) << 4) + ((col & 3) << 2));
  }
  static __device__ __forceinline__ float4 row4(const char* lds, int row, int u, int h) {
    return *reinterpret_cast<const float4*>(lds + row * RBK + (((2 * u + h) ^ (row & 7)) << 4));
  }
  static __device__ __forceinline__ void run(const char* lq, const char* lk, const char* lv,
                                             const float* wtab, int wave, int lane, int kd,
                                             bool have_state, const float (&d0)[16],
                                             const float (&)[16], const float (&rd)[NT], float gn,
                                             f16v (&S)[KT], f16v (&O)[NT]) {
    const int m = lane & 31, h = lane >> 5;
    if constexpr (OUT) {
      f16v P;
#pragma unroll
      for (int r = 0; r < 16; ++r) O[0][r] = P[r] = 0.f;
#pragma unroll
      for (int u = 0; u < 4 * KT; ++u)
        if (8 * u < kd) {
          const float4 q = row4(lq, m, u, h), k = row4(lk, m, u, h);
          P = __builtin_amdgcn_mfma_f32_32x32x2f32(k.x, q.x, P, 0, 0, 0);
          P = __builtin_amdgcn_mfma_f32_32x32x2f32(k.y, q.y, P, 0, 0, 0);
          P = __builtin_amdgcn_mfma_f32_32x32x2f32(k.z, q.z, P, 0, 0, 0);
          P = __builtin_amdgcn_mfma_f32_32x32x2f32(k.w, q.w, P, 0, 0, 0);
          if (have_state) {
            const int t = u >> 2, r = 4 * (u & 3);
            O[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(S[t][r], q.x, O[0], 0, 0, 0);
            O[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(S[t][r + 1], q.y, O[0], 0, 0, 0);
            O[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(S[t][r + 2], q.z, O[0], 0, 0, 0);
            O[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(S[t][r + 3], q.w, O[0], 0, 0, 0);
          }
        }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        O[0][r] *= rd[0];
        P[r] *= d0[r];
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 8 * (r >> 2) + 4 * h + (r & 3);
        O[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(elem(lv, RBV, j, 32 * wave + m), P[r], O[0], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] *= gn;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = 8 * (r >> 2) + 4 * h + (r & 3);
      const float v = elem(lv, RBV, j, 32 * wave + m) * wtab[j];
#pragma unroll
      for (int t = 0; t < KT; ++t)
        if (32 * t < kd)
          S[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(elem(lk, RBK, j, 32 * t + m), v, S[t], 0, 0, 0);
    }
  }
};

template <typename T, int KT, int NW, bool OUT> struct ChunkOf;
template <int KT, int NW, bool OUT> struct ChunkOf<uint16_t, KT, NW, OUT> { using type = ChunkBf16<KT, NW, OUT>; };
template <int KT, int NW, bool OUT> struct ChunkOf<float, KT, NW, OUT> { using type = ChunkF32<KT, NW, OUT>; };

// LDS of one workgroup: q, k, v tiles and the update's decay table.
template <typename T, int KT, int NW, bool OUT>
constexpr int lds_bytes() {
  return Elem<T>::kChunk * 32 * (int)sizeof(T) * (KT * (OUT ? 2 : 1) + NW) + Elem<T>::kChunk * 4;
}

template <typename T, int KT, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW, NW == 1 ? 2 : 2) void decay_kernel(Args a) {
  using Chunk = typename ChunkOf<T, KT, NW, OUT>::type;
  constexpr int C = Chunk::C, NT = Chunk::NT, NTH = 64 * NW;
  constexpr int kTileK = C * Chunk::RBK, kTileV = C * Chunk::RBV;
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<T, KT, NW, OUT>()];
  char* lk = smem;
  char* lv = smem + kTileK;
  char* lq = smem + kTileK + kTileV;
  float* wtab = reinterpret_cast<float*>(smem + kTileK * (OUT ? 2 : 1) + kTileV);

  // Workgroups are dealt to the XCDs in turn; neighbours in (segment, head,
  // batch) order, whose rows share cache lines, are put on one XCD.
  const int per = (int)gridDim.x >> 3;
  const int id = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if (id >= a.groups) return;
  const Role& R = a.role[blockIdx.y];
  const int64_t bh = id % (a.groups / a.nseg);
  const int seg = id / (a.groups / a.nseg);
  const int64_t b = bh / a.H, hd = bh % a.H;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;

  const int64_t len = seq_len(a, b);
  const int64_t seg0 = (int64_t)seg * a.seg_len;
  const int64_t left = len - seg0;
  const int64_t n = left < 0 ? 0 : (left < a.seg_len ? left : a.seg_len);
  const int pad = (int)((C - n % C) % C);
  const int64_t nch = (n + pad) / C;
  const int64_t base = R.reverse ? len - 1 - seg0 : seg0;
  const float ld2 = a.log_decay[hd] * 1.44269504088896340736f;

  const T* qh = OUT ? reinterpret_cast<const T*>(R.q.p) + b * R.q.sb + (hd / R.q.hdiv) * R.q.sh : nullptr;
  const T* kh = reinterpret_cast<const T*>(R.k.p) + b * R.k.sb + (hd / R.k.hdiv) * R.k.sh;
  const T* vh = reinterpret_cast<const T*>(R.v.p) + b * R.v.sb + (hd / R.v.hdiv) * R.v.sh;

  // ---- the wave's slice of the state: lane = value column, registers = rows
  const int vc = 32 * wave + (sizeof(T) == 2 ? perm16(m) : m);
  auto krow = [&](int t, int r) {   // state row of accumulator register r
    return sizeof(T) == 2 ? 32 * t + 16 * (r >> 3) + 8 * h + (r & 7)
                          : 32 * t + 8 * (r >> 2) + 4 * h + (r & 3);
  };
  f16v S[KT];
  {
    const float* s0 = R.s0 ? R.s0 + bh * R.s0_bh + seg * R.s0_seg : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = krow(t, r);
        S[t][r] = s0 && kr < R.kd && vc < R.vd ? s0[kr * R.s_k + vc * R.s_v] : 0.f;
      }
  }
  float d0[16], d1[16];
  if constexpr (OUT) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = m, j = krow(0, r);
      d0[r] = i >= j ? powg(ld2, i - j) * R.p_scale : 0.f;
      d1[r] = powg(ld2, 32 + i - j) * R.p_scale;
    }
  }
  for (int j = threadIdx.x; j < C; j += NTH) wtab[j] = powg(ld2, C - 1 - j + R.delta) * R.upd_scale;

  bool have_state = R.s0 != nullptr;
  Stage<T, KT, NTH> sq, sk;
  Stage<T, NW, NTH> sv;
  if (nch > 0) {
    if constexpr (OUT) sq.load(R.q, qh, -pad, base, R.reverse, R.kd);
    sk.load(R.k, kh, -pad, base, R.reverse, R.kd);
    sv.load(R.v, vh, -pad, base, R.reverse, R.vd);
  }
  for (int64_t c = 0; c < nch; ++c) {
    __syncthreads();   // the last chunk's tiles are no longer read
    if constexpr (OUT) sq.store(lq);
    sk.store(lk);
    sv.store(lv);
    __syncthreads();
    if (c + 1 < nch) {
      const int64_t x0 = (c + 1) * C - pad;
      if constexpr (OUT) sq.load(R.q, qh, x0, base, R.reverse, R.kd);
      sk.load(R.k, kh, x0, base, R.reverse, R.kd);
      sv.load(R.v, vh, x0, base, R.reverse, R.vd);
    }
    const int padc = c == 0 ? pad : 0;
    float rd[NT];
#pragma unroll
    for (int it = 0; it < NT; ++it)
      rd[it] = powg(ld2, 32 * it + m - padc + 1 - R.delta) * R.read_scale;
    f16v O[NT];
    Chunk::run(lq, lk, lv, wtab, wave, lane, R.kd, have_state, d0, d1, rd, powg(ld2, C - padc), S, O);
    have_state = true;
    if constexpr (OUT) {
#pragma unroll
      for (int it = 0; it < NT; ++it) {
        const int64_t x = c * C + 32 * it + m - pad;
        if (x >= 0) {
          const int64_t tok = R.reverse ? base - x : base + x;
          const int64_t off = b * R.o_sb + tok * R.o_st + hd * R.o_sh;
          // registers E s .. E s + E - 1 are consecutive columns
          constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
          for (int s = 0; s < 16 / E; ++s) {
            const int c0 = 32 * wave + 2 * E * s + E * h;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = O[it][E * s + e];
            if (sizeof(T) == 4 || R.o_f32) {
              float* o = reinterpret_cast<float*>(R.o) + off + c0;
              if (R.o_vec && c0 + E <= R.vd) {
#pragma unroll
                for (int e = 0; e < E; e += 4) sldm::Vec<float, 4>::store(o + e, v + e);
              } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                  if (c0 + e < R.vd) o[e] = v[e];
              }
            } else {
              T* o = reinterpret_cast<T*>(R.o) + off + c0;
              if (R.o_vec && c0 + E <= R.vd) {
                sldm::Vec<T, E>::store(o, v);
              } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                  if (c0 + e < R.vd) sldm::Vec<T, 1>::store(o + e, v + e);
              }
            }
          }
        }
      }
    }
  }
  if (R.s1) {
    float* s1 = R.s1 + bh * R.s1_bh + seg * R.s1_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = krow(t, r);
        if (kr < R.kd && vc < R.vd) s1[kr * R.s_k + vc * R.s_v] = S[t][r];
      }
  }
  if constexpr (OUT) {
    // tokens behind the sequence's end: zeros
    const int64_t t1 = seg0 + a.seg_len < a.T ? seg0 + a.seg_len : a.T;
    const int64_t t0 = len > seg0 ? len : seg0;
    const int64_t todo = t1 > t0 ? (t1 - t0) * R.vd : 0;
    for (int64_t i = threadIdx.x; i < todo; i += NTH) {
      const int64_t off = b * R.o_sb + (t0 + i / R.vd) * R.o_st + hd * R.o_sh + i % R.vd;
      if (sizeof(T) == 4 || R.o_f32) reinterpret_cast<float*>(R.o)[off] = 0.f;
      else reinterpret_cast<T*>(R.o)[off] = T(0);
    }
  }
}

template <typename T, int KT, int NW, bool OUT>
void launch(const Args& a, int roles, hipStream_t stream) {
  const unsigned grid = (unsigned)((a.groups + 7) / 8 * 8);
  decay_kernel<T, KT, NW, OUT><<<dim3(grid, roles), 64 * NW, 0, stream>>>(a);
}

inline int tiles_of(int d) { return d <= 32 ? 1 : d <= 64 ? 2 : 4; }

template <typename T, bool OUT>
void dispatch(const Args& a, int roles, hipStream_t stream) {
  const int kt = tiles_of(a.role[0].kd), nw = tiles_of(a.role[0].vd);
#define SLDM_DECAY_NW(KT)                                          \
  (nw == 1 ? launch<T, KT, 1, OUT>(a, roles, stream)               \
           : nw == 2 ? launch<T, KT, 2, OUT>(a, roles, stream) : launch<T, KT, 4, OUT>(a, roles, stream))
  if (kt == 1) SLDM_DECAY_NW(1);
  else if (kt == 2) SLDM_DECAY_NW(2);
  else SLDM_DECAY_NW(4);
#undef SLDM_DECAY_NW
}

// One launch of `roles` roles whose kd and vd fall into the same tile classes
// (decay_bf16.hip, decay_f32.hip).  out: roles write outputs; else states only.
void run_bf16(const Args& a, int roles, bool out, hipStream_t stream);
void run_f32(const Args& a, int roles, bool out, hipStream_t stream);

}  // namespace sldm_decay
