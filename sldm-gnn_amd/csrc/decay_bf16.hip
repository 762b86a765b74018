// Decay attention in bf16 (mathematics: decay.hpp): chunks of 64 tokens on
// v_mfma_f32_32x32x16_bf16, fp32 accumulation.
//
// A workgroup owns one (batch, head, segment); a wave owns 32 value columns and
// keeps its Dk x 32 slice of the state in accumulators for the whole walk.  Q, K
// and V tiles are staged in LDS while the next chunk's loads are in flight; rows
// are padded so that row reads (16 bytes of eight rows) and transposed reads
// (ds_read_b64_tr_b16: 64 bytes of four rows) spread over the banks with plain
// offsets, no address arithmetic a read.
//
// Roundings.  P = Q K^T o D goes into P V as hi + lo (16 significant bits): the
// rows of a short sequence hang on single entries of P.  The state is held in
// fp32 and read as bf16 (each of the Dk products of an output is off by 2^-9 or
// so of itself, at random: together like the rounding of the output).  The
// state's update takes V g^{n-1-j} as hi + mid + lo (all 24 bits) where the state
// is an output, hi + mid where it only feeds outputs of this type.
#include "decay.hpp"

namespace sldm_decay {
namespace {

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int C = 64, NT = C / 32;

__device__ __forceinline__ f16v mfma(bf8v a, bf8v b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf8v as_bf8(sldm::bf16x8 v) { return __builtin_bit_cast(bf8v, v); }
__device__ __forceinline__ bf8v pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = sldm::pack_bf16x2(v[2 * e], v[2 * e + 1]);
  return __builtin_bit_cast(bf8v, make_uint4(w[0], w[1], w[2], w[3]));
}

// Bytes of an LDS row of 32 DT values: 20, 36 or 84 banks, so eight rows at one
// 16-byte column hit eight different groups of banks.
constexpr int row_bytes(int dt) { return dt == 1 ? 80 : dt == 2 ? 144 : 336; }

// One 16-byte granule (elements e0 ..) of a row of d elements; zeros past d.
__device__ __forceinline__ uint4 load_granule(const uint16_t* row, int e0, int d, bool vec) {
  if (vec && e0 + 8 <= d) return *reinterpret_cast<const uint4*>(row + e0);
  uint16_t tmp[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) tmp[e] = e0 + e < d ? row[e0 + e] : (uint16_t)0;
  uint4 w;
  __builtin_memcpy(&w, tmp, 16);
  return w;
}

// A tile of C rows on its way through the workgroup's registers to LDS.
template <int DT, int NTH>
struct Stage {
  static constexpr int GR = DT * 4, N = C * GR / NTH;
  static_assert(C * GR % NTH == 0, "whole granules a thread");
  uint4 w[N];
  // rows r of the tile are positions x0 + r of the segment (below 0: zeros)
  __device__ __forceinline__ void load(const Operand& t, const uint16_t* head, int64_t x0, int64_t base,
                                       int reverse, int d) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = (int)threadIdx.x + i * NTH, r = idx / GR, g = idx % GR;
      const int64_t x = x0 + r;
      w[i] = make_uint4(0, 0, 0, 0);
      if (x >= 0 && g * 8 < d) w[i] = load_granule(head + (reverse ? base - x : base + x) * t.st, g * 8, d, t.vec);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = (int)threadIdx.x + i * NTH;
      *reinterpret_cast<uint4*>(lds + idx / GR * row_bytes(DT) + idx % GR * 16) = w[i];
    }
  }
};

// lane -> column (or row) inside a 32-wide tile: the middle two bits of each
// 16-group swapped, which makes the accumulator rows 8 s .. 8 s + 7 of a half
// wave eight neighbours: 16 s + 8 h + e.
__device__ __forceinline__ int perm16(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// Operand whose rows are the tile's columns: lane m holds column perm16(m) of
// eight rows from 8 h (p: tr_base), all shifted by `off` bytes.
__device__ __forceinline__ int tr_base(int lane, int rs) {
  const int q = lane >> 4, r16 = lane & 15, blk = r16 & 3, b = ((blk & 1) << 1) | (blk >> 1);
  return (8 * (q >> 1) + (r16 >> 2)) * rs + 32 * (q & 1) + 8 * b;
}
__device__ __forceinline__ bf8v tr_frag(const char* p, int rs) {
  typedef __attribute__((address_space(3))) s4v* lp;
  const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
  const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * rs));
  return __builtin_bit_cast(bf8v, s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

template <int KT, int NW, bool OUT>
__global__ __launch_bounds__(64 * NW, 2) void decay_bf16_kernel(Args a) {
  constexpr int NTH = 64 * NW, RSK = row_bytes(KT), RSV = row_bytes(NW);
  __shared__ __attribute__((aligned(16))) char lk[C * RSK], lv[C * RSV], lq[OUT ? C * RSK : 16];
  __shared__ __attribute__((aligned(16))) float wtab[C], dtab[96];

  const int id = xcd_order();
  if (id >= a.groups) return;
  const Role& R = a.role[blockIdx.y];
  const Span sp = span_of(a, R, id);
  const int seg = (int)(sp.seg0 / a.seg_len);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;
  const int kd = R.kd, vd = R.vd;
  const int pad = (int)((C - sp.n % C) % C);
  const int64_t nch = (sp.n + pad) / C;
  const float ld2 = a.log_decay[sp.hd] * 1.44269504088896340736f;
  const bool exact = R.s1 != nullptr;

  const uint16_t* qh = OUT ? reinterpret_cast<const uint16_t*>(R.q.p) + sp.b * R.q.sb + (sp.hd / R.q.hdiv) * R.q.sh : nullptr;
  const uint16_t* kh = reinterpret_cast<const uint16_t*>(R.k.p) + sp.b * R.k.sb + (sp.hd / R.k.hdiv) * R.k.sh;
  const uint16_t* vh = reinterpret_cast<const uint16_t*>(R.v.p) + sp.b * R.v.sb + (sp.hd / R.v.hdiv) * R.v.sh;

  Stage<KT, NTH> sq, sk;
  Stage<NW, NTH> sv;
  if (nch > 0) {
    if constexpr (OUT) sq.load(R.q, qh, -pad, sp.base, R.reverse, kd);
    sk.load(R.k, kh, -pad, sp.base, R.reverse, kd);
    sv.load(R.v, vh, -pad, sp.base, R.reverse, vd);
  }
  // state: lane = value column, register 8 s + e of tile t = row 32 t + 16 s + 8 h + e
  const int vc = 32 * wave + perm16(m);
  f16v S[KT];
  {
    const float* s0 = R.s0 ? R.s0 + sp.bh * R.s0_bh + seg * R.s0_seg : nullptr;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = 32 * t + 16 * (r >> 3) + 8 * h + (r & 7);
        S[t][r] = s0 && kr < kd && vc < vd ? s0[kr * R.s_k + vc * R.s_v] : 0.f;
      }
  }
  // wtab[j]: the weight with which row j enters the state; dtab[32 + i - j]: D
  for (int j = threadIdx.x; j < C; j += NTH) wtab[j] = powg(ld2, C - 1 - j + R.delta) * R.upd_scale;
  for (int j = threadIdx.x; j < 96; j += NTH) dtab[j] = j < 32 ? 0.f : powg(ld2, j - 32) * R.p_scale;

  const char* pq = lq + m * RSK + 16 * h;                       // row m, columns 16 t + 8 h ..
  const char* pk = lk + perm16(m) * RSK + 16 * h;
  const char* tk = lk + tr_base(lane, RSK);
  const char* tv = lv + tr_base(lane, RSV) + 64 * wave;
  const float* pd = dtab + 9 + m - 8 * h;                       // + 23 - (16 s + e): entry 32 + m - j
  const float* pw = wtab + 8 * h;

  bool have_state = R.s0 != nullptr;
  for (int64_t c = 0; c < nch; ++c) {
    __syncthreads();                                            // the last chunk's tiles are no longer read
    if constexpr (OUT) sq.store(lq);
    sk.store(lk);
    sv.store(lv);
    __syncthreads();
    if (c + 1 < nch) {
      const int64_t x0 = (c + 1) * C - pad;
      if constexpr (OUT) sq.load(R.q, qh, x0, sp.base, R.reverse, kd);
      sk.load(R.k, kh, x0, sp.base, R.reverse, kd);
      sv.load(R.v, vh, x0, sp.base, R.reverse, vd);
    }
    const int padc = c == 0 ? pad : 0;
    bf8v vf[NT][2];
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
#pragma unroll
      for (int s = 0; s < 2; ++s) vf[jt][s] = tr_frag(tv + (32 * jt + 16 * s) * RSV, RSV);

    if constexpr (OUT) {
      f16v O[NT];
#pragma unroll
      for (int it = 0; it < NT; ++it)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[it][r] = 0.f;
      if (have_state) {
#pragma unroll
        for (int t = 0; t < 2 * KT; ++t)
          if (16 * t < kd) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = S[t >> 1][8 * (t & 1) + e];
            const bf8v sf = pack8(x);
#pragma unroll
            for (int it = 0; it < NT; ++it)
              O[it] = mfma(sf, *reinterpret_cast<const bf8v*>(pq + 32 * it * RSK + 32 * t), O[it]);
          }
#pragma unroll
        for (int it = 0; it < NT; ++it) {
          const float rd = powg(ld2, 32 * it + m - padc + 1 - R.delta) * R.read_scale;
#pragma unroll
          for (int r = 0; r < 16; ++r) O[it][r] *= rd;
        }
      }
#pragma unroll
      for (int it = 0; it < NT; ++it) {
#pragma unroll
        for (int jt = 0; jt <= it; ++jt) {
          f16v P;
#pragma unroll
          for (int r = 0; r < 16; ++r) P[r] = 0.f;
#pragma unroll
          for (int t = 0; t < 2 * KT; ++t)
            if (16 * t < kd)
              P = mfma(*reinterpret_cast<const bf8v*>(pk + 32 * jt * RSK + 32 * t),
                       *reinterpret_cast<const bf8v*>(pq + 32 * it * RSK + 32 * t), P);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = P[8 * s + e] * pd[32 * (it - jt) + 23 - 16 * s - e];
            sldm::bf16x8 hi, lo;
            sldm::split_bf16x8(x, hi, lo);
            O[it] = mfma(vf[jt][s], as_bf8(lo), O[it]);
            O[it] = mfma(vf[jt][s], as_bf8(hi), O[it]);
          }
        }
        // lane = token 32 it + m, registers 8 s + e = columns 16 s + 8 h + e
        const int64_t x = c * C + 32 * it + m - pad;
        if (x >= 0) {
          const int64_t tok = R.reverse ? sp.base - x : sp.base + x;
          const int64_t off = sp.b * R.o_sb + tok * R.o_st + sp.hd * R.o_sh;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int c0 = 32 * wave + 16 * s + 8 * h;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = O[it][8 * s + e];
            if (R.o_f32) {
              float* o = reinterpret_cast<float*>(R.o) + off + c0;
              if (R.o_vec && c0 + 8 <= vd) {
                sldm::Vec<float, 4>::store(o, y);
                sldm::Vec<float, 4>::store(o + 4, y + 4);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (c0 + e < vd) o[e] = y[e];
              }
            } else {
              uint16_t* o = reinterpret_cast<uint16_t*>(R.o) + off + c0;
              if (R.o_vec && c0 + 8 <= vd) {
                sldm::Vec<uint16_t, 8>::store(o, y);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (c0 + e < vd) o[e] = sldm::f32_to_bf16(y[e]);
              }
            }
          }
        }
      }
    }
    const float gn = powg(ld2, C - padc);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] *= gn;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float* w = pw + 32 * jt + 16 * s;
        const uint4 u = __builtin_bit_cast(uint4, vf[jt][s]);
        const float x[8] = {sldm::bf16_lo(u.x) * w[0], sldm::bf16_hi(u.x) * w[1], sldm::bf16_lo(u.y) * w[2],
                            sldm::bf16_hi(u.y) * w[3], sldm::bf16_lo(u.z) * w[4], sldm::bf16_hi(u.z) * w[5],
                            sldm::bf16_lo(u.w) * w[6], sldm::bf16_hi(u.w) * w[7]};
        sldm::bf16x8 hi, mid, lo;
        if (exact) sldm::split3_bf16x8(x, hi, mid, lo);
        else sldm::split_bf16x8(x, hi, mid);
#pragma unroll
        for (int t = 0; t < KT; ++t)
          if (32 * t < kd) {
            const bf8v kf = tr_frag(tk + (32 * jt + 16 * s) * RSK + 64 * t, RSK);
            if (exact) S[t] = mfma(kf, as_bf8(lo), S[t]);
            S[t] = mfma(kf, as_bf8(mid), S[t]);
            S[t] = mfma(kf, as_bf8(hi), S[t]);
          }
      }
    have_state = true;
  }
  if (R.s1) {
    float* s1 = R.s1 + sp.bh * R.s1_bh + seg * R.s1_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = 32 * t + 16 * (r >> 3) + 8 * h + (r & 7);
        if (kr < kd && vc < vd) s1[kr * R.s_k + vc * R.s_v] = S[t][r];
      }
  }
  if constexpr (OUT) {                                          // tokens behind the sequence's end: zeros
    const int64_t t1 = sp.seg0 + a.seg_len < a.T ? sp.seg0 + a.seg_len : a.T;
    const int64_t t0 = sp.len > sp.seg0 ? sp.len : sp.seg0;
    const int64_t todo = t1 > t0 ? (t1 - t0) * vd : 0;
    for (int64_t i = threadIdx.x; i < todo; i += NTH) {
      const int64_t off = sp.b * R.o_sb + (t0 + i / vd) * R.o_st + sp.hd * R.o_sh + i % vd;
      if (R.o_f32) reinterpret_cast<float*>(R.o)[off] = 0.f;
      else reinterpret_cast<uint16_t*>(R.o)[off] = 0;
    }
  }
}

template <int KT, int NW, bool OUT>
void launch(const Args& a, int roles, hipStream_t st) {
  decay_bf16_kernel<KT, NW, OUT><<<dim3((unsigned)((a.groups + 7) / 8 * 8), roles), 64 * NW, 0, st>>>(a);
}
template <int KT, bool OUT>
void by_cols(const Args& a, int nw, int roles, hipStream_t st) {
  if (nw == 1) launch<KT, 1, OUT>(a, roles, st);
  else if (nw == 2) launch<KT, 2, OUT>(a, roles, st);
  else launch<KT, 4, OUT>(a, roles, st);
}
template <bool OUT>
void by_rows(const Args& a, int roles, hipStream_t st) {
  const int kt = tiles_of(a.role[0].kd), nw = tiles_of(a.role[0].vd);
  if (kt == 1) by_cols<1, OUT>(a, nw, roles, st);
  else if (kt == 2) by_cols<2, OUT>(a, nw, roles, st);
  else by_cols<4, OUT>(a, nw, roles, st);
}

}  // namespace

void run_bf16(const Args& a, int roles, bool out, hipStream_t st) {
  out ? by_rows<true>(a, roles, st) : by_rows<false>(a, roles, st);
}

}  // namespace sldm_decay
