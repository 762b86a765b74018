// Decay attention in bf16 (mathematics: decay.hpp), kernel: chunks of 32 tokens on
// v_mfma_f32_32x32x16_bf16, fp32 accumulation.
//
// A workgroup owns one (batch, head, segment); a wave owns 32 value columns and
// keeps its Dk x 32 slice of the state in accumulators for the whole walk.  Q, K
// and V tiles come by LDS-DMA (no registers on the way) into two buffers, the
// next chunk's while this one is computed, with one barrier a chunk; an output
// chunk is stored behind the next barrier, so that its stores have a chunk's time
// before anything waits for memory.  The 16-byte granules of a row are
// XOR-swizzled through the DMA's source addresses, so that row reads (one granule
// of eight rows) and transposed reads (ds_read_b64_tr_b16: 64 bytes of four rows)
// spread over the banks.  Chunks of 64 (half as many state conversions) were
// slower: their tiles and accumulators leave two waves a SIMD and spill.
//
// Measured (MI355X; copies reach 4.6 to 6.3 TB/s).  1024 sequences of one head, 2048
// frames: 64-wide 226 us (4.7 TB/s), bound by memory; 128-wide 552 us (3.9 TB/s) by
// VALU and MFMA issue; 16-wide 84 us (3.2 TB/s) and few long heads by the chain of a
// chunk (about 1 us from its first read to its state).  8 heads of 128, 32768 frames:
// forward 43 us for the segments' states, 15 for the scan, 78 to 85 for the outputs,
// backward 43, 15 and 213 to 222 (MFMA 45 %, VALU 64 % of the time busy).
//
// Roundings.  The state is held in fp32 accumulators.  What the matrix instructions
// take from fp32 goes in as sums of bf16 terms: the state that is read, and P = Q K^T
// o D, as hi + lo (16 significant bits, so the products of an output are each off by
// at most 2^-16 of themselves, far below what rounding the output to bf16 costs), and
// V g^{n-1-j}, which enters the state, as hi + mid + lo (all 24).  One term for the
// state or for P would be as large an error as the output's own rounding (relative
// error 0.0024 instead of 0.0017), and more where the products cancel.  What the second
// terms cost: 32768 frames, 8 heads of 128, training 316 -> 391 us with the third term
// into the state (345 with two), 64-wide heads nothing that shows.
#pragma once

#include "decay.hpp"

namespace sldm_decay {
namespace {

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int C = 32;

__device__ __forceinline__ f16v mfma(bf8v a, bf8v b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf8v as_bf8(sldm::bf16x8 v) { return __builtin_bit_cast(bf8v, v); }

// LDS rows of 32 DT values (96 take the room of 128); swizzle: granule g of row r
// lies at g ^ swz(r).  Four neighbouring rows' transposed reads (64 bytes of
// each) fall into the four quarters of the banks, eight rows' granules into eight
// places.
constexpr int row_bytes(int dt) { return dt == 1 ? 64 : dt == 2 ? 128 : 256; }
template <int RB>
struct Swizzle {
  static __device__ __forceinline__ int of(int r) {
    const int low = ((r >> 2) & 1) | ((r >> 2) & 2);
    return RB == 64 ? low : RB == 128 ? ((r & 2) << 1) | low : ((r & 3) << 2) | low;
  }
};

// lane -> column (or row) inside a 32-wide tile: the middle two bits of each
// 16-group swapped, which makes the accumulator rows 8 s .. 8 s + 7 of a half
// wave eight neighbours: 16 s + 8 h + e.
__device__ __forceinline__ int perm16(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// Operand whose rows are a tile's rows: lane `row`, columns 16 t + 8 h .. + 7.
struct RowRead {
  uint32_t base, x;
  template <int RB>
  __device__ __forceinline__ void init(int row, int h) {
    base = row * RB;
    x = (h ^ Swizzle<RB>::of(row)) << 4;
  }
  __device__ __forceinline__ bf8v at(const char* lds, int t) const {
    return *reinterpret_cast<const bf8v*>(lds + base + (x ^ (32 * t)));
  }
};
// Operand whose rows are a tile's columns: lane m holds column 32 ct + perm16(m)
// of the eight rows 16 s + 8 h ..
struct ColRead {
  uint32_t base, x;
  template <int RB>
  __device__ __forceinline__ void init(int lane) {
    const int q = lane >> 4, r16 = lane & 15, blk = r16 & 3, b = ((blk & 1) << 1) | (blk >> 1);
    const int row = 8 * (q >> 1) + (r16 >> 2);
    base = row * RB + 8 * (b & 1);
    x = ((2 * (q & 1) + (b >> 1)) ^ Swizzle<RB>::of(row)) << 4;
  }
  template <int RB>
  __device__ __forceinline__ bf8v at(const char* lds, int ct, int s) const {
    typedef __attribute__((address_space(3))) s4v* lp;
    const char* p = lds + base + 16 * s * RB;      // rows + 4: bit 0 of the swizzle flips
    const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + (x ^ (64 * ct))));
    const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * RB + (x ^ (64 * ct) ^ 16)));
    return __builtin_bit_cast(bf8v, s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
};

// Instructions stay on their side: scheduled over a whole chunk, the operands of
// all products are in registers at once and spill.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// The state's update: S <- g^n S + K^T diag(w) V, V diag(w) in three parts.
template <int KT>
__device__ __forceinline__ void update(f16v (&S)[KT], const bf8v (&vf)[2], const char* lk, const ColRead& ck,
                                       const float* pw, float gn) {
  bf8v kf[2][KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) kf[0][t] = ck.at<row_bytes(KT)>(lk, t, 0);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float* w = pw + 16 * s;
    const uint4 u = __builtin_bit_cast(uint4, vf[s]);
    const float x[8] = {sldm::bf16_lo(u.x) * w[0], sldm::bf16_hi(u.x) * w[1], sldm::bf16_lo(u.y) * w[2],
                        sldm::bf16_hi(u.y) * w[3], sldm::bf16_lo(u.z) * w[4], sldm::bf16_hi(u.z) * w[5],
                        sldm::bf16_lo(u.w) * w[6], sldm::bf16_hi(u.w) * w[7]};
    sldm::bf16x8 hi, mid, lo;
    sldm::split3_bf16x8(x, hi, mid, lo);
    phase();
    if (s == 0)
#pragma unroll
      for (int t = 0; t < KT; ++t) kf[1][t] = ck.at<row_bytes(KT)>(lk, t, 1);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (s == 0)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] *= gn;
      S[t] = mfma(kf[s][t], as_bf8(lo), S[t]);
      S[t] = mfma(kf[s][t], as_bf8(mid), S[t]);
      S[t] = mfma(kf[s][t], as_bf8(hi), S[t]);
    }
    phase();
  }
}

// LDS of a workgroup's tiles, and the waves a SIMD that leaves (up to 4, and 3
// where the state alone takes 64 registers).
template <int KT, int NW, bool OUT>
constexpr int tile_bytes() { return 2 * C * (row_bytes(KT) * (OUT ? 2 : 1) + row_bytes(NW)); }
constexpr int waves_for(int lds, int kt, int nw) {
  const int w = (160 * 1024 / (lds + 512)) * nw / 4, most = kt == 4 ? 3 : 4;
  return w < 1 ? 1 : w > most ? most : w;
}

// OUT: outputs, else the state alone.  FAST: by DMA, else by Tile::slow.
template <int KT, int NW, bool OUT, bool FAST>
__global__ __launch_bounds__(64 * NW, waves_for(tile_bytes<KT, NW, OUT>(), KT, NW)) void decay_bf16_kernel(Args a) {
  using TK = Tile<uint16_t, C, row_bytes(KT), NW, Swizzle>;
  using TV = Tile<uint16_t, C, row_bytes(NW), NW, Swizzle>;
  constexpr int NTH = 64 * NW, RBK = TK::kRB, RBV = TV::kRB;
  constexpr int kBuf = TK::BYTES * (OUT ? 2 : 1) + TV::BYTES;       // k, v, q
  __shared__ __attribute__((aligned(1024))) char tiles[2 * kBuf];
  __shared__ __attribute__((aligned(16))) float wtab[C], dtab[2 * C];

  const int order = xcd_order(a);
  int role = order;
  const int id = a.by_roles.split(role);
  if (id >= a.groups) return;
  const Role R = a.role[role];
  const Span sp = span_of(a, R, id);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 31, h = lane >> 5;
  const int kd = R.kd, vd = R.vd;
  const int pad = -sp.n & (C - 1), nch = (sp.n + pad) / C, sign = R.reverse ? -1 : 1;
  const float ld2 = sp.ld2;

  const uint16_t* qh = OUT ? head_of<uint16_t>(a, R.q, sp.b, sp.hd) : nullptr;
  const uint16_t* kh = head_of<uint16_t>(a, R.k, sp.b, sp.hd);
  const uint16_t* vh = head_of<uint16_t>(a, R.v, sp.b, sp.hd);

  TK tq, tk;
  TV tv;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_vptr)tiles;
  auto fetch = [&](int c, int first) {
    const uint32_t at = lds0 + (uint32_t)(c & 1) * kBuf;
    tk.load(c, at, first);
    tv.load(c, at + TK::BYTES, first);
    if constexpr (OUT) tq.load(c, at + TK::BYTES + TV::BYTES, first);
  };
  if (FAST && nch > 0) {
    if (pad > 0 || kd < 32 * KT || vd < 32 * NW) {
      for (int i = threadIdx.x; i < 2 * kBuf / 16; i += NTH) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
    tk.init(R.k, kh, sp, sign, pad, kd);
    tv.init(R.v, vh, sp, sign, pad, vd);
    if constexpr (OUT) tq.init(R.q, qh, sp, sign, pad, kd);
    fetch(0, pad);
  }
  // state: lane = value column, register 8 s + e of tile t = row 32 t + 16 s + 8 h + e
  const int vc = 32 * wave + perm16(m);
  f16v S[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[t][r] = 0.f;
  const bool whole = kd == 32 * KT && vd == 32 * NW;
  if (R.s0) {
    const float* s0 = R.s0 + sp.bh * R.s0_bh + sp.seg * R.s0_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      float x[16];
      load_state(R, s0, vc, whole, [&](int r) { return 32 * t + 16 * (r >> 3) + 8 * h + (r & 7); }, x);
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] = x[r];
    }
  }
  // wtab[j]: the weight with which row j enters the state; dtab[32 + i - j]: D
  for (int j = threadIdx.x; j < C; j += NTH) wtab[j] = powg(ld2, C - 1 - j + R.delta) * R.upd_scale;
  for (int j = threadIdx.x; j < 2 * C; j += NTH) dtab[j] = j < C ? 0.f : powg(ld2, j - C) * R.p_scale;

  RowRead rq, rk;
  ColRead ck, cv;
  rq.init<RBK>(m, h);
  rk.init<RBK>(perm16(m), h);
  ck.init<RBK>(lane);
  cv.init<RBV>(lane);
  const float* pd = dtab + 9 + m - 8 * h;                       // + 23 - (16 s + e): entry 32 + m - j
  const float* pw = wtab + 8 * h;
  f16v O;
  float seen = 0.f;                                             // what mark() has found
  // chunk c's outputs: lane = token m, registers 8 s + e = columns 16 s + 8 h + e
  const int o_bytes = R.o_f32 ? 4 : 2;
  char* o_at = OUT ? reinterpret_cast<char*>(R.o) + (sp.b * R.o_sb + (int64_t)(sp.base + sign * (m - pad)) * R.o_st +
                                                     sp.hd * R.o_sh + 32 * wave + 8 * h) * o_bytes
                   : nullptr;
  const int64_t o_step = (int64_t)sign * C * R.o_st * o_bytes;
  auto put = [&](int c) {
    char* at = o_at;
    o_at += o_step;
    if (c * C + m < pad) return;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int c0 = 32 * wave + 16 * s + 8 * h;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = O[8 * s + e];
      if (o_bytes == 4) {
        float* o = reinterpret_cast<float*>(at) + 16 * s;
        if (FAST) {
          if (c0 < vd) {
            sldm::Vec<float, 4>::store(o, y);
            sldm::Vec<float, 4>::store(o + 4, y + 4);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + e < vd) o[e] = y[e];
        }
      } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(at) + 16 * s;
        if (FAST) {
          if (c0 < vd) sldm::Vec<uint16_t, 8>::store(o, y);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + e < vd) o[e] = sldm::f32_to_bf16(y[e]);
        }
      }
    }
  };
  // the first chunk's padding shortens what lies between the state and its rows
  const float rd_full = powg(ld2, m + 1 - R.delta) * R.read_scale, gn_full = powg(ld2, C);
  float rd = powg(ld2, m - pad + 1 - R.delta) * R.read_scale, gn = powg(ld2, C - pad);

  for (int c = 0; c < nch; ++c) {
    if constexpr (FAST) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this chunk's tiles (and older stores)
      __syncthreads();                                          // of all waves; the other buffer is free
      if (OUT && c > 0) put(c - 1);
      if (c + 1 < nch) fetch(c + 1, 0);
    } else {
      if (OUT && c > 0) put(c - 1);
      __syncthreads();
      const int x0 = c * C - pad;
      char* at = tiles + (c & 1) * kBuf;
      TK::slow(at, kh + (int64_t)sp.base * R.k.st, sign * R.k.st, x0, kd);
      TV::slow(at + TK::BYTES, vh + (int64_t)sp.base * R.v.st, sign * R.v.st, x0, vd);
      if constexpr (OUT) TK::slow(at + TK::BYTES + TV::BYTES, qh + (int64_t)sp.base * R.q.st, sign * R.q.st, x0, kd);
      __syncthreads();
    }
    // the tables are read, and the operands' places worked out, anew: not kept in registers
    asm volatile("" : "+v"(rq.x), "+v"(rk.x), "+v"(ck.x), "+v"(cv.x) :: "memory");
    const char* lk = tiles + (c & 1) * kBuf;
    const char* lv = lk + TK::BYTES;
    const char* lq = lv + TV::BYTES;
    bf8v vf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) vf[s] = cv.at<RBV>(lv, wave, s);
    if constexpr (OUT) {
      f16v P;
#pragma unroll
      for (int r = 0; r < 16; ++r) O[r] = P[r] = 0.f;
      constexpr int A = 2 * KT < 3 ? 2 * KT : 3;                // operands in flight
      bf8v qn[A], kn[A];
#pragma unroll
      for (int t = 0; t < A; ++t) {
        qn[t] = rq.at(lq, t);
        kn[t] = rk.at(lk, t);
      }
#pragma unroll
      for (int t = 0; t < 2 * KT; ++t) {
        const bf8v qf = qn[t % A], kf = kn[t % A];
        if (t + A < 2 * KT) {
          qn[t % A] = rq.at(lq, t + A);
          kn[t % A] = rk.at(lk, t + A);
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = S[t >> 1][8 * (t & 1) + e];
        sldm::bf16x8 hi, lo;
        sldm::split_bf16x8(x, hi, lo);
        O = mfma(as_bf8(lo), qf, O);
        P = mfma(kf, qf, P);
        O = mfma(as_bf8(hi), qf, O);
        phase();
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) O[r] *= rd;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = P[8 * s + e] * pd[23 - 16 * s - e];
        sldm::bf16x8 hi, lo;
        sldm::split_bf16x8(x, hi, lo);
        O = mfma(vf[s], as_bf8(lo), O);
        O = mfma(vf[s], as_bf8(hi), O);
      }
      mark<16>(seen, O);
    }
    update<KT>(S, vf, lk, ck, pw, gn);
    rd = rd_full;
    gn = gn_full;
  }
  if (OUT && nch > 0) put(nch - 1);
#pragma unroll
  for (int t = 0; t < KT; ++t) mark<16>(seen, S[t]);
  if (!__all(seen == 0.f)) {
    const int l = lane_again();
    walk_tokens<uint16_t, 16 * KT, 32, OUT>(a, order, 0, 32 * wave + perm16(l & 31),
                                            [&](int i) { return 16 * (i >> 3) + 8 * (l >> 5) + (i & 7); });
  } else if (R.s1) {
    float* s1 = R.s1 + sp.bh * R.s1_bh + sp.seg * R.s1_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = S[t][r];
      store_state(R, s1, vc, whole, [&](int r) { return 32 * t + 16 * (r >> 3) + 8 * h + (r & 7); }, x);
    }
  }
  if constexpr (OUT) zero_tail<NTH, FAST>(a, R, sp, R.o_f32 ? 4 : 2);
}

template <int KT, int NW, bool OUT, bool FAST = true>
void launch(const Args& a, hipStream_t st) {
  decay_bf16_kernel<KT, NW, OUT, FAST>
      <<<grid_of(a), 64 * NW, 0, st>>>(a);
}
template <int KT, bool OUT>
void by_cols(const Args& a, int nw, hipStream_t st) {
  if (nw == 1) launch<KT, 1, OUT>(a, st);
  else if (nw == 2) launch<KT, 2, OUT>(a, st);
  else launch<KT, 4, OUT>(a, st);
}
template <bool OUT>
void by_rows(const Args& a, hipStream_t st) {
  const int kt = row_tiles(a.role[0].kd), nw = tiles_of(a.role[0].vd);
  if (kt == 1) by_cols<1, OUT>(a, nw, st);
  else if (kt == 2) by_cols<2, OUT>(a, nw, st);
  else if (kt == 3) by_cols<3, OUT>(a, nw, st);
  else by_cols<4, OUT>(a, nw, st);
}
}  // namespace
}  // namespace sldm_decay
