// Decay attention in fp32 (mathematics: decay.hpp): chunks of 16 tokens on
// v_mfma_f32_16x16x4_f32.
//
// A workgroup owns one (batch, head, segment), a wave 16 or 32 value columns and
// their slice of the state, in accumulators for the whole walk.  Tiles of SUB
// chunks of q, k and v come by LDS-DMA into two buffers, the next tile's while
// this one is computed, with one barrier a tile.  An fp32 operand is one value a
// lane and product, so rows are read 16 bytes a lane (lane = row: four
// neighbouring columns are four products' contraction slots) and columns 4 bytes
// a lane.  The chunk is as short as the matrix tile: the products inside a chunk
// cost C (Dk + Dv) a token against 2 Dk Dv between chunks, and a 16-wide head
// wastes no part of a tile.
//
// Measured (MI355X; copies reach 4.6 to 6.3 TB/s, an fp32 matrix product 153 TFLOP/s).
// 1024 sequences of one head, 2048 frames: 16-wide 109 us (4.9 TB/s) and 64-wide 471 us
// (4.6 TB/s), bound by memory; 128-wide 1.47 ms, 123 TFLOP/s of issued products, bound
// by them.  57600 heads of 16, 100 frames: forward 270 us (5.7 TB/s), backward 630 to 670
// us (4.0 TB/s of q, k, v, do, dq, dk, dv once each, which is all that moves); in the
// first ten passes after a pause 315 and up to 870 us.
#include "decay.hpp"

namespace sldm_decay {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
constexpr int C = 16;

__device__ __forceinline__ f4v mfma(float a, float b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Granule g of row r lies at g ^ swz(r): a column read's rows 4 h + r (64 bytes of
// each) fall into different quarters of the banks where a row has four, the 16
// rows of a row read into 16 places.
template <int RB>
struct Swizzle {
  static __device__ __forceinline__ int of(int r) {
    return RB == 64 ? (r >> 2) & 3 : RB == 128 ? (r & 4) | ((r >> 1) & 1) | ((r >> 2) & 2) : (r & 12) | (r & 3);
  }
};

// KT: tiles of 16 state rows; NV: of 16 value columns a wave.  OUT: outputs, else
// the state alone.  FAST: by DMA, else by Tile::slow.  PAIR: two waves have a head each,
// neighbours whose rows lie side by side, and share the tiles.
template <int KT, int NV, int NW, int SUB, bool OUT, bool FAST, bool PAIR>
__global__ __launch_bounds__(64 * NW, KT <= 2 ? 4 : 3) void decay_f32_kernel(Args a) {
  static_assert(!PAIR || (KT == 1 && NV == 1 && NW == 2 && FAST), "pairs of narrow heads");
  constexpr int HEADS = PAIR ? 2 : 1, ROWS = C * SUB, NTH = 64 * NW;
  constexpr int RBK = KT > 4 ? 512 : KT == 3 ? 256 : 64 * KT * HEADS, RBV = (NW == 3 ? 4 : NW) * 64 * NV;   // powers of two
  using TK = Tile<float, ROWS, RBK, NW, Swizzle>;
  using TV = Tile<float, ROWS, RBV, NW, Swizzle>;
  constexpr int kBuf = TK::BYTES * (OUT ? 2 : 1) + TV::BYTES;       // k, v, q
  __shared__ __attribute__((aligned(1024))) char tiles[2 * kBuf];

  const int order = xcd_order(a);
  int role = order;
  const int id = a.by_roles.split(role);
  if (id >= a.groups) return;
  const Role R = a.role[role];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), which = PAIR ? wave : 0;
  const Span sp = span_of(a, R, id, which);
  const int lane = threadIdx.x & 63, m = lane & 15, h = lane >> 4;
  const int v0 = PAIR ? 0 : 16 * NV * wave;
  const int kd = R.kd, vd = R.vd;
  const int pad = -sp.n & (ROWS - 1), nt = (sp.n + pad) / ROWS, sign = R.reverse ? -1 : 1;
  const float ld2 = sp.ld2;

  const float* qh = OUT ? head_of<float>(a, R.q, sp.b, sp.hd - which) : nullptr;
  const float* kh = head_of<float>(a, R.k, sp.b, sp.hd - which);
  const float* vh = head_of<float>(a, R.v, sp.b, sp.hd - which);

  TK tq, tk;
  TV tv;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_vptr)tiles;
  auto fetch = [&](int c, int first) {
    const uint32_t at = lds0 + (uint32_t)(c & 1) * kBuf;
    tk.load(c, at, first);
    tv.load(c, at + TK::BYTES, first);
    if constexpr (OUT) tq.load(c, at + TK::BYTES + TV::BYTES, first);
  };
  if (FAST && nt > 0) {
    if (pad > 0 || kd * HEADS * 4 < RBK || vd * HEADS * 4 < RBV) {
      for (int i = threadIdx.x; i < 2 * kBuf / 16; i += NTH) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
    tk.init(R.k, kh, sp, sign, pad, kd * HEADS);
    tv.init(R.v, vh, sp, sign, pad, vd * HEADS);
    if constexpr (OUT) tq.init(R.q, qh, sp, sign, pad, kd * HEADS);
    fetch(0, pad);
  }

  // state: lane = value column, registers = state rows 16 t + 4 h + r
  f4v S[KT][NV];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int v = 0; v < NV; ++v) S[t][v] = f4v{0.f, 0.f, 0.f, 0.f};
  const bool whole = kd == 16 * KT && vd == 16 * NV * NW / HEADS;
  if (R.s0) {
    const float* s0 = R.s0 + sp.bh * R.s0_bh + sp.seg * R.s0_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x[4];
        load_state(R, s0, v0 + 16 * v + m, whole, [&](int r) { return 16 * t + 4 * h + r; }, x);
        S[t][v] = f4v{x[0], x[1], x[2], x[3]};
      }
  }
  float d[4], w[4];                                  // D (lane = i, registers = j), the update's weights
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = 4 * h + r;
    d[r] = m >= j ? powg(ld2, m - j) * R.p_scale : 0.f;
    w[r] = powg(ld2, C - 1 - j + R.delta) * R.upd_scale;
  }
  const float rd_full = powg(ld2, m + 1 - R.delta) * R.read_scale, gn_full = powg(ld2, C);

  // where a lane finds granule h of row m, and column m of row 4 h; the swizzles are
  // XORs of bits, so other tiles and rows flip constant bits of the places
  const int row_at = m * RBK, kcol_at = 4 * h * RBK + 4 * (m & 3), vcol_at = 4 * h * RBV + 4 * (m & 3);
  int row_x = (h ^ 4 * which ^ Swizzle<RBK>::of(m)) << 4, kcol_x = (m >> 2 ^ 4 * which ^ Swizzle<RBK>::of(4 * h)) << 4;
  const int vcol_x = (m >> 2 ^ Swizzle<RBV>::of(4 * h)) << 4;
  f4v O[SUB][NV];
  float seen = 0.f;                                  // what mark() has found
  float* o_at = OUT ? reinterpret_cast<float*>(R.o) + sp.b * R.o_sb + (int64_t)(sp.base + sign * (m - pad)) * R.o_st +
                          sp.hd * R.o_sh + v0 + 4 * h
                    : nullptr;
  const int64_t o_step = (int64_t)sign * C * R.o_st;
  auto put = [&](int c) {
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      float* o = o_at;
      o_at += o_step;
      if (c * ROWS + C * s + m < pad) continue;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c0 = v0 + 16 * v + 4 * h;
        if (FAST) {
          if (c0 < vd) *reinterpret_cast<f4v*>(o + 16 * v) = O[s][v];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c0 + r < vd) o[16 * v + r] = O[s][v][r];
        }
      }
    }
  };

  for (int c = 0; c < nt; ++c) {
    if constexpr (FAST) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this tile (and older stores)
      __syncthreads();                                          // of all waves; the other buffer is free
      if (OUT && c > 0) put(c - 1);
      if (c + 1 < nt) fetch(c + 1, 0);
    } else {
      if (OUT && c > 0) put(c - 1);
      __syncthreads();
      const int x0 = c * ROWS - pad;
      char* at = tiles + (c & 1) * kBuf;
      TK::slow(at, kh + (int64_t)sp.base * R.k.st, sign * R.k.st, x0, kd);
      TV::slow(at + TK::BYTES, vh + (int64_t)sp.base * R.v.st, sign * R.v.st, x0, vd);
      if constexpr (OUT) TK::slow(at + TK::BYTES + TV::BYTES, qh + (int64_t)sp.base * R.q.st, sign * R.q.st, x0, kd);
      __syncthreads();
    }
    asm volatile("" : "+v"(row_x), "+v"(kcol_x) :: "memory");   // operands' places are worked out anew, not kept
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int empty = c == 0 ? pad - C * s : 0;               // rows in front of the segment
      if (SUB > 1 && empty >= C) continue;
      const char* lk = tiles + (c & 1) * kBuf + C * s * RBK;
      const char* lv = tiles + (c & 1) * kBuf + TK::BYTES + C * s * RBV;
      const char* lq = tiles + (c & 1) * kBuf + TK::BYTES + TV::BYTES + C * s * RBK;
      const int padc = empty > 0 ? empty : 0;
      f4v vv[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          vv[v][r] = *reinterpret_cast<const float*>(
              lv + vcol_at + r * RBV + (vcol_x ^ (64 * (NV * wave + v)) ^ (Swizzle<RBV>::of(r) << 4)));
      auto kcol = [&](int t) {
        f4v x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[r] = *reinterpret_cast<const float*>(
              lk + kcol_at + r * RBK + (kcol_x ^ (64 * t) ^ (Swizzle<RBK>::of(r) << 4)));
        return x;
      };
      if constexpr (OUT) {
        f4v P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NV; ++v) O[s][v] = f4v{0.f, 0.f, 0.f, 0.f};
        f4v qn = *reinterpret_cast<const f4v*>(lq + row_at + row_x), kn = *reinterpret_cast<const f4v*>(lk + row_at + row_x);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const f4v q = qn, k = kn;
          if (t + 1 < KT) {
            qn = *reinterpret_cast<const f4v*>(lq + row_at + (row_x ^ 64 * (t + 1)));
            kn = *reinterpret_cast<const f4v*>(lk + row_at + (row_x ^ 64 * (t + 1)));
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            P = mfma(k[r], q[r], P);
#pragma unroll
            for (int v = 0; v < NV; ++v) O[s][v] = mfma(S[t][v][r], q[r], O[s][v]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        const float rd = padc ? powg(ld2, m - padc + 1 - R.delta) * R.read_scale : rd_full;
#pragma unroll
        for (int v = 0; v < NV; ++v) O[s][v] *= rd;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int v = 0; v < NV; ++v) O[s][v] = mfma(vv[v][r], P[r] * d[r], O[s][v]);
#pragma unroll
        for (int v = 0; v < NV; ++v) mark<4>(seen, O[s][v]);
      }
      const float gn = padc ? powg(ld2, C - padc) : gn_full;
      f4v kn = kcol(0);
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) vv[v][r] *= w[r];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const f4v k = kn;
        if (t + 1 < KT) kn = kcol(t + 1);
#pragma unroll
        for (int v = 0; v < NV; ++v) S[t][v] *= gn;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int v = 0; v < NV; ++v) S[t][v] = mfma(k[r], vv[v][r], S[t][v]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (OUT && nt > 0) put(nt - 1);
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int v = 0; v < NV; ++v) mark<4>(seen, S[t][v]);
  if (!__all(seen == 0.f)) {
    const int l = lane_again();
#pragma unroll 1
    for (int v = 0; v < NV; ++v)
      walk_tokens<float, 4 * KT, 16, OUT>(a, order, which, v0 + 16 * v + (l & 15),
                                          [&](int i) { return 16 * (i >> 2) + 4 * (l >> 4) + (i & 3); });
  } else if (R.s1) {
    float* s1 = R.s1 + sp.bh * R.s1_bh + sp.seg * R.s1_seg;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const float x[4] = {S[t][v][0], S[t][v][1], S[t][v][2], S[t][v][3]};
        store_state(R, s1, v0 + 16 * v + m, whole, [&](int r) { return 16 * t + 4 * h + r; }, x);
      }
  }
  if constexpr (OUT) zero_tail<PAIR ? 64 : NTH, FAST>(a, R, sp, 4);
}

template <int KT, int NV, int NW, int SUB, bool OUT, bool FAST = true, bool PAIR = false>
void launch(const Args& a, hipStream_t st) {
  decay_f32_kernel<KT, NV, NW, SUB, OUT, FAST, PAIR>
      <<<grid_of(a), 64 * NW, 0, st>>>(a);
}
// Tiles of 32 tokens while a head is narrow, of 16 where 32 would leave a CU short
// of workgroups.
// State rows in steps of 16 and value columns of 48 and 96 of their own: 9600 x 2
// heads of 48, 100 frames, training 1740 us padded to 64, 1410 us like this; 8 heads
// over 2 of 48 and 80, 5 x 1237 frames 154 and 125 us.
template <int KT, bool OUT>
void by_cols(const Args& a, int vd, hipStream_t st) {
  constexpr int SUB = KT == 1 ? 2 : 1;
  if (vd <= 16) launch<KT, 1, 1, SUB, OUT>(a, st);
  else if (vd <= 32) launch<KT, 2, 1, SUB, OUT>(a, st);
  else if (vd <= 48) launch<KT, 1, 3, 1, OUT>(a, st);
  else if (vd <= 64) launch<KT, 2, 2, 1, OUT>(a, st);
  else if (vd <= 96) launch<KT, 2, 3, 1, OUT>(a, st);
  else launch<KT, 2, 4, 1, OUT>(a, st);
}
// Pairs of 16-wide heads make rows of 128 bytes, a cache line: half lines bound the
// backward, whose roles read them nine times (57600 heads, 100 frames: 738 us by single
// heads, whatever the tiles in flight and the order of the products; 627 by pairs).
bool pairs(const Args& a) {
  bool ok = a.H % 2 == 0;
  for (int i = 0; i < a.roles; ++i) {
    const Role& r = a.role[i];
    ok = ok && r.kd == 16 && r.vd == 16;
    for (const Operand* t : {&r.q, &r.k, &r.v}) ok = ok && !t->shared && t->sh == 16;
  }
  return ok;
}
template <bool OUT>
void run(const Args& a, hipStream_t st) {
  int kd = 0, vd = 0;
  for (int i = 0; i < a.roles; ++i) {
    kd = a.role[i].kd > kd ? a.role[i].kd : kd;
    vd = a.role[i].vd > vd ? a.role[i].vd : vd;
  }
  if (!all_fast(a, OUT, 4)) {
    launch<8, 2, 4, 1, OUT, false>(a, st);
  } else if (pairs(a)) {
    Args two = a;
    two.hpw = 2;
    two.groups = a.groups / 2;
    two.unit = a.roles * (a.H % 4 ? 1 : 2);
    two.by_unit = Div(two.unit);
    two.by_all = Div(a.B * a.H / 2);
    two.by_h = Div(a.H / 2);
    launch<1, 1, 2, 2, OUT, true, true>(two, st);
  }
  else if (kd <= 16) by_cols<1, OUT>(a, vd, st);
  else if (kd <= 32) by_cols<2, OUT>(a, vd, st);
  else if (kd <= 48) by_cols<3, OUT>(a, vd, st);
  else if (kd <= 64) by_cols<4, OUT>(a, vd, st);
  else if (kd <= 80) by_cols<5, OUT>(a, vd, st);
  else if (kd <= 96) by_cols<6, OUT>(a, vd, st);
  else by_cols<8, OUT>(a, vd, st);
}

}  // namespace

void run_f32(const Args& a, bool out, hipStream_t st) { out ? run<true>(a, st) : run<false>(a, st); }

}  // namespace sldm_decay
