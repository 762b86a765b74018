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
// A product q_i k_j inside a chunk that is smaller than its type's smallest number is
// lost (bf16 and fp32: steps of 2^-133 and 2^-149), whatever v_j it meets.
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
// A sequence is aligned to the END of its chunks: the first chunk is padded with
// zero rows in front, which leaves every decay table a constant.  The matrix
// accumulator layout (lane = column, registers = rows) is at once an operand
// layout (rows = lane, contraction = register), so the state feeds Q S, and
// P = Q K^T o D, computed transposed, feeds P V, without leaving registers; the
// output comes out transposed too, lane = token, registers = neighbouring
// columns, which are 16-byte stores.  Kernels: decay_f32.hip, decay_bf16.hip.
#pragma once

#include "common.hpp"

namespace sldm_decay {

// Division of 0 <= n < 2^31 by a divisor that the launch knows: the upper half of a
// product, in scalar registers, instead of some thirty instructions.  With 2^s the
// power of two from d on, n / d = (n + (n m >> 32)) >> s for m = floor(2^32 (2^s - d) / d) + 1.
struct Div {
  uint32_t d, m;
  int s;
  Div() = default;
  explicit Div(int64_t by) : d((uint32_t)by), s(0) {
    while (((int64_t)1 << s) < by) ++s;
    m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - by)) / by + 1);
  }
  __device__ __forceinline__ int quotient(int n) const { return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s); }
  // n becomes the remainder
  __device__ __forceinline__ int split(int& n) const {
    const int q = quotient(n);
    n -= q * (int)d;
    return q;
  }
};

struct Operand {
  const void* p;
  int64_t sb, st, sh;   // element strides of batch, token, head; columns are contiguous
  int shared;           // head h reads head h / group
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
  int s_k, s_v;
  float read_scale, p_scale, upd_scale;
  int delta, reverse;
  int kd, vd;
};

struct Args {
  Role role[3];
  int64_t B, H, T, seg_len;
  int nseg, groups;     // groups = B H nseg / hpw
  int hpw;              // heads a workgroup has
  int roles, unit;      // unit: workgroups that stay together on an XCD
  int group;            // heads that share a key head
  Div by_unit, by_roles, by_all, by_h, by_group;   // by_all, by_h: B H / hpw, H / hpw
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

// Workgroups are dealt to the XCDs in turn.  Units of neighbours in (segment,
// batch, head, role) order stay on one XCD: the roles of a head read the same
// tensors, and narrow heads share cache lines.  The units themselves go round the
// XCDs, one place further each time, so that batches of uneven lengths do not
// load some XCDs alone (ragged prompts: whole ranges of units an XCD 105 us).
__device__ __forceinline__ int xcd_order(const Args& a) {
  int slot = (int)blockIdx.x >> 3;
  const int turn = a.by_unit.split(slot);
  return (turn * 8 + (((int)blockIdx.x + turn) & 7)) * a.unit + slot;
}

// What a (batch, head, segment) is made of.  All uniform, and said so: what comes
// from a vector load would otherwise live in vector registers.
struct Span {
  int64_t bh, b;
  int hd, len, seg, seg0, n, base;   // n: the segment's tokens; base: position x is token base +- x
  float ld2;                    // log2 of the decay
};
// which: of the workgroup's heads.
__device__ __forceinline__ Span span_of(const Args& a, const Role& R, int id, int which = 0) {
  Span s;
  s.seg = a.by_all.split(id);
  s.b = a.by_h.split(id);
  s.hd = id * a.hpw + which;
  s.bh = s.b * a.H + s.hd;
  s.len = __builtin_amdgcn_readfirstlane((int)seq_len(a, s.b));
  s.seg0 = s.seg * (int)a.seg_len;
  const int left = s.len - s.seg0, whole = (int)a.seg_len;
  s.n = left < 0 ? 0 : (left < whole ? left : whole);
  s.base = R.reverse ? s.len - 1 - s.seg0 : s.seg0;
  s.ld2 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(a.log_decay[s.hd]))) * 1.44269504088896340736f;
  return s;
}

template <typename T>
__device__ __forceinline__ const T* head_of(const Args& a, const Operand& t, int64_t b, int hd) {
  return reinterpret_cast<const T*>(t.p) + b * t.sb + (t.shared ? a.by_group.quotient(hd) : hd) * t.sh;
}

// The walk's state in memory: element (row, column) of a kd x vd state lies at
// row s_k + column s_v.  N registers a lane, register i at row row_of(i); elements
// outside the state are zeros.
template <int N, typename RowOf>
__device__ __forceinline__ void load_state(const Role& R, const float* s0, int col, bool whole, RowOf row_of, float (&v)[N]) {
  if (whole) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = s0[row_of(i) * R.s_k + col * R.s_v];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row_of(i);
      v[i] = 0.f;
      if (r < R.kd && col < R.vd) v[i] = s0[r * R.s_k + col * R.s_v];
    }
  }
}
template <int N, typename RowOf>
__device__ __forceinline__ void store_state(const Role& R, float* s1, int col, bool whole, RowOf row_of, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = row_of(i);
    if (whole || (r < R.kd && col < R.vd)) s1[r * R.s_k + col * R.s_v] = v[i];
  }
}

typedef __attribute__((address_space(3))) void* lds_vptr;

// A tile of ROWS rows of RB bytes in LDS, by LDS-DMA: 64 granules of 16 bytes an
// instruction, instruction i of the tile by wave i % NW; granule g of row r lies
// at g ^ SWZ<RB>::of(r), by choice of the source address.  Lanes without a source
// (columns past d, rows in front of the segment) stay out and leave their place
// as it is: zeros, written once.
template <typename T, int ROWS, int RB, int NW, template <int> class SWZ>
struct Tile {
  static constexpr int kRB = RB, GR = RB / 16, BYTES = ROWS * RB, INSTR = BYTES / 1024, E = 16 / (int)sizeof(T);
  static constexpr int N = (INSTR + NW - 1) / NW, STEP = 64 / GR;
  static_assert(BYTES % 1024 == 0 && GR <= 64, "whole instructions");
  const char* base;        // of the lowest-addressed row of chunk 0
  int64_t step;            // bytes from chunk to chunk
  uint32_t voff[N];
  uint32_t on;             // bit i: this lane takes part in instruction i
  static __device__ __forceinline__ int row_of(int i) {
    return (i * NW + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * STEP + (int)(threadIdx.x & 63) / GR;
  }
  __device__ __forceinline__ void init(const Operand& t, const T* head, const Span& s, int sign, int pad, int d) {
    const int64_t st = t.st;
    base = reinterpret_cast<const char*>(head + (int64_t)(s.base - sign * pad + (sign < 0 ? -(ROWS - 1) : 0)) * st);
    step = (int64_t)sign * ROWS * st * (int)sizeof(T);
    on = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row_of(i), g = (int)(threadIdx.x & 63) % GR ^ SWZ<RB>::of(r);
      voff[i] = (uint32_t)((sign < 0 ? ROWS - 1 - r : r) * st * (int)sizeof(T)) + 16 * g;
      on |= (r < ROWS && E * g < d ? 1u : 0u) << i;
    }
  }
  // chunk c, rows from `first` on, to LDS address `lds`
  __device__ __forceinline__ void load(int c, uint32_t lds, int first) const {
    const char* p = base + c * step;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((on >> i & 1) && row_of(i) >= first)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :: "v"(voff[i]), "s"(p), "s"(__builtin_amdgcn_readfirstlane(lds + (uint32_t)((i * NW + wave) * 1024)))
                     : "memory", "m0");
  }
  // any alignment: element by element; row r is position x0 + r (below 0: zeros)
  static __device__ __forceinline__ void slow(char* lds, const T* row0, int64_t st, int x0, int d) {
    constexpr int W = RB / (int)sizeof(T);
#pragma unroll 1
    for (int i = threadIdx.x; i < ROWS * W; i += 64 * NW) {
      const int r = i / W, e = i % W;
      const int x = x0 + r;
      *reinterpret_cast<T*>(lds + r * RB + ((e / E ^ SWZ<RB>::of(r)) << 4) + (int)sizeof(T) * (e % E)) =
          x >= 0 && e < d ? row0[x * st + e] : T(0);
    }
  }
};

// Tokens behind the sequence's end (of this segment's range): zeros, 16 bytes a
// thread where the rows allow it, by NTH threads (64: each wave for its own head).
template <int NTH, bool FAST>
__device__ __forceinline__ void zero_tail(const Args& a, const Role& R, const Span& s, int elem_bytes) {
  const int T = (int)a.T, whole = (int)a.seg_len, t1 = T - s.seg0 > whole ? s.seg0 + whole : T;
  const int t0 = s.len > s.seg0 ? s.len : s.seg0;
  if (t0 >= t1) return;
  constexpr int kLanes = 32;                     // across a row (of at most 512 bytes: 32 granules)
  const int col = (int)threadIdx.x % kLanes, row0 = (int)threadIdx.x % NTH / kLanes, bytes = R.vd * elem_bytes;
  char* o = reinterpret_cast<char*>(R.o) + (s.b * R.o_sb + s.hd * R.o_sh) * elem_bytes;
  for (int t = t0 + row0; t < t1; t += NTH / kLanes) {
    char* row = o + (int64_t)t * R.o_st * elem_bytes;
    if (FAST) {
      if (16 * col < bytes) *reinterpret_cast<uint4*>(row + 16 * col) = make_uint4(0, 0, 0, 0);
    } else {
      for (int i = 2 * col; i < bytes; i += 2 * kLanes) *reinterpret_cast<uint16_t*>(row + i) = 0;
    }
  }
}

// A chunk's products mix its tokens, and a state's parts.  An infinity or NaN in a
// token's v would reach the outputs of the tokens in front of it in the same chunk (as
// 0 times itself, in the masked half of P V), in k likewise; an infinity in q would
// meet those zeros too, where operands go in as sums of terms one would become a NaN
// (as the difference of two), and q k may leave fp32's range where q S does not.  All
// of that leaves a mark in an output, or in the state, where it lasts to the end of
// the walk; a wave that has seen one writes its columns' outputs and state anew by the
// recurrence itself, token by token.  SPREAD: lanes col + SPREAD, .. of the wave hold
// the other rows of a column.  Looking costs 1 % (57600 heads of 16, 100 frames, training: 907
// -> 918 us); a walk about 5 us a token and wave (1024 heads of 64, 2048 frames, a NaN in
// each: 9.9 ms).
// seen: 0 while all are finite (and their sum is), NaN from then on.  N: a power of two.
template <int N, typename V>
__device__ __forceinline__ void mark(float& seen, const V& v) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
#pragma unroll
  for (int n = N / 2; n; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) x[i] += x[i + n];
  seen = __builtin_fmaf(x[0], 0.f, seen);
}
// the lane's number, not kept in a register from the kernel's start
__device__ __forceinline__ int lane_again() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t & 63;
}
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(uint16_t v) { return sldm::bf16_to_f32(v); }
template <typename T, int N, int SPREAD, bool OUT, typename RowOf>
__device__ __forceinline__ void walk_tokens(const Args& a, int order, int which, int col, RowOf row_of) {
  asm volatile("" : "+s"(order));                // the role is read anew, not kept over the walk before
  const int id = a.by_roles.split(order);
  const Role R = a.role[order];
  const Span s = span_of(a, R, id, which);
  float S[N];
#pragma unroll
  for (int i = 0; i < N; ++i) S[i] = 0.f;
  if (R.s0) load_state(R, R.s0 + s.bh * R.s0_bh + s.seg * R.s0_seg, col, false, row_of, S);
  const T* q = OUT ? head_of<T>(a, R.q, s.b, s.hd) : nullptr;
  const T* k = head_of<T>(a, R.k, s.b, s.hd);
  const T* v = head_of<T>(a, R.v, s.b, s.hd);
  const float g = exp2f(s.ld2), before = R.delta ? 1.f : g, after = R.delta ? g : 1.f;
  // the chunks' outputs of this wave are in memory before these are
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll 1
  for (int x = 0; x < s.n; ++x) {
    const int64_t t = s.base + (R.reverse ? -x : x);
    const float vv = col < R.vd ? widen(v[t * R.v.st + col]) * R.upd_scale : 0.f;
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row_of(i);
      if (r < R.kd) {
        S[i] = S[i] * before + widen(k[t * R.k.st + r]) * vv;
        if (OUT) o += widen(q[t * R.q.st + r]) * S[i];
        S[i] *= after;
      }
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if (!OUT) continue;
#pragma unroll
    for (int d = SPREAD; d < 64; d <<= 1) o += __shfl_xor(o, d);
    o *= R.read_scale;
    if (col < R.vd && (int)(threadIdx.x & 63) < SPREAD) {
      const int64_t at = s.b * R.o_sb + t * R.o_st + s.hd * R.o_sh + col;
      if (sizeof(T) == 4 || R.o_f32) reinterpret_cast<float*>(R.o)[at] = o;
      else reinterpret_cast<uint16_t*>(R.o)[at] = sldm::f32_to_bf16(o);
    }
  }
  if (R.s1) store_state(R, R.s1 + s.bh * R.s1_bh + s.seg * R.s1_seg, col, false, row_of, S);
}

// Rows of a chunk within 32-bit byte offsets of each other.
inline bool near(const Operand& t) { return t.st >= 0 && t.st < ((int64_t)1 << 24); }
// Whether every operand can come by DMA: rows on 16-byte boundaries, whole granules.
inline bool all_fast(const Args& a, bool out, int granule) {
  bool ok = true;
  for (int i = 0; i < a.roles; ++i) {
    const Role& r = a.role[i];
    ok = ok && r.k.vec && r.v.vec && r.kd % granule == 0 && r.vd % granule == 0 && near(r.k) && near(r.v) &&
         (!out || (r.q.vec && r.o_vec && near(r.q)));
  }
  return ok;
}

// One launch of roles whose kd and vd fall into the same tile classes.
// out: roles write outputs; else states only.
void run_bf16(const Args& a, bool out, hipStream_t stream);
void run_f32(const Args& a, bool out, hipStream_t stream);
inline unsigned grid_of(const Args& a) {
  const int64_t n = (int64_t)a.groups * a.roles, u = 8 * a.unit;
  return (unsigned)((n + u - 1) / u * u);
}
inline int tiles_of(int d) { return d <= 32 ? 1 : d <= 64 ? 2 : 4; }   // waves across vd
inline int row_tiles(int d) { return (d + 31) / 32; }

}  // namespace sldm_decay
