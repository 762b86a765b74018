// Rotary positions over several axes.
//
// Pair p of a head belongs to axis a(p) (sections[0] pairs to axis 0, the next
// sections[1] to axis 1, ...) and is turned by angle = pos[token, a(p)] f[p]:
//   (u, v) -> (u cos - v sin, u sin + v cos)
// The gradient is the turn by -angle, so one kernel serves both.  Bound by
// memory: q and k in and out once.  A workgroup takes some tokens, computes
// their angles once for all heads of q and k into LDS, and then turns rows 16
// bytes a lane.  Angles are products in 64 bits, reduced to [-pi, pi] there
// (positions of 10^6 times a frequency of 1 leave fp32 an error of 0.06), and
// only then rounded for the fp32 sine and cosine.
//
// Measured (MI355X, copies at 4.6 to 6.3 TB/s): 960 000 tokens x 12 heads of 16, fp32,
// 291 us (5.1 TB/s); 32768 tokens x 20 heads of 128, bf16, 67 us (5.0 TB/s); 300
// tokens x 12 heads of 16, bf16, 4.7 us.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kBlock = 256;
constexpr int kMaxAxes = 8;
constexpr int kMaxDim = 1024;
constexpr int kMaxBlock = 64;   // tokens of a workgroup

typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4a4 __attribute__((ext_vector_type(4), aligned(4)));

template <typename T, int V>
__device__ __forceinline__ void load_any(const T* p, float (&r)[V]) {
  if constexpr (sizeof(T) * V == 16) {
    uint4 w;
    if constexpr (sizeof(T) == 2) w = __builtin_bit_cast(uint4, *reinterpret_cast<const u4a2*>(p));
    else w = __builtin_bit_cast(uint4, *reinterpret_cast<const u4a4*>(p));
    sldm::Vec<T, V>::load(reinterpret_cast<const T*>(&w), r);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float one[1];
      sldm::Vec<T, 1>::load(p + e, one);
      r[e] = one[0];
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_any(T* p, const float (&r)[V]) {
  if constexpr (sizeof(T) * V == 16) {
    uint4 w;
    sldm::Vec<T, V>::store(reinterpret_cast<T*>(&w), r);
    if constexpr (sizeof(T) == 2) *reinterpret_cast<u4a2*>(p) = __builtin_bit_cast(u4a2, w);
    else *reinterpret_cast<u4a4*>(p) = __builtin_bit_cast(u4a4, w);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) sldm::Vec<T, 1>::store(p + e, &r[e]);
  }
}

struct RotArgs {
  const void *q, *k;
  void *oq, *ok;                 // contiguous [B, T, H, D]
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
  int64_t B, T;
  int hq, hk, dim, pairs, axes;
  int end[kMaxAxes];             // pairs before the end of each axis
  const void* pos;
  int64_t pos_sb, pos_st, pos_sa;
  int pos_type;
  const double* freq;
  float sign;
  int block;                     // tokens a workgroup takes
};

__device__ __forceinline__ double position(const RotArgs& a, int64_t off) {
  switch (a.pos_type) {
    case SLDM_POS_I32: return (double)reinterpret_cast<const int32_t*>(a.pos)[off];
    case SLDM_POS_I64: return (double)reinterpret_cast<const int64_t*>(a.pos)[off];
    case SLDM_POS_F32: return (double)reinterpret_cast<const float*>(a.pos)[off];
    default: return reinterpret_cast<const double*>(a.pos)[off];
  }
}

// MIX: a pair is (2p, 2p + 1), else (p, p + pairs).  V elements a lane.
template <typename T, int V, bool MIX>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotArgs a) {
  extern __shared__ float2 turn[];               // [tokens][pairs]: cos, sin
  __shared__ int64_t q_at[kMaxBlock], k_at[kMaxBlock];   // where the tokens' rows start
  const int64_t n0 = (int64_t)blockIdx.x * a.block;
  const int64_t all = a.B * a.T;
  const int here = (int)(all - n0 < a.block ? all - n0 : a.block);
  for (int i = threadIdx.x; i < here * a.pairs; i += kBlock) {
    const int64_t n = n0 + i / a.pairs;
    const int p = i % a.pairs;
    int ax = 0;
    while (ax + 1 < a.axes && p >= a.end[ax]) ++ax;
    const double x = position(a, (n / a.T) * a.pos_sb + (n % a.T) * a.pos_st + ax * a.pos_sa) * a.freq[p];
    const double turns = rint(x * 0.15915494309189533577);
    double r = fma(-turns, 6.283185307179586232, x);
    r = fma(-turns, 2.4492935982947063545e-16, r);
    float s, c;
    sincosf((float)r, &s, &c);
    turn[i] = make_float2(c, a.sign * s);
  }
  for (int i = threadIdx.x; i < here; i += kBlock) {
    const int64_t b = (n0 + i) / a.T, t = (n0 + i) % a.T;
    q_at[i] = b * a.q_sb + t * a.q_st;
    k_at[i] = b * a.k_sb + t * a.k_st;
  }
  __syncthreads();
  constexpr int F = 16 / (int)sizeof(T);
  const int rest = a.dim - 2 * a.pairs;          // columns no axis turns: 16 bytes a lane where there are as many
  const int turned = MIX ? (2 * a.pairs + V - 1) / V : (a.pairs + V - 1) / V;
  const int per = turned + (rest >= F ? (rest + F - 1) / F : rest);   // pieces of a head
  const int row = (a.hq + a.hk) * per;
  for (int i = threadIdx.x; i < here * row; i += kBlock) {
    const int tk = i / row, in_row = i % row;
    const int head = in_row / per, piece = in_row % per;
    const bool is_q = head < a.hq;
    const int hd = is_q ? head : head - a.hq;
    const T* src = reinterpret_cast<const T*>(is_q ? a.q : a.k) + (is_q ? q_at[tk] + hd * a.q_sh : k_at[tk] + hd * a.k_sh);
    T* dst = reinterpret_cast<T*>(is_q ? a.oq : a.ok) + ((n0 + tk) * (is_q ? a.hq : a.hk) + hd) * a.dim;
    const float2* tr = turn + tk * a.pairs;
    if (piece >= turned) {
      if (rest >= F) {
        const int c0 = min(2 * a.pairs + (piece - turned) * F, a.dim - F);
        float x[F];
        load_any<T, F>(src + c0, x);
        store_any<T, F>(dst + c0, x);
      } else {
        const int c0 = 2 * a.pairs + piece - turned;
        dst[c0] = src[c0];
      }
    } else if constexpr (MIX) {
      // the last piece steps back to end with the last pair
      const int c0 = min(piece * V, 2 * a.pairs - V);
      float x[V], y[V];
      load_any<T, V>(src + c0, x);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 w = tr[(c0 + e) >> 1];
        y[e] = x[e] * w.x - x[e + 1] * w.y;
        y[e + 1] = x[e] * w.y + x[e + 1] * w.x;
      }
      store_any<T, V>(dst + c0, y);
    } else {
      const int p0 = min(piece * V, a.pairs - V);
      float u[V], v[V], x[V], y[V];
      load_any<T, V>(src + p0, u);
      load_any<T, V>(src + a.pairs + p0, v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 w = tr[p0 + e];
        x[e] = u[e] * w.x - v[e] * w.y;
        y[e] = u[e] * w.y + v[e] * w.x;
      }
      store_any<T, V>(dst + p0, x);
      store_any<T, V>(dst + a.pairs + p0, y);
    }
  }
}

template <typename T>
void go(const RotArgs& a, bool mix, unsigned grid, size_t lds, hipStream_t st) {
  const int w = mix ? 2 * a.pairs : a.pairs;
  constexpr int F = 16 / sizeof(T);
#define SLDM_GO(V, M) rotary_kernel<T, V, M><<<grid, kBlock, lds, st>>>(a)
  if (mix) {
    if (w >= F) SLDM_GO(F, true);
    else SLDM_GO(2, true);
  } else {
    if (w >= F) SLDM_GO(F, false);
    else if (F == 8 && w >= 4) SLDM_GO(4, false);
    else if (w >= 2) SLDM_GO(2, false);
    else SLDM_GO(1, false);
  }
#undef SLDM_GO
}

}  // namespace

extern "C" int sldm_rotary_axes(int dtype, const void* q, const int64_t* ld_q, int64_t heads_q, const void* k,
                                const int64_t* ld_k, int64_t heads_k, int64_t B, int64_t T, int64_t dim,
                                const void* positions, int pos_type, const int64_t* ld_pos, const double* inv_freq,
                                const int64_t* sections, int64_t num_axes, int interleaved, int inverse,
                                void* out_q, void* out_k, void* stream) {
  SLDM_REQUIRE(dtype == SLDM_F32 || dtype == SLDM_BF16, "sldm_rotary_axes: dtype must be fp32 or bf16");
  SLDM_REQUIRE(pos_type >= SLDM_POS_I32 && pos_type <= SLDM_POS_F64, "sldm_rotary_axes: position type %d", pos_type);
  SLDM_REQUIRE(num_axes >= 1 && num_axes <= kMaxAxes && sections, "sldm_rotary_axes: 1 to %d axes, got %lld",
               kMaxAxes, (long long)num_axes);
  SLDM_REQUIRE(B >= 0 && T >= 0 && heads_q >= 1 && heads_k >= 0 && dim >= 2 && dim <= kMaxDim,
               "sldm_rotary_axes: bad shape (head size %lld, 2 to %d)", (long long)dim, kMaxDim);
  RotArgs a{};
  int64_t pairs = 0;
  for (int64_t i = 0; i < num_axes; ++i) {
    SLDM_REQUIRE(sections[i] >= 0, "sldm_rotary_axes: negative section");
    pairs += sections[i];
    SLDM_REQUIRE(2 * pairs <= dim, "sldm_rotary_axes: sections turn %lld pairs or more, a head of %lld has %lld",
                 (long long)pairs, (long long)dim, (long long)(dim / 2));
    a.end[i] = (int)pairs;
  }
  SLDM_REQUIRE(pairs >= 1, "sldm_rotary_axes: no pair is turned");
  if (B * T == 0) return SLDM_OK;
  SLDM_REQUIRE(q && out_q && ld_q && positions && ld_pos && inv_freq && (!heads_k || (k && ld_k && out_k)),
               "sldm_rotary_axes: null argument");
  a.q = q; a.k = k; a.oq = out_q; a.ok = out_k;
  a.q_sb = ld_q[0]; a.q_st = ld_q[1]; a.q_sh = ld_q[2];
  if (heads_k) { a.k_sb = ld_k[0]; a.k_st = ld_k[1]; a.k_sh = ld_k[2]; }
  a.B = B; a.T = T;
  a.dim = (int)dim; a.pairs = (int)pairs; a.axes = (int)num_axes;
  a.pos = positions; a.pos_type = pos_type;
  a.pos_sb = ld_pos[0]; a.pos_st = ld_pos[1]; a.pos_sa = ld_pos[2];
  a.freq = inv_freq;
  a.sign = inverse ? -1.f : 1.f;
  // about 512 angles a workgroup, fewer tokens while that leaves CUs idle
  int64_t block = std::max<int64_t>(1, std::min<int64_t>(kMaxBlock, 512 / pairs));
  block = std::max<int64_t>(1, std::min<int64_t>(block, B * T / 1024));
  const int64_t per_head = dim;   // an upper bound of a head's pieces
  SLDM_REQUIRE((heads_q + heads_k) * per_head * block < ((int64_t)1 << 31), "sldm_rotary_axes: too many heads");
  a.hq = (int)heads_q; a.hk = (int)heads_k;
  a.block = (int)block;
  const int64_t grid = (B * T + block - 1) / block;
  SLDM_REQUIRE(grid * kBlock < ((int64_t)1 << 32), "sldm_rotary_axes: too many tokens (%lld)", (long long)(B * T));
  const size_t lds = (size_t)block * pairs * sizeof(float2);
  hipStream_t st = sldm::as_stream(stream);
  if (dtype == SLDM_F32) go<float>(a, interleaved != 0, (unsigned)grid, lds, st);
  else go<uint16_t>(a, interleaved != 0, (unsigned)grid, lds, st);
  SLDM_LAUNCH_CHECK("rotary_kernel");
  return SLDM_OK;
}
