// Host side of the decay attention operators (mathematics: decay.hpp, kernels:
// decay_f32.hip, decay_bf16.hpp), the scan that joins the segments of a long axis,
// the sum over shared heads, and the single-token step.
#include <algorithm>

#include "decay.hpp"

namespace sldm_decay {
namespace {

constexpr int kMaxDim = 128;
constexpr int64_t kMaxThreads = (int64_t)1 << 32;   // work-items of one launch, exclusive

constexpr int kCUs = 256;
constexpr int kChunk = 32;   // tokens of a segment are a multiple of this: no padding inside a sequence

// Segments of the time axis.  One workgroup walks a sequence alone unless that
// leaves the chip short of waves; then the axis is cut, at the price of a pass
// over k and v for the pieces' states, which are read and written too.  Fewer
// than four pieces do not pay for that pass (bf16, 64 heads of 64, 1024 frames:
// 51 us whole, 48 us in two, 33 in four; 128 heads, 512 frames: 29, 33, 32), nor
// do short ones, nor in fp32 so few waves missing that fewer than five would make them
// up (1024 heads of 16, 2048 frames: 115 us whole, 194 us in four).  Where only the
// length allows no more than four, those pay in fp32 for few heads (544 frames, 8 heads
// of 64: 66 us whole, 41 in four, training 130 and 83) and not quite for many (192
// heads: 66 and 81, 178 and 192).  Waves aimed at, of 8 / 12 / 16 a CU: bf16 (8 heads
// of 128, 32768 frames, training) 392 / 393 / 430 us, with 8 for the forward and 12 for
// the backward 380; fp32 (5 x 1237 frames, 8 over 2 heads of 48 and 80, training) 305 /
// 159 / 158 us.
struct Plan {
  int64_t seg_len;
  int nseg;
};
Plan plan(int dtype, int64_t B, int64_t H, int64_t T, int64_t dk, int64_t dv, int roles) {
  const int64_t C = kChunk;
  const int64_t waves = B * H * roles * std::max(tiles_of((int)dk), tiles_of((int)dv));
  const int64_t chunks = (T + C - 1) / C;
  const bool f32 = dtype == SLDM_F32;
  int64_t want = waves > 0 ? kCUs * (f32 ? 16 : roles == 3 ? 12 : 8) / waves : 1;
  if (f32 && want < 5) want = 1;
  want = std::min(want, chunks / (f32 ? 4 : 8));
  if (want < 4) return {std::max<int64_t>(T, 1), 1};
  const int64_t per = (chunks + want - 1) / want;
  return {per * C, (int)((chunks + per - 1) / per)};
}

// The backward's three walks need fewer, longer segments: whole multiples of the
// forward's, whose states they start from (m: forward segments in one of theirs).
struct Plans {
  Plan fwd, bwd;
  int m;
};
Plans plans(int dtype, int64_t B, int64_t H, int64_t T, int64_t dk, int64_t dv) {
  Plans p{plan(dtype, B, H, T, dk, dv, 1), plan(dtype, B, H, T, dk, dv, 3), 1};
  if (p.fwd.nseg == 1) p.bwd = p.fwd;
  if (p.bwd.nseg > 1) {
    p.m = (int)std::max<int64_t>(1, (p.bwd.seg_len + p.fwd.seg_len / 2) / p.fwd.seg_len);
    p.bwd = {p.fwd.seg_len * p.m, (p.fwd.nseg + p.m - 1) / p.m};
  }
  return p;
}

// loc[bh][s]: the states that segments add, each from zero -> the states
// before each segment, and the state behind the last one.  A segment's decay may be
// zero in fp32 where a token's is not: it leaves an infinity one.
__device__ __forceinline__ float faded(float s, float g, bool keeps) {
  const float r = s * g;
  return keeps && r != r ? s : r;
}
__global__ __launch_bounds__(256) void scan_kernel(float* loc, const float* s0, float* s1, Args a,
                                                   int64_t elems) {
  const int64_t bh = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (bh >= a.B * a.H || e >= elems) return;
  const int64_t len = seq_len(a, bh / a.H);
  const float ld2 = a.log_decay[bh % a.H] * 1.44269504088896340736f;
  float run = s0 ? s0[bh * elems + e] : 0.f;
  float* p = loc + bh * a.nseg * elems + e;
  const float g = exp2f(ld2 * (float)a.seg_len);
  const bool keeps = exp2f(ld2) > 0.f;
  const int whole = (int)(len / a.seg_len);   // segments without padding
  int s = 0;
  for (; s + 8 <= whole; s += 8) {             // eight loads in flight
    float add[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) add[i] = p[(s + i) * elems];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[(s + i) * elems] = run;
      run = faded(run, g, keeps) + add[i];
    }
  }
  for (; s < whole; ++s) {
    const float add = p[s * elems];
    p[s * elems] = run;
    run = faded(run, g, keeps) + add;
  }
  if (s < a.nseg) {
    const int64_t n = len - (int64_t)s * a.seg_len;
    const float add = p[s * elems];
    p[s * elems] = run;
    run = faded(run, powg(ld2, (int)n), keeps) + add;
    for (++s; s < a.nseg; ++s) p[s * elems] = run;
  }
  if (s1) s1[bh * elems + e] = run;
}

// out[b, t, hk, :] = sum over the group's heads of part[b, t, hk * group + g, :],
// for dk (blockIdx.y 0) and dv (1)
struct SumArgs {
  const float* part[2];
  void* out[2];
  int64_t heads;   // B T Hk
  int group, d[2];
};
template <typename T>
__global__ __launch_bounds__(256) void sum_heads_kernel(SumArgs a) {
  const int w = blockIdx.y, d = a.d[w];
  T* out = reinterpret_cast<T*>(a.out[w]);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.heads * d; i += (int64_t)gridDim.x * 256) {
    const int64_t head = i / d;
    const float* p = a.part[w] + head * a.group * d + i % d;
    float s = p[0];
    for (int g = 1; g < a.group; ++g) s += p[(int64_t)g * d];
    if constexpr (sizeof(T) == 4) out[i] = s;
    else out[i] = sldm::f32_to_bf16(s);
  }
}

// One token: S <- g S + k v^T and o = scale q S, the state read and written
// once (its 8 Dk Dv bytes are all that counts).  A workgroup owns one (batch,
// head); lanes hold V neighbouring value columns, the row groups' partial sums
// of o meet in LDS.  Measured: 512 x 16 states of 64 x 64 56 us a pass on states that
// change (4.9 TB/s), 43 us on the same ones (6.4 TB/s, partly from the Infinity Cache);
// 240 of 16 x 16 4.5 us.
struct StepArgs {
  const void *q, *k, *v;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
  void* o;
  float* state;
  const float* log_decay;
  int64_t H;
  int group, dk, dv, cols;   // cols: lanes across the value columns (a power of two)
  float scale;
};
template <typename T> __device__ __forceinline__ float as_f32(T v);
template <> __device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_f32<uint16_t>(uint16_t v) { return sldm::bf16_to_f32(v); }

template <typename T, int V, int NTH>
__global__ __launch_bounds__(NTH) void step_kernel(StepArgs a) {
  __shared__ float qs[kMaxDim], ks[kMaxDim], red[NTH * V];
  const int64_t bh = blockIdx.x, b = bh / a.H, hd = bh % a.H, hk = hd / a.group;
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.q_sb + hd * a.q_sh;
  const T* k = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T* v = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
  const int tid = threadIdx.x, col = tid & (a.cols - 1), grp = tid / a.cols, groups = NTH / a.cols;
  for (int i = tid; i < a.dk; i += NTH) {
    qs[i] = as_f32(q[i]) * a.scale;
    ks[i] = as_f32(k[i]);
  }
  const int c0 = col * V;
  const bool on = c0 < a.dv;
  float vv[V], acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    vv[e] = on ? as_f32(v[c0 + e]) : 0.f;
    acc[e] = 0.f;
  }
  const float g = expf(a.log_decay[hd]);
  __syncthreads();
  float* s = a.state + bh * a.dk * a.dv + c0;
  if (on) {
#pragma unroll 4
    for (int r = grp; r < a.dk; r += groups) {
      float w[V];
      sldm::Vec<float, V>::load(s + (int64_t)r * a.dv, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        w[e] = w[e] * g + ks[r] * vv[e];
        acc[e] += qs[r] * w[e];
      }
      sldm::Vec<float, V>::store(s + (int64_t)r * a.dv, w);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[grp * a.cols * V + c0 + e] = acc[e];
  __syncthreads();
  T* o = reinterpret_cast<T*>(a.o) + bh * a.dv;
  for (int c = tid; c < a.dv; c += NTH) {
    float sum = 0.f;
    for (int r = 0; r < groups; ++r) sum += red[r * a.cols * V + c];
    if constexpr (sizeof(T) == 4) o[c] = sum;
    else o[c] = sldm::f32_to_bf16(sum);
  }
}

Operand operand(const void* p, const int64_t* ld, bool shared, int esz) {
  Operand t{p, ld[0], ld[1], ld[2], shared, 1};
  for (int i = 0; i < 3; ++i) t.vec &= (ld[i] * esz) % 16 == 0;
  t.vec &= reinterpret_cast<uintptr_t>(p) % 16 == 0;
  return t;
}

void set_out(Role& r, void* o, int64_t T, int64_t H, int64_t d, bool f32, int esz) {
  r.o = o;
  r.o_sb = T * H * d;
  r.o_st = H * d;
  r.o_sh = d;
  r.o_f32 = f32;
  r.o_vec = (d * (f32 ? 4 : esz)) % 16 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0;
}

void launch_roles(int dtype, Args& a, const Role* const* roles, int n, bool out, hipStream_t st) {
  // roles of the same tile classes share a launch
  bool done[3] = {false, false, false};
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    int m = 0;
    for (int j = i; j < n; ++j)
      if (!done[j] && row_tiles(roles[j]->kd) == row_tiles(roles[i]->kd) &&
          tiles_of(roles[j]->vd) == tiles_of(roles[i]->vd)) {
        a.role[m++] = *roles[j];
        done[j] = true;
      }
    a.roles = m;
    // heads whose rows share 256 bytes
    const int64_t row = std::max<int64_t>(1, std::min(a.role[0].kd, a.role[0].vd)) * (dtype == SLDM_F32 ? 4 : 2);
    a.unit = m * (int)std::max<int64_t>(1, std::min<int64_t>(a.H, 256 / row));
    a.hpw = 1;
    a.by_unit = Div(a.unit);
    a.by_roles = Div(m);
    a.by_all = Div(a.B * a.H);
    a.by_h = Div(a.H);
    a.by_group = Div(a.group);
    if (dtype == SLDM_F32) run_f32(a, out, st);
    else run_bf16(a, out, st);
  }
}

int scan(float* loc, const float* s0, float* s1, const Args& a, int64_t elems, hipStream_t st) {
  const int64_t bh = a.B * a.H;
  const int64_t y = std::min<int64_t>(bh, 32768);
  scan_kernel<<<dim3((unsigned)((elems + 255) / 256), (unsigned)y, (unsigned)((bh + y - 1) / y)), 256, 0, st>>>(
      loc, s0, s1, a, elems);
  SLDM_LAUNCH_CHECK("decay scan_kernel");
  return SLDM_OK;
}

int check_shape(int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t dk, int64_t dv) {
  SLDM_REQUIRE(dtype == SLDM_F32 || dtype == SLDM_BF16, "decay attention: dtype must be fp32 or bf16");
  SLDM_REQUIRE(B >= 0 && T >= 0 && T < ((int64_t)1 << 31), "decay attention: B and T must be >= 0, T < 2^31");
  SLDM_REQUIRE(H >= 1 && Hk >= 1 && H % Hk == 0, "decay attention: %lld heads over %lld key heads",
               (long long)H, (long long)Hk);
  SLDM_REQUIRE(dk >= 1 && dk <= kMaxDim && dv >= 1 && dv <= kMaxDim,
               "decay attention: head sizes must be in [1, %d], got %lld and %lld", kMaxDim, (long long)dk,
               (long long)dv);
  SLDM_REQUIRE(B * H < kMaxThreads / 256 / 4, "decay attention: too many (batch, head) pairs: %lld",
               (long long)(B * H));
  return SLDM_OK;
}

}  // namespace
}  // namespace sldm_decay

using namespace sldm_decay;

extern "C" size_t sldm_decay_attention_states_bytes(int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk,
                                                    int64_t dk, int64_t dv) {
  if (check_shape(dtype, B, T, H, Hk, dk, dv) != SLDM_OK) return 0;
  const Plan p = plan(dtype, B, H, T, dk, dv, 1);
  return p.nseg > 1 ? (size_t)(B * H) * p.nseg * dk * dv * 4 : 0;
}

extern "C" size_t sldm_decay_attention_bwd_workspace_bytes(int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk,
                                                           int64_t dk, int64_t dv) {
  if (check_shape(dtype, B, T, H, Hk, dk, dv) != SLDM_OK) return 0;
  const Plans p = plans(dtype, B, H, T, dk, dv);
  size_t n = p.bwd.nseg > 1 ? (size_t)(B * H) * p.fwd.nseg * dk * dv : 0;
  if (H != Hk) n += (size_t)(B * T * H) * (dk + dv);
  return n * 4;
}

extern "C" int sldm_decay_attention_fwd(int dtype, const void* q, const int64_t* ld_q, const void* k,
                                        const int64_t* ld_k, const void* v, const int64_t* ld_v, int64_t B,
                                        int64_t T, int64_t H, int64_t Hk, int64_t dk, int64_t dv,
                                        const float* log_decay, float scale, const float* state,
                                        const void* lengths, int lengths_int64, void* out, float* state_out,
                                        float* states, size_t states_bytes, void* stream) {
  if (const int rc = check_shape(dtype, B, T, H, Hk, dk, dv)) return rc;
  if (B == 0) return SLDM_OK;
  SLDM_REQUIRE(ld_q && ld_k && ld_v && log_decay, "sldm_decay_attention_fwd: null argument");
  SLDM_REQUIRE(T == 0 || (q && k && v && out), "sldm_decay_attention_fwd: null argument");
  const size_t need = sldm_decay_attention_states_bytes(dtype, B, T, H, Hk, dk, dv);
  SLDM_REQUIRE(!need || (states && states_bytes >= need), "sldm_decay_attention_fwd: no room for the states");
  const int esz = dtype == SLDM_F32 ? 4 : 2, group = (int)(H / Hk);
  const Plan p = plan(dtype, B, H, T, dk, dv, 1);
  const int64_t elems = dk * dv;
  hipStream_t st = sldm::as_stream(stream);
  Args a{};
  a.B = B; a.H = H; a.T = T; a.group = group;
  a.seg_len = p.seg_len; a.nseg = p.nseg; a.groups = (int)(B * H * p.nseg);
  a.log_decay = log_decay; a.lengths = lengths; a.lengths64 = lengths_int64;
  Role r{};
  r.q = operand(q, ld_q, false, esz);
  r.k = operand(k, ld_k, group > 1, esz);
  r.v = operand(v, ld_v, group > 1, esz);
  set_out(r, out, T, H, dv, false, esz);
  r.kd = (int)dk; r.vd = (int)dv;
  r.s_k = (int)dv; r.s_v = 1;
  r.read_scale = r.p_scale = scale;
  r.upd_scale = 1.f;
  const Role* one[1] = {&r};
  if (p.nseg == 1) {
    r.s0 = state; r.s0_bh = elems;
    r.s1 = state_out; r.s1_bh = elems;
    launch_roles(dtype, a, one, 1, true, st);
    SLDM_LAUNCH_CHECK("decay_kernel");
    return SLDM_OK;
  }
  float* loc = states;
  r.s1 = loc; r.s1_bh = p.nseg * elems; r.s1_seg = elems;
  launch_roles(dtype, a, one, 1, false, st);
  SLDM_LAUNCH_CHECK("decay_kernel (states)");
  if (const int rc = scan(loc, state, state_out, a, elems, st)) return rc;
  r.s1 = nullptr;
  r.s0 = loc; r.s0_bh = p.nseg * elems; r.s0_seg = elems;
  launch_roles(dtype, a, one, 1, true, st);
  SLDM_LAUNCH_CHECK("decay_kernel");
  return SLDM_OK;
}

extern "C" int sldm_decay_attention_bwd(int dtype, const void* q, const int64_t* ld_q, const void* k,
                                        const int64_t* ld_k, const void* v, const int64_t* ld_v, const void* dout,
                                        const int64_t* ld_do, int64_t B, int64_t T, int64_t H, int64_t Hk,
                                        int64_t dk, int64_t dv, const float* log_decay, float scale,
                                        const float* state, const float* states, const float* dstate_out,
                                        const void* lengths, int lengths_int64, void* dq, void* dk_out, void* dv_out,
                                        float* dstate, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_shape(dtype, B, T, H, Hk, dk, dv)) return rc;
  if (B == 0) return SLDM_OK;
  SLDM_REQUIRE(ld_q && ld_k && ld_v && ld_do && log_decay, "sldm_decay_attention_bwd: null argument");
  SLDM_REQUIRE(T == 0 || (q && k && v && dout), "sldm_decay_attention_bwd: null argument");
  const size_t need = sldm_decay_attention_bwd_workspace_bytes(dtype, B, T, H, Hk, dk, dv);
  SLDM_REQUIRE(!need || (workspace && workspace_bytes >= need), "sldm_decay_attention_bwd: workspace too small");
  const int esz = dtype == SLDM_F32 ? 4 : 2, group = (int)(H / Hk);
  const Plans p = plans(dtype, B, H, T, dk, dv);
  const bool cut = p.bwd.nseg > 1;
  SLDM_REQUIRE(!cut || states, "sldm_decay_attention_bwd: the forward's states are needed");
  const int64_t elems = dk * dv;
  hipStream_t st = sldm::as_stream(stream);
  Args a{};
  a.B = B; a.H = H; a.T = T; a.group = group;
  a.log_decay = log_decay; a.lengths = lengths; a.lengths64 = lengths_int64;
  auto segments = [&](const Plan& s) {
    a.seg_len = s.seg_len; a.nseg = s.nseg; a.groups = (int)(B * H * s.nseg);
  };

  float* ws = reinterpret_cast<float*>(workspace);
  float *locR = nullptr, *part_k = nullptr, *part_v = nullptr;
  if (cut) {
    locR = ws; ws += B * H * p.fwd.nseg * elems;
  }
  if (group > 1) {
    part_k = ws; ws += B * T * H * dk;
    part_v = ws;
  }
  const Operand oq = operand(q, ld_q, false, esz), ok = operand(k, ld_k, group > 1, esz),
                ov = operand(v, ld_v, group > 1, esz), od = operand(dout, ld_do, false, esz);

  Role rq{}, rk{}, rv{};
  rq.q = od; rq.k = ov; rq.v = ok;               // dq_t = scale S_t do_t
  rq.kd = (int)dv; rq.vd = (int)dk;
  rq.s_k = 1; rq.s_v = (int)dv;
  rq.read_scale = rq.p_scale = scale; rq.upd_scale = 1.f;
  set_out(rq, dq, T, H, dk, false, esz);
  rv.q = ok; rv.k = oq; rv.v = od;               // dv_t = k_t G_t
  rv.kd = (int)dk; rv.vd = (int)dv;
  rv.s_k = (int)dv; rv.s_v = 1;
  rv.read_scale = 1.f; rv.p_scale = rv.upd_scale = scale;
  rv.delta = rv.reverse = 1;
  set_out(rv, group > 1 ? (void*)part_v : dv_out, T, H, dv, group > 1, esz);
  rk.q = ov; rk.k = od; rk.v = oq;               // dk_t = G_t v_t
  rk.kd = (int)dv; rk.vd = (int)dk;
  rk.s_k = 1; rk.s_v = (int)dv;
  rk.read_scale = 1.f; rk.p_scale = rk.upd_scale = scale;
  rk.delta = rk.reverse = 1;
  set_out(rk, group > 1 ? (void*)part_k : dk_out, T, H, dk, group > 1, esz);

  if (cut) {
    if (dk_out || dv_out || dstate) {            // the gradient that each segment adds to the state
      segments(p.fwd);
      Role g = rv;
      g.s1 = locR;
      g.s1_bh = p.fwd.nseg * elems;
      g.s1_seg = elems;
      const Role* one[1] = {&g};
      launch_roles(dtype, a, one, 1, false, st);
      SLDM_LAUNCH_CHECK("decay_kernel (states)");
      if (const int rc = scan(locR, dstate_out, dstate, a, elems, st)) return rc;
    }
    segments(p.bwd);
    rq.s0 = states; rk.s0 = rv.s0 = locR;
    rq.s0_bh = rk.s0_bh = rv.s0_bh = p.fwd.nseg * elems;
    rq.s0_seg = rk.s0_seg = rv.s0_seg = p.m * elems;
  } else {
    segments(p.bwd);
    rq.s0 = state; rk.s0 = rv.s0 = dstate_out;
    rq.s0_bh = rk.s0_bh = rv.s0_bh = elems;
    rv.s1 = dstate; rv.s1_bh = elems;
    if (dstate && !dv_out) {                     // the state's gradient alone
      const Role* one[1] = {&rv};
      launch_roles(dtype, a, one, 1, false, st);
      SLDM_LAUNCH_CHECK("decay_kernel (states)");
    }
  }
  const Role* roles[3];
  int n = 0;
  if (dq) roles[n++] = &rq;
  if (dk_out) roles[n++] = &rk;
  if (dv_out) roles[n++] = &rv;
  launch_roles(dtype, a, roles, n, true, st);
  SLDM_LAUNCH_CHECK("decay_kernel");
  if (group > 1 && T > 0 && (dk_out || dv_out)) {
    SumArgs s{{part_k, part_v}, {dk_out, dv_out}, B * T * Hk, group, {(int)dk, (int)dv}};
    if (!dk_out) s.part[0] = part_v, s.out[0] = dv_out, s.d[0] = (int)dv;
    const int64_t most = s.heads * std::max(s.d[0], s.d[1]);
    const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, 1 << 15), dk_out && dv_out ? 2 : 1);
    if (dtype == SLDM_F32) sum_heads_kernel<float><<<grid, 256, 0, st>>>(s);
    else sum_heads_kernel<uint16_t><<<grid, 256, 0, st>>>(s);
    SLDM_LAUNCH_CHECK("decay sum_heads_kernel");
  }
  return SLDM_OK;
}

extern "C" int sldm_decay_attention_step(int dtype, const void* q, const int64_t* ld_q, const void* k,
                                         const int64_t* ld_k, const void* v, const int64_t* ld_v, int64_t B,
                                         int64_t H, int64_t Hk, int64_t dk, int64_t dv, const float* log_decay,
                                         float scale, float* state, void* out, void* stream) {
  if (const int rc = check_shape(dtype, B, 1, H, Hk, dk, dv)) return rc;
  if (B == 0) return SLDM_OK;
  SLDM_REQUIRE(q && k && v && ld_q && ld_k && ld_v && log_decay && state && out,
               "sldm_decay_attention_step: null argument");
  StepArgs a{q, k, v, ld_q[0], ld_q[1], ld_k[0], ld_k[1], ld_v[0], ld_v[1], out, state, log_decay, H,
             (int)(H / Hk), (int)dk, (int)dv, 1, scale};
  const bool vec = dv % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
  while (a.cols * (vec ? 4 : 1) < dv) a.cols <<= 1;
  const bool small = dk * dv <= 1024;   // at most eight elements a lane of two waves; else four waves
  const unsigned grid = (unsigned)(B * H);
  hipStream_t st = sldm::as_stream(stream);
#define SLDM_STEP(T, V) \
  (small ? step_kernel<T, V, 128><<<grid, 128, 0, st>>>(a) : step_kernel<T, V, 256><<<grid, 256, 0, st>>>(a))
  if (dtype == SLDM_F32) vec ? SLDM_STEP(float, 4) : SLDM_STEP(float, 1);
  else vec ? SLDM_STEP(uint16_t, 4) : SLDM_STEP(uint16_t, 1);
#undef SLDM_STEP
  SLDM_LAUNCH_CHECK("step_kernel");
  return SLDM_OK;
}
