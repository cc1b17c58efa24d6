// dm_mixer_device.h -- device helpers of the token mixer's kernels: row types,
// the sequences of a call, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dm_device.h"
#include "dm_mixer.h"

namespace dm {

// (HIP's min of a 64-bit and a 32-bit integer is a double)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// ---- row types ----------------------------------------------------------------
typedef _Float16 half_t;
typedef __bf16 bf16_t;

// N consecutive elements, aligned as one is: global memory takes such an access
// of up to 16 bytes at any element's address as it does an aligned one, so rows
// need no alignment or pitch of their own.
template <typename T, int N>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T>
struct VecOf<T, 1> {
  typedef T type;
};
template <typename T, int N>
using Vec = typename VecOf<T, N>::type;
template <int N, typename T>
__device__ __forceinline__ Vec<T, N> load_raw(const T* p) {
  return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <int N, typename T>
__device__ __forceinline__ void to_f32(T v, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = (float)v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)v[i];
  }
}
template <int N, typename T>
__device__ __forceinline__ void load_f32(const T* p, float (&f)[N]) {
  to_f32<N>(load_raw<N>(p), f);
}
template <int N, typename T>
__device__ __forceinline__ void store_f32(T* p, const float (&f)[N]) {
  if constexpr (N == 1) {
    *p = (T)f[0];
  } else {
    Vec<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)f[i];
    *reinterpret_cast<Vec<T, N>*>(p) = r;
  }
}

// ---- sequences ------------------------------------------------------------------
struct SeqRange {
  int begin, end, slot;
  bool fresh, live;  // live: rows to work on and a state to keep
};

// Whether an offset before sequence i lies behind `begin`, its first row.  What lies
// before a sequence that is not skipped is that one's to find wrong, so the way back
// ends there; offsets of skipped ones come eight at a time, as no load then waits for
// the slot before it.  before, slot: the offset and slot of sequence i - 1.
__device__ __forceinline__ bool offsets_fall(const SeqDev& s, int i, int begin, int before,
                                             int slot) {
  bool fall = before > begin, last = slot >= 0;
  for (int j = i - 2; j >= 0 && !fall && !last; j -= 8) {
    int off[8], slots[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      off[u] = s.off[max(j - u, 0)];
      slots[u] = s.slots[max(j - u, 0)];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      fall = fall || (!last && off[u] > begin);
      last = last || slots[u] >= 0;
    }
  }
  return fall;
}

// Sequence i, with everything about it checked that it and the skipped ones before
// it show.  report: record what is wrong with it (one workgroup per sequence does).
__device__ __forceinline__ SeqRange seq_range(const SeqDev& s, int i, bool report) {
  SeqRange r;
  r.begin = s.off[i];
  r.end = s.off[i + 1];
  r.slot = s.slots ? s.slots[i] : i;
  r.fresh = s.fresh && s.fresh[i] != 0;
  const int before = i ? s.off[i - 1] : 0, slot = i && s.slots ? s.slots[i - 1] : 0;
  r.live = r.slot >= 0;
  uint32_t kind = kSqCount;
  if (r.live) {
    if (r.begin < 0 || r.end < r.begin || r.end > s.rows ||
        offsets_fall(s, i, r.begin, before, slot))
      kind = kSqOffsets;
    else if (r.end - r.begin > s.max_len) kind = kSqLength;
    else if (r.slot >= s.slots_n) kind = kSqSlot;
  }
  if (kind != kSqCount) {
    r.live = false;
    if (report) record_err(s.status, err_key(kPhSeq, 0, 0, (uint32_t)i, kind));
  }
  if (r.end == r.begin) r.live = false;
  return r;
}

// Whether an earlier sequence with rows names the state of sequence i; lanes of
// one wave look at 64 of them at a time.
__device__ __forceinline__ void report_shared_slot(const SeqDev& s, int i, int slot, int lane) {
  bool same = false;
  for (int j = lane; j < i; j += 64)
    same = same || (s.slots[j] == slot && s.off[j + 1] > s.off[j]);
  if (same) record_err(s.status, err_key(kPhSeq, 0, 0, (uint32_t)i, kSqTwice));
}

// ---- activations ------------------------------------------------------------------
// 1 / (1 + e^-z) from the hardware's exp2 and reciprocal.  -z log2(e) is taken
// as a rounded product and its remainder, so the exponential keeps 1e-7 at any
// size of z; beyond +-100 the result no longer changes.
__device__ __forceinline__ float sigmoid_hw(float z) {
  const float c = fminf(fmaxf(z, -100.0f), 100.0f);
  const float hi = c * -0x1.715476p+0f;
  float lo = __builtin_fmaf(c, -0x1.715476p+0f, -hi);
  lo = __builtin_fmaf(c, -0x1.4ae0cp-26f, lo);
  float e = __builtin_amdgcn_exp2f(hi);
  e = __builtin_fmaf(e, lo * 0x1.62e43p-1f, e);
  e = hi >= 128.0f ? __builtin_inff() : e;
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return z != z ? z : r;
}

// The gates of one row and head of the delta rule: loaded as they are, since a
// conversion or a branch would wait for them, and made from raw or final values
// once other loads are on their way.  softplus above 20 is its argument to fp32's
// last bit.
struct Gates {
  float log_decay, beta;
};
template <typename T>
struct RawGates {
  T a, b;
  float fa, fb, a_log, dt;
};
template <typename T>
__device__ __forceinline__ RawGates<T> load_gates(const dmh_gated_delta& d, int64_t t, int h) {
  RawGates<T> r = {};
  if (d.a_log) {
    r.a = static_cast<const T*>(d.a)[t * d.a_stride + h];
    r.b = static_cast<const T*>(d.b)[t * d.b_stride + h];
    r.a_log = d.a_log[h];
    if (d.dt_bias) r.dt = d.dt_bias[h];
  } else {
    r.fa = static_cast<const float*>(d.a)[t * d.a_stride + h];
    r.fb = static_cast<const float*>(d.b)[t * d.b_stride + h];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Gates gates_of(const dmh_gated_delta& d, const RawGates<T>& r) {
  if (!d.a_log) return {r.fa, r.fb};
  const float a = (float)r.a + r.dt;
  return {-expf(r.a_log) * (a > 20.0f ? a : log1pf(expf(a))), 1.0f / (1.0f + expf(-(float)r.b))};
}

// The sum over the lanes whose number is the lane's own but for bits 3 to 5, in
// all of them, without a way through LDS.
__device__ __forceinline__ float sum_eighths(float x) {
  const auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
  const int eight = __builtin_amdgcn_update_dpp(0, (int)bits(x), 0x128, 0xF, 0xF, false);
  x += __builtin_bit_cast(float, eight);
  auto p = __builtin_amdgcn_permlane16_swap(bits(x), bits(x), false, false);
  x = __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
  p = __builtin_amdgcn_permlane32_swap(bits(x), bits(x), false, false);
  return __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
}

// ---- the delta rule, row by row -----------------------------------------------------
// A wave keeps 32 columns of one head's state in registers for the length of a
// sequence: lane (rg, cg) holds columns 4 cg .. 4 cg + 3 of the RPL rows
// RPL rg .. RPL rg + RPL - 1.  Columns never meet, so waves share nothing.
// Both products with the old state, S^T k and S^T q, run in one pass over the
// registers, and the new state's S'^T q = g S^T q + (k . q) u needs no second
// one.  A row's three sums of squares and eight column sums are then added over
// the eight row groups.  One read and one write of the state bound a single row
// per sequence: 128 bytes per row and wave, whole lines; 250 sequences of 32
// heads, 1.05 GB, in 167 us, 6.3 TB/s.  Further rows are bound by the instructions
// of a wave, 620 a row: 1.15 us.
// Sequences of more than max_rows rows (64 at most) are left alone; block: of the workgroups
// that delta_rows_blocks counts.
inline unsigned delta_rows_blocks(const dmh_gated_delta& d, const SeqDev& s) {
  return (unsigned)(((int64_t)s.num * d.v_heads * ((d.v_dim + 31) / 32) + 3) / 4);
}
template <typename T, int RPL>
__device__ __forceinline__ void delta_rows(const dmh_gated_delta& d, const SeqDev& s, int max_rows,
                                           unsigned block) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cg = lane & 7, rg = lane >> 3;
  const int ncb = (d.v_dim + 31) / 32;
  const int64_t unit = (int64_t)block * 4 + wave;
  const int per_seq = ncb * d.v_heads;
  const int seq = (int)(unit / per_seq);
  if (seq >= s.num) return;
  const int in_seq = (int)(unit - (int64_t)seq * per_seq);
  const int h = in_seq / ncb, cb = in_seq - h * ncb;
  const SeqRange r = seq_range(s, seq, in_seq == 0 && lane == 0);
  if (!r.live) return;
  if (in_seq == 0 && s.slots) report_shared_slot(s, seq, r.slot, lane);
  const int len = r.end - r.begin;
  if (len > max_rows) return;

  const int kh = h / (d.v_heads / d.k_heads);
  const int row0 = rg * RPL, col0 = cb * 32 + cg * 4;
  const bool col_in = col0 < d.v_dim;
  // Loads are not conditional, so that none waits for another: what is not there
  // is read from the first row or column.  Of rows that are not there keys,
  // queries and state are zeros; columns that are not there meet no others.
  constexpr int B = RPL / 8;
  int at[B];  // (k_dim is a multiple of 8)
#pragma unroll
  for (int i = 0; i < B; ++i) at[i] = row0 + 8 * i < d.k_dim ? row0 + 8 * i : 0;
  const T* qp = static_cast<const T*>(d.q) + r.begin * d.q_stride + (int64_t)kh * d.k_dim;
  const T* kp = static_cast<const T*>(d.k) + r.begin * d.k_stride + (int64_t)kh * d.k_dim;
  const T* vp = static_cast<const T*>(d.v) + r.begin * d.v_stride + (int64_t)h * d.v_dim +
                (col_in ? col0 : 0);
  T* op = static_cast<T*>(d.o) + r.begin * d.o_stride + (int64_t)h * d.v_dim + col0;

  // the gates of all rows, a row per lane, on their way before the state
  const RawGates<T> raw = load_gates<T>(d, r.begin + min(lane, len - 1), h);
  Vec<T, 8> qn[B], kn[B];
  Vec<T, 4> vn;  // (as they come: a conversion would wait for them)
  const auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < B; ++i) {
      qn[i] = load_raw<8>(qp + t * d.q_stride + at[i]);
      kn[i] = load_raw<8>(kp + t * d.k_stride + at[i]);
    }
    vn = load_raw<4>(vp + t * d.v_stride);
  };
  fetch(0);
  float* sp = d.state + ((size_t)r.slot * d.v_heads + h) * d.k_dim * d.v_dim + (col_in ? col0 : 0);
  f32x4 S[RPL];
  if (r.fresh) {
#pragma unroll
    for (int i = 0; i < RPL; ++i) S[i] = f32x4{};
  } else {
#pragma unroll
    for (int i = 0; i < RPL; ++i)
      S[i] = *reinterpret_cast<const f32x4*>(sp + (size_t)(at[i / 8] + i % 8) * d.v_dim);
  }
  const Gates gates = gates_of(d, raw);
  const float decays = expf(gates.log_decay);
#pragma unroll
  for (int i = 0; i < RPL; ++i)
    if (row0 + i / 8 * 8 >= d.k_dim) S[i] = f32x4{};
  for (int t = 0; t < len; ++t) {
    float q[RPL], k[RPL], v[4];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const bool in = row0 + 8 * i < d.k_dim;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        q[8 * i + j] = in ? (float)qn[i][j] : 0.0f;
        k[8 * i + j] = in ? (float)kn[i][j] : 0.0f;
      }
    }
    to_f32<4>(vn, v);
    fetch(min(t + 1, len - 1));

    float sum[11] = {};  // k.k, q.q, k.q, and k.S and q.S of the four columns
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      sum[0] = __builtin_fmaf(k[i], k[i], sum[0]);
      sum[1] = __builtin_fmaf(q[i], q[i], sum[1]);
      sum[2] = __builtin_fmaf(k[i], q[i], sum[2]);
    }
#pragma unroll
    for (int i = 0; i < RPL; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[3 + j] = __builtin_fmaf(k[i], S[i][j], sum[3 + j]);
        sum[7 + j] = __builtin_fmaf(q[i], S[i][j], sum[7 + j]);
      }
#pragma unroll
    for (int j = 0; j < 11; ++j) sum[j] = sum_eighths(sum[j]);
    const float rk = d.qk_norm ? 1.0f / sqrtf(sum[0] + d.eps) : 1.0f;
    const float rq = d.qk_norm ? d.scale / sqrtf(sum[1] + d.eps) : d.scale;
    const float decay = __shfl(decays, t), beta = __shfl(gates.beta, t);
    float u[4], o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[j] = beta * (v[j] - decay * (rk * sum[3 + j])) * rk;
      o[j] = rq * (decay * sum[7 + j] + sum[2] * u[j]);
    }
#pragma unroll
    for (int i = 0; i < RPL; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf(k[i], u[j], decay * S[i][j]);
    if (rg == 0 && col_in) store_f32<4>(op + t * d.o_stride, o);
  }
  if (!col_in) return;
  // Past the L2, since it is read again in the model's next step: 250 sequences of
  // 32 heads in 167 us instead of 182 (32 of them: 21.7 and 21.2).
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (row0 + 8 * i >= d.k_dim) break;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      __builtin_nontemporal_store(S[8 * i + j],
                                  reinterpret_cast<f32x4*>(sp + (size_t)(at[i] + j) * d.v_dim));
  }
}

}  // namespace dm
