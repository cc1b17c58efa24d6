// dm_mixer_device.h -- device helpers of the token mixer's kernels: row types,
// the sequences of a call, activations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dm_device.h"
#include "dm_mixer.h"

namespace dm {

// ---- row types ----------------------------------------------------------------
typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <typename T, int N>
struct alignas(sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};

// N consecutive elements as fp32: one or two 16-byte loads where `wide`, else
// element by element.
template <int N, typename T>
__device__ __forceinline__ void load_f32(const T* p, bool wide, float (&f)[N]) {
  if (wide) {
    const Vec<T, N> r = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)p[i];
  }
}
template <int N, typename T>
__device__ __forceinline__ void store_f32(T* p, bool wide, const float (&f)[N]) {
  if (wide) {
    Vec<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)f[i];
    *reinterpret_cast<Vec<T, N>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = (T)f[i];
  }
}

// ---- sequences ------------------------------------------------------------------
struct SeqRange {
  int begin, end, slot;
  bool fresh, live;  // live: rows to work on and a state to keep
};

// Sequence i, with everything about it checked that this sequence alone shows.
// report: record what is wrong with it (one workgroup per sequence does).
__device__ __forceinline__ SeqRange seq_range(const SeqDev& s, int i, bool report) {
  SeqRange r;
  r.begin = s.off[i];
  r.end = s.off[i + 1];
  r.slot = s.slots ? s.slots[i] : i;
  r.fresh = s.fresh && s.fresh[i] != 0;
  r.live = r.slot >= 0;
  uint32_t kind = kSqCount;
  if (r.live) {
    if (r.begin < 0 || r.end < r.begin || r.end > s.rows) kind = kSqOffsets;
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

// The gates of one row and head of the delta rule, from raw or final values.
// softplus above 20 is its argument to fp32's last bit.
struct Gates {
  float log_decay, beta;
};
__device__ __forceinline__ Gates gates_of(float a_dt, float b, float a_log) {
  return {-expf(a_log) * (a_dt > 20.0f ? a_dt : log1pf(expf(a_dt))), 1.0f / (1.0f + expf(-b))};
}
template <typename T>
__device__ __forceinline__ Gates load_gates(const dmh_gated_delta& d, int64_t t, int h) {
  if (!d.a_log)
    return {static_cast<const float*>(d.a)[t * d.a_stride + h],
            static_cast<const float*>(d.b)[t * d.b_stride + h]};
  return gates_of((float)static_cast<const T*>(d.a)[t * d.a_stride + h] +
                      (d.dt_bias ? d.dt_bias[h] : 0.0f),
                  (float)static_cast<const T*>(d.b)[t * d.b_stride + h], d.a_log[h]);
}

}  // namespace dm
