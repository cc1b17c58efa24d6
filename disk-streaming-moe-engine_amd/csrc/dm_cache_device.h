// dm_cache_device.h -- device helpers of the kernels on the 4-bit cache.
#pragma once
#include "dm_cache.h"
#include "dm_mixer_device.h"

namespace dm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Two codes as bf16 values times the power of two whose exponent field `scale` holds
// (255: NaN), exactly.
template <int BYTE>
__device__ __forceinline__ uint32_t held_pair(uint32_t codes, uint32_t scale) {
  return __builtin_bit_cast(
      uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, u2f(scale), BYTE));
}

// 1 / (1 + e^-z), also where it is below fp32's normal numbers, which the hardware's
// reciprocal takes for 0.
__device__ __forceinline__ float sigmoid_all(float z) {
  const float e = expf(-__builtin_fabsf(z));
  return (z < 0.0f ? e : 1.0f) / (1.0f + e);
}

// A sequence's rows and the tokens before them, with everything about it checked that
// no page needs.
struct CacheSeq {
  int begin, n, past, slot;  // n 0: none to work on
};
__device__ __forceinline__ CacheSeq cache_seq(const CacheDev& c, const SeqDev& s, int i,
                                              bool report) {
  const SeqRange r = seq_range(s, i, report);
  CacheSeq q = {r.begin, 0, 0, r.slot};
  if (!r.live) return q;
  q.past = r.fresh ? 0 : c.past[r.slot];
  if (q.past < 0 || (int64_t)q.past + (r.end - r.begin) > ((int64_t)c.max_pages << c.page_shift)) {
    if (report) record_err(s.status, err_key(kPhSeq, 0, 0, (uint32_t)i, kSqPast));
    return q;
  }
  q.n = r.end - r.begin;
  return q;
}

// The page of a position (of a sequence that cache_seq found whole), or -1.
__device__ __forceinline__ int page_of(const CacheDev& c, int slot, int pos) {
  const int p = c.pages[(int64_t)slot * c.max_pages + (pos >> c.page_shift)];
  return (unsigned)p < (unsigned)c.num_pages ? p : -1;
}
// The number of a region, each of page_size positions.
__device__ __forceinline__ size_t region_of(const CacheDev& c, int page, int kind, int head) {
  return ((size_t)page * 2 + kind) * c.heads + head;
}

}  // namespace dm
