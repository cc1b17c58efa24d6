// dm_cache.hip -- rows of keys and values into the 4-bit cache and out of it.
//
// A thread takes 8 elements of one head's row, four threads a block of 32: they agree
// on its largest element and its scale, and each makes one word of codes.  The
// hardware converts both ways (round to nearest even, above 6 to 6), so the bytes
// bound both kernels.
#include <algorithm>
#include <type_traits>

#include "dm_cache_device.h"

namespace dm {
namespace {

template <typename F>
hipError_t with_type(int dtype, F f) {
  if (dtype == DMH_DTYPE_BF16) return f(bf16_t{});
  if (dtype == DMH_DTYPE_F16) return f(half_t{});
  return f(float{});
}

// The eight codes of element group u of a value, one bit field of each two per lane.
template <int NB>
__device__ __forceinline__ void store_value(uint8_t* region, size_t pos, int u, uint32_t w) {
  using L = CacheLay<NB>;
  if constexpr (L::pow2 && NB >= 4) {
    *reinterpret_cast<uint32_t*>(region + L::value_byte(pos, u * 4 / NB, u * 4 % NB)) = w;
  } else if constexpr (NB == 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<uint16_t*>(region + L::value_byte(pos, 2 * u + i, 0)) = (uint16_t)(w >> (16 * i));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      region[L::value_byte(pos, (u & 3) * 4 + i, NB == 1 ? 0 : u >> 2)] = (uint8_t)(w >> (8 * i));
  }
}
template <int NB>
__device__ __forceinline__ uint32_t load_value(const uint8_t* region, size_t pos, int u) {
  using L = CacheLay<NB>;
  if constexpr (L::pow2 && NB >= 4) {
    return *reinterpret_cast<const uint32_t*>(region + L::value_byte(pos, u * 4 / NB, u * 4 % NB));
  } else if constexpr (NB == 2) {
    const uint32_t lo = *reinterpret_cast<const uint16_t*>(region + L::value_byte(pos, 2 * u, 0));
    const uint32_t hi = *reinterpret_cast<const uint16_t*>(region + L::value_byte(pos, 2 * u + 1, 0));
    return lo | hi << 16;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w |= (uint32_t)region[L::value_byte(pos, (u & 3) * 4 + i, NB == 1 ? 0 : u >> 2)] << (8 * i);
    return w;
  }
}

template <typename T, int NB, bool WRITE>
__global__ __launch_bounds__(256) void k_kv_rows(CacheDev c, dmh_kv_rows r, SeqDev s,
                                                 int64_t block0) {
  using L = CacheLay<NB>;
  const int tid = threadIdx.x;
  constexpr int per_head = 4 * NB;
  const int per_row = 2 * c.heads * per_head;
  const int64_t at = (block0 + blockIdx.x) * 256;
  // (fewer than 2^30 rows)
  const int t0 = (int)(at / per_row), t = (int)((at + tid) / per_row);

  // the first sequence with a row at t0 or behind it, then this row's
  __shared__ int first_seq;
  if (tid == 0) first_seq = s.num;
  __syncthreads();
  int j0 = tid;
  while (j0 < s.num && s.off[j0 + 1] <= t0) j0 += 256;
  if (j0 < s.num) atomicMin(&first_seq, j0);
  __syncthreads();
  int q = first_seq;
  if (block0 + blockIdx.x < s.num) {
    // what is wrong with the call's sequences, a workgroup each (and those behind the
    // last workgroup: the launch has as many as there are sequences at least)
    if (tid < 64) {
      const int i = (int)(block0 + blockIdx.x);
      const CacheSeq cs = cache_seq(c, s, i, tid == 0);
      if (WRITE && cs.n && s.slots) report_shared_slot(s, i, cs.slot, tid);
    }
  }
  if (t >= s.rows) return;
  while (q < s.num && s.off[q + 1] <= t) ++q;
  if (q >= s.num) return;
  const CacheSeq cs = cache_seq(c, s, q, false);
  if (!cs.n || t < cs.begin) return;
  const int pos = cs.past + (t - cs.begin);
  const int page = page_of(c, cs.slot, pos);
  if (page < 0) {
    record_err(s.status, err_key(kPhSeq, 0, 0, (uint32_t)q, kSqPage));
    return;
  }
  int in_row = (int)(at + tid - (int64_t)t * per_row);
  const int kind = in_row >= per_row / 2;
  in_row -= kind * (per_row / 2);
  const int head = in_row / per_head, u = in_row - head * per_head;
  const size_t region = region_of(c, page, kind, head) << c.page_shift;
  const size_t in_page = pos & ((1 << c.page_shift) - 1);
  uint8_t* const codes = c.codes + region * L::row;
  uint8_t* const scales = c.scales + region * NB;
  uint8_t* const scale = scales + (kind ? L::value_scale(in_page, u >> 2) : L::key_scale(in_page, u >> 2));
  T* const x = static_cast<T*>(kind ? r.v : r.k) + (int64_t)t * (kind ? r.v_stride : r.k_stride) +
               head * (kind ? r.v_head_stride : r.k_head_stride) + 8 * u;
  if constexpr (WRITE) {
    float f[8];
    load_f32<8>(x, f);
    uint32_t most = 0;  // as bits: a NaN is larger than any number
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, f2u(f[i]) & 0x7FFFFFFFu);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1));
    most = max(most, (uint32_t)__shfl_xor((int)most, 2));
    // 2^X with |x| <= 7 * 2^X: X = floor(log2) - 2, or one more above 1.75 * 2^floor
    const int e = (int)(most >> 23) - 2 + ((most & 0x7FFFFFu) > 0x600000u);
    const bool finite = most < 0x7F800000u;
    const uint32_t byte = finite ? (uint32_t)min(max(e, 7), 252) : 255u;
    const float unit = u2f((finite ? byte : 127u) << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], unit, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], unit, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], unit, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], unit, 3);
    w = finite ? w : 0u;
    if (kind) store_value<NB>(codes, in_page, u, w);
    else *reinterpret_cast<uint32_t*>(codes + L::key_word(in_page, u)) = w;
    if ((u & 3) == 0) *scale = (uint8_t)byte;
  } else {
    const uint32_t w = kind ? load_value<NB>(codes, in_page, u)
                            : *reinterpret_cast<const uint32_t*>(codes + L::key_word(in_page, u));
    const uint32_t unit = (uint32_t)*scale << 23;
    const uint32_t p[4] = {held_pair<0>(w, unit), held_pair<1>(w, unit), held_pair<2>(w, unit),
                           held_pair<3>(w, unit)};
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16lo(p[i]);
      f[2 * i + 1] = bf16hi(p[i]);
    }
    store_f32<8>(x, f);
  }
}

template <bool WRITE>
hipError_t run(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s, hipStream_t st) {
  return with_type(r.dtype, [&](auto t) {
    return with_blocks(c.dim, [&](auto nb) {
      using T = decltype(t);
      constexpr int NB = decltype(nb)::value;
      const int64_t threads = (int64_t)s.rows * 2 * c.kv_heads * 4 * NB;
      const int64_t blocks = std::max<int64_t>((threads + 255) / 256, s.num);
      constexpr int64_t most = 1 << 23;  // 2^31 threads a launch
      for (int64_t b = 0; b < blocks; b += most)
        k_kv_rows<T, NB, WRITE><<<(unsigned)std::min(most, blocks - b), 256, 0, st>>>(
            cache_dev(c), r, s, b);
      return hipGetLastError();
    });
  });
}

}  // namespace

hipError_t launch_kv_write(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s,
                           hipStream_t st) {
  return run<true>(c, r, s, st);
}
hipError_t launch_kv_read(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s,
                          hipStream_t st) {
  return run<false>(c, r, s, st);
}

}  // namespace dm
