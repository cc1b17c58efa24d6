// dm_cache.hip -- rows of keys and values into the 4-bit cache and out of it.
//
// A thread takes 8 elements of one head's row, four threads a block of 32: they agree
// on its largest element and its scale, and each makes one word of codes.  The
// hardware converts both ways (round to nearest even, above 6 to 6).  A workgroup first
// finds where its rows lie in the cache, a chain of four loads one behind the other, and
// then has up to 16 words for each thread, two on their way at a time: bound by
// that chain for few rows (32 of 2 heads of 256: 5 us) and by bytes for many (16384 rows of 8
// heads of 128 in f16, 86 MB: 19 us, 4.5 TB/s; 25 where each word's place takes divisions, and
// 38 with one word a thread).  Four words on their way leave fewer waves a SIMD: 8192
// rows of 4 heads of 64, there and back, 14.2 us, and 12.9 with two.
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

// The size of the largest of eight elements, as fp32 bits: a NaN is larger than any number.
template <typename T>
__device__ __forceinline__ uint32_t largest(Vec<T, 8> raw) {
  if constexpr (sizeof(T) == 2) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const uint4 w = __builtin_bit_cast(uint4, raw);
    const auto size = [](uint32_t x) { return __builtin_bit_cast(u16x2, x & 0x7FFF7FFFu); };
    const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(size(w.x), size(w.y)),
                                              __builtin_elementwise_max(size(w.z), size(w.w)));
    return f2u((float)__builtin_bit_cast(T, m.x > m.y ? m.x : m.y));
  } else {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, f2u(raw[i]) & 0x7FFFFFFFu);
    return most;
  }
}

// Eight elements of a row and their place in the cache.
template <typename T, int NB>
struct Word {
  using L = CacheLay<NB>;
  T* x;
  uint8_t *codes, *scale;
  size_t pos;
  int u;
  bool value, in;  // in: there is such a row
  __device__ __forceinline__ Word() {}
  // in_row: words of keys of all heads, then of values.
  __device__ __forceinline__ Word(const CacheDev& c, const dmh_kv_rows& r, int t, int in_row, int page,
                                  int pos)
      : in(true) {
    const int half = c.heads * 4 * NB;
    value = in_row >= half;
    in_row -= value ? half : 0;
    const int head = in_row / (4 * NB);
    u = in_row - head * (4 * NB);
    place(c, region_of(c, page, value, head) << c.page_shift, pos);
    x = row(r, t, head);
  }
  __device__ __forceinline__ T* row(const dmh_kv_rows& r, int t, int head) const {
    return static_cast<T*>(value ? r.v : r.k) + (int64_t)t * (value ? r.v_stride : r.k_stride) +
           head * (value ? r.v_head_stride : r.k_head_stride) + 8 * u;
  }
  // region: the tokens in front of a page's of this head.
  __device__ __forceinline__ void place(const CacheDev& c, size_t region, int at) {
    pos = at;
    codes = c.codes + region * L::row;
    scale = c.scales + region * NB + (value ? L::value_scale(pos, u >> 2) : L::key_scale(pos, u >> 2));
  }
  // (four lanes with the words of one block together)
  __device__ __forceinline__ void write(Vec<T, 8> raw) const {
    float f[8];
    to_f32<8>(raw, f);
    uint32_t most = largest<T>(raw);
    most = max(most, (uint32_t)__shfl_xor((int)most, 1));
    most = max(most, (uint32_t)__shfl_xor((int)most, 2));
    // 2^X with |x| <= 7 * 2^X: X = floor(log2) - 2, or one more above 1.75 * 2^floor
    const int e = (int)(most >> 23) - 2 + ((most & 0x7FFFFFu) > 0x600000u);
    const bool finite = most < 0x7F800000u;
    const uint32_t byte = finite ? (uint32_t)min(max(e, 7), 252) : 255u;
    const float unit = u2f((finite ? byte : 127u) << 23);
    uint32_t z = 0;
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, f[0], f[1], unit, 0);
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, f[2], f[3], unit, 1);
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, f[4], f[5], unit, 2);
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, f[6], f[7], unit, 3);
    z = finite ? z : 0u;
    if (!in) return;
    if (value) store_value<NB>(codes, pos, u, z);
    else *reinterpret_cast<uint32_t*>(codes + L::key_word(pos, u)) = z;
    if ((u & 3) == 0) *scale = (uint8_t)byte;
  }
  __device__ __forceinline__ void fetch(uint32_t& z, uint32_t& unit) const {
    z = unit = 0;
    if (!in) return;
    z = value ? load_value<NB>(codes, pos, u)
              : *reinterpret_cast<const uint32_t*>(codes + L::key_word(pos, u));
    unit = (uint32_t)*scale << 23;
  }
  // PAST: past the L2, which many rows would fill.
  template <bool PAST>
  __device__ __forceinline__ void read(uint32_t z, uint32_t unit) const {
    if (!in) return;
    const uint32_t p[4] = {held_pair<0>(z, unit), held_pair<1>(z, unit), held_pair<2>(z, unit),
                           held_pair<3>(z, unit)};
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16lo(p[i]);
      f[2 * i + 1] = bf16hi(p[i]);
    }
    if constexpr (PAST) {
      Vec<T, 8> v;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
      __builtin_nontemporal_store(v, reinterpret_cast<Vec<T, 8>*>(x));
    } else {
      store_f32<8>(x, f);
    }
  }
};

constexpr int kMostWords = 16;                        // of a thread
constexpr int kMostRows = 4 * kMostWords * 8;  // of a workgroup: four rows have 32 words or more

// A thread has the same word of every fourth row, so that only the page changes from one to
// the next; the words of one head in four rows lie together, whose values are one piece of
// the cache.  Where four rows have fewer than 256 words, `side` of them lie side by side;
// where they have more, `chunks` workgroups share them.
template <typename T, int NB, bool WRITE>
__global__ __launch_bounds__(256) void k_kv_rows(CacheDev c, dmh_kv_rows r, SeqDev s, int words, int side,
                                                 int chunks, int64_t block0) {
  const int tid = threadIdx.x;
  const int per_four = 4 * 2 * c.heads * 4 * NB;
  const int64_t block = block0 + blockIdx.x;
  const int64_t rows_at = block / chunks;
  const int chunk = (int)(block - rows_at * chunks);
  // (fewer than 2^30 rows)
  const int t0 = (int)least(rows_at * (4 * words * side), s.rows);
  const int t1 = (int)least((int64_t)t0 + 4 * words * side, s.rows);

  __shared__ int found;
  __shared__ struct { int begin, end, past, slot, seq; } part[kMostRows];
  __shared__ int page_of_row[kMostRows], pos_of_row[kMostRows];
  if (tid == 0) found = 0;
  if (block < s.num && tid < 64) {
    // what is wrong with the call's sequences, a workgroup each
    const CacheSeq q = cache_seq(c, s, (int)block, tid == 0);
    if (WRITE && q.n && s.slots) report_shared_slot(s, (int)block, q.slot, tid);
  }
  __syncthreads();
  // the sequences with rows here
  for (int i = tid; i < s.num; i += 256) {
    if (s.off[i] >= t1 || s.off[i + 1] <= t0) continue;
    const CacheSeq q = cache_seq(c, s, i, false);
    if (!q.n) continue;
    // (ones that overlap, which nothing is said about, may be more than there is room for)
    const int at = atomicAdd(&found, 1);
    if (at < kMostRows) part[at] = {q.begin, q.begin + q.n, q.past, q.slot, i};
  }
  __syncthreads();
  const int parts = min(found, kMostRows);
  for (int t = t0 + tid; t < t1; t += 256) {
    int page = -1, pos = 0;
    for (int i = 0; i < parts; ++i) {
      if (t < part[i].begin || t >= part[i].end) continue;
      pos = part[i].past + (t - part[i].begin);
      page = page_of(c, part[i].slot, pos);
      if (page < 0) record_err(s.status, err_key(kPhSeq, 0, 0, (uint32_t)part[i].seq, kSqPage));
      break;
    }
    page_of_row[t - t0] = page;
    pos_of_row[t - t0] = pos & ((1 << c.page_shift) - 1);
  }
  __syncthreads();

  const int at = chunk * 256 + tid, beside = at / per_four, in_four = at - beside * per_four;
  const int in_head = in_four % (4 * 4 * NB), mine = 4 * beside + in_head / (4 * NB);
  Word<T, NB> first;
  int head = in_four / (4 * 4 * NB);
  first.value = head >= c.heads;
  const size_t head_at = (size_t)head << c.page_shift, page_tokens = (size_t)(2 * c.heads) << c.page_shift;
  head -= first.value ? c.heads : 0;
  first.u = in_head % (4 * NB);
  const int64_t step = 4 * side * (first.value ? r.v_stride : r.k_stride);
  first.x = first.row(r, t0 + mine, head);
  const auto word = [&](int k) {
    Word<T, NB> w = first;
    const int row = mine + 4 * side * k;
    w.in = beside < side && k < words && t0 + row < t1 && page_of_row[row] >= 0;
    const int from = w.in ? row : 0;
    w.place(c, (w.in ? page_of_row[from] : 0) * page_tokens + head_at, pos_of_row[from]);
    w.x = first.x + k * step;
    return w;
  };
  constexpr int B = 2;
  for (int k0 = 0; k0 < words; k0 += B) {
    Word<T, NB> w[B];
#pragma unroll
    for (int b = 0; b < B; ++b) w[b] = word(k0 + b);
    if constexpr (WRITE) {
      Vec<T, 8> raw[B];
#pragma unroll
      for (int b = 0; b < B; ++b) raw[b] = w[b].in ? load_raw<8>(w[b].x) : Vec<T, 8>{};
#pragma unroll
      for (int b = 0; b < B; ++b) w[b].write(raw[b]);
    } else {
      uint32_t z[B], unit[B];
#pragma unroll
      for (int b = 0; b < B; ++b) w[b].fetch(z[b], unit[b]);
#pragma unroll
      for (int b = 0; b < B; ++b) w[b].template read<true>(z[b], unit[b]);
    }
  }
}

// The same with one word a thread, each of which finds its own row: no way through LDS.
template <typename T, int NB, bool WRITE>
__global__ __launch_bounds__(256) void k_kv_few(CacheDev c, dmh_kv_rows r, SeqDev s) {
  const int tid = threadIdx.x;
  const uint32_t per_row = 2 * c.heads * 4 * NB;
  const uint32_t i = blockIdx.x * 256 + tid;  // (2^20 at most)
  const int t0 = min((int)(blockIdx.x * 256 / per_row), s.rows);
  const int t = min((int)(i / per_row), s.rows);

  // the first sequence with a row at t0 or behind it, then this row's
  __shared__ int first_seq;
  if (tid == 0) first_seq = s.num;
  __syncthreads();
  int j0 = tid;
  while (j0 < s.num && s.off[j0 + 1] <= t0) j0 += 256;
  if (j0 < s.num) atomicMin(&first_seq, j0);
  __syncthreads();
  int q = first_seq;
  if ((int)blockIdx.x < s.num && tid < 64) {
    const CacheSeq cs = cache_seq(c, s, blockIdx.x, tid == 0);
    if (WRITE && cs.n && s.slots) report_shared_slot(s, blockIdx.x, cs.slot, tid);
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
  const Word<T, NB> w(c, r, t, (int)(i - t * per_row), page,
                      pos & ((1 << c.page_shift) - 1));
  if constexpr (WRITE) {
    w.write(load_raw<8>(w.x));
  } else {
    uint32_t z, unit;
    w.fetch(z, unit);
    w.template read<false>(z, unit);
  }
}

template <bool WRITE>
hipError_t run(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s, hipStream_t st) {
  return with_type(r.dtype, [&](auto t) {
    return with_blocks(c.dim, [&](auto nb) {
      using T = decltype(t);
      constexpr int NB = decltype(nb)::value;
      const int64_t per_row = 2 * c.kv_heads * 4 * NB, all = s.rows * per_row;  // words
      // as many to a thread as leave four workgroups a CU (32 rows of 2 heads of 256: 4.4 us
      // with none, which the first kernel does in 6.5)
      const int words = (int)std::min<int64_t>(kMostWords, all / (256 * 1024));
      if (words == 0 && s.num < 4096) {
        const int64_t blocks = std::max<int64_t>((all + 255) / 256, s.num);
        k_kv_few<T, NB, WRITE><<<(unsigned)blocks, 256, 0, st>>>(cache_dev(c), r, s);
        return hipGetLastError();
      }
      const int some = std::max(words, 1), per_four = (int)(4 * per_row);
      const int side = std::max(256 / per_four, 1), chunks = (per_four + 255) / 256;
      const int64_t blocks =
          std::max<int64_t>((s.rows + (int64_t)(4 * some * side) - 1) / (4 * some * side) * chunks, s.num);
      constexpr int64_t most = 1 << 23;  // 2^31 threads a launch
      for (int64_t b = 0; b < blocks; b += most)
        k_kv_rows<T, NB, WRITE><<<(unsigned)std::min(most, blocks - b), 256, 0, st>>>(
            cache_dev(c), r, s, some, side, chunks, b);
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
