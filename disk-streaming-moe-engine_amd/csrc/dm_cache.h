// dm_cache.h -- the 4-bit cache of keys and values: where its bytes lie, and the
// host-side launchers of the kernels on it (dm_cache.hip, dm_attend.hip).
//
// Every array is device memory; sizes, strides and alignment have been checked
// (dm_cache_api.cpp).  Sequences and pages are checked by the kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "dm_layout.h"
#include "dm_mixer.h"

namespace dm {

constexpr int kBlock = 32;  // elements of one scale

// A region holds one head's keys or values of a page.  Attention takes 32 tokens at a
// time as operands of v_mfma_f32_16x16x32_bf16, whose lane (n = lane % 16, quad =
// lane / 16) gives 8 values of the summed index.  The bytes lie so that a lane's words
// for that are next to each other and a wave reads a region from end to end:
//
// Keys (summed over elements; lane n: token n of 16): a token's NB = dim / 32 words of
// quad 0, those of quad 1, ...; word j of quad u has the elements 32 j + 8 u + 0 .. 7.
// Scales: a token's NB bytes.
//
// Values (summed over tokens; lane n: elements): for each four tokens, lane n's 4 NB
// bytes, NB of each token.  Where NB is a power of two byte b of lane n has the elements
// 2 NB n + 2 b + 0, 1, all of one scale; else 32 b + 2 n + 0, 1, of scale b.  Quad u
// takes the tokens 4 u + 0 .. 3 of two 16s.  Scales: for each four tokens, 4 bytes of
// scale 0, 4 of scale 1, ...
//
// The first of two elements is the low half of a byte.
template <int NB>
struct CacheLay {
  static constexpr int dim = kBlock * NB;
  static constexpr bool pow2 = (NB & (NB - 1)) == 0;
  static constexpr int row = dim / 2;  // bytes of codes per token
  // the word with the elements 8 u .. 8 u + 7 of a key
  DM_HD static size_t key_word(size_t pos, int u) { return pos * row + ((u & 3) * NB + (u >> 2)) * 4; }
  DM_HD static size_t key_scale(size_t pos, int j) { return pos * NB + j; }
  DM_HD static size_t value_byte(size_t pos, int lane, int b) {
    return (pos >> 2) * (4 * row) + lane * (4 * NB) + (pos & 3) * NB + b;
  }
  DM_HD static size_t value_scale(size_t pos, int j) {
    return (pos >> 2) * (4 * NB) + j * 4 + (pos & 3);
  }
};

// The cache on the device.
struct CacheDev {
  int heads, page_shift, num_pages, max_pages;
  uint8_t* codes;
  uint8_t* scales;
  const int32_t* pages;
  const int32_t* past;
};
inline CacheDev cache_dev(const dmh_kv_cache& c) {
  return {c.kv_heads, __builtin_ctz((unsigned)c.page_size), c.num_pages, c.max_pages,
          c.codes,    c.scales, c.pages, c.past};
}

// Calls f with the number of scales of a row as a compile-time value.
template <typename F>
hipError_t with_blocks(int dim, F f) {
  switch (dim / kBlock) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 6: return f(std::integral_constant<int, 6>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}

hipError_t launch_kv_write(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s,
                           hipStream_t st);
hipError_t launch_kv_read(const dmh_kv_cache& c, const dmh_kv_rows& r, const SeqDev& s,
                          hipStream_t st);

// Attention; ws: attend_bytes of device memory.  attend_fits: whether a launch holds the
// call's work.
bool attend_fits(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s);
size_t attend_bytes(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s);
hipError_t launch_attend(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s, void* ws,
                         hipStream_t st);

}  // namespace dm
