// dm_attend.hip -- causal attention over the 4-bit cache.
//
// A unit is one key head of a sequence with up to 16 MT of its query rows (a row is one
// token and one of the R query heads that share the key head).  A wave takes 32
// tokens of the context a step:
//   S^T = K Q^T   on the matrix cores; the codes become bf16 in registers, exactly
//   P   = e^(scale (S - m)) with m the running maximum of each row
//   O^T += V^T P^T
// With S and O transposed, lane (n, quad) holds row n of S for tokens 4 quad .. + 3
// and 16 + 4 quad .. + 3, which is what the second product takes from it: P passes
// through no other lane, and each row's maximum and factor lie in its own lanes.
//
// What is rounded: queries of 16 or 32 bits enter as one to three bf16 parts that hold
// all of them, P as two parts (16 bits of it) for rows of 16 bits and three (24) for
// fp32; sums and maxima are fp32.
#include <algorithm>
#include <type_traits>

#include "dm_attend_walk.h"
#include "dm_cache_device.h"

namespace dm {
namespace {

template <typename F>
hipError_t with_type(int dtype, F f) {
  if (dtype == DMH_DTYPE_BF16) return f(bf16_t{});
  if (dtype == DMH_DTYPE_F16) return f(half_t{});
  return f(float{});
}

// A matrix product's result may be read only some cycles after its issue; the compiler
// counts instructions for that, but not across the end of a loop.
template <int A, int B>
__device__ __forceinline__ void settle(f32x4 (&c)[A][B]) {
#pragma unroll
  for (int i = 0; i < A * B; ++i) asm volatile("" : "+v"(c[i / B][i % B]));
  asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c[0][0]));
#pragma unroll
  for (int i = 0; i < A * B; ++i) asm volatile("" : "+v"(c[i / B][i % B]));
}

constexpr int kStep = 32;   // tokens of a step
constexpr int kTile = 128;  // tokens of a step of four waves
constexpr float kNone = -3.40282347e38f;  // the maximum of a row that has seen no token: no score is less

// What k_attend_few leaves to k_attend_join of a unit.
struct Meta {
  int group, parts, place;  // the first workgroup with a part, how many, and that one's place
  int begin, n;             // the sequence's rows
  int head, block, pad;     // (of k_attend_many's units)
};

struct AttendDev {
  dmh_attention a;
  CacheDev c;
  SeqDev s;
  int rep;       // query heads per key head
  int few_rows;  // sequences of up to so many rows are k_attend_few's
  int blocks;    // row blocks of a unit there, at most
  float c2;      // scale * log2(e)
  float* part;   // the workgroups' unfinished units
  struct Meta* meta;  // by unit
};

// N words at any word's address.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t u2v __attribute__((ext_vector_type(2), aligned(4)));
  int i = 0;
#pragma unroll
  for (; i + 4 <= N; i += 4) {
    const u4 v = *reinterpret_cast<const u4*>(p + 4 * i);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i + j] = v[j];
  }
  if (N % 4 >= 2) {
    const u2v v = *reinterpret_cast<const u2v*>(p + 4 * i);
    w[i] = v[0];
    w[i + 1] = v[1];
    i += 2;
  }
  if (N % 2) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
}
// NB bytes at a multiple of their number (of 16 bytes that belong to the same array).
template <int NB>
__device__ __forceinline__ void load_scales(const uint8_t* p, uint32_t (&w)[(NB + 3) / 4]) {
  if constexpr (NB == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else if constexpr (NB == 6) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    w[0] = h[0] | (uint32_t)h[1] << 16;
    w[1] = h[2];
  } else if constexpr (NB == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (NB == 3) {
    w[0] = p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16;
  } else if constexpr (NB == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
    w[0] = p[0];
  }
}
// Byte i of a word in the place of an exponent: the conversions look at nothing else of a
// scale.
__device__ __forceinline__ uint32_t exponent(uint32_t w, int i) {
  return i == 3 ? w >> 1 : w << (23 - 8 * i);
}

__device__ __forceinline__ float max_quads(float x) {
  const auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
  auto p = __builtin_amdgcn_permlane16_swap(bits(x), bits(x), false, false);
  x = fmaxf(u2f(p[0]), u2f(p[1]));
  p = __builtin_amdgcn_permlane32_swap(bits(x), bits(x), false, false);
  return fmaxf(u2f(p[0]), u2f(p[1]));
}
__device__ __forceinline__ float sum_quads(float x) {
  const auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
  auto p = __builtin_amdgcn_permlane16_swap(bits(x), bits(x), false, false);
  x = u2f(p[0]) + u2f(p[1]);
  p = __builtin_amdgcn_permlane32_swap(bits(x), bits(x), false, false);
  return u2f(p[0]) + u2f(p[1]);
}

// x as PARTS bf16 values whose sum it is, to 8 bits each.  (The first of three is cut off, not
// rounded: the largest fp32 values have no bf16 above them.)
template <int PARTS>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&out)[PARTS]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = PARTS == 3 && p == 0 ? f2u(r[2 * i]) >> 16 | (f2u(r[2 * i + 1]) & 0xFFFF0000u)
                                  : pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (p + 1 < PARTS) {
        r[2 * i] -= bf16lo(w[i]);
        r[2 * i + 1] -= bf16hi(w[i]);
      }
    }
    out[p] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// The same of probabilities: what a part leaves comes from one product of two with -1 and 0
// instead of a conversion and a difference for each, which is the same value (NaN in one
// of two tokens makes the row NaN in any case).  2048 rows 120 -> 118 us,
// ragged prompts 1015 -> 988.
template <int PARTS>
__device__ __forceinline__ void split_p(float (&r)[8], bf16x8 (&out)[PARTS]) {
  uint32_t first = 0x0000BF80u, second = 0xBF800000u;  // (as literals they are encoded wrong)
  asm("" : "+s"(first), "+s"(second));
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
      if (p + 1 < PARTS) {
        const bf16x2 h = __builtin_bit_cast(bf16x2, w[i]);
        r[2 * i] = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), r[2 * i], false);
        r[2 * i + 1] =
            __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), r[2 * i + 1], false);
      }
    }
    out[p] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Where a unit's bytes lie.  All of it is the same in a wave: addresses are a scalar base
// and the lane's own 32 bits.
template <int NB>
struct Unit {
  const uint8_t *codes, *scales;
  const int32_t* table;  // the slot's pages
  size_t page_bytes, head_bytes, value_bytes;  // of codes; scales have a 16th
  int shift, num_pages, len;
  bool bad;  // a page was not one of the cache's
  __device__ __forceinline__ void begin(const AttendDev& d, const CacheSeq& s, int h) {
    codes = d.c.codes;
    scales = d.c.scales;
    table = d.c.pages + (int64_t)s.slot * d.c.max_pages;
    shift = d.c.page_shift;
    value_bytes = ((size_t)d.c.heads << shift) * (16 * NB);
    page_bytes = 2 * value_bytes;
    head_bytes = ((size_t)h << shift) * (16 * NB);
    num_pages = d.c.num_pages;
    len = s.past + s.n;
    bad = false;
  }
  // The page of a position, the same in all lanes (at() sees to that: here it would wait for
  // this load and the codes' before it).
  __device__ __forceinline__ int page(int t) const { return table[min(t, len - 1) >> shift]; }
  // The keys' codes of position t, in page p.
  __device__ __forceinline__ size_t at(int p, int t) {
    p = __builtin_amdgcn_readfirstlane(p);
    if ((unsigned)p >= (unsigned)num_pages) {
      bad = true;
      p = 0;
    }
    return p * page_bytes + head_bytes + (size_t)(t & ((1 << shift) - 1)) * (16 * NB);
  }
};

// Scales of the values of four tokens (a byte each) without those behind the last token.
__device__ __forceinline__ uint32_t present(uint32_t x, int left) {
  return left >= 4 ? x : left <= 0 ? 0u : x & ((1u << (8 * left)) - 1);
}
// Whether a byte is 255, and the word with such bytes 0.
__device__ __forceinline__ bool any_nan(uint32_t x) {
  const uint32_t y = ~x;
  return ((y - 0x01010101u) & ~y & 0x80808080u) != 0;
}
__device__ __forceinline__ uint32_t no_nan(uint32_t x) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((x >> (8 * e) & 0xFFu) == 0xFFu) x &= ~(0xFFu << (8 * e));
  return x;
}
// 1.0 for each NaN of the eight tokens whose scales two words hold, as an operand.
__device__ __forceinline__ bf16x8 nan_marks(uint32_t x0, uint32_t x1) {
  uint32_t mark[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = (e < 2 ? x0 : x1) >> (16 * (e % 2));
    mark[e] = ((x & 0xFFu) == 0xFFu ? 0x3F80u : 0u) | ((x & 0xFF00u) == 0xFF00u ? 0x3F800000u : 0u);
  }
  return __builtin_bit_cast(bf16x8, make_uint4(mark[0], mark[1], mark[2], mark[3]));
}

// One word of a key's codes as an operand.
__device__ __forceinline__ bf16x8 key_operand(uint32_t c, uint32_t scale) {
  return __builtin_bit_cast(bf16x8, make_uint4(held_pair<0>(c, scale), held_pair<1>(c, scale),
                                               held_pair<2>(c, scale), held_pair<3>(c, scale)));
}
// A row of the results: where it goes, its gate's place and the factor 1 / l.
template <typename T>
struct Result {
  const T* gate;
  T* o;
  float f;
  __device__ __forceinline__ Result(const AttendDev& d, const CacheSeq& s, int h, int row, float l) {
    const int t = row / d.rep, hq = h * d.rep + (row - t * d.rep);
    const int64_t tok = s.begin + t;
    gate = d.a.gate ? static_cast<const T*>(d.a.gate) + tok * d.a.gate_stride + hq * d.a.gate_head_stride
                    : nullptr;
    o = static_cast<T*>(d.a.o) + tok * d.a.o_stride + hq * d.a.o_head_stride;
    f = 1.0f / l;
  }
  __device__ __forceinline__ Vec<T, 4> gates(int e0) const {
    return gate ? load_raw<4>(gate + e0) : Vec<T, 4>{};
  }
  __device__ __forceinline__ void store(int e0, const float (&v)[4], Vec<T, 4> g) const {
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = v[e] * f;
    if (gate) {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] *= sigmoid_all((float)g[e]);
    }
    store_f32<4>(o + e0, r);
  }
};

// The JG j from j0 on of a row's outputs that this lane holds, in runs of four elements;
// all of their gates are requested before the first is used.
template <typename T, int NB, int JG>
__device__ __forceinline__ void store_lane(int quad, int j0, const f32x4 (&o)[JG],
                                           const Result<T>& out) {
  constexpr bool pow2 = CacheLay<NB>::pow2, runs = pow2 && NB >= 2;
  const auto place = [&](int i) {  // of run i: four j of one e, or two j of two e
    const int j = j0 + (runs ? i % (JG / 4) * 4 : i % (JG / 2) * 2);
    const int e = runs ? i / (JG / 4) : i / (JG / 2) * 2;
    return pow2 ? (4 * quad + e) * 2 * NB + j : 32 * (j / 2) + 8 * quad + 2 * e + j % 2;
  };
  Vec<T, 4> gate[JG] = {};
  if (out.gate) {
#pragma unroll
    for (int i = 0; i < JG; ++i) gate[i] = load_raw<4>(out.gate + place(i));
  }
#pragma unroll
  for (int i = 0; i < JG; ++i) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = runs ? o[i % (JG / 4) * 4 + k][i / (JG / 4)]
                  : o[i % (JG / 2) * 2 + k % 2][i / (JG / 2) * 2 + k / 2];
    out.store(place(i), v, gate[i]);
  }
}

// 16 MT rows of a unit on their way through the context: queries, running maxima and
// sums, and outputs.
template <typename T, int NB, int MT>
struct Wave {
  using L = CacheLay<NB>;
  static constexpr int QP = std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, half_t>::value ? 2 : 3;
  static constexpr int PP = std::is_same<T, float>::value ? 3 : 2;
  bf16x8 q[MT][QP][NB];
  f32x4 o[MT][2 * NB];
  float m[MT], l[MT];  // m of scores before they are scaled; l of this lane's tokens
  int seen[MT];        // the last position that the row sees, -1: no such row

  // Rows row0 .. row0 + 16 MT - 1 of the sequence's n * rep.
  __device__ __forceinline__ void begin(const AttendDev& d, const CacheSeq& s, int h, int row0) {
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int row = row0 + 16 * i + n, t = row / d.rep;
      const bool in = t < s.n;
      seen[i] = in ? s.past + t : -1;
      m[i] = kNone;
      l[i] = 0.0f;
      const T* p = static_cast<const T*>(d.a.q) + (int64_t)(s.begin + (in ? t : 0)) * d.a.q_stride +
                   (int64_t)(h * d.rep + (in ? row - t * d.rep : 0)) * d.a.q_head_stride + 8 * quad;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float f[8];
        bf16x8 w[QP];
        load_f32<8>(p + 32 * j, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = in ? f[e] : 0.0f;
        split<QP>(f, w);
#pragma unroll
        for (int e = 0; e < QP; ++e) q[i][e][j] = w[e];
      }
#pragma unroll
      for (int j = 0; j < 2 * NB; ++j) o[i][j] = f32x4{};
    }
  }

  // The 16 TILES tokens from t0 on.  MASK: some row does not see some of them.
  //   key(a, j)                  operand j of the keys of the a-th 16 tokens
  //   value(g, b, first, second) operands of elements 2 b and 2 b + 1 of the values of the
  //                              g-th 32 tokens
  //   nan, marks(g, b)           whether a value is held as NaN, and which: such a value would
  //                              reach the rows that do not see it (0 * NaN), so it enters as
  //                              0, and rows that see it are made NaN behind the products
  template <bool MASK, int TILES, typename K, typename V, typename M>
  __device__ __forceinline__ void step(float c2, int t0, K key, V value, bool nan, M marks) {
    const int quad = (threadIdx.x & 63) >> 4;
    f32x4 s[MT][TILES];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int a = 0; a < TILES; ++a) s[i][a] = f32x4{};
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      bf16x8 k[TILES];
#pragma unroll
      for (int a = 0; a < TILES; ++a) k[a] = key(a, j);
#pragma unroll
      for (int e = 0; e < QP; ++e)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int a = 0; a < TILES; ++a) s[i][a] = mfma16(k[a], q[i][e][j], s[i][a]);
    }
    bf16x8 p[MT][TILES / 2][PP];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float most = -__builtin_inff();
#pragma unroll
      for (int a = 0; a < TILES; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (MASK && t0 + 16 * a + 4 * quad + e > seen[i]) s[i][a][e] = -__builtin_inff();
          most = fmaxf(most, s[i][a][e]);
        }
      const float now = fmaxf(m[i], max_quads(most));
      if (__any(now != m[i])) {
        const float f = __builtin_amdgcn_exp2f((m[i] - now) * c2);
        l[i] *= f;
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) o[i][j] *= f;
        m[i] = now;
      }
#pragma unroll
      for (int g = 0; g < TILES / 2; ++g) {
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // (the difference first: the largest score's is 0 at any size, where a product's
          // remainder would be more than fp32's exponents from 2^31 on)
          z[e] = __builtin_amdgcn_exp2f((s[i][2 * g + e / 4][e % 4] - now) * c2);
          l[i] += z[e];
        }
        split_p<PP>(z, p[i][g]);
      }
    }
    if (nan) {
#pragma unroll
      for (int g = 0; g < TILES / 2; ++g)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const bf16x8 a = marks(g, b);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t v[4];  // 1.0 of each token that the row sees
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = t0 + 32 * g + 16 * (e / 2) + 4 * quad + e % 2 * 2;
              v[e] = MASK ? (t <= seen[i] ? 0x3F80u : 0u) | (t + 1 <= seen[i] ? 0x3F800000u : 0u)
                          : 0x3F803F80u;
            }
            const f32x4 hit = mfma16(
                a, __builtin_bit_cast(bf16x8, make_uint4(v[0], v[1], v[2], v[3])), f32x4{});
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float add = hit[e] > 0.0f ? __builtin_nanf("") : 0.0f;
              o[i][2 * b][e] += add;
              o[i][2 * b + 1][e] += add;
            }
          }
        }
    }
#pragma unroll
    for (int g = 0; g < TILES / 2; ++g)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        bf16x8 v[2];
        value(g, b, v[0], v[1]);
#pragma unroll
        for (int e = 0; e < PP; ++e)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < MT; ++i)
              o[i][2 * b + half] = mfma16(v[half], p[i][g][e], o[i][2 * b + half]);
      }
  }

  __device__ __forceinline__ void results(int i, const Result<T>& out) const {
    store_lane<T, NB, 2 * NB>((threadIdx.x & 63) >> 4, 0, o[i], out);
  }

  // Element of o[i][j][e].
  __device__ __forceinline__ static int elem(int quad, int j, int e) {
    return L::pow2 ? (4 * quad + e) * 2 * NB + j : 32 * (j / 2) + 8 * quad + 2 * e + j % 2;
  }
};

// The codes and scales of 32 tokens, as they come.
template <int NB>
struct Held {
  using L = CacheLay<NB>;
  static constexpr int VS = L::pow2 ? 1 : NB;
  uint32_t k[2][NB], v[2][NB], ks[2][(NB + 3) / 4], vs[2][VS];

  __device__ __forceinline__ void load(Unit<NB>& u, int t0, int p0, int p1) {
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      // (the second 16 may lie behind the last page: those of the first are read again)
      const size_t at = u.at(a ? p1 : p0, t0 + 16 * a < u.len ? t0 + 16 * a : t0);
      load_words<NB>(u.codes + at + (unsigned)(n * L::row + quad * NB * 4), k[a]);
      load_words<NB>(u.codes + at + u.value_bytes + (unsigned)(quad * (4 * L::row) + n * (4 * NB)), v[a]);
      load_scales<NB>(u.scales + at / 16 + (unsigned)(n * NB), ks[a]);
      load_value_scales(u, at, vs[a]);
    }
  }
  __device__ __forceinline__ static void load_value_scales(const Unit<NB>& u, size_t at,
                                                           uint32_t (&x)[VS]) {
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
    const uint8_t* const p = u.scales + (at + u.value_bytes) / 16;
    if constexpr (L::pow2)
      x[0] = *reinterpret_cast<const uint32_t*>(p + (unsigned)(quad * (4 * NB) + n * NB / 16 * 4));
    else load_words<VS>(p + (unsigned)(quad * (4 * NB)), x);
  }
};

// Steps t0, t0 + stride, ... below end, straight from memory, the next step's bytes on
// their way.
template <typename T, int NB, int MT>
__device__ __forceinline__ void run_steps(Wave<T, NB, MT>& w, Unit<NB>& u, float c2, int t0, int end,
                                          int stride, int past) {
  using H = Held<NB>;
  const int quad = (threadIdx.x & 63) >> 4;
  if (t0 >= end) return;
  H next;
  next.load(u, t0, u.page(t0), u.page(t0 + 16));
  int p0 = u.page(t0 + stride), p1 = u.page(t0 + stride + 16);
  // (steps that every row sees all of come first, in a loop of their own: as two ways in
  // one loop they took twice the registers)
  const auto one = [&](auto mask) {
    constexpr bool MASK = decltype(mask)::value;
    const H h = next;
    if (t0 + stride < end) {
      next.load(u, t0 + stride, p0, p1);
      p0 = u.page(t0 + 2 * stride);
      p1 = u.page(t0 + 2 * stride + 16);
    }
    uint32_t vs[2][H::VS], clean[2][H::VS];
    bool nan = false;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < H::VS; ++g) {
        vs[a][g] = MASK ? present(h.vs[a][g], u.len - (t0 + 16 * a + 4 * quad)) : h.vs[a][g];
        clean[a][g] = vs[a][g];
        nan = nan || any_nan(vs[a][g]);
      }
    nan = __any(nan);
    if (nan) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int g = 0; g < H::VS; ++g) clean[a][g] = no_nan(vs[a][g]);
    }
    uint32_t x[8];
    w.template step<MASK, 2>(
        c2, t0,
        [&](int a, int j) { return key_operand(h.k[a][j], exponent(h.ks[a][j / 4], j % 4)); },
        [&](int, int b, bf16x8& first, bf16x8& second) {
          uint32_t c[8];
          if (b == 0 || !H::L::pow2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = exponent(clean[e / 4][H::L::pow2 ? 0 : b], e % 4);
          }
          uint32_t pair[8], f[4], g[4];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = (e % 4) * NB + b;
            c[e] = h.v[e / 4][at / 4];
            pair[e] = at % 4 == 0 ? held_pair<0>(c[e], x[e]) : at % 4 == 1 ? held_pair<1>(c[e], x[e])
                      : at % 4 == 2 ? held_pair<2>(c[e], x[e]) : held_pair<3>(c[e], x[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x05040100u);
            g[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x07060302u);
          }
          first = __builtin_bit_cast(bf16x8, make_uint4(f[0], f[1], f[2], f[3]));
          second = __builtin_bit_cast(bf16x8, make_uint4(g[0], g[1], g[2], g[3]));
        },
        nan, [&](int, int b) { return nan_marks(vs[0][H::L::pow2 ? 0 : b], vs[1][H::L::pow2 ? 0 : b]); });
    t0 += stride;
  };
  while (t0 < end && t0 + kStep - 1 <= past) one(std::false_type{});
  while (t0 < end) one(std::true_type{});
  settle(w.o);
}

// ---- few rows: contexts divided over the workgroups -------------------------------------
// All tiles of 128 tokens of all units, one behind the other, are divided evenly over
// the workgroups, so that one long context and many short ones fill the device alike; a
// workgroup's four waves take the steps of its tiles in turn and join what they have
// through LDS.  A unit that lies in one workgroup is done there, others leave O, m and
// l of their parts for k_attend_join.
struct Share {
  int64_t total, lo, hi;  // tiles in all, this workgroup's
  int groups;
};
__device__ __forceinline__ int64_t share_at(int64_t total, int groups, int w) {
  return total / groups * w + total % groups * w / groups;
}

__device__ __forceinline__ int tiles_of(const AttendDev& d, const CacheSeq& q, int rows_per_block,
                                        int* blocks) {
  const int64_t rows = (int64_t)q.n * d.rep;
  if (!q.n || rows > d.few_rows) return *blocks = 0;
  *blocks = ((int)rows + rows_per_block - 1) / rows_per_block;
  return (q.past + q.n + kTile - 1) / kTile;
}

template <int D, int ROWS>
constexpr int part_floats() { return ROWS * (D + 2); }

// Waves a SIMD and workgroups a CU: three where the registers hold them (128 elements of bf16
// 134 -> 130 us, 64 102 -> 96; 128 of f16, whose queries take twice the registers, 38 -> 44).
template <typename T>
constexpr int few_waves(int dim, int mt) {
  return mt == 1 && (dim <= 64 || (dim <= 128 && std::is_same<T, bf16_t>::value)) ? 3 : 2;
}

template <typename T, int NB, int MT>
__global__ __launch_bounds__(256, few_waves<T>(32 * NB, MT)) void k_attend_few(AttendDev d) {
  using W = Wave<T, NB, MT>;
  constexpr int D = 32 * NB, ROWS = 16 * MT;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = blockIdx.x;

  __shared__ int64_t ends[256];  // tiles to the end of each of 256 sequences
  __shared__ CacheSeq seqs[256];
  __shared__ int64_t wsum[4];
  __shared__ float om[4][ROWS], ol[4][ROWS];
  __shared__ __align__(16) float oo[4][16][D + 4];

  // The tiles of 256 sequences from i0 on, summed up in ends; their sum.
  const auto count = [&](int i0) {
    CacheSeq q = {};
    int64_t mine = 0;
    if (i0 + tid < d.s.num) {
      q = cache_seq(d.c, d.s, i0 + tid, group == 0);
      int blocks;
      const int tiles = tiles_of(d, q, ROWS, &blocks);
      mine = (int64_t)tiles * blocks * d.c.heads;
      // (units that nobody works on, of which each call's other ones may have left something)
      if (group == 0)
        for (int u = 0; u < d.c.heads * d.blocks; ++u)
          if (u % d.blocks >= blocks) d.meta[(int64_t)(i0 + tid) * d.c.heads * d.blocks + u].parts = 0;
    }
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t x = __shfl_up(sum, o);
      if (lane >= o) sum += x;
    }
    __syncthreads();
    if (lane == 63) wsum[wave] = sum;
    seqs[tid] = q;
    __syncthreads();
    int64_t before = 0;
    for (int i = 0; i < wave; ++i) before += wsum[i];
    ends[tid] = before + sum;
    __syncthreads();
    return ends[255];
  };

  int64_t total = count(0);
  for (int i0 = 256; i0 < d.s.num; i0 += 256) total += count(i0);
  const int groups = (int)least(gridDim.x, total);
  if (group >= groups) return;
  const int64_t lo = share_at(total, groups, group), hi = share_at(total, groups, group + 1);
  int64_t base = 0, at = lo;
  int slot = 0;  // unfinished units of this workgroup so far
  for (int i0 = 0; i0 < d.s.num && at < hi; i0 += 256) {
    const int64_t sum = d.s.num > 256 ? count(i0) : total;
    int i = 0;
    while (at < hi && at < base + sum) {
      // the sequence that tile `at` lies in
      int step = 128;
      for (i = 0; step; step /= 2)
        if (base + ends[i + step - 1] <= at) i += step;
      i = __builtin_amdgcn_readfirstlane(i);
      const CacheSeq q = seqs[i];
      const int64_t first = base + (i ? ends[i - 1] : 0);
      int blocks;
      const int tiles = tiles_of(d, q, ROWS, &blocks);
      const int unit = (int)((at - first) / tiles);
      const int64_t unit_at = first + (int64_t)unit * tiles;
      const int h = unit / blocks, block = unit - h * blocks;
      const int ta = (int)(at - unit_at), tb = (int)least(tiles, hi - unit_at);

      W w;
      Unit<NB> u;
      u.begin(d, q, h);
      w.begin(d, q, h, block * ROWS);
      run_steps(w, u, d.c2, ta * kTile + wave * kStep, min(tb * kTile, u.len), kTile, q.past);
      if (u.bad) record_err(d.s.status, err_key(kPhSeq, 0, 0, (uint32_t)(i0 + i), kSqPage));

      const bool whole = ta == 0 && tb == tiles;
      const int n = lane & 15, quad = lane >> 4;
      float* const part = d.part + (size_t)(2 * group + slot) * part_floats<D, ROWS>();
      const int64_t mi = ((int64_t)(i0 + i) * d.c.heads + h) * d.blocks + block;
      if (ta == 0 && tid == 0) {
        // the workgroup of the unit's last tile: the last one that begins before it
        const int64_t last = unit_at + tiles - 1;
        int g = (int)(last * groups / total);
        while (share_at(total, groups, g) > last) --g;
        while (share_at(total, groups, g + 1) <= last) ++g;
        d.meta[mi] = {group, whole ? 0 : g - group + 1, 2 * group + slot, q.begin, q.n, h, block, 0};
      }
#pragma unroll
      for (int b = 0; b < MT; ++b) {
        __syncthreads();
        const float l = sum_quads(w.l[b]);
        if (quad == 0) {
          om[wave][16 * b + n] = w.m[b];
          ol[wave][16 * b + n] = l;
        }
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) oo[wave][n][W::elem(quad, j, e)] = w.o[b][j][e];
        __syncthreads();
        for (int x = tid; x < 16 * D / 4; x += 256) {
          const int r = x / (D / 4), e0 = x % (D / 4) * 4;
          const int row = block * ROWS + 16 * b + r;
          if (row >= q.n * d.rep) break;
          float f[4], m = kNone, sum_l = 0.0f, v[4] = {};
#pragma unroll
          for (int k = 0; k < 4; ++k) m = fmaxf(m, om[k][16 * b + r]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f[k] = __builtin_amdgcn_exp2f((om[k][16 * b + r] - m) * d.c2);
            sum_l += f[k] * ol[k][16 * b + r];
            const f32x4 y = *reinterpret_cast<const f32x4*>(&oo[k][r][e0]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(f[k], y[e], v[e]);
          }
          if (whole) {
            const Result<T> out(d, q, h, row, sum_l);
            out.store(e0, v, out.gates(e0));
          } else {
            *reinterpret_cast<f32x4*>(part + (16 * b + r) * D + e0) = f32x4{v[0], v[1], v[2], v[3]};
            if (e0 == 0) {
              part[ROWS * D + 16 * b + r] = m;
              part[ROWS * D + ROWS + 16 * b + r] = sum_l;
            }
          }
        }
      }
      slot += !whole;
      at = unit_at + tb;
      __syncthreads();
    }
    base += sum;
  }
}

// The parts of a unit joined: a workgroup takes one row, D / 4 threads of 4 elements, as
// many parts at a time as it has threads for.
template <typename T, int NB, int MT>
__global__ __launch_bounds__(256) void k_attend_join(AttendDev d, int rows_per_unit) {
  constexpr int D = 32 * NB, ROWS = 16 * MT, X = D / 4, Y = 256 / X;
  const int tid = threadIdx.x, x = tid % X, y = tid / X;
  const int unit = blockIdx.x / rows_per_unit, r = blockIdx.x - unit * rows_per_unit;
  const Meta meta = d.meta[unit];
  if (meta.parts == 0) return;
  const int block = unit % d.blocks, h = unit / d.blocks % d.c.heads;
  const int row = block * ROWS + r;
  if (row >= meta.n * d.rep) return;
  constexpr int P = part_floats<D, ROWS>();
  float m = kNone, l = 0.0f;
  f32x4 v = {};
  if (y < Y) {  // (D of 96 and 192 leave some threads over)
    for (int i = y; i < meta.parts; i += Y) {
      // (a workgroup's parts lie at 2 g and 2 g + 1; all but the first begin with this unit)
      const float* p = d.part + (size_t)(i ? 2 * (meta.group + i) : meta.place) * P;
      const float pm = p[ROWS * D + r], pl = p[ROWS * D + ROWS + r];
      const f32x4 o = *reinterpret_cast<const f32x4*>(p + r * D + 4 * x);
      const float now = fmaxf(m, pm);
      const float a = __builtin_amdgcn_exp2f((m - now) * d.c2), b = __builtin_amdgcn_exp2f((pm - now) * d.c2);
      m = now;
      l = a * l + b * pl;
      v = a * v + b * o;
    }
  }
  __shared__ float sm[Y][X], sl[Y][X];
  __shared__ f32x4 so[Y][X];
  if (y < Y) {
    sm[y][x] = m;
    sl[y][x] = l;
    so[y][x] = v;
  }
  __syncthreads();
  if (y) return;
#pragma unroll
  for (int i = 1; i < Y; ++i) m = fmaxf(m, sm[i][x]);
  l = 0.0f;
  v = f32x4{};
#pragma unroll
  for (int i = 0; i < Y; ++i) {
    const float f = __builtin_amdgcn_exp2f((sm[i][x] - m) * d.c2);
    l = __builtin_fmaf(f, sl[i][x], l);
    v = f * so[i][x] + v;
  }
  const float out[4] = {v[0], v[1], v[2], v[3]};
  const CacheSeq q = {meta.begin, meta.n, 0, 0};
  const Result<T> to(d, q, h, row, l);
  to.store(4 * x, out, to.gates(4 * x));
}

// ---- many rows ------------------------------------------------------------------------------
// A workgroup takes 128 rows of a unit, 16 MT for each wave, and its context 64 tokens at a
// time.  The waves share the work of making codes into operands, which pass through LDS
// in the order in which a wave reads them: 64 lanes of 16 bytes each.  One buffer is
// filled while the other is read, and the codes of the tokens behind those are on their way.
template <int NB, int NW>
struct Share64 {
  using L = CacheLay<NB>;
  static constexpr int JK = 4 * NB / NW;             // key words of a lane: tile wave % 4
  static constexpr int JV = (2 * NB + NW - 1) / NW;  // value bytes: 32 tokens of wave % 2
  static constexpr bool word = NB == 8;  // a wave's bytes of a token lie in one word
  static_assert(!(word || NB == 4) || JV == 2, "a wave has two bytes of such tokens");
  static constexpr int VW = word ? 4 : NB, VS = Held<NB>::VS;
  static constexpr int buffer = 8 * NB * 1024;
  uint32_t k[JK], ks[(NB + 3) / 4], v[2][VW], vs[2][VS];

  // The pages of this wave's tokens: of its keys, and of its values' two 16s.
  struct Pages {
    int k, v[2];
  };
  __device__ __forceinline__ static Pages pages(const Unit<NB>& u, int wave, int t0) {
    return {u.page(t0 + 16 * (wave % 4)),
            {u.page(t0 + 32 * (wave % 2)), u.page(t0 + 32 * (wave % 2) + 16)}};
  }
  __device__ __forceinline__ void load(Unit<NB>& u, int wave, int t0, const Pages& p) {
    const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
    // (behind the last token, its own 16 are read again)
    const int last = (u.len - 1) & ~15;
    const size_t key = u.at(p.k, min(t0 + 16 * (wave % 4), last));
    load_words<JK>(u.codes + key + (unsigned)(n * L::row + (quad * NB + wave / 4 * JK) * 4), k);
    load_scales<NB>(u.scales + key / 16 + (unsigned)(n * NB), ks);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const size_t at = u.at(p.v[a], min(t0 + 32 * (wave % 2) + 16 * a, last));
      const uint8_t* const c = u.codes + at + u.value_bytes;
      const unsigned mine = quad * (4 * L::row) + n * (4 * NB);
      if constexpr (word) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[a][e] = *reinterpret_cast<const uint32_t*>(c + (mine + e * NB + wave / 2 * JV / 4 * 4));
      } else {
        load_words<VW>(c + mine, v[a]);
      }
      Held<NB>::load_value_scales(u, at, vs[a]);
    }
  }

  // The scales of the values, as they count.
  __device__ __forceinline__ void value_scales(const Unit<NB>& u, int t32, uint32_t (&x)[2][VS]) const {
    const int quad = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < VS; ++g) x[a][g] = present(vs[a][g], u.len - (t32 + 16 * a + 4 * quad));
  }

  // Into a buffer: operands (tile, j) of the keys, then (32 tokens, 2 b + half) of the
  // values; whether a value is NaN.
  __device__ __forceinline__ bool store(const Unit<NB>& u, int wave, int t0, uint8_t* lds) const {
    const int lane = threadIdx.x & 63;
    bf16x8* const out = reinterpret_cast<bf16x8*>(lds) + lane;
#pragma unroll
    for (int i = 0; i < JK; ++i) {
      const int j = wave / 4 * JK + i;
      uint32_t x;
      if constexpr (NW == 4) x = exponent(ks[i / 4], i % 4);
      else x = ((uint32_t)((ks[0] | (uint64_t)ks[1] << 32) >> (8 * j)) & 0xFFu) << 23;
      out[((wave % 4) * NB + j) * 64] = key_operand(k[i], x);
    }
    uint32_t x[2][VS];
    value_scales(u, t0 + 32 * (wave % 2), x);
    bool nan = false;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < VS; ++g) nan = nan || any_nan(x[a][g]);
    nan = __any(nan);
    if (nan) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int g = 0; g < VS; ++g) x[a][g] = no_nan(x[a][g]);
    }
    const auto put = [&](int b, auto byte) {
      // byte: of the words where byte b lies (4: not known when this is compiled)
      constexpr int B = decltype(byte)::value;
      uint32_t pair[8], f[4], g[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t c, s;
        if constexpr (B < 4) {
          c = v[e / 4][e % 4];
        } else {
          const int at = (e % 4) * NB + b;
          c = 0;
#pragma unroll
          for (int y = 0; y < VW; ++y)
            if (at / 4 == y) c = v[e / 4][y] >> (8 * (at % 4));
        }
        if constexpr (L::pow2) {
          s = exponent(x[e / 4][0], e % 4);
        } else {
          uint32_t y = 0;
#pragma unroll
          for (int z = 0; z < VS; ++z)
            if (z == b) y = x[e / 4][z];
          s = exponent(y, e % 4);
        }
        pair[e] = held_pair<B % 4>(c, s);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x05040100u);
        g[e] = __builtin_amdgcn_perm(pair[2 * e + 1], pair[2 * e], 0x07060302u);
      }
      const int at = 4 * NB + (wave % 2) * 2 * NB + 2 * b;
      out[at * 64] = __builtin_bit_cast(bf16x8, make_uint4(f[0], f[1], f[2], f[3]));
      out[(at + 1) * 64] = __builtin_bit_cast(bf16x8, make_uint4(g[0], g[1], g[2], g[3]));
    };
    const int b0 = wave / 2 * JV;
    if constexpr (word || NB == 4) {  // two bytes of a word, the first or the last
      if (b0 % 4 == 0) {
        put(b0, std::integral_constant<int, 0>{});
        put(b0 + 1, std::integral_constant<int, 1>{});
      } else {
        put(b0, std::integral_constant<int, 2>{});
        put(b0 + 1, std::integral_constant<int, 3>{});
      }
    } else {
#pragma unroll
      for (int i = 0; i < JV; ++i)
        if (b0 + i < NB) put(b0 + i, std::integral_constant<int, 4>{});
    }
    return nan;
  }
};

// Places of a unit's part: of 16 rows and j, 64 lanes of four outputs; then the rows' m, l.
template <int NB>
__device__ __forceinline__ size_t many_part(int place) {
  return (size_t)place * kManyRows * (32 * NB + 2);
}

template <typename T, int NB, int MT>
__global__ __launch_bounds__(4 * kManyRows / MT, 2) void k_attend_many(AttendDev d) {
  constexpr int NW = kManyRows / (16 * MT), D = 32 * NB;
  using W = Wave<T, NB, MT>;
  using S = Share64<NB, NW>;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = blockIdx.x;
  __shared__ __align__(16) uint8_t lds[2][S::buffer];
  __shared__ int nans[2][NW];
  __shared__ int64_t wsum[NW], ends[64 * NW];
  __shared__ CacheSeq seqs[64 * NW];
  const ManyCost cost(d.rep, d.few_rows);

  // The lengths of as many sequences as there are threads, from i0 on, summed up in ends.
  const auto count = [&](int i0) {
    CacheSeq q = {};
    int64_t sum = 0;
    if (i0 + tid < d.s.num) {
      q = cache_seq(d.c, d.s, i0 + tid, group == 0);
      sum = d.c.heads * ManyLine(cost, q.n, q.past).head();
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int64_t x = __shfl_up(sum, o);
      if (lane >= o) sum += x;
    }
    __syncthreads();
    if (lane == 63) wsum[wave] = sum;
    seqs[tid] = q;
    __syncthreads();
    int64_t before = 0;
    for (int i = 0; i < wave; ++i) before += wsum[i];
    ends[tid] = before + sum;
    __syncthreads();
    return ends[64 * NW - 1];
  };
  int64_t total = count(0);
  for (int i0 = 64 * NW; i0 < d.s.num; i0 += 64 * NW) total += count(i0);
  const ManyShares shares(cost, total, (int)gridDim.x);
  if (tid == 0) d.meta[group].parts = 0;
  if (group >= shares.groups) return;
  many_walk<64 * NW>(
    cost, shares, group, d.s.num, ends, count, [&](int i) { return seqs[i]; },
    [&](int i0, int i, const CacheSeq& q, const ManyPart& unit, int slot) {
      const int h = __builtin_amdgcn_readfirstlane(unit.head);
      const int b = __builtin_amdgcn_readfirstlane(unit.block);
      const int from = __builtin_amdgcn_readfirstlane(unit.from);
      const int to = __builtin_amdgcn_readfirstlane(unit.to);
      const bool starts = unit.starts, whole = unit.whole;
      const int64_t rows = (int64_t)q.n * d.rep, block0 = (int64_t)b * kManyRows;
      const int64_t row0 = block0 + wave * (16 * MT);
      const int first_seen = q.past + (int)(block0 / d.rep);
      const int last_seen =
          row0 < rows ? q.past + (int)((least(row0 + 16 * MT, rows) - 1) / d.rep) : -1;
      W w;
      Unit<NB> u;
      u.begin(d, q, h);
      w.begin(d, q, h, (int)least(row0, rows));
      int t0 = 64 * from, buf = 0;
      const int stop = 64 * to;
      S raw;
      typename S::Pages pages;
      if (t0 < stop) {
        raw.load(u, wave, t0, S::pages(u, wave, t0));
        pages = S::pages(u, wave, t0 + 64);
        const bool nan = raw.store(u, wave, t0, lds[0]);
        if (lane == 0) nans[0][wave] = nan;
        raw.load(u, wave, t0 + 64, pages);
        pages = S::pages(u, wave, t0 + 128);
      }
      __syncthreads();
      const auto tile = [&](auto mask) {
        if (t0 + 64 < stop) {
          const bool nan = raw.store(u, wave, t0 + 64, lds[buf ^ 1]);
          if (lane == 0) nans[buf ^ 1][wave] = nan;
          raw.load(u, wave, t0 + 128, pages);
          pages = S::pages(u, wave, t0 + 192);
        }
        const bf16x8* const in = reinterpret_cast<const bf16x8*>(lds[buf]) + lane;
        if (t0 <= last_seen) {
          int nan = 0;
#pragma unroll
          for (int k = 0; k < NW; ++k) nan |= nans[buf][k];
          w.template step<decltype(mask)::value, 4>(
              d.c2, t0, [&](int a, int j) { return in[(a * NB + j) * 64]; },
              [&](int g, int b, bf16x8& v0, bf16x8& v1) {
                v0 = in[(4 * NB + g * 2 * NB + 2 * b) * 64];
                v1 = in[(4 * NB + g * 2 * NB + 2 * b + 1) * 64];
              },
              __builtin_amdgcn_readfirstlane(nan) != 0,
              [&](int g, int b) {  // (rare: the scales once more)
                uint32_t x[2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                  uint32_t y[S::VS];
                  const int t = t0 + 32 * g + 16 * a, near = min(t, (u.len - 1) & ~15);
                  Held<NB>::load_value_scales(u, u.at(u.page(near), near), y);
                  x[a] = 0;
#pragma unroll
                  for (int z = 0; z < S::VS; ++z)
                    if (S::L::pow2 || z == b) x[a] = y[z];
                  x[a] = present(x[a], u.len - (t + 4 * quad));
                }
                return nan_marks(x[0], x[1]);
              });
        }
        __syncthreads();
        t0 += 64;
        buf ^= 1;
      };
      // (steps that every row sees all of, then the others)
      while (t0 < stop && t0 + 63 <= first_seen) tile(std::false_type{});
      while (t0 < stop) tile(std::true_type{});
      settle(w.o);
      if (u.bad) record_err(d.s.status, err_key(kPhSeq, 0, 0, (uint32_t)(i0 + i), kSqPage));
      if (starts && !whole && tid == 0)
        d.meta[group] = {group, shares.parts(group, unit.end), 2 * group + slot, q.begin, q.n, h, b, 0};
      float* const part = d.part + many_part<NB>(2 * group + slot);
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        const float l = sum_quads(w.l[k]);
        const int64_t row = row0 + 16 * k + n;
        if (whole) {
          if (row < rows) w.results(k, Result<T>(d, q, h, (int)row, l));
        } else {
          const int of = wave * MT + k;
#pragma unroll
          for (int j = 0; j < 2 * NB; ++j)
            *reinterpret_cast<f32x4*>(part + ((size_t)(of * 2 * NB + j) * 64 + lane) * 4) = w.o[k][j];
          if (quad == 0) {
            part[kManyRows * D + 16 * of + n] = w.m[k];
            part[kManyRows * D + kManyRows + 16 * of + n] = l;
          }
        }
      }
    });
}

// The parts of a unit joined: a workgroup takes 16 rows and JG of the j of their outputs, each of
// its waves every fourth part.
template <int NB>
constexpr int join_js() { return CacheLay<NB>::pow2 && NB >= 2 ? 4 : 2; }

template <typename T, int NB>
__global__ __launch_bounds__(256) void k_attend_many_join(AttendDev d) {
  constexpr int D = 32 * NB, JG = join_js<NB>();
  using L = CacheLay<NB>;
  const Meta meta = d.meta[blockIdx.x];
  if (meta.parts == 0) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4, wave = tid >> 6;
  const int of = blockIdx.y / (2 * NB / JG), j0 = blockIdx.y % (2 * NB / JG) * JG;
  const int64_t row = (int64_t)meta.block * kManyRows + 16 * of + n;
  const int64_t rows = (int64_t)meta.n * d.rep;
  if (row - n >= rows) return;
  float m = kNone, l = 0.0f;
  f32x4 v[JG] = {};
  for (int i = wave; i < meta.parts; i += 4) {
    // (a workgroup's parts lie at 2 g and 2 g + 1; all but the first begin with this unit)
    const float* const p = d.part + many_part<NB>(i ? 2 * (meta.group + i) : meta.place);
    const float pm = p[kManyRows * D + 16 * of + n], pl = p[kManyRows * D + kManyRows + 16 * of + n];
    f32x4 o[JG];
#pragma unroll
    for (int j = 0; j < JG; ++j)
      o[j] = *reinterpret_cast<const f32x4*>(p + ((size_t)(of * 2 * NB + j0 + j) * 64 + lane) * 4);
    const float now = fmaxf(m, pm);
    const float a = __builtin_amdgcn_exp2f((m - now) * d.c2), b = __builtin_amdgcn_exp2f((pm - now) * d.c2);
    m = now;
    l = a * l + b * pl;
#pragma unroll
    for (int j = 0; j < JG; ++j) v[j] = a * v[j] + b * o[j];
  }
  __shared__ float sm[4][64], sl[4][64];
  __shared__ f32x4 so[4][JG][64];
  sm[wave][lane] = m;
  sl[wave][lane] = l;
#pragma unroll
  for (int j = 0; j < JG; ++j) so[wave][j][lane] = v[j];
  __syncthreads();
  if (wave || row >= rows) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) m = fmaxf(m, sm[i][lane]);
  l = 0.0f;
#pragma unroll
  for (int j = 0; j < JG; ++j) v[j] = f32x4{};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = __builtin_amdgcn_exp2f((sm[i][lane] - m) * d.c2);
    l = __builtin_fmaf(f, sl[i][lane], l);
#pragma unroll
    for (int j = 0; j < JG; ++j) v[j] = f * so[i][j][lane] + v[j];
  }
  const CacheSeq q = {meta.begin, meta.n, 0, 0};
  const Result<T> out(d, q, meta.head, (int)row, l);
  store_lane<T, NB, JG>(quad, j0, v, out);
}

// Workgroups of k_attend_few: as many as there is room for.
int few_groups(int dtype, int dim, int mt) {
  const int waves = dtype == DMH_DTYPE_BF16  ? few_waves<bf16_t>(dim, mt)
                    : dtype == DMH_DTYPE_F16 ? few_waves<half_t>(dim, mt)
                                             : few_waves<float>(dim, mt);
  return 256 * waves;
}
constexpr int64_t kMostBlocks = 1 << 23;  // workgroups of a launch, of 2^31 threads

// Workgroups of k_attend_many: one a CU where its LDS fills that, else two.
int many_groups(int dim) { return dim > 128 ? 256 : 512; }

// Rows (tokens times query heads of a key head) up to which a sequence is k_attend_few's.  8
// sequences behind 80000 tokens in all, 16 heads on 2, bf16, at 24, 32, 40 and 64 rows: 18, 18, 20
// and 21 us of 64 elements here, 39 to 44 by k_attend_many; 23, 24, 26 and 28 of 128, and 45 to 53;
// 29, 29, 39 and 41 of 256, and 56 to 67.  One sequence behind 8000, 64 rows of 256: 25 and 48.
// (At 96 and 128 rows the order is still the same: 28 and 31 for 45 and 47, 55 and 61 for 84 and 93.)
int few_limit(const dmh_attention& a, const dmh_kv_cache& c) {
  return std::max(a.q_heads / c.kv_heads, 64);
}

// Blocks of 16 or 32 rows of a unit of k_attend_few.
int few_blocks(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s, int mt) {
  const int64_t rep = a.q_heads / c.kv_heads;
  const int64_t most = std::max<int64_t>(rep, std::min<int64_t>(64, s.max_len * rep));
  return (int)((most + 16 * mt - 1) / (16 * mt));
}
// Of how many 16s: one where sequences have 16 rows or fewer (two: 128 elements at 8 rows 18.1 ->
// 19.5 us in bf16, 18.8 -> 29.9 in fp32), and of 256 elements, which leave no registers for two.
// Two 16s make operands once: of 64 elements 64 rows take 21.3 us, one by one 23.2.  At 24 and 32
// rows both take 18; of 128 elements two are slower there (22.4 and 21.2, in fp32 32.7 and 23.2, at
// 64 rows 28.0 and 28.5, in fp32 38.9 and 32.6).
int few_tiles(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s) {
  const int64_t rep = a.q_heads / c.kv_heads;
  return c.dim <= 128 && s.max_len * rep > 16 ? 2 : 1;
}

// Workgroups of k_attend_join.
// (of a unit's rows as many as sequences can have)
int join_rows(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s, int mt) {
  return (int)std::min<int64_t>(16 * mt, (int64_t)s.max_len * (a.q_heads / c.kv_heads));
}
int64_t join_blocks(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s, int mt) {
  return (int64_t)s.num * c.kv_heads * few_blocks(a, c, s, mt) * join_rows(a, c, s, mt);
}

}  // namespace

bool attend_fits(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s) {
  // (rows, tokens times query heads of a key head, are counted in 32 bits)
  return (int64_t)s.rows * (a.q_heads / c.kv_heads) < (int64_t)1 << 30 &&
         join_blocks(a, c, s, few_tiles(a, c, s)) < kMostBlocks;
}

// The memory is the same for all lengths of sequences, so that any call of as many heads and
// sequences may stand before one that is captured.  (The kernels for few and for many rows
// come one after the other and share the place of parts; those for many rows, two of 128 rows
// a workgroup, take more than two of 16 or 32.)
size_t attend_parts(const dmh_kv_cache& c) {
  static_assert(3 * 256 * 32 <= 256 * kManyRows, "three waves a SIMD of k_attend_few");
  return (size_t)2 * many_groups(c.dim) * kManyRows * (c.dim + 2);
}
size_t attend_bytes(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s) {
  const size_t units = (size_t)s.num * c.kv_heads * ((few_limit(a, c) + 15) / 16);
  return attend_parts(c) * 4 + sizeof(Meta) * std::max(units, (size_t)many_groups(c.dim));
}

hipError_t launch_attend(const dmh_attention& a, const dmh_kv_cache& c, const SeqDev& s, void* ws,
                         hipStream_t st) {
  AttendDev d = {a, cache_dev(c), s};
  d.rep = a.q_heads / c.kv_heads;
  d.few_rows = few_limit(a, c);
  d.c2 = (float)((double)a.scale * 1.4426950408889634);
  const int mt = few_tiles(a, c, s);
  d.blocks = few_blocks(a, c, s, mt);
  d.part = static_cast<float*>(ws);
  d.meta = reinterpret_cast<Meta*>(d.part + attend_parts(c));
  return with_type(a.dtype, [&](auto t) {
    return with_blocks(c.dim, [&](auto nb) {
      using T = decltype(t);
      constexpr int NB = decltype(nb)::value;
      if ((int64_t)s.max_len * d.rep > d.few_rows) {
        constexpr int MT = NB > 4 ? 1 : 2;
        const int groups = many_groups(c.dim);
        k_attend_many<T, NB, MT><<<groups, 4 * kManyRows / MT, 0, st>>>(d);
        k_attend_many_join<T, NB><<<dim3(groups, 16 * NB / join_js<NB>()), 256, 0, st>>>(d);
      }
      const auto few = [&](auto m) {
        constexpr int MT = decltype(m)::value;
        k_attend_few<T, NB, MT><<<few_groups(a.dtype, c.dim, MT), 256, 0, st>>>(d);
        k_attend_join<T, NB, MT><<<(unsigned)join_blocks(a, c, s, MT), 256, 0, st>>>(
            d, join_rows(a, c, s, MT));
      };
      if constexpr (NB <= 4) {
        if (mt == 2) few(std::integral_constant<int, 2>{});
      }
      if (mt == 1) few(std::integral_constant<int, 1>{});
      return hipGetLastError();
    });
  });
}

}  // namespace dm
