// dm_linear.hip -- linear layers with 4-bit weights: y = W x + bias.
//
// W's codes become bf16 operands of the matrix cores as they are read, each the
// bf16 value that dequantising gives; rows of x that are not bf16 enter as two or three
// bf16 parts that hold all of their bits, so products are exact and sums fp32.
#include <algorithm>
#include <type_traits>

#include "dm_device.h"
#include "dm_linear.h"
#include "dm_mixer_device.h"

namespace dm {
namespace {

constexpr int64_t kMostBlocks = 1 << 23;  // workgroups of a launch, of 2^31 threads

__global__ __launch_bounds__(256) void k_linear_pack(const uint16_t* __restrict__ scales,
                                                     const uint8_t* __restrict__ packed, int n, int k,
                                                     int group, uint8_t* __restrict__ nib,
                                                     uint16_t* __restrict__ sc, int chunks,
                                                     int64_t block0, int64_t lanes,
                                                     unsigned long long* vkey) {
  const int64_t gid = (block0 + blockIdx.x) * 256 + threadIdx.x;
  if (gid >= lanes) return;
  const int lane = (int)(gid & 63);
  const int gq = (int)((gid >> 6) % chunks), rb = (int)((gid >> 6) / chunks);
  const int row = rb * kTileRows + (lane & 15), quad = lane >> 4;
  uint32_t out[4], s[4];
  uint64_t key = kNoError;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int col = gq * kQuadCols + c * kGroup + 8 * quad;
    out[c] = 0x88888888u;  // code 0
    s[c] = 0;
    if (row >= n || col >= k) continue;
    const int64_t e0 = (int64_t)row * k + col;
    const uint8_t* p = packed + e0 / 2;
    uint32_t w = 0;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const uint32_t code = (p[kk / 2] >> (4 * (kk & 1))) & 15u;
      if (code == 8u && key > (1ull << 60)) key = 1ull << 60;
      w |= (code ^ 8u) << (4 * a16_slot_of_kk(kk));
    }
    out[c] = w;
    const int64_t g = e0 / group;
    const uint32_t u = s[c] = scales[g];
    uint64_t bad = kNoError;
    if (((u >> 10) & 0x1Fu) == 0x1Fu) bad = 2ull * g;
    else if ((u & 0x8000u) || (u & 0x7FFFu) == 0) bad = 2ull * g + 1;
    if (bad < key) key = bad;
  }
  *reinterpret_cast<uint4*>(nib + a16_nib_offset(chunks, rb, gq, lane)) =
      make_uint4(out[0], out[1], out[2], out[3]);
  if (quad == 0)
    *reinterpret_cast<uint2*>(sc + a16_sc_offset(chunks, rb, gq, lane & 15)) =
        make_uint2(s[0] | s[1] << 16, s[2] | s[3] << 16);
  if (key != kNoError) atomicMin(vkey, (unsigned long long)key);
}

template <typename T>
constexpr int parts_of() {
  return std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, half_t>::value ? 2 : 3;
}

// Eight elements as PARTS bf16 values whose sum each is.
template <typename T, int PARTS>
__device__ __forceinline__ void to_parts(Vec<T, 8> v, bf16x8 (&out)[PARTS]) {
  if constexpr (PARTS == 1) {
    out[0] = __builtin_bit_cast(bf16x8, v);
  } else {
    float r[8];
    to_f32<8>(v, r);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (fp32 values are cut off first, as the largest have no bf16 above them)
        w[i] = PARTS == 3 && q == 0 ? f2u(r[2 * i]) >> 16 | (f2u(r[2 * i + 1]) & 0xFFFF0000u)
                                    : pack_bf16x2(r[2 * i], r[2 * i + 1]);
        r[2 * i] -= bf16lo(w[i]);
        r[2 * i + 1] -= bf16hi(w[i]);
      }
      out[q] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    }
  }
}

template <typename O>
__device__ __forceinline__ void store_out(const LinearDev& l, const dmh_linear_rows& r, int64_t token,
                                          int row, f32x4 v) {
  if (token >= r.rows || row >= l.n) return;
  O* const y = static_cast<O*>(r.y) + token * r.y_stride + row;
  if (l.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += l.bias[min(row + i, l.n - 1)];
  }
  const float f[4] = {v[0], v[1], v[2], v[3]};
  if (row + 4 <= l.n) {
    store_f32<4>(y, f);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (row + i < l.n) y[i] = (O)f[i];
  }
}

// ---- few rows -------------------------------------------------------------------------
// A workgroup takes 16 AT rows of W and 16 NT rows of x; its waves take W's chunks of 128
// columns in turn, one of them on its way ahead of the products, and add up through LDS.
// Bound by W's bytes.
template <typename T, typename O, int AT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_linear_few(LinearDev l, dmh_linear_rows r) {
  constexpr int P = parts_of<T>();
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rb0 = blockIdx.x * AT;
  const int64_t t0 = (int64_t)blockIdx.y * (16 * NT);
  const T* x[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    x[i] = static_cast<const T*>(r.x) + least(t0 + 16 * i + n, r.rows - 1) * r.x_stride + 8 * quad;
  const uint8_t* nib[AT];
  const uint16_t* sc[AT];
#pragma unroll
  for (int j = 0; j < AT; ++j) {
    const int rb = min(rb0 + j, l.row_blocks - 1);
    nib[j] = l.nib + a16_nib_offset(l.chunks, rb, 0, lane);
    sc[j] = l.sc + a16_sc_offset(l.chunks, rb, 0, n);
  }
  uint4 w[AT];
  uint2 s[AT];
  const auto load = [&](size_t g) {
#pragma unroll
    for (int j = 0; j < AT; ++j) {
      w[j] = *reinterpret_cast<const uint4*>(nib[j] + g * 1024);
      s[j] = *reinterpret_cast<const uint2*>(sc[j] + g * 64);
    }
  };
  f32x4 acc[AT][NT] = {};
  if (wave < l.chunks) load(wave);
  for (int g = wave; g < l.chunks; g += WAVES) {
    uint4 wn[AT];
    uint2 sn[AT];
#pragma unroll
    for (int j = 0; j < AT; ++j) {
      wn[j] = w[j];
      sn[j] = s[j];
    }
    load(min(g + WAVES, l.chunks - 1));
    // (rows that are not there are not read: their lines would cost as much as the others')
    Vec<T, 8> raw[4][NT] = {};
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (t0 + 16 * i + n < r.rows) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          raw[c][i] = load_raw<8>(x[i] + min(g * kQuadCols + c * kGroup, l.k - kGroup));
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (g * kQuadCols + c * kGroup >= l.k) break;
      bf16x8 b[NT][P];
#pragma unroll
      for (int i = 0; i < NT; ++i) to_parts<T, P>(raw[c][i], b[i]);
#pragma unroll
      for (int j = 0; j < AT; ++j) {
        const uint32_t word = c == 0 ? wn[j].x : c == 1 ? wn[j].y : c == 2 ? wn[j].z : wn[j].w;
        const uint32_t half = c < 2 ? sn[j].x : sn[j].y;
        const bf16x8 a = dequant8(word, fp16_bits_to_f32(c % 2 ? half >> 16 : half & 0xFFFFu));
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[j][i] = mfma16(a, b[i][p], acc[j][i]);
      }
    }
  }
  __shared__ f32x4 red[WAVES][AT][NT][64];
  // (a product's result is read some cycles after its issue, which the compiler does not
  // count over the end of a loop)
#pragma unroll
  for (int j = 0; j < AT; ++j)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      asm volatile("s_nop 7\n\ts_nop 7" : "+v"(acc[j][i]));
      red[wave][j][i][lane] = acc[j][i];
    }
  __syncthreads();
  for (int i = wave; i < AT * NT; i += WAVES) {
    f32x4 v = red[0][i / NT][i % NT][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += red[k][i / NT][i % NT][lane];
    store_out<O>(l, r, t0 + 16 * (i % NT) + n, (rb0 + i / NT) * kTileRows + 4 * quad, v);
  }
}

// ---- few rows of a large W ----------------------------------------------------------------
// Workgroups that stay: each takes a run of W's row blocks, its waves CW chunks of 128
// columns each.  A wave holds its chunks of x as operands in registers the whole time, so that
// x is read and taken apart once a workgroup instead of once in every 16 AT rows of W, and
// W's next row blocks are on their way over the joins through LDS, two row blocks at a time
// (four: up to 2 us slower).  Bound by W's bytes: 100003 x 2048, five rows, 26.8 us in bf16
// (4.3 TB/s), 29.9 in f16, 33.4 in fp32; with one chunk after the other by k_linear_few 31.4,
// 38.9 and 44.6.
constexpr int kJoinTiles = 2;
template <typename T, typename O, int CW>
__global__ __launch_bounds__(1024, 4) void k_linear_run(LinearDev l, dmh_linear_rows r) {
  constexpr int P = parts_of<T>(), JT = kJoinTiles;
  extern __shared__ f32x4 red[];  // [2][JT][waves][64]
  const int waves = blockDim.x / 64;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lo = (int)((int64_t)l.row_blocks * blockIdx.x / gridDim.x);
  const int hi = (int)((int64_t)l.row_blocks * (blockIdx.x + 1) / gridDim.x);
  uint4 w[JT][CW];
  uint2 s[JT][CW];
  const auto load = [&](int j, int rb) {
#pragma unroll
    for (int i = 0; i < CW; ++i) {
      const int g = min(wave * CW + i, l.chunks - 1);
      // (read once and not again before the next call: not kept in L2 over what is)
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      const u32x4 a = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(l.nib + a16_nib_offset(l.chunks, rb, g, lane)));
      w[j][i] = make_uint4(a.x, a.y, a.z, a.w);
      s[j][i] = *reinterpret_cast<const uint2*>(l.sc + a16_sc_offset(l.chunks, rb, g, n));
    }
  };
#pragma unroll
  for (int j = 0; j < JT; ++j)
    if (lo + j < hi) load(j, lo + j);
  // (rows and columns that are not there are 0)
  bf16x8 b[CW][4][P];
  {
    const T* const x = static_cast<const T*>(r.x) + least(n, r.rows - 1) * r.x_stride + 8 * quad;
    Vec<T, 8> raw[CW][4] = {};
#pragma unroll
    for (int i = 0; i < CW; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = (wave * CW + i) * kQuadCols + c * kGroup;
        if (n < r.rows && col < l.k) raw[i][c] = load_raw<8>(x + col);
      }
#pragma unroll
    for (int i = 0; i < CW; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) to_parts<T, P>(raw[i][c], b[i][c]);
  }
  int buf = 0, turn = wave;  // the waves add up in turn, JT of them at a time
  for (int t = lo; t < hi; t += JT, buf ^= 1) {
    f32x4 acc[JT] = {};
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      if (t + j >= hi) break;
#pragma unroll
      for (int i = 0; i < CW; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t word = c == 0 ? w[j][i].x : c == 1 ? w[j][i].y : c == 2 ? w[j][i].z : w[j][i].w;
          const uint32_t half = c < 2 ? s[j][i].x : s[j][i].y;
          const bf16x8 a = dequant8(word, fp16_bits_to_f32(c % 2 ? half >> 16 : half & 0xFFFFu));
#pragma unroll
          for (int p = 0; p < P; ++p) acc[j] = mfma16(a, b[i][c][p], acc[j]);
        }
      if (t + JT + j < hi) load(j, t + JT + j);
      // (a product's result is read some cycles after its issue, which the compiler does not
      // count over the end of a block)
      asm volatile("s_nop 7\n\ts_nop 7" : "+v"(acc[j]));
      red[((buf * JT + j) * waves + wave) * 64 + lane] = acc[j];
    }
    __syncthreads();
    for (; turn < JT; turn += waves) {
      if (t + turn >= hi) continue;
      const f32x4* const from = red + (buf * JT + turn) * waves * 64 + lane;
      f32x4 v = from[0];
#pragma unroll 4
      for (int k = 1; k < waves; ++k) v += from[k * 64];
      store_out<O>(l, r, n, (t + turn) * kTileRows + 4 * quad, v);
    }
    turn -= JT;
  }
}

// ---- many rows --------------------------------------------------------------------------
// A workgroup takes 64 AT rows of W and 16 BT rows of x.  Each of its four waves has
// 16 AT rows of W of its own, whose codes it makes into operands once, and all rows of
// x, 128 columns of which pass through LDS at a time by direct loads, one stage ahead.
// Segment s (16 bytes) of row t lies at s ^ (t % 16), so that the 16 rows of an operand
// lie in different banks.  Bound by the matrix cores.
template <typename O, int AT, int BT>
__global__ __launch_bounds__(256, 2) void k_linear_many(LinearDev l, dmh_linear_rows r,
                                                        const uint16_t* __restrict__ xb,
                                                        int64_t x_stride, int64_t part_stride,
                                                        int parts, int wtiles, int ttiles) {
  constexpr int ROWS = 16 * BT, STAGE = ROWS * 256;
  __shared__ __align__(16) uint8_t lds[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // workgroups come to the XCDs in turn: each gets a run of tiles, rows of x fastest
  const int all = wtiles * ttiles, per = (all + 7) / 8;
  const int tile = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if ((int)(blockIdx.x / 8) >= per || tile >= all) return;
  const int wt = tile / ttiles, tt = tile - wt * ttiles;
  const int rb0 = (wt * 4 + wave) * AT;
  const int64_t t0 = (int64_t)tt * ROWS;

  // steps: the whole chunks of each part, then the last ones that are not whole
  const int whole = l.k / kQuadCols, steps = whole * parts;
  const int all_steps = l.chunks * parts;
  const auto chunk_of = [&](int step) { return step < steps ? step % whole : whole; };
  const auto part_of = [&](int step) { return step < steps ? step / whole : step - steps; };

  // this lane's part of a stage: 16 bytes of every fourth row
  const uint32_t base = lds_u32(lds);
  const auto fetch = [&](int step, int buf) {
    const int g = chunk_of(step);
    const uint16_t* const x = xb + part_of(step) * part_stride + g * kQuadCols;
#pragma unroll
    for (int i = 0; i < BT; ++i) {
      const int row = 16 * i + 4 * wave + quad;  // a wave brings 4 rows, 256 bytes each
      const int seg = n ^ (row & 15);
      // (columns behind the last are not used; they are read from the row itself)
      const int col = min(8 * seg, l.k - 8 - g * kQuadCols);
      dma16_lds(x + least(t0 + row, r.rows - 1) * x_stride + col,
                base + buf * STAGE + (16 * i + 4 * wave) * 256);
    }
  };
  const uint8_t* nib[AT];
  const uint16_t* sc[AT];
#pragma unroll
  for (int a = 0; a < AT; ++a) {
    const int rb = min(rb0 + a, l.row_blocks - 1);
    nib[a] = l.nib + a16_nib_offset(l.chunks, rb, 0, lane);
    sc[a] = l.sc + a16_sc_offset(l.chunks, rb, 0, n);
  }
  uint4 w[AT];
  uint2 s[AT];
  f32x4 acc[AT][BT] = {};
  const auto weights = [&](int step) {
    const size_t g = chunk_of(step);
#pragma unroll
    for (int a = 0; a < AT; ++a) {
      w[a] = *reinterpret_cast<const uint4*>(nib[a] + g * 1024);
      s[a] = *reinterpret_cast<const uint2*>(sc[a] + g * 64);
    }
  };
  // Brings the next step on its way and does this one's `groups` of 32 columns.
  const auto go = [&](int i, int groups) {
    uint4 wn[AT];
    uint2 sn[AT];
#pragma unroll
    for (int a = 0; a < AT; ++a) {
      wn[a] = w[a];
      sn[a] = s[a];
    }
    wait_vm();
    __syncthreads();
    if (i + 1 < all_steps) {
      fetch(i + 1, (i + 1) & 1);
      weights(i + 1);
    }
    const uint8_t* const x = lds + (i & 1) * STAGE;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c >= groups) break;
      bf16x8 a[AT], b[BT];
#pragma unroll
      for (int j = 0; j < BT; ++j)
        b[j] = *reinterpret_cast<const bf16x8*>(x + (16 * j + n) * 256 + ((4 * c + quad) ^ n) * 16);
#pragma unroll
      for (int j = 0; j < AT; ++j) {
        const uint32_t word = c == 0 ? wn[j].x : c == 1 ? wn[j].y : c == 2 ? wn[j].z : wn[j].w;
        const uint32_t half = c < 2 ? sn[j].x : sn[j].y;
        a[j] = dequant8(word, fp16_bits_to_f32(c % 2 ? half >> 16 : half & 0xFFFFu));
      }
#pragma unroll
      for (int j = 0; j < AT; ++j)
#pragma unroll
        for (int k = 0; k < BT; ++k) acc[j][k] = mfma16(a[j], b[k], acc[j][k]);
    }
  };
  fetch(0, 0);
  weights(0);
  for (int i = 0; i < steps; ++i) go(i, 4);
  for (int i = steps; i < all_steps; ++i) go(i, (l.k - whole * kQuadCols) / kGroup);
#pragma unroll
  for (int j = 0; j < AT; ++j)
#pragma unroll
    for (int k = 0; k < BT; ++k) asm volatile("" : "+v"(acc[j][k]));
  asm volatile("s_nop 7\n\ts_nop 7" : "+v"(acc[0][0]));
#pragma unroll
  for (int j = 0; j < AT; ++j) {
    if (rb0 + j >= l.row_blocks) break;
#pragma unroll
    for (int k = 0; k < BT; ++k) {
      asm volatile("" : "+v"(acc[j][k]));
      store_out<O>(l, r, t0 + 16 * k + n, (rb0 + j) * kTileRows + 4 * quad, acc[j][k]);
    }
  }
}

// Rows of x as bf16 parts, [parts][rows][k].
template <typename T>
__global__ __launch_bounds__(256) void k_linear_split(const T* x, int64_t stride, int k, int64_t rows,
                                                      uint16_t* out) {
  constexpr int P = parts_of<T>();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = k / 8;
  if (i >= rows * per) return;
  const int64_t row = i / per;
  const int col = (int)(i - row * per) * 8;
  bf16x8 p[P];
  to_parts<T, P>(load_raw<8>(x + row * stride + col), p);
#pragma unroll
  for (int j = 0; j < P; ++j)
    *reinterpret_cast<bf16x8*>(out + (j * rows + row) * k + col) = p[j];
}

template <typename T>
bool direct(const dmh_linear_rows& r) {  // whether the kernel can bring x into LDS as it is
  return std::is_same<T, bf16_t>::value && (uintptr_t)r.x % 16 == 0 && r.x_stride % 8 == 0;
}

template <typename T, typename O>
hipError_t many(const LinearDev& l, const dmh_linear_rows& r, void* ws, hipStream_t st) {
  constexpr int P = parts_of<T>();
  const uint16_t* xb = static_cast<const uint16_t*>(r.x);
  int64_t x_stride = r.x_stride;
  if (!direct<T>(r)) {
    const int64_t n = (int64_t)r.rows * (l.k / 8);
    uint16_t* const out = static_cast<uint16_t*>(ws);
    k_linear_split<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(static_cast<const T*>(r.x),
                                                                  r.x_stride, l.k, r.rows, out);
    xb = out;
    x_stride = l.k;
  }
  const auto go = [&](auto at, auto bt) {
    constexpr int AT = decltype(at)::value, BT = decltype(bt)::value;
    const int wt = (l.row_blocks + 4 * AT - 1) / (4 * AT);
    const int tt = (r.rows + 16 * BT - 1) / (16 * BT);
    const unsigned blocks = (unsigned)(((int64_t)wt * tt + 7) / 8 * 8);
    k_linear_many<O, AT, BT><<<blocks, 256, 0, st>>>(l, r, xb, x_stride, r.rows * x_stride, P, wt, tt);
  };
  // Tiles of 192 by 128 take the least from memory for their products, as long as there
  // are enough of them; 128 by 64 fill the device sooner.  9216 x 2048, 512, 1024 and
  // 2048 rows: 33, 51 and 83 us with the large ones, 36, 59 and 107 with the small; 2048
  // x 4096, 1024 rows (88 large tiles): 55 and 32.
  using std::integral_constant;
  const int64_t large = (int64_t)((l.row_blocks + 11) / 12) * ((r.rows + 127) / 128);
  if (large >= 192) go(integral_constant<int, 3>{}, integral_constant<int, 8>{});
  else go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  return hipGetLastError();
}

// Tiles of 16 by 16 outputs.
int64_t units(const LinearDev& l, const dmh_linear_rows& r) {
  return (int64_t)l.row_blocks * ((r.rows + 15) / 16);
}
// Up to how many of them waves without LDS in between are the faster: 2048 x 4096 at 512
// rows (4096 tiles) 22 us, and 31 through LDS; 9216 x 2048 at 128 (4608) 18.9 and 18.0, at
// 256 (9216) 30 and 24.  32 rows and fewer are bound by W's bytes, which they read once.
bool few_rows(const LinearDev& l, const dmh_linear_rows& r) {
  return r.rows <= 32 || units(l, r) <= 4608;
}

// Chunks of W a wave of k_linear_run takes and the waves that takes.  Two chunks of fp32 rows
// do not fit its registers.
template <typename T>
int run_chunks(const LinearDev& l) {
  return l.chunks > 8 && parts_of<T>() < 3 ? 2 : 1;
}
template <typename T>
int run_waves(const LinearDev& l) {
  return (l.chunks + run_chunks<T>(l) - 1) / run_chunks<T>(l);
}
// Whether that kernel is the faster: a CU's 16 waves have to be in use (nine to eleven
// waves leave the others empty: 65536 x 2496 29 us, and 22.6 with k_linear_few), and W needs enough rows to
// read and take apart x for, fewer the more parts that takes.  In bf16 2048 row blocks, one
// row of 16384 x 2048 7.2 us and 7.1, five of 32768 x 2048 11.4 and 11.6; in f16 half as many,
// one row of 9216 x 2048 8.6 and 8.3, of 16384 x 2048 9.0 and 9.7; in fp32 a quarter,
// 9216 x 2048 7.9 and 10.3.
template <typename T>
bool stays(const LinearDev& l, const dmh_linear_rows& r) {
  const int waves = run_waves<T>(l);
  return r.rows <= 16 && waves <= 16 && 16 / waves * waves >= 12 &&
         l.row_blocks >= 2048 >> (parts_of<T>() - 1);
}

template <typename T, typename O>
hipError_t run(const LinearDev& l, const dmh_linear_rows& r, void* ws, hipStream_t st) {
  if (!few_rows(l, r)) return many<T, O>(l, r, ws, st);
  if (stays<T>(l, r)) {
    const auto stay = [&](auto k) {
      const int waves = run_waves<T>(l);
      k<<<16 / waves * 256, 64 * waves, 2 * kJoinTiles * waves * 64 * sizeof(f32x4), st>>>(l, r);
      return hipGetLastError();
    };
    if (run_chunks<T>(l) == 1) return stay(k_linear_run<T, O, 1>);
    if constexpr (parts_of<T>() < 3) return stay(k_linear_run<T, O, 2>);
  }
  const auto few = [&](auto at, auto nt, auto waves) {
    constexpr int AT = decltype(at)::value, NT = decltype(nt)::value, W = decltype(waves)::value;
    const dim3 grid((l.row_blocks + AT - 1) / AT, (r.rows + 16 * NT - 1) / (16 * NT));
    k_linear_few<T, O, AT, NT, W><<<grid, 64 * W, 0, st>>>(l, r);
    return hipGetLastError();
  };
  using std::integral_constant;
  const integral_constant<int, 1> one{};
  const integral_constant<int, 2> two{};
  const integral_constant<int, 4> four{};
  const integral_constant<int, 8> eight{};
  // More tiles to a workgroup reuse what is loaded and dequantised, more workgroups and
  // waves load sooner.  One row: 2048 x 4096 4.3 us with 16 waves and 4.7 with 8, 9216 x
  // 2048 5.7 with 8 and 6.5 with two tiles; five rows of 65536 x 8192 65 us with four tiles
  // or two and 82 with one, 16 rows 65 with four, 79 with two.  32 rows of 2048 x 4096 6.9 us
  // with one tile, 7.4 with two; 64 rows 7.6 with two, 11.0 with one; 128 rows 10.1 with
  // four, 12.4 with two; of 9216 x 2048 32 rows 8.6 with four times two, 64 rows 13.0, with
  // one 17.
  const int64_t u = units(l, r);
  if (r.rows <= 16) {
    if (l.row_blocks < 256) return few(one, one, integral_constant<int, 16>{});
    if (l.row_blocks < 1024) return few(one, one, eight);
    if (l.row_blocks >= 4096) return few(four, one, four);
    return few(two, one, four);
  }
  if (u < 512) return few(one, one, eight);
  if (u < 1024) return few(two, one, eight);
  if (u < 2048) return r.rows <= 32 ? few(four, two, eight) : few(four, one, eight);
  return few(four, two, four);
}

}  // namespace

hipError_t launch_linear_pack(const uint16_t* scales, const uint8_t* packed, int n, int k, int group,
                              uint8_t* nib, uint16_t* sc, unsigned long long* vkey, hipStream_t st) {
  const int chunks = linear_chunks(k);
  const int64_t lanes = (int64_t)linear_row_blocks(n) * chunks * 64;
  const int64_t blocks = (lanes + 255) / 256;
  for (int64_t b = 0; b < blocks; b += kMostBlocks)
    k_linear_pack<<<(unsigned)std::min(kMostBlocks, blocks - b), 256, 0, st>>>(
        scales, packed, n, k, group, nib, sc, chunks, b, lanes, vkey);
  return hipGetLastError();
}

bool linear_fits(const LinearDev& l, const dmh_linear_rows& r) {
  if (few_rows(l, r)) return true;
  return (int64_t)((l.row_blocks + 7) / 8) * ((r.rows + 63) / 64) < kMostBlocks &&
         (int64_t)r.rows * (l.k / 8) < kMostBlocks * 256;
}

size_t linear_bytes(const LinearDev& l, const dmh_linear_rows& r) {
  if (few_rows(l, r)) return 0;
  const size_t n = (size_t)r.rows * l.k * 2;
  if (r.dtype == DMH_DTYPE_F32) return parts_of<float>() * n;
  if (r.dtype == DMH_DTYPE_F16) return parts_of<half_t>() * n;
  return direct<bf16_t>(r) ? 0 : n;
}

hipError_t launch_linear(const LinearDev& l, const dmh_linear_rows& r, void* ws, hipStream_t st) {
  const bool f32 = r.out_dtype == DMH_DTYPE_F32;
  if (r.dtype == DMH_DTYPE_F32) return run<float, float>(l, r, ws, st);
  if (r.dtype == DMH_DTYPE_F16)
    return f32 ? run<half_t, float>(l, r, ws, st) : run<half_t, half_t>(l, r, ws, st);
  return f32 ? run<bf16_t, float>(l, r, ws, st) : run<bf16_t, bf16_t>(l, r, ws, st);
}

}  // namespace dm
