// dm_linear.hip -- linear layers with 4-bit weights: y = W x + bias.
//
// W's codes become bf16 operands of the matrix cores as they are read, each the
// bf16 value that dequantising gives; rows of x that are not bf16 enter as two or three
// bf16 parts that hold all of their bits, so products are exact and sums fp32.
#include <type_traits>

#include "dm_device.h"
#include "dm_linear.h"
#include "dm_mixer_device.h"

namespace dm {
namespace {

__global__ __launch_bounds__(256) void k_linear_pack(const uint16_t* __restrict__ scales,
                                                     const uint8_t* __restrict__ packed, int n, int k,
                                                     int group, uint8_t* __restrict__ nib,
                                                     uint16_t* __restrict__ sc, int chunks,
                                                     int64_t lanes, unsigned long long* vkey) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
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
__device__ __forceinline__ void load_parts(const T* p, bf16x8 (&out)[PARTS]) {
  if constexpr (PARTS == 1) {
    const Vec<T, 8> v = load_raw<8>(p);
    out[0] = __builtin_bit_cast(bf16x8, v);
  } else {
    float r[8];
    load_f32<8>(p, r);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack_bf16x2(r[2 * i], r[2 * i + 1]);
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
// A workgroup takes 16 rows of W and 16 NT rows of x; its waves take W's chunks of 128
// columns in turn and add up through LDS.  Bound by W's bytes.
template <typename T, typename O, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_linear_few(LinearDev l, dmh_linear_rows r) {
  constexpr int P = parts_of<T>();
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rb = blockIdx.x;
  const int64_t t0 = (int64_t)blockIdx.y * (16 * NT);
  const T* x[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
    x[i] = static_cast<const T*>(r.x) + least(t0 + 16 * i + n, r.rows - 1) * r.x_stride + 8 * quad;
  const uint8_t* const nib = l.nib + a16_nib_offset(l.chunks, rb, 0, lane);
  const uint16_t* const sc = l.sc + a16_sc_offset(l.chunks, rb, 0, n);
  f32x4 acc[NT] = {};
  for (int g = wave; g < l.chunks; g += WAVES) {
    const uint4 w4 = *reinterpret_cast<const uint4*>(nib + (size_t)g * 1024);
    const uint2 s2 = *reinterpret_cast<const uint2*>(sc + (size_t)g * 64);
    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
    const uint32_t s[4] = {s2.x & 0xFFFFu, s2.x >> 16, s2.y & 0xFFFFu, s2.y >> 16};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = g * kQuadCols + c * kGroup;
      if (col >= l.k) break;
      const bf16x8 a = dequant8(w[c], fp16_bits_to_f32(s[c]));
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        bf16x8 b[P];
        load_parts<T, P>(x[i] + col, b);
#pragma unroll
        for (int p = 0; p < P; ++p) acc[i] = mfma16(a, b[p], acc[i]);
      }
    }
  }
  __shared__ f32x4 red[WAVES][NT][64];
  // (a product's result is read some cycles after its issue, which the compiler does not
  // count over the end of a loop)
#pragma unroll
  for (int i = 0; i < NT; ++i) asm volatile("s_nop 7\n\ts_nop 7" : "+v"(acc[i]));
#pragma unroll
  for (int i = 0; i < NT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < NT; i += WAVES) {
    f32x4 v = red[0][i][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += red[k][i][lane];
    store_out<O>(l, r, t0 + 16 * i + n, rb * kTileRows + 4 * quad, v);
  }
}

template <typename T, typename O>
hipError_t run(const LinearDev& l, const dmh_linear_rows& r, hipStream_t st) {
  const auto few = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    const dim3 grid(l.row_blocks, (r.rows + 16 * NT - 1) / (16 * NT));
    k_linear_few<T, O, NT, 4><<<grid, 256, 0, st>>>(l, r);
    return hipGetLastError();
  };
  if (r.rows <= 16) return few(std::integral_constant<int, 1>{});
  if (r.rows <= 32) return few(std::integral_constant<int, 2>{});
  return few(std::integral_constant<int, 4>{});
}

}  // namespace

hipError_t launch_linear_pack(const uint16_t* scales, const uint8_t* packed, int n, int k, int group,
                              uint8_t* nib, uint16_t* sc, unsigned long long* vkey, hipStream_t st) {
  const int chunks = linear_chunks(k);
  const int64_t lanes = (int64_t)linear_row_blocks(n) * chunks * 64;
  k_linear_pack<<<(unsigned)((lanes + 255) / 256), 256, 0, st>>>(scales, packed, n, k, group, nib, sc,
                                                                chunks, lanes, vkey);
  return hipGetLastError();
}

hipError_t launch_linear(const LinearDev& l, const dmh_linear_rows& r, hipStream_t st) {
  const bool f32 = r.out_dtype == DMH_DTYPE_F32;
  if (r.dtype == DMH_DTYPE_F32) return run<float, float>(l, r, st);
  if (r.dtype == DMH_DTYPE_F16) return f32 ? run<half_t, float>(l, r, st) : run<half_t, half_t>(l, r, st);
  return f32 ? run<bf16_t, float>(l, r, st) : run<bf16_t, bf16_t>(l, r, st);
}

}  // namespace dm
