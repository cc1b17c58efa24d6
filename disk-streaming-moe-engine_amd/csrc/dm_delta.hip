// dm_delta.hip -- the gated delta rule 64 rows at a time.
//
// With G the running sum of the log decays inside a chunk of 64 rows, khat and
// qhat the normalised (and scaled) keys and queries, S the state before it:
//   A_ij = beta_i (khat_i . khat_j) e^(G_i - G_j)   for j < i, else 0
//   U    = (I + A)^-1 diag(beta) (V - diag(e^G) Khat S)
//   O    = diag(e^G) Qhat S + [(qhat_i . khat_j) e^(G_i - G_j), j <= i] U
//   S'   = e^G_last S + (diag(e^(G_last - G)) Khat)^T U
// k_delta_prep makes what does not depend on S, for all chunks at once; then
// k_delta_chunks walks each head's chunks in order.
//
// Precision.  The state is fp32 and so are all sums; products run on the bf16
// matrix cores with every fp32 factor split into bf16 parts of 8 bits each: x =
// x0 + x1 + x2 to 2^-26, and the products of parts i and j with i + j < 3 kept (all
// 24 bits).  Keys and queries enter the products as they came (one part for bf16
// rows, two for f16, three for f32), their norms and decays as factors of rows in
// fp32.  Sums of log decays are
// kept in 64 bits: e^(G_i - G_j) of two large sums would lose what the
// difference holds.
#include <algorithm>
#include <type_traits>

#include "dm_mixer_device.h"

namespace dm {
namespace {

constexpr int kChunk = kDeltaChunk;
constexpr int kPad = 68;  // floats per row of a 64 x 64 matrix in LDS
// 16 x 32 tiles of a lower triangular 64 x 64 matrix: rows 0-15 and 16-31 have
// one, the others two
constexpr int kTiles = 6;
__device__ __forceinline__ int tile_of(int row_blk, int half) {
  return row_blk < 2 ? row_blk : 2 * row_blk - 2 + half;
}

constexpr size_t frag_bytes(int n) { return (size_t)n * 1024; }  // 64 lanes of 16 bytes

// What k_delta_prep leaves per chunk: for each value head (I + A)^-1 diag(beta)
// and the query-key matrix in three parts each, and the rows' factors; for each
// key head K^T, K and Q (copied: rows a power of two apart meet in the same
// channels of the L2, and read in place they hold up all the other loads: a tenth
// of the chain's time for 2048 rows of 32 heads).
// The key dimension comes in steps of a matrix product, SW dimensions each, of
// which lane group g of a factor has SW / 4 in a row.  In the state, whose tiles
// of 16 rows are a right factor as they stand, row 4 g + i of a step's first tile
// is the lane group's dimension i, of its second one 4 + i.  At 64 dimensions a
// wave of the chain has only one tile, and its step is half empty.
template <int DKT, int NPK>
struct Layout {
  static constexpr int SW = DKT == 64 ? 16 : 32;
  static constexpr int KS = DKT / SW;
  // the dimension that row m of tile t is
  static __device__ __forceinline__ int dim(int t, int m) {
    return SW == 32 ? 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3) : 16 * t + m;
  }
  static constexpr size_t qk = frag_bytes(kTiles * 3);
  static constexpr size_t rows = qk + frag_bytes(kTiles * 3);
  static constexpr size_t v_head = rows + 4 * kChunk * sizeof(float);
  static constexpr size_t k_rows = frag_bytes(DKT / 16 * 2 * NPK);
  static constexpr size_t q_rows = k_rows + frag_bytes(4 * KS * NPK);
  static constexpr size_t k_head = q_rows + frag_bytes(4 * KS * NPK);
};

struct ChunkWork {
  uint8_t* v_heads;
  uint8_t* k_heads;
  int rank0, count;  // the chunks of this pass, counted over all long sequences
  int min_rows;      // sequences of fewer rows are not taken
};

__device__ __forceinline__ int chunks_of(const SeqDev& s, int i, int min_rows) {
  const SeqRange r = seq_range(s, i, false);
  const int n = r.end - r.begin;
  return r.live && n >= min_rows ? (n + kChunk - 1) / kChunk : 0;
}

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// A matrix product's result may be read only some cycles after the product was
// issued, which the compiler sees to by counting instructions.  It does not do
// so where a branch lies between the two: there, results of a wave that took the
// branch were read before they were written.  So wherever a branch or the end of
// a loop may come between a product and the first other use of its result, the
// result passes through here: 16 cycles, more than any product used takes.
__device__ __forceinline__ void settle(f32x4& c) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c)); }

// Several results with one wait: all of them pass through before it, as they are
// made, and behind it, before they are used (some 45 cycles for each wait less).
template <int A, int B>
__device__ __forceinline__ void settle(f32x4 (&c)[A][B]) {
#pragma unroll
  for (int i = 0; i < A * B; ++i) asm volatile("" : "+v"(c[i / B][i % B]));
  settle(c[0][0]);
#pragma unroll
  for (int i = 0; i < A * B; ++i) asm volatile("" : "+v"(c[i / B][i % B]));
}

// Four fp32 values as NP parts of four bf16.
template <int NP>
__device__ __forceinline__ void split4(f32x4 v, uint2 (&p)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    p[i] = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    if (i + 1 < NP) {
      v[0] -= bf16lo(p[i].x);
      v[1] -= bf16hi(p[i].x);
      v[2] -= bf16lo(p[i].y);
      v[3] -= bf16hi(p[i].y);
    }
  }
}
template <int NP>
__device__ __forceinline__ void split8(const float (&v)[8], uint4 (&p)[NP]) {
  uint2 lo[NP], hi[NP];
  split4<NP>(f32x4{v[0], v[1], v[2], v[3]}, lo);
  split4<NP>(f32x4{v[4], v[5], v[6], v[7]}, hi);
#pragma unroll
  for (int i = 0; i < NP; ++i) p[i] = make_uint4(lo[i].x, lo[i].y, hi[i].x, hi[i].y);
}

// c += a b over the parts whose product counts.
template <int NPA, int NPB>
__device__ __forceinline__ f32x4 mfma_parts(const bf16x8 (&a)[NPA], const bf16x8 (&b)[NPB],
                                            f32x4 c) {
#pragma unroll
  for (int i = 0; i < NPA; ++i)
#pragma unroll
    for (int j = 0; j < NPB; ++j)
      if (i + j < 3) c = mfma16(a[i], b[j], c);
  return c;
}

__device__ __forceinline__ bf16x8 load_frag(const void* base, size_t frag, int lane) {
  return *reinterpret_cast<const bf16x8*>(static_cast<const uint8_t*>(base) + frag * 1024 +
                                          lane * 16);
}
__device__ __forceinline__ void store_frag(void* base, size_t frag, int lane, uint4 v) {
  *reinterpret_cast<uint4*>(static_cast<uint8_t*>(base) + frag * 1024 + lane * 16) = v;
}

// ---- what does not depend on the state ---------------------------------------------
// One workgroup per chunk and HB value heads of a key head (two, where there
// are; their keys' products are the same up to factors); wave w has rows 16 w ..
// 16 w + 15.  Products of rows with rows are taken transposed: four consecutive
// keys of one row per lane are a piece of the left factor that k_delta_chunks
// loads, and of a row of A.  T = (I + A)^-1 comes by substitution in the 16 x 16
// diagonal blocks (a row per lane) and, as -T22 A21 T11, in the blocks below
// them, 16 and then 32 wide, on the fp32 matrix cores: products of powers of A
// would take fewer steps and lose all precision for keys that resemble each
// other.
// With few chunks the way through loads, products and substitution bounds it, so
// everything is loaded at once, unconditionally, and T takes A's place in LDS (57
// KB at 128 dimensions in bf16: two workgroups per CU): 2048 rows of 16 key and 32
// value heads in 18.5 us.  With many, what it writes does: 516 MB of factors for
// 16384 rows in 133 us, 5 TB/s with what it reads.
// The first `short_blocks` workgroups take the short sequences, row by row: they
// have the longest way, and no chunk waits for them.
template <typename T, int DKT, int NPK, int HB>
__global__ __launch_bounds__(256) void k_delta_prep(dmh_gated_delta d, SeqDev s, ChunkWork cw,
                                                    unsigned short_blocks) {
  if (blockIdx.x < short_blocks) {
    delta_rows<T, DKT / 8>(d, s, cw.min_rows - 1, blockIdx.x);
    return;
  }
  using L = Layout<DKT, NPK>;
  constexpr int KS = L::KS;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rep = d.v_heads / d.k_heads, groups = (rep + HB - 1) / HB;
  const int block = blockIdx.x - short_blocks, local = block / (d.k_heads * groups);
  const int unit = block - local * d.k_heads * groups;
  const int kh = unit / groups, group = unit - kh * groups;
  const int h0 = kh * rep + group * HB, heads = min(HB, rep - group * HB);

  constexpr int kMat = kChunk * kPad;
  constexpr int kPiece = L::SW / 2;  // bytes of a lane's part of a step: no empty half in LDS
  __shared__ __align__(16) uint8_t kfrag[4 * KS * NPK * 64 * kPiece];
  __shared__ __align__(16) uint8_t qfrag[frag_bytes(KS * NPK)];  // the last rows' queries
  __shared__ __align__(16) float am[HB * kMat];  // A, and then T in its place
  __shared__ __align__(16) float2 decay[HB][kChunk];
  __shared__ __align__(16) float beta_s[HB][kChunk], rk_s[kChunk];
  __shared__ float rq_s[kChunk];

  // the chunk: sequence and place in it
  const int rank = cw.rank0 + local;
  int begin = -1, end = 0;
  for (int j0 = 0, base = 0; j0 < s.num && begin < 0; j0 += 64) {
    const int own = j0 + lane < s.num ? chunks_of(s, j0 + lane, cw.min_rows) : 0;
    int sum = own;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int v = __shfl_up(sum, m);
      if (lane >= m) sum += v;
    }
    const unsigned long long past = __ballot(base + sum > rank);
    if (past) {
      const int at = __builtin_ctzll(past);
      begin = s.off[j0 + at] + (rank - base - __shfl(sum - own, at)) * kChunk;
      end = s.off[j0 + at + 1];
    }
    base += __shfl(sum, 63);
  }
  begin = __builtin_amdgcn_readfirstlane(begin);
  if (begin < 0) return;
  const int rows = min(__builtin_amdgcn_readfirstlane(end) - begin, kChunk);
  uint8_t* const vws = cw.v_heads + ((size_t)local * d.v_heads + h0) * L::v_head;
  uint8_t* const kws = cw.k_heads + ((size_t)local * d.k_heads + kh) * L::k_head;

  // the rows' values and gates, all loads at once; of a row or column that is not
  // there, another's, cleared below
  const int row = 16 * w + n;
  const bool row_in = row < rows;
  // (a wave without a head: another one's gates)
  const RawGates<T> raw = load_gates<T>(d, begin + min(lane, rows - 1), h0 + min(w, heads - 1));
  float kv[KS][8], qv[KS][8];
  {
    const int64_t at = begin + min(row, rows - 1);
    const T* kp = static_cast<const T*>(d.k) + at * d.k_stride + kh * d.k_dim;
    const T* qp = static_cast<const T*>(d.q) + at * d.q_stride + kh * d.k_dim;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      constexpr int N = L::SW / 4;
      const int c = L::SW * st + N * g < d.k_dim ? L::SW * st + N * g : 0;
      float kn[N], qn[N];
      load_f32<N>(kp + c, kn);
      load_f32<N>(qp + c, qn);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        kv[st][i] = kn[i];
        qv[st][i] = qn[i];
      }
    }
  }
  // gates and decays of head h0 + w, a row per lane; e^-10000 is 0 as well as
  // e^-inf, and does not turn into NaN in a difference
  double since = 0.0;
  if (w < heads) {
    const Gates gt = gates_of(d, raw);
    since = lane < rows ? (double)gt.log_decay : 0.0;
    if (since < -10000.0) since = -10000.0;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const double v = __shfl_up(since, m);
      if (lane >= m) since += v;
    }
    // in powers of two and two fp32 parts: a difference of two sums is then
    // exact to its own last bit
    const double e2 = since * 0x1.71547652b82fep+0;
    const float hi = (float)e2;
    decay[w][lane] = make_float2(hi, (float)(e2 - (double)hi));
    beta_s[w][lane] = lane < rows ? gt.beta : 0.0f;
  }

  // norms and parts of keys and queries
  bf16x8 qf[KS][NPK], kf[KS][NPK];
  float ksum = 0.0f, qsum = 0.0f;
#pragma unroll
  for (int st = 0; st < KS; ++st) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = row_in && i < L::SW / 4 && L::SW * st + L::SW / 4 * g < d.k_dim;
      kv[st][i] = in ? kv[st][i] : 0.0f;
      qv[st][i] = in ? qv[st][i] : 0.0f;
      ksum = __builtin_fmaf(kv[st][i], kv[st][i], ksum);
      qsum = __builtin_fmaf(qv[st][i], qv[st][i], qsum);
    }
    uint4 kp4[NPK], qp4[NPK];
    split8<NPK>(kv[st], kp4);
    split8<NPK>(qv[st], qp4);
#pragma unroll
    for (int p = 0; p < NPK; ++p) {
      if (w == 3) store_frag(qfrag, st * NPK + p, lane, qp4[p]);
      if constexpr (kPiece == 16)
        store_frag(kfrag, (w * KS + st) * NPK + p, lane, kp4[p]);
      else
        *reinterpret_cast<uint2*>(kfrag + (((w * KS + st) * NPK + p) * 64 + lane) * 8) =
            make_uint2(kp4[p].x, kp4[p].y);
      kf[st][p] = __builtin_bit_cast(bf16x8, kp4[p]);
      qf[st][p] = __builtin_bit_cast(bf16x8, qp4[p]);
      if (group == 0) {
        store_frag(kws + L::k_rows, (w * KS + st) * NPK + p, lane, kp4[p]);
        store_frag(kws + L::q_rows, (w * KS + st) * NPK + p, lane, qp4[p]);
      }
    }
  }
  ksum += __shfl_xor(ksum, 16);
  qsum += __shfl_xor(qsum, 16);
  ksum += __shfl_xor(ksum, 32);
  qsum += __shfl_xor(qsum, 32);
  const float rk = d.qk_norm ? 1.0f / sqrtf(ksum + d.eps) : 1.0f;
  const float rq = d.qk_norm ? d.scale / sqrtf(qsum + d.eps) : d.scale;
  if (g == 0) {
    rk_s[row] = rk;
    rq_s[row] = rq;
  }
  __syncthreads();

  const auto load_key = [&](int rb, int st, int p) -> bf16x8 {
    const int at = ((rb * KS + st) * NPK + p) * 64 + lane;
    if constexpr (kPiece == 16) {
      return load_frag(kfrag, (rb * KS + st) * NPK + p, lane);
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(kfrag + at * 8);
      return __builtin_bit_cast(bf16x8, make_uint4(v.x, v.y, 0, 0));
    }
  };
  // K^T: the products of the wave's rows with unit vectors give a dimension's
  // values for four rows in a row, exactly
  if (group == 0) {
#pragma unroll
    for (int t = 0; t < DKT / 16; ++t) {
      bf16x8 unit;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        unit[e] = (__bf16)(e < L::SW / 4 && L::SW / 4 * g + e == L::dim(t, n) % L::SW ? 1.0f : 0.0f);
#pragma unroll
      for (int p = 0; p < NPK; ++p) {
        f32x4 k4 = mfma16(kf[L::SW == 32 ? t >> 1 : t][p], unit, f32x4{});
        uint2 v[1];
        split4<1>(k4, v);
        *reinterpret_cast<uint2*>(kws + ((t * 2 + (w >> 1)) * NPK + p) * 1024 +
                                  (n + 16 * ((w & 1) * 2 + (g >> 1))) * 16 + (g & 1) * 8) = v[0];
      }
    }
  }

  // A and the query-key matrix: wave 0 takes the first two of the last rows' four
  // tiles, besides its own one
  const auto tiles = [&](int rb, int j0, int j1, float rk_row, float rq_row) {
    const int qrow = 16 * rb + n;
    const bool here = qrow < rows;
    for (int j = j0; j <= j1; ++j) {
      f32x4 kk = {}, kq = {};
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        bf16x8 b[NPK];
#pragma unroll
        for (int p = 0; p < NPK; ++p) b[p] = load_key(j, st, p);
        kk = mfma_parts(b, kf[st], kk);
        kq = mfma_parts(b, qf[st], kq);
      }
      settle(kk);
      settle(kq);
      const int c0 = 16 * j + 4 * g;  // the lane's keys c0 .. c0 + 3 of row qrow
      const f32x4 rkc = *reinterpret_cast<const f32x4*>(rk_s + c0);
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        if (i >= heads) break;
        const float2 dr = decay[i][qrow];
        const float bk = beta_s[i][qrow] * rk_row;
        f32x4 a, q;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 dc = decay[i][c0 + r];
          const float e = __builtin_amdgcn_exp2f((dr.x - dc.x) + (dr.y - dc.y)) * rkc[r];
          a[r] = c0 + r < qrow && here ? bk * (e * kk[r]) : 0.0f;
          q[r] = c0 + r <= qrow && here ? rq_row * (e * kq[r]) : 0.0f;
        }
        *reinterpret_cast<f32x4*>(am + i * kMat + qrow * kPad + c0) = a;
        uint2 p[3];
        split4<3>(q, p);
        uint8_t* const to = vws + i * L::v_head + L::qk +
                            (n + 16 * ((j & 1) * 2 + (g >> 1))) * 16 + (g & 1) * 8;
#pragma unroll
        for (int o = 0; o < 3; ++o)
          *reinterpret_cast<uint2*>(to + (tile_of(rb, j >> 1) * 3 + o) * 1024) = p[o];
      }
    }
  };
  tiles(w, w == 3 ? 2 : 0, w, rk, rq);
  if (w == 0) {
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int p = 0; p < NPK; ++p) {
        kf[st][p] = load_key(3, st, p);
        qf[st][p] = load_frag(qfrag, st * NPK + p, lane);
      }
    tiles(3, 0, 1, rk_s[48 + n], rq_s[48 + n]);
  }
  if ((w & 1) == 0) {  // the empty halves of the tiles on the diagonal
    for (int i = 0; i < heads; ++i) {
      *reinterpret_cast<f32x4*>(am + i * kMat + row * kPad + 16 * w + 16 + 4 * g) = f32x4{};
      uint8_t* const to = vws + i * L::v_head + L::qk + (n + 32 + 16 * (g >> 1)) * 16 + (g & 1) * 8;
#pragma unroll
      for (int o = 0; o < 3; ++o)
        *reinterpret_cast<uint2*>(to + (tile_of(w, w >> 1) * 3 + o) * 1024) = make_uint2(0, 0);
    }
  }
  __syncthreads();

  // the diagonal blocks of T from T (I + A) = I, a row per lane, a head per group
  // of lanes
  {
    float* const a = am + (HB == 2 ? g & 1 : 0) * kMat + 16 * w * kPad + 16 * w;
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = j == n ? 1.0f : 0.0f;
#pragma unroll
    for (int m = 15; m > 0; --m)
#pragma unroll
      for (int j = 0; j < m; ++j) x[j] = __builtin_fmaf(-x[m], a[m * kPad + j], x[j]);
    // (in place: the wave has read its block)
    if (g < HB) {
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<f32x4*>(a + n * kPad + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    }
  }
  __syncthreads();
  // block (bi, bj) from the left; C tiles as right factors: step r of a product
  // over 16 takes row 4 g + r of it
  const auto left = [&](const float* m, int bi, int bj, int k) {
    return m[(16 * bi + n) * kPad + 16 * bj + k];
  };
  if (w < 2 * HB) {
    float* const a = am + (w >> 1) * kMat;
    const int b0 = 2 * (w & 1), b1 = b0 + 1;
    f32x4 x = {}, y = {};
#pragma unroll
    for (int st = 0; st < 4; ++st)
      x = mfma_f32(left(a, b1, b0, 4 * st + g), a[(16 * b0 + 4 * st + g) * kPad + 16 * b0 + n], x);
#pragma unroll
    for (int r = 0; r < 4; ++r) y = mfma_f32(left(a, b1, b1, 4 * g + r), x[r], y);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[(16 * b1 + 4 * g + r) * kPad + 16 * b0 + n] = -y[r];
  }
  __syncthreads();
  // the 2 x 2 blocks below: with two heads, a wave has a long and a short one
  const int fi = HB == 2 ? w & 1 : 0;
  float* const fa = am + fi * kMat;
  f32x4 fy[HB] = {};
#pragma unroll
  for (int task = 0; task < HB; ++task) {
    const int bi = HB == 2 ? (task == 0) : w >> 1, bj = HB == 2 ? (w >> 1) ^ task : w & 1;
    for (int k = 0; k <= bi; ++k) {
      f32x4 x = {};
      for (int kk = bj; kk < 2; ++kk)
#pragma unroll
        for (int st = 0; st < 4; ++st)
          x = mfma_f32(left(fa, 2 + k, kk, 4 * st + g),
                       fa[(16 * kk + 4 * st + g) * kPad + 16 * bj + n], x);
      settle(x);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        fy[task] = mfma_f32(left(fa, 2 + bi, 2 + k, 4 * g + r), x[r], fy[task]);
    }
    settle(fy[task]);
  }
  __syncthreads();
#pragma unroll
  for (int task = 0; task < HB; ++task) {
    const int bi = HB == 2 ? (task == 0) : w >> 1, bj = HB == 2 ? (w >> 1) ^ task : w & 1;
#pragma unroll
    for (int r = 0; r < 4; ++r) fa[(32 + 16 * bi + 4 * g + r) * kPad + 16 * bj + n] = -fy[task][r];
  }
  __syncthreads();

  // T diag(beta) in parts, as a left factor
  for (int q = tid; q < heads * kTiles * 64; q += 256) {
    const int i = q / (kTiles * 64), tile = (q >> 6) % kTiles;  // (lane is q & 63)
    const int blk = tile < 2 ? tile : (tile + 2) / 2, half = tile < 2 ? 0 : tile & 1;
    const float* const t = am + i * kMat + (16 * blk + n) * kPad + 32 * half + 8 * g;
    const float* const b = beta_s[i] + 32 * half + 8 * g;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[e] * b[e];
    uint4 vp[3];
    split8<3>(v, vp);
#pragma unroll
    for (int p = 0; p < 3; ++p) store_frag(vws + i * L::v_head, tile * 3 + p, lane, vp[p]);
  }
  if (w < heads) {
    float* f = reinterpret_cast<float*>(vws + w * L::v_head + L::rows);
    const bool in = lane < rows;
    const double last = __shfl(since, 63);
    const float grown = expf((float)since);
    f[lane] = in ? grown * rk_s[lane] : 0.0f;
    f[kChunk + lane] = in ? grown * rq_s[lane] : 0.0f;
    f[2 * kChunk + lane] = in ? expf((float)(last - since)) * rk_s[lane] : 0.0f;
    f[3 * kChunk + lane] = expf((float)last);
  }
}

// ---- the chunks of a head, in order ----------------------------------------------
// One workgroup per head and 16 NC columns of its state, eight waves.  Waves 0-3
// walk the chain from chunk to chunk: each holds the rows of DKT / 64 tiles of
// 16 of the state in registers, where they are a right factor as they stand, and
//   1  P   of all 64 rows over its part of the key dimension, summed through LDS,
//   2  R = V - e^G P and
//   3  U = T R of rows 16 w .. 16 w + 15 (rows of R up to its own),
//   4  its rows of S' = e^G_last S + K^T U,
// with a barrier behind 1, 2 and 3.  Waves 4-7 bring the factors of the chain
// from memory into LDS, without registers where they fit (M::stage), and make the
// outputs of 16 rows each, O = e^G Q S + (Q K^T) U, from the parts of S and U that
// the others leave in LDS.  So the chain never waits for memory: with its loads
// its own, it took a third longer: their issue, 64 bytes a cycle and CU.  What
// bounds it is the way from barrier to barrier, 1.9 us a chunk with one column tile
// (2048 rows of 32 heads: 60 us) and 2.8 to 3.2 with two; the matrix cores are busy
// 18 to 20% of it.  Outputs from two parts instead of three take 0.2 us a chunk less
// and lose what lies below 2^-17 of their terms.  A wave for all rows of a tile
// needs no way through LDS, but its 132 products and their splits alone take 2.3 us.
// A factor is used in one step only, so one copy of each is enough: the next
// chunk's K arrives from the barrier behind step 1 to the one behind 3, K^T as
// well, T from there to the next one.  Where they do not fit, the chain loads K,
// T and K^T into registers itself.
constexpr size_t kLds = 160 * 1024 - 512;

template <int DKT, int NC, int NPK>
struct Shared {
  using L = Layout<DKT, NPK>;
  static constexpr int KS = L::KS;
  static constexpr size_t s = 0;                               // S: [step][column tile][part]
  static constexpr size_t p = s + frag_bytes(KS * NC * 3);     // P: [column tile][row block][wave]
  static constexpr size_t r = p + frag_bytes(16 * NC);         // R: [half][column tile][part]
  static constexpr size_t u = r + frag_bytes(3 * 2 * NC);      // U
  static constexpr size_t g = u + frag_bytes(3 * 2 * NC);      // U as S' takes it
  static constexpr size_t v = g + frag_bytes(3 * 2 * NC);      // V: [row][column] fp32
  static constexpr int vp = 16 * NC + 4;  // a row's pitch: four rows apart, other banks
  static constexpr size_t f = v + (size_t)kChunk * vp * 4;     // factors of rows, twice
  static constexpr size_t common = f + 2 * 3 * kChunk * 4;
  static constexpr size_t k = common;                          // K, T, K^T as k_delta_prep left them
  static constexpr size_t t = k + frag_bytes(4 * KS * NPK);
  static constexpr size_t kt = t + frag_bytes(kTiles * 3);
  static constexpr size_t all = kt + frag_bytes(DKT / 16 * 2 * NPK);
  static constexpr bool stage = all <= kLds;
  static constexpr size_t bytes = stage ? all : common;
};

template <typename T, int DKT, int NC, int NPK>
__global__ __launch_bounds__(512) void k_delta_chunks(dmh_gated_delta d, SeqDev s, ChunkWork cw) {
  using L = Layout<DKT, NPK>;
  using M = Shared<DKT, NC, NPK>;
  constexpr int KS = L::KS, KW = KS / 4, NT = DKT / 64;
  constexpr int kKT = DKT / 16 * 2 * NPK;  // fragments of K^T
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3;
  const int n = lane & 15, g = lane >> 4;
  // the column blocks of a head on one XCD (workgroups go round the XCDs): they
  // read the same factors
  const int ncb = (d.v_dim + 16 * NC - 1) / (16 * NC);
  const int unit = blockIdx.x / (8 * ncb) * 8 + (blockIdx.x & 7), cb = (blockIdx.x >> 3) % ncb;
  if (unit >= s.num * d.v_heads) return;
  const int seq = unit / d.v_heads, h = unit - seq * d.v_heads;
  const int kh = h / (d.v_heads / d.k_heads);
  const SeqRange r = seq_range(s, seq, false);
  if (!r.live || r.end - r.begin < cw.min_rows) return;

  __shared__ __align__(16) uint8_t lds[M::bytes];
  __shared__ int before;
  uint8_t* const sb = lds + M::s;
  uint8_t* const pb = lds + M::p;
  uint8_t* const rb = lds + M::r;
  uint8_t* const ub = lds + M::u;
  uint8_t* const gb = lds + M::g;
  float* const vb = reinterpret_cast<float*>(lds + M::v);
  float* const fb = reinterpret_cast<float*>(lds + M::f);  // [chunk & 1][R | U | fade][row]

  // chunks of the sequences before this one
  if (tid == 0) before = 0;
  __syncthreads();
  int mine = 0;
  for (int j = tid; j < seq; j += 512) mine += chunks_of(s, j, cw.min_rows);
  if (mine) atomicAdd(&before, mine);
  __syncthreads();
  // (of this pass, counted in this sequence)
  const int first = cw.rank0 - __builtin_amdgcn_readfirstlane(before);
  const int len = r.end - r.begin;
  const int c0 = max(first, 0), c1 = min((len + kChunk - 1) / kChunk, first + cw.count);
  if (c0 >= c1) return;

  // Loads have a uniform base per chunk and 32-bit offsets of the lane that hold
  // for all chunks, and are not conditional, so that none waits for another.
  size_t vws_at = ((size_t)(c0 - first) * d.v_heads + h) * L::v_head;
  size_t kws_at = ((size_t)(c0 - first) * d.k_heads + kh) * L::k_head;
  const uint8_t *vws = cw.v_heads + vws_at, *kws = cw.k_heads + kws_at;
  const auto step = [&](int c) {  // from chunk c to the next one's factors (the last one's again)
    vws_at += c + 1 < c1 ? (size_t)d.v_heads * L::v_head : 0;
    kws_at += c + 1 < c1 ? (size_t)d.k_heads * L::k_head : 0;
    asm("" : "+s"(vws_at), "+s"(kws_at));  // one base each: not one for every load
    vws = cw.v_heads + vws_at;
    kws = cw.k_heads + kws_at;
  };
  const uint32_t at16 = lane * 16;
  const auto frag = [](const uint8_t* base, uint32_t at) {
    return *reinterpret_cast<const bf16x8*>(base + at);
  };
  const bool two = w >= 2;  // rows 32 on: two tiles of the triangular factors
  const auto get = [&](const uint8_t* base, int st, int nc, auto& b) {
    constexpr int NP = sizeof(b) / sizeof(b[0]);
#pragma unroll
    for (int i = 0; i < NP; ++i) b[i] = load_frag(base, (st * NC + nc) * NP + i, lane);
  };

  if (wave >= 4) {  // ---- loads, and the outputs of rows 16 w .. 16 w + 15
    // O and V are held transposed: a row (n) and four columns per lane
    const int col = cb * 16 * NC + 4 * g, row = 16 * w + n;
    const uint32_t q_at = (uint32_t)L::q_rows + w * KS * NPK * 1024 + at16;
    const uint32_t a_at[2] = {(uint32_t)L::qk + tile_of(w, 0) * 3 * 1024 + at16,
                              (uint32_t)L::qk + tile_of(w, two) * 3 * 1024 + at16};
    // the rows' factors in one load: of lane group 0 for R, 1 for O, 2 for U, 3 fade
    const uint32_t f_at = (uint32_t)L::rows + (g * kChunk + (g < 3 ? row : 0)) * 4;
    T* const o0 = static_cast<T*>(d.o) + (int64_t)(r.begin + row) * d.o_stride + h * d.v_dim + col;
    const T* const v0 = static_cast<const T*>(d.v) + (int64_t)r.begin * d.v_stride + h * d.v_dim;
    bf16x8 qf[KS][NPK], af[2][3];
    float f;
    Vec<T, 4> v4[NC];  // (as it comes: a conversion would wait for it)
    const auto load_q = [&] {
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int i = 0; i < NPK; ++i) qf[st][i] = frag(kws, q_at + (st * NPK + i) * 1024);
    };
    const auto load_a = [&] {
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < 3; ++i) af[st][i] = frag(vws, a_at[st] + i * 1024);
    };
    const auto load_v = [&](int c) {
      f = *reinterpret_cast<const float*>(vws + f_at);
      // (a row or columns that are not there: the chunk's first)
      const T* const vp = v0 + ((int64_t)c * kChunk + (c * kChunk + row < len ? row : 0)) * d.v_stride;
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        const T* const at = vp + (col + 16 * nc < d.v_dim ? col + 16 * nc : 0);
        v4[nc] = load_raw<4>(at);
      }
    };
    const auto put_v = [&](int c) {
      const bool in = c * kChunk + row < len;
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = in ? (float)v4[nc][i] : 0.0f;
        }
        *reinterpret_cast<f32x4*>(vb + row * M::vp + 16 * nc + 4 * g) = x;
      }
      if (g != 1) fb[((c & 1) * 3 + (g == 0 ? 0 : g - 1)) * kChunk + row] = f;
    };
    // fragments of the chain, a quarter of them per wave
    const auto bring = [&](const uint8_t* from, size_t to, int count) {
#pragma unroll
      for (int i = 0; i < (count + 3) / 4; ++i) {
        const int j = 4 * i + w;
        if (count % 4 == 0 || j < count) dma16_lds(from + j * 1024 + at16, lds_u32(lds + to + j * 1024));
      }
    };
    load_q();
    load_a();
    load_v(c0);
    if constexpr (M::stage) {
      bring(kws + L::k_rows, M::k, 4 * KS * NPK);
      bring(vws, M::t, kTiles * 3);
    }
    put_v(c0);
    wait_vm();
    __builtin_amdgcn_s_waitcnt(0x0F70);  // (vmcnt 0, which the compiler takes note of)
    lds_barrier();
    for (int c = c0; c < c1; ++c) {
      const float pq = __shfl(f, 16 + n);
      lds_barrier();  // 1
      const uint8_t* const kt_from = kws;
      step(c);
      if constexpr (M::stage) {
        bring(kws + L::k_rows, M::k, 4 * KS * NPK);
        bring(kt_from, M::kt, kKT);
      }
      load_v(min(c + 1, c1 - 1));
      lds_barrier();  // 2
      f32x4 o[NC][2] = {};
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          bf16x8 b[3];
          get(sb, st, nc, b);
          o[nc][st & 1] = mfma_parts(b, qf[st], o[nc][st & 1]);
        }
      settle(o);
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) o[nc][0] = (o[nc][0] + o[nc][1]) * pq;
      load_q();
      // K and K^T are there: only what was issued behind them, Q, may be under way
      if constexpr (M::stage) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KS * NPK) : "memory");
      lds_barrier();  // 3
      if constexpr (M::stage) bring(vws, M::t, kTiles * 3);
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        bf16x8 b[3];
        get(ub, 0, nc, b);
        o[nc][0] = mfma_parts(b, af[0], o[nc][0]);
        if (two) {
          get(ub, 1, nc, b);
          o[nc][0] = mfma_parts(b, af[1], o[nc][0]);
        }
      }
      settle(o);
      load_a();
      put_v(c + 1);
      if (c * kChunk + row < len) {
        T* const op = o0 + (int64_t)c * kChunk * d.o_stride;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          const float y[4] = {o[nc][0][0], o[nc][0][1], o[nc][0][2], o[nc][0][3]};
          if (col + 16 * nc < d.v_dim) store_f32<4>(op + 16 * nc, y);
        }
      }
      // T is there: only what was issued behind it, the stores, may be under way
      if constexpr (M::stage) asm volatile("s_waitcnt vmcnt(1)" ::: "memory");
    }
    return;
  }

  // ---- the chain
  __builtin_amdgcn_s_setprio(3);
  // an element of a C tile: row 4 g + i of 16, column n
  const int col = cb * 16 * NC + n;
  float* const sp = d.state + ((size_t)r.slot * d.v_heads + h) * d.k_dim * d.v_dim + col;
  f32x4 S[NT][NC];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dim = L::dim(NT * w + t, 4 * g + i);
        const bool in = dim < d.k_dim && col + 16 * nc < d.v_dim;
        S[t][nc][i] = in && !(c0 == 0 && r.fresh) ? sp[(size_t)dim * d.v_dim + 16 * nc] : 0.0f;
      }
  // row block t of a right factor to LDS
  const auto put = [&](uint8_t* base, int t, int nc, f32x4 x) {
    uint2 p[3];
    split4<3>(x, p);
    const int at = (n + 16 * ((t & 1) * 2 + (g >> 1))) * 16 + (g & 1) * 8;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      *reinterpret_cast<uint2*>(base + (((t >> 1) * NC + nc) * 3 + i) * 1024 + at) = p[i];
  };

  // a factor: from LDS where a step begins, or into registers for the next chunk
  bf16x8 kf[4][KW][NPK], tf[2][3], gf[NT][2][NPK];
  const auto take_k = [&](const uint8_t* base) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < KW * NPK; ++i)
        kf[b][i / NPK][i % NPK] = frag(base, (b * KS + w * KW) * NPK * 1024 + i * 1024 + at16);
  };
  const auto take_t = [&](const uint8_t* base) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      tf[0][i] = frag(base, tile_of(w, 0) * 3 * 1024 + i * 1024 + at16);
      if (two || !M::stage) tf[1][i] = frag(base, tile_of(w, two) * 3 * 1024 + i * 1024 + at16);
    }
  };
  const auto take_kt = [&](const uint8_t* base) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2 * NPK; ++i)
        gf[t][i / NPK][i % NPK] = frag(base, (NT * w + t) * 2 * NPK * 1024 + i * 1024 + at16);
  };
  if constexpr (!M::stage) {
    take_k(kws + L::k_rows);
    take_t(vws);
    take_kt(kws);
    // All loads here (vmcnt 0): the waits that the compiler places in the loop
    // would otherwise have to hold for the order of these as well, and wait for
    // every load there.
    __builtin_amdgcn_s_waitcnt(0x0F70);
  }
  lds_barrier();
  if constexpr (M::stage) take_k(lds + M::k);
  for (int c = c0; c < c1; ++c) {
    const float* const fc = fb + (c & 1) * 3 * kChunk;
    f32x4 p[NC][4] = {};
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int kw = 0; kw < KW; ++kw) {
        uint2 lo[3], hi[3] = {};
        split4<3>(S[NT == 1 ? 0 : 2 * kw][nc], lo);
        if constexpr (NT > 1) split4<3>(S[2 * kw + 1][nc], hi);
        bf16x8 b[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const uint4 q = make_uint4(lo[i].x, lo[i].y, hi[i].x, hi[i].y);
          store_frag(sb, ((w * KW + kw) * NC + nc) * 3 + i, lane, q);
          b[i] = __builtin_bit_cast(bf16x8, q);
        }
#pragma unroll
        for (int i = 0; i < NPK; ++i)  // (part by part: four sums in turn)
#pragma unroll
          for (int j = 0; j < 3 - i; ++j)
#pragma unroll
            for (int blk = 0; blk < 4; ++blk) p[nc][blk] = mfma16(kf[blk][kw][i], b[j], p[nc][blk]);
      }
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
        *reinterpret_cast<f32x4*>(pb + ((nc * 4 + blk) * 4 + w) * 1024 + at16) = p[nc][blk];
    lds_barrier();
    // (all of the step's reads ahead of its arithmetic, T's for the next step last)
    const f32x4 pk = *reinterpret_cast<const f32x4*>(fc + 16 * w + 4 * g);
    f32x4 q[NC][4], x[NC];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[nc][i] = *reinterpret_cast<const f32x4*>(pb + ((nc * 4 + w) * 4 + i) * 1024 + at16);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[nc][i] = vb[(16 * w + 4 * g + i) * M::vp + 16 * nc + n];
    }
    const f32x4 pr = *reinterpret_cast<const f32x4*>(fc + kChunk + 16 * w + 4 * g);
    const float fade = fc[2 * kChunk + 16 * w];
    if constexpr (M::stage) take_t(lds + M::t);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      q[nc][0] = (q[nc][0] + q[nc][1]) + (q[nc][2] + q[nc][3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[nc][i] = __builtin_fmaf(-pk[i], q[nc][0][i], x[nc][i]);
      put(rb, w, nc, x[nc]);
    }
    lds_barrier();
    f32x4 u[NC][2] = {};
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      bf16x8 b[3], b1[3];
      get(rb, 0, nc, b);
      if (two) {
        get(rb, 1, nc, b1);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int j = 0; j < 3 - i; ++j) {
            u[nc][0] = mfma16(tf[0][i], b[j], u[nc][0]);
            u[nc][1] = mfma16(tf[1][i], b1[j], u[nc][1]);
          }
      } else {
        u[nc][0] = mfma_parts(tf[0], b, u[nc][0]);
      }
    }
    settle(u);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      u[nc][0] += u[nc][1];
      put(gb, w, nc, u[nc][0] * pr);
      put(ub, w, nc, u[nc][0]);
    }
    lds_barrier();
    if constexpr (M::stage) take_kt(lds + M::kt);
    bf16x8 ug[NC][2][3];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < 2; ++st) get(gb, st, nc, ug[nc][st]);
    if constexpr (M::stage) take_k(lds + M::k);  // (the next chunk's)
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int t = 0; t < NT; ++t) S[t][nc] *= fade;
    // (part by part: all the sums in turn)
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < NPK; ++i)
#pragma unroll
        for (int j = 0; j < 3 - i; ++j)
#pragma unroll
          for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              S[t][nc] = mfma16(gf[t][st][i], ug[nc][st][j], S[t][nc]);
    if constexpr (!M::stage) {
      step(c);
      take_k(kws + L::k_rows);
      take_t(vws);
      take_kt(kws);
    }
    settle(S);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dim = L::dim(NT * w + t, 4 * g + i);
        if (dim < d.k_dim && col + 16 * nc < d.v_dim)
          sp[(size_t)dim * d.v_dim + 16 * nc] = S[t][nc][i];
      }
}

// ---- launches ----------------------------------------------------------------------
template <typename T, typename F>
auto with_dims(const dmh_gated_delta& a, F f) {
  constexpr int NPK = std::is_same_v<T, bf16_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3;
  if (a.k_dim <= 64) return f(T{}, Layout<64, NPK>{});
  if (a.k_dim <= 128) return f(T{}, Layout<128, NPK>{});
  return f(T{}, Layout<256, NPK>{});
}
template <typename F>
auto with_form(const dmh_gated_delta& a, F f) {
  if (a.dtype == DMH_DTYPE_BF16) return with_dims<bf16_t>(a, f);
  if (a.dtype == DMH_DTYPE_F16) return with_dims<half_t>(a, f);
  return with_dims<float>(a, f);
}

template <typename T, int DKT, int NPK>
hipError_t run(T, Layout<DKT, NPK>, const dmh_gated_delta& a, const SeqDev& s,
               int min_rows, int64_t chunks, int64_t room, void* ws, hipStream_t st) {
  using L = Layout<DKT, NPK>;
  ChunkWork cw;
  cw.v_heads = static_cast<uint8_t*>(ws);
  cw.k_heads = cw.v_heads + (size_t)room * a.v_heads * L::v_head;
  cw.min_rows = min_rows;
  const int64_t units = ((int64_t)s.num * a.v_heads + 7) / 8 * 8;
  const int rep = a.v_heads / a.k_heads;
  // Two column tiles per workgroup take 1.5 times as long as one (2048 rows of 32
  // heads: 91 us instead of 60), so they pay where single tiles would come to
  // more than one workgroup per CU (four long prompts: 449 us instead of 630).
  const int64_t longs = std::min<int64_t>(s.num, s.rows / min_rows);
  const bool pairs = longs * a.v_heads * ((a.v_dim + 15) / 16) > 256;
  const auto chain = pairs ? k_delta_chunks<T, DKT, 2, NPK>
                           : k_delta_chunks<T, DKT, 1, NPK>;
  const int64_t ncb = pairs ? (a.v_dim + 31) / 32 : (a.v_dim + 15) / 16;
  for (int64_t at = 0; at < chunks; at += room) {
    cw.rank0 = (int)at;
    cw.count = (int)(chunks - at < room ? chunks - at : room);
    const unsigned blocks = (unsigned)cw.count * a.k_heads * (rep > 1 ? (rep + 1) / 2 : 1);
    const unsigned rows = at == 0 ? delta_rows_blocks(a, s) : 0;
    const auto prep = rep > 1 ? k_delta_prep<T, DKT, NPK, 2>
                              : k_delta_prep<T, DKT, NPK, 1>;
    prep<<<dim3(rows + blocks), 256, 0, st>>>(a, s, cw, rows);
    chain<<<dim3((unsigned)(units * ncb)), 512, 0, st>>>(a, s, cw);
  }
  return hipGetLastError();
}

}  // namespace

int64_t delta_chunk_count(const SeqDev& s, int min_rows) {
  const int64_t most = s.rows / min_rows;  // sequences that long
  return s.rows / kChunk + (most < s.num ? most : s.num);
}

size_t delta_chunk_bytes(const dmh_gated_delta& a) {
  return with_form(a, [&](auto, auto l) {
    using L = decltype(l);
    return a.v_heads * L::v_head + a.k_heads * L::k_head;
  });
}

hipError_t launch_delta(const dmh_gated_delta& a, const SeqDev& s, int min_rows, int64_t chunks,
                        int64_t room, void* ws, hipStream_t st) {
  return with_form(a, [&](auto t, auto l) {
    return run(t, l, a, s, min_rows, chunks, room, ws, st);
  });
}

}  // namespace dm
