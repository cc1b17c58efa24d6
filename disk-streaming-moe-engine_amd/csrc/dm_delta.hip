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
// x0 + x1 + x2 to 2^-26.  What reaches the state keeps the products of parts i
// and j with i + j < 3 (all 24 bits); what only reaches 16-bit outputs keeps i +
// j < 2 (2^-17, against their 2^-9 or 2^-12).  Keys and queries enter the
// products as they came (one part for bf16 rows, two for f16, three for f32),
// their norms and decays as factors of rows in fp32.  Sums of log decays are
// kept in 64 bits: e^(G_i - G_j) of two large sums would lose what the
// difference holds.
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
// in three parts, the query-key matrix in NPO, and the rows' factors; for each
// key head K^T, and K and Q where the rows cannot be read in place.
template <int DKT, int NPK, int NPO, bool DIRECT>
struct Layout {
  static constexpr int KS = DKT / 32;  // steps of 32 along the key dimension
  static constexpr int NPQ = NPK < NPO ? NPK : NPO;
  static constexpr size_t qk = frag_bytes(kTiles * 3);
  static constexpr size_t rows = qk + frag_bytes(kTiles * NPO);
  static constexpr size_t v_head = rows + 4 * kChunk * sizeof(float);
  static constexpr size_t k_rows = frag_bytes(DKT / 16 * 2 * NPK);
  static constexpr size_t q_rows = k_rows + (DIRECT ? 0 : frag_bytes(4 * KS * NPK));
  static constexpr size_t k_head = q_rows + (DIRECT ? 0 : frag_bytes(4 * KS * NPQ));
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
template <int LIM, int NPA, int NPB>
__device__ __forceinline__ f32x4 mfma_parts(const bf16x8 (&a)[NPA], const bf16x8 (&b)[NPB],
                                            f32x4 c) {
#pragma unroll
  for (int i = 0; i < NPA; ++i)
#pragma unroll
    for (int j = 0; j < NPB; ++j)
      if (i + j < LIM) c = mfma16(a[i], b[j], c);
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
// One workgroup per chunk and value head; wave w has rows 16 w .. 16 w + 15.
// The products of rows with rows take each wave's rows as the left factor and
// all waves' rows, from LDS, as the right one.  (I + A)^-1 comes by forward
// substitution in the 16 x 16 diagonal blocks (a column per lane) and, as
// -T22 A21 T11, in the blocks below them, 16 and then 32 wide, on the fp32
// matrix cores: products of powers of A would take fewer steps and lose all
// precision for keys that resemble each other.
template <typename T, int DKT, int NPK, int NPO, bool DIRECT>
__global__ __launch_bounds__(256) void k_delta_prep(dmh_gated_delta d, SeqDev s, ChunkWork cw) {
  using L = Layout<DKT, NPK, NPO, DIRECT>;
  constexpr int KS = L::KS;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int local = blockIdx.x / d.v_heads, h = blockIdx.x - local * d.v_heads;
  const int rep = d.v_heads / d.k_heads, kh = h / rep;

  __shared__ __align__(16) uint8_t kfrag[frag_bytes(4 * KS * NPK)];
  __shared__ __align__(16) float am[kChunk * kPad], qm[kChunk * kPad], tm[kChunk * kPad];
  __shared__ double decay[kChunk];
  __shared__ float beta_s[kChunk], rk_s[kChunk], rq_s[kChunk];
  __shared__ int scan[4], found[2];

  // the chunk: sequence and place in it
  const int rank = cw.rank0 + local;
  if (tid == 0) found[0] = -1;
  for (int j0 = 0, base = 0; j0 < s.num; j0 += 256) {
    const int own = j0 + tid < s.num ? chunks_of(s, j0 + tid, cw.min_rows) : 0;
    int sum = own;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const int v = __shfl_up(sum, m);
      if (lane >= m) sum += v;
    }
    __syncthreads();
    if (lane == 63) scan[w] = sum;
    __syncthreads();
    for (int i = 0; i < w; ++i) sum += scan[i];
    const int all = scan[0] + scan[1] + scan[2] + scan[3];
    if (rank < base + sum && rank >= base + sum - own) {
      found[0] = j0 + tid;
      found[1] = rank - (base + sum - own);
    }
    base += all;
    if (rank < base) break;
  }
  __syncthreads();
  if (found[0] < 0) return;
  const int begin = s.off[found[0]] + found[1] * kChunk;
  const int rows = min(s.off[found[0] + 1] - begin, kChunk);
  uint8_t* const vws = cw.v_heads + (size_t)blockIdx.x * L::v_head;
  uint8_t* const kws = cw.k_heads + ((size_t)local * d.k_heads + kh) * L::k_head;

  // gates and decays: a row per lane
  double since = 0.0;
  float beta = 0.0f;
  if (lane < rows) {
    const Gates gt = load_gates<T>(d, begin + lane, h);
    since = gt.log_decay < -10000.0f ? -10000.0 : (double)gt.log_decay;  // e^-10000 is 0 as well
    beta = gt.beta;
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const double v = __shfl_up(since, m);
    if (lane >= m) since += v;
  }
  const double last = __shfl(since, 63);
  if (w == 0) {
    decay[lane] = since;
    beta_s[lane] = beta;
  }

  // keys and queries of the wave's rows: norms and parts
  bf16x8 qf[KS][NPK], kf[KS][NPK];
  {
    const int row = 16 * w + n;
    const T* kp = static_cast<const T*>(d.k) + (int64_t)(begin + row) * d.k_stride + kh * d.k_dim;
    const T* qp = static_cast<const T*>(d.q) + (int64_t)(begin + row) * d.q_stride + kh * d.k_dim;
    float ksum = 0.0f, qsum = 0.0f;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const int c = 32 * st + 8 * g;
      float kv[8] = {}, qv[8] = {};
      if (row < rows && c < d.k_dim) {
        load_f32<8>(kp + c, DIRECT, kv);
        load_f32<8>(qp + c, DIRECT, qv);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ksum = __builtin_fmaf(kv[i], kv[i], ksum);
        qsum = __builtin_fmaf(qv[i], qv[i], qsum);
      }
      uint4 kp4[NPK], qp4[NPK];
      split8<NPK>(kv, kp4);
      split8<NPK>(qv, qp4);
#pragma unroll
      for (int p = 0; p < NPK; ++p) {
        store_frag(kfrag, (w * KS + st) * NPK + p, lane, kp4[p]);
        kf[st][p] = __builtin_bit_cast(bf16x8, kp4[p]);
        qf[st][p] = __builtin_bit_cast(bf16x8, qp4[p]);
        if (!DIRECT && h == kh * rep) {
          store_frag(kws + L::k_rows, (w * KS + st) * NPK + p, lane, kp4[p]);
          if (p < L::NPQ) store_frag(kws + L::q_rows, (w * KS + st) * L::NPQ + p, lane, qp4[p]);
        }
      }
    }
    ksum += __shfl_xor(ksum, 16);
    qsum += __shfl_xor(qsum, 16);
    ksum += __shfl_xor(ksum, 32);
    qsum += __shfl_xor(qsum, 32);
    if (g == 0) {
      rk_s[row] = d.qk_norm ? 1.0f / sqrtf(ksum + d.eps) : 1.0f;
      rq_s[row] = d.qk_norm ? d.scale / sqrtf(qsum + d.eps) : d.scale;
    }
  }
  __syncthreads();

  // A and the query-key matrix
  for (int j = 0; j <= w; ++j) {
    f32x4 kk = {}, qk = {};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      bf16x8 b[NPK];
#pragma unroll
      for (int p = 0; p < NPK; ++p) b[p] = load_frag(kfrag, (j * KS + st) * NPK + p, lane);
      kk = mfma_parts<3>(kf[st], b, kk);
      qk = mfma_parts<3>(qf[st], b, qk);
    }
    const int col = 16 * j + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * w + 4 * g + r;
      const float e = row >= col ? expf((float)(decay[row] - decay[col])) * rk_s[col] : 0.0f;
      am[row * kPad + col] = row > col && row < rows ? beta_s[row] * rk_s[row] * e * kk[r] : 0.0f;
      qm[row * kPad + col] = row >= col && row < rows ? rq_s[row] * e * qk[r] : 0.0f;
    }
  }
  if ((w & 1) == 0) {  // the upper halves of the tiles on the diagonal
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      qm[(16 * w + 4 * g + r) * kPad + 16 * w + 16 + n] = 0.0f;
      tm[(16 * w + 4 * g + r) * kPad + 16 * w + 16 + n] = 0.0f;
    }
  }
  __syncthreads();

  // the diagonal blocks of T = (I + A)^-1, a column per lane
  {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == n ? 1.0f : 0.0f;
#pragma unroll
      for (int m = 0; m < i; ++m)
        v = __builtin_fmaf(-am[(16 * w + i) * kPad + 16 * w + m], x[m], v);
      x[i] = v;
      if (g == 0) tm[(16 * w + i) * kPad + 16 * w + n] = v;
    }
  }
  __syncthreads();
  // C tiles as right factors: step r of a product over 16 takes row 4 g + r of it
  const auto a_blk = [&](const float* m, int bi, int bj, int st) {
    return m[(16 * bi + n) * kPad + 16 * bj + st];
  };
  if (w < 2) {
    const int b0 = 2 * w, b1 = b0 + 1;
    f32x4 x = {}, y = {};
#pragma unroll
    for (int st = 0; st < 4; ++st)
      x = mfma_f32(a_blk(am, b1, b0, 4 * st + g),
                   tm[(16 * b0 + 4 * st + g) * kPad + 16 * b0 + n], x);
#pragma unroll
    for (int r = 0; r < 4; ++r) y = mfma_f32(a_blk(tm, b1, b1, 4 * g + r), x[r], y);
#pragma unroll
    for (int r = 0; r < 4; ++r) tm[(16 * b1 + 4 * g + r) * kPad + 16 * b0 + n] = -y[r];
  }
  __syncthreads();
  {
    const int bi = w >> 1, bj = w & 1;
    f32x4 y = {};
    for (int k = 0; k <= bi; ++k) {
      f32x4 x = {};
      for (int kk = bj; kk < 2; ++kk)
#pragma unroll
        for (int st = 0; st < 4; ++st)
          x = mfma_f32(a_blk(am, 2 + k, kk, 4 * st + g),
                       tm[(16 * kk + 4 * st + g) * kPad + 16 * bj + n], x);
#pragma unroll
      for (int r = 0; r < 4; ++r) y = mfma_f32(a_blk(tm, 2 + bi, 2 + k, 4 * g + r), x[r], y);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) tm[(32 + 16 * bi + 4 * g + r) * kPad + 16 * bj + n] = -y[r];
  }
  __syncthreads();

  // parts of both matrices, as left factors
  for (int i = tid; i < kTiles * 64; i += 256) {
    const int tile = i >> 6;  // (lane is i & 63)
    const int blk = tile < 2 ? tile : (tile + 2) / 2, half = tile < 2 ? 0 : tile & 1;
    const int at = (16 * blk + n) * kPad + 32 * half + 8 * g;
    float v[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = tm[at + e] * beta_s[32 * half + 8 * g + e];
      q[e] = qm[at + e];
    }
    uint4 vp[3], qp[NPO];
    split8<3>(v, vp);
    split8<NPO>(q, qp);
#pragma unroll
    for (int p = 0; p < 3; ++p) store_frag(vws, tile * 3 + p, lane, vp[p]);
#pragma unroll
    for (int p = 0; p < NPO; ++p) store_frag(vws + L::qk, tile * NPO + p, lane, qp[p]);
  }
  if (w == 0) {
    float* f = reinterpret_cast<float*>(vws + L::rows);
    const bool in = lane < rows;
    const float grown = expf((float)since);
    f[lane] = in ? grown * rk_s[lane] : 0.0f;
    f[kChunk + lane] = in ? grown * rq_s[lane] : 0.0f;
    f[2 * kChunk + lane] = in ? expf((float)(last - since)) * rk_s[lane] : 0.0f;
    f[3 * kChunk + lane] = expf((float)last);
  }
  if (h == kh * rep) {
    for (int i = tid; i < DKT / 16 * 2 * NPK * 64; i += 256) {
      const int frag = i >> 6, p = frag % NPK, half = frag / NPK & 1, t = frag / (2 * NPK);
      const int c = 16 * t + n;  // key dimension
      uint16_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = 32 * half + 8 * g + e;
        const int from = (((row >> 4) * KS + (c >> 5)) * NPK + p) * 1024 +
                         ((row & 15) + 16 * ((c & 31) >> 3)) * 16 + (c & 7) * 2;
        v[e] = *reinterpret_cast<const uint16_t*>(kfrag + from);
      }
      store_frag(kws, frag, lane,
                 make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16,
                            v[6] | v[7] << 16));
    }
  }
}

// ---- the chunks of a head, in order ----------------------------------------------
// One workgroup per head and 16 NC columns of its state, which four waves hold
// in registers, each the rows of DKT / 64 tiles of 16.  In a chunk wave w
// computes rows 16 w .. 16 w + 15: K S and Q S (all of S needed), R = V - K S,
// U = T R (rows of R up to its own), O; and then its rows of K^T U (all of U).
// S, R and U pass between the waves through LDS, already split into parts and
// in the order in which a right factor is held, so a chunk has three barriers.
// Every left factor is loaded straight into registers, as soon as the previous
// chunk's is used up.  A chunk takes about as long as this chain of products and
// exchanges, whatever the number of columns; more heads or sequences run beside
// it.
template <typename T, int DKT, int NC, int NPK, int NPO, bool DIRECT>
__global__ __launch_bounds__(256) void k_delta_chunks(dmh_gated_delta d, SeqDev s, ChunkWork cw) {
  using L = Layout<DKT, NPK, NPO, DIRECT>;
  constexpr int KS = L::KS, NT = DKT / 64, NPQ = L::NPQ;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
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

  __shared__ __align__(16) uint8_t sb[frag_bytes(3 * KS * NC)];
  __shared__ __align__(16) uint8_t rb[frag_bytes(3 * 2 * NC)];
  __shared__ __align__(16) uint8_t ub[frag_bytes(NPO * 2 * NC)], gb[frag_bytes(3 * 2 * NC)];
  __shared__ int before;

  // chunks of the sequences before this one
  if (tid == 0) before = 0;
  __syncthreads();
  int mine = 0;
  for (int j = tid; j < seq; j += 256) mine += chunks_of(s, j, cw.min_rows);
  if (mine) atomicAdd(&before, mine);
  __syncthreads();
  const int first = cw.rank0 - before;  // of this pass, counted in this sequence
  const int c0 = max(first, 0);
  const int c1 = min((r.end - r.begin + kChunk - 1) / kChunk, first + cw.count);
  if (c0 >= c1) return;

  // an element of a C tile: row 4 g + i of 16, column n
  const int col = cb * 16 * NC + n;
  float* const sp = d.state + (((size_t)r.slot * d.v_heads + h) * d.k_dim + 16 * NT * w + 4 * g) *
                                  d.v_dim + col;
  f32x4 S[NT][NC];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = 16 * (NT * w + t) + 4 * g + i < d.k_dim && col + 16 * nc < d.v_dim;
        S[t][nc][i] = in && !(c0 == 0 && r.fresh) ? sp[(size_t)(16 * t + i) * d.v_dim + 16 * nc] : 0.0f;
      }

  bf16x8 kf[KS][NPK], qf[KS][NPQ], tf[2][3], af[2][NPO], gf[NT][2][NPK];
  float v[NC][4], pk[4], pq[4], pr[4], fade;
  const bool two = w >= 2;  // rows 32 on: two tiles of the triangular factors
  const auto v_ws = [&](int c) {
    return cw.v_heads + ((size_t)(c - first) * d.v_heads + h) * L::v_head;
  };
  const auto k_ws = [&](int c) {
    return cw.k_heads + ((size_t)(c - first) * d.k_heads + kh) * L::k_head;
  };
  const auto load_rows = [&](int c) {  // K and Q
    if constexpr (DIRECT) {
      const int row = r.begin + c * kChunk + 16 * w + n;
      const T* kp = static_cast<const T*>(d.k) + (int64_t)row * d.k_stride + kh * d.k_dim;
      const T* qp = static_cast<const T*>(d.q) + (int64_t)row * d.q_stride + kh * d.k_dim;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const int at = 32 * st + 8 * g;
        uint4 k4 = {}, q4 = {};
        if (row < r.end && at < d.k_dim) {
          k4 = *reinterpret_cast<const uint4*>(kp + at);
          q4 = *reinterpret_cast<const uint4*>(qp + at);
        }
        kf[st][0] = __builtin_bit_cast(bf16x8, k4);
        qf[st][0] = __builtin_bit_cast(bf16x8, q4);
      }
    } else {
      const uint8_t* p = k_ws(c);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
#pragma unroll
        for (int i = 0; i < NPK; ++i)
          kf[st][i] = load_frag(p + L::k_rows, (w * KS + st) * NPK + i, lane);
#pragma unroll
        for (int i = 0; i < NPQ; ++i)
          qf[st][i] = load_frag(p + L::q_rows, (w * KS + st) * NPQ + i, lane);
      }
    }
  };
  const auto load_v = [&](int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r.begin + c * kChunk + 16 * w + 4 * g + i;
      const T* vp = static_cast<const T*>(d.v) + (int64_t)row * d.v_stride + h * d.v_dim + col;
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
        v[nc][i] = row < r.end && col + 16 * nc < d.v_dim ? (float)vp[16 * nc] : 0.0f;
    }
  };
  const auto load_factors = [&](int c) {
    const float* f = reinterpret_cast<const float*>(v_ws(c) + L::rows);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pk[i] = f[16 * w + 4 * g + i];
      pq[i] = f[kChunk + 16 * w + 4 * g + i];
      pr[i] = f[2 * kChunk + 16 * w + 4 * g + i];
    }
    fade = f[3 * kChunk];
  };
  const auto load_t = [&](int c) {
    const uint8_t* p = v_ws(c);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      tf[0][i] = load_frag(p, tile_of(w, 0) * 3 + i, lane);
      if (two) tf[1][i] = load_frag(p, tile_of(w, 1) * 3 + i, lane);
    }
  };
  const auto load_a = [&](int c) {
    const uint8_t* p = v_ws(c) + L::qk;
#pragma unroll
    for (int i = 0; i < NPO; ++i) {
      af[0][i] = load_frag(p, tile_of(w, 0) * NPO + i, lane);
      if (two) af[1][i] = load_frag(p, tile_of(w, 1) * NPO + i, lane);
    }
  };
  const auto load_kt = [&](int c) {
    const uint8_t* p = k_ws(c);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < NPK; ++i)
          gf[t][st][i] = load_frag(p, ((NT * w + t) * 2 + st) * NPK + i, lane);
  };
  // tile t of a right factor's rows to LDS: fragment [step][column tile][part]
  const auto put = [&](uint8_t* base, int t, int nc, auto parts, f32x4 x) {
    constexpr int NP = decltype(parts)::value;
    uint2 p[NP];
    split4<NP>(x, p);
    const int at = (n + 16 * ((t & 1) * 2 + (g >> 1))) * 16 + (g & 1) * 8;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      *reinterpret_cast<uint2*>(base + (((t >> 1) * NC + nc) * NP + i) * 1024 + at) = p[i];
  };
  const auto get = [&](const uint8_t* base, int st, int nc, auto& b) {
    constexpr int NP = sizeof(b) / sizeof(b[0]);
#pragma unroll
    for (int i = 0; i < NP; ++i) b[i] = load_frag(base, (st * NC + nc) * NP + i, lane);
  };
  using P3 = std::integral_constant<int, 3>;
  using PO = std::integral_constant<int, NPO>;

  load_rows(c0);
  load_v(c0);
  load_factors(c0);
  load_t(c0);
  load_a(c0);
  load_kt(c0);
  for (int c = c0; c < c1; ++c) {
    const bool more = c + 1 < c1;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) put(sb, NT * w + t, nc, P3{}, S[t][nc]);
    lds_barrier();
    f32x4 p[NC] = {}, o[NC] = {};
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        bf16x8 b[3];
        get(sb, st, nc, b);
        p[nc] = mfma_parts<3>(kf[st], b, p[nc]);
        o[nc] = mfma_parts<NPO>(qf[st], b, o[nc]);
      }
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __builtin_fmaf(-pk[i], p[nc][i], v[nc][i]);
        o[nc][i] *= pq[i];
      }
      put(rb, w, nc, P3{}, x);
    }
    if (more) {
      load_rows(c + 1);
      load_v(c + 1);
    }
    lds_barrier();
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      f32x4 u = {};
      bf16x8 b[3];
      get(rb, 0, nc, b);
      u = mfma_parts<3>(tf[0], b, u);
      if (two) {
        get(rb, 1, nc, b);
        u = mfma_parts<3>(tf[1], b, u);
      }
      put(ub, w, nc, PO{}, u);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] *= pr[i];
      put(gb, w, nc, P3{}, u);
    }
    if (more) load_t(c + 1);
    lds_barrier();
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        bf16x8 b[3];
        get(gb, st, nc, b);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (st == 0) S[t][nc] *= fade;
          S[t][nc] = mfma_parts<3>(gf[t][st], b, S[t][nc]);
        }
      }
      bf16x8 b[NPO];
      get(ub, 0, nc, b);
      o[nc] = mfma_parts<NPO>(af[0], b, o[nc]);
      if (two) {
        get(ub, 1, nc, b);
        o[nc] = mfma_parts<NPO>(af[1], b, o[nc]);
      }
    }
    if (more) {
      load_kt(c + 1);
      load_a(c + 1);
      load_factors(c + 1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r.begin + c * kChunk + 16 * w + 4 * g + i;
      T* op = static_cast<T*>(d.o) + (int64_t)row * d.o_stride + h * d.v_dim + col;
      if (row < r.end)
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
          if (col + 16 * nc < d.v_dim) op[16 * nc] = (T)o[nc][i];
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (16 * (NT * w + t) + 4 * g + i < d.k_dim && col + 16 * nc < d.v_dim)
          sp[(size_t)(16 * t + i) * d.v_dim + 16 * nc] = S[t][nc][i];
}

// ---- launches ----------------------------------------------------------------------
template <typename T, bool DIRECT, typename F>
auto with_dims(const dmh_gated_delta& a, F f) {
  constexpr int NPK = std::is_same_v<T, bf16_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3;
  constexpr int NPO = std::is_same_v<T, float> ? 3 : 2;
  if (a.k_dim <= 64) return f(T{}, Layout<64, NPK, NPO, DIRECT>{});
  if (a.k_dim <= 128) return f(T{}, Layout<128, NPK, NPO, DIRECT>{});
  return f(T{}, Layout<256, NPK, NPO, DIRECT>{});
}
template <typename F>
auto with_form(const dmh_gated_delta& a, bool wide, F f) {
  if (a.dtype == DMH_DTYPE_BF16)
    return wide ? with_dims<bf16_t, true>(a, f) : with_dims<bf16_t, false>(a, f);
  if (a.dtype == DMH_DTYPE_F16) return with_dims<half_t, false>(a, f);
  return with_dims<float, false>(a, f);
}

template <typename T, int DKT, int NPK, int NPO, bool DIRECT>
hipError_t run(T, Layout<DKT, NPK, NPO, DIRECT>, const dmh_gated_delta& a, const SeqDev& s,
               int min_rows, int64_t chunks, int64_t room, void* ws, hipStream_t st) {
  using L = Layout<DKT, NPK, NPO, DIRECT>;
  ChunkWork cw;
  cw.v_heads = static_cast<uint8_t*>(ws);
  cw.k_heads = cw.v_heads + (size_t)room * a.v_heads * L::v_head;
  cw.min_rows = min_rows;
  const int64_t units = ((int64_t)s.num * a.v_heads + 7) / 8 * 8;
  for (int64_t at = 0; at < chunks; at += room) {
    cw.rank0 = (int)at;
    cw.count = (int)(chunks - at < room ? chunks - at : room);
    k_delta_prep<T, DKT, NPK, NPO, DIRECT>
        <<<dim3((unsigned)cw.count * a.v_heads), 256, 0, st>>>(a, s, cw);
    k_delta_chunks<T, DKT, 1, NPK, NPO, DIRECT>
        <<<dim3((unsigned)(units * ((a.v_dim + 15) / 16))), 256, 0, st>>>(a, s, cw);
  }
  return hipGetLastError();
}

}  // namespace

int64_t delta_chunk_count(const SeqDev& s, int min_rows) {
  const int64_t most = s.rows / min_rows;  // sequences that long
  return s.rows / kChunk + (most < s.num ? most : s.num);
}

size_t delta_chunk_bytes(const dmh_gated_delta& a, bool wide) {
  return with_form(a, wide, [&](auto, auto l) {
    using L = decltype(l);
    return a.v_heads * L::v_head + a.k_heads * L::k_head;
  });
}

hipError_t launch_delta_chunks(const dmh_gated_delta& a, const SeqDev& s, int min_rows,
                               int64_t chunks, int64_t room, void* ws, bool wide, hipStream_t st) {
  return with_form(a, wide, [&](auto t, auto l) {
    return run(t, l, a, s, min_rows, chunks, room, ws, st);
  });
}

}  // namespace dm
