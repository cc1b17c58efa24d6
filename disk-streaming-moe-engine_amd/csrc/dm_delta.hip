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
#include <cstdlib>
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
// key head K^T, and K and Q where the rows cannot be read in place (they are not
// bf16, or not aligned: WIDE is false).
template <int DKT, int NPK, int NPO, bool WIDE>
struct Layout {
  static constexpr bool direct = WIDE && NPK == 1;  // K and Q are read in place
  static constexpr int KS = DKT / 32;  // steps of 32 along the key dimension
  static constexpr int NPQ = NPK < NPO ? NPK : NPO;
  static constexpr size_t qk = frag_bytes(kTiles * 3);
  static constexpr size_t rows = qk + frag_bytes(kTiles * NPO);
  static constexpr size_t v_head = rows + 4 * kChunk * sizeof(float);
  static constexpr size_t k_rows = frag_bytes(DKT / 16 * 2 * NPK);
  static constexpr size_t q_rows = k_rows + (direct ? 0 : frag_bytes(4 * KS * NPK));
  static constexpr size_t k_head = q_rows + (direct ? 0 : frag_bytes(4 * KS * NPQ));
};

struct ChunkWork {
  uint8_t* v_heads;
  uint8_t* k_heads;
  int rank0, count;  // the chunks of this pass, counted over all long sequences
  int min_rows;      // sequences of fewer rows are not taken
  uint8_t* nowhere;  // 4 KB: where a lane without an output row stores
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
// The products of rows with rows take each wave's rows as one factor and all
// waves' rows, from LDS, as the other.  (I + A)^-1 comes by substitution in the
// 16 x 16 diagonal blocks (a row per lane) and, as -T22 A21 T11, in the blocks
// below them, 16 and then 32 wide, on the fp32 matrix cores: products of powers
// of A would take fewer steps and lose all precision for keys that resemble each
// other.  The chain of loads, products and substitution bounds it, so everything
// is loaded at once, unconditionally, and LDS is kept small for more workgroups
// per CU: T takes the place of the keys.
template <typename T, int DKT, int NPK, int NPO, bool WIDE>
__global__ __launch_bounds__(256) void k_delta_prep(dmh_gated_delta d, SeqDev s, ChunkWork cw) {
  using L = Layout<DKT, NPK, NPO, WIDE>;
  constexpr int KS = L::KS;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int local = blockIdx.x / d.v_heads, h = blockIdx.x - local * d.v_heads;
  const int rep = d.v_heads / d.k_heads, kh = h / rep;

  constexpr size_t kMat = kChunk * kPad * sizeof(float);
  constexpr size_t kKeys = frag_bytes(4 * KS * NPK);
  __shared__ __align__(16) uint8_t shared[kKeys > kMat ? kKeys : kMat];
  __shared__ __align__(16) float am[kChunk * kPad];
  uint8_t* const kfrag = shared;
  float* const tm = reinterpret_cast<float*>(shared);
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
      found[0] = s.off[j0 + tid] + (rank - (base + sum - own)) * kChunk;
      found[1] = s.off[j0 + tid + 1];
    }
    base += all;
    if (rank < base) break;
  }
  __syncthreads();
  const int begin = __builtin_amdgcn_readfirstlane(found[0]);
  if (begin < 0) return;
  const int rows = min(__builtin_amdgcn_readfirstlane(found[1]) - begin, kChunk);
  uint8_t* const vws = cw.v_heads + (size_t)blockIdx.x * L::v_head;
  uint8_t* const kws = cw.k_heads + ((size_t)local * d.k_heads + kh) * L::k_head;

  // the rows' values; of a row or column that is not there, another's, cleared
  // below
  const int row = 16 * w + n;
  const bool row_in = row < rows;
  float kv[KS][8], qv[KS][8];
  {
    const int64_t at = begin + min(row, rows - 1);
    const T* kp = static_cast<const T*>(d.k) + at * d.k_stride + kh * d.k_dim;
    const T* qp = static_cast<const T*>(d.q) + at * d.q_stride + kh * d.k_dim;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      const int c = 32 * st + 8 * g < d.k_dim ? 32 * st + 8 * g : 0;
      load_f32<8>(kp + c, WIDE, kv[st]);
      load_f32<8>(qp + c, WIDE, qv[st]);
    }
  }
  // gates and decays: a row per lane
  const Gates gt = load_gates<T>(d, begin + min(lane, rows - 1), h);
  double since = lane < rows ? (double)gt.log_decay : 0.0;
  if (since < -10000.0) since = -10000.0;  // (e^-10000 is 0 as well)
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const double v = __shfl_up(since, m);
    if (lane >= m) since += v;
  }
  const double last = __shfl(since, 63);
  if (w == 0) {
    decay[lane] = since;
    beta_s[lane] = lane < rows ? gt.beta : 0.0f;
  }

  // norms and parts of keys and queries
  bf16x8 qf[KS][NPK], kf[KS][NPK];
  float ksum = 0.0f, qsum = 0.0f;
#pragma unroll
  for (int st = 0; st < KS; ++st) {
    const bool in = row_in && 32 * st + 8 * g < d.k_dim;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
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
      store_frag(kfrag, (w * KS + st) * NPK + p, lane, kp4[p]);
      kf[st][p] = __builtin_bit_cast(bf16x8, kp4[p]);
      qf[st][p] = __builtin_bit_cast(bf16x8, qp4[p]);
      if (!L::direct && h == kh * rep) {
        store_frag(kws + L::k_rows, (w * KS + st) * NPK + p, lane, kp4[p]);
        if (p < L::NPQ) store_frag(kws + L::q_rows, (w * KS + st) * L::NPQ + p, lane, qp4[p]);
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

  // A, with the wave's rows on the left; and the transposed query-key matrix,
  // with its rows on the right: four consecutive keys of a row per lane, which
  // is a piece of the left factor that k_delta_chunks loads
  const double since_q = decay[row];
  for (int j = 0; j <= w; ++j) {
    f32x4 kk = {}, kq = {};
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      bf16x8 b[NPK];
#pragma unroll
      for (int p = 0; p < NPK; ++p) b[p] = load_frag(kfrag, (j * KS + st) * NPK + p, lane);
      kk = mfma_parts<3>(kf[st], b, kk);
      kq = mfma_parts<3>(b, qf[st], kq);
    }
    const int col = 16 * j + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int rr = 16 * w + 4 * g + r, cc = 16 * j + 4 * g + r;
      const float e = rr > col ? expf((float)(decay[rr] - decay[col])) : 0.0f;
      am[rr * kPad + col] =
          rr > col && rr < rows ? beta_s[rr] * rk_s[rr] * (e * rk_s[col]) * kk[r] : 0.0f;
      const float eq = row >= cc ? expf((float)(since_q - decay[cc])) : 0.0f;
      kq[r] = row >= cc && row_in ? rq * (eq * rk_s[cc]) * kq[r] : 0.0f;
    }
    uint2 p[NPO];
    split4<NPO>(kq, p);
    uint8_t* const to = vws + L::qk + (n + 16 * ((j & 1) * 2 + (g >> 1))) * 16 + (g & 1) * 8;
#pragma unroll
    for (int i = 0; i < NPO; ++i)
      *reinterpret_cast<uint2*>(to + (tile_of(w, j >> 1) * NPO + i) * 1024) = p[i];
  }
  if ((w & 1) == 0) {  // the empty half of the tile on the diagonal
    uint8_t* const to = vws + L::qk + (n + 32 + 16 * (g >> 1)) * 16 + (g & 1) * 8;
#pragma unroll
    for (int i = 0; i < NPO; ++i)
      *reinterpret_cast<uint2*>(to + (tile_of(w, w >> 1) * NPO + i) * 1024) = make_uint2(0, 0);
  }
  if (h == kh * rep) {  // K^T
    for (int i = tid; i < DKT / 16 * 2 * NPK * 64; i += 256) {
      const int frag = i >> 6, p = frag % NPK, half = frag / NPK & 1, t = frag / (2 * NPK);
      const int c = 16 * t + n;  // key dimension
      uint16_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int tok = 32 * half + 8 * g + e;
        const int from = (((tok >> 4) * KS + (c >> 5)) * NPK + p) * 1024 +
                         ((tok & 15) + 16 * ((c & 31) >> 3)) * 16 + (c & 7) * 2;
        v[e] = *reinterpret_cast<const uint16_t*>(kfrag + from);
      }
      store_frag(kws, frag, lane,
                 make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16,
                            v[6] | v[7] << 16));
    }
  }
  __syncthreads();

  // the diagonal blocks of T = (I + A)^-1 from T (I + A) = I, a row per lane
  {
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = j == n ? 1.0f : 0.0f;
#pragma unroll
    for (int m = 15; m > 0; --m) {
      const float* a = am + (16 * w + m) * kPad + 16 * w;
#pragma unroll
      for (int j = 0; j < m; ++j) x[j] = __builtin_fmaf(-x[m], a[j], x[j]);
    }
    if (g == 0) {
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<f32x4*>(tm + row * kPad + 16 * w + j) = f32x4{x[j], x[j + 1], x[j + 2],
                                                                        x[j + 3]};
    } else if (g == 1 && (w & 1) == 0) {  // the empty half of the tile on the diagonal
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<f32x4*>(tm + row * kPad + 16 * w + 16 + j) = f32x4{};
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

  // its parts, as a left factor
  for (int i = tid; i < kTiles * 64; i += 256) {
    const int tile = i >> 6;  // (lane is i & 63)
    const int blk = tile < 2 ? tile : (tile + 2) / 2, half = tile < 2 ? 0 : tile & 1;
    const int at = (16 * blk + n) * kPad + 32 * half + 8 * g;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tm[at + e] * beta_s[32 * half + 8 * g + e];
    uint4 vp[3];
    split8<3>(v, vp);
#pragma unroll
    for (int p = 0; p < 3; ++p) store_frag(vws, tile * 3 + p, lane, vp[p]);
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
template <typename T, int DKT, int NC, int NPK, int NPO, bool WIDE>
__global__ __launch_bounds__(256) void k_delta_chunks(dmh_gated_delta d, SeqDev s, ChunkWork cw) {
  using L = Layout<DKT, NPK, NPO, WIDE>;
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
  const int first = cw.rank0 - __builtin_amdgcn_readfirstlane(before);  // of this pass, counted in this sequence
  const int c0 = max(first, 0);
  const int c1 = min((r.end - r.begin + kChunk - 1) / kChunk, first + cw.count);
  if (c0 >= c1) return;

  // an element of a C tile: row 4 g + i of 16, column n.  O is held transposed, a
  // row and four columns per lane.
  const int col = cb * 16 * NC + n, ocol = cb * 16 * NC + 4 * g;
  T* const nowhere = reinterpret_cast<T*>(cw.nowhere + tid * 16);
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
  T v[NC][4];
  f32x4 pk, pr;
  float pq, fade;
  const bool two = w >= 2;  // rows 32 on: two tiles of the triangular factors
  // Loads are unconditional, so that none waits for another: behind the last row
  // or dimension they read one that is there (what comes of it meets a factor of
  // zero or is not stored).  Addresses are a uniform base of the chunk and 32-bit
  // offsets of the lane that hold for all chunks.
  const uint32_t at16 = lane * 16;
  const uint32_t t_at[2] = {tile_of(w, 0) * 3 * 1024 + at16, tile_of(w, two) * 3 * 1024 + at16};
  const uint32_t a_at[2] = {(uint32_t)L::qk + tile_of(w, 0) * NPO * 1024 + at16,
                            (uint32_t)L::qk + tile_of(w, two) * NPO * 1024 + at16};
  const uint32_t g_at = NT * w * 2 * NPK * 1024 + at16;
  const uint32_t kr_at = (uint32_t)L::k_rows + w * KS * NPK * 1024 + at16;
  const uint32_t qr_at = (uint32_t)L::q_rows + w * KS * NPQ * 1024 + at16;
  const uint32_t f4_at = (uint32_t)L::rows + (16 * w + 4 * g) * 4;
  const uint32_t f1_at = (uint32_t)L::rows + (kChunk + 16 * w + n) * 4;
  uint32_t k_at[KS], v_at[NC];
#pragma unroll
  for (int st = 0; st < KS; ++st)
    k_at[st] = (32 * st + 8 * g < d.k_dim ? 32 * st + 8 * g : 0) * sizeof(T);
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) v_at[nc] = min(col + 16 * nc, d.v_dim - 1) * sizeof(T);
  const auto frag = [](const uint8_t* base, uint32_t at) {
    return *reinterpret_cast<const bf16x8*>(base + at);
  };
  const uint8_t* const k0 = reinterpret_cast<const uint8_t*>(
      static_cast<const T*>(d.k) + (int64_t)r.begin * d.k_stride + kh * d.k_dim);
  const uint8_t* const q0 = reinterpret_cast<const uint8_t*>(
      static_cast<const T*>(d.q) + (int64_t)r.begin * d.q_stride + kh * d.k_dim);
  const uint8_t* const v0 = reinterpret_cast<const uint8_t*>(
      static_cast<const T*>(d.v) + (int64_t)r.begin * d.v_stride + h * d.v_dim);
  const int64_t k_pitch = d.k_stride * sizeof(T), q_pitch = d.q_stride * sizeof(T);
  const int64_t v_pitch = d.v_stride * sizeof(T);
  T* const o0 = static_cast<T*>(d.o) + (int64_t)r.begin * d.o_stride + h * d.v_dim + ocol;
  const int len = r.end - r.begin;
  const auto load_rows = [&](int c, const uint8_t* kws) {  // K and Q
    if constexpr (L::direct) {
      const int row = min(c * kChunk + 16 * w + n, len - 1);
      const uint8_t *kp = k0 + row * k_pitch, *qp = q0 + row * q_pitch;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        kf[st][0] = frag(kp, k_at[st]);
        qf[st][0] = frag(qp, k_at[st]);
      }
    } else {
#pragma unroll
      for (int st = 0; st < KS; ++st) {
#pragma unroll
        for (int i = 0; i < NPK; ++i) kf[st][i] = frag(kws, kr_at + (st * NPK + i) * 1024);
#pragma unroll
        for (int i = 0; i < NPQ; ++i) qf[st][i] = frag(kws, qr_at + (st * NPQ + i) * 1024);
      }
    }
  };
  const auto load_v = [&](int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* vp = v0 + min(c * kChunk + 16 * w + 4 * g + i, len - 1) * v_pitch;
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) v[nc][i] = *reinterpret_cast<const T*>(vp + v_at[nc]);
    }
  };
  const auto load_factors = [&](const uint8_t* vws) {
    pk = *reinterpret_cast<const f32x4*>(vws + f4_at);
    pq = *reinterpret_cast<const float*>(vws + f1_at);
    pr = *reinterpret_cast<const f32x4*>(vws + f4_at + 2 * kChunk * 4);
    fade = *reinterpret_cast<const float*>(vws + L::rows + 3 * kChunk * 4);
  };
  const auto load_t = [&](const uint8_t* vws) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < 3; ++i) tf[st][i] = frag(vws, t_at[st] + i * 1024);
  };
  const auto load_a = [&](const uint8_t* vws) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int i = 0; i < NPO; ++i) af[st][i] = frag(vws, a_at[st] + i * 1024);
  };
  const auto load_kt = [&](const uint8_t* kws) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int i = 0; i < NPK; ++i)
          gf[t][st][i] = frag(kws, g_at + ((t * 2 + st) * NPK + i) * 1024);
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

  size_t vws_at = ((size_t)(c0 - first) * d.v_heads + h) * L::v_head;
  size_t kws_at = ((size_t)(c0 - first) * d.k_heads + kh) * L::k_head;
  const uint8_t *vws = cw.v_heads + vws_at, *kws = cw.k_heads + kws_at;
  load_rows(c0, kws);
  load_v(c0);
  load_factors(vws);
  load_t(vws);
  load_a(vws);
  load_kt(kws);
  // All loads here (vmcnt 0): the waits that the compiler places in the loop
  // would otherwise have to hold for the order of these as well, and wait for
  // every load there.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  for (int c = c0; c < c1; ++c) {
    const int next = min(c + 1, c1 - 1), row0 = c * kChunk + 16 * w + 4 * g;
    vws_at += next > c ? (size_t)d.v_heads * L::v_head : 0;
    kws_at += next > c ? (size_t)d.k_heads * L::k_head : 0;
    asm("" : "+s"(vws_at), "+s"(kws_at));  // one base each: not one for every load
    vws = cw.v_heads + vws_at;
    kws = cw.k_heads + kws_at;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) put(sb, NT * w + t, nc, P3{}, S[t][nc]);
    lds_barrier();
    // (two chains each: a product waits for the last one of its own sum)
    f32x4 p[NC][2] = {}, o[NC][2] = {};
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        bf16x8 b[3];
        get(sb, st, nc, b);
        p[nc][st & 1] = mfma_parts<3>(kf[st], b, p[nc][st & 1]);
        o[nc][st & 1] = mfma_parts<NPO>(b, qf[st], o[nc][st & 1]);
      }
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      p[nc][0] += p[nc][1];
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = __builtin_fmaf(-pk[i], p[nc][0][i], row0 + i < len ? (float)v[nc][i] : 0.0f);
        o[nc][0][i] = (o[nc][0][i] + o[nc][1][i]) * pq;
      }
      put(rb, w, nc, P3{}, x);
    }
    load_rows(next, kws);
    load_v(next);
    lds_barrier();
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      f32x4 u = {};
      bf16x8 b[3];
      get(rb, 0, nc, b);
      u = mfma_parts<3>(tf[0], b, u);
      if (two) {
        f32x4 u1 = {};
        get(rb, 1, nc, b);
        u1 = mfma_parts<3>(tf[1], b, u1);
        u += u1;
      }
      put(ub, w, nc, PO{}, u);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] *= pr[i];
      put(gb, w, nc, P3{}, u);
    }
    load_t(vws);
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
      o[nc][0] = mfma_parts<NPO>(b, af[0], o[nc][0]);
      if (two) {
        get(ub, 1, nc, b);
        o[nc][0] = mfma_parts<NPO>(b, af[1], o[nc][0]);
      }
    }
    load_kt(kws);
    load_a(vws);
    load_factors(vws);
    // (not a branch, which would make the waits in the loop longer)
    const int row = c * kChunk + 16 * w + n;
    T* const op = o0 + row * d.o_stride;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const bool in = row < len && ocol + 16 * nc < d.v_dim;
      const float y[4] = {o[nc][0][0], o[nc][0][1], o[nc][0][2], o[nc][0][3]};
      store_f32<4>(in ? op + 16 * nc : nowhere, WIDE, y);
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
template <typename T, bool WIDE, typename F>
auto with_dims(const dmh_gated_delta& a, F f) {
  constexpr int NPK = std::is_same_v<T, bf16_t> ? 1 : std::is_same_v<T, half_t> ? 2 : 3;
  constexpr int NPO = std::is_same_v<T, float> ? 3 : 2;
  if (a.k_dim <= 64) return f(T{}, Layout<64, NPK, NPO, WIDE>{});
  if (a.k_dim <= 128) return f(T{}, Layout<128, NPK, NPO, WIDE>{});
  return f(T{}, Layout<256, NPK, NPO, WIDE>{});
}
template <typename F>
auto with_form(const dmh_gated_delta& a, bool wide, F f) {
  if (a.dtype == DMH_DTYPE_BF16)
    return wide ? with_dims<bf16_t, true>(a, f) : with_dims<bf16_t, false>(a, f);
  if (a.dtype == DMH_DTYPE_F16)
    return wide ? with_dims<half_t, true>(a, f) : with_dims<half_t, false>(a, f);
  return wide ? with_dims<float, true>(a, f) : with_dims<float, false>(a, f);
}

template <typename T, int DKT, int NPK, int NPO, bool WIDE>
hipError_t run(T, Layout<DKT, NPK, NPO, WIDE>, const dmh_gated_delta& a, const SeqDev& s,
               int min_rows, int64_t chunks, int64_t room, void* ws, hipStream_t st) {
  using L = Layout<DKT, NPK, NPO, WIDE>;
  ChunkWork cw;
  cw.v_heads = static_cast<uint8_t*>(ws);
  cw.k_heads = cw.v_heads + (size_t)room * a.v_heads * L::v_head;
  cw.min_rows = min_rows;
  cw.nowhere = cw.k_heads + (size_t)room * a.k_heads * L::k_head;
  const int64_t units = ((int64_t)s.num * a.v_heads + 7) / 8 * 8;
  for (int64_t at = 0; at < chunks; at += room) {
    cw.rank0 = (int)at;
    cw.count = (int)(chunks - at < room ? chunks - at : room);
    k_delta_prep<T, DKT, NPK, NPO, WIDE>
        <<<dim3((unsigned)cw.count * a.v_heads), 256, 0, st>>>(a, s, cw);
    const char* e = getenv("DM_NC");
    const int nc = e ? atoi(e) : 1;
    const unsigned ncb = (a.v_dim + 16 * nc - 1) / (16 * nc);
    if (nc == 1) k_delta_chunks<T, DKT, 1, NPK, NPO, WIDE><<<dim3((unsigned)(units * ncb)), 256, 0, st>>>(a, s, cw);
    if (nc == 2) k_delta_chunks<T, DKT, 2, NPK, NPO, WIDE><<<dim3((unsigned)(units * ncb)), 256, 0, st>>>(a, s, cw);
    if (nc == 4) k_delta_chunks<T, DKT, DKT == 256 ? 2 : 4, NPK, NPO, WIDE><<<dim3((unsigned)(units * ncb)), 256, 0, st>>>(a, s, cw);
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
