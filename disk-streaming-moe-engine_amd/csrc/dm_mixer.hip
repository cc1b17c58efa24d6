// dm_mixer.hip -- the token mixer around its chunked delta rule: the short
// causal convolution, the norms at a block's edges, and the gated delta rule
// row by row (decoding, short sequences).
//
// All three read their rows once, keep what they sum in fp32 registers and
// round once on the way out; all are bound by the memory they touch.
#include <algorithm>

#include "dm_mixer_device.h"

namespace dm {
namespace {

template <typename F>
hipError_t with_type(int dtype, F f) {
  if (dtype == DMH_DTYPE_BF16) return f(bf16_t{});
  if (dtype == DMH_DTYPE_F16) return f(half_t{});
  return f(float{});
}

// ---- short convolution ----------------------------------------------------------
// A workgroup takes TOK consecutive rows, each thread V channels of them with the
// last W - 1 rows in registers, and loads eight rows at a time; what is left of
// the channels over V goes to threads of one channel each.  A sequence's state is
// read and replaced by the workgroup with its first row, which also computes all
// rows that need the old state (the first W - 1, also where they reach past its
// rows): no other workgroup touches the state, so nothing has to wait.  Bound by
// the rows' bytes: 16384 rows of 8192 f16 channels in 121 us, 4.4 TB/s.
template <typename T, int V, int W>
__device__ __forceinline__ void conv_rows(const dmh_short_conv& a, const SeqDev& s, int ch, int t0,
                                          int t1, int first_seq) {
  const T* const x = static_cast<const T*>(a.x) + ch;
  T* const y = static_cast<T*>(a.y) + ch;
  float w[V][W], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? a.bias[ch + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[i][j] = a.weight[(size_t)(ch + i) * W + j];
  }
  for (int q = first_seq; q < s.num; ++q) {
    const int begin = s.off[q];
    if (begin >= t1) break;
    const bool first = begin >= t0;  // this workgroup has the sequence's first row
    const SeqRange r = seq_range(s, q, false);
    if (!r.live) continue;
    // rows of the sequence that this workgroup computes
    const int head = min(r.begin + W - 1, r.end);
    const int from = first ? r.begin : max(t0, head);
    const int to = first ? max(min(t1, r.end), head) : min(t1, r.end);
    if (from >= to) continue;
    float past[W - 1][V];
    if (first) {
      T* const sp = static_cast<T*>(a.state) + (size_t)r.slot * (W - 1) * a.channels + ch;
      Vec<T, V> old[W - 1], now[W - 1];
      const int len = r.end - r.begin;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        old[j] = load_raw<V>(sp + (size_t)j * a.channels);
        // the row that the new state's row j holds, if it is one of these
        now[j] = load_raw<V>(x + (int64_t)(r.begin + max(len - (W - 1) + j, 0)) * a.x_stride);
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (r.fresh) old[j] = Vec<T, V>{};
        to_f32<V>(old[j], past[j]);
      }
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        const int p = len - (W - 1) + j;  // its position; before 0 the old state's row W - 1 + p
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
          if (p < 0 && k == W - 1 + p) now[j] = old[k];
        *reinterpret_cast<Vec<T, V>*>(sp + (size_t)j * a.channels) = now[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        load_f32<V>(x + (int64_t)(from - (W - 1) + j) * a.x_stride, past[j]);
    }
    constexpr int B = 8;
    for (int t = from; t < to; t += B) {
      Vec<T, V> raw[B];
#pragma unroll
      for (int b = 0; b < B; ++b) raw[b] = load_raw<V>(x + (int64_t)min(t + b, to - 1) * a.x_stride);
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (t + b >= to) break;
        float row[V], out[V];
        to_f32<V>(raw[b], row);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float z = bias[i];
#pragma unroll
          for (int j = 0; j < W - 1; ++j) z = __builtin_fmaf(past[j][i], w[i][j], z);
          z = __builtin_fmaf(row[i], w[i][W - 1], z);
          out[i] = a.silu ? z * sigmoid_hw(z) : z;
#pragma unroll
          for (int j = 0; j < W - 2; ++j) past[j][i] = past[j + 1][i];
          past[W - 2][i] = row[i];
        }
        store_f32<V>(y + (int64_t)(t + b) * a.y_stride, out);
      }
    }
  }
}

template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(256) void k_short_conv(dmh_short_conv a, SeqDev s, int col_blocks,
                                                    int tile0) {
  const int tid = threadIdx.x;
  const int in_launch = blockIdx.x / col_blocks, col = blockIdx.x - in_launch * col_blocks;
  const int tile = tile0 + in_launch;
  const int t0 = tile * TOK, t1 = min(t0 + TOK, s.rows);

  // the first sequence with a row at t0 or behind it
  __shared__ int first_seq;
  if (tid == 0) first_seq = s.num;
  __syncthreads();
  int j0 = tid;
  while (j0 < s.num && s.off[j0 + 1] <= t0) j0 += 256;
  if (j0 < s.num) atomicMin(&first_seq, j0);
  __syncthreads();
  const int q0 = __builtin_amdgcn_readfirstlane(first_seq);

  const int full = a.channels / V, at = col * 256 + tid;
  if (at < full)
    conv_rows<T, V, W>(a, s, at * V, t0, t1, q0);
  else if (at - full < a.channels % V)
    conv_rows<T, 1, W>(a, s, full * V + at - full, t0, t1, q0);

  // what is wrong with the call's sequences, spread over the first launch's first
  // column of workgroups
  if (tile0 == 0 && col == 0 && tid < 64)
    for (int q = tile; q < s.num; q += gridDim.x / col_blocks) {
      const SeqRange r = seq_range(s, q, tid == 0);
      if (r.live && s.slots) report_shared_slot(s, q, r.slot, tid);
    }
}

template <typename T, int W>
hipError_t conv_w(const dmh_short_conv& a, const SeqDev& s, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int cb = (a.channels / V + a.channels % V + 255) / 256;
  const auto blocks = [&](int tok) { return (int64_t)cb * ((s.rows + tok - 1) / tok); };
  const auto run = [&](auto kernel, int tok) {
    const int64_t tiles = blocks(tok) / cb, most = (1 << 23) / cb;  // 2^31 threads a launch
    for (int64_t t = 0; t < tiles; t += most)
      kernel<<<dim3((unsigned)(std::min(most, tiles - t) * cb)), 256, 0, st>>>(a, s, cb, (int)t);
  };
  // Longer tiles read the weights and the rows before them less often, as long
  // as they leave four workgroups per CU (256 CUs); below one per CU, rows one by
  // one.
  if (blocks(64) >= 1024) run(k_short_conv<T, V, W, 64>, 64);
  else if (blocks(16) >= 256) run(k_short_conv<T, V, W, 16>, 16);
  else run(k_short_conv<T, V, W, 1>, 1);
  return hipGetLastError();
}

// ---- norms ------------------------------------------------------------------------
// The sum over a row of the lanes' sums of each of their N pieces; LPR 256: the
// four waves of a workgroup through LDS.  Below 64 lanes the pieces are added
// last, in the order of twice the lanes with half the pieces: the same bits.
template <int LPR, int N>
__device__ __forceinline__ float row_sum(const float (&s)[N], float* part) {
  float v = 0.0f;
  if constexpr (LPR < 64) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float x = s[n];
#pragma unroll
      for (int m = 1; m < LPR; m *= 2) x += __shfl_xor(x, m);
      v = n ? v + x : x;
    }
    return v;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) v = n ? v + s[n] : s[n];
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  if constexpr (LPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
  }
  return v;
}

// LPR lanes hold one group of a row in registers, N times V consecutive elements
// each, so that both norms run on the one read of it.  All loads come first and
// are whole; the one lane whose elements pass the end of the group reads and
// writes them one by one.  Bound by the rows' bytes: 16384 rows of 2048, bf16
// into an fp32 stream and its norm, in 94 us, 5.0 TB/s.
template <typename T, typename S, int LPR, int V, int N>
__global__ __launch_bounds__(256) void k_gated_norm(dmh_gated_norm a, int64_t unit0) {
  __shared__ float part[4];
  const int64_t units = (int64_t)a.rows * a.groups;
  const int64_t mine = unit0 + (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool in = mine < units;
  const int64_t unit = in ? mine : units - 1;  // (lanes behind the last row only read)
  // (a division of 64 bits takes longer than the row of a small group)
  const int64_t row = units >> 32 ? unit / a.groups : (uint32_t)unit / (uint32_t)a.groups;
  const int grp = (int)(unit - row * a.groups);
  const int lane = threadIdx.x % LPR;
  const int64_t at = (int64_t)grp * a.dim;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride + at;
  const T* gate = static_cast<const T*>(a.gate) + row * a.gate_stride + at;
  const S* res = static_cast<const S*>(a.residual) + row * a.residual_stride + at;

  Vec<T, V> xr[N], zr[N];
  Vec<S, V> rr[N];
  int c[N], left[N];  // the first element, and how many there are from it on
#pragma unroll
  for (int n = 0; n < N; ++n) {
    c[n] = (n * LPR + lane) * V;
    left[n] = a.dim - c[n];
    xr[n] = load_raw<V>(x + min(c[n], a.dim - V));
  }
  if (a.gate_act)
#pragma unroll
    for (int n = 0; n < N; ++n) zr[n] = load_raw<V>(gate + min(c[n], a.dim - V));
  if (a.residual)
#pragma unroll
    for (int n = 0; n < N; ++n) rr[n] = load_raw<V>(res + min(c[n], a.dim - V));
  float u[N][V];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    to_f32<V>(xr[n], u[n]);
    if (left[n] < V)
#pragma unroll
      for (int i = 0; i < V; ++i) u[n][i] = i < left[n] ? (float)x[c[n] + i] : 0.0f;
  }
  if (a.post) {
    float sums[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) sums[n] = __builtin_fmaf(u[n][i], u[n][i], sums[n]);
    const float q = 1.0f / sqrtf(row_sum<LPR>(sums, part) / (float)a.dim + a.eps);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float g[V];
      if (a.gamma) {
        load_f32<V>(a.gamma + min(c[n], a.dim - V), g);
        if (left[n] < V)
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] = i < left[n] ? a.gamma[c[n] + i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) u[n][i] = u[n][i] * q * (a.gamma ? g[i] : 1.0f);
    }
  }
  float sums[N] = {};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (a.gate_act) {
      float z[V];
      to_f32<V>(zr[n], z);
      if (left[n] < V)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = i < left[n] ? (float)gate[c[n] + i] : 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float sg = sigmoid_hw(z[i]);
        u[n][i] *= a.gate_act == DMH_GATE_SILU ? z[i] * sg : sg;
      }
    }
    float sv[V], r[V];
    if (a.scale_vec) {
      load_f32<V>(a.scale_vec + at + min(c[n], a.dim - V), sv);
      if (left[n] < V)
#pragma unroll
        for (int i = 0; i < V; ++i) sv[i] = i < left[n] ? a.scale_vec[at + c[n] + i] : 0.0f;
    }
    if (a.residual) {
      to_f32<V>(rr[n], r);
      if (left[n] < V)
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = i < left[n] ? (float)res[c[n] + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = u[n][i] * (a.scale_vec ? a.scale * sv[i] : a.scale);
      if (a.residual) v += r[i];
      u[n][i] = v;
      if (i < left[n]) sums[n] = __builtin_fmaf(v, v, sums[n]);
    }
  }
  const auto put = [&](void* base, int64_t stride) {
    S* const p = static_cast<S*>(base) + row * stride + at;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (in && left[n] >= V) store_f32<V>(p + c[n], u[n]);
      else if (in)
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i < left[n]) p[c[n] + i] = (S)u[n][i];
    }
  };
  if (a.stream) put(a.stream, a.stream_stride);
  if (!a.y) return;
  const float q = 1.0f / sqrtf(row_sum<LPR>(sums, part) / (float)a.dim + a.eps);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float g[V];
    if (a.edge_gamma) {
      load_f32<V>(a.edge_gamma + min(c[n], a.dim - V), g);
      if (left[n] < V)
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = i < left[n] ? a.edge_gamma[c[n] + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) u[n][i] = u[n][i] * q * (a.edge_gamma ? g[i] : 1.0f);
  }
  put(a.y, a.y_stride);
}

template <typename T, typename S, int LPR, int V, int N>
hipError_t norm_n(const dmh_gated_norm& a, hipStream_t st) {
  const int64_t units = (int64_t)a.rows * a.groups, per = 256 / LPR;
  constexpr int64_t kMost = 1 << 23;  // workgroups of a launch: 2^31 threads
  for (int64_t u = 0; u < units; u += kMost * per) {
    const int64_t left = (units - u + per - 1) / per;
    k_gated_norm<T, S, LPR, V, N><<<dim3((unsigned)(left < kMost ? left : kMost)), 256, 0, st>>>(a, u);
  }
  return hipGetLastError();
}
template <typename T, typename S>
hipError_t norm_ts(const dmh_gated_norm& a, hipStream_t st) {
  if (a.dim < 8) return norm_n<T, S, 16, 1, 1>(a, st);
  // As few lanes as hold a group.  Half of them with twice the elements each make
  // many rows faster (2048 rows of 4096 bf16, gated, in groups of 128, 256 or 512:
  // 13.8 us instead of 15) and few rows slower (32 rows: 4.1 instead of 3.5); 512
  // rows, 2^21 elements, take 5.4 us either way.  The sums are the same bits.
  const bool many = (int64_t)a.rows * a.groups * a.dim > 1 << 21;
  if (a.dim <= 64) return norm_n<T, S, 8, 8, 1>(a, st);
  if (a.dim <= 128) return many ? norm_n<T, S, 8, 8, 2>(a, st) : norm_n<T, S, 16, 8, 1>(a, st);
  if (a.dim <= 256) return many ? norm_n<T, S, 16, 8, 2>(a, st) : norm_n<T, S, 32, 8, 1>(a, st);
  if (a.dim <= 512) return many ? norm_n<T, S, 32, 8, 2>(a, st) : norm_n<T, S, 64, 8, 1>(a, st);
  if (a.dim <= 2048) return norm_n<T, S, 256, 8, 1>(a, st);
  if (a.dim <= 4096) return norm_n<T, S, 256, 8, 2>(a, st);
  return norm_n<T, S, 256, 8, 4>(a, st);
}

// ---- the delta rule, row by row -----------------------------------------------------
template <typename T, int RPL>
__global__ __launch_bounds__(256) void k_delta_rows(dmh_gated_delta d, SeqDev s, int max_rows) {
  delta_rows<T, RPL>(d, s, max_rows, blockIdx.x);
}

template <typename T>
hipError_t delta_rows_t(const dmh_gated_delta& a, const SeqDev& s, hipStream_t st) {
  const int max_rows = s.max_len;
  const dim3 grid(delta_rows_blocks(a, s));
  if (a.k_dim <= 64) k_delta_rows<T, 8><<<grid, 256, 0, st>>>(a, s, max_rows);
  else if (a.k_dim <= 128) k_delta_rows<T, 16><<<grid, 256, 0, st>>>(a, s, max_rows);
  else k_delta_rows<T, 32><<<grid, 256, 0, st>>>(a, s, max_rows);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_short_conv(const dmh_short_conv& a, const SeqDev& s, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.width == 4 ? conv_w<T, 4>(a, s, st)
           : a.width == 3 ? conv_w<T, 3>(a, s, st) : conv_w<T, 2>(a, s, st);
  });
}

hipError_t launch_gated_norm(const dmh_gated_norm& a, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.stream_dtype == DMH_DTYPE_F32 ? norm_ts<T, float>(a, st) : norm_ts<T, T>(a, st);
  });
}

hipError_t launch_delta_rows(const dmh_gated_delta& a, const SeqDev& s, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) { return delta_rows_t<decltype(t)>(a, s, st); });
}

}  // namespace dm
