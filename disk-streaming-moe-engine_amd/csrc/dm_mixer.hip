// dm_mixer.hip -- the token mixer around its chunked delta rule: the short
// causal convolution, the norms at a block's edges, and the gated delta rule
// row by row (decoding, short sequences).
//
// All three read their rows once, keep what they sum in fp32 registers and
// round once on the way out; all are bound by the memory they touch.
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
// A workgroup takes TOK consecutive rows of 256 * V channels, each thread V
// channels of them with the last W - 1 rows in registers.  A sequence's state is
// read and replaced by the workgroup with its first row, which also computes
// all rows that need the old state (the first W - 1, also where they reach past
// its rows): no other workgroup touches the state, so nothing has to wait.
template <typename T, int V, int W, int TOK>
__global__ __launch_bounds__(256) void k_short_conv(dmh_short_conv a, SeqDev s, int col_blocks) {
  const int tid = threadIdx.x;
  const int tile = blockIdx.x / col_blocks, col = blockIdx.x - tile * col_blocks;
  const int t0 = tile * TOK, t1 = min(t0 + TOK, s.rows);
  const int ch = (col * 256 + tid) * V;
  const bool mine = ch < a.channels;
  const T* x = static_cast<const T*>(a.x) + ch;
  T* y = static_cast<T*>(a.y) + ch;
  T* state = static_cast<T*>(a.state) + ch;

  // the first sequence with a row at t0 or behind it
  __shared__ int first_seq;
  if (tid == 0) first_seq = s.num;
  __syncthreads();
  int j0 = tid;
  while (j0 < s.num && s.off[j0 + 1] <= t0) j0 += 256;
  if (j0 < s.num) atomicMin(&first_seq, j0);

  float w[V][W], bias[V];
  if (mine) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bias[i] = a.bias ? a.bias[ch + i] : 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) w[i][j] = a.weight[(size_t)(ch + i) * W + j];
    }
  }
  __syncthreads();

  for (int q = first_seq; q < s.num; ++q) {
    const int begin = s.off[q];
    if (begin >= t1) break;
    const bool first = begin >= t0;  // this workgroup has the sequence's first row
    const SeqRange r = seq_range(s, q, false);
    if (!r.live || !mine) continue;
    // rows of the sequence that this workgroup computes
    const int head = min(r.begin + W - 1, r.end);
    const int from = first ? r.begin : max(t0, head);
    const int to = first ? max(min(t1, r.end), head) : min(t1, r.end);
    T* sp = state + (size_t)r.slot * (W - 1) * a.channels;
    float past[W - 1][V];
    if (first) {
      Vec<T, V> old[W - 1];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (r.fresh) {
#pragma unroll
          for (int i = 0; i < V; ++i) old[j].v[i] = (T)0.0f;
        } else {
          old[j] = *reinterpret_cast<const Vec<T, V>*>(sp + (size_t)j * a.channels);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) past[j][i] = (float)old[j].v[i];
      }
      const int len = r.end - r.begin;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        const int p = len - (W - 1) + j;  // position that the new state's row j holds
        Vec<T, V> v = old[W - 2];
        if (p >= 0) {
          v = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)(r.begin + p) * a.x_stride);
        } else {
#pragma unroll
          for (int k = 0; k < W - 1; ++k)
            if (k == W - 1 + p) v = old[k];
        }
        *reinterpret_cast<Vec<T, V>*>(sp + (size_t)j * a.channels) = v;
      }
    } else {
      if (from >= to) continue;
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        load_f32<V>(x + (int64_t)(from - (W - 1) + j) * a.x_stride, true, past[j]);
    }
#pragma unroll 4
    for (int t = from; t < to; ++t) {
      float row[V], out[V];
      load_f32<V>(x + (int64_t)t * a.x_stride, true, row);
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
      store_f32<V>(y + (int64_t)t * a.y_stride, true, out);
    }
  }
  // what is wrong with the call's sequences, spread over the first column of
  // workgroups
  if (col == 0 && tid < 64)
    for (int q = tile; q < s.num; q += gridDim.x / col_blocks) {
      const SeqRange r = seq_range(s, q, tid == 0);
      if (r.live && s.slots) report_shared_slot(s, q, r.slot, tid);
    }
}

template <typename T, int V, int W>
hipError_t conv_w(const dmh_short_conv& a, const SeqDev& s, hipStream_t st) {
  constexpr int kTok = 16;
  const int cb = (a.channels + 256 * V - 1) / (256 * V);
  const int tiles = (s.rows + kTok - 1) / kTok;
  // rows one by one where tiles of 16 would leave CUs idle (256 of them)
  if ((int64_t)cb * tiles < 256) {
    k_short_conv<T, V, W, 1><<<dim3(cb * s.rows), 256, 0, st>>>(a, s, cb);
  } else {
    k_short_conv<T, V, W, kTok><<<dim3(cb * tiles), 256, 0, st>>>(a, s, cb);
  }
  return hipGetLastError();
}
template <typename T, int V>
hipError_t conv_v(const dmh_short_conv& a, const SeqDev& s, hipStream_t st) {
  return a.width == 4 ? conv_w<T, V, 4>(a, s, st)
         : a.width == 3 ? conv_w<T, V, 3>(a, s, st) : conv_w<T, V, 2>(a, s, st);
}

// ---- norms ------------------------------------------------------------------------
// The sum over the LPR lanes of a row; LPR 256: the four waves of a workgroup
// through LDS.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int m = 1; m < (LPR < 64 ? LPR : 64); m *= 2) v += __shfl_xor(v, m);
  if constexpr (LPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
  }
  return v;
}

// LPR lanes hold one group of a row in registers, N times V consecutive
// elements each, so that both norms run on the one read of it.
template <typename T, typename S, int LPR, int V, int N>
__global__ __launch_bounds__(256) void k_gated_norm(dmh_gated_norm a, int64_t unit0) {
  __shared__ float part[4];
  const int64_t unit = unit0 + (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const bool in = unit < (int64_t)a.rows * a.groups;
  const int64_t row = in ? unit / a.groups : 0;
  const int grp = in ? (int)(unit - row * a.groups) : 0;
  const int lane = threadIdx.x % LPR;
  const int64_t at = (int64_t)grp * a.dim;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride + at;
  const T* gate = static_cast<const T*>(a.gate) + row * a.gate_stride + at;
  const S* res = static_cast<const S*>(a.residual) + row * a.residual_stride + at;

  float u[N][V], z[N][V], r[N][V];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * LPR + lane) * V;
    if (in && c < a.dim) {
      load_f32<V>(x + c, V > 1, u[n]);
      if (a.gate_act) load_f32<V>(gate + c, V > 1, z[n]);
      if (a.residual) load_f32<V>(res + c, V > 1, r[n]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) u[n][i] = 0.0f;
    }
  }
  if (a.post) {
    float q = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) q = __builtin_fmaf(u[n][i], u[n][i], q);
    q = 1.0f / sqrtf(row_sum<LPR>(q, part) / (float)a.dim + a.eps);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * LPR + lane) * V;
      float g[V];
      if (a.gamma && c < a.dim) load_f32<V>(a.gamma + c, V > 1, g);
#pragma unroll
      for (int i = 0; i < V; ++i) u[n][i] = u[n][i] * q * (a.gamma && c < a.dim ? g[i] : 1.0f);
    }
  }
  float q = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * LPR + lane) * V;
    if (!in || c >= a.dim) continue;
    float sv[V];
    if (a.scale_vec) load_f32<V>(a.scale_vec + at + c, V > 1, sv);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = u[n][i];
      if (a.gate_act) {
        const float sg = sigmoid_hw(z[n][i]);
        v *= a.gate_act == DMH_GATE_SILU ? z[n][i] * sg : sg;
      }
      v *= a.scale_vec ? a.scale * sv[i] : a.scale;
      if (a.residual) v += r[n][i];
      u[n][i] = v;
      q = __builtin_fmaf(v, v, q);
    }
    if (a.stream)
      store_f32<V>(static_cast<S*>(a.stream) + row * a.stream_stride + at + c, V > 1, u[n]);
  }
  if (!a.y) return;
  q = 1.0f / sqrtf(row_sum<LPR>(q, part) / (float)a.dim + a.eps);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = (n * LPR + lane) * V;
    if (!in || c >= a.dim) continue;
    float g[V];
    if (a.edge_gamma) load_f32<V>(a.edge_gamma + c, V > 1, g);
#pragma unroll
    for (int i = 0; i < V; ++i) u[n][i] = u[n][i] * q * (a.edge_gamma ? g[i] : 1.0f);
    store_f32<V>(static_cast<S*>(a.y) + row * a.y_stride + at + c, V > 1, u[n]);
  }
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
hipError_t norm_ts(const dmh_gated_norm& a, bool wide, hipStream_t st) {
  if (wide) {
    if (a.dim <= 128) return norm_n<T, S, 16, 8, 1>(a, st);
    if (a.dim <= 512) return norm_n<T, S, 64, 8, 1>(a, st);
    if (a.dim <= 2048) return norm_n<T, S, 256, 8, 1>(a, st);
    if (a.dim <= 4096) return norm_n<T, S, 256, 8, 2>(a, st);
    return norm_n<T, S, 256, 8, 4>(a, st);
  }
  if (a.dim <= 64) return norm_n<T, S, 64, 1, 1>(a, st);
  if (a.dim <= 512) return norm_n<T, S, 64, 1, 8>(a, st);
  if (a.dim <= 2048) return norm_n<T, S, 256, 1, 8>(a, st);
  return norm_n<T, S, 256, 1, 32>(a, st);
}

// ---- the delta rule, row by row -----------------------------------------------------
template <typename T, int RPL>
__global__ __launch_bounds__(256) void k_delta_rows(dmh_gated_delta d, SeqDev s, int max_rows,
                                                    bool wide) {
  delta_rows<T, RPL>(d, s, max_rows, wide, blockIdx.x);
}

template <typename T>
hipError_t delta_rows_t(const dmh_gated_delta& a, const SeqDev& s, bool wide, hipStream_t st) {
  const int max_rows = s.max_len;
  const dim3 grid(delta_rows_blocks(a, s));
  if (a.k_dim <= 64) k_delta_rows<T, 8><<<grid, 256, 0, st>>>(a, s, max_rows, wide);
  else if (a.k_dim <= 128) k_delta_rows<T, 16><<<grid, 256, 0, st>>>(a, s, max_rows, wide);
  else k_delta_rows<T, 32><<<grid, 256, 0, st>>>(a, s, max_rows, wide);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_short_conv(const dmh_short_conv& a, const SeqDev& s, bool wide, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = sizeof(T) == 2 ? 8 : 4;
    return wide ? conv_v<T, V>(a, s, st) : conv_v<T, 1>(a, s, st);
  });
}

hipError_t launch_gated_norm(const dmh_gated_norm& a, bool wide, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    return a.stream_dtype == DMH_DTYPE_F32 ? norm_ts<T, float>(a, wide, st)
                                           : norm_ts<T, T>(a, wide, st);
  });
}

hipError_t launch_delta_rows(const dmh_gated_delta& a, const SeqDev& s, bool wide, hipStream_t st) {
  return with_type(a.dtype, [&](auto t) { return delta_rows_t<decltype(t)>(a, s, wide, st); });
}

}  // namespace dm
