// dm_mixer_api.cpp -- C ABI of the token mixer: argument checks, the sequences
// of a call, staging of host arrays, and the launches.
//
// Arguments are checked before the context is touched.  What only the device
// can see (sequences in device memory) the kernels check themselves.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "dm_api_rows.h"

namespace {

using namespace dm;

// Sequences of up to kRowsMost rows take the delta rule row by row.  Measured for
// 1, 8 and 64 sequences at 32 heads of 128: 8 rows take 14, 16 and 74 us row by
// row, 16 rows 23, 26 and 115, 32 rows 41, 44 and 212; as a chunk all of these
// 18, 44 and 253 to 278.
constexpr int kRowsMost = 16;
// Chunks whose factors are in memory at once (40 KB to 330 KB a head).  Four
// sequences of 16384 rows at 32 heads take 3.4 ms with 256, 1.99 ms with 512 and
// 1.96 ms with 2048; one of 65536 rows 2.9, 2.8 and 2.8 ms.
constexpr int64_t kChunkRoom = 512;
}  // namespace

int dm::api_mixer_error(unsigned long long key, char* err, size_t errlen) {
  return seq_error({err, errlen, "mixer"}, key_kind(key), key_pos(key));
}

extern "C" {

int dmh_short_conv_forward(dmh_ctx* c, const dmh_short_conv* args, const dmh_seq_batch* batch,
                           unsigned flags, char* errp, size_t errlen) {
  const Err err{errp, errlen, "short_conv"};
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!args) return err.arg("args is NULL");
  dmh_short_conv a = *args;
  if (!known(a.dtype)) return err.arg("unknown dtype");
  if (a.channels < 1 || a.channels > 1 << 20 || a.width < 2 || a.width > 4)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR", "channels %d, width %d (need 1 to 2^20, 2 to 4)",
               a.channels, a.width);
  int rc = check_batch(batch, dev, err);
  if (rc) return rc;
  dmh_seq_batch b = *batch;
  if (b.num_seqs == 0 || b.total_tokens == 0) return c ? DMH_OK : err.arg("ctx is NULL");
  if (!a.x || !a.weight || !a.state || !a.y) return err.arg("x, weight, state or y is NULL");
  const size_t es = elem(a.dtype);
  const int64_t state_row = (int64_t)(a.width - 1) * a.channels;
  Rows x{a.x, b.total_tokens, a.channels, a.x_stride, es};
  Rows y{a.y, b.total_tokens, a.channels, a.y_stride, es};
  const Rows state{a.state, b.num_slots, state_row, state_row, es};
  if (!x.ok() || !y.ok() || !state.ok()) return err.arg("a stride is shorter than its row, or an array is misaligned");
  if (overlap(x, y) || overlap(state, x) || overlap(state, y))
    return err.arg("x, y and state must not overlap");
  if (!c) return err.arg("ctx is NULL");
  hipStream_t st;
  unsigned long long* status;
  if ((rc = dm::api_mixer_begin(c, &st, &status, errp, errlen))) return rc;
  Stage stage;
  if (!dev) {
    stage.add(a.x, x.bytes());
    stage.add(a.weight, 4 * (size_t)a.channels * a.width);
    stage.add(a.bias, 4 * (size_t)a.channels);
    stage.add_out(a.state, state);
    stage.add_out(a.y, y);
    stage_batch(stage, b);
    if ((rc = stage.in(c, st, check, err))) return rc;
  }
  if (check) return DMH_OK;
  const hipError_t e = dm::launch_short_conv(a, seq_dev(b, status), st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

int dmh_gated_delta_forward(dmh_ctx* c, const dmh_gated_delta* args, const dmh_seq_batch* batch,
                            unsigned flags, char* errp, size_t errlen) {
  const Err err{errp, errlen, "gated_delta"};
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!args) return err.arg("args is NULL");
  dmh_gated_delta a = *args;
  if (!known(a.dtype)) return err.arg("unknown dtype");
  if (a.k_heads < 1 || a.v_heads < 1 || a.v_heads > 4096 || a.v_heads % a.k_heads)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "k_heads %d, v_heads %d (need v_heads a multiple of k_heads, up to 4096)", a.k_heads,
               a.v_heads);
  if (a.k_dim < 8 || a.k_dim > 256 || a.k_dim % 8 || a.v_dim < 8 || a.v_dim > 256 || a.v_dim % 8)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR", "k_dim %d, v_dim %d (need multiples of 8, 8 to 256)",
               a.k_dim, a.v_dim);
  if (!std::isfinite(a.scale)) return err.arg("scale must be finite");
  if (a.qk_norm && !(a.eps >= 0.0f && std::isfinite(a.eps)))
    return err.arg("eps must be finite and not negative");
  if (a.dt_bias && !a.a_log) return err.arg("dt_bias without a_log");
  int rc = check_batch(batch, dev, err);
  if (rc) return rc;
  dmh_seq_batch b = *batch;
  if (b.num_seqs == 0 || b.total_tokens == 0) return c ? DMH_OK : err.arg("ctx is NULL");
  if (!a.q || !a.k || !a.v || !a.a || !a.b || !a.state || !a.o)
    return err.arg("q, k, v, a, b, state or o is NULL");
  if (!aligned(a.state, 16)) return err.arg("state must be 16-byte aligned");
  // (a launch holds fewer than 2^32 threads; that of the chunks, of 512 a unit, counts
  // its units in eights)
  int64_t units = (int64_t)b.num_seqs * a.v_heads;
  if (b.max_seq_len > kRowsMost) units = (units + 7) / 8 * 8;
  if (units * ((a.v_dim + 15) / 16) >= (int64_t)1 << 23)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR", "too many sequences for one call: %d", b.num_seqs);
  const size_t es = elem(a.dtype), gs = a.a_log ? es : 4;
  const int64_t kw = (int64_t)a.k_heads * a.k_dim, vw = (int64_t)a.v_heads * a.v_dim;
  const int64_t sw = vw * a.k_dim;
  Rows q{a.q, b.total_tokens, kw, a.q_stride, es}, k{a.k, b.total_tokens, kw, a.k_stride, es};
  Rows v{a.v, b.total_tokens, vw, a.v_stride, es}, o{a.o, b.total_tokens, vw, a.o_stride, es};
  const Rows ga{a.a, b.total_tokens, a.v_heads, a.a_stride, gs};
  const Rows gb{a.b, b.total_tokens, a.v_heads, a.b_stride, gs};
  const Rows state{a.state, b.num_slots, sw, sw, 4};
  for (const Rows* r : std::initializer_list<const Rows*>{&q, &k, &v, &o, &ga, &gb})
    if (!r->ok() || r->stride >= 1 << 24)
      return err.arg("a stride is shorter than its row, or 2^24 or more, or an array is misaligned");
  for (const Rows* r : std::initializer_list<const Rows*>{&q, &k, &v, &ga, &gb})
    if (overlap(o, *r) || overlap(state, *r))
      return err.arg("o and state must not overlap the inputs");
  if (overlap(o, state)) return err.arg("o and state must not overlap");
  if (!c) return err.arg("ctx is NULL");
  hipStream_t st;
  unsigned long long* status;
  if ((rc = dm::api_mixer_begin(c, &st, &status, errp, errlen))) return rc;
  Stage stage;
  if (!dev) {
    stage.add(a.q, q.bytes());
    stage.add(a.k, k.bytes());
    stage.add(a.v, v.bytes());
    stage.add(a.a, ga.bytes());
    stage.add(a.b, gb.bytes());
    stage.add(a.a_log, 4 * (size_t)a.v_heads);
    stage.add(a.dt_bias, 4 * (size_t)a.v_heads);
    stage.add_out(a.state, state);
    stage.add_out(a.o, o);
    stage_batch(stage, b);
    if ((rc = stage.in(c, st, check, err))) return rc;
  }
  const SeqDev s = seq_dev(b, status);
  const int64_t chunks = b.max_seq_len > kRowsMost ? dm::delta_chunk_count(s, kRowsMost + 1) : 0;
  const int64_t room = std::min(chunks, kChunkRoom);
  void* ws = nullptr;
  if (chunks && (rc = dm::api_mixer_buffer(c, dm::kMixerChunks, room * dm::delta_chunk_bytes(a),
                                           &ws, errp, errlen)))
    return rc;
  if (check) return DMH_OK;
  const hipError_t e = chunks ? dm::launch_delta(a, s, kRowsMost + 1, chunks, room, ws, st)
                              : dm::launch_delta_rows(a, s, st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

int dmh_gated_norm_forward(dmh_ctx* c, const dmh_gated_norm* args, unsigned flags, char* errp,
                           size_t errlen) {
  const Err err{errp, errlen, "gated_norm"};
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!args) return err.arg("args is NULL");
  dmh_gated_norm a = *args;
  if (!known(a.dtype) || (a.stream_dtype != a.dtype && a.stream_dtype != DMH_DTYPE_F32))
    return err.arg("dtype must be known and stream_dtype the same or F32");
  if (a.rows < 0 || a.groups < 1 || a.groups > 1 << 20 || a.dim < 1 || a.dim > 8192)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "rows %d, groups %d, dim %d (need groups 1 to 2^20, dim 1 to 8192)", a.rows, a.groups,
               a.dim);
  if (a.gate_act < DMH_GATE_NONE || a.gate_act > DMH_GATE_SIGMOID) return err.arg("unknown gate_act");
  // (rmsnorm's check of its eps)
  if (!(a.eps > 0.0f) || !std::isfinite(a.eps)) return err.arg("eps must be finite and positive");
  if (a.rows == 0) return c ? DMH_OK : err.arg("ctx is NULL");
  if (!a.x || (a.gate_act && !a.gate)) return err.arg("x or gate is NULL");
  if (!a.stream && !a.y) return err.arg("stream and y are both NULL");
  if (!a.gate_act) a.gate = nullptr;
  const size_t es = elem(a.dtype), ss = elem(a.stream_dtype);
  const int64_t w = (int64_t)a.groups * a.dim;
  Rows x{a.x, a.rows, w, a.x_stride, es}, gate{a.gate, a.rows, w, a.gate_stride, es};
  Rows res{a.residual, a.rows, w, a.residual_stride, ss};
  Rows stream{a.stream, a.rows, w, a.stream_stride, ss}, y{a.y, a.rows, w, a.y_stride, ss};
  for (const Rows* r : {&x, &gate, &res, &stream, &y})
    if (r->p && !r->ok()) return err.arg("a stride is shorter than its row, or an array is misaligned");
  // (a thread reads the elements that it writes before it writes them)
  const bool on_res = a.stream == a.residual && a.stream_stride == a.residual_stride;
  const bool on_x = a.stream == a.x && a.stream_stride == a.x_stride && es == ss;
  if ((!on_x && overlap(stream, x)) || overlap(stream, gate) || (!on_res && overlap(stream, res)) ||
      overlap(y, x) || overlap(y, gate) || overlap(y, res) || overlap(y, stream))
    return err.arg("stream and y must not overlap each other or the inputs");
  if (!c) return err.arg("ctx is NULL");
  hipStream_t st;
  unsigned long long* status;
  int rc = dm::api_mixer_begin(c, &st, &status, errp, errlen);
  if (rc) return rc;
  Stage stage;
  if (!dev) {
    stage.add(a.x, x.bytes());
    stage.add(a.gate, gate.bytes());
    stage.add(a.residual, res.bytes());
    stage.add_out(a.stream, stream);
    stage.add_out(a.y, y);
    stage.add(a.gamma, 4 * (size_t)a.dim);
    stage.add(a.edge_gamma, 4 * (size_t)a.dim);
    stage.add(a.scale_vec, 4 * (size_t)w);
    if ((rc = stage.in(c, st, check, err))) return rc;
  }
  if (check) return DMH_OK;
  const hipError_t e = dm::launch_gated_norm(a, st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

}  // extern "C"
