// dm_api_rows.h -- what the entry points that take plain arrays share: their error
// texts, row arrays and whether they meet, the sequences of a call, and the staging
// of host arrays.
#pragma once
#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "dm_api_internal.h"
#include "dm_layout.h"
#include "dm_mixer.h"

namespace dm {

// Rows of a call, whose numbers the kernels count on from in 32 bits.
constexpr int32_t kRowsLimit = 1 << 30;

struct Err {
  char* p;
  size_t n;
  const char* stage;
  // {"error_type":type,"detail":...,"stage":...}
  int operator()(int code, const char* type, const char* fmt, ...) const
      __attribute__((format(printf, 4, 5))) {
    if (p && n) {
      char d[512];
      va_list ap;
      va_start(ap, fmt);
      vsnprintf(d, sizeof(d), fmt, ap);
      va_end(ap);
      snprintf(p, n, "{\"error_type\":\"%s\",\"detail\":\"%s\",\"stage\":\"%s\"}", type, d, stage);
    }
    return code;
  }
  int arg(const char* what) const { return (*this)(DMH_ERR_INVALID_ARG, "CONFIG_ERROR", "%s", what); }
  int hip(hipError_t e) const {
    return (*this)(DMH_ERR_HIP, "HIP_ERROR", "%s", hipGetErrorString(e));
  }
};

inline const char* seq_text(uint32_t kind) {
  switch (kind) {
    case kSqOffsets: return "offsets decrease or leave the rows";
    case kSqLength: return "longer than max_seq_len";
    case kSqSlot: return "slot outside the states";
    case kSqPast: return "its tokens are more than its pages hold, or past is negative";
    case kSqPage: return "a page outside the cache";
    default: return "names the state of an earlier sequence";
  }
}

inline int seq_error(const Err& err, uint32_t kind, int64_t seq) {
  return err(DMH_ERR_INVALID_ARG, "SEQUENCE_ERROR", "sequence %lld: %s", (long long)seq,
             seq_text(kind));
}

inline size_t elem(int dtype) { return dtype == DMH_DTYPE_F32 ? 4 : 2; }
inline bool known(int dtype) {
  return dtype == DMH_DTYPE_F32 || dtype == DMH_DTYPE_F16 || dtype == DMH_DTYPE_BF16;
}
inline bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// `rows` rows of `width` elements, `stride` elements apart.  A row of several heads
// has its width from the first one's first element to the last one's last.
struct Rows {
  const void* p;
  int64_t rows, width, stride;
  size_t size;
  int64_t heads = 1, head_stride = 0;
  size_t bytes() const { return rows ? ((size_t)(rows - 1) * stride + width) * size : 0; }
  bool ok() const {
    return stride >= width && stride < ((int64_t)1 << 40) && aligned(p, size);
  }
  int64_t head_width() const { return width - (heads - 1) * head_stride; }
};

// Whether two row arrays share an element.  Rows of one pitch whose columns lie
// side by side (slices of one buffer) do not.
inline bool overlap(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || !a.rows || !b.rows) return false;
  const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  if (pa + a.bytes() <= pb || pb + b.bytes() <= pa) return false;
  // whether columns of wa and wb bytes at these addresses, repeated each `pitch` bytes, are apart
  const auto apart = [&](size_t pitch, size_t wa, size_t wb) {
    const size_t d = (size_t)((pb % pitch + pitch - pa % pitch) % pitch);
    return d >= wa && pitch - d >= wb;
  };
  const size_t pitch = a.stride * a.size;
  if (pitch != b.stride * b.size) return true;
  if (apart(pitch, a.width * a.size, b.width * b.size)) return false;
  // (heads side by side, and rows that keep to their pitch)
  const size_t heads = a.head_stride * a.size;
  return !(a.heads > 1 && b.heads > 1 && heads == b.head_stride * b.size && pitch % heads == 0 &&
           apart(heads, a.head_width() * a.size, b.head_width() * b.size));
}

// The call's sequences, as far as the host sees them (all of them, where they
// are host memory).  written: the call writes their states, which no two may share.
inline int check_batch(const dmh_seq_batch* b, bool dev, const Err& err, bool written = true) {
  if (!b) return err.arg("batch is NULL");
  if (b->num_seqs < 0 || b->total_tokens < 0 || b->num_slots < 0)
    return err.arg("num_seqs, total_tokens and num_slots must not be negative");
  if (b->total_tokens >= kRowsLimit) return err.arg("total_tokens must be below 2^30");
  if (b->num_seqs == 0) return DMH_OK;
  if (b->max_seq_len < 1) return err.arg("max_seq_len must be positive");
  if (!b->offsets) return err.arg("offsets is NULL");
  if (!b->slots && b->num_seqs > b->num_slots)
    return err.arg("without slots, num_slots must be num_seqs or more");
  if (dev) return DMH_OK;
  std::vector<uint8_t> taken;
  try {
    taken.assign(b->num_slots, 0);
  } catch (const std::bad_alloc&) {
    return err(DMH_ERR_NO_MEMORY, "HIP_ERROR", "out of host memory");
  }
  int64_t most = 0;  // the largest offset so far
  for (int64_t i = 0; i < b->num_seqs; ++i) {
    const int64_t begin = b->offsets[i], end = b->offsets[i + 1];
    most = std::max(most, begin);
    const int64_t slot = b->slots ? b->slots[i] : i;
    if (slot < 0) continue;
    if (begin < most || end < begin || end > b->total_tokens) return seq_error(err, kSqOffsets, i);
    if (end - begin > b->max_seq_len) return seq_error(err, kSqLength, i);
    if (slot >= b->num_slots) return seq_error(err, kSqSlot, i);
    if (end == begin) continue;
    if (taken[slot] && written) return seq_error(err, kSqTwice, i);
    taken[slot] = 1;
  }
  return DMH_OK;
}

// Host arrays of a call, laid out in one device block: all are copied there,
// the written ones come back, without what lies between their rows (another
// output, where two are slices of one buffer).
class Stage {
 public:
  template <typename P>
  void add(P*& p, size_t bytes) {
    if (!p || !bytes) return;
    items_[n_++] = {const_cast<void*>(static_cast<const void*>(p)), bytes, total_, nullptr,
                    [](void* field, void* v) { *static_cast<P**>(field) = static_cast<P*>(v); }, &p};
    total_ += (bytes + 255) & ~(size_t)255;
  }
  // (r outlives the stage)
  template <typename P>
  void add_out(P*& p, const Rows& r) {
    const int n = n_;
    add(p, r.bytes());
    if (n_ > n) items_[n].out = &r;
  }
  // (check: makes the block alone)
  int in(dmh_ctx* c, hipStream_t st, bool check, const Err& err) {
    void* base = nullptr;
    const int rc = api_mixer_buffer(c, kMixerStage, total_ ? total_ : 256, &base, err.p, err.n);
    if (rc || check) return rc;
    for (int i = 0; i < n_; ++i) {
      Item& it = items_[i];
      void* d = static_cast<uint8_t*>(base) + it.at;
      const hipError_t e = hipMemcpyAsync(d, it.host, it.bytes, hipMemcpyHostToDevice, st);
      if (e != hipSuccess) return err.hip(e);
      it.set(it.field, d);
      it.dev = d;
    }
    return DMH_OK;
  }
  int out(hipStream_t st, const Err& err) {
    for (int i = 0; i < n_; ++i) {
      const Item& it = items_[i];
      if (!it.out) continue;
      const Rows& r = *it.out;
      const bool packed = r.heads == 1 || r.head_stride == r.head_width();
      hipError_t e = hipSuccess;
      if (packed && (r.stride == r.width || r.rows == 1)) {
        e = hipMemcpyAsync(it.host, it.dev, it.bytes, hipMemcpyDeviceToHost, st);
      } else {
        const int64_t n = packed ? 1 : r.heads, w = packed ? r.width : r.head_width();
        for (int64_t h = 0; h < n && e == hipSuccess; ++h) {
          const size_t at = (size_t)h * r.head_stride * r.size;
          e = hipMemcpy2DAsync(static_cast<uint8_t*>(it.host) + at, r.stride * r.size,
                               static_cast<uint8_t*>(it.dev) + at, r.stride * r.size, w * r.size,
                               r.rows, hipMemcpyDeviceToHost, st);
        }
      }
      if (e != hipSuccess) return err.hip(e);
    }
    const hipError_t e = hipStreamSynchronize(st);
    return e == hipSuccess ? DMH_OK : err.hip(e);
  }

 private:
  struct Item {
    void* host;
    size_t bytes, at;
    const Rows* out;  // the rows to copy back, or NULL
    void (*set)(void*, void*);
    void* field;
    void* dev;
  };
  Item items_[16];
  int n_ = 0;
  size_t total_ = 0;
};

inline void stage_batch(Stage& s, dmh_seq_batch& b) {
  s.add(b.offsets, 4 * ((size_t)b.num_seqs + 1));
  s.add(b.slots, 4 * (size_t)b.num_seqs);
  s.add(b.fresh, 4 * (size_t)b.num_seqs);
}

inline SeqDev seq_dev(const dmh_seq_batch& b, unsigned long long* status) {
  return {b.num_seqs, b.total_tokens, b.max_seq_len, b.num_slots,
          b.offsets,  b.slots,        b.fresh,       status};
}

}  // namespace dm
