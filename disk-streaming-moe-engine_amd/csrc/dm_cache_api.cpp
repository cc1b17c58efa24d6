// dm_cache_api.cpp -- C ABI of the 4-bit cache and of attention over it: argument
// checks, staging of host arrays, and the launches.
//
// Arguments are checked before the context is touched.  What only the device can see
// (sequences, pages and past in device memory) the kernels check themselves.
#include <hip/hip_runtime.h>

#include <cmath>
#include <initializer_list>

#include "dm_api_rows.h"
#include "dm_cache.h"

namespace {

using namespace dm;

constexpr int64_t kMostTokens = 1 << 30;  // of a slot, whose positions are counted in 32 bits

int check_cache(const dmh_kv_cache* c, const Err& err) {
  if (!c) return err.arg("cache is NULL");
  const int d = c->dim;
  if (c->kv_heads < 1 || c->kv_heads > 1024 ||
      (d != 32 && d != 64 && d != 96 && d != 128 && d != 192 && d != 256))
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "kv_heads %d, dim %d (need 1 to 1024, and 32, 64, 96, 128, 192 or 256)", c->kv_heads, d);
  if (c->page_size < 16 || c->page_size & (c->page_size - 1) || c->num_pages < 1 || c->max_pages < 1 ||
      (int64_t)c->page_size * c->max_pages > kMostTokens)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "page_size %d, num_pages %d, max_pages %d (need a power of two from 16 on, 1 or more,"
               " at most 2^30 positions)", c->page_size, c->num_pages, c->max_pages);
  return DMH_OK;
}

size_t cache_rows(const dmh_kv_cache& c) {
  return (size_t)c.num_pages * 2 * c.kv_heads * c.page_size;
}

// The cache's arrays, which a call with rows needs.
int check_arrays(const dmh_kv_cache& c, const Err& err) {
  if (!c.codes || !c.scales || !c.pages || !c.past)
    return err.arg("codes, scales, pages or past is NULL");
  if (!aligned(c.codes, 16) || !aligned(c.scales, 16))
    return err.arg("codes and scales must be 16-byte aligned");
  if (!aligned(c.pages, 4) || !aligned(c.past, 4)) return err.arg("pages or past is misaligned");
  return DMH_OK;
}

// past and the pages of host memory, for sequences that check_batch passed.  all: from
// the first position on, not that of the rows alone.
int check_pages(const dmh_kv_cache& c, const dmh_seq_batch& b, bool all, const Err& err) {
  for (int64_t i = 0; i < b.num_seqs; ++i) {
    const int64_t slot = b.slots ? b.slots[i] : i;
    if (slot < 0) continue;
    const int64_t n = b.offsets[i + 1] - b.offsets[i];
    if (n == 0) continue;
    const int64_t past = b.fresh && b.fresh[i] ? 0 : c.past[slot];
    if (past < 0 || past + n > (int64_t)c.max_pages * c.page_size) return seq_error(err, kSqPast, i);
    for (int64_t p = all ? 0 : past / c.page_size; p <= (past + n - 1) / c.page_size; ++p) {
      const int32_t page = c.pages[slot * c.max_pages + p];
      if (page < 0 || page >= c.num_pages) return seq_error(err, kSqPage, i);
    }
  }
  return DMH_OK;
}

Rows head_rows(const void* p, int64_t rows, int64_t heads, int64_t dim, int64_t stride,
               int64_t head_stride, size_t size) {
  Rows r{p, rows, (heads - 1) * head_stride + dim, stride, size};
  r.heads = heads;
  r.head_stride = head_stride;
  return r;
}
bool heads_ok(const Rows& r, int64_t dim) {
  return (r.heads == 1 || (r.head_stride >= dim && r.head_stride < (int64_t)1 << 40)) && r.ok();
}
constexpr const char* kBadRows =
    "a head lies in another or behind its row's stride, or an array is misaligned";

void stage_cache(Stage& s, dmh_kv_cache& c, const dmh_seq_batch& b, const Rows* codes,
                 const Rows* scales) {
  const size_t rows = cache_rows(c);
  if (codes) {
    s.add_out(c.codes, *codes);
    s.add_out(c.scales, *scales);
  } else {
    s.add(c.codes, rows * (c.dim / 2));
    s.add(c.scales, rows * (c.dim / 32));
  }
  s.add(c.pages, (size_t)4 * b.num_slots * c.max_pages);
  s.add(c.past, (size_t)4 * b.num_slots);
}

int kv_rows(dmh_ctx* ctx, const dmh_kv_cache* cache, const dmh_kv_rows* rows,
            const dmh_seq_batch* batch, bool write, unsigned flags, const Err& err) {
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!rows) return err.arg("rows is NULL");
  int rc = check_cache(cache, err);
  if (rc) return rc;
  dmh_kv_cache c = *cache;
  dmh_kv_rows r = *rows;
  if (!known(r.dtype)) return err.arg("unknown dtype");
  if ((rc = check_batch(batch, dev, err, write))) return rc;
  dmh_seq_batch b = *batch;
  if (b.num_seqs == 0 || b.total_tokens == 0) return ctx ? DMH_OK : err.arg("ctx is NULL");
  if (!r.k || !r.v) return err.arg("k or v is NULL");
  if ((rc = check_arrays(c, err))) return rc;
  const size_t es = elem(r.dtype);
  const Rows k = head_rows(r.k, b.total_tokens, c.kv_heads, c.dim, r.k_stride, r.k_head_stride, es);
  const Rows v = head_rows(r.v, b.total_tokens, c.kv_heads, c.dim, r.v_stride, r.v_head_stride, es);
  if (!heads_ok(k, c.dim) || !heads_ok(v, c.dim)) return err.arg(kBadRows);
  const int64_t n = (int64_t)cache_rows(c);
  const Rows codes{c.codes, n, c.dim / 2, c.dim / 2, 1};
  const Rows scales{c.scales, n, c.dim / 32, c.dim / 32, 1};
  if (overlap(codes, scales)) return err.arg("codes and scales must not overlap");
  for (const Rows* x : {&k, &v})
    if (overlap(*x, codes) || overlap(*x, scales)) return err.arg("the cache must not overlap the rows");
  if (!write && overlap(k, v)) return err.arg("k and v must not overlap");
  if (!dev && (rc = check_pages(c, b, false, err))) return rc;
  if (!ctx) return err.arg("ctx is NULL");
  hipStream_t st;
  unsigned long long* status;
  if ((rc = api_mixer_begin(ctx, &st, &status, err.p, err.n))) return rc;
  Stage stage;
  if (!dev) {
    if (write) {
      stage.add(r.k, k.bytes());
      stage.add(r.v, v.bytes());
    } else {
      stage.add_out(r.k, k);
      stage.add_out(r.v, v);
    }
    stage_cache(stage, c, b, write ? &codes : nullptr, &scales);
    stage_batch(stage, b);
    if ((rc = stage.in(ctx, st, check, err))) return rc;
  }
  if (check) return DMH_OK;
  const SeqDev s = seq_dev(b, status);
  const hipError_t e = write ? launch_kv_write(c, r, s, st) : launch_kv_read(c, r, s, st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

}  // namespace

extern "C" {

int dmh_kv_write(dmh_ctx* ctx, const dmh_kv_cache* cache, const dmh_kv_rows* rows,
                 const dmh_seq_batch* batch, unsigned flags, char* err, size_t errlen) {
  return kv_rows(ctx, cache, rows, batch, true, flags, {err, errlen, "kv_write"});
}

int dmh_kv_read(dmh_ctx* ctx, const dmh_kv_cache* cache, const dmh_kv_rows* rows,
                const dmh_seq_batch* batch, unsigned flags, char* err, size_t errlen) {
  return kv_rows(ctx, cache, rows, batch, false, flags, {err, errlen, "kv_read"});
}

int dmh_attention_forward(dmh_ctx* ctx, const dmh_attention* args, const dmh_kv_cache* cache,
                          const dmh_seq_batch* batch, unsigned flags, char* errp, size_t errlen) {
  const Err err{errp, errlen, "attention"};
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!args) return err.arg("args is NULL");
  int rc = check_cache(cache, err);
  if (rc) return rc;
  dmh_kv_cache c = *cache;
  dmh_attention a = *args;
  if (!known(a.dtype)) return err.arg("unknown dtype");
  if (a.q_heads < 1 || a.q_heads > 4096 || a.q_heads % c.kv_heads)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "q_heads %d, kv_heads %d (need q_heads a multiple of kv_heads, up to 4096)", a.q_heads,
               c.kv_heads);
  // (within these the factor times log2(e) is a normal fp32 number)
  if (!(a.scale >= 1e-30f && a.scale <= 1e30f))
    return err.arg("scale must be positive, from 1e-30 to 1e30");
  if ((rc = check_batch(batch, dev, err, false))) return rc;
  dmh_seq_batch b = *batch;
  if (b.num_seqs == 0 || b.total_tokens == 0) return ctx ? DMH_OK : err.arg("ctx is NULL");
  if (!a.q || !a.o) return err.arg("q or o is NULL");
  if ((rc = check_arrays(c, err))) return rc;
  const size_t es = elem(a.dtype);
  const auto rows = [&](const void* p, int64_t stride, int64_t head_stride) {
    return head_rows(p, b.total_tokens, a.q_heads, c.dim, stride, head_stride, es);
  };
  const Rows q = rows(a.q, a.q_stride, a.q_head_stride), o = rows(a.o, a.o_stride, a.o_head_stride);
  const Rows gate = rows(a.gate, a.gate_stride, a.gate_head_stride);
  if (!heads_ok(q, c.dim) || !heads_ok(o, c.dim) || (a.gate && !heads_ok(gate, c.dim)))
    return err.arg(kBadRows);
  const int64_t n = (int64_t)cache_rows(c);
  const Rows codes{c.codes, n, c.dim / 2, c.dim / 2, 1};
  const Rows scales{c.scales, n, c.dim / 32, c.dim / 32, 1};
  for (const Rows* x : std::initializer_list<const Rows*>{&q, &gate, &codes, &scales})
    if (overlap(o, *x)) return err.arg("o must not overlap q, gate or the cache");
  if (!attend_fits(a, c, seq_dev(b, nullptr)))
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR", "too many rows or sequences for one call: %d, %d",
               b.total_tokens, b.num_seqs);
  if (!dev && (rc = check_pages(c, b, true, err))) return rc;
  if (!ctx) return err.arg("ctx is NULL");
  hipStream_t st;
  unsigned long long* status;
  if ((rc = api_mixer_begin(ctx, &st, &status, errp, errlen))) return rc;
  Stage stage;
  if (!dev) {
    stage.add(a.q, q.bytes());
    stage.add(a.gate, gate.bytes());
    stage.add_out(a.o, o);
    stage_cache(stage, c, b, nullptr, nullptr);
    stage_batch(stage, b);
    if ((rc = stage.in(ctx, st, check, err))) return rc;
  }
  const SeqDev s = seq_dev(b, status);
  void* ws = nullptr;
  if ((rc = api_mixer_buffer(ctx, kMixerParts, attend_bytes(a, c, s), &ws, errp, errlen))) return rc;
  if (check) return DMH_OK;
  const hipError_t e = launch_attend(a, c, s, ws, st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

}  // extern "C"
