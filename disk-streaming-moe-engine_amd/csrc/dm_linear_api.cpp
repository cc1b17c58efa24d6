// dm_linear_api.cpp -- C ABI of the linear layers with 4-bit weights.
#include <hip/hip_runtime.h>

#include <new>

#include "dm_api_rows.h"
#include "dm_linear.h"

namespace {

using namespace dm;

// Device memory that is freed at the end of its scope.
struct Temp {
  void* p = nullptr;
  ~Temp() {
    if (p) (void)hipFree(p);
  }
};

int check_weights(const dmh_linear_weights* w, const Err& err) {
  if (!w) return err.arg("weights is NULL");
  const int g = w->group_size;
  if ((g != 32 && g != 64 && g != 128 && g != 256) || w->out_features < 1 ||
      w->out_features > 1 << 24 || w->in_features < 1 || w->in_features > 1 << 20 || w->in_features % g)
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR",
               "out_features %d, in_features %d, group_size %d (need 1 to 2^24, a multiple of the"
               " group size up to 2^20, and 32, 64, 128 or 256)", w->out_features, w->in_features, g);
  if (!w->scales || !w->packed) return err.arg("scales or packed is NULL");
  if (!aligned(w->scales, 2) || !aligned(w->bias, 4)) return err.arg("scales or bias is misaligned");
  return DMH_OK;
}

}  // namespace

extern "C" {

int dmh_upload_linear(dmh_ctx* c, const dmh_linear_weights* w, unsigned flags, dmh_linear** out,
                      char* errp, size_t errlen) {
  const Err err{errp, errlen, "linear"};
  int rc = check_weights(w, err);
  if (rc) return rc;
  if (!c || !out) return err.arg("ctx or out is NULL");
  *out = nullptr;
  hipStream_t st;
  unsigned long long* vkey;
  if ((rc = api_upload_begin(c, &st, &vkey, errp, errlen))) return rc;
  const int64_t n = w->out_features, k = w->in_features;
  const size_t scale_bytes = (size_t)(n * k / w->group_size) * 2, packed_bytes = (size_t)(n * k / 2);
  const int rb = linear_row_blocks((int)n), chunks = linear_chunks((int)k);
  const size_t nib_bytes = (size_t)rb * chunks * 1024, sc_bytes = (size_t)rb * chunks * 128;
  dmh_linear* l = new (std::nothrow) dmh_linear{};
  if (!l) return err(DMH_ERR_NO_MEMORY, "HIP_ERROR", "out of host memory");
  const auto fail = [&](int code) {
    if (l->buf) (void)hipFree(l->buf);
    delete l;
    return code;
  };
  if ((rc = api_malloc(nib_bytes + sc_bytes + (size_t)(w->bias ? 4 * n : 0), &l->buf, errp, errlen)))
    return fail(rc);
  uint8_t* const nib = static_cast<uint8_t*>(l->buf);
  uint16_t* const sc = reinterpret_cast<uint16_t*>(nib + nib_bytes);
  float* const bias = reinterpret_cast<float*>(nib + nib_bytes + sc_bytes);
  l->ctx = c;
  l->dev = {(int)n, (int)k, rb, chunks, nib, sc, w->bias ? bias : nullptr};
  const uint16_t* scales = w->scales;
  const uint8_t* packed = w->packed;
  hipError_t e = hipSuccess;
  Temp temp;
  if (!(flags & DMH_F_DEVICE)) {
    const size_t at = (scale_bytes + 255) & ~(size_t)255;
    if ((rc = api_malloc(at + packed_bytes, &temp.p, errp, errlen))) return fail(rc);
    uint8_t* const t = static_cast<uint8_t*>(temp.p);
    e = hipMemcpyAsync(t, scales, scale_bytes, hipMemcpyHostToDevice, st);
    if (e == hipSuccess) e = hipMemcpyAsync(t + at, packed, packed_bytes, hipMemcpyHostToDevice, st);
    scales = reinterpret_cast<const uint16_t*>(t);
    packed = t + at;
  }
  unsigned long long key = kNoError;
  if (e == hipSuccess) e = hipMemcpyAsync(vkey, &key, 8, hipMemcpyHostToDevice, st);
  if (e == hipSuccess) e = launch_linear_pack(scales, packed, (int)n, (int)k, w->group_size, nib, sc,
                                              vkey, st);
  if (e == hipSuccess && w->bias) e = hipMemcpyAsync(bias, w->bias, 4 * n, hipMemcpyDefault, st);
  if (e == hipSuccess) e = hipMemcpyAsync(&key, vkey, 8, hipMemcpyDeviceToHost, st);
  if (e == hipSuccess) e = hipStreamSynchronize(st);
  if (e != hipSuccess) return fail(err.hip(e));
  // (the texts of src/quant/dequant_kernel.mojo:68-108)
  if (key == 1ull << 60)
    return fail(err(DMH_ERR_DEQUANT, "DEQUANT_ERROR",
                    "dequant_kernel: reserved nibble 0b1000 (-8) encountered"));
  if (key != kNoError)
    return fail(err(DMH_ERR_DEQUANT, "DEQUANT_ERROR", "dequant_kernel: scale is %s at group %llu",
                    key & 1 ? "non-positive" : "NaN or Inf", key >> 1));
  if ((rc = api_keep_linear(c, l, errp, errlen))) return fail(rc);
  *out = l;
  return DMH_OK;
}

int dmh_free_linear(dmh_ctx* c, dmh_linear* l) {
  if (!c || !l || !api_drop_linear(c, l)) return DMH_ERR_INVALID_ARG;
  (void)hipFree(l->buf);  // (waits for the work queued on it)
  delete l;
  return DMH_OK;
}

int dmh_linear_forward(dmh_ctx* c, const dmh_linear* l, const dmh_linear_rows* rows, unsigned flags,
                       char* errp, size_t errlen) {
  const Err err{errp, errlen, "linear"};
  const bool dev = flags & DMH_F_DEVICE, check = flags & DMH_F_CHECK;
  if (!rows) return err.arg("rows is NULL");
  dmh_linear_rows r = *rows;
  if (!known(r.dtype) || (r.out_dtype != r.dtype && r.out_dtype != DMH_DTYPE_F32))
    return err.arg("dtype must be known and out_dtype the same or F32");
  if (r.rows < 0 || r.rows >= kRowsLimit) return err.arg("rows must be from 0 to below 2^30");
  if (!c || !l) return err.arg("ctx or the linear layer is NULL");
  if (l->ctx != c) return err.arg("the linear layer is another context's");
  if (r.rows == 0) return DMH_OK;
  if (!r.x || !r.y) return err.arg("x or y is NULL");
  const Rows x{r.x, r.rows, l->dev.k, r.x_stride, elem(r.dtype)};
  const Rows y{r.y, r.rows, l->dev.n, r.y_stride, elem(r.out_dtype)};
  if (!x.ok() || !y.ok()) return err.arg("a stride is shorter than its row, or an array is misaligned");
  if (overlap(x, y)) return err.arg("x and y must not overlap");
  if (!linear_fits(l->dev, r))
    return err(DMH_ERR_CONFIG, "CONFIG_ERROR", "too many rows for one call: %d", r.rows);
  hipStream_t st;
  unsigned long long* status;
  int rc = api_mixer_begin(c, &st, &status, errp, errlen);
  if (rc) return rc;
  Stage stage;
  if (!dev) {
    stage.add(r.x, x.bytes());
    stage.add_out(r.y, y);
    if ((rc = stage.in(c, st, check, err))) return rc;
  }
  void* ws = nullptr;
  const size_t need = linear_bytes(l->dev, r);
  if (need && (rc = api_mixer_buffer(c, kMixerSplit, need, &ws, errp, errlen))) return rc;
  if (check) return DMH_OK;
  const hipError_t e = launch_linear(l->dev, r, ws, st);
  if (e != hipSuccess) return err.hip(e);
  return dev ? DMH_OK : stage.out(st, err);
}

}  // extern "C"
