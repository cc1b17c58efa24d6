// dm_linear.h -- a 4-bit linear layer on the device, and the host-side launchers of
// its kernels (dm_linear.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/dismoen_hip.h"
#include "dm_layout.h"

namespace dm {

// W [n][k] in the A16 layout, its rows padded to 16 and its columns to 128 with zeros.
struct LinearDev {
  int n, k, row_blocks, chunks;  // chunks of 128 columns
  const uint8_t* nib;
  const uint16_t* sc;
  const float* bias;  // [n] or NULL
};

inline int linear_row_blocks(int n) { return (n + kTileRows - 1) / kTileRows; }
inline int linear_chunks(int k) { return (k + kQuadCols - 1) / kQuadCols; }

// The caller's layout (fp16 scales [n * k / group], packed codes [n * k / 2]) to A16;
// what is wrong with it goes into *vkey as 2 * group + kind (0 NaN or infinite, 1 not
// positive), a reserved code as 1 << 60.
hipError_t launch_linear_pack(const uint16_t* scales, const uint8_t* packed, int n, int k, int group,
                              uint8_t* nib, uint16_t* sc, unsigned long long* vkey, hipStream_t st);

// Whether a launch holds the call's work.
bool linear_fits(const LinearDev& l, const dmh_linear_rows& r);
// ws: linear_bytes of device memory (0: none), 16-byte aligned.
size_t linear_bytes(const LinearDev& l, const dmh_linear_rows& r);
hipError_t launch_linear(const LinearDev& l, const dmh_linear_rows& r, void* ws, hipStream_t st);

}  // namespace dm

// A linear layer of a context.
struct dmh_linear {
  dmh_ctx* ctx;
  void* buf;
  dm::LinearDev dev;
};
