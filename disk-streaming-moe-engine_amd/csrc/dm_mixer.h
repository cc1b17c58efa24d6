// dm_mixer.h -- host-side launchers of the token mixer's kernels: the short
// convolution and the norms (dm_mixer.hip), the gated delta rule row by row
// (dm_mixer.hip) and in chunks (dm_delta.hip).
//
// Every array is device memory; sizes, strides and alignment have been checked
// (dm_mixer_api.cpp).  What only the device knows, the sequences, is checked by
// the kernels (seq_range) before any row or state is touched.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/dismoen_hip.h"

namespace dm {

// dmh_seq_batch on the device.
struct SeqDev {
  int num, rows, max_len, slots_n;
  const int32_t* off;
  const int32_t* slots;
  const int32_t* fresh;
  unsigned long long* status;
};

hipError_t launch_short_conv(const dmh_short_conv& a, const SeqDev& s, hipStream_t st);
hipError_t launch_gated_norm(const dmh_gated_norm& a, hipStream_t st);

// The delta rule row by row.
hipError_t launch_delta_rows(const dmh_gated_delta& a, const SeqDev& s, hipStream_t st);

// Sequences of min_rows rows and more in chunks of kDeltaChunk, the others row by
// row.  delta_chunk_count is the most chunks there can be; room of them are worked
// on at a time, in ws of room times delta_chunk_bytes.
constexpr int kDeltaChunk = 64;
int64_t delta_chunk_count(const SeqDev& s, int min_rows);
size_t delta_chunk_bytes(const dmh_gated_delta& a);
hipError_t launch_delta(const dmh_gated_delta& a, const SeqDev& s, int min_rows, int64_t chunks,
                        int64_t room, void* ws, hipStream_t st);

}  // namespace dm
