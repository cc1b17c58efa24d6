// dm_api_internal.h -- helpers shared by the C ABI's translation units.
#ifndef DM_API_INTERNAL_H
#define DM_API_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stddef.h>

#include "../../include/dismoen_hip.h"

namespace dm {

// CONFIG_ERROR unless the 4-bit layer dimensions are supported (group size
// in {32, 64, 128, 256}, H / I / I_sh multiples of 128, E <= 2048, K <= 32).
// Callers run it before any size arithmetic or allocation on the dims.
int api_moe_dims_check(const dmh_moe_dims* d, int layer, char* err, size_t errlen);

// ---- what the token mixer's entry points (dm_mixer_api.cpp) use of a context --
// Makes the context's device current; its stream and the status word of these
// calls.
int api_mixer_begin(dmh_ctx* c, hipStream_t* st, unsigned long long** status, char* err,
                    size_t errlen);
// Device memory of the context, kept and grown from call to call.  A buffer
// whose address a captured graph holds is not freed when it grows, and none is
// made while the stream is being captured (DMH_ERR_INVALID_ARG).
enum MixerBuffer { kMixerStage, kMixerChunks, kMixerParts, kMixerSplit, kMixerBuffers };
int api_mixer_buffer(dmh_ctx* c, MixerBuffer which, size_t bytes, void** p, char* err,
                     size_t errlen);
// The text of a key that these calls recorded.
int api_mixer_error(unsigned long long key, char* err, size_t errlen);

// ---- what the linear layers' entry points (dm_linear_api.cpp) use besides --------
// Makes the context's device current for an upload, which a capture cannot hold; its
// stream and the word that checks of weights report to.
int api_upload_begin(dmh_ctx* c, hipStream_t* st, unsigned long long** vkey, char* err,
                     size_t errlen);
// Device memory on the current device.
int api_malloc(size_t bytes, void** p, char* err, size_t errlen);
// The context's linear layers, which end with it at the latest.
int api_keep_linear(dmh_ctx* c, dmh_linear* l, char* err, size_t errlen);
bool api_drop_linear(dmh_ctx* c, dmh_linear* l);

}  // namespace dm

#endif
