// Attention of new tokens over a paged cache, a window and a few first tokens
// that stay visible (kda_paged_hip.h), by the kernels in kda_paged_attn.h.
#include "kda_paged_attn.h"

namespace kda {

size_t paged_attn_workspace(const SinkParams& p, int D) { return attn_workspace(p, D); }
hipError_t launch_paged_attn(const SinkParams& p, int D, hipStream_t stream) { return launch_attn(p, D, stream); }

}  // namespace kda
