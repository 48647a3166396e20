// Launchers of the norm over many tensors and the clipping (clip.cu) behind api.cu.
#pragma once

#include "common.cuh"

namespace llattn {
namespace clip {
size_t workspace_bytes(const llattn_clip_args& a);
int launches(const llattn_clip_args& a);
cudaError_t launch(const llattn_clip_args& a, cudaStream_t s);
}  // namespace clip
}  // namespace llattn
