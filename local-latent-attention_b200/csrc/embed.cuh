// Launchers of the token embedding (embed.cu) behind api.cu.
#pragma once

#include "common.cuh"

namespace llattn {
namespace embed {
size_t workspace_bytes(const llattn_embed_args& a);
int launches(const llattn_embed_args& a, bool backward);
cudaError_t launch_fwd(const llattn_embed_args& a, cudaStream_t s);
cudaError_t launch_bwd(const llattn_embed_args& a, cudaStream_t s);
}  // namespace embed
}  // namespace llattn
