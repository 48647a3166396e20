// Launchers of the gated feed-forward block (gated.cu) behind api.cu.
#pragma once

#include "common.cuh"

namespace llattn {
namespace gated {
size_t kept_bytes(const llattn_gated_args& a);
size_t workspace_bytes(const llattn_gated_args& a, bool backward);
int launches(const llattn_gated_args& a, bool backward);
cudaError_t launch(const llattn_gated_args& a, bool backward, volatile unsigned* fault, cudaStream_t s);
unsigned read_fault_word(bool reset);
}  // namespace gated
}  // namespace llattn
