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
// up to few_tokens, forward only, nothing kept (gated_few.cu); 2 launches
int few_tokens(const llattn_gated_args& a);
size_t few_workspace_bytes(const llattn_gated_args& a);
cudaError_t launch_few(const llattn_gated_args& a, cudaStream_t s);
}  // namespace gated
}  // namespace llattn
