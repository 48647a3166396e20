// Launchers of the training operators (xent.cu, orth.cu) behind api.cu.
#pragma once

#include "common.cuh"

namespace llattn {
namespace xent {
size_t workspace_bytes(const llattn_xent_args& a);
int launches(const llattn_xent_args& a);
cudaError_t launch(const llattn_xent_args& a, volatile unsigned* fault, cudaStream_t s);
cudaError_t launch_scale(void* a, int64_t na, void* b, int64_t nb, int dtype, const float* f, cudaStream_t s);
unsigned read_fault_word(bool reset);
}  // namespace xent
namespace orth {
size_t workspace_bytes(const llattn_orth_args& a);
int launches(const llattn_orth_args& a);
cudaError_t launch(const llattn_orth_args& a, volatile unsigned* fault, cudaStream_t s);
unsigned read_fault_word(bool reset);
}  // namespace orth
}  // namespace llattn
