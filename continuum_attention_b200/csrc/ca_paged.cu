// ca_paged.cu -- Continuum Attention of new tokens over a paged cache: the choice of kernels.
//
// bf16 and f16 run on the tensor cores (decoding and short chunks ca_paged_mma.cu, long
// chunks ca_paged_tc.cu), f32 on the FMA pipes (ca_paged_simt.cu), whose scores are exact to 32 bits as f32
// inputs ask.
#include "ca_paged.cuh"

namespace ca {
namespace paged {

size_t workspace_bytes(long long seqs, long long max_q_len, long long H, long long G, long long D, int dtype) {
  (void)seqs;
  return dtype == 0 ? simt_workspace_bytes(max_q_len, H, G, D) : mma_workspace_bytes(max_q_len, H, G, D);
}

int launches(const Args& a, int dtype) { return dtype == 0 ? simt_launches(a) : mma_launches(a); }

cudaError_t forward(const Args& a, int dtype, void* workspace) {
  return dtype == 0 ? simt_forward(a, workspace) : mma_forward(a, dtype, workspace);
}

cudaError_t read_status(int* out, bool reset) {
  int more[2] = {0, 0};
  cudaError_t e = mma_read_status(out, reset);
  if (e == cudaSuccess) e = tc_read_status(&more[0], reset);
  if (e == cudaSuccess) e = simt_read_status(&more[1], reset);
  if (*out == 0) *out = more[0] ? more[0] : more[1];
  return e;
}

}  // namespace paged
}  // namespace ca
