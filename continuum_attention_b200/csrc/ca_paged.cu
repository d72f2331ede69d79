// ca_paged.cu -- Continuum Attention of new tokens over a paged cache, for serving.
//
// The simplest form: one warp per (row, query head) walks the row's keys in order.
#include <algorithm>

#include "ca_common.cuh"
#include "ca_internal.h"
#include "ca_paged.cuh"

namespace ca {
namespace paged {

constexpr int kWarps = 8;

template <typename T>
__device__ void simple_row(const Args& a, int s, int t, int h) {
  const int lane = threadIdx.x & 31;
  const int start = a.q_starts[s], n = a.q_starts[s + 1] - start, len = a.kv_lens[s];
  if (start < 0 || n > a.rows - start) { record_invalid(); return; }
  T* o = (T*)a.o + ((size_t)(start + t) * a.H + h) * a.D;
  const int i = len - n + t;
  bool bad = len < 0 || len > (long long)a.pages_per_seq * a.page_size;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, vp[4] = {0.f, 0.f, 0.f, 0.f};
  const float scale = expf(a.log_gain[h]) * a.inv_sqrt_d;
  const T* q = (const T*)a.q + (size_t)(start + t) * a.q_token_stride + (size_t)h * a.q_head_stride;
#pragma unroll
  for (int u = 0; u < 4; ++u) qv[u] = lane + 32 * u < a.D ? to_f32<T>(q[lane + 32 * u]) : 0.f;
  const int g = h / (a.H / a.G);
  float m = -INFINITY, z = 0.f, sa = 0.f, ea = 0.f, right = 0.f;
  for (int j = 0; j <= i && !bad; ++j) {
    const int page = a.page_table[(size_t)s * a.page_table_stride + j / a.page_size];
    if (page < 0 || page >= a.num_pages) { bad = true; break; }
    const size_t at = (size_t)page * a.page_stride + (size_t)g * a.head_stride + (size_t)(j % a.page_size) * a.slot_stride;
    float dot = 0.f, vv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 32 * u;
      vv[u] = d < a.D ? to_f32<T>(((const T*)a.v_cache)[at + d]) : 0.f;
      if (d < a.D) dot = fmaf(qv[u], to_f32<T>(((const T*)a.k_cache)[at + d]), dot);
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float sb = dot * scale;
    if (sb > m) {
      const float f = j ? exp_rel(m - sb) : 0.f;
      m = sb;
      z *= f;
      ea *= f;
      right *= f;
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] *= f;
    }
    const float eb = exp_rel(sb - m);
    if (j == 0) {
      right = 0.5f * eb;   // the first key's cap
      z += right;
    } else {
      float M0, M1;
      seg_moments01(ea, eb, sb - sa, M0, M1);
      z += M0;
      const float wl = right + (M0 - M1);
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = fmaf(wl, vp[u], acc[u]);
      right = M1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) vp[u] = vv[u];
    sa = sb;
    ea = eb;
  }
  if (bad && lane == 0) record_invalid();
  z += 0.5f * ea;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + 32 * u;
    float y = i < 0 ? 0.f : fmaf(right + 0.5f * ea, vp[u], acc[u]) / z;
    if (bad) y = __int_as_float(0x7fffffff);
    if (d < a.D) o[d] = from_f32<T>(y);
  }
}

template <typename T>
__global__ void simple_kernel(Args a) {
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.y, n = a.q_starts[s + 1] - a.q_starts[s];
  const long long w = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= (long long)a.max_q_len * a.H) return;
  for (int t = (int)(w / a.H); t < n; t += a.max_q_len) simple_row<T>(a, s, t, (int)(w % a.H));
}

size_t workspace_bytes(long long seqs, long long max_q_len, long long H, long long G, long long D, int dtype) {
  (void)seqs;
  return dtype == 0 ? 0 : mma_workspace_bytes(max_q_len, H, G, D);
}
int launches(const Args& a, int dtype) { return dtype == 0 ? 1 : mma_launches(a); }

template <typename T>
static cudaError_t forward_t(const Args& a) {
  const long long warps = (long long)a.max_q_len * a.H;
  return launch_pdl(simple_kernel<T>, dim3((unsigned)((warps + kWarps - 1) / kWarps), (unsigned)a.seqs),
                    dim3(kWarps * 32), 0, a.stream, a);
}

cudaError_t forward(const Args& a, int dtype, void* workspace) {
  return dtype == 0 ? forward_t<float>(a) : mma_forward(a, dtype, workspace);
}

cudaError_t read_status(int* out, bool reset) {
  int own = 0;
  cudaError_t e = mma_read_status(out, reset);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&own, g_status, sizeof(int));
  if (e != cudaSuccess) return e;
  if (*out == 0) *out = own;
  if (!reset || own == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
}

}  // namespace paged
}  // namespace ca
