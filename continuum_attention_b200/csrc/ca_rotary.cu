// ca_rotary.cu -- rotary positions in their general form, beside the decoder's own
// unpacking kernel (ca_rope.cu): interleaved or half layout, the first R of D head
// values, shared key heads, explicit positions, any cos/sin table (so any stretching
// of the context), for training (forward, gradient) and for serving (turned keys and
// values written straight into a paged cache).
//
// Pair p < R/2 of a head at position t is turned by the table's angle,
//   (x, y) -> (x c - y s, y c + x s),   (c, s) = table[t][p]  (float32, computed in 64 bits),
// with (x, y) = (h_{2p}, h_{2p+1}) interleaved or (h_p, h_{p+R/2}) in halves; values from R
// on and the value heads pass through.  The gradient is the transposed turn.  Arithmetic
// is fp32 with one rounding per output.
//
// HBM-bound: each element of [tokens][H + 2G][D] is read once and written once: 8 x 2048 tokens of 48
// heads of 64 in bf16 take 34.5 us forward and 36.6 backward for 201 MB each (5.8 and 5.5 TB/s), 1731 tokens
// of 20 heads in f32 3.9 and 4.3 us, 1540 tokens of 48 heads of 128 into a cache 8.8 us for 38 MB (14 where
// nothing of it is in L2), the 64 tokens of a decoding step 2.8 us (latency; 4.1).  An item
// is two vectors of W elements of one head: the two that a turn in halves combines, else
// two adjacent ones.  A thread keeps its item for several heads, so that it reads the
// table once, and loads kHeads heads before it stores the first.
#include <algorithm>

#include "ca_common.cuh"
#include "ca_internal.h"

namespace ca {
namespace rotary {

// set to CA_ERR_INVALID_ARGUMENT by a token whose position, length or page lies outside its table
__device__ int g_status = 0;
__device__ __forceinline__ void record_invalid() { atomicCAS(&g_status, 0, 1); }

// W consecutive elements as they are; p aligned to W elements (at least; 16 bytes where W is 8)
template <typename T, int W>
struct Raw {
  static constexpr int kBytes = W * (int)sizeof(T);
  alignas(kBytes < 16 ? kBytes : 16) T e[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
    } else {
      e[0] = p[0];
    }
  }
  __device__ __forceinline__ void get(float (&x)[W]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = to_f32<T>(e[i]);
  }
};

template <typename T, int W>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[W]) {
  constexpr int kBytes = W * (int)sizeof(T);
  alignas(16) T e[W];
#pragma unroll
  for (int i = 0; i < W; ++i) e[i] = from_f32<T>(x[i]);
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
  } else {
    p[0] = e[0];
  }
}

// One item: the vectors at a and b (b < 0: none) of a head, and whether they are turned.
// In halves the two vectors are the x and y of W pairs; interleaved each holds W/2 pairs.
template <int W, bool kHalf>
struct Item {
  int a, b;
  bool turn;
  float c[W], s[W];   // half: pair i of the item; interleaved: pair i of vector a (i < W/2), then of b

  __device__ __forceinline__ Item(int it, int D, int R) {
    const int np = R / (2 * W);
    if (kHalf && it < np) {
      a = it * W;
      b = R / 2 + it * W;
      turn = true;
    } else {
      // 2 np vectors are paired (kHalf), the others follow in order
      a = 2 * it * W;
      b = a + W < D ? a + W : -1;
      turn = !kHalf && a < R;
    }
  }
  // row: the position's [R/2][2] of the table; bad: NaN instead (a position outside the table)
  __device__ __forceinline__ void angles(const float2* row, bool bad, float sign, int R) {
    if (!turn) return;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int pair = kHalf ? a + i : a / 2 + i;
      float2 w = make_float2(1.f, 0.f);
      if (bad) w = make_float2(__int_as_float(0x7fffffff), 0.f);
      else if (kHalf || 2 * pair < R) w = row[pair];
      c[i] = w.x;
      s[i] = sign * w.y;
    }
  }
  __device__ __forceinline__ void apply(float (&x)[W], float (&y)[W], int R) const {
    if (!turn) return;
    if constexpr (kHalf) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float e = x[i], o = y[i];
        x[i] = fmaf(e, c[i], -o * s[i]);
        y[i] = fmaf(o, c[i], e * s[i]);
      }
    } else if constexpr (W > 1) {
#pragma unroll
      for (int i = 0; i < W / 2; ++i) {
        const float e = x[2 * i], o = x[2 * i + 1];
        x[2 * i] = fmaf(e, c[i], -o * s[i]);
        x[2 * i + 1] = fmaf(o, c[i], e * s[i]);
      }
      if (b >= 0 && b < R) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const float e = y[2 * i], o = y[2 * i + 1];
          y[2 * i] = fmaf(e, c[W / 2 + i], -o * s[W / 2 + i]);
          y[2 * i + 1] = fmaf(o, c[W / 2 + i], e * s[W / 2 + i]);
        }
      }
    }
  }
};

__host__ __device__ __forceinline__ int items_per_head(int D, int W) { return (D / W + 1) / 2; }

// the position's row of the table, or bad
__device__ __forceinline__ const float2* table_row(const float2* cs, long long pos, int rows, int R, bool& bad) {
  bad = pos < 0 || pos >= rows;
  return cs + (bad ? 0 : (size_t)pos * (R / 2));
}

// heads of a thread whose loads are in flight at once: one is 50% slower on a training batch, four are as
// fast as two in 32 bits and 60% slower in 16 (registers)
constexpr int kHeads = 2;

// training, forward: qkv [B*T rows][(H+2G) D] -> q [B,H,T,D], k, v [B,G,T,D] (q, k turned);
// backward: the other way with the transposed turn.  A block takes a token: four, whose
// rows of one head lie side by side in q, k and v, ran 4 to 9% slower.
template <typename T, int W, bool kHalf, bool kBack>
__global__ void qkv_kernel(const __grid_constant__ QkvArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int ni = items_per_head(a.D, W), heads = a.H + 2 * a.G;
  const int it = (int)threadIdx.x % ni, step = (int)blockDim.x / ni;
  const long long token = blockIdx.x;
  const int b = (int)(token / a.T), t = (int)(token - (long long)b * a.T);
  const long long pos = a.positions ? (long long)a.positions[(size_t)b * a.pos_stride + t] : t;
  bool bad;
  const float2* row = table_row((const float2*)a.cos_sin, pos, a.table_rows, a.R, bad);
  if (bad && threadIdx.x == 0) record_invalid();
  Item<W, kHalf> item(it, a.D, a.R);
  T* packed = (T*)a.qkv + (size_t)token * a.qkv_stride;
  auto split = [&](int h) {
    if (h < a.H) return (T*)a.q + (((size_t)b * a.H + h) * a.T + t) * a.D;
    if (h < a.H + a.G) return (T*)a.k + (((size_t)b * a.G + (h - a.H)) * a.T + t) * a.D;
    return (T*)a.v + (((size_t)b * a.G + (h - a.H - a.G)) * a.T + t) * a.D;
  };
  bool angles = false;
  for (int h0 = (int)threadIdx.x / ni; h0 < heads; h0 += step * kHeads) {
    Raw<T, W> x[kHeads], y[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * step;
      if (h >= heads) continue;
      const T* src = kBack ? split(h) : packed + (size_t)h * a.D;
      x[u].load(src + item.a);
      if (item.b >= 0) y[u].load(src + item.b);
    }
    if (!angles) item.angles(row, bad, kBack ? -1.f : 1.f, a.R);
    angles = true;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * step;
      if (h >= heads) continue;
      float v[W], w[W];
      x[u].get(v);
      y[u].get(w);
      if (h < a.H + a.G) item.apply(v, w, a.R);
      T* dst = kBack ? packed + (size_t)h * a.D : split(h);
      store_vec<T, W>(dst + item.a, v);
      if (item.b >= 0) store_vec<T, W>(dst + item.b, w);
    }
  }
}

// serving: token n of sequence s (q_starts[s] <= n < q_starts[s+1]) sits at position
// kv_lens[s] - (q_starts[s+1] - n); its queries go to q [N,H,D], its keys and values to
// slot pos % page_size of page page_table[s][pos / page_size].  The first heads' loads are
// issued before the sequence is looked up.
template <typename T, int W, bool kHalf>
__global__ void append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int ni = items_per_head(a.D, W), heads = a.H + 2 * a.G;
  const int it = (int)threadIdx.x % ni, step = (int)blockDim.x / ni;
  const int n = (int)blockIdx.x;
  Item<W, kHalf> item(it, a.D, a.R);
  const T* src0 = (const T*)a.qkv + (size_t)n * a.qkv_stride;
  Raw<T, W> x[kHeads], y[kHeads];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * step;
      if (h >= heads) continue;
      x[u].load(src0 + (size_t)h * a.D + item.a);
      if (item.b >= 0) y[u].load(src0 + (size_t)h * a.D + item.b);
    }
  };
  int h0 = (int)threadIdx.x / ni;
  fetch(h0);
  // The thread that finds the token's sequence looks its place up.  (Starts that decrease could let
  // several find one; each writes a place that is in range.)
  __shared__ long long s_pos, s_cache;   // s_pos = -1: no key; s_cache = -1: a page or position out of range
  __shared__ int s_found;
  if (threadIdx.x == 0) s_found = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < a.seqs; s += blockDim.x) {
    const int start = a.q_starts[s], end = a.q_starts[s + 1], len = a.kv_lens[s];
    const bool outside = start < 0 || end > a.tokens || start > end;   // rows that the buffers do not have
    if (outside && n == 0) record_invalid();
    if (outside || start > n || n >= end) continue;
    const long long p = (long long)len - end + n;
    long long cache = -1;
    if (p >= 0 && p < a.table_rows) {
      const long long col = p / a.page_size;
      int page = -1;
      if (col < a.pages_per_seq) page = a.page_table[(size_t)s * a.page_table_stride + col];
      if (page >= 0 && page < a.num_pages)
        cache = (long long)page * a.page_stride + (p - col * a.page_size) * a.slot_stride;
    }
    s_pos = p < 0 ? -1 : cache < 0 ? 0 : p;   // in the table whoever wrote s_cache
    s_cache = cache;
    s_found = 1;
  }
  __syncthreads();
  if (!s_found) return;   // a row behind the last sequence
  const bool none = s_pos < 0;   // more rows than keys: no key to write, no row to answer
  const bool bad = !none && s_cache < 0;
  const size_t cache = none || bad ? 0 : (size_t)s_cache;
  const float2* row = (const float2*)a.cos_sin + (none || bad ? 0 : (size_t)s_pos * (a.R / 2));
  if (bad && threadIdx.x == 0) record_invalid();
  item.angles(row, bad, 1.f, a.R);
  for (; h0 < heads; h0 += step * kHeads, fetch(h0)) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int h = h0 + u * step;
      if (h >= heads || (h >= a.H && (none || bad))) continue;
      T* dst;
      if (h < a.H) dst = (T*)a.q + ((size_t)n * a.H + h) * a.D;
      else if (h < a.H + a.G) dst = (T*)a.k_cache + cache + (size_t)(h - a.H) * a.head_stride;
      else dst = (T*)a.v_cache + cache + (size_t)(h - a.H - a.G) * a.head_stride;
      float v[W], w[W];
      x[u].get(v);
      y[u].get(w);
      if (none || bad) {
        const float fill = bad ? __int_as_float(0x7fffffff) : 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = w[i] = fill;
      } else if (h < a.H + a.G) {
        item.apply(v, w, a.R);
      }
      store_vec<T, W>(dst + item.a, v);
      if (item.b >= 0) store_vec<T, W>(dst + item.b, w);
    }
  }
}

// Elements per vector: the widest of 8 (16-bit types), 4, 2, 1 that the layout's pairs divide into (halves
// start at R/2, so a vector may not straddle it; interleaved pairs lie within a vector).  Eight f32 values
// and their angles cost registers that four do not (5.1 against 3.9 us on 1731 tokens of 20 heads).
int vector_width(int R, int half, bool f32) {
  const int m = half ? R / 2 : R;
  return m % 8 == 0 && !f32 ? 8 : m % 4 == 0 ? 4 : m % 2 == 0 ? 2 : 1;
}

// threads per token: whole heads of items, about `want` threads at most, each with `at_once` heads a round, and
// no more than the rounds need
static int token_threads(int heads, int ni, int want, int at_once) {
  int per = std::max(1, std::min(want / ni, (heads + at_once - 1) / at_once));
  const int rounds = (heads + per * at_once - 1) / (per * at_once);
  per = (heads + rounds * at_once - 1) / (rounds * at_once);
  return per * ni;
}

template <typename T, int W, bool kHalf>
static cudaError_t qkv_t(const QkvArgs& a, bool back) {
  const int lanes = token_threads(a.H + 2 * a.G, items_per_head(a.D, W), 256, kHeads);
  const dim3 grid((unsigned)((long long)a.B * a.T)), block((unsigned)lanes);
  return back ? launch_pdl(qkv_kernel<T, W, kHalf, true>, grid, block, 0, a.stream, a)
              : launch_pdl(qkv_kernel<T, W, kHalf, false>, grid, block, 0, a.stream, a);
}

template <typename T, int W, bool kHalf>
static cudaError_t append_t(const AppendArgs& a) {
  const int threads = token_threads(a.H + 2 * a.G, items_per_head(a.D, W), 256, kHeads);
  return launch_pdl(append_kernel<T, W, kHalf>, dim3((unsigned)a.tokens), dim3((unsigned)threads), 0, a.stream, a);
}

// dispatch on type, layout and vector width; FN<T, W, kHalf>
#define CA_ROTARY_W(FN, T, HALF, ...)                     \
  switch (vector_width(a.R, a.half, sizeof(T) == 4)) {    \
    case 8: return FN<T, sizeof(T) == 4 ? 4 : 8, HALF>(__VA_ARGS__); \
    case 4: return FN<T, 4, HALF>(__VA_ARGS__);           \
    case 2: return FN<T, 2, HALF>(__VA_ARGS__);           \
    default: return FN<T, HALF ? 1 : 2, HALF>(__VA_ARGS__); \
  }
#define CA_ROTARY_T(FN, T, ...)                                    \
  if (a.half) { CA_ROTARY_W(FN, T, true, __VA_ARGS__) }            \
  CA_ROTARY_W(FN, T, false, __VA_ARGS__)

template <typename T>
static cudaError_t qkv_type(const QkvArgs& a, bool back) {
  CA_ROTARY_T(qkv_t, T, a, back)
}
template <typename T>
static cudaError_t append_type(const AppendArgs& a) {
  CA_ROTARY_T(append_t, T, a)
}
#undef CA_ROTARY_T
#undef CA_ROTARY_W

cudaError_t qkv(const QkvArgs& a, int dtype, bool back) {
  switch (dtype) {
    case 0: return qkv_type<float>(a, back);
    case 1: return qkv_type<__nv_bfloat16>(a, back);
    default: return qkv_type<__half>(a, back);
  }
}

cudaError_t append(const AppendArgs& a, int dtype) {
  switch (dtype) {
    case 0: return append_type<float>(a);
    case 1: return append_type<__nv_bfloat16>(a);
    default: return append_type<__half>(a);
  }
}

cudaError_t read_status(int* out, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
  if (e != cudaSuccess || !reset || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
}

}  // namespace rotary
}  // namespace ca
