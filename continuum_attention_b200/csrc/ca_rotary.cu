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
// HBM-bound: each element of [tokens][H + 2G][D] is read once and written once.  An item
// is two vectors of W elements of one head: the two that a turn in halves combines, else
// two adjacent ones, so either layout keeps two independent loads of 16 bytes (16-bit
// types) or 32 (fp32) in flight per item.  A block takes one token and its threads stride over the token's
// heads by whole heads, so that a thread keeps its item and reads the table once.
#include "ca_common.cuh"
#include "ca_internal.h"

namespace ca {
namespace rotary {

// set to CA_ERR_INVALID_ARGUMENT by a token whose position, length or page lies outside its table
__device__ int g_status = 0;
__device__ __forceinline__ void record_invalid() { atomicCAS(&g_status, 0, 1); }

// W consecutive elements in 32 bits; p aligned to W elements (at least; 16 bytes where W is 8)
template <typename T, int W>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[W]) {
  constexpr int kBytes = W * (int)sizeof(T);
  alignas(16) T e[W];
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
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = to_f32<T>(e[i]);
}

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

// training, forward: qkv [B*T rows][(H+2G) D] -> q [B,H,T,D], k, v [B,G,T,D] (q, k turned);
// backward: the other way with the transposed turn
template <typename T, int W, bool kHalf, bool kBack>
__global__ void qkv_kernel(QkvArgs a) {
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
  item.angles(row, bad, kBack ? -1.f : 1.f, a.R);
  T* packed = (T*)a.qkv + (size_t)token * a.qkv_stride;
  for (int h = (int)threadIdx.x / ni; h < heads; h += step) {
    T* split;
    if (h < a.H) split = (T*)a.q + (((size_t)b * a.H + h) * a.T + t) * a.D;
    else if (h < a.H + a.G) split = (T*)a.k + (((size_t)b * a.G + (h - a.H)) * a.T + t) * a.D;
    else split = (T*)a.v + (((size_t)b * a.G + (h - a.H - a.G)) * a.T + t) * a.D;
    T* flat = packed + (size_t)h * a.D;
    const T* src = kBack ? split : flat;
    T* dst = kBack ? flat : split;
    if (h < a.H + a.G) {
      float x[W], y[W];
      load_vec<T, W>(src + item.a, x);
      if (item.b >= 0) load_vec<T, W>(src + item.b, y);
      item.apply(x, y, a.R);
      store_vec<T, W>(dst + item.a, x);
      if (item.b >= 0) store_vec<T, W>(dst + item.b, y);
    } else {
      float x[W];
      load_vec<T, W>(src + item.a, x);
      store_vec<T, W>(dst + item.a, x);
      if (item.b >= 0) {
        load_vec<T, W>(src + item.b, x);
        store_vec<T, W>(dst + item.b, x);
      }
    }
  }
}

// serving: token n of sequence s (q_starts[s] <= n < q_starts[s+1]) sits at position
// kv_lens[s] - (q_starts[s+1] - n); its queries go to q [N,H,D], its keys and values to
// slot pos % page_size of page page_table[s][pos / page_size]
template <typename T, int W, bool kHalf>
__global__ void append_kernel(AppendArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int ni = items_per_head(a.D, W), heads = a.H + 2 * a.G;
  const int it = (int)threadIdx.x % ni, step = (int)blockDim.x / ni;
  const int n = (int)blockIdx.x;
  __shared__ int s_seq;
  if (threadIdx.x == 0) s_seq = -1;
  __syncthreads();
  for (int s = threadIdx.x; s < a.seqs; s += blockDim.x)
    if (a.q_starts[s] <= n && n < a.q_starts[s + 1]) atomicMax(&s_seq, s);
  __syncthreads();
  const int s = s_seq;
  if (s < 0) return;   // a row behind the last sequence
  const long long pos = (long long)a.kv_lens[s] - a.q_starts[s + 1] + n;
  const bool none = pos < 0;   // more rows than keys: no key to write, no row to answer
  bool bad = false;
  const float2* row = table_row((const float2*)a.cos_sin, none ? 0 : pos, a.table_rows, a.R, bad);
  size_t cache = 0;
  if (!none && !bad) {
    const long long col = pos / a.page_size;
    int page = -1;
    if (col < a.pages_per_seq) page = a.page_table[(size_t)s * a.page_table_stride + col];
    bad = page < 0 || page >= a.num_pages;
    if (!bad) cache = (size_t)page * a.page_stride + (size_t)(pos - col * a.page_size) * a.slot_stride;
  }
  if (bad && threadIdx.x == 0) record_invalid();
  Item<W, kHalf> item(it, a.D, a.R);
  item.angles(row, bad, 1.f, a.R);
  const T* src0 = (const T*)a.qkv + (size_t)n * a.qkv_stride;
  for (int h = (int)threadIdx.x / ni; h < heads; h += step) {
    if (h >= a.H && (none || bad)) break;
    const T* src = src0 + (size_t)h * a.D;
    T* dst;
    if (h < a.H) dst = (T*)a.q + ((size_t)n * a.H + h) * a.D;
    else if (h < a.H + a.G) dst = (T*)a.k_cache + cache + (size_t)(h - a.H) * a.head_stride;
    else dst = (T*)a.v_cache + cache + (size_t)(h - a.H - a.G) * a.head_stride;
    float x[W], y[W];
    load_vec<T, W>(src + item.a, x);
    if (item.b >= 0) load_vec<T, W>(src + item.b, y);
    if (none || bad) {
      const float fill = bad ? __int_as_float(0x7fffffff) : 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = y[i] = fill;
    } else if (h < a.H + a.G) {
      item.apply(x, y, a.R);
    }
    store_vec<T, W>(dst + item.a, x);
    if (item.b >= 0) store_vec<T, W>(dst + item.b, y);
  }
}

// Elements per vector: the widest of 8, 4, 2, 1 that the layout's pairs divide into (halves start
// at R/2, so a vector may not straddle it; interleaved pairs lie within a vector).
int vector_width(int R, int half) {
  const int m = half ? R / 2 : R;
  return m % 8 == 0 ? 8 : m % 4 == 0 ? 4 : m % 2 == 0 ? 2 : 1;
}

// threads per block: whole heads of items, about `want` threads at most
static unsigned block_threads(int heads, int ni, int want) {
  int per = want / ni;
  if (per < 1) per = 1;
  if (per > heads) per = heads;
  // the same number of rounds with no more heads at a time than they need
  const int rounds = (heads + per - 1) / per;
  per = (heads + rounds - 1) / rounds;
  return (unsigned)(per * ni);
}

template <typename T, int W, bool kHalf>
static cudaError_t qkv_t(const QkvArgs& a, bool back) {
  const unsigned threads = block_threads(a.H + 2 * a.G, items_per_head(a.D, W), 256);
  const dim3 grid((unsigned)((long long)a.B * a.T));
  return back ? launch_pdl(qkv_kernel<T, W, kHalf, true>, grid, dim3(threads), 0, a.stream, a)
              : launch_pdl(qkv_kernel<T, W, kHalf, false>, grid, dim3(threads), 0, a.stream, a);
}

template <typename T, int W, bool kHalf>
static cudaError_t append_t(const AppendArgs& a) {
  const unsigned threads = block_threads(a.H + 2 * a.G, items_per_head(a.D, W), 256);
  return launch_pdl(append_kernel<T, W, kHalf>, dim3((unsigned)a.tokens), dim3(threads), 0, a.stream, a);
}

// dispatch on type, layout and vector width; FN<T, W, kHalf>
#define CA_ROTARY_W(FN, T, HALF, ...)                     \
  switch (vector_width(a.R, a.half)) {                    \
    case 8: return FN<T, 8, HALF>(__VA_ARGS__);           \
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
