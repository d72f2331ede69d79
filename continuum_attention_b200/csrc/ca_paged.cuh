// ca_paged.cuh -- how the kernels over a paged cache divide their work: units (row tile,
// key head, sequence), their tiles of keys, and equal ranges of all tiles for the workers.
//
// Entering and leaving a unit costs as much as some tiles (row set-up, query loads, the
// output), so a unit takes `unit_cost` places in the stream before its first tile: a tile is
// done by the worker in whose range its place lies.  Without them a batch with many short
// sequences left 40% of the SMs' time unused behind the workers that had got those.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ca_common.cuh"
#include "ca_internal.h"

namespace ca {
namespace paged {

// set to CA_ERR_INVALID_ARGUMENT by a length, row range or page that is out of range (one word per
// source file that includes this; ca_paged.cu reads them all)
static __device__ int g_status = 0;
__device__ __forceinline__ void record_invalid() { atomicCAS(&g_status, 0, 1); }

struct Plan {
  int group;              // query heads per key head
  int page_shift;         // log2(page_size), or -1
  int page_size;
  int capacity;           // keys that a page-table row covers
  int row_lo, row_hi;     // rows (tokens * group) of the sequences that this launch takes
  unsigned min_places;     // places of a worker's range, at least
  int unit_cost;          // places that a unit takes before its first tile
  int unit_rows;          // rows that one copy brings
  unsigned long long wait_ns;   // after which a wait gives up

  __device__ __forceinline__ int page_of(int key) const { return page_shift >= 0 ? key >> page_shift : key / page_size; }
  __device__ __forceinline__ unsigned places_per_worker(unsigned total, int workers) const {
    return max((total + workers - 1) / (unsigned)workers, min_places);
  }
};

inline Plan make_plan(const Args& a) {
  Plan p;
  p.group = a.H / a.G;
  p.page_size = a.page_size;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (a.page_size == 1 << s) p.page_shift = s;
  p.capacity = a.pages_per_seq * a.page_size;
  p.row_lo = 0;
  p.row_hi = 0x7fffffff;
  p.min_places = 1;
  p.unit_cost = 0;
  p.unit_rows = 1;
  p.wait_ns = a.wait_ns;
  return p;
}

// bf16 and f16 (ca_paged_mma.cu), f32 (ca_paged_simt.cu)
size_t mma_workspace_bytes(long long max_q_len, long long H, long long G, long long D);
int mma_launches(const Args& a);
cudaError_t mma_forward(const Args& a, int dtype, void* workspace);
cudaError_t mma_read_status(int* out, bool reset);
size_t simt_workspace_bytes(long long max_q_len, long long H, long long G, long long D);
int simt_launches(const Args& a);
cudaError_t simt_forward(const Args& a, void* workspace);
cudaError_t simt_read_status(int* out, bool reset);

// long chunks in bf16 and f16 on tcgen05 (ca_paged_tc.cu): units of tc_br() rows, tc_groups() workers per SM
struct Pieces;
int tc_br();
int tc_groups(int dp);
// false where the caches' strides do not suit it: nothing was launched
bool tc_launch(const Args& a, const Plan& plan, int dtype, const Pieces& pc, cudaError_t& e);
cudaError_t tc_read_status(int* out, bool reset);

// What merge_kernel does for a worker: nothing (pieces 0), join the pieces of a unit that starts in the worker's range
// and goes on behind it, or (-1) give NaN to the rows of a launch that was refused, those of the sequences
// with `start` to `rows` rows.
struct Meta {
  int pieces, slot, start, rows, h, rt;
};

// Prefix sums of the sequences' places in shared memory (all threads of the block take part in the
// constructor), and cursors into the stream of tiles: sequence, key head, row tile, key tile.
template <int BR, int TK>
struct Schedule {
  const Args& a;
  const Plan& plan;
  unsigned* prefix;    // [seqs + 1]
  unsigned total;

  struct Cursor {
    int s, h, rt, kt, nt;
    unsigned at;       // the tile's place in the stream
    int start, n, len, bad;
    int tiles_rt;      // row tiles
  };

  // tiles of a unit whose last row stands at position i
  static __device__ __forceinline__ int tiles_to(int i) { return i < 0 ? 1 : i / TK + 1; }

  __device__ __forceinline__ int unit_tiles(int rt, int rows, int lead) const {
    return tiles_to(lead + (min(rows, (rt + 1) * BR) - 1) / plan.group);
  }

  // n = 0 for a sequence that this launch does not take
  __device__ __forceinline__ void load(int s, int& start, int& n, int& len, int& bad) const {
    start = a.q_starts[s];
    const int end = a.q_starts[s + 1];
    len = a.kv_lens[s];
    n = 0;
    bad = 0;
    if (start < 0 || end > a.rows || start > end) {
      record_invalid();
      return;
    }
    const int rows = (end - start) * plan.group;
    if (rows < plan.row_lo || rows > plan.row_hi) return;
    n = end - start;
    if (n > 0 && (len < 0 || len > plan.capacity)) {
      record_invalid();
      bad = 1;
      len = 0;
    }
  }

  __device__ Schedule(const Args& a_, const Plan& plan_, unsigned* prefix_) : a(a_), plan(plan_), prefix(prefix_) {
    const int lane = threadIdx.x & 31;
    // whole warps walk the sequences, so that several row tiles are summed by all lanes
    for (int s0 = (threadIdx.x >> 5) * 32; s0 < a.seqs; s0 += blockDim.x) {
      const int s = s0 + lane;
      int start = 0, n = 0, len = 0, bad = 0;
      if (s < a.seqs) load(s, start, n, len, bad);
      const int rows = n * plan.group;
      const int nrt = (rows + BR - 1) / BR;
      unsigned long long tiles = nrt == 1 ? unit_tiles(0, rows, len - n) + plan.unit_cost : 0;
      unsigned many = __ballot_sync(0xffffffffu, nrt > 1);
      while (many) {
        const int b = __ffs(many) - 1;
        many &= many - 1;
        const int rows_b = __shfl_sync(0xffffffffu, rows, b), lead_b = __shfl_sync(0xffffffffu, len - n, b);
        const int nrt_b = __shfl_sync(0xffffffffu, nrt, b);
        unsigned long long sum = 0;
        for (int rt = lane; rt < nrt_b; rt += 32) sum += unit_tiles(rt, rows_b, lead_b) + plan.unit_cost;
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane == b) tiles = sum;
      }
      tiles *= (unsigned)a.G;
      if (s < a.seqs) prefix[s + 1] = (unsigned)min(tiles, 0x7fffffffull);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      unsigned long long carry = 0;
      for (int s0 = 0; s0 < a.seqs; s0 += 32) {
        const int s = s0 + lane;
        unsigned long long v = s < a.seqs ? prefix[s + 1] : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const unsigned long long u = __shfl_up_sync(0xffffffffu, v, off);
          if (lane >= off) v += u;
        }
        v += carry;
        if (s < a.seqs) prefix[s + 1] = (unsigned)min(v, 0x7fffffffull);
        carry = __shfl_sync(0xffffffffu, v, 31);
      }
      if (lane == 0) {
        const bool refused = carry >= 0x7fffffffull;   // more tiles than the stream's index holds: none is done
        prefix[0] = refused;
        if (refused) {
          record_invalid();
          prefix[a.seqs] = 0;
        }
      }
    }
    __syncthreads();
    total = prefix[a.seqs];
  }

  // a worker's record before it has any tile: the join reads it of every worker, also of one whose wait gave up
  __device__ __forceinline__ Meta none() const { return Meta{-(int)prefix[0], 0, plan.row_lo, plan.row_hi, 0, 0}; }

  __device__ __forceinline__ void enter(Cursor& c) const {   // a new sequence
    load(c.s, c.start, c.n, c.len, c.bad);
    c.tiles_rt = (c.n * plan.group + BR - 1) / BR;
  }

  // the first tile at place x or behind it, in the unit that has x; whole warps call this
  __device__ Cursor locate(unsigned x) const {
    Cursor c;
    int lo = 0, hi = a.seqs;               // the sequence with prefix[s] <= x < prefix[s + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid;
    }
    c.s = lo;
    enter(c);
    const unsigned per_head = (prefix[lo + 1] - prefix[lo]) / (unsigned)a.G;
    unsigned y = x - prefix[lo];
    c.h = (int)(y / per_head);
    y -= (unsigned)c.h * per_head;
    c.rt = 0;
    const int rows = c.n * plan.group, lead = c.len - c.n;
    if (c.tiles_rt > 1) {
      const int lane = threadIdx.x & 31;
      for (int r0 = 0; r0 < c.tiles_rt; r0 += 32) {
        const int rt = r0 + lane;
        const unsigned own = rt < c.tiles_rt ? (unsigned)(unit_tiles(rt, rows, lead) + plan.unit_cost) : 0;
        unsigned v = own;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const unsigned u = __shfl_up_sync(0xffffffffu, v, off);
          if (lane >= off) v += u;
        }
        const unsigned in = __ballot_sync(0xffffffffu, v > y);
        if (in) {
          const int b = __ffs(in) - 1;
          c.rt = r0 + b;
          y -= __shfl_sync(0xffffffffu, v - own, b);
          break;
        }
        y -= __shfl_sync(0xffffffffu, v, 31);
      }
    }
    c.kt = max((int)y - plan.unit_cost, 0);
    c.at = x + max(plan.unit_cost - (int)y, 0);
    c.nt = unit_tiles(c.rt, rows, lead);
    return c;
  }

  __device__ __forceinline__ void advance(Cursor& c) const {
    ++c.at;
    if (++c.kt < c.nt) return;
    c.kt = 0;
    c.at += plan.unit_cost;
    if (++c.rt == c.tiles_rt) {
      c.rt = 0;
      if (++c.h == a.G) {
        c.h = 0;
        do ++c.s;
        while (c.s < a.seqs && prefix[c.s + 1] == prefix[c.s]);
        if (c.s == a.seqs) return;      // behind the last tile; `at` is behind every range
        enter(c);
      }
    }
    c.nt = unit_tiles(c.rt, c.n * plan.group, c.len - c.n);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// two neighbouring outputs
template <typename T>
__device__ __forceinline__ void store2(T* p, float x, float y) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(x, y);
  else *reinterpret_cast<uint32_t*>(p) = pack2<T>(x, y);
}

// A score that no exponential feels: what masked keys and the key before key 0 get.  Their segments'
// moments vanish without a select: the closed form divides by 1e30, and between two of them both
// exponentials are 0.  (Finite, since infinities would meet as NaN.)
constexpr float kMasked = -1e30f;

// Joins the pieces of a cut unit: piece 0 is in this worker's slot, the others are the first pieces of the
// workers that follow.  A block takes up to 4 W rows of a unit, a warp four of them; where rows are fewer than
// warps, several warps share a row's pieces, each sums its own in order, and then the warps' sums are added
// in order.

struct Sum {
  float m = -INFINITY, z = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
  // adds a piece with maximum m2, mass z2 and row y2.  A piece without a key that the row sees has m = -inf
  // and no mass, or the NaN of a bad page or length.
  __device__ __forceinline__ void add(float m2, float z2, float4 y2) {
    const bool none = m2 == -INFINITY;
    const float top = fmaxf(m, m2);
    const float fa = none ? 1.f : exp_rel(m - top), fb = none ? 0.f : exp_rel(m2 - top);
    z = none ? z + z2 : fmaf(z, fa, z2 * fb);
    y[0] = fmaf(y[0], fa, none ? 0.f : y2.x * fb);
    y[1] = fmaf(y[1], fa, none ? 0.f : y2.y * fb);
    y[2] = fmaf(y[2], fa, none ? 0.f : y2.z * fb);
    y[3] = fmaf(y[3], fa, none ? 0.f : y2.w * fb);
    m = top;
  }
};

// the pieces of one launch: units of br rows
struct Pieces {
  float* o;
  float2* mz;
  Meta* meta;
  int br, workers;
};

template <typename T, int DP, int W>
static __global__ void __launch_bounds__(W * 32) merge_kernel(const __grid_constant__ Args a, int group,
                                                                 const __grid_constant__ Pieces one,
                                                                 const __grid_constant__ Pieces two) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int RB = 4 * W;
  const int slices = (one.br + RB - 1) / RB;         // (the second launch's units have 16 rows at most)
  const bool second = (int)blockIdx.x >= one.workers * slices;
  const Pieces& pc = second ? two : one;
  const float* part_o = pc.o;
  const float2* part_mz = pc.mz;
  const int BR = pc.br;
  constexpr int VL = DP / 32;                        // values per lane: 2 or 4
  __shared__ float4 sum_y[W][32];
  __shared__ float2 sum_mz[W];
  const int w = second ? (int)blockIdx.x - one.workers * slices : (int)blockIdx.x / slices;
  const int row0 = second ? 0 : (int)blockIdx.x % slices * RB;   // of the unit
  const Meta mt = pc.meta[w];
  if (mt.pieces == 0) return;
  if (mt.pieces < 0) {
    // more tiles than the stream's index holds: no row of the launch is left as it was
    const int blocks = second ? two.workers : one.workers * slices;
    const int block = second ? w : (int)blockIdx.x;
    for (int s = 0; s < a.seqs; ++s) {
      const int start = a.q_starts[s], end = a.q_starts[s + 1];
      if (start < 0 || end > a.rows || start > end) continue;
      const int rows = (end - start) * group;
      if (rows < mt.start || rows > mt.rows) continue;
      const size_t last = (size_t)end * a.H * a.D;
      for (size_t x = (size_t)start * a.H * a.D + block * blockDim.x + threadIdx.x; x < last; x += blocks * blockDim.x)
        ((T*)a.o)[x] = from_f32<T>(__int_as_float(0x7fffffff));
    }
    return;
  }
  const int nrows = min(min(BR, mt.rows - mt.rt * BR) - row0, RB);
  if (nrows <= 0) return;
  int share = 1;                                     // warps per row
  while (share * 2 * nrows <= W && share * 4 <= mt.pieces) share *= 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % share;
  auto load = [&](int p, int r, float2& mz, float4& y) {
    const long long row = ((long long)(w + p) * 2 + (p == 0 ? mt.slot : 0)) * BR + row0 + r;
    mz = part_mz[row];
    if constexpr (VL == 4) {
      y = *reinterpret_cast<const float4*>(part_o + row * DP + 4 * lane);
    } else {
      const float2 t = *reinterpret_cast<const float2*>(part_o + row * DP + 2 * lane);
      y = make_float4(t.x, t.y, 0.f, 0.f);
    }
  };
  auto store = [&](const Sum& acc, int r) {
    const float inv = acc.z == 0.f ? 0.f : 1.f / acc.z;   // y is 0 then
    const int row = mt.rt * BR + row0 + r, t = row / group;
    T* dst = (T*)a.o + ((size_t)(mt.start + t) * a.H + (size_t)mt.h * group + (row - t * group)) * a.D + VL * lane;
    if (VL * lane < a.D) {
      store2<T>(dst, acc.y[0] * inv, acc.y[1] * inv);
      if constexpr (VL == 4) store2<T>(dst + 2, acc.y[2] * inv, acc.y[3] * inv);
    }
  };
  if (share == 1) {
    // four rows of a warp side by side: one after the other each would wait for its own loads
    Sum acc[4];
#pragma unroll 2
    for (int p = 0; p < mt.pieces; ++p) {
      float2 mz[4];
      float4 y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (warp + u * W < nrows) load(p, warp + u * W, mz[u], y[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (warp + u * W < nrows) acc[u].add(mz[u].x, mz[u].y, y[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (warp + u * W < nrows) store(acc[u], warp + u * W);
    return;
  }
  const int r = warp / share;                        // nrows * share <= W
  if (r >= nrows) return;
  Sum acc;
#pragma unroll 4
  for (int p = part; p < mt.pieces; p += share) {
    float2 mz;
    float4 y;
    load(p, r, mz, y);
    acc.add(mz.x, mz.y, y);
  }
  sum_y[warp][lane] = make_float4(acc.y[0], acc.y[1], acc.y[2], acc.y[3]);
  if (lane == 0) sum_mz[warp] = make_float2(acc.m, acc.z);
  asm volatile("bar.sync 1, %0;" ::"r"(nrows * share * 32) : "memory");
  if (part > 0) return;
  for (int q = 1; q < share; ++q) acc.add(sum_mz[warp + q].x, sum_mz[warp + q].y, sum_y[warp + q][lane]);
  store(acc, r);
}

// workspace of a launch of `per_sm` workers per SM whose units have br rows
inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

template <int DP>
inline size_t pieces_bytes(int br, int per_sm) {
  const size_t w = (size_t)num_sms_cached() * per_sm;
  return up256(w * 2 * br * DP * sizeof(float)) + up256(w * 2 * br * sizeof(float2)) + up256(w * sizeof(Meta));
}

template <int DP>
inline Pieces carve(char* ws, int br, int per_sm) {
  const size_t w = (size_t)num_sms_cached() * per_sm;
  const size_t o = up256(w * 2 * br * DP * sizeof(float)), mz = up256(w * 2 * br * sizeof(float2));
  return Pieces{(float*)ws, (float2*)(ws + o), (Meta*)(ws + o + mz), br, (int)w};
}

// few rows a unit: sixteen warps share their pieces; else blocks of four, 16 rows each
template <typename T, int DP>
inline cudaError_t launch_merge(const Args& a, const Plan& plan, const Pieces& one, const Pieces& two) {
  auto launch = [&](auto w) {
    constexpr int W = decltype(w)::value;
    const int slices = (one.br + 4 * W - 1) / (4 * W);
    return launch_pdl(merge_kernel<T, DP, W>, dim3((unsigned)(one.workers * slices + two.workers)), dim3(W * 32), 0,
                      a.stream, a, plan.group, one, two);
  };
  return one.br <= 16 ? launch(std::integral_constant<int, 16>{}) : launch(std::integral_constant<int, 4>{});
}

}  // namespace paged
}  // namespace ca
