// ca_paged_simt.cu -- Continuum Attention over a paged cache in f32, on the FMA pipes.
//
// Work is divided as in ca_paged_mma.cu (units, places, pieces, merge); a worker is a block.
// A tile of TK keys is three steps between barriers: scores S = Q K^T in register tiles, the
// rows' moments (a few threads per row, consecutive keys each), O += P V in register tiles.
// Tiles arrive by cp.async, one ahead, gathered row by row through the page table, V one
// row early so that the weights of keys a-1 .. a+TK-2 meet it where they lie.
//
// Exponentials and reciprocals are the special-function unit's (2^-22 of the value, and e^x another |x| 2^-24 of
// its argument's rounding), all sums are in 32 bits: outputs of short prompts are 2.7e-7 of their norm from 64 bits,
// where torch's exp and division in 32 bits leave 3.6e-7; of decoding 3.9e-8 against 3.7e-8.
//
// What bounds it: decoding reads 2 D f32 values a key and key head and comes to 70% of the copy
// rate, held by the latency of a tile's three steps at ten warps an SM; chunks are bound by the FMA pipe and the
// shared-memory reads that feed it (scores: 6 16-byte reads for 32 FMAs of a thread; P V: 8 for 64).  8 prompts of 40 .. 192 tokens
// (4 heads of 64) take 25 us, nearly all of it latency: launch, a unit's few tiles, the join.
#include "ca_paged.cuh"

namespace ca {
namespace paged {

namespace {

__device__ float4 g_nan16 = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};

__device__ __forceinline__ void cp_async16(float* dst, const float* src, bool zero) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(zero ? 0 : 16) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// DP padded head values; BR rows of a unit; threads in TR x TC: scores are RT rows x KT keys a thread (row
// tr + TR i, key tc + TC j), outputs RT rows x DP/TC neighbouring columns
template <int DP_, int BR_, int TR_, int TC_, int PER_SM_>
struct Config {
  static constexpr int DP = DP_, BR = BR_, TR = TR_, TC = TC_, PER_SM = PER_SM_, TK = 32;
  static constexpr int NT = TR * TC, RT = BR / TR, KT = TK / TC, CT = DP / TC;
  static constexpr int TPR = NT / BR, KPT = TK / TPR;   // the moments: threads per row, keys per thread
  static constexpr int LD = DP + 4, LS = TK + 4;        // rows of tiles and of scores, on 16 bytes
  static constexpr int TILE = (TK + 1) * LD;            // floats; row TK is the halo
  static constexpr int FLOATS = 4 * TILE + BR * LD + BR * LS + 2 * BR;
  static constexpr int SMEM = FLOATS * 4 + 3 * (TK + 1) * 8;   // and the prefix sums behind it
  static_assert(TPR >= 1 && 32 % TPR == 0 && CT % 2 == 0, "");
  static constexpr int VW = CT % 4 == 0 ? 4 : 2;        // output columns of one access
  static constexpr int SW = KPT < 4 ? KPT : 4;          // scores of one access
};

template <int N>
struct alignas(N * 4) Vec {
  float x[N];
  static __device__ __forceinline__ Vec load(const float* p) { return *reinterpret_cast<const Vec*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<Vec*>(p) = *this; }
};

struct Tile {      // what the block knows of a tile (the same in all threads)
  int kt, nt, start, n, len, h, rt, bad;
  bool first, last, end;
};

template <typename C>
__global__ void __launch_bounds__(C::NT, C::PER_SM)
    simt_kernel(const __grid_constant__ Args a, const __grid_constant__ Plan plan, float* __restrict__ part_o,
                float2* __restrict__ part_mz, Meta* __restrict__ meta) {
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  constexpr int TK = C::TK, DP = C::DP, BR = C::BR, LD = C::LD, LS = C::LS, RT = C::RT, KT = C::KT, CT = C::CT;
  float* kv = reinterpret_cast<float*>(smem);            // stages: K, V, K, V
  float* sq = kv + 4 * C::TILE;                          // Q [BR][LD]
  float* ss = sq + BR * LD;                              // S, then P [BR][LS]
  float* row_f = ss + BR * LS;                           // per row: factor on O, then weight of the last key
  float* row_z = row_f + BR;                             // its mass
  long long* offs = reinterpret_cast<long long*>(smem + C::FLOATS * 4);   // [3][TK + 1]: rows a-1 .. a+TK-1
  unsigned* prefix = reinterpret_cast<unsigned*>(smem + C::SMEM);
  const int tid = threadIdx.x, tr = tid / C::TC, tc = tid % C::TC;

  Schedule<BR, TK> sched(a, plan, prefix);
  const unsigned total = sched.total;
  const int worker = blockIdx.x;
  const unsigned per = plan.places_per_worker(total, gridDim.x);
  const unsigned x0 = (unsigned)min((unsigned long long)worker * per, (unsigned long long)total);
  const unsigned x1 = (unsigned)min((unsigned long long)x0 + per, (unsigned long long)total);
  typename Schedule<BR, TK>::Cursor cur;
  cur.at = x1;
  if (x0 < x1) cur = sched.locate(x0);
  if (cur.at >= x1) {
    if (tid == 0) meta[worker] = sched.none();
    return;
  }

  // the next tile of the stream, and its rows' offsets in the cache (-1: none, -2: a bad page)
  int ring = 0;
  bool more = true, opening = true;
  unsigned at = 0;
  auto describe = [&](Tile& t) {
    const int base = cur.kt * TK;
    for (int r = tid; r <= TK; r += C::NT) {
      const int key = base - 1 + r;
      long long off = -1;
      if (key >= 0 && key < cur.len) {
        const int col = plan.page_of(key);
        const int page = a.page_table[(size_t)cur.s * a.page_table_stride + col];
        if (page < 0 || page >= a.num_pages) {
          off = -2;
          record_invalid();
        } else {
          off = (long long)page * a.page_stride + (long long)cur.h * a.head_stride +
                (long long)(key - col * a.page_size) * a.slot_stride;
        }
      }
      offs[ring * (TK + 1) + r] = off;
    }
    at = cur.at;
    more = cur.at + 1 < x1;
    t.kt = cur.kt;
    t.nt = cur.nt;
    t.start = cur.start;
    t.n = cur.n;
    t.len = cur.len;
    t.h = cur.h;
    t.rt = cur.rt;
    t.bad = cur.bad;
    t.first = opening || cur.kt == 0;
    t.last = !more || cur.kt + 1 == cur.nt;
    opening = false;
    if (more) {
      sched.advance(cur);
      more = cur.at < x1;
    }
    t.end = !more;
  };
  auto copy = [&](const Tile& t, int stage, int slot) {
    const long long* of = offs + slot * (TK + 1);
    float* kd = kv + stage * 2 * C::TILE;
    float* vd = kd + C::TILE;
    constexpr int C4 = DP / 4;
    const float* kc = (const float*)a.k_cache;
    const float* vc = (const float*)a.v_cache;
    for (int x = tid; x < (TK + 1) * C4; x += C::NT) {
      const int r = x / C4, c = (x - r * C4) * 4;
      const bool pad = c >= a.D;
      // K row r is key a + r, the halo (row TK) key a - 1; V row r is key a - 1 + r
      const long long ok = of[r < TK ? r + 1 : 0], ov = of[r];
      const float* nan = reinterpret_cast<const float*>(&g_nan16);
      cp_async16(kd + r * LD + c, ok < -1 ? nan : kc + (ok < 0 ? 0 : ok + c), ok == -1 || pad);
      cp_async16(vd + r * LD + c, ov < -1 ? nan : vc + (ov < 0 ? 0 : ov + c), ov == -1 || pad);
    }
  };

  // a row's moments: threads [row][part] in one warp
  const int mrow = tid / C::TPR, mpart = tid % C::TPR;
  float m = -INFINITY, z = 0.f, carry_s = kMasked, carry_b = 0.f, scale = 0.f;
  int pos = -1, kt0 = 0;
  bool in_first = true, first_piece = true;
  float o[RT][CT];

  Tile cur_t, next_t;
  describe(cur_t);
  __syncthreads();
  copy(cur_t, 0, 0);
  cp_commit();
  int stage = 0, slot = 0;
  unsigned at_now = at;
  while (true) {
    const Tile t = cur_t;
    const unsigned at_t = at_now;
    ring = slot == 2 ? 0 : slot + 1;
    if (!t.end) {
      describe(next_t);
      at_now = at;
    }
    const int base = t.kt * TK, rows = t.n * plan.group, row0 = t.rt * BR;
    if (t.first) {
      kt0 = t.kt;
      in_first = first_piece;
      first_piece = false;
      for (int x = tid; x < BR * (DP / 4); x += C::NT) {
        const int r = x / (DP / 4), c = (x % (DP / 4)) * 4, row = row0 + r;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < rows && c < a.D) {
          const int tk = row / plan.group;
          v = *reinterpret_cast<const float4*>((const float*)a.q + (size_t)(t.start + tk) * a.q_token_stride +
                                               (size_t)(t.h * plan.group + row - tk * plan.group) * a.q_head_stride + c);
        }
        *reinterpret_cast<float4*>(sq + r * LD + c) = v;
      }
      const int row = row0 + mrow;
      pos = -1;
      scale = 0.f;
      if (row < rows) {
        const int tk = row / plan.group;
        pos = t.len - t.n + tk;
        scale = expf(a.log_gain[t.h * plan.group + row - tk * plan.group]) * a.inv_sqrt_d;
      }
      m = -INFINITY;
      z = 0.f;
      carry_s = kMasked;
      carry_b = 0.f;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c) o[i][c] = 0.f;
    }
    cp_wait<0>();
    __syncthreads();                 // this tile, Q and the next tile's offsets are there
    if (!t.end) copy(next_t, stage ^ 1, ring);
    cp_commit();
    const float* ks = kv + stage * 2 * C::TILE;
    const float* vs = ks + C::TILE;

    {
      // scores: even and odd positions of the head in the two halves of packed FMAs
      float2 acc[RT][KT];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < KT; ++j) acc[i][j] = splat2(0.f);
#pragma unroll 4
      for (int d = 0; d < DP; d += 4) {
        float4 q[RT], k[KT];
#pragma unroll
        for (int i = 0; i < RT; ++i) q[i] = *reinterpret_cast<const float4*>(sq + (tr + C::TR * i) * LD + d);
#pragma unroll
        for (int j = 0; j < KT; ++j) k[j] = *reinterpret_cast<const float4*>(ks + (tc + C::TC * j) * LD + d);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            acc[i][j] = fma2(make_float2(q[i].x, q[i].y), make_float2(k[j].x, k[j].y), acc[i][j]);
            acc[i][j] = fma2(make_float2(q[i].z, q[i].w), make_float2(k[j].z, k[j].w), acc[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < KT; ++j) ss[(tr + C::TR * i) * LS + tc + C::TC * j] = acc[i][j].x + acc[i][j].y;
    }
    if (t.first && t.kt > 0) {
      // the score that the first segment starts from, by the row's threads
      float s = 0.f;
      for (int d = 4 * mpart; d < DP; d += 4 * C::TPR) {
        const float4 q = *reinterpret_cast<const float4*>(sq + mrow * LD + d);
        const float4 k = *reinterpret_cast<const float4*>(ks + TK * LD + d);
        s = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s))));
      }
#pragma unroll
      for (int off = C::TPR / 2; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (base - 1 <= pos) m = carry_s = s * scale;
    }
    __syncthreads();

    {
      // the row's weights
      float* sr = ss + mrow * LS + mpart * C::KPT;
      const int kc = base + mpart * C::KPT;
      float s[C::KPT];
      float top = kMasked;
#pragma unroll
      for (int x = 0; x < C::KPT; x += C::SW) {
        const Vec<C::SW> v = Vec<C::SW>::load(sr + x);
#pragma unroll
        for (int e = 0; e < C::SW; ++e) s[x + e] = v.x[e];
      }
#pragma unroll
      for (int x = 0; x < C::KPT; ++x) {
        s[x] = kc + x <= pos ? s[x] * scale : kMasked;
        top = fmaxf(top, s[x]);
      }
#pragma unroll
      for (int off = C::TPR / 2; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      float f = 1.f;
      if (top > kMasked && top > m) {
        f = exp_rel(m - top);
        m = top;
        z *= f;
        carry_b *= f;
      }
      const float mm = m == -INFINITY ? 0.f : m;
      float got = __shfl_up_sync(0xffffffffu, s[C::KPT - 1], 1, C::TPR);
      float sa = mpart == 0 ? carry_s : got;
      float ea = exp_rel(sa - mm), right = 0.f, p[C::KPT], eb[C::KPT], M0[C::KPT], M1[C::KPT];
      const int lowest = t.first ? base : base - 1;      // key `pos` has its cap here from this key on
      // both forms of each moment, selected: a branch would run both for a warp anyway, key after key
#pragma unroll
      for (int x = 0; x < C::KPT; ++x) eb[x] = exp_rel(s[x] - mm);
#pragma unroll
      for (int x = 0; x < C::KPT; ++x) {
        const float a0 = x ? eb[x - 1] : ea, d = s[x] - (x ? s[x - 1] : sa);
        const float r = rcp_approx(d);
        const float m0 = (eb[x] - a0) * r, near = a0 * series_j1(d);
        const bool use = fabsf(d) < kSeriesMax;
        M1[x] = use ? near : (eb[x] - m0) * r;
        M0[x] = use ? fmaf(-d, near, eb[x]) : m0;
      }
#pragma unroll
      for (int x = 0; x < C::KPT; ++x) {
        z += M0[x];
        p[x] = right + (M0[x] - M1[x]);
        const int key = kc + x - 1;                      // the key this weight belongs to
        const float half = (key == 0 && pos >= 0 ? 0.5f : 0.f) + (key == pos && key >= lowest ? 0.5f : 0.f);
        if (half > 0.f) {
          p[x] = fmaf(half, x ? eb[x - 1] : ea, p[x]);
          z = fmaf(half, x ? eb[x - 1] : ea, z);
        }
        right = M1[x];
      }
      sa = s[C::KPT - 1];
      got = __shfl_up_sync(0xffffffffu, right, 1, C::TPR);
      p[0] += mpart == 0 ? carry_b : got;
      carry_s = __shfl_sync(0xffffffffu, sa, C::TPR - 1, C::TPR);
      carry_b = __shfl_sync(0xffffffffu, right, C::TPR - 1, C::TPR);
#pragma unroll
      for (int x = 0; x < C::KPT; x += C::SW) {
        Vec<C::SW> v;
#pragma unroll
        for (int e = 0; e < C::SW; ++e) v.x[e] = p[x + e];
        v.store(sr + x);
      }
      if (mpart == 0) row_f[mrow] = f;
    }
    __syncthreads();

#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const float f = row_f[tr + C::TR * i];
#pragma unroll
      for (int c = 0; c < CT; ++c) o[i][c] *= f;
    }
#pragma unroll 2
    for (int k = 0; k < TK; k += 4) {
      float4 p[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) p[i] = *reinterpret_cast<const float4*>(ss + (tr + C::TR * i) * LS + k);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int c = 0; c < CT; c += C::VW) {
          const Vec<C::VW> v = Vec<C::VW>::load(vs + (k + u) * LD + tc * CT + c);
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
#pragma unroll
            for (int e = 0; e < C::VW; e += 2) {
              const float2 y = fma2(splat2(w), make_float2(v.x[e], v.x[e + 1]), make_float2(o[i][c + e], o[i][c + e + 1]));
              o[i][c + e] = y.x;
              o[i][c + e + 1] = y.y;
            }
          }
        }
      }
    }

    if (t.last) {
      const bool whole = kt0 == 0 && t.kt + 1 == t.nt;
      const int key = base + TK - 1;                     // the key whose weight is still carried
      const long long slot_row = ((long long)worker * 2 + (in_first ? 0 : 1)) * BR;
      const float mm = m == -INFINITY ? 0.f : m;
      const float cap = key == pos ? 0.5f * exp_rel(carry_s - mm) : 0.f;
      float zz = z;
#pragma unroll
      for (int off = C::TPR / 2; off; off >>= 1) zz += __shfl_xor_sync(0xffffffffu, zz, off);
      zz += cap;
      if (t.bad) zz = __int_as_float(0x7fffffff);
      __syncthreads();                                   // row_f has been read
      if (mpart == 0) {
        // a key beyond the row's own has no weight, and its V may hold anything
        row_f[mrow] = key <= pos ? carry_b + cap : 0.f;
        row_z[mrow] = zz;
        if (!whole && row0 + mrow < rows) part_mz[slot_row + mrow] = make_float2(m, zz);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = tr + C::TR * i, row = row0 + r;
        if (row >= rows) continue;
        const float w = row_f[r], zr = row_z[r], inv = 1.f / zr;
        const int tk = row / plan.group;
        float* dst = (float*)a.o +
                     ((size_t)(t.start + tk) * a.H + (size_t)t.h * plan.group + (row - tk * plan.group)) * a.D;
#pragma unroll
        for (int c = 0; c < CT; c += C::VW) {
          const int col = tc * CT + c;
          Vec<C::VW> y = Vec<C::VW>::load(vs + TK * LD + col);
#pragma unroll
          for (int e = 0; e < C::VW; ++e) y.x[e] = w != 0.f ? fmaf(w, y.x[e], o[i][c + e]) : o[i][c + e];
          if (!whole) {
            y.store(part_o + (slot_row + r) * DP + col);
          } else if (col < a.D) {
            // z = 0: the row sees no key
#pragma unroll
            for (int e = 0; e < C::VW; ++e) y.x[e] = zr == 0.f ? 0.f : y.x[e] * inv;
            y.store(dst + col);
          }
        }
      }
      if (t.end && tid == 0) {
        // this worker joins the unit that starts in its range and goes on behind it
        Meta mt;
        mt.pieces = kt0 == 0 && t.kt + 1 < t.nt ? 1 + (int)((at_t + (t.nt - 1 - t.kt)) / per) - worker : 0;
        mt.slot = in_first ? 0 : 1;
        mt.start = t.start;
        mt.rows = rows;
        mt.h = t.h;
        mt.rt = t.rt;
        meta[worker] = mt;
      }
    }
    if (t.end) break;
    __syncthreads();                 // scores, Q and this tile's stage are free
    cur_t = next_t;
    stage ^= 1;
    slot = ring;
  }
  cp_wait<0>();
}

// Rows of a unit: 4 or 16 for decoding, 64 for chunks.  In the decoding forms a warp's lanes are the tile's 32
// keys, then its output columns.  64 sequences of one row over 8192 keys (16 heads of 64): units of 4 rows 958 us
// (4.5 TB/s; on one warp 1220, on four 1050), of 16 rows 3230; 16 rows over 4096 keys (16 sequences, 32 heads on
// 2 of 64): 46 us, with threads in 16 x 8 75.  Prompts of 2 x 1024 tokens, 16 heads of 128: 371 us in 8 x 32, 395 in
// 16 x 16, which is better with 64 values (2 x 2048 tokens 639 and 708).
template <int DP> using One = Config<DP, 4, 2, 32, DP == 64 ? 5 : 3>;
template <int DP> using Few = Config<DP, 16, 4, 32, DP == 64 ? 4 : 2>;
template <int DP> using Many = Config<DP, 64, DP == 64 ? 16 : 8, DP == 64 ? 16 : 32, DP == 64 ? 2 : 1>;
constexpr int kUnitCost = 1;

template <int DP, typename F>
auto with_form(long long rows, F f) {
  return rows <= 4 ? f(One<DP>{}) : rows <= 16 ? f(Few<DP>{}) : f(Many<DP>{});
}

template <typename C>
cudaError_t launch_main(const Args& a, const Plan& plan, const Pieces& pc) {
  // (with the prefix sums of 200 sequences; with more, fewer blocks run at once)
  static_assert((C::SMEM + 200 * 4 + 1024) * C::PER_SM <= 233472, "shared memory of an SM");
  const size_t smem = C::SMEM + (size_t)(a.seqs + 1) * sizeof(unsigned);
  cudaError_t e = cudaFuncSetAttribute(simt_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       C::SMEM + (kMaxSeqs + 1) * (int)sizeof(unsigned));
  if (e != cudaSuccess) return e;
  return launch_pdl(simt_kernel<C>, dim3((unsigned)pc.workers), dim3(C::NT), smem, a.stream, a, plan, pc.o, pc.mz,
                    pc.meta);
}

// Whether a batch with chunks gives its short sequences (at most One's rows) a launch of their own: where they have to
// be the most, since there are fewer than 32 rows a sequence.  63 sequences of one row and one of 200 over 8192 keys,
// 16 heads of 64: 1253 us, in one launch 4981; 8 prompts of 40 .. 192 rows would pay 2 of their 25 us for it.
bool splits(const Args& a) {
  const long long group = a.H / a.G;
  return a.max_q_len * group > 16 && a.seqs > 1 && a.rows * group < 32LL * a.seqs;
}

template <int DP>
cudaError_t forward_dp(const Args& a, void* workspace) {
  Plan plan = make_plan(a);
  plan.unit_cost = kUnitCost;
  char* ws = (char*)workspace;
  const long long rows = (long long)a.max_q_len * plan.group;
  auto run = [&](auto form) {
    using C = decltype(form);
    Pieces pc = carve<DP>(ws, C::BR, C::PER_SM), few{};
    Plan tall = plan;
    if (splits(a)) tall.row_lo = One<DP>::BR + 1;
    cudaError_t e = launch_main<C>(a, tall, pc);
    if (e == cudaSuccess && splits(a)) {
      few = carve<DP>(ws + pieces_bytes<DP>(C::BR, C::PER_SM), One<DP>::BR, One<DP>::PER_SM);
      plan.row_hi = One<DP>::BR;
      e = launch_main<One<DP>>(a, plan, few);
    }
    return e != cudaSuccess ? e : launch_merge<float, DP>(a, plan, pc, few);
  };
  return with_form<DP>(rows, run);
}

}  // namespace

size_t simt_workspace_bytes(long long max_q_len, long long H, long long G, long long D) {
  auto bytes = [](auto form) {
    using C = decltype(form);
    // (a batch with chunks may take two launches)
    return pieces_bytes<C::DP>(C::BR, C::PER_SM) +
           (C::BR > 16 ? pieces_bytes<C::DP>(One<C::DP>::BR, One<C::DP>::PER_SM) : 0);
  };
  return D <= 64 ? with_form<64>(max_q_len * (H / G), bytes) : with_form<128>(max_q_len * (H / G), bytes);
}

int simt_launches(const Args& a) { return splits(a) ? 3 : 2; }

cudaError_t simt_forward(const Args& a, void* workspace) {
  return a.D <= 64 ? forward_dp<64>(a, workspace) : forward_dp<128>(a, workspace);
}

cudaError_t simt_read_status(int* out, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
  if (e != cudaSuccess || !reset || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
}

}  // namespace paged
}  // namespace ca
