// ca_paged_mma.cu -- Continuum Attention over a paged cache, bf16 and f16.
//
// Work.  A unit is a tile of BR query rows (row = token * group + head in group) of one
// sequence and key head; it has ceil((last row's position + 1) / TK) tiles of TK keys, one
// at least.  All units' tiles are laid end to end and cut into equal ranges, one per
// worker, so that a batch of any lengths, one long sequence or many short ones, keeps every
// SM busy to the end.  A worker walks its range as one stream of tiles: the copies of the
// next tiles are in flight across unit borders.  A unit that lies in one range is written
// directly; the pieces of a cut one (row maximum, mass, accumulator, all fp32) go to the
// workspace and merge_kernel joins them in order, so results do not depend on timing.
//
// A worker of the decoding form is one warp with up to 16 rows: four run on an SM, each
// with a ring of its own, and no barrier couples them.  The form for chunks is a block of
// four warps with 16 rows each that share the ring.
//
// Cutting keys.  Segments, not keys, are divided: the segment from key j-1 to key j belongs
// to the tile of j.  A tile with keys a .. a+TK-1 therefore weighs keys a-1 .. a+TK-2, V is
// staged one row early, and only the mass that ends at key a+TK-1 is carried on.  The first
// tile of a piece also stages K row a-1 (its score starts the first segment), the last one
// V row a+TK-1 (for the carried mass, and the row's own cap).
//
// Registers.  The products run on mma.sync m16n8k16 with scores in registers: the bound of
// this operator is the scalar work per score (one exp2, one reciprocal, about 17 other
// instructions), not the tensor pipe, and register scores spare the trip through tensor
// memory.  B fragments may come from any rows, so keys are dealt to lanes in runs: column
// 2c + e of score tile j is key (TK/4) c + j + (TK/8) e.  A lane's pair (j, j + TK/8) then
// has the pair (j-1, j-1 + TK/8) as its left neighbours, every step of the moments is one
// packed f32x2 instruction for two keys, and neighbours in other lanes are needed once per
// run.  The weights leave as A fragments with the same dealing of V rows.  Each weight is
// split into two 16-bit parts (hi + lo, 16 bits or more): one rounding to bf16 would put
// 1.1e-3 of the output's size on every row.  With 8 rows or fewer hi and lo are the two
// halves of one fragment and cost one product.
#include <algorithm>

#include "ca_common.cuh"
#include "ca_paged.cuh"

namespace ca {
namespace paged {

namespace {

constexpr float kRescaleNats = 8.f;   // the reference maximum moves when it grows by more

__device__ uint4 g_nan16 = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};   // NaN in bf16, f16 and f32

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool fill) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 0 : 16));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// a weight pair as two 16-bit parts: hi + lo keeps 16 bits (bf16) or 21 (f16)
template <typename T>
__device__ __forceinline__ void split2(float2 w, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float2 w, uint32_t& hi, uint32_t& lo) {
  const uint32_t u0 = __float_as_uint(w.x), u1 = __float_as_uint(w.y);
  hi = __byte_perm(u0, u1, 0x7632);   // bf16 by truncation; the remainder is exact
  const float2 r = sub2(w, make_float2(__uint_as_float(u0 & 0xffff0000u), __uint_as_float(u1 & 0xffff0000u)));
  const __nv_bfloat162 l = __floats2bfloat162_rn(r.x, r.y);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
template <>
__device__ __forceinline__ void split2<__half>(float2 w, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(w.x, w.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(w.x - f.x, w.y - f.y);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
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

// Weights of one lane's run of one row.  raw[j] = unscaled scores of keys (kc + j, kc + NJ + j), sL the
// scaled score of key kc - 1, m2 the reference maximum in log2 units.  On return W[j] weighs keys
// (kc - 1 + j, kc + NJ - 1 + j), but for the mass that ends at key kc - 1, which the lane to the
// left adds to W[0].x; last is the mass that ends at the run's last key.
// kEdge: keys beyond position i are masked by selects (their exponentials may overflow), segment
// k counts for 1 <= k <= i, keys 0 and i have half caps; key i's belongs to this piece when i >= lowest
// (the piece before it has weighed its own last key to the end).
template <bool kEdge, int NJ>
__device__ __forceinline__ void weigh(const float2 (&raw)[NJ], float scale, float m2, int kc, int i, int lowest,
                                      float sL, float2 (&W)[NJ], float& last, float2& z2) {
  const float2 l2e = splat2(kLog2e), nm2 = splat2(-m2), sc = splat2(scale);
  float2 sv[NJ], ev[NJ], M1[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    sv[j] = mul2(raw[j], sc);
    const float2 arg = fma2(sv[j], l2e, nm2);
    ev[j] = make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
  }
  const float eL0 = ex2_approx(fmaf(sL, kLog2e, -m2));
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const float2 sl = j ? sv[j - 1] : make_float2(sL, sv[NJ - 1].x);
    const float2 eL = j ? ev[j - 1] : make_float2(eL0, ev[NJ - 1].x);
    const float2 nd = sub2(sl, sv[j]);                                          // -d
    const float2 rn = make_float2(rcp_approx(nd.x), rcp_approx(nd.y));         // -1/d
    float2 ps = fma2(splat2(-1.f / 30.f), nd, splat2(1.f / 8.f));              // J1's series in -nd
    ps = fma2(ps, nd, splat2(-1.f / 3.f));
    ps = mul2(fma2(ps, nd, splat2(1.f / 2.f)), eL);
    const float2 m0c = mul2(sub2(eL, ev[j]), rn);
    const float2 m1c = mul2(sub2(m0c, ev[j]), rn);
    float2 m1 = make_float2(fabsf(nd.x) < kSeriesMaxFwd ? ps.x : m1c.x, fabsf(nd.y) < kSeriesMaxFwd ? ps.y : m1c.y);
    float2 m0 = fma2(nd, m1, ev[j]);
    if (kEdge) {
      const int kx = kc + j, ky = kc + NJ + j;
      const bool okx = kx >= 1 && kx <= i, oky = ky <= i;
      m0 = make_float2(okx ? m0.x : 0.f, oky ? m0.y : 0.f);
      m1 = make_float2(okx ? m1.x : 0.f, oky ? m1.y : 0.f);
    }
    M1[j] = m1;
    W[j] = sub2(m0, m1);
    z2 = add2(z2, m0);
    if (kEdge) {
      const int kx = kc + j - 1, ky = kc + NJ + j - 1;   // the keys these weights belong to
      const float nx = (kx == 0 && i >= 0 ? 0.5f : 0.f) + (kx == i && i >= lowest ? 0.5f : 0.f);
      const float2 cap = make_float2(nx > 0.f ? nx * eL.x : 0.f, ky == i ? 0.5f * eL.y : 0.f);
      W[j] = add2(W[j], cap);
      z2 = add2(z2, cap);
    }
  }
#pragma unroll
  for (int j = NJ - 1; j >= 1; --j) W[j] = add2(W[j], M1[j - 1]);
  W[0].y += M1[NJ - 1].x;
  last = M1[NJ - 1].y;
}

// ------------------------------------------------------------------ the kernel

// RPW rows per warp (8 or 16), RW warps that share a ring (1 or 4), GROUPS rings per block,
// NST stages of TK keys of DP (padded) values
template <typename T, int DP_, int RPW_, int RW_, int GROUPS_, int NST_>
struct Config {
  static constexpr int DP = DP_, TK = DP_ == 64 ? 64 : 32, RPW = RPW_, RW = RW_, GROUPS = GROUPS_, NST = NST_;
  static constexpr int NT = RW * 32;                    // threads of a group
  static constexpr int BR = RPW * RW;                   // rows of a unit
  static constexpr int NJ = TK / 8;                     // score tiles of 8 keys; half a lane's run
  static constexpr int CH = DP / 8;                     // 16-byte chunks of a row
  static constexpr int ROWB = DP * 2;
  static constexpr bool kStageQ = RW == 1 && RPW == 8 && DP == 64;   // as far as shared memory goes
  static constexpr int KV_BYTES = (TK + 1) * ROWB;      // row TK: the halo
  static constexpr int Q_BYTES = kStageQ ? RPW * ROWB : 0;
  static constexpr int STAGE = 2 * KV_BYTES + Q_BYTES;
  static constexpr int RING = NST + 1;                  // descriptors and row offsets live one tile longer
  static constexpr int OFFS = TK + 1;
  static constexpr int GROUP_BYTES = NST * STAGE + RING * (OFFS * 8 + 40);
  static constexpr int GROUP_STRIDE = (GROUP_BYTES + 255) / 256 * 256;
  static constexpr int SMEM = GROUPS * GROUP_STRIDE;    // and the prefix sums behind it
};

struct Desc {   // one tile of the stream
  int kt, nt;         // tile in its unit, tiles of the unit
  int first, last;    // of the piece
  int start, n, len;  // the sequence
  int h, rt;          // key head, row tile
  int bad;            // the sequence's length is out of range
};
static_assert(sizeof(Desc) == 40, "");

template <int RW>
__device__ __forceinline__ void group_sync() {
  if constexpr (RW == 1) __syncwarp();
  else __syncthreads();
}

template <typename T, typename C>
__global__ void __launch_bounds__(C::NT* C::GROUPS, C::RW == 1 ? 1 : 3)
    mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Plan plan, float* __restrict__ part_o, float2* __restrict__ part_mz, Meta* __restrict__ meta) {
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  constexpr int TK = C::TK, NJ = C::NJ, DP = C::DP, ROWB = C::ROWB, CH = C::CH, NST = C::NST;
  constexpr int NKK = DP / 16;                 // k-steps of Q K^T
  constexpr int NN = DP / 8;                   // column tiles of the output
  const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
  const int group = threadIdx.x / C::NT, gt = threadIdx.x % C::NT, warp = gt >> 5;
  unsigned* prefix = reinterpret_cast<unsigned*>(smem + C::SMEM);

  Schedule<C::BR, TK> sched(a, plan, prefix);
  const unsigned total = sched.total;
  const int worker = blockIdx.x * C::GROUPS + group, workers = gridDim.x * C::GROUPS;
  const unsigned per = plan.tiles_per_worker(total, workers);
  const unsigned long long x0l = (unsigned long long)worker * per;
  if (x0l >= total) {
    if (gt == 0) meta[worker].pieces = 0;
    return;
  }
  const unsigned x0 = (unsigned)x0l, x1 = min(total, x0 + per);

  uint8_t* gsm = smem + (size_t)group * C::GROUP_STRIDE;
  long long* offs_ring = reinterpret_cast<long long*>(gsm + NST * C::STAGE);
  Desc* desc_ring = reinterpret_cast<Desc*>(offs_ring + C::RING * C::OFFS);

  // ---- the loader's side: where the stream's next tile lies
  typename Schedule<C::BR, TK>::Cursor cur = sched.locate(x0);
  unsigned xa = x0;          // the tile `cur` stands at: the next to be described
  int slot_a = 0;            // xa % RING
  unsigned xb = x0;          // the next tile to be copied
  int slot_b = 0, stage_b = 0;

  // describe tile xa: its rows' offsets in the cache (keys a-1 .. a+TK-1; -1: none, -2: bad page)
  auto describe = [&]() {
    if (xa < x1) {
      const int base = cur.kt * TK;
      for (int r = gt; r < C::OFFS; r += C::NT) {
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
        offs_ring[slot_a * C::OFFS + r] = off;
      }
      if (gt == 0) {
        Desc d;
        d.kt = cur.kt;
        d.nt = cur.nt;
        d.first = xa == x0 || cur.kt == 0;
        d.last = xa + 1 == x1 || cur.kt + 1 == cur.nt;
        d.start = cur.start;
        d.n = cur.n;
        d.len = cur.len;
        d.h = cur.h;
        d.rt = cur.rt;
        d.bad = cur.bad;
        desc_ring[slot_a] = d;
      }
      if (xa + 1 < x1) sched.advance(cur);
    }
    ++xa;
    if (++slot_a == C::RING) slot_a = 0;
  };

  // copy tile xb into its stage
  auto copy = [&]() {
    if (xb < x1) {
      const long long* offs = offs_ring + slot_b * C::OFFS;
      const Desc& d = desc_ring[slot_b];
      const uint32_t ks = smem_addr(gsm + stage_b * C::STAGE), vs = ks + C::KV_BYTES;
      const T* kc = (const T*)a.k_cache + (gt % CH) * 8;
      const T* vc = (const T*)a.v_cache + (gt % CH) * 8;
      const bool pad = (gt % CH) * 8 >= a.D;
      const int ch = gt % CH;
#pragma unroll 8
      for (int r = gt / CH; r < TK; r += C::NT / CH) {
        const long long ov = offs[r], ok = offs[r + 1];
        const uint32_t dst = (uint32_t)r * ROWB + (uint32_t)((ch ^ (r / NJ)) << 4);
        cp_async16(ks + dst, ok < -1 ? (const void*)&g_nan16 : (const void*)(kc + (ok < 0 ? 0 : ok)), ok == -1 || pad);
        cp_async16(vs + dst, ov < -1 ? (const void*)&g_nan16 : (const void*)(vc + (ov < 0 ? 0 : ov)), ov == -1 || pad);
      }
      if (gt < CH) {
        if (d.first) {
          const long long ok = offs[0];
          cp_async16(ks + TK * ROWB + (ch << 4), ok < -1 ? (const void*)&g_nan16 : (const void*)(kc + (ok < 0 ? 0 : ok)),
                     ok == -1 || pad);
        }
        if (d.last) {
          const long long ov = offs[TK];
          cp_async16(vs + TK * ROWB + (ch << 4), ov < -1 ? (const void*)&g_nan16 : (const void*)(vc + (ov < 0 ? 0 : ov)),
                     ov == -1 || pad);
        }
      }
      if constexpr (C::kStageQ) {
        if (d.first) {
          for (int x = gt; x < C::RPW * CH; x += C::NT) {
            const int r = x / CH, q = x % CH;
            const int row = d.rt * C::BR + r;
            const bool none = row >= d.n * plan.group || q * 8 >= a.D;
            const int t = none ? 0 : row / plan.group, hh = none ? 0 : row - t * plan.group;
            const T* src = (const T*)a.q + (none ? 0 : (size_t)(d.start + t) * a.q_token_stride +
                                                          (size_t)(d.h * plan.group + hh) * a.q_head_stride + q * 8);
            cp_async16(vs + C::KV_BYTES + r * ROWB + (q << 4), src, none);
          }
        }
      }
    }
    cp_commit();
    ++xb;
    if (++slot_b == C::RING) slot_b = 0;
    if (++stage_b == NST) stage_b = 0;
  };

  // ---- the consumer's state
  constexpr int RS = C::RPW == 8 ? 1 : 2;      // row sets per lane: rows r8 (and r8 + 8)
  uint32_t qf[NKK][4];
  float o[NN][4];
  float m[RS], carry_s[RS], carry_b[RS], scale[RS];
  float2 z2[RS];
  int pos[RS];
  int i_min = 0, i_max = -1, kt0 = 0;
  bool in_first = true;                         // the piece starts the worker's range

  // lanes' addresses within a stage: B fragments of K (score tile j: + j rows) and of V
  const int mi = lane >> 3, rr = lane & 7;
  const uint32_t k_lane = (uint32_t)((2 * NJ * (rr >> 1) + NJ * (rr & 1)) * ROWB + ((mi ^ rr) << 4));
  const uint32_t v_lane = (uint32_t)((2 * NJ * (rr >> 1) + NJ * (rr & 1) + (mi & 1)) * ROWB + (((mi >> 1) ^ rr) << 4));

  describe();
  group_sync<C::RW>();
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) {
    copy();
    describe();
    group_sync<C::RW>();
  }

  int slot = 0, stage = 0;
  for (unsigned x = x0; x < x1; ++x) {
    cp_wait<NST - 2>();
    group_sync<C::RW>();     // this tile has arrived, and every warp has left the stage filled next
    copy();
    describe();

    const Desc& d = desc_ring[slot];
    const uint32_t ks = smem_addr(gsm + stage * C::STAGE), vs = ks + C::KV_BYTES;
    const int base = d.kt * TK;
    const int rows = d.n * plan.group;
    if (d.first) {
      kt0 = d.kt;
      in_first = x == x0;
      const int row0 = d.rt * C::BR + warp * C::RPW;
      const int row_last = min(rows, row0 + C::RPW) - 1;    // < row0: the warp has no row
      const int lead = d.len - d.n;                         // position of the sequence's first row
      i_min = lead + row0 / plan.group;
      i_max = row_last >= row0 ? lead + row_last / plan.group : -1;
      const T* qrow[RS];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        const int row = row0 + r8 + 8 * u;
        const bool none = row > row_last;
        const int t = (none ? max(row_last, 0) : row) / plan.group;
        const int head = d.h * plan.group + (none ? 0 : row - t * plan.group);
        pos[u] = lead + t;
        scale[u] = expf(a.log_gain[head]) * a.inv_sqrt_d;
        m[u] = -INFINITY;
        z2[u] = splat2(0.f);
        carry_s[u] = carry_b[u] = 0.f;
        qrow[u] = none ? nullptr : (const T*)a.q + (size_t)(d.start + t) * a.q_token_stride +
                                       (size_t)head * a.q_head_stride;
      }
#pragma unroll
      for (int n = 0; n < NN; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < NKK; ++k) {
        if constexpr (C::kStageQ) {
          const uint8_t* qs = gsm + stage * C::STAGE + 2 * C::KV_BYTES + r8 * ROWB + (16 * k + 2 * c4) * 2;
          qf[k][0] = *reinterpret_cast<const uint32_t*>(qs);
          qf[k][2] = *reinterpret_cast<const uint32_t*>(qs + 16);
          qf[k][1] = qf[k][3] = 0u;
        } else {
#pragma unroll
          for (int u = 0; u < RS; ++u) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int col = 16 * k + 8 * w + 2 * c4;
              qf[k][u + 2 * w] = qrow[u] && col < a.D ? *reinterpret_cast<const uint32_t*>(qrow[u] + col) : 0u;
            }
          }
          if (RS == 1) qf[k][1] = qf[k][3] = 0u;
        }
      }
      if (d.kt > 0 && base - 1 <= i_max) {
        // the score of key base - 1, in every column of one score tile
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t addr = ks + TK * ROWB + (mi << 4);
#pragma unroll
        for (int kp = 0; kp < NKK / 2; ++kp) {
          uint32_t b[4];
          ldsm4(b, addr + (kp << 6));
          mma<T>(s, qf[2 * kp][0], qf[2 * kp][1], qf[2 * kp][2], qf[2 * kp][3], b[0], b[1]);
          mma<T>(s, qf[2 * kp + 1][0], qf[2 * kp + 1][1], qf[2 * kp + 1][2], qf[2 * kp + 1][3], b[2], b[3]);
        }
#pragma unroll
        for (int u = 0; u < RS; ++u) {
          carry_s[u] = s[2 * u] * scale[u];
          if (base - 1 <= pos[u]) m[u] = carry_s[u];
        }
      }
    }

    // a warp none of whose rows sees a segment of this tile, or its first weight, has nothing to do
    if (base - 1 <= i_max && i_max >= 0) {
      float2 s[RS][NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < NKK / 2; ++kp) {
          uint32_t b[4];
          ldsm4(b, (ks + k_lane + j * ROWB) ^ (kp << 6));
          mma<T>(acc, qf[2 * kp][0], qf[2 * kp][1], qf[2 * kp][2], qf[2 * kp][3], b[0], b[1]);
          mma<T>(acc, qf[2 * kp + 1][0], qf[2 * kp + 1][1], qf[2 * kp + 1][2], qf[2 * kp + 1][3], b[2], b[3]);
        }
#pragma unroll
        for (int u = 0; u < RS; ++u) s[u][j] = make_float2(acc[2 * u], acc[2 * u + 1]);
      }
      const bool edge = base == 0 || base + TK - 1 > i_min;
      const int kc = base + 2 * NJ * c4;        // first key of the lane's run
      const int lowest = d.first ? base : base - 1;
      uint32_t hi[RS][NJ], lo[RS][NJ];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        float top = -INFINITY;
        if (edge) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            if (kc + j <= pos[u]) top = fmaxf(top, s[u][j].x);
            if (kc + NJ + j <= pos[u]) top = fmaxf(top, s[u][j].y);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NJ; ++j) top = max3f(top, s[u][j].x, s[u][j].y);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * scale[u];
        const bool move = top > m[u] + kRescaleNats || (m[u] == -INFINITY && top > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float to = move ? top : m[u];
          const float f = move ? exp_rel(m[u] - to) : 1.f;
          m[u] = to;
          carry_b[u] *= f;
          z2[u] = mul2(z2[u], splat2(f));
#pragma unroll
          for (int n = 0; n < NN; ++n) {
            o[n][2 * u] *= f;
            o[n][2 * u + 1] *= f;
            if (RS == 1) {
              o[n][2] *= f;
              o[n][3] *= f;
            }
          }
        }
        const float m2 = m[u] == -INFINITY ? 0.f : m[u] * kLog2e;
        const int left = (lane & ~3) | ((lane + 3) & 3);
        float got = __shfl_sync(0xffffffffu, s[u][NJ - 1].y * scale[u], left);
        const float sL = c4 == 0 ? carry_s[u] : got;
        if (c4 == 0) carry_s[u] = got;
        float2 W[NJ];
        float last;
        if (edge) weigh<true, NJ>(s[u], scale[u], m2, kc, pos[u], lowest, sL, W, last, z2[u]);
        else weigh<false, NJ>(s[u], scale[u], m2, kc, pos[u], lowest, sL, W, last, z2[u]);
        got = __shfl_sync(0xffffffffu, last, left);
        W[0].x += c4 == 0 ? carry_b[u] : got;
        if (c4 == 0) carry_b[u] = got;
#pragma unroll
        for (int j = 0; j < NJ; ++j) split2<T>(W[j], hi[u][j], lo[u][j]);
      }
#pragma unroll
      for (int kk = 0; kk < TK / 16; ++kk) {
#pragma unroll
        for (int np = 0; np < NN / 2; ++np) {
          uint32_t b[4];
          ldsm4_t(b, (vs + v_lane + 2 * kk * ROWB) ^ (np << 5));
          if constexpr (RS == 1) {
            mma<T>(o[2 * np], hi[0][2 * kk], lo[0][2 * kk], hi[0][2 * kk + 1], lo[0][2 * kk + 1], b[0], b[1]);
            mma<T>(o[2 * np + 1], hi[0][2 * kk], lo[0][2 * kk], hi[0][2 * kk + 1], lo[0][2 * kk + 1], b[2], b[3]);
          } else {
            mma<T>(o[2 * np], hi[0][2 * kk], hi[RS - 1][2 * kk], hi[0][2 * kk + 1], hi[RS - 1][2 * kk + 1], b[0], b[1]);
            mma<T>(o[2 * np + 1], hi[0][2 * kk], hi[RS - 1][2 * kk], hi[0][2 * kk + 1], hi[RS - 1][2 * kk + 1], b[2],
                   b[3]);
            mma<T>(o[2 * np], lo[0][2 * kk], lo[RS - 1][2 * kk], lo[0][2 * kk + 1], lo[RS - 1][2 * kk + 1], b[0], b[1]);
            mma<T>(o[2 * np + 1], lo[0][2 * kk], lo[RS - 1][2 * kk], lo[0][2 * kk + 1], lo[RS - 1][2 * kk + 1], b[2],
                   b[3]);
          }
        }
      }
    }

    if (d.last) {
      const bool whole = kt0 == 0 && d.kt + 1 == d.nt;
      const int row0 = d.rt * C::BR + warp * C::RPW;
      const int key = base + TK - 1;             // the key whose weight is still carried
      const long long slot_row = ((long long)worker * 2 + (in_first ? 0 : 1)) * C::BR + warp * C::RPW;
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        const int row = row0 + r8 + 8 * u;
        const float m2 = m[u] == -INFINITY ? 0.f : m[u] * kLog2e;
        float w = __shfl_sync(0xffffffffu, carry_b[u], lane & ~3);
        const float ls = __shfl_sync(0xffffffffu, carry_s[u], lane & ~3);
        const float cap = key == pos[u] ? 0.5f * ex2_approx(fmaf(ls, kLog2e, -m2)) : 0.f;
        w += cap;
        float z = z2[u].x + z2[u].y + (c4 == 0 ? cap : 0.f);
        z += __shfl_xor_sync(0xffffffffu, z, 1);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        if (d.bad) z = __int_as_float(0x7fffffff);
        if (row >= rows) continue;
        const bool seen = key <= pos[u];         // else the weight is 0, and V may hold anything
        const int t = row / plan.group;
        T* dst = (T*)a.o + ((size_t)(d.start + t) * a.H + (size_t)d.h * plan.group + (row - t * plan.group)) * a.D;
        float* po = part_o + (slot_row + r8 + 8 * u) * DP;
        // z = 0: the row sees no key
        const float inv = 1.f / z;
        const uint8_t* vrow = gsm + stage * C::STAGE + C::KV_BYTES + TK * ROWB + 4 * c4;
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          const int col = 8 * n + 2 * c4;
          float2 y = make_float2(o[n][2 * u], o[n][2 * u + 1]);
          if (RS == 1) {
            y.x += o[n][2];
            y.y += o[n][3];
          }
          if (seen) {
            const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t*>(vrow + 16 * n));
            y.x = fmaf(w, v.x, y.x);
            y.y = fmaf(w, v.y, y.y);
          }
          if (whole) {
            if (col < a.D) *reinterpret_cast<uint32_t*>(dst + col) = z == 0.f ? 0u : pack2<T>(y.x * inv, y.y * inv);
          } else {
            *reinterpret_cast<float2*>(po + col) = y;
          }
        }
        if (!whole && c4 == 0) part_mz[slot_row + r8 + 8 * u] = make_float2(m[u], z);
      }
    }
    if (x + 1 == x1 && gt == 0) {
      // this worker joins the unit that starts in its range and goes on behind it
      Meta mt;
      mt.pieces = kt0 == 0 && d.kt + 1 < d.nt ? 1 + (d.nt - d.kt - 2 + (int)per) / (int)per : 0;
      mt.slot = in_first ? 0 : 1;
      mt.start = d.start;
      mt.rows = rows;
      mt.h = d.h;
      mt.rt = d.rt;
      meta[worker] = mt;
    }
    if (++slot == C::RING) slot = 0;
    if (++stage == NST) stage = 0;
  }
  cp_wait<0>();
}

// Joins the pieces of a cut unit in the order of their keys: piece 0 is in this worker's slot, the others
// are the first pieces of the workers that follow.
template <typename T, int DP, int BR>
__global__ void __launch_bounds__(128) merge_kernel(Args a, int group, const float* __restrict__ part_o,
                                                    const float2* __restrict__ part_mz,
                                                    const Meta* __restrict__ meta) {
  pdl_wait();
  pdl_launch_dependents();
  const int w = blockIdx.x;
  const Meta mt = meta[w];
  if (mt.pieces == 0) return;
  const int nrows = min(BR, mt.rows - mt.rt * BR);
  constexpr int V = DP / 4;
  for (int x = threadIdx.x; x < nrows * V; x += blockDim.x) {
    const int r = x / V, d0 = (x - r * V) * 4;
    float m = -INFINITY, z = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < mt.pieces; ++p) {
      const long long row = ((long long)(w + p) * 2 + (p == 0 ? mt.slot : 0)) * BR + r;
      const float2 mz = part_mz[row];
      const float4 v = *reinterpret_cast<const float4*>(part_o + row * DP + d0);
      if (mz.x == -INFINITY) {   // no key seen: no mass, or the NaN of a bad page or length
        z += mz.y;
        continue;
      }
      const float top = fmaxf(m, mz.x);
      const float fa = exp_rel(m - top), fb = exp_rel(mz.x - top);
      z = fmaf(z, fa, mz.y * fb);
      y = make_float4(fmaf(y.x, fa, v.x * fb), fmaf(y.y, fa, v.y * fb), fmaf(y.z, fa, v.z * fb), fmaf(y.w, fa, v.w * fb));
      m = top;
    }
    const float inv = z == 0.f ? 0.f : 1.f / z;   // y is 0 then
    const int row = mt.rt * BR + r, t = row / group;
    T* dst = (T*)a.o + ((size_t)(mt.start + t) * a.H + (size_t)mt.h * group + (row - t * group)) * a.D + d0;
    if (d0 < a.D) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
    }
  }
}

}  // namespace

// ------------------------------------------------------------------ host side

namespace {

// The forms: decoding with 8 or 16 rows a warp, and chunks
template <typename T, int DP> using Decode8 = Config<T, DP, 8, 1, 4, 3>;
template <typename T, int DP> using Decode16 = Config<T, DP, 16, 1, 4, 3>;
template <typename T, int DP> using Chunk = Config<T, DP, 16, 4, 1, 3>;

size_t part_bytes(long long workers, int br, int dp) {
  return (size_t)workers * 2 * br * (dp * sizeof(float) + sizeof(float2)) + (size_t)workers * sizeof(Meta) + 768;
}

template <typename T, typename C>
cudaError_t launch(const Args& a, Plan plan, void* workspace) {
  static_assert(C::SMEM + (kMaxSeqs + 1) * (int)sizeof(unsigned) <= 232448, "shared memory of a block");
  const size_t smem = C::SMEM + (size_t)(a.seqs + 1) * sizeof(unsigned);
  static thread_local int set_dev = -1;    // the attribute belongs to the device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (set_dev != dev) {
    e = cudaFuncSetAttribute(mma_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::SMEM + (kMaxSeqs + 1) * (int)sizeof(unsigned));
    if (e != cudaSuccess) return e;
    set_dev = dev;
  }
  const int blocks = num_sms_cached() * (C::RW == 1 ? 1 : kChunkBlocksPerSM);
  const long long workers = (long long)blocks * C::GROUPS;
  char* ws = (char*)workspace;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  float* po = (float*)ws;
  float2* mz = (float2*)(ws + up((size_t)workers * 2 * C::BR * C::DP * sizeof(float)));
  Meta* meta = (Meta*)((char*)mz + up((size_t)workers * 2 * C::BR * sizeof(float2)));
  e = launch_pdl(mma_kernel<T, C>, dim3(blocks), dim3(C::NT * C::GROUPS), smem, a.stream, a, plan, po, mz, meta);
  if (e != cudaSuccess) return e;
  return launch_pdl(merge_kernel<T, C::DP, C::BR>, dim3((unsigned)workers), dim3(128), 0, a.stream, a, plan.group,
                    (const float*)po, (const float2*)mz, (const Meta*)meta);
}

template <typename T, int DP>
cudaError_t forward_dp(const Args& a, void* workspace) {
  Plan plan = make_plan(a);
  const long long rows = (long long)a.max_q_len * plan.group;
  if (rows <= 16) {
    // every sequence, whatever its rows: max_q_len may be wrong
    return rows <= 8 ? launch<T, Decode8<T, DP>>(a, plan, workspace) : launch<T, Decode16<T, DP>>(a, plan, workspace);
  }
  // sequences of up to 16 rows in the decoding form, the others as chunks; both use the workspace, one
  // after the other
  plan.min_tiles = 4;
  plan.row_lo = 17;
  cudaError_t e = launch<T, Chunk<T, DP>>(a, plan, workspace);
  if (e != cudaSuccess || a.seqs == 1) return e;
  plan.min_tiles = 1;
  plan.row_lo = 0;
  plan.row_hi = 16;
  return launch<T, Decode16<T, DP>>(a, plan, workspace);
}

}  // namespace

size_t mma_workspace_bytes(long long max_q_len, long long H, long long G, long long D) {
  const int dp = D <= 64 ? 64 : 128;
  const long long sms = num_sms_cached(), rows = max_q_len * (H / G);
  const size_t decode = part_bytes(sms * 4, 16, dp);
  return rows <= 16 ? decode : std::max(decode, part_bytes(sms * kChunkBlocksPerSM, 64, dp));
}

cudaError_t mma_read_status(int* out, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
  if (e != cudaSuccess || !reset || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
}

int mma_launches(const Args& a) {
  const long long rows = (long long)a.max_q_len * (a.H / a.G);
  return rows <= 16 || a.seqs == 1 ? 2 : 4;
}

cudaError_t mma_forward(const Args& a, int dtype, void* workspace) {
  if (a.D <= 64)
    return dtype == 1 ? forward_dp<__nv_bfloat16, 64>(a, workspace) : forward_dp<__half, 64>(a, workspace);
  return dtype == 1 ? forward_dp<__nv_bfloat16, 128>(a, workspace) : forward_dp<__half, 128>(a, workspace);
}

}  // namespace paged
}  // namespace ca
