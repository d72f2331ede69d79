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
// A worker is RW consumer warps with 16 (or 8) rows each that share a ring of key tiles, and
// one producer warp that walks the stream ahead of them: it looks pages up, issues the copies
// and describes each tile.  With the copies in the consumers' own hands their warp 0 did a
// third more work than the others, who waited for it at every tile.  In the decoding form
// a worker has one consumer and 8 or 16 rows, for chunks four and 64 rows.
//
// Cutting keys.  Segments, not keys, are divided: the segment from key j-1 to key j belongs
// to the tile of j.  A tile of keys a .. a+TK-1 therefore weighs keys a-1 .. a+TK-2, and only
// the mass that ends at key a+TK-1 is carried on.  The first tile of a piece brings K and V
// row a-1 along (the score that the first segment starts from, the row it weighs); later
// tiles keep the V row of the tile before.
//
// Registers.  The products run on mma.sync m16n8k16 with scores in registers: the bound of
// this operator is the scalar work per score (one exp2, one reciprocal, about 13 packed or
// single instructions), not the tensor pipe, and register scores spare the trip through tensor
// memory.  B fragments may come from any rows, so keys are dealt to lanes in runs: column
// 2c + e of score tile j is key (TK/4) c + j + NJ e, NJ = TK/8.  A lane's pair (j, j + NJ)
// then has the pair (j-1, j-1 + NJ) as its left neighbours, every step of the moments is one
// packed f32x2 instruction for two keys, and neighbours in other lanes are needed once per
// run.  The weights leave as A fragments with the same dealing of V rows.  Each weight is
// split into two 16-bit parts (hi + lo: 16 bits in bf16, 21 in f16): one rounding to bf16 would put
// 1.1e-3 of the output's size on every row.  Against weights in 32 bits, 2 to 5 of a thousand bf16 outputs, and 2 of
// a hundred f16 ones, are another rounding of a value that lies within 7e-5 of the outputs' size from the border
// (prompts of 2 x 2048 tokens, 511 rows over 16001 keys); the error against 64 bits is the same to three digits.  With 8 rows or fewer hi and lo are the two
// halves of one fragment and cost one product.
//
// Shared memory.  The eight rows of a fragment lie NJ rows apart, so every NJ rows are
// followed by 16 bytes: the eight land in different banks without any address arithmetic, and
// each NJ rows (512 or 1024 bytes) are one bulk copy where the page holds them in one run,
// else one copy per row.
//
// What bounds it.  Decoding reads every visible key's K and V once and is bound by that: 2 sequences
// over 90001 .. 131071 keys (f16, 32 heads on 8 of 64, pages of 16) 97 us for 506 MB, 5.2 TB/s (on the
// same inputs again, some of them still in L2, 91); 17 sequences of 1 .. 4 rows over up to 20000 keys (bf16, 32
// heads on 8 of 128) 98 us for 484 MB, 4.9 TB/s; 64 sequences over 1 .. 8192 keys (bf16, 16 heads of 64) 51 us for
// 231 MB, 4.5 TB/s; a single sequence of 2048 keys is all latency, 13 us (launch, page look-ups, one round of
// copies, the join).
// Chunks are bound by the scalar work and its dependences (885 issue slots a warp for 1024 scores, 40% of
// the cycles issue); those of more than 64 rows are ca_paged_tc.cu's.
#include <algorithm>
#include <type_traits>

#include "ca_common.cuh"
#include "ca_paged.cuh"
#include "ca_paged_math.cuh"

namespace ca {
namespace paged {

namespace {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Whole warp; gives up after limit_ns (the barrier of copies that never land): records the timeout and
// raises the group's flag, which ends the others' waits too.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up,
                                         unsigned long long limit_ns) {
  bool ok = bar_try(bar, parity);
  if (!ok) {
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    while (!(ok = bar_try(bar, parity)) && !*gave_up) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t - t0 > limit_ns) {
        atomicCAS(&g_status, 0, 5);
        *gave_up = 1;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
// the producer's wait for room: with no limit at all it gives up at once, so that a call can be made to
__device__ __forceinline__ bool room_wait(uint32_t bar, uint32_t parity, volatile int* gave_up,
                                          unsigned long long limit_ns) {
  if (limit_ns > 0) return bar_wait(bar, parity, gave_up, limit_ns);
  atomicCAS(&g_status, 0, 5);
  *gave_up = 1;
  return false;
}
// a wait that no other warp's giving up ends (whole warp)
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  do asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  while (!bar_try(bar, parity) && t - t0 < kWaitNs);
  __syncwarp();
}
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// orders this thread's shared-memory writes before later bulk copies into the same place
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------------ the kernel

// Tiles of TK keys of DP (padded) values; RPW rows per warp (8 or 16); RW consumer warps that share a
// ring of NST stages (1 or 4); GROUPS rings per block.  One block per SM.  REGS_C and REGS_P: registers of a
// consumer and a producer thread, 0 where the launch's even share suffices.
template <int DP_, int TK_, int RPW_, int RW_, int GROUPS_, int NST_, int REGS_C_, int REGS_P_>
struct Config {
  static constexpr int DP = DP_, TK = TK_, RPW = RPW_, RW = RW_, GROUPS = GROUPS_, NST = NST_;
  static constexpr int REGS_C = REGS_C_, REGS_P = REGS_P_;
  static constexpr int CONSUMERS = GROUPS * RW;                          // warps
  static constexpr int THREADS = (CONSUMERS + (GROUPS + 3) / 4 * 4) * 32;   // producers in whole warpgroups
  static constexpr int BR = RPW * RW;                   // rows of a unit
  static constexpr int NJ = TK / 8;                     // score tiles of 8 keys; half a lane's run
  static constexpr int CH = DP / 8;                     // 16-byte chunks of a row
  static constexpr int ROWB = DP * 2;
  static constexpr int PITCH = NJ * ROWB + 16;          // of NJ rows
  static constexpr int KV_BYTES = 8 * PITCH;
  static constexpr bool kStageQ = RW == 1;
  static constexpr int HALO = 2 * KV_BYTES;             // K row, then V row before the tile
  static constexpr int Q_AT = HALO + 2 * ROWB;
  static constexpr int STAGE = Q_AT + (kStageQ ? RPW * ROWB : 0);
  static constexpr int RING = NST + 1;                  // descriptors live one tile longer
  // behind the stages: each warp's V row of the tile before (in the banks that the fragments leave free),
  // descriptors, barriers, the flag of a wait that gave up
  static constexpr int WARP_HALO = ROWB + 128;
  // several warps: query fragments wait here for the next tile (16 registers that the moments need more)
  static constexpr int Q_FRAG = RW > 1 ? DP * 32 : 0;   // bytes of a warp
  static constexpr int QF_AT = NST * STAGE + RW * WARP_HALO;
  static constexpr int DESC_AT = QF_AT + RW * Q_FRAG;
  static constexpr int BAR_AT = DESC_AT + RING * 32;
  static constexpr int GROUP_STRIDE = (BAR_AT + 2 * NST * 8 + 16 + 127) / 128 * 128;
  static constexpr int SMEM = GROUPS * GROUP_STRIDE;    // and the prefix sums behind it
  static_assert(KV_BYTES % 128 == 0 && STAGE % 128 == 0 && DESC_AT % 16 == 0, "");
  // setmaxnreg draws on what the block was launched with
  static constexpr int REGS_LAUNCH = 65536 / THREADS / 8 * 8;
  static_assert(REGS_C == 0 || (CONSUMERS % 4 == 0 && CONSUMERS * REGS_C + (THREADS / 32 - CONSUMERS) * REGS_P <=
                                                          THREADS / 32 * REGS_LAUNCH), "");
};

// one tile of the stream; consumers read the first four words of every tile, the others at a piece's ends
struct alignas(16) Desc {
  int kt, flags, len, nt;   // tile in its unit, flags, keys of the sequence, tiles of the unit
  int start, n, h, rt;      // the sequence's rows; key head; row tile
};
// of the piece: its first tile, its last; the sequence's length or a page is out of range; the worker's last
// tile; the worker has none
enum : int { kFirst = 1, kLast = 2, kBad = 4, kEnd = 8, kNone = 16 };

template <typename T, typename C>
__global__ void __launch_bounds__(C::THREADS, 1)
    mma_kernel(const __grid_constant__ Args a, const __grid_constant__ Plan plan, float* __restrict__ part_o,
               float2* __restrict__ part_mz, Meta* __restrict__ meta, int after_chunks) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // after_chunks: the kernel before this one in the stream is the chunks' launch of the same call.  Nothing
  // here depends on it, and what both depend on was complete before it let this one start; so this one
  // fills the SMs that it leaves, and waits for it at the end (every warp that leaves), since the merge
  // that follows waits for this kernel only.
  if (!after_chunks) pdl_wait();
  pdl_launch_dependents();
  constexpr int TK = C::TK, NJ = C::NJ, DP = C::DP, ROWB = C::ROWB, CH = C::CH, NST = C::NST;
  constexpr int NKK = DP / 16;                 // k-steps of Q K^T
  constexpr int NN = DP / 8;                   // column tiles of the output
  const int lane = threadIdx.x & 31, c4 = lane & 3, r8 = lane >> 2;
  const int wid = threadIdx.x >> 5;
  const bool producer = wid >= C::CONSUMERS;
  const int group = producer ? wid - C::CONSUMERS : wid / C::RW, warp = wid % C::RW;
  unsigned* prefix = reinterpret_cast<unsigned*>(smem + C::SMEM);
  uint8_t* gsm = smem + (size_t)group * C::GROUP_STRIDE;
  const uint32_t g0 = smem_addr(gsm);
  Desc* descs = reinterpret_cast<Desc*>(gsm + C::DESC_AT);
  const uint32_t full = g0 + C::BAR_AT, empty = full + 8 * NST;
  volatile int* gave_up = reinterpret_cast<volatile int*>(gsm + C::BAR_AT + 16 * NST);

  if (producer && group < C::GROUPS) {
    if (lane == 0) {
      for (int i = 0; i < NST; ++i) {
        bar_init(full + 8 * i, 1);
        bar_init(empty + 8 * i, C::RW);
      }
      *gave_up = 0;
    }
    // values behind D stay 0 (copies write D values a row)
    if (a.D < DP) {
      for (int x = lane; x < NST * C::STAGE / 16; x += 32)
        *reinterpret_cast<uint4*>(gsm + 16 * x) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_async();
  }
  Schedule<C::BR, TK> sched(a, plan, prefix);   // a barrier of the block among other things
  const unsigned total = sched.total;
  const int worker = blockIdx.x * C::GROUPS + group, workers = gridDim.x * C::GROUPS;
  const unsigned per = plan.places_per_worker(total, workers);
  const unsigned x0 = (unsigned)min((unsigned long long)worker * per, (unsigned long long)total);
  const unsigned x1 = (unsigned)min((unsigned long long)x0 + per, (unsigned long long)total);

  if (producer) {
    if constexpr (C::REGS_C > 0) regs_down<C::REGS_P>();
    if (group >= C::GROUPS) {
      if (after_chunks) pdl_wait();
      return;
    }
    if (lane == 0) meta[worker] = sched.none();
    // `cur` stands at the next tile to be described; a tile's pages are fetched when it is described, one tile
    // before its copies are issued.  Every instruction here counts: the producer shares a scheduler with
    // the consumers.
    typename Schedule<C::BR, TK>::Cursor cur;
    cur.at = x1;
    if (x0 < x1) cur = sched.locate(x0);
    if (cur.at >= x1) {            // no tile's place lies in this range
      if (lane == 0) {
        descs[0].flags = kNone;
        bar_expect(full, 0);
      }
      if (after_chunks) pdl_wait();
      return;
    }
    int kt0 = 0;                   // the first tile of the piece
    bool more = true, first = true, in_first = true;
    constexpr int NP = TK / 32;
    int pg[NP];                    // page of a lane's rows
    long long in_page[NP];         // and their offset in it
    int halo_page = -1;            // of the key before a piece that does not start at key 0
    Desc d;                        // the described tile

  auto in_page_of = [&](int key, int col, int h) {
    return (long long)h * a.head_stride + (long long)(key - col * a.page_size) * a.slot_stride;
  };
  auto describe = [&]() {
    const int* pages = a.page_table + (size_t)cur.s * a.page_table_stride;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int row = plan.unit_rows == 1 ? lane + 32 * k : (k == 0 && lane < 8 ? lane * NJ : TK);
      const int key = cur.kt * TK + row;
      pg[k] = -1;
      if (row < TK && key < cur.len) {
        const int col = plan.page_of(key);
        pg[k] = pages[col];
        in_page[k] = in_page_of(key, col, cur.h);
      }
    }
    d.kt = cur.kt;
    d.nt = cur.nt;
    d.flags = cur.bad ? kBad : 0;
    if (first || cur.kt == 0) {
      d.flags |= kFirst;
      kt0 = cur.kt;
      in_first = first;
      first = false;
      halo_page = cur.kt > 0 ? pages[plan.page_of(cur.kt * TK - 1)] : -1;
    }
    d.start = cur.start;
    d.n = cur.n;
    d.len = cur.len;
    d.h = cur.h;
    d.rt = cur.rt;
    const unsigned at = cur.at;
    more = at + 1 < x1;
    if (!more || cur.kt + 1 == cur.nt) d.flags |= kLast;
    if (more) {
      sched.advance(cur);
      more = cur.at < x1;        // the next unit's first tile may lie behind the range
    }
    if (!more) {
      d.flags |= kEnd;
      if (lane == 0) {
        // this worker joins the unit that starts in its range and goes on behind it
        Meta mt;
        mt.pieces = kt0 == 0 && d.kt + 1 < d.nt ? 1 + (int)((at + (d.nt - 1 - d.kt)) / per) - worker : 0;
        mt.slot = in_first ? 0 : 1;
        mt.start = d.start;
        mt.rows = d.n * plan.group;
        mt.h = d.h;
        mt.rt = d.rt;
        meta[worker] = mt;
      }
    }
  };

  int slot_b = 0, stage_b = 0;
  uint32_t empty_parity = 1;      // of the stage's previous use
  describe();
  int k = 0;
  for (int end = 0; !end; ++k) {
    if (k >= NST && !room_wait(empty + 8 * stage_b, empty_parity, gave_up, plan.wait_ns)) break;
    {
      const uint32_t st = g0 + stage_b * C::STAGE, bar = full + 8 * stage_b;
      const int base = d.kt * TK;
      end = d.flags & kEnd;
      const uint32_t row_bytes = (uint32_t)a.D * 2;
      const uint32_t unit_bytes = plan.unit_rows * row_bytes;
      bool go[NP], bad = false;
      uint32_t bytes = 0;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int row = plan.unit_rows == 1 ? lane + 32 * k : (k == 0 && lane < 8 ? lane * NJ : TK);
        go[k] = pg[k] >= 0 && pg[k] < a.num_pages;      // -1 where there is nothing to fetch
        bad |= !go[k] && row < TK && base + row < d.len;
        bytes += __popc(__ballot_sync(0xffffffffu, go[k])) * 2 * unit_bytes;
      }
      bool halo = false;
      int q_row = -1;
      if (d.flags & kFirst) {
        halo = base > 0 && base - 1 < d.len;
        const bool in = halo_page >= 0 && halo_page < a.num_pages;
        bad |= halo && !in;
        halo = halo && in;
        if (halo) bytes += 2 * row_bytes;
        if constexpr (C::kStageQ) {
          if (lane < C::RPW && d.rt * C::BR + lane < d.n * plan.group) q_row = d.rt * C::BR + lane;
          bytes += __popc(__ballot_sync(0xffffffffu, q_row >= 0)) * row_bytes;
        }
      }
      bad = __any_sync(0xffffffffu, bad);
      if (lane == 0) {
        if (bad) {
          d.flags |= kBad;
          record_invalid();
        }
        int4* to = reinterpret_cast<int4*>(&descs[slot_b]);
        to[0] = make_int4(d.kt, d.flags, d.len, d.nt);
        to[1] = make_int4(d.start, d.n, d.h, d.rt);
        bar_expect(bar, bytes);
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        if (go[k]) {
          const int row = plan.unit_rows == 1 ? lane + 32 * k : lane * NJ;
          const long long at = (long long)pg[k] * a.page_stride + in_page[k];
          const uint32_t dst = st + (row / NJ) * C::PITCH + (row % NJ) * ROWB;
          bulk_load(dst, (const T*)a.k_cache + at, unit_bytes, bar);
          bulk_load(dst + C::KV_BYTES, (const T*)a.v_cache + at, unit_bytes, bar);
        }
      }
      if (halo && lane == 31) {
        const long long at = (long long)halo_page * a.page_stride +
                             in_page_of(base - 1, plan.page_of(base - 1), d.h);
        bulk_load(st + C::HALO, (const T*)a.k_cache + at, row_bytes, bar);
        bulk_load(st + C::HALO + ROWB, (const T*)a.v_cache + at, row_bytes, bar);
      }
      if (q_row >= 0) {
        const int t = q_row / plan.group;
        bulk_load(st + C::Q_AT + lane * ROWB,
                  (const T*)a.q + (size_t)(d.start + t) * a.q_token_stride +
                      (size_t)(d.h * plan.group + q_row - t * plan.group) * a.q_head_stride,
                  row_bytes, bar);
      }
    }
    if (++slot_b == C::RING) slot_b = 0;
    if (++stage_b == NST) {
      stage_b = 0;
      empty_parity ^= 1;
    }
    if (!end) describe();
  }
  // every copy has to land before this block's shared memory is another's, where the consumers gave up too
  for (int u = max(k - NST, 0); u < k; ++u) bar_drain(full + 8 * (u % NST), (u / NST) & 1);
  if (after_chunks) pdl_wait();
  return;
  }

  if constexpr (C::REGS_C > 0) regs_up<C::REGS_C>();
  // ---- the consumers' state
  constexpr int RS = C::RPW == 8 ? 1 : 2;      // row sets per lane: rows r8 (and r8 + 8)
  uint32_t qf[NKK][4];
  float o[NN][4];
  float m[RS], carry_s[RS], carry_b[RS], scale[RS];
  float2 z2[RS];
  int pos[RS];
  int i_min = 0, i_max = -1, kt0 = 0, piece_bad = 0;
  bool in_first = true;                         // the piece starts the worker's range

  // lanes' addresses within a stage: B fragments of K (score tile j: + j rows) and of V (k-step kk: + 2 kk
  // rows, one row early; place 0 of a run is the row before it)
  const int mi = lane >> 3, rr = lane & 7;
  const uint32_t k_lane = (uint32_t)(rr * C::PITCH + mi * 16);
  const uint32_t v_lane = (uint32_t)(C::KV_BYTES + rr * C::PITCH + ((mi & 1) - 1) * ROWB + (mi >> 1) * 16);
  const uint32_t my_halo = g0 + NST * C::STAGE + warp * C::WARP_HALO + 112;
  uint8_t* my_halo_p = gsm + NST * C::STAGE + warp * C::WARP_HALO + 112;

  uint8_t* my_qf = gsm + C::QF_AT + warp * C::Q_FRAG + 16 * lane;

  int slot = 0, stage = 0;
  uint32_t parity = 0;
  bool first_tile = true;
  for (int end = 0; !end;) {
    if (!bar_wait(full + 8 * stage, parity, gave_up, plan.wait_ns)) break;
    const Desc& d = descs[slot];
    const int4 head = *reinterpret_cast<const int4*>(&d);
    const int kt = head.x, flags = head.y, len = head.z;
    end = flags & (kEnd | kNone);
    if (flags & kNone) break;
    uint8_t* sm = gsm + stage * C::STAGE;
    const uint32_t st = g0 + stage * C::STAGE;
    const int base = kt * TK;
    if (flags & kFirst) {
      kt0 = kt;
      const int rows = d.n * plan.group;
      piece_bad = 0;
      in_first = first_tile;
      first_tile = false;
      const int row0 = d.rt * C::BR + warp * C::RPW;
      const int row_last = min(rows, row0 + C::RPW) - 1;    // < row0: the warp has no row
      const int lead = len - d.n;                         // position of the sequence's first row
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
        carry_s[u] = kMasked;
        carry_b[u] = 0.f;
        qrow[u] = none ? nullptr : (const T*)a.q + (size_t)(d.start + t) * a.q_token_stride +
                                       (size_t)head * a.q_head_stride;
      }
#pragma unroll
      for (int n = 0; n < NN; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < NKK; ++k) {
        if constexpr (C::kStageQ) {
          const uint8_t* qs = sm + C::Q_AT + r8 * ROWB + (16 * k + 2 * c4) * 2;
          qf[k][0] = *reinterpret_cast<const uint32_t*>(qs);
          qf[k][2] = *reinterpret_cast<const uint32_t*>(qs + 16);
          qf[k][1] = RS == 2 ? *reinterpret_cast<const uint32_t*>(qs + 8 * ROWB) : 0u;
          qf[k][3] = RS == 2 ? *reinterpret_cast<const uint32_t*>(qs + 8 * ROWB + 16) : 0u;
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
      if constexpr (C::Q_FRAG > 0) {
#pragma unroll
        for (int k = 0; k < NKK; ++k)
          *reinterpret_cast<uint4*>(my_qf + 512 * k) = make_uint4(qf[k][0], qf[k][1], qf[k][2], qf[k][3]);
      }
      if (kt > 0 && base - 1 <= i_max) {
        // the score of key base - 1, in every column of one score tile
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < NKK / 2; ++kp) {
          uint32_t b[4];
          ldsm4(b, st + C::HALO + mi * 16 + kp * 64);
          mma<T>(s, qf[2 * kp][0], qf[2 * kp][1], qf[2 * kp][2], qf[2 * kp][3], b[0], b[1]);
          mma<T>(s, qf[2 * kp + 1][0], qf[2 * kp + 1][1], qf[2 * kp + 1][2], qf[2 * kp + 1][3], b[2], b[3]);
        }
#pragma unroll
        for (int u = 0; u < RS; ++u) {
          if (base - 1 <= pos[u]) m[u] = carry_s[u] = s[2 * u] * scale[u];
        }
      }
      if (lane < CH)
        *reinterpret_cast<uint4*>(my_halo_p + 16 * lane) =
            kt > 0 ? *reinterpret_cast<const uint4*>(sm + C::HALO + ROWB + 16 * lane) : make_uint4(0u, 0u, 0u, 0u);
    }
    piece_bad |= flags & kBad;
    if (base + TK > len) {
      // V behind the sequence's end may hold anything, and 0 times it has to be 0.  The warps of a group
      // write the same zeros.
      for (int r = max(len - base, 0) * CH + lane; r < TK * CH; r += 32) {
        const int row = r / CH;
        *reinterpret_cast<uint4*>(sm + C::KV_BYTES + (row / NJ) * C::PITCH + (row % NJ) * ROWB + (r % CH) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async();
    }
    __syncwarp();

    // a warp none of whose rows sees a segment of this tile, or its first weight, has nothing to do
    if (base - 1 <= i_max && i_max >= 0) {
      float2 s[RS][NJ];
      const uint32_t ka = st + k_lane;
      if constexpr (C::Q_FRAG > 0) {
#pragma unroll
        for (int k = 0; k < NKK; ++k) {
          const uint4 t = *reinterpret_cast<const uint4*>(my_qf + 512 * k);
          qf[k][0] = t.x;
          qf[k][1] = t.y;
          qf[k][2] = t.z;
          qf[k][3] = t.w;
        }
      }
      // score tiles side by side, so that no product waits for the one before it
      float acc[NJ][4];
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
      for (int kp = 0; kp < NKK / 2; ++kp) {
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
          uint32_t b[2][4];
          ldsm4(b[0], ka + j * ROWB + kp * 64);
          ldsm4(b[1], ka + (j + 1) * ROWB + kp * 64);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma<T>(acc[j], qf[2 * kp + e][0], qf[2 * kp + e][1], qf[2 * kp + e][2], qf[2 * kp + e][3], b[0][2 * e],
                   b[0][2 * e + 1]);
            mma<T>(acc[j + 1], qf[2 * kp + e][0], qf[2 * kp + e][1], qf[2 * kp + e][2], qf[2 * kp + e][3], b[1][2 * e],
                   b[1][2 * e + 1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int u = 0; u < RS; ++u) s[u][j] = mul2(make_float2(acc[j][2 * u], acc[j][2 * u + 1]), splat2(scale[u]));
      // keys beyond a row's own, or caps among the weights
      const bool edge = base == 0 || base + TK - 1 > i_min;
      const int kc = base + 2 * NJ * c4;        // first key of the lane's run
      if (edge) {
#pragma unroll
        for (int u = 0; u < RS; ++u) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            if (kc + j > pos[u]) s[u][j].x = kMasked;
            if (kc + NJ + j > pos[u]) s[u][j].y = kMasked;
          }
        }
      }
      uint32_t hi[RS][NJ], lo[RS][NJ];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        float top = max3f(s[u][0].x, s[u][0].y, s[u][1].x);
        top = fmaxf(top, s[u][1].y);
#pragma unroll
        for (int j = 2; j < NJ; ++j) top = max3f(top, s[u][j].x, s[u][j].y);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool move = top > kMasked && top > m[u] + kRescaleNats;
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
        const float m2 = reference2<T>(m[u]);
        const int left = (lane & ~3) | ((lane + 3) & 3);
        float got = __shfl_sync(0xffffffffu, s[u][NJ - 1].y, left);
        const float sL = c4 == 0 ? carry_s[u] : got;
        carry_s[u] = got;                       // of use to the quad's first lane only
        float2 first;
        float last;
        weigh<T, NJ>(s[u], m2, sL, edge, kc, pos[u], flags & kFirst ? base : base - 1, hi[u], lo[u], first, last,
                     z2[u]);
        got = __shfl_sync(0xffffffffu, last, left);
        first.x += c4 == 0 ? carry_b[u] : got;
        carry_b[u] = got;
        split2<T>(first, hi[u][0], lo[u][0]);
      }
      const uint32_t va = st + v_lane;
      const uint32_t va0 = lane == 0 || lane == 16 ? my_halo + (mi >> 1) * 16
                           : (mi & 1) || rr == 0 ? va : va - C::PITCH + NJ * ROWB;
#pragma unroll
      for (int kk = 0; kk < TK / 16; ++kk) {
#pragma unroll
        for (int np = 0; np < NN / 2; np += 2) {
          uint32_t b[2][4];
          ldsm4_t(b[0], (kk == 0 ? va0 : va + 2 * kk * ROWB) + np * 32);
          ldsm4_t(b[1], (kk == 0 ? va0 : va + 2 * kk * ROWB) + np * 32 + 32);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t b0 = b[t >> 1][2 * (t & 1)], b1 = b[t >> 1][2 * (t & 1) + 1];
            if constexpr (RS == 1)
              mma<T>(o[2 * np + t], hi[0][2 * kk], lo[0][2 * kk], hi[0][2 * kk + 1], lo[0][2 * kk + 1], b0, b1);
            else
              mma<T>(o[2 * np + t], hi[0][2 * kk], hi[RS - 1][2 * kk], hi[0][2 * kk + 1], hi[RS - 1][2 * kk + 1], b0, b1);
          }
          if constexpr (RS == 2) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              mma<T>(o[2 * np + t], lo[0][2 * kk], lo[RS - 1][2 * kk], lo[0][2 * kk + 1], lo[RS - 1][2 * kk + 1],
                     b[t >> 1][2 * (t & 1)], b[t >> 1][2 * (t & 1) + 1]);
          }
        }
      }
    }

    const uint8_t* vlast = sm + C::KV_BYTES + 7 * C::PITCH + (NJ - 1) * ROWB;   // V of the tile's last key
    if (flags & kLast) {
      const bool whole = kt0 == 0 && kt + 1 == head.w;
      const int rows = d.n * plan.group;
      const int row0 = d.rt * C::BR + warp * C::RPW;
      const int key = base + TK - 1;             // the key whose weight is still carried
      const long long slot_row = ((long long)worker * 2 + (in_first ? 0 : 1)) * C::BR + warp * C::RPW;
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        const int row = row0 + r8 + 8 * u;
        const float m2 = reference2<T>(m[u]);
        float w = __shfl_sync(0xffffffffu, carry_b[u], lane & ~3);
        const float ls = __shfl_sync(0xffffffffu, carry_s[u], lane & ~3);
        const float cap = key == pos[u] ? 0.5f * ex2_approx(fmaf(ls, kLog2e, -m2)) : 0.f;
        w += cap;
        float z = z2[u].x + z2[u].y + (c4 == 0 ? cap : 0.f);
        z += __shfl_xor_sync(0xffffffffu, z, 1);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        if (piece_bad) z = __int_as_float(0x7fffffff);
        if (row >= rows) continue;
        const bool seen = key <= pos[u];         // else the weight is 0, and V may hold anything
        const int t = row / plan.group;
        T* dst = (T*)a.o + ((size_t)(d.start + t) * a.H + (size_t)d.h * plan.group + (row - t * plan.group)) * a.D;
        float* po = part_o + (slot_row + r8 + 8 * u) * DP;
        const float inv = 1.f / z;
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          const int col = 8 * n + 2 * c4;
          float2 y = make_float2(o[n][2 * u], o[n][2 * u + 1]);
          if (RS == 1) {
            y.x += o[n][2];
            y.y += o[n][3];
          }
          if (seen) {
            const float2 v = unpack2<T>(*reinterpret_cast<const uint32_t*>(vlast + 4 * c4 + 16 * n));
            y.x = fmaf(w, v.x, y.x);
            y.y = fmaf(w, v.y, y.y);
          }
          if (whole) {
            // z = 0: the row sees no key
            if (col < a.D) *reinterpret_cast<uint32_t*>(dst + col) = z == 0.f ? 0u : pack2<T>(y.x * inv, y.y * inv);
          } else {
            *reinterpret_cast<float2*>(po + col) = y;
          }
        }
        if (!whole && c4 == 0) part_mz[slot_row + r8 + 8 * u] = make_float2(m[u], z);
      }
    } else {
      __syncwarp();
      if (lane < CH) *reinterpret_cast<uint4*>(my_halo_p + 16 * lane) = *reinterpret_cast<const uint4*>(vlast + 16 * lane);
    }
    __syncwarp();
    if (lane == 0) bar_arrive(empty + 8 * stage);
    if (++slot == C::RING) slot = 0;
    if (++stage == NST) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (after_chunks) pdl_wait();
}

}  // namespace

// ------------------------------------------------------------------ host side

namespace {

// The forms: decoding with 8 or 16 rows a warp, and chunks
template <int DP> using Decode8 = std::conditional_t<DP == 64, Config<64, 32, 8, 1, 8, 2, 184, 72>, Config<128, 32, 8, 1, 4, 2, 0, 0>>;
template <int DP> using Decode16 = std::conditional_t<DP == 64, Config<64, 32, 16, 1, 8, 2, 184, 72>, Config<128, 32, 16, 1, 4, 2, 0, 0>>;
template <int DP> using Chunk = Config<DP, DP == 64 ? 64 : 32, 16, 4, 3, 3, 152, 56>;

constexpr int kDecodeUnitCost = 2, kChunkUnitCost = 2;

template <typename T, typename C>
cudaError_t launch_main(const Args& a, Plan plan, const Pieces& pc, bool after_chunks) {
  static_assert(C::SMEM + (kMaxSeqs + 1) * (int)sizeof(unsigned) <= 232448, "shared memory of a block");
  const size_t smem = C::SMEM + (size_t)(a.seqs + 1) * sizeof(unsigned);
  cudaError_t e = cudaFuncSetAttribute(mma_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       C::SMEM + (kMaxSeqs + 1) * (int)sizeof(unsigned));
  if (e != cudaSuccess) return e;
  plan.unit_rows = a.D == C::DP && a.slot_stride == C::DP && a.page_size % C::NJ == 0 ? C::NJ : 1;
  return launch_pdl(mma_kernel<T, C>, dim3(num_sms_cached()), dim3(C::THREADS), smem, a.stream, a, plan, pc.o, pc.mz,
                    pc.meta, (int)after_chunks);
}

// 128-row units on tcgen05 (ca_paged_tc.cu) where the longest sequence fills more than half of one; else units of 64
// rows on mma.sync.  16 heads of 64, tcgen05 against mma.sync: 16 sequences of 64 rows over 4096 keys 173 and 139 us,
// of 80 rows 178 and 251; 1 of 128 rows over 16000 keys 77 and 81; 4 pieces of 256 rows over 512 keys 35 and 31.
// Heads of 128: 80 rows 270 and 372, 128 rows 99 and 116, 256 rows 43 and 47.
bool use_tc(long long rows) { return rows > 64; }

template <typename T, int DP>
cudaError_t forward_dp(const Args& a, void* workspace) {
  Plan plan = make_plan(a);
  char* ws = (char*)workspace;
  const long long rows = (long long)a.max_q_len * plan.group;
  plan.unit_cost = kDecodeUnitCost;
  if (rows <= 16) {
    // every sequence, whatever its rows: max_q_len may be wrong
    const Pieces pc = rows <= 8 ? carve<DP>(ws, Decode8<DP>::BR, Decode8<DP>::GROUPS) : carve<DP>(ws, Decode16<DP>::BR, Decode16<DP>::GROUPS);
    cudaError_t e = rows <= 8 ? launch_main<T, Decode8<DP>>(a, plan, pc, false)
                              : launch_main<T, Decode16<DP>>(a, plan, pc, false);
    return e != cudaSuccess ? e : launch_merge<T, DP>(a, plan, pc, Pieces{});
  }
  // sequences of up to 16 rows in the decoding form, the others as chunks
  Plan chunks = plan;
  chunks.min_places = 2;
  chunks.unit_cost = kChunkUnitCost;
  chunks.row_lo = 17;
  // (a single sequence is all in one form, whatever its rows)
  if (a.seqs == 1) chunks.row_lo = 0;
  const bool tall = use_tc(rows);
  const int br = tall ? tc_br() : Chunk<DP>::BR, groups = tall ? tc_groups(DP) : Chunk<DP>::GROUPS;
  Pieces pc = carve<DP>(ws, br, groups);
  cudaError_t e;
  if (!tall || !tc_launch(a, chunks, std::is_same_v<T, __nv_bfloat16> ? 1 : 2, pc, e)) {
    pc = carve<DP>(ws, Chunk<DP>::BR, Chunk<DP>::GROUPS);   // its units are the smaller ones
    e = launch_main<T, Chunk<DP>>(a, chunks, pc, false);
  }
  if (e != cudaSuccess) return e;
  if (a.seqs == 1) return launch_merge<T, DP>(a, plan, pc, Pieces{});
  plan.row_hi = 16;
  const Pieces few = carve<DP>(ws + pieces_bytes<DP>(br, groups), Decode16<DP>::BR, Decode16<DP>::GROUPS);
  e = launch_main<T, Decode16<DP>>(a, plan, few, true);
  return e != cudaSuccess ? e : launch_merge<T, DP>(a, plan, pc, few);
}

}  // namespace

size_t mma_workspace_bytes(long long max_q_len, long long H, long long G, long long D) {
  const long long rows = max_q_len * (H / G);
  auto bytes = [&](auto d8, auto d16, auto chunk) {
    using D8 = decltype(d8);
    using D16 = decltype(d16);
    using Ck = decltype(chunk);
    constexpr int DP = D8::DP;
    const size_t few = pieces_bytes<DP>(D16::BR, D16::GROUPS);
    return rows <= 8 ? pieces_bytes<DP>(D8::BR, D8::GROUPS)
                     : rows <= 16 ? few
                                  : few + (use_tc(rows) ? pieces_bytes<DP>(tc_br(), tc_groups(DP))
                                                            : pieces_bytes<DP>(Ck::BR, Ck::GROUPS));
  };
  return D <= 64 ? bytes(Decode8<64>{}, Decode16<64>{}, Chunk<64>{}) : bytes(Decode8<128>{}, Decode16<128>{}, Chunk<128>{});
}

cudaError_t mma_read_status(int* out, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
  if (e != cudaSuccess || !reset || *out == 0) return e;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
}

int mma_launches(const Args& a) {
  const long long rows = (long long)a.max_q_len * (a.H / a.G);
  return rows <= 16 || a.seqs == 1 ? 2 : 3;
}

cudaError_t mma_forward(const Args& a, int dtype, void* workspace) {
  if (a.D <= 64)
    return dtype == 1 ? forward_dp<__nv_bfloat16, 64>(a, workspace) : forward_dp<__half, 64>(a, workspace);
  return dtype == 1 ? forward_dp<__nv_bfloat16, 128>(a, workspace) : forward_dp<__half, 128>(a, workspace);
}

}  // namespace paged
}  // namespace ca
