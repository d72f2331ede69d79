// ca_paged_tc.cu -- Continuum Attention of chunks over a paged cache on tcgen05: bf16 and f16,
// units of 128 rows.
//
// Work is divided as in ca_paged_mma.cu (units, places, pieces, merge).  One block runs on an SM,
// with three workers (two where heads have more than 64 values) that share nothing but the tensor
// pipe: each has four math warps (a thread is a row, its TMEM lane), a warp that issues the products
// and a warp that loads.
//
// A worker's tensor memory: three regions of 32 columns and O in 64 or 128.  Tile t of 32 keys has its
// scores S = Q K^T in region t mod 3; its weights P overwrite them in place, each 16 keys as 8
// columns of hi pairs and 8 of lo pairs (two 16-bit parts, see ca_paged_mma.cu); then
// O += P_hi V + P_lo V with P as the A operand from tensor memory.  The products run in issue
// order, so S of tile t + 3 is issued behind P V of tile t into the same region, and the math
// warps find the next tiles' scores done.  O is rescaled in place, only when a row's maximum
// has grown by more than 8 nats.
//
// Columns: S column 16 c + 2 j + s is key 16 c + j + 8 s (K rows are gathered in that order),
// so a register pair of the score load is the pair (j, j + 8), whose left neighbours are the pair
// before it, and every step of the moments is one packed instruction for two keys.  P keeps
// the order, and V's rows are gathered in it, one key early (ca_paged_mma.cu: cutting keys).
// Being one thread's, a row needs no exchange between lanes at all.
//
// The loader brings rows by TMA, four rows of any page a copy (tile::gather4), in the 128-byte swizzle
// that the matrix descriptors name; the caches are maps of rows one common divisor of all strides
// apart, so any page size and any strides do, and a row that no key fills is one outside the map,
// zeros.  (One 16-byte cp.async per lane and a shuffled 64-bit address each took 2400 cycles a tile
// and 16000 for a unit's queries: prompts of 2 x 2048 tokens 155 us, with TMA 126.)
//
// What bounds it: the scalar work per score, 23.6 instructions with everything, of which the schedulers
// issue one in 55% of the cycles, with three math warps on each (counters at 511 rows over
// 16001 keys; tensor pipe 13% busy, transcendental pipe 35%, HBM 5%).  Without the moments that case
// takes 127 us, without moments and copies 91.  Tried and slower: two workers with tiles of 64 keys (205
// against 189 us at that case), tiles of 48 keys (189 against 170), four workers with 96 registers a thread
// (216) or with one warp for products and copies (220), one such warp for each of three workers (187
// against 179).
// Measured (16 heads of 64): prompts of 2 x 2048 tokens 115 us (mma.sync form 148), 511 rows over
// 16001 keys 173 us (235), 23 sequences of 0 .. 300 rows over up to 4000 keys, 4 query heads a key
// head, 84 us (102).  Heads of 128, with two workers and one unit's queries at a time: the first two 171 (226)
// and 262 us (352).
#include <cuda.h>

#include <numeric>

#include "ca_common.cuh"
#include "ca_paged.cuh"
#include "ca_paged_math.cuh"
#include "ca_sm100_ptx.cuh"

namespace ca {
namespace paged {

namespace {

using namespace sm100;

constexpr int TK = 32, BR = 128, NREG = 3, NST = 4, RING = NST + 1;

// head values padded to DP, in halves of 64 (128 bytes, a swizzled row)
template <int DP_>
struct Config {
  static constexpr int DP = DP_, HALVES = DP / 64;
  static constexpr int GROUPS = DP == 64 ? 3 : 2;
  static constexpr int MATH_WARPS = 4 * GROUPS, THREADS = (MATH_WARPS + 8) * 32;   // and a warpgroup of issuers, one of loaders
  // the moments of 16 pairs want 120 registers (112: 189 us at 511 rows over 16001 keys, 120: 180, 128: 179), which the
  // loaders and issuers give up
  static constexpr int REGS_MATH = DP == 64 ? 128 : 168, REGS_OTHER = DP == 64 ? 48 : 88;
  static_assert(GROUPS * REGS_MATH + 2 * REGS_OTHER <= THREADS / 128 * (65536 / THREADS / 8 * 8), "registers of the launch");
  static constexpr uint32_t COL_O = DP == 64 ? 96 : 128, COLS = COL_O + DP;   // a worker's columns: regions at 0, 32, 64
  static_assert(GROUPS * COLS <= 512, "tensor memory");
  static constexpr int QBUF = DP == 64 ? 2 : 1;       // units whose queries are held at once
  static constexpr uint32_t Q_HALF = BR * 128, Q_BYTES = HALVES * Q_HALF;
  static constexpr uint32_t KV_HALF = TK * 128, KV_BYTES = HALVES * KV_HALF;

  struct alignas(16) Slot {     // what a tile's readers need beside its stage
    int kt, flags, len, nt;     // tile in its unit, flags, keys of the sequence, tiles of the unit
    int start, n, h, rt;        // the sequence's rows; key head; row tile
    uint8_t k_before[2 * DP];   // K of the key before a piece
    uint8_t v_last[2 * DP];     // V of a piece's last key
  };

  struct alignas(1024) Group {
    uint8_t q[QBUF][Q_BYTES];
    uint8_t k[NST][KV_BYTES];
    uint8_t v[NST][KV_BYTES];
  };

  struct alignas(16) Control {
    uint64_t full[NST];         // a tile's rows and descriptor are there                 (1: the loader)
    uint64_t free_[NST];        // its products have read them                              (1: commit)
    uint64_t s_full[NREG];      // its scores are in tensor memory                          (1: commit)
    uint64_t p_ready[NREG];     // its weights are                                          (4: math warps)
    uint64_t pv_done[2];        // P V of tile t and all before it: barrier t & 1           (1: commit)
    uint64_t drained;           // every product                                            (1: commit)
    int gave_up;
    Slot ring[RING];
  };

  static constexpr size_t SMEM = GROUPS * (sizeof(Group) + sizeof(Control)) + 16;   // and the prefix sums behind it
};

enum : int { kFirst = 1, kLast = 2, kBad = 4, kEnd = 8, kNone = 16, kQ1 = 32 };   // kQ1: Q is in buffer 1

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// whether the phase has completed, at once (a try_wait may sleep for microseconds before it says no); whole warp
__device__ __forceinline__ bool mbar_test_warp(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, done != 0);
}
// a wait that no other warp's giving up ends; whole warp
__device__ __forceinline__ void mbar_drain_warp(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitNs) {}
  __syncwarp();
}
// the loader's wait for room: with no limit at all it gives up at once, so that a call can be made to; whole warp
__device__ __forceinline__ bool room_wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up,
                                               unsigned long long limit_ns) {
  if (limit_ns > 0) return mbar_wait_warp(bar, parity, gave_up, limit_ns);
  atomicCAS(&g_device_status, 0, 5);
  *gave_up = 1;
  return false;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// The caches and q as 2-D maps of rows: the strides' greatest common divisor apart, so that a row's number
// is a sum of products of small integers, whatever the strides.
struct Maps {
  CUtensorMap q, k, v;
  int q_box;                         // a unit's rows are those of whole tokens: q is a map of tokens and heads
  int q_token, q_head;               // else rows between tokens, heads
  int page, slot, head;              // rows between pages, slots, key heads
  long long unit;                    // values between a cache's rows
};

// ------------------------------------------------------------------ the loader

template <typename T, typename C>
__device__ __forceinline__ void load_warp(const Args& a, const Plan& plan, const Maps& maps,
                                          const Schedule<BR, TK>& sched, int worker, unsigned per, unsigned x0,
                                          unsigned x1, typename C::Group& gm, typename C::Control& ct,
                                          Meta* __restrict__ meta) {
  const int lane = threadIdx.x & 31;
  volatile int* ab = &ct.gave_up;
  if (lane == 0) meta[worker] = sched.none();
  typename Schedule<BR, TK>::Cursor cur;
  cur.at = x1;
  if (x0 < x1) cur = sched.locate(x0);
  if (cur.at >= x1) {              // no tile's place lies in this range
    if (lane == 0) {
      ct.ring[0].flags = kNone;
      mbar_arrive(&ct.full[0]);
    }
    return;
  }
  auto page_at = [&](int key) {                       // of this sequence, -1 beyond its keys
    return key < cur.len ? a.page_table[(size_t)cur.s * a.page_table_stride + plan.page_of(key)] : -1;
  };
  auto row_of = [&](int page, int key, int h) {       // of the maps
    return page * maps.page + (key - plan.page_of(key) * a.page_size) * maps.slot + h * maps.head;
  };
  // this lane's four rows of the stage: K and V, each half, eight lanes.  Row r is the key at
  // 16 (r / 16) + (r % 16) / 2 + 8 (r % 2): K of it, V of the key before it
  constexpr int KL = 8 * C::HALVES;
  const bool is_v = lane >= KL;
  const int half = C::HALVES == 1 ? 0 : (lane >> 3) & 1;
  const uint32_t dst = (is_v ? smem_u32(gm.v) : smem_u32(gm.k)) + half * C::KV_HALF + (lane & 7) * 512;
  const int p0 = ((lane & 4) << 2) + ((lane & 3) << 1);    // of its first row: + 0, 8, 1, 9 for the four
  const CUtensorMap* map = is_v ? &maps.v : &maps.k;
  const uint32_t row_bytes = a.D * sizeof(T);

  bool first = true, in_first = true;
  int kt0 = 0, qbuf = C::QBUF - 1;
  int last_tile[2] = {-1, -1};   // the last tiles of the unit before this one and of that before it
  int before = -1;               // the row of the key before the tile (-1: none)
  int pg = page_at(cur.kt * TK + lane);
  int pg_before = cur.kt > 0 ? page_at(cur.kt * TK - 1) : -1;
  bool end = false;
  int t = 0;
  for (; !end; ++t) {
    const int st = t % NST;
    if (t >= NST && !room_wait_warp(&ct.free_[st], (t / NST - 1) & 1, ab, plan.wait_ns)) break;
    const int base = cur.kt * TK;
    const bool opens = first || cur.kt == 0;
    int flags = cur.bad ? kBad : 0;
    typename C::Slot& slot = ct.ring[t % RING];
    const uint32_t bar = smem_u32(&ct.full[st]);
    uint32_t bytes = 2 * C::KV_BYTES;
    const int key = base + lane;
    bool bad = key < cur.len && (pg < 0 || pg >= a.num_pages);
    const int row = key < cur.len && !bad ? row_of(pg, key, cur.h) : -1;
    if (opens) {
      flags |= kFirst;
      kt0 = cur.kt;
      in_first = first;
      first = false;
      if (C::QBUF == 2) qbuf ^= 1;
      // Q of an earlier unit lay in this buffer: its products have to be done (they are known to be where the
      // stage of its last tile has been filled again since)
      const int u = last_tile[C::QBUF - 1];
      if (u >= 0 && u + NST > t && !room_wait_warp(&ct.free_[u % NST], (u / NST) & 1, ab, plan.wait_ns)) break;
      bytes += C::Q_BYTES;
      before = -1;
      if (base > 0 && base - 1 < cur.len) {
        if (pg_before < 0 || pg_before >= a.num_pages) bad = true;
        else before = row_of(pg_before, base - 1, cur.h);
      }
      if (before >= 0) bytes += row_bytes;
    }
    if (qbuf) flags |= kQ1;
    bad = __any_sync(0xffffffffu, bad);
    if (bad) flags |= kBad;
    const int behind = __shfl_sync(0xffffffffu, row, 31);
    const unsigned at = cur.at;
    bool more = at + 1 < x1;
    if (!more || cur.kt + 1 == cur.nt) {
      flags |= kLast;
      last_tile[1] = last_tile[0];
      last_tile[0] = t;
      if (behind >= 0) bytes += row_bytes;
    }
    const int kt = cur.kt, nt = cur.nt, start = cur.start, n = cur.n, len = cur.len, h = cur.h, rt = cur.rt;
    if (more) {
      sched.advance(cur);
      more = cur.at < x1;        // the next unit's first tile may lie behind the range
    }
    if (more) {
      pg = page_at(cur.kt * TK + lane);
      pg_before = -1;            // a unit that is entered here starts at key 0
    } else {
      flags |= kEnd;
      end = true;
    }
    if (lane == 0) {
      if (bad) record_invalid();
      int4* to = reinterpret_cast<int4*>(&slot);
      to[0] = make_int4(kt, flags, len, nt);
      to[1] = make_int4(start, n, h, rt);
      if (end) {
        // this worker joins the unit that starts in its range and goes on behind it
        Meta mt;
        mt.pieces = kt0 == 0 && kt + 1 < nt ? 1 + (int)((at + (nt - 1 - kt)) / per) - worker : 0;
        mt.slot = in_first ? 0 : 1;
        mt.start = start;
        mt.rows = n * plan.group;
        mt.h = h;
        mt.rt = rt;
        meta[worker] = mt;
      }
    }
    mbar_arrive_expect_tx(&ct.full[st], bytes);
    __syncwarp();
    int r[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int p = p0 + (x >> 1) + 8 * (x & 1) - (is_v ? 1 : 0);
      r[x] = __shfl_sync(0xffffffffu, row, p & 31);
      if (p < 0) r[x] = before;
    }
    if (lane < 2 * KL) tma_gather4(dst + st * C::KV_BYTES, map, bar, 64 * half, r[0], r[1], r[2], r[3]);
    if (opens) {
      const int rows = n * plan.group;
      if (maps.q_box) {
        // (rows behind the sequence's last are another's or zeros: nothing of theirs is kept)
#pragma unroll
        for (int x = 0; x < C::HALVES; ++x)
          tma_load_3d(gm.q[qbuf] + x * C::Q_HALF, &maps.q, &ct.full[st], 64 * x, h * plan.group,
                      start + rt * maps.q_box);
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = rt * BR + 4 * lane + x, tk = i / plan.group;
          r[x] = i < rows ? (start + tk) * maps.q_token + (h * plan.group + i - tk * plan.group) * maps.q_head : -1;
        }
#pragma unroll
        for (int x = 0; x < C::HALVES; ++x)
          tma_gather4(smem_u32(gm.q[qbuf]) + x * C::Q_HALF + lane * 512, &maps.q, bar, 64 * x, r[0], r[1], r[2], r[3]);
      }
      if (lane == 0 && before >= 0)
        bulk_load(smem_u32(slot.k_before), (const T*)a.k_cache + before * maps.unit, row_bytes, bar);
    }
    if (lane == 0 && (flags & kLast) && behind >= 0)
      bulk_load(smem_u32(slot.v_last), (const T*)a.v_cache + behind * maps.unit, row_bytes, bar);
    before = behind;
  }
  // every copy has to land before this block's shared memory is another's
  for (int u = max(t - NST, 0); u < t; ++u) mbar_drain_warp(&ct.full[u % NST], (u / NST) & 1);
}

// ------------------------------------------------------------------ the issuer

template <bool kBF16, typename C>
__device__ __forceinline__ void issue_warp(const Plan& plan, typename C::Group& gm, typename C::Control& ct, uint32_t tmem) {
  volatile int* ab = &ct.gave_up;
  const uint32_t id_s = make_idesc(BR, TK, kBF16, false), id_o = make_idesc(BR, 64, kBF16, true);
  const uint32_t q0 = smem_u32(gm.q), k0 = smem_u32(gm.k), v0 = smem_u32(gm.v);
  int issued = 0;
  bool more = true, good = true;
  // S of tile `issued` into its region; its rows are there
  auto issue_s = [&]() {
    const int st = issued % NST, flags = ct.ring[issued % RING].flags;
    if (flags & kNone) {
      more = false;
      return;
    }
    more = !(flags & kEnd);
    const uint64_t qd = sdesc_sw128(q0 + (flags & kQ1 ? C::Q_BYTES : 0), 16, 1024);
    const uint64_t kd = sdesc_sw128(k0 + st * C::KV_BYTES, 16, 1024);
    tc_fence_after();
#pragma unroll
    for (int kk = 0; kk < 4 * C::HALVES; ++kk)
      mma_ss(tmem + TK * (issued % NREG), qd + (kk >> 2) * (C::Q_HALF >> 4) + 2 * (kk & 3),
             kd + (kk >> 2) * (C::KV_HALF >> 4) + 2 * (kk & 3), id_s, kk > 0 ? 1u : 0u);
    mma_commit(&ct.s_full[issued % NREG]);
    ++issued;
  };
  // scores up to three tiles ahead of the weights, as far as rows are there.  Only where no weights are
  // awaited may this wait for them: the loader itself waits for a unit's last products before it
  // overwrites its Q, and with units of one tile those are the next that this warp issues.
  auto scores = [&](int upto, int awaited) {
    while (more && good && issued < upto) {
      uint64_t* bar = &ct.full[issued % NST];
      const uint32_t parity = (issued / NST) & 1;
      if (!mbar_test_warp(bar, parity)) {
        if (issued > awaited) return;
        good = mbar_wait_warp(bar, parity, ab, plan.wait_ns);
        if (!good) return;
      }
      issue_s();
    }
  };
  scores(NREG, 0);
  for (int t = 0; good && t < issued; ++t) {
    good = mbar_wait_warp(&ct.p_ready[t % NREG], (t / NREG) & 1, ab, plan.wait_ns);
    if (!good) break;
    const int st = t % NST;
    const bool first = ct.ring[t % RING].flags & kFirst;
    const uint64_t vd = sdesc_sw128(v0 + st * C::KV_BYTES, 16384, 1024);
    const uint32_t p = tmem + TK * (t % NREG);
    tc_fence_after();
#pragma unroll
    for (int x = 0; x < C::HALVES; ++x)
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int kk = 0; kk < TK / 16; ++kk)
          mma_ts(tmem + C::COL_O + 64 * x, p + 16 * kk + 8 * part, vd + x * (C::KV_HALF >> 4) + 128 * kk, id_o,
                 first && part == 0 && kk == 0 ? 0u : 1u);
    mma_commit(&ct.pv_done[t & 1]);
    mma_commit(&ct.free_[st]);
    scores(t + 1 + NREG, t + 1);
  }
  if (issued > 0) {
    // products may still be running where a wait gave up, the math warps' or this one's: they end before tensor
    // memory is given back
    mma_commit(&ct.drained);
    mbar_drain_warp(&ct.drained, 0);
  }
}

// ------------------------------------------------------------------ the math warps

template <typename T, typename C>
__device__ __forceinline__ void math_warp(const Args& a, const Plan& plan, int worker, typename C::Group& gm,
                                          typename C::Control& ct, uint32_t tmem, float* __restrict__ part_o, float2* __restrict__ part_mz) {
  volatile int* ab = &ct.gave_up;
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, r = warp * 32 + lane;
  const uint32_t lanes = (uint32_t)(warp * 32) << 16, t_o = tmem + C::COL_O + lanes;
  float m = -INFINITY, carry_s = kMasked, carry_b = 0.f, scale = 0.f;
  float2 z2 = splat2(0.f);
  int pos = -1, i_min = 0, i_max = -1, kt0 = 0, bad = 0;
  bool in_first = true, first_tile = true;
  for (int t = 0;; ++t) {
    if (!mbar_wait_warp(&ct.full[t % NST], (t / NST) & 1, ab, plan.wait_ns)) return;
    const typename C::Slot& d = ct.ring[t % RING];
    const int4 head = *reinterpret_cast<const int4*>(&d);
    const int kt = head.x, flags = head.y, base = kt * TK;
    if (flags & kNone) return;
    if (flags & kFirst) {
      kt0 = kt;
      bad = 0;
      in_first = first_tile;
      first_tile = false;
      const int rows = d.n * plan.group, row0 = d.rt * BR + warp * 32, lead = head.z - d.n;
      const int row_last = min(rows, row0 + 32) - 1;          // < row0: the warp has no row
      i_min = lead + row0 / plan.group;
      i_max = row_last >= row0 ? lead + row_last / plan.group : -1;
      const int row = max(min(row0 + lane, row_last), 0);
      const int tk = row / plan.group;
      pos = lead + tk;
      scale = expf(a.log_gain[d.h * plan.group + row - tk * plan.group]) * a.inv_sqrt_d;
      m = -INFINITY;
      z2 = splat2(0.f);
      carry_s = kMasked;
      carry_b = 0.f;
      if (kt > 0 && base - 1 <= i_max) {
        // the score of the key before the piece, this row's
        const uint8_t* q = gm.q[flags & kQ1 ? 1 : 0] + r * 128;
        float2 s = splat2(0.f);
#pragma unroll
        for (int c = 0; c < C::DP / 8; ++c) {
          const uint4 x = *reinterpret_cast<const uint4*>(q + (c >> 3) * C::Q_HALF + (((c & 7) ^ (r & 7)) << 4));
          const uint4 y = *reinterpret_cast<const uint4*>(d.k_before + 16 * c);
          s = fma2(unpack2<T>(x.x), unpack2<T>(y.x), s);
          s = fma2(unpack2<T>(x.y), unpack2<T>(y.y), s);
          s = fma2(unpack2<T>(x.z), unpack2<T>(y.z), s);
          s = fma2(unpack2<T>(x.w), unpack2<T>(y.w), s);
        }
        if (base - 1 <= pos) m = carry_s = (s.x + s.y) * scale;
      }
    }
    bad |= flags & kBad;
    if (!mbar_wait_warp(&ct.s_full[t % NREG], (t / NREG) & 1, ab, plan.wait_ns)) return;
    tc_fence_after();
    const uint32_t t_s = tmem + TK * (t % NREG) + lanes;
    if (base - 1 <= i_max && i_max >= 0) {
      uint32_t raw[32];
      tmem_ld32(t_s, raw);
      tmem_ld_wait();
      tmem_reg_fence(raw);
      float2 s[2][8];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        s[j >> 3][j & 7] = mul2(make_float2(__uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1])), splat2(scale));
      const bool edge = base == 0 || base + TK - 1 > i_min;     // keys beyond a row's own, or caps
      if (edge) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = base + 16 * (j >> 3) + (j & 7);
          if (key > pos) s[j >> 3][j & 7].x = kMasked;
          if (key + 8 > pos) s[j >> 3][j & 7].y = kMasked;
        }
      }
      float top = max3f(s[0][0].x, s[0][0].y, s[0][1].x);
      top = fmaxf(top, s[0][1].y);
#pragma unroll
      for (int j = 2; j < 16; ++j) top = max3f(top, s[j >> 3][j & 7].x, s[j >> 3][j & 7].y);
      const bool move = top > kMasked && top > m + kRescaleNats;
      if (__any_sync(0xffffffffu, move)) {
        const float to = move ? top : m, f = move ? exp_rel(m - to) : 1.f;
        m = to;
        carry_b *= f;
        z2 = mul2(z2, splat2(f));
        if (!(flags & kFirst)) {
          // O holds P V of the piece's tiles so far: the last of them has to have landed.  Its barrier is
          // neither a phase further on (that needs P of tile t + 1) nor behind (P V of tile t - 3
          // completed before the scores of tile t)
          if (!mbar_wait_warp(&ct.pv_done[(t - 1) & 1], ((t - 1) >> 1) & 1, ab, plan.wait_ns)) return;
          tc_fence_after();
#pragma unroll
          for (int half = 0; half < C::DP / 32; ++half) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * half, o);
            tmem_ld_wait();
            tmem_reg_fence(o);
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tmem_st32(t_o + 32 * half, o);
          }
          tmem_st_wait();
        }
      }
      const float m2 = reference2<T>(m);
      const int lowest = flags & kFirst ? base : base - 1;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t hi[8], lo[8];
        float2 lead;
        float last;
        weigh<T, 8>(s[c], m2, carry_s, edge, base + 16 * c, pos, lowest, hi, lo, lead, last, z2);
        lead.x += carry_b;
        split2<T>(lead, hi[0], lo[0]);
        carry_s = s[c][7].y;
        carry_b = last;
        tmem_st8(t_s + 16 * c, hi);
        tmem_st8(t_s + 16 * c + 8, lo);
      }
    } else if (i_max >= 0) {
      // no row of this warp sees a segment or a weight here
      uint32_t zero[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st8(t_s + 8 * c, zero);
    }
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive_warp(&ct.p_ready[t % NREG]);

    if (flags & kLast) {
      // (P V of tile t - 1 first: only then can this tile's phase be told from the one before)
      if (t > 0 && !mbar_wait_warp(&ct.pv_done[(t - 1) & 1], ((t - 1) >> 1) & 1, ab, plan.wait_ns)) return;
      if (!mbar_wait_warp(&ct.pv_done[t & 1], (t >> 1) & 1, ab, plan.wait_ns)) return;
      tc_fence_after();
      const int rows = d.n * plan.group, row = d.rt * BR + r;
      const bool whole = kt0 == 0 && kt + 1 == head.w;
      const int key = base + TK - 1;                      // the key whose weight is still carried
      const float m2 = reference2<T>(m);
      const float cap = key == pos ? 0.5f * ex2_approx(fmaf(carry_s, kLog2e, -m2)) : 0.f;
      // beyond the row's own key the weight is 0, and V may hold anything
      const float w = key <= pos ? carry_b + cap : 0.f;
      float z = z2.x + z2.y + cap;
      if (bad) z = __int_as_float(0x7fffffff);
      const float inv = 1.f / z;
      const long long prow = ((long long)worker * 2 + (in_first ? 0 : 1)) * BR + r;
      const int tk = row / plan.group;
      T* dst = (T*)a.o + ((size_t)(d.start + tk) * a.H + (size_t)d.h * plan.group + (row - tk * plan.group)) * a.D;
      // 64 columns at a time
#pragma unroll
      for (int half = 0; half < C::HALVES; ++half) {
        uint32_t o[2][32];
        tmem_ld32(t_o + 64 * half, o[0]);
        tmem_ld32(t_o + 64 * half + 32, o[1]);
        tmem_ld_wait();
        tmem_reg_fence(o[0]);
        tmem_reg_fence(o[1]);
        if (row < rows) {
#pragma unroll
          for (int c8 = 0; c8 < 8; ++c8) {
            const int c = 8 * half + c8;
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = __uint_as_float(o[(8 * c8 + x) >> 5][(8 * c8 + x) & 31]);
            if (w != 0.f) {
              const uint4 v = *reinterpret_cast<const uint4*>(d.v_last + 16 * c);
              const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 vv = unpack2<T>(vw[x]);
                y[2 * x] = fmaf(w, vv.x, y[2 * x]);
                y[2 * x + 1] = fmaf(w, vv.y, y[2 * x + 1]);
              }
            }
            if (!whole) {
              *reinterpret_cast<float4*>(part_o + prow * C::DP + 8 * c) = make_float4(y[0], y[1], y[2], y[3]);
              *reinterpret_cast<float4*>(part_o + prow * C::DP + 8 * c + 4) = make_float4(y[4], y[5], y[6], y[7]);
            } else if (8 * c < a.D) {
              // z = 0: the row sees no key
              const bool none = z == 0.f;
              *reinterpret_cast<uint4*>(dst + 8 * c) =
                  none ? make_uint4(0u, 0u, 0u, 0u)
                       : make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv),
                                    pack2<T>(y[4] * inv, y[5] * inv), pack2<T>(y[6] * inv, y[7] * inv));
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (!whole && row < rows) part_mz[prow] = make_float2(m, z);
      __syncwarp();
    }
    if (flags & kEnd) return;
  }
}

// ------------------------------------------------------------------ the kernel

template <typename T, typename C>
__global__ void __launch_bounds__(C::THREADS, 1)
    tc_kernel(const __grid_constant__ Args a, const __grid_constant__ Plan plan, const __grid_constant__ Maps maps,
              float* __restrict__ part_o, float2* __restrict__ part_mz, Meta* __restrict__ meta) {
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  using Group = typename C::Group;
  using Control = typename C::Control;
  constexpr int GROUPS = C::GROUPS, MATH_WARPS = C::MATH_WARPS;
  Group* groups = reinterpret_cast<Group*>(smem);
  Control* controls = reinterpret_cast<Control*>(smem + GROUPS * sizeof(Group));
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(smem + GROUPS * (sizeof(Group) + sizeof(Control)));
  unsigned* prefix = reinterpret_cast<unsigned*>(smem + C::SMEM);
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int role = wid < MATH_WARPS ? 0 : wid < MATH_WARPS + 4 ? 1 : 2;
  const int group = role == 0 ? wid >> 2 : wid & 3;

  if (role == 2 && group < GROUPS) {
    // values behind D stay 0 (copies write D values a row)
    Control& ct = controls[group];
    constexpr int CH = C::DP / 8;
    for (int x = lane; x < RING * CH; x += 32) {
      reinterpret_cast<uint4*>(ct.ring[x / CH].k_before)[x % CH] = make_uint4(0u, 0u, 0u, 0u);
      reinterpret_cast<uint4*>(ct.ring[x / CH].v_last)[x % CH] = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  if (role == 2 && group < GROUPS && lane == 0) {
    Control& ct = controls[group];
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
    for (int i = 0; i < NST; ++i) {
      mbar_init(&ct.full[i], 1);
      mbar_init(&ct.free_[i], 1);
    }
    for (int i = 0; i < NREG; ++i) {
      mbar_init(&ct.s_full[i], 1);
      mbar_init(&ct.p_ready[i], 4);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&ct.pv_done[i], 1);
    mbar_init(&ct.drained, 1);
    ct.gave_up = 0;
    fence_mbar_init();
  }
  if (role == 1 && group == 3) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  Schedule<BR, TK> sched(a, plan, prefix);   // a barrier of the block among other things
  tc_fence_after();
  const uint32_t tmem = *tmem_at + C::COLS * (group < GROUPS ? group : 0);
  const unsigned total = sched.total;
  const int worker = blockIdx.x * GROUPS + group, workers = gridDim.x * GROUPS;
  const unsigned per = plan.places_per_worker(total, workers);

  if (role == 0) {
    regs_up<C::REGS_MATH>();
    math_warp<T, C>(a, plan, worker, groups[group], controls[group], tmem, part_o, part_mz);
  } else {
    regs_down<C::REGS_OTHER>();
    if (group < GROUPS) {
      if (role == 1) {
        issue_warp<std::is_same<T, __nv_bfloat16>::value, C>(plan, groups[group], controls[group], tmem);
      } else {
        const unsigned x0 = (unsigned)min((unsigned long long)worker * per, (unsigned long long)total);
        const unsigned x1 = (unsigned)min((unsigned long long)x0 + per, (unsigned long long)total);
        load_warp<T, C>(a, plan, maps, sched, worker, per, x0, x1, groups[group], controls[group], meta);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (role == 1 && group == 3) {
    tc_fence_after();
    tmem_dealloc(*tmem_at, 512);
  }
}

}  // namespace

int tc_br() { return BR; }
int tc_groups(int dp) { return dp == 64 ? Config<64>::GROUPS : Config<128>::GROUPS; }

namespace {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  }
  return fn;
}

struct Axis {
  long long count, stride;
};

// a map of rows of D values over the places that the axes reach, and how many rows a step along each is;
// false where the rows are too many for a coordinate
template <int N>
bool make_rows(CUtensorMap* map, const void* base, long long D, bool bf16, const Axis (&axes)[N], int* const (&step)[N],
               long long* unit) {
  long long g = 0, rows = 1;
  for (const Axis& x : axes) g = x.count > 1 ? std::gcd(g, x.stride) : g;
  if (g == 0) g = D;
  for (int i = 0; i < N; ++i) {
    const long long s = axes[i].count > 1 ? axes[i].stride / g : 0;
    if (s > 0x7fffffffll) return false;
    *step[i] = (int)s;
    rows += (axes[i].count - 1) * s;           // (counts are below 2^31)
    if (rows > 0x7fffffffll) return false;
  }
  *unit = g;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows}, pitch[1] = {(cuuint64_t)(g * 2)};
  const cuuint32_t box[2] = {64, 1}, one[2] = {1, 1};
  return encode_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                     const_cast<void*>(base), dims, pitch, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_maps(const Args& a, bool bf16, Maps& m) {
  if (!encode_fn() || a.num_pages < 1 || a.rows < 1) return false;
  // a unit's rows are one box where it has whole tokens, else 32 copies of four (a prompt of 400 tokens: 27 or 29 us)
  m.q_box = BR % (a.H / a.G) == 0 ? BR / (a.H / a.G) : 0;
  if (m.q_box) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.rows};
    const cuuint64_t pitch[2] = {(cuuint64_t)(a.q_head_stride * 2), (cuuint64_t)(a.q_token_stride * 2)};
    const cuuint32_t box[3] = {64, (cuuint32_t)(a.H / a.G), (cuuint32_t)m.q_box}, one[3] = {1, 1, 1};
    if (encode_fn()(&m.q, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                    const_cast<void*>(a.q), dims, pitch, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      m.q_box = 0;
  }
  long long q_unit;
  return (m.q_box || make_rows(&m.q, a.q, a.D, bf16, {Axis{a.rows, a.q_token_stride}, {a.H, a.q_head_stride}},
                   {&m.q_token, &m.q_head}, &q_unit)) &&
         make_rows(&m.k, a.k_cache, a.D, bf16, {Axis{a.num_pages, a.page_stride}, {a.page_size, a.slot_stride}, {a.G, a.head_stride}},
                   {&m.page, &m.slot, &m.head}, &m.unit) &&
         make_rows(&m.v, a.v_cache, a.D, bf16, {Axis{a.num_pages, a.page_stride}, {a.page_size, a.slot_stride}, {a.G, a.head_stride}},
                   {&m.page, &m.slot, &m.head}, &m.unit);
}

template <typename T, typename C>
cudaError_t launch(const Args& a, const Plan& plan, const Maps& maps, const Pieces& pc) {
  static_assert(C::SMEM + (kMaxSeqs + 1) * sizeof(unsigned) <= 232448, "shared memory of a block");
  const cudaError_t e = cudaFuncSetAttribute(tc_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(C::SMEM + (kMaxSeqs + 1) * sizeof(unsigned)));
  if (e != cudaSuccess) return e;
  const size_t smem = C::SMEM + (size_t)(a.seqs + 1) * sizeof(unsigned);
  return launch_pdl(tc_kernel<T, C>, dim3(num_sms_cached()), dim3(C::THREADS), smem, a.stream, a, plan, maps, pc.o,
                    pc.mz, pc.meta);
}

}  // namespace

bool tc_launch(const Args& a, const Plan& plan, int dtype, const Pieces& pc, cudaError_t& e) {
  // a thread that has made no runtime call yet has no context, which the encoder asks for
  int dev;
  e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e != cudaSuccess) return true;
  Maps maps;
  if (!make_maps(a, dtype == 1, maps)) return false;
  if (a.D <= 64) e = dtype == 1 ? launch<__nv_bfloat16, Config<64>>(a, plan, maps, pc) : launch<__half, Config<64>>(a, plan, maps, pc);
  else e = dtype == 1 ? launch<__nv_bfloat16, Config<128>>(a, plan, maps, pc) : launch<__half, Config<128>>(a, plan, maps, pc);
  return true;
}

cudaError_t tc_read_status(int* out, bool reset) {
  int word[2] = {0, 0};
  cudaError_t e = cudaMemcpyFromSymbol(&word[0], g_status, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&word[1], sm100::g_device_status, sizeof(int));
  if (e != cudaSuccess) return e;
  *out = word[1] ? word[1] : word[0];
  if (!reset || *out == 0) return e;
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
  return e != cudaSuccess ? e : cudaMemcpyToSymbol(sm100::g_device_status, &zero, sizeof(int));
}

}  // namespace paged
}  // namespace ca
