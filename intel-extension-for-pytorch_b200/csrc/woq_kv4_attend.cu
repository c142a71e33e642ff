// Attention of a few query rows a sequence over the paged 4-bit cache (layout: woq_kv4_common.cuh):
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys j that the row sees, in one pass over the cache.
//
// The work is one long sequence of units, 32 keys of one (sequence, kv head, tile of query rows) each, dealt to the
// CTAs in equal shares whatever the lengths; the warps of a CTA take its units in turn.  A warp computes S^T = K Q^T
// and O^T += V^T P^T, so that up to eight query rows (the heads of a kv head, times tokens) fill the n side of
// m16n8k16 and dequantised codes are A fragments as they come from the cache.  P^T is S^T transposed in registers
// (movmatrix).  A running reference of the maximum is raised only when a score passes it by 8 (log2): P is at most 256.
// When a tile of rows ends, the warps' sums are joined in shared memory; a tile that several CTAs share is joined
// through the workspace by the last one, in the order of the keys, so that results do not depend on who is last.
#include <algorithm>

#include "woq_kernels.h"
#include "woq_kv4_common.cuh"
#include "woq_kv4_dequant.cuh"

namespace woq {

namespace {

// Seven warps compute and one loads: sixteen an SM may have 128 registers each, eighteen only 96.
constexpr int kWarps = 7;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kJoinBar = 1;
constexpr int kMaxCtas = 512;
constexpr int kUnitKeys = 32;  // keys of a unit: two blocks

// What an item costs beside its units (queries, joining the warps), in units: 222 units over 32 short sequences took
// three times as long as over two long ones.
constexpr int kItemCost = 24;

// Two CTAs an SM where the registers allow it (their accumulators are D x 8 NT / 32 a lane), and as many ring slots as
// fit: one SM then has up to 150 KB of copies in flight.
constexpr int ctas_per_sm(int d, int nt) { return nt * d <= 128 ? 2 : 1; }
template <int D, int G, int NT>
struct Smem {
  static constexpr int kCtas = ctas_per_sm(D, NT), kBlock = kv4_block_bytes(D, G);
  static constexpr size_t kBudget = kCtas == 2 ? 112 * 1024 : 226 * 1024;
  static constexpr size_t join = 0;                              // [kWarps][kJoinD][8] sums of the values
  static constexpr int kJoinD = kCtas == 2 || D == 64 ? 64 : 128;
  static_assert(D % kJoinD == 0, "whole slices");
  static constexpr size_t kJoinBytes = kWarps * kJoinD * 8 * 4;
  static constexpr size_t query = join + kJoinBytes;             // [8 NT][D] of T, where registers do not hold them
  static constexpr bool kQInRegs = NT * D <= 128;
  static constexpr size_t stats = query + (kQInRegs ? 0 : 8 * NT * D * 2);  // [kWarps][8 NT]{max, sum}
  static constexpr size_t totals = stats + kWarps * 8 * NT * 8;  // [8 NT]{max, sum}
  static constexpr size_t full = totals + 8 * NT * 8;            // [kWarps][kRing] barriers: the slot holds its block
  static constexpr size_t empty = full + kWarps * 8 * 8;         // the warp has read it
  static constexpr size_t left_out = empty + kWarps * 8 * 8;     // words: nothing was loaded
  static constexpr size_t ring = left_out + kWarps * 8 * 4;
  static constexpr int kFit = static_cast<int>((kBudget - ring) / (kWarps * kBlock)), kRing = kFit >= 8 ? 8 : kFit / 2 * 2;
  static constexpr size_t total = ring + static_cast<size_t>(kWarps) * kRing * kBlock;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Where a unit is: sequence b, kv head h, tile r of its query rows, unit blk of the item.  All lanes hold the same.
struct Cursor {
  int b, h, r, blk;
  int blocks, tiles;  // units of an item and tiles of the sequence
  int q0, rows_tok;   // first query row, number of them
  int len;
  int load;           // blocks of 16 keys that some row of the tile sees
};

template <int ROWS>
__device__ __forceinline__ void load_sequence(const Kv4AttendParams& p, Cursor& c) {
  int len = p.lens[c.b];
  len = min(max(len, 0), p.max_blocks * kKv4Tokens);
  c.len = len;
  c.blocks = max(1, (len + kUnitKeys - 1) / kUnitKeys);
  if (p.starts) {
    const int s0 = min(max(p.starts[c.b], 0), p.tokens), s1 = min(max(p.starts[c.b + 1], s0), p.tokens);
    c.q0 = s0;
    c.rows_tok = s1 - s0;
  } else {
    c.q0 = c.b;
    c.rows_tok = 1;
  }
  c.tiles = (c.rows_tok * p.heads + ROWS - 1) / ROWS;
}
// {items, units of an item}
template <int ROWS>
__device__ __forceinline__ int2 sequence_items(const Kv4AttendParams& p, int b) {
  if (b >= p.batch) return make_int2(0, 0);
  Cursor c;
  c.b = b;
  load_sequence<ROWS>(p, c);
  return make_int2(c.tiles * p.kv_heads, c.blocks);
}
template <int ROWS>
__device__ __forceinline__ void enter_item(const Kv4AttendParams& p, Cursor& c) {
  int limit = c.len;  // keys that the last row of the tile sees
  if (p.causal && p.starts) limit += (min(c.rows_tok * p.heads, (c.r + 1) * ROWS) - 1) / p.heads + 1 - c.rows_tok;
  c.load = max(0, limit + kKv4Tokens - 1) / kKv4Tokens;
}
// `steps` units on; the caller stays within the units there are
template <int ROWS>
__device__ __forceinline__ void advance(const Kv4AttendParams& p, Cursor& c, int steps) {
  c.blk += steps;
  if (c.blk < c.blocks) return;
  do {
    c.blk -= c.blocks;
    if (++c.r < c.tiles) continue;
    c.r = 0;
    if (++c.h < p.kv_heads) continue;
    c.h = 0;
    do {
      if (++c.b >= p.batch) return;  // past the last unit
      load_sequence<ROWS>(p, c);
    } while (c.tiles == 0);
  } while (c.blk >= c.blocks);
  enter_item<ROWS>(p, c);
}

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, NT)) kv4_attend_kernel(const __grid_constant__ Kv4AttendParams p) {
  using S = Smem<D, G, NT>;
  constexpr int kRows = 8 * NT, kRing = S::kRing, kBlock = S::kBlock, W = kv4_width(D), nw = W / 32, kHalves = D / W;
  constexpr int ng = D / G, kGroups = ng / kHalves, kWordsPerGroup = G / 32, kMt = D / 16;
  constexpr bool kQInRegs = S::kQInRegs;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_share, s_item;  // share of a CTA; where the first item begins (both with kItemCost an item)
  __shared__ int s_b, s_in_b, s_units, s_last;
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::full);
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem + S::empty);
  volatile uint32_t* left_out = reinterpret_cast<volatile uint32_t*>(smem + S::left_out);
  uint8_t* ring = smem + S::ring;
  float* join = reinterpret_cast<float*>(smem + S::join);
  float2* stats = reinterpret_cast<float2*>(smem + S::stats);
  float2* totals = reinterpret_cast<float2*>(smem + S::totals);
  uint16_t* qs = reinterpret_cast<uint16_t*>(smem + S::query);

  if (threadIdx.x < kWarps * kRing) {
    mbar_init(full + threadIdx.x, 1);
    mbar_init(empty + threadIdx.x, 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) s_abort = 0;
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- this CTA's share: [begin, end) of all items' units, every item preceded by kItemCost that nobody computes ----
  if (warp == 0) {
    const int2 chunk0 = sequence_items<kRows>(p, lane);
    auto chunk = [&](int b0) { return b0 == 0 ? chunk0 : sequence_items<kRows>(p, b0 + lane); };
    int64_t total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      const int2 c = chunk(b0);
      int64_t u = static_cast<int64_t>(c.x) * (c.y + kItemCost);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      total += u;
    }
    const int64_t share = max(int64_t(kWarps), (total + gridDim.x - 1) / gridDim.x);
    const int64_t begin = share * blockIdx.x, end = min(total, begin + share);
    int64_t units = 0;
    if (begin < total) {
      int64_t before = 0, before_units = 0, first_unit = 0;  // of the sequences before b0
      bool first = false;
      for (int b0 = 0;; b0 += 32) {
        const int2 c = chunk(b0);
        const int64_t cost = static_cast<int64_t>(c.x) * (c.y + kItemCost), u = static_cast<int64_t>(c.x) * c.y;
        int64_t cost_end = cost, u_end = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, cost_end, o), y = __shfl_up_sync(0xffffffffu, u_end, o);
          if (lane >= o) {
            cost_end += x;
            u_end += y;
          }
        }
        // units before a place in the lane's sequence
        const int64_t start = before + cost_end - cost, start_units = before_units + u_end - u;
        const int length = c.y + kItemCost;
        auto units_before = [&](int64_t place) {
          const int64_t item = (place - start) / length;
          return start_units + item * c.y + max(int64_t(0), place - start - item * length - kItemCost);
        };
        if (!first) {
          const uint32_t hit = __ballot_sync(0xffffffffu, start + cost > begin);
          if (hit) {
            first = true;
            const int src = __ffs(hit) - 1;
            if (lane == src) {
              const int64_t item = (begin - start) / length;
              first_unit = units_before(begin);
              s_b = b0 + lane;
              s_item = start + item * length;
              s_in_b = static_cast<int>(item);
            }
            first_unit = __shfl_sync(0xffffffffu, first_unit, src);
          }
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, start + cost >= end);
        if (hit) {
          const int src = __ffs(hit) - 1;
          units = (lane == src ? units_before(end) : 0) - first_unit;
          units = __shfl_sync(0xffffffffu, units, src);
          break;
        }
        before += __shfl_sync(0xffffffffu, cost_end, 31);
        before_units += __shfl_sync(0xffffffffu, u_end, 31);
      }
    }
    if (lane == 0) {
      s_share = share;
      s_units = static_cast<int>(units);
    }
  }
  __syncthreads();
  const int units = s_units;
  if (units == 0) return;
  const int64_t share = s_share, begin = share * blockIdx.x;
  int64_t item_at = s_item;  // where the current item begins

  Cursor cc;  // of the item that the CTA is at; blk: the CTA's next unit
  cc.b = s_b;
  load_sequence<kRows>(p, cc);
  cc.h = s_in_b / cc.tiles;
  cc.r = s_in_b % cc.tiles;
  cc.blk = static_cast<int>(max(int64_t(0), begin - item_at - kItemCost));
  enter_item<kRows>(p, cc);

  // ---- the loading warp: lane 4 w + c brings blocks c, c + 4, .. of warp w's sequence, which are half c & 1 of units
  // w + 7 (c / 2), and every 14th after it, into the slots of w's ring as they come free.  A pass over the lanes costs
  // as much for one block as for eight, so it waits between passes.  Page numbers are fetched one block ahead ----
  if (warp == kWarps) {
    constexpr int kNone = INT32_MIN;  // no row sees the block
    const int w = lane >> 2, half = lane & 1;
    int unit = w < kWarps ? w + kWarps * ((lane >> 1) & 1) : INT32_MAX, at = lane & 3;
    auto fetch = [&]() -> int {
      const int blk = 2 * cc.blk + half;
      if (blk >= cc.load) return kNone;
      const int page = p.page_shift >= 0 ? blk >> p.page_shift : blk / p.page_blocks;
      return p.table[static_cast<int64_t>(cc.b) * p.table_ld + page];
    };
    int next_page = kNone;
    if (unit < units) {
      advance<kRows>(p, cc, unit);
      next_page = fetch();
    }
    long long since = clock64();
    while (__any_sync(0xffffffffu, unit < units)) {
      const int slot = w * kRing + at % kRing, use = at / kRing;
      const bool go = unit < units && (use == 0 || mbar_test(empty + slot, (use - 1) & 1));
      if (go) {
        int page = next_page;
        if (page != kNone && (page < 0 || page >= p.num_pages)) {
          atomicCAS(p.status, 0, kStatusBadPage);
          page = kNone;
        }
        left_out[slot] = page == kNone;
        if (page != kNone) {
          const int blk = 2 * cc.blk + half;
          const int inner = p.page_shift >= 0 ? blk & (p.page_blocks - 1) : blk % p.page_blocks;
          mbar_arrive_expect_tx(full + slot, kBlock);
          bulk_g2s(ring + slot * kBlock,
                   p.cache + ((static_cast<int64_t>(page) * p.kv_heads + cc.h) * p.page_blocks + inner) * kBlock, kBlock,
                   full + slot);
        } else {
          mbar_arrive(full + slot);
        }
        at += 4;
        unit += 2 * kWarps;
        if (unit < units) {
          advance<kRows>(p, cc, 2 * kWarps);
          next_page = fetch();
        }
      }
      if (__any_sync(0xffffffffu, go)) since = clock64();
      if (!__any_sync(0xffffffffu, go && at < kRing)) __nanosleep(100);
      if (clock64() - since > kWaitLimitCycles) {
        s_abort = 1;
        atomicCAS(p.status, 0, 911);
        break;
      }
    }
    return;
  }

  int at = 0;           // blocks of the warp's sequence so far
  int done = 0;         // units of the share before the current item's
  uint4 qf[kQInRegs ? NT * D / 32 : 1];
  // query row i of a tile is token (r * kRows + i) / heads, head (r * kRows + i) % heads
  auto query = [&](const Cursor& c, int row, int e) {
    const int i = c.r * kRows + row;
    if (i >= c.rows_tok * p.heads) return make_uint4(0, 0, 0, 0);
    const int token = p.starts ? i / p.heads : 0;
    return *reinterpret_cast<const uint4*>(p.q + static_cast<int64_t>(c.q0 + token) * p.q_tok +
                                           static_cast<int64_t>(c.h * p.heads + i - token * p.heads) * p.q_head + e);
  };
  auto load_queries = [&](const Cursor& c) {
#pragma unroll
    for (int i = 0; i < NT * D / 32; ++i) qf[i] = query(c, i / (D / 32) * 8 + g, i % (D / 32) * 32 + t * 8);
  };
  if (kQInRegs) load_queries(cc);
  while (done < units) {
    // ---- one item (or the part of it that is this CTA's): units done .. done + n - 1 ----
    const int n = min(units - done, cc.blocks - cc.blk);
    const bool whole = cc.blk == 0 && n == cc.blocks;
    if (!kQInRegs) {
      named_bar_sync(kJoinBar, kWarps * 32);
      for (int i = threadIdx.x; i < kRows * D / 8; i += kWarps * 32)
        *reinterpret_cast<uint4*>(qs + i * 8) = query(cc, i / (D / 8), i % (D / 8) * 8);
      named_bar_sync(kJoinBar, kWarps * 32);
    }
    auto q_frag = [&](int nt, int w) {
      return *reinterpret_cast<const uint4*>(qs + (nt * 8 + g) * D + w * 32 + t * 8);
    };
    int sees[NT][2];  // keys that rows 2 t and 2 t + 1 of every 8 see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = cc.r * kRows + nt * 8 + 2 * t + e;
        sees[nt][e] = p.causal ? cc.len - cc.rows_tok + at / p.heads + 1 : cc.len;
        if (at >= cc.rows_tok * p.heads) sees[nt][e] = cc.len;  // (a row of zeros that nobody reads)
        sees[nt][e] = min(sees[nt][e], cc.len);
      }
    int all_see = sees[0][0];  // keys that every row of the tile sees: below, nothing is masked
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) all_see = min(all_see, sees[nt][e]);
    all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 1));
    all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 2));

    float o[NT][kMt][4];
    float top[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      top[nt][0] = top[nt][1] = -INFINITY;
      sum[nt][0] = sum[nt][1] = 0.f;
    }

    // the warp's units of the item: those with (unit % kWarps) == warp
    for (int u = done + (warp - done % kWarps + kWarps) % kWarps; u < done + n; u += kWarps) {
      const int key0 = (cc.blk + u - done) * kUnitKeys;
      const int slot0 = warp * kRing + at % kRing, use = (at / kRing) & 1;  // the unit's other block is in the next slot
      at += 2;
      mbar_wait(full + slot0, use, &s_abort, p.status, 910);
      mbar_wait(full + slot0 + 1, use, &s_abort, p.status, 910);
      const bool have0 = !left_out[slot0], have1 = !left_out[slot0 + 1];
      // ---- scores: s[i][nt] = keys g, g + 8 of block i and rows 2 t, 2 t + 1.  Both blocks side by side: their
      // products do not wait for one another ----
      float s[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][nt][e] = 0.f;
#pragma unroll
      for (int hh = 0; hh < kHalves; ++hh) {
        // (a block that was not loaded holds anything: its scores are masked below)
        uint32_t kw[2][2][nw], wp[2][2][kGroups];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* blk = ring + (slot0 + i) * kBlock;
          load_words(blk + g * (D / 2) + hh * 64 + t * nw * 4, kw[i][0]);
          load_words(blk + (g + 8) * (D / 2) + hh * 64 + t * nw * 4, kw[i][1]);
          load_words(blk + kv4_key_params(D) + (g * ng + hh * kGroups) * 4, wp[i][0]);
          load_words(blk + kv4_key_params(D) + ((g + 8) * ng + hh * kGroups) * 4, wp[i][1]);
        }
        Dequant<T> dq[2][2];
#pragma unroll
        for (int j = 0; j < nw; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (j % kWordsPerGroup == 0) {
              dq[i][0].same(wp[i][0][j / kWordsPerGroup]);
              dq[i][1].same(wp[i][1][j / kWordsPerGroup]);
            }
            uint32_t xa[4], xb[4];
            dq[i][0].values(kw[i][0][j], xa);
            dq[i][1].values(kw[i][1][j], xb);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {xa[2 * e], xb[2 * e], xa[2 * e + 1], xb[2 * e + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint4 q = kQInRegs ? qf[nt * (D / 32) + hh * nw + j] : q_frag(nt, hh * nw + j);
                T::mma(s[i][nt], a, e ? q.z : q.x, e ? q.w : q.y);
              }
            }
          }
      }
      // ---- softmax ----
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][nt][e] *= p.scale;
        if (key0 + kUnitKeys > all_see || !have0 || !have1) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(i ? have1 : have0) || key0 + i * 16 + g + (e >> 1) * 8 >= sees[nt][e & 1]) s[i][nt][e] = -INFINITY;
        }
        float m[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) m[e] = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
        const float over = fmaxf(m[0] - top[nt][0], m[1] - top[nt][1]);
        // (no score yet: -inf less -inf is NaN and stays; the first score is infinitely above)
        if (__any_sync(0xffffffffu, over > 8.f)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 4));
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 8));
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 16));
            m[e] = fmaxf(m[e], top[nt][e]);
            const float f = top[nt][e] == m[e] ? 1.f : exp2_approx(top[nt][e] - m[e]);
            top[nt][e] = m[e];
            sum[nt][e] *= f;
#pragma unroll
            for (int i = 0; i < kMt; ++i) {
              o[nt][i][e] *= f;
              o[nt][i][e + 2] *= f;
            }
          }
        }
        // a row without a score yet has -inf for both: less 0 then, so that its weights are 0
        const float t0 = top[nt][0] == -INFINITY ? 0.f : top[nt][0], t1 = top[nt][1] == -INFINITY ? 0.f : top[nt][1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x0 = exp2_approx(s[i][nt][0] - t0), x1 = exp2_approx(s[i][nt][1] - t1);
          const float x2 = exp2_approx(s[i][nt][2] - t0), x3 = exp2_approx(s[i][nt][3] - t1);
          sum[nt][0] += x0 + x2;
          sum[nt][1] += x1 + x3;
          pb[i][nt][0] = transpose8x8(T::pack(x0, x1));
          pb[i][nt][1] = transpose8x8(T::pack(x2, x3));
        }
      }
      // ---- values ----
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!(i ? have1 : have0)) continue;
        const uint8_t* blk = ring + (slot0 + i) * kBlock;
        const int left = cc.len - key0 - i * 16;  // tokens behind the last one hold anything
#pragma unroll
        for (int hh = 0; hh < kHalves; ++hh) {
          uint32_t va[nw], vb[nw];
          const uint8_t* base = blk + 8 * D + hh * W * 8 + g * 8 * (nw * 4);
          load_words(base + (t ^ kv4_swap(D, g)) * (nw * 4), va);
          load_words(base + ((t + 4) ^ kv4_swap(D, g)) * (nw * 4), vb);
          uint32_t x[4][kGroups];  // of tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int token = 2 * t + (e & 1) + (e >> 1) * 8;
            load_words(blk + kv4_value_params(D, G) + (token * ng + hh * kGroups) * 4, x[e]);
          }
          if (left < kKv4Tokens) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int k = 0; k < kGroups; ++k)
                if (2 * t + (e & 1) + (e >> 1) * 8 >= left) x[e][k] = 0;
          }
          Dequant<T> da, db;
#pragma unroll
          for (int j = 0; j < nw; ++j) {
            if (j % kWordsPerGroup == 0) {
              da.pair(x[0][j / kWordsPerGroup], x[1][j / kWordsPerGroup]);
              db.pair(x[2][j / kWordsPerGroup], x[3][j / kWordsPerGroup]);
            }
            uint32_t xa[4], xb[4];
            da.values(va[j], xa);
            db.values(vb[j], xb);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t a[4] = {xa[2 * e], xa[2 * e + 1], xb[2 * e], xb[2 * e + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) T::mma(o[nt][hh * 8 + 2 * j + e], a, pb[i][nt][0], pb[i][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane < 2) mbar_arrive(empty + slot0 + lane);
    }

    // ---- the next item's queries are on their way while the warps are joined ----
    Cursor next = cc;
    const bool more = done + n < units;
    if (more) {
      advance<kRows>(p, next, n);
      if (kQInRegs) load_queries(next);
    }

    // ---- join the warps ----
    // partial results of this CTA and item: [max, sum of every row][D x rows]
    constexpr int kPartial = kRows * (D + 2);
    const int64_t item_units = item_at + kItemCost;
    float* part = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (item_units < begin ? 0 : 1)) * kPartial;
    auto store = [&](int row, int d, float sum_pv, float sum_p) {
      const int i = cc.r * kRows + row;
      if (i >= cc.rows_tok * p.heads) return;
      const int token = p.starts ? i / p.heads : 0;
      p.out[static_cast<int64_t>(cc.q0 + token) * p.o_tok + static_cast<int64_t>(cc.h * p.heads + i - token * p.heads) * p.o_head +
            d] = T::from_float(sum_p == 0.f ? 0.f : sum_pv / sum_p * Dequant<T>::kBack);
    };
    constexpr int kJoinD = S::kJoinD;
#pragma unroll
    for (int step = 0; step < NT * D / kJoinD; ++step) {
      const int nt = step / (D / kJoinD), d0 = step % (D / kJoinD) * kJoinD;
      named_bar_sync(kJoinBar, kWarps * 32);  // (what was joined before is read)
      if (d0 == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = sum[nt][e];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (g == 0) stats[warp * 8 + 2 * t + e] = make_float2(top[nt][e], l);
        }
      }
#pragma unroll
      for (int i = 0; i < kJoinD / 16; ++i) {
        const float* x = o[nt][d0 / 16 + i];
        float* dst = join + (warp * kJoinD + 16 * i + g) * 8 + 2 * t;
        *reinterpret_cast<float2*>(dst) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(dst + 64) = make_float2(x[2], x[3]);
      }
      named_bar_sync(kJoinBar, kWarps * 32);
      // a thread has rows 4 (tid & 1) .. + 3 of elements tid / 2, + 112, ..
      const int row0 = (threadIdx.x & 1) * 4;
      float f[kWarps][4], m[4], l[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = -INFINITY;
        l[e] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m[e] = fmaxf(m[e], stats[w * 8 + row0 + e].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 st = stats[w * 8 + row0 + e];
          // (a warp without a score has sums of zero, or of NaN)
          f[w][e] = st.x == -INFINITY ? 1.f : exp2_approx(st.x - m[e]);
          l[e] = fmaf(st.y, f[w][e], l[e]);
        }
      }
      for (int i = threadIdx.x; i < kJoinD * 2; i += kWarps * 32) {
        const int d = d0 + i / 2;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(join + w * kJoinD * 8 + i * 4);
          v[0] = fmaf(x.x, f[w][0], v[0]);
          v[1] = fmaf(x.y, f[w][1], v[1]);
          v[2] = fmaf(x.z, f[w][2], v[2]);
          v[3] = fmaf(x.w, f[w][3], v[3]);
        }
        if (whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e) store(nt * 8 + row0 + e, d, v[e], l[e]);
        } else {
          *reinterpret_cast<float4*>(part + 2 * kRows + d * kRows + nt * 8 + row0) = make_float4(v[0], v[1], v[2], v[3]);
          if (d == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(part + 2 * (nt * 8 + row0 + e)) = make_float2(m[e], l[e]);
          }
        }
      }
    }
    if (!whole) {
      // ---- the last CTA of the item joins the parts ----
      const int first = static_cast<int>(item_units / share);
      const int parts = static_cast<int>((item_units + cc.blocks - 1) / share) - first + 1;
      __threadfence();
      named_bar_sync(kJoinBar, kWarps * 32);
      if (threadIdx.x == 0) {
        const uint32_t before = atomicAdd(p.counters + first, 1u);
        s_last = before == static_cast<uint32_t>(parts - 1);
        if (s_last) p.counters[first] = 0;
      }
      named_bar_sync(kJoinBar, kWarps * 32);
      if (s_last) {
        __threadfence();
        auto part_of = [&](int c) {
          return p.partials + (static_cast<int64_t>(first + c) * 2 + (item_units < (first + c) * share ? 0 : 1)) * kPartial;
        };
        // weights of the parts, [part][row] for as many parts at a time as the joining buffer takes
        float* wt = join;
        constexpr int kChunk = static_cast<int>(S::kJoinBytes) / (kRows * 4), kQuads = (D * 2 * NT + kWarps * 32 - 1) / (kWarps * 32);
        float mm = -INFINITY, l = 0.f;
        if (threadIdx.x < kRows)
          for (int c = 0; c < parts; ++c) mm = fmaxf(mm, __ldcg(part_of(c) + 2 * threadIdx.x));
        float4 v[kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c0 = 0; c0 < parts; c0 += kChunk) {
          const int c1 = min(parts, c0 + kChunk);
          if (c0) named_bar_sync(kJoinBar, kWarps * 32);
          if (threadIdx.x < kRows)
            for (int c = c0; c < c1; ++c) {
              const float2 st = __ldcg(reinterpret_cast<const float2*>(part_of(c) + 2 * threadIdx.x));
              const float f = st.x == -INFINITY ? 0.f : exp2_approx(st.x - mm);
              wt[(c - c0) * kRows + threadIdx.x] = f;
              l += st.x == -INFINITY ? st.y : st.y * f;
            }
          named_bar_sync(kJoinBar, kWarps * 32);
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
            const int at = threadIdx.x + i * kWarps * 32;
            if (at >= D * 2 * NT) break;
            for (int c = c0; c < c1; ++c) {
              const float4 x = __ldcg(reinterpret_cast<const float4*>(part_of(c) + 2 * kRows + at * 4));
              const float4 f = *reinterpret_cast<const float4*>(wt + (c - c0) * kRows + at % (2 * NT) * 4);
              v[i].x = fmaf(x.x, f.x, v[i].x);
              v[i].y = fmaf(x.y, f.y, v[i].y);
              v[i].z = fmaf(x.z, f.z, v[i].z);
              v[i].w = fmaf(x.w, f.w, v[i].w);
            }
          }
        }
        if (threadIdx.x < kRows) totals[threadIdx.x] = make_float2(mm, l);
        named_bar_sync(kJoinBar, kWarps * 32);
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const int quad = threadIdx.x + i * kWarps * 32;
          if (quad >= D * 2 * NT) break;
          const int d = quad / (2 * NT), row0 = quad % (2 * NT) * 4;
          const float r[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) store(row0 + e, d, r[e], totals[row0 + e].y);
        }
      }
    }
    item_at += cc.blocks + kItemCost;
    done += n;
    cc = next;
  }
}

template <typename T, int D, int G, int NT>
cudaError_t launch_one(const Kv4AttendParams& p, int ctas, cudaStream_t stream) {
  using S = Smem<D, G, NT>;
  static_assert(S::kFit >= 4 && S::ring % 16 == 0, "shared memory");
  auto kernel = kv4_attend_kernel<T, D, G, NT>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::total)))
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::total;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (dependent_launch_enabled()) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int NT>
cudaError_t launch_shape(const Kv4AttendParams& p, int d, int g, int ctas, cudaStream_t stream) {
  if (d == 64 && g == 32) return launch_one<T, 64, 32, NT>(p, ctas, stream);
  if (d == 64 && g == 64) return launch_one<T, 64, 64, NT>(p, ctas, stream);
  if constexpr (NT <= 2) {
    if (d == 128 && g == 32) return launch_one<T, 128, 32, NT>(p, ctas, stream);
    if (d == 128 && g == 64) return launch_one<T, 128, 64, NT>(p, ctas, stream);
    if (d == 128 && g == 128) return launch_one<T, 128, 128, NT>(p, ctas, stream);
    if (d == 256 && g == 32) return launch_one<T, 256, 32, NT>(p, ctas, stream);
    if (d == 256 && g == 64) return launch_one<T, 256, 64, NT>(p, ctas, stream);
    if (d == 256 && g == 128) return launch_one<T, 256, 128, NT>(p, ctas, stream);
  }
  return cudaErrorInvalidValue;
}

int ctas_for(int nt, int d, int num_sms) { return std::min(kMaxCtas, num_sms * ctas_per_sm(d, nt)); }

}  // namespace

// eights of query rows in a tile: what an average sequence brings
int kv4_attend_tiles(int batch, int64_t tokens, int heads, int d) {
  const int64_t rows = ceil_div(tokens, batch) * heads;
  if (rows <= 8) return 1;
  if (rows <= 16 || d >= 128) return 2;
  return 4;
}

size_t kv4_attend_partial_bytes(int batch, int64_t tokens, int heads, int d, int num_sms) {
  const int nt = kv4_attend_tiles(batch, tokens, heads, d);
  return static_cast<size_t>(ctas_for(nt, d, num_sms)) * 2 * 8 * nt * (d + 2) * 4;
}

// Whether the prompt kernel takes a call: its tiles have 128 rows, the ones above 8, 16 or 32.
bool kv4_attend_prompt(int batch, int64_t tokens, int heads) { return ceil_div(tokens, batch) * heads > 32; }

cudaError_t launch_kv4_attend(const Kv4AttendParams& p, int f16, int d, int g, int num_sms, cudaStream_t stream) {
  Kv4AttendParams q = p;
  q.page_shift = (p.page_blocks & (p.page_blocks - 1)) ? -1 : __builtin_ctz(static_cast<unsigned>(p.page_blocks));
  q.scale *= f16 ? Dequant<Kv4Fp16>::kBack : Dequant<Kv4Bf16>::kBack;
  if (p.starts && kv4_attend_prompt(p.batch, p.tokens, p.heads)) return launch_kv4_prompt(q, f16, d, g, stream);
  const int nt = kv4_attend_tiles(p.batch, p.tokens, p.heads, d);
  const int ctas = ctas_for(nt, d, num_sms);
#define KV4_NT(NT) f16 ? launch_shape<Kv4Fp16, NT>(q, d, g, ctas, stream) : launch_shape<Kv4Bf16, NT>(q, d, g, ctas, stream)
  return nt == 1 ? KV4_NT(1) : nt == 2 ? KV4_NT(2) : KV4_NT(4);
#undef KV4_NT
}

}  // namespace woq
