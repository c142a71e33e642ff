// Attention of a few query rows a sequence over the paged 4-bit cache (layout: woq_kv4_common.cuh):
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys j that the row sees, in one pass over the cache.
//
// The work is one long sequence of units, 32 keys of one (sequence, kv head, tile of query rows) each, dealt to the
// CTAs in equal shares whatever the lengths; the warps of a CTA take its units in turn.  A warp computes S^T = K Q^T
// and O^T += V^T P^T, so that up to eight query rows (the heads of a kv head, times tokens) fill the n side of
// m16n8k16 and dequantised codes are A fragments as they come from the cache.  P^T is S^T transposed in registers
// (movmatrix).  The softmax's reference runs behind the maximum (woq_kv4_common.cuh).
// When a tile of rows ends, the warps' sums are joined in shared memory; a tile that several CTAs share is joined
// through the workspace by the last one, in a fixed order, so that results do not depend on who is last.
//
// Bound by latency inside a warp's units (dequantise, products, maximum, exponentials, transpose, products, one behind the
// other) at 14 computing warps an SM: about 350 instructions for a block of 16 keys at half of the issue slots, DRAM at 42 %.
// 64 sequences of 1 to 8192 tokens, 64 heads of 128 on 8, 84 us = 3.6 TB/s of 6.6; two of 100,000 in fp16 68 us.  Small calls
// are bound by what comes one after another (lengths, page numbers, blocks, joining warps and CTAs), each part from a cold
// instruction cache: one sequence of 1025 tokens 10.8 us.
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

// What an item costs beside its units (queries, joining the warps), in units.  64 sequences of 1 to 8192 tokens take
// 84.8 / 83.8 / 84.0 / 85.6 us with 10 / 14 / 18 / 24, 16 drafts of 3 to 6 tokens (D = 256) 43.1 / 41.3 / 41.1 / 42.1, 1024
// sequences of 100 to 300 tokens 152 / 156 / 155 / 159.
constexpr int kItemCost = 18;

// Two CTAs an SM where the registers allow it (their accumulators are D x 8 NT / 32 a lane), and as many ring slots as
// fit: one SM then has up to 150 KB of copies in flight.
constexpr int ctas_per_sm(int d, int nt) { return nt * d <= 128 ? 2 : 1; }
template <int D, int G, int NT>
struct Smem {
  // CTAs that share an item, what their statistics leave room for.  More of them are joined longer and read faster: one
  // sequence of 100,000 tokens of one kv head takes 35.6 us with 36 CTAs, 26.4 with 64 and 23.6 with 112.
  static constexpr int kMaxParts = NT > 2 ? 48 : 112;
  static constexpr int kCtas = ctas_per_sm(D, NT), kBlock = kv4_block_bytes(D, G);
  static constexpr size_t kBudget = kCtas == 2 ? 112 * 1024 : 226 * 1024;
  static constexpr size_t join = 0;                              // [kWarps][D][8] sums of the values
  static constexpr size_t kJoinBytes = kWarps * D * 8 * 4;
  static constexpr size_t query = join + kJoinBytes;             // [8 NT][D] of T, where registers do not hold them
  static constexpr bool kQInRegs = NT * D <= 128;
  static constexpr size_t stats = query + (kQInRegs ? 0 : 8 * NT * D * 2);  // [kWarps][8 NT]{max, sum}
  static constexpr size_t totals = stats + kWarps * 8 * NT * 8;  // [8 NT]{max, sum}
  static constexpr size_t row_at = totals + 8 * NT * 8;          // [8 NT] places in the output
  static constexpr size_t full = row_at + 8 * NT * 8;            // [kWarps][kRing] barriers: the slot holds its block
  static constexpr size_t empty = full + kWarps * 8 * 8;         // the warp has read it
  static constexpr size_t weight = empty + kWarps * 8 * 8;       // [kMaxParts][8 NT] of the parts of an item
  static constexpr size_t left_out = weight + kMaxParts * 8 * NT * 4;  // words: nothing was loaded
  static constexpr size_t ring = left_out + kWarps * 8 * 4;
  static constexpr int kFit = static_cast<int>((kBudget - ring) / (kWarps * kBlock)), kRing = kFit >= 8 ? 8 : kFit;
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
  constexpr int kMaxParts = S::kMaxParts;
  constexpr int kRows = 8 * NT, kRing = S::kRing, kBlock = S::kBlock, W = kv4_width(D), nw = W / 32, kHalves = D / W;
  constexpr int ng = D / G, kGroups = ng / kHalves, kWordsPerGroup = G / 32, kMt = D / 16;
  constexpr bool kQInRegs = S::kQInRegs;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_run[kThreads / 32][3];  // {cost, units, longest item} of the sequences of a warp
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
  int64_t* row_at = reinterpret_cast<int64_t*>(smem + S::row_at);
  uint16_t* qs = reinterpret_cast<uint16_t*>(smem + S::query);

  if (threadIdx.x < kWarps * kRing) {
    mbar_init(full + threadIdx.x, 1);
    mbar_init(empty + threadIdx.x, 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) s_abort = 0;
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- this CTA's share: [begin, end) of all items' units, every item preceded by kItemCost that nobody computes.  Every
  // warp adds up a run of the sequences (their lengths all on their way at once), the first one looks into two of the
  // runs for the ends of the share ----
  const int run = (p.batch + kThreads - 1) / kThreads * 32;  // sequences of a warp
  {
    int64_t cost = 0, u = 0;
    int longest = 0;
#pragma unroll 4
    for (int b = warp * run + lane; b < min(p.batch, (warp + 1) * run); b += 32) {
      const int2 c = sequence_items<kRows>(p, b);
      cost += static_cast<int64_t>(c.x) * (c.y + kItemCost);
      u += static_cast<int64_t>(c.x) * c.y;
      if (c.x > 0) longest = max(longest, c.y);
    }
    if (warp * run < p.batch) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        cost += __shfl_xor_sync(0xffffffffu, cost, o);
        u += __shfl_xor_sync(0xffffffffu, u, o);
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
      }
    }
    if (lane == 0) {
      s_run[warp][0] = cost;
      s_run[warp][1] = u;
      s_run[warp][2] = longest;
    }
  }
  const int runs = (p.batch + run - 1) / run;
  if (runs > 1)
    __syncthreads();
  else
    __syncwarp();  // (the first warp has them all)
  if (warp == 0) {
    int64_t total = 0, longest = 0;
    for (int w = 0; w < runs; ++w) {
      total += s_run[w][0];
      longest = max(longest, s_run[w][2]);
    }
    // (few long items: as many parts as are joined in less time than they save)
    const int64_t share = max(max(int64_t(kWarps), (total + gridDim.x - 1) / gridDim.x), longest / (kMaxParts - 2) + 1);
    const int64_t begin = share * blockIdx.x, end = min(total, begin + share);
    int64_t units = 0;
    if (begin < total) {
      // the units before `place` of the sequence of all items; the sequence, item within it and its beginning
      auto locate = [&](int64_t place, int64_t& item_begin, int& b_out, int& item_out) -> int64_t {
        int64_t before = 0, before_units = 0;  // of the sequences before b0
        int b0 = 0;
        for (int w = 0; w + 1 < runs && before + s_run[w][0] <= place; ++w) {
          before += s_run[w][0];
          before_units += s_run[w][1];
          b0 += run;
        }
        for (;; b0 += 32) {
          const int2 c = sequence_items<kRows>(p, b0 + lane);
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
          const uint32_t hit = __ballot_sync(0xffffffffu, before + cost_end > place);
          if (hit) {
            const int src = __ffs(hit) - 1, length = c.y + kItemCost;
            const int64_t start = before + cost_end - cost, x = place - start;
            // (a 64-bit division takes a hundred instructions)
            const int64_t item = lane != src ? 0 : x >> 32 ? x / length : static_cast<uint32_t>(x) / static_cast<uint32_t>(length);
            const int64_t at = before_units + u_end - u + item * c.y + max(int64_t(0), x - item * length - kItemCost);
            item_begin = __shfl_sync(0xffffffffu, start + item * length, src);
            item_out = static_cast<int>(__shfl_sync(0xffffffffu, item, src));
            b_out = b0 + src;
            return __shfl_sync(0xffffffffu, at, src);
          }
          before += __shfl_sync(0xffffffffu, cost_end, 31);
          before_units += __shfl_sync(0xffffffffu, u_end, 31);
        }
      };
      int64_t item_begin, unused;
      int b, in_b, unused_b, unused_in;
      units = -locate(begin, item_begin, b, in_b);
      if (end < total) {
        units += locate(end, unused, unused_b, unused_in);
      } else {
        for (int w = 0; w < runs; ++w) units += s_run[w][1];
      }
      if (lane == 0) {
        s_b = b;
        s_in_b = in_b;
        s_item = item_begin;
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
          p.status[kBadPageWord] = 1;
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
      const int slot0 = warp * kRing + at % kRing, slot1 = warp * kRing + (at + 1) % kRing;  // of the unit's two blocks
      mbar_wait(full + slot0, (at / kRing) & 1, &s_abort, p.status, 910);
      mbar_wait(full + slot1, ((at + 1) / kRing) & 1, &s_abort, p.status, 910);
      at += 2;
      const bool have0 = !left_out[slot0], have1 = !left_out[slot1];
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
          const uint8_t* blk = ring + (i ? slot1 : slot0) * kBlock;
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
        if (__any_sync(0xffffffffu, over > T::kRaise)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 4));
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 8));
            m[e] = fmaxf(m[e], __shfl_xor_sync(0xffffffffu, m[e], 16));
            m[e] = fmaxf(m[e] - T::kTopWeight, top[nt][e]);
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
        const uint8_t* blk = ring + (i ? slot1 : slot0) * kBlock;
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
      if (lane < 2) mbar_arrive(empty + (lane ? slot1 : slot0));
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
    auto store = [&](int row0, int d, const float4& v) {
      const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t at = row_at[row0 + e];
        const float l = totals[row0 + e].y;
        if (at >= 0) p.out[at + d] = T::from_float(l == 0.f ? 0.f : __fdividef(r[e], l) * Dequant<T>::kBack);
      }
    };
    auto add_warps = [&](int i) {  // element i / 2, rows 4 (i & 1) to + 3
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(join + w * D * 8 + i * 4);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      return v;
    };
    // eight rows at a time: every warp's sums against the rows' common maximum, added in the order of the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[nt][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) stats[warp * 8 + 2 * t + e] = make_float2(top[nt][e], l);
      }
      named_bar_sync(kJoinBar, kWarps * 32);  // (what was joined before is read, too)
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, stats[w * 8 + 2 * t + e].x);
        // (a warp without a score has sums of zero, or of NaN)
        f[e] = top[nt][e] == -INFINITY ? 1.f : exp2_approx(top[nt][e] - m);
      }
#pragma unroll
      for (int i = 0; i < kMt; ++i) {
        const float* x = o[nt][i];
        float* dst = join + (warp * D + 16 * i + g) * 8 + 2 * t;
        *reinterpret_cast<float2*>(dst) = make_float2(x[0] * f[0], x[1] * f[1]);
        *reinterpret_cast<float2*>(dst + 64) = make_float2(x[2] * f[0], x[3] * f[1]);
      }
      // (where rows go is looked up once: the code of a small call runs from a cold instruction cache)
      if (nt == 0 && threadIdx.x < kRows) {
        const int i = cc.r * kRows + threadIdx.x, token = p.starts ? i / p.heads : 0;
        row_at[threadIdx.x] = i < cc.rows_tok * p.heads ? static_cast<int64_t>(cc.q0 + token) * p.o_tok +
                                                            static_cast<int64_t>(cc.h * p.heads + i - token * p.heads) * p.o_head
                                                      : -1;
      }
      if (threadIdx.x < 8) {
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, stats[w * 8 + threadIdx.x].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 st = stats[w * 8 + threadIdx.x];
          l = fmaf(st.y, st.x == -INFINITY ? 1.f : exp2_approx(st.x - m), l);
        }
        totals[nt * 8 + threadIdx.x] = make_float2(m, l);
        if (!whole) *reinterpret_cast<float2*>(part + 2 * (nt * 8 + threadIdx.x)) = make_float2(m, l);
      }
      named_bar_sync(kJoinBar, kWarps * 32);
      for (int i = threadIdx.x; i < D * 2; i += kWarps * 32) {
        const int d = i / 2, row0 = (i & 1) * 4;
        const float4 v = add_warps(i);
        if (whole) {
          store(nt * 8 + row0, d, v);
        } else {
          *reinterpret_cast<float4*>(part + 2 * kRows + d * kRows + nt * 8 + row0) = v;
        }
      }
      if (nt + 1 < NT) named_bar_sync(kJoinBar, kWarps * 32);  // (the statistics' place is written again)
    }
    if (!whole) {
      // ---- the last CTA of the item joins the parts ----
      const int first = static_cast<int>(item_units / share);
      const int parts = static_cast<int>((item_units + cc.blocks - 1) / share) - first + 1;
      named_bar_sync(kJoinBar, kWarps * 32);
      if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t before = atomicAdd(p.counters + first, 1u);
        s_last = before == static_cast<uint32_t>(parts - 1);
        if (s_last) p.counters[first] = 0;
        __threadfence();
      }
      named_bar_sync(kJoinBar, kWarps * 32);
      if (s_last) {
        // Statistics of all parts at once, eight lanes a row weigh them, then the sums in the order of the parts, four in
        // flight.  Small code: it runs once, from a cold instruction cache.
        // (the item begins in its first CTA's share and before all others')
        auto part_of = [&](int c) { return p.partials + (2 * (first + c) + (c == 0)) * kPartial; };
        float2* ps = reinterpret_cast<float2*>(join);               // [part][row]
        float* weight = reinterpret_cast<float*>(smem + S::weight);  // [part][row]
        static_assert(2 * kMaxParts * kRows * 4 <= S::kJoinBytes, "joining buffer");
        for (int i = threadIdx.x; i < parts * kRows; i += kWarps * 32)
          ps[i] = __ldcg(reinterpret_cast<const float2*>(part_of(i / kRows)) + i % kRows);
        named_bar_sync(kJoinBar, kWarps * 32);
        for (int row = threadIdx.x >> 3; row < kRows; row += kWarps * 4) {  // (four rows a warp: it stays together)
          const int sub = threadIdx.x & 7;
          float m = -INFINITY, l = 0.f;
          for (int c = sub; c < parts; c += 8) m = fmaxf(m, ps[c * kRows + row].x);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          for (int c = sub; c < parts; c += 8) {
            const float2 st = ps[c * kRows + row];
            const float f = st.x == -INFINITY ? 1.f : exp2_approx(st.x - m);  // (nothing seen: sums of zero, or of NaN)
            weight[c * kRows + row] = f;
            l = fmaf(st.y, f, l);
          }
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          if (sub == 0) totals[row] = make_float2(m, l);
        }
        named_bar_sync(kJoinBar, kWarps * 32);
        // a warp adds every seventh part, all of it in flight; then the warps as above
#pragma unroll 1
        for (int nt = 0; nt < NT; ++nt) {
          float4 v[kMt];
#pragma unroll
          for (int k = 0; k < kMt; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
          for (int c = warp; c < parts; c += kWarps) {
            const float4 f = *reinterpret_cast<const float4*>(weight + c * kRows + nt * 8 + (lane & 1) * 4);
            const float4* src = reinterpret_cast<const float4*>(part_of(c) + 2 * kRows + lane / 2 * kRows + nt * 8) + (lane & 1);
            float4 x[kMt];
#pragma unroll
            for (int k = 0; k < kMt; ++k) x[k] = __ldcg(src + k * 4 * kRows);
#pragma unroll
            for (int k = 0; k < kMt; ++k) {
              v[k].x = fmaf(x[k].x, f.x, v[k].x);
              v[k].y = fmaf(x[k].y, f.y, v[k].y);
              v[k].z = fmaf(x[k].z, f.z, v[k].z);
              v[k].w = fmaf(x[k].w, f.w, v[k].w);
            }
          }
#pragma unroll
          for (int k = 0; k < kMt; ++k) *reinterpret_cast<float4*>(join + warp * D * 8 + (lane + 32 * k) * 4) = v[k];
          named_bar_sync(kJoinBar, kWarps * 32);
          for (int i = threadIdx.x; i < D * 2; i += kWarps * 32) store(nt * 8 + (i & 1) * 4, i / 2, add_warps(i));
          if (nt + 1 < NT) named_bar_sync(kJoinBar, kWarps * 32);
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

// Whether the prompt kernel takes a call.  Its tiles have 128 rows, the ones above 8, 16 or 32, but its CTAs are long to
// fill and to join.  With a tile for every SM it wins from the second small tile on (32 sequences of 1000 tokens, 8 kv
// heads of 4 query heads and 128 elements, 9 new tokens: 54.8 us against 72.2), with fewer from about the fifth (one
// sequence of 20,000 tokens: 12 new tokens 68 us against 37, 16 68 against 44, 32 68 against 76; 8 sequences of 2000: 16
// new tokens 44.4 against 45.3, 24 44.7 against 62.1).  Elements of 64 and 256 divide alike.  The rows are an average, since
// lengths are not known here: 64 sequences of 4096 tokens with one new token each and a prompt of 1000 take 367 us in one call,
// 88 and 32 in two.
static int64_t kv4_small_tile_rows(int batch, int kv_heads, int num_sms) {
  return static_cast<int64_t>(batch) * kv_heads >= num_sms ? 32 : 64;
}
static bool kv4_attend_prompt(int batch, int64_t tokens, int heads, int kv_heads, int num_sms) {
  return ceil_div(tokens, batch) * heads > kv4_small_tile_rows(batch, kv_heads, num_sms);
}

static size_t few_rows_bytes(int nt, int d, int num_sms) {
  return static_cast<size_t>(ctas_for(nt, d, num_sms)) * 2 * 8 * nt * (d + 2) * 4;
}

size_t kv4_attend_partial_bytes(int batch, int64_t tokens, int heads, int kv_heads, int d, int num_sms) {
  const size_t few = few_rows_bytes(kv4_attend_tiles(batch, tokens, heads, d), d, num_sms);
  return kv4_attend_prompt(batch, tokens, heads, kv_heads, num_sms) ? std::max(few, kv4_prompt_partial_bytes(batch, tokens, heads, kv_heads, d, num_sms)) : few;
}

// The most that any call of up to `tokens` rows takes: a workspace made for a large call serves every smaller one.  (Large
// calls share nothing between CTAs; of the prompts the fewest rows of one sequence are shared first.)
size_t kv4_attend_partial_bytes_up_to(int64_t tokens, int heads, int kv_heads, int d, int num_sms) {
  size_t most = 0;
  for (int nt = 1; nt <= kv4_attend_tiles(1, tokens, heads, d); nt *= 2) most = std::max(most, few_rows_bytes(nt, d, num_sms));
  const int64_t shortest = kv4_small_tile_rows(1, kv_heads, num_sms) / heads + 1;  // prompt
  return tokens < shortest ? most : std::max(most, kv4_prompt_partial_bytes(1, shortest, heads, kv_heads, d, num_sms));
}

cudaError_t launch_kv4_attend(const Kv4AttendParams& p, int f16, int d, int g, int num_sms, cudaStream_t stream) {
  Kv4AttendParams q = p;
  q.page_shift = (p.page_blocks & (p.page_blocks - 1)) ? -1 : __builtin_ctz(static_cast<unsigned>(p.page_blocks));
  q.scale *= f16 ? Dequant<Kv4Fp16>::kBack : Dequant<Kv4Bf16>::kBack;
  if (p.starts && kv4_attend_prompt(p.batch, p.tokens, p.heads, p.kv_heads, num_sms)) {
    q.splits = kv4_prompt_splits(p.batch, p.tokens, p.heads, p.kv_heads, d, static_cast<int64_t>(p.max_blocks) * kKv4Tokens, num_sms);
    return launch_kv4_prompt(q, f16, d, g, stream);
  }
  const int nt = kv4_attend_tiles(p.batch, p.tokens, p.heads, d);
  const int ctas = ctas_for(nt, d, num_sms);
#define KV4_NT(NT) f16 ? launch_shape<Kv4Fp16, NT>(q, d, g, ctas, stream) : launch_shape<Kv4Bf16, NT>(q, d, g, ctas, stream)
  return nt == 1 ? KV4_NT(1) : nt == 2 ? KV4_NT(2) : KV4_NT(4);
#undef KV4_NT
}

}  // namespace woq
