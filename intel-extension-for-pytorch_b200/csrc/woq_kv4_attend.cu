// Attention of a few query rows a sequence over the paged 4-bit cache (layout: woq_kv4_common.cuh):
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys j that the row sees, in one pass over the cache.
//
// The work is one long sequence of units, 16 keys of one (sequence, kv head, tile of query rows) each, dealt to the
// CTAs in equal shares whatever the lengths; the warps of a CTA take its units in turn.  A warp computes S^T = K Q^T
// and O^T += V^T P^T, so that up to eight query rows (the heads of a kv head, times tokens) fill the n side of
// m16n8k16 and dequantised codes are A fragments as they come from the cache.  P^T is S^T transposed in registers
// (movmatrix).  A running reference of the maximum is raised only when a score passes it by 8 (log2): P is at most 256.
// When a tile of rows ends, the warps' sums are joined in shared memory; a tile that several CTAs share is joined
// through the workspace by the last one, in the order of the keys, so that results do not depend on who is last.
#include <algorithm>

#include "woq_kernels.h"
#include "woq_kv4_common.cuh"

namespace woq {

namespace {

constexpr int kWarps = 8;
constexpr int kMaxCtas = 512;

// joined in slices of 64 elements x 8 rows a warp
constexpr int kJoinD = 64;
constexpr size_t kJoinBytes = kWarps * kJoinD * 8 * 4;

// Two CTAs an SM where the registers allow it (their accumulators are D x 8 NT / 32 a lane), and as many ring slots as
// fit: one SM then has up to 150 KB of copies in flight.
template <int D, int G, int NT>
struct Smem {
  static constexpr int kCtas = NT * D <= 256 ? 2 : 1, kBlock = kv4_block_bytes(D, G);
  static constexpr size_t kBudget = kCtas == 2 ? 112 * 1024 : 226 * 1024;
  static constexpr size_t join = 0;
  static constexpr size_t query = join + kJoinBytes;             // [8 NT][D] of T
  static constexpr size_t stats = query + 8 * NT * D * 2;        // [kWarps][8 NT]{max, sum}
  static constexpr size_t totals = stats + kWarps * 8 * NT * 8;  // [8 NT]{max, sum}
  static constexpr size_t bars = totals + 8 * NT * 8;            // [kWarps][8]
  static constexpr size_t ring = bars + kWarps * 8 * 8;
  static constexpr int kFit = static_cast<int>((kBudget - ring) / (kWarps * kBlock)), kRing = kFit < 8 ? kFit : 8;
  static constexpr size_t total = ring + static_cast<size_t>(kWarps) * kRing * kBlock;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Where a unit is: sequence b, kv head h, tile r of its query rows, block of 16 keys.  All lanes hold the same.
struct Cursor {
  int b, h, r, blk;
  int blocks, tiles;  // units of an item and tiles of the sequence
  int q0, rows_tok;   // first query row, number of them
  int len;
};

template <int ROWS>
__device__ __forceinline__ void load_sequence(const Kv4AttendParams& p, Cursor& c) {
  int len = p.lens[c.b];
  len = min(max(len, 0), p.max_blocks * kKv4Tokens);
  c.len = len;
  c.blocks = max(1, (len + kKv4Tokens - 1) / kKv4Tokens);
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
template <int ROWS>
__device__ __forceinline__ int64_t sequence_units(const Kv4AttendParams& p, int b) {
  Cursor c;
  c.b = b;
  load_sequence<ROWS>(p, c);
  return static_cast<int64_t>(c.blocks) * c.tiles * p.kv_heads;
}
// `steps` units on; the caller stays within the units there are
template <int ROWS>
__device__ __forceinline__ void advance(const Kv4AttendParams& p, Cursor& c, int steps) {
  c.blk += steps;
  while (c.blk >= c.blocks) {
    c.blk -= c.blocks;
    if (++c.r < c.tiles) continue;
    c.r = 0;
    if (++c.h < p.kv_heads) continue;
    c.h = 0;
    do {
      if (++c.b >= p.batch) return;  // past the last unit
      load_sequence<ROWS>(p, c);
    } while (c.tiles == 0);
  }
}
// keys that the last row of the tile sees
template <int ROWS>
__device__ __forceinline__ int tile_limit(const Kv4AttendParams& p, const Cursor& c) {
  if (!p.causal) return c.len;
  const int last = min(c.rows_tok * p.heads, (c.r + 1) * ROWS) - 1;
  return c.len - c.rows_tok + last / p.heads + 1;
}

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT * D <= 256 ? 2 : 1) kv4_attend_kernel(const __grid_constant__ Kv4AttendParams p) {
  using S = Smem<D, G, NT>;
  constexpr int kRows = 8 * NT, kRing = S::kRing, kBlock = S::kBlock, W = kv4_width(D), nw = W / 32, kHalves = D / W;
  constexpr int ng = D / G, kWordsPerGroup = G / 32, kMt = D / 16;
  constexpr bool kQInRegs = NT * D <= 128;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_total;
  __shared__ int64_t s_first_unit;
  __shared__ int s_first_b, s_last;
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::bars) + warp * 8;
  uint8_t* ring = smem + S::ring + static_cast<size_t>(warp) * kRing * kBlock;
  float* join = reinterpret_cast<float*>(smem + S::join);
  float2* stats = reinterpret_cast<float2*>(smem + S::stats);
  float2* totals = reinterpret_cast<float2*>(smem + S::totals);
  uint16_t* qs = reinterpret_cast<uint16_t*>(smem + S::query);

  if (lane == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(bars + i, 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) s_abort = 0;
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- this CTA's share ----
  if (warp == 0) {
    int64_t total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
      int64_t u = b0 + lane < p.batch ? sequence_units<kRows>(p, b0 + lane) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      total += u;
    }
    const int64_t most = max(int64_t(1), min(int64_t(gridDim.x), (total + kWarps - 1) / kWarps));
    const int64_t share = ((total + most - 1) / most + kWarps - 1) / kWarps * kWarps;
    const int64_t begin = share * blockIdx.x;
    if (begin < total) {
      int64_t before = 0;  // units of the sequences before b0
      for (int b0 = 0;; b0 += 32) {
        const int64_t u = b0 + lane < p.batch ? sequence_units<kRows>(p, b0 + lane) : 0;
        int64_t end = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += x;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, before + end > begin);
        if (hit) {
          const int at = __ffs(hit) - 1;
          if (lane == at) {
            s_first_b = b0 + at;
            s_first_unit = before + end - u;  // of the sequence
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, end, 31);
      }
    }
    if (lane == 0) s_total = begin < total ? total : -1;
    if (lane == 0) s_last = static_cast<int>(share);
  }
  __syncthreads();
  if (s_total < 0) return;
  const int64_t total = s_total, share = s_last, begin = share * blockIdx.x, end = min(total, begin + share);
  const int units = static_cast<int>(end - begin);

  Cursor cc;  // of the item that the CTA is at; blk: block of the CTA's next unit
  cc.b = s_first_b;
  load_sequence<kRows>(p, cc);
  {
    const int64_t rest = begin - s_first_unit;
    const int64_t item = rest / cc.blocks;
    cc.blk = static_cast<int>(rest - item * cc.blocks);
    cc.h = static_cast<int>(item / cc.tiles);
    cc.r = static_cast<int>(item % cc.tiles);
  }

  // ---- loads: the warp's units warp, warp + 8, .. of the share, kRing ahead ----
  Cursor pc = cc;
  int produced = warp;
  if (produced < units) advance<kRows>(p, pc, warp);
  int slot_in = 0;
  auto page_of = [&](const Cursor& c) -> int {  // -1: nothing to load
    if (c.blk * kKv4Tokens >= tile_limit<kRows>(p, c)) return -1;
    return p.table[static_cast<int64_t>(c.b) * p.table_ld + c.blk / p.page_blocks];
  };
  uint32_t loaded = 0;  // by ring slot: a copy was started
  auto produce = [&]() {
    if (produced >= units) return;
    const bool want = pc.blk * kKv4Tokens < tile_limit<kRows>(p, pc);
    int page = want ? page_of(pc) : -1;
    if (want && (page < 0 || page >= p.num_pages)) {
      if (lane == 0) atomicCAS(p.status, 0, kStatusBadPage);
      page = -1;
    }
    if (page >= 0) {
      loaded |= 1u << slot_in;
      if (lane == 0) {
        const uint8_t* src = p.cache + ((static_cast<int64_t>(page) * p.kv_heads + pc.h) * p.page_blocks +
                                        pc.blk % p.page_blocks) * kBlock;
        mbar_arrive_expect_tx(bars + slot_in, kBlock);
        bulk_g2s(ring + slot_in * kBlock, src, kBlock, bars + slot_in);
      }
    } else {
      loaded &= ~(1u << slot_in);
    }
    slot_in = slot_in + 1 == kRing ? 0 : slot_in + 1;
    produced += kWarps;
    if (produced < units) advance<kRows>(p, pc, kWarps);
  };
  for (int i = 0; i < kRing; ++i) produce();

  uint32_t parity = 0;  // by ring slot
  int slot_out = 0;
  int done = 0;         // units of the share before the current item's
  while (done < units) {
    // ---- one item (or the part of it that is this CTA's): units done .. done + n - 1 ----
    const int n = min(units - done, cc.blocks - cc.blk);
    const bool whole = cc.blk == 0 && n == cc.blocks;
    // query rows: row i of the tile is token (r * kRows + i) / heads, head (r * kRows + i) % heads
    for (int i = threadIdx.x; i < kRows * D / 8; i += kWarps * 32) {
      const int row = i / (D / 8), at = cc.r * kRows + row;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (at < cc.rows_tok * p.heads)
        v = *reinterpret_cast<const uint4*>(p.q + static_cast<int64_t>(cc.q0 + at / p.heads) * p.q_tok +
                                            static_cast<int64_t>(cc.h * p.heads + at % p.heads) * p.q_head + (i % (D / 8)) * 8);
      *reinterpret_cast<uint4*>(qs + i * 8) = v;
    }
    __syncthreads();
    uint4 qf[kQInRegs ? NT * D / 32 : 1];
    auto q_frag = [&](int nt, int w) {
      return *reinterpret_cast<const uint4*>(qs + (nt * 8 + g) * D + w * 32 + t * 8);
    };
    if (kQInRegs) {
#pragma unroll
      for (int i = 0; i < NT * D / 32; ++i) qf[i] = q_frag(i / (D / 32), i % (D / 32));
    }
    int sees[NT][2];  // keys that rows 2 t and 2 t + 1 of every 8 see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = cc.r * kRows + nt * 8 + 2 * t + e;
        sees[nt][e] = p.causal ? cc.len - cc.rows_tok + at / p.heads + 1 : cc.len;
        if (at >= cc.rows_tok * p.heads) sees[nt][e] = 0;
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

    // the warp's units of the item: those with (unit % 8) == warp
    for (int u = done + ((warp - done) & (kWarps - 1)); u < done + n; u += kWarps) {
      const int key0 = (cc.blk + u - done) * kKv4Tokens;
      const bool have = (loaded >> slot_out) & 1;
      if (have) {
        mbar_wait(bars + slot_out, (parity >> slot_out) & 1, &s_abort, p.status, 910);
        parity ^= 1u << slot_out;
        const uint8_t* blk = ring + slot_out * kBlock;
        // ---- scores ----
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int hh = 0; hh < kHalves; ++hh) {
          uint32_t ka[nw], kb[nw];
          const uint8_t* row = blk + g * (D / 2) + hh * 64 + t * nw * 4;
          if (nw == 4) {
            *reinterpret_cast<uint4*>(ka) = *reinterpret_cast<const uint4*>(row);
            *reinterpret_cast<uint4*>(kb) = *reinterpret_cast<const uint4*>(row + 4 * D);
          } else {
            *reinterpret_cast<uint2*>(ka) = *reinterpret_cast<const uint2*>(row);
            *reinterpret_cast<uint2*>(kb) = *reinterpret_cast<const uint2*>(row + 4 * D);
          }
          uint32_t sa = 0, ma = 0, sb = 0, mb = 0;
#pragma unroll
          for (int j = 0; j < nw; ++j) {
            if (j % kWordsPerGroup == 0) {
              const int group = (hh * nw + j) / kWordsPerGroup;
              const uint32_t pa = *reinterpret_cast<const uint32_t*>(blk + kv4_key_params(D) + (g * ng + group) * 4);
              const uint32_t pb = *reinterpret_cast<const uint32_t*>(blk + kv4_key_params(D) + ((g + 8) * ng + group) * 4);
              sa = __byte_perm(pa, 0, 0x1010);
              ma = __byte_perm(pa, 0, 0x3232);
              sb = __byte_perm(pb, 0, 0x1010);
              mb = __byte_perm(pb, 0, 0x3232);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a[4];
              a[0] = kv4_dequant2<T>(ka[j] >> (8 * e), sa, ma);
              a[1] = kv4_dequant2<T>(kb[j] >> (8 * e), sb, mb);
              a[2] = kv4_dequant2<T>(ka[j] >> (8 * e + 4), sa, ma);
              a[3] = kv4_dequant2<T>(kb[j] >> (8 * e + 4), sb, mb);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint4 q = kQInRegs ? qf[nt * (D / 32) + hh * nw + j] : q_frag(nt, hh * nw + j);
                T::mma(s[nt], a, e ? q.z : q.x, e ? q.w : q.y);
              }
            }
          }
        }
        // ---- softmax: s[nt] = keys g, g + 8 of rows 2 t, 2 t + 1 ----
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] *= p.scale;
          if (key0 + kKv4Tokens > all_see) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + g + (e >> 1) * 8 >= sees[nt][e & 1]) s[nt][e] = -INFINITY;
          }
          const float over = fmaxf(fmaxf(s[nt][0], s[nt][2]) - top[nt][0], fmaxf(s[nt][1], s[nt][3]) - top[nt][1]);
          // (no score yet: -inf less -inf is NaN and stays; the first score is infinitely above)
          if (__any_sync(0xffffffffu, over > 8.f)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float m = fmaxf(s[nt][e], s[nt][e + 2]);
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              m = fmaxf(m, top[nt][e]);
              const float f = top[nt][e] == m ? 1.f : exp2_approx(top[nt][e] - m);
              top[nt][e] = m;
              sum[nt][e] *= f;
#pragma unroll
              for (int i = 0; i < kMt; ++i) {
                o[nt][i][e] *= f;
                o[nt][i][e + 2] *= f;
              }
            }
          }
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // a row without a score yet: top is -inf, and so is the score
            x[e] = top[nt][e & 1] == -INFINITY ? (s[nt][e] == -INFINITY ? 0.f : s[nt][e]) : exp2_approx(s[nt][e] - top[nt][e & 1]);
          }
          sum[nt][0] += x[0] + x[2];
          sum[nt][1] += x[1] + x[3];
          pb[nt][0] = transpose8x8(T::pack(x[0], x[1]));
          pb[nt][1] = transpose8x8(T::pack(x[2], x[3]));
        }
        // ---- values ----
        const bool ragged = key0 + kKv4Tokens > cc.len;  // tokens behind the last one hold anything
#pragma unroll
        for (int hh = 0; hh < kHalves; ++hh) {
          uint32_t va[nw], vb[nw];
          const uint8_t* base = blk + 8 * D + hh * W * 8 + g * 8 * (nw * 4);
          const uint8_t* ra = base + (t ^ kv4_swap(D, g)) * (nw * 4);
          const uint8_t* rb = base + ((t + 4) ^ kv4_swap(D, g)) * (nw * 4);
          if (nw == 4) {
            *reinterpret_cast<uint4*>(va) = *reinterpret_cast<const uint4*>(ra);
            *reinterpret_cast<uint4*>(vb) = *reinterpret_cast<const uint4*>(rb);
          } else {
            *reinterpret_cast<uint2*>(va) = *reinterpret_cast<const uint2*>(ra);
            *reinterpret_cast<uint2*>(vb) = *reinterpret_cast<const uint2*>(rb);
          }
          uint32_t sa = 0, ma = 0, sb = 0, mb = 0;
#pragma unroll
          for (int j = 0; j < nw; ++j) {
            if (j % kWordsPerGroup == 0) {
              const int group = (hh * nw + j) / kWordsPerGroup;
              const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + kv4_value_params(D, G));
              uint32_t x[4] = {vp[(2 * t) * ng + group], vp[(2 * t + 1) * ng + group], vp[(2 * t + 8) * ng + group],
                               vp[(2 * t + 9) * ng + group]};
              if (ragged) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key0 + 2 * t + (e & 1) + (e >> 1) * 8 >= cc.len) x[e] = 0;
              }
              sa = __byte_perm(x[0], x[1], 0x5410);
              ma = __byte_perm(x[0], x[1], 0x7632);
              sb = __byte_perm(x[2], x[3], 0x5410);
              mb = __byte_perm(x[2], x[3], 0x7632);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a[4];
              a[0] = kv4_dequant2<T>(va[j] >> (8 * e), sa, ma);
              a[1] = kv4_dequant2<T>(va[j] >> (8 * e + 4), sa, ma);
              a[2] = kv4_dequant2<T>(vb[j] >> (8 * e), sb, mb);
              a[3] = kv4_dequant2<T>(vb[j] >> (8 * e + 4), sb, mb);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) T::mma(o[nt][hh * 8 + 2 * j + e], a, pb[nt][0], pb[nt][1]);
            }
          }
        }
      }
      __syncwarp();
      slot_out = slot_out + 1 == kRing ? 0 : slot_out + 1;
      produce();
    }

    // ---- join the warps ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[nt][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) stats[warp * kRows + nt * 8 + 2 * t + e] = make_float2(top[nt][e], l);
      }
    __syncthreads();
    if (threadIdx.x < kRows) {
      float mm = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, stats[w * kRows + threadIdx.x].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 st = stats[w * kRows + threadIdx.x];
        l += st.x == -INFINITY ? st.y : st.y * exp2_approx(st.x - mm);
      }
      totals[threadIdx.x] = make_float2(mm, l);
    }
    // partial results of this CTA and item: [max, sum of every row][D x rows]
    const int64_t item_begin = begin + done - cc.blk;  // in the sequence of all units
    constexpr int kPartial = kRows * (D + 2);
    const int slot = item_begin < begin ? 0 : 1;
    float* part = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * kPartial;
    constexpr int kSlices = D / kJoinD, kSliceD = kJoinD;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float m[2], f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[e] = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m[e] = fmaxf(m[e], stats[w * kRows + nt * 8 + 2 * t + e].x);
        f[e] = top[nt][e] == -INFINITY ? 0.f : exp2_approx(top[nt][e] - m[e]);
      }
#pragma unroll
      for (int sl = 0; sl < kSlices; ++sl) {
        if (nt > 0 || sl > 0) __syncthreads();
        // [warp][kSliceD][8]
#pragma unroll
        for (int i = 0; i < kSliceD / 16; ++i) {
          const float* x = o[nt][sl * (kSliceD / 16) + i];
          float* dst = join + (warp * kSliceD + 16 * i + g) * 8 + 2 * t;
          *reinterpret_cast<float2*>(dst) = make_float2(x[0] * f[0], x[1] * f[1]);
          *reinterpret_cast<float2*>(dst + 64) = make_float2(x[2] * f[0], x[3] * f[1]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kSliceD * 2; i += kWarps * 32) {  // element i / 2, four rows
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(join + w * kSliceD * 8 + i * 4);
            v.x += x.x;
            v.y += x.y;
            v.z += x.z;
            v.w += x.w;
          }
          const int d = sl * kSliceD + i / 2, row0 = nt * 8 + (i & 1) * 4;
          if (whole) {
            const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = cc.r * kRows + row0 + e;
              const float l = totals[row0 + e].y;
              if (at < cc.rows_tok * p.heads)
                p.out[static_cast<int64_t>(cc.q0 + at / p.heads) * p.o_tok +
                      static_cast<int64_t>(cc.h * p.heads + at % p.heads) * p.o_head + d] = T::from_float(l == 0.f ? 0.f : r[e] / l);
            }
          } else {
            *reinterpret_cast<float4*>(part + 2 * kRows + d * kRows + row0) = v;
          }
        }
      }
    }
    if (!whole) {
      if (threadIdx.x < kRows) *reinterpret_cast<float2*>(part + 2 * threadIdx.x) = totals[threadIdx.x];
      // ---- the last CTA of the item joins the parts ----
      const int first = static_cast<int>(item_begin / share), parts = static_cast<int>((item_begin + cc.blocks - 1) / share) - first + 1;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const uint32_t before = atomicAdd(p.counters + first, 1u);
        s_last = before == static_cast<uint32_t>(parts - 1);
        if (s_last) p.counters[first] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        auto part_of = [&](int c) {
          return p.partials + (static_cast<int64_t>(first + c) * 2 + (item_begin < (first + c) * share ? 0 : 1)) * kPartial;
        };
        // weights of the parts, [part][row] for as many parts at a time as the joining buffer takes
        float* wt = join;
        constexpr int kChunk = static_cast<int>(kJoinBytes) / (kRows * 4), kQuads = (D * 2 * NT + kWarps * 32 - 1) / (kWarps * 32);
        float mm = -INFINITY, l = 0.f;
        if (threadIdx.x < kRows)
          for (int c = 0; c < parts; ++c) mm = fmaxf(mm, __ldcg(part_of(c) + 2 * threadIdx.x));
        float4 v[kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c0 = 0; c0 < parts; c0 += kChunk) {
          const int c1 = min(parts, c0 + kChunk);
          if (c0) __syncthreads();
          if (threadIdx.x < kRows)
            for (int c = c0; c < c1; ++c) {
              const float2 st = __ldcg(reinterpret_cast<const float2*>(part_of(c) + 2 * threadIdx.x));
              const float f = st.x == -INFINITY ? 0.f : exp2_approx(st.x - mm);
              wt[(c - c0) * kRows + threadIdx.x] = f;
              l += st.x == -INFINITY ? st.y : st.y * f;
            }
          __syncthreads();
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
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
          const int quad = threadIdx.x + i * kWarps * 32;
          if (quad >= D * 2 * NT) break;
          const int d = quad / (2 * NT), row0 = quad % (2 * NT) * 4;
          const float r[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = cc.r * kRows + row0 + e;
            const float sum_e = totals[row0 + e].y;
            if (at < cc.rows_tok * p.heads)
              p.out[static_cast<int64_t>(cc.q0 + at / p.heads) * p.o_tok +
                    static_cast<int64_t>(cc.h * p.heads + at % p.heads) * p.o_head + d] =
                  T::from_float(sum_e == 0.f ? 0.f : r[e] / sum_e);
          }
        }
      }
    }
    __syncthreads();  // the query, the statistics and the joining buffer serve the next item
    done += n;
    if (done < units) advance<kRows>(p, cc, n);
  }
}

template <typename T, int D, int G, int NT>
cudaError_t launch_one(const Kv4AttendParams& p, int ctas, cudaStream_t stream) {
  using S = Smem<D, G, NT>;
  static_assert(S::kRing >= 2 && S::ring % 16 == 0, "shared memory");
  auto kernel = kv4_attend_kernel<T, D, G, NT>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::total)))
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kWarps * 32);
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
  if (d == 128 && g == 32) return launch_one<T, 128, 32, NT>(p, ctas, stream);
  if (d == 128 && g == 64) return launch_one<T, 128, 64, NT>(p, ctas, stream);
  if (d == 128 && g == 128) return launch_one<T, 128, 128, NT>(p, ctas, stream);
  if constexpr (NT <= 2) {
    if (d == 256 && g == 32) return launch_one<T, 256, 32, NT>(p, ctas, stream);
    if (d == 256 && g == 64) return launch_one<T, 256, 64, NT>(p, ctas, stream);
    if (d == 256 && g == 128) return launch_one<T, 256, 128, NT>(p, ctas, stream);
  }
  return cudaErrorInvalidValue;
}

int ctas_for(int nt, int d, int num_sms) { return std::min(kMaxCtas, num_sms * (nt * d <= 256 ? 2 : 1)); }

}  // namespace

// eights of query rows in a tile: what an average sequence brings
int kv4_attend_tiles(int batch, int64_t tokens, int heads, int d) {
  const int64_t rows = ceil_div(tokens, batch) * heads;
  if (rows <= 8) return 1;
  if (rows <= 16 || d == 256) return 2;
  return 4;
}

size_t kv4_attend_partial_bytes(int batch, int64_t tokens, int heads, int d, int num_sms) {
  const int nt = kv4_attend_tiles(batch, tokens, heads, d);
  return static_cast<size_t>(ctas_for(nt, d, num_sms)) * 2 * 8 * nt * (d + 2) * 4;
}

cudaError_t launch_kv4_attend(const Kv4AttendParams& p, int f16, int d, int g, int num_sms, cudaStream_t stream) {
  const int nt = kv4_attend_tiles(p.batch, p.tokens, p.heads, d);
  const int ctas = ctas_for(nt, d, num_sms);
#define KV4_NT(NT) f16 ? launch_shape<Kv4Fp16, NT>(p, d, g, ctas, stream) : launch_shape<Kv4Bf16, NT>(p, d, g, ctas, stream)
  return nt == 1 ? KV4_NT(1) : nt == 2 ? KV4_NT(2) : KV4_NT(4);
#undef KV4_NT
}

}  // namespace woq
