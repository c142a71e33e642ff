// Attention of prompts over the paged 4-bit cache (layout: woq_kv4_common.cuh) on the tensor cores (tcgen05):
//   o = sum_j softmax_j(scale * q . k_j) v_j, causal from the last token backwards or over all keys.
//
// A CTA takes one kv head of one sequence and NQ tiles of 128 query rows (a row is a token's query head; the heads
// of a kv head lie next to one another, so they share its keys), and walks over the keys in tiles of KT:
//   warps 0 .. 4 NQ - 1   softmax: thread = query row.  Scores from tensor memory, probabilities back over them
//   4 warps               codes of a tile to T in shared memory, K-major with 128-byte swizzle; values transposed (a row
//                         per element, its keys next to one another)
//   1 warp                issues S = Q K^T and O += P V; allocates tensor memory
// The products of one tile of rows run while the other tile's softmax does.  Codes are loaded straight into
// registers, one tile ahead; the dequantised values (bf16: times 2^-64, see Dequant) never leave the SM.
// The softmax's reference runs behind the maximum (woq_kv4_common.cuh), so that O is rescaled seldom.
//
// Bound by the softmax warps (two passes over the scores in tensor memory, an exponential an element) and, as much, by
// the dequantising warps: each takes about 4100 cycles a tile of 256 x 128, whose products take 2048 (the tensor pipe is
// active for 35 % of the time).  Prompts of 4096 and 3000 tokens, 32 heads of 128 on 8, some behind cached ones: 346 us,
// 720 TFLOP/s.
#include <algorithm>

#include "woq_kernels.h"
#include "woq_kv4_common.cuh"
#include "woq_kv4_dequant.cuh"
#include "woq_tc_common.cuh"

namespace woq {

namespace {

template <int D>
struct Shape {
  static constexpr int kNQ = D == 256 ? 1 : 2;    // tiles of 128 rows
  static constexpr int kKeys = D == 256 ? 64 : 128;
  static constexpr int kRows = 128 * kNQ;
  static constexpr int kSoftmaxWarps = 4 * kNQ, kDequantWarp0 = kSoftmaxWarps, kMmaWarp = kDequantWarp0 + 4;
  static constexpr int kThreads = (kMmaWarp + 1) * 32;
  static constexpr int kQBytes = 128 * D * 2, kKBytes = kKeys * D * 2;  // of a tile of queries, of keys or values
  static constexpr int q = 1024, k = q + kNQ * kQBytes, v = k + 2 * kKBytes, used = v + 2 * kKBytes + 1024;
  static constexpr int total = used < 116 * 1024 ? 116 * 1024 : used;  // one CTA an SM: it takes all of tensor memory
};
static_assert(Shape<64>::total <= 227 * 1024 && Shape<128>::total <= 227 * 1024 && Shape<256>::total <= 227 * 1024, "shared memory");

struct Header {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_full[2], q_full[2];
  uint32_t tmem;
  int abort_flag;
  int bad_page;  // a page of the sequence does not exist
  int last[2];   // this CTA joins the parts of the tile of rows
  int b, tile;
};
static_assert(sizeof(Header) <= 1024, "header");
// two 32-bit operations an instruction
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void halves_of(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// waits for the loads issued so far; the registers pass through, so that nothing that reads them moves ahead of it
__device__ __forceinline__ void wait_ld_x32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void umma_f16_ss_plain(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_plain(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 32 columns of scores: those of keys that the row does not see to -inf
__device__ __forceinline__ void mask32(uint32_t (&x)[32], int sees, uint32_t gone) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (e >= sees || ((gone >> (e / 16)) & 1)) x[e] = 0xff800000u;
}
// Calls work(x, c) for the KT columns from t_s, 32 at a time, with the next 32 on their way.  A short loop: the roles'
// code together has to stay in the instruction cache (unrolled, a third of all stalls were instruction fetches).
template <int KT, typename Work>
__device__ __forceinline__ void over_columns(uint32_t t_s, Work work) {
  uint32_t a[32], b[32];
  tmem_ld_x32(t_s, a);
#pragma unroll 1
  for (int c = 0; c < KT / 32; c += 2) {
    wait_ld_x32(a);
    tmem_ld_x32(t_s + (c + 1) * 32, b);
    work(a, c);
    wait_ld_x32(b);
    if (c + 2 < KT / 32) tmem_ld_x32(t_s + (c + 2) * 32, a);
    work(b, c + 1);
  }
}
// the largest score of a row; `sees`: how many of the tile's keys the row sees, `gone`: blocks of 16 that do not exist
template <int KT, bool MASKED>
__device__ __forceinline__ float tile_max(uint32_t t_s, int sees, uint32_t gone) {
  float most = -INFINITY;
  over_columns<KT>(t_s, [&](uint32_t(&x)[32], int c) {
    if (MASKED) mask32(x, sees - c * 32, gone >> (2 * c));
#pragma unroll
    for (int e = 0; e < 32; e += 2) most = fmaxf(most, fmaxf(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
  });
  return most;
}
// probabilities 2^(score * scale + base) of a row, in T over the scores; returns their sum
template <typename T, int KT, bool MASKED>
__device__ __forceinline__ float tile_exp(uint32_t t_s, float scale, float base, int sees, uint32_t gone) {
  const uint64_t scale2 = pair_of(__float_as_uint(scale), __float_as_uint(scale));
  const uint64_t base2 = pair_of(__float_as_uint(base), __float_as_uint(base));
  uint64_t part = 0;
  over_columns<KT>(t_s, [&](uint32_t(&x)[32], int c) {
    if (MASKED) mask32(x, sees - c * 32, gone >> (2 * c));
    uint32_t out[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float y0, y1;
      halves_of(fma_x2(pair_of(x[e], x[e + 1]), scale2, base2), y0, y1);
      if (MASKED) {  // (-inf times a scale of 0)
        if (x[e] == 0xff800000u) y0 = -INFINITY;
        if (x[e + 1] == 0xff800000u) y1 = -INFINITY;
      }
      y0 = exp2_approx(y0);
      y1 = exp2_approx(y1);
      part = add_x2(part, pair_of(__float_as_uint(y0), __float_as_uint(y1)));
      out[e / 2] = T::pack(y0, y1);
    }
    tmem_st_x16(t_s + c * 16, out);
  });
  float s0, s1;
  halves_of(part, s0, s1);
  return s0 + s1;
}

// The sequence and tile of rows of a CTA (b = batch: none), found by one warp.  A sequence's last rows see most keys:
// they go first.
template <int ROWS>
__device__ __forceinline__ void find_tile(const Kv4AttendParams& p, int64_t at, int& b_out, int& tile_out) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  b_out = p.batch;
  tile_out = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int64_t tiles = 0;
    if (b0 + lane < p.batch) {
      const int s0 = min(max(p.starts[b0 + lane], 0), p.tokens), s1 = min(max(p.starts[b0 + lane + 1], s0), p.tokens);
      tiles = (static_cast<int64_t>(s1 - s0) * p.heads + ROWS - 1) / ROWS;
    }
    int64_t end = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + end > at);
    if (hit) {
      const int src = __ffs(hit) - 1;
      b_out = b0 + src;
      tile_out = static_cast<int>(__shfl_sync(0xffffffffu, before + end - 1 - at, src));
      return;
    }
    before += __shfl_sync(0xffffffffu, end, 31);
  }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1) kv4_prompt_kernel(const __grid_constant__ Kv4AttendParams p) {
  using S = Shape<D>;
  constexpr int NQ = S::kNQ, KT = S::kKeys, kRows = S::kRows, kBlock = kv4_block_bytes(D, G), ng = D / G;
  constexpr int W = kv4_width(D), nw = W / 32, kHalves = D / W, kGroups = ng / kHalves, kWordsPerGroup = G / 32;
  constexpr uint32_t kFormat = T::kIsBf16 ? 1 : 0;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  Header* hd = reinterpret_cast<Header*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &hd->abort_flag;

  if (warp == S::kMmaWarp) {
    tmem_alloc(&hd->tmem, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&hd->k_full[i], 128);
      mbar_init(&hd->k_empty[i], 1);
      mbar_init(&hd->v_full[i], 128);
      mbar_init(&hd->v_empty[i], 1);
      mbar_init(&hd->s_full[i], 1);
      mbar_init(&hd->p_full[i], 128);
      mbar_init(&hd->o_full[i], 1);
    }
    for (int i = 0; i < NQ; ++i) mbar_init(&hd->q_full[i], 128);
    mbar_fence_init();
    hd->abort_flag = 0;
    hd->bad_page = 0;
  }
  tc_fence_before_sync();
  __syncthreads();
  // Only now, with the tensor memory in hand: a dependent that allocates too and then waits for this grid must not find
  // this CTA without it, since the two would wait for one another.
  grid_launch_dependents();
  grid_dependency_wait();
  const int part = blockIdx.x % p.splits, item = blockIdx.x / p.splits, h = item % p.kv_heads;
  if (warp == 0) {
    int b, tile;
    find_tile<kRows>(p, item / p.kv_heads, b, tile);
    if (lane == 0) {
      hd->b = b;
      hd->tile = tile;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = hd->tmem;
  const int b = hd->b, tile = hd->tile;
  if (b < p.batch) {
    const int q0 = min(max(p.starts[b], 0), p.tokens), n_tok = min(max(p.starts[b + 1], q0), p.tokens) - q0;
    const int len = min(max(p.lens[b], 0), p.max_blocks * kKv4Tokens);
    const int rows = n_tok * p.heads;                 // of the sequence
    const int row_base = tile * kRows;
    int tiles_of[NQ], n_max = 0;                      // tiles of keys that a tile of rows sees
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int last = min(rows, row_base + (i + 1) * 128) - 1;
      int limit = p.causal ? len - n_tok + last / p.heads + 1 : len;
      if (last < row_base + i * 128) limit = 0;       // no rows
      tiles_of[i] = (max(0, min(limit, len)) + KT - 1) / KT;
      n_max = max(n_max, tiles_of[i]);
    }
    // with few tiles of rows several CTAs share one: each takes a run of the tiles of keys, from tile `first`
    const int first = p.splits > 1 ? static_cast<int>(static_cast<int64_t>(n_max) * part / p.splits) : 0;
    if (p.splits > 1) {
      const int end = static_cast<int>(static_cast<int64_t>(n_max) * (part + 1) / p.splits);
      n_max = end - first;
#pragma unroll
      for (int i = 0; i < NQ; ++i) tiles_of[i] = max(0, min(tiles_of[i], end) - first);
    }
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_ld;

    if (warp < S::kSoftmaxWarps) {
      // ==== softmax ====
      const int i = warp >> 2, quarter = warp & 3, row = row_base + i * 128 + quarter * 32 + lane;
      const int token = row / p.heads, head = h * p.heads + row - token * p.heads;
      {
        // ---- the warp's 32 query rows: K-major, 64 elements a 128-byte row, 16-byte chunks swizzled.  D / 8 lanes read a
        // row; lane r knows where row r is ----
        const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u;  // the scale's, so that the largest product is the largest score
        const int64_t at = row < rows ? static_cast<int64_t>(q0 + token) * p.q_tok + static_cast<int64_t>(head) * p.q_head : -1;
        uint8_t* dst = smem + S::q + i * S::kQBytes + quarter * 32 * 128;
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 8 * kAtOnce) {
          uint4 x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int64_t from = __shfl_sync(0xffffffffu, at, (r0 + k * kAtOnce + lane / kLanes) & 31);
            x[k] = from >= 0 ? *reinterpret_cast<const uint4*>(p.q + from + lane % kLanes * 8) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = r0 + k * kAtOnce + lane / kLanes, ch = lane % kLanes;
            if (r < 32)
              *reinterpret_cast<uint4*>(dst + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) =
                  make_uint4(x[k].x ^ sign, x[k].y ^ sign, x[k].z ^ sign, x[k].w ^ sign);
          }
        }
        fence_async_proxy();
        mbar_arrive(&hd->q_full[i]);
      }
      const uint32_t t_s = tmem + i * 256 + (static_cast<uint32_t>(quarter * 32) << 16), t_o = t_s + 128;
      const int n = NQ == 1 || i == 0 ? tiles_of[0] : tiles_of[NQ - 1];
      int sees = p.causal ? len - n_tok + row / p.heads + 1 : len;
      if (row >= rows) sees = len;  // (a row of zeros that nobody reads)
      sees = min(sees, len);
      int all_see = sees;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, o));
      const float scale = fabsf(p.scale);
      float top = -INFINITY, sum = 0.f;
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int key0 = (first + j) * KT;
        mbar_wait(&hd->s_full[i], j & 1, abort_flag, p.status, 920);
        tc_fence_after_sync();
        uint32_t gone = 0;  // blocks of the tile whose page does not exist: masked (looked up if the sequence has any)
        if (*static_cast<volatile int*>(&hd->bad_page)) {
          const int blk = key0 / kKv4Tokens + lane;
          if (lane < KT / kKv4Tokens && blk * kKv4Tokens < len) {
            const int page = table[p.page_shift >= 0 ? blk >> p.page_shift : blk / p.page_blocks];
            gone = page < 0 || page >= p.num_pages;
          }
          gone = __ballot_sync(0xffffffffu, gone);
        }
        const bool masked = key0 + KT > all_see || gone;
        // once over the tile for its maximum, once for the probabilities, which are stored over the scores that have been
        // read; the next 16 columns are on their way while the last ones are worked on
        float most = masked ? tile_max<KT, true>(t_s, sees - key0, gone) : tile_max<KT, false>(t_s, 0, 0);
        most *= scale;  // (NaN for a row that sees nothing of the tile at a scale of 0: ignored)
        if (__any_sync(0xffffffffu, most - top > T::kRaise)) {
          const float m = fmaxf(most - T::kTopWeight, top), f = top == m ? 1.f : exp2_approx(top - m);
          top = m;
          sum *= f;
          if (j > 0) {
            mbar_wait(&hd->o_full[i], (j - 1) & 1, abort_flag, p.status, 921);
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t x[32];
              tmem_ld_x32(t_o + c * 32, x);
              wait_ld_x32(x);
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
              tmem_st_x32(t_o + c * 32, x);
            }
          }
        }
        const float base = top == -INFINITY ? 0.f : -top;
        sum += masked ? tile_exp<T, KT, true>(t_s, scale, base, sees - key0, gone) : tile_exp<T, KT, false>(t_s, scale, base, 0, 0);
        tc_wait_st();
        tc_fence_before_sync();
        mbar_arrive(&hd->p_full[i]);
      }
      // ---- the rows' results ----
      bool last = true;
      if (n > 0) {
        mbar_wait(&hd->o_full[i], (n - 1) & 1, abort_flag, p.status, 922);
        tc_fence_after_sync();
      }
      // Parts of a row: {maximum, sum}, then its sums of values, four at a time, a row next to the other.  The last CTA adds
      // them in the order of the keys, two parts' sums on their way at a time.
      constexpr int kPart = 128 * (D + 2);
      const float* parts = p.partials + (static_cast<int64_t>(item) * NQ + i) * p.splits * kPart;
      if (p.splits > 1) {
        const int r = quarter * 32 + lane;
        float* mine = p.partials + ((static_cast<int64_t>(item) * NQ + i) * p.splits + part) * kPart;
        *reinterpret_cast<float2*>(mine + 2 * r) = make_float2(top, sum);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t x[32];
          if (n > 0) {
            tmem_ld_x32(t_o + c * 32, x);
            wait_ld_x32(x);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(mine + 256 + (c * 8 + e) * 512 + r * 4) = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        }
        named_bar_sync(1 + i, 128);
        if (quarter == 0 && lane == 0) {
          __threadfence();
          const uint32_t before = atomicAdd(p.counters + item * NQ + i, 1u);
          hd->last[i] = before == static_cast<uint32_t>(p.splits - 1);
          if (hd->last[i]) p.counters[item * NQ + i] = 0;
          __threadfence();
        }
        named_bar_sync(1 + i, 128);
        last = hd->last[i];
        if (last) {
          top = -INFINITY;
          sum = 0.f;
#pragma unroll 1
          for (int k = 0; k < p.splits; ++k) top = fmaxf(top, __ldcg(parts + k * kPart + 2 * r));
#pragma unroll 1
          for (int k = 0; k < p.splits; ++k) {
            const float2 st = __ldcg(reinterpret_cast<const float2*>(parts + k * kPart + 2 * r));
            sum = fmaf(st.y, st.x == -INFINITY ? 1.f : exp2_approx(st.x - top), sum);
          }
        }
      }
      const float inv = sum == 0.f ? 0.f : Dequant<T>::kBack / sum;
      if (last) {
        // to the place of the warp's query rows (their products are done) and from there, a row by D / 8 lanes
        uint8_t* stage = smem + S::q + i * S::kQBytes + quarter * 32 * 128;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (p.splits > 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
#pragma unroll 2
            for (int k = 0; k < p.splits; ++k) {
              const float* from = parts + k * kPart;
              const int rr = quarter * 32 + lane;
              const float2 st = __ldcg(reinterpret_cast<const float2*>(from + 2 * rr));
              const float f = st.x == -INFINITY ? 1.f : exp2_approx(st.x - top);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(from + 256 + (c * 8 + e) * 512 + rr * 4));
                const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) r[4 * e + q] = __float_as_uint(fmaf(xs[q], f, __uint_as_float(r[4 * e + q])));
              }
            }
          } else if (n > 0) {
            tmem_ld_x32(t_o + c * 32, r);
            wait_ld_x32(r);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = sum != 0.f ? T::pack(__uint_as_float(r[e * 8 + k * 2]) * inv, __uint_as_float(r[e * 8 + k * 2 + 1]) * inv) : 0u;
            const int ch = c * 4 + e;
            *reinterpret_cast<uint4*>(stage + (ch >> 3) * (128 * 128) + lane * 128 + (((ch & 7) ^ (lane & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        {
          const int64_t at = row < rows ? static_cast<int64_t>(q0 + token) * p.o_tok + static_cast<int64_t>(head) * p.o_head : -1;
          constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
#pragma unroll 4
          for (int r0 = 0; r0 < 32; r0 += kAtOnce) {
            const int r = r0 + lane / kLanes, ch = lane % kLanes;
            const int64_t to = __shfl_sync(0xffffffffu, at, r);
            const uint4 x = *reinterpret_cast<const uint4*>(stage + (ch >> 3) * (128 * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
            if (to >= 0) *reinterpret_cast<uint4*>(p.out + to + ch * 8) = x;
          }
        }
      }
      tc_fence_before_sync();
    } else if (warp < S::kMmaWarp) {
      const int dw = warp - S::kDequantWarp0;
      // lane i < KT / 16 has the page of block i of a tile; fetched a tile before it is needed
      auto fetch_pages = [&](int j) -> int {
        const int key = (first + j) * KT + lane * kKv4Tokens, blk = key / kKv4Tokens;
        if (lane >= KT / kKv4Tokens || key >= len) return -1;
        const int page = table[p.page_shift >= 0 ? blk >> p.page_shift : blk / p.page_blocks];
        if (page < 0 || page >= p.num_pages) {
          *static_cast<volatile int*>(&hd->bad_page) = 1;
          p.status[kBadPageWord] = 1;
        }
        return page;
      };
      // block `at` of tile j (for key `at` < len); null: no key, or its page does not exist
      auto block_at = [&](int pages, int j, int at) -> const uint8_t* {
        const int page = __shfl_sync(0xffffffffu, pages, at), blk = (first + j) * (KT / kKv4Tokens) + at;
        if (page < 0 || page >= p.num_pages) return nullptr;
        const int inner = p.page_shift >= 0 ? blk & (p.page_blocks - 1) : blk % p.page_blocks;
        return p.cache + ((static_cast<int64_t>(page) * p.kv_heads + h) * p.page_blocks + inner) * kBlock;
      };
      // ==== keys: a thread has words [t][..] of four rows (and halves) of a tile.  Lanes: 8 rows x 4 words, so that eight
      // lanes of one t write eight rows' chunks to different banks ====
      constexpr int kItems = KT * 4 * kHalves / 128;
      uint32_t kw[kItems][nw], kpar[kItems][kGroups];
      auto row_of = [&](int it) { return (it / kHalves * 4 + dw) * 8 + (lane & 7); };
      const int t = lane >> 3;
      auto load_keys = [&](int j, int pages) {
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
          const int hh = it % kHalves, r = row_of(it) % kKv4Tokens;
          const uint8_t* blk = block_at(pages, j, row_of(it) / kKv4Tokens);
          if (blk) {
            load_words(blk + r * (D / 2) + hh * 64 + t * nw * 4, kw[it]);
            load_words(blk + kv4_key_params(D) + (r * ng + hh * kGroups) * 4, kpar[it]);
          } else {
#pragma unroll
            for (int k = 0; k < nw; ++k) kw[it][k] = 0;
#pragma unroll
            for (int k = 0; k < kGroups; ++k) kpar[it][k] = 0;
          }
        }
      };
      auto put_keys = [&](int j) {
        uint8_t* dst = smem + S::k + (j & 1) * S::kKBytes;
        if (j >= 2) mbar_wait(&hd->k_empty[j & 1], ((j >> 1) - 1) & 1, abort_flag, p.status, 923);
#pragma unroll
        for (int it = 0; it < kItems; ++it) {
          const int row = row_of(it), hh = it % kHalves;
          Dequant<T> dq;
#pragma unroll
          for (int k = 0; k < nw; ++k) {
            if (k % kWordsPerGroup == 0) dq.same(kpar[it][k / kWordsPerGroup]);
            uint32_t x[4];
            dq.values(kw[it][k], x);
            const int ch = hh * 16 + 4 * k + t;  // 8 elements from 8 ch
            *reinterpret_cast<uint4*>(dst + (ch >> 3) * (KT * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) =
                make_uint4(x[0], x[1], x[2], x[3]);
          }
        }
        fence_async_proxy();
        mbar_arrive(&hd->k_full[j & 1]);
      };
      // ==== values: a thread has elements g + 8 n + 32 k (of a half) of eight tokens of a tile ====
      const int id = dw * 4 + (lane >> 3), g = lane & 7;
      const int hh = id % kHalves, eight = id / kHalves;  // half of the head, eight tokens
      uint32_t vw[4][nw], vpar[8][kGroups];
      auto load_values = [&](int j, int pages) {
        const int key = (first + j) * KT + eight * 8;
        const uint8_t* blk = block_at(pages, j, eight >> 1);
        const int p0 = (eight & 1) * 4;  // first pair of tokens in its block
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (blk) {
            load_words(blk + 8 * D + hh * W * 8 + (g * 8 + ((p0 + k) ^ kv4_swap(D, g))) * (nw * 4), vw[k]);
          } else {
#pragma unroll
            for (int e = 0; e < nw; ++e) vw[k][e] = 0;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (blk && key + k < len) {
            load_words(blk + kv4_value_params(D, G) + ((p0 * 2 + k) * ng + hh * kGroups) * 4, vpar[k]);
          } else {
#pragma unroll
            for (int e = 0; e < kGroups; ++e) vpar[k][e] = 0;  // tokens behind the last one hold anything
          }
        }
      };
      auto put_values = [&](int j) {
        uint8_t* dst = smem + S::v + (j & 1) * S::kKBytes;
        if (j >= 2) mbar_wait(&hd->v_empty[j & 1], ((j >> 1) - 1) & 1, abort_flag, p.status, 924);
        Dequant<T> dq[4];
#pragma unroll
        for (int k = 0; k < nw; ++k) {
          if (k % kWordsPerGroup == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dq[e].pair(vpar[2 * e][k / kWordsPerGroup], vpar[2 * e + 1][k / kWordsPerGroup]);
          }
          uint32_t x[4][4];  // [pair of tokens][n]
#pragma unroll
          for (int e = 0; e < 4; ++e) dq[e].values(vw[e][k], x[e]);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int d = hh * 128 + 32 * k + 8 * n + g;
            *reinterpret_cast<uint4*>(dst + (eight >> 3) * (D * 128) + d * 128 + (((eight & 7) ^ g) << 4)) =
                make_uint4(x[0][n], x[1][n], x[2][n], x[3][n]);
          }
        }
        fence_async_proxy();
        mbar_arrive(&hd->v_full[j & 1]);
      };
      // (the first keys' products start while the values are on their way; later loads are a tile ahead)
      int pages0 = fetch_pages(0), pages1 = fetch_pages(1), pages2 = -1;  // of tiles j, j + 1, j + 2
      if (n_max > 0) {
        load_keys(0, pages0);
        load_values(0, pages0);
        put_keys(0);
        if (n_max > 1) load_keys(1, pages1);
      }
#pragma unroll 1
      for (int j = 0; j < n_max; ++j) {
        pages2 = fetch_pages(j + 2);
        if (j + 1 < n_max) put_keys(j + 1);
        if (j + 2 < n_max) load_keys(j + 2, pages2);
        put_values(j);
        if (j + 1 < n_max) load_values(j + 1, pages1);
        pages1 = pages2;
      }
    } else {
      // ==== products.  The warp stays together and one lane issues: descriptors live in uniform registers ====
      const uint32_t id_s = umma_idesc(KT, kFormat, kFormat, 1), id_o = umma_idesc(D, kFormat, kFormat, 1);
      const uint32_t t = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint64_t q_desc = umma_desc_k128(base + S::q), k_desc = umma_desc_k128(base + S::k), v_desc = umma_desc_k128(base + S::v);
      const int n0 = __shfl_sync(0xffffffffu, tiles_of[0], 0), n1 = __shfl_sync(0xffffffffu, tiles_of[NQ - 1], 0);
      const int n_all = max(n0, n1);
      // (a descriptor's low bits are the address / 16)
      auto scores = [&](int i, int j) {
        const uint64_t q = q_desc + i * (S::kQBytes / 16), k = k_desc + (j & 1) * (S::kKBytes / 16);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            umma_f16_ss_plain(t + i * 256, q + ((s >> 2) * (128 * 128) + (s & 3) * 32) / 16, k + ((s >> 2) * (KT * 128) + (s & 3) * 32) / 16,
                        id_s, s > 0);
          tc_commit(&hd->s_full[i]);
        }
        __syncwarp();
      };
      auto values = [&](int i, int j) {
        const uint64_t v = v_desc + (j & 1) * (S::kKBytes / 16);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < KT / 16; ++s)
            umma_f16_ts_plain(t + i * 256 + 128, t + i * 256 + s * 8, v + ((s >> 2) * (D * 128) + (s & 3) * 32) / 16, id_o, j > 0 || s > 0);
          tc_commit(&hd->o_full[i]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
      };
      if (n_all > 0) {
        mbar_wait(&hd->k_full[0], 0, abort_flag, p.status, 925);
#pragma unroll 1
        for (int i = 0; i < NQ; ++i) {
          mbar_wait(&hd->q_full[i], 0, abort_flag, p.status, 930);
          tc_fence_after_sync();
          if ((i ? n1 : n0) > 0) scores(i, 0);
        }
        commit(&hd->k_empty[0]);
      }
#pragma unroll 1
      for (int j = 0; j < n_all; ++j) {
        mbar_wait(&hd->v_full[j & 1], (j >> 1) & 1, abort_flag, p.status, 926);
        if (j + 1 < n_all) mbar_wait(&hd->k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, abort_flag, p.status, 927);
#pragma unroll 1
        for (int i = 0; i < NQ; ++i) {
          const int n = i ? n1 : n0;
          if (j < n) {
            mbar_wait(&hd->p_full[i], j & 1, abort_flag, p.status, 928);
            tc_fence_after_sync();
            values(i, j);
          }
          if (j + 1 < n) scores(i, j + 1);
        }
        commit(&hd->v_empty[j & 1]);
        if (j + 1 < n_all) commit(&hd->k_empty[(j + 1) & 1]);
      }
      // the last commits of the barriers that nobody waits for end with the products before them
      if (n_all > 0) mbar_wait(&hd->v_empty[(n_all - 1) & 1], ((n_all - 1) >> 1) & 1, abort_flag, p.status, 929);
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (warp == S::kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// tiles of rows times kv heads, at most
int64_t prompt_items(int batch, int64_t tokens, int heads, int kv_heads, int d) {
  return (ceil_div(tokens * heads, d == 256 ? 128 : 256) + batch) * kv_heads;
}

template <typename T, int D, int G>
cudaError_t launch_one(const Kv4AttendParams& p, cudaStream_t stream) {
  using S = Shape<D>;
  auto kernel = kv4_prompt_kernel<T, D, G>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::total)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(prompt_items(p.batch, p.tokens, p.heads, p.kv_heads, D) * p.splits));
  cfg.blockDim = dim3(S::kThreads);
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

template <typename T>
cudaError_t launch_shape(const Kv4AttendParams& p, int d, int g, cudaStream_t stream) {
  if (d == 64 && g == 32) return launch_one<T, 64, 32>(p, stream);
  if (d == 64 && g == 64) return launch_one<T, 64, 64>(p, stream);
  if (d == 128 && g == 32) return launch_one<T, 128, 32>(p, stream);
  if (d == 128 && g == 64) return launch_one<T, 128, 64>(p, stream);
  if (d == 128 && g == 128) return launch_one<T, 128, 128>(p, stream);
  if (d == 256 && g == 32) return launch_one<T, 256, 32>(p, stream);
  if (d == 256 && g == 64) return launch_one<T, 256, 64>(p, stream);
  if (d == 256 && g == 128) return launch_one<T, 256, 128>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

// CTAs that share a tile of rows: as many as there are SMs for, where the cache can hold four tiles of keys for each.
// 100 tokens of 32 heads behind 5000 cached ones take 42.8 us with six CTAs a tile and 99.6 with one, 64 of 8 heads behind
// 60,000 105 us against 1038.  Two tiles of keys for each: 200 tokens of 8 heads behind 3000 38.4 us against 35.6 with
// four, 100 tokens of 32 heads behind 1000 27.6 against 29.8.
int kv4_prompt_splits(int batch, int64_t tokens, int heads, int kv_heads, int d, int64_t max_keys, int num_sms) {
  const int64_t by_sms = num_sms / prompt_items(batch, tokens, heads, kv_heads, d), by_keys = max_keys / (4 * (d == 256 ? 64 : 128));
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({by_sms, by_keys, 16})));
}
size_t kv4_prompt_partial_bytes(int batch, int64_t tokens, int heads, int kv_heads, int d, int num_sms) {
  const int64_t items = prompt_items(batch, tokens, heads, kv_heads, d);
  return items * 2 > num_sms ? 0 : static_cast<size_t>(num_sms) * (d == 256 ? 1 : 2) * 128 * (d + 2) * 4;
}

cudaError_t launch_kv4_prompt(const Kv4AttendParams& p, int f16, int d, int g, cudaStream_t stream) {
  return f16 ? launch_shape<Kv4Fp16>(p, d, g, stream) : launch_shape<Kv4Bf16>(p, d, g, stream);
}

}  // namespace woq
