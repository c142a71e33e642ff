// Writing tokens to the paged 4-bit key/value cache, with the position rotation of queries and keys on the way, and
// reading them back.  Layout: woq_kv4_common.cuh.
//
//   x = rotated row, rounded to its type T (keys), or the row as it is (values); for every group of G elements
//   m = min x,  s = T toward zero((max x - m) / 15),  c = clamp(rint((x - m) / s), 0, 15)  (0 where s is 0)
// s is rounded toward zero so that no c * s + m passes T's largest value.
#include "woq_kernels.h"
#include "woq_kv4_common.cuh"

namespace woq {

namespace {

__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// a * c - b * s for two pairs with an error below two units of the result's last place, whatever cancels
// (Kahan's difference of products): rotated keys decide codes, and a product rounded on its own would move some of them.
__device__ __forceinline__ float2 diff_of_products(uint64_t a, uint64_t c, uint64_t b, uint64_t s) {
  const uint64_t p = mul2(b, s) ^ 0x8000000080000000ull;  // -(b s)
  return halves2(fma2(fma2(b, s, p), pair2(-1.f, -1.f), fma2(a, c, p)));
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = T::lo(w[i]);
    x[2 * i + 1] = T::hi(w[i]);
  }
}

// Codes of 8 neighbouring elements of a row whose group is spread over LG lanes, and the group's parameters.
// Differences are taken of halves: max - min of T's extremes passes the largest fp32.
template <typename T, int LG>
__device__ __forceinline__ void quantise8(const float (&x)[8], uint32_t (&c)[8], uint32_t& param, bool& finite) {
  float lo = x[0], hi = x[0];
  finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite = finite && fabsf(x[i]) < T::kTooLarge;
  }
#pragma unroll
  for (int o = 1; o < LG; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // Toward zero: 15 times a number of T has at most 15 digits, so the range in 32 bits, cut, reaches it where the true one does,
  // and a quotient that was rounded up to a number of T is told by its product.
  const float range = __fsub_rz(hi * 0.5f, lo * 0.5f);
  uint16_t s16 = T::from_float_rz(__fdiv_rn(range, 7.5f));
  if (T::to_float(s16) * 7.5f > range) --s16;
  const float s = T::to_float(s16) * 0.5f, m = lo * 0.5f;
  // The quotient by the scale's reciprocal is within 2^-19 of the true one (two roundings of a number up to 15.2): where it
  // is that near a tie, the division decides, and everywhere for steps of up to 2^-127, whose halves have no finite
  // reciprocal.  Adding 1.5 2^23 leaves the rounded quotient in the low bits.
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  const float clear = inv < INFINITY ? 0.5f - 1.f / 131072.f : -1.f;
  bool near_tie = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = fminf(fmaf(x[i], 0.5f, -m) * inv, 15.f), r = t + 12582912.f;
    c[i] = __float_as_uint(r) & 15u;
    near_tie = near_tie || !(fabsf(t - (r - 12582912.f)) <= clear);
  }
  if (near_tie && s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = fminf(__fdiv_rn(fmaf(x[i], 0.5f, -m), s), 15.f);
      c[i] = __float_as_uint(t + 12582912.f) & 15u;
    }
  }
  param = static_cast<uint32_t>(s16) | static_cast<uint32_t>(T::from_float(lo)) << 16;
}

// One CTA per token (and part of its rows): D / 8 lanes a row, 8 elements a lane.  Rows are the query heads, then the
// key heads, then the value heads; a thread keeps its 8 elements' angles over all rows.  Bound by the latency of a CTA's trips
// to memory (slot and position, angles, queries, keys and values), which 28 warps an SM do not cover: nearly half of the
// stalls are waits for loads, 63 % of the issue slots are used, DRAM is at a third.  8000 tokens of 64 + 2 x 8 heads of 128
// 93 us (3.3 TB/s of 6.6), 1001 of 25 + 2 x 5 heads of 64 7.7 us, 8 tokens 2.8 us.
template <typename T, int D, int G>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(Kv4AppendParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, LG = G / 8, ng = D / G;
  const int64_t token = blockIdx.x;
  const int sub = threadIdx.x % kLanes, row0 = threadIdx.x / kLanes;
  grid_launch_dependents();
  grid_dependency_wait();
  const int step = kRows * gridDim.y, start = row0 + static_cast<int>(blockIdx.y) * kRows;
  // the first rows are on their way while slots, positions and angles are looked up
  const uint16_t* q_src = p.q + token * p.q_tok + sub * 8;
  const int q_last = p.q_heads - 1;
  uint4 ahead = make_uint4(0, 0, 0, 0);
  if (p.q_heads > 0) ahead = *reinterpret_cast<const uint4*>(q_src + min(start, q_last) * p.q_head);
  const int64_t slot = p.slots[token], pos = p.positions ? p.positions[token] : 0;
  const bool bad_pos = p.rot > 0 && (pos < 0 || pos >= p.max_pos);
  const bool store = !bad_pos && slot >= 0 && slot < p.num_slots;

  // angles of the lane's elements: x[i] * c[i] - partner * s[i], the sign of s says which of the pair it is
  uint64_t cs[4], sn[4];
  const int half = p.rot / 2, lane_rot = p.rot / 8;
  const bool turns = sub < lane_rot;
  if (turns && !bad_pos) {
    const float* t = p.cos_sin + pos * p.rot;
    if (p.interleaved) {  // (table rows start at multiples of 16 bytes: rot is a multiple of 16)
      const float4 c = *reinterpret_cast<const float4*>(t + sub * 4), s = *reinterpret_cast<const float4*>(t + half + sub * 4);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = pair2(cc[i], cc[i]);
        sn[i] = pair2(ss[i], -ss[i]);
      }
    } else {
      const bool second = sub >= lane_rot / 2;
      const float4* c = reinterpret_cast<const float4*>(t + (second ? sub - lane_rot / 2 : sub) * 8);
      const float4* s = reinterpret_cast<const float4*>(t + half + (second ? sub - lane_rot / 2 : sub) * 8);
      const float sign = second ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 a = c[i], b = s[i];
        cs[2 * i] = pair2(a.x, a.y);
        cs[2 * i + 1] = pair2(a.z, a.w);
        sn[2 * i] = pair2(sign * b.x, sign * b.y);
        sn[2 * i + 1] = pair2(sign * b.z, sign * b.w);
      }
    }
  }
  // lane of the row that holds the partners (rotation of halves): whole lanes, since rot is a multiple of 16
  const int mate = (threadIdx.x & 31) - sub % kLanes + (sub < lane_rot / 2 ? sub + lane_rot / 2 : turns ? sub - lane_rot / 2 : sub);

  // what a lane holds of a row, rotated
  auto rotate = [&](const uint4& raw) -> uint4 {
    uint4 other;
    if (p.interleaved) {  // the neighbour within the pair
      other = make_uint4(__byte_perm(raw.x, 0, 0x1032), __byte_perm(raw.y, 0, 0x1032), __byte_perm(raw.z, 0, 0x1032),
                         __byte_perm(raw.w, 0, 0x1032));
    } else {
      other.x = __shfl_sync(0xffffffffu, raw.x, mate);
      other.y = __shfl_sync(0xffffffffu, raw.y, mate);
      other.z = __shfl_sync(0xffffffffu, raw.z, mate);
      other.w = __shfl_sync(0xffffffffu, raw.w, mate);
    }
    if (!turns || bad_pos) return raw;
    const uint32_t a[4] = {raw.x, raw.y, raw.z, raw.w}, b[4] = {other.x, other.y, other.z, other.w};
    uint32_t z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 y = diff_of_products(pair2(T::lo(a[i]), T::hi(a[i])), cs[i], pair2(T::lo(b[i]), T::hi(b[i])), sn[i]);
      z[i] = T::pack(y.x, y.y);
    }
    return make_uint4(z[0], z[1], z[2], z[3]);
  };
  // ---- queries.  (The whole warp takes part in every round: shuffles; rows past the end repeat the last one and store
  // nothing.)  The next round's row is on its way while this one is rotated ----
  if (p.q_heads > 0) {
    uint16_t* dst = p.q_out + token * p.q_heads * D + sub * 8;
    for (int head = start; head - row0 <= q_last; head += step) {
      const uint4 raw = ahead;
      ahead = *reinterpret_cast<const uint4*>(q_src + min(head + step, q_last) * p.q_head);
      uint4 out = p.rot > 0 ? rotate(raw) : raw;
      if (bad_pos) out = make_uint4(T::kNan * 0x10001u, T::kNan * 0x10001u, T::kNan * 0x10001u, T::kNan * 0x10001u);
      if (head <= q_last) *reinterpret_cast<uint4*>(dst + head * D) = out;
    }
  }
  // ---- keys, then values ----
  if (!store) return;  // (the token's, not the lane's)
  const int64_t block = slot / kKv4Tokens;
  const int r = static_cast<int>(slot % kKv4Tokens);
  const int64_t page = block / p.page_blocks, inner = block % p.page_blocks;
  const int rows = 2 * p.kv_heads;
  // (CTAs that the queries leave idle first: the rounds go on where those ended)
  for (int row = row0 + static_cast<int>((gridDim.y - 1 - blockIdx.y)) * kRows; row - row0 < rows; row += step) {
    const bool live = row < rows;
    const int rr = live ? row : rows - 1;
    const bool is_k = rr < p.kv_heads;
    const int head = is_k ? rr : rr - p.kv_heads;
    const uint4 value = *reinterpret_cast<const uint4*>(p.v + token * p.v_tok + head * p.v_head + sub * 8);
    uint4 raw = value;
    if (is_k) raw = *reinterpret_cast<const uint4*>(p.k + token * p.k_tok + head * p.k_head + sub * 8);
    if (p.rot > 0) {
      const uint4 turned = rotate(raw);
      if (is_k) raw = turned;
    }
    float x[8];
    unpack8<T>(raw, x);
    uint32_t c[8], param;
    bool finite;
    quantise8<T, LG>(x, c, param, finite);
    // Nothing non-finite is kept among the values: a masked row multiplies them by zero.  The token's key says it
    // instead (its scores are NaN for the rows that see it, and only for those).
    if (is_k) {
      float y[8];
      unpack8<T>(value, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) finite = finite && fabsf(y[i]) < T::kTooLarge;
    }
    const uint32_t bad = __ballot_sync(0xffffffffu, !finite);
    const uint32_t row_mask = kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1) << ((threadIdx.x & 31) / kLanes * kLanes);
    if (bad & row_mask) {
      param = is_k ? T::kNan * 0x10001u : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = 0;
    }
    uint8_t* blk = p.cache + ((page * p.kv_heads + head) * p.page_blocks + inner) * kv4_block_bytes(D, G);
    // four lanes 4 j .. 4 j + 3 hold elements 32 j + 8 n + g of nibble n: each leaves with two g of all four
    uint32_t w[4];
    const int n = sub & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (c[2 * i] | c[2 * i + 1] << 16) << (4 * n);
    const uint32_t give = n & 2 ? w[0] : w[2], give2 = n & 2 ? w[1] : w[3];
    const uint32_t a = (n & 2 ? w[2] : w[0]) | __shfl_xor_sync(0xffffffffu, give, 2);
    const uint32_t b = (n & 2 ? w[3] : w[1]) | __shfl_xor_sync(0xffffffffu, give2, 2);
    const uint32_t mine = (n & 1 ? b : a) | __shfl_xor_sync(0xffffffffu, n & 1 ? a : b, 1);
    if (live && is_k) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) word |= c[i] << (4 * ((i >> 1) + 4 * (i & 1)));
      *reinterpret_cast<uint32_t*>(blk + kv4_key_word(D, r, sub)) = word;
      if (sub % LG == 0) *reinterpret_cast<uint32_t*>(blk + kv4_key_params(D) + (r * ng + sub / LG) * 4) = param;
    } else if (live) {
      const int g0 = 2 * n, hh = sub / 16, j = (sub % 16) / 4;
      *reinterpret_cast<uint16_t*>(blk + kv4_value_half(D, r, hh, j, g0)) = static_cast<uint16_t>(mine & 0xffffu);
      *reinterpret_cast<uint16_t*>(blk + kv4_value_half(D, r, hh, j, g0 + 1)) = static_cast<uint16_t>(mine >> 16);
      if (sub % LG == 0) *reinterpret_cast<uint32_t*>(blk + kv4_value_params(D, G) + (r * ng + sub / LG) * 4) = param;
    }
  }
}

// One CTA per 16 listed slots and head (slots that follow one another share a block, whose sectors then come from
// L1): D / 8 lanes a row.  Slots outside the cache give zeros.  Bound by its instructions and the trips in front of them (a
// value's eight codes come in eight loads of two bytes, behind the slot's): three quarters of the issue slots are used, the
// bytes pass at 3.8 of 6.6 TB/s.  8000 tokens of 8 heads of 128 11 us.
template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4ReadParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, LG = G / 8, ng = D / G;
  const int sub = threadIdx.x % kLanes, row0 = threadIdx.x / kLanes;
  const int head = blockIdx.y;
  grid_launch_dependents();
  grid_dependency_wait();
  for (int row = row0; row < 2 * kKv4Tokens; row += kRows) {
    const int64_t token = static_cast<int64_t>(blockIdx.x) * kKv4Tokens + (row & 15);
    const bool value = row >= kKv4Tokens;
    if (token >= p.tokens) continue;
    const int64_t slot = p.slots[token];
    uint4 out = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot < p.num_slots) {
      const int64_t block = slot / kKv4Tokens, page = block / p.page_blocks, inner = block % p.page_blocks;
      const int r = static_cast<int>(slot % kKv4Tokens);
      const uint8_t* blk = p.cache + ((page * p.kv_heads + head) * p.page_blocks + inner) * kv4_block_bytes(D, G);
      const uint32_t param = *reinterpret_cast<const uint32_t*>(
          blk + (value ? kv4_value_params(D, G) : kv4_key_params(D)) + (r * ng + sub / LG) * 4);
      const uint32_t s2 = __byte_perm(param, 0, 0x1010), m2 = __byte_perm(param, 0, 0x3232);
      uint32_t w[4];
      if (!value) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + kv4_key_word(D, r, sub));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = word >> (4 * i);
      } else {
        const int hh = sub / 16, j = (sub % 16) / 4, n = sub & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = *reinterpret_cast<const uint16_t*>(blk + kv4_value_half(D, r, hh, j, 2 * i));
          const uint32_t b = *reinterpret_cast<const uint16_t*>(blk + kv4_value_half(D, r, hh, j, 2 * i + 1));
          w[i] = (a | b << 16) >> (4 * n);
        }
      }
      out = make_uint4(kv4_dequant2<T>(w[0], s2, m2), kv4_dequant2<T>(w[1], s2, m2), kv4_dequant2<T>(w[2], s2, m2),
                       kv4_dequant2<T>(w[3], s2, m2));
    }
    uint16_t* dst = value ? p.v : p.k;
    *reinterpret_cast<uint4*>(dst + (token * p.kv_heads + head) * D + sub * 8) = out;
  }
}

template <typename P>
cudaError_t launch(void (*kernel)(P), dim3 grid, cudaStream_t stream, const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
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

// the instance for a head width and group, or null
template <typename P, template <typename, int, int> class K>
void (*pick(int dtype_f16, int d, int g))(P) {
#define KV4_CASE(D, G) if (d == D && g == G) return dtype_f16 ? K<Kv4Fp16, D, G>::kernel() : K<Kv4Bf16, D, G>::kernel()
  KV4_CASE(64, 32);
  KV4_CASE(64, 64);
  KV4_CASE(128, 32);
  KV4_CASE(128, 64);
  KV4_CASE(128, 128);
  KV4_CASE(256, 32);
  KV4_CASE(256, 64);
  KV4_CASE(256, 128);
#undef KV4_CASE
  return nullptr;
}
template <typename T, int D, int G>
struct AppendKernel {
  static void (*kernel())(Kv4AppendParams) { return kv4_append_kernel<T, D, G>; }
};
template <typename T, int D, int G>
struct ReadKernel {
  static void (*kernel())(Kv4ReadParams) { return kv4_read_kernel<T, D, G>; }
};

}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendParams& p, int f16, int d, int g, int64_t tokens, cudaStream_t stream) {
  const int rows = p.q_heads + 2 * p.kv_heads, per = 256 / (d / 8);
  // few tokens: a token's rows over several CTAs, as many as find room at two an SM (8 tokens 2.8 us against 3.5 with one;
  // eight an SM: 148 tokens 4.4 us against 3.5, 300 5.3 against 5.8)
  int parts = (rows + per - 1) / per;
  while (parts > 1 && tokens * parts > 2 * 148) parts = (parts + 1) / 2;
  return launch(pick<Kv4AppendParams, AppendKernel>(f16, d, g), dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(parts)), stream, p);
}

cudaError_t launch_kv4_read(const Kv4ReadParams& p, int f16, int d, int g, cudaStream_t stream) {
  return launch(pick<Kv4ReadParams, ReadKernel>(f16, d, g),
                dim3(static_cast<unsigned>(ceil_div(p.tokens, kKv4Tokens)), static_cast<unsigned>(p.kv_heads)), stream, p);
}

}  // namespace woq
