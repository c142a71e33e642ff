// The paged 4-bit key/value cache: layout of a block and the arithmetic on its codes.  sm_100a only.
#pragma once
#include <cuda_fp16.h>

#include "woq_common.cuh"

namespace woq {

// ---------------------------------------------------------------------------------------
// The cache is [page][kv head][page size / 16] blocks.  A block holds 16 tokens of one head of D elements in
// groups of G (`ng` = D / G groups a row), one contiguous range for a bulk copy:
//   8 D bytes      codes of the keys
//   8 D bytes      codes of the values
//   64 ng bytes    {scale, lowest} of the keys, [token][group], 16-bit floats of the keys' type T
//   64 ng bytes    {scale, lowest} of the values
// A code c stands for T(c * scale + lowest), one rounding.
//
// Both code areas are fragments of m16n8k16 A operands (keys as rows, or transposed values as rows), so that a lane
// fetches its nibbles with wide loads and (word >> 4 n) & 0x000f000f is one register of two codes.  Rows of 256
// elements are two halves of 128; W = min(D, 128), nw = W / 32.
//   keys:   row of token r at r * D / 2; inside it [half][t][j] 32-bit words, t = 0..3, j < nw, of elements
//           128 half + 32 j + 8 t + e: nibble e / 2 for even e, 4 + e / 2 for odd e (two neighbours a register)
//   values: [half][g][slot][j] words, g = 0..7, of elements 128 half + 32 j + 8 n + g in nibble n (n = 0..3) of a
//           half-word: the low one of token 2 p, the high one of token 2 p + 1; slot = p ^ kv4_swap(D, g), which
//           spreads the four pairs that a quarter of a warp reads over all banks
// A token's codes of one element row never share a byte with another token's.
// ---------------------------------------------------------------------------------------
constexpr int kKv4Tokens = 16;

__host__ __device__ constexpr int kv4_width(int d) { return d < 128 ? d : 128; }
__host__ __device__ constexpr int kv4_block_bytes(int d, int g) { return 16 * d + 128 * (d / g); }
__host__ __device__ constexpr int kv4_key_params(int d) { return 16 * d; }
__host__ __device__ constexpr int kv4_value_params(int d, int g) { return 16 * d + 64 * (d / g); }
__host__ __device__ constexpr int kv4_swap(int d, int g) { return d < 128 ? ((g >> 1) & 1) * 4 : (g & 1) * 4; }
// byte of the word that holds keys 8 i .. 8 i + 7 of token r
__host__ __device__ constexpr int kv4_key_word(int d, int r, int i) {
  const int nw = kv4_width(d) / 32, half = i / 16, ii = i % 16;
  return r * (d / 2) + half * 64 + ((ii & 3) * nw + (ii >> 2)) * 4;
}
// byte of the half-word that holds elements 128 half + 32 j + 8 n + g (n = 0..3) of token r
__host__ __device__ constexpr int kv4_value_half(int d, int r, int half, int j, int g) {
  const int w = kv4_width(d), nw = w / 32;
  return 8 * d + half * w * 8 + (g * 8 + ((r >> 1) ^ kv4_swap(d, g))) * (nw * 4) + j * 4 + (r & 1) * 2;
}

// Arithmetic of the two 16-bit types.
// Weights of the softmax are kept in the type as 2^(score - reference), in one pass with a running maximum (Milakov and
// Gimelshein, "Online normalizer calculation for softmax", 2018).  Any reference gives the same quotients; it is set
// kTopWeight below the maximum and raised when a score passes it by kRaise, so that sums are seldom rescaled.  bf16 has room
// below: weights of 1 to 2^8 at the top.  fp16 has none, and tens of thousands of small weights may be most of a result: 2^11
// to 2^15 at the top, so that weights down to 2^-25 of the largest keep all their digits and down to 2^-35 some.
struct Kv4Bf16 {
  using type = __nv_bfloat16;
  static constexpr bool kIsBf16 = true;
  static constexpr uint32_t kMagic = 0x43004300u;  // 128 + c with the code in the low bits
  static constexpr float kTooLarge = 2305843009213693952.f;  // 2^61: the attention kernel scales by 2^69
  static constexpr uint32_t kNan = 0x7fffu;
  static constexpr float kTopWeight = 0.f, kRaise = 8.f;
  static __device__ __forceinline__ float to_float(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  static __device__ __forceinline__ uint16_t from_float_rz(float v) { return __bfloat16_as_ushort(__float2bfloat16_rz(v)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {  // a in the low half
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) { return bf16x2_sub(a, b); }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ void mma(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    // (not volatile: independent products may move past one another)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
struct Kv4Fp16 {
  using type = __half;
  static constexpr bool kIsBf16 = false;
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + c
  static constexpr float kTooLarge = INFINITY;
  static constexpr uint32_t kNan = 0x7fffu;
  static constexpr float kTopWeight = 11.f, kRaise = 15.f;
  static __device__ __forceinline__ float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ float lo(uint32_t v) { return to_float(static_cast<uint16_t>(v & 0xffffu)); }
  static __device__ __forceinline__ float hi(uint32_t v) { return to_float(static_cast<uint16_t>(v >> 16)); }
  static __device__ __forceinline__ uint16_t from_float(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ uint16_t from_float_rz(float v) { return __half_as_ushort(__float2half_rz(v)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ void mma(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Two codes (`w` shifted so that they are at bits 0..3 and 16..19) to two values of T: c exactly, then one fma.
template <typename T>
__device__ __forceinline__ uint32_t kv4_dequant2(uint32_t w, uint32_t s2, uint32_t m2) {
  return T::fma2(T::sub2(lop3_and_or(w, 0x000f000fu, T::kMagic), T::kMagic), s2, m2);
}

}  // namespace woq
