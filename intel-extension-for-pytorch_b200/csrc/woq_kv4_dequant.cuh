// Codes of the paged 4-bit cache to the attention kernels' operands.  sm_100a only.
#pragma once
#include "woq_kv4_common.cuh"

namespace woq {

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// {scale, lowest} words of 16-bit floats -> what values() takes, and back from there.
//
// bf16: a nibble at bits 0..3 (4..7) of a half-word, the rest masked, is the bf16 number c 2^-133 (c 2^-129) exactly:
// the encoding is linear that far down.  Multiplied by scale 2^69 (2^65), plus lowest 2^-64, one fma gives the value
// times 2^-64 with the very rounding that it has without: two instructions for two codes, and one shift for eight.
// Scores and results are multiplied by 2^64 again in 32 bits.  (Appended values are below 2^61, so scales stay finite;
// below 2^-62 values lose digits.)
// fp16 has no such room: 1024 + c, less 1024, then the fma.
template <typename T>
struct Dequant;
template <>
struct Dequant<Kv4Bf16> {
  static constexpr float kBack = 18446744073709551616.f;  // 2^64
  uint32_t se, so, m;
  static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) { return bf16x2_mul(a, b); }
  // both halves from one word
  __device__ __forceinline__ void same(uint32_t param) {
    const uint32_t x = mul2(param, 0x1f806200u);  // {2^69, 2^-64}
    se = __byte_perm(x, 0, 0x1010);
    m = __byte_perm(x, 0, 0x3232);
    so = mul2(se, 0x3d803d80u);  // 2^-4
  }
  // the low half from one word, the high half from another
  __device__ __forceinline__ void pair(uint32_t lo, uint32_t hi) {
    se = mul2(__byte_perm(lo, hi, 0x5410), 0x62006200u);
    m = mul2(__byte_perm(lo, hi, 0x7632), 0x1f801f80u);
    so = mul2(se, 0x3d803d80u);
  }
  // nibbles 0 .. 3 of both half-words
  __device__ __forceinline__ void values(uint32_t w, uint32_t (&v)[4]) const {
    const uint32_t u = w >> 8;
    v[0] = Kv4Bf16::fma2(w & 0x000f000fu, se, m);
    v[1] = Kv4Bf16::fma2(w & 0x00f000f0u, so, m);
    v[2] = Kv4Bf16::fma2(u & 0x000f000fu, se, m);
    v[3] = Kv4Bf16::fma2(u & 0x00f000f0u, so, m);
  }
};
template <>
struct Dequant<Kv4Fp16> {
  static constexpr float kBack = 1.f;
  uint32_t s, m;
  __device__ __forceinline__ void same(uint32_t param) {
    s = __byte_perm(param, 0, 0x1010);
    m = __byte_perm(param, 0, 0x3232);
  }
  __device__ __forceinline__ void pair(uint32_t lo, uint32_t hi) {
    s = __byte_perm(lo, hi, 0x5410);
    m = __byte_perm(lo, hi, 0x7632);
  }
  __device__ __forceinline__ void values(uint32_t w, uint32_t (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = kv4_dequant2<Kv4Fp16>(w >> (4 * i), s, m);
  }
};

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4)
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (N == 2)
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  else
    w[0] = *reinterpret_cast<const uint32_t*>(p);
}

}  // namespace woq
