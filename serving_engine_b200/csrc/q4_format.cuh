// The 4-bit KV pool's format, shared by the kernels that write, read back and attend
// over it.
//
// A plane (K or V of one layer) is [num_blocks][num_kv_heads][9 * head_dim] bytes: a
// row is one kv head of one 16-token block. Every 64 values of a token's head are a
// group, x ~ scale * n + low with n = 0..15 and scale, low in fp16: 4.5 bits a value.
// Bytes [0, 8 * head_dim) of a row are codes, bytes [8 * head_dim, 9 * head_dim) the
// (scale, low) pairs. Both are cut in panels of W = min(head_dim, 128) dims, and with
// G = W / 64 groups to a panel:
//   K: token r has W / 2 bytes; dims [16 t, 16 t + 16) of every group are neighbours,
//      4 chunks t of 8 G bytes; 8 dims are one 32-bit word, its low half dims 0, 2, 4,
//      6 and its high half dims 1, 3, 5, 7 (4 bits each, lowest first).
//   V: tokens 2p and 2p + 1 share W bytes; dims [8 c, 8 c + 8) of every group are
//      neighbours, 8 chunks of 8 G bytes, chunk c at place c ^ turn(p); 4 dims are one
//      32-bit word, its low half token 2p's and its high half token 2p + 1's.
//   pairs: token by token, the panel's groups in order, 4 bytes each.
// This is the order in which the lanes of an m16n8k16 tensor-core operand need them:
// masking a word with 0x000f000f or 0x00f000f0 leaves two operand elements (as fp16
// numbers, n * 2^-24 and n * 2^-20), and each lane's words of a block are one or two
// 8- or 16-byte loads that meet no bank twice (what turn() is for). No byte holds
// codes of two tokens, so tokens of one block can be written at the same time.
#pragma once

#include "seb_common.cuh"

namespace seb {
namespace q4 {

constexpr int kGroup = 64;

template <int D>
struct Layout {
  static constexpr int kWidth = D < 128 ? D : 128;       // dims of a panel
  static constexpr int kGroups = kWidth / kGroup;        // groups of a panel
  static constexpr int kPanels = D / kWidth;
  static constexpr int kCodes = 8 * D;                   // bytes of a row before its pairs
  static constexpr int kRow = 9 * D;

  static __device__ __forceinline__ int turn(int pair) {
    return kGroups == 2 ? 2 * (pair & 3) : 4 * ((pair >> 1) & 1);
  }
  // Byte of the word of K codes of token r, dims [dim, dim + 8).
  static __device__ __forceinline__ int k_word(int r, int dim) {
    const int p = dim / kWidth, g = dim % kWidth / kGroup, c = dim % kGroup;
    return p * 8 * kWidth + r * (kWidth / 2) + (c >> 4) * (8 * kGroups) + g * 8 + ((c >> 3) & 1) * 4;
  }
  // Byte of token r's 16 bits of V codes of dims [dim, dim + 4); those of the next four dims are 4 bytes on.
  static __device__ __forceinline__ int v_half(int r, int dim) {
    const int p = dim / kWidth, g = dim % kWidth / kGroup, c = dim % kGroup;
    return p * 8 * kWidth + (r >> 1) * kWidth + ((c >> 3) ^ turn(r >> 1)) * (8 * kGroups) + g * 8 +
           ((c >> 2) & 1) * 4 + (r & 1) * 2;
  }
  // Byte of the (scale, low) pair of token r's group that holds `dim`.
  static __device__ __forceinline__ int pair(int r, int dim) {
    const int p = dim / kWidth, g = dim % kWidth / kGroup;
    return kCodes + p * (64 * kGroups) + (r * kGroups + g) * 4;
  }
};

// Codes 0..7 of a word of K (dims 0..7) and of V's two 16-bit pieces.
__device__ __forceinline__ uint32_t k_pack(const uint32_t (&n)[8]) {
  return n[0] | n[2] << 4 | n[4] << 8 | n[6] << 12 | n[1] << 16 | n[3] << 20 | n[5] << 24 | n[7] << 28;
}
__device__ __forceinline__ uint32_t k_code(uint32_t word, int i) { return (word >> (16 * (i & 1) + 4 * (i >> 1))) & 15u; }
__device__ __forceinline__ uint32_t v_pack(const uint32_t* n) { return n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12; }
__device__ __forceinline__ uint32_t v_code(uint32_t half, int i) { return (half >> (4 * i)) & 15u; }

// min and max that return NaN where an operand is one
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A group's parameters from its extremes. scale and low are rounded to fp16 and the
// codes are taken against the rounded values, so that rounding costs the group no
// more than its ends; low is clamped to +-65504 and scale to 65504. A group that holds
// an infinity or a NaN reads back as NaN in every value.
struct Params {
  uint32_t bits;  // scale, then low
  float low, inverse;
};
__device__ __forceinline__ Params params_of(float lo, float hi) {
  Params p;
  const bool finite = fabsf(lo) < INFINITY && fabsf(hi) < INFINITY;
  const float range = __fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f);
  const __half s = finite ? __float2half_rn(fminf(range, 65504.f)) : __ushort_as_half(0x7fff);
  const __half l = finite ? __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f)) : __ushort_as_half(0x7fff);
  const float sf = __half2float(s);
  p.low = __half2float(l);
  p.inverse = sf > 0.f ? __fdiv_rn(1.f, sf) : 0.f;
  p.bits = (uint32_t)__half_as_ushort(s) | (uint32_t)__half_as_ushort(l) << 16;
  return p;
}
// The code of x, ties to even. Adding 1.5 * 2^23 leaves the rounded integer in the low bits.
__device__ __forceinline__ uint32_t code_of(float x, const Params& p) {
  const float y = __fmul_rn(__fsub_rn(x, p.low), p.inverse);
  return __float_as_uint(__fadd_rn(fminf(fmaxf(y, 0.f), 15.f), 12582912.f)) & 15u;
}
// The value that code n stands for.
__device__ __forceinline__ float value_of(uint32_t n, float scale, float low) {
  return __fadd_rn(__fmul_rn((float)n, scale), low);
}

}  // namespace q4
}  // namespace seb
