// Arithmetic of the softmax warps of the tcgen05 attention kernels, and their bounded wait.
#pragma once

#include "seb_common.cuh"

namespace seb {

// 2^x by the MUFU instruction (ex2.approx.ftz: 2^-22 relative error, -inf -> +0).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed fp32 pairs (sm_100 f32x2 instructions: one issue slot for the two
// lanes of an FMA, add, subtract or multiply), so that the softmax, which is
// bound by issue slots and the MUFU, spends half the slots on its fp32 work.
__device__ __forceinline__ uint64_t f2_pack(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(f2_pack(a)), "l"(f2_pack(b)), "l"(f2_pack(c)));
  return f2_unpack(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_pack(a)), "l"(f2_pack(b)));
  return f2_unpack(d);
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_pack(a)), "l"(f2_pack(b)));
  return f2_unpack(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_pack(a)), "l"(f2_pack(b)));
  return f2_unpack(d);
}
__device__ __forceinline__ float2 splat2(float v) { return make_float2(v, v); }

// max(a, b, c) in one instruction (sm_100); NaN operands are dropped as fmaxf drops them.
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for two scores on the FMA pipe, so that part of a tile's exponentials
// run beside the MUFU's. Cody-Waite range reduction: 2^x = 2^j * 2^f with
// j = rint(x) (the 1.5 * 2^23 addition leaves j in the low mantissa bits) and
// f = x - j in [-1/2, 1/2], exact; 2^f by the degree-3 polynomial that minimises
// the relative error on that interval (coefficients fitted for this kernel by a
// linear program: 7.5e-5 relative error in fp32, against 2^-9 for the 16-bit P
// it feeds). Valid for x <= 127. It is used only on unmasked tiles (no -inf
// scores); there a score more than 126 below the row's reference maximum weighs
// about 1.2e-38 instead of ex2's 0. max.NaN keeps a NaN score NaN, as ex2 does.
__device__ __forceinline__ float2 poly_exp2x2(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));  // max(x, -126)
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
  const float2 t = add2(x, splat2(12582912.f));
  const float2 f = sub2(x, sub2(t, splat2(12582912.f)));
  float2 p = fma2(splat2(0x1.c3f76p-5f), f, splat2(0x1.f0de1ap-3f));
  p = fma2(p, f, splat2(0x1.62f31ap-1f));
  p = fma2(p, f, splat2(0x1.fff692p-1f));
  const float2 scale = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                                   __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000));  // 2^j
  return mul2(p, scale);
}

// A bounded wait that, once one has run out, waits no more.
__device__ __forceinline__ bool wait_or_flag(uint32_t bar, uint32_t parity, bool& failed) {
  if (failed) return false;
  if (!mbar_wait_bounded(bar, parity)) {
    failed = true;
    return false;
  }
  return true;
}

}  // namespace seb
