// What the tensor-core attention kernels share: bf16 pairs, exponentials on the
// fp32 pipe, and V tiles without what a row must not meet.
#pragma once

#include "tcgen05.cuh"

namespace mtpb {

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// 2^x of two values on the fp32 pipe: x = n + f with n the nearest integer
// (read off the low bits of x + 1.5 * 2^23) and |f| <= 1/2, 2^f by the cubic
// of least relative error there (7.5e-5 by the Remez exchange, a fiftieth of
// bf16's half step), n added to the exponent. For x <= 126; below -125 the
// result is 2^-125.
__device__ __forceinline__ float2 exp2_cubic(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
  x.x = fmaxf(x.x, -125.f);
  x.y = fmaxf(x.y, -125.f);
  const float2 r = add2(x, magic);
  const float2 f = fma2(add2(r, back), make_float2(-1.f, -1.f), x);
  float2 q = fma2(f, make_float2(0.0551716685295105f, 0.0551716685295105f),
                  make_float2(0.2426111251115799f, 0.2426111251115799f));
  q = fma2(q, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
  q = fma2(q, f, make_float2(0.9999280571937561f, 0.9999280571937561f));
  return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(q.y) + (__float_as_int(r.y) << 23)));
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

constexpr uint32_t kTcSub = 128 * 64 * 2;  // a 128 x 64 bf16 subtile

// Row r of a V tile: behind the range it becomes zeros; one that not every
// token sees loses its NaN and infinities, and *odd = mark tells of them. (A call, to
// take no registers from the softmax.)
template <int HD>
__device__ __noinline__ void tc_clean_row(unsigned char* tile, int r, bool behind, bool unseen, int* odd, int mark = 1) {
  auto at = [&](int i) { return reinterpret_cast<uint4*>(tile + (i >> 3) * kTcSub + r * 128 + (((i ^ r) & 7) << 4)); };
  if (behind) {
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) *at(i) = make_uint4(0, 0, 0, 0);
  } else if (unseen) {
    uint32_t nan = 0;  // two bf16, NaN when a value was not finite
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      const uint4 v = *at(i);
      nan = fma_bf16x2(v.x, 0u, fma_bf16x2(v.y, 0u, fma_bf16x2(v.z, 0u, fma_bf16x2(v.w, 0u, nan))));
    }
    if (nan & 0x7FFF7FFFu) {
      *static_cast<volatile int*>(odd) = mark;
      __threadfence_block();
#pragma unroll 1
      for (int i = 0; i < HD; ++i) {
        uint16_t* h = reinterpret_cast<uint16_t*>(at(i >> 3)) + (i & 7);
        if ((*h & 0x7F80u) == 0x7F80u) *h = 0;
      }
    }
  }
}

}  // namespace mtpb
