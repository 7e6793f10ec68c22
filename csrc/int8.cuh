// What the kernels of 8-bit integer projections share: the arithmetic of a row's integers and the order in which a row's squares are
// added up, so that a row has the same integers and the same scale, bit for bit, in whichever kernel it is quantised.
#pragma once
#include "common.cuh"

namespace {

constexpr float I8_MOST = 127.f;          // of activations and weights
constexpr float I16_MOST = 32512.f;       // of gradients, two digits of 8 bits: 127 * 256
constexpr float I8_LEAST = 0x1p-110f;     // rows whose largest magnitude is below count as zeros: (1 / m) * 32512 is finite above

// What a row's values are multiplied with; 0 for a row of zeros, one with an infinity or NaN too.  Magnitudes are compared as the integers
// that their bits are, in which a NaN is the largest.
__device__ __forceinline__ float i8_factor(uint32_t most_bits, float most_int) {
  const float m = __uint_as_float(most_bits);
  return most_bits >= 0x7f800000u || m < I8_LEAST ? 0.f : __fmul_rn(__frcp_rn(m), most_int);
}
// The row's scale (before a norm's factor).  `part` is 1 / most_int rounded to fp32.
__device__ __forceinline__ float i8_scale(uint32_t most_bits, float part) {
  const float m = __uint_as_float(most_bits);
  return most_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : m < I8_LEAST ? 0.f : __fmul_rn(m, part);
}
__device__ __forceinline__ uint32_t i8_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The nearest integer of t * factor (ties to even), in the low bits, of which a signed byte or 16 bits may be taken: behind the sum with 1.5 * 2^23
// a float's last bit stands for one.
__device__ __forceinline__ uint32_t i8_round_bits(float t, float factor) { return __float_as_uint(__fadd_rn(__fmul_rn(t, factor), 12582912.f)); }
__device__ __forceinline__ uint32_t i8_pack(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Order of a row's squares: vectors of eight values one after the other; the 32 vectors of a group of 256 values by halving (xor 16, 8, 4,
// 2, 1); then the groups, of which lane l of a warp adds l, l + 32, ... in that order before the lanes are halved again.
constexpr int I8_GROUP = 256;
__device__ __forceinline__ float i8_groups_sum(const float* groups, int n) {
  float s = 0.f;
  for (int g = threadIdx.x & 31; g < n; g += 32) s += groups[g];
  return warp_sum(s);
}
__device__ __forceinline__ uint32_t i8_warp_most(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// A product's result from its sum of integers: the sum in fp32 (rounded above 2^24) times the product of both scales.  The same operations
// in the same order in every kernel: a row's results do not depend on which one the number of rows leads to.
__device__ __forceinline__ float i8_value(int acc, float scale) { return __fmul_rn(__int2float_rn(acc), scale); }
__device__ __forceinline__ float i8_swiglu(float gate, float up) { return __fmul_rn(__fdividef(gate, 1.f + __expf(-gate)), up); }

enum { I8_STORE = 0, I8_RESIDUAL = 1, I8_SWIGLU = 2, I8_STORE_F32 = 3 };

// SMs of the current device (host).
inline int i8_sms() {
  static TrlPerDevice<int> counts;
  int& n = counts.here();
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

}  // namespace
