// Rows that a training step keeps in 8 bits between its passes, and SwiGLU from and to them.
//
// A row goes in groups of 128 values (its last one may be shorter): scale = amax * (1 / 127), q = rint(x * ((1 / amax) * 127)), all
// quotients and products in fp32, so that any two forms of it give the same bytes; the row stands for q * scale.  A group that holds an infinity or
// NaN stands for NaN as a whole (its scale is NaN): a gradient through it shows it.  Groups whose largest magnitude is under 2^-120, whose
// 1 / amax would come near the end of the range, are kept as zeros.
//
//   pack      x -> (q, scale)                    unpack     (q, scale) -> x^
//   swiglu    y = g sig(g) u of interleaved (g, u) pairs, and the pairs packed, in one pass over them
//   its gradient   dg = dy u sig(g) (1 + g (1 - sig(g))), du = dy g sig(g) from the packed pairs
//
// All are bound by memory.  A warp takes four groups, all of their loads on their way before the first is worked on: of a group four values a lane
// (16 bytes of fp32, 4 of q), the largest magnitude by one reduction over the bits of |x| (whose order is that of the values, NaN above
// all), the quotients a lane a group.  8192 x 5120, us (TB/s, launch included): pack 41 (5.1), unpack 39 (5.4), SwiGLU 57 (5.1), its gradient 53 (5.5); with one
// group a warp 72, 51, 85, 65, with eight 40, 39, 55, 64.
// The reference keeps the inputs of its checkpointed segments as they are (src/tilerl/autograd.py:34); no counterpart.
#include "common.cuh"

namespace {

constexpr int KP_GROUP = 128, KP_U = 4;             // values a group, groups a warp
constexpr float KP_LEAST = 0x1p-120f, KP_MOST = 0x1.020406p+121f;      // KP_MOST: the largest scale 127 times which is finite

__device__ __forceinline__ float4 kp_ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float kp_sigm(float x) { return 1.f / (1.f + expf(-x)); }

// The values of a lane in its group: columns lane * 4 .. + 3 of `len` (VEC), else one by one.
template <bool VEC>
__device__ __forceinline__ float4 kp_load(const float* p, int c, int len) {
  if (VEC) return c < len ? kp_ld4(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c < len ? p[c] : 0.f, c + 1 < len ? p[c + 1] : 0.f, c + 2 < len ? p[c + 2] : 0.f, c + 3 < len ? p[c + 3] : 0.f);
}
template <bool VEC>
__device__ __forceinline__ void kp_store(float* p, int c, int len, float4 v) {
  if (VEC) {
    if (c < len) *reinterpret_cast<float4*>(p + c) = v;
    return;
  }
  if (c < len) p[c] = v.x;
  if (c + 1 < len) p[c + 1] = v.y;
  if (c + 2 < len) p[c + 2] = v.z;
  if (c + 3 < len) p[c + 3] = v.w;
}
template <bool VEC>
__device__ __forceinline__ char4 kp_load_q(const signed char* p, int c, int len) {
  if (VEC) return c < len ? *reinterpret_cast<const char4*>(p + c) : make_char4(0, 0, 0, 0);
  return make_char4(c < len ? p[c] : 0, c + 1 < len ? p[c + 1] : 0, c + 2 < len ? p[c + 2] : 0, c + 3 < len ? p[c + 3] : 0);
}

// The bits of the largest magnitude of a group; what values are multiplied with, and the scale, from them.
__device__ __forceinline__ uint32_t kp_most(float4 v) {
  return __reduce_max_sync(0xffffffffu, max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                                            max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
}
__device__ __forceinline__ float kp_inverse(uint32_t most) {
  return most >= 0x7f800000u || __uint_as_float(most) < KP_LEAST ? 0.f : 1.f / __uint_as_float(most) * 127.f;
}
__device__ __forceinline__ float kp_scale(uint32_t most) {
  if (most >= 0x7f800000u) return NAN;
  return __uint_as_float(most) < KP_LEAST ? 0.f : fminf(__uint_as_float(most) * (1.f / 127.f), KP_MOST);
}
// (0 times an infinity or NaN converts to 0)
__device__ __forceinline__ char4 kp_pack(float4 v, float inv) {
  return make_char4((signed char)__float2int_rn(v.x * inv), (signed char)__float2int_rn(v.y * inv), (signed char)__float2int_rn(v.z * inv),
                    (signed char)__float2int_rn(v.w * inv));
}
template <bool VEC>
__device__ __forceinline__ void kp_store_q(signed char* p, int c, int len, char4 q) {
  if (VEC) {
    if (c < len) *reinterpret_cast<char4*>(p + c) = q;
    return;
  }
  if (c < len) p[c] = q.x;
  if (c + 1 < len) p[c + 1] = q.y;
  if (c + 2 < len) p[c + 2] = q.z;
  if (c + 3 < len) p[c + 3] = q.w;
}

// KIND: 0 pack, 1 unpack, 2 SwiGLU, 3 its gradient.  f: fp32 rows in (pack, swiglu) or out (unpack, gradient); h: rows of half the
// width, out (swiglu) or in (gradient).  WHOLE: rows are whole groups, and so lie one group behind the other; VEC: 16-byte vectors.
template <int KIND, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(256) kp_kernel(float* f, signed char* q, float* scale, float* h, long groups, int width, int per_row) {
  constexpr int U = KP_U;
  const int lane = threadIdx.x & 31, c = lane * 4;
  const long g0 = ((long)blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
  if (g0 >= groups) return;
  // U groups a warp, all that they need on its way at once
  long at[U];
  int len[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const long g = g0 + j;
    if (WHOLE) {
      at[j] = g * KP_GROUP, len[j] = g < groups ? KP_GROUP : 0;
    } else {
      const long row = g / per_row;
      const int k = (int)(g - row * per_row) * KP_GROUP;
      at[j] = row * width + k, len[j] = g < groups ? min(KP_GROUP, width - k) : 0;
    }
  }
  if (KIND == 0 || KIND == 2) {
    float4 v[U];
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = kp_load<VEC>(f + at[j], c, len[j]);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const uint32_t most = kp_most(v[j]);
      if (lane == j) mine = most;
    }
    const float inv = kp_inverse(mine);              // (a lane a group)
    if (lane < U && g0 + lane < groups) scale[g0 + lane] = kp_scale(mine);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      kp_store_q<VEC>(q + at[j], c, len[j], kp_pack(v[j], __shfl_sync(0xffffffffu, inv, j)));
      if (KIND == 2) {
        const float2 y = make_float2(v[j].x * kp_sigm(v[j].x) * v[j].y, v[j].z * kp_sigm(v[j].z) * v[j].w);
        float* o = h + at[j] / 2 + c / 2;
        if (VEC) {
          if (c < len[j]) *reinterpret_cast<float2*>(o) = y;
        } else {
          if (c < len[j]) o[0] = y.x;
          if (c + 2 < len[j]) o[1] = y.y;
        }
      }
    }
  } else {
    char4 b[U];
    float2 up[U];
    const float mine = lane < U && g0 + lane < groups ? scale[g0 + lane] : 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      b[j] = kp_load_q<VEC>(q + at[j], c, len[j]);
      if (KIND == 3) {
        const float* e = h + at[j] / 2 + c / 2;
        up[j] = make_float2(0.f, 0.f);
        if (VEC) {
          if (c < len[j]) up[j] = *reinterpret_cast<const float2*>(e);
        } else {
          if (c < len[j]) up[j].x = e[0];
          if (c + 2 < len[j]) up[j].y = e[1];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float s = __shfl_sync(0xffffffffu, mine, j);
      float4 v = make_float4((float)b[j].x * s, (float)b[j].y * s, (float)b[j].z * s, (float)b[j].w * s);
      if (KIND == 3) {
        const float a = kp_sigm(v.x), z = kp_sigm(v.z);
        v = make_float4(up[j].x * v.y * a * (1.f + v.x * (1.f - a)), up[j].x * v.x * a, up[j].y * v.w * z * (1.f + v.z * (1.f - z)), up[j].y * v.z * z);
      }
      kp_store<VEC>(f + at[j], c, len[j], v);
    }
  }
}

template <int KIND>
int kp_launch(void* f, void* q, void* scale, void* h, long rows, int width, cudaStream_t st) {
  if (rows < 1 || width < 1 || ((KIND >= 2) && width % 2)) return (int)cudaErrorInvalidValue;
  const int per_row = (width + KP_GROUP - 1) / KP_GROUP;
  const long groups = rows * per_row, blocks = (groups + 8 * KP_U - 1) / (8 * KP_U);
  if (blocks >= 1l << 31) return (int)cudaErrorInvalidValue;
  const bool vec = width % 4 == 0 && !((reinterpret_cast<uintptr_t>(f) | reinterpret_cast<uintptr_t>(q) * 4 | reinterpret_cast<uintptr_t>(h) * 2) & 15);
  auto kern = !vec ? kp_kernel<KIND, false, false> : width % KP_GROUP ? kp_kernel<KIND, true, false> : kp_kernel<KIND, true, true>;
  kern<<<(unsigned)blocks, 256, 0, st>>>((float*)f, (signed char*)q, (float*)scale, (float*)h, groups, width, per_row);
  return (int)cudaGetLastError();
}

}  // namespace

// Rows of `width` values: f fp32 [rows, width], q int8 as f, scale fp32 [rows, ceil(width / 128)].
TRL_API int trl_keep_pack(const void* f, void* q, void* scale, long rows, int width, void* stream) {
  return kp_launch<0>(const_cast<void*>(f), q, scale, nullptr, rows, width, (cudaStream_t)stream);
}
TRL_API int trl_keep_unpack(const void* q, const void* scale, void* f, long rows, int width, void* stream) {
  return kp_launch<1>(f, const_cast<void*>(q), const_cast<void*>(scale), nullptr, rows, width, (cudaStream_t)stream);
}
// gu [rows, width] of (gate, up) pairs, out [rows, width / 2]
TRL_API int trl_keep_swiglu(const void* gu, void* q, void* scale, void* out, long rows, int width, void* stream) {
  return kp_launch<2>(const_cast<void*>(gu), q, scale, out, rows, width, (cudaStream_t)stream);
}
TRL_API int trl_keep_swiglu_grad(const void* q, const void* scale, const void* up, void* dgu, long rows, int width, void* stream) {
  return kp_launch<3>(dgu, const_cast<void*>(q), const_cast<void*>(scale), const_cast<void*>(up), rows, width, (cudaStream_t)stream);
}
