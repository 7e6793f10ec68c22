// Rows into 8-bit integers with a scale each (activations, weights), and gradients into 16 bits as two digits of 8.
//
//   t = x * w (w: norm weight or none),  m = max |t|,  q = rint(t * ((1 / m) * 127)),  s = m * (1 / 127) [* rsqrt(mean x^2 + eps)]
//   u = g * ws,                          m = max |u|,  Q = rint(u * ((1 / m) * 32512)) = 256 hi + lo,  s = m * (1 / 32512)
//
// A norm's factor is the same for a whole row, so it cancels out of the integers and goes into the scale alone.  One pass: a block a
// row, the row stays in registers between its maximum and its integers (up to 8 vectors of 8 values a thread; longer rows are read a
// second time, out of L2).  Bound by memory for many rows, by latency (two block barriers) for few.
//
// The reference quantises activations per token for its FP8 products (`quant_fp8`, packages/tilerl-kernels/src/tilerl_kernels/
// kernels_linear.py:1547-1590); it has no integer form.
#include "int8.cuh"

namespace {

struct RowsParams {
  const void* x;
  const float* w;        // norm weight, or the channels' scales of a gradient; may be null
  int8_t* q;             // [rows][ldq]; gradients: rows 2r (high digits) and 2r + 1 (low)
  float* s;
  long long ldx, ldq;
  int K;
  float eps;
  int norm;
  int weights;           // q and s are a weight: products may read one before they wait for the kernel ahead of them
};

template <typename T, bool VEC>
__device__ __forceinline__ void rows_load(const T* x, int k, int K, float (&v)[8]) {
  if (VEC && k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = __ldcg(reinterpret_cast<const uint4*>(x + k));
      const float2 a = bf162_bits_to_f2(u.x), b = bf162_bits_to_f2(u.y), c = bf162_bits_to_f2(u.z), d = bf162_bits_to_f2(u.w);
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
    } else {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(x + k)), b = __ldcg(reinterpret_cast<const float4*>(x + k) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
    if (k + i < K) {
      if constexpr (sizeof(T) == 2) v[i] = __bfloat162float(__ldcg(x + k + i));
      else v[i] = __ldcg(x + k + i);
    }
  }
}

// CH: vectors that a thread keeps; 0: a row of any length, read twice.  W16: two digits.
template <typename T, int CH, bool VEC, bool W16>
__global__ void __launch_bounds__(1024) rows_i8_kernel(const RowsParams p) {
  extern __shared__ float groups[];              // sums of squares of 256 values each
  __shared__ uint32_t most_s[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5, K = p.K;
  // A product behind this kernel loads weights before it waits.  So the dependents are let in only once all that came before is through
  // (it may have written those weights), and by a weight's quantiser not before its end.
  pdl_enter();
  pdl_wait();
  if (!p.weights) pdl_trigger();
  const T* x = reinterpret_cast<const T*>(p.x) + (long long)blockIdx.x * p.ldx;
  constexpr int KEEP = CH ? CH : 1;
  float t[KEEP][8];
  uint32_t most = 0;
  const bool squares = !W16 && p.norm;
  auto weight = [&](int k, float (&v)[8]) {
    if (p.w == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? __fmul_rn(v[i], p.w[k + i]) : 0.f;
  };
  auto take = [&](int c, float (&v)[8]) {
    const int k = (c * (int)blockDim.x + (int)threadIdx.x) * 8;
    rows_load<T, VEC>(x, k, K, v);
    if (squares) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
      ss = warp_sum(ss);
      const int g = c * nw + warp;
      if (lane == 0 && g * I8_GROUP < K) groups[g] = ss;
    }
    weight(k, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, i8_abs_bits(v[i]));
  };
  const int chunks = CH ? CH : (K + (int)blockDim.x * 8 - 1) / ((int)blockDim.x * 8);
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c) take(c, t[c]);
  } else {
    for (int c = 0; c < chunks; ++c) take(c, t[0]);
  }
  most = i8_warp_most(most);
  if (lane == 0) most_s[warp] = most;
  __syncthreads();
  most = i8_warp_most(lane < nw ? most_s[lane] : 0u);
  constexpr float MOST = W16 ? I16_MOST : I8_MOST, PART = 1.f / MOST;
  const float f = i8_factor(most, MOST);
  auto give = [&](int c, float (&v)[8]) {
    const int k = (c * (int)blockDim.x + (int)threadIdx.x) * 8;
    if (k >= K) return;
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = i8_round(v[i], f);
    auto store = [&](int8_t* out, const int (&d)[8]) {
      if (k + 8 <= K) {
        *reinterpret_cast<uint2*>(out + k) = make_uint2(i8_pack(d[0], d[1], d[2], d[3]), i8_pack(d[4], d[5], d[6], d[7]));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) out[k + i] = (int8_t)d[i];
      }
    };
    if constexpr (W16) {
      int hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) hi[i] = (q[i] + 128) >> 8, lo[i] = q[i] - hi[i] * 256;
      int8_t* out = p.q + 2ll * blockIdx.x * p.ldq;
      store(out, hi), store(out + p.ldq, lo);
    } else {
      store(p.q + (long long)blockIdx.x * p.ldq, q);
    }
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c) give(c, t[c]);
  } else {
    for (int c = 0; c < chunks; ++c) {
      rows_load<T, VEC>(x, (c * (int)blockDim.x + (int)threadIdx.x) * 8, K, t[0]);
      weight((c * (int)blockDim.x + (int)threadIdx.x) * 8, t[0]);
      give(c, t[0]);
    }
  }
  if (warp == 0) {
    float s = i8_scale(most, PART);
    if (squares) s = __fmul_rn(s, rsqrtf(i8_groups_sum(groups, (K + I8_GROUP - 1) / I8_GROUP) / (float)K + p.eps));
    if (lane == 0) p.s[blockIdx.x] = s;
  }
}

template <typename T, bool VEC, bool W16>
cudaError_t rows_launch(const RowsParams& p, long long rows, cudaStream_t stream) {
  const int vecs = (p.K + 7) / 8;
  // vectors a thread: more of them keep more loads in flight a block, fewer leave more threads for a short row
  const int ch = vecs <= 256 ? 1 : vecs <= 1280 ? 2 : vecs <= 2560 ? 4 : vecs <= 8192 ? 8 : 0;
  const int threads = ch ? max(32, ((vecs + ch - 1) / ch + 31) / 32 * 32) : 1024;
  const size_t smem = (size_t)((p.K + I8_GROUP - 1) / I8_GROUP) * sizeof(float);
  if (smem > 48 * 1024) return cudaErrorInvalidValue;
  switch (ch) {
    case 1: return trl_launch(rows_i8_kernel<T, 1, VEC, W16>, dim3((unsigned)rows), dim3(threads), smem, stream, p);
    case 2: return trl_launch(rows_i8_kernel<T, 2, VEC, W16>, dim3((unsigned)rows), dim3(threads), smem, stream, p);
    case 4: return trl_launch(rows_i8_kernel<T, 4, VEC, W16>, dim3((unsigned)rows), dim3(threads), smem, stream, p);
    case 8: return trl_launch(rows_i8_kernel<T, 8, VEC, W16>, dim3((unsigned)rows), dim3(threads), smem, stream, p);
    default: return trl_launch(rows_i8_kernel<T, 0, VEC, W16>, dim3((unsigned)rows), dim3(threads), smem, stream, p);
  }
}

}  // namespace

// x [rows, K] (type 0: fp32, 1: bf16; rows ldx apart) -> q int8 [rows, ldq], s fp32 [rows].  w: fp32 [K] or null; norm: w is a norm's
// weight, and the row's 1 / rms goes into s.  digits 2: q has two rows of digits a row, 16 bits in all, and w is not a norm's.
// weights: q and s are a weight's.  ldq and q on 8-byte boundaries.
TRL_API int trl_rows_i8(const void* x, int type, long ldx, const void* w, int norm, float eps, void* q, long ldq, void* s, long rows, int K,
                        int digits, int weights, void* stream) {
  if (rows <= 0 || rows > 0x7fffffffl || K <= 0 || ldq < K || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8 || (type != 0 && type != 1) ||
      (digits != 1 && digits != 2) || (norm && (w == nullptr || digits == 2)))
    return (int)cudaErrorInvalidValue;
  RowsParams p{x, (const float*)w, (int8_t*)q, (float*)s, ldx, ldq, K, eps, norm, weights};
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (type ? 8 : 4) == 0;
  if (type) {
    if (digits == 2) return (int)(vec ? rows_launch<bf16, true, true>(p, rows, st) : rows_launch<bf16, false, true>(p, rows, st));
    return (int)(vec ? rows_launch<bf16, true, false>(p, rows, st) : rows_launch<bf16, false, false>(p, rows, st));
  }
  if (digits == 2) return (int)(vec ? rows_launch<float, true, true>(p, rows, st) : rows_launch<float, false, true>(p, rows, st));
  return (int)(vec ? rows_launch<float, true, false>(p, rows, st) : rows_launch<float, false, false>(p, rows, st));
}
