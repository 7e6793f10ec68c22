// Products of 8-bit integers with a scale for each token and each channel.
//
//   y[t, n]  = epi((sum_k q[t, k] W[n, k]) * s[t] * ws[n])                              (W: int8 [N, K], q: rows_i8.cu)
//   dx[t, k] = s[t] * (256 sum_n hi[t, n] W[n, k] + sum_n lo[t, n] W[n, k])             (gradient of y's input, rows in two digits)
//
// Simple form: a block 64 x 64 results, 64 bytes of the summed dimension at a time through shared memory, dp4a.
//
// The reference has no integer product; in the place of its `linear_fp8` (packages/tilerl-kernels/src/tilerl_kernels/
// kernels_linear.py:1777-1813) for weights in this format.
#include "int8.cuh"

namespace {

enum { I8_STORE = 0, I8_RESIDUAL = 1, I8_SWIGLU = 2, I8_STORE_F32 = 3 };

struct I8Params {
  const int8_t* w;       // [N, K]
  const float* ws;       // [N]
  const int8_t* q;       // [T, ldq]
  const float* s;        // [T]
  const bf16* residual;
  void* out;
  long long ldw, ldq, ldr, ldo;
  int T, N, K, epi;
};

__device__ __forceinline__ void i8_out(const I8Params& p, int t, int n, float v, float up) {
  const size_t at = (size_t)t * p.ldo;
  if (p.epi == I8_SWIGLU) {
    if (!(n & 1)) reinterpret_cast<bf16*>(p.out)[at + (n >> 1)] = __float2bfloat16(__fdividef(v, 1.f + __expf(-v)) * up);
  } else if (p.epi == I8_STORE_F32) {
    reinterpret_cast<float*>(p.out)[at + n] = v;
  } else {
    if (p.epi == I8_RESIDUAL) v += __bfloat162float(__ldcg(p.residual + (size_t)t * p.ldr + n));
    reinterpret_cast<bf16*>(p.out)[at + n] = __float2bfloat16(v);
  }
}

// GRAD: results are [T, K], summed over N; q has two rows a token.
template <bool GRAD>
__global__ void __launch_bounds__(256) i8_simple_kernel(const I8Params p) {
  __shared__ int ws_[16][65], qs[16][65], ql[GRAD ? 16 : 1][65];       // [4-byte step][feature or token]
  pdl_launch_dependents();
  pdl_wait();
  const int f0 = blockIdx.x * 64, t0 = blockIdx.y * 64, features = GRAD ? p.K : p.N, depth = GRAD ? p.N : p.K;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {}, low[GRAD ? 4 : 1][4] = {};
  for (int d0 = 0; d0 < depth; d0 += 64) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int r = i / 16, j = i % 16;
      uint32_t w = 0, q = 0, l = 0;
      for (int b = 0; b < 4; ++b) {
        const int d = d0 + j * 4 + b, f = f0 + r, t = t0 + r;
        if (d < depth && f < features) w |= (uint32_t)(uint8_t)(GRAD ? p.w[(size_t)d * p.ldw + f] : p.w[(size_t)f * p.ldw + d]) << (8 * b);
        if (d < depth && t < p.T) {
          q |= (uint32_t)(uint8_t)__ldcg(p.q + (size_t)t * (GRAD ? 2 : 1) * p.ldq + d) << (8 * b);
          if (GRAD) l |= (uint32_t)(uint8_t)__ldcg(p.q + ((size_t)t * 2 + 1) * p.ldq + d) << (8 * b);
        }
      }
      ws_[j][r] = (int)w, qs[j][r] = (int)q;
      if (GRAD) ql[j][r] = (int)l;
    }
    __syncthreads();
    for (int j = 0; j < 16; ++j)
      for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b) {
          acc[a][b] = __dp4a(qs[j][ty * 4 + a], ws_[j][tx * 4 + b], acc[a][b]);
          if (GRAD) low[a][b] = __dp4a(ql[j][ty * 4 + a], ws_[j][tx * 4 + b], low[a][b]);
        }
    __syncthreads();
  }
  for (int a = 0; a < 4; ++a) {
    const int t = t0 + ty * 4 + a;
    if (t >= p.T) continue;
    const float s = __ldcg(p.s + t);
    float v[5] = {};
    for (int b = 0; b < 4; ++b) {
      const int f = f0 + tx * 4 + b;
      if (f < features) v[b] = GRAD ? fmaf(256.f, (float)acc[a][b], (float)low[a][b]) * s : (float)acc[a][b] * (s * p.ws[f]);
    }
    for (int b = 0; b < 4; ++b)
      if (f0 + tx * 4 + b < features) i8_out(p, t, f0 + tx * 4 + b, v[b], v[b + 1]);
  }
}

}  // namespace

// out[t, n] = epi(...).  K and N up to 131072 (sums of 32 bits); SwiGLU: N even, rows of w in (gate, up) pairs, out [T, N / 2].
TRL_API int trl_gemm_i8(const void* w, long ldw, const void* ws, const void* q, long ldq, const void* s, const void* residual, long ldr, void* out,
                        long ldo, int T, int N, int K, int epi, void* stream) {
  if (T <= 0 || N <= 0 || K <= 0 || K > 131072 || epi < 0 || epi > 3 || (epi == I8_SWIGLU && N % 2)) return (int)cudaErrorInvalidValue;
  const I8Params p{(const int8_t*)w, (const float*)ws, (const int8_t*)q, (const float*)s, (const bf16*)residual, out, ldw, ldq, ldr, ldo, T, N, K, epi};
  return (int)trl_launch(i8_simple_kernel<false>, dim3((N + 63) / 64, (T + 63) / 64), dim3(256), 0, (cudaStream_t)stream, p);
}

// dx[t, k], fp32, of rows in two digits: q [2 T, ldq].
TRL_API int trl_gemm_i8_grad(const void* w, long ldw, const void* q, long ldq, const void* s, void* dx, long ldo, int T, int N, int K, void* stream) {
  if (T <= 0 || N <= 0 || K <= 0 || N > 131072) return (int)cudaErrorInvalidValue;
  const I8Params p{(const int8_t*)w, nullptr, (const int8_t*)q, (const float*)s, nullptr, dx, ldw, ldq, 0, ldo, T, N, K, I8_STORE_F32};
  return (int)trl_launch(i8_simple_kernel<true>, dim3((K + 63) / 64, (T + 63) / 64), dim3(256), 0, (cudaStream_t)stream, p);
}
