// Products of 8-bit integers with up to eight rows: y[t, n] = epi((sum_k q[t, k] W[n, k]) * s[t] * ws[n]), as gemm_i8.cu, bound by the read of
// W.  The rows are quantised here as rows_i8.cu does it (same integers, same scales), by every block for itself, while its first weights are
// on their way; or they come quantised.
//
// One block an SM with an even share of W's rows, to the row pair, so that all SMs read as long.  Its 16 warps share the row groups (16
// rows, the A operand of mma.m16n8k32) and the steps along K (64 bytes: 16 a lane, of rows g and g + 8, four steps in flight); tokens
// are the B operand.  A lane's 16 bytes are used as they lie: both operands permute K the same way.  Sums go into shared memory by
// integer atomics: exact, so their order changes nothing.
//
// The reference's FP8 form for few rows is `linear_fp8_gemv` (packages/tilerl-kernels/src/tilerl_kernels/kernels_linear.py:1442-1494).
#include "int8.cuh"

namespace {

constexpr int GV_THREADS = 512, GV_WARPS = GV_THREADS / 32, GV_DEPTH = 4, GV_TOKENS = 8;
constexpr int GV_STEP = 64;

struct GemvI8Params {
  const int8_t* w;
  const float* ws;
  const void* x;         // FUSED: bf16 rows; else int8 rows
  const float* s;        // rows' scales (not FUSED)
  const float* norm_w;
  const bf16* residual;
  void* out;
  long long ldw, ldx, ldr, ldo;
  int T, N, K, epi, kw;  // kw: warps that share K (a power of two; the others share row groups)
  float eps;
};

__host__ __device__ constexpr int gv_row(int K) { return (K + 127) / 128 * 128 + 64; }     // bytes of a token in shared memory: lanes of two tokens hit all banks

__device__ __forceinline__ void gv_mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool FUSED>
__global__ void __launch_bounds__(GV_THREADS, 1) gemv_i8_kernel(const GemvI8Params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_s[GV_TOKENS];
  __shared__ uint32_t most_s[GV_TOKENS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = p.K, T = p.T, ldx = gv_row(K);
  // this block's rows, in pairs
  const int r0 = (int)((long long)blockIdx.x * (p.N + 1) / 2 / gridDim.x) * 2, r1 = min(p.N, (int)((long long)(blockIdx.x + 1) * (p.N + 1) / 2 / gridDim.x) * 2);
  int8_t* xs = reinterpret_cast<int8_t*>(smem);                          // [T][ldx]
  int* acc = reinterpret_cast<int*>(smem + (size_t)T * ldx);             // [r1 - r0][8]
  pdl_launch_dependents();

  const int KW = p.kw, GW = GV_WARPS / KW, kw = warp % KW, gw = warp / KW;
  const int steps = (K + GV_STEP - 1) / GV_STEP, groups = (r1 - r0 + 15) / 16;
  const int my_steps = kw < steps ? (steps - kw + KW - 1) / KW : 0, my_groups = gw < groups ? (groups - gw + GW - 1) / GW : 0, items = my_steps * my_groups;
  uint4 ring[GV_DEPTH][2];
  int ld_g = gw, ld_s = kw;
  auto load = [&](uint4 (&v)[2], bool there) {
    const int row = r0 + ld_g * 16 + (lane >> 2), k = ld_s * GV_STEP + (lane & 3) * 16;
    const int8_t* src = p.w + (long long)row * p.ldw + k;
    const bool in = there && k < K;
    v[0] = in && row < r1 ? ldg_stream_16(src) : make_uint4(0u, 0u, 0u, 0u);
    v[1] = in && row + 8 < r1 ? ldg_stream_16(src + 8 * p.ldw) : make_uint4(0u, 0u, 0u, 0u);
    if ((ld_s += KW) >= steps) ld_s = kw, ld_g += GW;
  };
#pragma unroll
  for (int d = 0; d < GV_DEPTH; ++d) load(ring[d], d < items);           // weights do not depend on the kernel ahead (rows_i8.cu)

  for (int i = threadIdx.x; i < (r1 - r0) * GV_TOKENS; i += GV_THREADS) acc[i] = 0;
  if (threadIdx.x < GV_TOKENS) most_s[threadIdx.x] = 0;
  const int pieces = (K + I8_GROUP - 1) / I8_GROUP;                      // of 256 values: a warp's lanes have eight each
  pdl_wait();
  if constexpr (FUSED) {
    uint4* raw = reinterpret_cast<uint4*>(acc + (size_t)(r1 - r0) * GV_TOKENS);      // [T][pieces * 32] as they came
    float* sums = reinterpret_cast<float*>(raw + (size_t)T * pieces * 32);           // [T][pieces]
    auto times = [&](int k, const uint4& u, float (&v)[8]) {
      const float2 a = bf162_bits_to_f2(u.x), b = bf162_bits_to_f2(u.y), c = bf162_bits_to_f2(u.z), d = bf162_bits_to_f2(u.w);
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
      if (p.norm_w == nullptr || k >= K) return;
      const float4 w0 = *reinterpret_cast<const float4*>(p.norm_w + k), w1 = *reinterpret_cast<const float4*>(p.norm_w + k + 4);
      v[0] = __fmul_rn(v[0], w0.x), v[1] = __fmul_rn(v[1], w0.y), v[2] = __fmul_rn(v[2], w0.z), v[3] = __fmul_rn(v[3], w0.w);
      v[4] = __fmul_rn(v[4], w1.x), v[5] = __fmul_rn(v[5], w1.y), v[6] = __fmul_rn(v[6], w1.z), v[7] = __fmul_rn(v[7], w1.w);
    };
    __syncthreads();                                 // most_s is zero
    for (int i = warp; i < T * pieces; i += GV_WARPS) {
      const int t = i / pieces, k = (i % pieces) * I8_GROUP + lane * 8;
      const uint4 u = k < K ? __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(p.x) + (long long)t * p.ldx + k)) : make_uint4(0u, 0u, 0u, 0u);
      raw[i * 32 + lane] = u;
      if (p.norm_w != nullptr) {
        const float2 a = bf162_bits_to_f2(u.x), b = bf162_bits_to_f2(u.y), c = bf162_bits_to_f2(u.z), d = bf162_bits_to_f2(u.w);
        float ss = fmaf(a.y, a.y, fmaf(a.x, a.x, 0.f));
        ss = fmaf(b.y, b.y, fmaf(b.x, b.x, ss)), ss = fmaf(c.y, c.y, fmaf(c.x, c.x, ss)), ss = fmaf(d.y, d.y, fmaf(d.x, d.x, ss));
        ss = warp_sum(ss);
        if (lane == 0) sums[i] = ss;
      }
      float v[8];
      times(k, u, v);
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, i8_abs_bits(v[e]));
      most = i8_warp_most(most);
      if (lane == 0) atomicMax(&most_s[t], most);
    }
    __syncthreads();
    for (int i = warp; i < T * pieces; i += GV_WARPS) {
      const int t = i / pieces, k = (i % pieces) * I8_GROUP + lane * 8;
      float v[8];
      times(k, raw[i * 32 + lane], v);
      const float f = i8_factor(most_s[t], I8_MOST);
      uint32_t q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = f == 0.f ? 0u : i8_round_bits(v[e], f);
      if (k < K) *reinterpret_cast<uint2*>(xs + (size_t)t * ldx + k) = make_uint2(i8_pack(q[0], q[1], q[2], q[3]), i8_pack(q[4], q[5], q[6], q[7]));
    }
    if (warp < T) {
      float s = i8_scale(most_s[warp], 1.f / I8_MOST);
      if (p.norm_w != nullptr) s = __fmul_rn(s, rsqrtf(i8_groups_sum(sums + warp * pieces, pieces) / (float)K + p.eps));
      if (lane == 0) s_s[warp] = s;
    }
  } else {
    const int vecs = K / 16;
    for (int i = threadIdx.x; i < T * vecs; i += GV_THREADS) {
      const int t = i / vecs, k = (i % vecs) * 16;
      *reinterpret_cast<uint4*>(xs + (size_t)t * ldx + k) = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const int8_t*>(p.x) + (long long)t * p.ldx + k));
    }
    if (threadIdx.x < T) s_s[threadIdx.x] = __ldcg(p.s + threadIdx.x);
  }
  __syncthreads();

  // (columns past the last token repeat it: their sums are left out)
  const int8_t* xb = xs + (size_t)min(lane >> 2, T - 1) * ldx + (lane & 3) * 16;
  int c[4] = {}, g = gw, st = kw;
  auto step = [&](const uint4 (&w)[2]) {
    const uint4 b = *reinterpret_cast<const uint4*>(xb + st * GV_STEP);     // (past K: whatever it is, the weights are zeros)
    gv_mma(c, w[0].x, w[1].x, w[0].y, w[1].y, b.x, b.y);
    gv_mma(c, w[0].z, w[1].z, w[0].w, w[1].w, b.z, b.w);
    if ((st += KW) >= steps) {                       // this group's share of K is through
      const int row = g * 16 + (lane >> 2), col = (lane & 3) * 2;
      if (r0 + row < r1) {
        if (col < T) atomicAdd(&acc[row * GV_TOKENS + col], c[0]);
        if (col + 1 < T) atomicAdd(&acc[row * GV_TOKENS + col + 1], c[1]);
      }
      if (r0 + row + 8 < r1) {
        if (col < T) atomicAdd(&acc[(row + 8) * GV_TOKENS + col], c[2]);
        if (col + 1 < T) atomicAdd(&acc[(row + 8) * GV_TOKENS + col + 1], c[3]);
      }
      c[0] = c[1] = c[2] = c[3] = 0, st = kw, g += GW;
    }
  };
  for (int i = 0; i < items; i += GV_DEPTH) {
#pragma unroll
    for (int d = 0; d < GV_DEPTH; ++d) {
      if (i + d < items) step(ring[d]);
      load(ring[d], i + d + GV_DEPTH < items);
    }
  }
  __syncthreads();

  // results: neighbouring threads have neighbouring rows
  const int rows = r1 - r0, per = p.epi == I8_SWIGLU ? 2 : 1, outs = rows / per;
  for (int i = threadIdx.x; i < outs * T; i += GV_THREADS) {
    const int t = i / outs, r = (i % outs) * per, n = r0 + r;
    const float s = s_s[t], v = i8_value(acc[r * GV_TOKENS + t], __fmul_rn(s, p.ws[n]));
    const size_t at = (size_t)t * p.ldo;
    if (p.epi == I8_SWIGLU) {
      const float up = i8_value(acc[(r + 1) * GV_TOKENS + t], __fmul_rn(s, p.ws[n + 1]));
      reinterpret_cast<bf16*>(p.out)[at + (n >> 1)] = __float2bfloat16(i8_swiglu(v, up));
    } else if (p.epi == I8_STORE_F32) {
      reinterpret_cast<float*>(p.out)[at + n] = v;
    } else {
      reinterpret_cast<bf16*>(p.out)[at + n] =
          __float2bfloat16(p.epi == I8_RESIDUAL ? __fadd_rn(v, __bfloat162float(__ldcg(p.residual + (size_t)t * p.ldr + n))) : v);
    }
  }
}

constexpr size_t GV_SMEM = 220 * 1024;
size_t gv_smem(int T, int N, int K, int ctas, bool fused) {
  const size_t rows = ((N + 1) / 2 + ctas - 1) / ctas * 2 + 2, pieces = (K + I8_GROUP - 1) / I8_GROUP;
  return (size_t)T * gv_row(K) + rows * GV_TOKENS * 4 + (fused ? T * pieces * (512 + 4) : 0);
}
int gv_ctas(int N) {
  int sms = 0, dev = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return min(sms, (N + 1) / 2);
}

template <bool FUSED>
int gv_launch(GemvI8Params p, cudaStream_t stream) {
  const int ctas = gv_ctas(p.N);
  const size_t smem = gv_smem(p.T, p.N, p.K, ctas, FUSED);
  if (smem > GV_SMEM) return (int)cudaErrorInvalidValue;
  p.kw = GV_WARPS;
  while (p.kw > 1 && p.kw > (p.K + GV_STEP - 1) / GV_STEP) p.kw /= 2;     // (no warp without a step, where K has a few)
  static TrlPerDevice<bool> set;
  bool& configured = set.here();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemv_i8_kernel<FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GV_SMEM);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return (int)trl_launch(gemv_i8_kernel<FUSED>, dim3(ctas), dim3(GV_THREADS), smem, stream, p);
}

}  // namespace

// Whether trl_gemv_i8 takes T rows: 1 as they are (bf16), 2 quantised, 0 not.
int gemv_i8_takes(int T, int N, int K) {
  if (T > GV_TOKENS) return 0;
  const int ctas = gv_ctas(N);
  if (gv_smem(T, N, K, ctas, true) <= GV_SMEM) return 1;
  return gv_smem(T, N, K, ctas, false) <= GV_SMEM ? 2 : 0;
}

// quantised: x is int8 with scales s; else bf16, quantised here (of rmsnorm(x) * norm_w where that is given).
int gemv_i8_launch(const void* w, long ldw, const void* ws, const void* x, long ldx, const void* s, const void* norm_w, float eps, const void* residual,
                   long ldr, void* out, long ldo, int T, int N, int K, int epi, int quantised, cudaStream_t stream) {
  GemvI8Params p{(const int8_t*)w, (const float*)ws, x, (const float*)s, (const float*)norm_w, (const bf16*)residual, out, ldw, ldx, ldr, ldo, T, N, K, epi, 0, eps};
  return quantised ? gv_launch<false>(p, stream) : gv_launch<true>(p, stream);
}
