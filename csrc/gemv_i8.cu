// Products of 8-bit integers with one to four rows: y[t, n] = epi((sum_k q[t, k] W[n, k]) * s[t] * ws[n]), as gemm_i8.cu, bound by the read of
// W (reached through trl_linear_i8 there).  The rows are quantised here as rows_i8.cu does it (same integers, same scales), by every
// block for itself, while its first weights are on their way.
//
// One block an SM with an even share of W's rows, in groups of eight, so that all SMs read as long.  A unit is 32 rows x 128 bytes: one copy
// into the ring of the warp that multiplies it (16 warps, two or three stages each: 128 to 192 KB on their way an SM); units go round the warps
// along K, then down the rows.  Rows of W are the A operand of mma.m16n8k32, tokens B.  Sums go into shared memory by integer atomics: exact, so
// their order changes nothing.
//
// Bound by latency: launch, the row's read, its maximum and its integers (two block barriers), sums, results (1 x 5120 x 1024: 4.9 us, of which the
// 5 MB take 0.8).
//
// The reference's FP8 form for few rows is `linear_fp8_gemv` (packages/tilerl-kernels/src/tilerl_kernels/kernels_linear.py:1442-1494).
#include <cuda.h>

#include "int8.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int GV_WARPS = 16, GV_THREADS = GV_WARPS * 32, GV_TOKENS = 4, GV_MOST_STAGES = 3;
constexpr int GV_ROWS = 32, GV_STEP = 128, GV_UNIT = GV_ROWS * GV_STEP;
constexpr int GV_PIECES = 2, GV_MOST_K = GV_PIECES * GV_WARPS * I8_GROUP;      // of 256 values, that a warp keeps of a token
constexpr size_t GV_SMEM = 224 * 1024;

struct GemvI8Params {
  const float* ws;
  const bf16* x;
  const float* norm_w;
  const bf16* residual;
  void* out;
  long long ldx, ldr, ldo;
  int T, N, K, epi, stages;
  float eps;
};

__host__ __device__ constexpr int gv_row(int K) { return (K + 127) / 128 * 128 + 16; }      // bytes of a token in shared memory: eight tokens' 16 bytes hit all banks

__device__ __forceinline__ void gv_mma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void gv_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// TOK: room for so many tokens.
template <int TOK>
__global__ void __launch_bounds__(GV_THREADS, 1)
gemv_i8_kernel(const __grid_constant__ CUtensorMap map32, const __grid_constant__ CUtensorMap map8, const GemvI8Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bars[GV_WARPS * GV_MOST_STAGES];
  __shared__ float s_s[GV_TOKENS];
  __shared__ uint32_t most_s[GV_TOKENS];
  __shared__ int abort_s;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = p.K, T = p.T, S = p.stages, ldx = gv_row(K);
  const int eights = (p.N + 7) / 8;                // this block's rows
  const int r0 = (int)((long long)blockIdx.x * eights / gridDim.x) * 8, r8 = (int)((long long)(blockIdx.x + 1) * eights / gridDim.x) * 8, r1 = min(p.N, r8);
  const int pieces = (K + I8_GROUP - 1) / I8_GROUP;                      // of 256 values: a warp's lanes have eight each
  unsigned char* ring = smem;                                            // [warp][stage][32 rows x 128 bytes]
  int8_t* xs = reinterpret_cast<int8_t*>(ring + (size_t)GV_WARPS * S * GV_UNIT);      // [T][ldx]
  int* acc = reinterpret_cast<int*>(xs + (size_t)T * ldx);               // [r8 - r0][4]
  float* sums = reinterpret_cast<float*>(acc + (r8 - r0) * GV_TOKENS);   // [T][pieces]
  volatile int* abort_flag = &abort_s;

  const int steps = (K + GV_STEP - 1) / GV_STEP, blocks = (r8 - r0 + GV_ROWS - 1) / GV_ROWS, units = steps * blocks;
  const int mine = warp < units ? (units - warp + GV_WARPS - 1) / GV_WARPS : 0;
  const uint32_t ring0 = smem_u32(ring + (size_t)warp * S * GV_UNIT), bar0 = smem_u32(bars + warp * GV_MOST_STAGES);
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(bar0 + 8u * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) abort_s = 0;
  if (threadIdx.x < GV_TOKENS) most_s[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < (r8 - r0) * GV_TOKENS; i += GV_THREADS) acc[i] = 0;
  pdl_launch_dependents();
  __syncthreads();

  auto load = [&](int u, int st) {                 // (one lane) this warp's unit u
    const uint32_t dst = ring0 + (uint32_t)st * GV_UNIT, bar = bar0 + 8u * st;
    const int unit = warp + u * GV_WARPS, k = unit % steps * GV_STEP, row = r0 + unit / steps * GV_ROWS, rows = min(GV_ROWS, r8 - row);
    mbar_expect_tx(bar, (uint32_t)rows * GV_STEP);
    if (rows == GV_ROWS) {
      tma_load_2d(dst, &map32, k, row, bar);
    } else {                                       // the last of this block's rows, eight at a time
      for (int r = 0; r < rows; r += 8) tma_load_2d(dst + (uint32_t)r * GV_STEP, &map8, k, row + r, bar);
    }
  };
  pdl_wait();                                      // (the kernel ahead may have written the weights)
  if (elect_one())
    for (int u = 0; u < min(S, mine); ++u) load(u, u);
  __syncwarp();

  // ---- the rows into integers: a warp has up to two pieces of 256 values of every token, and the norm's factors of those ----
  uint4 raw[GV_PIECES][TOK];
  float w[GV_PIECES][8];
#pragma unroll
  for (int i = 0; i < GV_PIECES; ++i) {
    const int k = (warp + i * GV_WARPS) * I8_GROUP + lane * 8;
#pragma unroll
    for (int t = 0; t < TOK; ++t)
      raw[i][t] = t < T && k < K ? __ldcg(reinterpret_cast<const uint4*>(p.x + (long long)t * p.ldx + k)) : make_uint4(0u, 0u, 0u, 0u);
    float4 a = make_float4(1.f, 1.f, 1.f, 1.f), b = a;                   // (without a norm times 1: exact)
    if (p.norm_w != nullptr && k < K) a = __ldcg(reinterpret_cast<const float4*>(p.norm_w + k)), b = __ldcg(reinterpret_cast<const float4*>(p.norm_w + k) + 1);
    w[i][0] = a.x, w[i][1] = a.y, w[i][2] = a.z, w[i][3] = a.w, w[i][4] = b.x, w[i][5] = b.y, w[i][6] = b.z, w[i][7] = b.w;
  }
  auto values = [&](const uint4& u, float (&v)[8]) {
    const float2 a = bf162_bits_to_f2(u.x), b = bf162_bits_to_f2(u.y), c = bf162_bits_to_f2(u.z), d = bf162_bits_to_f2(u.w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
  };
#pragma unroll
  for (int t = 0; t < TOK; ++t) {
    if (t >= T) break;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < GV_PIECES; ++i) {
      const int piece = warp + i * GV_WARPS;
      if (piece >= pieces) break;
      float v[8];
      values(raw[i][t], v);
      if (p.norm_w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
        ss = warp_sum(ss);
        if (lane == 0) sums[t * pieces + piece] = ss;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, i8_abs_bits(__fmul_rn(v[e], w[i][e])));
    }
    most = i8_warp_most(most);
    if (lane == 0) atomicMax(&most_s[t], most);
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < TOK; ++t) {
    if (t >= T) break;
    const float f = i8_factor(most_s[t], I8_MOST);
#pragma unroll
    for (int i = 0; i < GV_PIECES; ++i) {
      const int k = (warp + i * GV_WARPS) * I8_GROUP + lane * 8;
      float v[8];
      values(raw[i][t], v);
      uint32_t q[8] = {};
      if (f != 0.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = i8_round_bits(__fmul_rn(v[e], w[i][e]), f);
      }
      if (k < K) *reinterpret_cast<uint2*>(xs + (size_t)t * ldx + k) = make_uint2(i8_pack(q[0], q[1], q[2], q[3]), i8_pack(q[4], q[5], q[6], q[7]));
    }
  }
  if (warp < T) {
    float s = i8_scale(most_s[warp], 1.f / I8_MOST);
    if (p.norm_w != nullptr) s = __fmul_rn(s, rsqrtf(i8_groups_sum(sums + warp * pieces, pieces) / (float)K + p.eps));
    if (lane == 0) s_s[warp] = s;
  }
  __syncthreads();

  // ---- this warp's units ----
  // (columns past the last token repeat it: their sums are left out; past K the weights are zeros, whatever the row holds there)
  const uint32_t xb = smem_u32(xs) + (uint32_t)min(lane & 7, T - 1) * ldx + (uint32_t)(lane >> 3) * 16;
  const uint32_t arow = (uint32_t)(lane & 15) * GV_STEP, achunk = (uint32_t)lane >> 4, aswap = (uint32_t)lane & 7;
  int c[2][4] = {}, step = warp % steps, block = warp / steps, st = 0;
  uint32_t ph = 0;
  auto flush = [&] {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int row = block * GV_ROWS + m * 16 + (lane >> 2), col = (lane & 3) * 2;
      if (col < T) {
        const bool two = col + 1 < T;
        if (r0 + row < r1) {
          atomicAdd(&acc[row * GV_TOKENS + col], c[m][0]);
          if (two) atomicAdd(&acc[row * GV_TOKENS + col + 1], c[m][1]);
        }
        if (r0 + row + 8 < r1) {
          atomicAdd(&acc[(row + 8) * GV_TOKENS + col], c[m][2]);
          if (two) atomicAdd(&acc[(row + 8) * GV_TOKENS + col + 1], c[m][3]);
        }
      }
      c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0;
    }
  };
  for (int u = 0; u < mine; ++u) {
    if (!__all_sync(0xffffffffu, mbar_wait(bar0 + 8u * st, ph, abort_flag))) break;
    const uint32_t src = ring0 + (uint32_t)st * GV_UNIT, xk = xb + (uint32_t)step * GV_STEP;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t b[4];
      gv_ldmatrix(b, xk + h * 64);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const uint32_t chunk = ((uint32_t)(h * 4 + s2 * 2) + achunk) ^ aswap;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          uint32_t a[4];
          gv_ldmatrix(a, src + (uint32_t)m * 16 * GV_STEP + arow + chunk * 16);
          gv_mma(c[m], a, b[s2 * 2], b[s2 * 2 + 1]);
        }
      }
    }
    __syncwarp();                                  // all lanes have read the stage
    if (u + S < mine && elect_one()) load(u + S, st);
    __syncwarp();
    if (++st == S) st = 0, ph ^= 1u;
    int next = block;
    step += GV_WARPS;
    while (step >= steps) step -= steps, ++next;
    if (next != block || u + 1 == mine) flush();
    block = next;
  }
  __syncthreads();
  if (*abort_flag) {                               // copies still in flight must land before the memory goes away
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
    return;
  }

  // ---- results: neighbouring threads have neighbouring rows ----
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

int gv_ctas(int N) { return min(i8_sms(), (N + 7) / 8); }
size_t gv_smem(int T, int N, int K, int stages) {
  const int ctas = gv_ctas(N);
  const size_t rows = (size_t)(((N + 7) / 8 + ctas - 1) / ctas + 1) * 8, pieces = (K + I8_GROUP - 1) / I8_GROUP;
  return 1024 + (size_t)GV_WARPS * stages * GV_UNIT + (size_t)T * gv_row(K) + rows * GV_TOKENS * 4 + T * pieces * 4;
}
int gv_stages(int T, int N, int K) {
  for (int s = GV_MOST_STAGES; s >= 2; --s)
    if (gv_smem(T, N, K, s) <= GV_SMEM) return s;
  return 0;
}

template <int TOK>
int gv_launch(const CUtensorMap& m32, const CUtensorMap& m8, const GemvI8Params& p, cudaStream_t stream) {
  static TrlPerDevice<bool> set;
  bool& configured = set.here();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemv_i8_kernel<TOK>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GV_SMEM);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return (int)trl_launch(gemv_i8_kernel<TOK>, dim3(gv_ctas(p.N)), dim3(GV_THREADS), gv_smem(p.T, p.N, p.K, p.stages), stream, m32, m8, p);
}

}  // namespace

bool i8_tensor(CUtensorMap* m, const void* base, long long width, long long rows, long long ld, int box_rows);

// Whether gemv_i8_launch takes T rows.  Weights up to 16 MB, of three or four rows 8: there a launch less counts more than that the pair form's first weights are on their way
// while its rows are quantised (us in a row of products here and in two launches, one row: 320 x 256 3.4 and 5.5, 5120 x 1024 4.9 and 7.2,
// 4096 x 4096 8.3 and 10.7, 5120 x 5120 11.7 and 11.8, 16480 x 5120 19.5 and 19.4; two rows, 5120 x 5120 12.6 and 11.8; three, 5120 x 1600 7.1 and 8.2,
// 16000 x 1024 9.7 and 9.3; four, 5120 x 1024 6.7 and 7.2, 16480 x 5120 22.1 and 19.2).
bool gemv_i8_takes(int T, int N, int K) { return T <= GV_TOKENS && (long long)N * K <= (T > 2 ? 8 : 16) << 20 && K <= GV_MOST_K && gv_stages(T, N, K) > 0; }

// x: bf16 rows, on 16-byte boundaries, quantised here (of rmsnorm(x) * norm_w where that is given).
int gemv_i8_launch(const void* w, long ldw, const void* ws, const void* x, long ldx, const void* norm_w, float eps, const void* residual, long ldr,
                   void* out, long ldo, int T, int N, int K, int epi, cudaStream_t stream) {
  CUtensorMap m32, m8;
  if (!i8_tensor(&m32, w, K, N, ldw, GV_ROWS) || !i8_tensor(&m8, w, K, N, ldw, 8)) return (int)cudaErrorInvalidValue;
  GemvI8Params p{(const float*)ws, (const bf16*)x, (const float*)norm_w, (const bf16*)residual, out, ldx, ldr, ldo, T, N, K, epi, gv_stages(T, N, K), eps};
  return T == 1 ? gv_launch<1>(m32, m8, p, stream) : T == 2 ? gv_launch<2>(m32, m8, p, stream) : gv_launch<4>(m32, m8, p, stream);
}
