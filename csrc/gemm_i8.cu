// Products of 8-bit integers with a scale for each token and each channel, on pairs of SMs (tcgen05.mma.cta_group::2.kind::i8).
//
//   y[t, n]  = epi((sum_k q[t, k] W[n, k]) * s[t] * ws[n])                              (W: int8 [N, K], q: rows_i8.cu)
//   dx[t, k] = s[t] * (256 sum_n hi[t, n] W[n, k] + sum_n lo[t, n] W[n, k])             (gradient of y's input, rows in two digits)
//
// Sums are of 32-bit integers: exact, whatever the order, so K may be shared between SMs without a change of the result.
//
// A tile is 256 features x BN columns.  Features are the A operand: 128 of them a SM, of y's rows of W (K-major), of dx's columns of W
// (M-major: the same copies of 128 x 128 bytes, read across, so the gradient needs no second layout of the weight).  Columns are tokens,
// two a token for dx (high and low digit side by side, put together in the epilogue); each SM holds half of them and the MMA hands them to
// both.  A stage is 128 bytes of the summed dimension: 16 KB of W and BN / 2 x 128 bytes of q a SM, one copy each, four MMAs.  Two
// accumulators in TMEM: the epilogue of a tile runs beside the next one's MMAs.  It turns the values round through shared memory, so that
// they leave as 16-byte pieces of a token's row.  With fewer tiles than pairs, two to four pairs of a cluster share a tile along the summed
// dimension and add their parts through each other's shared memory.
//
// What bounds it.  Many tokens: the tensor cores, at the clocks that the power cap leaves them (2000 x 16 480 x 5120: 116 us alone, tensor pipe 88 % of its
// active cycles; a second of it 144 us, 2.3 POP/s; on another GPU 175).  An MMA of 128 x 256 x 32 takes 128 clocks, as fp8 does and bf16
// with half of K.  Few: the read of W (eight rows of 34 816 x 5120: 35 us from an empty L2 cache, 5.1 TB/s; 32.6 us with the quantiser in a row of
// products, whose first stages are on their way while the rows between them are quantised; it lets them start behind its own wait, for weights
// that were just written, which costs 0.5 to 1 us).  Measured and not taken: W on its way before TMEM
// is taken (the quantiser's few loads then wait behind it: 32.8), half a SM a CTA, so that the next product moves in earlier (four
// stages are too few: 35.6), the head of W fetched into L2 by the quantiser (33.0).
//
// The reference has no integer product; in the place of its `linear_fp8` (packages/tilerl-kernels/src/tilerl_kernels/
// kernels_linear.py:1777-1813) for weights in this format.
#include "int8.cuh"
#include "tcgen05_pair.cuh"

typedef CUresult (*EncodeTiledFnI)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A tensor map of [rows, width] bytes, rows ld apart, in pieces of 128 bytes x box_rows; what lies outside reads as zero
bool i8_tensor(CUtensorMap* m, const void* base, long long width, long long rows, long long ld, int box_rows) {
  static EncodeTiledFnI encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn) return false;
    encode = (EncodeTiledFnI)fn;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int GI_ROWS = 128;                      // features a SM
constexpr int GI_KT = 128;                        // bytes of the summed dimension a stage
constexpr int GI_THREADS = 320;
constexpr int GI_TR_STRIDE = 36;                  // words a token in a warp's turning piece: 32 features, and 4 so that reads spread
constexpr int GI_TR_BYTES = 16 * GI_TR_STRIDE * 4;
constexpr int GI_MAX_PARTS = 4;

template <int BN>
struct I8Cfg {
  static constexpr int A_BYTES = GI_ROWS * GI_KT, B_BYTES = BN / 2 * GI_KT, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 200 * 1024 / STAGE < 9 ? 200 * 1024 / STAGE : 9;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int SMEM = (RING < 160 * 1024 ? 160 * 1024 : RING) + 8 * GI_TR_BYTES + 512 + 1024;
  static constexpr int TMEM_COLS = BN <= 64 ? 128 : BN <= 128 ? 256 : 512;
  static_assert(SMEM <= 227 * 1024 && 2 * BN <= TMEM_COLS && STAGE % 1024 == 0, "layout");
  static_assert(SMEM > 227 * 1024 / 2 + 1024, "no other kernel with TMEM fits beside it on an SM");
  static_assert(BN * GI_ROWS * 4 <= RING, "parts of a shared tile lie in the ring");
};

struct I8Params {
  const float* ws;       // [N]
  const float* s;        // [T]
  const bf16* residual;
  void* out;
  long long ldr, ldo;
  int features, tokens, depth, nk, r_tiles, c_tiles, epi;
  int rows;              // features that a SM's 128 rows hold: fewer, in steps of eight, where the pairs of SMs share W more evenly that way
  int vec;               // 8 features of a token are one aligned vector of the output (of SwiGLU four results) and of the residual
  int parts;             // pairs that share a tile (a cluster), each a part of the summed dimension; 1: a pair goes through whole tiles
};

__device__ __forceinline__ void gi_mma(uint32_t d_tmem, uint32_t alo, uint32_t blo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 da, db;\n"
      "  mov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};\n"
      "  setp.ne.b32 p, %5, 0;\n"
      "  tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %4, p; }\n"
      ::"r"(d_tmem), "r"(alo), "r"(blo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ int4 gi_ld_cluster(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Eight features of a token (of both its columns, J = 2), summed over the parts; all of them are asked for before the first is added.
template <int PARTS, int J>
__device__ __forceinline__ void gi_join(uint32_t at, int rank, int (&y)[J][8]) {
  int4 x[PARTS][J][2];
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
    const uint32_t src = gp_map(at, 2 * q + rank);
#pragma unroll
    for (int j = 0; j < J; ++j) x[q][j][0] = gi_ld_cluster(src + j * GI_ROWS * 4), x[q][j][1] = gi_ld_cluster(src + j * GI_ROWS * 4 + 16);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[j][e] = 0;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      const int4 a = x[q][j][0], b = x[q][j][1];
      y[j][0] += a.x, y[j][1] += a.y, y[j][2] += a.z, y[j][3] += a.w, y[j][4] += b.x, y[j][5] += b.y, y[j][6] += b.z, y[j][7] += b.w;
    }
  }
}

// The residual's eight features of a token, asked for well before they are added.
__device__ __forceinline__ uint4 gi_residual8(const I8Params& p, int tok, int f) {
  if (tok >= p.tokens || f >= p.features) return make_uint4(0u, 0u, 0u, 0u);
  return __ldcg(reinterpret_cast<const uint4*>(p.residual + (size_t)tok * p.ldr + f));
}
// Eight features of a token out as one vector (v: results before the residual, which is u or still to be read).
template <bool READ>
__device__ __forceinline__ void gi_store8(const I8Params& p, int tok, int f, const float (&v)[8], uint4 u) {
  if (tok >= p.tokens || f >= p.features) return;
  const size_t at = (size_t)tok * p.ldo;
  if (p.epi == I8_SWIGLU) {                          // features in (gate, up) pairs
    *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.out) + at + (f >> 1)) =
        make_uint2(f2_to_bf162_bits(i8_swiglu(v[0], v[1]), i8_swiglu(v[2], v[3])), f2_to_bf162_bits(i8_swiglu(v[4], v[5]), i8_swiglu(v[6], v[7])));
  } else if (p.epi == I8_STORE_F32) {
    float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at + f);
    o[0] = make_float4(v[0], v[1], v[2], v[3]), o[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = v[i];
    if (p.epi == I8_RESIDUAL) {
      if (!READ) u = gi_residual8(p, tok, f);
      const float2 a = bf162_bits_to_f2(u.x), b = bf162_bits_to_f2(u.y), c = bf162_bits_to_f2(u.z), d = bf162_bits_to_f2(u.w);
      y[0] = __fadd_rn(y[0], a.x), y[1] = __fadd_rn(y[1], a.y), y[2] = __fadd_rn(y[2], b.x), y[3] = __fadd_rn(y[3], b.y);
      y[4] = __fadd_rn(y[4], c.x), y[5] = __fadd_rn(y[5], c.y), y[6] = __fadd_rn(y[6], d.x), y[7] = __fadd_rn(y[7], d.y);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(p.out) + at + f) =
        make_uint4(f2_to_bf162_bits(y[0], y[1]), f2_to_bf162_bits(y[2], y[3]), f2_to_bf162_bits(y[4], y[5]), f2_to_bf162_bits(y[6], y[7]));
  }
}
// N results out one by one, for outputs that take no vectors: `there` of them, tok_step tokens and f_step features apart.  SwiGLU: v and up are a
// pair's.  (All values are at hand before the first store: a shuffle or a load between the stores would wait for each of them.)
template <int N>
__device__ __forceinline__ void gi_store_each(const I8Params& p, int tok, int tok_step, int f, int f_step, int there, const float (&v)[N], const float (&up)[N]) {
  const size_t at = (size_t)tok * p.ldo + (p.epi == I8_SWIGLU ? f >> 1 : f);
  const size_t step = (size_t)tok_step * p.ldo + (p.epi == I8_SWIGLU ? f_step >> 1 : f_step);
  if (p.epi == I8_SWIGLU) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) reinterpret_cast<bf16*>(p.out)[at + i * step] = __float2bfloat16(i8_swiglu(v[i], up[i]));
  } else if (p.epi == I8_STORE_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) reinterpret_cast<float*>(p.out)[at + i * step] = v[i];
  } else if (p.epi == I8_RESIDUAL) {
    float r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = i < there ? __bfloat162float(__ldcg(p.residual + (size_t)(tok + i * tok_step) * p.ldr + f + i * f_step)) : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) reinterpret_cast<bf16*>(p.out)[at + i * step] = __float2bfloat16(__fadd_rn(v[i], r[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < there) reinterpret_cast<bf16*>(p.out)[at + i * step] = __float2bfloat16(v[i]);
  }
}

// GRAD: results are dx; two columns a token.  SPLIT: a cluster's pairs share a tile.
template <int BN, bool GRAD, bool SPLIT>
__global__ void __launch_bounds__(GI_THREADS, 1)
gemm_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, const I8Params p) {
  using C = I8Cfg<BN>;
  constexpr int STAGES = C::STAGES, J = GRAD ? 2 : 1;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* turn = smem + C::RING;
  uint64_t* bars = reinterpret_cast<uint64_t*>(turn + 8 * GI_TR_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int part = SPLIT ? pair % p.parts : 0, even = 2 * part;          // even: the cluster's CTA that issues for this pair
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };                              // the even SM's counts both SMs' copies
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };   // of the even SM: both SMs' epilogue warps

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 16);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // (TMEM of a pair is taken by both SMs together: only once both CTAs are known to run)
  gp_cluster_sync();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  gp_cluster_sync();                                // both halves are allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();

  // Whole tiles, every `pairs`-th one; columns run fastest, so that the pairs at work share a few tiles' features and all columns, and the
  // L2 cache holds both while they do.
  const int tiles = p.r_tiles * p.c_tiles, tile0 = SPLIT ? pair / p.parts : pair, tile1 = SPLIT ? tile0 + 1 : tiles, tile_step = SPLIT ? 1 : pairs;
  const int my_tiles = tile1 > tile0 ? (tile1 - tile0 + tile_step - 1) / tile_step : 0;
  const int k0 = SPLIT ? (int)((long long)part * p.nk / p.parts) : 0, k1 = SPLIT ? (int)((long long)(part + 1) * p.nk / p.parts) : p.nk;

  // Parts of a shared tile: this pair adds up tokens join_t .. join_t1 of it, a thread of the epilogue's eight features of every sixteenth one.  What
  // that needs besides the parts is asked for before the tile's sums are waited for (a barrier of the cluster waits for loads, too).
  constexpr int TOKENS = BN / J, JOIN_STEP = (GI_THREADS - 64) / 16;
  const int join_r = (threadIdx.x & 15) * 8;
  int join_t = 0, join_t1 = 0, join_f = 0;
  float join_ws[8], join_scale = 0.f;
  uint4 join_res = make_uint4(0u, 0u, 0u, 0u);
  auto scale_of = [&](int t) { return t < join_t1 ? __ldcg(p.s + tile0 % p.c_tiles * TOKENS + t) : 0.f; };
  auto residual_of = [&](int t) {
    return !GRAD && p.epi == I8_RESIDUAL && p.vec && t < join_t1 ? gi_residual8(p, tile0 % p.c_tiles * TOKENS + t, join_f) : make_uint4(0u, 0u, 0u, 0u);
  };

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      const uint32_t smem0 = smem_u32(smem);
      const int units = my_tiles * (k1 - k0);
      auto load_w = [&](int rt, int kt, int st) {
        const uint32_t dst = smem0 + (uint32_t)st * C::STAGE, bar = gp_map(full(st), even);
        const int f = (rt * 2 + rank) * p.rows;
        if (rank == 0) mbar_expect_tx(full(st), 2u * (uint32_t)(p.rows * GI_KT + C::B_BYTES));
        gp_load_2d(dst, &map_w, GRAD ? f : kt * GI_KT, GRAD ? kt * GI_KT : f, bar);
      };
      auto load_q = [&](int ct, int kt, int st) {
        gp_load_2d(smem0 + (uint32_t)st * C::STAGE + C::A_BYTES, &map_q, kt * GI_KT, ct * BN + rank * (BN / 2), gp_map(full(st), even));
      };
      int w_tile = tile0, w_rt = tile0 / p.c_tiles, w_kt = k0, q_tile = tile0, q_ct = tile0 % p.c_tiles, q_kt = k0, st = 0;
      uint32_t ph = 0;
      auto next_w = [&] { if (++w_kt == k1) w_kt = k0, w_tile += tile_step, w_rt = w_tile / p.c_tiles; };
      const int pre = min(STAGES, units);
      for (int u = 0; u < pre; ++u) load_w(w_rt, w_kt, u), next_w();       // the kernel ahead, the rows' quantiser, runs: what wrote the weights has ended (rows_i8.cu)
      pdl_wait();
      for (int u = 0; u < units; ++u) {
        if (u >= pre) {
          if (!mbar_wait(empty(st), ph ^ 1u, abort_flag)) break;
          load_w(w_rt, w_kt, st), next_w();
        }
        load_q(q_ct, q_kt, st);
        if (++q_kt == k1) q_kt = k0, q_tile += tile_step, q_ct = q_tile % p.c_tiles;
        if (++st == STAGES) st = 0, ph ^= 1u;
      }
      // the last arrivals of the even SM's MMAs on this CTA's barriers, before its memory goes away
      for (int s = 0; s < pre; ++s) {
        const int u = units - pre + s;              // the last unit of its stage
        if (!mbar_wait(empty(u % STAGES), (uint32_t)(u / STAGES) & 1u, abort_flag)) break;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (for both SMs) ----------------
    pdl_wait();
    if (rank == 0 && elect_one()) {
      // sums of 32 bits, both operands signed; dx: A with the features side by side
      constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((GRAD ? 1u : 0u) << 15) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((2 * GI_ROWS) >> 4) << 24);
      // 32 bytes of a row further along K; across, 32 rows of 128 bytes (and 1024 bytes from eight rows to the next eight either way)
      constexpr uint32_t A_STEP = GRAD ? 32 * GI_KT >> 4 : 2;
      const uint64_t d_op = desc_sw128(smem_u32(smem));
      const uint32_t op_lo = (uint32_t)d_op, op_hi = (uint32_t)(d_op >> 32);
      int st = 0;
      uint32_t ph = 0;
      const uint16_t both = (uint16_t)(3u << even);
      bool ok = true;
      for (int n = 0; ok && n < my_tiles; ++n) {
        const int buf = n & 1;
        if (n >= 2) {
          ok = mbar_wait(acc_empty(buf), (uint32_t)((n >> 1) - 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        const uint32_t acc = tmem_base + (uint32_t)buf * BN;
        for (int kt = k0; kt < k1; ++kt) {
          ok = mbar_wait(full(st), ph, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t off = (uint32_t)st * (uint32_t)(C::STAGE >> 4);
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
            gi_mma(acc, op_lo + off + kb * A_STEP, op_lo + off + (C::A_BYTES >> 4) + kb * 2, op_hi, idesc, kt > k0 || kb ? 1u : 0u);
          gp_commit(empty(st), both);
          if (++st == STAGES) st = 0, ph ^= 1u;
        }
        if (ok) gp_commit(acc_full(buf), both);
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..9) ----------------
    pdl_wait();
    const int quad = warp & 3, half = (warp - 2) >> 2;
    constexpr int COLS = BN / 2, CHUNKS = COLS / 32, TOK = 32 / J;      // a warp's columns, in pieces of 32
    int* tr = reinterpret_cast<int*>(turn + (warp - 2) * GI_TR_BYTES);
    int* sum = reinterpret_cast<int*>(smem);        // parts: [column][128 features] of this CTA's, in the ring, which is through by then
    const uint32_t even_empty = gp_map(acc_empty(0), even);
    if (SPLIT) {
      const int tokens = min(TOKENS, p.tokens - tile0 % p.c_tiles * TOKENS);
      join_t = part * tokens / p.parts + (int)((threadIdx.x - 64) >> 4), join_t1 = (part + 1) * tokens / p.parts;
      join_f = join_r < p.rows ? (tile0 / p.c_tiles * 2 + rank) * p.rows + join_r : p.features;
#pragma unroll
      for (int e = 0; e < 8; ++e) join_ws[e] = !GRAD && join_f + e < p.features ? p.ws[join_f + e] : 0.f;
      join_scale = scale_of(join_t), join_res = residual_of(join_t);
    }
    for (int n = 0; n < my_tiles; ++n) {
      const int tile = tile0 + n * tile_step, buf = n & 1, rt = tile / p.c_tiles, ct = tile % p.c_tiles;
      const int row = quad * 32 + (p.vec ? (lane & 3) * 8 : lane), f0 = row < p.rows ? (rt * 2 + rank) * p.rows + row : p.features;      // this lane's first feature as they leave
      const int tok0 = (ct * BN + half * COLS) / J;
      float ws[8], s[CHUNKS];
#pragma unroll
      for (int i = 0; i < 8; ++i) ws[i] = !GRAD && !SPLIT && f0 + i < p.features && (p.vec || i == 0) ? p.ws[f0 + i] : 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) s[c] = !SPLIT && lane < TOK && tok0 + c * TOK + lane < p.tokens ? __ldcg(p.s + tok0 + c * TOK + lane) : 0.f;
      // (the warps of a group do not meet: each has its own barrier phase and its own piece of shared memory)
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full(buf), (uint32_t)(n >> 1) & 1u, abort_flag))) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + half * COLS);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        uint32_t r[32];
        // (wider tiles read the residual where it is added: behind long sums the other accumulator's MMAs hide that wait, behind a few stages nothing does)
        constexpr bool EARLY = BN <= 128;
        uint4 res[TOK / 8];
        if (!GRAD && !SPLIT && EARLY && p.epi == I8_RESIDUAL && p.vec) {
#pragma unroll
          for (int i = 0; i < TOK / 8; ++i) res[i] = gi_residual8(p, tok0 + c * TOK + i * 8 + (lane >> 2), f0);
        }
        tc_ld32(taddr + (uint32_t)(c * 32), r);
        tc_wait_ld();
        if (c == CHUNKS - 1) {                       // read out: the accumulator goes back
          tc_fence_before();
          __syncwarp();
          if (lane == 0)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(even_empty + 8u * buf) : "memory");
        }
        if (SPLIT) {
          if (tok0 + c * TOK >= p.tokens) continue;
#pragma unroll
          for (int t = 0; t < 32; ++t) sum[(size_t)(half * COLS + c * 32 + t) * GI_ROWS + quad * 32 + lane] = (int)r[t];
        } else {
#pragma unroll
          for (int h = 0; h < TOK; h += 16) {        // 16 tokens at a time
            if (tok0 + c * TOK + h >= p.tokens) break;
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const int x = h + u;
              tr[u * GI_TR_STRIDE + lane] = GRAD ? __float_as_int(fmaf(256.f, (float)(int)r[x * J], (float)(int)r[x * J + J - 1])) : (int)r[x];
            }
            __syncwarp();
            auto value = [&](int x, float st, float scale) { return GRAD ? __fmul_rn(__int_as_float(x), st) : i8_value(x, __fmul_rn(st, scale)); };
            if (p.vec) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int u = i * 8 + (lane >> 2);
                const float st = __shfl_sync(0xffffffffu, s[c], h + u);
                const int* src = tr + u * GI_TR_STRIDE + (lane & 3) * 8;
                const int4 a = reinterpret_cast<const int4*>(src)[0], b = reinterpret_cast<const int4*>(src)[1];
                const int x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = value(x[e], st, ws[e]);
                gi_store8<EARLY>(p, tok0 + c * TOK + h + u, f0, v, EARLY ? res[h / 8 + i] : make_uint4(0u, 0u, 0u, 0u));
              }
            } else {
              float v[16], up[16];
#pragma unroll
              for (int u = 0; u < 16; ++u) v[u] = value(tr[u * GI_TR_STRIDE + lane], __shfl_sync(0xffffffffu, s[c], h + u), ws[0]);
              if (p.epi == I8_SWIGLU) {
#pragma unroll
                for (int u = 0; u < 16; ++u) up[u] = __shfl_down_sync(0xffffffffu, v[u], 1);
              }
              const int tok = tok0 + c * TOK + h;
              if (f0 < p.features && !(p.epi == I8_SWIGLU && (lane & 1))) gi_store_each<16>(p, tok, 1, f0, 0, p.tokens - tok, v, up);
            }
          }
        }
      }
    }
  }

  if constexpr (SPLIT) {
    // each pair of the cluster adds up its share of the tokens
    gp_cluster_sync();
    for (int t = join_t; warp >= 2 && t < join_t1; t += JOIN_STEP, join_scale = scale_of(t), join_res = residual_of(t)) {
      const int tok = tile0 % p.c_tiles * TOKENS + t, f = join_f;
      int y[J][8];
      const uint32_t src = smem_u32(smem) + (uint32_t)(t * J * GI_ROWS + join_r) * 4u;
      if (p.parts == 2) gi_join<2, J>(src, rank, y);
      else if (p.parts == 3) gi_join<3, J>(src, rank, y);
      else gi_join<4, J>(src, rank, y);
      if (f >= p.features) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = GRAD ? __fmul_rn(fmaf(256.f, (float)y[0][e], (float)y[J - 1][e]), join_scale) : i8_value(y[0][e], __fmul_rn(join_scale, join_ws[e]));
      if (p.vec) {
        gi_store8<true>(p, tok, f, v, join_res);
      } else if (p.epi == I8_SWIGLU) {
        const float gate[4] = {v[0], v[2], v[4], v[6]}, up[4] = {v[1], v[3], v[5], v[7]};
        gi_store_each<4>(p, tok, 0, f, 2, (p.features - f + 1) / 2, gate, up);
      } else {
        gi_store_each<8>(p, tok, 0, f, 1, p.features - f, v, v);
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // give copies that are still in flight time to land before the CTAs' memory goes away
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
  }
  gp_cluster_sync();                                // nothing of the pair is in flight towards the other SM any more
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  gp_cluster_sync();                                // no CTA leaves while the other's half is being given back
}

template <int BN, bool GRAD, bool SPLIT>
cudaError_t gi_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int ctas, int parts, cudaStream_t stream) {
  auto kern = gemm_i8_kernel<BN, GRAD, SPLIT>;
  static TrlPerDevice<bool> set;
  bool& configured = set.here();
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, I8Cfg<BN>::SMEM);
    if (e != cudaSuccess) return e;
    configured = true;
  }
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(GI_THREADS), cfg.dynamicSmemBytes = I8Cfg<BN>::SMEM, cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * parts, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = g_trl_use_pdl ? 2 : 1;
  return cudaSuccess;
}

// Clusters of `parts` pairs that fit the GPU at a time.
int gi_clusters(int parts) {
  static TrlPerDevice<int> counts[GI_MAX_PARTS + 1];
  int& known = counts[parts].here();
  if (known == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (gi_config<64, false, true>(cfg, attr, 2 * parts, parts, nullptr) != cudaSuccess) return 0;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_i8_kernel<64, false, true>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    known = n > 0 ? n : -1;
  }
  return known;
}

struct I8Plan {
  int bn, parts, pairs, rows;
};

// Columns a tile and pairs a tile, by the least of: what a launch costs (us), rounds x stages x the time of a stage, putting parts together.
// Measured with the row quantiser, us: 24 rows of 5120 x 17408 with one pair a tile 33.0, two 24.6, three 23.2; of 5120 x 1024 7.4, 8.4, 8.7; 1024 rows of
// 5120 x 6144 with 64, 128, 192, 256 columns 61.7, 46.0, 41.8, 48.4; 512 rows of 34816 x 5120 125, 86.2, 78.9, 70.9.
// One tile of columns: a launch reads W once and is over when the pair with the most of it is, so tiles may have 192 to 240 of 256 features: where the
// tiles are more than pairs (eight rows of 20 000 x 2992 19.3 -> 17.8 us), or few enough that three quarters of the pairs have one afterwards
// (of 10 000 x 4096 13.9 -> 13.2).  From there on memory is busy, and more pairs are no gain (16 480 x 5120, 224 features on 74 pairs instead of 256 on
// 65: 18.6 -> 19.0).
I8Plan gi_plan(int cols, int features, int nk, bool narrow) {
  const int pairs = i8_sms() / 2;
  static const struct { int bn; double launch, stage; } forms[] = {{64, 5.25, 0.2}, {128, 6, 0.25}, {192, 6.65, 0.33}, {256, 7.35, 0.4}};
  static const double join[GI_MAX_PARTS + 1] = {0, 0, 2.5, 3.2, 3.8};
  I8Plan best{0, 1, pairs, GI_ROWS};
  double least = 0;
  for (const auto& f : forms) {
    for (int R = GI_ROWS; R >= (narrow && cols <= 64 ? 96 : GI_ROWS); R -= 8) {
      const long long T = (long long)((features + 2 * R - 1) / (2 * R)) * ((cols + f.bn - 1) / f.bn);
      for (int S = 1; S <= GI_MAX_PARTS; ++S) {
        if (S > 1 && (nk < 4 * S || T * S > pairs || T > gi_clusters(S))) break;
        if (R < GI_ROWS && T <= pairs && T * S * 4 > pairs * 3) continue;
        const double stage = f.stage * (R * GI_KT + f.bn / 2 * GI_KT) / (GI_ROWS * GI_KT + f.bn / 2 * GI_KT);
        const double cost = f.launch + (double)((T + pairs - 1) / pairs) * ((nk + S - 1) / S) * stage + join[S];
        if (!best.bn || cost < (R < GI_ROWS ? 0.97 : 1) * least) best = I8Plan{f.bn, S, pairs, R}, least = cost;
      }
    }
    if (cols <= f.bn) break;
  }
  return best;
}

template <int BN, bool GRAD>
int gi_launch(const void* w, long long ldw, const void* q, long long ldq, int width, int rows, I8Params p, const I8Plan& plan, cudaStream_t stream) {
  constexpr int J = GRAD ? 2 : 1;
  CUtensorMap mw, mq;
  if (!i8_tensor(&mw, w, width, rows, ldw, GRAD ? GI_KT : plan.rows) || !i8_tensor(&mq, q, p.depth, (long long)p.tokens * J, ldq, BN / 2)) return (int)cudaErrorInvalidValue;
  p.rows = plan.rows, p.r_tiles = (p.features + 2 * p.rows - 1) / (2 * p.rows), p.c_tiles = (p.tokens * J + BN - 1) / BN, p.parts = plan.parts;
  const long long tiles = (long long)p.r_tiles * p.c_tiles;
  if (tiles > 0x7fffffffll / p.nk) return (int)cudaErrorInvalidValue;
  const int pairs = plan.parts > 1 ? (int)tiles * plan.parts : (int)(tiles < plan.pairs ? tiles : plan.pairs);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const cudaError_t e = plan.parts > 1 ? gi_config<BN, GRAD, true>(cfg, attr, 2 * pairs, plan.parts, stream) : gi_config<BN, GRAD, false>(cfg, attr, 2 * pairs, 1, stream);
  if (e != cudaSuccess) return (int)e;
  return (int)(plan.parts > 1 ? cudaLaunchKernelEx(&cfg, gemm_i8_kernel<BN, GRAD, true>, mw, mq, p) : cudaLaunchKernelEx(&cfg, gemm_i8_kernel<BN, GRAD, false>, mw, mq, p));
}

template <bool GRAD>
int gi_launch(const void* w, long long ldw, const void* q, long long ldq, int width, int rows, I8Params& p, cudaStream_t stream) {
  constexpr int J = GRAD ? 2 : 1;
  p.nk = (p.depth + GI_KT - 1) / GI_KT;
  const I8Plan plan = gi_plan(p.tokens * J, p.features, p.nk, !GRAD);
  switch (plan.bn) {
    case 64: return gi_launch<64, GRAD>(w, ldw, q, ldq, width, rows, p, plan, stream);
    case 128: return gi_launch<128, GRAD>(w, ldw, q, ldq, width, rows, p, plan, stream);
    case 192: return gi_launch<192, GRAD>(w, ldw, q, ldq, width, rows, p, plan, stream);
    default: return gi_launch<256, GRAD>(w, ldw, q, ldq, width, rows, p, plan, stream);
  }
}

// Values a sum: activations go up to 127 and weights to 128 in magnitude, and 127 * 128 times as many is below 2^31.  A gradient's low digits go down
// to -128, but that of its row's largest value, which is at 127 * 256, is 0, and 128 * 128 times one less is below 2^31 too.
constexpr int GI_MOST = 131072, GI_WIDEST = 1 << 24;      // (and channels)
bool gi_operands(const void* w, long long ldw, int K, const void* q, long long ldq) {
  return reinterpret_cast<uintptr_t>(w) % 16 == 0 && ldw % 16 == 0 && ldw >= K && reinterpret_cast<uintptr_t>(q) % 16 == 0 && ldq % 16 == 0;
}

}  // namespace

// out[t, n] = epi(...).  w and q: rows on 16-byte boundaries.  K up to 131072 (sums of 32 bits); SwiGLU: N even, rows of w in (gate, up)
// pairs, out [T, N / 2].
static int gi_linear(const void* w, long ldw, const void* ws, const void* q, long ldq, const void* s, const void* residual, long ldr, void* out,
                        long ldo, int T, int N, int K, int epi, void* stream) {
  if (T <= 0 || T > (1 << 30) || N <= 0 || N > GI_WIDEST || K <= 0 || K > GI_MOST || epi < 0 || epi > 3 || (epi == I8_SWIGLU && N % 2) ||
      (epi == I8_RESIDUAL) != (residual != nullptr) || !gi_operands(w, ldw, K, q, ldq) || ldq < K)
    return (int)cudaErrorInvalidValue;
  I8Params p{};
  p.ws = (const float*)ws, p.s = (const float*)s, p.residual = (const bf16*)residual, p.out = out, p.ldr = ldr, p.ldo = ldo;
  p.features = N, p.tokens = T, p.depth = K, p.epi = epi;
  const uintptr_t o = reinterpret_cast<uintptr_t>(out), r = reinterpret_cast<uintptr_t>(residual);
  p.vec = N % 8 == 0 && (epi == I8_SWIGLU ? o % 8 == 0 && ldo % 4 == 0 : epi == I8_STORE_F32 ? o % 16 == 0 && ldo % 4 == 0 : o % 16 == 0 && ldo % 8 == 0) &&
          (epi != I8_RESIDUAL || (r % 16 == 0 && ldr % 8 == 0));
  return gi_launch<false>(w, ldw, q, ldq, K, N, p, (cudaStream_t)stream);
}

// dx[t, k], fp32, of rows in two digits: q [2 T, ldq].
static int gi_grad(const void* w, long ldw, const void* q, long ldq, const void* s, void* dx, long ldo, int T, int N, int K, void* stream) {
  if (T <= 0 || T > (1 << 29) || N <= 0 || N > GI_MOST || K <= 0 || K > GI_MOST || !gi_operands(w, ldw, K, q, ldq) || ldq < N) return (int)cudaErrorInvalidValue;
  I8Params p{};
  p.s = (const float*)s, p.out = dx, p.ldo = ldo, p.features = K, p.tokens = T, p.depth = N, p.epi = I8_STORE_F32;
  p.vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(dx) % 16 == 0 && ldo % 4 == 0;
  return gi_launch<true>(w, ldw, q, ldq, K, N, p, (cudaStream_t)stream);
}

bool gemv_i8_takes(int T, int N, int K);
int gemv_i8_launch(const void* w, long ldw, const void* ws, const void* x, long ldx, const void* norm_w, float eps, const void* residual, long ldr,
                   void* out, long ldo, int T, int N, int K, int epi, cudaStream_t stream);
extern "C" int trl_rows_i8(const void* x, int type, long ldx, const void* w, int norm, float eps, void* q, long ldq, void* s, long rows, int K, int digits,
                           void* scratch, void* stream);

// out[t, n] = epi(norm(x) . w): rows of x (type 0: fp32, 1: bf16) quantised, multiplied.  norm_w: a norm's weight, or null.  scratch: T * K
// bytes for the integers and 4 * T for the scales, on a 16-byte boundary, K % 16 == 0.  Otherwise as above.  Returns minus the number of launches,
// or an error.
TRL_API int trl_linear_i8(const void* x, int type, long ldx, const void* norm_w, float eps, const void* w, long ldw, const void* ws, const void* residual,
                          long ldr, void* out, long ldo, void* scratch, int T, int N, int K, int epi, void* stream) {
  if (T <= 0 || T > (1 << 30) || N <= 0 || N > GI_WIDEST || K <= 0 || K > GI_MOST || K % 16 || epi < 0 || epi > 3 || (epi == I8_SWIGLU && N % 2) ||
      (epi == I8_RESIDUAL) != (residual != nullptr) || !gi_operands(w, ldw, K, scratch, K))
    return (int)cudaErrorInvalidValue;
  // (in one launch every block reads all of x, while others write results already: not into the same memory)
  const int width = epi == I8_SWIGLU ? N / 2 : N, size = epi == I8_STORE_F32 ? 4 : 2;
  const char *x0 = (const char*)x, *y0 = (const char*)out, *x1 = x0 + 2 * ((long long)(T - 1) * ldx + K), *y1 = y0 + size * ((long long)(T - 1) * ldo + width);
  const bool whole = (x1 <= y0 || y1 <= x0) && type == 1 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx % 8 == 0) && reinterpret_cast<uintptr_t>(norm_w) % 16 == 0;
  if (whole && gemv_i8_takes(T, N, K)) {
    const int rc = gemv_i8_launch(w, ldw, ws, x, ldx, norm_w, eps, residual, ldr, out, ldo, T, N, K, epi, (cudaStream_t)stream);
    return rc ? rc : -1;
  }
  void* s = (int8_t*)scratch + (size_t)T * K;
  int rc = trl_rows_i8(x, type, ldx, norm_w, norm_w != nullptr, eps, scratch, K, s, T, K, 1, nullptr, stream);
  if (!rc) rc = gi_linear(w, ldw, ws, scratch, K, s, residual, ldr, out, ldo, T, N, K, epi, stream);
  return rc ? rc : -2;
}

// dx[t, k] of g [T, N] (type 0: fp32, 1: bf16).  scratch on a 16-byte boundary: 2 * T rows of N rounded up to 16 bytes, 4 * T for the scales, and 4 * T
// for every 2048 channels.
TRL_API int trl_linear_i8_grad(const void* g, int type, long ldg, const void* w, long ldw, const void* ws, void* dx, long ldo, void* scratch, int T, int N, int K,
                               void* stream) {
  if (T <= 0 || N <= 0 || N > GI_MOST) return (int)cudaErrorInvalidValue;
  const long ldq = (N + 15) / 16 * 16;
  char* s = (char*)scratch + 2 * (size_t)T * ldq;
  const int rc = trl_rows_i8(g, type, ldg, ws, 0, 0.f, scratch, ldq, s, T, N, 2, s + 4 * (size_t)T, stream);
  return rc ? rc : gi_grad(w, ldw, scratch, ldq, s, dx, ldo, T, N, K, stream);
}
