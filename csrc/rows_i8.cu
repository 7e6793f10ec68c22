// Rows into 8-bit integers with a scale each (activations, weights), and gradients into 16 bits as two digits of 8.
//
//   t = x * w (w: norm weight or none),  m = max |t|,  q = rint(t * ((1 / m) * 127)),  s = m * (1 / 127) [* rsqrt(mean x^2 + eps)]
//   u = g * ws,                          m = max |u|,  Q = rint(u * ((1 / m) * 32512)) = 256 hi + lo,  s = m * (1 / 32512)
//
// A norm's factor is the same for a whole row, so it cancels out of the integers and goes into the scale alone.  One pass: a block takes
// row after row, which stays in registers between its maximum and its integers.  Bound by instructions for many rows (2000 x 5120 bf16: 13 us, 64 % of
// the issue slots, 31 MB; packed fp32 arithmetic takes 8 % of them away and no time), by latency for few (2.5 us).  Bounds of 640 threads twice and of 1024
// leave 48 and 64 registers a thread, and 38 of the 48 forms spill some of what they hold (aligned fp32 of two vectors 72 bytes stored and 48 read a
// thread, unaligned fp32 of five 680 and 296).
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
  long long ldx, ldq, rows;
  int K;
  float eps;
  int norm;
};

// Products ask for their first weights before they wait for the quantiser of their rows (gemm_i8.cu).  So a quantiser lets them start only once it
// has itself waited for all that is ahead of it: whatever wrote the weight (a copy, a quantiser of weights, an optimiser) has then ended, and
// what it wrote can be seen.
__device__ __forceinline__ void rows_enter() {
  pdl_enter();
  pdl_wait();
  pdl_trigger();
}

// Eight values as they lie in memory.
template <typename T>
struct RowsRaw {
  uint4 u[sizeof(T) / 2];
};
template <typename T, bool VEC>
__device__ __forceinline__ RowsRaw<T> rows_load(const T* x, int k, int K) {
  RowsRaw<T> r;
  if (VEC && k + 8 <= K) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = __ldcg(reinterpret_cast<const uint4*>(x + k) + i);
    return r;
  }
  if constexpr (!VEC && sizeof(T) == 4) {
    // a row off its boundary (gradients of an odd number of channels): the three aligned vectors that the eight values lie in, where all of
    // them are the row's.  One by one, 32 bytes from lane to lane, every sector would be asked for eight times.
    if (k >= 4 && k + 12 <= K) {
      const int m = (int)(reinterpret_cast<uintptr_t>(x) >> 2 & 3);
      const uint4* p = reinterpret_cast<const uint4*>(x + k - m);
      const uint4 a = __ldcg(p), b = __ldcg(p + 1), c = __ldcg(p + 2);
      switch (m) {
        case 0: r.u[0] = a, r.u[1] = b; break;
        case 1: r.u[0] = make_uint4(a.y, a.z, a.w, b.x), r.u[1] = make_uint4(b.y, b.z, b.w, c.x); break;
        case 2: r.u[0] = make_uint4(a.z, a.w, b.x, b.y), r.u[1] = make_uint4(b.z, b.w, c.x, c.y); break;
        default: r.u[0] = make_uint4(a.w, b.x, b.y, b.z), r.u[1] = make_uint4(b.w, c.x, c.y, c.z);
      }
      return r;
    }
  }
  T* v = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? __ldcg(x + k + i) : T(0.f);
  return r;
}
template <typename T>
__device__ __forceinline__ void rows_values(const RowsRaw<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const float2 a = bf162_bits_to_f2(r.u[0].x), b = bf162_bits_to_f2(r.u[0].y), c = bf162_bits_to_f2(r.u[0].z), d = bf162_bits_to_f2(r.u[0].w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
  } else {
    const uint32_t b[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(b[i]);
  }
}

// The digits of eight values (rounded: bits) out: byte `digit` of each.
__device__ __forceinline__ void rows_store(int8_t* out, int k, int K, const uint32_t (&q)[8], int digit) {
  const uint32_t pick = digit ? 0x0051u : 0x0040u;
  const uint2 b = make_uint2(__byte_perm(__byte_perm(q[0], q[1], pick), __byte_perm(q[2], q[3], pick), 0x5410),
                             __byte_perm(__byte_perm(q[4], q[5], pick), __byte_perm(q[6], q[7], pick), 0x5410));
  if (k + 8 <= K) {
    *reinterpret_cast<uint2*>(out + k) = b;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) out[k + i] = (int8_t)((i < 4 ? b.x : b.y) >> (8 * (i & 3)));
  }
}
template <bool W16>
__device__ __forceinline__ void rows_give(const RowsParams& p, long long row, int k, const float (&v)[8], float f) {
  uint32_t q[8] = {};
  if (f != 0.f) {                                  // (of a row with an infinity or NaN the products would be NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = i8_round_bits(v[i], f);
  }
  int8_t* out = p.q + (W16 ? 2 : 1) * row * p.ldq;
  if constexpr (W16) {
    rows_store(out + p.ldq, k, p.K, q, 0);         // the low digit is the low byte, a signed one
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] += 128u;      // the high digit goes up where that one is negative
    rows_store(out, k, p.K, q, 1);
  } else {
    rows_store(out, k, p.K, q, 0);
  }
}

// CH: vectors of eight that a thread keeps; 0: a row of any length, read twice.  One vector a thread: the next row's values are on their way
// while this one's maximum is found and its integers leave.  W16: two digits.
template <typename T, int CH, bool VEC, bool W16>
__global__ void __launch_bounds__(CH == 1 ? 640 : 1024, CH == 1 ? 2 : 1) rows_i8_kernel(const RowsParams p) {
  extern __shared__ float groups_s[];            // sums of squares of 256 values each, of two rows in turn
  __shared__ uint32_t most_s[2][32];
  rows_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5, K = p.K, pieces = (K + I8_GROUP - 1) / I8_GROUP;
  const bool squares = !W16 && p.norm;
  constexpr int KEEP = CH ? CH : 1;
  constexpr float MOST = W16 ? I16_MOST : I8_MOST, PART = 1.f / MOST;
  const int chunks = CH ? CH : (K + (int)blockDim.x * 8 - 1) / ((int)blockDim.x * 8);
  auto at = [&](int c) { return (c * (int)blockDim.x + (int)threadIdx.x) * 8; };
  auto source = [&](long long row) { return reinterpret_cast<const T*>(p.x) + row * p.ldx; };
  constexpr int HOLD = CH && CH <= 2 ? CH : 0;   // the factors of a thread's values stay too: all blocks read the same few lines of the L2 cache
  float wreg[HOLD ? HOLD : 1][8];
  auto factors = [&](int c, float (&w)[8]) { rows_values<float>(rows_load<float, VEC>(p.w, at(c), K), w); };
  auto weight = [&](int c, float (&v)[8]) {
    if (p.w == nullptr) return;
    float w[8];
    if constexpr (HOLD == 0) factors(c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], HOLD ? wreg[HOLD ? c : 0][i] : w[i]);
  };
  RowsRaw<T> next[KEEP];
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c) next[c] = rows_load<T, VEC>(source(blockIdx.x), at(c), K);
  }
  if constexpr (HOLD > 0) {
    if (p.w != nullptr) {
#pragma unroll
      for (int c = 0; c < HOLD; ++c) factors(c, wreg[c]);
    }
  }
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    float* groups = groups_s + turn * pieces;
    float t[KEEP][8];
    uint32_t most = 0;
    auto take = [&](int c, const RowsRaw<T>& r, float (&v)[8]) {
      rows_values<T>(r, v);
      if (squares) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
        ss = warp_sum(ss);
        const int g = c * nw + warp;
        if (lane == 0 && g < pieces) groups[g] = ss;
      }
      weight(c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, i8_abs_bits(v[i]));
    };
    if constexpr (CH > 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c) take(c, next[c], t[c]);
      if (CH == 1 && row + gridDim.x < p.rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c) next[c] = rows_load<T, VEC>(source(row + gridDim.x), at(c), K);
      }
    } else {
      for (int c = 0; c < chunks; ++c) take(c, rows_load<T, VEC>(source(row), at(c), K), t[0]);
    }
    most = i8_warp_most(most);
    if (lane == 0) most_s[turn][warp] = most;
    __syncthreads();                               // (one a row: what the next row writes is the other half)
    most = i8_warp_most(lane < nw ? most_s[turn][lane] : 0u);
    const float f = i8_factor(most, MOST);
    auto give = [&](int c, const float (&v)[8]) {
      if (at(c) < K) rows_give<W16>(p, row, at(c), v, f);
    };
    if constexpr (CH > 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c) give(c, t[c]);
      if (CH > 1 && row + gridDim.x < p.rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c) next[c] = rows_load<T, VEC>(source(row + gridDim.x), at(c), K);
      }
    } else {
      for (int c = 0; c < chunks; ++c) {
        rows_values<T>(rows_load<T, VEC>(source(row), at(c), K), t[0]);
        weight(c, t[0]);
        give(c, t[0]);
      }
    }
    if (warp == 0) {
      float s = i8_scale(most, PART);
      if (squares) s = __fmul_rn(s, rsqrtf(i8_groups_sum(groups, pieces) / (float)K + p.eps));
      if (lane == 0) p.s[row] = s;
    }
  }
}

// Long rows in two digits, many of them: what a SM can hold of such a row leaves it idle between the row's maximum and its integers.  So two
// passes, a block 2048 or 8192 channels of every few rows, whose factors stay in registers: the maxima of pieces of 2048, then the
// integers.
constexpr int RL_THREADS = 256, RL_PIECE = RL_THREADS * 8, RL_VECS = 4, RL_ROWS = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(RL_THREADS, 3) rows_most_kernel(const RowsParams p, uint32_t* most) {      // most: [pieces][rows]
  __shared__ uint32_t most_s[2][RL_ROWS][RL_THREADS / 32];
  rows_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = p.K, k = min(blockIdx.x * RL_PIECE + threadIdx.x * 8, K);
  float w[8];
  rows_values<float>(rows_load<float, VEC>(p.w, k, K), w);
  int turn = 0;
  for (long long r0 = blockIdx.y * RL_ROWS; r0 < p.rows; r0 += gridDim.y * RL_ROWS, turn ^= 1) {
    RowsRaw<T> raw[RL_ROWS];
#pragma unroll
    for (int r = 0; r < RL_ROWS; ++r) raw[r] = rows_load<T, VEC>(reinterpret_cast<const T*>(p.x) + min(r0 + r, p.rows - 1) * p.ldx, k, K);
#pragma unroll
    for (int r = 0; r < RL_ROWS; ++r) {
      float v[8];
      rows_values<T>(raw[r], v);
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, i8_abs_bits(__fmul_rn(v[e], w[e])));      // (past the row's end: zeros)
      m = i8_warp_most(m);
      if (lane == 0) most_s[turn][r][warp] = m;
    }
    __syncthreads();                                 // (the next rows' go into the other half)
    if (warp < RL_ROWS && r0 + warp < p.rows) {
      const uint32_t m = i8_warp_most(lane < RL_THREADS / 32 ? most_s[turn][warp][lane] : 0u);
      if (lane == 0) most[(size_t)blockIdx.x * p.rows + r0 + warp] = m;
    }
  }
}
template <typename T, bool VEC>
__global__ void __launch_bounds__(RL_THREADS, 2) rows_digits_kernel(const RowsParams p, const uint32_t* most, int pieces) {
  pdl_launch_dependents();                           // (it runs: the first pass has waited)
  pdl_wait();
  const int lane = threadIdx.x & 31, K = p.K;
  int k[RL_VECS];
  float w[RL_VECS][8];
#pragma unroll
  for (int c = 0; c < RL_VECS; ++c) {
    k[c] = min((blockIdx.x * RL_VECS + c) * RL_PIECE + (int)threadIdx.x * 8, K);
    rows_values<float>(rows_load<float, VEC>(p.w, k[c], K), w[c]);
  }
  // (from the last row on, which the first pass read last)
  for (long long row = p.rows - 1 - blockIdx.y; row >= 0; row -= gridDim.y) {
    RowsRaw<T> raw[RL_VECS];
    const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
#pragma unroll
    for (int c = 0; c < RL_VECS; ++c) raw[c] = rows_load<T, VEC>(x, k[c], K);
    uint32_t m = 0;
    for (int j = lane; j < pieces; j += 32) m = max(m, __ldcg(most + (size_t)j * p.rows + row));
    m = i8_warp_most(m);
    const float f = i8_factor(m, I16_MOST);
#pragma unroll
    for (int c = 0; c < RL_VECS; ++c) {
      float v[8];
      rows_values<T>(raw[c], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(v[e], w[c][e]);
      if (k[c] < K) rows_give<true>(p, row, k[c], v, f);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.s[row] = i8_scale(m, 1.f / I16_MOST);
  }
}
int rows_long_pieces(int K) { return (K + RL_PIECE - 1) / RL_PIECE; }
// (fp32 2000 x 34816: 137 us, 223 in one pass; 1024 x 5120, which one pass holds, 10)
bool rows_long(long long rows, int K, int digits) { return digits == 2 && K > 10240 && rows >= 64; }

template <typename T, bool VEC>
cudaError_t rows_long_launch(const RowsParams& p, void* most, cudaStream_t stream) {
  const int pieces = rows_long_pieces(p.K), wide = (pieces + RL_VECS - 1) / RL_VECS;
  const long long fit = 3 * i8_sms(), fit2 = 2 * i8_sms();
  const cudaError_t e = trl_launch(rows_most_kernel<T, VEC>, dim3(pieces, (unsigned)min((p.rows + RL_ROWS - 1) / RL_ROWS, max(1ll, fit / pieces))), dim3(RL_THREADS), 0,
                                   stream, p, (uint32_t*)most);
  if (e != cudaSuccess) return e;
  return trl_launch(rows_digits_kernel<T, VEC>, dim3(wide, (unsigned)min(p.rows, max(1ll, fit2 / wide))), dim3(RL_THREADS), 0, stream, p, (const uint32_t*)most, pieces);
}

template <typename T, int CH, bool VEC, bool W16>
cudaError_t rows_launch(const RowsParams& p, int threads, cudaStream_t stream) {
  auto kern = rows_i8_kernel<T, CH, VEC, W16>;
  const size_t smem = 2 * (size_t)((p.K + I8_GROUP - 1) / I8_GROUP) * sizeof(float);
  if (smem > 48 * 1024) return cudaErrorInvalidValue;
  // blocks that fit the GPU at a time
  static TrlPerDevice<int> fit[33];
  int& known = fit[threads / 32].here();
  if (known == 0) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem);
    if (e != cudaSuccess) return e;
    known = i8_sms() * max(n, 1);
  }
  return trl_launch(kern, dim3((unsigned)min(p.rows, (long long)known)), dim3(threads), smem, stream, p);
}
template <typename T, bool VEC, bool W16>
cudaError_t rows_launch(const RowsParams& p, cudaStream_t stream) {
  const int vecs = (p.K + 7) / 8;
  // Rows up to 5120 values: a vector a thread, two blocks or more a SM, the next row on its way (2000 x 5120 bf16 13 us; five vectors a thread in
  // blocks of 128 15).  Longer ones: as few vectors a thread as there are threads for.  From 40960 values on a row is read a second time, out of L2.
  const int ch = vecs <= 640 ? 1 : vecs <= 2048 ? 2 : vecs <= 5120 ? (vecs + 1023) / 1024 : 0, threads = ch ? max(32, ((vecs + ch - 1) / ch + 31) / 32 * 32) : 1024;
  switch (ch) {
    case 1: return rows_launch<T, 1, VEC, W16>(p, threads, stream);
    case 2: return rows_launch<T, 2, VEC, W16>(p, threads, stream);
    case 3: return rows_launch<T, 3, VEC, W16>(p, threads, stream);
    case 4: return rows_launch<T, 4, VEC, W16>(p, threads, stream);
    case 5: return rows_launch<T, 5, VEC, W16>(p, threads, stream);
    default: return rows_launch<T, 0, VEC, W16>(p, threads, stream);
  }
}

}  // namespace

// x [rows, K] (type 0: fp32, 1: bf16; rows ldx apart) -> q int8 [rows, ldq], s fp32 [rows].  w: fp32 [K] or null; norm: w is a norm's
// weight, and the row's 1 / rms goes into s.  digits 2: q has two rows of digits a row, 16 bits in all, and w is the channels' scales.
// scratch: 4 bytes a row for every 2048 of its values (two digits only).  ldq and q on 8-byte boundaries.
TRL_API int trl_rows_i8(const void* x, int type, long ldx, const void* w, int norm, float eps, void* q, long ldq, void* s, long rows, int K,
                        int digits, void* scratch, void* stream) {
  if (rows <= 0 || rows > 0x7fffffffl || K <= 0 || ldq < K || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8 || (type != 0 && type != 1) ||
      (digits != 1 && digits != 2) || (norm && (w == nullptr || digits == 2)) || (digits == 2 && w == nullptr) ||
      (scratch == nullptr && digits == 2))
    return (int)cudaErrorInvalidValue;
  RowsParams p{x, (const float*)w, (int8_t*)q, (float*)s, ldx, ldq, rows, K, eps, norm};
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || ldx % (type ? 8 : 4) == 0) && reinterpret_cast<uintptr_t>(w) % 16 == 0;
  if (rows_long(rows, K, digits)) {
    if (type) return (int)(vec ? rows_long_launch<bf16, true>(p, scratch, st) : rows_long_launch<bf16, false>(p, scratch, st));
    return (int)(vec ? rows_long_launch<float, true>(p, scratch, st) : rows_long_launch<float, false>(p, scratch, st));
  }
  if (type) {
    if (digits == 2) return (int)(vec ? rows_launch<bf16, true, true>(p, st) : rows_launch<bf16, false, true>(p, st));
    return (int)(vec ? rows_launch<bf16, true, false>(p, st) : rows_launch<bf16, false, false>(p, st));
  }
  if (digits == 2) return (int)(vec ? rows_launch<float, true, true>(p, st) : rows_launch<float, false, true>(p, st));
  return (int)(vec ? rows_launch<float, true, false>(p, st) : rows_launch<float, false, false>(p, st));
}
