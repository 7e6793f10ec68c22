// Losses over the rows of logits that policy and preference training form, with their gradients: the clipped policy loss with a KL
// term, and the preference loss of pairs of sequences.
//
//   m = max x, s = sum exp(x - m), lp = x[t] - m - log s                  a row, its target t
//   policy      rho = exp(lp - old), u = min(rho A, clip(rho) A), kl = e^d - d - 1 with d = ref - lp, loss = scale sum (-u + beta kl)
//               w = scale (A rho [not clipped] - beta (1 - e^d))
//   preference  S = sum (or mean) of lp - ref over a sequence, z = beta (S_chosen - S_rejected),
//               loss = scale sum (-(1 - e) log sigmoid(z) - e log sigmoid(-z)), w = -+ beta dloss/dz
//   gradient    dx[c] = w (exp(x[c] - m) / s - [c == t]);  rows that are not scored: zeros, and nothing of them is read
//
// Bound by memory: a row is read, and its gradient written, once each at best.  Sums over a row are fp32 in
// short runs and fp64 over them; what follows from them is
// a handful of operations a row, done in fp64: d is a difference of two log-probabilities near each other, kl the third-order rest
// of an exponential, and the border of the clipping decides about a whole row.  Sums over rows are fp64, in a fixed order.  No atomics.
//
// Targets out of range: the row's loss and gradient are NaN and the error word says which.
// In the place of the reference's weighted cross-entropy (tilerl_kernels/reference.py:1511-1603) and its per-token weights
// (src/tilerl/train.py:805-864).
#include "common.cuh"

namespace {

constexpr int PL_SITE = 16;                          // of trl_set_error

// What a row's loss needs besides its logits.
struct PolicyRow {
  const float *adv, *old, *ref;                      // old, ref: a row each, or null
  int adv_rows;                                      // rows that share an advantage
  double lo, hi, kl, scale;                          // 1 - eps, 1 + eps_high
  float *lp, *ratio, *klv, *weight;                  // results, a row each
  unsigned char* clipped;
  double* loss;                                      // a row's, unscaled
};
struct Rows {
  const unsigned char* mask;                         // null: every row is scored
  const long long* target;
  long n, V;
};

// A row as vectors of 16 bytes with what is left at both ends (rows may start anywhere): `head` values, nv vectors, `tail` values.
template <typename T>
struct Span {
  static constexpr int E = 16 / sizeof(T);           // values a vector
  int head, tail;
  long nv;
  __device__ Span(const T* p, long V) {
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    head = (int)min((long)((E - off) % E), V);
    nv = (V - head) / E;
    tail = (int)(V - head - nv * E);
  }
  // the value at an end that thread k of a row's looks after, or -1
  __device__ long end_of(int k) const {
    if (k < head) return k;
    const int j = k - 16;
    return j >= 0 && j < tail ? head + nv * E + j : -1;
  }
};

__device__ __forceinline__ float pl_float(float x) { return x; }
__device__ __forceinline__ float pl_float(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T pl_round(float x);
template <>
__device__ __forceinline__ float pl_round<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 pl_round<bf16>(float x) { return __float2bfloat16(x); }
__device__ __forceinline__ void pl_unpack(uint4 v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void pl_unpack(uint4 v, float (&x)[8]) {
  const float2 a = bf162_bits_to_f2(v.x), b = bf162_bits_to_f2(v.y), c = bf162_bits_to_f2(v.z), d = bf162_bits_to_f2(v.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}
__device__ __forceinline__ uint4 pl_pack(const float (&x)[4]) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pl_pack(const float (&x)[8]) {
  return make_uint4(f2_to_bf162_bits(x[0], x[1]), f2_to_bf162_bits(x[2], x[3]), f2_to_bf162_bits(x[4], x[5]), f2_to_bf162_bits(x[6], x[7]));
}

// exp(x - m) where m may still be -inf: values of -inf count nothing, NaN stays.
__device__ __forceinline__ float pl_base(float m) { return m == -INFINITY ? 0.f : m; }

// log-probability of the target, in fp64; NaN for a target out of range.
__device__ __forceinline__ double pl_logprob(float xt, float m, double s) { return (double)xt - (double)m - log(s); }
template <typename T>
__device__ __forceinline__ float pl_target(const T* row, long long t, long V, long r) {
  if (t < 0 || t >= V) {
    trl_set_error(TRL_ERR_BOUNDS, PL_SITE, (int)t, (int)V);
    return NAN;
  }
  return pl_float(row[t]);
}

// A scored row's terms from its log-probability; the weight of its gradient comes back.
__device__ __forceinline__ float pl_policy(const PolicyRow& a, long r, double lp) {
  const double A = (double)a.adv[r / a.adv_rows];
  const double rho = a.old ? exp(lp - (double)a.old[r]) : 1.0;
  const bool clip = (rho > a.hi && A > 0.0) || (rho < a.lo && A < 0.0);
  // (an advantage of nothing has no part in the loss, whatever the ratio)
  double w = A == 0.0 ? 0.0 : clip ? 0.0 : A * rho, loss = A == 0.0 ? 0.0 : clip ? -A * (A > 0.0 ? a.hi : a.lo) : -A * rho, kl = 0.0;
  if (lp != lp) w = loss = lp;                       // (NaN stays where the advantage or the clipping would hide it)
  if (a.ref) {
    const double d = (double)a.ref[r] - lp, e = expm1(d);
    kl = e - d;
    if (a.kl != 0.0) w += a.kl * e, loss += a.kl * kl;
  }
  const float weight = (float)(w * a.scale);
  a.lp[r] = (float)lp, a.ratio[r] = (float)rho, a.klv[r] = (float)kl, a.weight[r] = weight, a.clipped[r] = clip, a.loss[r] = loss;
  return weight;
}
__device__ __forceinline__ void pl_policy_skip(const PolicyRow& a, long r) {
  a.lp[r] = a.ratio[r] = a.klv[r] = a.weight[r] = 0.f, a.clipped[r] = 0, a.loss[r] = 0.0;
}

// Sum over a block of W warps through `red` (W doubles), in a fixed order; the result in thread 0.
template <int W>
__device__ __forceinline__ double pl_block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < W; ++i) t += red[i];
  return t;
}

// ---- rows of any length, in two kernels -----------------------------------------------------------------------------------
// A block a row: (m, s) into ms, and its log-probability (POLICY: its terms).
template <typename T, bool POLICY>
__global__ void __launch_bounds__(512) pl_stats_kernel(const T* x, const Rows rows, float2* ms, double* lps, const PolicyRow a) {
  using S = Span<T>;
  __shared__ __align__(8) float red[32];
  const long r = blockIdx.x;
  if (rows.mask && !rows.mask[r]) {
    if (threadIdx.x == 0) {
      if (POLICY) pl_policy_skip(a, r);
      else lps[r] = 0.0;
    }
    return;
  }
  const T* row = x + (size_t)r * rows.V;
  const S sp(row, rows.V);
  const uint4* body = reinterpret_cast<const uint4*>(row + sp.head);
  float m = -INFINITY;
  double s = 0.0;                                    // (a thread adds up to V / 512 values: fp32 would lose 1e-6 of 250 000)
  const long e = sp.end_of(threadIdx.x);
  if (e >= 0) {
    m = pl_float(row[e]);
    s = expf(m - pl_base(m));
    if (m != m) m = -INFINITY;
  }
  constexpr int U = 16 / S::E;                        // vectors in flight: 16 values
  auto add = [&](const uint4 (&u)[U], int cnt) {
    float v[U][S::E], n = m, t = 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k >= cnt) break;
      pl_unpack(u[k], v[k]);
#pragma unroll
      for (int j = 0; j < S::E; ++j) n = fmaxf(n, v[k][j]);
    }
    if (n > m) s *= (double)expf(m - n), m = n;
    const float b = pl_base(m);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k >= cnt) break;
#pragma unroll
      for (int j = 0; j < S::E; j += 2) t += expf(v[k][j] - b) + expf(v[k][j + 1] - b);
    }
    s += (double)t;
  };
  long i = threadIdx.x;
  for (; i + (U - 1) * 512 < sp.nv; i += U * 512) {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k) u[k] = body[i + k * 512];
    add(u, U);
  }
  for (; i < sp.nv; i += 512) {
    uint4 u[U];
    u[0] = body[i];
    add(u, 1);
  }
  const float all = block_max(m, red);
  s = pl_block_sum<16>(s * (double)expf(m - all), reinterpret_cast<double*>(red));
  if (threadIdx.x == 0) {
    const double lp = pl_logprob(pl_target(row, rows.target[r], rows.V, r), all, s);
    ms[r] = make_float2(all, (float)s);
    if (POLICY) pl_policy(a, r, lp);
    else lps[r] = lp;
  }
}

// Gradients: a block a slice of a row.  weight of row r: weight[r / per].  The last rows first: they are what L2 still holds.
constexpr int PL_SLICE = 2048;                       // vectors a block
template <typename T>
__global__ void __launch_bounds__(256) pl_grad_kernel(const T* x, const Rows rows, const float2* ms, const float* weight, long per, T* grad, int slices) {
  using S = Span<T>;
  const long r = rows.n - 1 - blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  T* out = grad + (size_t)r * rows.V;
  const T* row = x + (size_t)r * rows.V;
  const S sp(row, rows.V);                           // (the gradient lies as the logits do)
  const bool scored = !rows.mask || rows.mask[r];
  const float w = scored ? weight[r / per] : 0.f;
  const float2 st = scored ? ms[r] : make_float2(0.f, 1.f);
  const float inv = 1.f / st.y;
  const long long t = scored ? rows.target[r] : -1;
  if (slice == 0) {
    const long e = sp.end_of(threadIdx.x);
    if (e >= 0) out[e] = pl_round<T>(scored ? (expf(pl_float(row[e]) - st.x) * inv - (e == t ? 1.f : 0.f)) * w : 0.f);
  }
  const uint4* body = reinterpret_cast<const uint4*>(row + sp.head);
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  const long end = min(sp.nv, (long)(slice + 1) * PL_SLICE);
#pragma unroll 4
  for (long i = (long)slice * PL_SLICE + threadIdx.x; i < end; i += 256) {
    float v[S::E] = {};
    if (scored) {
      pl_unpack(body[i], v);
#pragma unroll
      for (int j = 0; j < S::E; ++j) v[j] = expf(v[j] - st.x) * inv;
      const long long at = t - sp.head - i * S::E;
#pragma unroll
      for (int j = 0; j < S::E; ++j) v[j] = (v[j] - (at == j ? 1.f : 0.f)) * w;
    }
    dst[i] = pl_pack(v);
  }
}

// ---- sums over rows, and pairs of sequences ----------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pl_sum_kernel(const double* v, long n, double scale, float* out) {
  __shared__ double red[8];
  double s = 0.0;
#pragma unroll 4
  for (long i = threadIdx.x; i < n; i += 256) s += v[i];
  s = pl_block_sum<8>(s, red);
  if (threadIdx.x == 0) *out = (float)(s * scale);
}

// log(1 + e^y)
__device__ __forceinline__ double pl_softplus(double y) { return fmax(y, 0.0) + log1p(exp(-fabs(y))); }
// A block a pair: rows [2p T, 2p T + T) chosen, the T behind them rejected.  Results: sums of log-probabilities, margins, a pair's
// loss, and each sequence's weight for its rows' gradients.
__global__ void __launch_bounds__(256) pl_pairs_kernel(const double* lps, const float* ref, const unsigned char* mask, long T, double beta, double smooth,
                                                       int average, double scale, float* totals, float* margins, double* loss, float* weight) {
  __shared__ double red[8];
  const long p = blockIdx.x;
  double total[2], gap[2], div[2];
  for (int k = 0; k < 2; ++k) {
    const long at = (2 * p + k) * T;
    double a = 0.0, b = 0.0, c = 0.0;
    for (long i = threadIdx.x; i < T; i += 256)
      if (!mask || mask[at + i]) a += lps[at + i], b += lps[at + i] - (ref ? (double)ref[at + i] : 0.0), c += 1.0;
    total[k] = pl_block_sum<8>(a, red), gap[k] = pl_block_sum<8>(b, red), c = pl_block_sum<8>(c, red);
    div[k] = average ? fmax(c, 1.0) : 1.0;
  }
  if (threadIdx.x) return;
  const double z = beta * (gap[0] / div[0] - gap[1] / div[1]), e = smooth;
  const double dz = e / (1.0 + exp(-z)) - (1.0 - e) / (1.0 + exp(z));
  totals[2 * p] = (float)(total[0] / div[0]), totals[2 * p + 1] = (float)(total[1] / div[1]);
  margins[p] = (float)z;
  loss[p] = (1.0 - e) * pl_softplus(-z) + (e != 0.0 ? e * pl_softplus(z) : 0.0);
  // (the row's gradient is weight (p - onehot): minus that of its log-probability)
  weight[2 * p] = (float)(-dz * scale * beta / div[0]), weight[2 * p + 1] = (float)(dz * scale * beta / div[1]);
}

// x times *up; no pass over the values where that is 1.
template <typename T>
__global__ void __launch_bounds__(256) pl_scale_kernel(T* x, const float* up, long n) {
  const float u = *up;
  if (u == 1.f) return;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) x[i] = pl_round<T>(pl_float(x[i]) * u);
}

template <typename T>
int grad_launch(const void* x, const Rows& rows, const float2* ms, const float* weight, long per, void* grad, cudaStream_t st) {
  const long nv = rows.V / Span<T>::E, slices = nv < PL_SLICE ? 1 : (nv + PL_SLICE - 1) / PL_SLICE;
  if (rows.n * slices >= 1l << 31) return (int)cudaErrorInvalidValue;
  pl_grad_kernel<T><<<(unsigned)(rows.n * slices), 256, 0, st>>>((const T*)x, rows, ms, weight, per, (T*)grad, (int)slices);
  return (int)cudaGetLastError();
}

bool rows_ok(long n, long V) { return n >= 1 && n < 1l << 31 && V >= 1 && V < 1l << 31; }

}  // namespace

// n rows of V logits, contiguous (type 0: fp32, 1: bf16), anywhere; the gradient (null: not wanted) lies at the same offset from a 16-byte boundary.
// terms: [4, n] floats: log-probability, ratio, kl, weight; work: n doubles, then (n float2) what the kernels keep.
TRL_API int trl_policy_loss(const void* x, int type, long n, long V, const void* target, const void* mask, const void* adv, long adv_rows, const void* old,
                            const void* ref, double lo, double hi, double kl, double scale, void* terms, void* clipped, void* loss, void* grad, void* work,
                            void* stream) {
  if (!rows_ok(n, V) || adv_rows < 1 || adv_rows >= 1l << 31) return (int)cudaErrorInvalidValue;
  if (grad && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(grad)) & 15)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  float* f = (float*)terms;
  double* row_loss = (double*)work;
  float2* ms = (float2*)(row_loss + n);
  const Rows rows{(const unsigned char*)mask, (const long long*)target, n, V};
  const PolicyRow a{(const float*)adv, (const float*)old, (const float*)ref, (int)adv_rows, lo, hi, kl, scale, f, f + n, f + 2 * n, f + 3 * n,
                    (unsigned char*)clipped, row_loss};
  if (type) pl_stats_kernel<bf16, true><<<(int)n, 512, 0, st>>>((const bf16*)x, rows, ms, nullptr, a);
  else pl_stats_kernel<float, true><<<(int)n, 512, 0, st>>>((const float*)x, rows, ms, nullptr, a);
  if (grad) {
    const int rc = type ? grad_launch<bf16>(x, rows, ms, a.weight, 1, grad, st) : grad_launch<float>(x, rows, ms, a.weight, 1, grad, st);
    if (rc) return rc;
  }
  pl_sum_kernel<<<1, 256, 0, st>>>(row_loss, n, scale, (float*)loss);
  return (int)cudaGetLastError();
}

// 2 pairs sequences of T rows, chosen and rejected in turn.  totals [2 pairs], margins [pairs]; work: 2 pairs T doubles, as many
// float2, then pairs doubles and 2 pairs floats.
TRL_API int trl_preference_loss(const void* x, int type, long pairs, long T, long V, const void* target, const void* mask, const void* ref, double beta,
                                double smooth, int average, double scale, void* totals, void* margins, void* loss, void* grad, void* work, void* stream) {
  const long n = 2 * pairs * T;
  if (pairs < 1 || T < 1 || pairs >= 1l << 30 || T >= 1l << 31 || !rows_ok(n, V)) return (int)cudaErrorInvalidValue;
  if (grad && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(grad)) & 15)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  double* lps = (double*)work;
  float2* ms = (float2*)(lps + n);
  double* pair_loss = (double*)(ms + n);
  float* weight = (float*)(pair_loss + pairs);
  const Rows rows{(const unsigned char*)mask, (const long long*)target, n, V};
  if (type) pl_stats_kernel<bf16, false><<<(int)n, 512, 0, st>>>((const bf16*)x, rows, ms, lps, PolicyRow{});
  else pl_stats_kernel<float, false><<<(int)n, 512, 0, st>>>((const float*)x, rows, ms, lps, PolicyRow{});
  pl_pairs_kernel<<<(int)pairs, 256, 0, st>>>(lps, (const float*)ref, rows.mask, T, beta, smooth, average, scale, (float*)totals, (float*)margins, pair_loss,
                                              weight);
  if (grad) {
    const int rc = type ? grad_launch<bf16>(x, rows, ms, weight, T, grad, st) : grad_launch<float>(x, rows, ms, weight, T, grad, st);
    if (rc) return rc;
  }
  pl_sum_kernel<<<1, 256, 0, st>>>(pair_loss, pairs, scale, (float*)loss);
  return (int)cudaGetLastError();
}

TRL_API int trl_loss_scale(void* x, int type, const void* up, long n, void* stream) {
  if (n < 1) return (int)cudaErrorInvalidValue;
  const long blocks = (n + 1023) / 1024;
  const int grid = (int)(blocks < 148 * 16 ? blocks : 148 * 16);
  if (type) pl_scale_kernel<bf16><<<grid, 256, 0, (cudaStream_t)stream>>>((bf16*)x, (const float*)up, n);
  else pl_scale_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>((float*)x, (const float*)up, n);
  return (int)cudaGetLastError();
}
