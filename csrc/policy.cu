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
// Bound by memory: a row is read, and its gradient written, once each at best.  Sums over a row are fp32, 16 values and more at a time in a
// tree; what follows from them is a handful of operations a row, done in fp64: d is a difference of two log-probabilities near each other, kl the third-order rest
// of an exponential, and the border of the clipping decides about a whole row.  Sums over rows are fp64, in a fixed order.  No atomics.
//
// Targets out of range: the row's loss and gradient are NaN and the error word says which.
// In the place of the reference's weighted cross-entropy (tilerl_kernels/reference.py:1511-1603) and its per-token weights
// (src/tilerl/train.py:805-864).
#include <cuda.h>

#include <type_traits>

#include "tcgen05.cuh"

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

// ---- exponentials ------------------------------------------------------------------------------------------------------------
// Sums are of 2^(x log2 e - B) with a whole number B, the row's largest x log2 e rounded up: one fused multiply-add, rounded once, and
// ex2.approx, where expf(x - m) has ten instructions; instructions were these kernels' time.  A whole B makes it no matter which B: the rounding
// of a product m log2 e would go into every value of the row.  ex2.approx is off by 2^-22, and the multiply-add's rounding moves a value at a distance
// of d by d 2^-24 of itself, both at random over a row.  fp32's log2 e is off by PL_OFF of itself, as if all of x were: lp by PL_OFF times the distance
// of x[t] from the row's mean, 1e-7 of the same sign in every row, which a sequence's sum or a divergence shows.  So the mean, u / s with
// u = sum 2^y y, comes out of the pass over the row too (one multiply-add more), and lp without that.  ex2.approx is low by some 4e-8 in the mean
// (measured against 64 bits: 2 to 5e-8, by the spread of the logits), which lp is given back.
constexpr float PL_L2E = 1.4426950408889634f;
constexpr double PL_LN2 = 0.693147180559945309417, PL_OFF = (double)PL_L2E * PL_LN2 - 1.0, PL_LESS = 3.5e-8;
__device__ __forceinline__ float pl_exp2(float y) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return e;
}
__device__ __forceinline__ float pl_exp(float x, float base) { return pl_exp2(fmaf(x, PL_L2E, -base)); }
// into s and u  (0 times -inf is not meant; 2^-256 is 0)
__device__ __forceinline__ void pl_add(float x, float base, float& s, float& u) {
  const float y = fmaf(x, PL_L2E, -base), e = pl_exp2(y);
  s += e, u = fmaf(e, fmaxf(y, -256.f), u);
}
// B for a largest value.  From below it is bounded: threads that see nothing but masked words (-inf, -1e30) have sums of 0 there.  A row whose B is
// that bound, or so large that whole numbers near it have gaps, is far: gone through once more, slowly, with x - m.
constexpr float PL_FAR = 2097152.f;
__device__ __forceinline__ float pl_base(float most) { return fmaxf(ceilf(most * PL_L2E), -PL_FAR); }
__device__ __forceinline__ bool pl_far(float base) { return !(fabsf(base) < PL_FAR); }
// (B, s, u) of some of a row's values.
struct Part {
  float base, s, u;
  // at a base that is not below its own
  __device__ __forceinline__ void move(float to) {
    const float d = base - to, f = pl_exp2(d);
    u = fmaf(d, s, u) * f, s *= f, base = to;
  }
  __device__ __forceinline__ void join_warp() {
    move(warp_max(base));
    s = warp_sum(s), u = warp_sum(u);
  }
};
// The log-probability of a value x but for the logarithm of the sum, in fp64.  (x itself goes in as it is: a target at the type's lowest value has
// an old log-probability as low, and 1e-16 of 1e38 between them would be a ratio of infinity.)
__device__ __forceinline__ double pl_low(float x, float base, float mean) {
  return (double)x + (PL_OFF * (double)mean - (double)base) * (1.0 / (double)PL_L2E) - PL_LESS;
}
// N parts, in order: the sum and, through it, a value's pl_low.  base: at first one that the result's is not to be below.
template <int N>
__device__ __forceinline__ double pl_join(const Part* parts, float& base, float& mean) {
#pragma unroll
  for (int k = 0; k < N; ++k) base = fmaxf(base, parts[k].base);
  double sum = 0.0;
  float u = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    Part q = parts[k];
    q.move(base);
    sum += (double)q.s, u += q.u;
  }
  mean = u / (float)sum;
  return sum;
}

template <typename T>
__device__ __forceinline__ float pl_target(const T* row, long long t, long V) {
  if (t < 0 || t >= V) {
    trl_set_error(TRL_ERR_BOUNDS, PL_SITE, (int)t, (int)V);
    return NAN;
  }
  return pl_float(row[t]);
}

// What a scored row's terms need, and they from its target's logit, less what the sum's exponentials have less, and the sum.  Two warps share the
// chain: the three exponentials go side by side over a warp's lanes and give the weight, which every thread waits for; the logarithm, which only the written
// terms need, is another warp's.  8192 x 4000 83 us, 2048 x 32 768 103 (one thread for
// all of it 95, 108; all of it in fp32 81, 101).
struct PolicyIn {
  float adv, old, ref;
  __device__ PolicyIn() : adv(0.f), old(0.f), ref(0.f) {}
  __device__ PolicyIn(const PolicyRow& a, long r) : adv(a.adv[a.adv_rows == 1 ? (unsigned)r : (unsigned)r / (unsigned)a.adv_rows]), old(a.old ? a.old[r] : 0.f), ref(a.ref ? a.ref[r] : 0.f) {}
};
struct PolicyMid {                                   // of a row, in shared memory
  double low, log_sum, rho, kle;                     // kle: e^d
  float adv, ref;
};
__device__ __forceinline__ bool pl_clips(const PolicyRow& a, double A, double rho) { return (rho > a.hi && A > 0.0) || (rho < a.lo && A < 0.0); }
// By a whole warp, four lanes a row, all of which have its values: (weight over the sum, the target's gradient weight (p - 1)).
// (Inlined: a function of its own would read the kernel's arguments through memory: 2048 x 32 768 120 us.)
__device__ __forceinline__ float2 pl_weigh(const PolicyRow& a, const PolicyIn in, double low, double sum, PolicyMid* mid, float* weight_of) {
  const int lane = threadIdx.x & 31, j = lane & 3, lead = lane & ~3;
  const double A = (double)in.adv, part = 1.0 / sum, e = exp(j == 1 ? low - (double)in.old : j == 2 ? (double)in.ref - low : low);
  const double p = __shfl_sync(0xffffffffu, e, lead) * part, by_old = __shfl_sync(0xffffffffu, e, lead + 1), by_ref = __shfl_sync(0xffffffffu, e, lead + 2);
  const double rho = a.old ? by_old * part : 1.0, kle = by_ref * sum;      // (1e-16 of cancellation in kl: d^2 / 2 from |d| of 1e-5 on)
  // (an advantage of nothing has no part in the loss, whatever the ratio; NaN stays where the advantage or the clipping would hide it)
  double w = A == 0.0 || pl_clips(a, A, rho) ? 0.0 : A * rho;
  if (low != low || sum != sum) w = low + sum;
  if (a.ref && a.kl != 0.0) w += a.kl * (kle - 1.0);
  const float weight = (float)(w * a.scale);
  if (j == 0 && mid) mid->low = low, mid->rho = rho, mid->kle = kle, mid->adv = in.adv, mid->ref = in.ref, *weight_of = weight;
  return make_float2((float)((double)weight * part), (float)((p - 1.0) * (double)weight));
}
// The rest of a row's terms, written.
__device__ __forceinline__ void pl_write(const PolicyRow& a, long r, const PolicyMid& mid) {
  const double A = (double)mid.adv, lp = mid.low - mid.log_sum, rho = mid.rho;
  const bool clip = pl_clips(a, A, rho);
  double loss = A == 0.0 ? 0.0 : clip ? -A * (A > 0.0 ? a.hi : a.lo) : -A * rho, kl = 0.0;
  if (lp != lp) loss = lp;
  if (a.ref) {
    kl = mid.kle - ((double)mid.ref - lp) - 1.0;
    if (a.kl != 0.0) loss += a.kl * kl;
  }
  a.lp[r] = (float)lp, a.ratio[r] = (float)rho, a.klv[r] = (float)kl, a.clipped[r] = clip, a.loss[r] = loss;
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

// ---- the two passes over a row --------------------------------------------------------------------------------------------------
// G vectors a thread at a time, NT threads apart: f(vectors, first one's place, whether all are there).  Those past the end are -inf.
// HINT: L2 is told whether it should keep them (the second pass reads them again: 1.5 % less time at 1024 x 248 320) or they are not needed
// any more.
__device__ __forceinline__ uint64_t pl_policy_of(bool keep) {
  uint64_t last, first;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(last));
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
  return keep ? last : first;
}
template <bool HINT>
__device__ __forceinline__ uint4 pl_load(const uint4* p, uint64_t policy) {
  if (!HINT) return *p;
  uint4 v;
  asm volatile("ld.global.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
  return v;
}
template <typename T, int NT, int G, bool HINT = false, typename F>
__device__ __forceinline__ void pl_each(const uint4* body, int cnt, F f, bool keep = false) {
  const uint64_t policy = HINT ? pl_policy_of(keep) : 0;
  int i = threadIdx.x;
  const uint4* p = body + i;
  uint4 z[G];
#pragma unroll 1
  for (; i + (G - 1) * NT < cnt; i += G * NT, p += G * NT) {
#pragma unroll
    for (int k = 0; k < G; ++k) z[k] = pl_load<HINT>(p + k * NT, policy);
    f(z, i, true);
  }
  if (i < cnt) {
    constexpr uint32_t low = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int k = 0; k < G; ++k) z[k] = i + k * NT < cnt ? pl_load<HINT>(p + k * NT, policy) : make_uint4(low, low, low, low);
    f(z, i, false);
  }
}
// x = -inf if a == b  (written so that arrays of x stay in registers)
__device__ __forceinline__ void pl_lower(float& x, int a, int b) {
  asm("{ .reg .pred p; setp.eq.s32 p, %1, %2; @p mov.b32 %0, 0fFF800000; }" : "+f"(x) : "r"(a), "r"(b));
}
// A thread's part of a row: of its vectors and the value xe at one of its ends (-inf: none).  SKIP: without value `skip % E` of vector
// `skip / E` of the row.
template <typename T, int NT, int G, bool HINT = false, bool SKIP = false>
__device__ __forceinline__ Part pl_sums(const uint4* body, int cnt, float xe, bool keep = false, int skip = -1) {
  constexpr int E = Span<T>::E, C = E == 4 ? G : G / 2 < 1 ? 1 : G / 2;        // vectors that are unpacked at a time
  Part p = {pl_base(xe == xe ? xe : -INFINITY), 0.f, 0.f};
  pl_add(xe, p.base, p.s, p.u);
  const int place = SKIP && skip >= 0 && skip / E % NT == threadIdx.x ? skip / E : -1;
  pl_each<T, NT, G, HINT>(body, cnt, [&](const uint4 (&z)[G], int i, bool) {
#pragma unroll
    for (int k0 = 0; k0 < G; k0 += C) {
      float v[C][E], top = -INFINITY, q[4] = {}, w[2] = {};
#pragma unroll
      for (int k = 0; k < C; ++k) pl_unpack(z[k0 + k], v[k]);
      if (SKIP && place >= i + k0 * NT && place < i + (k0 + C) * NT) {
        const int which = (place - (i + k0 * NT)) / NT * E + skip % E;
#pragma unroll
        for (int k = 0; k < C * E; ++k) pl_lower(v[k / E][k % E], which, k);
      }
#pragma unroll
      for (int k = 0; k < C; ++k) {
#pragma unroll
        for (int e = 0; e < E; e += 2) top = fmaxf(top, fmaxf(v[k][e], v[k][e + 1]));
      }
      const float b = pl_base(top);
      if (b > p.base) p.move(b);
#pragma unroll
      for (int k = 0; k < C; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) pl_add(v[k][e], p.base, q[e & 3], w[e & 1]);
      p.s += (q[0] + q[1]) + (q[2] + q[3]), p.u += w[0] + w[1];
    }
  }, keep);
  return p;
}
// The gradients of a thread's vectors, c 2^(x log2 e - B).
template <typename T, int NT, int G, bool HINT = false>
__device__ __forceinline__ void pl_grads(const uint4* body, uint4* dst, int cnt, float base, float c) {
  constexpr int E = Span<T>::E;
  pl_each<T, NT, G, HINT>(body, cnt, [&](const uint4 (&z)[G], int i, bool whole) {
    uint4* o = dst + i;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      float v[E];
      pl_unpack(z[k], v);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = pl_exp(v[e], base) * c;
      if (whole || i + k * NT < cnt) __stcs(o + k * NT, pl_pack(v));
    }
  });
}
// Of far rows: a thread's largest value, its sum of e^(x - m), its gradients c e^(x - m).
template <typename T, int NT>
__device__ float pl_far_most(const uint4* body, int cnt, float xe) {
  float m = xe;
  pl_each<T, NT, 1>(body, cnt, [&](const uint4 (&z)[1], int, bool) {
    float v[Span<T>::E];
    pl_unpack(z[0], v);
    for (int e = 0; e < Span<T>::E; ++e) m = fmaxf(m, v[e]);
  });
  return m;
}
template <typename T, int NT>
__device__ float pl_far_sum(const uint4* body, int cnt, float xe, bool end, float m) {
  float s = end ? expf(xe - m) : 0.f;
  pl_each<T, NT, 1>(body, cnt, [&](const uint4 (&z)[1], int i, bool) {
    float v[Span<T>::E];
    pl_unpack(z[0], v);
    for (int e = 0; e < Span<T>::E; ++e) s += expf(v[e] - m);
  });
  return s;
}
template <typename T, int NT>
__device__ void pl_far_grads(const uint4* body, uint4* dst, int cnt, float m, float c) {
  pl_each<T, NT, 1>(body, cnt, [&](const uint4 (&z)[1], int i, bool) {
    float v[Span<T>::E];
    pl_unpack(z[0], v);
    for (int e = 0; e < Span<T>::E; ++e) v[e] = expf(v[e] - m) * c;
    dst[i] = pl_pack(v);
  });
}
__device__ __forceinline__ void pl_store_zero(uint4* p) { __stcs(p, make_uint4(0u, 0u, 0u, 0u)); }
// Whether this thread wrote the target's gradient: it is at one of its ends, or among its vectors lo + k, lo + k + NT, ...
__device__ __forceinline__ bool pl_wrote(long long t, long end, int head, int E, long lo, int cnt, int k, int NT) {
  const long tv = (long)(t - head) / E - lo;
  return t >= 0 && (t == end || (t >= head && tv >= 0 && tv < cnt && tv % NT == k));
}

__device__ __forceinline__ uint32_t pl_map(uint32_t addr, int cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ void pl_cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void pl_cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  __syncwarp();
}

// The values of thread k of a short row's NT: N of its vectors; -inf where there are none.
constexpr int PL_SHORT = 16;
template <typename T, int NT>
__device__ __forceinline__ void pl_short_load(const uint4* body, int nv, int k, float (&v)[PL_SHORT]) {
  constexpr int E = Span<T>::E;
#pragma unroll
  for (int i = 0; i < PL_SHORT / E; ++i) {
    constexpr uint32_t low = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;       // -inf
    float u[E];
    pl_unpack(k + i * NT < nv ? body[k + i * NT] : make_uint4(low, low, low, low), u);
#pragma unroll
    for (int j = 0; j < E; ++j) v[i * E + j] = u[j];
  }
}
// v as 2^((v - less) log2 e), and with the value at an end their sums over the warp.  (The largest value is known before the first exponential here, and the two
// more instructions of (x - m) log2 e are not what counts.)
__device__ __forceinline__ Part pl_short_sums(float (&v)[PL_SHORT], float& end, float most, float less) {
  float s[4] = {}, u[2] = {};
#pragma unroll
  for (int i = 0; i < PL_SHORT; ++i) {
    const float y = (v[i] - less) * PL_L2E;
    v[i] = pl_exp2(y), s[i & 3] += v[i], u[i & 1] = fmaf(v[i], fmaxf(y, -256.f), u[i & 1]);
  }
  const float y = (end - less) * PL_L2E;
  end = pl_exp2(y);
  return {most, warp_sum(((s[0] + s[1]) + (s[2] + s[3])) + end), warp_sum(u[0] + u[1] + end * fmaxf(y, -256.f))};
}
__device__ __forceinline__ float pl_short_most(const float (&v)[PL_SHORT], float end) {
#pragma unroll
  for (int i = 0; i < PL_SHORT; i += 2) end = fmaxf(end, fmaxf(v[i], v[i + 1]));
  return warp_max(end);
}
// W parts at the base of their largest values to one at `top` (not below them).  Without a finite value nothing is a number here.
template <int W>
__device__ __forceinline__ double pl_short_join(const Part* q, float top, float& u) {
  double s = 0.0;
  u = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float d = fmaxf((q[i].base - top) * PL_L2E, -256.f), f = pl_exp2(d);
    s += (double)(q[i].s * f), u += fmaf(d, q[i].s, q[i].u) * f;
  }
  return s;
}
template <int W>
__device__ __forceinline__ float pl_short_top(const Part* q) {
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) top = fmaxf(top, q[i].base);
  return top;
}

// ---- policy loss -----------------------------------------------------------------------------------------------------------------
// Up to 4096 values: NT threads a row, which waits in registers, 16 values a thread, as exponentials until its sum and weight are known; the rows of a
// block have theirs formed side by side, four lanes of a warp and a lane of another a row.  A row's chain (target, its logit, exponentials in fp64) is some 5 us, so what
// counts is how many are on their way: 40 warps an SM.  (A warp a row, 32 values a lane, each its own weight: 16 384 x 1000 69 us, this 50.)
template <typename T, int NT>
__global__ void __launch_bounds__(256, 5) pl_policy_short_kernel(const T* x, const Rows rows, T* grad, const __grid_constant__ PolicyRow a, float* whole) {
  using S = Span<T>;
  constexpr int E = S::E, VPT = PL_SHORT / E, W = NT / 32, R = 256 / NT;
  __shared__ Part sums[8];                           // (at the base of the largest value itself)
  __shared__ float3 found[R];                        // the largest value, weight over the sum, the target's gradient
  __shared__ PolicyMid mid[R];
  pdl_launch_dependents();                           // (only the sum, which waits for all of this)
  const int k = threadIdx.x % NT, mine = threadIdx.x / NT, warp = threadIdx.x >> 5;
  const long r0 = (long)blockIdx.x * R, r = r0 + mine;
  const bool there = r < rows.n, scored = there && (!rows.mask || rows.mask[r]);
  // lanes 4 i .. of the first warp, and lane i of the second, look after row r0 + i
  const int q = warp == 0 ? threadIdx.x / 4 : threadIdx.x % 32;
  const long rw = r0 + q;
  const bool forms = warp < 2 && q < R && rw < rows.n, weighs = forms && (!rows.mask || rows.mask[rw]);
  PolicyIn in;
  float xt = 0.f;
  if (weighs) {
    if (warp == 0) in = PolicyIn(a, rw);
    const long long t = rows.target[rw];
    if (warp == 1) pl_target(x + (size_t)rw * rows.V, t, rows.V);
    xt = t >= 0 && t < rows.V ? pl_float(x[(size_t)rw * rows.V + t]) : NAN;
  }
  const T* row = x + (size_t)r * rows.V;
  T* out = grad + (size_t)r * rows.V;
  const S sp(row, rows.V);
  const int nv = there ? (int)sp.nv : 0;
  const uint4* body = reinterpret_cast<const uint4*>(row + sp.head);
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  const long ie = there ? sp.end_of(k) : -1;
  float v[PL_SHORT], end = scored && ie >= 0 ? pl_float(row[ie]) : -INFINITY;
  pl_short_load<T, NT>(body, scored ? nv : 0, k, v);
  const float most = pl_short_most(v, end), less = most == -INFINITY ? 0.f : most;
  const Part part = pl_short_sums(v, end, most, less);
  if (threadIdx.x % 32 == 0) sums[warp] = part;
  __syncthreads();
  if (warp < 2) {
    double low = 0.0, all = 1.0;
    float top = 0.f;
    if (weighs) {
      const Part* of = sums + q * W;
      float all_u;
      top = pl_short_top<W>(of), all = pl_short_join<W>(of, top, all_u);
      const float mean = all_u / (float)all, others = 1.f - 1.f / (float)all;      // (the largest value's is 1 exactly)
      low = (double)xt - (double)top + PL_OFF * PL_LN2 * (double)mean - PL_LESS * (double)others;
    }
    if (warp == 0) {
      const float2 f = pl_weigh(a, in, low, all, weighs ? mid + q : nullptr, a.weight + rw);
      if (weighs && threadIdx.x % 4 == 0) found[q] = make_float3(top, f.x, f.y);
    } else if (weighs) {
      mid[q].log_sum = log(all);
    }
  }
  __syncthreads();
  if (weighs && warp == 1) pl_write(a, rw, mid[q]);
  else if (forms && warp == 1) pl_policy_skip(a, rw);
  if (whole) pl_cluster_arrive();
  if (grad && there) {
    const float3 f = scored ? found[mine] : make_float3(0.f, 0.f, 0.f);
    // (a warp that saw no word that can be has exponentials of 0 at a base of 0, which may lie above f.x by more than a float holds)
    const float c = scored ? pl_exp2((most - f.x) * PL_L2E) * f.y : 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float u[E];
#pragma unroll
      for (int j = 0; j < E; ++j) u[j] = scored ? v[i * E + j] * c : 0.f;
      if (k + i * NT < nv) __stcs(dst + k + i * NT, pl_pack(u));
    }
    if (ie >= 0) out[ie] = pl_round<T>(scored ? end * c : 0.f);
    if (scored) {
      const long long t = rows.target[r];
      if (t < rows.V && pl_wrote(t, ie, sp.head, E, 0, nv, k, NT)) out[t] = pl_round<T>(f.z);
    }
  }
  if (!whole) return;
  pl_cluster_wait();                                 // (every row's loss is written)
  if (blockIdx.x || warp) return;
  double sum = 0.0;
  for (long i = threadIdx.x; i < rows.n; i += 32) sum += a.loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x == 0) *whole = (float)(sum * a.scale);
}

// Longer rows: a cluster of CL blocks goes through a row twice, for its sum and for its gradient; the second time the row is still in L2, as long as
// those in work fit there.  Between the passes the blocks send each other their (B, s, u); each adds them up in a fixed order and forms the row's weight for
// itself.  The cluster's first barrier is passed before another block's shared memory is touched, no block's is after the second.  Both end:
// every thread of a scored row's cluster comes to them, and nothing before them waits.
// What a block works on: its vectors of a row, and its threads' values at the row's ends.
template <typename T, int CL>
struct PolicyPart {
  const T* row;
  T* out;
  Span<T> sp;
  long lo, ie;
  int rank, cnt;
  const uint4* body;
  uint4* dst;
  __device__ PolicyPart(const T* x, T* grad, long r, long V)
      : row(x + (size_t)r * V), out(grad + (size_t)r * V), sp(row, V), rank(CL > 1 ? blockIdx.x % CL : 0) {
    const long per = (sp.nv + CL - 1) / CL;
    lo = min(sp.nv, rank * per), cnt = (int)(min(sp.nv, lo + per) - lo);
    body = reinterpret_cast<const uint4*>(row + sp.head) + lo, dst = reinterpret_cast<uint4*>(out + sp.head) + lo;
    ie = rank == 0 ? sp.end_of(threadIdx.x) : -1;
  }
};

// A far row.  All blocks of its cluster come here, behind the same barriers.
template <typename T, int CL, int NT>
__device__ __noinline__ void pl_policy_far(const T* x, const Rows& rows, T* grad, const PolicyRow& a, long r, Part* sums, Part* peers, float4* found, PolicyMid* mid) {
  const PolicyPart<T, CL> p(x, grad, r, rows.V);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto meet = [&] {
    if (CL > 1) pl_cluster_arrive(), pl_cluster_wait();
    else __syncthreads();
  };
  auto join = [&](float v, auto warps, auto op, float none) {       // of all threads of the cluster
    v = warps(v);
    meet();                                          // (what was there before has been read)
    if (lane == 0) sums[warp].s = v;
    __syncthreads();
    if (warp == 0) {
      v = warps(lane < NT / 32 ? sums[lane].s : none);
      if (CL > 1) {
        if (lane < CL) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(pl_map(smem_u32(&peers[p.rank].s), lane)), "f"(v) : "memory");
      } else if (lane == 0) {
        peers[0].s = v;
      }
    }
    meet();
    v = peers[0].s;
    for (int k = 1; k < CL; ++k) v = op(v, peers[k].s);
    return v;
  };
  const float xe = p.ie >= 0 ? pl_float(p.row[p.ie]) : -INFINITY;
  const float m = join(pl_far_most<T, NT>(p.body, p.cnt, xe), [](float v) { return warp_max(v); }, [](float v, float w) { return fmaxf(v, w); }, -INFINITY);
  const float sum = join(pl_far_sum<T, NT>(p.body, p.cnt, xe, p.ie >= 0, m), [](float v) { return warp_sum(v); }, [](float v, float w) { return v + w; }, 0.f);
  const long long t = rows.target[r];
  if (warp == 0) {
    const float xt = t >= 0 && t < rows.V ? pl_float(p.row[t]) : NAN;
    const float2 f = pl_weigh(a, PolicyIn(a, r), (double)xt - (double)m, (double)sum, mid, a.weight + r);
    if (tid == 0) *found = make_float4(0.f, f.x, f.y, 0.f), mid->log_sum = log((double)sum);
  }
  __syncthreads();
  if (tid == 0 && p.rank == 0) pl_write(a, r, *mid);
  if (grad) {
    pl_far_grads<T, NT>(p.body, p.dst, p.cnt, m, found->y);
    if (p.ie >= 0) p.out[p.ie] = pl_round<T>(expf(xe - m) * found->y);
    if (t < rows.V && pl_wrote(t, p.ie, p.sp.head, Span<T>::E, p.lo, p.cnt, tid, NT)) p.out[t] = pl_round<T>(found->z);
  }
  meet();                                            // (no block leaves while another reads what it sent)
}

template <typename T, int CL, int NT, int G, int BLOCKS>
__global__ void __launch_bounds__(NT, BLOCKS) pl_policy_kernel(const T* x, const __grid_constant__ Rows rows, T* grad, const __grid_constant__ PolicyRow a) {
  constexpr int W = NT / 32;
  __shared__ Part sums[W], peers[CL];
  __shared__ float4 found;                           // base, weight over the sum, the target's gradient, whether the row is far
  __shared__ PolicyMid mid;
  pdl_launch_dependents();                           // (only the sum, which waits for all of this)
  const long r = blockIdx.x / CL;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PolicyPart<T, CL> p(x, grad, r, rows.V);
  if (rows.mask && !rows.mask[r]) {
    if (tid == 0 && p.rank == 0) pl_policy_skip(a, r);
    if (grad) {
      for (int i = tid; i < p.cnt; i += NT) pl_store_zero(p.dst + i);
      if (p.ie >= 0) p.out[p.ie] = pl_round<T>(0.f);
    }
    return;
  }
  if (CL > 1) pl_cluster_arrive();
  const long long t = rows.target[r];
  PolicyIn in;
  float xt = 0.f;
  if (warp == 0) in = PolicyIn(a, r), xt = t >= 0 && t < rows.V ? pl_float(p.row[t]) : NAN;
  if (tid == 0 && p.rank == 0) pl_target(p.row, t, rows.V);
  const float xe = p.ie >= 0 ? pl_float(p.row[p.ie]) : -INFINITY;
  Part part = pl_sums<T, NT, G, true>(p.body, p.cnt, xe, grad != nullptr);
  part.join_warp();
  if (lane == 0) sums[warp] = part;
  __syncthreads();
  if (CL > 1) pl_cluster_wait();
  if (warp == 0) {
    part = lane < W ? sums[lane] : Part{-PL_FAR, 0.f, 0.f};
    part.join_warp();
    if (CL > 1) {
      if (lane < CL) {
        const uint32_t to = pl_map(smem_u32(&peers[p.rank]), lane);
        asm volatile("st.shared::cluster.f32 [%0], %1; st.shared::cluster.f32 [%0 + 4], %2; st.shared::cluster.f32 [%0 + 8], %3;" ::"r"(to), "f"(part.base), "f"(part.s), "f"(part.u) : "memory");
      }
    } else if (lane == 0) {
      peers[0] = part;
    }
  }
  if (CL > 1) pl_cluster_arrive(), pl_cluster_wait();
  else __syncthreads();
  if (warp < 2) {
    float all = -PL_FAR, mean;
    const double sum = pl_join<CL>(peers, all, mean);
    if (pl_far(all)) {
      if (tid == 0) found.w = 1.f;
    } else if (warp == 0) {
      const float2 f = pl_weigh(a, in, pl_low(xt, all, mean), sum, &mid, a.weight + r);
      if (lane == 0) found = make_float4(all, f.x, f.y, 0.f);
    } else if (lane == 0 && p.rank == 0) {
      mid.log_sum = log(sum);
    }
  }
  __syncthreads();
  if (found.w != 0.f) {
    pl_policy_far<T, CL, NT>(x, rows, grad, a, r, sums, peers, &found, &mid);
    return;
  }
  if (tid == 32 && p.rank == 0) pl_write(a, r, mid);
  if (!grad) return;
  pl_grads<T, NT, G, true>(p.body, p.dst, p.cnt, found.x, found.y);
  if (p.ie >= 0) p.out[p.ie] = pl_round<T>(pl_exp(xe, found.x) * found.y);
  if (t < rows.V && pl_wrote(t, p.ie, p.sp.head, Span<T>::E, p.lo, p.cnt, tid, NT)) p.out[t] = pl_round<T>(found.z);
}

// ---- preference loss: a row's weight needs its whole sequence -------------------------------------------------------------------
// A block a row: what its gradient needs into `rest`, and its log-probability.  `rest`: base, p - 1 of the target, sum, 0; of far rows p - 1, the largest
// value, sum, 1.  p - 1 is the others' share, formed as that: a quotient less 1 would have fp32's rounding of 1, 6 % of a share of 1e-6.
template <typename T>
__global__ void __launch_bounds__(256, 4) pl_stats_kernel(const T* x, const Rows rows, float4* rest, double* lps) {
  using S = Span<T>;
  constexpr int NT = 256, G = sizeof(T) == 4 ? 8 : 4;
  __shared__ Part sums[NT / 32];
  __shared__ float red[32];
  __shared__ int far;
  pdl_launch_dependents();
  const long r = blockIdx.x;
  if (rows.mask && !rows.mask[r]) {
    if (threadIdx.x == 0) lps[r] = 0.0;
    return;
  }
  const T* row = x + (size_t)r * rows.V;
  const S sp(row, rows.V);
  const uint4* body = reinterpret_cast<const uint4*>(row + sp.head);
  float xt = 0.f;
  const long long t = rows.target[r];
  if (threadIdx.x == 0) xt = pl_target(row, t, rows.V);
  const long ie = sp.end_of(threadIdx.x);
  const float xe = ie >= 0 ? pl_float(row[ie]) : -INFINITY;
  // A sequence's sum takes in every row's error.  Where the target is likely, that is its exponential's and what additions to it lose: 6e-8 a row (a
  // plain softmax in fp32: 9e-8), without it 8e-9.  So the target stays out of the sums and comes in in fp64.
  Part part = pl_sums<T, NT, G, false, true>(body, (int)sp.nv, ie == t ? -INFINITY : xe, false,
                                             t >= sp.head && t < sp.head + sp.nv * S::E ? (int)(t - sp.head) : -1);
  part.join_warp();
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = pl_base(xt == xt ? xt : -INFINITY), mean;
    const double rest_of = pl_join<NT / 32>(sums, all, mean);
    const double y = (double)xt * (double)PL_L2E - (double)all, e = exp(y * PL_LN2), sum = rest_of + e;
    const float most = (float)e / (float)sum;
    // (the mean of the others, and the target's share)
    const float of_all = rest_of > 0.0 ? mean + most * (fmaxf((float)y, -256.f) - mean) : (float)y;
    rest[r] = make_float4(all, (float)(-rest_of / sum), (float)sum, 0.f), lps[r] = pl_low(xt, all, of_all) + PL_LESS * (double)most - log(sum);
    far = pl_far(all);
  }
  __syncthreads();
  if (!far) return;
  const float m = block_max(pl_far_most<T, NT>(body, (int)sp.nv, xe), red);
  const float s = block_sum(pl_far_sum<T, NT>(body, (int)sp.nv, xe, ie >= 0, m), red);
  if (threadIdx.x == 0) {
    const double low = (double)xt - (double)m;
    rest[r] = make_float4((float)(exp(low) / (double)s - 1.0), m, s, 1.f), lps[r] = low - log((double)s);
  }
}

// Up to 4096 values, as the policy loss has them: NT threads a row.  `rest` as of far rows.
template <typename T, int NT>
__global__ void __launch_bounds__(256, 5) pl_stats_short_kernel(const T* x, const Rows rows, float4* rest, double* lps) {
  constexpr int E = Span<T>::E, W = NT / 32, R = 256 / NT;
  __shared__ Part sums[8];
  pdl_launch_dependents();
  const int k = threadIdx.x % NT;
  const long r0 = (long)blockIdx.x * R, r = r0 + threadIdx.x / NT, rw = r0 + threadIdx.x;
  const bool scored = r < rows.n && (!rows.mask || rows.mask[r]);
  const bool forms = threadIdx.x < R && rw < rows.n, weighs = forms && (!rows.mask || rows.mask[rw]);
  float xt = 0.f;
  if (weighs) xt = pl_target(x + (size_t)rw * rows.V, rows.target[rw], rows.V);
  else if (forms) lps[rw] = 0.0;
  const T* row = x + (size_t)r * rows.V;
  const Span<T> sp(row, rows.V);
  const long ie = scored ? sp.end_of(k) : -1;
  const long long t = scored ? rows.target[r] : -1;
  float v[PL_SHORT], end = ie >= 0 && ie != t ? pl_float(row[ie]) : -INFINITY;
  pl_short_load<T, NT>(reinterpret_cast<const uint4*>(row + sp.head), scored ? (int)sp.nv : 0, k, v);
  if (t >= sp.head && t < sp.head + sp.nv * E && (int)(t - sp.head) / E % NT == k) {       // (the target comes in below)
    const int which = (int)(t - sp.head) / E / NT * E + (int)(t - sp.head) % E;
#pragma unroll
    for (int i = 0; i < PL_SHORT; ++i) pl_lower(v[i], which, i);
  }
  const float most = pl_short_most(v, end), less = most == -INFINITY ? 0.f : most;
  const Part part = pl_short_sums(v, end, most, less);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = part;
  __syncthreads();
  if (!weighs) return;
  const Part* q = sums + threadIdx.x * W;
  const float others = pl_short_top<W>(q), top = fmaxf(others, xt);
  float u;
  const double rest_of = pl_short_join<W>(q, top, u), low = (double)xt - (double)top, e = exp(low), sum = rest_of + e;
  const float mean = (u + (float)e * fmaxf((float)low * PL_L2E, -256.f)) / (float)sum;
  const float rough = (float)(rest_of - (others == top ? 1.0 : 0.0)) / (float)sum;       // (what exponentials that are not exact have of the sum)
  rest[rw] = make_float4((float)(-rest_of / sum), top, (float)sum, 1.f);
  lps[rw] = low + PL_OFF * PL_LN2 * (double)mean - PL_LESS * (double)rough - log(sum);
}
template <typename T, int NT>
__global__ void __launch_bounds__(256, 5) pl_grad_short_kernel(const T* x, const Rows rows, const float4* rest, const float* weight, long per, T* grad) {
  constexpr int E = Span<T>::E, R = 256 / NT;
  pdl_launch_dependents();
  pdl_wait();
  const long r = rows.n - 1 - ((long)blockIdx.x * R + threadIdx.x / NT);
  const int k = threadIdx.x % NT;
  if (r < 0) return;
  const bool scored = !rows.mask || rows.mask[r];
  const T* row = x + (size_t)r * rows.V;
  T* out = grad + (size_t)r * rows.V;
  const Span<T> sp(row, rows.V);
  const int nv = (int)sp.nv;
  const long ie = sp.end_of(k);
  float v[PL_SHORT];
  pl_short_load<T, NT>(reinterpret_cast<const uint4*>(row + sp.head), scored ? nv : 0, k, v);
  const float w = scored ? weight[(unsigned)r / (unsigned)per] : 0.f;
  const float4 st = scored ? rest[r] : make_float4(0.f, 0.f, 1.f, 0.f);
  const float c = w / st.z;
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  auto one = [&](float x) { return pl_exp2((x - st.y) * PL_L2E); };
#pragma unroll
  for (int i = 0; i < PL_SHORT / E; ++i) {
    float u[E];
#pragma unroll
    for (int j = 0; j < E; ++j) u[j] = scored ? one(v[i * E + j]) * c : 0.f;
    if (k + i * NT < nv) __stcs(dst + k + i * NT, pl_pack(u));
  }
  if (ie >= 0) out[ie] = pl_round<T>(scored ? one(pl_float(row[ie])) * c : 0.f);
  if (!scored) return;
  const long long t = rows.target[r];
  if (t < rows.V && pl_wrote(t, ie, sp.head, E, 0, nv, k, NT)) out[t] = pl_round<T>(st.x * w);
}

// Gradients: a block a slice of a row.  weight of row r: weight[r / per].  The last rows first: they are what L2 still holds.
constexpr int PL_SLICE = 4096;                       // vectors a block
template <typename T>
__global__ void __launch_bounds__(256, 4) pl_grad_kernel(const T* x, const Rows rows, const float4* rest, const float* weight, long per, T* grad, int slices) {
  using S = Span<T>;
  constexpr int NT = 256, G = sizeof(T) == 4 ? 8 : 4;
  pdl_launch_dependents();
  pdl_wait();
  const long r = rows.n - 1 - blockIdx.x / slices, lo = (long)(blockIdx.x % slices) * PL_SLICE;
  T* out = grad + (size_t)r * rows.V;
  const T* row = x + (size_t)r * rows.V;
  const S sp(row, rows.V);                           // (the gradient lies as the logits do)
  const int cnt = (int)max(0l, min(sp.nv - lo, (long)PL_SLICE)), k = threadIdx.x;
  const long ie = lo == 0 ? sp.end_of(k) : -1;
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head) + lo;
  if (rows.mask && !rows.mask[r]) {
    for (int i = k; i < cnt; i += NT) pl_store_zero(dst + i);
    if (ie >= 0) out[ie] = pl_round<T>(0.f);
    return;
  }
  const float w = weight[(unsigned)r / (unsigned)per];
  const float4 st = rest[r];
  const long long t = rows.target[r];
  const uint4* body = reinterpret_cast<const uint4*>(row + sp.head) + lo;
  const float c = w / st.z;
  auto one = [&](float x) { return st.w != 0.f ? expf(x - st.y) : pl_exp(x, st.x); };
  if (st.w != 0.f) pl_far_grads<T, NT>(body, dst, cnt, st.y, c);
  else pl_grads<T, NT, G>(body, dst, cnt, st.x, c);
  if (ie >= 0) out[ie] = pl_round<T>(one(pl_float(row[ie])) * c);
  if (t < rows.V && pl_wrote(t, ie, sp.head, S::E, lo, cnt, k, NT)) out[t] = pl_round<T>((st.w != 0.f ? st.x : st.y) * w);
}

// ---- sums over rows, and pairs of sequences ----------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) pl_sum_kernel(const double* v, long n, double scale, float* out) {
  __shared__ double red[32];
  double s = 0.0;
  pdl_wait();                                        // (launched while the rows' kernel runs)
#pragma unroll 8
  for (long i = threadIdx.x; i < n; i += 1024) s += v[i];
  s = pl_block_sum<32>(s, red);
  if (threadIdx.x == 0) *out = (float)(s * scale);
}

// A block a pair: rows [2p T, 2p T + T) chosen, the T behind them rejected.  Results: sums of log-probabilities, margins, a pair's
// loss, and each sequence's weight for its rows' gradients.  `whole` (few pairs: the blocks are one cluster): the sum of the losses too, in place of a launch more.
constexpr int PL_PAIRS = 8;
__global__ void __launch_bounds__(1024) pl_pairs_kernel(const double* lps, const float* ref, const unsigned char* mask, long T, double beta, double smooth,
                                                       int average, double scale, float* totals, float* margins, double* loss, float* weight, float* whole) {
  __shared__ double red[32][6], losses[PL_PAIRS];
  pdl_launch_dependents();
  if (whole) pl_cluster_arrive();
  pdl_wait();
  const long p = blockIdx.x;
  double v[6] = {};                                  // log-probabilities, their differences to the reference's, scored tokens; chosen, rejected
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long at = (2 * p + k) * T;
#pragma unroll 4
    for (long i = threadIdx.x; i < T; i += blockDim.x)
      if (!mask || mask[at + i]) v[3 * k] += lps[at + i], v[3 * k + 1] += lps[at + i] - (ref ? (double)ref[at + i] : 0.0), v[3 * k + 2] += 1.0;
  }
#pragma unroll
  for (int q = 0; q < 6; ++q) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32][q] = v[q];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int q = 0; q < 6; ++q) {
      v[q] = 0.0;
      for (int w = 0; w < (int)blockDim.x / 32; ++w) v[q] += red[w][q];
    }
    const double by0 = average ? 1.0 / fmax(v[2], 1.0) : 1.0, by1 = average ? 1.0 / fmax(v[5], 1.0) : 1.0;
    const double z = beta * (v[1] * by0 - v[4] * by1), e = smooth;
    // with u = e^-|z|: sigmoid(|z|) = 1 / (1 + u), -log of it log(1 + u), and |z| more the other way round
    const double u = exp(-fabs(z)), l = log1p(u), near = 1.0 / (1.0 + u), up = z >= 0.0 ? near : u * near, down = z >= 0.0 ? u * near : near;
    const double dz = z == z ? e * up - (1.0 - e) * down : z;
    totals[2 * p] = (float)(v[0] * by0), totals[2 * p + 1] = (float)(v[3] * by1);
    margins[p] = (float)z;
    const double of = z != z ? z : (e != 1.0 ? (1.0 - e) * (l + fmax(-z, 0.0)) : 0.0) + (e != 0.0 ? e * (l + fmax(z, 0.0)) : 0.0);
    loss[p] = losses[0] = of;
    // (the row's gradient is weight (p - onehot): minus that of its log-probability)
    weight[2 * p] = (float)(-dz * scale * beta * by0), weight[2 * p + 1] = (float)(dz * scale * beta * by1);
  }
  if (!whole) return;
  pl_cluster_wait();                                 // every block runs
  if (threadIdx.x == 0 && p) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(pl_map(smem_u32(&losses[p]), 0)), "d"(losses[0]) : "memory");
  pl_cluster_arrive(), pl_cluster_wait();
  if (p || threadIdx.x) return;
  double sum = 0.0;
  for (long k = 0; k < gridDim.x; ++k) sum += losses[k];
  *whole = (float)(sum * scale);
}

// x times *up; no pass over the values where that is 1.
template <typename T>
__global__ void __launch_bounds__(256) pl_scale_kernel(T* x, const float* up, long n) {
  const float u = *up;
  if (u == 1.f) return;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) x[i] = pl_round<T>(pl_float(x[i]) * u);
}

// f(NT as a type) for rows of up to 4096 values, 16 a thread.
template <typename F>
int short_form(long V, F f) {
  if (V <= 512) return f(std::integral_constant<int, 32>());
  if (V <= 1024) return f(std::integral_constant<int, 64>());
  if (V <= 2048) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 256>());
}
constexpr long PL_SHORT_ROW = 4096;
unsigned short_blocks(long n, int threads) { return (unsigned)((n + 256 / threads - 1) / (256 / threads)); }

template <typename T>
int stats_launch(const T* x, const Rows& rows, float4* rest, double* lps, cudaStream_t st) {
  if (rows.V > PL_SHORT_ROW) {
    pl_stats_kernel<T><<<(unsigned)rows.n, 256, 0, st>>>(x, rows, rest, lps);
    return (int)cudaGetLastError();
  }
  return short_form(rows.V, [&](auto nt) {
    pl_stats_short_kernel<T, nt.value><<<short_blocks(rows.n, nt.value), 256, 0, st>>>(x, rows, rest, lps);
    return (int)cudaGetLastError();
  });
}
template <typename T>
int grad_launch(const void* x, const Rows& rows, const float4* rest, const float* weight, long per, void* grad, cudaStream_t st) {
  if (rows.V <= PL_SHORT_ROW)
    return short_form(rows.V, [&](auto nt) {
      return (int)trl_launch(pl_grad_short_kernel<T, nt.value>, dim3(short_blocks(rows.n, nt.value)), dim3(256), 0, st, (const T*)x, rows, rest, weight, per, (T*)grad);
    });
  const long nv = rows.V / Span<T>::E, slices = nv < PL_SLICE ? 1 : (nv + PL_SLICE - 1) / PL_SLICE;
  if (rows.n * slices >= 1l << 31) return (int)cudaErrorInvalidValue;
  return (int)trl_launch(pl_grad_kernel<T>, dim3((unsigned)(rows.n * slices)), dim3(256), 0, st, (const T*)x, rows, rest, weight, per, (T*)grad, (int)slices);
}

template <typename T, int CL, int NT, int G, int BLOCKS>
int policy_launch(const T* x, const Rows& rows, T* grad, const PolicyRow& a, cudaStream_t st) {
  if (rows.n * CL >= 1l << 31) return (int)cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows.n * CL)), cfg.blockDim = dim3(NT), cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, pl_policy_kernel<T, CL, NT, G, BLOCKS>, x, rows, grad, a);
}
// The form by a row's length.
template <typename T>
int policy_rows(const T* x, const Rows& rows, T* grad, const PolicyRow& a, float* loss, bool& summed, cudaStream_t st) {
  constexpr int E = Span<T>::E;
  const long V = rows.V;
  if (V <= PL_SHORT_ROW)
    return short_form(V, [&](auto nt) {
      // (few blocks are a cluster, which adds the rows' losses up as well: a launch less)
      const unsigned blocks = short_blocks(rows.n, nt.value);
      summed = blocks <= 8;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(blocks), cfg.blockDim = dim3(256), cfg.stream = st;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = blocks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr, cfg.numAttrs = summed ? 1 : 0;
      return (int)cudaLaunchKernelEx(&cfg, pl_policy_short_kernel<T, nt.value>, x, rows, grad, a, summed ? loss : nullptr);
    });
  // By a row's bytes, since those in work have to stay in L2 (some 50 MB) and blocks to be many: the longer a row, the more blocks share it.  Measured best,
  // us, before the pass summed the mean too, which takes 2 % (and the next): 4096 x 8192 57 (two blocks a row 68), 2048 x 32 768 107 (one block of 384 threads 110, two of 192 108), 1024 x 65 536 110 (two of 256 113),
  // 1024 x 248 320 382 (four of 256 415, four blocks an SM in place of three 437); bf16 2048 x 49 999 99 (one of 128 107), 1024 x 131 072 116 (four of 128
  // 118), 1024 x 248 320 213 (eight of 256 222).
  const long bytes = V * (long)sizeof(T);
  if (bytes <= 64 << 10) return policy_launch<T, 1, 128, 8, 8>(x, rows, grad, a, st);
  if (bytes <= 192 << 10) return policy_launch<T, E == 4 ? 4 : 2, 128, 8, 8>(x, rows, grad, a, st);
  if (bytes <= 384 << 10) return policy_launch<T, 4, 256, 4, 5>(x, rows, grad, a, st);
  return policy_launch<T, E == 4 ? 8 : 4, 256, 8, 3>(x, rows, grad, a, st);
}

bool rows_ok(long n, long V) { return n >= 1 && n < 1l << 31 && V >= 1 && V < 1l << 31; }

}  // namespace

// n rows of V logits, contiguous (type 0: fp32, 1: bf16), anywhere; the gradient (null: not wanted) lies at the same offset from a 16-byte boundary.
// terms: [4, n] floats: log-probability, ratio, kl, weight; work: n doubles.
TRL_API int trl_policy_loss(const void* x, int type, long n, long V, const void* target, const void* mask, const void* adv, long adv_rows, const void* old,
                            const void* ref, double lo, double hi, double kl, double scale, void* terms, void* clipped, void* loss, void* grad, void* work,
                            void* stream) {
  if (!rows_ok(n, V) || adv_rows < 1 || adv_rows >= 1l << 31) return (int)cudaErrorInvalidValue;
  if (grad && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(grad)) & 15)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  float* f = (float*)terms;
  double* row_loss = (double*)work;
  const Rows rows{(const unsigned char*)mask, (const long long*)target, n, V};
  const PolicyRow a{(const float*)adv, (const float*)old, (const float*)ref, (int)adv_rows, lo, hi, kl, scale, f, f + n, f + 2 * n, f + 3 * n,
                    (unsigned char*)clipped, row_loss};
  bool summed = false;
  const int rc = type ? policy_rows((const bf16*)x, rows, (bf16*)grad, a, (float*)loss, summed, st) : policy_rows((const float*)x, rows, (float*)grad, a, (float*)loss, summed, st);
  if (rc || summed) return rc;
  return (int)trl_launch(pl_sum_kernel, dim3(1), dim3(1024), 0, st, row_loss, n, scale, (float*)loss);
}

// 2 pairs sequences of T rows, chosen and rejected in turn.  totals [2 pairs], margins [pairs]; work: 2 pairs T float4, as many
// doubles, then pairs doubles and 2 pairs floats.
TRL_API int trl_preference_loss(const void* x, int type, long pairs, long T, long V, const void* target, const void* mask, const void* ref, double beta,
                                double smooth, int average, double scale, void* totals, void* margins, void* loss, void* grad, void* work, void* stream) {
  const long n = 2 * pairs * T;
  if (pairs < 1 || T < 1 || pairs >= 1l << 30 || T >= 1l << 31 || !rows_ok(n, V)) return (int)cudaErrorInvalidValue;
  if (grad && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(grad)) & 15)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  float4* rest = (float4*)work;
  double* lps = (double*)(rest + n);
  double* pair_loss = lps + n;
  float* weight = (float*)(pair_loss + pairs);
  const Rows rows{(const unsigned char*)mask, (const long long*)target, n, V};
  const int stated = type ? stats_launch((const bf16*)x, rows, rest, lps, st) : stats_launch((const float*)x, rows, rest, lps, st);
  if (stated) return stated;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)pairs), cfg.blockDim = dim3(T > 4096 ? 1024 : 256), cfg.stream = st;       // (a pair of 2 x 32 768 rows of 500: 103 us, with 256 threads 128; of 2 x 2048 rows of 2000 34, 30)
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_trl_use_pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)pairs, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = pairs <= PL_PAIRS ? 2 : 1;
  const cudaError_t paired = cudaLaunchKernelEx(&cfg, pl_pairs_kernel, (const double*)lps, (const float*)ref, rows.mask, T, beta, smooth, average, scale,
                                                (float*)totals, (float*)margins, pair_loss, weight, pairs <= PL_PAIRS ? (float*)loss : nullptr);
  if (paired != cudaSuccess) return (int)paired;
  if (grad) {
    const int rc = type ? grad_launch<bf16>(x, rows, rest, weight, T, grad, st) : grad_launch<float>(x, rows, rest, weight, T, grad, st);
    if (rc) return rc;
  }
  if (pairs <= PL_PAIRS) return 0;
  return (int)trl_launch(pl_sum_kernel, dim3(1), dim3(1024), 0, st, pair_loss, pairs, scale, (float*)loss);
}

TRL_API int trl_loss_scale(void* x, int type, const void* up, long n, void* stream) {
  if (n < 1) return (int)cudaErrorInvalidValue;
  const long blocks = (n + 1023) / 1024;
  const int grid = (int)(blocks < 148 * 16 ? blocks : 148 * 16);
  if (type) pl_scale_kernel<bf16><<<grid, 256, 0, (cudaStream_t)stream>>>((bf16*)x, (const float*)up, n);
  else pl_scale_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>((float*)x, (const float*)up, n);
  return (int)cudaGetLastError();
}
