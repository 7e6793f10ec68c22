// Log-probabilities of given tokens (and entropies) from hidden rows and the head, without the logits: x = h W^T stays in TMEM.
//
//   of a tile of 256 rows by 256 words, a row's (m, s[, u]) = (max x, sum e^(x - m)[, sum e^(x - m) (x - m)]), and x[t] where the target is
//   among them;  then over a row's tiles  M = max m, S = sum s e^(m - M), lp = x[t] - M - log S, entropy = log S - U / S
//
// A product of matrices with an epilogue that gives back 8 bytes (12 with entropies) for 128 logits: bound by the tensor cores from a
// few hundred rows on, by the reading of W below.  Pairs of SMs (`cta_group::2`) share a tile: 128 hidden rows each as the MMA's A, half of the
// 256 words each as its B, so that a k-block of 64 brings 32 KB to an SM for 512 clocks of MMAs (one SM alone: 48 KB, more than L2
// gives to all of them).  Two accumulators of 256 columns fill TMEM: a tile's epilogue runs beside the next one's products.  Rows are the
// TMEM lanes, so a thread has a row's values and no two threads meet.  The tensor cores cut off what they add up, so that 5120 terms in one accumulator
// lose 1e-6 of lp; an accumulator has at most 2048 of them, and the epilogue adds the accumulators in registers (1 to 3 % of the time; with 1024
// 3 to 5 %).  Where there is one, it goes through a row's values as they come from TMEM.  The tiles go round the pairs words by words over up to 2048
// rows at a time: pairs that run together read the same words, and W comes from memory once for 2048 rows.
//
// Exponentials are ex2.approx of (x - m) log2(e): its 2^-22 and the rounding of far arguments are averages over the words of a row, below
// fp32's rounding of lp.  (One fused x log2(e) - m log2(e) would carry the rounding of the second product into every word: 1e-6 of lp at
// logits of 30, infinity at 1e38.)  Sums of a row's tiles are fp32, their logarithm fp64.
//
// Only scored rows are worked on: their indices are gathered first, on the device.  Roles (10 warps): warp 0 = TMA producer, warp 1 = TMEM
// owner and MMA issuer (even SM), warps 2-9 = epilogue, two groups of four with 128 columns each.  Waits: see tcgen05_pair.cuh.
// In the place of the reference's log-probabilities over full logits (tilerl_kernels/reference.py:1511-1603).
#include "tcgen05_pair.cuh"

namespace {

constexpr int SC_ROWS = 128, SC_WORDS = 256, SC_KT = 64;       // rows an SM, words a tile, k a stage
constexpr int SC_THREADS = 320, SC_STAGES = 7, SC_STAGE = 2 * SC_ROWS * SC_KT * 2;
constexpr int SC_SMEM = SC_STAGES * SC_STAGE + 1024 + 256;
constexpr int SC_SEGMENT = 2048;                                // values of k whose products an accumulator adds up
constexpr int SC_GROUP = 8;                                     // tiles of 256 rows that go through the words together
static_assert(SC_SMEM >= 208 * 1024 && SC_SMEM <= 227 * 1024, "no other kernel with TMEM fits beside it on an SM");
constexpr int SC_SITE = 17;                                     // of trl_set_error

struct ScoreArgs {
  const int* count;            // scored rows, on the device (null: n of them)
  const int* index;            // of a scored row among all (null: itself)
  const long long* target;     // of all rows
  float2* part;                // [n, parts] (m, s)
  float* part_u;               // [n, parts], or null
  float* xt;                   // [n]
  int n, V, nk, v_tiles, parts, segments;
};

__device__ __forceinline__ void sc_mma(uint32_t d, uint32_t alo, uint32_t blo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 da, db;\n"
      "  mov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};\n"
      "  setp.ne.b32 p, %5, 0;\n"
      "  tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p; }\n"
      ::"r"(d), "r"(alo), "r"(blo), "r"(hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float sc_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The tile of unit u: words fastest over rows of a group.
__device__ __forceinline__ void sc_unit(int u, int r_tiles, int v_tiles, int& rt, int& vt) {
  const int whole = SC_GROUP * v_tiles, g = u / whole, left = u - g * whole, rows = min(SC_GROUP, r_tiles - g * SC_GROUP);
  vt = left / rows, rt = g * SC_GROUP + left - vt * rows;
}

// WHOLE: one accumulator a tile.
template <bool ENTROPY, bool WHOLE>
__global__ void __launch_bounds__(SC_THREADS, 1)
score_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, const ScoreArgs p) {
  constexpr int S = SC_STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * SC_STAGE);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t bar0 = smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };                              // the even SM's counts both SMs' copies
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * S + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * S + 2 + b); };           // of the even SM: both SMs' epilogue warps
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
    for (int b = 0; b < 2; ++b) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 16);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  gp_cluster_sync();                                // both CTAs run, before TMEM is asked for
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  gp_cluster_sync();                                // both halves are allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();                          // (the joining blocks, which wait for all of this)
  pdl_wait();                                       // (the rows and their number come from the kernels before)
  const int n = p.count ? min(*p.count, p.n) : p.n, r_tiles = (n + 2 * SC_ROWS - 1) / (2 * SC_ROWS), units = r_tiles * p.v_tiles;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      const uint32_t smem0 = smem_u32(smem);
      int st = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs) {
        int rt, vt;
        sc_unit(u, r_tiles, p.v_tiles, rt, vt);
        for (int kt = 0; kt < p.nk; ++kt, ++issued) {
          if (issued >= S && !(ok = mbar_wait(empty(st), ph ^ 1u, abort_flag))) break;
          const uint32_t dst = smem0 + (uint32_t)st * SC_STAGE, bar = gp_map(full(st), 0);
          if (rank == 0) mbar_expect_tx(full(st), 2u * SC_STAGE);
          gp_load_2d(dst, &map_h, kt * SC_KT, (rt * 2 + rank) * SC_ROWS, bar);
          gp_load_2d(dst + SC_STAGE / 2, &map_w, kt * SC_KT, vt * SC_WORDS + rank * (SC_WORDS / 2), bar);
          if (++st == S) st = 0, ph ^= 1u;
        }
      }
      // the last arrivals of the even SM's MMAs on this CTA's barriers, before its memory goes away
      const int pre = min(S, issued);
      for (int s = 0; ok && s < pre; ++s) {
        const int i = issued - pre + s;             // the last use of its stage
        ok = mbar_wait(empty(i % S), (uint32_t)(i / S) & 1u, abort_flag);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (for both SMs) ----------------
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(SC_WORDS >> 3) << 17) | ((uint32_t)((2 * SC_ROWS) >> 4) << 24);
      const uint64_t d0 = desc_sw128(smem_u32(smem));
      const uint32_t lo0 = (uint32_t)d0, hi = (uint32_t)(d0 >> 32);
      int st = 0, count = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = pair; ok && u < units; u += pairs) {
        for (int seg = 0; ok && seg < p.segments; ++seg, ++count) {
          const int buf = count & 1, k0 = seg * p.nk / p.segments, k1 = (seg + 1) * p.nk / p.segments;
          if (count >= 2) {
            if (!(ok = mbar_wait(acc_empty(buf), (uint32_t)((count >> 1) - 1) & 1u, abort_flag))) break;
            tc_fence_after();
          }
          const uint32_t acc = tmem_base + (uint32_t)buf * SC_WORDS;
          for (int kt = k0; kt < k1; ++kt) {
            if (!(ok = mbar_wait(full(st), ph, abort_flag))) break;
            tc_fence_after();
            const uint32_t a = lo0 + (uint32_t)st * (uint32_t)(SC_STAGE >> 4), b = a + (uint32_t)(SC_STAGE / 2 >> 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc_mma(acc, a + i * 2, b + i * 2, hi, idesc, kt > k0 || i ? 1u : 0u);
            gp_commit(empty(st), 3);
            if (++st == S) st = 0, ph ^= 1u;
          }
          if (ok) gp_commit(acc_full(buf), 3);
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..9): a thread a row, 128 words ----------------
    const int quad = warp & 3, half = (warp - 2) >> 2;
    constexpr float L2E = 1.4426950408889634f;
    const uint32_t even_empty = gp_map(acc_empty(0), 0);
    int count = 0;
    bool ok = true;
    for (int u = pair; ok && u < units; u += pairs) {
      int rt, vt;
      sc_unit(u, r_tiles, p.v_tiles, rt, vt);
      const int row = (rt * 2 + rank) * SC_ROWS + quad * 32 + lane, col0 = vt * SC_WORDS + half * (SC_WORDS / 2);
      const bool mine = row < n;
      const long long t = mine ? p.target[p.index ? p.index[row] : row] : -1;
      float m = -INFINITY, s = 0.f, w = 0.f;
      auto take = [&](float (&x)[32], int c) {      // 32 of the row's values, from word col0 + c on
        if (col0 + c + 32 > p.V) {                  // past the last word
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (col0 + c + i >= p.V) x[i] = -INFINITY;
        }
        const long long at = t - col0 - c;
        if (at >= 0 && at < 32 && t < p.V) {
          float xt = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (at == i) xt = x[i];
          p.xt[row] = xt;
        }
        float best = m;
#pragma unroll
        for (int i = 0; i < 32; ++i) best = fmaxf(best, x[i]);
        const float base = best == -INFINITY ? 0.f : best;
        if (best > m) {
          const float f = sc_exp2((m - base) * L2E);       // (0 for the first)
          if (ENTROPY) w = s > 0.f ? f * (w + s * (m - base)) : w;
          s *= f, m = best;
        }
        float a0 = 0.f, a1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float d = x[i] - base, g = x[i + 1] - base, e = sc_exp2(d * L2E), f = sc_exp2(g * L2E);
          a0 += e, a1 += f;
          if (ENTROPY) b0 += e > 0.f ? e * d : 0.f, b1 += f > 0.f ? f * g : 0.f;     // (no -inf times 0)
        }
        s += a0 + a1;
        if (ENTROPY) w += b0 + b1;
      };
      auto tmem = [&](int buf) { return tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * SC_WORDS + half * (SC_WORDS / 2)); };
      auto wait = [&](int buf) {
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full(buf), (uint32_t)(count >> 1) & 1u, abort_flag));
        tc_fence_after();
        return ok;
      };
      auto give_back = [&](int buf) {               // read out: the accumulator goes back
        tc_fence_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(even_empty + 8u * buf) : "memory");
      };
      if (WHOLE) {
        const int buf = count & 1;
        if (!wait(buf)) break;
#pragma unroll
        for (int c = 0; c < SC_WORDS / 2; c += 32) {
          uint32_t r[32];
          float x[32];
          __syncwarp();                             // (the branches in `take` part the lanes)
          tc_ld32(tmem(buf) + (uint32_t)c, r);
          tc_wait_ld();
          if (c + 32 == SC_WORDS / 2) give_back(buf);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
          take(x, c);
        }
        ++count;
      } else {
        float x[SC_WORDS / 64][32] = {};            // the thread's logits: the sums of the accumulators, as they come
        for (int seg = 0; seg < p.segments; ++seg, ++count) {
          const int buf = count & 1;
          if (!wait(buf)) break;
#pragma unroll
          for (int c = 0; c < SC_WORDS / 64; ++c) {
            uint32_t r[32];
            tc_ld32(tmem(buf) + (uint32_t)c * 32, r);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) x[c][i] += __uint_as_float(r[i]);
          }
          give_back(buf);
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < SC_WORDS / 64; ++c) take(x[c], c * 32);
      }
      if (mine) {
        const size_t o = (size_t)row * p.parts + vt * 2 + half;
        p.part[o] = make_float2(m, s);
        if (ENTROPY) p.part_u[o] = w;
      }
      __syncwarp();
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
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  gp_cluster_sync();                                // no CTA leaves while the other's half is being given back
}

// The log-probability and the entropy of a row whose words' (m, s, u) are joined.
__device__ __forceinline__ void score_write(const ScoreArgs& p, int to, float xt, float m, float s, float u, float* lp, float* entropy) {
  const long long t = p.target[to];
  const double log_s = log((double)s);
  if (t < 0 || t >= p.V) {
    trl_set_error(TRL_ERR_BOUNDS, SC_SITE, (int)t, p.V);
    lp[to] = NAN;
  } else {
    lp[to] = (float)((double)xt - (double)m - log_s);
  }
  if (entropy) entropy[to] = (float)(log_s - (double)u / (double)s);
}

// (s, u) of values whose largest is `from` as those of values whose largest is `to`, not below it
__device__ __forceinline__ void score_move(float& s, float& u, float from, float to) {
  const float f = from == -INFINITY ? 0.f : expf(from - to);
  u = f == 0.f ? 0.f : f * (u + s * (from - to)), s *= f;
}

// A block a scored row: its tiles together, read once, two a thread at a time (2048 rows of 256 tiles: eight at a time 2 us more).
__global__ void __launch_bounds__(128) score_join_kernel(const ScoreArgs p, float* lp, float* entropy) {
  constexpr int U = 2;
  __shared__ float red[32];
  pdl_wait();
  const int row = blockIdx.x, n = p.count ? *p.count : p.n;
  if (row >= n) return;
  const float2* part = p.part + (size_t)row * p.parts;
  const float* part_u = p.part_u + (size_t)row * p.parts;
  const int to = threadIdx.x || !p.index ? row : p.index[row];
  const float xt = threadIdx.x ? 0.f : p.xt[row];
  float m = -INFINITY, s = 0.f, u = 0.f;
  for (int i = threadIdx.x; i < p.parts; i += U * 128) {
    float2 v[U];
    float w[U], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const bool there = i + k * 128 < p.parts;
      v[k] = there ? part[i + k * 128] : make_float2(-INFINITY, 0.f);
      w[k] = there && entropy ? part_u[i + k * 128] : 0.f;
      top = fmaxf(top, v[k].x);
    }
    if (top > m) score_move(s, u, m, top), m = top;
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float f = expf(v[k].x - base);
      s += v[k].y * f;
      if (entropy && v[k].y != 0.f) u += f * (w[k] + v[k].y * (v[k].x - base));
    }
  }
  const float most = block_max(m, red);
  score_move(s, u, m, most);
  s = block_sum(s, red);
  if (entropy) u = block_sum(u, red);
  if (threadIdx.x == 0) score_write(p, to, xt, most, s, u, lp, entropy);
}

// Few rows, whose logits [n, ldo] are there: a cluster of blocks a row, each goes through its part of the words once and sends the first its (m, s, u).
constexpr int SC_SPREAD = 8;
__global__ void __cluster_dims__(SC_SPREAD, 1, 1) __launch_bounds__(256) score_few_kernel(const float* x, long ldo, const ScoreArgs p, float* lp, float* entropy) {
  __shared__ float red[32];
  __shared__ float parts[SC_SPREAD][3];
  pdl_wait();
  const int row = blockIdx.x / SC_SPREAD, rank = blockIdx.x % SC_SPREAD, n = p.count ? *p.count : p.n;
  if (row >= n) return;                              // (the whole cluster, before its first barrier)
  const float* at = x + (size_t)row * ldo;
  const int nv = (int)(ldo / 4), per = (nv + SC_SPREAD - 1) / SC_SPREAD, end = min(nv, (rank + 1) * per);
  float m = -INFINITY, s = 0.f, u = 0.f;
  for (int i = rank * per + threadIdx.x; i < end; i += 4 * 256) {
    float4 v[4];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = i + k * 256;
      v[k] = j < end ? reinterpret_cast<const float4*>(at)[j] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (j == nv - 1) {                             // (the last vector may reach past the words)
        if (4 * j + 1 >= p.V) v[k].y = -INFINITY;
        if (4 * j + 2 >= p.V) v[k].z = -INFINITY;
        if (4 * j + 3 >= p.V) v[k].w = -INFINITY;
      }
      top = fmaxf(top, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
    }
    if (top > m) {
      score_move(s, u, m, top);
      m = top;
    }
    const float base = m == -INFINITY ? 0.f : m;
    auto one = [&](float x) {
      const float d = x - base, e = expf(d);
      s += e;
      if (e > 0.f) u += e * d;
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) one(v[k].x), one(v[k].y), one(v[k].z), one(v[k].w);
  }
  const float most = block_max(m, red);
  score_move(s, u, m, most);
  s = block_sum(s, red);
  if (entropy) u = block_sum(u, red);
  gp_cluster_sync();                                 // all blocks run
  if (threadIdx.x == 0) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(parts[rank])));
    asm volatile("st.shared::cluster.f32 [%0], %1; st.shared::cluster.f32 [%0 + 4], %2; st.shared::cluster.f32 [%0 + 8], %3;" ::"r"(to), "f"(most), "f"(s), "f"(u) : "memory");
  }
  gp_cluster_sync();
  if (rank || threadIdx.x) return;
  m = -INFINITY, s = 0.f, u = 0.f;
  for (int k = 0; k < SC_SPREAD; ++k) m = fmaxf(m, parts[k][0]);
  for (int k = 0; k < SC_SPREAD; ++k) {
    float sk = parts[k][1], uk = parts[k][2];
    score_move(sk, uk, parts[k][0], m);
    s += sk, u += uk;
  }
  const int to = p.index ? p.index[row] : row;
  const long long t = p.target[to];
  score_write(p, to, t >= 0 && t < p.V ? at[t] : 0.f, m, s, u, lp, entropy);
}

// The scored rows in bf16, one behind the other in order, their indices, and their number; results of the others are 0.  A warp a row; a block counts
// the scored rows before its own for itself (some KB of mask bytes from L2; one block that counted for all took 8 us on its own, a block a row
// with the copy 9).
constexpr int SC_PACK = 8;                           // rows a block
template <typename T>
__global__ void __launch_bounds__(SC_PACK * 32) score_pack_kernel(const T* h, bf16* out, int n, int H, const unsigned char* mask, int* index, int* count, float* lp, float* entropy) {
  __shared__ int sums[SC_PACK];
  pdl_launch_dependents();
  const int first = blockIdx.x * SC_PACK, warp = threadIdx.x / 32, lane = threadIdx.x % 32, i = first + warp;
  int row = i;
  if (mask) {
    const unsigned on = __ballot_sync(0xffffffffu, lane < SC_PACK && first + lane < n && mask[first + lane]);
    int before = 0;
    if (on || first + SC_PACK >= n) {                // (the last block says how many there are)
      if (reinterpret_cast<uintptr_t>(mask) % 4 == 0) {
        const uint32_t* four = reinterpret_cast<const uint32_t*>(mask);
#pragma unroll 4
        for (int k = threadIdx.x; k < first / 4; k += SC_PACK * 32) before += __popc(__vsetne4(four[k], 0u));
      } else {
        for (int k = threadIdx.x; k < first; k += SC_PACK * 32) before += mask[k] != 0;
      }
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) sums[warp] = before;
      __syncthreads();
      before = 0;
#pragma unroll
      for (int w = 0; w < SC_PACK; ++w) before += sums[w];
    }
    if (first + SC_PACK >= n && threadIdx.x == 0) *count = before + __popc(on);
    if (i >= n) return;
    if (!(on >> warp & 1u)) {
      if (lane == 0) {
        lp[i] = 0.f;
        if (entropy) entropy[i] = 0.f;
      }
      return;
    }
    row = before + __popc(on & ((1u << warp) - 1u));
    if (lane == 0) index[row] = i;
  }
  if (i >= n) return;
  const T* src = h + (size_t)i * H;
  bf16* dst = out + (size_t)row * H;
#pragma unroll 4
  for (int c = lane * 8; c < H; c += 256) {
    uint4 v;
    if (sizeof(T) == 2) {
      v = *reinterpret_cast<const uint4*>(src + c);
    } else {
      const float4 a = reinterpret_cast<const float4*>(src + c)[0], b = reinterpret_cast<const float4*>(src + c)[1];
      v = make_uint4(f2_to_bf162_bits(a.x, a.y), f2_to_bf162_bits(a.z, a.w), f2_to_bf162_bits(b.x, b.y), f2_to_bf162_bits(b.z, b.w));
    }
    *reinterpret_cast<uint4*>(dst + c) = v;
  }
}

typedef CUresult (*EncodeTiledFnS)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [rows, K] bf16, boxes of 64 values x 128 rows; what lies past either end reads as zero
bool score_map(CUtensorMap* m, const void* base, long rows, long K) {
  static EncodeTiledFnS encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn) return false;
    encode = (EncodeTiledFnS)fn;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K * 2};
  const cuuint32_t b[2] = {SC_KT, SC_ROWS}, estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Pairs of SMs that run at a time.
template <bool ENTROPY, bool WHOLE>
int score_pairs() {
  static TrlPerDevice<int> counts;
  int& known = counts.here();
  if (known == 0) {
    auto kern = score_kernel<ENTROPY, WHOLE>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2), cfg.blockDim = dim3(SC_THREADS), cfg.dynamicSmemBytes = SC_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SC_SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    known = n > 0 ? n : -1;
  }
  return known;
}

template <bool ENTROPY, bool WHOLE>
int score_launch(const CUtensorMap& mh, const CUtensorMap& mw, const ScoreArgs& p, cudaStream_t st) {
  const int most = score_pairs<ENTROPY, WHOLE>();
  if (most < 1) return (int)cudaErrorInvalidConfiguration;
  const long units = (long)((p.n + 2 * SC_ROWS - 1) / (2 * SC_ROWS)) * p.v_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(units < most ? units : most)), cfg.blockDim = dim3(SC_THREADS), cfg.dynamicSmemBytes = SC_SMEM, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = g_trl_use_pdl ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, score_kernel<ENTROPY, WHOLE>, mh, mw, p);
}

// Up to so many rows the head's kernel for decode ticks streams the words (its MMA has them as rows, and as many columns as there are hidden rows), and
// their logits, 1 MB a row of 248 320, go through L2: an MMA of 256 rows here, most of them empty, takes longer than the words from memory.  Pairs and
// this, us, in turn: 248 320 x 5120 1 row 562, 379 (389 to read W at the measured copy rate), 33 rows 467 to 488, 445, 64 rows 543 to 591, 472; 128 000 x 4096
// 33 rows 190, 190, 64 rows 223 to 236, 203; 32 768 x 1024 1 row 40, 29, 33 rows 27, 29, 48 rows 24, 25, 64 rows 22, 26.  Above 32 rows, up to
// the 64 that the head's kernel takes, small heads are better off with pairs and large ones with this: a rule by rows alone ends where neither loses much.
constexpr int SC_FEW = 32;
int score_parts(int V) { return (V + SC_WORDS - 1) / SC_WORDS * 2; }

}  // namespace

TRL_API int trl_head_bf16_after(const void* x, const void* w, void* out, long ldo, int M, int N, int K, void* stream);

// Bytes of workspace for n rows (of which the scored ones are gathered, `packed`), a multiple of 256.
TRL_API long trl_score_workspace(int n, int H, int V, int packed, int entropy) {
  long b = 4l * n * 2 + 512;
  if (packed) b += 2l * n * H + 512;
  b += n <= SC_FEW ? 4l * n * ((V + 3) / 4 * 4) : (long)n * score_parts(V) * (entropy ? 12 : 8);
  return (b + 255) / 256 * 256;
}
// h [n, H] (type 0: fp32, 1: bf16), w [V, H] bf16, both contiguous and 16-byte aligned, H % 8 == 0; target int64 [n]; mask bytes [n] or null; lp and entropy
// (or null) fp32 [n]; n * parts of the words' tiles below 2^31.
TRL_API int trl_score(const void* h, int type, const void* w, const void* target, const void* mask, int n, int H, int V, void* lp, void* entropy, void* work,
                      void* stream) {
  if (n < 1 || V < 1 || H < 8 || H % 8 || ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(work)) & 15))
    return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  const bool packed = mask || type == 0;
  const int v_tiles = (V + SC_WORDS - 1) / SC_WORDS, parts = 2 * v_tiles;
  if ((long)n * parts >= 1l << 31) return (int)cudaErrorInvalidValue;
  unsigned char* at = (unsigned char*)work;
  auto take = [&](long bytes) {
    void* r = at;
    at += (bytes + 15) / 16 * 16;
    return r;
  };
  int* index = mask ? (int*)take(4l * n) : nullptr;
  int* count = mask ? (int*)take(4) : nullptr;
  bf16* rows = packed ? (bf16*)take(2l * n * H) : nullptr;
  if (packed) {
    if (type == 0) score_pack_kernel<float><<<(n + SC_PACK - 1) / SC_PACK, SC_PACK * 32, 0, st>>>((const float*)h, rows, n, H, (const unsigned char*)mask, index, count, (float*)lp, (float*)entropy);
    else score_pack_kernel<bf16><<<(n + SC_PACK - 1) / SC_PACK, SC_PACK * 32, 0, st>>>((const bf16*)h, rows, n, H, (const unsigned char*)mask, index, count, (float*)lp, (float*)entropy);
    const cudaError_t rc = cudaGetLastError();
    if (rc != cudaSuccess) return (int)rc;
  }
  if (n <= SC_FEW) {
    const long ldo = (V + 3) / 4 * 4;
    float* logits = (float*)take(4l * n * ldo);
    const ScoreArgs p{count, index, (const long long*)target, nullptr, nullptr, nullptr, n, V, 0, 0, 0, 0};
    const int rc = trl_head_bf16_after(packed ? rows : h, w, logits, ldo, n, V, H, stream);
    return rc ? rc : (int)trl_launch(score_few_kernel, dim3(SC_SPREAD * n), dim3(256), 0, st, (const float*)logits, ldo, p, (float*)lp, (float*)entropy);
  }
  float2* part = (float2*)take(8l * n * parts);
  float* part_u = entropy ? (float*)take(4l * n * parts) : nullptr;
  float* xt = (float*)take(4l * n);
  CUtensorMap mh, mw;
  if (!score_map(&mh, packed ? rows : h, n, H) || !score_map(&mw, w, V, H)) return (int)cudaErrorInvalidValue;
  const ScoreArgs p{count, index, (const long long*)target, part, part_u, xt, n, V, (H + SC_KT - 1) / SC_KT, v_tiles, parts, (H + SC_SEGMENT - 1) / SC_SEGMENT};
  const int rc = p.segments == 1 ? (entropy ? score_launch<true, true>(mh, mw, p, st) : score_launch<false, true>(mh, mw, p, st))
                                 : (entropy ? score_launch<true, false>(mh, mw, p, st) : score_launch<false, false>(mh, mw, p, st));
  if (rc) return rc;
  return (int)trl_launch(score_join_kernel, dim3(n), dim3(128), 0, st, p, (float*)lp, (float*)entropy);
}
