// Log-probability of given tokens, entropy of their distribution and its n likeliest alternatives, from logits, and the
// gradient of all three.
//
// With M = max z, x_j = (z_j - M) log2(e) / temperature, S = sum 2^x, X = sum 2^x x, everything in one pass:
//   logprob = (z_tok - M) / temperature - ln S,   entropy = (log2 S - X / S) ln 2
// (all relative to the maximum: no difference of two large numbers, and no overflow of logits at the type's lowest value).
//
// Alternatives without a second pass over the row: a warp notes the maximum of each stretch of the row that it reads (512
// or 1024 logits; where the block reads little, each thread that of its own logits).  The n-th largest of the warps' few
// largest maxima is reached by n logits, so it bounds the n-th largest logit from below; the stretches whose maximum
// reaches it, hardly more than n, are looked at again, and what reaches it there is ranked.  Where those are too many (rows
// of equal or rising logits): at most n stretches hold the n largest logits, those with the n largest maxima, and of equal
// logits no more than n have to be looked at.  Order: larger logit first, then lower index.
//
// A row is read by a cluster of 1 to 8 blocks, which write their sums and lists into the first block's shared memory.
//
// 128 rows of 152 k fp32 logits with 8 alternatives: 20.3 us, 3.8 TB/s; of bf16 logits 20.0 us, half the bytes.  What
// bounds it there is not the bytes alone: instructions are issued in 48 % of the cycles for either type, waits are for the
// loads (fp32), at the barriers of the selection (3 us that nothing hides) and for busy pipes (bf16; exponentials one a
// logit, conversions, packed fp32 sums).  1,024 rows of bf16 with 16, and the gradient: 200 us, 623 MB without the second
// read of the logits, 4.7 TB/s with it.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>

#include <type_traits>

#include "q8.cuh"

using namespace cl;
namespace cg = cooperative_groups;

namespace {

constexpr int kSmThreads = 1024;                  // threads that an SM holds of it: 2 blocks of 512, or 4 of 256
constexpr int kMaxTop = 64;
constexpr int kUnroll = 4;                        // vectors of 16 bytes a lane loads at once
constexpr int kCand = 4096;                       // n (n + 1) / 2 candidates when all logits are equal, and room; a power of two
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1000.f;                   // 2^kFar is 0: -inf logits stay out of 0 * inf

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// unique key: larger logit first, then lower index; NaN counts as -inf, -0 as 0
__device__ __forceinline__ uint64_t key_of(float v, int idx) {
  v = v == v ? v + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(v);
  return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)(~idx);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

template <typename T> struct Wide { static constexpr int N = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void load16(const T* p, float* f) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < Wide<T>::N; ++i) f[i] = q8::to_float(t[i]);
}

// maximum over the warp, NaN left out
__device__ __forceinline__ float warp_max_f32(float v) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}
// two fp32 in one register pair
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes of logits
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
template <typename T>
__device__ __forceinline__ uint4 raw_lowest() {  // -inf everywhere
  const uint32_t x = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(x, x, x, x);
}
template <typename T>
__device__ __forceinline__ void expand(const uint4& u, float* f) {
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < Wide<T>::N; ++i) f[i] = q8::to_float(t[i]);
}
// largest of a vector, NaN left out
template <typename T>
__device__ __forceinline__ float raw_max(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(&u);
    return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
}

struct Sums { float m, s, x; };                   // M, S, X
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -INFINITY) { r.s = a.s + b.s; r.x = a.x + b.x; return r; }   // 0, or NaN
  const float da = fmaxf((a.m - r.m) * c, kFar), db = fmaxf((b.m - r.m) * c, kFar);
  const float ea = exp2_approx(da), eb = exp2_approx(db);
  r.s = a.s * ea + b.s * eb;
  r.x = ea * (a.x + a.s * da) + eb * (b.x + b.s * db);
  return r;
}

constexpr int kSmall = 96;                        // candidates that are ranked by counting; more are sorted

// The block sorts `count` keys, largest first (bitonic; zeros fill up to a power of two).
template <int kThreads>
__device__ __forceinline__ void sort_keys(uint64_t* keys, int count) {
  int size = 64;
  while (size < count) size *= 2;
  for (int i = count + threadIdx.x; i < size; i += kThreads) keys[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const uint64_t x = keys[lo], y = keys[hi];
        if ((x < y) == ((lo & k) == 0)) { keys[lo] = y; keys[hi] = x; }
      }
      __syncthreads();
    }
}

template <int kThreads>
struct __align__(16) Shared {
  static constexpr int kWarps = kThreads / 32, kMaxStretch = kThreads;
  float stretch[kMaxStretch];
  uint64_t cand[kCand];
  uint64_t best[8 * kMaxTop];                     // the cluster's lists, in the first block
  int chosen[kMaxTop];
  float firsts[2 * kMaxTop + kWarps];
  Sums warp_sums[kWarps], part_sums[8];
  Sums sums;
  uint64_t round;
  float bound;
  int count;
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads)
token_logprob_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ tokens, int V, int n, float c,
                     float inv_temp, float* __restrict__ lp, float* __restrict__ ent, float* __restrict__ stats, float* __restrict__ top_lp,
                     int64_t* __restrict__ top_id) {
  __shared__ Shared<kThreads> sh;
  constexpr int kWarps = kThreads / 32;
  constexpr int kMaxStretch = kThreads;            // stretches of a block: 32 of a warp
  constexpr int N = Wide<T>::N;
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* z = logits + row * stride;
  // 16-byte vectors from the first aligned element on; what is in front and behind them belongs to the first block
  const int mis = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int head = min(V, mis ? N - mis : 0), vecs = (V - head) / N, tail = head + vecs * N;
  const T* body = z + head;
  const int batches = (vecs + 32 * kUnroll - 1) / (32 * kUnroll);
  const int b0 = (int)((int64_t)part * batches / parts), b1 = (int)((int64_t)(part + 1) * batches / parts);
  const int per = max(1, (b1 - b0 + kMaxStretch - 1) / kMaxStretch);          // batches of a stretch: a lane for each of a warp's
  const int stretches = (b1 - b0 + per - 1) / per, length = per * 32 * kUnroll;      // length in vectors
  const int v_end = min(b1 * 32 * kUnroll, vecs);
  const bool little = b1 - b0 <= 2 * kWarps;       // at most two batches of a warp
  if (parts > 1) cluster.barrier_arrive();         // the first block has begun, for the writes into its shared memory
  // the token's logit on its way
  const int64_t tok = tokens[row];
  const bool real = tok >= 0 && tok < V;
  float z_tok = 0.f;
  if (tid == 0 && part == 0 && real) z_tok = q8::to_float(z[tok]);

  // ---- the pass over the row
  Sums a{-INFINITY, 0.f, 0.f};                     // m is the warp's
  // two logits at a time: S and X of the even and the odd ones
  uint64_t s2 = 0, x2 = 0;
  const uint64_t c2 = pair(c, c);
  auto take = [&](const float* f, auto count) {
    const float ref = a.m == -INFINITY ? 0.f : -a.m;
    const uint64_t ref2 = pair(ref, ref);
#pragma unroll
    for (int i = 0; i < decltype(count)::value; i += 2) {
      const float2 y = unpair(mul2(add2(pair(f[i], f[i + 1]), ref2), c2));
      const float x0 = max_nan(y.x, kFar), x1 = max_nan(y.y, kFar);
      const uint64_t e = pair(exp2_approx(x0), exp2_approx(x1));
      s2 = add2(s2, e);
      x2 = fma2(e, pair(x0, x1), x2);
    }
  };
  auto raise = [&](float y) {                      // a new warp maximum
    if (y > a.m) {
      if (a.m != -INFINITY) {
        const float d = fmaxf((a.m - y) * c, kFar), e = exp2_approx(d);
        const uint64_t e2 = pair(e, e);
        x2 = mul2(e2, fma2(s2, pair(d, d), x2));
        s2 = mul2(s2, e2);
      }
      a.m = y;
    }
  };
  // the warp's batches in order, the next one on its way while this one is summed up
  auto fetch = [&](int b, uint4 (&raw)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = (b * kUnroll + u) * 32 + lane;
      raw[u] = v < v_end ? load_raw(body + (int64_t)v * N) : raw_lowest<T>();
    }
  };
  int run = warp, b = b0 + warp * per;
  uint4 next[kUnroll];
  fetch(b, next);                                  // (behind the end: nothing is loaded)
  float most = -INFINITY;
  float maxima = -INFINITY;                        // lane i: of the warp's i-th stretch (where `little`: of the lane's logits)
  int nth = 0;
  while (run < stretches) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = next[u];
    const bool last = b + 1 >= min(b0 + (run + 1) * per, b1);
    if (last) { run += kWarps; b = b0 + run * per; } else ++b;
    if (run < stretches) fetch(b, next);
    const float mine = fmaxf(fmaxf(raw_max<T>(raw[0]), raw_max<T>(raw[1])), fmaxf(raw_max<T>(raw[2]), raw_max<T>(raw[3])));
    const float all = warp_max_f32(mine);
    if (little) maxima = fmaxf(maxima, mine);
    raise(all);
    most = fmaxf(most, all);
    if (last) {
      if (!little && lane == nth) maxima = most;
      ++nth;
      most = -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[N];
      expand<T>(raw[u], f);
      take(f, std::integral_constant<int, N>{});
    }
  }
  if (part == 0 && warp == kWarps - 1) {           // the unaligned ends
    float f[2] = {-INFINITY, -INFINITY};
    if (lane < head) f[0] = q8::to_float(z[lane]);
    if (lane >= 16 && tail + lane - 16 < V) f[0] = q8::to_float(z[tail + lane - 16]);
    raise(warp_max(f[0]));
    take(f, std::integral_constant<int, 2>{});
  }
  {
    const float2 s = unpair(s2), x = unpair(x2);
    a.s = s.x + s.y;
    a.x = x.x + x.y;
  }
  a.s = warp_sum(a.s);
  a.x = warp_sum(a.x);
  if (lane == 0) sh.warp_sums[warp] = a;
  // maxima that a warp contributes to the bound: twice n in all
  const int warps = max(1, min(kWarps, stretches)), firsts = min(32, (2 * n + warps - 1) / warps);
  if (n > 0) {
    float rest = maxima;
    for (int k = 0; k < firsts; ++k) {
      const float top = warp_max_f32(rest);
      if (lane == 0 && warp < warps) sh.firsts[warp * firsts + k] = top;
      const uint32_t at = __ballot_sync(0xffffffffu, rest == top);
      if (lane == __ffs(at) - 1) rest = -INFINITY;
    }
  }
  if (tid == 0) { sh.count = 0; sh.bound = -INFINITY; }
  for (int i = tid; i < n; i += kThreads) sh.best[i] = 0;
  __syncthreads();
  if (warp == kWarps - 1) {                        // (the warp with the least to do below)
    Sums t = lane < kWarps ? sh.warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll 1
    for (int o = kWarps / 2; o > 0; o /= 2) {
      const Sums y{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o), __shfl_xor_sync(0xffffffffu, t.x, o)};
      t = lane & o ? join(y, t, c) : join(t, y, c);
    }
    if (lane == 0) sh.sums = t;
  }

  // ---- the block's n best
  if (n > 0) {
    // the bound, by every warp for itself
    float bound = -INFINITY;
    for (int i0 = 0; i0 < warps * firsts; i0 += 32) {
      const int i = i0 + lane;
      const float v = i < warps * firsts ? sh.firsts[i] : -INFINITY;
      int rank = i < warps * firsts ? 0 : kMaxStretch;
#pragma unroll 4
      for (int j = 0; j < warps * firsts; ++j) {
        const float w = sh.firsts[j];
        rank += w > v || (w == v && j < i);
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, rank == n - 1);
      if (hit) bound = __shfl_sync(0xffffffffu, v, __ffs(hit) - 1);
    }
    auto push = [&](float v, int idx) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCand) sh.cand[at] = key_of(v, idx);
    };
    auto ends = [&](auto take_one) {
      if (part == 0 && warp == kWarps - 1) {
        if (lane < head) take_one(q8::to_float(z[lane]), lane);
        if (lane >= 16 && tail + lane - 16 < V) take_one(q8::to_float(z[tail + lane - 16]), tail + lane - 16);
      }
    };
    // what reaches it (where nothing does: NaN too, whose vectors have NaN for a maximum)
    auto look = [&](const uint4& u, int v) {
      if (!(raw_max<T>(u) < bound)) {
        float f[N];
        expand<T>(u, f);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (f[e] >= bound || (bound == -INFINITY && f[e] != f[e])) push(f[e], head + v * N + e);
      }
    };
    if (little) {
      if (maxima >= bound) {                       // the lane's own logits again
        for (int b = b0 + warp; b < b1; b += kWarps) {
          uint4 u[kUnroll];
          fetch(b, u);
#pragma unroll
          for (int x = 0; x < kUnroll; ++x)
            if ((b * kUnroll + x) * 32 + lane < v_end) look(u[x], (b * kUnroll + x) * 32 + lane);
        }
      }
    } else {
      uint32_t todo = __ballot_sync(0xffffffffu, lane < nth && maxima >= bound);
      while (todo) {                               // two stretches at a time: their loads overlap
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        const int j = todo ? __ffs(todo) - 1 : i;
        const bool two = todo != 0;
        todo &= todo - 1;
        const int v0 = b0 * 32 * kUnroll + (warp + i * kWarps) * length, v1 = b0 * 32 * kUnroll + (warp + j * kWarps) * length;
        for (int at = lane; at < length; at += 32 * kUnroll) {
          uint4 u[2][kUnroll];
#pragma unroll
          for (int x = 0; x < kUnroll; ++x) {
            u[0][x] = v0 + at + 32 * x < v_end ? load_raw(body + (int64_t)(v0 + at + 32 * x) * N) : raw_lowest<T>();
            u[1][x] = two && v1 + at + 32 * x < v_end ? load_raw(body + (int64_t)(v1 + at + 32 * x) * N) : raw_lowest<T>();
          }
#pragma unroll
          for (int x = 0; x < kUnroll; ++x) {
            if (v0 + at + 32 * x < v_end) look(u[0][x], v0 + at + 32 * x);
            if (two && v1 + at + 32 * x < v_end) look(u[1][x], v1 + at + 32 * x);
          }
        }
      }
    }
    ends(push);
    __syncthreads();
    int count = sh.count, chosen = 0;
    if (count > kCand) {                           // too many: the n stretches with the largest maxima, equal logits counted
      if (little) {
        for (int i = 0; i < nth; ++i) {            // a stretch is one batch
          uint4 u[kUnroll];
          fetch(b0 + warp + i * kWarps, u);
          const float m = warp_max_f32(fmaxf(fmaxf(raw_max<T>(u[0]), raw_max<T>(u[1])), fmaxf(raw_max<T>(u[2]), raw_max<T>(u[3]))));
          if (lane == 0) sh.stretch[warp + i * kWarps] = fmaxf(m, -INFINITY);        // of nothing but NaN: -inf
        }
      } else if (lane < nth) {
        sh.stretch[warp + lane * kWarps] = maxima;
      }
      __syncthreads();
      for (int i = tid; i < stretches; i += kThreads) {
        const float v = sh.stretch[i];
        int rank = 0;
        for (int j = 0; j < stretches; ++j) {
          const float w = sh.stretch[j];
          rank += w > v || (w == v && j < i);
        }
        if (rank < n) sh.chosen[rank] = i;
        if (rank == n - 1) sh.bound = v;
      }
      if (tid == 0) sh.count = 0;
      __syncthreads();
      bound = sh.bound;
      chosen = min(n, stretches);
      for (int r = warp; r < chosen; r += kWarps) {
        int equal = 0;                             // logits equal to the bound so far; no more than n - r can matter
        const int v0 = b0 * 32 * kUnroll + sh.chosen[r] * length, v1 = min(v0 + length, v_end);
        for (int v = v0 + lane; v - lane < v1; v += 32) {
          float f[N];
          int mine = 0;
          if (v < v1) {
            load16(body + (int64_t)v * N, f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              f[i] = f[i] == f[i] ? f[i] : -INFINITY;
              mine += f[i] == bound;
              if (f[i] > bound) push(f[i], head + v * N + i);
            }
          }
          if (__any_sync(0xffffffffu, mine > 0)) {
            int inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int p = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += p;
            }
            int to = equal + inc - mine;
            if (mine > 0)
#pragma unroll
              for (int i = 0; i < N; ++i)
                if (f[i] == bound) {
                  if (to < n - r) push(f[i], head + v * N + i);
                  ++to;
                }
            equal += __shfl_sync(0xffffffffu, inc, 31);
          }
        }
      }
      ends(push);
      __syncthreads();
      count = sh.count;
    }
    if (count <= kSmall) {
      if (tid < count) {                           // (kSmall < kThreads)
        const uint64_t k = sh.cand[tid];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += sh.cand[j] > k;
        if (rank < n) sh.best[rank] = k;
      }
      __syncthreads();
    } else if (count <= kCand) {
      sort_keys<kThreads>(sh.cand, count);
      if (tid < n && tid < count) sh.best[tid] = sh.cand[tid];
      __syncthreads();
    } else {
      // thousands of logits of few stretches above the bound (ascending rows, for one): n rounds of the largest key
      // below the last one, over the chosen stretches
      uint64_t last = ~0ull;
      for (int k = 0; k < n; ++k) {
        uint64_t mine = 0;
        auto see = [&](float v, int idx) {
          const uint64_t x = key_of(v, idx);
          if (x < last && x > mine) mine = x;
        };
        for (int r = warp; r < chosen; r += kWarps) {
          const int v0 = b0 * 32 * kUnroll + sh.chosen[r] * length, v1 = min(v0 + length, v_end);
          for (int v = v0 + lane; v < v1; v += 32) {
            float f[N];
            load16(body + (int64_t)v * N, f);
#pragma unroll
            for (int i = 0; i < N; ++i) see(f[i], head + v * N + i);
          }
        }
        ends(see);
        if (tid == 0) sh.round = 0;
        __syncthreads();
        if (mine) atomicMax(reinterpret_cast<unsigned long long*>(&sh.round), (unsigned long long)mine);
        __syncthreads();
        last = sh.round;
        if (tid == 0) sh.best[k] = last;
        __syncthreads();
      }
    }
  }

  // ---- the cluster's parts meet in its first block
  if (parts > 1) {
    __syncthreads();
    cluster.barrier_wait();
    if (part > 0) {
      Shared<kThreads>* to = cluster.map_shared_rank(&sh, 0);
      if (tid < n) to->best[part * n + tid] = sh.best[tid];
      if (tid == 0) to->part_sums[part] = sh.sums;
    }
    cluster.barrier_arrive();                      // what was written is there for those who wait
    if (part > 0) return;
    cluster.barrier_wait();
    const int total = parts * n;
    for (int i = tid; i < total; i += kThreads) {
      const uint64_t k = sh.best[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < total; ++j) rank += sh.best[j] > k;
      if (k && rank < n) sh.cand[rank] = k;
    }
    if (warp == kWarps - 1) {
      Sums t = lane == 0 ? sh.sums : lane < parts ? sh.part_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll 1
      for (int o = 4; o > 0; o /= 2) {
        const Sums y{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o), __shfl_xor_sync(0xffffffffu, t.x, o)};
        t = lane & o ? join(y, t, c) : join(t, y, c);
      }
      if (lane == 0) sh.sums = t;
    }
  }
  const uint64_t* best = parts > 1 ? sh.cand : sh.best;
  __syncthreads();
  const Sums t = sh.sums;
  const bool empty = t.m == -INFINITY && t.s == 0.f;                          // nothing but -inf
  const float ls = log2f(t.s);
  auto logprob = [&](float v) { return empty ? -INFINITY : fmaf(v - t.m, inv_temp, -ls * kLn2); };
  if (tid == 0) {
    lp[row] = real ? logprob(z_tok) : 0.f;
    ent[row] = empty ? 0.f : (ls - t.x / t.s) * kLn2;
    stats[2 * row] = t.m;
    stats[2 * row + 1] = ls;
  }
  if (tid < n) {
    const uint64_t k = best[tid];
    top_lp[row * n + tid] = logprob(value_of(k));
    top_id[row * n + tid] = index_of(k);
  }
}

// dz_j = 1/temperature [ g_lp d(j = token) + sum_k g_top_k d(j = top_k) - p_j (g_lp + sum_k g_top_k) - g_ent p_j (ln p_j + H) ]
// One read of the logits, one write of the gradient; the columns of the token and the alternatives are written again
// after the stretch that holds them.  Bound by the two passes' bytes: 1,024 x 152 k bf16 115 us, 5.4 TB/s.
constexpr int kGradThreads = 256, kGradVecs = 4;   // vectors of a thread, all on their way at a time
constexpr int kGradSpan = kGradThreads * kGradVecs * 16;                    // bytes of a row that a block handles

template <typename T>
__global__ void __launch_bounds__(kGradThreads)
token_logprob_grad_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ tokens, int V, int n,
                          int spans, float c, float inv_temp, const float* __restrict__ ent, const float* __restrict__ stats,
                          const int64_t* __restrict__ top_id, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                          const float* __restrict__ g_top, T* __restrict__ dz, int64_t dz_stride) {
  constexpr int N = Wide<T>::N;
  pdl_trigger();
  pdl_wait();
  // last rows first: the forward pass has left them in L2
  const int64_t row = (gridDim.x - 1 - blockIdx.x) / spans;
  const int span = (int)((gridDim.x - 1 - blockIdx.x) % spans), tid = threadIdx.x, lane = tid & 31;
  const T* z = logits + row * stride;
  T* d = dz + row * dz_stride;
  // both rows at the same place inside 16 bytes: vectors; else single elements
  const int mis = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int head = same ? min(V, mis ? N - mis : 0) : 0, vecs = same ? (V - head) / N : 0, tail = head + vecs * N;
  constexpr int kVecs = kGradSpan / 16;
  const int v0 = span * kVecs + tid;
  uint4 raw[kGradVecs];
#pragma unroll
  for (int i = 0; i < kGradVecs; ++i)
    if (v0 + i * kGradThreads < vecs) raw[i] = load_raw(z + head + (int64_t)(v0 + i * kGradThreads) * N);
  const int64_t tok = tokens[row];
  const float M = stats[2 * row], ls = stats[2 * row + 1], H = ent[row];
  const bool empty = M == -INFINITY && ls == -INFINITY;                       // log2 of an empty sum
  const float gl = g_lp && tok >= 0 && tok < V ? g_lp[row] : 0.f, ge = g_ent ? g_ent[row] : 0.f;
  float g_all = 0.f;                               // every warp for itself
  if (g_top) {
    for (int i = lane; i < n; i += 32) g_all += g_top[row * n + i];
    g_all = warp_sum(g_all);
  }
  // p (A x + B) with x = log2 p
  const float A = -inv_temp * ge * kLn2, B = -inv_temp * (gl + g_all + ge * H);
  auto grad = [&](float v) {
    const float x = max_nan(fmaf(v - M, c, -ls), kFar);
    return empty ? 0.f : exp2_approx(x) * fmaf(x, A, B);
  };
  int lo, hi;                                      // columns of this block
  if (same) {
    // what lies behind the last whole vector is the last span's, though an earlier one may reach over it
    lo = span == 0 ? 0 : min(tail, head + span * kVecs * N);
    hi = span == spans - 1 ? V : min(tail, head + (span + 1) * kVecs * N);
    if (span == 0 && tid < head) d[tid] = q8::from_float<T>(grad(q8::to_float(z[tid])));
#pragma unroll
    for (int i = 0; i < kGradVecs; ++i)
      if (v0 + i * kGradThreads < vecs) {
        float f[N];
        expand<T>(raw[i], f);
        uint4 u;
        T* o = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = q8::from_float<T>(grad(f[e]));
        __stcs(reinterpret_cast<uint4*>(d + head + (int64_t)(v0 + i * kGradThreads) * N), u);
      }
    if (span == spans - 1)
      for (int i = tail + tid; i < V; i += kGradThreads) d[i] = q8::from_float<T>(grad(q8::to_float(z[i])));
  } else {
    lo = min(V, span * kVecs * N);
    hi = span == spans - 1 ? V : min(V, lo + kVecs * N);
    for (int i = lo + tid; i < hi; i += kGradThreads) d[i] = q8::from_float<T>(grad(q8::to_float(z[i])));
  }
  // thread n: the token; an alternative that is the token is its job
  const int64_t col = tid < n ? top_id[row * n + tid] : tok;
  const bool own = tid <= n && !empty && col >= lo && col < hi && !(tid < n && col == tok);
  __syncthreads();
  if (own) {
    float add = tid < n ? (g_top ? g_top[row * n + tid] : 0.f) : gl;
    if (tid == n && g_top)
      for (int i = 0; i < n; ++i)
        if (top_id[row * n + i] == tok) add += g_top[row * n + i];
    d[col] = q8::from_float<T>(fmaf(add, inv_temp, grad(q8::to_float(z[col]))));
  }
}

// Threads of a block: 512 (more to read for each of what a block does once); 256 where rows are so short that this is most
// of the time (300 rows, 512 and 256 threads: 4000 fp32 logits with 20 alternatives 13.7 and 9.9 us, 32 k with 5 16.4 and
// 15.3 us; 128 rows of 152 k bf16 logits with 8 20.0 and 26.4 us).
constexpr int kShortRow = 160 << 10;
// blocks that share a row: as many as the GPU holds at a time, each with some to read (1 / 16 / 64 rows of 152 k fp32 logits
// with 8 alternatives: 15.0 / 16.7 / 24.3 us with one block a row, 11.3 / 11.0 / 13.9 us with clusters)
constexpr int kLeast = 32768;
int cluster_for(int64_t rows, int64_t row_bytes, int threads) {
  const int kBlocks = kSmThreads / threads;
  int parts = 1;
  while (parts < 8 && rows * parts * 2 <= kBlocks * 148 && row_bytes >= parts * 2 * kLeast) parts *= 2;
  return parts;
}

}  // namespace

// {log-prob, entropy, alternatives' log-probs, their ids, statistics for the gradient}; empty where the arguments are not as
// the kernel takes them.
std::vector<at::Tensor> token_logprob_fwd(const at::Tensor& z, const at::Tensor& tokens, int64_t n, double inv_temp) {
  const auto type = z.scalar_type();
  const bool fits = z.is_cuda() && z.dim() == 2 && (type == at::kBFloat16 || type == at::kHalf || type == at::kFloat) && z.size(1) > 0 &&
                    (z.size(1) == 1 || z.stride(1) == 1) && z.size(0) < (int64_t)1 << 28 && z.size(1) < (int64_t)1 << 30 && n >= 0 &&
                    n <= std::min<int64_t>(kMaxTop, z.size(1)) && inv_temp > 0.0 && tokens.scalar_type() == at::kLong && tokens.dim() == 1 &&
                    tokens.size(0) == z.size(0) && tokens.is_contiguous() && tokens.device() == z.device() &&
                    !z._fw_grad(0).defined();
  if (!fits) return {};
  const c10::cuda::CUDAGuard guard(z.device());
  const int64_t R = z.size(0), V = z.size(1);
  auto f = z.options().dtype(at::kFloat);
  auto lp = at::empty({R}, f), ent = at::empty({R}, f), stats = at::empty({R, 2}, f), top = at::empty({R, n}, f);
  auto ids = at::empty({R, n}, z.options().dtype(at::kLong));
  if (R == 0) return {lp, ent, top, ids, stats};
  const int64_t row_bytes = V * (int64_t)z.element_size();
  const int threads = row_bytes <= kShortRow ? 256 : 512;
  const int parts = cluster_for(R, row_bytes, threads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(R * parts)); cfg.blockDim = dim3(threads); cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const float c = (float)(inv_temp * 1.4426950408889634);
#define LAUNCH(T)                                                                                                        \
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, threads == 256 ? token_logprob_kernel<T, 256> : token_logprob_kernel<T, 512>, (const T*)z.data_ptr(), z.stride(0),                   \
                                    (const int64_t*)tokens.data_ptr<int64_t>(), (int)V, (int)n, c, (float)inv_temp, lp.data_ptr<float>(),  \
                                    ent.data_ptr<float>(), stats.data_ptr<float>(), top.data_ptr<float>(), ids.data_ptr<int64_t>()))
  if (z.scalar_type() == at::kFloat) LAUNCH(float);
  else if (z.scalar_type() == at::kHalf) LAUNCH(__half);
  else LAUNCH(__nv_bfloat16);
#undef LAUNCH
  return {lp, ent, top, ids, stats};
}

at::Tensor token_logprob_bwd(const at::Tensor& z, const at::Tensor& tokens, const at::Tensor& ent, const at::Tensor& stats,
                             const at::Tensor& ids, const c10::optional<at::Tensor>& g_lp, const c10::optional<at::Tensor>& g_ent,
                             const c10::optional<at::Tensor>& g_top, double inv_temp) {
  const c10::cuda::CUDAGuard guard(z.device());
  const int64_t R = z.size(0), V = z.size(1), n = ids.size(1);
  // rows at the places that the logits' rows have inside 16 bytes, so that both go in vectors (a little padding stays)
  const int64_t stride = z.stride(0) >= V && z.stride(0) - V <= 128 ? z.stride(0) : V;
  auto dz = at::empty({R, stride}, z.options()).narrow(1, 0, V);
  if (R == 0 || V == 0) return dz;
  const int esize = (int)z.element_size();
  const int spans = (int)((V * esize + kGradSpan - 1) / kGradSpan);
  auto ptr = [](const c10::optional<at::Tensor>& t) { return t.has_value() && t->numel() ? (const float*)t->data_ptr<float>() : nullptr; };
  const float c = (float)(inv_temp * 1.4426950408889634);
  auto st = at::cuda::getCurrentCUDAStream();
#define LAUNCH(T)                                                                                                          \
  C10_CUDA_CHECK(launch_pdl(token_logprob_grad_kernel<T>, dim3((unsigned)(R * spans)), dim3(kGradThreads), 0, st,           \
                            (const T*)z.data_ptr(), z.stride(0), (const int64_t*)tokens.data_ptr<int64_t>(), (int)V, (int)n, \
                            spans, c, (float)inv_temp, (const float*)ent.data_ptr<float>(), (const float*)stats.data_ptr<float>(), \
                            (const int64_t*)ids.data_ptr<int64_t>(), ptr(g_lp), ptr(g_ent), ptr(g_top), (T*)dz.data_ptr(), dz.stride(0)))
  if (z.scalar_type() == at::kFloat) LAUNCH(float);
  else if (z.scalar_type() == at::kHalf) LAUNCH(__half);
  else LAUNCH(__nv_bfloat16);
#undef LAUNCH
  return dz;
}
