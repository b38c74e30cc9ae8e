// Appending to the paged key/value cache held in 8 bits.
//
// One power-of-two scale s per (page, kv head, K or V); a cached value is s times an e4m3 code.  New rows of a page need
//   need = 2^ceil(log2(amax / 448)), clamped to [2^-24, 2^64],  amax over the finite |x| of the page's new rows;
//   s'   = need where the page begins with them (slot 0 is among them), else max(s, need).
// Where s' > s the page's older codes become RN(code * s / s'); the new rows are RN_sat(x / s').  e4m3 is a floating
// format, so a power-of-two scale costs no precision, dividing by it is exact, and a grown scale moves the exponents of
// the older codes: only codes that leave the normal range (below 2^-6) lose bits, once per growth.
//
// The rows are named by sequence (block table, length, new tokens), so one block owns all rows of a page that a call
// writes: the page's maximum is taken and its rows are written in one pass over them, with no atomics and no second
// launch.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "q8.cuh"
#include "q8_attention.h"

using namespace cl;
using namespace q8;

namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const void* x[2];              // new keys, new values
  int64_t row[2], head[2];       // strides in elements
  uint8_t* codes[2];             // [pages, nkv, bs, D]
  float* scale[2];               // [pages, nkv]
  const int* tables;             // [B, width]
  const int* lens;               // [B] lengths with the new tokens
  const int* news;               // [B] new tokens (null: one each)
  int B, width, T, nkv, D, bs;
  int64_t pages;
};

// 8 consecutive elements as they are, and as fp32; `vec`: the address is 16-byte aligned
template <typename T>
struct __align__(16) Raw {
  T x[8];
};
template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p, bool vec) {
  Raw<T> r;
  if (vec) {
#pragma unroll
    for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) *reinterpret_cast<uint4*>(&r.x[i]) = *reinterpret_cast<const uint4*>(p + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = p[i];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void expand(const Raw<T>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_float(r.x[i]);
}

// Largest magnitude, NaN left out, infinities not; and the largest finite one, for where there are infinities.  (bf16 and
// fp16 two at a time: an and and a maximum for two elements.)
__device__ __forceinline__ float magnitude(const Raw<float>& r) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(r.x[i]));
  return m;
}
__device__ __forceinline__ float magnitude(const Raw<__nv_bfloat16>& r) {
  const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(r.x);
  const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(x[0]), __habs2(x[1])), __hmax2(__habs2(x[2]), __habs2(x[3])));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float magnitude(const Raw<__half>& r) {
  const __half2* x = reinterpret_cast<const __half2*>(r.x);
  const __half2 m = __hmax2(__hmax2(__habs2(x[0]), __habs2(x[1])), __hmax2(__habs2(x[2]), __habs2(x[3])));
  return fmaxf(__low2float(m), __high2float(m));
}
template <typename T>
__device__ __forceinline__ float finite_magnitude(const Raw<T>& r) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(to_float(r.x[i]));
    m = a < INFINITY ? fmaxf(m, a) : m;
  }
  return m;
}

__device__ __forceinline__ void store8(uint8_t* p, const float (&f)[8], float inv) {
  uint2 u;
  u.x = pack_e4m3(f[0] * inv, f[1] * inv) | (uint32_t)pack_e4m3(f[2] * inv, f[3] * inv) << 16;
  u.y = pack_e4m3(f[4] * inv, f[5] * inv) | (uint32_t)pack_e4m3(f[6] * inv, f[7] * inv) << 16;
  *reinterpret_cast<uint2*>(p) = u;
}

// older codes of a page under its grown scale; n is a multiple of 8
__device__ __forceinline__ void regrade(uint8_t* codes, int n, float ratio, int tid, int step) {
  for (int i = tid * 8; i < n; i += step * 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(codes + i);
    float f[8];
    unpack_e4m3(u.x, f);
    unpack_e4m3(u.y, f + 4);
    store8(codes + i, f, ratio);
  }
}

// One token per sequence: a warp per (sequence, kv head, K or V).  The chain length -> table -> scale of dependent
// loads is all there is to wait for; the row itself is loaded beside it.  128 sequences (8 kv heads of 128): 3.0 us, 5.3
// from the caller's side.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_step_kernel(const AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5);
  const int b = (int)(item / (2 * a.nkv)), h = (int)(item / 2 % a.nkv), kv = (int)(item & 1);
  if (b >= min(a.B, a.T)) return;
  const T* x = static_cast<const T*>(a.x[kv]) + b * a.row[kv] + h * a.head[kv];
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  Raw<T> kept;                                     // D <= 256: 8 elements of a lane
  float amax = 0.f;
  const bool mine = lane * 8 < a.D;
  if (mine) {
    kept = load8(x + lane * 8, vec);
    amax = magnitude(kept);
  }
  amax = warp_max(amax);
  if (!(amax < INFINITY)) amax = warp_max(mine ? finite_magnitude(kept) : 0.f);
  const int pos = a.lens[b] - 1;
  if (pos < 0 || pos / a.bs >= a.width) return;
  const int page = a.tables[(int64_t)b * a.width + pos / a.bs], off = pos % a.bs;
  if (page < 0 || page >= a.pages) return;
  const int64_t ph = (int64_t)page * a.nkv + h;
  uint8_t* codes = a.codes[kv] + ph * a.bs * a.D;
  float s = scale_for(amax);
  if (off > 0) {
    const float old = a.scale[kv][ph];
    if (s > old) regrade(codes, off * a.D, old / s, lane, 32);
    else s = old;
  }
  __syncwarp();
  if (lane == 0) a.scale[kv][ph] = s;
  const float inv = 1.f / s;
  if (mine) {
    float f[8];
    expand(kept, f);
    store8(codes + (int64_t)off * a.D + lane * 8, f, inv);
  }
}

// Any number of tokens per sequence: a block per (page that gets new rows, kv head, K or V).  The rows of a page of 64 x
// 128 fit the block's registers (kKeep vectors of 8 a thread), so they are read once; longer pages read the rest again,
// out of L2.  Blocks of the same rows run side by side (heads, then K and V): a row's heads lie beside each other.
// 16 prompts of 900 to 1,152 tokens (100 MB in bf16 rows and codes): 22.4 us, 4.5 TB/s.  Bound by the chain in each block:
// find the page, load (rows and page id beside each other), block maximum, store.  So many small blocks: 128 threads, 8
// blocks an SM 22.4 us; 64 threads, 10 blocks 23.6; 256 threads, 6 or 5 blocks 24.3 and 27.3; 512 threads, 4 blocks 33.
constexpr int kPageThreads = 128, kKeep = 8;

template <typename T>
__global__ void __launch_bounds__(kPageThreads, sizeof(T) == 4 ? 5 : 8) append_pages_kernel(const AppendArgs a) {
  __shared__ int sh_found[5];
  __shared__ float sh_max[kPageThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x % a.nkv, kv = blockIdx.x / a.nkv & 1, run = blockIdx.x / (2 * a.nkv);
  // which (sequence, page) is this block's: prefix sums of the pages and rows that the sequences add
  if (warp == 0) {
    if (lane == 0) sh_found[0] = -1;
    __syncwarp();
    int pages = 0, rows = 0;                       // before these 32 sequences
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + lane;
      const int len = b < a.B ? a.lens[b] : 0, n = b < a.B ? max(0, a.news[b]) : 0, begin = max(len - n, 0);
      const int cnt = n > 0 && len > 0 ? (len - 1) / a.bs - begin / a.bs + 1 : 0;
      int ip = cnt, ir = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(0xffffffffu, ip, o), r = __shfl_up_sync(0xffffffffu, ir, o);
        if (lane >= o) { ip += p; ir += r; }
      }
      const int first = pages + ip - cnt;
      if (cnt > 0 && first <= run && run < first + cnt) {
        const int pg = begin / a.bs + (run - first);
        const int lo = max(begin, pg * a.bs), hi = min(len, (pg + 1) * a.bs);
        const int row = rows + ir - n + (lo - (len - n));      // row of the page's first new token
        sh_found[1] = lo - pg * a.bs;
        sh_found[2] = min(hi - lo, a.T - row);                 // rows that the tensors really hold
        sh_found[3] = row;
        sh_found[4] = pg;
        if (sh_found[2] > 0 && pg < a.width) sh_found[0] = b;
      }
      pages += __shfl_sync(0xffffffffu, ip, 31);
      rows += __shfl_sync(0xffffffffu, ir, 31);
      if (pages > run) break;
    }
  }
  __syncthreads();
  const int seq = sh_found[0], off = sh_found[1], m = sh_found[2], row = sh_found[3];
  if (seq < 0) return;
  const int page = a.tables[(int64_t)seq * a.width + sh_found[4]];       // on its way while the rows are
  const T* x = static_cast<const T*>(a.x[kv]) + row * a.row[kv] + h * a.head[kv];
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(a.row[kv] * sizeof(T))) & 15) == 0;
  const int shift = a.D == 64 ? 3 : a.D == 128 ? 4 : 5, total = m << shift;
  // the thread's vectors, tid + i * kPageThreads; those of a row lie side by side
  auto at = [&](int c) { return (c >> shift) * a.row[kv] + (c & ((1 << shift) - 1)) * 8; };
  Raw<T> kept[kKeep];
  float amax = 0.f, f[8];
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (i * kPageThreads + tid < total) kept[i] = load8(x + at(i * kPageThreads + tid), vec);
  if (page < 0 || page >= a.pages) return;
  const int64_t ph = (int64_t)page * a.nkv + h;
  const float old = off > 0 ? a.scale[kv][ph] : 0.f;
  auto largest = [&](auto of) {                    // over the block, by `of` each vector
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
      if (i * kPageThreads + tid < total) m = fmaxf(m, of(kept[i]));
    for (int c = kKeep * kPageThreads + tid; c < total; c += kPageThreads) m = fmaxf(m, of(load8(x + at(c), vec)));
    m = warp_max(m);
    if (lane == 0) sh_max[warp] = m;
    __syncthreads();                               // every thread has read the old scale, too
#pragma unroll
    for (int w = 0; w < kPageThreads / 32; ++w) m = fmaxf(m, sh_max[w]);
    return m;
  };
  amax = largest([](const Raw<T>& r) { return magnitude(r); });
  if (!(amax < INFINITY)) {
    __syncthreads();
    amax = largest([](const Raw<T>& r) { return finite_magnitude(r); });
  }
  const float s = fmaxf(scale_for(amax), old), inv = 1.f / s;
  uint8_t* codes = a.codes[kv] + ph * a.bs * a.D;
  if (off > 0 && s > old) regrade(codes, off * a.D, old / s, tid, kPageThreads);
  if (tid == 0) a.scale[kv][ph] = s;
  uint8_t* to = codes + (int64_t)off * a.D;
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (i * kPageThreads + tid < total) {
      expand(kept[i], f);
      store8(to + (i * kPageThreads + tid) * 8, f, inv);
    }
  for (int c = kKeep * kPageThreads + tid; c < total; c += kPageThreads) {
    expand(load8(x + at(c), vec), f);
    store8(to + c * 8, f, inv);
  }
}

template <typename T>
void launch_append(const AppendArgs& a, cudaStream_t st) {
  if (!a.news) {
    const int64_t items = (int64_t)std::min(a.B, a.T) * a.nkv * 2;
    const int64_t grid = (items + kThreads / 32 - 1) / (kThreads / 32);
    C10_CUDA_CHECK(launch_pdl(append_step_kernel<T>, dim3((unsigned)grid), dim3(kThreads), 0, st, a));
  } else {
    // a sequence with n new tokens adds to at most (n - 1) / bs + 2 pages
    const int64_t runs = std::min<int64_t>(a.T, a.T / a.bs + 2 * (int64_t)a.B);
    C10_CUDA_CHECK(launch_pdl(append_pages_kernel<T>, dim3((unsigned)(runs * a.nkv * 2)), dim3(kPageThreads), 0, st, a));
  }
}

}  // namespace

// False, and nothing done, where the arguments are not as the kernels take them.
bool kv_append_q8(const at::Tensor& k, const at::Tensor& v, at::Tensor kc, at::Tensor vc, at::Tensor ks, at::Tensor vs,
                  const at::Tensor& tables, const at::Tensor& lens, const c10::optional<at::Tensor>& news) {
  const auto type = k.scalar_type();
  const bool fits = k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes() && v.scalar_type() == type && v.device() == k.device() &&
                    (type == at::kBFloat16 || type == at::kHalf || type == at::kFloat) && k.stride(2) == 1 && v.stride(2) == 1 &&
                    q8::cache_fits(kc, vc, ks, vs, tables, lens, news, k.device()) && kc.size(1) == k.size(1) && kc.size(3) == k.size(2) &&
                    (k.size(2) == 64 || k.size(2) == 128 || k.size(2) == 256) && k.size(0) < (int64_t)1 << 31 &&
                    (news.has_value() || k.size(0) >= lens.size(0));
  if (!fits) return false;
  const c10::cuda::CUDAGuard guard(k.device());
  AppendArgs a;
  a.x[0] = k.data_ptr(); a.x[1] = v.data_ptr();
  a.row[0] = k.stride(0); a.row[1] = v.stride(0);
  a.head[0] = k.stride(1); a.head[1] = v.stride(1);
  a.codes[0] = (uint8_t*)kc.data_ptr(); a.codes[1] = (uint8_t*)vc.data_ptr();
  a.scale[0] = ks.data_ptr<float>(); a.scale[1] = vs.data_ptr<float>();
  a.tables = tables.data_ptr<int>(); a.lens = lens.data_ptr<int>();
  a.news = news.has_value() ? news->data_ptr<int>() : nullptr;
  a.B = (int)lens.size(0); a.width = (int)tables.size(1); a.T = (int)k.size(0);
  a.nkv = (int)kc.size(1); a.bs = (int)kc.size(2); a.D = (int)kc.size(3); a.pages = kc.size(0);
  if (a.B == 0 || a.T == 0 || a.width == 0) return true;
  auto st = at::cuda::getCurrentCUDAStream();
  if (k.scalar_type() == at::kBFloat16) launch_append<__nv_bfloat16>(a, st);
  else if (k.scalar_type() == at::kHalf) launch_append<__half>(a, st);
  else launch_append<float>(a, st);
  return true;
}
