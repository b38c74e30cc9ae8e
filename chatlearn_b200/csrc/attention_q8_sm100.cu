// Attention of many new tokens per sequence over the paged 8-bit cache, on the 5th-generation tensor cores.
//
// Continuation chunks of a prefill attend over everything cached before them: with hundreds of new tokens per sequence
// the two products bound the work, not the cache's bytes.  A CTA owns G groups of 128 query rows of one sequence and one
// kv head: 128 G / rep tokens times the rep query heads that share the head, so a cached tile is dequantised once for all
// of them.  Warps, for G = 2 (one CTA to an SM) and G = 1 (two, but for elements of 256):
//   4 G   softmax, thread = query row: first the row itself, rescaled by a power of two to fp16, into shared memory;
//         then per tile of 64 keys the scores out of tensor memory, running maximum (lazily applied, as soon as it has
//         run ahead by 2^8) and sum, P as fp16 back over the scores; at the end O / l to the output.  Two groups take
//         turns at the exponentials: one's run beside the other's maxima (both at once had the special-function units
//         wait on them first and then stand idle: 389 -> 351 us at the case below)
//   4     dequantisation: e4m3 codes from the pages, copied to shared memory a tile ahead, to fp16 tiles (exact) in the
//         128-byte swizzle.  K's scales stay out of the tiles: S takes them, one for each 16 keys where pages end inside a
//         tile, so that scales of any distance leave each other's keys alone.  V's too (P takes it) where a page covers
//         the tile.  Of other pages V is brought to the largest of its scales where they are within 2^8 (exact: its
//         smallest code is then 2^-17), else V becomes bf16 values (exact) and P two bf16, the second what the first's
//         rounding leaves (16 bits in all), as fp16 has not the range for scales far apart.
//         (8 x 256 tokens on pages of 16: 277 us, where every tile's scales are far apart 316)
//   1     one elected thread issues, for each group, S = Q K^T (128x64x16) into one of two accumulators and O += P V
//         (128xDx16, P from tensor memory, V as an MN-major operand straight from its row-major tile), one tile behind
// O is kept in units of a V scale that follows the tiles' scales where they are far apart (as in the decode kernel).
// The queries are causal inside their sequence's new tokens.  Every mbarrier wait is bounded; one that runs out records a
// status, the CTA drains and frees its tensor memory.
//
// P is rounded to fp16 (or two bf16) once, as the matrix instruction takes it: 2^-11 of each probability; the sum is fp32.
//
// 8 sequences of 512 new tokens after 3,300 to 3,800, 32 / 8 heads of 128: 363 us, 700 TFLOP/s of the visible pairs (42 % of
// a library product's rate); the tensor pipe is 40 % busy while a CTA runs.  What bounds it: a softmax thread's chain of
// dependent instructions over its tile (2 warps to a scheduler), and 512 CTAs on 148 SMs, of whose fourth wave half is idle.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAException.h>

#include <atomic>
#include <type_traits>

#include "q8.cuh"
#include "q8_attention.h"
#include "sm100.cuh"

using namespace cl;
using namespace q8;
using namespace sm100;

namespace {

constexpr int BM = 128, BN = 64, kStages = 2, kInfo = 8;
constexpr uint32_t kChunk = BN * 128;             // 64 keys x 64 elements of fp16
constexpr float kRescale = 8.f;                   // bits that the maximum may run ahead
constexpr float kShift = 7.f;                     // P times 2^7: at most 2^15, and normal down to 2^-21 of a row's largest
// Scores (in bits) from which a score's product is rounded before the maximum is taken off.  The exact product inside a
// fused multiply-add is off the rounded maximum by up to half a step of it: 2^-4 at 2^20, more than P has room for from 2^24 on
constexpr float kFarScore = 0x1p20f;

struct TileInfo { float ks, vs, log2_vs, per_vs; uint32_t seen[2], bf; };      // scales of the tile, keys that exist, P and V in bf16

// G: groups of 128 query rows
template <int D, int G>
struct Smem {
  uint8_t q[G][D / 64][BM * 128];
  uint8_t k[kStages][D / 64][kChunk];
  uint8_t v[kStages][D / 64][kChunk];
  uint4 raw[2][BN * D / 16];                        // the codes of the tile to come, each piece read by the thread that copied it
  TileInfo info[kInfo];
  float4 ks[kInfo];                                 // K's scale of each 16 keys, where pages end inside a tile
  float red[2][4];
  uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[G][2], p_full[G][2], pv_done[G], turn[2];
  uint32_t tmem_base;
  int seq, tile, row0, len, n;
};

__device__ int g_q8_status = 0;
enum : int { ST_OK = 0, ST_CONVERT = 1, ST_MMA = 2, ST_SOFTMAX = 3, ST_SMEM_ALIGN = 4 };

// bf: 0 fp16 operands, 1 bf16
__host__ __device__ constexpr uint32_t idesc_of(int M, int N, int b_mn, int bf) {
  return (1u << 4) | ((uint32_t)bf << 7) | ((uint32_t)bf << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t y;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(y));
  return y != 0;
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D += A B with A in tensor memory, two 16-bit elements of a row to a column
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// loads that stay where they are written: the compiler would move them down to the use of their value, and wait there
__device__ __forceinline__ float load_here(const float* at) {
  float x;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(x) : "l"(at));
  return x;
}
__device__ __forceinline__ int load_here(const int* at) {
  int x;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(x) : "l"(at));
  return x;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t half2_mul(uint32_t a, __half2 b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// SMALL: pages that are no multiple of 64 tokens
template <int D, bool SMALL, int G>
__global__ void __launch_bounds__(128 * G + 160, D == 256 || G == 2 ? 1 : 2) chunk_q8_kernel(const ChunkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  Smem<D, G>* sm = reinterpret_cast<Smem<D, G>*>(smem_raw);
  constexpr int kOCol = 2 * BN, kGroupCols = kOCol + D, kTmemCols = G * kGroupCols > 256 ? 512 : 256;
  static_assert(G * kGroupCols <= 512, "tensor memory has 512 columns");
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int rep = a.nq / a.nkv, tokens = G * BM / rep;     // tokens of a tile

  // ---- which (sequence, tile) is this CTA's; a sequence's tiles are listed last-first: those with the most keys begin first
  if (warp == 0) {
    int left = blockIdx.x, rows = 0, seq = -1;
    for (int s0 = 0; s0 < a.B; s0 += 32) {
      const int s = s0 + lane;
      const int n = s < a.B ? max(a.news[s], 0) : 0;
      int ir = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, ir, o);
        if (lane >= o) ir += y;
      }
      const int held = min(n, a.T - (rows + ir - n));      // rows that the tensor really holds
      const int nt = n >= a.min_new && held > 0 ? (held + tokens - 1) / tokens : 0;
      int it = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, it, o);
        if (lane >= o) it += x;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, it > left && it - nt <= left);
      if (hit) {
        if (hit >> lane & 1) {
          sm->tile = nt - 1 - (left - (it - nt));
          sm->row0 = rows + ir - n;
          sm->n = n;
          sm->len = a.lens[s];
        }
        seq = s0 + __ffs(hit) - 1;
        break;
      }
      left -= __shfl_sync(0xffffffffu, it, 31);
      rows += __shfl_sync(0xffffffffu, ir, 31);
    }
    if (lane == 0) {
      sm->seq = seq;
      if ((smem_u32(smem_raw) & 1023u) != 0u) { sm->seq = -1; atomicCAS(&g_q8_status, ST_OK, ST_SMEM_ALIGN); }
    }
  }
  __syncthreads();
  const int seq = sm->seq;
  if (seq < 0) return;                             // surplus CTA of the over-sized grid (nothing allocated yet)
  const int n = sm->n, len = sm->len, row0 = sm->row0, t0 = sm->tile * tokens;
  const int first_pos = len - n + t0;              // position of the tile's first token
  const int keys = max(0, min(min(len, a.width * a.bs), first_pos + min(tokens, n - t0)));
  const int nblk = (keys + BN - 1) / BN;

  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) mbar_init(&sm->turn[g], 4);
    mbar_init(&sm->q_full, 128 * G);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm->k_full[s], 128); mbar_init(&sm->k_empty[s], 1);
      mbar_init(&sm->v_full[s], 128); mbar_init(&sm->v_empty[s], 1);
    }
    for (int g = 0; g < G; ++g) {
      for (int b = 0; b < 2; ++b) { mbar_init(&sm->s_full[g][b], 1); mbar_init(&sm->p_full[g][b], 128); }
      mbar_init(&sm->pv_done[g], 1);
    }
    fence_barrier_init();
  }
  if (warp == 4 * G + 4) {
    tmem_alloc(&sm->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = sm->tmem_base;

  if (warp >= 4 * G && warp < 4 * G + 4) {
    // ------------------------------------------------ dequantisation
    // thread: element chunk `col` (16 codes) of rows tid / CH + i * ROWS
    constexpr int CH = D / 16, ROWS = 128 / CH, N = BN / ROWS;
    const int tid = threadIdx.x - 128 * G, col = tid % CH, row = tid / CH;
    const int* table = a.tables + (int64_t)seq * a.width;
    const int64_t page_bytes = (int64_t)a.bs * D;
    constexpr int P = SMALL ? N : 1;                // pages of a thread's rows
    struct Ids { int page[P], id[P]; };             // their places in the table and what stands there, loaded two tiles ahead
    auto ids_of = [&](int j) {
      Ids x;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int tok = j * BN + (SMALL ? row + i * ROWS : 0);
        x.page[i] = tok / a.bs;
        x.id[i] = -1;
        if (tok < keys) x.id[i] = load_here(table + x.page[i]);
      }
      return x;
    };
    // addresses, scales and validity of the thread's rows of tile j
    struct Where { int64_t at[P]; float ks[P], vs[P]; uint32_t ok; };
    auto where = [&](int j, const Ids& x) {
      Where w;
      w.ok = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int tok = j * BN + (SMALL ? row + i * ROWS : 0);
        const bool ok = (uint32_t)x.id[i] < (uint32_t)a.pages;
        const int ph = ok ? x.id[i] * a.nkv + kvh : 0;
        w.at[i] = ph * page_bytes + (int64_t)(tok - x.page[i] * a.bs) * D + col * 16;
        w.ks[i] = w.vs[i] = 0.f;
        if (ok) {
          w.ks[i] = load_here(a.ks + ph);
          w.vs[i] = load_here(a.vs + ph);
        }
        if constexpr (SMALL) {
          w.ok |= (ok ? 1u : 0u) << i;
        } else if (ok) {
#pragma unroll
          for (int y = 0; y < N; ++y) w.ok |= (tok + row + y * ROWS < keys ? 1u : 0u) << y;
        }
      }
      return w;
    };
    // the thread's pieces of a tile on their way to shared memory: registers would have to be waited for at the end of the
    // iteration, where they change names
    auto fetch = [&](uint4* raw, const uint8_t* from, const Where& w) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint8_t* at = from + (SMALL ? w.at[SMALL ? i : 0] : w.at[0] + (row + i * ROWS) * D);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(raw + i * 128 + tid)), "l"(at), "r"((w.ok >> i & 1) * 16) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto all = [&](bool x) {                        // whether it holds for all 128 threads
      uint32_t y;
      asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.and.pred q, 1, 128, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(y) : "r"((uint32_t)x) : "memory");
      return y != 0;
    };
    auto put = [&](uint8_t (*to)[kChunk], const uint4* raw, const float* scale, float ref, bool bf, auto values) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = row + i * ROWS;
        uint32_t h[8];
        uint4 x = raw[i * 128 + tid];
        if (!SMALL && decltype(values)::value && !(ref > 0.f)) x = make_uint4(0, 0, 0, 0);     // an empty scale: zeros, whatever the codes are
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) e4m3x4_to_half2(w[e], h[2 * e], h[2 * e + 1]);
        if (SMALL && decltype(values)::value && bf) {                // bf16 values
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale[i], f.y * scale[i]);
            h[e] = *reinterpret_cast<const uint32_t*>(&b);
          }
        } else if constexpr (SMALL && decltype(values)::value) {     // codes under the tile's largest scale
          const __half2 f = __float2half2_rn(ref > 0.f ? scale[i] / ref : 0.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] = half2_mul(h[e], f);
        }
        uint8_t* box = to[col / 4] + at * 128;
        const int c = col % 4 * 2;
        // the chunks of the second 64 elements in the other order: 8 neighbours then store to 8 different chunks of a row
        const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
        const int odd = col >> 2 & 1;
        *reinterpret_cast<uint4*>(box + (((c + odd) ^ (at & 7)) << 4)) = odd ? hi : lo;
        *reinterpret_cast<uint4*>(box + (((c + 1 - odd) ^ (at & 7)) << 4)) = odd ? lo : hi;
      }
    };
    bool ok = true;
    Where w = {};
    Ids ids = {};
    if (nblk > 0) {
      w = where(0, ids_of(0));
      ids = ids_of(1);
      fetch(sm->raw[0], a.kc, w);
      fetch(sm->raw[1], a.vc, w);
    }
    for (int j = 0; j < nblk; ++j) {
      const uint32_t stage = j % kStages, phase = (j / kStages) & 1;
      const Where next = where(j + 1, ids);
      ids = ids_of(j + 2);
      float ref_v = w.vs[0];
      bool bf = false;
      if constexpr (SMALL) {
        float low = INFINITY;                      // smallest V scale of the tile
#pragma unroll
        for (int i = 0; i < N; ++i) {
          ref_v = fmaxf(ref_v, w.vs[i]);
          if (w.vs[i] > 0.f) low = fminf(low, w.vs[i]);
        }
        // (order of numbers from 0 on: that of their bits)
        ref_v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(ref_v, 0.f))));
        low = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(low)));
        if (lane == 0) {
          sm->red[0][warp - 4 * G] = ref_v;
          sm->red[1][warp - 4 * G] = low;
        }
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
        const float (&r)[2][4] = sm->red;
        ref_v = fmaxf(fmaxf(r[0][0], r[0][1]), fmaxf(r[0][2], r[0][3]));
        low = fminf(fminf(r[1][0], r[1][1]), fminf(r[1][2], r[1][3]));
        bf = low < ref_v * 0x1p-8f;
        if (bf) ref_v = 1.f;
      }
      ok = mbar_wait(&sm->k_empty[stage], phase ^ 1) && ok;
      TileInfo& info = sm->info[j % kInfo];
      if (tid < 2) info.seen[tid] = SMALL || (w.ok & 1u) ? 0xffffffffu : 0u;
      if constexpr (SMALL) {
        if (col == 0)
#pragma unroll
          for (int i = 0; i < N; ++i)
            if ((row + i * ROWS) % 16 == 0) reinterpret_cast<float*>(&sm->ks[j % kInfo])[(row + i * ROWS) / 16] = w.ks[i];
      }
      if (tid == 0) {
        info.ks = w.ks[0];
        info.vs = ref_v;
        info.log2_vs = log2f(ref_v);
        info.per_vs = 1.f / ref_v;
        info.bf = bf;
      }
      if constexpr (SMALL) {
        ok = all(ok);                              // the waits of all ran out, or of none: everybody leaves together
        if (!ok) break;
        if (col == 0 && w.ok != (1u << N) - 1u) {  // keys without a page
          uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (!(w.ok >> i & 1)) bits[(row + i * ROWS) >> 5] &= ~(1u << ((row + i * ROWS) & 31));
          atomicAnd(&info.seen[0], bits[0]);
          atomicAnd(&info.seen[1], bits[1]);
        }
      } else if (!ok) {
        break;
      }
      put(sm->k[stage], sm->raw[0], w.ks, 1.f, false, std::false_type{});
      fence_proxy_async();
      mbar_arrive(&sm->k_full[stage]);
      fetch(sm->raw[0], a.kc, next);
      ok = mbar_wait(&sm->v_empty[stage], phase ^ 1);
      put(sm->v[stage], sm->raw[1], w.vs, ref_v, bf, std::true_type{});
      fence_proxy_async();
      mbar_arrive(&sm->v_full[stage]);
      fetch(sm->raw[1], a.vc, next);
      w = next;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!ok) atomicCAS(&g_q8_status, ST_OK, ST_CONVERT);
  } else if (warp == 4 * G + 4) {
    // ------------------------------------------------ MMA issuer
    if (nblk > 0 && elect_one()) {
      constexpr uint32_t idesc_qk = idesc_of(BM, BN, 0, 0), idesc_pv_half = idesc_of(BM, D, 1, 0), idesc_pv_bf = idesc_of(BM, D, 1, 1);
      bool ok = mbar_wait(&sm->q_full, 0);
      tc_fence_after_sync();
      // O += P(i) V(i) is issued one tile behind the scores: the tensor core has the next S = Q K^T to run while the
      // softmax warps turn tile i into P
      auto issue_pv = [&](int i) -> bool {
        const uint32_t st = i % kStages, ph = (i / kStages) & 1;
        if (!mbar_wait(&sm->v_full[st], ph)) return false;
        const bool bf = SMALL && sm->info[i % kInfo].bf;
        const uint32_t idesc_pv = bf ? idesc_pv_bf : idesc_pv_half;
        const uint64_t dv = make_mnmajor_sw128_desc(smem_u32(sm->v[st][0]), kChunk);
        for (int g = 0; g < G; ++g) {
          if (!mbar_wait(&sm->p_full[g][i & 1], (i >> 1) & 1)) return false;
          tc_fence_after_sync();
          const uint32_t base = tmem_base + g * kGroupCols, p_tmem = base + (i & 1) * BN;
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk) {
            const uint32_t p = p_tmem + (bf ? 32 * (kk >> 1) + 8 * (kk & 1) : 8 * kk);
            umma_ts(base + kOCol, p, dv + 128ull * kk, idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
            if (bf) umma_ts(base + kOCol, p + 16, dv + 128ull * kk, idesc_pv, 1u);
          }
          umma_commit(&sm->pv_done[g]);
        }
        umma_commit(&sm->v_empty[st]);
        return true;
      };
      for (int j = 0; j < nblk && ok; ++j) {
        const uint32_t st = j % kStages, ph = (j / kStages) & 1, b = j & 1;
        if (!mbar_wait(&sm->k_full[st], ph)) { ok = false; break; }
        for (int g = 0; g < G && ok; ++g) {
          if (j > 1 && !mbar_wait(&sm->pv_done[g], j & 1)) { ok = false; break; }      // P(j - 2) lies where S(j) goes
          tc_fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t dq = make_kmajor_sw128_desc(smem_u32(sm->q[g][kk >> 2])) + 2ull * (kk & 3);
            const uint64_t dk = make_kmajor_sw128_desc(smem_u32(sm->k[st][kk >> 2])) + 2ull * (kk & 3);
            umma_bf16(tmem_base + g * kGroupCols + b * BN, dq, dk, idesc_qk, kk > 0 ? 1u : 0u);
          }
          umma_commit(&sm->s_full[g][b]);
        }
        if (!ok) break;
        umma_commit(&sm->k_empty[st]);
        if (j > 0 && !issue_pv(j - 1)) { ok = false; break; }
      }
      if (ok) ok = issue_pv(nblk - 1);
      if (!ok) atomicCAS(&g_q8_status, ST_OK, ST_MMA);
    }
  } else {
    // ------------------------------------------------ softmax and epilogue: thread = query row
    const int g = warp >> 2, row = (warp & 3) * 32 + lane, tok = threadIdx.x / rep, hr = threadIdx.x - tok * rep;
    const bool real = tok < tokens && t0 + tok < n && row0 + t0 + tok < a.T;
    const int last = real ? min(first_pos + tok, keys - 1) : -1;     // last visible key
    // the row as fp16, its largest in [2^10, 2^11); the sign of the softmax scale goes with it
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + (real ? (row0 + t0 + tok) * a.q_row + (int64_t)(kvh * rep + hr) * D : 0);
    float big = 0.f;
    if (real)
#pragma unroll 8
      for (int c = 0; c < D; c += 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(q + c);
        const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&u);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(to_float(x[e])));
      }
    const int e2 = big > 0.f ? min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 120) : 0;
    const float up = copysignf(__uint_as_float((uint32_t)(127 + 10 - e2) << 23), a.scale);
    const float sc = fabsf(a.scale) * __uint_as_float((uint32_t)(127 - 10 + e2) << 23);
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (real) u = *reinterpret_cast<const uint4*>(q + c * 8);
      const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&u);
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = half2_bits(to_float(x[2 * e]) * up, to_float(x[2 * e + 1]) * up);
      *reinterpret_cast<uint4*>(sm->q[g][c >> 3] + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    fence_proxy_async();
    mbar_arrive(&sm->q_full);

    const uint32_t lane_addr = tmem_base + g * kGroupCols + ((uint32_t)((warp & 3) * 32) << 16);
    float m = -INFINITY, l = 0.f, unit = 0.f, per_unit = 0.f, log2_unit = 0.f;
    bool ok = true, far = false;                            // far: a row of the warp has a maximum of kFarScore or more
    // a tile; false: it has to be done again, as the maximum turned out to be far (or a wait ran out)
    auto take = [&](int j, auto from_far) {
      const uint32_t b = j & 1;
      if (!mbar_wait(&sm->s_full[g][b], (j >> 1) & 1)) return ok = false;
      tc_fence_after_sync();
      const TileInfo info = sm->info[j % kInfo];
      const int k0 = j * BN;
      // keys behind the row's own position, and keys without a page
      uint32_t see[2] = {0xffffffffu, 0xffffffffu};
      const bool partly = k0 + BN - 1 > last || (info.seen[0] & info.seen[1]) != 0xffffffffu;
      if (partly) {
        const int room = last - k0;                         // keys 0 .. room of the tile are at or before it
        see[0] = (room >= 31 ? 0xffffffffu : room < 0 ? 0u : (2u << room) - 1u) & info.seen[0];
        see[1] = (room >= 63 ? 0xffffffffu : room < 32 ? 0u : (2u << (room - 32)) - 1u) & info.seen[1];
      }
      // 32 scores at a time.  With one group they are read twice, for the maximum and for P: two CTAs leave a thread 96
      // registers, too few for 64 scores beside the addresses (a spill of 30 loads a tile)
      auto scores = [&](int half, uint32_t (&s)[32]) {
        tmem_ld_32x32(lane_addr + b * BN + 32 * half, s);
        tmem_ld_wait();
        if (partly) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see[half] >> i & 1)) s[i] = 0xff800000u;
        }
      };
      constexpr int NF = SMALL ? 4 : 1;
      float f[NF];                                          // scales of the scores; above 0: masked ones stay -inf at a softmax scale of 0 too
      if constexpr (SMALL) {
        const float4 ks = sm->ks[j % kInfo];
        f[0] = fmaxf(sc * ks.x, 1e-37f); f[1] = fmaxf(sc * ks.y, 1e-37f); f[2] = fmaxf(sc * ks.z, 1e-37f); f[3] = fmaxf(sc * ks.w, 1e-37f);
      }
      uint32_t kept[2][G == 2 ? 32 : 1];
      float mx = -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t s[32];
        scores(half, s);
        if constexpr (G == 2) {
#pragma unroll
          for (int i = 0; i < 32; ++i) kept[half][i] = s[i];
        }
        // four chains: one is bound by its instructions' latency (SMALL: 0 and 1 the first 16 keys, 2 and 3 the others)
        float top[4] = {SMALL ? -INFINITY : mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float& t = top[SMALL ? i >> 4 << 1 | (i >> 1 & 1) : i >> 1 & 3];
          t = max3(t, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        }
        if constexpr (SMALL) mx = max3(mx, fmaxf(top[0], top[1]) * f[2 * half], fmaxf(top[2], top[3]) * f[2 * half + 1]);
        else mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      }
      if constexpr (!SMALL) {
        f[0] = fmaxf(sc * info.ks, 1e-37f);
        mx *= f[0];
      }
      // units of the tile's P V: O's own, where the scales are near enough
      float change = 1.f, shift = 0.f, back = 1.f;
      if (info.vs > 0.f) {
        const float ratio = info.vs * per_unit;
        if (ratio <= 1.f && ratio >= 0.0625f) {
          shift = info.log2_vs - log2_unit;
          back = unit * info.per_vs;
        } else {
          change = unit * info.per_vs;
          unit = info.vs;
          per_unit = info.per_vs;
          log2_unit = info.log2_vs;
        }
      }
      const bool need = mx > m + kRescale;                  // the first visible key's too
      const bool rescale = change != 1.f || __any_sync(0xffffffffu, need);
      // O must be at rest before it is rescaled.  The barrier is in the phase of P(j - 1) V(j - 1) or behind it: S(j) was
      // issued after P(j - 2) V(j - 2) was done, and P(j) is not given yet.  The last tile waits too, so that the wait after
      // the loop finds it one phase on.
      if (j > 0 && (rescale || j == nblk - 1) && !mbar_wait(&sm->pv_done[g], (j - 1) & 1)) return ok = false;
      if (rescale) {
        const float alpha = need ? exp2_approx(m - mx) : 1.f;
        if (need) m = mx;
        far = __any_sync(0xffffffffu, fabsf(m) >= kFarScore && m != -INFINITY);
        l *= alpha;
        const float by = alpha * change;
        tc_fence_after_sync();
#pragma unroll 1
        for (int cc = 0; cc < (j > 0 ? D : 0); cc += 32) {
          uint32_t o[32];
          tmem_ld_32x32(lane_addr + kOCol + cc, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
          tmem_st_32x32(lane_addr + kOCol + cc, o);
        }
        tmem_st_wait();
        if (far && !decltype(from_far)::value) return false;
      }
      const float base = m == -INFINITY ? 0.f : m, off = m == -INFINITY ? 0.f : kShift - m + shift;
      if (G == 2 && (g == 1 || j > 0) && !mbar_wait(&sm->turn[g], (j + g - 1) & 1)) return ok = false;
      float2 sum2[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t s[32], w[16];
        if constexpr (G == 2) {
#pragma unroll
          for (int i = 0; i < 32; ++i) s[i] = kept[half][i];
        } else {
          scores(half, s);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float by = f[NF == 4 ? 2 * half + (i >> 3) : 0], s0 = __uint_as_float(s[2 * i]), s1 = __uint_as_float(s[2 * i + 1]);
          float2 y;
          if constexpr (decltype(from_far)::value)
            y = {__fadd_rn(__fmul_rn(s0, by), -base) + (kShift + shift), __fadd_rn(__fmul_rn(s1, by), -base) + (kShift + shift)};
          else
            y = fma2({s0, s1}, {by, by}, {off, off});
          const float p0 = exp2_approx(y.x), p1 = exp2_approx(y.y);
          sum2[i & 1] = add2(sum2[i & 1], {p0, p1});
          s[2 * i] = __float_as_uint(p0);
          s[2 * i + 1] = __float_as_uint(p1);
        }
        // over scores that are in registers already
        if (SMALL && info.bf) {                             // P and what its rounding leaves, side by side
          uint32_t rest[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p0 = __uint_as_float(s[2 * i]), p1 = __uint_as_float(s[2 * i + 1]);
            const __nv_bfloat162 x = __floats2bfloat162_rn(p0, p1);
            const __nv_bfloat162 y = __floats2bfloat162_rn(p0 - __low2float(x), p1 - __high2float(x));
            w[i] = *reinterpret_cast<const uint32_t*>(&x);
            rest[i] = *reinterpret_cast<const uint32_t*>(&y);
          }
          tmem_st_32x16(lane_addr + b * BN + 32 * half, w);
          tmem_st_32x16(lane_addr + b * BN + 32 * half + 16, rest);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = half2_bits(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
          tmem_st_32x16(lane_addr + b * BN + 16 * half, w);
        }
      }
      if (G == 2) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm->turn[g ^ 1]);
      }
      const float sum = sum2[0].x + sum2[0].y + (sum2[1].x + sum2[1].y);
      l = fmaf(sum, back, l);
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&sm->p_full[g][b]);
      return true;
    };
    for (int j = 0; j < nblk && ok;) j += far ? take(j, std::true_type{}) : take(j, std::false_type{});
    if (ok && nblk > 0 && !mbar_wait(&sm->pv_done[g], (nblk - 1) & 1)) ok = false;
    if (ok) {
      tc_fence_after_sync();
      const float inv = l == 0.f ? 0.f : unit / l;
      // through the Q tile (no product reads it any more; without keys, when other warps may still be writing it, there is
      // nothing to stage): 16-byte chunk c of row r at chunk c ^ (r % CH), free of bank
      // conflicts row by row and in row segments
      constexpr int CH = D / 8;
      uint8_t* stage = sm->q[g][0];
#pragma unroll 1
      for (int cc = 0; cc < (nblk > 0 ? D : 0); cc += 32) {
        uint32_t o[32];
        tmem_ld_32x32(lane_addr + kOCol + cc, o);
        tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          __nv_bfloat16 w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = from_float<__nv_bfloat16>(inv == 0.f ? 0.f : __uint_as_float(o[x * 8 + i]) * inv);
          *reinterpret_cast<uint4*>(stage + row * D * 2 + (((cc / 8 + x) ^ (row & (CH - 1))) << 4)) = *reinterpret_cast<const uint4*>(w);
        }
      }
      __syncwarp();
      constexpr int RW = 256 / D;                           // rows that the warp writes at a time (D = 256: one)
#pragma unroll 1
      for (int i = 0; i < 32 / RW; ++i) {
        const int r = (warp & 3) * 32 + i * RW + lane / CH, chunk = lane % CH, all = g * BM + r, tk = all / rep;
        if (tk < tokens && t0 + tk < n && row0 + t0 + tk < a.T) {
          uint4 val = make_uint4(0, 0, 0, 0);
          if (nblk > 0) val = *reinterpret_cast<const uint4*>(stage + r * D * 2 + ((chunk ^ (r & (CH - 1))) << 4));
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + ((int64_t)(row0 + t0 + tk) * a.nq + kvh * rep + (all - tk * rep)) * D + chunk * 8) = val;
        }
      }
    }
    if (!ok && lane == 0) atomicCAS(&g_q8_status, ST_OK, ST_SOFTMAX);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 4 * G + 4) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D, bool SMALL, int G>
void launch(const ChunkArgs& a, int dev, cudaStream_t st) {
  static std::atomic<bool> ready[64] = {};
  if (!ready[dev].load()) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(chunk_q8_kernel<D, SMALL, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D, G>)));
    C10_CUDA_CHECK(cudaFuncSetAttribute(chunk_q8_kernel<D, SMALL, G>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                        (int)cudaSharedmemCarveoutMaxShared));
    ready[dev].store(true);
  }
  const int tokens = G * BM / (a.nq / a.nkv);
  const int64_t tiles = std::min<int64_t>(a.T / tokens + a.B, a.T / std::max(a.min_new, 1) + a.T / tokens);
  if (tiles > 0)
    C10_CUDA_CHECK(launch_pdl(chunk_q8_kernel<D, SMALL, G>, dim3((unsigned)tiles, a.nkv), dim3(128 * G + 160), sizeof(Smem<D, G>), st, a));
}

template <int D, bool SMALL>
void launch_rows(const ChunkArgs& a, bool wide, int dev, cudaStream_t st) {
  wide ? launch<D, SMALL, 2>(a, dev, st) : launch<D, SMALL, 1>(a, dev, st);
}

}  // namespace

bool q8::chunk_supported(int rep) { return rep <= BM; }

void q8::launch_chunk(const ChunkArgs& a, int D, int dev, cudaStream_t st) {
  TORCH_CHECK(dev >= 0 && dev < 64, "paged_attention_q8: device index out of range");
  const bool small = a.bs % BN != 0;
  // two groups of rows where the sequences have more than one on average.  A CTA of two takes 1.5 times as long as the two
  // of one that an SM holds: 32 sequences of 32 / 48 / 64 / 128 new tokens (4 heads to a kv head: 128 to 512 rows) after
  // 4,000 take 120 / 225 / 220 / 411 us with one group, 185 / 182 / 187 / 355 us with two; 320 rows 323 and 355 us
  const bool wide = (int64_t)a.T * (a.nq / a.nkv) * 4 >= (int64_t)a.B * 5 * BM;
  if (D == 64) small ? launch_rows<64, true>(a, wide, dev, st) : launch_rows<64, false>(a, wide, dev, st);
  else if (D == 128) small ? launch_rows<128, true>(a, wide, dev, st) : launch_rows<128, false>(a, wide, dev, st);
  else small ? launch<256, true, 1>(a, dev, st) : launch<256, false, 1>(a, dev, st);
}

int64_t paged_attention_q8_last_status() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_q8_status, sizeof(int));
  cudaMemcpyToSymbol(g_q8_status, &zero, sizeof(int));
  return v;
}
