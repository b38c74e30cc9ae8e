// Attention of many new tokens per sequence over the paged 8-bit cache, on the 5th-generation tensor cores.
//
// Continuation chunks of a prefill attend over everything cached before them: with hundreds of new tokens per sequence
// the two products bound the work, not the cache's bytes.  A CTA owns 128 query rows of one sequence and one kv head:
// 128 / rep tokens times the rep query heads that share the head, so a cached tile is dequantised once for all of them.
// Warps:
//   0..3  softmax, thread = query row: first the row itself, rescaled by a power of two to fp16, into shared memory;
//         then per tile of 64 keys the scores out of tensor memory, running maximum (lazily applied, as soon as it has
//         run ahead by 2^8) and sum, P as fp16 into shared memory; at the end O / l to the output
//   4..7  dequantisation: e4m3 codes from the pages to fp16 tiles (exact) in the 128-byte swizzle, one tile ahead in
//         registers.  Pages of a multiple of 64 tokens keep their scales out of the tiles (S and P take them).  Of other
//         pages a tile holds several: K is brought to the largest of its scales (what that loses is 2^-34 of the tile's
//         largest keys), V becomes bf16 values (exact) and P bf16, as fp16 has not the range for scales far apart.
//   8     one thread issues S = Q K^T (128x64x16) into one of two S accumulators and O += P V (128xDx16, V as an
//         MN-major operand straight from its row-major tile)
// O is kept in units of a V scale that follows the tiles' scales where they are far apart (as in the decode kernel).
// The queries are causal inside their sequence's new tokens.  Every mbarrier wait is bounded; one that runs out records a
// status, the CTA drains and frees its tensor memory.
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

constexpr int BM = 128, BN = 64, kStages = 2, kThreads = 288, kInfo = 8;
constexpr uint32_t kChunk = BN * 128;             // 64 keys x 64 elements of fp16
constexpr float kRescale = 8.f;                   // bits that the maximum may run ahead
constexpr float kShift = 7.f;                     // P times 2^7: at most 2^15, and normal down to 2^-21 of a row's largest

struct TileInfo { float ks, vs; uint32_t seen[2]; };      // scales of the tile, keys that exist

template <int D>
struct Smem {
  uint8_t q[D / 64][BM * 128];
  uint8_t k[kStages][D / 64][kChunk];
  uint8_t v[kStages][D / 64][kChunk];
  uint8_t p[BM * 128];
  TileInfo info[kInfo];
  float red[4];
  uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], s_empty[2], p_full, pv_done;
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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
template <int D, bool SMALL>
__global__ void __launch_bounds__(kThreads, D == 256 ? 1 : 2) chunk_q8_kernel(const ChunkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  Smem<D>* sm = reinterpret_cast<Smem<D>*>(smem_raw);
  constexpr int kTmemCols = D == 256 ? 512 : 256, kOCol = 2 * BN;
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int rep = a.nq / a.nkv, tokens = BM / rep;         // tokens of a tile

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
    mbar_init(&sm->q_full, 128);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm->k_full[s], 128); mbar_init(&sm->k_empty[s], 1);
      mbar_init(&sm->v_full[s], 128); mbar_init(&sm->v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) { mbar_init(&sm->s_full[b], 1); mbar_init(&sm->s_empty[b], 4); }
    mbar_init(&sm->p_full, 128);
    mbar_init(&sm->pv_done, 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(&sm->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = sm->tmem_base;

  if (warp >= 4 && warp < 8) {
    // ------------------------------------------------ dequantisation
    // thread: element chunk `col` (16 codes) of rows tid / CH + i * ROWS
    constexpr int CH = D / 16, ROWS = 128 / CH, N = BN / ROWS;
    const int tid = threadIdx.x - 128, col = tid % CH, row = tid / CH;
    const int* table = a.tables + (int64_t)seq * a.width;
    const int64_t page_bytes = (int64_t)a.bs * D;
    struct Raw { uint4 x[N]; };
    constexpr int P = SMALL ? N : 1;                // pages of a thread's rows
    struct Ids { int page[P], id[P]; };             // their places in the table and what stands there, loaded two tiles ahead
    auto ids_of = [&](int j) {
      Ids x;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int tok = j * BN + (SMALL ? row + i * ROWS : 0);
        x.page[i] = tok / a.bs;
        x.id[i] = tok < keys ? table[x.page[i]] : -1;
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
        w.ks[i] = ok ? a.ks[ph] : 0.f;
        w.vs[i] = ok ? a.vs[ph] : 0.f;
        if constexpr (SMALL) {
          w.ok |= (ok ? 1u : 0u) << i;
        } else if (ok) {
#pragma unroll
          for (int y = 0; y < N; ++y) w.ok |= (tok + row + y * ROWS < keys ? 1u : 0u) << y;
        }
      }
      return w;
    };
    auto fetch = [&](const uint8_t* from, const Where& w) {
      Raw r;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        r.x[i] = make_uint4(0, 0, 0, 0);
        if (w.ok >> i & 1) r.x[i] = __ldg(reinterpret_cast<const uint4*>(from + (SMALL ? w.at[SMALL ? i : 0] : w.at[0] + (row + i * ROWS) * D)));
      }
      return r;
    };
    auto all = [&](bool x) {                        // whether it holds for all 128 threads
      uint32_t y;
      asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.and.pred q, 1, 128, p;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(y) : "r"((uint32_t)x) : "memory");
      return y != 0;
    };
    auto put = [&](uint8_t (*to)[kChunk], const Raw& r, const float* scale, float ref, auto values) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = row + i * ROWS;
        uint32_t h[8];
        const uint32_t w[4] = {r.x[i].x, r.x[i].y, r.x[i].z, r.x[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) e4m3x4_to_half2(w[e], h[2 * e], h[2 * e + 1]);
        if constexpr (SMALL && decltype(values)::value) {            // V: bf16 values
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale[i], f.y * scale[i]);
            h[e] = *reinterpret_cast<const uint32_t*>(&b);
          }
        } else if constexpr (SMALL) {                                // K: codes under the tile's largest scale
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
    Raw rk = {}, rv = {};
    if (nblk > 0) {
      w = where(0, ids_of(0));
      ids = ids_of(1);
      rk = fetch(a.kc, w);
      rv = fetch(a.vc, w);
    }
    for (int j = 0; j < nblk; ++j) {
      const uint32_t stage = j % kStages, phase = (j / kStages) & 1;
      const Where next = where(j + 1, ids);
      ids = ids_of(j + 2);
      float ref_k = w.ks[0];
      const float ref_v = SMALL ? 1.f : w.vs[0];
      if constexpr (SMALL) {
#pragma unroll
        for (int i = 1; i < N; ++i) ref_k = fmaxf(ref_k, w.ks[i]);
        ref_k = warp_max(ref_k);
        if (lane == 0) sm->red[warp - 4] = ref_k;
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
        ref_k = fmaxf(fmaxf(sm->red[0], sm->red[1]), fmaxf(sm->red[2], sm->red[3]));
      }
      ok = mbar_wait(&sm->k_empty[stage], phase ^ 1) && ok;
      TileInfo& info = sm->info[j % kInfo];
      if (tid < 2) info.seen[tid] = 0u;
      if (tid == 0) { info.ks = ref_k; info.vs = ref_v; }
      ok = all(ok);                                // the waits of all ran out, or of none: everybody leaves together
      if (!ok) break;
      if (col == 0) {                              // keys that exist: a bit for each row
        uint32_t bits[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (w.ok >> i & 1) bits[(row + i * ROWS) >> 5] |= 1u << ((row + i * ROWS) & 31);
        atomicOr(&info.seen[0], bits[0]);
        atomicOr(&info.seen[1], bits[1]);
      }
      put(sm->k[stage], rk, w.ks, ref_k, std::false_type{});
      fence_proxy_async();
      mbar_arrive(&sm->k_full[stage]);
      rk = fetch(a.kc, next);
      ok = mbar_wait(&sm->v_empty[stage], phase ^ 1);
      if (!SMALL && !(ref_v > 0.f)) rv = Raw{};    // an empty scale: zeros, whatever the codes are
      put(sm->v[stage], rv, w.vs, ref_v, std::true_type{});
      fence_proxy_async();
      mbar_arrive(&sm->v_full[stage]);
      rv = fetch(a.vc, next);
      w = next;
    }
    if (!ok) atomicCAS(&g_q8_status, ST_OK, ST_CONVERT);
  } else if (warp == 8) {
    // ------------------------------------------------ MMA issuer
    if (lane == 0 && nblk > 0) {
      constexpr uint32_t idesc_qk = idesc_of(BM, BN, 0, 0), idesc_pv = idesc_of(BM, D, 1, SMALL);
      const uint32_t o_tmem = tmem_base + kOCol;
      bool ok = mbar_wait(&sm->q_full, 0);
      tc_fence_after_sync();
      // O += P(i) V(i) is issued one tile behind the scores: the tensor core has the next S = Q K^T to run while the
      // softmax warps turn tile i into P
      auto issue_pv = [&](int i) -> bool {
        const uint32_t st = i % kStages, ph = (i / kStages) & 1;
        if (!mbar_wait(&sm->v_full[st], ph)) return false;
        if (!mbar_wait(&sm->p_full, i & 1)) return false;
        tc_fence_after_sync();
        const uint64_t dp = make_kmajor_sw128_desc(smem_u32(sm->p));
        const uint64_t dv = make_mnmajor_sw128_desc(smem_u32(sm->v[st][0]), kChunk);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          umma_bf16(o_tmem, dp + 2ull * kk, dv + 128ull * kk, idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&sm->v_empty[st]);
        umma_commit(&sm->pv_done);
        return true;
      };
      for (int j = 0; j < nblk && ok; ++j) {
        const uint32_t st = j % kStages, ph = (j / kStages) & 1, b = j & 1;
        if (!mbar_wait(&sm->k_full[st], ph)) { ok = false; break; }
        if (!mbar_wait(&sm->s_empty[b], ((j >> 1) & 1) ^ 1)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t dq = make_kmajor_sw128_desc(smem_u32(sm->q[kk >> 2])) + 2ull * (kk & 3);
          const uint64_t dk = make_kmajor_sw128_desc(smem_u32(sm->k[st][kk >> 2])) + 2ull * (kk & 3);
          umma_bf16(tmem_base + b * BN, dq, dk, idesc_qk, kk > 0 ? 1u : 0u);
        }
        umma_commit(&sm->k_empty[st]);
        umma_commit(&sm->s_full[b]);
        if (j > 0 && !issue_pv(j - 1)) { ok = false; break; }
      }
      if (ok) ok = issue_pv(nblk - 1);
      if (!ok) atomicCAS(&g_q8_status, ST_OK, ST_MMA);
    }
  } else {
    // ------------------------------------------------ softmax and epilogue: thread = query row
    const int row = warp * 32 + lane, tok = row / rep, hr = row - tok * rep;
    const bool real = tok < tokens && t0 + tok < n && row0 + t0 + tok < a.T;
    const int last = real ? first_pos + tok : -1;          // last visible key
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
      *reinterpret_cast<uint4*>(sm->q[c >> 3] + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    fence_proxy_async();
    mbar_arrive(&sm->q_full);

    const uint32_t lane_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, l = 0.f, unit = 0.f, per_unit = 0.f;
    bool ok = true;
    for (int j = 0; j < nblk; ++j) {
      const uint32_t b = j & 1;
      if (!mbar_wait(&sm->s_full[b], (j >> 1) & 1)) { ok = false; break; }
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
      // the scores are read twice, 32 at a time, once for the maximum and once for P: 64 of them in registers all the
      // while were too many beside the addresses (a spill of 30 loads a tile)
      auto scores = [&](int half, uint32_t (&s)[32]) {
        tmem_ld_32x32(lane_addr + b * BN + 32 * half, s);
        tmem_ld_wait();
        if (partly) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see[half] >> i & 1)) s[i] = 0xff800000u;
        }
      };
      float mx = -INFINITY;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t s[32];
        scores(half, s);
#pragma unroll
        for (int i = 0; i < 32; ++i) mx = fmaxf(mx, __uint_as_float(s[i]));
      }
      const float f = fmaxf(sc * info.ks, 1e-37f);          // above 0: masked scores stay -inf at a softmax scale of 0 too
      mx *= f;
      // P(j-1) must have been consumed before the tile is overwritten, and O must be at rest before it is rescaled
      if (j > 0 && !mbar_wait(&sm->pv_done, (j - 1) & 1)) { ok = false; break; }
      float change = 1.f, ratio = info.vs > 0.f ? info.vs * per_unit : 1.f;
      if (!(ratio <= 1.f && ratio >= 0.0625f)) {
        change = unit / info.vs;
        unit = info.vs;
        per_unit = 1.f / unit;
        ratio = 1.f;
      }
      const bool need = mx > m + kRescale || (m == -INFINITY && mx > m);
      const float alpha = need ? exp2_approx(m - mx) : 1.f;
      if (need) { m = mx; l *= alpha; }
      if (j > 0 && (change != 1.f || __any_sync(0xffffffffu, need))) {
        tc_fence_after_sync();
        const float by = alpha * change;
#pragma unroll 1
        for (int cc = 0; cc < D; cc += 32) {
          uint32_t o[32];
          tmem_ld_32x32(lane_addr + kOCol + cc, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
          tmem_st_32x32(lane_addr + kOCol + cc, o);
        }
        tmem_st_wait();
      }
      float off = m == -INFINITY ? 0.f : kShift - m;
      if (ratio != 1.f) off += log2f(ratio);
      float sum = 0.f;
      uint8_t* prow = sm->p + row * 128;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t s[32];
        scores(half, s);
        if (half == 1) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm->s_empty[b]);      // the scores are in registers: the buffer may be overwritten
        }
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p0 = exp2_approx(fmaf(__uint_as_float(s[ch * 8 + 2 * i]), f, off));
            const float p1 = exp2_approx(fmaf(__uint_as_float(s[ch * 8 + 2 * i + 1]), f, off));
            sum += p0 + p1;
            if constexpr (SMALL) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(p0, p1);
              w[i] = *reinterpret_cast<const uint32_t*>(&x);
            } else {
              w[i] = half2_bits(p0, p1);
            }
          }
          *reinterpret_cast<uint4*>(prow + (((half * 4 + ch) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      l += ratio == 1.f ? sum : sum / ratio;
      fence_proxy_async();          // written through the generic proxy, read through the async one
      tc_fence_before_sync();
      mbar_arrive(&sm->p_full);
    }
    if (ok && nblk > 0 && !mbar_wait(&sm->pv_done, (nblk - 1) & 1)) ok = false;
    if (ok) {
      tc_fence_after_sync();
      const float inv = l == 0.f ? 0.f : unit / l;
      // through the Q tile (no product reads it any more): 16-byte chunk c of row r at chunk c ^ (r % CH), free of bank
      // conflicts row by row and in row segments
      constexpr int CH = D / 8;
      uint8_t* stage = sm->q[0];
#pragma unroll 1
      for (int cc = 0; cc < D; cc += 32) {
        uint32_t o[32];
        if (nblk > 0) {
          tmem_ld_32x32(lane_addr + kOCol + cc, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          __nv_bfloat16 w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = from_float<__nv_bfloat16>(inv == 0.f ? 0.f : __uint_as_float(o[g * 8 + i]) * inv);
          *reinterpret_cast<uint4*>(stage + row * D * 2 + (((cc / 8 + g) ^ (row & (CH - 1))) << 4)) = *reinterpret_cast<const uint4*>(w);
        }
      }
      __syncwarp();
      constexpr int RW = 256 / D;                           // rows that the warp writes at a time (D = 256: one)
#pragma unroll 1
      for (int i = 0; i < 32 / RW; ++i) {
        const int r = warp * 32 + i * RW + lane / CH, chunk = lane % CH, tk = r / rep;
        if (tk < tokens && t0 + tk < n && row0 + t0 + tk < a.T) {
          const uint4 val = *reinterpret_cast<const uint4*>(stage + r * D * 2 + ((chunk ^ (r & (CH - 1))) << 4));
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + ((int64_t)(row0 + t0 + tk) * a.nq + kvh * rep + (r - tk * rep)) * D + chunk * 8) = val;
        }
      }
    }
    if (!ok && lane == 0) atomicCAS(&g_q8_status, ST_OK, ST_SOFTMAX);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D, bool SMALL>
void launch(const ChunkArgs& a, int dev, cudaStream_t st) {
  static std::atomic<bool> ready[64] = {};
  if (!ready[dev].load()) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(chunk_q8_kernel<D, SMALL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D>)));
    C10_CUDA_CHECK(cudaFuncSetAttribute(chunk_q8_kernel<D, SMALL>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                        (int)cudaSharedmemCarveoutMaxShared));
    ready[dev].store(true);
  }
  const int tokens = BM / (a.nq / a.nkv);
  const int64_t tiles = std::min<int64_t>(a.T / tokens + a.B, a.T / std::max(a.min_new, 1) + a.T / tokens);
  if (tiles > 0)
    C10_CUDA_CHECK(launch_pdl(chunk_q8_kernel<D, SMALL>, dim3((unsigned)tiles, a.nkv), dim3(kThreads), sizeof(Smem<D>), st, a));
}

}  // namespace

bool q8::chunk_supported(int rep) { return rep <= BM; }

void q8::launch_chunk(const ChunkArgs& a, int D, int dev, cudaStream_t st) {
  TORCH_CHECK(dev >= 0 && dev < 64, "paged_attention_q8: device index out of range");
  const bool small = a.bs % BN != 0;
  if (D == 64) small ? launch<64, true>(a, dev, st) : launch<64, false>(a, dev, st);
  else if (D == 128) small ? launch<128, true>(a, dev, st) : launch<128, false>(a, dev, st);
  else small ? launch<256, true>(a, dev, st) : launch<256, false>(a, dev, st);
}

int64_t paged_attention_q8_last_status() {
  int v = 0, zero = 0;
  cudaMemcpyFromSymbol(&v, g_q8_status, sizeof(int));
  cudaMemcpyToSymbol(g_q8_status, &zero, sizeof(int));
  return v;
}
