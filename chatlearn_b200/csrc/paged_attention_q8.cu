// Attention over the paged key/value cache held in 8 bits (e4m3 codes, one power-of-two scale per page and kv head).
//
//   o = softmax(scale * q (s_k C_k)^T) (s_v C_v)
//
// One unit of work is (query row set, kv head): the query heads that share a kv head are the columns of m16n8k16 tiles
// whose rows are cached tokens (S^T = K Q^T) or head elements (O^T = V^T P^T), so that up to 8 heads waste nothing, each
// cached byte is read once per unit and dequantised once.  Codes become halves by one conversion (exact: e4m3 is a
// subset of fp16); the scales are powers of two and stay out of the products: s_k joins the softmax scale, s_v the
// probabilities.  (Products of e4m3 operands are no way around the conversions: mma.sync carries them out in halves.)
// Queries are rescaled per row by a power of two to 2^10..2^11, so that their fp16 form loses nothing that counts (bf16
// has 8 significant bits, fp16 11; what falls below 2^-24 of a row's largest is lost).
//
// The bytes of the cache bound it.  The tokens of all units form one line that is cut evenly over the resident blocks
// (whatever the lengths are), 64 at a time; a unit that a cut divides is written as partial (o, m, l) and joined by a
// second kernel.  The cut goes by the lengths alone, so results do not depend on timing.  Inside a block each warp owns
// 16 of the 64 tokens with its own cp.async ring, running maximum and sum: no barrier in the loop; the four streams meet
// at the end of a unit.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_pipeline.h>

#include <atomic>
#include <type_traits>

#include "q8.cuh"

using namespace cl;
using namespace q8;

namespace {

constexpr int kThreads = 128, kWarps = 4;
// tokens that a warp takes at a time: 8 KB of keys and values at head dims 128 and 256
__host__ __device__ constexpr int warp_tokens(int D) { return D >= 256 ? 16 : 32; }
__host__ __device__ constexpr int tile_tokens(int D) { return kWarps * warp_tokens(D); }
// probabilities are carried times 2^10: fp16 keeps 11 bits of them down to 2^-24 of the largest
constexpr float kProbShift = 10.f;

struct Args {
  const void* q;                 // [T, nq, D], row stride q_row
  int64_t q_row;
  const uint8_t *kc, *vc;        // [pages, nkv, bs, D]
  const float *ks, *vs;          // [pages, nkv]
  const int* tables;             // [B, width]
  const int* row_seq;            // [rows] sequence of a query row (null: the row's own number)
  const int* row_len;            // [rows] tokens it sees
  void* out;                     // [T, nq, D]
  float *part_o, *part_ml;       // [2 * grid, 16, D], [2 * grid, 16, 2]
  int rows, T, width, nq, nkv, bs;
  int pages;
  int grid;                      // blocks that the line is cut over
  int unit_rows;                 // query heads of a unit: 8 or 16
  float scale;                   // softmax scale times log2 e
};

template <int TILE>
__device__ __forceinline__ int tiles_of(const Args& a, int r) {
  const int len = min(a.row_len[r], a.width * a.bs);
  return len > 0 ? (len + TILE - 1) / TILE : 0;
}

// The line is cut into min(blocks, tiles) shares, the first ones a tile longer where it does not come out even: none is
// empty, and their bounds go by the lengths alone.
struct Place {
  int64_t total;                 // tiles of the line
  int shares, longer;            // shares, and how many of them have share + 1 tiles
  int64_t share;
  int64_t pos;                   // where share `index` begins (total, if there is no such share)
  int row;                       // row set that holds this position
  int64_t base;                  // where that row set begins
  __device__ __forceinline__ int64_t begin(int i) const { return i * share + min(i, longer); }
};

// Exclusive prefix sums over the rows' tiles, `per_row` units each.  All threads of the block take part.
template <int TILE>
__device__ Place locate(const Args& a, int per_row, int index, int64_t* sh) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.rows + kThreads - 1) / kThreads;
  const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  int64_t sum = 0;
  for (int r = r0; r < r1; ++r) sum += tiles_of<TILE>(a, r);
  sum *= per_row;
  int64_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t p = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += p;
  }
  if (lane == 31) sh[warp] = inc;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh[w];
    total += sh[w];
  }
  Place p;
  p.total = total;
  p.shares = (int)max((int64_t)1, min((int64_t)a.grid, total));
  if (total >> 31) {
    p.share = total / p.shares;
    p.longer = (int)(total - p.share * p.shares);
  } else {
    p.share = (uint32_t)total / (uint32_t)p.shares;
    p.longer = (int)((uint32_t)total - (uint32_t)p.share * p.shares);
  }
  p.pos = index < p.shares ? p.begin(index) : total;
  const int64_t first = before + inc - sum;
  if (first <= p.pos && p.pos < first + sum) {
    int64_t at = first;
    int r = r0;
    for (; r < r1; ++r) {
      const int64_t n = (int64_t)tiles_of<TILE>(a, r) * per_row;
      if (p.pos < at + n) break;
      at += n;
    }
    sh[4] = r;
    sh[5] = at;
  }
  __syncthreads();
  p.row = (int)sh[4];
  p.base = sh[5];
  return p;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// lane (g, t) gives elements 2 t, 2 t + 1 of row g of an 8 x 8 matrix of halves and gets those of column g
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16-byte chunk of a row after the swizzle that keeps both reads below free of bank conflicts: eight lanes that read in
// one phase are two neighbouring rows x four chunks (keys), or rows 0, 2, 4, 6 x the chunks c and c + 4 (values)
template <int D>
__device__ __forceinline__ int swizzled(int r, int chunk) {
  if (D >= 128) return chunk ^ (((r & 1) << 2) | ((r >> 1) & 3));
  return chunk ^ ((r >> 1) & 3);
}

// A warp's position on the line: row set, kv head and row tile of it, tile; the page that holds the warp's first token.
template <int TILE, int WT>
struct Cursor {
  int row, head, rt, tile, tiles, len;
  int page, off;                                 // number in the sequence's table, token inside the page
  int step_page, step_off;                       // of a tile
  const int* table;
  __device__ __forceinline__ int token(int warp) const { return tile * TILE + warp * WT; }
  __device__ __forceinline__ void rewind(const Args& a, int warp) {
    page = token(warp) / a.bs;
    off = token(warp) - page * a.bs;
  }
  __device__ __forceinline__ void enter(const Args& a, int r) {
    row = r;
    tiles = 0;
    while (row < a.rows && (tiles = tiles_of<TILE>(a, row)) == 0) ++row;
    if (row >= a.rows) return;
    len = min(a.row_len[row], a.width * a.bs);
    table = a.tables + (int64_t)(a.row_seq ? a.row_seq[row] : row) * a.width;
  }
  __device__ __forceinline__ void next(const Args& a, int row_tiles, int warp) {
    if (++tile < tiles) {
      page += step_page;
      off += step_off;
      if (off >= a.bs) { off -= a.bs; ++page; }
      return;
    }
    tile = 0;
    rewind(a, warp);
    if (++rt < row_tiles) return;
    rt = 0;
    if (++head < a.nkv) return;
    head = 0;
    enter(a, row + 1);
  }
};

template <int D, int ST>
struct WarpRing {
  uint8_t k[ST][warp_tokens(D) * D];
  uint8_t v[ST][warp_tokens(D) * D];
  float s[ST][4];                                // scales of the 16-token halves: K, V, K, V
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {       // the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// H: 1 for units of at most 8 rows, 2 for up to 16.  PG: pages that a warp's tokens can lie in (2: 32 tokens, page length
// no multiple of 32).
template <typename T, int D, int ST, int H, int PG>
__global__ void __launch_bounds__(kThreads)
paged_q8_kernel(const Args a) {
  constexpr int WT = warp_tokens(D), TILE = tile_tokens(D), PIECES = WT / 16, PT = WT / PG;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t sh_place[8];
  __shared__ float sh_m[kWarps][16], sh_l[kWarps][16];
  pdl_wait();
  pdl_trigger();                                   // after the wait: the joining kernel reads the lengths before its own
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  auto& ring = reinterpret_cast<WarpRing<D, ST>*>(smem)[warp];
  float* red = reinterpret_cast<float*>(smem + sizeof(WarpRing<D, ST>) * kWarps);   // [2][rows of a unit][D]
  const int rep = a.nq / a.nkv, row_tiles = (rep + 8 * H - 1) / (8 * H), per_row = a.nkv * row_tiles, red_rows = min(rep, 8 * H);
  T* out = static_cast<T*>(a.out);

  const Place place = locate<TILE>(a, per_row, blockIdx.x, sh_place);
  const int64_t pos = place.pos;
  // rows that see nothing are zero
  for (int r = blockIdx.x * kWarps + warp; r < a.T; r += gridDim.x * kWarps)
    if (r >= a.rows || tiles_of<TILE>(a, r) == 0)
      for (int i = lane * 8; i < a.nq * D; i += 256) *reinterpret_cast<uint4*>(&out[(int64_t)r * a.nq * D + i]) = make_uint4(0, 0, 0, 0);
  if (pos >= place.total) return;
  int left = (int)(place.begin(blockIdx.x + 1) - pos), left_load = left;
  Cursor<TILE, WT> use;
  use.step_page = TILE / a.bs;
  use.step_off = TILE % a.bs;
  use.enter(a, place.row);
  {
    const uint32_t in_row = (uint32_t)(pos - place.base);        // a row set has less than 2^31 tiles
    const int unit = (int)(in_row / (uint32_t)use.tiles);
    use.tile = (int)in_row - unit * use.tiles;
    use.head = unit / row_tiles;
    use.rt = unit - use.head * row_tiles;
  }
  use.rewind(a, warp);
  Cursor<TILE, WT> load = use;

  // a lane copies the 16-byte chunks lane, lane + 32, ... of PT rows that lie one behind the other
  constexpr int CH = D / 16, COPIES = PT * CH / 32;
  const uint32_t k_base = shared_address(&ring.k[0][0]);
  uint32_t k_to[16 * CH / 32];                     // of the first 16 rows: the swizzle repeats behind them
#pragma unroll
  for (int i = 0; i < 16 * CH / 32; ++i) {
    const int c = i * 32 + lane, r = c / CH;
    k_to[i] = k_base + r * D + swizzled<D>(r, c % CH) * 16;
  }
  constexpr uint32_t kToV = sizeof(ring.k);
  const uint32_t s_to = shared_address(&ring.s[0][lane & 1]);
  const float* s_from = lane & 1 ? a.vs : a.ks;
  const int64_t page_bytes = (int64_t)a.bs * D;
  struct Pages { int id[PG]; };                    // -1: none
  auto pages_of = [&](const Cursor<TILE, WT>& c) {
    Pages p;
    const int tok = c.token(warp);
    p.id[0] = tok < c.len ? c.table[c.page] : -1;
    if constexpr (PG == 2) p.id[1] = tok + PT >= c.len ? -1 : c.off + PT < a.bs ? p.id[0] : c.table[c.page + 1];
    return p;
  };
  Pages pages = pages_of(load);
  constexpr uint32_t kAll = (1u << PG) - 1;
  uint32_t active = 0;                             // pages of the stages that hold tokens
  auto issue = [&](int st) {
    if (left_load > 0) {
      uint32_t have = 0;
#pragma unroll
      for (int x = 0; x < PG; ++x)
        if ((uint32_t)pages.id[x] < (uint32_t)a.pages) {
          have |= 1u << x;
          int off = load.off + PT * x;
          if (x > 0 && off >= a.bs) off -= a.bs;
          const int ph = pages.id[x] * a.nkv + load.head, valid = load.len - load.token(warp) - PT * x;
          const int64_t at = ph * page_bytes + off * D + lane * 16;
          const uint8_t *k = a.kc + at, *v = a.vc + at;
          const uint32_t stage = (st * WT + x * PT) * D;
          if (valid >= PT) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              const uint32_t to = k_to[i % (16 * CH / 32)] + stage + i / (16 * CH / 32) * 16 * D;
              copy16(to, k + i * 512);
              copy16(to + kToV, v + i * 512);
            }
          } else {                                 // rows behind the end become zeros: 0 * garbage must not be NaN
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              const uint32_t to = k_to[i % (16 * CH / 32)] + stage + i / (16 * CH / 32) * 16 * D;
              const int bytes = (i * 32 + lane) / CH < valid ? 16 : 0;
              copy16(to, k + i * 512, bytes);
              copy16(to + kToV, v + i * 512, bytes);
            }
          }
          if (lane < 2) copy4(s_to + st * 16 + x * 8, s_from + ph);
        }
      active = (active & ~(kAll << (st * PG))) | have << (st * PG);
      load.next(a, row_tiles, warp);
      if (--left_load > 0) pages = pages_of(load);
    }
    __pipeline_commit();
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(s);

  int st = 0;
  bool first_unit = true;
  while (left > 0) {
    // ---------------- a unit, or the part of it in this block's share
    const int head = use.head, rt = use.rt, rows_here = min(8 * H, rep - rt * 8 * H);
    const int from_tile = use.tile, n = min(use.tiles - use.tile, left);
    const int row = use.row, tiles = use.tiles, len = use.len;
    const T* q = static_cast<const T*>(a.q) + row * a.q_row + (int64_t)(head * rep + rt * 8 * H) * D;
    // Q fragments: k-step e of chunk i holds elements 16 (t + 4 i) + 4 e .. + 3 of head g (+ 8 h); the order of the
    // contraction is free as long as K's fragments follow it
    constexpr int KI = D / 64;
    uint32_t qb[H][KI * 4][2];
    float sc[H][2];                                // softmax scale of heads 2 t, 2 t + 1 (+ 8 h) times what q was divided by
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int r = g + 8 * h;
      float f[KI][16], big = 0.f;
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (r < rows_here) u = *reinterpret_cast<const uint4*>(q + (int64_t)r * D + 16 * (t + 4 * i) + e);
          const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int j = 0; j < 8; ++j) { f[i][e + j] = to_float(x[j]); big = fmaxf(big, fabsf(f[i][e + j])); }
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // power of two that brings the row's largest to [2^10, 2^11); the sign of the softmax scale goes with it
      const int e = big > 0.f ? min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 120) : 0;
      const float up = copysignf(__uint_as_float((uint32_t)(127 + 10 - e) << 23), a.scale);
      const float down = fabsf(a.scale) * __uint_as_float((uint32_t)(127 - 10 + e) << 23);
      sc[h][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      sc[h][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          qb[h][i * 4 + s][0] = half2_bits(f[i][4 * s] * up, f[i][4 * s + 1] * up);
          qb[h][i * 4 + s][1] = half2_bits(f[i][4 * s + 2] * up, f[i][4 * s + 3] * up);
        }
    }
    // accumulator j: elements 2 j, 2 j + 1 of a lane's piece of the head, heads 2 t, 2 t + 1
    constexpr int NT = D / 16;
    float o[H][NT][4];
    float m[H][2], l[H][2], shift[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int j = 0; j < NT; ++j) o[h][j][0] = o[h][j][1] = o[h][j][2] = o[h][j][3] = 0.f;
      m[h][0] = m[h][1] = -INFINITY;
      l[h][0] = l[h][1] = 0.f;
      shift[h][0] = shift[h][1] = 0.f;
    }
    float unit_v = 0.f, per_unit = 0.f;            // o is kept in units of this V scale; 1 / unit_v

    for (int i = 0; i < n; ++i) {
      __pipeline_wait_prior(ST - 2);
      __syncwarp();                                // every lane's copies of this stage are in, every lane is done with the last
      const uint32_t now = active >> (st * PG) & kAll;
      issue(st == 0 ? ST - 1 : st - 1);
      if (now) {
        const uint8_t *ks = ring.k[st], *vs = ring.v[st];
        float k_scale[PG], v_scale[PG];
#pragma unroll
        for (int x = 0; x < PG; ++x) {
          const float2 u = *reinterpret_cast<const float2*>(&ring.s[st][2 * x]);
          k_scale[x] = u.x;
          v_scale[x] = u.y;
        }
        // ---- S^T = K Q^T, 16 tokens at a time: tokens g (elements 0, 1) and g + 8 (2, 3), heads 2 t and 2 t + 1
        float s[H][PIECES][4];
#pragma unroll
        for (int x = 0; x < PIECES; ++x) {
#pragma unroll
          for (int h = 0; h < H; ++h) s[h][x][0] = s[h][x][1] = s[h][x][2] = s[h][x][3] = 0.f;
#pragma unroll
          for (int c = 0; c < KI; ++c) {
            const int r = x * 16 + g;              // row r + 8 has the same swizzle
            const uint8_t* at = ks + r * D + swizzled<D>(r, t + 4 * c) * 16;
            const uint4 u = *reinterpret_cast<const uint4*>(at), v = *reinterpret_cast<const uint4*>(at + 8 * D);
            const uint32_t lo[4] = {u.x, u.y, u.z, u.w}, hi[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t ka[4];
              e4m3x4_to_half2(lo[e], ka[0], ka[2]);
              e4m3x4_to_half2(hi[e], ka[1], ka[3]);
#pragma unroll
              for (int h = 0; h < H; ++h) mma_f16(s[h][x], ka, qb[h][c * 4 + e][0], qb[h][c * 4 + e][1]);
            }
          }
        }
        const int valid = len - (from_tile + i) * TILE - warp * WT;
        if (valid < WT || now != kAll) {
#pragma unroll
          for (int x = 0; x < PIECES; ++x) {
            const bool page_in = now >> (x * PG / PIECES) & 1;
            if (!page_in) k_scale[x * PG / PIECES] = 1.f;
            const bool out0 = x * 16 + g >= valid || !page_in, out1 = x * 16 + g + 8 >= valid || !page_in;
#pragma unroll
            for (int h = 0; h < H; ++h) {
              if (out0) s[h][x][0] = s[h][x][1] = -INFINITY;
              if (out1) s[h][x][2] = s[h][x][3] = -INFINITY;
            }
          }
        }
        // ---- running softmax
        float f[H][2][PG], mx[H][2];
        bool grown = false;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float best[PG];
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
              const float b = fmaxf(s[h][x][y], s[h][x][2 + y]);
              best[x * PG / PIECES] = x * PG % PIECES == 0 ? b : fmaxf(best[x * PG / PIECES], b);
            }
#pragma unroll
            for (int x = 0; x < PG; ++x) {
              f[h][y][x] = fmaxf(sc[h][y] * k_scale[x], 1e-37f);     // above 0: masked scores stay -inf at a softmax scale of 0 too
              best[x] *= f[h][y][x];
            }
            mx[h][y] = PG == 2 ? fmaxf(best[0], best[PG - 1]) : best[0];
            mx[h][y] = fmaxf(mx[h][y], __shfl_xor_sync(0xffffffffu, mx[h][y], 4));
            mx[h][y] = fmaxf(mx[h][y], __shfl_xor_sync(0xffffffffu, mx[h][y], 8));
            mx[h][y] = fmaxf(mx[h][y], __shfl_xor_sync(0xffffffffu, mx[h][y], 16));
            grown |= mx[h][y] > m[h][y];
          }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float top = fmaxf(m[h][y], mx[h][y]);
              const float alpha = top == m[h][y] ? 1.f : exp2_approx(m[h][y] - top);
              m[h][y] = top;
              shift[h][y] = top == -INFINITY ? 0.f : kProbShift - top;
              l[h][y] *= alpha;
#pragma unroll
              for (int j = 0; j < NT; ++j) { o[h][j][y] *= alpha; o[h][j][2 + y] *= alpha; }
            }
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
              s[h][x][y] = exp2_approx(fmaf(s[h][x][y], f[h][y][x * PG / PIECES], shift[h][y]));
              s[h][x][2 + y] = exp2_approx(fmaf(s[h][x][2 + y], f[h][y][x * PG / PIECES], shift[h][y]));
              l[h][y] += s[h][x][y] + s[h][x][2 + y];
            }
        // ---- O^T += V^T P^T, 16 tokens at a time: lane g holds the elements of its piece of V's rows
        constexpr int VB = D >= 128 ? 16 : 8;      // bytes of a piece
        const int piece = ((g & 1) << 2) | (g >> 1);
#pragma unroll
        for (int x = 0; x < PIECES; ++x) {
          if (PG == 2 && !(now >> x & 1)) continue;
          // V's scale joins the probabilities, relative to the unit that o is kept in; the unit follows the scale where
          // they are far apart, so that the probabilities stay inside fp16's normal range
          const float vs_x = v_scale[x * PG / PIECES];
          float ratio = vs_x * per_unit;
          if (vs_x > 0.f && !(ratio <= 1.f && ratio >= 0.0625f)) {             // the same for the whole warp
            const float change = unit_v / vs_x;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h][j][e] *= change;
            unit_v = vs_x;
            per_unit = 1.f / vs_x;
            ratio = 1.f;
          }
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[h][x][e] *= ratio;
          uint32_t pb[H][2];
#pragma unroll
          for (int h = 0; h < H; ++h) {
            pb[h][0] = transpose8(half2_bits(s[h][x][0], s[h][x][1]));
            pb[h][1] = transpose8(half2_bits(s[h][x][2], s[h][x][3]));
          }
#pragma unroll
          for (int c = 0; c < D / (8 * VB); ++c) {
            uint32_t w[4][VB / 4];                 // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int r = x * 16 + 2 * t + (y & 1) + (y >> 1) * 8;
              if constexpr (VB == 16) {
                const uint4 u = *reinterpret_cast<const uint4*>(vs + r * D + swizzled<D>(r, piece + 8 * c) * 16);
                w[y][0] = u.x; w[y][1] = u.y; w[y][2] = u.z; w[y][3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(vs + r * D + swizzled<D>(r, piece >> 1) * 16 + (piece & 1) * 8);
                w[y][0] = u.x; w[y][1] = u.y;
              }
            }
#pragma unroll
            for (int y = 0; y < VB / 4; ++y) {
              uint32_t lo[4], hi[4];
              e4m3x4_to_half2(__byte_perm(w[0][y], w[1][y], 0x5140), lo[0], lo[1]);
              e4m3x4_to_half2(__byte_perm(w[0][y], w[1][y], 0x7362), lo[2], lo[3]);
              e4m3x4_to_half2(__byte_perm(w[2][y], w[3][y], 0x5140), hi[0], hi[1]);
              e4m3x4_to_half2(__byte_perm(w[2][y], w[3][y], 0x7362), hi[2], hi[3]);
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const uint32_t va[4] = {lo[e], lo[e + 1], hi[e], hi[e + 1]};
#pragma unroll
                for (int h = 0; h < H; ++h) mma_f16(o[h][(c * VB + y * 4 + e) / 2], va, pb[h][0], pb[h][1]);
              }
            }
          }
        }
      }
      st = st + 1 == ST ? 0 : st + 1;
    }
    left -= n;
    use.tile += n - 1;
    use.next(a, row_tiles, warp);

    // ---------------- the four streams of the unit meet
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h][y] += __shfl_xor_sync(0xffffffffu, l[h][y], d);
        if (g == 0) { sh_m[warp][8 * h + 2 * t + y] = m[h][y]; sh_l[warp][8 * h + 2 * t + y] = l[h][y]; }
      }
    __syncthreads();
    float w[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWarps; ++x) top = fmaxf(top, sh_m[x][8 * h + 2 * t + y]);
        w[h][y] = m[h][y] == -INFINITY && l[h][y] == 0.f ? 0.f : exp2_approx(m[h][y] - top) * unit_v;
      }
    constexpr int VB = D >= 128 ? 16 : 8;
    const int piece = ((g & 1) << 2) | (g >> 1);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      if ((warp >> 1) == pass) {
        float* to = red + (warp & 1) * red_rows * D;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (8 * h + 2 * t + y < rows_here)
#pragma unroll
              for (int j = 0; j < NT; j += 2) {
                float4& x = *reinterpret_cast<float4*>(&to[(8 * h + 2 * t + y) * D + (j * 2 / VB) * 8 * VB + piece * VB + j * 2 % VB]);
                float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                if (w[h][y] != 0.f)
                  z = make_float4(o[h][j][y] * w[h][y], o[h][j][2 + y] * w[h][y], o[h][j + 1][y] * w[h][y], o[h][j + 1][2 + y] * w[h][y]);
                if (pass) { z.x += x.x; z.y += x.y; z.z += x.z; z.w += x.w; }
                x = z;
              }
      }
      __syncthreads();
    }
    const bool whole = from_tile == 0 && n == tiles;
    const int slot = 2 * blockIdx.x + (first_unit && from_tile > 0 ? 0 : 1);
    for (int i = tid * 2; i < rows_here * D; i += kThreads * 2) {
      const int r = i / D, d = i % D;
      float big = -INFINITY, sum = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) big = fmaxf(big, sh_m[x][r]);
#pragma unroll
      for (int x = 0; x < kWarps; ++x)
        if (sh_l[x][r] != 0.f) sum += sh_l[x][r] * exp2_approx(sh_m[x][r] - big);
      const float2 u = *reinterpret_cast<const float2*>(&red[i]), v = *reinterpret_cast<const float2*>(&red[red_rows * D + i]);
      const float2 val = make_float2(u.x + v.x, u.y + v.y);
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T pair[2] = {from_float<T>(val.x * inv), from_float<T>(val.y * inv)};
        *reinterpret_cast<uint32_t*>(&out[((int64_t)row * a.nq + head * rep + rt * 8 * H + r) * D + d]) = *reinterpret_cast<const uint32_t*>(pair);
      } else {
        *reinterpret_cast<float2*>(&a.part_o[((int64_t)slot * 16 + r) * D + d]) = val;
        if (d == 0) {
          a.part_ml[(slot * 16 + r) * 2] = big;
          a.part_ml[(slot * 16 + r) * 2 + 1] = sum;
        }
      }
    }
    first_unit = false;
    __syncthreads();
  }
}

// Joins the parts of the units that the cuts divide: block c looks after the cut in front of block c + 1's share, if it
// is the first cut inside its unit.  A warp joins a query head; where the cut lies is found while the attention kernel
// still runs (it lets this one start only after the lengths are there).
constexpr int kMostParts = 64;                    // weights of so many parts at a time

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_q8_join_kernel(const Args a) {
  __shared__ int64_t sh_place[8];
  __shared__ float sh_w[kWarps][kMostParts];
  pdl_trigger();
  const int rep = a.nq / a.nkv, row_tiles = (rep + a.unit_rows - 1) / a.unit_rows, per_row = a.nkv * row_tiles;
  const int c = blockIdx.x + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place place = locate<tile_tokens(D)>(a, per_row, c, sh_place);
  const int64_t pos = place.pos;
  bool mine = pos < place.total;
  int tiles = 1, unit = 0, parts = 0;
  if (mine) {
    tiles = tiles_of<tile_tokens(D)>(a, place.row);
    unit = (int)((uint32_t)(pos - place.base) / (uint32_t)tiles);
    const int64_t start = place.base + (int64_t)unit * tiles, stop = start + tiles;
    mine = pos != start && place.begin(c - 1) <= start;
    if (mine) {                                    // parts: the end of share c - 1 and the shares from c on that begin before `stop`
      int last = c + (int)((uint32_t)(stop - 1 - pos) / (uint32_t)min(place.share + 1, (int64_t)1 << 31));      // no share is longer
      while (last + 1 < place.shares && place.begin(last + 1) < stop) ++last;
      parts = last - c + 2;
    }
  }
  pdl_wait();
  if (!mine) return;
  const int head = unit / row_tiles, rt = unit % row_tiles, rows_here = min(a.unit_rows, rep - rt * a.unit_rows);
  auto slot = [&](int x) { return (x == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + x)) * 16; };
  for (int r = warp; r < rows_here; r += kWarps) {
    float big = -INFINITY;
    for (int x = lane; x < parts; x += 32) big = fmaxf(big, a.part_ml[(slot(x) + r) * 2]);
    big = warp_max(big);
    constexpr int E = D / 32;
    float num[E], den = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) num[e] = 0.f;
    for (int x0 = 0; x0 < parts; x0 += kMostParts) {
      const int here = min(kMostParts, parts - x0);
      __syncwarp();
      for (int x = lane; x < here; x += 32) {
        const float2 ml = *reinterpret_cast<const float2*>(&a.part_ml[(slot(x0 + x) + r) * 2]);
        const float w = ml.y == 0.f ? 0.f : exp2_approx(ml.x - big);
        sh_w[warp][x] = w;
        den += w * ml.y;
      }
      __syncwarp();
#pragma unroll 8
      for (int x = 0; x < here; ++x) {
        const float w = sh_w[warp][x];
        const float* from = a.part_o + (int64_t)(slot(x0 + x) + r) * D + lane;
#pragma unroll
        for (int e = 0; e < E; ++e) num[e] += w == 0.f ? 0.f : w * from[32 * e];
      }
    }
    den = warp_sum(den);
    T* out = static_cast<T*>(a.out) + ((int64_t)place.row * a.nq + head * rep + rt * a.unit_rows + r) * D + lane;
#pragma unroll
    for (int e = 0; e < E; ++e) out[32 * e] = from_float<T>(den == 0.f ? 0.f : num[e] / den);
  }
}

// tokens that every query row sees, and its sequence: trailing q_len tokens of each sequence, causal
__global__ void __launch_bounds__(kThreads)
q8_rows_kernel(const int* __restrict__ lens, const int* __restrict__ news, int B, int T, int* __restrict__ row_seq, int* __restrict__ row_len) {
  pdl_wait();
  pdl_trigger();
  __shared__ int sh[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // rows before this block's sequence
  const int b = blockIdx.x;
  int before = 0;
  for (int i = tid; i < b; i += kThreads) before += max(news[i], 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) sh[warp] = before;
  __syncthreads();
  before = sh[0] + sh[1] + sh[2] + sh[3];
  if (b == B) {                                    // rows behind the last sequence
    for (int r = before + tid; r < T; r += kThreads) { row_seq[r] = 0; row_len[r] = 0; }
    return;
  }
  const int n = max(news[b], 0);
  for (int i = tid; i < n && before + i < T; i += kThreads) {
    row_seq[before + i] = b;
    row_len[before + i] = max(lens[b] - n + 1 + i, 0);
  }
}

template <typename T, int D>
void launch_q8(Args a, const at::Tensor& q, cudaStream_t st) {
  constexpr int ST = D == 64 ? 5 : 3;
  const int rep = a.nq / a.nkv;
  a.unit_rows = rep <= 8 ? 8 : 16;
  const int row_tiles = (rep + a.unit_rows - 1) / a.unit_rows, red_rows = std::min(rep, a.unit_rows);
  constexpr int kMostPG = warp_tokens(D) / 16;
  const int pg = a.bs % warp_tokens(D) ? kMostPG : 1;
  void (*kernel)(const Args) = a.unit_rows == 8 ? (pg == 1 ? paged_q8_kernel<T, D, ST, 1, 1> : paged_q8_kernel<T, D, ST, 1, kMostPG>)
                                                : (pg == 1 ? paged_q8_kernel<T, D, ST, 2, 1> : paged_q8_kernel<T, D, ST, 2, kMostPG>);
  auto smem_of = [](int rows) { return sizeof(WarpRing<D, ST>) * kWarps + 2 * rows * D * sizeof(float); };
  const size_t smem = smem_of(red_rows);
  static std::atomic<int> residents[64][2][17] = {};  // blocks that an SM holds, per device, pages of a warp, rows of a unit
  const int dev = q.get_device();
  TORCH_CHECK(dev >= 0 && dev < 64, "paged_attention_q8: device index out of range");
  int resident = residents[dev][pg - 1][red_rows].load();
  if (!resident) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(16)));
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, smem));
    resident = std::max(resident, 1);
    residents[dev][pg - 1][red_rows].store(resident);
  }
  const int64_t most = (int64_t)a.rows * a.nkv * row_tiles * (((int64_t)a.width * a.bs + tile_tokens(D) - 1) / tile_tokens(D));
  a.grid = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)resident * at::cuda::getCurrentDeviceProperties()->multiProcessorCount, most));
  auto part_o = at::empty({2 * a.grid, 16, D}, q.options().dtype(at::kFloat));
  auto part_ml = at::empty({2 * a.grid, 16, 2}, q.options().dtype(at::kFloat));
  a.part_o = part_o.data_ptr<float>();
  a.part_ml = part_ml.data_ptr<float>();
  C10_CUDA_CHECK(launch_pdl(kernel, dim3(a.grid), dim3(kThreads), smem, st, a));
  if (a.grid > 1)
    C10_CUDA_CHECK(launch_pdl(paged_q8_join_kernel<T, D>, dim3(a.grid - 1), dim3(kThreads), 0, st, a));
}

}  // namespace

at::Tensor paged_attention_q8(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                              const at::Tensor& vs, const at::Tensor& tables, const at::Tensor& lens,
                              const c10::optional<at::Tensor>& news, double scale) {
  const c10::cuda::CUDAGuard guard(q.device());
  Args a = {};
  const int D = (int)q.size(2);
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  if (q.size(0) == 0) return out;
  a.q = q.data_ptr(); a.q_row = q.stride(0);
  a.kc = (const uint8_t*)kc.data_ptr(); a.vc = (const uint8_t*)vc.data_ptr();
  a.ks = ks.data_ptr<float>(); a.vs = vs.data_ptr<float>();
  a.tables = tables.data_ptr<int>();
  a.out = out.data_ptr();
  a.T = (int)q.size(0); a.nq = (int)q.size(1); a.nkv = (int)kc.size(1); a.bs = (int)kc.size(2); a.pages = (int)kc.size(0);
  TORCH_CHECK_VALUE(kc.size(0) * kc.size(1) < (int64_t)1 << 31, "paged_attention_q8: fewer than 2^31 pages times heads");
  a.width = (int)tables.size(1);
  a.scale = (float)(scale * 1.4426950408889634);
  auto st = at::cuda::getCurrentCUDAStream();
  const int B = (int)lens.size(0);
  at::Tensor row_seq, row_len;
  if (news.has_value()) {
    row_seq = at::empty({a.T}, lens.options());
    row_len = at::empty({a.T}, lens.options());
    a.rows = a.T;
    C10_CUDA_CHECK(launch_pdl(q8_rows_kernel, dim3(B + 1), dim3(kThreads), 0, st, (const int*)lens.data_ptr<int>(),
                              (const int*)news->data_ptr<int>(), B, a.T, row_seq.data_ptr<int>(), row_len.data_ptr<int>()));
    a.row_seq = row_seq.data_ptr<int>();
    a.row_len = row_len.data_ptr<int>();
  } else {
    a.rows = std::min(a.T, B);
    a.row_len = lens.data_ptr<int>();
  }
  const bool bf = q.scalar_type() == at::kBFloat16;
  if (D == 64) bf ? launch_q8<__nv_bfloat16, 64>(a, q, st) : launch_q8<__half, 64>(a, q, st);
  else if (D == 128) bf ? launch_q8<__nv_bfloat16, 128>(a, q, st) : launch_q8<__half, 128>(a, q, st);
  else bf ? launch_q8<__nv_bfloat16, 256>(a, q, st) : launch_q8<__half, 256>(a, q, st);
  return out;
}
