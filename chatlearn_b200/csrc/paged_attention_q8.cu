// Attention over the paged key/value cache held in 8 bits (e4m3 codes, one power-of-two scale per page and kv head).
//
//   o = softmax(scale * q (s_k C_k)^T) (s_v C_v)
//
// One unit of work is (query row set, kv head): the query heads that share a kv head are the columns of m16n8k16 tiles
// whose rows are cached tokens (S^T = K Q^T) or head elements (O^T = V^T P^T), so that up to 8 heads waste nothing, each
// cached byte is read once per unit and dequantised once.  Codes become halves by one conversion (exact: e4m3 is a
// subset of fp16); the scales are powers of two and stay out of the products: s_k joins the softmax scale, s_v the
// probabilities.  (Products of e4m3 operands are no way around the conversions: mma.sync carries them out in halves.)
// The probabilities are rounded to fp16 once, as the product beside exact codes takes them (2^-11 of each); their sum is
// taken in fp32 before.
// Queries are rescaled per row by a power of two to 2^10..2^11, so that their fp16 form loses nothing that counts (bf16
// has 8 significant bits, fp16 11; what falls below 2^-24 of a row's largest is lost).
//
// The bytes of the cache bound it.  The tokens of all units form one line that is cut evenly over the resident blocks
// (whatever the lengths are) and inside a block over its warps, 32 tokens at a time (16 at head dim 256).  A warp works
// alone: its own cp.async ring, running maximum and sum, no barrier until its block's share is done.  A unit that lies
// inside a warp's stretch is finished by the warp; parts of divided units meet at the end of the block, and a second
// kernel joins what a cut between blocks divides.  The cuts go by the lengths alone, so results do not depend on timing.
//
// Measured, 32 / 8 heads of 128, from box to box: 128 sequences of 128 to 2,600 tokens (344 MB) 71 to 82 us, 4.2 to 4.8 TB/s;
// 4 of 30 to 65 thousand (331 MB) 70 to 78 us; one of 750 9.9 us.  About 10 us stand still (lengths -> tables -> tiles ->
// parts -> join).  The rest is a warp's own chain over a tile, which has to end before its stage is filled again: with two
// warps to a scheduler (162 registers, 98 KB of ring a block) an instruction is issued in 35 % of the cycles, DRAM is 57 %
// busy, no pipe above 34 % (the conversions'), and the warps wait for the instruction before (1.7 of 5 cycles), for the
// copies (0.8) and for shared memory (0.7).  Shorter tiles, more or fewer stages or blocks did not change it.  (Of the cuts
// tried, more shares than resident blocks cost more in parts than they even out.)
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_pipeline.h>

#include <atomic>
#include <type_traits>

#include "q8.cuh"
#include "q8_attention.h"

using namespace cl;
using namespace q8;

namespace {

constexpr int kThreads = 128, kWarps = 4;
// tokens of a tile, which a warp takes at a time: 8 KB of keys and values at head dims 128 and 256
__host__ __device__ constexpr int tile_tokens(int D) { return D >= 256 ? 16 : 32; }
// probabilities are carried times 2^10: fp16 keeps 11 bits of them down to 2^-24 of the largest
constexpr float kProbShift = 10.f;
// scores (in bits) from which a score's product is rounded before the maximum is taken off: the exact product in a fused
// multiply-add is off the rounded maximum by up to half a step of it, 2^-4 here, but 2^6 and more from 2^30 on
constexpr float kFarScore = 0x1p20f;

struct Args {
  const void* q;                 // [T, nq, D], row stride q_row
  int64_t q_row;
  const uint8_t *kc, *vc;        // [pages, nkv, bs, D]
  const float *ks, *vs;          // [pages, nkv]
  const int* tables;             // [B, width]
  // the query rows: row of q and out (-1: none), its sequence (both null: the row's own number), the tokens that it sees
  const int *row_id, *row_seq;
  const int* row_len;
  void* out;                     // [T, nq, D]
  // parts of divided units, unit_rows each: 2 of every block (the unit that its share begins in, the one it ends in),
  // behind them one of every warp (the unit that its stretch begins in)
  float *part_o, *part_ml;       // [6 * grid, unit_rows, D], [6 * grid, unit_rows, 2]: maximum and sum
  int rows, T, width, nq, nkv, bs;  // T: rows of out that this kernel looks after, the ones behind `rows` being empty
  int pages;
  int grid;                      // blocks that the line is cut over
  int unit_rows;                 // query heads of a unit: 8 or 16
  float scale;                   // softmax scale times log2 e
};

// Sequences with fewer new tokens go row by row, each row reading its cache; the others in tiles of 128 / rep tokens, which
// read it once but walk it alone, 64 keys in 1.6 us.  Many sequences fill the GPU with tiles: 32 of 2 / 3 / 4 / 7 new
// tokens after 4,096 (32 / 8 heads of 128) take 107 / 153 / 197 / 316 us by rows, 129 us in tiles.  Where all new tokens
// beyond one a sequence are few, the rows of one pass are cheaper than one tile's walk: 2 sequences of 7 after 2,048 take 25
// us by rows, 54 us in tiles.
constexpr int kChunkTokens = 3;
constexpr int64_t kChunkWork = 60000;              // (new tokens - sequences) x kv heads x head_dim from which tiles pay

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
  int64_t pos, end;              // stretch of the line
  int row;                       // row set that holds `pos`
  int64_t base;                  // where that row set begins
  __device__ __forceinline__ int64_t begin(int i) const { return i * share + min(i, longer); }
};

// Exclusive prefix sums over the rows' tiles, `per_row` units each: the warp's stretch of share `index`, or all of the
// share where `whole`; pos == end if there is none.  Every warp for itself.
template <int TILE>
__device__ Place locate(const Args& a, int per_row, int index, bool whole) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.rows + 31) / 32;
  const int r0 = min(lane * per, a.rows), r1 = min(r0 + per, a.rows);
  int64_t sum = 0;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) sum += tiles_of<TILE>(a, r);
  sum *= per_row;
  int64_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t p = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += p;
  }
  Place p;
  p.total = __shfl_sync(0xffffffffu, inc, 31);
  // at least a tile for each warp of a share
  p.shares = (int)max((int64_t)1, min((int64_t)a.grid, (p.total + kWarps - 1) / kWarps));
  if (p.total >> 31) {
    p.share = p.total / p.shares;
    p.longer = (int)(p.total - p.share * p.shares);
  } else {
    p.share = (uint32_t)p.total / (uint32_t)p.shares;
    p.longer = (int)((uint32_t)p.total - (uint32_t)p.share * p.shares);
  }
  p.pos = p.end = p.total;
  if (index < p.shares) {
    const int64_t n = p.share + (index < p.longer), first = p.begin(index);
    p.pos = whole ? first : first + n * warp / kWarps;
    p.end = whole ? first + n : first + n * (warp + 1) / kWarps;
  }
  const int64_t first = inc - sum;
  const uint32_t mine = __ballot_sync(0xffffffffu, first <= p.pos && p.pos < inc);
  int r = r0;
  int64_t at = first;
  if (mine >> lane & 1)
    for (; r < r1; ++r) {
      const int64_t n = (int64_t)tiles_of<TILE>(a, r) * per_row;
      if (p.pos < at + n) break;
      at += n;
    }
  const int from = mine ? __ffs(mine) - 1 : 0;
  p.row = __shfl_sync(0xffffffffu, r, from);
  p.base = __shfl_sync(0xffffffffu, at, from);
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

// A warp's position on the line: row set, kv head and row tile of it, tile; the page that holds the tile's first token.
template <int TILE>
struct Cursor {
  int row, head, rt, tile, tiles, len;
  int page, off;                                 // number in the sequence's table, token inside the page
  int step_page, step_off;                       // of a tile
  const int* table;
  __device__ __forceinline__ void rewind(const Args& a) {
    page = tile * TILE / a.bs;
    off = tile * TILE - page * a.bs;
  }
  __device__ __forceinline__ void enter(const Args& a, int r) {
    row = r;
    tiles = 0;
    while (row < a.rows && (tiles = tiles_of<TILE>(a, row)) == 0) ++row;
    if (row >= a.rows) return;
    len = min(a.row_len[row], a.width * a.bs);
    table = a.tables + (int64_t)(a.row_seq ? a.row_seq[row] : row) * a.width;
    // the first 1024 pages' numbers on their way
    const int line = (threadIdx.x & 31) * 32;
    if (line < a.width) asm volatile("prefetch.global.L1 [%0];" ::"l"(table + line));
  }
  // whether a new unit begins
  __device__ __forceinline__ bool next(const Args& a, int row_tiles) {
    if (++tile < tiles) {
      page += step_page;
      off += step_off;
      if (off >= a.bs) { off -= a.bs; ++page; }
      return false;
    }
    tile = page = off = 0;
    if (++rt < row_tiles) return true;
    rt = 0;
    if (++head < a.nkv) return true;
    head = 0;
    enter(a, row + 1);
    return true;
  }
};

template <int D, int ST>
struct WarpRing {
  uint8_t k[ST][tile_tokens(D) * D];
  uint8_t v[ST][tile_tokens(D) * D];
  float s[ST][4];                                // scales of the 16-token halves: K, V, K, V
};

// Parts that a warp leaves to its block: of the unit that its stretch begins in (if it ended there), and of the one that
// it ends in (if it did not).
struct Left {
  int head, tail;                                // 1: there is such a part; tail 2: the unit began in an earlier stretch
  int row[2], col[2], rows[2];                   // row of out, first query head, heads of the unit
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
  constexpr int TILE = tile_tokens(D), PIECES = TILE / 16, PT = TILE / PG;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float2 sh_ml[kWarps][2][8 * H];       // maximum and sum of the parts left to the block
  __shared__ Left sh_left[kWarps];
  pdl_wait();
  pdl_trigger();                                   // after the wait: the joining kernel reads the lengths before its own
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  auto& ring = reinterpret_cast<WarpRing<D, ST>*>(smem)[warp];
  const int rep = a.nq / a.nkv, row_tiles = (rep + 8 * H - 1) / (8 * H), per_row = a.nkv * row_tiles;
  T* out = static_cast<T*>(a.out);

  const Place place = locate<TILE>(a, per_row, blockIdx.x, false);
  int left = (int)(place.end - place.pos), left_load = left;
  Cursor<TILE> use;
  use.step_page = TILE / a.bs;
  use.step_off = TILE % a.bs;
  if (left > 0) {
    use.enter(a, place.row);
    const uint32_t in_row = (uint32_t)(place.pos - place.base);        // a row set has less than 2^31 tiles
    const int unit = (int)(in_row / (uint32_t)use.tiles);
    use.tile = (int)in_row - unit * use.tiles;
    use.head = unit / row_tiles;
    use.rt = unit - use.head * row_tiles;
    use.rewind(a);
  }
  Cursor<TILE> load = use;

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
  auto pages_of = [&](const Cursor<TILE>& c) {
    Pages p;
    const int tok = c.tile * TILE;
    p.id[0] = c.table[c.page];
    if constexpr (PG == 2) p.id[1] = tok + PT >= c.len ? -1 : c.off + PT < a.bs ? p.id[0] : c.table[c.page + 1];
    return p;
  };
  Pages pages = {};
  if (left > 0) pages = pages_of(load);
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
          const int ph = pages.id[x] * a.nkv + load.head, valid = load.len - load.tile * TILE - PT * x;
          const int64_t at = ph * page_bytes + off * D + lane * 16;
          const uint8_t *k = a.kc + at, *v = a.vc + at;
          const uint32_t stage = (st * TILE + x * PT) * D;
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
      const bool fresh = load.next(a, row_tiles);
      if (--left_load > 0) {
        pages = pages_of(load);
        if (fresh) {                               // the next unit's queries on their way
          const int first = load.head * rep + load.rt * 8 * H, bytes = min(8 * H, rep - load.rt * 8 * H) * D * 2;
          const int id = a.row_id ? a.row_id[load.row] : load.row;
          const char* q = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + id * a.q_row + (int64_t)first * D);
          for (int i = lane * 128; i < bytes; i += 32 * 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + i));
        }
      }
    }
    __pipeline_commit();
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(s);

  int st = 0;
  if (lane == 0) sh_left[warp].head = sh_left[warp].tail = 0;
  while (left > 0) {
    // ---------------- a unit, or the part of it in this warp's stretch
    const int head = use.head, rt = use.rt, rows_here = min(8 * H, rep - rt * 8 * H);
    const int from_tile = use.tile, n = min(use.tiles - use.tile, left);
    const int row = use.row, tiles = use.tiles, len = use.len;
    const int id = a.row_id ? a.row_id[row] : row;
    const T* q = static_cast<const T*>(a.q) + id * a.q_row + (int64_t)(head * rep + rt * 8 * H) * D;
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
    bool far = false;                              // of the whole warp

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
        const int valid = len - (from_tile + i) * TILE;
        if (valid < TILE || now != kAll) {
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
              far |= fabsf(top) >= kFarScore && top != -INFINITY;
              shift[h][y] = top == -INFINITY ? 0.f : kProbShift - top;
              l[h][y] *= alpha;
#pragma unroll
              for (int j = 0; j < NT; ++j) { o[h][j][y] *= alpha; o[h][j][2 + y] *= alpha; }
            }
          far = __any_sync(0xffffffffu, far);
        }
        if (far) {                                 // scores become their distances to the maximum
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              if (m[h][y] == -INFINITY) continue;
#pragma unroll
              for (int x = 0; x < PIECES; ++x) {
                s[h][x][y] = __fadd_rn(__fmul_rn(s[h][x][y], f[h][y][x * PG / PIECES]), -m[h][y]);
                s[h][x][2 + y] = __fadd_rn(__fmul_rn(s[h][x][2 + y], f[h][y][x * PG / PIECES]), -m[h][y]);
              }
#pragma unroll
              for (int x = 0; x < PG; ++x) f[h][y][x] = 1.f;
            }
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
              const float off = far && m[h][y] != -INFINITY ? kProbShift : shift[h][y];
              s[h][x][y] = exp2_approx(fmaf(s[h][x][y], f[h][y][x * PG / PIECES], off));
              s[h][x][2 + y] = exp2_approx(fmaf(s[h][x][2 + y], f[h][y][x * PG / PIECES], off));
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
    use.next(a, row_tiles);

    // ---------------- the end of the unit, or of the stretch
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h][y] += __shfl_xor_sync(0xffffffffu, l[h][y], d);
    // accumulators j and j + 1 of a head: 4 neighbouring elements
    constexpr int VB = D >= 128 ? 16 : 8;
    const int piece = ((g & 1) << 2) | (g >> 1);
    auto column = [&](int j) { return j * 2 / VB * 8 * VB + piece * VB + j * 2 % VB; };
    const bool begins = from_tile == 0, ends = from_tile + n == tiles;
    if (begins && ends) {
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = 8 * h + 2 * t + y;
          if (r >= rows_here) continue;
          const float w = l[h][y] == 0.f ? 0.f : unit_v / l[h][y];
          T* to = out + ((int64_t)id * a.nq + head * rep + rt * 8 * H + r) * D;
#pragma unroll
          for (int j = 0; j < NT; j += 4) {        // 8 elements
            T x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[2 * e] = from_float<T>(o[h][j + e][y] * w);
              x[2 * e + 1] = from_float<T>(o[h][j + e][2 + y] * w);
            }
            *reinterpret_cast<uint4*>(to + column(j)) = *reinterpret_cast<const uint4*>(x);
          }
        }
    } else {
      // a part: the stretch's first unit goes to memory (the ring is in use), its last one into the ring
      float* to;
      if (ends) {
        to = a.part_o + (int64_t)(2 * a.grid + blockIdx.x * kWarps + warp) * a.unit_rows * D;
      } else {
        __pipeline_wait_prior(0);
        __syncwarp();
        to = reinterpret_cast<float*>(&ring);
      }
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int r = 8 * h + 2 * t + y;
          if (r >= rows_here) continue;
          if (g == 0) sh_ml[warp][ends ? 0 : 1][r] = make_float2(m[h][y], l[h][y]);
#pragma unroll
          for (int j = 0; j < NT; j += 2)
            *reinterpret_cast<float4*>(&to[r * D + column(j)]) =
                make_float4(o[h][j][y] * unit_v, o[h][j][2 + y] * unit_v, o[h][j + 1][y] * unit_v, o[h][j + 1][2 + y] * unit_v);
        }
      if (lane == 0) {
        Left& x = sh_left[warp];
        const int i = ends ? 0 : 1;
        if (ends) x.head = 1;
        else x.tail = begins ? 1 : 2;
        x.row[i] = id;
        x.col[i] = head * rep + rt * 8 * H;
        x.rows[i] = rows_here;
      }
    }
  }
  __pipeline_wait_prior(0);

  // ---------------- parts of the block's warps meet; the list is in the order of the line
  __syncthreads();
  auto join_parts = [&](int first, int last, bool continued, bool finished) {        // part 2 w: warp w's head, 2 w + 1: its tail
    const Left& x = sh_left[last >> 1];
    const int i = last & 1, rows_here = x.rows[i];
    for (int e = tid * 4; e < rows_here * D; e += kThreads * 4) {
      const int r = e / D;
      float big = -INFINITY, den = 0.f;
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = first; p <= last; ++p)
        if (p & 1 ? sh_left[p >> 1].tail : sh_left[p >> 1].head) big = fmaxf(big, sh_ml[p >> 1][p & 1][r].x);
      for (int p = first; p <= last; ++p) {
        if (!(p & 1 ? sh_left[p >> 1].tail : sh_left[p >> 1].head)) continue;
        const float2 ml = sh_ml[p >> 1][p & 1][r];
        if (ml.y == 0.f) continue;
        const float* from = p & 1 ? reinterpret_cast<const float*>(&reinterpret_cast<WarpRing<D, ST>*>(smem)[p >> 1])
                                  : a.part_o + (int64_t)(2 * a.grid + blockIdx.x * kWarps + (p >> 1)) * a.unit_rows * D;
        const float4 v = *reinterpret_cast<const float4*>(&from[e]);
        const float w = exp2_approx(ml.x - big);
        den += w * ml.y;
        num.x += w * v.x; num.y += w * v.y; num.z += w * v.z; num.w += w * v.w;
      }
      if (finished && !continued) {
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const T y[4] = {from_float<T>(num.x * inv), from_float<T>(num.y * inv), from_float<T>(num.z * inv), from_float<T>(num.w * inv)};
        *reinterpret_cast<uint2*>(&out[((int64_t)x.row[i] * a.nq + x.col[i]) * D + e]) = *reinterpret_cast<const uint2*>(y);
      } else {
        const int64_t slot = 2 * blockIdx.x + (continued ? 0 : 1);
        *reinterpret_cast<float4*>(&a.part_o[slot * a.unit_rows * D + e]) = num;
        if (e % D == 0) *reinterpret_cast<float2*>(&a.part_ml[(slot * a.unit_rows + r) * 2]) = make_float2(big, den);
      }
    }
  };
  int first = -1;
  bool continued = false;
  for (int w = 0; w < kWarps; ++w) {
    if (sh_left[w].head) {
      if (first < 0) { first = 2 * w; continued = true; }
      join_parts(first, 2 * w, continued, true);
      first = -1;
    }
    if (sh_left[w].tail && first < 0) { first = 2 * w + 1; continued = sh_left[w].tail == 2; }
  }
  if (first >= 0) {
    int last = kWarps - 1;
    while (!sh_left[last].tail) --last;            // warps behind it have no stretch
    join_parts(first, 2 * last + 1, continued, false);
  }
  // rows that see nothing are zero
  for (int r = blockIdx.x * kWarps + warp; r < a.T; r += gridDim.x * kWarps)
    if (r >= a.rows || tiles_of<TILE>(a, r) == 0) {
      const int to = a.row_id ? a.row_id[r] : r;
      for (int i = lane * 8; to >= 0 && i < a.nq * D; i += 256) *reinterpret_cast<uint4*>(&out[(int64_t)to * a.nq * D + i]) = make_uint4(0, 0, 0, 0);
    }
}

// Joins the parts of the units that the cuts between blocks divide: block (c, r) looks after query head r of the unit that
// the cut in front of share c + 1 divides, if it is the first cut inside its unit.  Where the cut lies is found while the
// attention kernel still runs, ahead of the wait: from the lengths alone, which are there, because every block of the
// attention kernel triggers this one behind its own wait for the kernels that wrote them.  Few and short loops: a handful
// of warps run through here once, and waiting for code to arrive is a good part of what that takes.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_q8_join_kernel(const Args a) {
  __shared__ float sh_num[kWarps][D], sh_den[kWarps];
  pdl_trigger();
  const int rep = a.nq / a.nkv, row_tiles = (rep + a.unit_rows - 1) / a.unit_rows, per_row = a.nkv * row_tiles;
  const int c = blockIdx.x + 1, r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place place = locate<tile_tokens(D)>(a, per_row, c, true);
  const int64_t pos = place.pos;
  bool mine = pos < place.total;
  const int tiles = mine ? tiles_of<tile_tokens(D)>(a, place.row) : 1;
  const int unit = (int)((uint32_t)(pos - place.base) / (uint32_t)tiles);
  const int64_t start = place.base + (int64_t)unit * tiles, stop = start + tiles;
  const int head = unit / row_tiles, rt = unit - head * row_tiles;
  mine = mine && pos != start && place.begin(c - 1) <= start && r < min(a.unit_rows, rep - rt * a.unit_rows);
  // parts: the end of share c - 1 and the shares from c on that begin before `stop`
  int last = c + (int)((uint32_t)(stop - 1 - pos) / (uint32_t)min(place.share + 1, (int64_t)1 << 31));      // no share is longer
  while (mine && last + 1 < place.shares && place.begin(last + 1) < stop) ++last;
  const int parts = last - c + 2;
  pdl_wait();                                      // blocks without a cut wait too: this grid's end says that the outputs are there
  if (!mine) return;
  auto slot = [&](int x) { return (x == 0 ? 2 * (c - 1) + 1 : 2 * (c - 1 + x)) * a.unit_rows + r; };
  float big = -INFINITY;
  for (int x = lane; x < parts; x += 32) big = fmaxf(big, a.part_ml[slot(x) * 2]);
  big = warp_max(big);
  constexpr int E = D / 32;                        // neighbouring elements of a lane
  float num[E], den = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) num[e] = 0.f;
#pragma unroll 4
  for (int x = warp; x < parts; x += kWarps) {     // a warp takes every fourth part
    const float2 ml = *reinterpret_cast<const float2*>(&a.part_ml[slot(x) * 2]);
    const float* from = a.part_o + (int64_t)slot(x) * D + lane * E;
    const float w = ml.y == 0.f ? 0.f : exp2_approx(ml.x - big);
    den = fmaf(w, ml.y, den);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(from + e);
      num[e] = fmaf(w, v.x, num[e]);
      num[e + 1] = fmaf(w, v.y, num[e + 1]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sh_num[warp][lane * E + e] = num[e];
  if (lane == 0) sh_den[warp] = den;
  __syncthreads();
  den = (sh_den[0] + sh_den[1]) + (sh_den[2] + sh_den[3]);
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int id = a.row_id ? a.row_id[place.row] : place.row;
  T* out = static_cast<T*>(a.out) + ((int64_t)id * a.nq + head * rep + rt * a.unit_rows + r) * D;
  for (int d = threadIdx.x; d < D; d += kThreads)
    out[d] = from_float<T>(((sh_num[0][d] + sh_num[1][d]) + (sh_num[2][d] + sh_num[3][d])) * inv);
}

// The rows that go one by one: those of sequences with fewer than `min_chunk` new tokens, packed one behind the other,
// `room` places in all.  A block per sequence; the last one empties the places behind them and the rows of out behind the
// last sequence.
__global__ void __launch_bounds__(kThreads)
q8_rows_kernel(const int* __restrict__ lens, const int* __restrict__ news, int B, int T, int min_chunk, int room, int* __restrict__ row_id,
               int* __restrict__ row_seq, int* __restrict__ row_len, uint4* __restrict__ out, int out_row) {
  pdl_wait();
  pdl_trigger();
  __shared__ int sh[2][kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
  int rows = 0, at = 0;                            // rows before this sequence, and those of them that are in the list
  for (int i = tid; i < b; i += kThreads) {
    const int n = max(news[i], 0);
    rows += n;
    at += n < min_chunk ? n : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
    at += __shfl_xor_sync(0xffffffffu, at, o);
  }
  if (lane == 0) { sh[0][warp] = rows; sh[1][warp] = at; }
  __syncthreads();
  rows = sh[0][0] + sh[0][1] + sh[0][2] + sh[0][3];
  at = sh[1][0] + sh[1][1] + sh[1][2] + sh[1][3];
  if (b == B) {
    for (int r = at + tid; r < room; r += kThreads) { row_id[r] = -1; row_seq[r] = 0; row_len[r] = 0; }
    for (int64_t i = (int64_t)rows * out_row + tid; i < (int64_t)T * out_row; i += kThreads) out[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int n = max(news[b], 0), len = lens[b];
  if (n >= min_chunk) return;
  for (int i = tid; i < n && at + i < room; i += kThreads) {
    const bool held = rows + i < T;                // there is such a row
    row_id[at + i] = held ? rows + i : -1;
    row_seq[at + i] = b;
    row_len[at + i] = held ? max(len - n + 1 + i, 0) : 0;
  }
}

template <typename T, int D>
void launch_q8(Args a, const at::Tensor& q, cudaStream_t st) {
  // stages of a ring: as much on its way at D = 64, where a tile has half the bytes (64 x 4096 tokens of 8 kv heads: 75 us
  // with 3, 64 us with 5); more than 3 cost the second resident block elsewhere
  constexpr int ST = D == 64 ? 5 : 3;
  const int rep = a.nq / a.nkv;
  // More than 8 query heads to a kv head: 16 of them to a unit read the cache once, 8 twice, but faster (at head dim 256 16
  // rows do not fit the registers).  One kv head in two of B sequences of L tokens, 16 heads each, us with 8 / 16 rows:
  //   B x L      1 x 1024     8 x 4096     32 x 4096    64 x 4096
  //   D = 64     14.4 / 13.8  15.8 / 17.3  26.3 / 23.3
  //   D = 128    10.9 / 14.0  19.1 / 23.9  33.6 / 33.6  56.4 / 49.7
  //   D = 256    15.0 / 21.3  28.3 / 39.1  56.0 / 66.7
  // so 16 at D = 64, and at D = 128 where the tables have room for 64 MB (32 x 4096 above)
  constexpr bool kBoth = D < 256;
  a.unit_rows = kBoth && rep > 8 && (D == 64 || (int64_t)a.rows * a.nkv * a.width * a.bs * 2 * D >= 64 << 20) ? 16 : 8;
  const int row_tiles = (rep + a.unit_rows - 1) / a.unit_rows;
  constexpr int kMostPG = tile_tokens(D) / 16;
  const int pg = a.bs % tile_tokens(D) ? kMostPG : 1;
  void (*kernel)(const Args) = pg == 1 ? paged_q8_kernel<T, D, ST, 1, 1> : paged_q8_kernel<T, D, ST, 1, kMostPG>;
  if constexpr (kBoth)
    if (a.unit_rows == 16) kernel = pg == 1 ? paged_q8_kernel<T, D, ST, 2, 1> : paged_q8_kernel<T, D, ST, 2, kMostPG>;
  constexpr size_t smem = sizeof(WarpRing<D, ST>) * kWarps;
  static_assert(sizeof(WarpRing<D, ST>) >= 16 * D * sizeof(float), "a part fits the ring");
  static std::atomic<int> residents[64][4] = {};   // blocks that a device holds, per kernel
  const int dev = q.get_device();
  TORCH_CHECK(dev >= 0 && dev < 64, "paged_attention_q8: device index out of range");
  std::atomic<int>& known = residents[dev][(pg - 1) * 2 + a.unit_rows / 16];
  int resident = known.load();
  if (!resident) {
    int sms = 0;
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, smem));
    resident = std::max(resident, 1) * sms;
    known.store(resident);
  }
  const int64_t most = (int64_t)a.rows * a.nkv * row_tiles * (((int64_t)a.width * a.bs + tile_tokens(D) - 1) / tile_tokens(D));
  a.grid = (int)std::max<int64_t>(1, std::min<int64_t>(resident, (most + kWarps - 1) / kWarps));
  const int64_t rows = (int64_t)(2 + kWarps) * a.grid * a.unit_rows;
  auto part = at::empty({rows * (D + 2)}, q.options().dtype(at::kFloat));
  a.part_o = part.data_ptr<float>();
  a.part_ml = a.part_o + rows * D;
  C10_CUDA_CHECK(launch_pdl(kernel, dim3(a.grid), dim3(kThreads), smem, st, a));
  if (a.grid > 1) C10_CUDA_CHECK(launch_pdl(paged_q8_join_kernel<T, D>, dim3(a.grid - 1, std::min(rep, a.unit_rows)), dim3(kThreads), 0, st, a));
}

}  // namespace

bool q8::cache_fits(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& tables,
                    const at::Tensor& lens, const c10::optional<at::Tensor>& news, c10::Device dev) {
  auto codes = [&](const at::Tensor& x) {
    return x.scalar_type() == at::kFloat8_e4m3fn && x.device() == dev && x.is_contiguous() && (uintptr_t)x.data_ptr() % 16 == 0;
  };
  auto scales = [&](const at::Tensor& x) {
    return x.scalar_type() == at::kFloat && x.dim() == 2 && x.size(0) == kc.size(0) && x.size(1) == kc.size(1) && x.device() == dev && x.is_contiguous();
  };
  auto ints = [&](const at::Tensor& x, int64_t dims) { return x.scalar_type() == at::kInt && x.dim() == dims && x.device() == dev && x.is_contiguous(); };
  return dev.is_cuda() && kc.dim() == 4 && codes(kc) && codes(vc) && vc.sizes() == kc.sizes() && kc.size(1) > 0 && kc.size(2) > 0 &&
         kc.size(2) % 16 == 0 && scales(ks) && scales(vs) && ints(tables, 2) && ints(lens, 1) && tables.size(0) == lens.size(0) &&
         (!news.has_value() || (ints(*news, 1) && news->size(0) == lens.size(0))) && kc.size(0) > 0 &&
         kc.size(0) * kc.size(1) < (int64_t)1 << 31 && tables.size(1) * kc.size(2) < (int64_t)1 << 30;
}

// No tensor where the arguments are not as the kernels take them (the caller then says what is wrong, or lays them out).
c10::optional<at::Tensor> paged_attention_q8(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                              const at::Tensor& vs, const at::Tensor& tables, const at::Tensor& lens,
                              const c10::optional<at::Tensor>& news, double scale) {
  const int64_t D64 = q.dim() == 3 ? q.size(2) : 0;
  const bool fits =
      (D64 == 64 || D64 == 128 || D64 == 256) && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && q.stride(2) == 1 &&
      (q.size(1) == 1 || q.stride(1) == D64) && (q.size(0) <= 1 || q.stride(0) % 8 == 0) && (uintptr_t)q.data_ptr() % 16 == 0 &&
      cache_fits(kc, vc, ks, vs, tables, lens, news, q.device()) && kc.size(3) == D64 && q.size(1) > 0 && q.size(1) % kc.size(1) == 0 &&
      q.size(0) < (int64_t)1 << 31 && (news.has_value() || q.size(0) >= lens.size(0));
  if (!fits) return c10::nullopt;
  const c10::cuda::CUDAGuard guard(q.device());
  Args a = {};
  const int D = (int)D64;
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  if (q.size(0) == 0) return out;
  a.q = q.data_ptr(); a.q_row = q.stride(0);
  a.kc = (const uint8_t*)kc.data_ptr(); a.vc = (const uint8_t*)vc.data_ptr();
  a.ks = ks.data_ptr<float>(); a.vs = vs.data_ptr<float>();
  a.tables = tables.data_ptr<int>();
  a.out = out.data_ptr();
  a.T = (int)q.size(0); a.nq = (int)q.size(1); a.nkv = (int)kc.size(1); a.bs = (int)kc.size(2); a.pages = (int)kc.size(0);
  a.width = (int)tables.size(1);
  a.scale = (float)(scale * 1.4426950408889634);
  auto st = at::cuda::getCurrentCUDAStream();
  const int B = (int)lens.size(0);
  at::Tensor row_list;
  const bool bf = q.scalar_type() == at::kBFloat16;
  if (news.has_value()) {
    // (fp16 queries keep to the rows: the tiles' outputs are bf16)
    const bool chunks = bf && (int64_t)(a.T - B) * a.nkv * D >= kChunkWork && q8::chunk_supported(a.nq / a.nkv);
    a.rows = chunks ? (int)std::min<int64_t>(a.T, (int64_t)B * (kChunkTokens - 1)) : a.T;
    row_list = at::empty({3, std::max(a.rows, 1)}, lens.options());
    int* list = row_list.data_ptr<int>();
    const int room = (int)row_list.size(1);
    C10_CUDA_CHECK(launch_pdl(q8_rows_kernel, dim3(B + 1), dim3(kThreads), 0, st, (const int*)lens.data_ptr<int>(),
                              (const int*)news->data_ptr<int>(), B, a.T, chunks ? kChunkTokens : 1 << 30, room, list, list + room,
                              list + 2 * room, (uint4*)a.out, (int)(a.nq * D / 8)));
    a.row_id = list;
    a.row_seq = list + room;
    a.row_len = list + 2 * room;
    if (chunks) {
      q8::ChunkArgs c = {};
      c.q = a.q; c.q_row = a.q_row; c.kc = a.kc; c.vc = a.vc; c.ks = a.ks; c.vs = a.vs; c.tables = a.tables; c.out = a.out;
      c.lens = lens.data_ptr<int>(); c.news = news->data_ptr<int>();
      c.B = B; c.T = a.T; c.width = a.width; c.nq = a.nq; c.nkv = a.nkv; c.bs = a.bs; c.pages = a.pages;
      c.min_new = kChunkTokens; c.scale = a.scale;
      q8::launch_chunk(c, D, q.get_device(), st);
    }
    a.T = a.rows;
    if (a.rows == 0) return out;
  } else {
    a.rows = std::min(a.T, B);
    a.row_len = lens.data_ptr<int>();
  }
  if (D == 64) bf ? launch_q8<__nv_bfloat16, 64>(a, q, st) : launch_q8<__half, 64>(a, q, st);
  else if (D == 128) bf ? launch_q8<__nv_bfloat16, 128>(a, q, st) : launch_q8<__half, 128>(a, q, st);
  else bf ? launch_q8<__nv_bfloat16, 256>(a, q, st) : launch_q8<__half, 256>(a, q, st);
  return out;
}
