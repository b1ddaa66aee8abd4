// Decode attention over the 4-bit paged key/value cache (layout: include/kv4.cuh).
//
//   q    [B rows, Hq, d] bf16: the last `rows` tokens of every request; row i of a request of L cached tokens sees L - rows + 1 + i
//   out  [B rows, Hq, d] bf16 = sum_t p_t v_t,  p = softmax_t(scale q k_t),  k_t and v_t = code * step + lowest
//   weights[t] = decay * weights[t] + sum over the rows and the query heads of a key/value head of p_t
//
// Codes go to the tensor cores as whole numbers, exactly, and steps multiply fp32 numbers:
//   q k_t = sum over groups  step_t (sum q code) + lowest_t (sum q)
//   out   = sum over groups  sum_t (step_t p_t) (code - 8)  +  sum_t p_t (lowest_t + 8 step_t)
// so keys and values are never rounded.  Behind the exponent of 1024 a code is an fp16 number with an offset (kv4_code below).  Queries become fp16
// numbers without loss (a power of two for each row); the weights of the second product, step p_t, are rounded to fp16 once, after a
// factor for each row and group that follows the largest of them: 11 bits against the 8 of the result, whatever the sizes of other groups and
// tokens are.  Of the error against 64 bits, 1.66e-3 of a result, that makes under 1%.  Values go in around 0: their offset would cost the
// fp32 sums over a long cache the bits that they need.
//
// A token takes 144 bytes of keys and values at d = 128 and a tile of 16 tokens serves 8 query rows per product.  Instructions bound the
// kernel, though none of its units is full: 344 of them a tile of 16 tokens and 8 rows (some 150 integer, 48 packed fp16, 90 fp32, 16 products).  2 x 131,067
// tokens of 8 heads in 80 us fill 58% of the issue slots, integer pipes to 50%, tensor pipes to 22%, and read at 59% of a copy's rate.  Of the 4.5
// cycles that a warp takes an instruction, 1 issues it, 1 waits out a fixed latency, 0.9 wait for a busy pipe, 0.75 for other warps and 0.5 for
// data; an SM quarter has 3 warps for that.  Two and three blocks an SM run equally fast.
// Products in e4m3, in which a code needs no offset, are slower: they are carried out as four times as many fp16 ones (130 us when fp16 took 82).
//
// The query rows of a key/value head (rows x heads of its group, in tiles of 8) are the columns of the products (mma.sync m16n8k16), tokens and
// then columns of the head their rows: S = K Q^T, O^T = V^T P^T.  So a group of 8 heads wastes nothing, and P^T, which wants tokens along its
// rows, is what movmatrix makes of S.  tcgen05 products would want 64 or 128 rows and the unpacked codes in shared memory:
// 128 rows a head over 30,011 tokens twice took 105 us that way when they took 99 in tiles of 16 rows here (the softmax of a thread a row, and its waits for
// products, unpacked tiles and tensor memory, took longer than unpacking a tile 8 times).
//
// Each warp walks tiles of 64 tokens (32 at d = 256) by itself: bulk copies of the tile's codes and scales two tiles ahead, an mbarrier
// for each stage.  No block-wide wait stands in the loop.  The warps' results meet in shared memory at the end, those of the parts of a
// long request in a second kernel, the weights come from a third, each started while the one ahead of it ends: from scores that the first
// kept, or, where those would take too much memory, from the keys once more.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../include/kv4.cuh"
#include "../include/omni_ptx.cuh"
#include "../include/score_mod.cuh"
#include "../include/tma_host.h"

namespace omni {

constexpr int KV4_SITE_DECODE = 84, KV4_SITE_TILE = 85, KV4_SITE_WEIGHTS = 86;
constexpr int KV4_WARPS = 4, KV4_STAGES = 2, KV4_MAX_BLOCKS = 4096;
constexpr int KV4_WEIGHTS_ROWS = 256;       // most query rows a key/value head of a call that yields weights

struct Kv4Decode {
  const __nv_bfloat16* q;
  long long q_row;
  int q_head, q_wide;               // q_wide: rows and heads start on 16 bytes
  const int *table, *seq_lens;
  int table_ld, table_w, rows, hq;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;                       // [B, Hq, rows] in units of log 2, or null
  float* weights;
  float decay;
  int piece;                        // tokens of a copy: the largest of 64, 32, 16 that divides the block
  int min_tiles;                    // fewest tiles of a block's share; 0: a block takes one item, whole
  float* o_part;                    // [blocks, 2, 8 NT, d]: what a block has of the item that it starts with, and of the one it ends with
  float* lse_part;                  // [blocks, 2, 8 NT]
  float* scores;                    // [B, Hkv, chunks, score_places, 8 NT] in units of log 2, or null
  int score_places;                 // table_w blocks up to a multiple of 64
  int2* shared;                     // [B, Hkv, chunks]: where the parts of an item start (2 block + which), and how many there are
};

__device__ __forceinline__ int kv4_length(const Kv4Decode& a, int block, int b, OmniStatus* st) {
  const int n = max(a.seq_lens[b], 0);
  if (n <= a.table_w * block) return n;
  if (threadIdx.x == 0) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_DECODE, b);
  return a.table_w * block;
}
// Work is cut into equal shares.  An item is a tile of query rows of a key/value head of a request (in the weights kernel all rows).  With
// few items each is cut into parts of its own, so that no block has to change items: of `share` tiles at most, where share is the least that
// surely leaves no more parts than blocks (parts are at most total / share and one for each item).  Otherwise the tiles of all items are
// numbered through, items of a request one after the other, and block i takes those from i * share on: what it has of the item that
// it starts with and of the one that it ends with are parts of these.  A warp finds its block's tiles by a scan of the lengths.
struct Kv4Work {
  int b, item, tile0, n_tiles, parts;       // parts: of the item, where the block has it alone to itself; else 0
  long long left, share;
};
__device__ __forceinline__ int kv4_tiles(const Kv4Decode& a, int block, int tokens, int b) {
  return (min(max(a.seq_lens[b], 0), a.table_w * block) + tokens - 1) / tokens;
}
__device__ __forceinline__ long long kv4_ceil(long long x, long long by) {       // a 64-bit division takes as long as a load
  return ((x | by) >> 31) == 0 ? (long long)(((unsigned)x + (unsigned)by - 1) / (unsigned)by) : (x + by - 1) / by;
}
// Request that has unit i when request b has of(b) of them, and the units ahead of it; -1 behind the last
template <typename F>
__device__ __forceinline__ int kv4_find(int B, long long i, F of, long long& ahead) {
  const int lane = threadIdx.x & 31;
  ahead = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const long long mine = b0 + lane < B ? of(b0 + lane) : 0;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, ahead + upto > i);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      ahead += __shfl_sync(0xffffffffu, upto - mine, l);
      return b0 + l;
    }
    ahead += __shfl_sync(0xffffffffu, upto, 31);
  }
  return -1;
}
__device__ __forceinline__ bool kv4_work(const Kv4Decode& a, int block, int tokens, int items, int B, int least, Kv4Work& w) {
  long long all = 0;
  int busy = 0;
  for (int b = threadIdx.x & 31; b < B; b += 32) {
    const int n = kv4_tiles(a, block, tokens, b);
    all += n;
    busy += n > 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    busy += __shfl_xor_sync(0xffffffffu, busy, o);
  }
  all *= items;
  const long long some = (long long)busy * items, blocks = gridDim.x;
  long long ahead;
  if (some * 2 <= blocks) {                 // of 444 blocks, 32 uneven items take 14 us against 17 and 124 48 against 51; above half, waste
    w.share = max((long long)least, kv4_ceil(all, blocks - some));
    w.b = kv4_find(B, blockIdx.x, [&](int b) { return items * kv4_ceil(kv4_tiles(a, block, tokens, b), w.share); }, ahead);
    if (w.b < 0) return false;
    w.n_tiles = kv4_tiles(a, block, tokens, w.b);
    w.parts = (int)kv4_ceil(w.n_tiles, w.share);
    const int i = blockIdx.x - (int)ahead;
    w.item = i / w.parts;
    const int part = i - w.item * w.parts, each = w.n_tiles / w.parts, more = w.n_tiles - each * w.parts;
    w.tile0 = part * each + min(part, more);
    w.left = each + (part < more ? 1 : 0);
    return true;
  }
  w.parts = 0;
  w.share = max((long long)least, kv4_ceil(all, blocks));
  const long long g = blockIdx.x * w.share;
  if (g >= all) return false;
  w.b = kv4_find(B, g, [&](int b) { return (long long)items * kv4_tiles(a, block, tokens, b); }, ahead);
  w.n_tiles = kv4_tiles(a, block, tokens, w.b);
  w.item = (int)((g - ahead) / w.n_tiles);
  w.tile0 = (int)(g - ahead - (long long)w.item * w.n_tiles);
  w.left = min(w.share, all - g);
  return true;
}

// The codes minus 8 of the nibbles I of both halves of a word, as an fp16 pair, exactly.  Behind the exponent of 1024 a code in bits
// 0 .. 3 makes 1024 + code and one in bits 4 .. 7 makes 1024 + 16 code; the fp16 multiply-add that takes the offset off runs on
// another pipe than the integer operations.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t kv4_bits(uint32_t x) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(y) : "r"(x), "n"(MASK));      // (x & MASK) | 0x64006400
  return y;
}
template <int I>
__device__ __forceinline__ uint32_t kv4_code(uint32_t w) {
  if (I >= 2) w >>= 8;
  __half2 v;
  if (I & 1) {
    const uint32_t x = kv4_bits<0x00f000f0u>(w);
    v = __hfma2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
  } else {
    const uint32_t x = kv4_bits<0x000f000fu>(w);
    v = __hadd2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(-1032.f));
  }
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void kv4_mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// The same into d, from c
__device__ __forceinline__ void kv4_mma_from(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t kv4_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t kv4_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t kv4_max2(uint32_t x, uint32_t y) {             // of fp16 pairs; a NaN gives way to a number
  const __half2 v = __hmax2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void kv4_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
template <int N>
__device__ __forceinline__ void kv4_lds(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  }
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
}

template <int NG, bool VALUES, int TOK = NG == 4 ? 32 : 64>
struct Kv4Tile {
  static constexpr int PER = NG > 1 ? 2 : 1, PLANES = NG / PER;
  static constexpr int TOKENS = TOK;
  static constexpr int CODES = TOKENS * 32 * NG, SCALES = TOKENS * 4 * NG;
  static constexpr int V0 = CODES, KS0 = VALUES ? 2 * CODES : CODES, VS0 = KS0 + SCALES;
  static constexpr int BYTES = VALUES ? 2 * (CODES + SCALES) : CODES + SCALES;
  static constexpr int TOKEN_BYTES = BYTES / TOKENS;
  static constexpr int KINDS = VALUES ? 2 * PLANES + 2 : PLANES + 1;      // copies of a run of tokens
};

// The copies of a warp's tiles: lane l copies one kind of data (a plane of codes, the scales) of one run of `piece` tokens of a tile,
// which lies in one block.  The block ids of 32 runs are fetched by one load, another 32 runs ahead of their use: with the copies of
// all warps under way, a load that is waited for takes microseconds.
template <int NG, bool VALUES, int TOK = NG == 4 ? 32 : 64>
struct Kv4Feed {
  using T = Kv4Tile<NG, VALUES, TOK>;
  const uint8_t* base;              // of this lane's kind and head, in block 0
  long long blk_bytes;
  const int* table;
  int tok_bytes, dst, run;          // bytes a token, place in the stage, first token of the run in the tile (TOKENS: no copy)
  int off, step, step_off;          // token of the run in its block; tokens from one tile to the next, and what they are in a block
  int ids, ids_next;                // block ids of run lane % runs of step lane / runs, of these steps and the next ones
  int at, ahead;                    // steps of `ids` behind us; first token of the tile that ids_next starts with
  int runs;

  __device__ __forceinline__ int fetch(const Kv4Decode& a, const Kv4Cache& c, int first, int end) const {
    const int lane = threadIdx.x & 31, t = first + lane / runs * step + lane % runs * a.piece;
    return t < end && lane % runs * a.piece < T::TOKENS ? table[t / c.block] : -1;
  }
  __device__ __forceinline__ void init(const Kv4Decode& a, const Kv4Cache& c, int b, int h, int tile, int stride, int end) {
    const int lane = threadIdx.x & 31, kind = lane % T::KINDS;
    table = a.table + (long long)b * a.table_ld;
    step = stride * T::TOKENS;
    runs = a.piece >= T::TOKENS ? 1 : T::TOKENS / a.piece;
    at = 0;
    ids = fetch(a, c, tile * T::TOKENS, end);
    ahead = tile * T::TOKENS + 32 / runs * step;
    ids_next = fetch(a, c, ahead, end);
    run = min(lane / T::KINDS * a.piece, T::TOKENS);
    const bool values = VALUES && ((kind >= T::PLANES && kind < 2 * T::PLANES) || kind == 2 * T::PLANES + 1);
    const bool scales = kind >= (VALUES ? 2 : 1) * T::PLANES;
    const int plane = values ? kind - T::PLANES : kind;
    tok_bytes = scales ? 4 * NG : 32 * T::PER;
    base = (values ? c.v : c.k) + c.at(0, h) + (scales ? c.block * (32 * NG) : plane * c.block * (32 * T::PER));
    dst = scales ? (values ? T::VS0 : T::KS0) + run * (4 * NG) : (values ? T::V0 : 0) + (plane * T::TOKENS + run) * (32 * T::PER);
    blk_bytes = c.hkv * c.piece();
    step_off = step % c.block;
    off = (tile * T::TOKENS + run) % c.block;
  }
  // Start the copies of the tile in turn, `tokens` of it (a multiple of 16), and go on to the next one
  __device__ __forceinline__ void start(const Kv4Decode& a, const Kv4Cache& c, int tokens, int end, uint8_t* stage, uint64_t* bar, OmniStatus* st) {
    if ((threadIdx.x & 31) == 0) mbar_expect_tx(bar, tokens * T::TOKEN_BYTES);
    int blk = __shfl_sync(0xffffffffu, ids, at * runs + (threadIdx.x & 31) / T::KINDS % runs);
    if (run < tokens) {
      if (blk < 0 || blk >= c.blocks) {
        report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_DECODE, blk);
        blk = 0;                    // in bounds; the result is reported as wrong
      }
      kv4_bulk(smem_u32(stage) + dst, base + blk * blk_bytes + off * tok_bytes, min(a.piece, tokens - run) * tok_bytes, bar);
    }
    off += step_off;
    if (off >= c.block) off -= c.block;
    if (++at == 32 / runs) {
      at = 0;
      ids = ids_next;
      ahead += 32 / runs * step;
      ids_next = fetch(a, c, ahead, end);
    }
  }
};

// Fragments of 8 query rows (row r: query token r / rep, head h rep + r % rep) as fp16 numbers, each row times a power of two that
// brings its largest number to 2^13 .. 2^14: bf16 numbers keep all their bits down to 2^-26 of the largest.  qs are the sums of the
// groups, unit what brings scores to units of log 2 (its sign is that of the query), for the rows 2 c and 2 c + 1.
// Key codes of odd columns are left as 16 (64 + code): their queries are a 16th.  The products start from `base`, which takes off what
// the codes have too much: 64 for the odd columns, and too little: 8 for the even ones.
template <int NG>
struct Kv4Query {
  uint32_t b[NG][4][2];
  float qs[NG][2], base[NG][4], unit[2];
  // pairs of neighbouring columns as they are
  static __device__ __forceinline__ void fetch(const Kv4Decode& a, int rep, int b0, int h, int r, int total, uint32_t (&w)[NG][8]) {
    const int c = threadIdx.x & 3;
    const __nv_bfloat16* q = a.q + ((long long)b0 * a.rows + r / rep) * a.q_row + (long long)(h * rep + r % rep) * a.q_head + c * 16;
    if (r >= total) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[g][i] = 0u;
    } else if (a.q_wide) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(q + g * 64 + i * 8);
          w[g][4 * i] = v.x; w[g][4 * i + 1] = v.y; w[g][4 * i + 2] = v.z; w[g][4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[g][i] = (uint32_t)__bfloat16_as_ushort(q[g * 64 + 2 * i]) | (uint32_t)__bfloat16_as_ushort(q[g * 64 + 2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ void make(const uint32_t (&w)[NG][8], float scale_log2) {
    const int c = threadIdx.x & 3;
    float most = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[g][i] << 16)), fabsf(__uint_as_float(w[g][i] & 0xffff0000u))));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // exponent of the factor: 13 - that of the largest, within what a factor and its inverse can be
    const int e = min(max(13 - ((int)(__float_as_uint(most) >> 23) - 127), -120), 120);
    const float up = copysignf(__uint_as_float((uint32_t)(127 + e) << 23), scale_log2);
    const float exact = fabsf(scale_log2) * __uint_as_float((uint32_t)(127 - e) << 23), un = exact < 0x1p-120f ? 0x1p-120f : exact;      // a NaN stays one
    unit[0] = __shfl_sync(0xffffffffu, un, c * 8);
    unit[1] = __shfl_sync(0xffffffffu, un, c * 8 + 4);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float even = 0.f, odd = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {                                        // columns i, i + 4 and i + 1, i + 5 of a word, i = 2 (s & 1)
        const uint32_t u = w[g][(s >> 1) * 4 + (s & 1)], v = w[g][(s >> 1) * 4 + (s & 1) + 2];
        const float u0 = __uint_as_float(u << 16) * up, u1 = __uint_as_float(u & 0xffff0000u) * up;
        const float v0 = __uint_as_float(v << 16) * up, v1 = __uint_as_float(v & 0xffff0000u) * up;
        b[g][s][0] = kv4_pack(u0, v0);
        b[g][s][1] = kv4_pack(u1 * 0.0625f, v1 * 0.0625f);
        even += u0 + v0;
        odd += u1 + v1;
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        even += __shfl_xor_sync(0xffffffffu, even, d);
        odd += __shfl_xor_sync(0xffffffffu, odd, d);
      }
      const float sum = even + odd, from = fmaf(odd, -64.f, even * 8.f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        qs[g][x] = __shfl_sync(0xffffffffu, sum, c * 8 + 4 * x);
        base[g][x] = base[g][2 + x] = __shfl_sync(0xffffffffu, from, c * 8 + 4 * x);
      }
    }
  }
};

// Key codes of 16 tokens of a staged tile, minus 8 those of even columns and 16 (64 + code) those of odd ones
template <int NG, bool VALUES, int TOK = NG == 4 ? 32 : 64>
struct Kv4Keys {
  using T = Kv4Tile<NG, VALUES, TOK>;
  uint32_t w[T::PLANES][2][2 * T::PER], sc[2][NG];
  __device__ __forceinline__ void load(const uint8_t* stage, int sub) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      kv4_lds<NG>(sc[e], stage + T::KS0 + (sub * 16 + r + 8 * e) * (4 * NG));
#pragma unroll
      for (int p = 0; p < T::PLANES; ++p)
        kv4_lds<2 * T::PER>(w[p][e], stage + (p * T::TOKENS + sub * 16 + r + 8 * e) * (32 * T::PER) + c * (8 * T::PER));
    }
  }
  __device__ __forceinline__ void fragment(int g, int s, uint32_t (&a)[4]) const {       // s: 16 columns of the group
    const uint32_t w0 = w[g / T::PER][0][g % T::PER * 2 + (s >> 1)], w1 = w[g / T::PER][1][g % T::PER * 2 + (s >> 1)];
    if (s & 1) {
      a[0] = kv4_code<2>(w0); a[1] = kv4_code<2>(w1); a[2] = kv4_bits<0x00f000f0u>(w0 >> 8); a[3] = kv4_bits<0x00f000f0u>(w1 >> 8);
    } else {
      a[0] = kv4_code<0>(w0); a[1] = kv4_code<0>(w1); a[2] = kv4_bits<0x00f000f0u>(w0); a[3] = kv4_bits<0x00f000f0u>(w1);
    }
  }
};

// Adds a group's part to the scores of tokens r and r + 8 and rows 2 c and 2 c + 1
__device__ __forceinline__ void kv4_score(float (&s)[4], const float (&acc)[4], const uint32_t (&word)[2], const float (&qs)[2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float step = kv4_step(word[e]), low = kv4_low(word[e]);
#pragma unroll
    for (int x = 0; x < 2; ++x) s[2 * e + x] = fmaf(step, acc[2 * e + x], fmaf(low, qs[x], s[2 * e + x]));
  }
}

// What a warp carries along the cache for its query rows: running maxima, sums of weights, and the two parts of the result
template <int NG, int NT>
struct Kv4Sums {
  using T = Kv4Tile<NG, true>;
  static constexpr int HALF = 32, SUBS = HALF / 16;
  float m[NT][2], l[NT][2], o[NT][NG][4][4], z[NT][NG][2];                 // m in the scores' own units
  // o is in units of 1 / c: the largest of a row's weights times a group's steps becomes an fp16 number of 2^7 .. 2^15, whatever other rows, groups
  // and tokens without weight have.  One factor for all, by the largest step, is 4% faster (2 x 131,067 tokens: 80.5 us against 84), but takes the
  // codes from a group beside one 2^24 times as large, and from all tokens behind one that is and has no weight.
  float c[NT][2][NG];
  static constexpr float C_MOST = 0x1p118f;                                // times a weight still finite

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[n][x] = -INFINITY;
        l[n][x] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          z[n][g][x] = 0.f;
          c[n][x][g] = C_MOST;                                             // what the first tokens have lowers it
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][g][j][x] = o[n][g][j][x + 2] = 0.f;
        }
      }
  }

  // 32 tokens from `t0` on, from sub `sub0` of the stage.  EDGE: some row does not see all of them.  KEEP: scores go to memory as well.
  template <bool EDGE, bool KEEP>
  __device__ __forceinline__ void add(const uint8_t* stage, int sub0, int t0, int end, const int (&sees)[NT][2], const Kv4Query<NG> (&q)[NT], float* scores) {
    const int lane = threadIdx.x & 31, r = lane >> 2, cc = lane & 3;
    float s[SUBS][NT][4], top[NT][2];
    uint32_t vs[SUBS][2][NG];
#pragma unroll
    for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      Kv4Keys<NG, true> k;
      k.load(stage, sub0 + u);
#pragma unroll
      for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[NT][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t f[4];
          k.fragment(g, x, f);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (x == 0) kv4_mma_from(acc[n], f, q[n].b[g][x], q[n].base[g]);
            else kv4_mma(acc[n], f, q[n].b[g][x]);
          }
        }
        const uint32_t word[2] = {k.sc[0][g], k.sc[1][g]};
#pragma unroll
        for (int n = 0; n < NT; ++n) kv4_score(s[u][n], acc[n], word, q[n].qs[g]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = t0 + u * 16 + r + 8 * e;
        kv4_lds<NG>(vs[u][e], stage + T::VS0 + ((sub0 + u) * 16 + r + 8 * e) * (4 * NG));
        if (EDGE) {
          if (t >= end) {                                                  // what lies there is not of this request
#pragma unroll
            for (int g = 0; g < NG; ++g) vs[u][e][g] = 0u;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (t >= sees[n][x]) s[u][n][2 * e + x] = -INFINITY;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) top[n][x] = fmaxf(top[n][x], fmaxf(s[u][n][x], s[u][n][2 + x]));
    }
    if (KEEP) {
#pragma unroll
      for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float2*>(scores + (long long)(t0 + u * 16 + r + 8 * e) * (8 * NT) + n * 8 + cc * 2) =
                make_float2(s[u][n][2 * e] * q[n].unit[0], s[u][n][2 * e + 1] * q[n].unit[1]);
    }
    // The maximum is followed only when a score exceeds it by 2^8: weights in fp32 bear that.
    bool more = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) more |= (top[n][0] - m[n][0]) * q[n].unit[0] > 8.f || (top[n][1] - m[n][1]) * q[n].unit[1] > 8.f;
    if (__any_sync(0xffffffffu, more)) rescale(top, q);
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float sub = EDGE && m[n][x] == -INFINITY ? 0.f : m[n][x] * q[n].unit[x];
          s[u][n][x] = ex2_fast(fmaf(s[u][n][x], q[n].unit[x], -sub));
          s[u][n][2 + x] = ex2_fast(fmaf(s[u][n][2 + x], q[n].unit[x], -sub));
          if (EDGE) {                                                      // whatever the scale is
            if (t0 + u * 16 + r >= sees[n][x]) s[u][n][x] = 0.f;
            if (t0 + u * 16 + r + 8 >= sees[n][x]) s[u][n][2 + x] = 0.f;
          }
          l[n][x] += s[u][n][x] + s[u][n][2 + x];
        }
    }
    uint32_t pt[SUBS][NG][NT][2], most = 0u;
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float step = kv4_step(vs[u][e][g]), mid = fmaf(step, 8.f, kv4_low(vs[u][e][g]));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float p0 = s[u][n][2 * e], p1 = s[u][n][2 * e + 1];
            if (EDGE) {                                                    // an unseen token adds nothing, whatever its value
              const int t = t0 + u * 16 + r + 8 * e;
              z[n][g][0] += t < sees[n][0] ? p0 * mid : 0.f;
              z[n][g][1] += t < sees[n][1] ? p1 * mid : 0.f;
            } else {
              z[n][g][0] = fmaf(p0, mid, z[n][g][0]);
              z[n][g][1] = fmaf(p1, mid, z[n][g][1]);
            }
            pt[u][g][n][e] = product<EDGE>(p0, p1, step, n, g, t0 + u * 16 + r + 8 * e, sees);
            most = kv4_max2(most, pt[u][g][n][e]);
          }
        }
    // One of 2^15 or more.  Weights and products ahead of a single vote for maxima and factors were slower (more registers, or scores made again).
    if (__any_sync(0xffffffffu, ((most + 0x08000800u) & 0x80008000u) != 0u)) {
      lower(s, vs);
#pragma unroll
      for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              pt[u][g][n][e] = product<EDGE>(s[u][n][2 * e], s[u][n][2 * e + 1], kv4_step(vs[u][e][g]), n, g, t0 + u * 16 + r + 8 * e, sees);
    }
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
#pragma unroll
      for (int p = 0; p < T::PLANES; ++p) {
        uint32_t w[2][2 * T::PER];                                         // pairs of tokens c and c + 4: even (groups), odd (groups)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int pair = cc + 4 * e;
          const int ch = T::PER == 2 ? r ^ ((pair & 3) << 1) : r ^ (((pair >> 1) & 1) << 2);
          kv4_lds<2 * T::PER>(w[e], stage + T::V0 + (p * T::TOKENS + (sub0 + u) * 16 + pair * 2) * (32 * T::PER) + ch * (8 * T::PER));
        }
#pragma unroll
        for (int gp = 0; gp < T::PER; ++gp) {
          const int g = p * T::PER + gp;
          uint32_t b[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) b[n][e] = kv4_transpose(pt[u][g][n][e]);
          const uint32_t x0 = __byte_perm(w[0][gp], w[0][T::PER + gp], 0x5410), y0 = __byte_perm(w[0][gp], w[0][T::PER + gp], 0x7632);
          const uint32_t x1 = __byte_perm(w[1][gp], w[1][T::PER + gp], 0x5410), y1 = __byte_perm(w[1][gp], w[1][T::PER + gp], 0x7632);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t v0 = j < 2 ? x0 : y0, v1 = j < 2 ? x1 : y1;
            const uint32_t f[4] = {j & 1 ? kv4_code<2>(v0) : kv4_code<0>(v0), j & 1 ? kv4_code<3>(v0) : kv4_code<1>(v0),
                                   j & 1 ? kv4_code<2>(v1) : kv4_code<0>(v1), j & 1 ? kv4_code<3>(v1) : kv4_code<1>(v1)};
#pragma unroll
            for (int n = 0; n < NT; ++n) kv4_mma(o[n][g][j], f, b[n]);
          }
        }
      }
    }
  }

  // step p of rows 2 c and 2 c + 1, a token that is not seen has 0 whatever its value
  template <bool EDGE>
  __device__ __forceinline__ uint32_t product(float p0, float p1, float step, int n, int g, int t, const int (&sees)[NT][2]) const {
    float f0 = p0 * c[n][0][g] * step, f1 = p1 * c[n][1][g] * step;
    if (EDGE) {
      f0 = t < sees[n][0] ? f0 : 0.f;
      f1 = t < sees[n][1] ? f1 : 0.f;
    }
    return kv4_pack(f0, f1);
  }
  // Where 32 tokens have products of 2^14 or more, the largest of them becomes 2^7 .. 2^8
  __device__ __forceinline__ void lower(const float (&p)[SUBS][NT][4], const uint32_t (&vs)[SUBS][2][NG]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float v = 0.f;
#pragma unroll
          for (int u = 0; u < SUBS; ++u) v = fmaxf(v, fmaxf(p[u][n][x] * kv4_step(vs[u][0][g]), p[u][n][2 + x] * kv4_step(vs[u][1][g])));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
          if (v * c[n][x][g] >= 0x1p14f) {
            const float next = __uint_as_float((261u - (__float_as_uint(v) >> 23)) << 23), by = next * rcp_fast(c[n][x][g]);
            c[n][x][g] = next;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[n][g][j][x] *= by;
              o[n][g][j][x + 2] *= by;
            }
          }
        }
  }

  // New maxima.  o stays as it is while c can grow by what the weights lose.
  __device__ __forceinline__ void rescale(const float (&top)[NT][2], const Kv4Query<NG> (&q)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v = top[n][x];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
        v = fmaxf(v, m[n][x]);
        const float f = v == -INFINITY ? 1.f : ex2_fast((m[n][x] - v) * q[n].unit[x]), up = v == -INFINITY ? 1.f : ex2_fast((v - m[n][x]) * q[n].unit[x]);
        m[n][x] = v;
        l[n][x] *= f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          z[n][g][x] *= f;
          const float next = c[n][x][g] * up;
          if (next < C_MOST) {
            c[n][x][g] = next;
          } else {
            const float by = f * C_MOST * rcp_fast(c[n][x][g]);
            c[n][x][g] = C_MOST;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[n][g][j][x] *= by;
              o[n][g][j][x + 2] *= by;
            }
          }
        }
      }
  }
};

template <int NG, int NT, bool KEEP>
__global__ void __launch_bounds__(KV4_WARPS * 32, NT * NG > 2 ? 2 : 3) kv4_decode_kernel(Kv4Decode a, Kv4Cache c, int B, OmniStatus* st) {
  using T = Kv4Tile<NG, true>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[KV4_WARPS * KV4_STAGES];
  __shared__ int abort_flag;
  constexpr int D = NG * 64, NQ = 8 * NT;
  const int rep = a.hq / c.hkv, total = a.rows * rep, chunks = (total + NQ - 1) / NQ, items = c.hkv * chunks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cc = lane & 3;
  uint8_t* stages = smem + warp * (KV4_STAGES * T::BYTES);
  uint64_t* bar = bars + warp * KV4_STAGES;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < KV4_STAGES; ++s) mbar_init(bar + s, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;");

  Kv4Work w;
  if (a.min_tiles == 0) {
    w.b = blockIdx.x / items;
    w.item = blockIdx.x - w.b * items;
    w.tile0 = w.parts = 0;
    w.left = w.n_tiles = kv4_tiles(a, c.block, T::TOKENS, w.b);
  } else if (!kv4_work(a, c.block, T::TOKENS, items, B, a.min_tiles, w)) {
    return;
  }
  int uses = 0, turn = 0;                                                  // of this warp's stages so far; the warp that the next tile falls to
  for (bool first = true;; first = false) {
    const int b = w.b, h = w.item / chunks, row0 = (w.item - h * chunks) * NQ, tile0 = w.tile0, n_tiles = w.n_tiles;
    const int len = kv4_length(a, c.block, b, st);
    const int first_sees = len - a.rows + 1 + row0 / rep;                  // of the item's first and last rows
    const int end = len - a.rows + 1 + (min(total, row0 + NQ) - 1) / rep;
    const int end_tile = (int)min((long long)n_tiles, tile0 + w.left);
    if (a.min_tiles != 0 && tile0 == 0 && threadIdx.x == 0) {              // the blocks behind this one take a share each of what is left
      const int parts = w.parts > 0 ? w.parts : end_tile == n_tiles ? 1 : 1 + (int)kv4_ceil(n_tiles - end_tile, w.share);
      a.shared[(long long)b * items + w.item] = make_int2(2 * blockIdx.x + (first ? 0 : 1), parts);
    }
    const int stop = min(end, end_tile * T::TOKENS);                       // first token behind this part
    const int stop_tile = stop > 0 ? (stop + T::TOKENS - 1) / T::TOKENS : 0;
    int tile = tile0 + ((warp - turn) & (KV4_WARPS - 1)), next = tile;
    Kv4Feed<NG, true> feed;
    feed.init(a, c, b, h, tile, KV4_WARPS, stop);
    uint32_t raw[NT][NG][8];                                               // asked for ahead of the copies, which would hold them up
#pragma unroll
    for (int n = 0; n < NT; ++n) Kv4Query<NG>::fetch(a, rep, b, h, row0 + n * 8 + r, total, raw[n]);
#pragma unroll
    for (int s = 0; s < KV4_STAGES; ++s, next += KV4_WARPS) {
      const int i = (uses + s) % KV4_STAGES;
      if (next < stop_tile) feed.start(a, c, min(T::TOKENS, (end - next * T::TOKENS + 15) & ~15), stop, stages + i * T::BYTES, bar + i, st);
    }
    Kv4Query<NG> q[NT];
    int sees[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      q[n].make(raw[n], a.scale_log2);
#pragma unroll
      for (int x = 0; x < 2; ++x) sees[n][x] = len - a.rows + 1 + min(row0 + n * 8 + cc * 2 + x, total - 1) / rep;
    }
    float* scores = KEEP ? a.scores + ((long long)b * items + w.item) * a.score_places * NQ : nullptr;
    Kv4Sums<NG, NT> sum;
    sum.clear();
    for (; tile < stop_tile; tile += KV4_WARPS, next += KV4_WARPS, ++uses) {
      const int i = uses % KV4_STAGES;
      uint8_t* stage = stages + i * T::BYTES;
      if (!__all_sync(0xffffffffu, mbar_wait(bar + i, (uses / KV4_STAGES) & 1, &abort_flag, st, KV4_SITE_TILE, tile))) break;
#pragma unroll 1
      for (int sub = 0; sub < T::TOKENS / 16; sub += 2) {
        const int t0 = tile * T::TOKENS + sub * 16;
        if (t0 + 32 <= first_sees) sum.template add<false, KEEP>(stage, sub, t0, end, sees, q, scores);
        else if (t0 < end) sum.template add<true, KEEP>(stage, sub, t0, end, sees, q, scores);
      }
      __syncwarp();                                                        // every lane has read the stage
      if (next < stop_tile) feed.start(a, c, min(T::TOKENS, (end - next * T::TOKENS + 15) & ~15), stop, stage, bar + i, st);
    }

    // ---- the sums over the lanes that share a query row, then over the warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          sum.l[n][x] += __shfl_xor_sync(0xffffffffu, sum.l[n][x], d);
#pragma unroll
          for (int g = 0; g < NG; ++g) sum.z[n][g][x] += __shfl_xor_sync(0xffffffffu, sum.z[n][g][x], d);
        }
    __syncthreads();
    if (abort_flag != 0) {                                                 // copies may still be under way: leave the memory alone
      if (threadIdx.x == 0) report_abort(&abort_flag, st);
      for (int s = 0; s < KV4_STAGES; ++s) {
        const int i = uses + s;                                            // what this warp has started and not seen: its phases
        if (tile + s * KV4_WARPS < stop_tile) {
          for (int k = 0; k < 1 << 16 && !mbar_try_wait(bar + i % KV4_STAGES, (i / KV4_STAGES) & 1); ++k) {}
        }
      }
      return;
    }
    float* s_o = reinterpret_cast<float*>(smem);                           // [warps][NQ][D]
    float* s_m = s_o + KV4_WARPS * NQ * D;                                 // [warps][NQ], and the sums likewise
    float* s_l = s_m + KV4_WARPS * NQ;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int i = warp * NQ + n * 8 + cc * 2 + x;
        if (r == 0) {
          s_m[i] = sum.m[n][x] == -INFINITY ? -INFINITY : sum.m[n][x] * q[n].unit[x];
          s_l[i] = sum.l[n][x];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float unit = 1.f / sum.c[n][x][g];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(s_o + (size_t)i * D + g * 64 + r * 8 + j * 2) =
                make_float2(fmaf(sum.o[n][g][j][x], unit, sum.z[n][g][x]), fmaf(sum.o[n][g][j][x + 2], unit, sum.z[n][g][x]));
        }
      }
    __syncthreads();
    const bool whole = tile0 == 0 && end_tile == n_tiles;
    if (threadIdx.x < NQ) {                                                // a warp's factor in place of its maximum; 1 / sum and sum
      const int row = threadIdx.x;
      float mm = -INFINITY, total_l = 0.f;
#pragma unroll
      for (int w = 0; w < KV4_WARPS; ++w) mm = fmaxf(mm, s_m[w * NQ + row]);
#pragma unroll
      for (int w = 0; w < KV4_WARPS; ++w) {
        const float mw = s_m[w * NQ + row], lw = s_l[w * NQ + row];
        const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : ex2_fast(mw - mm);       // a sum without a maximum is NaN
        s_m[w * NQ + row] = f;
        total_l += lw * f;
      }
      s_l[row] = total_l == 0.f ? 0.f : 1.f / total_l;
      const float lse = total_l == 0.f ? -INFINITY : mm + __log2f(total_l);
      if (row0 + row < total) {
        const int head = h * rep + (row0 + row) % rep, tok = (row0 + row) / rep;
        if (!whole) a.lse_part[((long long)blockIdx.x * 2 + (first ? 0 : 1)) * NQ + row] = lse;
        else if (a.lse != nullptr) a.lse[((long long)b * a.hq + head) * a.rows + tok] = lse;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NQ * D / 4; i += KV4_WARPS * 32) {
      const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
      if (row0 + row >= total) break;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KV4_WARPS; ++w) {
        const float f = s_m[w * NQ + row];
        const float4 v = *reinterpret_cast<const float4*>(s_o + ((size_t)w * NQ + row) * D + d);
        acc[0] = fmaf(v.x, f, acc[0]);
        acc[1] = fmaf(v.y, f, acc[1]);
        acc[2] = fmaf(v.z, f, acc[2]);
        acc[3] = fmaf(v.w, f, acc[3]);
      }
      const float by = s_l[row];
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[x] = by == 0.f ? 0.f : acc[x] * by;
      if (whole) {
        const int head = h * rep + (row0 + row) % rep, tok = (row0 + row) / rep;
        const __nv_bfloat162 lo = __floats2bfloat162_rn(acc[0], acc[1]), hi = __floats2bfloat162_rn(acc[2], acc[3]);
        *reinterpret_cast<uint2*>(a.out + (((long long)b * a.rows + tok) * a.hq + head) * D + d) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        *reinterpret_cast<float4*>(a.o_part + (((long long)blockIdx.x * 2 + (first ? 0 : 1)) * NQ + row) * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      }
    }
    // ---- the next item
    w.left -= end_tile - tile0;
    if (w.left <= 0) return;
    turn += max(0, stop_tile - tile0);
    w.tile0 = 0;
    if (++w.item == items) {
      w.item = 0;
      do w.n_tiles = kv4_tiles(a, c.block, T::TOKENS, ++w.b);              // tiles are left, so there is a request that has some
      while (w.n_tiles == 0);
    }
    fence_proxy_async_smem();                                              // the sums in shared memory come before the next copies
    __syncthreads();
  }
}

// Items that several blocks have worked on, and requests of no tokens: one block for a query row and head, a thread a column.
template <int NT>
__global__ void __launch_bounds__(256) kv4_join_kernel(Kv4Decode a, Kv4Cache c, int blocks) {
  constexpr int NQ = 8 * NT;
  extern __shared__ float s_f[];                                           // [blocks]
  asm volatile("griddepcontrol.launch_dependents;");
  const int rep = a.hq / c.hkv, total = a.rows * rep, chunks = (total + NQ - 1) / NQ;
  const int h = blockIdx.x / total, row = blockIdx.x - h * total, b = blockIdx.y, d = threadIdx.x, lane = d & 31;
  const int head = h * rep + row % rep, tok = row / rep;
  const bool none = a.table_w == 0 || a.seq_lens[b] <= 0;
  // Every block waits, those without work too: a kernel that follows this one may then count on the one ahead of it being done.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int2 shared = none ? make_int2(0, 0) : a.shared[((long long)b * c.hkv + h) * chunks + row / NQ];
  // after a wait that ran out it may be anything
  const int parts = shared.x >= 0 && shared.y >= 0 && shared.x / 2 + shared.y <= blocks ? shared.y : 0;
  if (parts == 1) return;                                                  // written by its only block
  // the first part is where its block says, those of the blocks behind it are their first ones
  const int first = shared.x, next = (first | 1) + 1, in = row % NQ;
  auto slot = [&](int s) -> long long { return (long long)(s == 0 ? first : next + 2 * (s - 1)) * NQ + in; };
  constexpr int AHEAD = 16;                                                // partial results that are asked for together with the sums
  float v[AHEAD];
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) v[s] = s < parts ? a.o_part[slot(s) * c.d + d] : 0.f;
  // every warp finds the maximum and the sum of the parts by itself
  float mm = -INFINITY, sum = 0.f;
  for (int s = lane; s < parts; s += 32) mm = fmaxf(mm, a.lse_part[slot(s)]);
  mm = warp_max(mm);
  for (int s = lane; s < parts; s += 32) {
    const float x = a.lse_part[slot(s)], f = x == -INFINITY ? 0.f : exp2f(x - mm);
    sum += f;
    if (d < 32) s_f[s] = f;
  }
  sum = warp_sum(sum);
  __syncthreads();
  float acc = 0.f;                                                         // a part that sees nothing is 0; 0 times a NaN that is seen is NaN
#pragma unroll
  for (int s = 0; s < AHEAD; ++s)
    if (s < parts) acc = fmaf(s_f[s], v[s], acc);
#pragma unroll 8
  for (int s = AHEAD; s < parts; ++s) acc = fmaf(s_f[s], a.o_part[slot(s) * c.d + d], acc);
  a.out[(((long long)b * a.rows + tok) * a.hq + head) * c.d + d] = __float2bfloat16(sum == 0.f ? 0.f : acc / sum);
  if (d == 0 && a.lse != nullptr) a.lse[((long long)b * a.hq + head) * a.rows + tok] = sum == 0.f ? -INFINITY : mm + __log2f(sum);
}

// The weights that the rows give a request's tokens by kept scores and the finished sums.  With one tile of 8 rows a lane takes a token (32 requests of
// up to 4099 tokens: 9 us, by two lanes a token 12), with tiles of 16 rows 4 of them, so that a warp reads 512 bytes in a row (128 rows, 30,011
// tokens twice: 36 us, by a lane a token 39).
template <int NQ>
__global__ void __launch_bounds__(256) kv4_add_kernel(Kv4Decode a, Kv4Cache c) {
  constexpr int LANES = NQ == 8 ? 1 : NQ / 4, TOKENS = 256 / LANES, EACH = NQ / LANES / 4;
  __shared__ __align__(16) float s_lse[256 + NQ];
  const int rep = a.hq / c.hkv, total = a.rows * rep, chunks = (total + NQ - 1) / NQ;
  const int h = blockIdx.y, b = blockIdx.z, part = threadIdx.x % LANES;
  const int len = min(max(a.seq_lens[b], 0), a.table_w * c.block);          // longer ones are reported by the kernel ahead
  int t = blockIdx.x * TOKENS + threadIdx.x / LANES;
  float *to, old;
  auto look = [&] {
    const int blk = t < len ? a.table[(long long)b * a.table_ld + t / c.block] : -1;
    to = blk >= 0 && blk < c.blocks ? a.weights + ((long long)blk * c.hkv + h) * c.block + t % c.block : nullptr;
    old = to != nullptr && a.decay != 0.f ? *to : 0.f;
  };
  look();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x * TOKENS >= len) return;
  for (int row = threadIdx.x; row < chunks * NQ; row += 256)                // rows beyond the last have a weight of 0
    s_lse[row] = row < total ? a.lse[((long long)b * a.hq + h * rep + row % rep) * a.rows + row / rep] : INFINITY;
  __syncthreads();
  const int all_see = len - a.rows + 1;                                     // tokens that every row sees
  const float* scores = a.scores + ((long long)b * c.hkv + h) * chunks * a.score_places * NQ + part * (EACH * 4);
  for (; t - (int)threadIdx.x / LANES < len; t += gridDim.x * TOKENS, look()) {
    float sum = 0.f;
    if (t < len) {
#pragma unroll 4
      for (int ch = 0; ch < chunks; ++ch) {
        const float4* from = reinterpret_cast<const float4*>(scores + ((long long)ch * a.score_places + t) * NQ);
        float4 v[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) v[j] = from[j];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          const int row = ch * NQ + (part * EACH + j) * 4;
          const float4 l = *reinterpret_cast<const float4*>(s_lse + row);
          float p[4] = {ex2_fast(v[j].x - l.x), ex2_fast(v[j].y - l.y), ex2_fast(v[j].z - l.z), ex2_fast(v[j].w - l.w)};
          if (t >= all_see) {                                               // scores that are not there are dropped as well
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (row + x >= total || t >= all_see + (row + x) / rep) p[x] = 0.f;
          }
          sum += (p[0] + p[1]) + (p[2] + p[3]);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (part == 0 && to != nullptr) *to = a.decay == 0.f ? sum : fmaf(a.decay, old, sum);
  }
}

// The same without kept scores: those of the staged keys once more, against the finished sums.  32 tokens (16 at d = 256) are unpacked
// once for all rows, whose fragments stand in shared memory.  128 rows a key/value head over 30,011 tokens twice take 55 us (16 tokens at a time,
// one product and one row after the other: 67), bound by the latencies of 12 warps an SM: issue slots are 38% full, tensor pipes 36%.
template <int NG, int TOK>
__global__ void __launch_bounds__(KV4_WARPS * 32, 3) kv4_weights_kernel(Kv4Decode a, Kv4Cache c, int B, OmniStatus* st) {
  using T = Kv4Tile<NG, false, TOK>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[KV4_WARPS * KV4_STAGES];
  __shared__ int abort_flag;
  __shared__ float s_w[KV4_WARPS][TOK];
  constexpr int ROW = 1 + NG, EACH = TOK / 32, SUBS = NG == 4 ? 1 : 2;
  const int rep = a.hq / c.hkv, total = a.rows * rep, chunks = (total + 7) / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cc = lane & 3;
  uint8_t* stages = smem + warp * (KV4_STAGES * T::BYTES);
  uint4* s_q = reinterpret_cast<uint4*>(smem + KV4_WARPS * KV4_STAGES * T::BYTES);      // [chunks][NG][2][32]
  float4* s_row = reinterpret_cast<float4*>(s_q + chunks * NG * 64);                     // [chunks][ROW][4]: see below
  uint64_t* bar = bars + warp * KV4_STAGES;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int s = 0; s < KV4_STAGES; ++s) mbar_init(bar + s, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncthreads();
  Kv4Work w;
  if (!kv4_work(a, c.block, TOK, c.hkv, B, KV4_WARPS, w)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");                    // as in the join
    return;
  }
  int uses = 0, turn = 0;
  for (bool first = true;; first = false) {
    const int b = w.b, h = w.item, tile0 = w.tile0;
    const int len = kv4_length(a, c.block, b, st), end_tile = (int)min((long long)w.n_tiles, tile0 + w.left), stop = min(len, end_tile * TOK);
    int tile = tile0 + ((warp - turn) & (KV4_WARPS - 1)), next = tile;
    Kv4Feed<NG, false, TOK> feed;
    feed.init(a, c, b, h, tile, KV4_WARPS, stop);
#pragma unroll
    for (int s = 0; s < KV4_STAGES; ++s, next += KV4_WARPS) {
      const int i = (uses + s) % KV4_STAGES;
      if (next < end_tile) feed.start(a, c, min(TOK, (len - next * TOK + 15) & ~15), stop, stages + i * T::BYTES, bar + i, st);
    }
    // the blocks of a lane's tokens of the next tile
    int place[EACH];
    auto look = [&](int of) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int t = of * TOK + i * 32 + lane;
        place[i] = t < stop ? a.table[(long long)b * a.table_ld + t / c.block] : -1;
      }
    };
    look(tile);
    for (int ch = warp; ch < chunks; ch += KV4_WARPS) {
      Kv4Query<NG> q;
      uint32_t raw[NG][8];
      Kv4Query<NG>::fetch(a, rep, b, h, ch * 8 + r, total, raw);
      q.make(raw, a.scale_log2);
#pragma unroll
      for (int g2 = 0; g2 < NG; ++g2)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          s_q[(ch * NG * 2 + g2 * 2 + x) * 32 + lane] = make_uint4(q.b[g2][2 * x][0], q.b[g2][2 * x][1], q.b[g2][2 * x + 1][0], q.b[g2][2 * x + 1][1]);
      if (r == 0) {                 // of the rows 2 c and 2 c + 1: minus their sums (below), their units, and for each group qs and base
        s_row[(ch * ROW) * 4 + cc] = make_float4(-INFINITY, -INFINITY, q.unit[0], q.unit[1]);
#pragma unroll
        for (int g2 = 0; g2 < NG; ++g2) s_row[(ch * ROW + 1 + g2) * 4 + cc] = make_float4(q.qs[g2][0], q.qs[g2][1], q.base[g2][0], q.base[g2][1]);
      }
    }
    __syncthreads();
    if (first) asm volatile("griddepcontrol.wait;" ::: "memory");         // the sums are there
    for (int row = threadIdx.x; row < total; row += KV4_WARPS * 32)
      reinterpret_cast<float*>(&s_row[(row / 8 * ROW) * 4 + row % 8 / 2])[row & 1] = -a.lse[((long long)b * a.hq + h * rep + row % rep) * a.rows + row / rep];
    __syncthreads();
    for (; tile < end_tile; tile += KV4_WARPS, next += KV4_WARPS, ++uses) {
      const int st_i = uses % KV4_STAGES;
      uint8_t* stage = stages + st_i * T::BYTES;
      float* to[EACH];
      float old[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int t = tile * TOK + i * 32 + lane;
        to[i] = place[i] >= 0 && place[i] < c.blocks ? a.weights + ((long long)place[i] * c.hkv + h) * c.block + t % c.block : nullptr;
        old[i] = to[i] != nullptr && a.decay != 0.f ? *to[i] : 0.f;
      }
      look(tile + KV4_WARPS);
      if (!__all_sync(0xffffffffu, mbar_wait(bar + st_i, (uses / KV4_STAGES) & 1, &abort_flag, st, KV4_SITE_WEIGHTS, tile))) break;
#pragma unroll 1
      for (int u = 0; u < TOK / 16; u += SUBS) {
        const int t0 = tile * TOK + u * 16;
        if (t0 >= len) break;
        uint32_t f[SUBS][NG][4][4];
        f32x2 step[SUBS][2][NG], low[SUBS][2][NG], sum[SUBS][2];
#pragma unroll
        for (int x = 0; x < SUBS; ++x) {
          Kv4Keys<NG, false, TOK> k;
          k.load(stage, u + x);
#pragma unroll
          for (int g2 = 0; g2 < NG; ++g2) {
#pragma unroll
            for (int y = 0; y < 4; ++y) k.fragment(g2, y, f[x][g2][y]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              step[x][e][g2] = pack_f32x2(kv4_step(k.sc[e][g2]), kv4_step(k.sc[e][g2]));
              low[x][e][g2] = pack_f32x2(kv4_low(k.sc[e][g2]), kv4_low(k.sc[e][g2]));
            }
          }
          sum[x][0] = sum[x][1] = 0ull;
        }
        // EDGE: some row does not see all of these tokens.  Rows beyond the last have a weight of 0 by their sums.
        auto rows = [&](auto edge) {
#pragma unroll 1
          for (int ch = 0; ch < chunks; ++ch) {
            const float4 row = s_row[ch * ROW * 4 + cc];
            f32x2 s[SUBS][2];
#pragma unroll
            for (int g2 = 0; g2 < NG; ++g2) {
              const float4 sums = s_row[(ch * ROW + 1 + g2) * 4 + cc];
              const float base[4] = {sums.z, sums.w, sums.z, sums.w};
              const f32x2 qs = pack_f32x2(sums.x, sums.y);
              const uint4 v0 = s_q[(ch * NG * 2 + g2 * 2) * 32 + lane], v1 = s_q[(ch * NG * 2 + g2 * 2 + 1) * 32 + lane];
              const uint32_t bq[4][2] = {{v0.x, v0.y}, {v0.z, v0.w}, {v1.x, v1.y}, {v1.z, v1.w}};
              float acc[SUBS][4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int x = 0; x < SUBS; ++x) {
                  if (y == 0) kv4_mma_from(acc[x], f[x][g2][y], bq[y], base);
                  else kv4_mma(acc[x], f[x][g2][y], bq[y]);
                }
#pragma unroll
              for (int x = 0; x < SUBS; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  s[x][e] = fma_f32x2(step[x][e][g2], pack_f32x2(acc[x][2 * e], acc[x][2 * e + 1]), fma_f32x2(low[x][e][g2], qs, g2 == 0 ? 0ull : s[x][e]));
            }
#pragma unroll
            for (int x = 0; x < SUBS; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float p[2];
                unpack_f32x2(fma_f32x2(s[x][e], pack_f32x2(row.z, row.w), pack_f32x2(row.x, row.y)), p[0], p[1]);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  p[y] = ex2_fast(p[y]);
                  if (decltype(edge)::value) {
                    const int i = ch * 8 + cc * 2 + y;
                    if (i >= total || t0 + x * 16 + r + 8 * e >= len - a.rows + 1 + i / rep) p[y] = 0.f;
                  }
                }
                sum[x][e] = add_f32x2(sum[x][e], pack_f32x2(p[0], p[1]));
              }
          }
        };
        if (t0 + SUBS * 16 > len - a.rows + 1) rows(std::true_type{});
        else rows(std::false_type{});
#pragma unroll
        for (int x = 0; x < SUBS; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float p0, p1;
            unpack_f32x2(sum[x][e], p0, p1);
            p0 += p1;
            p0 += __shfl_xor_sync(0xffffffffu, p0, 1);
            p0 += __shfl_xor_sync(0xffffffffu, p0, 2);
            if (cc == 0) s_w[warp][(u + x) * 16 + r + 8 * e] = p0;
          }
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (to[i] != nullptr) *to[i] = a.decay == 0.f ? s_w[warp][i * 32 + lane] : fmaf(a.decay, old[i], s_w[warp][i * 32 + lane]);
      __syncwarp();
      if (next < end_tile) feed.start(a, c, min(TOK, (len - next * TOK + 15) & ~15), stop, stage, bar + st_i, st);
    }
    __syncthreads();
    if (abort_flag != 0) {
      if (threadIdx.x == 0) report_abort(&abort_flag, st);
      for (int s = 0; s < KV4_STAGES; ++s) {
        const int i = uses + s;
        if (tile + s * KV4_WARPS < end_tile) {
          for (int k = 0; k < 1 << 16 && !mbar_try_wait(bar + i % KV4_STAGES, (i / KV4_STAGES) & 1); ++k) {}
        }
      }
      return;
    }
    w.left -= end_tile - tile0;
    if (w.left <= 0) return;
    turn += end_tile - tile0;
    w.tile0 = 0;
    if (++w.item == c.hkv) {
      w.item = 0;
      do w.n_tiles = kv4_tiles(a, c.block, TOK, ++w.b);
      while (w.n_tiles == 0);
    }
  }
}

// A launch that may begin while the kernel ahead of it ends; it waits for that one's results itself.
template <typename... Args>
static cudaError_t kv4_follow(void (*kernel)(Args...), dim3 grid, int threads, int bytes, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

template <int NG, int NT, bool KEEP>
static cudaError_t kv4_launch(const Kv4Decode& a, const Kv4Cache& c, int B, int blocks, int max_len, OmniStatus* st, cudaStream_t stream) {
  using T = Kv4Tile<NG, true>;
  constexpr int merge = KV4_WARPS * 8 * NT * (NG * 64 + 2) * 4, stages = KV4_WARPS * KV4_STAGES * T::BYTES, bytes = merge > stages ? merge : stages;
  const int total = a.rows * (a.hq / c.hkv), chunks = (total + 8 * NT - 1) / (8 * NT);
  const long long grid = a.min_tiles == 0 ? (long long)B * c.hkv * chunks : blocks;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  static bool asked[64] = {false};
  cudaError_t e = (cudaError_t)ensure_dyn_smem((const void*)kv4_decode_kernel<NG, NT, KEEP>, bytes, asked);
  if (e != cudaSuccess) return e;
  kv4_decode_kernel<NG, NT, KEEP><<<(unsigned)grid, KV4_WARPS * 32, bytes, stream>>>(a, c, B, st);
  e = cudaGetLastError();
  if (e == cudaSuccess && a.min_tiles > 0) e = kv4_follow(kv4_join_kernel<NT>, dim3(c.hkv * total, B), c.d, blocks * 4, stream, a, c, blocks);
  if (e != cudaSuccess || !KEEP) return e;
  // as many blocks as the longest request has tokens for, while that is no more than two rounds of them
  const int tokens = NT == 1 ? 256 : 64, want = (max_len + tokens - 1) / tokens, most_x = 148 * 16 / (c.hkv * B), x = want < most_x ? want : most_x;
  return kv4_follow(kv4_add_kernel<8 * NT>, dim3(x < 1 ? 1 : x, c.hkv, B), 256, 0, stream, a, c);
}
template <int NG, int NT>
static cudaError_t kv4_launch(const Kv4Decode& a, const Kv4Cache& c, int B, int blocks, int max_len, OmniStatus* st, cudaStream_t stream) {
  return a.scores != nullptr ? kv4_launch<NG, NT, true>(a, c, B, blocks, max_len, st, stream) : kv4_launch<NG, NT, false>(a, c, B, blocks, max_len, st, stream);
}

template <int NG, int TOK>
static cudaError_t kv4_launch_weights(const Kv4Decode& a, const Kv4Cache& c, int B, int max_len, OmniStatus* st, cudaStream_t stream) {
  const int total = a.rows * (a.hq / c.hkv), chunks = (total + 7) / 8;
  constexpr int stages = KV4_WARPS * KV4_STAGES * Kv4Tile<NG, false, TOK>::BYTES, each = NG * 64 * 16 + (1 + NG) * 4 * 16;
  const int bytes = stages + chunks * each;
  // the most that any call needs: threads whose calls have different rows set the same limit
  static bool asked[64] = {false};
  cudaError_t e = (cudaError_t)ensure_dyn_smem((const void*)kv4_weights_kernel<NG, TOK>, stages + KV4_WEIGHTS_ROWS / 8 * each, asked);
  if (e != cudaSuccess) return e;
  const long long shares = ((long long)B * c.hkv * ((max_len + TOK - 1) / TOK) + KV4_WARPS - 1) / KV4_WARPS, resident = 148 * 3;
  const unsigned grid = (unsigned)(shares < 1 ? 1 : shares < resident ? shares : resident);
  return kv4_follow(kv4_weights_kernel<NG, TOK>, dim3(grid), KV4_WARPS * 32, bytes, stream, a, c, B, st);
}

}  // namespace omni

using namespace omni;

// The arguments come in a block, as the caller packs them; 8-byte fields first, so that there are no gaps.
// row_tile: query rows that share a pass over the cache, 8, or 16 for d <= 128.  min_tiles 0: a block for every item (a row_tile of a
// key/value head of a request); else `blocks_at_once` blocks share all tiles of 64 tokens (32 for d = 256) equally, at least min_tiles each,
// and o_part [blocks_at_once, 2, row_tile, d] and lse_part [blocks_at_once, 2, row_tile] take what they have of shared items, `shared` where that is.
struct Kv4DecodeArgs {
  const void *q, *k_cache, *v_cache;
  const int *table, *seq_lens;
  void* out;
  float *o_part, *lse_part, *lse, *weights;
  void* shared;                     // int32 [batch, hkv, row tiles, 2]
  float* scores;                    // [batch, hkv, row tiles, table_w blocks up to a multiple of 64, row_tile]; null: scores are made twice
  long long q_row, blocks;
  int q_head, block, hkv, d, table_ld, table_w, batch, rows, hq, max_len, row_tile, blocks_at_once, min_tiles;
  float scale, decay;
  int reserved;
};
extern "C" int omni_kv4_decode(const Kv4DecodeArgs* p, void* status, cudaStream_t stream) {
  const int d = p->d, B = p->batch, rep = p->hkv > 0 ? p->hq / p->hkv : 0;
  const Kv4Cache c = {(uint8_t*)p->k_cache, (uint8_t*)p->v_cache, p->blocks, p->block, p->hkv, d};
  if (!kv4_shape_ok(c) || p->hq < 1 || p->hq % p->hkv != 0 || p->rows < 1 || p->hkv > 65535 || B > 65535 || p->min_tiles < 0 ||
      (p->row_tile != 8 && (p->row_tile != 16 || d > 128)))
    return -1;
  if (p->weights != nullptr && (p->lse == nullptr || p->rows * rep > KV4_WEIGHTS_ROWS)) return -2;
  if (p->min_tiles > 0 && (p->o_part == nullptr || p->lse_part == nullptr || p->shared == nullptr || p->blocks_at_once < 1 || p->blocks_at_once > KV4_MAX_BLOCKS)) return -3;
  if (B <= 0) return 0;
  const int wide_q = (uintptr_t)p->q % 16 == 0 && p->q_row % 8 == 0 && p->q_head % 8 == 0;
  const Kv4Decode a = {(const __nv_bfloat16*)p->q, p->q_row, p->q_head, wide_q, p->table, p->seq_lens, p->table_ld, p->table_w, p->rows, p->hq,
                       p->scale * 1.4426950408889634f, (__nv_bfloat16*)p->out, p->lse, p->weights, p->decay,
                       p->block % 64 == 0 ? 64 : p->block % 32 == 0 ? 32 : 16, p->min_tiles, p->o_part, p->lse_part, p->weights != nullptr ? p->scores : nullptr, (p->table_w * p->block + 63) / 64 * 64, (int2*)p->shared};
  OmniStatus* st = (OmniStatus*)status;
  const bool wide = p->row_tile == 16;
  const int n = p->blocks_at_once;
  cudaError_t e = d == 64    ? wide ? kv4_launch<1, 2>(a, c, B, n, p->max_len, st, stream) : kv4_launch<1, 1>(a, c, B, n, p->max_len, st, stream)
                  : d == 128 ? wide ? kv4_launch<2, 2>(a, c, B, n, p->max_len, st, stream) : kv4_launch<2, 1>(a, c, B, n, p->max_len, st, stream)
                             : kv4_launch<4, 1>(a, c, B, n, p->max_len, st, stream);
  if (e != cudaSuccess || p->weights == nullptr || p->scores != nullptr) return (int)e;
  e = d == 64    ? kv4_launch_weights<1, 64>(a, c, B, p->max_len, st, stream)
      : d == 128 ? kv4_launch_weights<2, 64>(a, c, B, p->max_len, st, stream)
                 : kv4_launch_weights<4, 32>(a, c, B, p->max_len, st, stream);
  return (int)e;
}
