// What the attention kernels over the 4-bit paged key/value cache share: their arguments, how work is shared out, codes as fp16 numbers, and
// the copies of tiles of tokens into shared memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kv4.cuh"
#include "omni_ptx.cuh"
#include "score_mod.cuh"

namespace omni {

constexpr int KV4_SITE_DECODE = 84, KV4_SITE_TILE = 85, KV4_SITE_WEIGHTS = 86;
constexpr int KV4_WARPS = 4, KV4_STAGES = 2, KV4_MAX_BLOCKS = 4096;

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
  if (some * 2 <= blocks) {                 // up to 218 uneven items of 444 blocks: 14 us against 17, 48 against 51; above, waste
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
__device__ __forceinline__ uint32_t kv4_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
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

// Shared memory beyond 48 KB is asked for once a device and kernel; `most` remembers how much.
inline cudaError_t kv4_smem(const void* kernel, int bytes, int (&most)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && most[dev] >= bytes)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) most[dev] = bytes;
  return e;
}

// Many rows on tcgen05 (kv4_rows.cu): the first of the launches, in the place of the decode kernel, with row tiles of 128
cudaError_t kv4_launch_rows(const Kv4Decode& a, const Kv4Cache& c, int B, int blocks, OmniStatus* st, cudaStream_t stream);

}  // namespace omni
