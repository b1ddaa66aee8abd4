// Layout of the 4-bit paged key/value cache.
//
// A cache is [blocks, Hkv, block_size * 9 d / 16] bytes.  The piece of one block and head holds the codes of its tokens (d / 2
// bytes each) and behind them, for every token and group of 64 columns, one 32-bit word of two bf16 values: the step and the
// lowest value.  value = code * step + lowest.  A kernel that reads a run of tokens therefore reads two contiguous ranges (three
// for d = 256), which is what the bulk copies of the decode kernel want.
//
// Codes lie in planes of up to two groups; eight columns make a 32-bit word, column j of them in bits 4j .. 4j + 3.
//   keys    a token's words in a row; in the row, lane c of four owns the words of the columns 16 c .. 16 c + 15 of every group, so
//           that it fetches them with one 16-byte read (8 bytes with one group)
//   values  two tokens share a row: chunk r of eight holds the columns 8 r .. 8 r + 7 of every group, of the even token and then of
//           the odd one; a matrix fragment wants both tokens of a pair in one lane.  The chunks of a row are permuted by the row's
//           number, so that the 32 lanes of such a read touch every bank once per wavefront.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace omni {

constexpr int KV4_GROUP = 64;

struct Kv4Cache {
  uint8_t *k, *v;
  long long blocks;
  int block, hkv, d;
  __host__ __device__ int groups() const { return d / KV4_GROUP; }
  __host__ __device__ int per() const { return d > KV4_GROUP ? 2 : 1; }                 // groups of a plane
  __host__ __device__ long long piece() const { return (long long)block * (d * 9 / 16); }
  __host__ __device__ long long at(long long blk, int h) const { return (blk * hkv + h) * piece(); }
  // byte of word u (columns 8 u .. 8 u + 7) of token t of the block, from the piece's start
  __host__ __device__ int k_word(int t, int u) const {
    const int p = per(), g = u >> 3, i = u & 7, gp = g & (p - 1);
    return (g / p * block + t) * 32 * p + ((i >> 1) * 2 * p + gp * 2 + (i & 1)) * 4;
  }
  __host__ __device__ int v_word(int t, int u) const {
    const int p = per(), g = u >> 3, r = u & 7, gp = g & (p - 1), pair = t >> 1;
    const int chunk = p == 2 ? r ^ ((pair & 3) << 1) : r ^ (((pair >> 1) & 1) << 2);
    return (g / p * block + pair * 2) * 32 * p + chunk * 8 * p + (t & 1) * 4 * p + gp * 4;
  }
  __host__ __device__ int scale_word(int t, int g) const { return block * d / 2 + (t * groups() + g) * 4; }
};

// step and lowest value of a group, from its word
__device__ __forceinline__ float kv4_step(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float kv4_low(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

inline bool kv4_shape_ok(const Kv4Cache& c) {
  return c.blocks > 0 && c.hkv > 0 && c.block >= 16 && c.block <= 1 << 20 && c.block % 16 == 0 && (c.d == 64 || c.d == 128 || c.d == 256) &&
         ((uintptr_t)c.k | (uintptr_t)c.v) % 16 == 0;
}

}  // namespace omni
