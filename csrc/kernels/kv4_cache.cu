// Rows of the 4-bit paged key/value cache: written, read back, chosen for eviction and moved (layout: include/kv4.cuh).
//
// Formulas.  A group of 64 columns x of one token and head is stored as lo = min x, step = (max x - min x) / 15 rounded up to
// bf16 and codes = round((x - lo) / step) (to nearest, ties to even, 0 where step = 0); it stands for code * step + lo.  lo is one
// of the bf16 inputs and therefore exact; the step is rounded up so that 15 steps always reach the maximum, and code * step + lo has
// one rounding in fp32 (code * step has 12 bits).  A group with a NaN, an infinity or a range beyond fp32 is NaN as a whole.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../include/kv4.cuh"
#include "../include/omni_ptx.cuh"
#include "../include/score_mod.cuh"

namespace omni {

constexpr int KV4_SITE_ROWS = 81, KV4_SITE_KEEP = 82, KV4_SITE_MOVE = 83;

// ------------------------------------------------------------------------------------------------ write and read
struct Kv4Rows {
  const __nv_bfloat16 *k, *v;       // write: sources; element strides below
  __nv_bfloat16 *k_out, *v_out;     // read: [n, Hkv, d] contiguous
  long long k_row, v_row;
  int k_head, v_head;
  const long long* slots;           // [n]; negative: skipped (write), zeros (read)
  long long n;
  float* weights;                   // write: [blocks, Hkv, block] or null, set to zero
  int* positions;                   // write: [blocks, Hkv, block] or null, set to token_positions[i]
  const long long* token_positions;
  int parts, span;                  // warps of a token, and their heads
};

// A warp takes a token at a time and walks its heads.  Which word (8 columns) of the keys or of the values a lane has is the same for all
// heads, so that its addresses are worked out once a token and then go on by a stride.  At d = 128 the 32 lanes have the two rows of a
// head, at d = 64 those of two heads, at d = 256 the keys' row and then the values'.  Where there are few tokens, several warps share one.
struct Kv4Place {
  long long blk;                    // -1: no row
  int t;
};
__device__ __forceinline__ Kv4Place kv4_place(const Kv4Cache& c, long long slot, OmniStatus* st, long long tok) {
  if (slot < 0) return {-1, 0};
  Kv4Place p;
  if (slot < 0x7fffffffll) {        // a 64-bit division costs as much as the rest of the row
    p.blk = (unsigned)slot / (unsigned)c.block;
    p.t = (int)slot - (int)p.blk * c.block;
  } else {
    p.blk = slot / c.block;
    p.t = (int)(slot - p.blk * c.block);
  }
  if (p.blk < c.blocks) return p;
  if ((threadIdx.x & 31) == 0) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_ROWS, (int)tok);
  return {-1, 0};
}

// Word of the codes round((x - low) / step), ties to even, of 8 columns, all times `lift` (a power of two that leaves step and inverse normal).
// The inverse is at most 2^-20 of it too small, never too large, so that code = floor((x - low) inverse) is the quotient's floor or one less, which
// an addition that rounds down leaves in the lowest bits.  The remainder off = x - low - code step is exact (code step has 12 bits, and no bit
// of the rest lies below those of x - low and of step); it is not negative and one more is right where it is more than half a step, or
// half a step and the code odd: a comparison of their bits as whole numbers.
__device__ __forceinline__ uint32_t kv4_word(const __nv_bfloat162 (&x)[4], float low, float step, float lift) {
  const float unit = step * lift, inverse = rcp_fast(unit) * (1.f - 0x1p-21f);
  const int half = __float_as_int(0.5f * unit);
  uint32_t word = 0, over = 0;      // over: the sums' exponents, shifted along with the codes
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float v = __fsub_rn(i & 1 ? __high2float(x[i / 2]) : __low2float(x[i / 2]), low) * lift;
    const float sum = __fmaf_rd(v, inverse, 12582912.f), off = __fmaf_rn(12582912.f - sum, unit, v);
    const uint32_t code = __float_as_uint(sum);
    word = word * 16u + code + ((uint32_t)(half - __float_as_int(off) - (int)(code & 1u)) >> 31);
    over = over * 16u + 0x4b400000u;
  }
  return word - over;
}

template <int D>
struct Kv4Lane {
  static constexpr int WORDS = D / 8, SIDES = WORDS == 32 ? 2 : 1, HEADS = WORDS == 8 ? 2 : 1;      // steps of a head, heads of a step
  int u, head;
  bool values;                      // of the first side
  __device__ __forceinline__ Kv4Lane() {
    const int lane = threadIdx.x & 31;
    u = lane & (WORDS - 1);
    values = SIDES == 1 && ((lane / WORDS) & 1);
    head = HEADS == 2 ? lane >> 4 : 0;
  }
  __device__ __forceinline__ long long word(const Kv4Cache& c, const Kv4Place& p, bool of_values, int h) const {
    return c.at(p.blk, h) + (of_values ? c.v_word(p.t, u) : c.k_word(p.t, u));
  }
  __device__ __forceinline__ long long scale(const Kv4Cache& c, const Kv4Place& p, int h) const { return c.at(p.blk, h) + c.scale_word(p.t, u >> 3); }
};
// Token and heads of unit `unit`
__device__ __forceinline__ long long kv4_unit(const Kv4Rows& a, const Kv4Cache& c, long long unit, int& from, int& to) {
  const long long tok = a.parts == 1 ? unit : unit < 0x7fffffffll ? (long long)((unsigned)unit / (unsigned)a.parts) : unit / a.parts;
  from = (int)(unit - tok * a.parts) * a.span;
  to = min(c.hkv, from + a.span);
  return tok;
}

// The 8 lanes of a group find its range, as the smallest of x and of -x, with three shuffles.  Reads 2 d bytes and writes 9 d / 16 a row; bound
// by its instructions: 4099 tokens of 8 heads in 12 us, 30,000 in 58 (2.5 TB/s).  32 registers a thread (8 blocks an SM) beat 48 and 56.
template <int D, bool VEC>
__global__ void __launch_bounds__(256, 8) kv4_write_kernel(Kv4Rows a, Kv4Cache c, OmniStatus* st) {
  using L = Kv4Lane<D>;
  const L lane;
  const long long warps = (long long)gridDim.x * 8, head_bytes = c.piece() * L::HEADS;
  for (long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); unit < a.n * a.parts; unit += warps) {
    int from, to;
    const long long tok = kv4_unit(a, c, unit, from, to);
    const Kv4Place p = kv4_place(c, a.slots[tok], st, tok);
    if (p.blk < 0) continue;
#pragma unroll
    for (int side = 0; side < L::SIDES; ++side) {
      const bool values = L::SIDES == 2 ? side == 1 : lane.values;
      const int h = from + lane.head;
      const long long head_step = (long long)(values ? a.v_head : a.k_head);
      const __nv_bfloat16* src = (values ? a.v + tok * a.v_row : a.k + tok * a.k_row) + lane.u * 8 + h * head_step;
      uint8_t* cache = values ? c.v : c.k;
      uint8_t *codes = cache + lane.word(c, p, values, h), *scales = cache + lane.scale(c, p, h);
      int left = to - h;                                                    // heads of this lane that there are to write
      for (int h0 = from; h0 < to; h0 += L::HEADS) {
        __nv_bfloat162 x[4];
        if (left <= 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = __float2bfloat162_rn(0.f);
        } else if (VEC) {
          *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = __halves2bfloat162(src[2 * j], src[2 * j + 1]);
        }
        const __nv_bfloat162 lo2 = __hmin2_nan(__hmin2_nan(x[0], x[1]), __hmin2_nan(x[2], x[3]));
        const __nv_bfloat162 hi2 = __hmax2_nan(__hmax2_nan(x[0], x[1]), __hmax2_nan(x[2], x[3]));
        auto least = [](uint32_t p, uint32_t q) {
          const __nv_bfloat162 m = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&p), *reinterpret_cast<__nv_bfloat162*>(&q));
          return *reinterpret_cast<const uint32_t*>(&m);
        };
        const uint32_t lo = *reinterpret_cast<const uint32_t*>(&lo2), hi = *reinterpret_cast<const uint32_t*>(&hi2) ^ 0x80008000u;
        uint32_t ends = least(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));      // smallest, minus the largest
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ends = least(ends, __shfl_xor_sync(0xffffffffu, ends, o));
        const float low = __uint_as_float(ends << 16), range = __fsub_rn(__uint_as_float((ends & 0xffff0000u) ^ 0x80000000u), low);
        float step = __uint_as_float((__float_as_uint(__fdiv_rn(range, 15.f)) + 0xffffu) & 0xffff0000u);
        if (!(range < INFINITY)) step = __uint_as_float(0x7fc00000u);                                     // NaN or infinite
        uint32_t word = 0;
        if (step >= 0x1p-100f) word = kv4_word(x, low, step, 1.f);
        else if (step > 0.f) word = kv4_word(x, low, step, 0x1p60f);
        if (left > 0) {
          *reinterpret_cast<uint32_t*>(codes) = word;
          if ((lane.u & 7) == 0) *reinterpret_cast<uint32_t*>(scales) = (__float_as_uint(step) >> 16) | ends << 16;
          if (lane.u == 0 && !values && a.weights != nullptr) a.weights[(p.blk * c.hkv + h0 + lane.head) * c.block + p.t] = 0.f;
          if (lane.u == 0 && !values && a.positions != nullptr) a.positions[(p.blk * c.hkv + h0 + lane.head) * c.block + p.t] = (int)a.token_positions[tok];
        }
        codes += head_bytes;
        scales += head_bytes;
        src += L::HEADS * head_step;
        left -= L::HEADS;
      }
    }
  }
}

// The inverse: a word of codes and its group's word to 8 bf16 values, four words a lane under way.  Reads 9 d / 16 bytes and writes 2 d a row:
// 40,003 tokens of 8 heads in 39 us, 5.4 TB/s; 32 registers a thread (8 blocks an SM) beat 42 and 57 of them.
template <int D>
__global__ void __launch_bounds__(256, 8) kv4_read_kernel(Kv4Rows a, Kv4Cache c, OmniStatus* st) {
  using L = Kv4Lane<D>;
  constexpr int AT_ONCE = 4;
  const L lane;
  const long long warps = (long long)gridDim.x * 8, head_bytes = c.piece() * L::HEADS;
  for (long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); unit < a.n * a.parts; unit += warps) {
    int from, to;
    const long long tok = kv4_unit(a, c, unit, from, to);
    const Kv4Place p = kv4_place(c, a.slots[tok], st, tok);
#pragma unroll
    for (int side = 0; side < L::SIDES; ++side) {
      const bool values = L::SIDES == 2 ? side == 1 : lane.values;
      const int h = from + lane.head;
      const uint8_t* cache = values ? c.v : c.k;
      const uint8_t *codes = cache + lane.word(c, p, values, h), *scales = cache + lane.scale(c, p, h);
      __nv_bfloat16* to_row = (values ? a.v_out : a.k_out) + (tok * c.hkv + h) * D + lane.u * 8;
      int left = p.blk < 0 ? 0 : to - h;                                    // heads of this lane that there are to read
      for (int h0 = from; h0 < to; h0 += L::HEADS * AT_ONCE) {
        uint32_t w[AT_ONCE], s[AT_ONCE];
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
          w[x] = s[x] = 0u;
          if (x * L::HEADS < left) {
            w[x] = *reinterpret_cast<const uint32_t*>(codes + x * head_bytes);
            s[x] = *reinterpret_cast<const uint32_t*>(scales + x * head_bytes);
          }
        }
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
          const float step = kv4_step(s[x]), low = kv4_low(s[x]);
          __nv_bfloat162 y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // the byte in both halves; 1024 + code and 1024 + 16 code as fp16 numbers, whose conversion runs beside the integer operations
            const uint32_t pair = (__byte_perm(w[x], 0u, j | 0x4040 | j << 8) & 0x00f0000fu) | 0x64006400u;
            const float2 code = __half22float2(__hfma2(*reinterpret_cast<const __half2*>(&pair), __floats2half2_rn(1.f, 0.0625f), __floats2half2_rn(-1024.f, -64.f)));
            y[j] = __floats2bfloat162_rn(fmaf(code.x, step, low), fmaf(code.y, step, low));
          }
          if (h0 + x * L::HEADS + lane.head < to) *reinterpret_cast<uint4*>(to_row + x * (L::HEADS * D)) = *reinterpret_cast<uint4*>(y);
        }
        codes += head_bytes * AT_ONCE;
        scales += head_bytes * AT_ONCE;
        to_row += L::HEADS * AT_ONCE * D;
        left -= L::HEADS * AT_ONCE;
      }
    }
  }
}
// Blocks of 8 warps, as many as fit the card four times over at most.  A token's heads are shared out to several warps while there are fewer
// warps than `want`: 64 tokens of 4 heads are written and read back in 7 us, by a warp a token in 14; 1000 tokens of 8 heads written take
// 5.6 us, by a warp a token 8.2; 4099 take 12, by a warp a head 16.
static unsigned kv4_row_blocks(Kv4Rows& a, const Kv4Cache& c, long long want) {
  const int heads = c.d == 64 ? 2 : 1, steps = (c.hkv + heads - 1) / heads;
  const long long share = (want + a.n - 1) / a.n;
  const int parts = share < steps ? (int)share : steps, each = (steps + parts - 1) / parts;
  a.parts = (steps + each - 1) / each;
  a.span = each * heads;
  const long long blocks = (a.n * a.parts + 7) / 8, most = 148 * 8 * 4;
  return (unsigned)(blocks < most ? blocks : most);
}

// ------------------------------------------------------------------------------------------------ eviction
// Order of eviction: larger keys stay.  Places of the first and last positions come before all weights, a NaN before the numbers.
__device__ __forceinline__ uint32_t kv4_keep_key(float w, int pos, int first, int last_from) {
  if (pos < first || pos >= last_from) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(w + 0.f);                      // -0 counts as 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum over a block of that many threads
template <int THREADS>
__device__ __forceinline__ int kv4_block_scan(int x) {
  constexpr int WARPS = THREADS / 32;
  __shared__ int part[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) part[warp] = v;
  __syncthreads();
  int sum = lane < WARPS ? part[lane] : 0;                          // every warp scans the warps' sums by itself
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  const int base = __shfl_sync(0xffffffffu, sum, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? base : 0) + v - x;
}

struct Kv4Keep {
  const float* weights;
  const int *positions, *table, *seq_lens, *seen;
  long long blocks;
  int table_ld, table_w, block, hkv, budget, first, last;
  int *keep, *lens, *scratch;       // [B, Hkv, budget], [B], scratch as keep (null where no request has over 2 KV4_BINS places)
};

// A cluster of blocks for a request and head, each with a run of its places.  The keys are read from memory once and kept in shared
// memory (`cap` of them a block; those beyond are made again when they are needed).  The key of the budget-th heaviest place is
// found 11, 11 and 10 bits at a time: histograms in shared memory, which every block of the cluster adds up for itself.  Then a
// warp walks its own run of places, and ranks (of equal keys, of the places to fill, of the tokens that fill them) are counts of its
// votes and sums over the warps and blocks ahead.  Reads 8 bytes a place; bound by the latency of its some ten steps.
constexpr int KV4_BINS = 2048, KV4_MOST_BLOCKS = 8, KV4_MOST_KEYS = 40000;
__host__ __device__ constexpr int kv4_keep_run(int n, int size) { return ((n + size - 1) / size + 3) & ~3; }      // places of a block
struct Kv4KeepShared {
  int hist[2][KV4_BINS];            // highest keys first
  int run[3][32];                   // of the warps' runs: equal keys, places to fill, tokens that fill some
  int count[2];                     // of this block: places to fill, tokens that fill some
  int equal;                        // keys equal to the last that stays in the blocks ahead
  uint32_t prefix;
  int left, all;
};
// ALL: the keys of a run find room in shared memory.  VEC: places that are read at once, 4 where blocks and addresses allow (15 keys a thread and
// 32 warps an SM are bound by instructions, not bytes).
template <bool ALL, int VEC, int N>
__device__ __forceinline__ void kv4_keep_body(const Kv4Keep& a, int n, int cap, uint32_t* s_keys, Kv4KeepShared& sh, OmniStatus* st) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.y, h = blockIdx.x / size, tid = threadIdx.x;
  int* keep = a.keep + ((long long)b * a.hkv + h) * a.budget;
  const int chunk = kv4_keep_run(n, size), j0 = rank * chunk, count = max(0, min(chunk, n - j0));
  const int last_from = a.seen[b] - a.last;
  const int* table = a.table + (long long)b * a.table_ld;
  auto make_at = [&](int page, int off) -> uint32_t {
    const int blk = table[page];
    if (blk < 0 || blk >= a.blocks) {
      report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_KEEP, b);
      return 0u;
    }
    const long long at = ((long long)blk * a.hkv + h) * a.block + off;
    return kv4_keep_key(a.weights[at], a.positions[at], a.first, last_from);
  };
  auto make = [&](int i) -> uint32_t { return make_at((j0 + i) / a.block, (j0 + i) % a.block); };
  auto key = [&](int i) -> uint32_t { return ALL || i < cap ? s_keys[i] : make(i); };
  for (int i = tid; i < KV4_BINS; i += N) sh.hist[0][i] = sh.hist[1][i] = 0;
  __syncthreads();
  {
    constexpr int AT_ONCE = VEC == 4 ? 4 : 8, STEP = N * VEC;        // loads under way a thread: block ids, then weights and positions
    const int pages = STEP / a.block, rest = STEP - pages * a.block, stride = a.hkv * a.block, base = h * a.block;
    int page = (j0 + tid * VEC) / a.block, off = (j0 + tid * VEC) - page * a.block;
    for (int i0 = tid * VEC; i0 < count; i0 += STEP * AT_ONCE) {
      int blk[AT_ONCE], at[AT_ONCE], pos[AT_ONCE][VEC];
      float w[AT_ONCE][VEC];
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        at[x] = base + off;
        blk[x] = i0 + x * STEP < count ? table[page] : 0;
        page += pages;
        off += rest;
        if (off >= a.block) {
          off -= a.block;
          ++page;
        }
      }
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        const bool in = blk[x] >= 0 && blk[x] < a.blocks;
        const long long from = (long long)(in ? blk[x] : 0) * stride + at[x];
        if (VEC == 4) {
          *reinterpret_cast<float4*>(w[x]) = *reinterpret_cast<const float4*>(a.weights + from);
          *reinterpret_cast<int4*>(pos[x]) = *reinterpret_cast<const int4*>(a.positions + from);
        } else {
          w[x][0] = a.weights[from];
          pos[x][0] = a.positions[from];
        }
      }
#pragma unroll
      for (int x = 0; x < AT_ONCE; ++x) {
        const int i = i0 + x * STEP;
        if (i >= count) break;
        const bool in = blk[x] >= 0 && blk[x] < a.blocks;
        if (!in) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_KEEP, b);
        uint32_t k[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          k[e] = in ? kv4_keep_key(w[x][e], pos[x][e], a.first, last_from) : 0u;
          if (VEC == 1 || i + e < count) atomicAdd(&sh.hist[0][KV4_BINS - 1 - (k[e] >> 21)], 1);
        }
        if (ALL || i < cap) {                                       // cap is a multiple of 4
          if (VEC == 4) *reinterpret_cast<uint4*>(s_keys + i) = *reinterpret_cast<uint4*>(k);
          else s_keys[i] = k[0];
        }
      }
    }
  }
  uint32_t prefix = 0, mask = 0;
  int left = a.budget;                                              // of the places whose key starts with the prefix, so many stay
  bool all_stay = false;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    int* mine = sh.hist[pass & 1];
    if (pass > 0) {
      for (int i = tid; i < count; i += N) {
        const uint32_t k = key(i);
        if ((k & mask) == prefix) atomicAdd(&mine[bins - 1 - ((k >> shift) & (bins - 1))], 1);
      }
    }
    cluster.sync();
    constexpr int MOST = KV4_BINS / N;                              // bins of a thread, or half as many
    const int each = bins / N;
    int v[MOST], all = 0;
#pragma unroll
    for (int d = 0; d < MOST; ++d) v[d] = 0;
#pragma unroll
    for (int r = 0; r < KV4_MOST_BLOCKS; ++r) {
      if (r >= size) continue;
      const int* theirs = cluster.map_shared_rank(mine, r) + tid * each;
      if (each == 4) {
        const int4 x = *reinterpret_cast<const int4*>(theirs);
        v[0] += x.x; v[1] += x.y; v[MOST - 2] += x.z; v[MOST - 1] += x.w;
      } else if (each == 2) {
        const int2 x = *reinterpret_cast<const int2*>(theirs);
        v[0] += x.x; v[1] += x.y;
      } else {
        v[0] += *theirs;
      }
    }
#pragma unroll
    for (int d = 0; d < MOST; ++d) all += v[d];
    int above = kv4_block_scan<N>(all);
#pragma unroll
    for (int d = 0; d < MOST; ++d) {
      if (above < left && left <= above + v[d]) {
        sh.prefix = prefix | (uint32_t)(bins - 1 - tid * each - d) << shift;
        sh.left = left - above;
        sh.all = v[d];
      }
      above += v[d];
    }
    if (pass == 1)                                                  // nobody reads the first histogram any more: it serves once more
      for (int i = tid; i < KV4_BINS; i += N) sh.hist[0][i] = 0;
    __syncthreads();
    prefix = sh.prefix;
    left = sh.left;
    all_stay = left == sh.all;
    mask |= (uint32_t)(bins - 1) << shift;
    __syncthreads();
    if (all_stay) break;                                            // no need to tell the places of this prefix apart
  }
  // `prefix` begins the keys of the last places that stay; `left` of the places with such keys do, the lowest first.  A warp walks a run of the
  // block's places, 32 at a time, so that a place's rank is a count of votes.
  const int warp = tid >> 5, lane = tid & 31;
  const uint32_t below = (1u << lane) - 1u;
  const int each = (count + N - 1) / N * 32, i0 = min(warp * each, count), i1 = min(i0 + each, count);
  auto ahead = [&](int x) -> int { return __reduce_add_sync(0xffffffffu, lane < warp ? sh.run[x][lane] : 0); };
  int equal0 = 0;
  if (!all_stay) {                                                  // all bits are known: the keys are equal
    if (tid < 32) {                                                 // their number in the blocks ahead is in the last histograms
      const int x = __reduce_add_sync(0xffffffffu, tid < rank ? cluster.map_shared_rank(sh.hist[0], tid)[1023 - (prefix & 1023)] : 0);
      if (tid == 0) sh.equal = x;
    }
    int mine = 0;
#pragma unroll 4
    for (int i = i0 + lane; i < i0 + each; i += 32) mine += __popc(__ballot_sync(0xffffffffu, i < i1 && key(i) == prefix));
    if (lane == 0) sh.run[0][warp] = mine;
    __syncthreads();
    equal0 = sh.equal + ahead(0);
  }
  // Which of a warp's next 32 places stay.  Later walks find the votes where the run's first keys were: a word for 32 keys.
  auto decide = [&](int i, int& equal) -> uint32_t {
    const uint32_t k = i < i1 ? key(i) & mask : 0u;
    const bool above = i < i1 && k > prefix, last = i < i1 && k == prefix;
    if (all_stay) return __ballot_sync(0xffffffffu, above || last);
    const uint32_t votes = __ballot_sync(0xffffffffu, last);
    const bool s = above || (last && equal + __popc(votes & below) < left);
    equal += __popc(votes);
    return __ballot_sync(0xffffffffu, s);
  };
  auto again = [&](int i, int& equal) -> uint32_t { return ALL ? s_keys[i0 + (i - i0) / 32] : decide(i, equal); };
  const int near = max(0, min(i1 - i0, a.budget - j0 - i0));        // the run's first places are to be filled, the others may fill some
  auto near_of = [&](int i) -> uint32_t {                           // of the 32 with i
    const int x = near - (i - i0 - lane);
    return x >= 32 ? 0xffffffffu : x <= 0 ? 0u : (1u << x) - 1u;
  };
  int holes = 0, far = 0, equal = equal0;
#pragma unroll 4
  for (int i = i0 + lane; i < i0 + each; i += 32) {
    const uint32_t stay = decide(i, equal), first = near_of(i);
    holes += __popc(~stay & first);
    far += __popc(stay & ~first);
    if (ALL && lane == 0 && i < i1) s_keys[i0 + (i - i0) / 32] = stay;      // the vote was behind the reads of these keys
  }
  if (lane == 0) {
    sh.run[1][warp] = holes;
    sh.run[2][warp] = far;
  }
  __syncthreads();
  int hole = ahead(1), source = ahead(2);
  if (tid == N - 32) {
    sh.count[0] = hole + holes;
    sh.count[1] = source + far;
  }
  cluster.sync();
  if (rank > 0) {
    const int* theirs = cluster.map_shared_rank(sh.count, lane < rank ? lane : 0);
    hole += __reduce_add_sync(0xffffffffu, lane < rank ? theirs[0] : 0);
    source += __reduce_add_sync(0xffffffffu, lane < rank ? theirs[1] : 0);
  }
  // The places to fill, in order: at most half of all places, so that those of up to 4096 find room in the histograms
  int* list = size == 1 && n <= 2 * KV4_BINS ? sh.hist[0] : a.scratch + ((long long)b * a.hkv + h) * a.budget;
  equal = equal0;
#pragma unroll 4
  for (int i = i0 + lane; i - lane < i0 + near; i += 32) {
    const uint32_t stay = again(i, equal), open = ~stay & near_of(i);
    if (i < i0 + near) {
      if (stay >> lane & 1u) keep[j0 + i] = j0 + i;
      else list[hole + __popc(open & below)] = j0 + i;
    }
    hole += __popc(open);
  }
  cluster.sync();                                                   // the list is there, and nobody reads another's memory any more
  if (far == 0) return;
  constexpr int AT_ONCE = 8;                                        // loads under way a thread
  equal = equal0;
  for (int i = i0 + lane; i < i0 + each; i += 32 * AT_ONCE) {
    int to[AT_ONCE];
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const int at = i + x * 32;
      to[x] = -1;
      if (at - lane < i1) {
        const uint32_t fill = again(at, equal) & ~near_of(at);
        if (fill >> lane & 1u) to[x] = list[source + __popc(fill & below)];
        source += __popc(fill);
      }
    }
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x)
      if (to[x] >= 0) keep[to[x]] = j0 + i + x * 32;
  }
}

template <int VEC, int N>
__global__ void __launch_bounds__(N, 1024 / N) kv4_keep_kernel(Kv4Keep a, int cap, OmniStatus* st) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ __align__(16) Kv4KeepShared sh;
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.y, h = blockIdx.x / size, tid = threadIdx.x;
  int n = max(a.seq_lens[b], 0);
  if (n > a.table_w * a.block) {
    if (tid == 0) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_KEEP, b);
    n = a.table_w * a.block;
  }
  int* keep = a.keep + ((long long)b * a.hkv + h) * a.budget;
  if (blockIdx.x == 0 && tid == 0) a.lens[b] = min(n, a.budget);
  if (n <= a.budget) {
    for (int j = rank * N + tid; j < a.budget; j += size * N) keep[j] = j < n ? j : -1;
    return;
  }
  if (kv4_keep_run(n, size) <= cap) kv4_keep_body<true, VEC, N>(a, n, cap, s_keys, sh, st);
  else kv4_keep_body<false, VEC, N>(a, n, cap, s_keys, sh, st);
}

struct Kv4Move {
  const int *table, *keep;
  int table_ld, table_w, budget;
  float* weights;
  int* positions;
};

// Eight lanes for a place; those of a place that is filled from elsewhere copy the row, all loads ahead of the stores.  Sources lie behind
// the budget and places below it, so no row is both and the order of the copies does not matter.  Bound by latency: a place's keep entry,
// the two block ids, the row.
template <int GROUPS>
__global__ void __launch_bounds__(256) kv4_move_kernel(Kv4Move a, Kv4Cache c, OmniStatus* st) {
  constexpr int PER = GROUPS > 1 ? 2 : 1, PLANES = GROUPS / PER;
  using Chunk = typename std::conditional<PER == 2, uint2, uint32_t>::type;         // what a lane has of a plane of a row
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 7, j = blockIdx.x * 32 + (threadIdx.x >> 3);
  if (j >= a.budget) return;
  const int s = a.keep[((long long)b * c.hkv + h) * a.budget + j];
  if (s < 0 || s == j) return;
  const int* table = a.table + (long long)b * a.table_ld;
  const int w0 = s / c.block, w1 = j / c.block, ft = s - w0 * c.block, tt = j - w1 * c.block;
  bool ok = s >= a.budget && w0 < a.table_w && w1 < a.table_w;
  const int fb = ok ? table[w0] : -1, tb = ok ? table[w1] : -1;
  ok = fb >= 0 && fb < c.blocks && tb >= 0 && tb < c.blocks;
  if (!ok) {
    if (lane == 0) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_MOVE, b);
    return;
  }
  const long long fp = c.at(fb, h), tp = c.at(tb, h);
  Chunk k[PLANES], v[PLANES];
  uint32_t scale = 0u, number = 0u;
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    k[p] = *reinterpret_cast<const Chunk*>(c.k + fp + (p * c.block + ft) * (32 * PER) + lane * (4 * PER));
    v[p] = *reinterpret_cast<const Chunk*>(c.v + fp + c.v_word(ft, p * 8 * PER + lane));
  }
  const bool of_k = lane < GROUPS, of_v = lane >= 4 && lane - 4 < GROUPS;
  if (of_k || of_v) scale = *reinterpret_cast<const uint32_t*>((of_k ? c.k : c.v) + fp + c.scale_word(ft, lane & 3));
  const long long x = ((long long)fb * c.hkv + h) * c.block + ft, y = ((long long)tb * c.hkv + h) * c.block + tt;
  if (lane == 0 && a.weights != nullptr) number = __float_as_uint(a.weights[x]);
  if (lane == 1 && a.positions != nullptr) number = (uint32_t)a.positions[x];
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    *reinterpret_cast<Chunk*>(c.k + tp + (p * c.block + tt) * (32 * PER) + lane * (4 * PER)) = k[p];
    *reinterpret_cast<Chunk*>(c.v + tp + c.v_word(tt, p * 8 * PER + lane)) = v[p];
  }
  if (of_k || of_v) *reinterpret_cast<uint32_t*>((of_k ? c.k : c.v) + tp + c.scale_word(tt, lane & 3)) = scale;
  if (lane == 0 && a.weights != nullptr) a.weights[y] = __uint_as_float(number);
  if (lane == 1 && a.positions != nullptr) a.positions[y] = (int)number;
}

}  // namespace omni

using namespace omni;

// The calls take their arguments in a block, as the caller packs them: a call with thirty arguments of their own costs more than the
// launch.  8-byte fields come first, so that there are no gaps.
struct Kv4WriteArgs {
  const void *k, *v;
  const long long* slots;
  void *k_cache, *v_cache;
  float* weights;
  int* positions;
  const long long* token_positions;
  long long k_row, v_row, n, blocks;
  int k_head, v_head, block, hkv, d, reserved;
};
extern "C" int omni_kv4_write(const Kv4WriteArgs* p, void* status, cudaStream_t stream) {
  const Kv4Cache c = {(uint8_t*)p->k_cache, (uint8_t*)p->v_cache, p->blocks, p->block, p->hkv, p->d};
  if (!kv4_shape_ok(c)) return -1;
  if ((p->positions == nullptr) != (p->token_positions == nullptr)) return -2;
  if (p->n <= 0) return 0;
  Kv4Rows a = {};
  a.k = (const __nv_bfloat16*)p->k;
  a.v = (const __nv_bfloat16*)p->v;
  a.k_row = p->k_row;
  a.v_row = p->v_row;
  a.k_head = p->k_head;
  a.v_head = p->v_head;
  a.slots = p->slots;
  a.n = p->n;
  a.weights = p->weights;
  a.positions = p->positions;
  a.token_positions = p->token_positions;
  const unsigned grid = kv4_row_blocks(a, c, 148 * 32);
  const bool vec = ((uintptr_t)p->k | (uintptr_t)p->v) % 16 == 0 && (p->k_row | p->v_row) % 8 == 0 && (p->k_head | p->v_head) % 8 == 0;
  const auto kernel = p->d == 64    ? vec ? kv4_write_kernel<64, true> : kv4_write_kernel<64, false>
                      : p->d == 128 ? vec ? kv4_write_kernel<128, true> : kv4_write_kernel<128, false>
                                    : vec ? kv4_write_kernel<256, true> : kv4_write_kernel<256, false>;
  kernel<<<grid, 256, 0, stream>>>(a, c, (OmniStatus*)status);
  return (int)cudaGetLastError();
}

struct Kv4ReadArgs {
  const void *k_cache, *v_cache;
  const long long* slots;
  void *k_out, *v_out;
  long long n, blocks;
  int block, hkv, d, reserved;
};
extern "C" int omni_kv4_read(const Kv4ReadArgs* p, void* status, cudaStream_t stream) {
  const Kv4Cache c = {(uint8_t*)p->k_cache, (uint8_t*)p->v_cache, p->blocks, p->block, p->hkv, p->d};
  if (!kv4_shape_ok(c)) return -1;
  if (p->n <= 0) return 0;
  Kv4Rows a = {};
  a.k_out = (__nv_bfloat16*)p->k_out;
  a.v_out = (__nv_bfloat16*)p->v_out;
  a.slots = p->slots;
  a.n = p->n;
  const unsigned grid = kv4_row_blocks(a, c, 148 * 64);
  const auto kernel = p->d == 64 ? kv4_read_kernel<64> : p->d == 128 ? kv4_read_kernel<128> : kv4_read_kernel<256>;
  kernel<<<grid, 256, 0, stream>>>(a, c, (OmniStatus*)status);
  return (int)cudaGetLastError();
}

struct Kv4KeepArgs {
  const float* weights;
  const int *positions, *table, *seq_lens, *seen;
  int *keep, *lens, *scratch;
  long long blocks;
  int block, hkv, table_ld, table_w, batch, budget, first, last, max_len, reserved;
};
extern "C" int omni_kv4_keep(const Kv4KeepArgs* p, void* status, cudaStream_t stream) {
  if (p->blocks <= 0 || p->block < 1 || p->hkv < 1 || p->hkv > 65535 || p->batch > 65535 || p->budget < 1 || p->max_len < 0 || p->first < 0 || p->last < 0 ||
      p->first + p->last > p->budget || (long long)p->hkv * p->block > 0x7fffffffll)
    return -1;
  if (p->scratch == nullptr && (long long)p->table_w * p->block > 2 * KV4_BINS) return -2;
  if (p->batch <= 0) return 0;
  const Kv4Keep a = {p->weights, p->positions, p->table, p->seq_lens, p->seen, p->blocks, p->table_ld, p->table_w, p->block, p->hkv,
                     p->budget, p->first, p->last, p->keep, p->lens, p->scratch};
  // Blocks of a cluster: one for every 8192 places, at most 8, while all clusters find room at once (an SM takes one block of 1024 threads,
  // and the SMs that are left where clusters of 8 do not fit lie idle): 32 items of 60001 places take 25 us with 4 blocks each, 57 with 8; 64 items
  // 41 with 2 and 51 with 4; 16 of 130000 41 with 4 and 53 with 8; 8 of 20000 20 with 4 and 22 with 2.  A block keeps 40,000 keys;
  // beyond 8 times that they are made again.
  const long long items = (long long)p->hkv * p->batch;
  int size = 1;
  while (size < KV4_MOST_BLOCKS &&
         (p->max_len > KV4_MOST_KEYS * size || (p->max_len > 8192 * size && items * size * 2 <= (size == 4 ? 112 : 128))))
    size *= 2;
  const int run = kv4_keep_run(p->max_len, size), cap = run < 1024 ? 1024 : run > KV4_MOST_KEYS ? KV4_MOST_KEYS : run;
  // 128 items of 8000 places take 20 us with 1024 threads each and 22 with 512, 128 of 2176 14 and 13.
  const bool large = p->max_len > 4096, vec = p->block % 4 == 0 && ((uintptr_t)p->weights | (uintptr_t)p->positions) % 16 == 0;
  const auto kernel = large ? vec ? kv4_keep_kernel<4, 1024> : kv4_keep_kernel<1, 1024> : vec ? kv4_keep_kernel<4, 512> : kv4_keep_kernel<1, 512>;
  static bool asked[4][64] = {{false}};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !asked[2 * large + vec][dev])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KV4_MOST_KEYS * 4);
    if (e == cudaSuccess && dev < 64) asked[2 * large + vec][dev] = true;
  }
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p->hkv * size, p->batch);
  config.blockDim = dim3(large ? 1024 : 512);
  config.dynamicSmemBytes = cap * 4;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)size, 1, 1};
  config.attrs = &attr;
  config.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&config, kernel, a, cap, (OmniStatus*)status);
}

struct Kv4MoveArgs {
  void *k_cache, *v_cache;
  const int *table, *keep;
  float* weights;
  int* positions;
  long long blocks;
  int block, hkv, d, table_ld, table_w, batch, budget, reserved;
};
extern "C" int omni_kv4_move(const Kv4MoveArgs* p, void* status, cudaStream_t stream) {
  const Kv4Cache c = {(uint8_t*)p->k_cache, (uint8_t*)p->v_cache, p->blocks, p->block, p->hkv, p->d};
  if (!kv4_shape_ok(c) || p->hkv > 65535 || p->batch > 65535 || p->budget < 1) return -1;
  if (p->batch <= 0) return 0;
  const Kv4Move a = {p->table, p->keep, p->table_ld, p->table_w, p->budget, p->weights, p->positions};
  const dim3 grid((p->budget + 31) / 32, p->hkv, p->batch);
  if (p->d == 64) kv4_move_kernel<1><<<grid, 256, 0, stream>>>(a, c, (OmniStatus*)status);
  else if (p->d == 128) kv4_move_kernel<2><<<grid, 256, 0, stream>>>(a, c, (OmniStatus*)status);
  else kv4_move_kernel<4><<<grid, 256, 0, stream>>>(a, c, (OmniStatus*)status);
  return (int)cudaGetLastError();
}
