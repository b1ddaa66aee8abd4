// Attention of many query rows over the 4-bit paged key/value cache on the 5th-generation tensor cores (layout: include/kv4.cuh).
//
// The same sums as in kv4_decode.cu, for requests that bring several rows at once (a window of a prompt's last tokens, many heads to a key/value
// head): 128 rows of a key/value head are one operand of 128 rows, so that a tile of tokens is unpacked once for all of them.
//   S_g = Q_g (K_g - 8)^T    Q_g [128, 64] in shared memory (fp16, each row times a power of two), K_g: codes minus 8 of 64 tokens (fp16)
//   p   = exp(scale (sum_g step S_g + (lowest + 8 step) (sum q)) - m)         a thread for each row: no sums across threads
//   O_g += (p step) (V_g - 8)   p step in TMEM (fp16 after a power of two that follows the largest step) over the S_g that it came from
//   out = (sum_g O_g + sum_t p (lowest + 8 step)) / sum_t p
// Both products run in groups of 64 columns, because each group of a token has its own step.
//
// Four warps hold a query row a thread; three unpack (72 bytes of a token's keys, and values, to 256 in the 128-byte swizzle that the
// products read); one copies tiles into shared memory two ahead and issues the products.  104 KB of shared memory and 256 columns of TMEM: two
// blocks share an SM, and the softmax of one runs beside the products and the unpacking of the other.  Bound by the softmax:
// some 16 instructions a row and token.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../include/kv4_tile.cuh"

namespace omni {

constexpr int KV4_ROWS = 128, KV4_ROWS_THREADS = 256, KV4_SITE_ROWS_TILE = 87;

template <int NG>
struct Kv4RowsLayout {
  using T = Kv4Tile<NG, true, 64>;
  static constexpr int CHUNK = 64 * 128;                                    // 64 tokens of a group
  static constexpr int Q = 0, K = Q + NG * KV4_ROWS * 128, V = K + NG * CHUNK, RAW = V + 2 * NG * CHUNK, PAR = RAW + 2 * T::BYTES;
  static constexpr int PAR_SIDE = 64 * 2 * NG * 4, END = PAR + 4 * PAR_SIDE;      // numbers of a tile's tokens: [tile & 1][keys, values]
  static constexpr int BYTES = END + 1024;                                  // and room to start on 1024 bytes
  static constexpr int T_S = 0, T_O = 64 * NG, T_COLS = 128 * NG;
};

__device__ __forceinline__ void kv4_umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) { umma_bf16(d, a, b, idesc, accumulate); }
__device__ __forceinline__ void kv4_umma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void kv4_tmem_ld8(uint32_t at, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void kv4_tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Column of place i among 8: codes come out of a word as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
__host__ __device__ constexpr int kv4_column(int i) { return (i >> 1) + 4 * (i & 1); }
// A word's 8 codes minus 8, in that order
__device__ __forceinline__ uint4 kv4_codes(uint32_t w) { return make_uint4(kv4_code<0>(w), kv4_code<1>(w), kv4_code<2>(w), kv4_code<3>(w)); }

template <int NG>
__global__ void __launch_bounds__(KV4_ROWS_THREADS, 2) kv4_rows_kernel(Kv4Decode a, Kv4Cache c, int B, OmniStatus* st) {
  using L = Kv4RowsLayout<NG>;
  using T = typename L::T;
  constexpr int D = NG * 64, TOK = 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  // a phase a tile; where there are two, of tiles with that parity
  __shared__ __align__(8) uint64_t raw_full[2], raw_empty[2], k_full, v_full[2], v_empty[2], qk_done, p_full, pv_done;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ float s_most[2][2];                                            // largest value step of a tile, of each half of its tokens
  const int rep = a.hq / c.hkv, total = a.rows * rep, chunks = (total + KV4_ROWS - 1) / KV4_ROWS, items = c.hkv * chunks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 3);
      mbar_init(&v_full[i], 3);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(&k_full, 3);
    mbar_init(&qk_done, 1);
    mbar_init(&p_full, 4);
    mbar_init(&pv_done, 1);
    abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 7) {
    tmem_alloc(&tmem_slot, L::T_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;");
  auto wait = [&](uint64_t* bar, int phase, int n) -> bool { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, &abort_flag, st, KV4_SITE_ROWS_TILE, n)); };

  Kv4Work w;
  bool some = true;
  if (a.min_tiles == 0) {
    w.b = blockIdx.x / items;
    w.item = blockIdx.x - w.b * items;
    w.tile0 = w.parts = 0;
    w.left = w.n_tiles = kv4_tiles(a, c.block, TOK, w.b);
  } else {
    some = kv4_work(a, c.block, TOK, items, B, a.min_tiles, w);
  }
  int n0 = 0;                                                               // tiles that are behind this block
  bool ok = true;
  for (bool first = true; some; first = false) {
    const int b = w.b, h = w.item / chunks, row0 = (w.item - h * chunks) * KV4_ROWS, tile0 = w.tile0;
    const int len = kv4_length(a, c.block, b, st);
    const int first_sees = len - a.rows + 1 + row0 / rep, end = len - a.rows + 1 + (min(total, row0 + KV4_ROWS) - 1) / rep;
    const int end_tile = (int)min((long long)w.n_tiles, tile0 + w.left);
    const int stop = min(end, end_tile * TOK), n = stop > tile0 * TOK ? (stop + TOK - 1) / TOK - tile0 : 0;        // tiles of this part
    const bool whole = tile0 == 0 && end_tile == w.n_tiles;
    if (a.min_tiles != 0 && tile0 == 0 && threadIdx.x == 0) {               // as in kv4_decode.cu
      const int parts = w.parts > 0 ? w.parts : whole ? 1 : 1 + (int)kv4_ceil(w.n_tiles - end_tile, w.share);
      a.shared[(long long)b * items + w.item] = make_int2(2 * blockIdx.x + (first ? 0 : 1), parts);
    }
    Kv4Feed<NG, true, 64> feed;
    auto copy = [&](int i) {                                                // tile i of the part, into the place of the tile two ahead of it
      const int k = n0 + i;
      if (k >= 2 && !wait(&raw_empty[k & 1], (k - 2) >> 1, k)) return false;
      feed.start(a, c, min(TOK, (end - (tile0 + i) * TOK + 15) & ~15), stop, smem + L::RAW + (k & 1) * T::BYTES, &raw_full[k & 1], st);
      return true;
    };
    // a thread's query row
    const int row = row0 + threadIdx.x;
    float qs[NG], unit = 0.f;
    if (warp < 4) {
      const __nv_bfloat16* src = a.q + ((long long)b * a.rows + row / rep) * a.q_row + (long long)(h * rep + row % rep) * a.q_head;
      auto eight = [&](int at, float (&f)[8]) {                             // columns at .. at + 7
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < total && a.q_wide) {
          v = *reinterpret_cast<const uint4*>(src + at);
        } else if (row < total) {
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = (uint32_t)__bfloat16_as_ushort(src[at + 2 * j]) | (uint32_t)__bfloat16_as_ushort(src[at + 2 * j + 1]) << 16;
          v = make_uint4(x[0], x[1], x[2], x[3]);
        }
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] = __uint_as_float(x[j] << 16);
          f[2 * j + 1] = __uint_as_float(x[j] & 0xffff0000u);
        }
      };
      float most = 0.f, f[8];
#pragma unroll 4
      for (int at = 0; at < D; at += 8) {
        eight(at, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[j]));
      }
      const int e = min(max(13 - ((int)(__float_as_uint(most) >> 23) - 127), -120), 120);      // as in kv4_decode.cu
      const float up = copysignf(__uint_as_float((uint32_t)(127 + e) << 23), a.scale_log2);
      unit = fmaxf(fabsf(a.scale_log2) * __uint_as_float((uint32_t)(127 - e) << 23), 0x1p-120f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        qs[g] = 0.f;
#pragma unroll 4
        for (int i = 0; i < 8; ++i) {
          eight(g * 64 + i * 8, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            f[j] *= up;
            qs[g] += f[j];
          }
          const uint4 v = make_uint4(kv4_pack(f[kv4_column(0)], f[kv4_column(1)]), kv4_pack(f[kv4_column(2)], f[kv4_column(3)]),
                                     kv4_pack(f[kv4_column(4)], f[kv4_column(5)]), kv4_pack(f[kv4_column(6)], f[kv4_column(7)]));
          *reinterpret_cast<uint4*>(smem + L::Q + g * (KV4_ROWS * 128) + threadIdx.x * 128 + ((i ^ (threadIdx.x & 7)) << 4)) = v;
        }
      }
      fence_proxy_async_smem();
    } else if (warp == 7) {
      feed.init(a, c, b, h, tile0, 1, stop);
      for (int i = 0; i < 2 && i < n; ++i) ok = ok && copy(i);
    }
    __syncthreads();                                                        // the queries are there

    if (warp == 7) {
      constexpr uint32_t qk = umma_idesc(128, 64, 0, 0, 0, 0), pv = umma_idesc(128, 64, 0, 0, 0, 1);
      for (int i = 0; i < n && ok; ++i) {
        const int k = n0 + i;
        if (!(ok = wait(&k_full, k, k))) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint64_t qd = umma_desc_kmajor_sw128(smem_u32(smem + L::Q) + g * (KV4_ROWS * 128)), kd = umma_desc_kmajor_sw128(smem_u32(smem + L::K) + g * L::CHUNK);
#pragma unroll
            for (int s = 0; s < 4; ++s) kv4_umma(tmem + L::T_S + g * 64, qd + 2 * s, kd + 2 * s, qk, s > 0);
          }
          umma_commit(&qk_done);
        }
        __syncwarp();
        if (i + 2 < n && !(ok = copy(i + 2))) break;
        if (!(ok = wait(&p_full, k, k) && wait(&v_full[k & 1], k >> 1, k))) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int s = 0; s < 4; ++s)
              kv4_umma_tmem(tmem + L::T_O + g * 64, tmem + L::T_S + g * 64 + s * 8,
                            umma_desc_mnmajor_sw128(smem_u32(smem + L::V) + ((k & 1) * NG + g) * L::CHUNK + s * 2048, L::CHUNK, 1024), pv, i > 0 || s > 0);
          umma_commit(&v_empty[k & 1]);
          umma_commit(&pv_done);
        }
        __syncwarp();
      }
    } else if (warp >= 4) {
      const int id = threadIdx.x - 128;                                     // of 96
      for (int i = 0; i < n && ok; ++i) {
        const int k = n0 + i;
        const uint8_t* raw = smem + L::RAW + (k & 1) * T::BYTES;
        float* par = reinterpret_cast<float*>(smem + L::PAR + (k & 1) * 2 * L::PAR_SIDE);
        const bool there = (tile0 + i) * TOK + id < end;                    // what lies behind is not of this request
        if (!(ok = wait(&raw_full[k & 1], k >> 1, k) && (k == 0 || wait(&qk_done, k - 1, k)))) break;
        for (int x = id; x < 64 * 4; x += 96) {
          const int t = x >> 2, cc = x & 3;
          uint32_t v[2 * NG];
          kv4_lds<2 * NG>(v, raw + t * (32 * NG) + cc * (8 * NG));
#pragma unroll
          for (int y = 0; y < 2 * NG; ++y)
            *reinterpret_cast<uint4*>(smem + L::K + (y >> 1) * L::CHUNK + t * 128 + (((2 * cc + (y & 1)) ^ (t & 7)) << 4)) = kv4_codes(v[y]);
        }
        if (id < 64) {
          uint32_t v[NG];
          kv4_lds<NG>(v, raw + T::KS0 + id * (4 * NG));
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float step = there ? kv4_step(v[g]) : 0.f;
            par[id * 2 * NG + g] = step;
            par[id * 2 * NG + NG + g] = there ? fmaf(step, 8.f, kv4_low(v[g])) : 0.f;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full);
        if (k >= 2 && !(ok = wait(&v_empty[k & 1], (k - 2) >> 1, k))) break;
        uint8_t* values = smem + L::V + (k & 1) * NG * L::CHUNK;
        for (int x = id; x < 32 * 8; x += 96) {
          const int pair = x >> 3, r = x & 7, ch = NG == 2 ? r ^ ((pair & 3) << 1) : r ^ (((pair >> 1) & 1) << 2);
          uint32_t v[2 * NG];
          kv4_lds<2 * NG>(v, raw + T::V0 + pair * (64 * NG) + ch * (8 * NG));
#pragma unroll
          for (int y = 0; y < 2 * NG; ++y) {
            const int t = pair * 2 + y / NG;
            *reinterpret_cast<uint4*>(values + (y % NG) * L::CHUNK + t * 128 + ((r ^ (t & 7)) << 4)) = kv4_codes(v[y]);
          }
        }
        if (id < 64) {
          uint32_t v[NG];
          kv4_lds<NG>(v, raw + T::VS0 + id * (4 * NG));
          float most = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float step = there ? kv4_step(v[g]) : 0.f;
            par[(64 + id) * 2 * NG + g] = step;
            par[(64 + id) * 2 * NG + NG + g] = there ? fmaf(step, 8.f, kv4_low(v[g])) : 0.f;
            most = fmaxf(most, step);
          }
          most = warp_max(most);
          if (lane == 0) s_most[k & 1][warp - 4] = most;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_full[k & 1]);
          mbar_arrive(&raw_empty[k & 1]);
        }
      }
    } else {
      const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
      const int sees = len - a.rows + 1 + min(row, total - 1) / rep;
      float m = -INFINITY, l = 0.f, z[NG], most = 0.f, to_one = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) z[g] = 0.f;
      for (int i = 0; i < n && ok; ++i) {
        const int k = n0 + i, t0 = (tile0 + i) * TOK;
        const float* par = reinterpret_cast<const float*>(smem + L::PAR + (k & 1) * 2 * L::PAR_SIDE);
        if (!(ok = wait(&qk_done, k, k) && wait(&v_full[k & 1], k >> 1, k))) break;
        tc_fence_after();
        float s[TOK];
#pragma unroll
        for (int x = 0; x < TOK; x += 8) {
          uint32_t v[NG][8];
#pragma unroll
          for (int g = 0; g < NG; ++g) kv4_tmem_ld8(mine + L::T_S + g * 64 + x, v[g]);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float p[2 * NG];
            if (NG == 2) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(par + (x + j) * 4);
            else *reinterpret_cast<float2*>(p) = *reinterpret_cast<const float2*>(par + (x + j) * 2);
            float y = p[NG] * qs[0];
            if (NG == 2) y = fmaf(p[3], qs[NG - 1], y);
#pragma unroll
            for (int g = 0; g < NG; ++g) y = fmaf(p[g], __uint_as_float(v[g][j]), y);
            s[x + j] = y;
          }
        }
        const bool edge = t0 + TOK > first_sees;                            // some row does not see all of the tile
        if (edge) {
#pragma unroll
          for (int j = 0; j < TOK; ++j)
            if (t0 + j >= sees) s[j] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < TOK; ++j) top = fmaxf(top, s[j]);
        const float steps = fmaxf(s_most[k & 1][0], s_most[k & 1][1]);
        // maxima and steps are followed as in kv4_decode.cu
        if (__any_sync(0xffffffffu, (top - m) * unit > 8.f || steps > most)) {
          const float to = fmaxf(top, m);
          float f = to == -INFINITY ? 1.f : ex2_fast((m - to) * unit);
          m = to;
          l *= f;
#pragma unroll
          for (int g = 0; g < NG; ++g) z[g] *= f;
          if (steps > most) {
            const float next = fmaxf(__uint_as_float((__float_as_uint(steps) + 0x007fffffu) & 0x7f800000u), 0x1p-110f);
            to_one = __uint_as_float(0x7f000000u - __float_as_uint(next)) * 128.f;
            f *= most * to_one * 0.0078125f;
            most = next;
          }
          if (i > 0) {
            if (!(ok = wait(&pv_done, k - 1, k))) break;
            tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
              uint32_t o[16];
              tmem_ld_x16(mine + L::T_O + x, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_x16(mine + L::T_O + x, o);
            }
            tmem_st_wait();
          }
        }
        const float sub = m == -INFINITY ? 0.f : m * unit;
        par += 64 * 2 * NG;
#pragma unroll
        for (int x = 0; x < TOK; x += 16) {
          uint32_t pk[NG][8];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float f[NG][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float pt = ex2_fast(fmaf(s[x + j + e], unit, -sub));
              l += pt;
              float v[2 * NG];
              if (NG == 2) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(par + (x + j + e) * 4);
              else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(par + (x + j + e) * 2);
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                f[g][e] = pt * (v[g] * to_one);
                if (edge && pt == 0.f) f[g][e] = 0.f;                       // an unseen token adds nothing, whatever its value
                else z[g] = fmaf(pt, v[NG + g], z[g]);
              }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) pk[g][j / 2] = kv4_pack(f[g][0], f[g][1]);
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) kv4_tmem_st8(mine + L::T_S + g * 64 + x / 2, pk[g]);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full);
      }
      if (ok && n > 0) ok = wait(&pv_done, n0 + n - 1, n);
      if (ok) {
        tc_fence_after();
        const float by = l == 0.f ? 0.f : 1.f / l, o_by = by * (most * 0.0078125f), lse = l == 0.f ? -INFINITY : m * unit + __log2f(l);
        const int head = h * rep + row % rep, tok = row / rep;
        const long long part = ((long long)blockIdx.x * 2 + (first ? 0 : 1)) * KV4_ROWS + threadIdx.x;
        if (row < total) {
          if (!whole) a.lse_part[part] = lse;
          else if (a.lse != nullptr) a.lse[((long long)b * a.hq + head) * a.rows + tok] = lse;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll 1
          for (int x = 0; x < 64; x += 16) {
            uint32_t o[16];
            if (n > 0) {
              tmem_ld_x16(mine + L::T_O + g * 64 + x, o);
              tmem_ld_wait();
            }
            if (row < total) {
              float f[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) f[(j & 8) + kv4_column(j & 7)] = by == 0.f ? 0.f : fmaf(__uint_as_float(o[j]), o_by, z[g] * by);
              if (whole) {
                uint32_t y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                  y[j] = *reinterpret_cast<const uint32_t*>(&v);
                }
                uint4* to = reinterpret_cast<uint4*>(a.out + (((long long)b * a.rows + tok) * a.hq + head) * D + g * 64 + x);
                to[0] = make_uint4(y[0], y[1], y[2], y[3]);
                to[1] = make_uint4(y[4], y[5], y[6], y[7]);
              } else {
                float4* to = reinterpret_cast<float4*>(a.o_part + part * D + g * 64 + x);
#pragma unroll
                for (int j = 0; j < 4; ++j) to[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
              }
            }
            __syncwarp();
          }
        }
        tc_fence_before();
      }
    }
    __syncthreads();                                                        // all roles are through with this part
    tc_fence_after();
    if (abort_flag != 0) break;
    n0 += n;
    w.left -= end_tile - tile0;
    if (w.left <= 0) break;
    w.tile0 = 0;
    if (++w.item == items) {
      w.item = 0;
      do w.n_tiles = kv4_tiles(a, c.block, TOK, ++w.b);                     // tiles are left, so there is a request that has some
      while (w.n_tiles == 0);
    }
  }
  if (abort_flag != 0) {                                                    // copies and products may still be under way: give them time
    if (threadIdx.x == 0) report_abort(&abort_flag, st);
    const uint64_t since = globaltimer_ns();
    while (globaltimer_ns() - since < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 7) {
    tc_fence_after();
    tmem_dealloc(tmem, L::T_COLS);
  }
}

template <int NG>
static cudaError_t kv4_rows_launch(const Kv4Decode& a, const Kv4Cache& c, long long grid, int B, OmniStatus* st, cudaStream_t stream) {
  static int most[64] = {0};
  const cudaError_t e = kv4_smem((const void*)kv4_rows_kernel<NG>, Kv4RowsLayout<NG>::BYTES, most);
  if (e != cudaSuccess) return e;
  kv4_rows_kernel<NG><<<(unsigned)grid, KV4_ROWS_THREADS, Kv4RowsLayout<NG>::BYTES, stream>>>(a, c, B, st);
  return cudaGetLastError();
}

cudaError_t kv4_launch_rows(const Kv4Decode& a, const Kv4Cache& c, int B, int blocks, OmniStatus* st, cudaStream_t stream) {
  const int total = a.rows * (a.hq / c.hkv);
  const long long grid = a.min_tiles == 0 ? (long long)B * c.hkv * ((total + KV4_ROWS - 1) / KV4_ROWS) : blocks;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return c.d == 64 ? kv4_rows_launch<1>(a, c, grid, B, st, stream) : kv4_rows_launch<2>(a, c, grid, B, st, stream);
}

}  // namespace omni
