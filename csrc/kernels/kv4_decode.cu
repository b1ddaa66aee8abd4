// Decode attention over the 4-bit paged key/value cache (layout: include/kv4.cuh).
//
//   q    [B rows, Hq, d] bf16: the last `rows` tokens of every request; row i of a request of L cached tokens sees L - rows + 1 + i
//   out  [B rows, Hq, d] bf16 = sum_t p_t v_t,  p = softmax_t(scale q k_t),  k_t and v_t = code * step + lowest
//   weights[t] = decay * weights[t] + sum over the rows and the query heads of a key/value head of p_t
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../include/kv4.cuh"
#include "../include/omni_ptx.cuh"

namespace omni {

constexpr int KV4_SITE_DECODE = 84;

struct Kv4Decode {
  const __nv_bfloat16* q;
  long long q_row;
  int q_head;
  const int *table, *seq_lens;
  int table_ld, table_w, rows, hq;
  float scale_log2;
  __nv_bfloat16* out;
  float* lse;                       // [B, Hq, rows] in units of log 2, or null
  float* weights;
  float decay;
};

__device__ __forceinline__ int kv4_length(const Kv4Decode& a, int block, int b, OmniStatus* st) {
  const int n = max(a.seq_lens[b], 0);
  if (n <= a.table_w * block) return n;
  if (threadIdx.x == 0) report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_DECODE, b);
  return a.table_w * block;
}

// q k of one token, or -inf for one in no valid block
__device__ __forceinline__ float kv4_score(const Kv4Decode& a, const Kv4Cache& c, const float* q, int b, int h, int t, OmniStatus* st) {
  const int blk = a.table[(long long)b * a.table_ld + t / c.block];
  if (blk < 0 || blk >= c.blocks) {
    report_status(st, OMNI_ERR_BOUNDS, KV4_SITE_DECODE, b);
    return -INFINITY;
  }
  const uint8_t* piece = c.k + c.at(blk, h);
  float s = 0.f;
  for (int u = 0; u < c.d / 8; ++u) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(piece + c.k_word(t % c.block, u));
    const uint32_t p = *reinterpret_cast<const uint32_t*>(piece + c.scale_word(t % c.block, u >> 3));
    for (int j = 0; j < 8; ++j) s = fmaf(q[u * 8 + j], fmaf((float)((w >> (4 * j)) & 15u), kv4_step(p), kv4_low(p)), s);
  }
  return s * a.scale_log2;
}

// One block for a query row: tiles of 128 tokens, a thread for each of them in the scores and for each column in the sums.
__global__ void __launch_bounds__(128) kv4_decode_kernel(Kv4Decode a, Kv4Cache c, OmniStatus* st) {
  const int b = blockIdx.z, row = blockIdx.y, hq = blockIdx.x, h = hq / (a.hq / c.hkv);
  __shared__ float q[256], p[128], red[4];
  const int sees = kv4_length(a, c.block, b, st) - a.rows + 1 + row;
  const long long at = (long long)b * a.rows + row;
  for (int i = threadIdx.x; i < c.d; i += 128) q[i] = __bfloat162float(a.q[at * a.q_row + (long long)hq * a.q_head + i]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int t0 = 0; t0 < sees; t0 += 128) {
    const int t = t0 + threadIdx.x;
    const float s = t < sees ? kv4_score(a, c, q, b, h, t, st) : -INFINITY;
    float top = warp_max(s);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float f = top == -INFINITY ? 1.f : exp2f(m - top), w = s == -INFINITY ? 0.f : exp2f(s - top);
    m = top;
    p[threadIdx.x] = w;
    const float part = warp_sum(w);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = part;
    __syncthreads();
    l = l * f + red[0] + red[1] + red[2] + red[3];
    for (int e = 0; e < 2; ++e) {
      const int d = threadIdx.x + 128 * e;
      if (d >= c.d) break;
      o[e] *= f;
      for (int i = 0; i < 128 && t0 + i < sees; ++i) {
        const int blk = a.table[(long long)b * a.table_ld + (t0 + i) / c.block];
        if (blk < 0 || blk >= c.blocks) continue;
        const uint8_t* piece = c.v + c.at(blk, h);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(piece + c.v_word((t0 + i) % c.block, d >> 3));
        const uint32_t g = *reinterpret_cast<const uint32_t*>(piece + c.scale_word((t0 + i) % c.block, d >> 6));
        o[e] = fmaf(p[i], fmaf((float)((w >> (4 * (d & 7))) & 15u), kv4_step(g), kv4_low(g)), o[e]);
      }
    }
    __syncthreads();
  }
  for (int e = 0; e < 2; ++e) {
    const int d = threadIdx.x + 128 * e;
    if (d < c.d) a.out[(at * a.hq + hq) * c.d + d] = __float2bfloat16(l == 0.f ? 0.f : o[e] / l);
  }
  if (a.lse != nullptr && threadIdx.x == 0) a.lse[((long long)b * a.hq + hq) * a.rows + row] = l == 0.f ? INFINITY : m + log2f(l);
}

// A thread for a token and head: its scores once more, against the finished softmax denominators.
__global__ void __launch_bounds__(128) kv4_weights_kernel(Kv4Decode a, Kv4Cache c, OmniStatus* st) {
  const int b = blockIdx.z, h = blockIdx.y, rep = a.hq / c.hkv;
  __shared__ float q[256];
  const int n = kv4_length(a, c.block, b, st), tiles = (n + 127) / 128;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int t = tile * 128 + threadIdx.x;
    float sum = 0.f;
    for (int r = 0; r < a.rows * rep; ++r) {
      const int row = r / rep, hq = h * rep + r % rep;
      const long long at = (long long)b * a.rows + row;
      __syncthreads();
      for (int i = threadIdx.x; i < c.d; i += 128) q[i] = __bfloat162float(a.q[at * a.q_row + (long long)hq * a.q_head + i]);
      __syncthreads();
      if (t < n - a.rows + 1 + row) sum += exp2f(kv4_score(a, c, q, b, h, t, st) - a.lse[((long long)b * a.hq + hq) * a.rows + row]);
    }
    if (t >= n) continue;
    const int blk = a.table[(long long)b * a.table_ld + t / c.block];
    if (blk < 0 || blk >= c.blocks) continue;
    float* w = a.weights + ((long long)blk * c.hkv + h) * c.block + t % c.block;
    *w = a.decay == 0.f ? sum : fmaf(a.decay, *w, sum);
  }
}

}  // namespace omni

using namespace omni;

extern "C" int omni_kv4_decode(const void* q, long long q_row, int q_head, const void* k_cache, const void* v_cache, long long blocks, int block,
                               int hkv, int d, const int* table, int table_ld, int table_w, const int* seq_lens, int B, int rows, int hq,
                               float scale, int max_len, void* out, float* lse, float* weights, float decay, void* status, cudaStream_t stream) {
  const Kv4Cache c = {(uint8_t*)k_cache, (uint8_t*)v_cache, blocks, block, hkv, d};
  if (!kv4_shape_ok(c) || hq % hkv != 0 || rows < 1 || hkv > 65535 || B > 65535 || rows > 65535) return -1;
  if (weights != nullptr && lse == nullptr) return -2;
  if (B <= 0) return 0;
  const Kv4Decode a = {(const __nv_bfloat16*)q, q_row, q_head, table, seq_lens, table_ld, table_w, rows, hq,
                       scale * 1.4426950408889634f, (__nv_bfloat16*)out, lse, weights, decay};
  kv4_decode_kernel<<<dim3(hq, rows, B), 128, 0, stream>>>(a, c, (OmniStatus*)status);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || weights == nullptr) return (int)e;
  const int tiles = (max_len + 127) / 128;
  kv4_weights_kernel<<<dim3(tiles < 1 ? 1 : tiles, hkv, B), 128, 0, stream>>>(a, c, (OmniStatus*)status);
  return (int)cudaGetLastError();
}
