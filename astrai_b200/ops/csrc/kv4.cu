// The 4-bit KV cache (format: kv4.cuh): storing rows, reading rows back, decode attention on the codes, copying pages.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv4.cuh"
#include "launchers.h"

namespace ab {

// ------------------------------------------------------------------------------------------------------- store rows
// D / 8 lanes a row, blockIdx.y = 0 for keys, 1 for values.  A slot outside the pool is skipped.
template <int D, typename Loc>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v,
                                                         uint8_t* __restrict__ k_codes, uint32_t* __restrict__ k_meta,
                                                         uint8_t* __restrict__ v_codes, uint32_t* __restrict__ v_meta,
                                                         const Loc* __restrict__ loc, long long rows, int heads, long long n_slots,
                                                         long long k_tok, long long k_head, long long v_tok, long long v_head) {
  constexpr int LPR = D / 8;
  const bool key = blockIdx.y == 0;
  const int l = threadIdx.x % LPR;
  const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / LPR;
  const long long t = r / heads;
  const int h = (int)(r - t * heads);
  const long long slot = r < rows ? (long long)loc[t] : -1;
  const bool live = slot >= 0 && slot < n_slots;
  const long long at = live ? slot * heads + h : 0;
  const __nv_bfloat16* src = key ? k + t * k_tok + h * k_head : v + t * v_tok + h * v_head;
  kv4_store_row<D>(live, key, l, src, (key ? k_codes : v_codes) + at * (D / 2), (key ? k_meta : v_meta) + at * (D / 32));
}

int kv4_append(const void* k, const void* v, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* loc, bool loc64,
               long long tokens, int heads, int head_dim, long long n_slots, long long k_tok, long long k_head, long long v_tok,
               long long v_head, cudaStream_t st) {
  const long long rows = tokens * heads;
  if (rows == 0) return 0;
  const long long blocks = (rows * (head_dim / 8) + 255) / 256;
  if (blocks > 0x7fffffffLL) return -4;
  const dim3 grid((unsigned)blocks, 2);
#define AB_APPEND(DD, LL)                                                                                                     \
  kv4_append_kernel<DD, LL><<<grid, 256, 0, st>>>((const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (uint8_t*)k_codes,         \
                                                  (uint32_t*)k_meta, (uint8_t*)v_codes, (uint32_t*)v_meta, (const LL*)loc,     \
                                                  rows, heads, n_slots, k_tok, k_head, v_tok, v_head)
#define AB_APPEND_D(DD) \
  if (loc64) AB_APPEND(DD, long long); else AB_APPEND(DD, int)
  switch (head_dim) {
    case 32: AB_APPEND_D(32); break;
    case 64: AB_APPEND_D(64); break;
    case 128: AB_APPEND_D(128); break;
    case 256: AB_APPEND_D(256); break;
    default: return -3;
  }
#undef AB_APPEND_D
#undef AB_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// -------------------------------------------------------------------------------------------------------- read rows
// The reverse, as bf16 rows [tokens, heads, D].  A slot outside the pool reads as zeros.
template <int D, typename Loc>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const uint8_t* __restrict__ k_codes, const uint32_t* __restrict__ k_meta,
                                                         const uint8_t* __restrict__ v_codes, const uint32_t* __restrict__ v_meta,
                                                         const Loc* __restrict__ loc, __nv_bfloat16* __restrict__ k,
                                                         __nv_bfloat16* __restrict__ v, long long rows, int heads, long long n_slots) {
  constexpr int LPR = D / 8;
  const bool key = blockIdx.y == 0;
  const int l = threadIdx.x % LPR;
  const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / LPR;
  if (r >= rows) return;
  const long long t = r / heads;
  const int h = (int)(r - t * heads);
  const long long slot = (long long)loc[t];
  Vec8<__nv_bfloat16> out;
  out.raw = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < n_slots) {
    const long long at = slot * heads + h;
    const uint8_t* codes = (key ? k_codes : v_codes) + at * (D / 2);
    const uint32_t ms = (key ? k_meta : v_meta)[at * (D / 32) + (l >> 2)];
    uint32_t word;
    if (key) {
      word = reinterpret_cast<const uint32_t*>(codes)[kv4_key_word<D>(l >> 2, l & 3)];
    } else {
      const uint16_t* halves = reinterpret_cast<const uint16_t*>(codes);
      word = halves[kv4_value_half<D>(l >> 2, 2 * (l & 3))] | ((uint32_t)halves[kv4_value_half<D>(l >> 2, 2 * (l & 3) + 1)] << 16);
    }
    const float m = __uint_as_float(ms << 16), s = __uint_as_float(ms & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fma_ieee(s, (float)((int)((word >> (4 * j)) & 15) - 8), m);
    out.pack(x);
  }
  out.store((key ? k : v) + r * D + 8 * l);
}

int kv4_gather(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const void* loc, bool loc64, void* k,
               void* v, long long tokens, int heads, int head_dim, long long n_slots, cudaStream_t st) {
  const long long rows = tokens * heads;
  if (rows == 0) return 0;
  const long long blocks = (rows * (head_dim / 8) + 255) / 256;
  if (blocks > 0x7fffffffLL) return -4;
  const dim3 grid((unsigned)blocks, 2);
#define AB_GATHER(DD, LL)                                                                                                       \
  kv4_gather_kernel<DD, LL><<<grid, 256, 0, st>>>((const uint8_t*)k_codes, (const uint32_t*)k_meta, (const uint8_t*)v_codes,     \
                                                  (const uint32_t*)v_meta, (const LL*)loc, (__nv_bfloat16*)k, (__nv_bfloat16*)v, \
                                                  rows, heads, n_slots)
#define AB_GATHER_D(DD) \
  if (loc64) AB_GATHER(DD, long long); else AB_GATHER(DD, int)
  switch (head_dim) {
    case 32: AB_GATHER_D(32); break;
    case 64: AB_GATHER_D(64); break;
    case 128: AB_GATHER_D(128); break;
    case 256: AB_GATHER_D(256); break;
    default: return -3;
  }
#undef AB_GATHER_D
#undef AB_GATHER
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// -------------------------------------------------------------------------------------------------- decode attention
// One CTA per (kv head, request, split of the keys), a warp per key, a lane per D / 32 numbers.  With k_new / v_new the
// CTA whose share ends at the last position first stores that position's rows.
constexpr int K4_WARPS = 4;

template <int D, int G>
__global__ void __launch_bounds__(K4_WARPS * 32)
kv4_decode_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* k_codes, const uint32_t* k_meta, const uint8_t* v_codes,
                  const uint32_t* v_meta, const int* __restrict__ req_to_token, const int* __restrict__ req_pool_indices,
                  const long long* __restrict__ seq_lens, const __nv_bfloat16* __restrict__ k_new,
                  const __nv_bfloat16* __restrict__ v_new, float* __restrict__ o_part, float* __restrict__ ml_part,
                  int* __restrict__ counters, __nv_bfloat16* __restrict__ out, int n_kv_heads, int max_ctx, int table_rows,
                  long long n_slots, float scale_log2, int max_splits) {
  constexpr int E = D / 32;  // numbers of a lane
  const int kvh = blockIdx.x, b = blockIdx.y, split = blockIdx.z, splits = gridDim.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // lengths beyond the table row are cut to the row, a row outside the table attends to nothing
  long long len = seq_lens[b];
  len = len < 0 ? 0 : (len > max_ctx ? (long long)max_ctx : len);
  int row = req_pool_indices[b];
  if (row < 0 || row >= table_rows) row = 0, len = 0;
  const int* table = req_to_token + (long long)row * max_ctx;
  const long long chunk = ((len + splits - 1) / splits + 31) / 32 * 32;
  const long long begin = split * chunk, end = min(len, begin + chunk);
  const int n_q_heads = n_kv_heads * G;

  if (k_new != nullptr && end == len && begin < len) {
    const long long slot = table[len - 1];
    if (slot >= 0 && slot < n_slots && warp < 2) {
      const long long at = slot * n_kv_heads + kvh, src = ((long long)b * n_kv_heads + kvh) * D;
      const bool key = warp == 0;
      const int l = lane % (D / 8);
      kv4_store_row<D>(lane < D / 8, key, l, (key ? k_new : v_new) + src,
                       const_cast<uint8_t*>(key ? k_codes : v_codes) + at * (D / 2),
                       const_cast<uint32_t*>(key ? k_meta : v_meta) + at * (D / 32));
    }
    __syncthreads();
  }

  float qf[G][E], acc[G][E], m[G], sum[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY, sum[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[g][e] = 0.f;
      qf[g][e] = to_f(q[((long long)b * n_q_heads + kvh * G + g) * D + e * 32 + lane]) * scale_log2;
    }
  }
  for (long long t = begin + warp; t < end; t += K4_WARPS) {
    const long long slot = table[t];
    if (slot < 0 || slot >= n_slots) continue;
    const long long at = slot * n_kv_heads + kvh;
    float s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) s[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {  // number lane of group e
      const uint32_t ms = k_meta[at * E + e];
      const uint32_t w = reinterpret_cast<const uint32_t*>(k_codes + at * (D / 2))[kv4_key_word<D>(e, lane >> 3)];
      const float x = __uint_as_float(ms << 16) + __uint_as_float(ms & 0xffff0000u) * (float)((int)((w >> (4 * (lane & 7))) & 15) - 8);
#pragma unroll
      for (int g = 0; g < G; ++g) s[g] += qf[g][e] * x;
    }
    float vx[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t ms = v_meta[at * E + e];
      const uint32_t w = reinterpret_cast<const uint16_t*>(v_codes + at * (D / 2))[kv4_value_half<D>(e, lane >> 2)];
      vx[e] = __uint_as_float(ms << 16) + __uint_as_float(ms & 0xffff0000u) * (float)((int)((w >> (4 * (lane & 3))) & 15) - 8);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sc = warp_sum(s[g]);
      const float nm = fmaxf(m[g], sc), base = nm == -INFINITY ? 0.f : nm;
      const float alpha = exp2f(m[g] - base), p = exp2f(sc - base);
      sum[g] = sum[g] * alpha + p;
      m[g] = nm;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = acc[g][e] * alpha + p * vx[e];
    }
  }

  __shared__ float s_acc[K4_WARPS][G][D];
  __shared__ float s_ml[K4_WARPS][G][2];
  __shared__ int s_last;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_acc[warp][g][e * 32 + lane] = acc[g][e];
    if (lane == 0) s_ml[warp][g][0] = m[g], s_ml[warp][g][1] = sum[g];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    const int g = i / D, d = i % D;
    float mm = -INFINITY, o = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < K4_WARPS; ++w) mm = fmaxf(mm, s_ml[w][g][0]);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < K4_WARPS; ++w) {
      const float f = exp2f(s_ml[w][g][0] - base);
      o += s_acc[w][g][d] * f;
      ll += s_ml[w][g][1] * f;
    }
    const long long head = (long long)b * n_q_heads + kvh * G + g;
    o_part[(head * max_splits + split) * D + d] = o;
    if (d == 0) {
      ml_part[(head * max_splits + split) * 2] = mm;
      ml_part[(head * max_splits + split) * 2 + 1] = ll;
    }
  }
  // the last CTA of this (request, kv head) combines the splits
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int done = atomicAdd(&counters[b * n_kv_heads + kvh], 1);
    s_last = done == splits - 1;
    if (s_last) counters[b * n_kv_heads + kvh] = 0;  // ready for the next launch
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int i = threadIdx.x; i < G * D; i += blockDim.x) {
    const int g = i / D, d = i % D;
    const long long head = (long long)b * n_q_heads + kvh * G + g;
    float mm = -INFINITY, o = 0.f, ll = 0.f;
    for (int s = 0; s < splits; ++s) mm = fmaxf(mm, ml_part[(head * max_splits + s) * 2]);
    const float base = mm == -INFINITY ? 0.f : mm;
    for (int s = 0; s < splits; ++s) {
      const float f = exp2f(ml_part[(head * max_splits + s) * 2] - base);
      o += o_part[(head * max_splits + s) * D + d] * f;
      ll += ml_part[(head * max_splits + s) * 2 + 1] * f;
    }
    out[head * D + d] = __float2bfloat16_rn(ll == 0.f ? 0.f : o / ll);
  }
}

int kv4_decode_splits(int batch, int n_kv_heads, long long max_len, int max_splits) {
  const long long base = (long long)batch * n_kv_heads;
  long long s = (148 * 2) / (base < 1 ? 1 : base);
  const long long by_len = (max_len + 127) / 128;
  if (s > by_len) s = by_len;
  if (s > max_splits) s = max_splits;
  return (int)(s < 1 ? 1 : s);
}

int kv4_decode(const void* q, const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const int* req_to_token,
               const int* req_pool_indices, const long long* seq_lens, const void* k_new, const void* v_new, float* o_part, float* ml_part,
               int* counters, void* out, int batch, int n_q_heads, int n_kv_heads, int head_dim, int max_ctx, int table_rows,
               long long n_slots, float scale, int splits, int max_splits, cudaStream_t st) {
  if (batch == 0) return 0;
  if (n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 8) return -1;
  if (splits < 1 || splits > max_splits) return -2;
  if (batch > 65535 || splits > 65535) return -4;
  const dim3 grid(n_kv_heads, batch, splits);
#define AB_K4(DD, GG)                                                                                                              \
  kv4_decode_kernel<DD, GG><<<grid, K4_WARPS * 32, 0, st>>>(                                                                       \
      (const __nv_bfloat16*)q, (const uint8_t*)k_codes, (const uint32_t*)k_meta, (const uint8_t*)v_codes, (const uint32_t*)v_meta, \
      req_to_token, req_pool_indices, seq_lens, (const __nv_bfloat16*)k_new, (const __nv_bfloat16*)v_new, o_part, ml_part,         \
      counters, (__nv_bfloat16*)out, n_kv_heads, max_ctx, table_rows, n_slots, scale * 1.4426950408889634f, max_splits)
#define AB_K4_G(DD)               \
  switch (n_q_heads / n_kv_heads) { \
    case 1: AB_K4(DD, 1); break;    \
    case 2: AB_K4(DD, 2); break;    \
    case 3: AB_K4(DD, 3); break;    \
    case 4: AB_K4(DD, 4); break;    \
    case 5: AB_K4(DD, 5); break;    \
    case 6: AB_K4(DD, 6); break;    \
    case 7: AB_K4(DD, 7); break;    \
    default: AB_K4(DD, 8); break;   \
  }
  switch (head_dim) {
    case 32: AB_K4_G(32); break;
    case 64: AB_K4_G(64); break;
    case 128: AB_K4_G(128); break;
    case 256: AB_K4_G(256); break;
    default: return -3;
  }
#undef AB_K4_G
#undef AB_K4
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// ------------------------------------------------------------------------------------------------------- copy pages
// Page dst[i] of every layer of every pool becomes a copy of page src[i].  The page numbers travel in the launch's
// parameters, so the call keeps no buffer alive and can be captured into a graph as it stands.
template <typename Unit>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageCopies c) {
  const int pool = blockIdx.z, layer = blockIdx.y, pair = blockIdx.x;
  const long long page = c.page_bytes[pool];
  char* base = static_cast<char*>(c.base[pool]) + layer * c.layer_bytes[pool];
  const Unit* src = reinterpret_cast<const Unit*>(base + c.src[pair] * page);
  Unit* dst = reinterpret_cast<Unit*>(base + c.dst[pair] * page);
  const long long n = page / (long long)sizeof(Unit);
  for (long long i = threadIdx.x; i < n; i += blockDim.x) dst[i] = src[i];
}

int copy_pages(const PageCopies& c, int pairs, int layers, int pools, cudaStream_t st) {
  if (pairs == 0 || layers == 0 || pools == 0) return 0;
  if (layers > 65535) return -4;
  uintptr_t bits = 0;  // the widest unit that divides every address and every size
  for (int p = 0; p < pools; ++p)
    bits |= reinterpret_cast<uintptr_t>(c.base[p]) | (uintptr_t)c.page_bytes[p] | (uintptr_t)c.layer_bytes[p];
  const dim3 grid(pairs, layers, pools);
  if (bits % 16 == 0) copy_pages_kernel<uint4><<<grid, 256, 0, st>>>(c);
  else if (bits % 4 == 0) copy_pages_kernel<uint32_t><<<grid, 256, 0, st>>>(c);
  else copy_pages_kernel<uint8_t><<<grid, 256, 0, st>>>(c);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // namespace ab
