// The 4-bit KV cache (format: kv4.cuh): storing rows, reading rows back, decode attention on the codes, copying pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
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
// Attention of one query per request on the codes themselves.  With c the codes (0..15), s / m the steps and middles and
// lo = m - 8 s, for key k, group g and head h:
//   logit = sum_g s_kg (q_hg . c_kg) + lo_kg sum(q_hg)       out_d = sum_k (p_k s_kg) c_kd + sum_k p_k lo_kg   (d in g)
// so the big products take the codes as they are: a code in the low bits of an fp16 IS the number c 2^-24 (a subnormal),
// and one shifted left by four is c 2^-20, so a pair of numbers costs one AND (and every second pair a shift).  The
// other operand is the query times a power of two that puts its largest number below 2^14 (exact), or p s times a power
// of two that puts the tile's largest step below 2^15 (rounded to fp16: 2^-11 of each product; the query's and the
// steps' own sizes cost nothing).  Products go to m16n8k16 tensor instructions with fp32 sums: a tile's share of `out` is
// summed from zero and added to the running sum in fp32 registers, so a long context loses nothing to the tensor
// accumulator's rounding.  lo_kg sum(q_hg) is a product of the (m, s) words as they lie in memory with (sum q, -8 sum q)
// split into three bf16 parts (24 bits).
//
// Work: the keys of every (request, kv head) are cut into units of 32 W keys; the units of the whole batch, laid end to
// end, are divided evenly over the CTAs of one wave, whatever the lengths.  A CTA of W warps walks its range segment by
// segment; warp w takes every W-th tile of 32 keys, streams it through a ring of its own in shared memory (cp.async, no
// barrier between warps) and the warps' sums meet at the end of the segment.  A segment that several CTAs share is joined
// by the one that finishes last.
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
  const int n = live ? N : 0;  // 0: zeros are written and nothing is read
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

struct Kv4Attn {
  const __nv_bfloat16* q;
  uint8_t *k_codes, *v_codes;
  uint32_t *k_meta, *v_meta;
  const int *table, *rows;
  const long long* lens;
  const __nv_bfloat16 *k_new, *v_new;
  float *o_part, *ml_part;
  int* counters;
  __nv_bfloat16* out;
  int batch, heads, group, max_ctx, table_rows;  // heads: kv heads; group: query heads of one
  long long n_slots;
  float scale_log2;
};

template <int N> struct Words { uint32_t w[N]; };
template <int N> __device__ __forceinline__ Words<N> lds_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 1) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); r.w[0] = v.x, r.w[1] = v.y; }
  else { const uint4 v = *reinterpret_cast<const uint4*>(p); r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w; }
  return r;
}

template <int D> struct Kv4Tile {  // a tile of 32 keys in shared memory
  static constexpr int NG = D / 32, KEYS = 32, CODES = KEYS * D / 2, META = KEYS * NG * 4;
  static constexpr int K = 0, V = CODES, KM = 2 * CODES, VM = 2 * CODES + META, BYTES = 2 * (CODES + META);
  static constexpr int STAGES = D == 256 ? 2 : 3;
  // 16-byte pieces of a row are swapped by the row's number so that neither the lanes' reads of keys (two rows at a time)
  // nor those of values (four rows, a quarter of each) meet in a bank
  static __device__ __forceinline__ int swap(int r) { return D == 128 ? (r & 2) : D == 256 ? (((r & 1) << 2) | (r & 2)) : 0; }
};

template <int D, int W>
__global__ void __launch_bounds__(W * 32, D == 256 ? 2 : 3) kv4_attn_kernel(const Kv4Attn p) {
  using T = Kv4Tile<D>;
  constexpr int NG = T::NG, NB = NG < 4 ? NG : 4, BATCHES = NG / NB, STAGES = T::STAGES, UNIT = 32 * W;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t s_mask[W][STAGES];
  __shared__ float s_ml[W][8][2], s_z[W][8][NG];
  __shared__ long long s_scan[W + 1], s_found[2];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = smem + warp * STAGES * T::BYTES;

  // a length beyond the table row is cut to the row, a row outside the table attends to nothing
  auto length = [&](int b) -> long long {
    const int row = p.rows[b];
    const long long n = p.lens[b];
    return row < 0 || row >= p.table_rows || n < 0 ? 0 : n > p.max_ctx ? p.max_ctx : n;
  };
  auto units = [&](long long n) -> long long { return n <= UNIT ? 1 : (n + UNIT - 1) / UNIT; };

  // this CTA's share [u, u_end) of all units, and the request that u lies in
  long long total, u, u_end;
  int b;
  long long seg_start;  // first unit of the current segment (request b, head kvh)
  int kvh;
  {
    const int per = (p.batch + W * 32 - 1) / (W * 32);
    const int b0 = threadIdx.x * per;
    long long mine = 0;
    for (int i = 0; i < per && b0 + i < p.batch; ++i) mine += units(length(b0 + i));
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    total *= p.heads;
    before *= p.heads;
    const long long n = min((long long)gridDim.x, total);
    if (blockIdx.x >= n) return;
    u = blockIdx.x * total / n;
    u_end = (blockIdx.x + 1) * total / n;
    if (u >= before && u < before + mine * p.heads) {
      long long at = before;
      int i = 0;
      for (;; ++i) {
        const long long here = units(length(b0 + i)) * p.heads;
        if (u < at + here) break;
        at += here;
      }
      s_found[0] = b0 + i, s_found[1] = at;
    }
    __syncthreads();
    b = (int)s_found[0];
    const long long nu = units(length(b));
    kvh = (int)((u - s_found[1]) / nu);
    seg_start = s_found[1] + kvh * nu;
  }
  const long long n_ctas = min((long long)gridDim.x, total);

  while (u < u_end) {
    const long long len = length(b), nu = units(len);
    const long long seg_end = seg_start + nu, stop = min(u_end, seg_end);
    const int seg = b * p.heads + kvh;
    const int* table = p.table + (long long)(len > 0 ? p.rows[b] : 0) * p.max_ctx;
    const long long key_end = min(len, (stop - seg_start) * UNIT);
    long long key = (u - seg_start) * UNIT + warp * 32;  // first key of this warp's next tile

    // ---- copies: a tile's slots, then its rows
    auto slot_of = [&](long long k0) -> int { return k0 + lane < key_end ? table[k0 + lane] : -1; };
    auto issue = [&](long long k0, int slot, int stage) {
      if (p.k_new != nullptr && k0 < len && k0 + 32 >= len) {  // the step's own rows: stored before they are read
        const int at = __shfl_sync(0xffffffffu, slot, (int)(len - 1 - k0));
        const bool ok = at >= 0 && at < p.n_slots;
        constexpr int LPR = D / 8;
        const long long to = ((long long)(ok ? at : 0) * p.heads + kvh), from = ((long long)b * p.heads + kvh) * D;
#pragma unroll
        for (int pass = 0; pass < (D == 256 ? 2 : 1); ++pass) {
          const int which = D == 256 ? pass : lane / LPR;
          kv4_store_row<D>(ok && which < 2, which == 0, lane % LPR, (which == 0 ? p.k_new : p.v_new) + from,
                           (which == 0 ? p.k_codes : p.v_codes) + to * (D / 2), (which == 0 ? p.k_meta : p.v_meta) + to * NG);
        }
        __threadfence();
        __syncwarp();
      }
      const bool live = slot >= 0 && slot < p.n_slots;
      const uint32_t mask = __ballot_sync(0xffffffffu, live);
      if (lane == 0) s_mask[warp][stage] = mask;
      const uint32_t base = smem_addr(ring + stage * T::BYTES);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int c = i * 32 + lane, r = c / NG, piece = c % NG;
        const int s = __shfl_sync(0xffffffffu, live ? slot : 0, r);
        const bool on = (mask >> r) & 1;
        const long long from = ((long long)s * p.heads + kvh) * (D / 2) + piece * 16;
        const uint32_t to = base + r * (D / 2) + ((piece ^ T::swap(r)) * 16);
        cp_async<16>(to + T::K, p.k_codes + from, on);
        cp_async<16>(to + T::V, p.v_codes + from, on);
      }
      const long long from = ((long long)(live ? slot : 0) * p.heads + kvh) * NG;
      constexpr int PIECE = NG < 4 ? NG * 4 : 16;
#pragma unroll
      for (int i = 0; i < NG * 4 / PIECE; ++i) {
        cp_async<PIECE>(base + T::KM + lane * NG * 4 + i * PIECE, reinterpret_cast<const uint8_t*>(p.k_meta + from) + i * PIECE, live);
        cp_async<PIECE>(base + T::VM + lane * NG * 4 + i * PIECE, reinterpret_cast<const uint8_t*>(p.v_meta + from) + i * PIECE, live);
      }
    };
    int slot = slot_of(key);
    long long ahead = key;  // first key of the next tile to copy
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (ahead < key_end) {
        const int cur = slot;
        slot = slot_of(ahead + UNIT);
        issue(ahead, cur, s);
        ahead += UNIT;
      }
      cp_commit();
    }

    // ---- the query as operand A: row gid = head, numbers 32 w + 8 tig + (0 4 | 1 5 | 2 6 | 3 7) as pairs
    uint32_t qa[NG][4], qs[BATCHES][3];
    float back;  // undoes the query's power of two
    {
      float x[NG][8], big = 0.f;
      const bool on = gid < p.group;
      const __nv_bfloat16* src = p.q + (((long long)b * p.heads + kvh) * p.group + (on ? gid : 0)) * D + 8 * tig;
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        Vec8<__nv_bfloat16> v;
        v.load(src + 32 * w);
        v.unpack(x[w]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!on) x[w][j] = 0.f;
          big = fmaxf(big, fabsf(x[w][j]));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int e = min(126, 140 - (int)(__float_as_uint(big) >> 23));
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      back = __uint_as_float((uint32_t)(127 - e) << 23);
      float sums[NG];
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) t += x[w][j];
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        sums[w] = t * p.scale_log2;
        const float odd = up * 0.0625f;
        qa[w][0] = half2_bits(x[w][0] * up, x[w][4] * up), qa[w][1] = half2_bits(x[w][1] * odd, x[w][5] * odd);
        qa[w][2] = half2_bits(x[w][2] * up, x[w][6] * up), qa[w][3] = half2_bits(x[w][3] * odd, x[w][7] * odd);
      }
#pragma unroll
      for (int h = 0; h < BATCHES; ++h) {  // lane tig: (sum, -8 sum) of group 4 h + tig, in three parts
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NB; ++w) t = tig == w ? sums[h * NB + w] : t;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const float part = __bfloat162float(__float2bfloat16_rn(t));
          const __nv_bfloat162 pair = __floats2bfloat162_rn(part, -8.f * part);
          qs[h][i] = *reinterpret_cast<const uint32_t*>(&pair);
          t -= part;
        }
      }
    }

    float o[NG][2][4], z[NG], mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      z[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i >> 2][i & 3] = 0.f;
    }
    const int key_row = (gid & 1) ? ((gid >> 1) ^ 1) + 4 : gid >> 1;  // row of a block of 8 keys that column gid stands for
    const int row_e[2] = {tig, (tig ^ 1) + 4};                        // rows of columns 2 tig and 2 tig + 1

    for (int stage = 0; key < key_end; key += UNIT) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      const uint8_t* tile = ring + stage * T::BYTES;
      const uint32_t mask = s_mask[warp][stage];
      {  // the tile after the ones in flight goes into the stage that the previous turn has read
        const int next = stage == 0 ? STAGES - 1 : stage - 1;
        if (ahead < key_end) {
          const int cur = slot;
          slot = slot_of(ahead + UNIT);
          issue(ahead, cur, next);
          ahead += UNIT;
        }
        cp_commit();
      }
      // ---- logits of 4 blocks of 8 keys: this lane's head is gid, its keys row_e[0] and row_e[1] of each block
      float s[4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = 8 * n + key_row;
        float term[4] = {0.f, 0.f, 0.f, 0.f}, acc[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < BATCHES; ++h) {
          const uint32_t word = tig < NB ? *reinterpret_cast<const uint32_t*>(tile + T::KM + (r * NG + h * NB + (tig < NB ? tig : 0)) * 4) : 0u;
          mma_bf16(term, qs[h][0], 0u, qs[h][1], 0u, word, word);
          mma_bf16(term, qs[h][2], 0u, 0u, 0u, word, 0u);
          Words<NB> ms[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) ms[e] = lds_words<NB>(tile + T::KM + ((8 * n + row_e[e]) * NG + h * NB) * 4);
          Words<NB> codes;
          if constexpr (NG >= 4) codes = lds_words<NB>(tile + T::K + r * (D / 2) + (((4 * h + tig) ^ T::swap(r)) * 16));
          else codes = lds_words<NB>(tile + T::K + r * (D / 2) + tig * NB * 4);
#pragma unroll
          for (int w = 0; w < NB; ++w) {
            const uint32_t x = codes.w[w], y = x >> 8;
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(part, qa[h * NB + w][0], 0u, qa[h * NB + w][1], 0u, x & 0x000f000fu, x & 0x00f000f0u);
            mma_f16(part, qa[h * NB + w][2], 0u, qa[h * NB + w][3], 0u, y & 0x000f000fu, y & 0x00f000f0u);
            acc[0] = fmaf(part[0], high_bf16(ms[0].w[w]), acc[0]);
            acc[1] = fmaf(part[1], high_bf16(ms[1].w[w]), acc[1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float logit = fmaf(acc[e] * back, p.scale_log2 * 0x1p24f, term[e]);
          s[n][e] = (mask >> (8 * n + row_e[e])) & 1 ? logit : -INFINITY;
        }
      }
      // ---- softmax of the tile
      float top = mx;
#pragma unroll
      for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(s[n][0], s[n][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float base = top == -INFINITY ? 0.f : top;
      if (__any_sync(0xffffffffu, top != mx)) {
        const float alpha = exp2f(mx - base);
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * tig), a1 = __shfl_sync(0xffffffffu, alpha, 8 * tig + 4);
        sum *= alpha;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          z[g] *= alpha;
#pragma unroll
          for (int t = 0; t < 2; ++t) o[g][t][0] *= a0, o[g][t][1] *= a1, o[g][t][2] *= a0, o[g][t][3] *= a1;
        }
        mx = top;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][e] = exp2f(s[n][e] - base);
          sum += s[n][e];
        }
      // ---- the power of two that puts the largest step of the tile into [2^14, 2^15)
      uint32_t largest = 0;
#pragma unroll
      for (int h = 0; h < BATCHES; ++h) {
        const Words<NB> ms = lds_words<NB>(tile + T::VM + (lane * NG + h * NB) * 4);
#pragma unroll
        for (int w = 0; w < NB; ++w) largest = max(largest, ms.w[w]);
      }
      largest = __reduce_max_sync(0xffffffffu, largest);
      const uint32_t ex = min(254u, 268u - min(254u, (largest >> 23) & 0xffu));
      const float up = __uint_as_float(ex << 23);
      const float down = __uint_as_float((278u - ex) << 23);  // 2^24 / up
      // ---- out
#pragma unroll
      for (int h = 0; h < BATCHES; ++h) {
        float t[NB][2][4];
#pragma unroll
        for (int g = 0; g < NB; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) t[g][i >> 2][i & 3] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          constexpr int VW = NB < 2 ? 1 : NB / 2;  // words of a lane's share of a row
          Words<NB> ms[2][2];
          Words<VW> codes[2][2];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = 16 * j + 8 * n + row_e[e];
              ms[n][e] = lds_words<NB>(tile + T::VM + (r * NG + h * NB) * 4);
              const uint8_t* row = tile + T::V + r * (D / 2);
              if constexpr (D == 256) codes[n][e] = lds_words<VW>(row + ((gid ^ T::swap(r)) * 16) + h * 8);
              else if constexpr (D == 128) codes[n][e] = lds_words<VW>(row + (((gid >> 1) ^ T::swap(r)) * 16) + (gid & 1) * 8);
              else if constexpr (D == 64) codes[n][e] = lds_words<VW>(row + gid * 4);
              else codes[n][e].w[0] = *reinterpret_cast<const uint16_t*>(row + gid * 2);
            }
#pragma unroll
          for (int g = 0; g < NB; ++g) {
            uint32_t pb[2], pair[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float ps[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float step = high_bf16(ms[n][e].w[g]), prob = s[2 * j + n][e];
                z[h * NB + g] = fmaf(prob, fmaf(-8.f, step, low_bf16(ms[n][e].w[g])), z[h * NB + g]);
                ps[e] = prob * (step * up);
              }
              pb[n] = half2_bits(ps[0], ps[1]);
              pair[n] = __byte_perm(codes[n][0].w[g >> 1], codes[n][1].w[g >> 1], (g & 1) ? 0x7632 : 0x5410);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = i ? pair[0] >> 8 : pair[0], y = i ? pair[1] >> 8 : pair[1];
              mma_f16(t[g][i], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[0], pb[1]);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < NB; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float(&to)[4] = o[h * NB + g][i];
            to[0] = fmaf(t[g][i][0], down, to[0]), to[1] = fmaf(t[g][i][1], down, to[1]);
            to[2] = fmaf(t[g][i][2], down * 0.0625f, to[2]), to[3] = fmaf(t[g][i][3], down * 0.0625f, to[3]);
          }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncwarp();

    // ---- the warps' sums meet: out of each warp [8 heads][D] in its own ring
    float* mine = reinterpret_cast<float*>(ring);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      z[g] += __shfl_xor_sync(0xffffffffu, z[g], 1);
      z[g] += __shfl_xor_sync(0xffffffffu, z[g], 2);
      if (tig == 0) s_z[warp][gid][g] = z[g];
#pragma unroll
      for (int h = 0; h < 2; ++h)  // heads 2 tig and 2 tig + 1; numbers 32 g + 4 gid .. + 3
        *reinterpret_cast<float4*>(mine + (2 * tig + h) * D + 32 * g + 4 * gid) = make_float4(o[g][0][h], o[g][0][2 + h], o[g][1][h], o[g][1][2 + h]);
    }
    if (tig == 0) s_ml[warp][gid][0] = mx, s_ml[warp][gid][1] = sum;
    __syncthreads();
    const bool whole = u == seg_start && stop == seg_end;
    const long long cta0 = whole ? 0 : ((seg_start + 1) * n_ctas - 1) / total, cta1 = whole ? 0 : (seg_end * n_ctas - 1) / total;
    float* part = p.o_part + (blockIdx.x + (long long)seg) * p.group * D;
    float* part_ml = p.ml_part + (blockIdx.x + (long long)seg) * p.group * 2;
    __nv_bfloat16* out = p.out + (long long)seg * p.group * D;
    for (int i = threadIdx.x; i < p.group * (D / 4); i += W * 32) {
      const int h = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][h][0]);
      const float base = top == -INFINITY ? 0.f : top;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = exp2f(s_ml[w][h][0] - base), zz = s_z[w][h][d >> 5];
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * STAGES * T::BYTES) + h * D + d);
        l = fmaf(s_ml[w][h][1], f, l);
        a.x = fmaf(v.x + zz, f, a.x), a.y = fmaf(v.y + zz, f, a.y), a.z = fmaf(v.z + zz, f, a.z), a.w = fmaf(v.w + zz, f, a.w);
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        __nv_bfloat162 r[2] = {__floats2bfloat162_rn(a.x * inv, a.y * inv), __floats2bfloat162_rn(a.z * inv, a.w * inv)};
        *reinterpret_cast<uint2*>(out + h * D + d) = *reinterpret_cast<const uint2*>(r);
      } else {
        *reinterpret_cast<float4*>(part + h * D + d) = a;
        if (d == 0) part_ml[2 * h] = top, part_ml[2 * h + 1] = l;
      }
    }
    if (!whole) {  // the CTA that finishes a shared segment last joins its parts
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int done = atomicAdd(&p.counters[seg], 1);
        s_last = done == (int)(cta1 - cta0);
        if (s_last) p.counters[seg] = 0;  // ready for the next launch
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        const int parts = (int)(cta1 - cta0) + 1;
        const float* from = p.o_part + (cta0 + seg) * p.group * D;
        const float* from_ml = p.ml_part + (cta0 + seg) * p.group * 2;
        for (int i = threadIdx.x; i < p.group * (D / 4); i += W * 32) {
          const int h = i / (D / 4), d = (i % (D / 4)) * 4;
          float top = -INFINITY, l = 0.f;
          for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(from_ml + ((long long)k * p.group + h) * 2));
          const float base = top == -INFINITY ? 0.f : top;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int k = 0; k < parts; ++k) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(from_ml + ((long long)k * p.group + h) * 2));
            const float4 v = __ldcg(reinterpret_cast<const float4*>(from + ((long long)k * p.group + h) * D + d));
            const float f = exp2f(ml.x - base);
            l = fmaf(ml.y, f, l);
            a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
          }
          const float inv = l == 0.f ? 0.f : 1.f / l;
          __nv_bfloat162 r[2] = {__floats2bfloat162_rn(a.x * inv, a.y * inv), __floats2bfloat162_rn(a.z * inv, a.w * inv)};
          *reinterpret_cast<uint2*>(out + h * D + d) = *reinterpret_cast<const uint2*>(r);
        }
      }
    }
    __syncthreads();  // the rings and the sums are free again

    u = stop;
    seg_start = seg_end;
    if (++kvh == p.heads) kvh = 0, ++b;
  }
}

// Parts that the workspace holds for each (request, kv head) bound the CTAs: the part of CTA c of segment g is number
// c + g, which no other pair has.
template <int D, int W> static int kv4_attn_launch(const Kv4Attn& p, int parts, long long max_len, cudaStream_t st) {
  constexpr int bytes = W * Kv4Tile<D>::STAGES * Kv4Tile<D>::BYTES;
  static_assert(Kv4Tile<D>::STAGES * Kv4Tile<D>::BYTES >= 8 * D * 4, "a warp's ring holds its sums");
  if (cudaFuncSetAttribute(kv4_attn_kernel<D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -5;
  const long long segments = (long long)p.batch * p.heads, room = segments * (parts - 1) + 1;
  const long long most = segments * ((max_len + 32 * W - 1) / (32 * W));  // units, if no request is longer
  long long ctas = 148 * (D == 256 ? 2 : 3);
  if (ctas > room) ctas = room;
  if (ctas > most) ctas = most;
  kv4_attn_kernel<D, W><<<(unsigned)ctas, W * 32, bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

int kv4_decode(const void* q, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const int* req_to_token, const int* req_pool_indices,
               const long long* seq_lens, const void* k_new, const void* v_new, float* o_part, float* ml_part, int* counters, void* out,
               int batch, int n_q_heads, int n_kv_heads, int head_dim, int max_ctx, int table_rows, long long n_slots, float scale, int parts,
               long long max_len, cudaStream_t st) {
  if (batch == 0) return 0;
  if (n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 8) return -1;
  if (parts < 1) return -2;
  const Kv4Attn p{(const __nv_bfloat16*)q, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_meta, (uint32_t*)v_meta, req_to_token,
                  req_pool_indices, seq_lens, (const __nv_bfloat16*)k_new, (const __nv_bfloat16*)v_new, o_part, ml_part, counters,
                  (__nv_bfloat16*)out, batch, n_kv_heads, n_q_heads / n_kv_heads, max_ctx, table_rows, n_slots, scale * 1.4426950408889634f};
  const long long longest = max_len > 0 && max_len < max_ctx ? max_len : max_ctx;
  switch (head_dim) {
    case 32: return kv4_attn_launch<32, 4>(p, parts, longest, st);
    case 64: return kv4_attn_launch<64, 4>(p, parts, longest, st);
    case 128: return kv4_attn_launch<128, 4>(p, parts, longest, st);
    case 256: return kv4_attn_launch<256, 4>(p, parts, longest, st);
    default: return -3;
  }
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
