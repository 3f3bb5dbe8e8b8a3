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
// Work: a (request, kv head) is a segment of ceil(len / 32) tiles of 32 keys and one turn of set-up; the segments of the
// whole batch, laid end to end, are divided evenly over the warps of one wave, whatever the lengths.  A warp walks its
// range alone: tiles stream through a ring of its own in shared memory (cp.async, across the ends of segments, no
// barrier), and a segment that begins and ends in its range is written out from its registers.  Of the others a warp has
// one that ends in its range at most (its sums go to the workspace) and one that goes on behind it (its sums stay in the
// ring); when all warps of a CTA are done they are joined, and what several CTAs share is joined by the one that is last.
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
  const int n = live ? N : 0;  // 0: zeros are written and nothing is read
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d = a b + c; the upper 8 rows of A are a1 / a3
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(0u), "r"(a2), "r"(0u), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// two fp32 numbers at a time
struct Pair { float x, y; };
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("{ .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("{ .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ uint32_t bf162_bits(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
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
  int n_slots;
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

template <int D> struct Kv4Shape { static constexpr int W = D == 256 ? 8 : 12; };  // warps of a CTA, one CTA per SM

template <int D>
__global__ void __launch_bounds__(Kv4Shape<D>::W * 32, 1) kv4_attn_kernel(const Kv4Attn p) {
  using T = Kv4Tile<D>;
  constexpr int W = Kv4Shape<D>::W, NG = T::NG, NB = NG < 4 ? NG : 4, BATCHES = NG / NB, STAGES = T::STAGES;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t s_mask[W][STAGES];
  __shared__ float s_ml[W][8][2];
  __shared__ int s_scan[W], s_found[W][2], s_end[W][3], s_open[W][4], s_last[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = smem + warp * STAGES * T::BYTES;

  // a length beyond the table row is cut to the row, a row outside the table attends to nothing
  auto length = [&](int b) -> int {
    const int row = p.rows[b];
    const long long n = p.lens[b];
    return row < 0 || row >= p.table_rows || n < 0 ? 0 : n > p.max_ctx ? p.max_ctx : (int)n;
  };
  auto turns = [&](int len) -> int { return ((len + 31) >> 5) + 1; };

  // this warp's share [u, u_end) of all turns: the first `extra` warps of the grid take one more than `base`
  int u, u_end, base, extra, n_workers;
  {
    const int per = (p.batch + W * 32 - 1) / (W * 32);
    const int b0 = threadIdx.x * per;
    int mine = 0;
    for (int i = 0; i < per && b0 + i < p.batch; ++i) mine += turns(length(b0 + i));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    total *= p.heads;
    before *= p.heads;
    n_workers = min((int)gridDim.x * W, total);
    base = total / n_workers, extra = total % n_workers;
    if (blockIdx.x * W >= n_workers) return;
    // where each of this CTA's warps begins: the request, and the request's first turn
#pragma unroll 1
    for (int w = 0; w < W; ++w) {
      const int i = blockIdx.x * W + w, at_w = i * base + min(i, extra);
      if (i < n_workers && at_w >= before && at_w < before + mine * p.heads) {
        int at = before, k = b0;
        for (;; ++k) {
          const int here = turns(length(k)) * p.heads;
          if (at_w < at + here) break;
          at += here;
        }
        s_found[w][0] = k, s_found[w][1] = at;
      }
    }
    const int i = blockIdx.x * W + warp;
    u = i < n_workers ? i * base + min(i, extra) : 0;
    u_end = i < n_workers ? u + base + (i < extra) : 0;
    if (lane == 0) s_end[warp][0] = s_open[warp][0] = -1;
    __syncthreads();
  }
  auto cta_of = [&](int x) -> int {
    return (x < extra * (base + 1) ? x / (base + 1) : extra + (x - extra * (base + 1)) / base) / W;
  };
  const int n_ctas = (n_workers + W - 1) / W;
  const float* const o_part = p.o_part;
  // parts: number CTA + segment for a CTA's share of a segment (no other pair has that number); behind them one for each
  // segment's end
  const int ends = n_ctas + p.batch * p.heads - 1;

  // A walk over the segments of [u, u_end): the tiles [tile, tile_end) of (b, kvh), whose first turn is `start`.
  struct Walk { int b, kvh, start, row, len, tile, tile_end; };
  auto enter = [&](Walk& w) {
    w.tile = max(u - w.start - 1, 0);
    w.tile_end = min(u_end - w.start - 1, (w.len + 31) >> 5);
  };
  auto next_segment = [&](Walk& w) {
    w.start += turns(w.len);
    if (++w.kvh == p.heads) {
      w.kvh = 0, ++w.b;
      if (w.start < u_end) w.row = p.rows[w.b], w.len = length(w.b);
    }
    enter(w);
  };
  Walk get{}, put{};  // the tiles that are computed, and those that are copied ahead of them
  if (u < u_end) {
    get.b = s_found[warp][0];
    get.row = p.rows[get.b], get.len = length(get.b);
    const int nt = turns(get.len);
    get.kvh = (u - s_found[warp][1]) / nt;
    get.start = s_found[warp][1] + get.kvh * nt;
    enter(get);
    put = get;
  }

  // ---- copies: a tile's slots, then its rows.  A slot outside the pool counts as none: its row is filled with zeros.
  auto settle = [&]() {  // put: on to a segment that has tiles left, if there is one
    while (put.tile >= put.tile_end && put.start + turns(put.len) < u_end) next_segment(put);
    return put.tile < put.tile_end;
  };
  auto slot_of = [&]() -> int {
    const int key = put.tile * 32 + lane;
    if (key >= put.len) return -1;
    const int s = p.table[(long long)put.row * p.max_ctx + key];
    return s < p.n_slots ? s : -1;
  };
  auto issue = [&](int slot, int stage) {
    if (p.k_new != nullptr && put.tile == (put.len - 1) >> 5) {  // the step's own rows: stored before they are read
      const int dst = __shfl_sync(0xffffffffu, slot, (put.len - 1) & 31);
      constexpr int LPR = D / 8;
      const long long to = (long long)max(dst, 0) * p.heads + put.kvh, from = ((long long)put.b * p.heads + put.kvh) * D;
#pragma unroll
      for (int pass = 0; pass < (D == 256 ? 2 : 1); ++pass) {
        const int which = D == 256 ? pass : lane / LPR;
        kv4_store_row<D>(dst >= 0 && which < 2, which == 0, lane % LPR, (which == 0 ? p.k_new : p.v_new) + from,
                         (which == 0 ? p.k_codes : p.v_codes) + to * (D / 2), (which == 0 ? p.k_meta : p.v_meta) + to * NG);
      }
      __threadfence();
      __syncwarp();
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, slot >= 0);
    if (lane == 0) s_mask[warp][stage] = mask;
    // a row's codes are NG pieces of 16 bytes, its middles and steps NG words: one number counts both
    const uint32_t row = slot >= 0 ? ((uint32_t)slot * (uint32_t)p.heads + (uint32_t)put.kvh) * NG : 0u;
    const uint32_t at = smem_addr(ring + stage * T::BYTES);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int r = i * (32 / NG) + lane / NG;
      const uint32_t from = __shfl_sync(0xffffffffu, row, r) + lane % NG;
      const uint32_t to = at + r * (D / 2) + (((lane % NG) ^ T::swap(r)) * 16);
      const bool live = (mask >> r) & 1;
      cp_async<16>(to + T::K, p.k_codes + (uint64_t)from * 16, live);
      cp_async<16>(to + T::V, p.v_codes + (uint64_t)from * 16, live);
    }
    constexpr int PIECE = NG < 4 ? NG * 4 : 16;  // bytes of the middles and steps that one copy takes
#pragma unroll
    for (int i = 0; i < NG * 4 / PIECE; ++i) {
      const uint32_t to = at + lane * NG * 4 + i * PIECE;
      cp_async<PIECE>(to + T::KM, p.k_meta + (uint64_t)row + i * (PIECE / 4), slot >= 0);
      cp_async<PIECE>(to + T::VM, p.v_meta + (uint64_t)row + i * (PIECE / 4), slot >= 0);
    }
  };
  bool more = settle();
  int slot = more ? slot_of() : -1;
  auto copy_next = [&](int stage) {  // issues the tile at `put`, whose slots are at hand, and fetches the slots of the next
    if (more) {
      issue(slot, stage);
      ++put.tile;
      more = settle();
      slot = more ? slot_of() : -1;
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) copy_next(s);

  for (int stage = 0; u < u_end; u = get.start) {
    const int b = get.b, kvh = get.kvh, seg = b * p.heads + kvh;
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

    // out: numbers 32 g + 4 gid + 2 i (+ 1: elements 2 and 3) of heads 2 tig and 2 tig + 1; z: sum p m of group gid, the same heads
    float o[NG][2][4], mx = -INFINITY, sum = 0.f;
    Pair z = {0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i >> 2][i & 3] = 0.f;
    const int key_row = (gid & 1) ? ((gid >> 1) ^ 1) + 4 : gid >> 1;  // row of a block of 8 keys that column gid stands for
    const int row_e[2] = {tig, (tig ^ 1) + 4};                        // rows of columns 2 tig and 2 tig + 1

    for (; get.tile < get.tile_end; ++get.tile) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      const uint8_t* tile = ring + stage * T::BYTES;
      const uint32_t mask = s_mask[warp][stage];
      copy_next(stage == 0 ? STAGES - 1 : stage - 1);  // into the stage that the previous turn has read
      // ---- logits of 4 blocks of 8 keys: this lane's head is gid, its keys row_e[0] and row_e[1] of each block
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      Pair s[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = 8 * n + key_row;
        float term[4] = {0.f, 0.f, 0.f, 0.f};
        Pair acc = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < BATCHES; ++h) {
          const uint32_t word = tig < NB ? *reinterpret_cast<const uint32_t*>(tile + T::KM + (r * NG + h * NB + (tig < NB ? tig : 0)) * 4) : 0u;
          mma_bf16(term, qs[h][0], qs[h][1], word, word, term);
          mma_bf16(term, qs[h][2], 0u, word, 0u, term);
          Words<NB> ms[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) ms[e] = lds_words<NB>(tile + T::KM + ((8 * n + row_e[e]) * NG + h * NB) * 4);
          Words<NB> codes;
          if constexpr (NG >= 4) codes = lds_words<NB>(tile + T::K + r * (D / 2) + (((4 * h + tig) ^ T::swap(r)) * 16));
          else codes = lds_words<NB>(tile + T::K + r * (D / 2) + tig * NB * 4);
#pragma unroll
          for (int w = 0; w < NB; ++w) {
            const uint32_t x = codes.w[w], y = x >> 8;
            float part[4];
            mma_f16(part, qa[h * NB + w][0], 0u, qa[h * NB + w][1], 0u, x & 0x000f000fu, x & 0x00f000f0u, none);
            mma_f16(part, qa[h * NB + w][2], 0u, qa[h * NB + w][3], 0u, y & 0x000f000fu, y & 0x00f000f0u, part);
            acc = fma2({part[0], part[1]}, {high_bf16(ms[0].w[w]), high_bf16(ms[1].w[w])}, acc);
          }
        }
        s[n] = fma2(mul2(acc, {back, back}), {p.scale_log2 * 0x1p24f, p.scale_log2 * 0x1p24f}, {term[0], term[1]});
      }
      if (mask != 0xffffffffu) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (!((mask >> (8 * n + row_e[0])) & 1)) s[n].x = -INFINITY;
          if (!((mask >> (8 * n + row_e[1])) & 1)) s[n].y = -INFINITY;
        }
      }
      // ---- softmax of the tile
      float top = mx;
#pragma unroll
      for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(s[n].x, s[n].y));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float zero = top == -INFINITY ? 0.f : top;
      if (__any_sync(0xffffffffu, top != mx)) {
        const float alpha = exp2f(mx - zero);
        const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * tig), a1 = __shfl_sync(0xffffffffu, alpha, 8 * tig + 4);
        sum *= alpha;
        z.x *= a0, z.y *= a1;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int t = 0; t < 2; ++t) o[g][t][0] *= a0, o[g][t][1] *= a1, o[g][t][2] *= a0, o[g][t][3] *= a1;
        mx = top;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        s[n].x = exp2f(s[n].x - zero), s[n].y = exp2f(s[n].y - zero);
        sum += s[n].x + s[n].y;
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
      // ---- sum p m: rows of A are the groups (bf16 words of the cache as they are), p in two bf16 parts (16 bits)
      float zt[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t a[2], hi[2], lo[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            w[e] = gid < NG ? *reinterpret_cast<const uint32_t*>(tile + T::VM + ((16 * j + 8 * n + row_e[e]) * NG + (gid < NG ? gid : 0)) * 4) : 0u;
          a[n] = __byte_perm(w[0], w[1], 0x5410);
          const Pair q = s[2 * j + n];
          hi[n] = bf162_bits(q.x, q.y);
          lo[n] = bf162_bits(q.x - low_bf16(hi[n]), q.y - high_bf16(hi[n]));
        }
        mma_bf16(zt, a[0], a[1], hi[0], hi[1], zt);
        mma_bf16(zt, a[0], a[1], lo[0], lo[1], zt);
      }
      z.x += zt[0], z.y += zt[1];
#pragma unroll
      for (int n = 0; n < 4; ++n) s[n] = mul2(s[n], {up, up});
      // ---- sum (p s) (c - 8), PB groups at a time; -8 enters as a product with a constant operand
      constexpr int PB = NG < 2 ? 1 : 2;
#pragma unroll
      for (int h = 0; h < NG / PB; ++h) {
        Words<PB> ms[4][2];
        uint32_t codes[4][2];  // a lane's numbers of two groups (D = 32: of one, a half word)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + row_e[e];
            ms[n][e] = lds_words<PB>(tile + T::VM + (r * NG + h * PB) * 4);
            const uint8_t* row = tile + T::V + r * (D / 2);
            if constexpr (D == 256) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + ((gid ^ T::swap(r)) * 16) + h * 4);
            else if constexpr (D == 128) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + (((gid >> 1) ^ T::swap(r)) * 16) + (gid & 1) * 8 + h * 4);
            else if constexpr (D == 64) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + gid * 4);
            else codes[n][e] = *reinterpret_cast<const uint16_t*>(row + gid * 2);
          }
#pragma unroll
        for (int g = 0; g < PB; ++g) {
          uint32_t pb[4], pair[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const Pair ps = mul2(s[n], {high_bf16(ms[n][0].w[g]), high_bf16(ms[n][1].w[g])});
            pb[n] = half2_bits(ps.x, ps.y);
            pair[n] = __byte_perm(codes[n][0], codes[n][1], g ? 0x7632 : 0x5410);
          }
          float eight[4], t[4];  // -8 sum p s: 0x80088008 is -8 2^-24 twice, 0x80808080 -8 2^-20
          mma_f16(eight, 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pb[0], pb[1], none);
          mma_f16(eight, 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, pb[2], pb[3], eight);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t x = i ? pair[2 * j] >> 8 : pair[2 * j], y = i ? pair[2 * j + 1] >> 8 : pair[2 * j + 1];
              if (j == 0) mma_f16(t, x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[0], pb[1], eight);
              else mma_f16(t, x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pb[2], pb[3], t);
            }
            float(&to)[4] = o[h * PB + g][i];
            const Pair lo = fma2({t[0], t[1]}, {down, down}, {to[0], to[1]});
            const Pair hi = fma2({t[2], t[3]}, {down * 0.0625f, down * 0.0625f}, {to[2], to[3]});
            to[0] = lo.x, to[1] = lo.y, to[2] = hi.x, to[3] = hi.y;
          }
        }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    // ---- the end of the segment, or of what this warp has of it
    const int first = get.start, behind = first + turns(get.len);
    const bool began = u <= first, ended = behind <= u_end;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float zx = __shfl_sync(0xffffffffu, z.x, 4 * g + tig), zy = __shfl_sync(0xffffffffu, z.y, 4 * g + tig);
#pragma unroll
      for (int i = 0; i < 2; ++i) o[g][i][0] += zx, o[g][i][1] += zy, o[g][i][2] += zx, o[g][i][3] += zy;
    }
    if (began && ended) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float l = __shfl_sync(0xffffffffu, sum, 8 * tig + 4 * h), inv = l == 0.f ? 0.f : 1.f / l;
        if (2 * tig + h < p.group) {
          __nv_bfloat16* out = p.out + ((long long)seg * p.group + 2 * tig + h) * D + 4 * gid;
#pragma unroll
          for (int g = 0; g < NG; ++g)
            *reinterpret_cast<uint2*>(out + 32 * g) = make_uint2(bf162_bits(o[g][0][h] * inv, o[g][0][2 + h] * inv), bf162_bits(o[g][1][h] * inv, o[g][1][2 + h] * inv));
        }
      }
    } else {
      float *to, *ml;
      if (ended) {
        to = p.o_part + (long long)(ends + seg) * p.group * D, ml = p.ml_part + (long long)(ends + seg) * p.group * 2;
        if (lane == 0) s_end[warp][0] = seg, s_end[warp][1] = first, s_end[warp][2] = behind;
      } else {  // the last of the range: nothing is on its way into the ring any more
        cp_wait<0>();
        __syncwarp();
        to = reinterpret_cast<float*>(ring), ml = &s_ml[warp][0][0];
        if (lane == 0) s_open[warp][0] = seg, s_open[warp][1] = first, s_open[warp][2] = behind, s_open[warp][3] = began;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * tig + h < p.group) {
#pragma unroll
          for (int g = 0; g < NG; ++g)
            *reinterpret_cast<float4*>(to + (2 * tig + h) * D + 32 * g + 4 * gid) = make_float4(o[g][0][h], o[g][0][2 + h], o[g][1][h], o[g][1][2 + h]);
        }
      }
      if (tig == 0 && gid < p.group) ml[2 * gid] = mx, ml[2 * gid + 1] = sum;
    }
    next_segment(get);
  }
  __syncthreads();

  // ---- join the parts of this CTA's warps, a warp for each segment: those that end in warp w's range, and (w = W) the one
  // that goes on behind the CTA
  const int last_warp = min(W, n_workers - (int)blockIdx.x * W) - 1;
  auto joined_here = [&](int w, int& seg, int& first, int& behind) -> bool {  // false: none, or not all of it is here
    const int* from = w < W ? s_end[w] : s_open[last_warp];
    seg = from[0], first = from[1], behind = from[2];
    return seg >= 0 && cta_of(first) == (int)blockIdx.x && cta_of(behind - 1) == (int)blockIdx.x;
  };
  auto weigh = [&](float m, float l, float4 v, float zero, float& sum_l, float4& a) {
    const float f = exp2f(m - zero);
    sum_l = fmaf(l, f, sum_l);
    a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
  };
  auto write_out = [&](int seg, int h, int d, float l, float4 a) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + ((long long)seg * p.group + h) * D + d) = make_uint2(bf162_bits(a.x * inv, a.y * inv), bf162_bits(a.z * inv, a.w * inv));
  };
  for (int w = warp; w <= W; w += W) {
    int seg, first, behind;
    const bool whole = joined_here(w, seg, first, behind);
    if (seg < 0 || (w < W && w > last_warp)) continue;
    const float* end_o = o_part + (long long)(ends + seg) * p.group * D;
    const float* end_ml = p.ml_part + (long long)(ends + seg) * p.group * 2;
    for (int i = lane; i < p.group * (D / 4); i += 32) {
      const int h = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = w < W ? __ldcg(end_ml + 2 * h) : -INFINITY, l = 0.f;
      for (int k = 0; k <= last_warp; ++k)
        if (s_open[k][0] == seg) top = fmaxf(top, s_ml[k][h][0]);
      const float zero = top == -INFINITY ? 0.f : top;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k <= last_warp; ++k)
        if (s_open[k][0] == seg)
          weigh(s_ml[k][h][0], s_ml[k][h][1], *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + k * STAGES * T::BYTES) + h * D + d), zero, l, a);
      if (w < W) weigh(__ldcg(end_ml + 2 * h), __ldcg(end_ml + 2 * h + 1), __ldcg(reinterpret_cast<const float4*>(end_o + h * D + d)), zero, l, a);
      if (whole) {
        write_out(seg, h, d, l, a);
      } else {
        const long long part = ((long long)blockIdx.x + seg) * p.group + h;
        *reinterpret_cast<float4*>(p.o_part + part * D + d) = a;
        if (d == 0) p.ml_part[2 * part] = top, p.ml_part[2 * part + 1] = l;
      }
    }
  }
  // ---- segments that other CTAs have a part of: one that came from the CTA before, one that goes on behind this one
  __threadfence();
  __syncthreads();
  int shared_seg[2], shared_cta[2], shared_n[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    shared_seg[k] = -1;
    int seg, first, behind;
    if (k == 0) {  // the only one that can have come from before is the first that ends here
      int w = 0;
      while (w < last_warp && s_end[w][0] < 0) ++w;
      if (joined_here(w, seg, first, behind) || seg < 0) continue;
    } else {
      if (joined_here(W, seg, first, behind) || seg < 0) continue;
    }
    shared_seg[k] = seg, shared_cta[k] = cta_of(first), shared_n[k] = cta_of(behind - 1) - cta_of(first) + 1;
  }
  if (threadIdx.x < 2) {
    const int k = threadIdx.x, seg = k ? shared_seg[1] : shared_seg[0], n = k ? shared_n[1] : shared_n[0];
    bool mine = false;
    if (seg >= 0) {
      mine = atomicAdd(&p.counters[seg], 1) == n - 1;
      if (mine) p.counters[seg] = 0;  // ready for the next launch
    }
    s_last[k] = mine;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!s_last[k]) continue;
    __threadfence();
    const long long from = (long long)shared_cta[k] + shared_seg[k];
    for (int i = threadIdx.x; i < p.group * (D / 4); i += W * 32) {
      const int h = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = -INFINITY, l = 0.f;
#pragma unroll 8
      for (int c = 0; c < shared_n[k]; ++c) top = fmaxf(top, __ldcg(p.ml_part + ((from + c) * p.group + h) * 2));
      const float zero = top == -INFINITY ? 0.f : top;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int c = 0; c < shared_n[k]; ++c) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.ml_part + ((from + c) * p.group + h) * 2));
        weigh(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(o_part + ((from + c) * p.group + h) * D + d)), zero, l, a);
      }
      write_out(shared_seg[k], h, d, l, a);
    }
  }
}

template <int D> static int kv4_attn_launch(const Kv4Attn& p, int parts, long long max_len, cudaStream_t st) {
  constexpr int W = Kv4Shape<D>::W, bytes = W * Kv4Tile<D>::STAGES * Kv4Tile<D>::BYTES;
  static_assert(Kv4Tile<D>::STAGES * Kv4Tile<D>::BYTES >= 8 * D * 4, "a warp's ring holds its sums");
  if (cudaFuncSetAttribute(kv4_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -5;
  const long long segments = (long long)p.batch * p.heads;
  if (p.max_ctx > 0x7fffff00 || segments * (p.max_ctx / 32 + 2) > 0x3fffffffLL) return -4;
  // the workspace holds a part for each segment's end and one for each (CTA, segment) that meet
  const long long room = segments * (parts - 2) + 1, turns = segments * ((max_len + 31) / 32 + 1);
  long long ctas = (turns + W - 1) / W;
  if (ctas > 148) ctas = 148;
  if (ctas > room) ctas = room;
  kv4_attn_kernel<D><<<(unsigned)ctas, W * 32, bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

int kv4_decode(const void* q, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const int* req_to_token, const int* req_pool_indices,
               const long long* seq_lens, const void* k_new, const void* v_new, float* o_part, float* ml_part, int* counters, void* out,
               int batch, int n_q_heads, int n_kv_heads, int head_dim, int max_ctx, int table_rows, long long n_slots, float scale, int parts,
               long long max_len, cudaStream_t st) {
  if (batch == 0) return 0;
  if (n_q_heads % n_kv_heads || n_q_heads / n_kv_heads > 8) return -1;
  if (parts < 2) return -2;
  if (n_slots * n_kv_heads * (head_dim / 32) > 0xffffffffLL) return -4;
  const Kv4Attn p{(const __nv_bfloat16*)q, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_meta, (uint32_t*)v_meta, req_to_token,
                  req_pool_indices, seq_lens, (const __nv_bfloat16*)k_new, (const __nv_bfloat16*)v_new, o_part, ml_part, counters,
                  (__nv_bfloat16*)out, batch, n_kv_heads, n_q_heads / n_kv_heads, max_ctx, table_rows, (int)(n_slots < 0x7fffffffLL ? n_slots : 0x7fffffffLL), scale * 1.4426950408889634f};
  const long long longest = max_len > 0 && max_len < max_ctx ? max_len : max_ctx;
  switch (head_dim) {
    case 32: return kv4_attn_launch<32>(p, parts, longest, st);
    case 64: return kv4_attn_launch<64>(p, parts, longest, st);
    case 128: return kv4_attn_launch<128>(p, parts, longest, st);
    case 256: return kv4_attn_launch<256>(p, parts, longest, st);
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
