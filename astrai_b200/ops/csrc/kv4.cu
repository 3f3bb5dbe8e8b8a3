// The 4-bit KV cache (format: kv4.cuh): storing rows, reading rows back, decode attention on the codes, copying pages.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "kv4.cuh"
#include "launchers.h"

namespace ab {

// ------------------------------------------------------------------------------------------------------- store rows
// D / 8 lanes a row, a key row and a value row each, both on their way before the first is worked on.  A slot outside the
// pool is skipped.  Bound by its instructions, 420 a warp for 2 x 256 numbers: 8192 tokens of 8 heads of 128 numbers take
// 16.6 us, of which 12 are issue slots, 6.7 the 44 MB that move; 16 tokens take 2 us (a launch).
template <int D, typename Loc>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v,
                                                         uint8_t* __restrict__ k_codes, uint32_t* __restrict__ k_meta,
                                                         uint8_t* __restrict__ v_codes, uint32_t* __restrict__ v_meta,
                                                         const Loc* __restrict__ loc, int rows, int heads, long long n_slots,
                                                         long long k_tok, long long k_head, long long v_tok, long long v_head) {
  constexpr int LPR = D / 8;
  const int l = threadIdx.x % LPR;
  const int r = (blockIdx.x * 256 + threadIdx.x) / LPR, t = r / heads, h = r - t * heads;
  const long long slot = r < rows ? (long long)loc[t] : -1;
  const bool live = slot >= 0 && slot < n_slots;
  const long long at = live ? slot * heads + h : 0;
  const Vec8<__nv_bfloat16> kv = kv4_load_numbers(live, l, k + t * k_tok + h * k_head), vv = kv4_load_numbers(live, l, v + t * v_tok + h * v_head);
  kv4_store_numbers<D>(live, true, l, kv, k_codes + at * (D / 2), k_meta + at * (D / 32));
  kv4_store_numbers<D>(live, false, l, vv, v_codes + at * (D / 2), v_meta + at * (D / 32));
}

// -------------------------------------------------------------------------------------------------------- read rows
// The reverse, as bf16 rows [tokens, heads, D].  A slot outside the pool reads as zeros.  Bound by memory: 131072 tokens of
// 8 heads of 128 numbers (705 MB) take 122 us, 5.8 TB/s (88% of a copy's rate).  The rows are written past the caches: they
// would push out the codes of the next call.
__device__ __forceinline__ uint4 kv4_numbers(uint32_t word, uint32_t ms) {
  const float m = __uint_as_float(ms << 16), s = __uint_as_float(ms & 0xffff0000u);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)  // c in the low bits of 2^23 makes the number 2^23 + c
    x[j] = fma_ieee(s, __uint_as_float(0x4b000000u | ((word >> (4 * j)) & 15u)) - 8388616.f, m);
  Vec8<__nv_bfloat16> out;
  out.pack(x);
  return out.raw;
}

template <int D, typename Loc>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const uint8_t* __restrict__ k_codes, const uint32_t* __restrict__ k_meta,
                                                         const uint8_t* __restrict__ v_codes, const uint32_t* __restrict__ v_meta,
                                                         const Loc* __restrict__ loc, __nv_bfloat16* __restrict__ k,
                                                         __nv_bfloat16* __restrict__ v, int rows, int heads, long long n_slots) {
  constexpr int LPR = D / 8, NG = D / 32, DEEP = 2;  // DEEP: rows of a lane that are on their way at a time
  const int l = threadIdx.x % LPR, g = l >> 2;
  const int r0 = blockIdx.x * (256 / LPR * DEEP) + threadIdx.x / LPR;
  uint32_t kw[DEEP], vw[DEEP], kms[DEEP], vms[DEEP];
#pragma unroll
  for (int i = 0; i < DEEP; ++i) {
    const int r = r0 + i * (256 / LPR), t = r / heads, h = r - t * heads;
    const long long slot = r < rows ? (long long)loc[t] : -1;
    kw[i] = vw[i] = 0x88888888u, kms[i] = vms[i] = 0;
    if (slot >= 0 && slot < n_slots) {
      const long long at = slot * heads + h;
      kw[i] = reinterpret_cast<const uint32_t*>(k_codes + at * (D / 2))[kv4_key_word<D>(g, l & 3)];
      vw[i] = reinterpret_cast<const uint32_t*>(v_codes + at * (D / 2))[l];
      kms[i] = k_meta[at * NG + g], vms[i] = v_meta[at * NG + g];
    }
  }
  // numbers 8 l .. of a value row are the half words of group g, eighths 2 (l & 3) and the next: with two lanes
  const int base = (threadIdx.x & 31) - l, h0 = kv4_value_half<D>(g, 2 * (l & 3)), h1 = kv4_value_half<D>(g, 2 * (l & 3) + 1);
#pragma unroll
  for (int i = 0; i < DEEP; ++i) {
    const int r = r0 + i * (256 / LPR);
    const uint32_t w0 = __shfl_sync(0xffffffffu, vw[i], base + (h0 >> 1)), w1 = __shfl_sync(0xffffffffu, vw[i], base + (h1 >> 1));
    const uint32_t word = __byte_perm(w0, w1, (h0 & 1 ? 0x0032 : 0x0010) | (h1 & 1 ? 0x7600 : 0x5400));
    if (r < rows) {
      const long long to = (long long)r * D + 8 * l;
      __stcs(reinterpret_cast<uint4*>(k + to), kv4_numbers(kw[i], kms[i]));
      __stcs(reinterpret_cast<uint4*>(v + to), kv4_numbers(word, vms[i]));
    }
  }
}

// Rows of one launch: their lanes are counted in 32 bits.
constexpr long long kKv4Rows = 1 << 25;

int kv4_append(const void* k, const void* v, void* k_codes, void* k_meta, void* v_codes, void* v_meta, const void* loc, bool loc64,
               long long tokens, int heads, int head_dim, long long n_slots, long long k_tok, long long k_head, long long v_tok,
               long long v_head, cudaStream_t st) {
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return -3;
  if (tokens == 0 || heads == 0) return 0;
  if (heads > kKv4Rows) return -4;
  const long long step = kKv4Rows / heads;
  for (long long t = 0; t < tokens; t += step) {
    const int rows = (int)((tokens - t < step ? tokens - t : step) * heads);
    const int grid = ceil_div((long long)rows * (head_dim / 8), 256);
#define AB_APPEND(DD, LL)                                                                                                       \
  kv4_append_kernel<DD, LL><<<grid, 256, 0, st>>>((const __nv_bfloat16*)k + t * k_tok, (const __nv_bfloat16*)v + t * v_tok,      \
                                                  (uint8_t*)k_codes, (uint32_t*)k_meta, (uint8_t*)v_codes, (uint32_t*)v_meta,    \
                                                  (const LL*)loc + t, rows, heads, n_slots, k_tok, k_head, v_tok, v_head)
#define AB_APPEND_D(DD) \
  if (loc64) AB_APPEND(DD, long long); else AB_APPEND(DD, int)
    switch (head_dim) {
      case 32: AB_APPEND_D(32); break;
      case 64: AB_APPEND_D(64); break;
      case 128: AB_APPEND_D(128); break;
      default: AB_APPEND_D(256); break;
    }
#undef AB_APPEND_D
#undef AB_APPEND
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

int kv4_gather(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, const void* loc, bool loc64, void* k,
               void* v, long long tokens, int heads, int head_dim, long long n_slots, cudaStream_t st) {
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return -3;
  if (tokens == 0 || heads == 0) return 0;
  if (heads > kKv4Rows) return -4;
  const long long step = kKv4Rows / heads;
  for (long long t = 0; t < tokens; t += step) {
    const int rows = (int)((tokens - t < step ? tokens - t : step) * heads);
    const int grid = ceil_div((long long)rows * (head_dim / 8), 512);
    const long long to = t * heads * head_dim;
#define AB_GATHER(DD, LL)                                                                                                          \
  kv4_gather_kernel<DD, LL><<<grid, 256, 0, st>>>((const uint8_t*)k_codes, (const uint32_t*)k_meta, (const uint8_t*)v_codes,        \
                                                  (const uint32_t*)v_meta, (const LL*)loc + t, (__nv_bfloat16*)k + to,              \
                                                  (__nv_bfloat16*)v + to, rows, heads, n_slots)
#define AB_GATHER_D(DD) \
  if (loc64) AB_GATHER(DD, long long); else AB_GATHER(DD, int)
    switch (head_dim) {
      case 32: AB_GATHER_D(32); break;
      case 64: AB_GATHER_D(64); break;
      case 128: AB_GATHER_D(128); break;
      default: AB_GATHER_D(256); break;
    }
#undef AB_GATHER_D
#undef AB_GATHER
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// -------------------------------------------------------------------------------------------------- decode attention
// Attention of one query per request on the codes themselves.  With c the codes (0..15), s / m the steps and middles and
// lo = m - 8 s, for key k, group g and head h:
//   logit = sum_g s_kg (q_hg . c_kg) + lo_kg sum(q_hg)       out_d = sum_k (p_k s_kg) c_kd + sum_k p_k lo_kg   (d in g)
// so the big products take the codes as they are: a code in the low bits of an fp16 IS the number c 2^-24 (a subnormal),
// and one shifted left by four is c 2^-20, so a pair of numbers costs one AND (and every second pair a shift).  The
// other operand is the query times a power of two that puts its largest number into [2^13, 2^14), or p s times a power of two
// that puts the largest step of the tile's 32 rows into [2^14, 2^15), rounded to fp16.  What that costs (p: the weight
// relative to the largest so far, 1):
//   p s      2^-11 of it, and 2^-39 of the tile's largest step where it is below 2^-28 of that step
//   query    nothing down to 2^-26 of the head's largest number, 2^-34 of that number below
// so the sizes of queries, keys and values cost nothing by themselves, and ranges inside a head or a tile nothing that
// bf16 numbers of one model come near.  Products go to m16n8k16 tensor instructions with fp32 sums: a tile's share of `out` is
// summed from zero and added to the running sum in fp32 registers, so a long context loses nothing to the tensor
// accumulator's rounding.  lo_kg sum(q_hg) is a product of the (m, s) words as they lie in memory with (sum q, -8 sum q)
// split into three bf16 parts (24 bits).
//
// Work: a request is ceil(len / UNIT) turns of UNIT = 32 W keys and SETUP empty ones (what it costs to begin and end one);
// the requests of the batch, laid end to end, are divided evenly over groups of CTAs, whatever the lengths.  A group has a
// CTA for each kv head: the rows of a token's heads lie side by side in memory and are read at about the same time (with
// the heads' parts cut independently a batch of 16 x 65521 tokens took 211 us).  A CTA walks its range request by request:
// warp w takes every W-th tile of 32 keys, streams it through a ring of its own in shared memory (cp.async, no barrier
// between warps), and the warps' sums meet at the end of the request.  What several groups share of a request is joined by
// the one that finishes last.
//
// What it takes, and what bounds it.  16 requests of 65521 tokens, 16 query over 4 kv heads, D = 128 (671 MB of codes and
// steps): 157 us, 4.3 TB/s, 65% of a copy's rate.  The loop without its copies takes 137 us, the copies without the
// arithmetic 123 us.  The arithmetic waits more than it works: with three warps a scheduler (162 registers a thread) half
// of the issue slots are taken, 43% of the integer pipe's, 33% of the shared memory's, 19% of the tensor pipe's (a tile
// of 32 keys has a chain of products, a maximum over lanes, exponentials and products again).  Four warps a scheduler at
// 128 registers spilled and took 190 us.  A launch begins with some 5 us of lengths, table, slots and first tiles and ends
// with 3 to 4 us in which sums meet, and shorter work is bound by those: one request of 65521 tokens over 8 kv heads
// 34.7 us (floor 12.8), 128 requests of 16 to 4608 tokens over 4 28.8 us (floor 11.8), 32 of 2049 to 8191 over 4 of 64
// numbers 26.8 us (floor 7.0), 64 of 1000 over 4 of 256 numbers 34.5 us, one of 8192 over 4 12.4 us, 4 of 1 to 33 6.2 us.
//
// Keys are the rows of the logits' product and queries its columns: a lane then holds two keys' steps, and eight query heads
// fill the columns (with queries as rows, half of them empty, the 16 requests took 177 us).  The products of the weights
// take queries as columns too, so the weights are turned round in registers (movmatrix).
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d = a b + c; rows 0-7 of A are a.x / a.z, rows 8-15 a.y / a.w
__device__ __forceinline__ void mma_f16(float (&d)[4], uint4 a, uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint4 a, uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
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
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("{ .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
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
template <int N> struct Floats { float f[N]; };
template <int N> __device__ __forceinline__ Floats<N> lds_floats(const float* p) {
  const Words<N> w = lds_words<N>(reinterpret_cast<const uint8_t*>(p));
  Floats<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.f[i] = __uint_as_float(w.w[i]);
  return r;
}
template <int N> __device__ __forceinline__ void sts_floats(float* p, const Floats<N>& v) {
  if constexpr (N == 1) *p = v.f[0];
  else if constexpr (N == 2) *reinterpret_cast<float2*>(p) = make_float2(v.f[0], v.f[1]);
  else *reinterpret_cast<float4*>(p) = make_float4(v.f[0], v.f[1], v.f[2], v.f[3]);
}
// An 8 x 8 matrix of 16-bit numbers, row gid and columns 2 tig, 2 tig + 1 to a lane, turned round.
__device__ __forceinline__ uint32_t transpose(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// A tile of 32 keys in shared memory.  STAGES: tiles of a warp's ring; three, two where three do not fit (with two, D = 128,
// 16 requests of 65521 tokens: 161 us instead of 158).
template <int D> struct Kv4Tile {
  static constexpr int NG = D / 32, KEYS = 32, CODES = KEYS * D / 2, META = KEYS * NG * 4;
  static constexpr int K = 0, V = CODES, KM = 2 * CODES, VM = 2 * CODES + META, BYTES = 2 * (CODES + META);
  static constexpr int STAGES = D == 256 ? 2 : 3, RING = STAGES * BYTES, QUERY = 512 * (NG + (NG < 4 ? 1 : NG / 4)), STEPS = 2 * KEYS * NG * 4;
  // behind a warp's ring: a tile's steps, or four heads of its sums when they meet those of the other warps
  static constexpr int SPACE = STEPS > 16 * D ? (STEPS > 1024 ? STEPS : 1024) : (16 * D > 1024 ? 16 * D : 1024);
  static constexpr int WARP = RING + SPACE;  // bytes of a warp; the query's are the CTA's
  // 16-byte pieces of a row are swapped by the row's number so that neither the lanes' reads of keys (two rows at a time)
  // nor those of values (four rows, a quarter of each) meet in a bank
  static __device__ __forceinline__ int swap(int r) { return D == 128 ? (r & 2) : D == 256 ? (((r & 1) << 2) | (r & 2)) : 0; }
};

__device__ __forceinline__ void weigh(float m, float l, float4 v, float zero, float& sum_l, float4& a) {
  const float f = exp2f(m - zero);
  sum_l = fmaf(l, f, sum_l);
  a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
}
template <int D> __device__ __forceinline__ void write_out(const Kv4Attn& p, int seg, int h, int d, float l, float4 a) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + ((long long)seg * p.group + h) * D + d) = make_uint2(bf162_bits(a.x * inv, a.y * inv), bf162_bits(a.z * inv, a.w * inv));
}

// Joins `n` parts of a (request, kv head), `from` the first one's first head and `step` from one to the next: `copies` threads share a number's parts, eight of them on
// their way at a time, and meet in shared memory.
template <int D, int W> __device__ __forceinline__ void kv4_join(const Kv4Attn& p, int seg, long long from, long long step, int n, uint8_t* smem) {
  const int items = p.group * (D / 4), copies = max(1, W * 32 / items);
  auto meet = [&](int i) -> float* { return reinterpret_cast<float*>(smem + (i >> 5) * Kv4Tile<D>::WARP + Kv4Tile<D>::RING) + (i & 31) * 8; };
  for (int i = threadIdx.x; i < items * copies; i += W * 32) {
    const int item = i % items, h = item / (D / 4), d = (item % (D / 4)) * 4;
    float top = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int c = i / items; c < n; c += 8 * copies) {
      float2 ml[8];
      float4 v[8];
      float most = top;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool on = c + j * copies < n;
        const long long part = from + (on ? c + j * copies : c) * step + h;
        ml[j] = __ldcg(reinterpret_cast<const float2*>(p.ml_part + 2 * part)), v[j] = __ldcg(reinterpret_cast<const float4*>(p.o_part + part * D + d));
        if (!on) ml[j] = make_float2(-INFINITY, 0.f), v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, ml[j].x);
      const float zero = most == -INFINITY ? 0.f : most, f = exp2f(top - zero);
      l *= f, a.x *= f, a.y *= f, a.z *= f, a.w *= f;
      top = most;
#pragma unroll
      for (int j = 0; j < 8; ++j) weigh(ml[j].x, ml[j].y, v[j], zero, l, a);
    }
    if (copies == 1) {
      write_out<D>(p, seg, h, d, l, a);
    } else {
      *reinterpret_cast<float4*>(meet(i)) = a;
      meet(i)[4] = top, meet(i)[5] = l;
    }
  }
  if (copies == 1) return;
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += W * 32) {
    float top = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < copies; ++c) top = fmaxf(top, meet(c * items + i)[4]);
    const float zero = top == -INFINITY ? 0.f : top;
    for (int c = 0; c < copies; ++c) {
      const float* at = meet(c * items + i);
      weigh(at[4], at[5], *reinterpret_cast<const float4*>(at), zero, l, a);
    }
    write_out<D>(p, seg, i / (D / 4), (i % (D / 4)) * 4, l, a);
  }
}

// What beginning and ending a request costs, in turns, and how far a cut is moved to spare one (both: 128 mixed lengths of 16
// to 4608 took 28.8 us with 1 turn, 30.9 with 2, 34.5 with 3; 128 requests of 100 tokens 13.2, 11.5 and 13.0; cuts that are
// not moved: 30.8 and 13.0).
constexpr int KV4_SETUP = 1, KV4_TOL = 1;
// W warps a CTA; `per_sm` CTAs fit an SM: 128, 168 and 255 registers a thread for D up to 64, 128 and 256 (D = 64, 16
// requests of 65521 tokens: three CTAs 116 us, four 105; shared memory that does not begin on a 128-byte line: 137).
template <int D, int W> constexpr int kv4_per_sm() { return W == 12 ? 1 : D == 256 ? 2 : D == 128 ? 3 : 4; }

template <int D, int W>
__global__ void __launch_bounds__(W * 32, kv4_per_sm<D, W>()) kv4_attn_kernel(const Kv4Attn p) {
  using T = Kv4Tile<D>;
  constexpr int NG = T::NG, NB = NG < 4 ? NG : 4, BATCHES = NG / NB, STAGES = T::STAGES, UNIT = 32 * W;
  constexpr int SETUP = KV4_SETUP, TOL = KV4_TOL;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_mask[W][STAGES];
  __shared__ float s_ml[W][8][2];
  __shared__ int s_scan[W], s_found[2][2], s_last;
  // what is the same in all lanes is passed through a shuffle, so that the compiler can hold it in uniform registers
  auto same = [](int x) -> int { return __shfl_sync(0xffffffffu, x, 0); };
  const int warp = same(threadIdx.x >> 5), lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = smem + warp * T::WARP;
  // a tile's steps (times a power of two) and lows of the values in fp32, [key][group]
  float *v_step = reinterpret_cast<float*>(ring + T::RING), *v_low = v_step + 32 * NG;
  float* space = v_step;
  // the query as operand B, a lane's registers at a time: two steps of every group, then (sum q, -8 sum q) in three parts
  uint4* q_frag = reinterpret_cast<uint4*>(smem + W * T::WARP);

  // a length beyond the table row is cut to the row, a row outside the table attends to nothing
  auto length = [&](int b) -> int {
    const int row = p.rows[b];
    const long long n = p.lens[b];
    return row < 0 || row >= p.table_rows || n < 0 ? 0 : n > p.max_ctx ? p.max_ctx : (int)n;
  };
  auto turns = [&](int len) -> int { return (len + UNIT - 1) / UNIT + SETUP; };

  // Group i has the turns from cut i to cut i + 1, where cut i lies at turn i base + min(i, extra), moved to the end of its
  // request if that is `tol` turns away or less: a cut costs a join.
  const int group = blockIdx.x / p.heads, kvh = blockIdx.x - group * p.heads;
  int u, u_end, b, start, base, extra;  // start: first turn of the current request b
  auto tol_of = [&](int n) -> int { return min(min(TOL, base >> 1), (n - 1) >> 1); };  // n: turns of the request
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
    total = same(total);
    const int n_groups = min((int)gridDim.x / p.heads, (total + SETUP) / (SETUP + 1));
    if (group >= n_groups) return;
    base = total / n_groups, extra = total % n_groups;
    int cut[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = group + k;
      cut[k] = i * base + min(i, extra);
      const int x = min(cut[k], total - 1);
      if (x >= before && x < before + mine) {  // the request that the cut lies in, and the request's first turn
        int at = before, r = b0;
        if (per > 1) {
          for (;; ++r) {
            const int here = turns(length(r));
            if (x < at + here) break;
            at += here;
          }
        }
        s_found[k][0] = r, s_found[k][1] = at;
      }
    }
    __syncthreads();
    u = u_end = total;
#pragma unroll
    for (int k = 1; k >= 0; --k) {
      if (cut[k] == total) continue;
      b = same(s_found[k][0]), start = same(s_found[k][1]);
      const int n = turns(same(length(b))), tol = tol_of(n);
      (k ? u_end : u) = cut[k] <= start + tol ? start : cut[k] >= start + n - tol ? start + n : cut[k];
      if (k == 0 && u == start + n) start = u, ++b;  // moved to the start of the next request
    }
  }
  auto group_of = [&](int x) -> int { return x < extra * (base + 1) ? x / (base + 1) : extra + (x - extra * (base + 1)) / base; };

  // A request, and what this CTA has of it: the keys up to key_end; `key` is the first one of this warp's next tile.
  struct Part { int b, row, len, start, behind, key, key_end; };
  Part cur{}, next{};
  auto enter = [&](Part& r, int request, int first) {
    r.b = request, r.start = first;
    r.len = same(length(request)), r.row = same(p.rows[request]);
    r.behind = first + turns(r.len);
    r.key_end = u_end >= r.behind ? r.len : max(0, u_end - first - SETUP) * UNIT;
    r.key = max(0, u - first - SETUP) * UNIT + warp * 32;
  };

  // ---- copies: a tile's slots, then its rows.  A key whose slot is outside the pool takes the row of one that is not
  // (nothing, if there is none): its weight will be zero, but what it is multiplied with has to be a number.
  auto slot_of = [&](const Part& r, int k0) -> int {
    const int s = k0 + lane < r.key_end ? p.table[(long long)r.row * p.max_ctx + k0 + lane] : -1;
    return s < p.n_slots ? s : -1;
  };
  auto issue = [&](const Part& r, int k0, int slot, int stage) {
    if (p.k_new != nullptr && k0 + 32 >= r.len) {  // the step's own rows: stored before they are read
      const int dst = __shfl_sync(0xffffffffu, slot, (r.len - 1) & 31);
      constexpr int LPR = D / 8;
      const long long to = (long long)max(dst, 0) * p.heads + kvh, from = ((long long)r.b * p.heads + kvh) * D;
#pragma unroll 1
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
    if (mask == 0) return;
    if (mask != 0xffffffffu) {
      const int other = __shfl_sync(0xffffffffu, slot, __ffs(mask) - 1);
      if (slot < 0) slot = other;
    }
    // a row's codes are NG pieces of 16 bytes, its middles and steps NG words: one number counts both
    const uint32_t at_row = ((uint32_t)slot * (uint32_t)p.heads + (uint32_t)kvh) * NG;
    const uint32_t at = smem_addr(ring + stage * T::BYTES);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int row = i * (32 / NG) + lane / NG;
      const uint32_t from = __shfl_sync(0xffffffffu, at_row, row) + lane % NG;
      const uint32_t to = at + row * (D / 2) + (((lane % NG) ^ T::swap(row)) * 16);
      cp_async<16>(to + T::K, p.k_codes + (uint64_t)from * 16);
      cp_async<16>(to + T::V, p.v_codes + (uint64_t)from * 16);
    }
    constexpr int PIECE = NG < 4 ? NG * 4 : 16;  // bytes of the middles and steps that one copy takes
#pragma unroll
    for (int i = 0; i < NG * 4 / PIECE; ++i) {
      const uint32_t to = at + lane * NG * 4 + i * PIECE;
      cp_async<PIECE>(to + T::KM, p.k_meta + (uint64_t)at_row + i * (PIECE / 4));
      cp_async<PIECE>(to + T::VM, p.v_meta + (uint64_t)at_row + i * (PIECE / 4));
    }
  };
  int ahead = 0, slot = -1, slot_after = -1;  // the next tile to copy, its slots and those of the one behind it
  auto copy_next = [&](const Part& r, int stage) {
    if (ahead < r.key_end) {
      const int now = slot;
      slot = slot_after, slot_after = slot_of(r, ahead + 2 * UNIT);
      issue(r, ahead, now, stage);
      ahead += UNIT;
    }
    cp_commit();
  };

  // Of everything a lane has heads 2 tig and 2 tig + 1, as pairs.  back undoes the query's power of two; o: numbers 32 g +
  // 4 gid + 2 i (+ 1: elements 2 and 3); sum, z: sums of p and p lo over this lane's keys.
  float o[NG][2][4];
  Pair back{}, mx{}, z[NG], sum{};
  const int key_row = (gid & 1) ? ((gid >> 1) ^ 1) + 4 : gid >> 1;  // the key that row gid of a block of 8 stands for
  const int row_e[2] = {tig, (tig ^ 1) + 4};                        // those of rows 2 tig and 2 tig + 1
  bool began = false, going = false;  // going: a request (cur) is in hand, its tiles are done; began: it began in this CTA
  if (u < u_end) enter(next, b, start);
  for (;;) {
    // ---- the first tiles of the next request are on their way while the one in hand ends
    const bool more = going ? cur.behind < u_end : u < u_end;
    if (more) {
      if (going) u = cur.behind, enter(next, cur.b + 1, cur.behind);
      ahead = next.key, slot = slot_of(next, ahead), slot_after = slot_of(next, ahead + UNIT);
#pragma unroll 1
      for (int t = 0; t < STAGES - 1; ++t) copy_next(next, t);
    }
    if (going) {
      // ---- the warps' sums meet, four heads at a time
      const int seg = cur.b * p.heads + kvh;
      const bool whole = began && cur.behind <= u_end;
      auto over_keys = [](Pair v) -> Pair {
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) v.x += __shfl_xor_sync(0xffffffffu, v.x, i), v.y += __shfl_xor_sync(0xffffffffu, v.y, i);
        return v;
      };
      const Pair l = over_keys(sum);
      if (gid == 0) {
        s_ml[warp][2 * tig][0] = mx.x, s_ml[warp][2 * tig][1] = l.x;
        s_ml[warp][2 * tig + 1][0] = mx.y, s_ml[warp][2 * tig + 1][1] = l.y;
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const Pair zz = over_keys(z[g]);
#pragma unroll
        for (int i = 0; i < 2; ++i) o[g][i][0] += zz.x, o[g][i][1] += zz.y, o[g][i][2] += zz.x, o[g][i][3] += zz.y;
      }
#pragma unroll 1
      for (int h0 = 0; h0 < p.group; h0 += 4) {
        if ((tig & 2) * 2 == h0) {  // heads 2 tig and 2 tig + 1; numbers 32 g + 4 gid .. + 3
          float* to = space + (tig & 1) * 2 * D + 4 * gid;
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<float4*>(to + h * D + 32 * g) = make_float4(o[g][0][h], o[g][0][2 + h], o[g][1][h], o[g][1][2 + h]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < min(4, p.group - h0) * (D / 4); i += W * 32) {
          const int h = h0 + i / (D / 4), d = (i % (D / 4)) * 4;
          float top = -INFINITY, ls = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][h][0]);
          const float zero = top == -INFINITY ? 0.f : top;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w)
            weigh(s_ml[w][h][0], s_ml[w][h][1], *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * T::WARP + T::RING) + (h - h0) * D + d), zero, ls, a);
          if (whole) {
            write_out<D>(p, seg, h, d, ls, a);
          } else {  // part number group + request of the head: no other pair has it
            const long long part = (((long long)group + cur.b) * p.heads + kvh) * p.group + h;
            *reinterpret_cast<float4*>(p.o_part + part * D + d) = a;
            if (d == 0) p.ml_part[2 * part] = top, p.ml_part[2 * part + 1] = ls;
          }
        }
        __syncthreads();
      }
      if (!whole) {  // the CTA that finishes a shared request last joins its parts
        const int tol = tol_of(cur.behind - cur.start), group0 = group_of(cur.start + tol), parts = group_of(cur.behind - 1 - tol) - group0 + 1;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          s_last = atomicAdd(&p.counters[seg], 1) == parts - 1;
          if (s_last) p.counters[seg] = 0;  // ready for the next launch
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          kv4_join<D, W>(p, seg, (((long long)group0 + cur.b) * p.heads + kvh) * p.group, (long long)p.heads * p.group, parts, smem);
          __syncthreads();
        }
      }
    }
    if (!more) break;
    began = u <= next.start;
    cur = next;
    going = true;
    // ---- the query as operand B: column gid = head, numbers 32 w + 8 tig + (0 4 | 1 5 | 2 6 | 3 7) as pairs
    {
      float x[NG][8], big = 0.f;
      const bool on = gid < p.group;
      const __nv_bfloat16* src = p.q + (((long long)cur.b * p.heads + kvh) * p.group + (on ? gid : 0)) * D + 8 * tig;
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
      const float undo = __uint_as_float((uint32_t)(127 - e) << 23);
      back = {__shfl_sync(0xffffffffu, undo, 8 * tig), __shfl_sync(0xffffffffu, undo, 8 * tig + 4)};
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
        if (w % W != warp) continue;  // every warp has all of them, each brings its share
        q_frag[w * 32 + lane] = make_uint4(half2_bits(x[w][0] * up, x[w][4] * up), half2_bits(x[w][1] * odd, x[w][5] * odd),
                                           half2_bits(x[w][2] * up, x[w][6] * up), half2_bits(x[w][3] * odd, x[w][7] * odd));
      }
#pragma unroll
      for (int h = 0; h < BATCHES; ++h) {  // lane tig: (sum, -8 sum) of group 4 h + tig, in three parts
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NB; ++w) t = tig == w ? sums[h * NB + w] : t;
        uint32_t parts[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const float part = __bfloat162float(__float2bfloat16_rn(t));
          parts[i] = bf162_bits(part, -8.f * part);
          t -= part;
        }
        if (warp != W - 1) continue;
        q_frag[(NG + h) * 32 + lane] = make_uint4(parts[0], parts[1], parts[2], 0u);
      }
    }
    mx = {-INFINITY, -INFINITY}, sum = {0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      z[g] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) o[g][i >> 2][i & 3] = 0.f;
    }
    __syncthreads();
    for (int t = 0; cur.key < cur.key_end; t = t + 1 == STAGES ? 0 : t + 1, cur.key += UNIT) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      copy_next(cur, t == 0 ? STAGES - 1 : t - 1);  // into the stage that the previous turn has read
      const uint8_t* tile = ring + t * T::BYTES;
      const uint32_t mask = same(s_mask[warp][t]);
      if (mask == 0) continue;
      // ---- steps of the values: lane = key
      float down;
      {
        uint32_t largest = 0;
        Words<NB> v[BATCHES];
#pragma unroll
        for (int h = 0; h < BATCHES; ++h) {
          v[h] = lds_words<NB>(tile + T::VM + (lane * NG + h * NB) * 4);
#pragma unroll
          for (int w = 0; w < NB; ++w) largest = max(largest, v[h].w[w]);
        }
        // the power of two that puts the tile's largest step into [2^14, 2^15)
        largest = __reduce_max_sync(0xffffffffu, largest);
        const uint32_t ex = min(254u, 268u - min(254u, (largest >> 23) & 0xffu));
        const float up = __uint_as_float(ex << 23);
        down = __uint_as_float((278u - ex) << 23);  // 2^24 / up
#pragma unroll
        for (int h = 0; h < BATCHES; ++h) {
          Floats<NB> step, low;
#pragma unroll
          for (int w = 0; w < NB; ++w) {
            step.f[w] = high_bf16(v[h].w[w]);
            low.f[w] = fmaf(-8.f, step.f[w], low_bf16(v[h].w[w]));
            step.f[w] *= up;
          }
          sts_floats<NB>(v_step + lane * NG + h * NB, step);
          sts_floats<NB>(v_low + lane * NG + h * NB, low);
        }
        __syncwarp();
      }
      // ---- logits: keys are the rows of A (blocks 2 j and 2 j + 1 of 8), this lane has key key_row of each block
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      Pair s[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
      float term[2][4];
#pragma unroll
      for (int h = 0; h < BATCHES; ++h) {
        Words<NB> codes[4], meta[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int r = 8 * n + key_row;
          if constexpr (NG >= 4) codes[n] = lds_words<NB>(tile + T::K + r * (D / 2) + (((4 * h + tig) ^ T::swap(r)) * 16));
          else codes[n] = lds_words<NB>(tile + T::K + r * (D / 2) + tig * NB * 4);
          meta[n] = lds_words<NB>(tile + T::KM + (r * NG + h * NB) * 4);
        }
#pragma unroll
        for (int w = 0; w < NB; ++w) {
          const uint4 q = q_frag[(h * NB + w) * 32 + lane];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x0 = codes[2 * j].w[w], x1 = codes[2 * j + 1].w[w], y0 = x0 >> 8, y1 = x1 >> 8;
            float part[4];
            mma_f16(part, make_uint4(x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u), q.x, q.y, none);
            mma_f16(part, make_uint4(y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u), q.z, q.w, part);
            const float s0 = high_bf16(meta[2 * j].w[w]), s1 = high_bf16(meta[2 * j + 1].w[w]);
            s[2 * j].x = fmaf(part[0], s0, s[2 * j].x), s[2 * j].y = fmaf(part[1], s0, s[2 * j].y);
            s[2 * j + 1].x = fmaf(part[2], s1, s[2 * j + 1].x), s[2 * j + 1].y = fmaf(part[3], s1, s[2 * j + 1].y);
          }
        }
        const uint4 q = q_frag[(NG + h) * 32 + lane];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t word[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            word[i] = tig < NB ? *reinterpret_cast<const uint32_t*>(tile + T::KM + ((16 * j + 8 * i + key_row) * NG + h * NB + (tig < NB ? tig : 0)) * 4) : 0u;
          const uint4 a = make_uint4(word[0], word[1], word[0], word[1]);
          if (h == 0) mma_bf16(term[j], a, q.x, q.y, none);
          else mma_bf16(term[j], a, q.x, q.y, term[j]);
          mma_bf16(term[j], a, q.z, 0u, term[j]);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n)
        s[n] = fma2(mul2(s[n], back), {p.scale_log2 * 0x1p24f, p.scale_log2 * 0x1p24f}, {term[n >> 1][2 * (n & 1)], term[n >> 1][2 * (n & 1) + 1]});
      if (mask != 0xffffffffu) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (!((mask >> (8 * n + key_row)) & 1)) s[n] = {-INFINITY, -INFINITY};
      }
      // ---- softmax of the tile
      Pair top = mx;
#pragma unroll
      for (int n = 0; n < 4; ++n) top.x = fmaxf(top.x, s[n].x), top.y = fmaxf(top.y, s[n].y);
#pragma unroll
      for (int i = 4; i < 32; i <<= 1) top.x = fmaxf(top.x, __shfl_xor_sync(0xffffffffu, top.x, i)), top.y = fmaxf(top.y, __shfl_xor_sync(0xffffffffu, top.y, i));
      const Pair zero = {top.x == -INFINITY ? 0.f : top.x, top.y == -INFINITY ? 0.f : top.y};
      if (__any_sync(0xffffffffu, top.x != mx.x || top.y != mx.y)) {
        const Pair alpha = {exp2f(mx.x - zero.x), exp2f(mx.y - zero.y)};
        sum = mul2(sum, alpha);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          z[g] = mul2(z[g], alpha);
#pragma unroll
          for (int i = 0; i < 2; ++i) o[g][i][0] *= alpha.x, o[g][i][1] *= alpha.y, o[g][i][2] *= alpha.x, o[g][i][3] *= alpha.y;
        }
        mx = top;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        s[n].x = exp2f(s[n].x - zero.x), s[n].y = exp2f(s[n].y - zero.y);
        sum = add2(sum, s[n]);
      }
      // ---- sum p lo, and sum (p s) c with p s in fp16; PB groups at a time
      constexpr int PB = NG < 2 ? 1 : 2;
#pragma unroll
      for (int h = 0; h < NG / PB; ++h) {
        uint32_t codes[4][2], pb[4][PB];  // codes: a lane's numbers of two groups (D = 32: of one, a half word)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const Floats<PB> step = lds_floats<PB>(v_step + (8 * n + key_row) * NG + h * PB), low = lds_floats<PB>(v_low + (8 * n + key_row) * NG + h * PB);
#pragma unroll
          for (int g = 0; g < PB; ++g) {
            pb[n][g] = transpose(half2_bits(s[n].x * step.f[g], s[n].y * step.f[g]));
            z[h * PB + g].x = fmaf(s[n].x, low.f[g], z[h * PB + g].x), z[h * PB + g].y = fmaf(s[n].y, low.f[g], z[h * PB + g].y);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + row_e[e];
            const uint8_t* row = tile + T::V + r * (D / 2);
            if constexpr (D == 256) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + ((gid ^ T::swap(r)) * 16) + h * 4);
            else if constexpr (D == 128) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + (((gid >> 1) ^ T::swap(r)) * 16) + (gid & 1) * 8 + h * 4);
            else if constexpr (D == 64) codes[n][e] = *reinterpret_cast<const uint32_t*>(row + gid * 4);
            else codes[n][e] = *reinterpret_cast<const uint16_t*>(row + gid * 2);
          }
        }
#pragma unroll
        for (int g = 0; g < PB; ++g) {
          uint32_t pair[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) pair[n] = __byte_perm(codes[n][0], codes[n][1], g ? 0x7632 : 0x5410);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float t[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t x = i ? pair[2 * j] >> 8 : pair[2 * j], y = i ? pair[2 * j + 1] >> 8 : pair[2 * j + 1];
              const uint4 a = make_uint4(x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u);
              if (j == 0) mma_f16(t, a, pb[0][g], pb[1][g], none);
              else mma_f16(t, a, pb[2][g], pb[3][g], t);
            }
            float(&to)[4] = o[h * PB + g][i];
            const Pair lo = fma2({t[0], t[1]}, {down, down}, {to[0], to[1]});
            const Pair hi = fma2({t[2], t[3]}, {down * 0.0625f, down * 0.0625f}, {to[2], to[3]});
            to[0] = lo.x, to[1] = lo.y, to[2] = hi.x, to[3] = hi.y;
          }
        }
      }
    }
    __syncwarp();  // the ring is free
  }
}

static_assert(kKv4Positions <= 0x7fffffffLL - 4 * 32 * 12, "no position that a warp asks for passes 32 bits");
template <int D, int W> static int kv4_attn_launch(const Kv4Attn& p, long long room, long long max_len, cudaStream_t st) {
  constexpr int bytes = W * Kv4Tile<D>::WARP + Kv4Tile<D>::QUERY;
  static_assert(Kv4Tile<D>::SPACE >= 4 * D * 4 && Kv4Tile<D>::SPACE >= 32 * 32, "a warp's space holds four heads of its sums");
  static std::atomic<unsigned long long> ready{0};  // devices that have been told (a tenth of a small call's time)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -5;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kv4_attn_kernel<D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -5;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  // positions are counted in 32 bits, up to three turns behind a request's last one
  if (p.max_ctx > kKv4Positions || p.batch * (p.max_ctx / (32LL * W) + 4) > 0x3fffffffLL) return -4;
  const long long most = p.batch * ((max_len - 1) / (32 * W) + 1);  // units, if no request is longer
  long long groups = 148 * kv4_per_sm<D, W>() / p.heads;
  if (groups > room) groups = room;
  if (groups > most) groups = most;
  if (groups < 1) groups = 1;
  if (groups * p.heads > 0x7fffffffLL) return -4;
  kv4_attn_kernel<D, W><<<(unsigned)(groups * p.heads), W * 32, bytes, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

// Where the workspace has fewer parts than a wave of CTAs would make (few long requests), each is made by more warps: one
// request of 65521 tokens over 8 kv heads, 32 parts, takes 34.7 us with 12 warps a CTA and 37.3 with 4.  Elsewhere a cut
// every 128 keys divides the work better than one every 384: 128 mixed requests 28.8 us with 4 warps, 39.1 with 12.
template <int D> static int kv4_attn_pick(const Kv4Attn& p, int parts, long long max_len, cudaStream_t st) {
  const long long room = (long long)p.batch * (parts - 1) + 1;
  if constexpr (D <= 128) {
    const long long shares = p.batch * ((max_len - 1) / 128 + 1 + KV4_SETUP) / (KV4_SETUP + 1), wave = 148 * kv4_per_sm<D, 4>() / p.heads;
    if (room < (shares < wave ? shares : wave)) return kv4_attn_launch<D, 12>(p, room, max_len, st);
  }
  return kv4_attn_launch<D, 4>(p, room, max_len, st);
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
    case 32: return kv4_attn_pick<32>(p, parts, longest, st);
    case 64: return kv4_attn_pick<64>(p, parts, longest, st);
    case 128: return kv4_attn_pick<128>(p, parts, longest, st);
    case 256: return kv4_attn_pick<256>(p, parts, longest, st);
    default: return -3;
  }
}

// ------------------------------------------------------------------------------------------------------- copy pages
// Page dst[i] of every layer of every pool becomes a copy of page src[i].  The page numbers travel in the launch's
// parameters, so the call keeps no buffer alive and can be captured into a graph as it stands.  Bound by memory: 192 pages
// of 16 tokens in 32 layers of 8 heads of 128 numbers in 4 bits (252 MB read and written) take 40 us, 96% of a copy's rate.
template <typename Unit>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageCopies c) {
  const int pool = blockIdx.z, layer = blockIdx.y, pair = blockIdx.x;
  const long long page = c.page_bytes[pool];
  char* base = static_cast<char*>(c.base[pool]) + layer * c.layer_bytes[pool];
  const Unit* src = reinterpret_cast<const Unit*>(base + c.src[pair] * page);
  Unit* dst = reinterpret_cast<Unit*>(base + c.dst[pair] * page);
  const long long n = page / (long long)sizeof(Unit);
  constexpr int DEEP = 4;  // units of a thread that are on their way at a time
  for (long long i = threadIdx.x; i < n; i += DEEP * 256) {
    Unit unit[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k)
      if (i + k * 256 < n) unit[k] = src[i + k * 256];
#pragma unroll
    for (int k = 0; k < DEEP; ++k)
      if (i + k * 256 < n) dst[i + k * 256] = unit[k];
  }
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
