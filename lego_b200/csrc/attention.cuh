// Shared by the attention kernels: the problem as the device sees it, which key a query
// sees, and what the tiles of 128 x 128 scores are made of.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace lego {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 128;            // queries and keys of one tile
constexpr int kBoxBytes = kTile * 128;   // 64 values of 128 tokens: one TMA box
// Limit of one wait, in cycles of the SM clock: about a second.
constexpr long long kAttnWait = 2000000000LL;

struct AttnProblem {
  int batch, q_len, k_len, q_heads, k_heads, dim, group;   // group: query heads of one key head
  int offset;                                              // position of query 0: k_len - q_len
  int causal;
  float scale, softcap;
  long long q_stride[3], k_stride[3], v_stride[3];         // batch, token, head, in elements
  const float* slopes;
  const int* prefix;
  const int* documents;
  // of every tile of keys, then of every tile of queries, [batch][tile]: smallest and largest
  // document number that is not negative (min > max: there is none), whether a token is padding
  const int4* key_docs;
  const int4* query_docs;
};

inline __host__ __device__ int tiles_of(int n) { return (n + kTile - 1) / kTile; }

// Refuses what the attention kernels do not take and fills in the device's view of the rest.
int32_t attention_problem(const lego_attention_t* d, AttnProblem* out);
// Bytes of the document summaries; 0 without documents.
int64_t attention_docs_bytes(const AttnProblem& p);
// Enqueues the kernel that writes them to `where` and points the problem at them.
int32_t attention_docs(AttnProblem* p, void* where, cudaStream_t s);

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(u), given 2 log2(e) u: 1 - 2 / (1 + e^2u), off by a few 2^-24 absolutely.
__device__ __forceinline__ float tanh_of(float twice_log2e_u) { return fmaf(-2.f, rcp(1.f + ex2(twice_log2e_u)), 1.f); }

// ---- which key a query sees --------------------------------------------------------------

// The query at position pos sees keys 0 .. last_key(pos) of its document.
__device__ __forceinline__ int last_key(const AttnProblem& p, int prefix, int pos) {
  if (!p.causal) return p.k_len - 1;
  const int last = pos > prefix - 1 ? pos : prefix - 1;
  return last < p.k_len - 1 ? last : p.k_len - 1;
}
__device__ __forceinline__ int prefix_of(const AttnProblem& p, int b) {
  if (!p.prefix) return 0;
  const int n = p.prefix[b];
  return n < 0 ? 0 : n > p.k_len ? p.k_len : n;
}
__device__ __forceinline__ bool docs_meet(const int4& a, const int4& b) { return a.x <= b.y && b.x <= a.y; }
// both tiles are one and the same document throughout
__device__ __forceinline__ bool docs_same(const int4& a, const int4& b) {
  return a.x == a.y && b.x == b.y && a.x == b.x && !a.z && !b.z;
}

// Bits c (0 .. 31 of word w) of the columns of a tile up to column `last`.
__device__ __forceinline__ uint32_t bits_upto(int last, int w) {
  const int n = last + 1 - 32 * w;
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
}
// Clears the columns whose document differs from this lane's: other[w] is the document of
// column 32 w + lane, own this lane's row's.  All lanes of the warp take part.
template <int W>
__device__ __forceinline__ void mask_documents(uint32_t (&m)[W], const int (&other)[W], int own) {
  uint32_t same[W] = {};
  uint32_t todo = __ballot_sync(~0u, own >= 0);
  while (todo) {
    const int d = __shfl_sync(~0u, own, __ffs(todo) - 1);
    const bool mine = own == d;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t eq = __ballot_sync(~0u, other[w] == d);
      if (mine) same[w] = eq;
    }
    todo &= ~__ballot_sync(~0u, mine);
  }
#pragma unroll
  for (int w = 0; w < W; ++w) m[w] &= same[w];
}

// ---- tiles in shared memory ----------------------------------------------------------------

// A tile is DP / 64 boxes of [128 tokens][64 values], rows of 128 bytes under the 128-byte
// swizzle: as a K-major operand its 16-value steps are 32 bytes apart inside a box, as an
// MN-major one 16 tokens are 2 KiB and 64 values one box apart.
template <int DP> constexpr int tile_bytes() { return DP / 64 * kBoxBytes; }
// The descriptors of a tile differ in the low word only, by a constant per step: one addition.
__device__ __forceinline__ uint64_t tile_desc(uint32_t low) {
  constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29);    // smem_desc_sw128: stride 1024, swizzle
  return (uint64_t)high << 32 | low;
}
__device__ __forceinline__ uint32_t low_k_major(uint32_t tile) { return (tile >> 4) + (1u << 16); }
__device__ __forceinline__ uint32_t low_mn_major(uint32_t tile) { return (tile >> 4) + ((uint32_t)(kBoxBytes >> 4) << 16); }
__device__ __forceinline__ uint64_t desc_k_major(uint32_t low, int step) {    // step: 16 values
  return tile_desc(low + (((step >> 2) * kBoxBytes + (step & 3) * 32) >> 4));
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t low, int step) {   // step: 16 tokens
  return tile_desc(low + ((step * 2048) >> 4));
}
template <bool BF16>
__device__ __forceinline__ uint32_t idesc_of(int n, bool b_mn) {
  return BF16 ? ptx::idesc_bf16(kTile, n, 0, b_mn) : ptx::idesc_f16(kTile, n, 0, b_mn);
}

// One warp's copy of a tile by plain loads, zeros in the place of padding tokens (negative
// documents) and past the ends: for tiles that hold padding, whose values may be anything
// while a product 0 * NaN must not come about.  base: value (token 0, this head and batch).
// docs: document of token 0.  The caller arrives on the tile's barrier afterwards.
template <int DP>
__device__ __forceinline__ void copy_tile_clean(uint8_t* tile, const uint16_t* base, long long token_stride, int dim,
                                                int first, int len, const int* docs, int lane) {
  constexpr int CH = DP / 8;   // 16-byte pieces of a row
  for (int i = lane; i < kTile * CH; i += 32) {
    const int r = i / CH, c = i % CH, tok = first + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (tok < len && c * 8 < dim && docs[tok] >= 0) v = *reinterpret_cast<const uint4*>(base + tok * token_stride + c * 8);
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  ptx::fence_proxy_async();
  __syncwarp();
}

// ---- a tile of scores to weights ---------------------------------------------------------------

// log2 of the growth a row's reference value may lag behind its maximum: weights stay below
// 2^8, their sum is kept in 32 bits, and O in TMEM is rarely rescaled.
constexpr float kRescale = 8.f;

// A row's reference value m for a tile whose maximum is mt (log2 units).  Not the first tile:
// where some row of the warp outgrew its reference value, its sums, in two registers and over DP
// columns of o_tmem, follow it.
template <int DP>
__device__ __forceinline__ void follow_maximum(float mt, bool first, float* m, float* sum, float* sum2, uint32_t o_tmem) {
  if (first) {
    *m = mt;
  } else if (__any_sync(~0u, mt > *m + kRescale)) {
    const float mn = fmaxf(*m, mt);
    const float f = mn == -INFINITY ? 1.f : ex2(*m - mn);
    *m = mn;
    *sum *= f;
    *sum2 *= f;
#pragma unroll
    for (int c = 0; c < DP; c += 16) {     // rare, and the scores fill the registers
      uint32_t o[16];
      ptx::tmem_ld_32x16(o_tmem + c, o);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
      ptx::tmem_st_32x16(o_tmem + c, o);
    }
  }
}

// One thread per row: the row's 128 scores s (hidden ones -inf) become weights
// 2^(s by - m) (SCALED: s is in log2 units already), packed to 16 bits over columns 0 .. 63 of
// s_tmem.  `sum` takes the weights as they are, for the row's logarithm; `packed_sum` as they
// were rounded: divided by it, the result's weights add up to one, so an error all of them
// share, above all that of a row's one large weight, falls out.  by > 0.
template <int DP, bool BF16, bool SCALED>
__device__ __forceinline__ void weigh_tile(const float (&s)[kTile], float by, bool first, float* m, float* sum,
                                           float* packed_sum, uint32_t s_tmem, uint32_t o_tmem) {
  float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int c = 4; c < kTile; ++c) top[c & 3] = fmaxf(top[c & 3], s[c]);
  float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  if (!SCALED) mt *= by;
  follow_maximum<DP>(mt, first, m, sum, packed_sum, o_tmem);
  const float mu = *m == -INFINITY ? 0.f : *m;
  float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, packed_add[2] = {add[0], add[0]};
  const float2 by2 = make_float2(by, by), mu2 = make_float2(-mu, -mu);
#pragma unroll
  for (int c = 0; c < kTile; c += 32) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float2 z = make_float2(s[c + i], s[c + i + 1]);
      z = SCALED ? ptx::add2(z, mu2) : ptx::fma2(z, by2, mu2);
      const float2 x = make_float2(ex2(z.x), ex2(z.y));
      const int k = (i >> 1) & 1;
      add[k] = ptx::add2(add[k], x);
      w[i >> 1] = pack2<BF16>(x.x, x.y);
      packed_add[k] = ptx::add2(packed_add[k], unpack2<BF16>(w[i >> 1]));
    }
    ptx::tmem_st_32x16(s_tmem + c / 2, w);
  }
  *sum += (add[0].x + add[0].y) + (add[1].x + add[1].y);
  *packed_sum += (packed_add[0].x + packed_add[0].y) + (packed_add[1].x + packed_add[1].y);
  ptx::tmem_st_wait();
}

__device__ __forceinline__ void attn_fail(uint32_t* status, volatile uint32_t* abort_flag, uint32_t code) {
  *abort_flag = 1;
  atomicCAS(status, 0u, code);
}

}  // namespace lego
