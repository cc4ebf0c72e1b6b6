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

// Pieces a long loop is cut into when a call has fewer CTAs than SMs: enough to fill one wave, or,
// where a causal or document mask makes the loops unequal, two CTAs per SM; none shorter than four
// steps (a piece costs its start and its sums' way through memory).  148 SMs whatever the device,
// so that the workspace follows from the call alone.  Measured: backward, 16384 causal tokens on one
// key head (128 CTAs), 2392 -> 1580 us; equal loops of that number cut the same way were slower
// (2944 -> 3322 us), and so was a forward pass of 192 CTAs (81 -> 116 us), although calls of 149 to some 300
// unequal CTAs take two waves whose longest CTAs set the time.
inline int pieces_of(const AttnProblem& p, long long ctas, long long steps) {
  if (ctas >= 148) return 1;
  const long long want = p.causal || p.documents ? (2 * 148 + ctas - 1) / ctas : 148 / ctas, most = steps / 4;
  return (int)(want < most ? want : most > 1 ? most : 1);
}

// Whether a scale and a cap (0: none) are numbers the kernels can work with.
bool scores_ok(float scale, float softcap);
// Refuses what the attention kernels do not take and fills in the device's view of the rest.
int32_t attention_problem(const lego_attention_t* d, AttnProblem* out);
// Bytes of the document summaries; 0 without documents.
int64_t attention_docs_bytes(const AttnProblem& p);
// Workspace of the forward pass.
int64_t attention_fwd_bytes(const AttnProblem& p);
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// The largest of N values: three to an instruction, four chains.
template <int N>
__device__ __forceinline__ float max_of(const float (&s)[N]) {
  float top[4] = {max3(s[0], s[1], s[2]), max3(s[3], s[4], s[5]), max3(s[6], s[7], s[8]), max3(s[9], s[10], s[11])};
#pragma unroll
  for (int c = 12; c + 1 < N; c += 2) top[(c >> 1) & 3] = max3(top[(c >> 1) & 3], s[c], s[c + 1]);
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(u) for |u| <= 1: an odd polynomial of degree 13, off by 2e-8 (1e-7 in 32 bits).  Scores under
// a cap rarely reach it, and the exact way below takes two of the 16 per cycle.
__device__ __forceinline__ float2 tanh_near(float2 u) {
  const float2 w = ptx::mul2(u, u);
  float2 p = make_float2(9.637710173e-04f, 9.637710173e-04f);
  p = ptx::fma2(p, w, make_float2(-5.951276980e-03f, -5.951276980e-03f));
  p = ptx::fma2(p, w, make_float2(1.997327805e-02f, 1.997327805e-02f));
  p = ptx::fma2(p, w, make_float2(-5.326583236e-02f, -5.326583236e-02f));
  p = ptx::fma2(p, w, make_float2(1.331958324e-01f, 1.331958324e-01f));
  p = ptx::fma2(p, w, make_float2(-3.333213031e-01f, -3.333213031e-01f));
  p = ptx::fma2(p, w, make_float2(9.999997020e-01f, 9.999997020e-01f));
  return ptx::mul2(p, u);
}
// Whether tanh_near does for all scores of the warp's rows.
template <int N>
__device__ __forceinline__ bool all_near(const float (&s)[N], float to_u) {
  float top[2] = {fabsf(s[0]), fabsf(s[1])};
#pragma unroll
  for (int c = 2; c < N; ++c) top[c & 1] = fmaxf(top[c & 1], fabsf(s[c]));
  return __all_sync(~0u, fmaxf(top[0], top[1]) * fabsf(to_u) <= 1.f);
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

// A row's weights are 2^(s - m) for a reference value m that moves only when the row's maximum outgrows it by
// kLag, so O in TMEM is rarely rescaled.  bf16: m is the maximum of its time, weights stay below 2^8.
// fp16 has no range to spare: a weight loses bits below 2^-14 and is zero below 2^-25, and many keys far below
// the largest can make up much of a row.  There m is the maximum less kLift and lags by less, so
// the weights stand times 2^11 and more and stay below 2^15: 17 nats under the largest still have all bits, what becomes
// zero is under 2^-36 of it, and 2^20 such keys together under a thirtieth of the result's rounding.
// (Lags of 2^2, 2^4 and 2^8: 2 x 4096 causal tokens x 32/8 heads of 128 255, 246 and 247 us; documents of 45 to
// 2162 tokens with a cap no difference.)
template <bool BF16> constexpr float kLag = BF16 ? 8.f : 4.f;
template <bool BF16> constexpr float kLift = BF16 ? 0.f : 11.f;
static_assert(kLag<false> + kLift<false> <= 15.f, "weights have to stay in fp16's range");

// A row's reference value m for a tile whose maximum is mt (log2 units).  Not the first tile:
// where some row of the warp outgrew its reference value, its sums, in two registers and over DP
// columns of o_tmem, follow it.
template <int DP, bool BF16>
__device__ __forceinline__ void follow_maximum(float mt, bool first, float* m, float* sum, float* sum2, uint32_t o_tmem) {
  mt -= kLift<BF16>;
  if (first) {
    *m = mt;
  } else if (__any_sync(~0u, mt > *m + kLag<BF16>)) {
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
// The natural logarithm of a row's sum of exp(s).
template <bool BF16>
__device__ __forceinline__ float log_of_sum(float m, float sum) {
  constexpr float by = BF16 ? 1.f : 1.f / (1 << (int)kLift<false>);
  return (m + kLift<BF16> + log2f(sum * by)) * kLn2;
}

// Raw scores to log2 units: z = cap tanh(scale s / cap) - slope distance, times log2(e).  first:
// position minus that of the first key.
struct Scores {
  float by;              // scale log2(e)
  float to_u, cap_by;    // scale / cap, cap log2(e)
  float slope;           // slope log2(e)
};
template <bool CAP>
__device__ __forceinline__ Scores scores_of(float scale, float softcap, const float* slopes, int h) {
  Scores s;
  s.by = scale * kLog2e;
  s.to_u = CAP ? scale / softcap : 0.f;
  s.cap_by = softcap * kLog2e;
  s.slope = slopes ? slopes[h] * kLog2e : 0.f;
  return s;
}
// The bias where no key is ahead: linear in the column, and no conversion per key (an integer to a
// float costs as much as an exponential); 8192 causal tokens of 16 heads of 128 355 -> 319 us.  The
// product slope * from is rounded by 2^-24 of itself, that is of the bias 128 keys on at most, and
// alike for all the columns.
template <int N, bool CAP>
__device__ __forceinline__ void bias_behind(float (&s)[N], const Scores& sc, float from) {
  const float2 slope2 = make_float2(sc.slope, sc.slope), base2 = make_float2(-sc.slope * from, -sc.slope * from);
  const float2 by2 = make_float2(sc.by, sc.by);
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const float2 off = ptx::fma2(slope2, make_float2((float)c, (float)(c + 1)), base2);
    const float2 z = make_float2(s[c], s[c + 1]);
    const float2 r = CAP ? ptx::add2(z, off) : ptx::fma2(z, by2, off);
    s[c] = r.x;
    s[c + 1] = r.y;
  }
}
template <int N, bool CAP, bool BIAS>
__device__ __forceinline__ void score(float (&s)[N], const Scores& sc, int first) {
  if (CAP) {
    if (all_near(s, sc.to_u)) {
#pragma unroll
      for (int c = 0; c < N; c += 2) {
        const float2 z = ptx::mul2(tanh_near(ptx::mul2(make_float2(s[c], s[c + 1]), make_float2(sc.to_u, sc.to_u))),
                                   make_float2(sc.cap_by, sc.cap_by));
        s[c] = z.x;
        s[c + 1] = z.y;
      }
    } else {
      const float by = 2.f * kLog2e * sc.to_u;
#pragma unroll
      for (int c = 0; c < N; ++c) s[c] = sc.cap_by * tanh_of(s[c] * by);
    }
  }
  if (BIAS) {
    const float from = (float)first;      // past 2^24 a distance is rounded, by 2^-24 of itself
    if (__all_sync(~0u, first >= N - 1)) {
      bias_behind<N, CAP>(s, sc, from);
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c) s[c] = fmaf(-sc.slope, fabsf(from - (float)c), CAP ? s[c] : s[c] * sc.by);
    }
  }
}

// Both 16-bit values of a pair, added to 32-bit sums.
template <bool BF16>
__device__ __forceinline__ void add_packed(uint32_t pair, float* lo, float* hi) {
  if constexpr (BF16)
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; add.f32.bf16 %0, l, %0; add.f32.bf16 %1, h, %1;}" : "+f"(*lo), "+f"(*hi) : "r"(pair));
  else
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; add.f32.f16 %0, l, %0; add.f32.f16 %1, h, %1;}" : "+f"(*lo), "+f"(*hi) : "r"(pair));
}

// One thread per row: the row's 128 scores s (hidden ones -inf) become weights
// 2^(s by - m) (SCALED: s is in log2 units already), packed to 16 bits over columns 0 .. 63 of
// s_tmem; ready[i] gets the warp's arrival when 64 of them are in place.  `sum` takes the weights as
// they are, for the row's logarithm, `packed_sum` as they were rounded: divided by it, the result's
// weights add up to one, so an error all of them share, above all that of a row's one large weight,
// falls out.  (Two sums cost 2 %: 16384 causal tokens x 8 heads of 128 415 -> 422 us; 426 where a pair is added
// before its group is stored, 440 with pairs unpacked to 32 bits first.)  by > 0.
template <bool BF16, bool SCALED>
__device__ __forceinline__ void weigh(const float (&s)[kTile], float by, float m, float* sum, float* packed_sum,
                                      uint32_t s_tmem, uint64_t* ready, int lane) {
  const float mu = m == -INFINITY ? 0.f : m;
  float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, packed_add[2] = {add[0], add[0]};
  const float2 by2 = make_float2(by, by), mu2 = make_float2(-mu, -mu);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int c = half * 64; c < half * 64 + 64; c += 32) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float2 z = make_float2(s[c + i], s[c + i + 1]);
        z = SCALED ? ptx::add2(z, mu2) : ptx::fma2(z, by2, mu2);
        const float2 x = make_float2(ex2(z.x), ex2(z.y));
        add[(i >> 1) & 1] = ptx::add2(add[(i >> 1) & 1], x);
        w[i >> 1] = pack2<BF16>(x.x, x.y);
      }
      ptx::tmem_st_32x16(s_tmem + c / 2, w);
#pragma unroll
      for (int i = 0; i < 16; ++i) add_packed<BF16>(w[i], &packed_add[i & 1].x, &packed_add[i & 1].y);
    }
    ptx::tmem_st_wait();
    ptx::tc_fence_before();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ready[half]));
  }
  *sum += (add[0].x + add[0].y) + (add[1].x + add[1].y);
  *packed_sum += (packed_add[0].x + packed_add[0].y) + (packed_add[1].x + packed_add[1].y);
}
template <int DP, bool BF16, bool SCALED>
__device__ __forceinline__ void weigh_tile(const float (&s)[kTile], float by, bool first, float* m, float* sum,
                                           float* packed_sum, uint32_t s_tmem, uint32_t o_tmem, uint64_t* ready, int lane) {
  float mt = max_of(s);
  if (!SCALED) mt *= by;
  follow_maximum<DP, BF16>(mt, first, m, sum, packed_sum, o_tmem);
  weigh<BF16, SCALED>(s, by, *m, sum, packed_sum, s_tmem, ready, lane);
}

__device__ __forceinline__ void attn_fail(uint32_t* status, volatile uint32_t* abort_flag, uint32_t code) {
  *abort_flag = 1;
  atomicCAS(status, 0u, code);
}

}  // namespace lego
