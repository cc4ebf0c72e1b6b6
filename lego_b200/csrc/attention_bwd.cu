// Attention backward on tcgen05 (sm_100a).
//
//   P = exp(s - lse), dV = P^T dO, dP = dO V^T, dS = P (dP - delta) (1 - tanh^2 of a cap),
//   dQ = scale dS K, dK = scale dS^T Q, delta = row sum of dO O.
//
// Three launches.  A preparation writes delta and the rows' log-sums in the form the others
// use.  The key kernel takes a tile of 128 keys per CTA and walks the tiles of queries of
// all heads that share the key head: dK and dV stay in TMEM from the first to the last, so
// shared heads are summed in a fixed order.  The query kernel takes a tile of 128 queries
// and walks the keys: dQ stays in TMEM.  Scores are computed in both, seven products instead
// of the five that one kernel with a sum of dQ over CTAs in memory would take; in return no
// addition depends on the order in which CTAs happen to run, and there is no dQ in 32 bits to
// clear, add to and convert.
//
// Where the tiles are too few to load the SMs alike (short or shared key heads; few queries), a
// CTA's loop is cut into pieces whose sums go through the workspace in 32 bits and are added in
// order by one more launch.
//
// Key kernel: S^T = K Q^T and dP^T = V dO^T into TMEM, one thread per key and half the
// columns (two warpgroups); P^T and dS^T go back over them as 16-bit pairs and are the TMEM
// operands of dV += P^T dO and dK += dS^T Q.  The order of issue is dV(n), S(n + 1), dK(n),
// dP(n + 1): the products of one kind run while the warps work on the other.  All 512
// columns of TMEM are in use (64-wide heads: 384).  Query kernel: S in two buffers, so the
// weights of a tile are ready when its dP is.
//
// fp16: P is kept times 2^14 (weights of long rows fall below the type's normal range) and dS times a
// power of two that a bound on it leaves in range, |dS| <= |dP - delta| <= max|dO_i| sum|V_j| + |delta_i|.  The
// query kernel has one per row, from the keys it walks.  In the key kernel the rows of a sum are queries: one
// per step (128 queries of one head), and where the next step's is another, dK in TMEM follows, which
// a power of two does exactly.  So a token's gradients do not depend on how large dO is elsewhere, but for
// dK from queries of one tile: what is 2^-29 of the tile's bound still has all bits.  All powers are taken out of
// the 32-bit sums at the end.
//
// What bounds it: the tensor pipe (67 % and 60 % busy at heads of 128, 28 % at 64) and the warps that feed it (issue
// slots 47 % and 39 %, under a cap 53 %) take turns; memory is idle.  Counting 10 flop per visible pair and value, from
// a cold L2: 16384 causal tokens x 8/1 heads of 128, bf16 1.60 ms (0.86 PFLOP/s), all keys, fp16 3.30 ms (0.83);
// 2 x 4096 causal x 32/8 heads, bf16 0.90 ms (0.76), fp16 0.96; 8192 causal x 16 heads of 64, fp16 0.84 ms (0.41), bf16
// 0.77, with a cap, fp16 1.20 ms.  The key kernels of 64-wide heads spill 4 or 5 registers, as do the query kernels
// under a cap.  Slower: products of 64 columns in the key kernel (858 -> 1143 us).
#include <cuda.h>

#include <type_traits>

#include "attention.cuh"
#include "tma_host.cuh"

namespace lego {
namespace {

constexpr int kBwdThreads = 384;
constexpr int kBwdRegs = 168, kMathRegs = 216, kBwdOtherRegs = 72;
static_assert(2 * kMathRegs + kBwdOtherRegs <= 3 * kBwdRegs, "more registers than the launch has would wait forever");
constexpr int kWeightShift = 14;     // fp16: log2 of the factor on P
constexpr int kStats = 264;          // floats of a step's rows: -lse, -delta, and in fp16 4 x (peak of dO, of |delta|)

struct BwdArgs {
  CUtensorMap q, k, v, d_o;          // boxes of 128 tokens
  CUtensorMap dq, dk, dv;            // boxes of 32 tokens
  AttnProblem p;
  const uint16_t *q_raw, *k_raw, *o_raw, *low_raw, *do_raw, *v_raw;    // low_raw: what o's rounding left, or null
  const float* lse;
  float *neg_lse, *neg_delta;        // [batch][q_heads][q_len up to whole tiles], log2 units
  // fp16: max|dO| of every row; of 32 rows, and the largest |delta|; the largest sum|V| of 32 keys
  float *row_peak;                   // like neg_lse
  float2 *query_peaks;               // [batch][q_heads][query tiles][4]
  float *key_peaks;                  // [batch][k_heads][key tiles][4]
  uint32_t* status;
  int key_pieces, query_pieces;
  float *key_part, *query_part;      // [piece][tile CTA](dV, dK)[128][DP]; [piece][tile CTA][128][DP]
  uint16_t *dq_raw, *dk_raw, *dv_raw;
};

__device__ __forceinline__ long long row_slot(const AttnProblem& p, int b, int h) {
  return ((long long)b * p.q_heads + h) * tiles_of(p.q_len) * kTile;
}

// fp16: log2 of the factor that brings a bound on dS to 2^14 .. 2^15, half of the type's range; false
// where there is none (nothing but zeros; an infinity or a NaN, which no factor mends).
__device__ __forceinline__ bool factor_log2(float bound, int* e) {
  if (!(bound > 1e-30f) || !(bound < 1e30f)) return false;
  *e = 14 - ((int)(__float_as_uint(bound) >> 23) - 127);
  return true;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float max_of4(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }

// ---- preparation -----------------------------------------------------------------------------

// Per row delta and the negated log-sum, and in fp16 the peaks of dO, delta and V.  Rows past q_len (whole
// tiles) and padding get weight zero: -inf.  A warp takes 32 tokens of one head, a block the same
// tokens of eight heads, which lie together in memory; four rows are under way at a time, and lane i
// keeps token i's results so they leave as one line.  Memory bound at heads of 128 (4.6 TB/s); at 64 half the lanes
// have nothing to load, and in fp16 it is 1.7 TB/s (2 x 4096 tokens x 16 heads 40 us).
struct PrepGrid {
  int q_chunks, q_blocks, k_blocks;     // of 32 tokens; of 8 heads x 32 tokens
};
__host__ __device__ inline PrepGrid prep_grid(const AttnProblem& p, bool peaks) {
  PrepGrid g;
  g.q_chunks = tiles_of(p.q_len) * 4;
  g.q_blocks = p.batch * g.q_chunks * ((p.q_heads + 7) / 8);
  g.k_blocks = peaks ? p.batch * tiles_of(p.k_len) * 4 * ((p.k_heads + 7) / 8) : 0;
  return g;
}
template <bool BF16>
__global__ void __launch_bounds__(256) attn_bwd_prep_kernel(const __grid_constant__ BwdArgs a) {
  const AttnProblem& p = a.p;
  const PrepGrid g = prep_grid(p, !BF16);
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool mine = lane * 4 < p.dim;
  if ((int)blockIdx.x < g.q_blocks) {
    const int groups = (p.q_heads + 7) / 8;
    const int h = (int)(blockIdx.x % groups) * 8 + warp, chunk = (int)(blockIdx.x / groups) % g.q_chunks;
    const int b = (int)(blockIdx.x / groups) / g.q_chunks;
    if (h >= p.q_heads) return;
    const int i0 = chunk * 32, own = i0 + lane;
    const bool real = own < p.q_len && (!p.documents || p.documents[(long long)b * p.k_len + p.offset + own] >= 0);
    const uint32_t rows = __ballot_sync(~0u, real);
    float kept = 0.f, own_peak = 0.f;
    const long long stride = (long long)p.q_heads * p.dim;
    const long long at0 = ((long long)b * p.q_len + i0) * stride + (long long)h * p.dim + lane * 4;
    for (int r = 0; r < 32; r += 4) {
      if (((rows >> r) & 15u) == 0) continue;
      uint2 x[4], d[4], y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool load = mine && ((rows >> (r + k)) & 1u);
        const long long at = at0 + (r + k) * stride;
        x[k] = load ? __ldg(reinterpret_cast<const uint2*>(a.o_raw + at)) : make_uint2(0, 0);
        d[k] = load ? __ldg(reinterpret_cast<const uint2*>(a.do_raw + at)) : make_uint2(0, 0);
        y[k] = load && a.low_raw ? __ldg(reinterpret_cast<const uint2*>(a.low_raw + at)) : make_uint2(0, 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x0 = ptx::add2(unpack2<BF16>(x[k].x), unpack2<BF16>(y[k].x));
        const float2 x1 = ptx::add2(unpack2<BF16>(x[k].y), unpack2<BF16>(y[k].y));
        const float2 d0 = unpack2<BF16>(d[k].x), d1 = unpack2<BF16>(d[k].y);
        float delta = fmaf(x0.x, d0.x, fmaf(x0.y, d0.y, fmaf(x1.x, d1.x, x1.y * d1.y)));
        uint32_t peak = 0;
        if (!BF16)
          peak = __reduce_max_sync(~0u, __float_as_uint(fmaxf(fmaxf(fabsf(d0.x), fabsf(d0.y)), fmaxf(fabsf(d1.x), fabsf(d1.y)))));
#pragma unroll
        for (int o = 16; o; o >>= 1) delta += __shfl_xor_sync(~0u, delta, o);
        if (lane == r + k) {
          kept = delta;
          own_peak = __uint_as_float(peak);
        }
      }
    }
    float nl = -INFINITY;
    if (real) {
      const float ls = a.lse[((long long)b * p.q_heads + h) * p.q_len + own];
      if (ls > -INFINITY) nl = -ls * kLog2e + (BF16 ? 0.f : (float)kWeightShift);
      else own_peak = 0.f;      // sees nothing: no gradient passes it
    }
    const long long at = row_slot(p, b, h) + own;
    a.neg_lse[at] = nl;
    a.neg_delta[at] = -kept;
    if (!BF16) {
      a.row_peak[at] = own_peak;
      const float top = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(own_peak)));
      const float most = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(fabsf(kept))));
      if (lane == 0) a.query_peaks[at / 32] = make_float2(top, most);
    }
    return;
  }
  if (BF16) return;
  const int id = (int)blockIdx.x - g.q_blocks, groups = (p.k_heads + 7) / 8, chunks = tiles_of(p.k_len) * 4;
  const int h = id % groups * 8 + warp, i0 = id / groups % chunks * 32, b = id / groups / chunks;
  if (h >= p.k_heads) return;
  float peak = 0.f;
#pragma unroll 4
  for (int r = 0; r < 32; ++r) {
    const int j = i0 + r;
    if (j >= p.k_len || (p.documents && p.documents[(long long)b * p.k_len + j] < 0)) continue;     // the same for the warp
    uint2 x = make_uint2(0, 0);
    if (mine) x = __ldg(reinterpret_cast<const uint2*>(a.v_raw + b * p.v_stride[0] + j * p.v_stride[1] + h * p.v_stride[2] + lane * 4));
    const float2 x0 = unpack2<BF16>(x.x), x1 = unpack2<BF16>(x.y);
    float sum = (fabsf(x0.x) + fabsf(x0.y)) + (fabsf(x1.x) + fabsf(x1.y));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    peak = fmaxf(peak, sum);
  }
  if (lane == 0) a.key_peaks[((long long)b * p.k_heads + h) * chunks + i0 / 32] = peak;
}

// ---- shared by the two product kernels ---------------------------------------------------------

// A pair of raw scores -> weights x = 2^(z + nl) and what the score gradient is multiplied by,
// w = x (1 - tanh^2).  far: distances; NEAR: tanh_near does.
template <bool CAP, bool BIAS, bool NEAR>
__device__ __forceinline__ void weights(float2 s, float2 nl, const Scores& sc, float2 far, float2* x, float2* w) {
  float2 z;
  float2 bend = make_float2(1.f, 1.f);
  if (CAP) {
    const float by = 2.f * kLog2e * sc.to_u;
    const float2 t = NEAR ? tanh_near(ptx::mul2(s, make_float2(sc.to_u, sc.to_u)))
                          : make_float2(tanh_of(s.x * by), tanh_of(s.y * by));
    z = ptx::fma2(t, make_float2(sc.cap_by, sc.cap_by), nl);
    bend = ptx::fma2(make_float2(-t.x, -t.y), t, bend);
  } else {
    z = ptx::fma2(s, make_float2(sc.by, sc.by), nl);
  }
  if (BIAS) z = ptx::fma2(make_float2(-sc.slope, -sc.slope), far, z);
  *x = make_float2(ex2(z.x), ex2(z.y));
  *w = CAP ? ptx::mul2(*x, bend) : *x;
}

// 16-bit rows of 32 lanes x DP columns of TMEM, times `by`, staged and stored by TMA.
template <int DP, bool BF16>
__device__ __forceinline__ void store_rows(const CUtensorMap* map, uint32_t tmem, bool any, float by, uint8_t* stage,
                                           int row0, int head, int b, int lane) {
#pragma unroll
  for (int c = 0; c < DP; c += 32) {
    uint32_t o[32];
    if (any) {
      ptx::tmem_ld_32x32(tmem + c, o);
      ptx::tmem_ld_wait();
    }
    uint8_t* dst = stage + (c >> 6) * kBoxBytes + lane * 128;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = any ? pack2<BF16>(__uint_as_float(o[8 * i + 2 * k]) * by, __uint_as_float(o[8 * i + 2 * k + 1]) * by) : 0u;
      *reinterpret_cast<uint4*>(dst + (((((c & 32) >> 3) + i) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  ptx::fence_proxy_async();
  __syncwarp();
  if (lane == 0) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
      const int32_t at[5] = {c * 64, row0, head, b, 0};
      ptx::tma_store_nd(4, map, at, ptx::smem_u32(stage) + c * kBoxBytes);
    }
    ptx::bulk_commit_group();
    ptx::bulk_wait_group_read<0>();
  }
}

// The same rows in 32 bits, to the workspace.
template <int DP>
__device__ __forceinline__ void keep_rows(float* to, uint32_t tmem, bool any, float by, int lane) {
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    uint32_t o[32];
    if (any) {
      ptx::tmem_ld_32x32(tmem + c, o);
      ptx::tmem_ld_wait();
    }
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<float4*>(to + lane * DP + c + i) =
          any ? make_float4(__uint_as_float(o[i]) * by, __uint_as_float(o[i + 1]) * by, __uint_as_float(o[i + 2]) * by,
                            __uint_as_float(o[i + 3]) * by)
              : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// The pieces of one result added up in order.  Tiles are numbered [tile][batch][head], `sums` of
// them side by side (dV, dK); a thread takes four values of a row.
template <int DP, bool BF16>
__global__ void __launch_bounds__(256) attn_add_kernel(const float* part, int pieces, int sums, int batch, int heads, int len,
                                                       int dim, bool reversed, uint16_t* out0, uint16_t* out1) {
  ptx::grid_dependency_wait();
  const long long tiles = (long long)tiles_of(len) * batch * heads * sums, per = tiles * kTile * (DP / 4);
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= per) return;
  const int c = (int)(id % (DP / 4)) * 4, r = (int)(id / (DP / 4) % kTile);
  const long long slot = id / (DP / 4) / kTile;
  const int which = (int)(slot % sums);
  const long long cta = slot / sums;
  const int h = (int)(cta % heads), b = (int)(cta / heads % batch), n = (int)(cta / heads / batch);
  const int row = (reversed ? tiles_of(len) - 1 - n : n) * kTile + r;
  if (row >= len || c >= dim) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int x = 0; x < pieces; ++x) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(part) + per * x + id);
    sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
  }
  uint16_t* out = which ? out1 : out0;
  *reinterpret_cast<uint2*>(out + (((long long)b * len + row) * heads + h) * dim + c) =
      make_uint2(pack2<BF16>(sum.x, sum.y), pack2<BF16>(sum.z, sum.w));
}

// What the rounding of a pair to 16 bits left.
template <bool BF16>
__device__ __forceinline__ uint32_t rest_of(float2 x, uint32_t packed) {
  const float2 y = unpack2<BF16>(packed);
  return pack2<BF16>(x.x - y.x, x.y - y.y);
}

// TMEM column of 16 tokens' packed pairs: a warpgroup's half of the columns lies over the
// scores that this warpgroup has read, the first half at 0, the second at 64.
__device__ __forceinline__ uint32_t packed_at(int step) { return (step < 4 ? 0 : 64) + (step & 3) * 8; }

// ---- dK, dV --------------------------------------------------------------------------------------

template <int DP> constexpr int key_stages() { return DP == 128 ? 2 : 4; }
template <int DP> constexpr int key_smem() {
  return (2 + 2 * key_stages<DP>()) * tile_bytes<DP>() + key_stages<DP>() * kStats * 4 + 1024 + 512;
}

struct KeyShared {
  uint64_t kv_full[2], s_full, p_full, dp_full, ds_full, acc_full;
  uint64_t q_full[4], q_empty[4], do_full[4], do_empty[4];
  int lo, hi;
  uint32_t tmem_base, abort_flag;
};

template <int DP, bool BF16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1) attn_bwd_keys_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int TILE = tile_bytes<DP>(), NS = key_stages<DP>();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  // K, V, ring of Q, ring of dO, ring of the rows' (-lse, -delta, peaks)
  float* stats = reinterpret_cast<float*>(smem + (2 + 2 * NS) * TILE);
  KeyShared* sh = reinterpret_cast<KeyShared*>(smem + (2 + 2 * NS) * TILE + NS * kStats * 4);
  volatile uint32_t* abort_flag = &sh->abort_flag;
  const uint32_t k_smem = ptx::smem_u32(smem), v_smem = k_smem + TILE, q_smem = v_smem + TILE, do_smem = q_smem + NS * TILE;
  const AttnProblem& p = a.p;

  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int heads = p.batch * p.k_heads;
  const int piece = a.key_pieces > 1 ? (int)(blockIdx.x % a.key_pieces) : 0;
  const int cta = a.key_pieces > 1 ? (int)(blockIdx.x / a.key_pieces) : (int)blockIdx.x;
  const int kt = cta / heads;      // the first keys, which most queries see, come first
  const int b = cta % heads / p.k_heads, hk = cta % heads % p.k_heads;
  const int j0 = kt * kTile;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) ptx::mbar_init(ptx::smem_u32(&sh->kv_full[t]), 1);
    ptx::mbar_init(ptx::smem_u32(&sh->s_full), 1);
    ptx::mbar_init(ptx::smem_u32(&sh->p_full), 8);
    ptx::mbar_init(ptx::smem_u32(&sh->dp_full), 1);
    ptx::mbar_init(ptx::smem_u32(&sh->ds_full), 8);
    ptx::mbar_init(ptx::smem_u32(&sh->acc_full), 1);
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->q_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->q_empty[s]), 1 + 8);    // the MMAs, and the warps done with the row sums
      ptx::mbar_init(ptx::smem_u32(&sh->do_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->do_empty[s]), 1);
    }
    sh->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&a.q);
    ptx::prefetch_tensormap(&a.k);
    ptx::prefetch_tensormap(&a.v);
    ptx::prefetch_tensormap(&a.d_o);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&sh->tmem_base), 512);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  const int prefix = prefix_of(p, b);
  if (warp == 0) {   // tiles of queries that see some key of the tile
    const int nq = tiles_of(p.q_len);
    int lo = 0, hi = nq;
    if (p.causal && j0 >= prefix) {      // from the query at position j0 on
      const int first = j0 - p.offset;
      lo = first <= 0 ? 0 : first >= p.q_len ? nq : first / kTile;
    }
    if (p.documents && lo < hi) {
      const int4 mine = p.key_docs[(long long)b * tiles_of(p.k_len) + kt];
      const int4* qd = p.query_docs + (long long)b * nq;
      int first = hi, last = -1;
      for (int i = lo + lane; i < hi; i += 32)
        if (docs_meet(qd[i], mine)) {
          if (i < first) first = i;
          last = i;
        }
      lo = __reduce_min_sync(~0u, first);
      hi = __reduce_max_sync(~0u, last) + 1;
    }
    if (lane == 0) {
      sh->lo = lo;
      sh->hi = hi > lo ? hi : lo;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ptx::uniform(sh->tmem_base);
  const uint32_t s_at = tmem, dp_at = tmem + kTile, dv_at = tmem + 2 * kTile, dk_at = dv_at + DP;
  const int lo = ptx::uniform(sh->lo), per_head = ptx::uniform(sh->hi) - lo, all_steps = per_head * p.group;
  const int step0 = (int)((long long)all_steps * piece / a.key_pieces);      // this CTA's steps
  const int steps = (int)((long long)all_steps * (piece + 1) / a.key_pieces) - step0;

  if (warp >= 8) {
    ptx::regs_less<kBwdOtherRegs>();
    if (warp == 8 && steps > 0) {
      // ---------------- loads ----------------
      bool ok = true;
      if (lane == 0)
        for (int t = 0; t < 2; ++t) {
          const uint32_t bar = ptx::smem_u32(&sh->kv_full[t]);
          ptx::mbar_arrive_expect_tx(bar, TILE);
          for (int c = 0; c < DP / 64; ++c) {
            const int32_t at[5] = {c * 64, j0, hk, b, 0};
            ptx::tma_load_nd(4, (t ? v_smem : k_smem) + c * kBoxBytes, t ? &a.v : &a.k, at, bar);
          }
        }
      const int4* qd = p.documents ? p.query_docs + (long long)b * tiles_of(p.q_len) : nullptr;
      int n = 0;
      for (; ok && n < steps; ++n) {
        const int h = hk * p.group + (step0 + n) / per_head, i = lo + (step0 + n) % per_head;
        const uint32_t slot = n % NS, parity = ((n / NS) & 1) ^ 1;
        const bool dirty = qd && qd[i].z;
        for (int g = 0; g < 2; ++g) {       // Q with the rows' sums, then dO
          const uint32_t full = ptx::smem_u32(g ? &sh->do_full[slot] : &sh->q_full[slot]);
          if (lane == 0)
            ok = ptx::mbar_wait_bounded(ptx::smem_u32(g ? &sh->do_empty[slot] : &sh->q_empty[slot]), parity, abort_flag, kAttnWait);
          ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
          if (!ok) {
            if (lane == 0) attn_fail(a.status, abort_flag, 0x510000u | slot);
            break;
          }
          const uint32_t tile = (g ? do_smem : q_smem) + slot * TILE;
          if (dirty) {     // padding among the queries must not meet a zero weight
            const uint16_t* base = g ? a.do_raw + ((long long)b * p.q_len * p.q_heads + h) * p.dim
                                     : a.q_raw + b * p.q_stride[0] + h * p.q_stride[2];
            copy_tile_clean<DP>(smem + (tile - k_smem), base, g ? (long long)p.q_heads * p.dim : p.q_stride[1], p.dim,
                                i * kTile, p.q_len, p.documents + (long long)b * p.k_len + p.offset, lane);
          }
          if (lane == 0) {
            const uint32_t bytes = (dirty ? 0 : TILE) + (g ? 0 : BF16 ? 1024 : 1024 + 32);
            if (bytes) ptx::mbar_arrive_expect_tx(full, bytes);
            else ptx::mbar_arrive(full);
            if (!dirty)
              for (int c = 0; c < DP / 64; ++c) {
                const int32_t at[5] = {c * 64, i * kTile, h, b, 0};
                ptx::tma_load_nd(4, tile + c * kBoxBytes, g ? &a.d_o : &a.q, at, full);
              }
            if (!g) {
              const long long at = row_slot(p, b, h) + i * kTile;
              ptx::bulk_load(ptx::smem_u32(stats + slot * kStats), a.neg_lse + at, 512, full);
              ptx::bulk_load(ptx::smem_u32(stats + slot * kStats + 128), a.neg_delta + at, 512, full);
              if (!BF16) ptx::bulk_load(ptx::smem_u32(stats + slot * kStats + 256), a.query_peaks + at / 32, 32, full);
            }
          }
        }
      }
      if (lane == 0 && *abort_flag) {   // leave no copy in flight
        uint32_t never = 0;
        for (int t = 0; t < 2; ++t) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->kv_full[t]), 0, &never, kAttnWait);
        for (int s = 0; s < NS; ++s)
          if (n > s) {
            ptx::mbar_wait_bounded(ptx::smem_u32(&sh->q_full[s]), ((n - 1 - s) / NS) & 1, &never, kAttnWait);
            ptx::mbar_wait_bounded(ptx::smem_u32(&sh->do_full[s]), ((n - 1 - s) / NS) & 1, &never, kAttnWait);
          }
      }
    } else if (warp == 9 && steps > 0) {
      // ---------------- MMA issue ----------------
      const uint32_t leader = ptx::elect_one();
      const uint32_t id_s = idesc_of<BF16>(kTile, false), id_d = idesc_of<BF16>(DP, true);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (ok && !__all_sync(~0u, ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait))) {
          if (leader) attn_fail(a.status, abort_flag, code);
          ok = false;
        }
        ptx::tc_fence_after();
      };
      auto score_product = [&](uint32_t d, uint32_t own, uint32_t other, uint64_t* bar) {
        const uint32_t a_low = low_k_major(own), b_low = low_k_major(other);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) ptx::mma_f16_ss_by(leader, d, desc_k_major(a_low, s), desc_k_major(b_low, s), id_s, s != 0);
        ptx::mma_commit_by(leader, ptx::smem_u32(bar));
      };
      auto sum_product = [&](uint32_t d, uint32_t w, uint32_t other, bool add, uint64_t* bar) {
        const uint32_t b_low = low_mn_major(other);
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s) ptx::mma_f16_ts_by(leader, d, w + packed_at(s), desc_mn_major(b_low, s), id_d, add || s != 0);
        ptx::mma_commit_by(leader, ptx::smem_u32(bar));
      };
      wait(&sh->kv_full[0], 0, 0x520000u);
      wait(&sh->q_full[0], 0, 0x520001u);
      if (ok) score_product(s_at, k_smem, q_smem, &sh->s_full);
      wait(&sh->kv_full[1], 0, 0x520002u);
      wait(&sh->do_full[0], 0, 0x520003u);
      if (ok) score_product(dp_at, v_smem, do_smem, &sh->dp_full);
      uint32_t slot = 0, parity = 0;
      for (int n = 0; ok && n < steps; ++n) {
        const uint32_t next = slot + 1 == NS ? 0 : slot + 1, next_parity = slot + 1 == NS ? parity ^ 1 : parity;
        const bool more = n + 1 < steps;
        wait(&sh->p_full, n & 1, 0x530000u);
        if (!ok) break;
        sum_product(dv_at, s_at, do_smem + slot * TILE, n != 0, &sh->do_empty[slot]);
        if (more) {
          wait(&sh->q_full[next], next_parity, 0x530001u);
          if (!ok) break;
          score_product(s_at, k_smem, q_smem + next * TILE, &sh->s_full);
        }
        wait(&sh->ds_full, n & 1, 0x530002u);
        if (!ok) break;
        sum_product(dk_at, dp_at, q_smem + slot * TILE, n != 0, &sh->q_empty[slot]);
        if (more) {
          wait(&sh->do_full[next], next_parity, 0x530003u);
          if (!ok) break;
          score_product(dp_at, v_smem, do_smem + next * TILE, &sh->dp_full);
        }
        slot = next;
        parity = next_parity;
      }
      if (ok) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->acc_full));
    }
  } else {
    ptx::regs_more<kMathRegs>();
    // ---------------- weights and score gradients, epilogue ----------------
    const int half = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = s_at + lanes + half * 64, dp_tmem = dp_at + lanes + half * 64;
    const int key = j0 + quarter * 32 + lane;
    // fp16: log2 of the factor on dS, and the smallest so far
    int factor = 0, least = 1000;
    const float key_peak = BF16 ? 0.f : max_of4(reinterpret_cast<const float4*>(a.key_peaks)[((long long)b * p.k_heads + hk) * tiles_of(p.k_len) + kt]);
    int own_doc = -1;
    int4 tile_docs = make_int4(0, 0, 0, 0);
    const int* docs = nullptr;      // of query 0 on
    const int4* qd = nullptr;
    if (p.documents && steps > 0) {
      docs = p.documents + (long long)b * p.k_len + p.offset;
      qd = p.query_docs + (long long)b * tiles_of(p.q_len);
      if (key < p.k_len) own_doc = p.documents[(long long)b * p.k_len + key];
      tile_docs = p.key_docs[(long long)b * tiles_of(p.k_len) + kt];
    }
    const bool behind = !p.causal || key < prefix;       // seen from every position
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait)) ok = false;
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(a.status, abort_flag, code);
        ok = false;
      }
      ptx::tc_fence_after();
      return ok;
    };
    for (int n = 0; n < steps; ++n) {
      const int h = hk * p.group + (step0 + n) / per_head, i = lo + (step0 + n) % per_head, i0 = i * kTile;
      const uint32_t slot = n % NS;
      const Scores sc = scores_of<CAP>(p.scale, p.softcap, p.slopes, h);
      // seen whole: the first query sees the last key (queries past the end have weight zero)
      bool masked = p.causal && last_key(p, prefix, i0 + p.offset) < j0 + kTile - 1;
      if (qd) masked = masked || !docs_same(qd[i], tile_docs);
      const float4* nl4 = reinterpret_cast<const float4*>(stats + slot * kStats + half * 64);
      const float4* nd4 = nl4 + 32;
      // the row sums arrive with Q, before the scores made from it
      if (!wait(&sh->q_full[slot], (n / NS) & 1, 0x540000u) || !wait(&sh->s_full, n & 1, 0x540001u)) break;
      float w[64];
#pragma unroll
      for (int c = 0; c < 64; c += 32) ptx::tmem_ld_32x32(s_tmem + c, reinterpret_cast<uint32_t*>(w) + c);
      ptx::tmem_ld_wait();
      uint32_t see[2] = {~0u, ~0u};
      if (masked) {
        if (!behind) {
          const int first = key - p.offset - i0 - half * 64;      // column of the first query at the key's position or past it
          see[0] = ~bits_upto(first - 1, 0);
          see[1] = ~bits_upto(first - 1, 1);
        }
        if (docs) {
          int other[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int i = i0 + half * 64 + x * 32 + lane;
            other[x] = i < p.q_len ? docs[i] : -1;
          }
          mask_documents(see, other, own_doc);
        }
      }
      auto weigh = [&](auto near_tag) {
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 nl = nl4[(c + e) >> 2];
          float2 far[2];
          if (BIAS) {
            const float d = (float)(i0 + half * 64 + c + e + p.offset - key);
            far[0] = make_float2(fabsf(d), fabsf(d + 1.f));
            far[1] = make_float2(fabsf(d + 2.f), fabsf(d + 3.f));
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int at = c + e + 2 * x;
            float2 px, pw;
            weights<CAP, BIAS, decltype(near_tag)::value>(make_float2(w[at], w[at + 1]), x ? make_float2(nl.z, nl.w) : make_float2(nl.x, nl.y), sc,
                               far[x], &px, &pw);
            if (masked) {
              if (!((see[at >> 5] >> (at & 31)) & 1u)) px.x = pw.x = 0.f;
              if (!((see[at >> 5] >> ((at + 1) & 31)) & 1u)) px.y = pw.y = 0.f;
            }
            packed[(e + 2 * x) >> 1] = pack2<BF16>(px.x, px.y);
            w[at] = pw.x;
            w[at + 1] = pw.y;
          }
        }
        ptx::tmem_st_32x16(s_tmem + c / 2, packed);
      }
      };
      if (CAP && all_near(w, sc.to_u)) weigh(std::true_type{});
      else weigh(std::false_type{});
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->p_full));

      const int before = factor;
      if (!BF16) {
        const float4* peaks = reinterpret_cast<const float4*>(stats + slot * kStats + 256);
        const float4 x = peaks[0], y = peaks[1];
        int best;
        if (factor_log2(fmaxf(fmaxf(x.x, x.z), fmaxf(y.x, y.z)) * key_peak + fmaxf(fmaxf(x.y, x.w), fmaxf(y.y, y.w)), &best)) {
          // Steps whose bounds differ little share a factor: one that leaves the bound at 2^11 or more and below
          // 2^15 stays.  None is more than 2^48 times the smallest, so the sums, 2^51 at that one, stay in range.
          if (least == 1000 || factor > best || factor < best - 3) factor = best - 1;
          factor = factor < least + 48 ? factor : least + 48;
          least = factor < least ? factor : least;
        }
      }
      const float w_by = BF16 ? 1.f : power_of_two(factor - kWeightShift);
      if (!wait(&sh->dp_full, n & 1, 0x540002u)) break;
      if (!BF16 && n > 0 && factor != before) {      // dP came after dK's last product, and the next one waits for this dS
        const float by = power_of_two(factor - before);
#pragma unroll 1
        for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {
          uint32_t o[16];
          ptx::tmem_ld_32x16(dk_at + lanes + c, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
          ptx::tmem_st_32x16(dk_at + lanes + c, o);
        }
      }
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        float d[32];
        ptx::tmem_ld_32x32(dp_tmem + c, reinterpret_cast<uint32_t*>(d));
        ptx::tmem_ld_wait();
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 nd = nd4[(c + e) >> 2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int at = c + e + 2 * x;
            float2 f = make_float2(w[at], w[at + 1]);
            if (!BF16) f = ptx::mul2(f, make_float2(w_by, w_by));
            float2 g = ptx::add2(make_float2(d[e + 2 * x], d[e + 2 * x + 1]), x ? make_float2(nd.z, nd.w) : make_float2(nd.x, nd.y));
            g = ptx::mul2(f, g);
            if (masked) {     // not 0 * infinity
              if (!((see[at >> 5] >> (at & 31)) & 1u)) g.x = 0.f;
              if (!((see[at >> 5] >> ((at + 1) & 31)) & 1u)) g.y = 0.f;
            }
            packed[(e + 2 * x) >> 1] = pack2<BF16>(g.x, g.y);
          }
        }
        // over the columns this warp has read: 0 .. 15 first, then 16 .. 31 of its half
        ptx::tmem_st_32x16(dp_tmem + c / 2, packed);
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(ptx::smem_u32(&sh->ds_full));
        ptx::mbar_arrive(ptx::smem_u32(&sh->q_empty[slot]));    // done with the row sums
      }
    }
    if (ok && steps > 0) wait(&sh->acc_full, 0, 0x550000u);
    const int row0 = j0 + quarter * 32;
    const float dv_by = BF16 ? 1.f : ldexpf(1.f, -kWeightShift), dk_by = p.scale * power_of_two(-factor);
    if (ok && a.key_pieces > 1) {
      const long long slot = ((long long)piece * (gridDim.x / a.key_pieces) + cta) * 2 + half;
      keep_rows<DP>(a.key_part + (slot * kTile + quarter * 32) * DP, (half ? dk_at : dv_at) + lanes, steps > 0,
                    half ? dk_by : dv_by, lane);
    } else if (ok && row0 < p.k_len) {      // staged where K and V were
      if (half == 0)
        store_rows<DP, BF16>(&a.dv, dv_at + lanes, steps > 0, dv_by,
                             smem + TILE + quarter * 4096, row0, hk, b, lane);
      else
        store_rows<DP, BF16>(&a.dk, dk_at + lanes, steps > 0, dk_by, smem + quarter * 4096, row0, hk, b, lane);
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- dQ --------------------------------------------------------------------------------------------

template <int DP> constexpr int query_k_stages() { return DP == 128 ? 3 : 4; }
template <int DP> constexpr int query_v_stages() { return DP == 128 ? 2 : 3; }
template <int DP> constexpr int query_smem() {
  return (2 + query_k_stages<DP>() + query_v_stages<DP>()) * tile_bytes<DP>() + 1024 + 512;
}

struct QueryShared {
  uint64_t q_full[2], s_full[2], dp_full, ds_full, acc_full;
  uint64_t k_full[4], k_empty[4], v_full[3], v_empty[3];
  int lo, hi;
  uint32_t tmem_base, abort_flag;
};

template <int DP, bool BF16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1) attn_bwd_queries_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int TILE = tile_bytes<DP>(), NK = query_k_stages<DP>(), NV = query_v_stages<DP>();
  // dS in 16 bits makes dQ's error 1.41 to 1.66 times that of its own rounding, little as scores differ (deviations
  // of 0.3 to 8, capped or not); with what the rounding left as a product of its own it is 1.02 to 1.24 times.
  // Under a cap the warps' arithmetic bounds this kernel and the tensor pipe waits: there the product costs 3 %
  // (8192 causal tokens x 16 heads of 64 backward 1120 -> 1160 us) and is taken; without a cap the pipe is in
  // its way and it costs 13 % (2 x 4096 causal tokens x 32/8 heads of 128 970 -> 1100 us).
  constexpr bool REST = CAP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  QueryShared* sh = reinterpret_cast<QueryShared*>(smem + (2 + NK + NV) * TILE);
  volatile uint32_t* abort_flag = &sh->abort_flag;
  const uint32_t q_smem = ptx::smem_u32(smem), do_smem = q_smem + TILE, k_smem = do_smem + TILE, v_smem = k_smem + NK * TILE;
  const AttnProblem& p = a.p;

  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int heads = p.batch * p.q_heads;
  const int piece = a.query_pieces > 1 ? (int)(blockIdx.x % a.query_pieces) : 0;
  const int cta = a.query_pieces > 1 ? (int)(blockIdx.x / a.query_pieces) : (int)blockIdx.x;
  const int qt = tiles_of(p.q_len) - 1 - cta / heads;
  const int b = cta % heads / p.q_heads, h = cta % heads % p.q_heads, hk = h / p.group;
  const int q0 = qt * kTile;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(&sh->q_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->s_full[t]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&sh->dp_full), 1);
    ptx::mbar_init(ptx::smem_u32(&sh->ds_full), 8);
    ptx::mbar_init(ptx::smem_u32(&sh->acc_full), 1);
    for (int s = 0; s < NK; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->k_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->k_empty[s]), 1);
    }
    for (int s = 0; s < NV; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->v_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->v_empty[s]), 1);
    }
    sh->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&a.q);
    ptx::prefetch_tensormap(&a.k);
    ptx::prefetch_tensormap(&a.v);
    ptx::prefetch_tensormap(&a.d_o);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&sh->tmem_base), 512);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  const int prefix = prefix_of(p, b);
  const int4* kd = p.documents ? p.key_docs + (long long)b * tiles_of(p.k_len) : nullptr;
  if (warp == 0) {
    const int last_row = q0 + kTile - 1 < p.q_len - 1 ? q0 + kTile - 1 : p.q_len - 1;
    int lo = 0, hi = tiles_of(last_key(p, prefix, last_row + p.offset) + 1);
    if (hi < 0) hi = 0;
    if (kd) {
      const int4 mine = p.query_docs[(long long)b * tiles_of(p.q_len) + qt];
      int first = hi, last = -1;
      for (int j = lane; j < hi; j += 32)
        if (docs_meet(kd[j], mine)) {
          if (j < first) first = j;
          last = j;
        }
      lo = __reduce_min_sync(~0u, first);
      hi = __reduce_max_sync(~0u, last) + 1;
    }
    if (lane == 0) {
      sh->lo = lo;
      sh->hi = hi > lo ? hi : lo;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ptx::uniform(sh->tmem_base);
  const uint32_t s_at = tmem, dp_at = tmem + 2 * kTile, dq_at = tmem + 3 * kTile;
  const int lo_all = ptx::uniform(sh->lo), all_steps = ptx::uniform(sh->hi) - lo_all;
  const int lo = lo_all + (int)((long long)all_steps * piece / a.query_pieces);      // this CTA's tiles
  const int steps = lo_all + (int)((long long)all_steps * (piece + 1) / a.query_pieces) - lo;

  if (warp >= 8) {
    ptx::regs_less<kBwdOtherRegs>();
    if (warp == 8 && steps > 0) {
      // ---------------- loads ----------------
      bool ok = true;
      if (lane == 0)
        for (int t = 0; t < 2; ++t) {
          const uint32_t bar = ptx::smem_u32(&sh->q_full[t]);
          ptx::mbar_arrive_expect_tx(bar, TILE);
          for (int c = 0; c < DP / 64; ++c) {
            const int32_t at[5] = {c * 64, q0, h, b, 0};
            ptx::tma_load_nd(4, (t ? do_smem : q_smem) + c * kBoxBytes, t ? &a.d_o : &a.q, at, bar);
          }
        }
      int n = 0;
      for (; ok && n < steps; ++n) {
        const int j = lo + n;
        for (int g = 0; g < 2; ++g) {
          const uint32_t slot = n % (g ? NV : NK), parity = ((n / (g ? NV : NK)) & 1) ^ 1;
          const uint32_t full = ptx::smem_u32(g ? &sh->v_full[slot] : &sh->k_full[slot]);
          if (lane == 0)
            ok = ptx::mbar_wait_bounded(ptx::smem_u32(g ? &sh->v_empty[slot] : &sh->k_empty[slot]), parity, abort_flag, kAttnWait);
          ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
          if (!ok) {
            if (lane == 0) attn_fail(a.status, abort_flag, 0x610000u | slot);
            break;
          }
          if (!g && kd && kd[j].z) {   // padding among the keys must not meet a zero score gradient
            copy_tile_clean<DP>(smem + (2 + slot) * TILE, a.k_raw + b * p.k_stride[0] + hk * p.k_stride[2], p.k_stride[1],
                                p.dim, j * kTile, p.k_len, p.documents + (long long)b * p.k_len, lane);
            if (lane == 0) ptx::mbar_arrive(full);
          } else if (lane == 0) {
            ptx::mbar_arrive_expect_tx(full, TILE);
            for (int c = 0; c < DP / 64; ++c) {
              const int32_t at[5] = {c * 64, j * kTile, hk, b, 0};
              ptx::tma_load_nd(4, (g ? v_smem : k_smem) + slot * TILE + c * kBoxBytes, g ? &a.v : &a.k, at, full);
            }
          }
        }
      }
      if (lane == 0 && *abort_flag) {   // leave no copy in flight
        uint32_t never = 0;
        for (int t = 0; t < 2; ++t) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->q_full[t]), 0, &never, kAttnWait);
        for (int s = 0; s < NK; ++s)
          if (n > s) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->k_full[s]), ((n - 1 - s) / NK) & 1, &never, kAttnWait);
        for (int s = 0; s < NV; ++s)
          if (n > s) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->v_full[s]), ((n - 1 - s) / NV) & 1, &never, kAttnWait);
      }
    } else if (warp == 9 && steps > 0) {
      // ---------------- MMA issue ----------------
      const uint32_t leader = ptx::elect_one();
      const uint32_t id_s = idesc_of<BF16>(kTile, false), id_d = idesc_of<BF16>(DP, true);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (ok && !__all_sync(~0u, ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait))) {
          if (leader) attn_fail(a.status, abort_flag, code);
          ok = false;
        }
        ptx::tc_fence_after();
      };
      uint32_t k_slot = 0, k_parity = 0, v_slot = 0, v_parity = 0;      // of the next K, V
      auto score = [&](int n) {        // S(n) = Q K(n)
        if (n >= steps) return;
        wait(&sh->k_full[k_slot], k_parity, 0x620000u);
        if (!ok) return;
        const uint32_t a_low = low_k_major(q_smem), b_low = low_k_major(k_smem + k_slot * TILE);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          ptx::mma_f16_ss_by(leader, s_at + (n & 1) * kTile, desc_k_major(a_low, s), desc_k_major(b_low, s), id_s, s != 0);
        ptx::mma_commit_by(leader, ptx::smem_u32(&sh->s_full[n & 1]));
        if (++k_slot == NK) {
          k_slot = 0;
          k_parity ^= 1;
        }
      };
      auto grad = [&](int n) {         // dP(n) = dO V(n)
        if (n >= steps) return;
        wait(&sh->v_full[v_slot], v_parity, 0x620001u);
        if (!ok) return;
        const uint32_t a_low = low_k_major(do_smem), b_low = low_k_major(v_smem + v_slot * TILE);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          ptx::mma_f16_ss_by(leader, dp_at, desc_k_major(a_low, s), desc_k_major(b_low, s), id_s, s != 0);
        ptx::mma_commit_by(leader, ptx::smem_u32(&sh->dp_full));
        ptx::mma_commit_by(leader, ptx::smem_u32(&sh->v_empty[v_slot]));
        if (++v_slot == NV) {
          v_slot = 0;
          v_parity ^= 1;
        }
      };
      wait(&sh->q_full[0], 0, 0x620002u);
      if (ok) score(0);
      wait(&sh->q_full[1], 0, 0x620003u);
      if (ok) grad(0);
      if (ok) score(1);
      uint32_t slot = 0;               // of K(n)
      for (int n = 0; ok && n < steps; ++n) {
        wait(&sh->ds_full, n & 1, 0x630000u);
        if (!ok) break;
        const uint32_t b_low = low_mn_major(k_smem + slot * TILE);
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          ptx::mma_f16_ts_by(leader, dq_at, dp_at + packed_at(s), desc_mn_major(b_low, s), id_d, n != 0 || s != 0);
        if (REST) {
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            ptx::mma_f16_ts_by(leader, dq_at, dp_at + packed_at(s) + 32, desc_mn_major(b_low, s), id_d, true);
        }
        ptx::mma_commit_by(leader, ptx::smem_u32(&sh->k_empty[slot]));
        if (++slot == NK) slot = 0;
        grad(n + 1);
        if (ok) score(n + 2);
      }
      if (ok) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->acc_full));
    }
  } else {
    ptx::regs_more<kMathRegs>();
    // ---------------- score gradients, epilogue ----------------
    const int half = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t dp_tmem = dp_at + lanes + half * 64;
    const int row = q0 + quarter * 32 + lane, pos = row + p.offset;
    const int last = last_key(p, prefix, pos), last_first = last_key(p, prefix, q0 + p.offset);
    const Scores sc = scores_of<CAP>(p.scale, p.softcap, p.slopes, h);
    const long long slot = row_slot(p, b, h) + row;
    const float nl = a.neg_lse[slot], nd = a.neg_delta[slot];
    int factor = 0;        // fp16: log2 of the factor on the row's dS
    if (!BF16) {
      const float4* peaks = reinterpret_cast<const float4*>(a.key_peaks) + ((long long)b * p.k_heads + hk) * tiles_of(p.k_len) + lo;
      float peak = 0.f;
#pragma unroll 4
      for (int j = lane; j < steps; j += 32) peak = fmaxf(peak, max_of4(peaks[j]));
      peak = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(peak)));
      factor_log2(fmaf(a.row_peak[slot], peak, fabsf(nd)), &factor);
    }
    const float w_by = BF16 ? 1.f : power_of_two(factor - kWeightShift), dq_by = p.scale * power_of_two(-factor);
    const float2 nl2 = make_float2(nl, nl), nd2 = make_float2(nd, nd);
    int own_doc = -1;
    int4 tile_docs = make_int4(0, 0, 0, 0);
    const int* docs = nullptr;
    if (kd && steps > 0) {
      docs = p.documents + (long long)b * p.k_len;
      if (row < p.q_len) own_doc = docs[pos];
      tile_docs = p.query_docs[(long long)b * tiles_of(p.q_len) + qt];
    }
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait)) ok = false;
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(a.status, abort_flag, code);
        ok = false;
      }
      ptx::tc_fence_after();
      return ok;
    };
    for (int n = 0; n < steps; ++n) {
      const int j0 = (lo + n) * kTile;
      bool masked = j0 + kTile - 1 > last_first;
      if (kd) masked = masked || !docs_same(kd[lo + n], tile_docs);
      if (!wait(&sh->s_full[n & 1], (n >> 1) & 1, 0x640000u)) break;
      const uint32_t s_tmem = s_at + lanes + (n & 1) * kTile + half * 64;
      float w[64];
#pragma unroll
      for (int c = 0; c < 64; c += 32) ptx::tmem_ld_32x32(s_tmem + c, reinterpret_cast<uint32_t*>(w) + c);
      ptx::tmem_ld_wait();
      auto weigh = [&](auto near_tag) {
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        float2 far, px, pw;
        if (BIAS) {
          const float d = (float)(pos - j0 - half * 64 - c);
          far = make_float2(fabsf(d), fabsf(d - 1.f));
        }
        weights<CAP, BIAS, decltype(near_tag)::value>(make_float2(w[c], w[c + 1]), nl2, sc, far, &px, &pw);
        if (!BF16) pw = ptx::mul2(pw, make_float2(w_by, w_by));
        w[c] = pw.x;
        w[c + 1] = pw.y;
      }
      };
      if (CAP && all_near(w, sc.to_u)) weigh(std::true_type{});
      else weigh(std::false_type{});
      uint32_t see[2] = {~0u, ~0u};
      if (masked) {
        see[0] = bits_upto(last - j0 - half * 64, 0);
        see[1] = bits_upto(last - j0 - half * 64, 1);
        if (docs) {
          int other[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = j0 + half * 64 + x * 32 + lane;
            other[x] = j < p.k_len ? docs[j] : -1;
          }
          mask_documents(see, other, own_doc);
        }
      }
      if (!wait(&sh->dp_full, n & 1, 0x640001u)) break;
      uint32_t rest[REST ? 2 : 1][16];
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        float d[32];
        ptx::tmem_ld_32x32(dp_tmem + c, reinterpret_cast<uint32_t*>(d));
        ptx::tmem_ld_wait();
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const int at = c + e;
          float2 g = ptx::add2(make_float2(d[e], d[e + 1]), nd2);
          g = ptx::mul2(make_float2(w[at], w[at + 1]), g);
          if (masked) {
            if (!((see[at >> 5] >> (at & 31)) & 1u)) g.x = 0.f;
            if (!((see[at >> 5] >> ((at + 1) & 31)) & 1u)) g.y = 0.f;
          }
          packed[e >> 1] = pack2<BF16>(g.x, g.y);
          if (REST) rest[c >> 5][e >> 1] = rest_of<BF16>(g, packed[e >> 1]);
        }
        ptx::tmem_st_32x16(dp_tmem + c / 2, packed);
      }
      if (REST) {     // over columns that have been read by now
        ptx::tmem_st_32x16(dp_tmem + 32, rest[0]);
        ptx::tmem_st_32x16(dp_tmem + 48, rest[REST ? 1 : 0]);
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->ds_full));
    }
    if (ok && steps > 0) wait(&sh->acc_full, 0, 0x650000u);
    const int row0 = q0 + quarter * 32;
    if (ok && half == 0 && a.query_pieces > 1) {
      const long long slot = (long long)piece * (gridDim.x / a.query_pieces) + cta;
      keep_rows<DP>(a.query_part + (slot * kTile + quarter * 32) * DP, dq_at + lanes, steps > 0, dq_by, lane);
    } else if (ok && half == 0 && row0 < p.q_len)      // staged where Q was
      store_rows<DP, BF16>(&a.dq, dq_at + lanes, steps > 0, dq_by, smem + quarter * 4096, row0, h, b, lane);
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- launches ----------------------------------------------------------------------------------------

template <int DP, bool BF16, bool CAP, bool BIAS>
int32_t launch_bwd(const BwdArgs& a, int device, cudaStream_t s) {
  static PerDeviceFlag ready;
  auto keys = attn_bwd_keys_kernel<DP, BF16, CAP, BIAS>;
  auto queries = attn_bwd_queries_kernel<DP, BF16, CAP, BIAS>;
  if (!ready.test(device)) {
    LEGO_CUDA_TRY(cudaFuncSetAttribute(keys, cudaFuncAttributeMaxDynamicSharedMemorySize, key_smem<DP>()));
    LEGO_CUDA_TRY(cudaFuncSetAttribute(queries, cudaFuncAttributeMaxDynamicSharedMemorySize, query_smem<DP>()));
    ready.set(device);
  }
  const long long key_ctas = (long long)tiles_of(a.p.k_len) * a.p.batch * a.p.k_heads;
  const long long query_ctas = (long long)tiles_of(a.p.q_len) * a.p.batch * a.p.q_heads;
  if (key_ctas > 0x7fffffffLL || query_ctas > 0x7fffffffLL) return LEGO_ERR_SIZE;
  // (pieces are only made of calls with few CTAs: the products below stay small)
  auto add = [&](const float* part, int pieces, int sums, long long ctas, int heads, int len, bool reversed, uint16_t* o0, uint16_t* o1) {
    const long long blocks = (ctas * sums * kTile * (DP / 4) + 255) / 256;
    return launch_overlapped(attn_add_kernel<DP, BF16>, dim3((unsigned)blocks), dim3(256), 0, s, part, pieces, sums, a.p.batch,
                             heads, len, a.p.dim, reversed, o0, o1);
  };
  LEGO_CUDA_TRY(launch_overlapped(keys, dim3((unsigned)(key_ctas * a.key_pieces)), dim3(kBwdThreads), key_smem<DP>(), s, a));
  if (a.key_pieces > 1)
    LEGO_CUDA_TRY(add(a.key_part, a.key_pieces, 2, key_ctas, a.p.k_heads, a.p.k_len, false, a.dv_raw, a.dk_raw));
  LEGO_CUDA_TRY(launch_overlapped(queries, dim3((unsigned)(query_ctas * a.query_pieces)), dim3(kBwdThreads), query_smem<DP>(), s, a));
  if (a.query_pieces > 1)
    LEGO_CUDA_TRY(add(a.query_part, a.query_pieces, 1, query_ctas, a.p.q_heads, a.p.q_len, true, a.dq_raw, nullptr));
  return LEGO_OK;
}

template <int DP, bool BF16>
int32_t launch_bwd_scores(const BwdArgs& a, int device, cudaStream_t s) {
  const bool cap = a.p.softcap > 0.f, bias = a.p.slopes != nullptr;
  if (cap) return bias ? launch_bwd<DP, BF16, true, true>(a, device, s) : launch_bwd<DP, BF16, true, false>(a, device, s);
  return bias ? launch_bwd<DP, BF16, false, true>(a, device, s) : launch_bwd<DP, BF16, false, false>(a, device, s);
}

// Workspace of the backward pass: document summaries, row sums, peaks, the pieces' sums (those of dQ
// are written after those of dK, dV have been added up, and use their place).
struct BwdLayout {
  int64_t neg_lse, neg_delta, row_peak, query_peaks, key_peaks, part, bytes;
  int key_pieces, query_pieces;
};
BwdLayout bwd_layout(const AttnProblem& p, bool fp16) {
  BwdLayout l;
  const int64_t rows = (int64_t)p.batch * p.q_heads * tiles_of(p.q_len) * kTile;
  l.neg_lse = attention_docs_bytes(p);
  l.neg_delta = l.neg_lse + rows * 4;
  l.row_peak = l.neg_delta + rows * 4;
  l.query_peaks = l.row_peak + (fp16 ? rows * 4 : 0);
  l.key_peaks = l.query_peaks + (fp16 ? rows / 32 * 8 : 0);
  l.part = l.key_peaks + (fp16 ? (int64_t)p.batch * p.k_heads * tiles_of(p.k_len) * 16 : 0);
  const int64_t key_ctas = (int64_t)tiles_of(p.k_len) * p.batch * p.k_heads, query_ctas = (int64_t)tiles_of(p.q_len) * p.batch * p.q_heads;
  l.key_pieces = pieces_of(p, key_ctas, (int64_t)tiles_of(p.q_len) * p.group);
  l.query_pieces = pieces_of(p, query_ctas, tiles_of(p.k_len));
  const int64_t tile = (int64_t)kTile * (p.dim <= 64 ? 64 : 128) * 4;
  const int64_t keys = l.key_pieces > 1 ? key_ctas * l.key_pieces * 2 * tile : 0;
  const int64_t queries = l.query_pieces > 1 ? query_ctas * l.query_pieces * tile : 0;
  l.bytes = l.part + (keys > queries ? keys : queries);
  return l;
}

}  // namespace
}  // namespace lego

using namespace lego;

extern "C" {

int64_t lego_attention_workspace_bytes(const lego_attention_t* d, int32_t backward) {
  AttnProblem p;
  const int32_t st = attention_problem(d, &p);
  if (st != LEGO_OK) return st;
  return backward ? bwd_layout(p, d->dtype == LEGO_F16).bytes : attention_fwd_bytes(p);
}

int32_t lego_attention_bwd(const lego_attention_t* d, const void* q, const void* k, const void* v, const void* o,
                           const void* o_low, const float* lse, const void* d_o, void* dq, void* dk, void* dv,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  BwdArgs a = {};
  int32_t st = attention_problem(d, &a.p);
  if (st != LEGO_OK) return st;
  if (!q || !k || !v || !o || !lse || !d_o || !dq || !dk || !dv || !workspace) return LEGO_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)o_low | (uintptr_t)d_o | (uintptr_t)dq | (uintptr_t)dk |
       (uintptr_t)dv | (uintptr_t)workspace) & 15)
    return LEGO_ERR_ALIGN;
  const AttnProblem& p = a.p;
  const BwdLayout l = bwd_layout(p, d->dtype == LEGO_F16);
  if (workspace_bytes < l.bytes) return LEGO_ERR_SIZE;
  DeviceCtx* ctx = device_ctx(&st);
  if (!ctx) return st;
  EncodeFn enc = encode_fn(&st);
  if (!enc) return st;
  const bool bf16 = d->dtype == LEGO_BF16;
  const long long q_dense[3] = {(long long)p.q_len * p.q_heads * p.dim, (long long)p.q_heads * p.dim, p.dim};
  const long long k_dense[3] = {(long long)p.k_len * p.k_heads * p.dim, (long long)p.k_heads * p.dim, p.dim};
  if (make_tmap_heads(enc, &a.q, bf16, q, p.dim, p.q_len, p.q_heads, p.batch, p.q_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.k, bf16, k, p.dim, p.k_len, p.k_heads, p.batch, p.k_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.v, bf16, v, p.dim, p.k_len, p.k_heads, p.batch, p.v_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.d_o, bf16, d_o, p.dim, p.q_len, p.q_heads, p.batch, q_dense, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.dq, bf16, dq, p.dim, p.q_len, p.q_heads, p.batch, q_dense, 32) != LEGO_OK ||
      make_tmap_heads(enc, &a.dk, bf16, dk, p.dim, p.k_len, p.k_heads, p.batch, k_dense, 32) != LEGO_OK ||
      make_tmap_heads(enc, &a.dv, bf16, dv, p.dim, p.k_len, p.k_heads, p.batch, k_dense, 32) != LEGO_OK)
    return LEGO_ERR_UNSUPPORTED;
  cudaStream_t s = (cudaStream_t)stream;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.q_raw = (const uint16_t*)q;
  a.k_raw = (const uint16_t*)k;
  a.v_raw = (const uint16_t*)v;
  a.o_raw = (const uint16_t*)o;
  a.low_raw = (const uint16_t*)o_low;
  a.do_raw = (const uint16_t*)d_o;
  a.lse = lse;
  a.neg_lse = reinterpret_cast<float*>(ws + l.neg_lse);
  a.neg_delta = reinterpret_cast<float*>(ws + l.neg_delta);
  a.row_peak = reinterpret_cast<float*>(ws + l.row_peak);
  a.query_peaks = reinterpret_cast<float2*>(ws + l.query_peaks);
  a.key_peaks = reinterpret_cast<float*>(ws + l.key_peaks);
  a.key_pieces = l.key_pieces;
  a.query_pieces = l.query_pieces;
  a.key_part = a.query_part = reinterpret_cast<float*>(ws + l.part);
  a.dq_raw = (uint16_t*)dq;
  a.dk_raw = (uint16_t*)dk;
  a.dv_raw = (uint16_t*)dv;
  a.status = ctx->status_word;
  if ((int64_t)p.batch * (tiles_of(p.q_len) * 4LL * ((p.q_heads + 7) / 8) + tiles_of(p.k_len) * 4LL * ((p.k_heads + 7) / 8)) > 0x7fffffffLL)
    return LEGO_ERR_SIZE;
  const PrepGrid grid = prep_grid(p, !bf16);
  const int blocks = grid.q_blocks + grid.k_blocks;
  st = attention_docs(&a.p, workspace, s);
  if (st != LEGO_OK) return st;
  LEGO_CUDA_TRY(launch_overlapped(bf16 ? attn_bwd_prep_kernel<true> : attn_bwd_prep_kernel<false>, dim3((unsigned)blocks),
                                  dim3(256), 0, s, a));
  if (p.dim <= 64)
    return bf16 ? launch_bwd_scores<64, true>(a, ctx->device, s) : launch_bwd_scores<64, false>(a, ctx->device, s);
  return bf16 ? launch_bwd_scores<128, true>(a, ctx->device, s) : launch_bwd_scores<128, false>(a, ctx->device, s);
}

}  // extern "C"
