// Attention forward on tcgen05 (sm_100a): O = softmax(cap / bias / mask of scale Q K^T) V
// without the scores in memory.
//
// One CTA takes 256 queries of one head as two tiles of 128 rows and walks the tiles of 128
// keys that some of its rows see.  Per tile of scores: S = Q K^T into TMEM (both operands
// from shared memory), a warpgroup with one thread per row turns S into weights
// P = exp2(s - m) and writes them over S in TMEM as packed 16-bit pairs, and O += P V takes
// P from TMEM.  The two row tiles alternate: while one's scores are in its warpgroup, the
// tensor core works for the other.  Warps: 0-3 and 4-7 softmax of row tile 0 and 1 (and
// their epilogue), 8 TMA loads, 9 MMA issue (10 and 11 fill up their warpgroup).
//
// Few queries and many keys: the tiles of keys are cut into pieces, a CTA each; a piece leaves its
// sums in 32 bits and (m, sums) of its rows in the workspace, a second kernel joins them in the
// order of the keys.
//
// Running maximum: the reference value m of a row moves only when a tile's maximum outgrows it by more
// than 2^8 (fp16 2^4, its weights stand times 2^11: see attention.cuh), so O in TMEM is rarely rescaled;
// the row sums are kept in 32 bits.  The rounding of the weights to 16 bits, half a step of the type
// each, and the one of the result are the only ones below 32 bits.  What the last one takes
// away goes to a second output where the caller wants it: the backward pass subtracts dO O
// from terms of nearly the same size wherever a row has one large weight.
//
// Tiles no row of the CTA sees are not loaded (causal and prefix limits, document ranges);
// the mask is evaluated only on tiles that are not seen whole, as 128 bits per row.
//
// What bounds it: the way of a row tile from scores to weights to the product.  The tensor pipe and the
// exponentials' unit are each 63 % busy (4 x 4096 tokens, 16/4 heads of 128, no mask), and two row tiles are what TMEM
// and the registers hold.  Heads of 64 have half the products for the same exponentials: 28 % and 57 % (2 x 4096
// causal tokens, 16 heads); under a cap 15 % and 30 %, issue slots 46 %, so there it is the length of a warp's way, a
// polynomial of 9 instructions on a pair of scores in it, with two such warps per scheduler.  From a cold L2: 16384
// causal tokens x 8 heads of 128, bf16 465 us (1.18 PFLOP/s; 417 us, 1.32, where K and V are in L2); 2 x 4096
// causal x 32/8 heads 272 us (1.01); 8192 causal x 16 heads of 64, fp16 219 us (0.63), with a cap 426 us.  (The capped
// instances without a bias spill 2 to 6 registers.)  Slower, 16384 x 16384 x 8 heads, PFLOP/s where this form had 1.21:
// steps of 64 keys 0.72, two issuing threads 0.83, four softmax warpgroups 1.11, K and V released together 1.18.
#include <cuda.h>

#include "attention.cuh"
#include "tma_host.cuh"

namespace lego {
namespace {

constexpr int kFwdThreads = 384;
// Registers: the launch gives every thread of the three warpgroups 168 (64512 in all); a
// softmax thread holds a row of 128 scores, the loads and the MMA issue need few.
constexpr int kFwdRegs = 168, kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kFwdRegs, "more registers than the launch has would wait forever");

template <int DP> constexpr int fwd_stages() { return DP == 128 ? 5 : 8; }
template <int DP> constexpr int fwd_smem() { return (2 + fwd_stages<DP>()) * tile_bytes<DP>() + 1024 + 512; }

struct FwdArgs {
  CUtensorMap q, k, v, o, o_low;
  bool low;             // o_low is wanted
  AttnProblem p;
  const uint16_t* v_raw;
  float* lse;
  uint32_t* status;
  int q_tiles;          // of 256 queries
  int pieces;
  float* part;          // pieces > 1: [piece][batch][q_heads][q_len][DP], then 4 floats for every row: m, sum, packed sum
  uint16_t *o_raw, *low_raw;
};
__host__ __device__ inline long long part_rows(const AttnProblem& p) { return (long long)p.batch * p.q_heads * p.q_len; }

struct FwdShared {
  uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2];      // p_full: by halves of the keys
  uint64_t kv_full[8], kv_empty[8];
  int lo[2], hi[2];     // tiles of keys that row tile t sees
  uint32_t tmem_base, abort_flag;
};

template <int DP, bool BF16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kFwdThreads, 1) attn_fwd_kernel(const __grid_constant__ FwdArgs a) {
  constexpr int TILE = tile_bytes<DP>(), NS = fwd_stages<DP>();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  FwdShared* sh = reinterpret_cast<FwdShared*>(smem + (2 + NS) * TILE);
  volatile uint32_t* abort_flag = &sh->abort_flag;
  const uint32_t q_smem = ptx::smem_u32(smem), kv_smem = q_smem + 2 * TILE;
  const AttnProblem& p = a.p;

  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // the last queries, which see the most keys of a causal mask, come first
  const int heads = p.batch * p.q_heads;
  const int piece = a.pieces > 1 ? (int)(blockIdx.x % a.pieces) : 0, cta = a.pieces > 1 ? (int)(blockIdx.x / a.pieces) : (int)blockIdx.x;
  const int qt = a.q_tiles - 1 - cta / heads;
  const int bh = cta % heads, b = bh / p.q_heads, h = bh % p.q_heads, hk = h / p.group;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(&sh->q_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->s_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->p_full[t][0]), 4);
      ptx::mbar_init(ptx::smem_u32(&sh->p_full[t][1]), 4);
      ptx::mbar_init(ptx::smem_u32(&sh->o_full[t]), 1);
    }
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->kv_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->kv_empty[s]), 1);
    }
    sh->abort_flag = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    ptx::prefetch_tensormap(&a.q);
    ptx::prefetch_tensormap(&a.k);
    ptx::prefetch_tensormap(&a.v);
    ptx::prefetch_tensormap(&a.o);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&sh->tmem_base), 512);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  const int prefix = prefix_of(p, b);
  if (warp < 2) {   // range of key tiles of row tile `warp`
    const int q0 = qt * 2 * kTile + warp * kTile;
    int lo = 0, hi = 0;
    if (q0 < p.q_len) {
      const int last_row = q0 + kTile - 1 < p.q_len - 1 ? q0 + kTile - 1 : p.q_len - 1;
      hi = tiles_of(last_key(p, prefix, last_row + p.offset) + 1);   // last_key may be negative: no tile
      if (hi < 0) hi = 0;
      if (p.documents) {
        const int4 mine = p.query_docs[(long long)b * tiles_of(p.q_len) + q0 / kTile];
        const int4* kd = p.key_docs + (long long)b * tiles_of(p.k_len);
        int first = hi, last = -1;
        for (int j = lane; j < hi; j += 32)
          if (docs_meet(kd[j], mine)) {
            if (j < first) first = j;
            last = j;
          }
        lo = __reduce_min_sync(~0u, first);
        hi = __reduce_max_sync(~0u, last) + 1;
      }
    }
    if (lane == 0) {
      sh->lo[warp] = lo;
      sh->hi[warp] = hi > lo ? hi : lo;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ptx::uniform(sh->tmem_base);
  int lo0 = ptx::uniform(sh->lo[0]), hi0 = ptx::uniform(sh->hi[0]);
  int lo1 = ptx::uniform(sh->lo[1]), hi1 = ptx::uniform(sh->hi[1]);
  bool any0 = lo0 < hi0, any1 = lo1 < hi1;
  int lo = !any0 ? lo1 : !any1 ? lo0 : lo0 < lo1 ? lo0 : lo1;
  int hi = !any0 ? hi1 : !any1 ? hi0 : hi0 > hi1 ? hi0 : hi1;
  if (a.pieces > 1) {     // this CTA's piece of them
    const int first = lo, n = hi - lo;
    lo = first + (int)((long long)n * piece / a.pieces);
    hi = first + (int)((long long)n * (piece + 1) / a.pieces);
    lo0 = lo0 > lo ? lo0 : lo;
    lo1 = lo1 > lo ? lo1 : lo;
    hi0 = hi0 < hi ? hi0 : hi;
    hi1 = hi1 < hi ? hi1 : hi;
    any0 = lo0 < hi0;
    any1 = lo1 < hi1;
  }

  if (warp >= 8) {
  ptx::regs_less<kOtherRegs>();
  if (warp == 8) {
    // ---------------- loads ----------------
    bool ok = true;
    if (lane == 0) {
      for (int t = 0; t < 2; ++t) {
        if (!(t ? any1 : any0)) continue;
        const uint32_t bar = ptx::smem_u32(&sh->q_full[t]);
        ptx::mbar_arrive_expect_tx(bar, TILE);
        for (int c = 0; c < DP / 64; ++c) {
          const int32_t at[5] = {c * 64, qt * 2 * kTile + t * kTile, h, b, 0};
          ptx::tma_load_nd(4, q_smem + t * TILE + c * kBoxBytes, &a.q, at, bar);
        }
      }
    }
    const int4* kd = p.documents ? p.key_docs + (long long)b * tiles_of(p.k_len) : nullptr;
    uint32_t n = 0;      // ring slots filled so far
    for (int j = lo; ok && j < hi; ++j) {
      const bool dirty = kd && kd[j].z;
      for (int kv = 0; kv < 2; ++kv, ++n) {
        const uint32_t slot = n % NS, round = n / NS;
        const uint32_t full = ptx::smem_u32(&sh->kv_full[slot]);
        if (lane == 0)
          ok = ptx::mbar_wait_bounded(ptx::smem_u32(&sh->kv_empty[slot]), (round & 1) ^ 1, abort_flag, kAttnWait);
        ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
        if (!ok) {
          if (lane == 0) attn_fail(a.status, abort_flag, 0x410000u | slot);
          break;
        }
        if (kv == 1 && dirty) {   // padding among these keys: their values must not meet a zero weight
          copy_tile_clean<DP>(smem + (2 + slot) * TILE, a.v_raw + b * p.v_stride[0] + hk * p.v_stride[2], p.v_stride[1],
                              p.dim, j * kTile, p.k_len, p.documents + (long long)b * p.k_len, lane);
          if (lane == 0) ptx::mbar_arrive(full);
        } else if (lane == 0) {
          ptx::mbar_arrive_expect_tx(full, TILE);
          for (int c = 0; c < DP / 64; ++c) {
            const int32_t at[5] = {c * 64, j * kTile, hk, b, 0};
            ptx::tma_load_nd(4, kv_smem + slot * TILE + c * kBoxBytes, kv ? &a.v : &a.k, at, full);
          }
        }
      }
    }
    if (lane == 0 && *abort_flag) {   // leave no copy in flight
      uint32_t never = 0;
      for (int t = 0; t < 2; ++t)
        if (t ? any1 : any0) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->q_full[t]), 0, &never, kAttnWait);
      for (uint32_t s = 0; s < (uint32_t)NS; ++s)
        if (n > s) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->kv_full[s]), ((n - 1 - s) / NS) & 1, &never, kAttnWait);
    }
  } else if (warp == 9) {
    // ---------------- MMA issue ----------------
    {
      const uint32_t leader = ptx::elect_one();
      const uint32_t id_s = idesc_of<BF16>(kTile, false), id_o = idesc_of<BF16>(DP, true);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (ok && !__all_sync(~0u, ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait))) {
          if (leader) attn_fail(a.status, abort_flag, code);
          ok = false;
        }
      };
      uint32_t slot = 0, phase = 0, v_slot = 0, v_phase = 0;     // ring: the next tile's, V's of the step before
      bool have_q[2] = {false, false};
      for (int j = lo; ok && j <= hi && lo < hi; ++j) {
        const uint32_t k_slot = slot;
        if (j < hi) wait(&sh->kv_full[slot], phase, 0x420000u);
        if (j > lo) wait(&sh->kv_full[v_slot], v_phase, 0x420001u);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t v_tile = low_mn_major(kv_smem + v_slot * TILE), k_tile = low_k_major(kv_smem + k_slot * TILE);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int l = t ? lo1 : lo0, e = t ? hi1 : hi0;
          const uint32_t s_tmem = tmem + t * kTile, o_tmem = tmem + 2 * kTile + t * DP;
          if (j - 1 >= l && j - 1 < e) {     // O += P V(j - 1)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              wait(&sh->p_full[t][half], (j - 1 - l) & 1, 0x430000u | t);
              if (!ok) break;
              ptx::tc_fence_after();
#pragma unroll
              for (int s = half * 4; s < half * 4 + 4; ++s)
                ptx::mma_f16_ts_by(leader, o_tmem, s_tmem + s * 8, desc_mn_major(v_tile, s), id_o, j - 1 != l || s != 0);
            }
            if (!ok) break;
            if (j == e) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->o_full[t]));
          }
          if (j >= l && j < e) {             // S = Q K(j)
            if (!have_q[t]) {
              wait(&sh->q_full[t], 0, 0x440000u | t);
              if (!ok) break;
              have_q[t] = true;
              ptx::tc_fence_after();
            }
            const uint32_t q_tile = low_k_major(q_smem + t * TILE);
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
              ptx::mma_f16_ss_by(leader, s_tmem, desc_k_major(q_tile, s), desc_k_major(k_tile, s), id_s, s != 0);
            ptx::mma_commit_by(leader, ptx::smem_u32(&sh->s_full[t]));
          }
        }
        if (!ok) break;
        if (j > lo) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->kv_empty[v_slot]));
        if (j < hi) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->kv_empty[k_slot]));
        // K, V alternate in the ring
        v_slot = slot + 1 == NS ? 0 : slot + 1;
        v_phase = slot + 1 == NS ? phase ^ 1 : phase;
        slot = v_slot + 1 == NS ? 0 : v_slot + 1;
        phase = v_slot + 1 == NS ? v_phase ^ 1 : v_phase;
      }
    }
  }
  } else {
    ptx::regs_more<kSoftmaxRegs>();
    // ---------------- softmax, epilogue ----------------
    const int t = warp >> 2, quarter = warp & 3;
    const int l = t ? lo1 : lo0, e = t ? hi1 : hi0;
    const int q0 = qt * 2 * kTile + t * kTile;
    const int row = q0 + quarter * 32 + lane, pos = row + p.offset;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + t * kTile, o_tmem = tmem + lanes + 2 * kTile + t * DP;
    const int last = last_key(p, prefix, pos);
    const int last_first = last_key(p, prefix, q0 + p.offset);      // of the tile's first row: the smallest
    int own_doc = -1;
    int4 tile_docs = make_int4(0, 0, 0, 0);
    const int* docs = nullptr;
    const int4* kd = nullptr;
    if (p.documents && l < e) {
      docs = p.documents + (long long)b * p.k_len;
      kd = p.key_docs + (long long)b * tiles_of(p.k_len);
      if (row < p.q_len) own_doc = docs[pos];
      tile_docs = p.query_docs[(long long)b * tiles_of(p.q_len) + q0 / kTile];
    }
    const Scores sc = scores_of<CAP>(p.scale, p.softcap, p.slopes, h);
    float m = -INFINITY, sum = 0.f, packed_sum = 0.f;
    bool ok = true;
    for (int j = l; j < e; ++j) {
      const int j0 = j * kTile;
      bool masked = j0 + kTile - 1 > last_first;
      if (kd) masked = masked || !docs_same(kd[j], tile_docs);
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(&sh->s_full[t]), (j - l) & 1, abort_flag, kAttnWait)) {
        ok = false;
      }
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(a.status, abort_flag, 0x450000u | t);
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      float s[kTile];
#pragma unroll
      for (int c = 0; c < kTile; c += 32) ptx::tmem_ld_32x32(s_tmem + c, reinterpret_cast<uint32_t*>(s) + c);
      ptx::tmem_ld_wait();
      score<kTile, CAP, BIAS>(s, sc, pos - j0);
      if (masked) {
        uint32_t see[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) see[w] = bits_upto(last - j0, w);
        if (docs) {
          int other[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int c = j0 + 32 * w + lane;
            other[w] = c < p.k_len ? docs[c] : -1;
          }
          mask_documents(see, other, own_doc);
        }
#pragma unroll
        for (int c = 0; c < kTile; ++c) s[c] = (see[c >> 5] >> (c & 31)) & 1u ? s[c] : -INFINITY;
      }
      weigh_tile<DP, BF16, CAP || BIAS>(s, sc.by, j == l, &m, &sum, &packed_sum, s_tmem, o_tmem, sh->p_full[t], lane);
    }
    // result
    const bool has = sum > 0.f || sum != sum;
    const float inv = has ? 1.f / packed_sum : 0.f;
    if (ok && l < e) {
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(&sh->o_full[t]), 0, abort_flag, kAttnWait)) ok = false;
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(a.status, abort_flag, 0x460000u | t);
        ok = false;
      }
      ptx::tc_fence_after();
    }
    if (a.pieces > 1) {
      const long long at = part_rows(p) * piece + ((long long)b * p.q_heads + h) * p.q_len + row;
      if (ok && l < e && q0 + quarter * 32 < p.q_len) {
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(o_tmem + c, o);
          ptx::tmem_ld_wait();
          if (row < p.q_len)
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4*>(a.part + at * DP + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      if (ok && row < p.q_len)
        reinterpret_cast<float4*>(a.part + part_rows(p) * a.pieces * DP)[at] = make_float4(m, sum, packed_sum, 0.f);
      ok = false;      // the second kernel writes the results
    }
    if (row < p.q_len && ok)
      a.lse[((long long)b * p.q_heads + h) * p.q_len + row] = has ? log_of_sum<BF16>(m, sum) : -INFINITY;
    for (int low = 0; ok && low <= (a.low ? 1 : 0) && q0 + quarter * 32 < p.q_len; ++low) {   // the tile's own queries are no longer needed: stage there
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        if (l < e) {
          ptx::tmem_ld_32x32(o_tmem + c, o);
          ptx::tmem_ld_wait();
        }
        uint8_t* dst = smem + t * TILE + (c >> 6) * kBoxBytes + (quarter * 32 + lane) * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = __uint_as_float(o[8 * i + 2 * k]) * inv, y = __uint_as_float(o[8 * i + 2 * k + 1]) * inv;
            w[k] = inv != 0.f ? pack2<BF16>(x, y) : 0u;
            if (low) {
              const float2 z = unpack2<BF16>(w[k]);
              w[k] = inv != 0.f ? pack2<BF16>(x - z.x, y - z.y) : 0u;
            }
          }
          *reinterpret_cast<uint4*>(dst + (((((c & 32) >> 3) + i) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          const int32_t at[5] = {c * 64, q0 + quarter * 32, h, b, 0};
          ptx::tma_store_nd(4, low ? &a.o_low : &a.o, at, q_smem + t * TILE + c * kBoxBytes + quarter * 4096);
        }
        ptx::bulk_commit_group();
        ptx::bulk_wait_group_read<0>();
      }
      __syncwarp();
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// A warp per row: the pieces' sums brought to the largest reference value and added in order.
template <int DP, bool BF16>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ FwdArgs a) {
  const AttnProblem& p = a.p;
  ptx::grid_dependency_wait();
  const long long rows = part_rows(p), row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float4* stats = reinterpret_cast<const float4*>(a.part + rows * a.pieces * DP);
  float top = -INFINITY;
  for (int x = lane; x < a.pieces; x += 32) top = fmaxf(top, stats[rows * x + row].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  const float mu = top == -INFINITY ? 0.f : top;
  constexpr int V = DP / 32;
  float sum = 0.f, packed_sum = 0.f, acc[V] = {};
#pragma unroll 4
  for (int x = 0; x < a.pieces; ++x) {
    const float4 st = stats[rows * x + row];
    const float f = ex2(st.x - mu);
    if (st.y == 0.f) continue;      // saw nothing: its sums were not written
    sum = fmaf(st.y, f, sum);
    packed_sum = fmaf(st.z, f, packed_sum);
    const float* o = a.part + (rows * x + row) * DP + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = fmaf(o[i], f, acc[i]);
  }
  const bool has = sum > 0.f || sum != sum;
  const float inv = has ? 1.f / packed_sum : 0.f;
  const int i = (int)(row % p.q_len), h = (int)(row / p.q_len % p.q_heads), b = (int)(row / p.q_len / p.q_heads);
  const long long at = (((long long)b * p.q_len + i) * p.q_heads + h) * p.dim + lane * V;
  if (lane * V < p.dim) {
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      const float x = acc[k] * inv, y = acc[k + 1] * inv;
      const uint32_t w = has ? pack2<BF16>(x, y) : 0u;
      *reinterpret_cast<uint32_t*>(a.o_raw + at + k) = w;
      if (a.low) {
        const float2 z = unpack2<BF16>(w);
        *reinterpret_cast<uint32_t*>(a.low_raw + at + k) = has ? pack2<BF16>(x - z.x, y - z.y) : 0u;
      }
    }
  }
  if (lane == 0) a.lse[row] = has ? log_of_sum<BF16>(top, sum) : -INFINITY;
}

// Pieces of a call's loop over the keys, and the workspace they take.
int fwd_pieces(const AttnProblem& p) {
  return pieces_of(p, (long long)((p.q_len + 2 * kTile - 1) / (2 * kTile)) * p.batch * p.q_heads, tiles_of(p.k_len));
}

template <int DP, bool BF16, bool CAP, bool BIAS>
int32_t launch_fwd(const FwdArgs& a, int device, cudaStream_t s) {
  static PerDeviceFlag ready;
  auto kernel = attn_fwd_kernel<DP, BF16, CAP, BIAS>;
  if (!ready.test(device)) {
    LEGO_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fwd_smem<DP>()));
    ready.set(device);
  }
  const long long ctas = (long long)a.q_tiles * a.p.batch * a.p.q_heads * a.pieces;
  if (ctas > 0x7fffffffLL) return LEGO_ERR_SIZE;
  LEGO_CUDA_TRY(launch_overlapped(kernel, dim3((unsigned)ctas), dim3(kFwdThreads), fwd_smem<DP>(), s, a));
  if (a.pieces > 1)
    LEGO_CUDA_TRY(launch_overlapped(attn_join_kernel<DP, BF16>, dim3((unsigned)((part_rows(a.p) + 3) / 4)), dim3(128), 0, s, a));
  return LEGO_OK;
}

template <int DP, bool BF16>
int32_t launch_fwd_scores(const FwdArgs& a, int device, cudaStream_t s) {
  // The instance without cap and bias compares raw scores and scales them afterwards, which
  // needs a positive scale; the bias instance takes the others with a slope of zero.
  const bool cap = a.p.softcap > 0.f, bias = a.p.slopes || (!cap && !(a.p.scale > 0.f));
  if (cap) return bias ? launch_fwd<DP, BF16, true, true>(a, device, s) : launch_fwd<DP, BF16, true, false>(a, device, s);
  return bias ? launch_fwd<DP, BF16, false, true>(a, device, s) : launch_fwd<DP, BF16, false, false>(a, device, s);
}

}  // namespace

int64_t attention_fwd_bytes(const AttnProblem& p) {
  const int pieces = fwd_pieces(p);
  return attention_docs_bytes(p) + (pieces > 1 ? part_rows(p) * pieces * ((p.dim <= 64 ? 64 : 128) + 4) * 4 : 0);
}

}  // namespace lego

using namespace lego;

extern "C" int32_t lego_attention_fwd(const lego_attention_t* d, const void* q, const void* k, const void* v, void* o,
                                      void* o_low, float* lse, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  FwdArgs a = {};
  int32_t st = attention_problem(d, &a.p);
  if (st != LEGO_OK) return st;
  if (!q || !k || !v || !o || !lse) return LEGO_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)o_low | (uintptr_t)workspace) & 15) return LEGO_ERR_ALIGN;
  const int64_t need = attention_fwd_bytes(a.p);
  if (need && !workspace) return LEGO_ERR_NULL;
  if (workspace_bytes < need) return LEGO_ERR_SIZE;
  DeviceCtx* ctx = device_ctx(&st);
  if (!ctx) return st;
  EncodeFn enc = encode_fn(&st);
  if (!enc) return st;
  const AttnProblem& p = a.p;
  const bool bf16 = d->dtype == LEGO_BF16;
  const long long o_stride[3] = {(long long)p.q_len * p.q_heads * p.dim, (long long)p.q_heads * p.dim, p.dim};
  if (make_tmap_heads(enc, &a.q, bf16, q, p.dim, p.q_len, p.q_heads, p.batch, p.q_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.k, bf16, k, p.dim, p.k_len, p.k_heads, p.batch, p.k_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.v, bf16, v, p.dim, p.k_len, p.k_heads, p.batch, p.v_stride, kTile) != LEGO_OK ||
      make_tmap_heads(enc, &a.o, bf16, o, p.dim, p.q_len, p.q_heads, p.batch, o_stride, 32) != LEGO_OK ||
      (o_low && make_tmap_heads(enc, &a.o_low, bf16, o_low, p.dim, p.q_len, p.q_heads, p.batch, o_stride, 32) != LEGO_OK))
    return LEGO_ERR_UNSUPPORTED;
  a.low = o_low != nullptr;
  cudaStream_t s = (cudaStream_t)stream;
  st = attention_docs(&a.p, workspace, s);
  if (st != LEGO_OK) return st;
  a.v_raw = (const uint16_t*)v;
  a.lse = lse;
  a.status = ctx->status_word;
  a.q_tiles = (p.q_len + 2 * kTile - 1) / (2 * kTile);
  a.pieces = fwd_pieces(p);
  a.part = reinterpret_cast<float*>((uint8_t*)workspace + attention_docs_bytes(p));
  a.o_raw = (uint16_t*)o;
  a.low_raw = (uint16_t*)o_low;
  if (p.dim <= 64)
    return bf16 ? launch_fwd_scores<64, true>(a, ctx->device, s) : launch_fwd_scores<64, false>(a, ctx->device, s);
  return bf16 ? launch_fwd_scores<128, true>(a, ctx->device, s) : launch_fwd_scores<128, false>(a, ctx->device, s);
}
