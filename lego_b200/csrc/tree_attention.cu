// Attention of drafted token trees over a paged cache (sm_100a); one drafted token is plain
// decoding.
//
// The cache is read once and that is the bound: per 128 keys of 128 values 64 KiB arrive in
// about 2800 cycles of an SM's share of the memory, while the products of 128 rows take 1024
// and their weights about 1400.  So one form serves every number of rows: the drafted tokens
// and the query heads of a key head are the rows of one tile of 128 (the rest idle), more
// rows are more tiles.  The tensor core does the products as in the forward pass: S = Q K^T
// in TMEM, weights over S as packed pairs, O += P V.
//
// Work: the tiles of 128 keys of all sequences, key heads and row tiles, in one line, are cut
// into equal runs, one per CTA (one CTA per SM), so sequences of any lengths load every SM
// alike.  A run is a list of pieces: tile ranges of one (sequence, key head, row tile).
// A piece that covers all its tiles is finished by its CTA; the others, at most the first and
// the last of a run, leave (m, sum, O) in the workspace and a second kernel joins them in the
// order of the keys.  Which runs a sequence is in follows from the lengths, which only the
// device knows: every CTA adds them up.
//
// Few rows would leave most lanes of TMEM, and the warps that can read them, idle while one
// warp works through 128 scores per row.  Up to 16 rows the queries therefore stand in the tile
// four times, up to 64 twice: every copy weighs its own quarter or half of a tile's keys (its
// weights of the others are zero) with its own m, sum and O, and the copies are put together
// at a piece's end.
//
// Warps: 0-3 and 4-7 weights of the even and the odd tiles of a piece (each with its own m, sum
// and O, put together at the piece's end), 8-11 loads of the cache, 12 MMA issue, 13-15 the run's
// pieces with their trees and queries, one piece ahead (64 sequences 261 -> 257 us, 2 x 131072 tokens
// 157 -> 156, against loads that did this in between; their waits are long suspends, polling took
// slots from capped weights).  Each loading lane looks up the place of one row of a tile.  Tiles come by TMA, in
// boxes of as many rows as stand together in a page (a common divisor of the page size and 32, at
// least 8); pages of other sizes come as 16-byte copies.  Keys that do not exist (past the end, of
// a page number outside the cache, of an unused drafted token) are hidden by a mask that the loads
// leave with the tile, and their values, which may be NaN and must not meet a zero weight, are
// zeros in shared memory: a box past the cache reads as zeros, other rows are cleared by the
// loading warp before it hands the tile on.
//
// Measured, calls in turn: 64 sequences of 1024 .. 8192 tokens x 32/8 heads of 128, bf16, one token 257 us (5.1 TB/s);
// 8 of 8192 .. 65536 tokens 260 us (5.8, what a plain sum reads here: the difference is the change of sequence and
// the join, a launch of 8 us that starts when the last run has ended); 2 x 131072 tokens x 64 rows with a
// bias 157 us (4.7).  8 x 16384 x 37 tokens of 2 heads with a cap 100 us: no unit is half busy (issue slots 39 %, FMA 18 %,
// exponentials 16 %, memory 25 %); above 64 rows a warp takes 128 columns in four chunks, each read from TMEM, written
// back and read again, and two warps per scheduler do not hide that.  Slower: scores and weights of one copy in
// registers (drafts 95 -> 104 us).
#include <cuda.h>

#include "attention.cuh"
#include "tma_host.cuh"

namespace lego {
namespace {

constexpr int kMaxDraft = LEGO_MAX_DRAFT;
constexpr int kTreeThreads = 512;
constexpr int kTreeRegs = 128, kTreeMathRegs = 176, kTreeOtherRegs = 80;
static_assert(2 * kTreeMathRegs + 2 * kTreeOtherRegs <= 4 * kTreeRegs, "more registers than the launch has would wait forever");

struct TreeProblem {
  int batch, drafted, q_heads, k_heads, dim, group;
  int pages, page_size, max_pages;
  int rows, row_tiles;          // rows of a key head: drafted * group; tiles of 128 of them
  int copies;                   // of the rows in a tile: 4, 2 or 1
  long long table_stride;
  long long q_stride[3], k_stride[3], v_stride[3];
  float scale, softcap;
  const int* table;
  const int* lengths;
  const int* parents;
  const float* slopes;
  const uint16_t *q, *k, *v;
  uint16_t* o;
  float* partial;               // [2 * runs][128][dim rounded up to 64], then [2 * runs][128] (m, sum)
  uint32_t* status;
  int runs;                     // CTAs of the main kernel
  int box_rows;                 // rows of a TMA box of the cache; 0: 16-byte copies only
  FastDiv by_page, by_group;
};

struct TreeMaps {
  CUtensorMap k, v;
};

int32_t tree_problem(const lego_tree_attention_t* d, TreeProblem* p) {
  if (!d) return LEGO_ERR_NULL;
  if (d->dtype != LEGO_F16 && d->dtype != LEGO_BF16) return LEGO_ERR_UNSUPPORTED;
  if (d->batch < 1 || d->drafted < 1 || d->q_heads < 1 || d->k_heads < 1 || d->head_dim < 1 || d->pages < 1 ||
      d->page_size < 1 || d->max_pages < 1)
    return LEGO_ERR_DIM;
  if (d->drafted > kMaxDraft || d->q_heads % d->k_heads || d->head_dim % 8 || d->head_dim > 128) return LEGO_ERR_SIZE;
  if (d->batch > 65535 || d->q_heads > 65535 || d->pages > 0x7fffffffLL || d->page_size > (1 << 30) ||
      d->max_pages > (1 << 30) / d->page_size || d->table_stride < d->max_pages)
    return LEGO_ERR_SIZE;
  if (!scores_ok(d->scale, d->softcap)) return LEGO_ERR_SIZE;
  p->batch = (int)d->batch;
  p->drafted = (int)d->drafted;
  p->q_heads = (int)d->q_heads;
  p->k_heads = (int)d->k_heads;
  p->dim = (int)d->head_dim;
  p->group = p->q_heads / p->k_heads;
  p->rows = p->drafted * p->group;
  p->row_tiles = tiles_of(p->rows);
  p->copies = p->rows <= 16 ? 4 : p->rows <= 64 ? 2 : 1;
  if ((int64_t)p->batch * p->k_heads * p->row_tiles > 0x7fffffffLL) return LEGO_ERR_SIZE;
  p->pages = (int)d->pages;
  p->page_size = (int)d->page_size;
  p->max_pages = (int)d->max_pages;
  p->table_stride = d->table_stride;
  for (int i = 0; i < 3; ++i) {
    p->q_stride[i] = d->q_stride[i];
    p->k_stride[i] = d->k_stride[i];
    p->v_stride[i] = d->v_stride[i];
    if (d->q_stride[i] % 8 || d->k_stride[i] % 8 || d->v_stride[i] % 8) return LEGO_ERR_ALIGN;
  }
  // every tile of the longest sequences the table has room for, in 31 bits
  if ((int64_t)p->batch * p->k_heads * p->row_tiles * tiles_of(p->max_pages * p->page_size) > 0x7fffffffLL) return LEGO_ERR_SIZE;
  p->by_page = make_fastdiv((uint64_t)p->page_size);
  p->by_group = make_fastdiv((uint64_t)p->group);
  p->scale = d->scale;
  p->softcap = d->softcap;
  return LEGO_OK;
}

// ---- the line of tiles and its runs --------------------------------------------------------------

// Places of a sequence of `len` cached tokens that may be seen: those and the drafted ones, within
// the table.
__device__ __forceinline__ int tree_places(const TreeProblem& p, int len) {
  if (len < 0) return 0;
  const int room = p.max_pages * p.page_size;      // at most 2^30
  return len < room - p.drafted ? len + p.drafted : room;
}
__device__ __forceinline__ int run_begin(int total, int runs, int c) { return total / runs * c + total % runs * c / runs; }

struct Piece {
  int b, hk, rt;         // sequence (-1: no more pieces), key head, row tile
  int first, last;       // tiles [first, last)
  int len, places;       // of the sequence
};

// Sum over the block's threads of v and what the threads before this one add to; a word of shared
// memory per warp.  Every thread takes part.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* before, int* words) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) words[warp] = x;
  __syncthreads();
  int base = 0, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    const int w = words[i];
    if (i < warp) base += w;
    total += w;
  }
  *before = base + x - v;
  return total;
}

// ---- the draft's tree -------------------------------------------------------------------------------

struct Tree {
  unsigned long long seen[kMaxDraft];   // ancestors of a token and itself; 0: unused
  uint8_t depth[kMaxDraft];
};

// One warp, two tokens a lane: every token's set, depth and next ancestor double their reach
// six times.
__device__ void grow_tree(const TreeProblem& p, int b, Tree* out, int lane) {
  int up[2], depth[2];
  unsigned long long seen[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = lane + 32 * i;
    up[i] = -2;
    if (t < p.drafted) {
      up[i] = p.parents ? p.parents[(long long)b * p.drafted + t] : t - 1;
      if (up[i] < -1 || up[i] >= t) up[i] = -2;
    }
    seen[i] = 1ull << t;
    depth[i] = up[i] >= 0;
  }
  for (int reach = 1; reach < p.drafted; reach *= 2) {
    int nu[2], nd[2];
    unsigned long long ns[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = up[i] & 31;
      const bool high = up[i] >= 32;
      const int u0 = __shfl_sync(~0u, up[0], from), u1 = __shfl_sync(~0u, up[1], from);
      const int d0 = __shfl_sync(~0u, depth[0], from), d1 = __shfl_sync(~0u, depth[1], from);
      const unsigned long long s0 = __shfl_sync(~0u, seen[0], from), s1 = __shfl_sync(~0u, seen[1], from);
      nu[i] = up[i] < 0 ? up[i] : high ? u1 : u0;
      nd[i] = up[i] < 0 ? depth[i] : depth[i] + (high ? d1 : d0);
      ns[i] = up[i] < 0 ? seen[i] : seen[i] | (high ? s1 : s0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      up[i] = nu[i];
      depth[i] = nd[i];
      seen[i] = ns[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = lane + 32 * i;
    out->seen[t] = up[i] == -1 ? seen[i] : 0;
    out->depth[t] = (uint8_t)depth[i];
  }
}

// ---- main kernel --------------------------------------------------------------------------------------

template <int DP> constexpr int tree_stages() { return DP == 128 ? 5 : 10; }
constexpr int kMaskRing = 8;    // see the note at its use
struct TreeShared {
  Tree tree[2];
  Piece piece[2];
  uint32_t exist[kMaskRing][4];
  uint64_t exist_full[kMaskRing], full[10], empty[10], cleared[4];
  uint64_t piece_full[2], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], odd_done, o_free, merged;
  int words[16];
  int start_b, start_hr, start_tile, start_left;
  uint32_t tmem_base, abort_flag;
};
template <int DP> constexpr int tree_smem() { return (2 + tree_stages<DP>()) * tile_bytes<DP>() + 1024 + (int)sizeof(TreeShared); }
static_assert(tree_smem<128>() <= 232448 && tree_smem<64>() <= 232448, "shared memory of a CTA");

template <int DP, bool BF16, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_attn_kernel(const __grid_constant__ TreeProblem p, const __grid_constant__ TreeMaps maps) {
  constexpr int TILE = tile_bytes<DP>(), NS = tree_stages<DP>();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  TreeShared* sh = reinterpret_cast<TreeShared*>(smem + (2 + NS) * TILE);
  volatile uint32_t* abort_flag = &sh->abort_flag;
  const uint32_t q_smem = ptx::smem_u32(smem), kv_smem = q_smem + 2 * TILE;
  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(&sh->piece_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->q_full[t]), 96);           // the copies of three warps' threads
      ptx::mbar_init(ptx::smem_u32(&sh->q_empty[t]), 1 + 8 + 4);   // the MMAs; the warps done with the piece and its tree
      ptx::mbar_init(ptx::smem_u32(&sh->s_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->p_full[t]), 4);
      ptx::mbar_init(ptx::smem_u32(&sh->o_full[t]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&sh->odd_done), 4);
    ptx::mbar_init(ptx::smem_u32(&sh->o_free), 4);
    ptx::mbar_init(ptx::smem_u32(&sh->merged), 4);
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->full[s]), 128);     // every loading thread's copies
      ptx::mbar_init(ptx::smem_u32(&sh->empty[s]), 1);
    }
    for (int s = 0; s < kMaskRing; ++s) ptx::mbar_init(ptx::smem_u32(&sh->exist_full[s]), 4);
    for (int s = 0; s < 4; ++s) ptx::mbar_init(ptx::smem_u32(&sh->cleared[s]), 1);
    sh->abort_flag = 0;
    sh->start_left = 0;
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  if (warp == 12) {
    ptx::tmem_alloc(ptx::smem_u32(&sh->tmem_base), 512);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_wait();
  {   // this CTA's run: where it starts and how long it is
    const int per_tile = p.k_heads * p.row_tiles;
    auto units_of = [&](int b) { return b < p.batch ? tiles_of(tree_places(p, p.lengths[b])) * per_tile : 0; };
    int total = 0, mine = 0, before = 0;
    for (int base = 0; base < p.batch; base += kTreeThreads) {
      mine = units_of(base + threadIdx.x);
      total += block_scan<kTreeThreads>(mine, &before, sh->words);
    }
    const int runs = total < (int)gridDim.x ? total : (int)gridDim.x;
    if ((int)blockIdx.x < runs) {
      const int u0 = run_begin(total, runs, blockIdx.x), u1 = run_begin(total, runs, blockIdx.x + 1);
      int passed = 0;
      for (int base = 0; base < p.batch; base += kTreeThreads) {
        int sum = total;
        if (p.batch > kTreeThreads) {     // not the sums of the last turn above
          mine = units_of(base + threadIdx.x);
          sum = block_scan<kTreeThreads>(mine, &before, sh->words);
        }
        const int at = u0 - passed - before;
        if (at >= 0 && at < mine) {
          const int tiles = mine / per_tile;
          sh->start_b = base + threadIdx.x;
          sh->start_hr = at / tiles;
          sh->start_tile = at % tiles;
          sh->start_left = u1 - u0;
        }
        passed += sum;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = ptx::uniform(sh->tmem_base);
  Piece pc;

  if (warp >= 12) {
    ptx::regs_less<kTreeOtherRegs>();
    if (warp == 12) {
      // ---------------- MMA issue ----------------
      const uint32_t leader = ptx::elect_one();
      const uint32_t id_s = idesc_of<BF16>(kTile, false), id_o = idesc_of<BF16>(DP, true);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (ok && !__all_sync(~0u, ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait))) {
          if (leader) attn_fail(p.status, abort_flag, code);
          ok = false;
        }
        ptx::tc_fence_after();
      };
      uint32_t pos = 0;                    // ring position of K(i)
      uint32_t weighed[2] = {0, 0};
      for (int n = 0; ok; ++n) {
        wait(&sh->piece_full[n & 1], (n >> 1) & 1, 0x720005u);
        pc = sh->piece[n & 1];
        if (!ok || pc.b < 0) break;
        const int count = pc.last - pc.first;
        const uint32_t q_tile = q_smem + (n & 1) * TILE;
        wait(&sh->q_full[n & 1], (n >> 1) & 1, 0x720000u);
        ptx::fence_proxy_async();      // the queries came as 16-byte copies, through the generic proxy
        for (int i = 0; ok && i <= count; ++i, pos += 2) {
          // the accumulators, and the place of the odd warps' statistics, have been read
          if (i == 1 && n > 0) wait(&sh->o_free, (n - 1) & 1, 0x720001u);
          if (!ok) break;
          if (i < count) {
            const uint32_t slot = pos % NS;
            wait(&sh->full[slot], (pos / NS) & 1, 0x720002u);
            if (!ok) break;
            if (!p.box_rows)
              ptx::fence_proxy_async();      // so did these keys
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
              ptx::mma_f16_ss_by(leader, tmem + (i & 1) * kTile, desc_k_major(low_k_major(q_tile), s), desc_k_major(low_k_major(kv_smem + slot * TILE), s), id_s, s != 0);
            ptx::mma_commit_by(leader, ptx::smem_u32(&sh->s_full[i & 1]));
            ptx::mma_commit_by(leader, ptx::smem_u32(&sh->empty[slot]));
            if (i == count - 1) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->q_empty[n & 1]));
          }
          if (i > 0) {
            const uint32_t t = (i - 1) & 1, vpos = pos - 1, slot = vpos % NS;
            wait(&sh->full[slot], (vpos / NS) & 1, 0x720003u);
            wait(&sh->p_full[t], weighed[t] & 1, 0x720004u);
            if (!ok) break;
            if (!p.box_rows) ptx::fence_proxy_async();
            ++weighed[t];
#pragma unroll
            for (int s = 0; s < kTile / 16; ++s)
              ptx::mma_f16_ts_by(leader, tmem + 2 * kTile + t * DP, tmem + t * kTile + s * 8, desc_mn_major(low_mn_major(kv_smem + slot * TILE), s), id_o,
                              i > 2 || s != 0);
            ptx::mma_commit_by(leader, ptx::smem_u32(&sh->empty[slot]));
            if (i >= count - 1) ptx::mma_commit_by(leader, ptx::smem_u32(&sh->o_full[t]));
          }
        }
        pos -= 2;     // the last turn had no K
      }
    } else {
      // ---------------- pieces (warp 13) and their queries ----------------
      constexpr int CH = DP / 8, PER = 32 / CH;    // 16-byte pieces of a row; rows per instruction
      const int chunk = lane % CH, first_row = (warp - 13) * PER + lane / CH;
      const bool chunk_real = chunk * 8 < p.dim;
      int next_b = sh->start_b, next_hr = sh->start_hr, next_tile = sh->start_tile, left = sh->start_left;
      int len = warp == 13 && left > 0 ? p.lengths[next_b] : 0;
      bool ok = true;
      auto bounded = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (lane == 0) ok = ptx::mbar_wait_bounded<true>(ptx::smem_u32(bar), parity, abort_flag, kAttnWait);
        ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
        if (!ok && lane == 0) attn_fail(p.status, abort_flag, code);
        return ok;
      };
      for (int n = 0; ok; ++n) {
        if (warp == 13) {
          if (!bounded(&sh->q_empty[n & 1], ((n >> 1) & 1) ^ 1, 0x710000u)) break;
          pc.b = -1;
          if (left > 0) {
            pc.b = next_b;
            pc.hk = next_hr / p.row_tiles;
            pc.rt = next_hr - pc.hk * p.row_tiles;
            pc.len = len;
            pc.places = tree_places(p, len);
            pc.first = next_tile;
            const int tiles = tiles_of(pc.places);
            pc.last = left < tiles - next_tile ? next_tile + left : tiles;
            left -= pc.last - pc.first;
            next_tile = 0;
            grow_tree(p, pc.b, &sh->tree[n & 1], lane);
          }
          if (lane == 0) sh->piece[n & 1] = pc;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->piece_full[n & 1]));
        } else {
          if (!bounded(&sh->piece_full[n & 1], (n >> 1) & 1, 0x710004u)) break;
          pc = sh->piece[n & 1];
        }
        if (pc.b < 0) break;
        const int per_copy = kTile / p.copies;
#pragma unroll 4
        for (int r = first_row; r < kTile; r += 3 * PER) {
          const int row = pc.rt * kTile + (r & (per_copy - 1));
          const bool copy = row < p.rows && chunk_real;
          const int t = (int)fd_div((uint32_t)row, p.by_group), h = pc.hk * p.group + row - t * p.group;
          const uint16_t* src = p.q + pc.b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2] + chunk * 8;
          ptx::cp_async_16(q_smem + (n & 1) * TILE + (chunk >> 3) * kBoxBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4),
                           copy ? src : p.q, copy);
        }
        ptx::cp_async_arrive(ptx::smem_u32(&sh->q_full[n & 1]));
        if (warp == 13 && ++next_hr == p.k_heads * p.row_tiles && left > 0) {
          next_hr = 0;
          do len = p.lengths[++next_b];      // units are left, so a sequence with tiles follows
          while (len < 0);
        }
      }
      ptx::cp_async_wait_all();
    }
  } else if (warp >= 8) {
    ptx::regs_less<kTreeOtherRegs>();
    // ---------------- loads ----------------
    constexpr int CH = DP / 8, PER = 32 / CH;    // 16-byte pieces of a row; rows per instruction
    const int w = warp - 8, chunk = lane % CH, sub = lane / CH;
    const bool chunk_real = chunk * 8 < p.dim;
    uint32_t issued = 0, tile_no = 0, clears = 0;
    bool ok = true;
    auto bounded = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (lane == 0) ok = ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait);
      ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
      if (!ok && lane == 0) attn_fail(p.status, abort_flag, code);
      return ok;
    };
    for (int n = 0; ok; ++n) {
      if (!bounded(&sh->piece_full[n & 1], (n >> 1) & 1, 0x710002u)) break;
      pc = sh->piece[n & 1];
      if (pc.b < 0) break;
      const Tree* tree = &sh->tree[n & 1];
      const int places = pc.places;
      const int* table = p.table + pc.b * p.table_stride;
      // page number of this lane's row of a tile, as the table has it; -1: past the end
      auto page_of = [&](int tile) {
        const int j = tile * kTile + w * 32 + lane;
        return tile < pc.last && j < places ? table[fd_div((uint32_t)j, p.by_page)] : -1;
      };
      int page = page_of(pc.first);
      for (int tile = pc.first; ok && tile < pc.last; ++tile, ++tile_no) {
        const int place = tile * kTile + w * 32 + lane;
        const int in_page = place - (int)fd_div((uint32_t)place, p.by_page) * p.page_size;
        const bool paged = page >= 0 && page < p.pages;
        const int here = paged ? page : p.pages;     // past the cache: a TMA box of zeros
        const bool real = paged && (place < pc.len || tree->seen[place - pc.len] != 0);
        page = page_of(tile + 1);                    // on its way while this tile's copies are issued
        const uint32_t word = __ballot_sync(~0u, real);
        for (int g = 0; g < 2; ++g, ++issued) {
          const uint32_t slot = issued % NS, full = ptx::smem_u32(&sh->full[slot]);
          if (!bounded(&sh->empty[slot], ((issued / NS) & 1) ^ 1, 0x710001u)) break;
          // The entry was read for the tile 8 before.  A free slot for this K means that the product
          // S of a tile at most 5 before is done (10 slots hold 5 tiles); it was issued after the
          // weights of the two tiles before it had been waited for, so those of 8 before are done.
          if (g == 0 && lane == 0) {
            sh->exist[tile_no % kMaskRing][w] = word;
            ptx::mbar_arrive(ptx::smem_u32(&sh->exist_full[tile_no % kMaskRing]));
          }
          const uint32_t dst = kv_smem + slot * TILE + w * 4096;     // this warp's rows in the first box
          if (p.box_rows) {
            const bool clear = g == 1 && word != ~0u;
            const uint32_t bar = clear ? ptx::smem_u32(&sh->cleared[w]) : full;
            if (lane == 0) {
              ptx::mbar_arrive_expect_tx(bar, TILE / 4);
              if (!clear) ptx::mbar_arrive_n(full, 31);      // 32 arrivals, as of a warp's copies
            }
            __syncwarp();
            constexpr int WIDE = DP / 64;
            const int r = lane / WIDE * p.box_rows, c = lane % WIDE;
            const int pg = __shfl_sync(~0u, here, r & 31), at_slot = __shfl_sync(~0u, in_page, r & 31);
            if (r < 32) {
              const int32_t at[5] = {c * 64, at_slot, pc.hk, pg, 0};
              ptx::tma_load_nd(4, dst + c * kBoxBytes + r * 128, g ? &maps.v : &maps.k, at, bar);
            }
            if (clear) {
              __syncwarp();
              if (!bounded(&sh->cleared[w], clears++ & 1, 0x710003u)) break;
              if (lane < CH)
                for (uint32_t dead = ~word; dead; dead &= dead - 1)
                  *reinterpret_cast<uint4*>(smem + (2 + slot) * TILE + (lane >> 3) * kBoxBytes + (w * 32 + __ffs(dead) - 1) * 128 +
                                            ((lane & 7) << 4)) = make_uint4(0, 0, 0, 0);
              ptx::fence_proxy_async();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive_n(full, 32);
            }
            continue;
          }
          const long long s0 = g ? p.v_stride[0] : p.k_stride[0], s1 = g ? p.v_stride[1] : p.k_stride[1],
                          s2 = g ? p.v_stride[2] : p.k_stride[2];
          const long long row_at = real ? here * s0 + in_page * s1 + pc.hk * s2 : 0;
          const uint16_t* src = g ? p.v : p.k;
#pragma unroll 4
          for (int i = 0; i < 32; i += PER) {
            const int r = i + sub;
            const long long at = __shfl_sync(~0u, row_at, r);
            const bool copy = ((word >> r) & 1u) && chunk_real;
            ptx::cp_async_16(dst + (chunk >> 3) * kBoxBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4),
                             src + (copy ? at + chunk * 8 : 0), copy);
          }
          ptx::cp_async_arrive(full);
        }
      }
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->q_empty[n & 1]));
    }
    ptx::cp_async_wait_all();
    if (*abort_flag && lane == 0) {      // leave no copy in flight: a tenth of a second for each slot at most
      uint32_t never = 0;
      for (uint32_t s = 0; s < (uint32_t)NS; ++s)
        if (issued > s) ptx::mbar_wait_bounded(ptx::smem_u32(&sh->full[s]), ((issued - 1 - s) / NS) & 1, &never, kAttnWait / 10);
    }
  } else {
    ptx::regs_more<kTreeMathRegs>();
    // ---------------- weights, epilogue ----------------
    const int t = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + t * kTile, o_tmem = tmem + lanes + 2 * kTile + t * DP;
    const float by = p.scale * kLog2e;
    const int per_copy = kTile / p.copies, chunks = 4 / p.copies;     // rows; chunks of 32 columns a copy weighs
    const int in_copy = (quarter * 32 + lane) & (per_copy - 1), copy = quarter * 32 / per_copy, chunk0 = copy * chunks;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait)) ok = false;
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(p.status, abort_flag, code);
        ok = false;
      }
      return ok;
    };
    uint32_t scored = 0, tile_no = 0, mine = 0, paired = 0, merges = 0;
    for (int n = 0; ok; ++n) {
      if (!wait(&sh->piece_full[n & 1], (n >> 1) & 1, 0x740000u)) break;
      pc = sh->piece[n & 1];
      if (pc.b < 0) break;
      const int count = pc.last - pc.first;
      const int row = pc.rt * kTile + in_copy;
      const bool real = row < p.rows, any_row = pc.rt * kTile + (quarter * 32 & (per_copy - 1)) < p.rows;
      const int tok = real ? (int)fd_div((uint32_t)row, p.by_group) : 0, h = pc.hk * p.group + (real ? row - tok * p.group : 0);
      const Tree* tree = &sh->tree[n & 1];
      const int len = pc.len;
      const unsigned long long seen = real ? tree->seen[tok] : 0;
      const int depth = tree->depth[tok];
      const Scores sc = scores_of<CAP>(p.scale, p.softcap, p.slopes, h);
      float m = -INFINITY, sum = 0.f;
      for (int i = t; i < count; i += 2) {
        const int j0 = (pc.first + i) * kTile;
        const uint32_t no = tile_no + i;
        if (!wait(&sh->exist_full[no % kMaskRing], (no / kMaskRing) & 1, 0x740001u) ||
            !wait(&sh->s_full[t], scored & 1, 0x740002u))
          break;
        ++scored;
        ptx::tc_fence_after();
        if (any_row) {       // else whatever the product makes of what stands there: nobody reads it
          // First the maximum; scores that are not used as the product leaves them go back to
          // their place.  Then the weights.
          float s[32], mt = -INFINITY;
          bool back = CAP || BIAS;
          for (int x = 0; x < chunks; ++x) {
            const int c0 = 32 * (chunk0 + x);
            ptx::tmem_ld_32x32(s_tmem + c0, reinterpret_cast<uint32_t*>(s));
            uint32_t see = sh->exist[no % kMaskRing][chunk0 + x];
            const int at = len - j0 - c0;      // column of the first drafted token
            if (at < 32) {
              const int shift = -at;           // draft token of column 0
              const uint32_t drafted = shift <= -32 || shift >= 64 ? 0u : shift >= 0 ? (uint32_t)(seen >> shift) : (uint32_t)(seen << -shift);
              see &= bits_upto(at - 1, 0) | drafted;
            }
            ptx::tmem_ld_wait();
            if (CAP || BIAS) {
              // cached tokens: none is ahead.  (A place past 2^24 is rounded, its distance by as little.)
              score<32, CAP, false>(s, sc, 0);
              if (BIAS) bias_behind<32, CAP>(s, sc, (float)at + (float)depth);
              if (BIAS && at < 32) {     // drafted tokens stand where their depth says, not their place
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                  const int d = c - at;
                  if (d >= 0 && d < p.drafted)
                    s[c] = fmaf(-sc.slope, fabsf((float)(depth - tree->depth[d])) - (float)(depth - d), s[c]);
                }
              }
            }
            const bool hide = __any_sync(~0u, see != ~0u);
            if (hide) {
#pragma unroll
              for (int c = 0; c < 32; ++c) s[c] = (see >> c) & 1u ? s[c] : -INFINITY;
            }
            mt = fmaxf(mt, max_of(s));
            if (chunks > 1 && (CAP || BIAS || hide)) {
              ptx::tmem_st_32x16(s_tmem + c0, reinterpret_cast<uint32_t*>(s));
              ptx::tmem_st_32x16(s_tmem + c0 + 16, reinterpret_cast<uint32_t*>(s) + 16);
              back = true;
            }
          }
          if (chunks > 1 && back) ptx::tmem_st_wait();
          if (!CAP && !BIAS) mt *= by;     // by > 0 in this instance
          float unused = 0.f;
          follow_maximum<DP, BF16>(mt, i == t, &m, &sum, &unused, o_tmem);
          const float mu = m == -INFINITY ? 0.f : m;
          const float2 by2 = make_float2(by, by), mu2 = make_float2(-mu, -mu);
          for (int x = 0; x < 4; ++x) {
            uint32_t w[16] = {};
            if (x >= chunk0 && x < chunk0 + chunks) {
              if (chunks > 1) {
                ptx::tmem_ld_32x32(s_tmem + 32 * x, reinterpret_cast<uint32_t*>(s));
                ptx::tmem_ld_wait();
              }
              float2 add[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                float2 z = make_float2(s[c], s[c + 1]);
                z = CAP || BIAS ? ptx::add2(z, mu2) : ptx::fma2(z, by2, mu2);
                w[c >> 1] = pack2<BF16>(ex2(z.x), ex2(z.y));
                add[(c >> 1) & 1] = ptx::add2(add[(c >> 1) & 1], unpack2<BF16>(w[c >> 1]));     // as they count in O
              }
              sum += (add[0].x + add[0].y) + (add[1].x + add[1].y);
            }
            ptx::tmem_st_32x16(s_tmem + 16 * x, w);      // over scores that have been read: chunk x / 2
          }
          ptx::tmem_st_wait();
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->p_full[t]));
      }
      if (!ok) break;
      tile_no += count;
      if (seen == 0) {        // an unused token: no weight, whatever it would have seen
        m = -INFINITY;
        sum = 0.f;
      }
      if (t == 1) {       // leave (m, sum) where the scores were, for the other warpgroup
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->q_empty[n & 1]));    // done with the tree
        if (count < 2) continue;
        if (!wait(&sh->o_full[1], mine & 1, 0x750000u)) break;
        ++mine;
        ptx::tc_fence_after();
        ptx::tmem_st_32x2(s_tmem, __float_as_uint(m), __float_as_uint(sum));
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->odd_done));
        continue;
      }
      if (!wait(&sh->o_full[0], mine & 1, 0x750001u)) break;
      ++mine;
      float m1 = -INFINITY, sum1 = 0.f;
      if (count >= 2) {
        if (!wait(&sh->odd_done, paired & 1, 0x750002u)) break;
        ++paired;
        ptx::tc_fence_after();
        uint32_t r[2];
        ptx::tmem_ld_32x2(s_tmem + kTile, r);
        ptx::tmem_ld_wait();
        m1 = __uint_as_float(r[0]);
        sum1 = __uint_as_float(r[1]);
      }
      ptx::tc_fence_after();
      float top = fmaxf(m, m1);
      float mu = top == -INFINITY ? 0.f : top;
      float f0 = ex2(m - mu), f1 = ex2(m1 - mu);
      float all = sum * f0 + sum1 * f1;
      // The copies of a row meet in the piece's place of queries, which no product reads any more
      // (o_full) and the loads get back only afterwards.
      uint8_t* scratch = smem + (n & 1) * TILE;
      auto meet = [&]() {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->merged));
        return wait(&sh->merged, merges++ & 1, 0x750003u);
      };
      if (p.copies > 1) {
        float2* stats = reinterpret_cast<float2*>(scratch);
        stats[copy * per_copy + in_copy] = make_float2(top, all);
        if (!meet()) break;
        const float own = top;
        for (int x = 0; x < p.copies; ++x) top = fmaxf(top, stats[x * per_copy + in_copy].x);
        mu = top == -INFINITY ? 0.f : top;
        all = 0.f;
        for (int x = 0; x < p.copies; ++x) {
          const float2 y = stats[x * per_copy + in_copy];
          all = fmaf(y.y, ex2(y.x - mu), all);
        }
        const float f = ex2(own - mu);
        f0 *= f;
        f1 *= f;
        if (!meet()) break;      // everyone has read them
      }
      const bool whole = pc.first == 0 && pc.last == tiles_of(pc.places);
      const bool has = all > 0.f || all != all;
      const float norm = whole ? (has ? 1.f / all : 0.f) : 1.f;
      const float g0 = sum != 0.f ? f0 * norm : 0.f, g1 = sum1 != 0.f ? f1 * norm : 0.f;
      // of an unfinished piece: the run's last when it starts its sequence, else the run's first
      const long long slot = 2 * (long long)blockIdx.x + (pc.first == 0 ? 1 : 0);
      // 32 columns of this thread's row, both warpgroups' parts
      auto combined = [&](int c, float (&v)[32]) {
        uint32_t o[32], o1[32];
        ptx::tmem_ld_32x32(o_tmem + c, o);
        if (count >= 2) ptx::tmem_ld_32x32(o_tmem + DP + c, o1);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          v[x] = g0 != 0.f ? __uint_as_float(o[x]) * g0 : 0.f;
          if (count >= 2 && g1 != 0.f) v[x] = fmaf(__uint_as_float(o1[x]), g1, v[x]);
        }
      };
      if (p.copies > 1) {
        // All copies put their part down, 128 threads add them up and write whole rows.  Two copies'
        // 64 rows fit in two turns.
        const int wide = p.copies == 4 ? DP : DP / 2, vecs = wide / 4;
        float4* meeting = reinterpret_cast<float4*>(scratch);      // [copy][row][wide / 4], rows under a swizzle
        for (int c0 = 0; ok && c0 < DP; c0 += wide) {
          if (any_row) {
#pragma unroll 1
            for (int c = 0; c < wide; c += 32) {
              float v[32];
              combined(c0 + c, v);
              if (real) {
                float4* to = meeting + (copy * p.rows + in_copy) * vecs + c / 4;
#pragma unroll
                for (int x = 0; x < 8; ++x) to[x ^ (in_copy & 7)] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
              }
            }
          }
          if (!meet()) break;
          for (int e = threadIdx.x; e < p.rows * vecs; e += 128) {
            const int r = e / vecs, at = e % vecs, from = at ^ (r & 7);
            float4 z = meeting[r * vecs + from];
            for (int y = 1; y < p.copies; ++y) {
              const float4 u = meeting[(y * p.rows + r) * vecs + from];
              z = make_float4(z.x + u.x, z.y + u.y, z.z + u.z, z.w + u.w);
            }
            const int c = c0 + 4 * at;
            if (whole) {
              const int tk = (int)fd_div((uint32_t)r, p.by_group);
              const long long head = (pc.b * (long long)p.drafted + tk) * p.q_heads + pc.hk * p.group + r - tk * p.group;
              if (c < p.dim) *reinterpret_cast<uint2*>(p.o + head * p.dim + c) = make_uint2(pack2<BF16>(z.x, z.y), pack2<BF16>(z.z, z.w));
            } else {
              *reinterpret_cast<float4*>(p.partial + (slot * kTile + r) * DP + c) = z;
            }
          }
          if (c0 + wide < DP && !meet()) break;     // before the next turn writes there
        }
      } else if (any_row) {
        float* part = p.partial + (slot * kTile + in_copy) * DP;
        uint16_t* out = p.o + (((long long)pc.b * p.drafted + tok) * p.q_heads + h) * p.dim;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float v[32];
          combined(c, v);
          if (!real) continue;
          if (whole) {
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              if (c + x < p.dim)
                *reinterpret_cast<uint4*>(out + c + x) = make_uint4(pack2<BF16>(v[x], v[x + 1]), pack2<BF16>(v[x + 2], v[x + 3]),
                                                                    pack2<BF16>(v[x + 4], v[x + 5]), pack2<BF16>(v[x + 6], v[x + 7]));
          } else {
#pragma unroll
            for (int x = 0; x < 32; x += 4) *reinterpret_cast<float4*>(part + c + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          }
        }
      }
      if (!ok) break;
      if (real && !whole && copy == 0) {
        float2* ms = reinterpret_cast<float2*>(p.partial + 2 * (long long)p.runs * kTile * DP);
        ms[slot * kTile + in_copy] = make_float2(top, all);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(ptx::smem_u32(&sh->o_free));
        ptx::mbar_arrive(ptx::smem_u32(&sh->q_empty[n & 1]));    // done with the tree and the place of the queries
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- joining the pieces ------------------------------------------------------------------------------

constexpr int kJoinThreads = 128;

// Block (x, y): rows y * 4 + warp, ... of (sequence, key head, row tile) x.  Writes what the main kernel
// did not: results whose tiles lie in several runs, and zeros where there is no tile.
template <int DP, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeProblem p) {
  __shared__ int words[kJoinThreads / 32];
  __shared__ int first_unit;
  ptx::grid_dependency_wait();
  const int per_tile = p.k_heads * p.row_tiles;
  const int b = blockIdx.x / per_tile, hr = blockIdx.x - b * per_tile, hk = hr / p.row_tiles, rt = hr - hk * p.row_tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = tiles_of(tree_places(p, p.lengths[b]));
  int total = 0, before;
  for (int base = 0; base < p.batch; base += kJoinThreads) {
    const int i = base + threadIdx.x;
    const int sum = block_scan<kJoinThreads>(i < p.batch ? tiles_of(tree_places(p, p.lengths[i])) * per_tile : 0, &before, words);
    if (i == b) first_unit = total + before + hr * tiles;
    total += sum;
  }
  __syncthreads();
  int c0 = 0, c1 = -1;
  if (tiles > 0) {
    const int runs = total < p.runs ? total : p.runs;
    auto run_of = [&](int u) {     // the run that holds unit u
      int c = (int)((float)u * runs / total);
      c = c < 0 ? 0 : c >= runs ? runs - 1 : c;
      while (c > 0 && run_begin(total, runs, c) > u) --c;
      while (c + 1 < runs && run_begin(total, runs, c + 1) <= u) ++c;
      return c;
    };
    c0 = run_of(first_unit);
    c1 = run_of(first_unit + tiles - 1);
    if (c0 == c1) return;                // finished by its run
  }
  const float2* ms = reinterpret_cast<const float2*>(p.partial + 2 * (long long)p.runs * kTile * DP);
  constexpr int V = DP / 32;             // values per lane
  for (int r = blockIdx.y * (kJoinThreads / 32) + warp; r < kTile && rt * kTile + r < p.rows;
       r += gridDim.y * (kJoinThreads / 32)) {
    const int row = rt * kTile + r;
    // the piece of the first run is its run's last (slot 1), the others are their runs' first (slot 0)
    auto slot_of = [&](int c) { return 2 * (long long)c + (c == c0 ? 1 : 0); };
    float top = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, ms[slot_of(c) * kTile + r].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float mu = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[V] = {};
#pragma unroll 8
    for (int c = c0; c <= c1; ++c) {
      const long long slot = slot_of(c) * kTile + r;
      const float2 x = ms[slot];
      const float f = ex2(x.x - mu);
      const float* o = p.partial + slot * DP + lane * V;
      sum = fmaf(x.y, f, sum);
      float v[V];
      if constexpr (V == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(o);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(o);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(v[e], f, acc[e]);
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int tok = (int)fd_div((uint32_t)row, p.by_group), h = hk * p.group + row - tok * p.group;
    uint16_t* out = p.o + (((long long)b * p.drafted + tok) * p.q_heads + h) * p.dim + lane * V;
    if (lane * V < p.dim) {
#pragma unroll
      for (int e = 0; e < V; e += 2)
        *reinterpret_cast<uint32_t*>(out + e) = inv != 0.f ? pack2<BF16>(acc[e] * inv, acc[e + 1] * inv) : 0u;
    }
  }
}

int padded_dim(const TreeProblem& p) { return p.dim <= 64 ? 64 : 128; }

// Runs of a call: one per SM.  (The device decides how many of them get work.)
int64_t tree_bytes(const TreeProblem& p, int runs) { return 2LL * runs * kTile * (padded_dim(p) + 2) * 4; }

template <int DP, bool BF16, bool CAP, bool BIAS>
int32_t launch_tree(const TreeProblem& p, const TreeMaps& maps, int device, cudaStream_t s) {
  static PerDeviceFlag ready;
  auto kernel = tree_attn_kernel<DP, BF16, CAP, BIAS>;
  if (!ready.test(device)) {
    LEGO_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tree_smem<DP>()));
    ready.set(device);
  }
  LEGO_CUDA_TRY(launch_overlapped(kernel, dim3((unsigned)p.runs), dim3(kTreeThreads), tree_smem<DP>(), s, p, maps));
  const int rows = p.rows < kTile ? p.rows : kTile;
  const int rows_per_block = kJoinThreads / 32, blocks = (rows + rows_per_block - 1) / rows_per_block;
  const dim3 grid((unsigned)(p.batch * p.k_heads * p.row_tiles), (unsigned)(blocks < 16 ? blocks : 16));
  LEGO_CUDA_TRY(launch_overlapped(tree_join_kernel<DP, BF16>, grid, dim3(kJoinThreads), 0, s, p));
  return LEGO_OK;
}

template <int DP, bool BF16>
int32_t launch_tree_scores(const TreeProblem& p, const TreeMaps& maps, int device, cudaStream_t s) {
  const bool cap = p.softcap > 0.f, bias = p.slopes || (!cap && !(p.scale > 0.f));   // as in the forward pass
  if (cap)
    return bias ? launch_tree<DP, BF16, true, true>(p, maps, device, s) : launch_tree<DP, BF16, true, false>(p, maps, device, s);
  return bias ? launch_tree<DP, BF16, false, true>(p, maps, device, s) : launch_tree<DP, BF16, false, false>(p, maps, device, s);
}

constexpr int kRunsAtMost = 160;    // the SMs of the device, for a caller that sizes the workspace without one

}  // namespace
}  // namespace lego

using namespace lego;

extern "C" {

int64_t lego_tree_attention_workspace_bytes(const lego_tree_attention_t* d) {
  TreeProblem p;
  const int32_t st = tree_problem(d, &p);
  return st != LEGO_OK ? st : tree_bytes(p, kRunsAtMost);
}

int32_t lego_tree_attention(const lego_tree_attention_t* d, const void* q, const void* k_cache, const void* v_cache,
                            const int32_t* page_table, const int32_t* lengths, const int32_t* parents,
                            const float* slopes, void* o, void* workspace, int64_t workspace_bytes, void* stream) {
  TreeProblem p = {};
  int32_t st = tree_problem(d, &p);
  if (st != LEGO_OK) return st;
  if (!q || !k_cache || !v_cache || !page_table || !lengths || !o || !workspace) return LEGO_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)o | (uintptr_t)workspace) & 15) return LEGO_ERR_ALIGN;
  if (workspace_bytes < tree_bytes(p, kRunsAtMost)) return LEGO_ERR_SIZE;
  DeviceCtx* ctx = device_ctx(&st);
  if (!ctx) return st;
  p.runs = ctx->sm_count < kRunsAtMost ? ctx->sm_count : kRunsAtMost;
  p.table = page_table;
  p.lengths = lengths;
  p.parents = parents;
  p.slopes = slopes;
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k_cache;
  p.v = (const uint16_t*)v_cache;
  p.o = (uint16_t*)o;
  p.partial = (float*)workspace;
  p.status = ctx->status_word;
  const bool bf16 = d->dtype == LEGO_BF16;
  TreeMaps maps = {};
  int rows = 32;
  while (rows >= 8 && p.page_size % rows) rows /= 2;
  if (rows >= 8) {
    EncodeFn enc = encode_fn(&st);
    if (!enc) return st;
    if (make_tmap_heads(enc, &maps.k, bf16, k_cache, p.dim, p.page_size, p.k_heads, p.pages, p.k_stride, rows) == LEGO_OK &&
        make_tmap_heads(enc, &maps.v, bf16, v_cache, p.dim, p.page_size, p.k_heads, p.pages, p.v_stride, rows) == LEGO_OK)
      p.box_rows = rows;
  }
  cudaStream_t s = (cudaStream_t)stream;
  if (p.dim <= 64)
    return bf16 ? launch_tree_scores<64, true>(p, maps, ctx->device, s) : launch_tree_scores<64, false>(p, maps, ctx->device, s);
  return bf16 ? launch_tree_scores<128, true>(p, maps, ctx->device, s) : launch_tree_scores<128, false>(p, maps, ctx->device, s);
}

}  // extern "C"
