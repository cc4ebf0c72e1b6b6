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
// Warps: 0-3 and 4-7 weights of the even and the odd tiles of a piece (each with its own m, sum
// and O, put together at the piece's end), 8-11 loads, 12 MMA issue (13-15 fill up their
// warpgroup).  Each loading lane looks up the place of one row of a tile.  Tiles of cached
// tokens come by TMA, in boxes of as many rows as stand together in a page (a common divisor
// of the page size and 32, at least 8).  The last tiles of a sequence, which hold drafted tokens
// and end somewhere, and pages of other sizes come as 16-byte copies.  Keys that do not exist
// (past the end, of a page number outside the cache, of an unused drafted token) are zeros in
// shared memory and hidden by a mask that the loads leave with the tile.
#include <cuda.h>

#include "attention.cuh"
#include "tma_host.cuh"

namespace lego {
namespace {

constexpr int kMaxDraft = LEGO_MAX_DRAFT;
constexpr int kTreeThreads = 512;
constexpr int kTreeRegs = 128, kTreeMathRegs = 200, kTreeOtherRegs = 56;
static_assert(2 * kTreeMathRegs + 2 * kTreeOtherRegs <= 4 * kTreeRegs, "more registers than the launch has would wait forever");

struct TreeProblem {
  int batch, drafted, q_heads, k_heads, dim, group;
  int pages, page_size, max_pages;
  int rows, row_tiles;          // rows of a key head: drafted * group; tiles of 128 of them
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
  if (!(d->softcap >= 0.f) || d->softcap > 3e38f || !(d->scale >= -3e38f && d->scale <= 3e38f)) return LEGO_ERR_SIZE;
  p->batch = (int)d->batch;
  p->drafted = (int)d->drafted;
  p->q_heads = (int)d->q_heads;
  p->k_heads = (int)d->k_heads;
  p->dim = (int)d->head_dim;
  p->group = p->q_heads / p->k_heads;
  p->rows = p->drafted * p->group;
  p->row_tiles = tiles_of(p->rows);
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
  p->scale = d->scale;
  p->softcap = d->softcap;
  return LEGO_OK;
}

// ---- the line of tiles and its runs --------------------------------------------------------------

// Places of sequence b that may be seen: cached and drafted tokens within the table.
__device__ __forceinline__ int tree_places(const TreeProblem& p, int b) {
  const int len = p.lengths[b];
  if (len < 0) return 0;
  const int room = p.max_pages * p.page_size;      // at most 2^30
  return len < room - p.drafted ? len + p.drafted : room;
}
__device__ __forceinline__ int tree_tiles(const TreeProblem& p, int b) { return tiles_of(tree_places(p, b)); }
__device__ __forceinline__ long long run_begin(long long total, int runs, int c) {
  return total / runs * c + total % runs * c / runs;
}

// Every key of a tile is a cached token within the table.
__device__ __forceinline__ bool all_cached(int tile, int len, int places) {
  const int end = (tile + 1) * kTile;
  return end <= len && end <= places;
}

struct Piece {
  int b, hk, rt;         // sequence, key head, row tile
  int first, last;       // tiles [first, last)
  int tiles;             // of the sequence
};

struct Walk {
  int b, hr, tile;       // next piece: sequence, key head * row tiles + row tile, tile
  long long left;        // tiles of the run still to come
};

__device__ __forceinline__ bool next_piece(const TreeProblem& p, Walk& w, Piece* out) {
  if (w.left <= 0) return false;
  const int tiles = tree_tiles(p, w.b);
  out->b = w.b;
  out->hk = w.hr / p.row_tiles;
  out->rt = w.hr % p.row_tiles;
  out->tiles = tiles;
  out->first = w.tile;
  out->last = w.left < tiles - w.tile ? w.tile + (int)w.left : tiles;
  w.left -= out->last - out->first;
  w.tile = 0;
  if (++w.hr == p.k_heads * p.row_tiles) {
    w.hr = 0;
    do ++w.b;
    while (w.b < p.batch && w.left > 0 && tree_tiles(p, w.b) == 0);
  }
  return true;
}

// Sum over the block's threads of v and what the threads before this one add to; `warps` words of
// shared memory.  Every thread takes part.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* before, long long* words) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) words[warp] = x;
  __syncthreads();
  long long base = 0, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) base += words[i];
    total += words[i];
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
  uint32_t exist[kMaskRing][4];
  uint64_t exist_full[kMaskRing], full[10], empty[10];
  uint64_t tree_full[2], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], odd_done, o_free;
  long long words[16];
  long long start_left;
  int start_b, start_hr, start_tile;
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(ptx::smem_u32(&sh->tree_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->q_full[t]), 4);
      ptx::mbar_init(ptx::smem_u32(&sh->q_empty[t]), 1 + 8);   // the MMAs; the warps done with the tree
      ptx::mbar_init(ptx::smem_u32(&sh->s_full[t]), 1);
      ptx::mbar_init(ptx::smem_u32(&sh->p_full[t]), 4);
      ptx::mbar_init(ptx::smem_u32(&sh->o_full[t]), 1);
    }
    ptx::mbar_init(ptx::smem_u32(&sh->odd_done), 4);
    ptx::mbar_init(ptx::smem_u32(&sh->o_free), 4);
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(ptx::smem_u32(&sh->full[s]), 128);     // every loading thread's copies
      ptx::mbar_init(ptx::smem_u32(&sh->empty[s]), 1);
    }
    for (int s = 0; s < kMaskRing; ++s) ptx::mbar_init(ptx::smem_u32(&sh->exist_full[s]), 4);
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
    const long long per_tile = (long long)p.k_heads * p.row_tiles;
    long long total = 0, before;
    for (int base = 0; base < p.batch; base += kTreeThreads) {
      const int b = base + threadIdx.x;
      total += block_scan<kTreeThreads>(b < p.batch ? tree_tiles(p, b) * per_tile : 0, &before, sh->words);
    }
    const int runs = total < gridDim.x ? (int)total : (int)gridDim.x;
    if ((int)blockIdx.x < runs) {
      const long long u0 = run_begin(total, runs, blockIdx.x), u1 = run_begin(total, runs, blockIdx.x + 1);
      long long passed = 0;
      for (int base = 0; base < p.batch; base += kTreeThreads) {
        const int b = base + threadIdx.x;
        const int tiles = b < p.batch ? tree_tiles(p, b) : 0;
        const long long mine = tiles * per_tile;
        const long long sum = block_scan<kTreeThreads>(mine, &before, sh->words);
        const long long at = u0 - passed - before;
        if (at >= 0 && at < mine) {
          sh->start_b = b;
          sh->start_hr = (int)(at / tiles);
          sh->start_tile = (int)(at % tiles);
          sh->start_left = u1 - u0;
        }
        passed += sum;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  Walk walk = {sh->start_b, sh->start_hr, sh->start_tile, sh->start_left};
  Piece pc;

  if (warp >= 12) {
    ptx::regs_less<kTreeOtherRegs>();
    if (warp == 12 && lane == 0) {
      // ---------------- MMA issue ----------------
      const uint32_t id_s = idesc_of<BF16>(kTile, false), id_o = idesc_of<BF16>(DP, true);
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        if (ok && !ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait)) {
          attn_fail(p.status, abort_flag, code);
          ok = false;
        }
        ptx::tc_fence_after();
      };
      uint32_t pos = 0;                    // ring position of K(i)
      uint32_t weighed[2] = {0, 0};
      for (int n = 0; ok && next_piece(p, walk, &pc); ++n) {
        const int count = pc.last - pc.first;
        const uint32_t q_tile = q_smem + (n & 1) * TILE;
        const int len = p.lengths[pc.b], places = tree_places(p, pc.b);
        wait(&sh->q_full[n & 1], (n >> 1) & 1, 0x720000u);
        for (int i = 0; ok && i <= count; ++i, pos += 2) {
          // the accumulators, and the place of the odd warps' statistics, have been read
          if (i == 1 && n > 0) wait(&sh->o_free, (n - 1) & 1, 0x720001u);
          if (!ok) break;
          if (i < count) {
            const uint32_t slot = pos % NS;
            wait(&sh->full[slot], (pos / NS) & 1, 0x720002u);
            if (!ok) break;
            if (!(p.box_rows && all_cached(pc.first + i, len, places)))
              ptx::fence_proxy_async();      // 16-byte copies go through the generic proxy
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
              ptx::mma_f16_ss(tmem + (i & 1) * kTile, desc_k_major(q_tile, s), desc_k_major(kv_smem + slot * TILE, s), id_s, s != 0);
            ptx::mma_commit(ptx::smem_u32(&sh->s_full[i & 1]));
            ptx::mma_commit(ptx::smem_u32(&sh->empty[slot]));
            if (i == count - 1) ptx::mma_commit(ptx::smem_u32(&sh->q_empty[n & 1]));
          }
          if (i > 0) {
            const uint32_t t = (i - 1) & 1, vpos = pos - 1, slot = vpos % NS;
            wait(&sh->full[slot], (vpos / NS) & 1, 0x720003u);
            wait(&sh->p_full[t], weighed[t] & 1, 0x720004u);
            if (!ok) break;
            if (!(p.box_rows && all_cached(pc.first + i - 1, len, places))) ptx::fence_proxy_async();
            ++weighed[t];
#pragma unroll
            for (int s = 0; s < kTile / 16; ++s)
              ptx::mma_f16_ts(tmem + 2 * kTile + t * DP, tmem + t * kTile + s * 8, desc_mn_major(kv_smem + slot * TILE, s), id_o,
                              i > 2 || s != 0);
            ptx::mma_commit(ptx::smem_u32(&sh->empty[slot]));
            if (i >= count - 1) ptx::mma_commit(ptx::smem_u32(&sh->o_full[t]));
          }
        }
        pos -= 2;     // the last turn had no K
      }
    }
  } else if (warp >= 8) {
    ptx::regs_less<kTreeOtherRegs>();
    // ---------------- loads ----------------
    constexpr int CH = DP / 8, PER = 32 / CH;    // 16-byte pieces of a row; rows per instruction
    const int w = warp - 8, chunk = lane % CH, sub = lane / CH;
    const bool chunk_real = chunk * 8 < p.dim;
    uint32_t issued = 0, tile_no = 0;
    bool ok = true;
    auto bounded = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (lane == 0) ok = ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait);
      ok = __shfl_sync(~0u, ok ? 1 : 0, 0);
      if (!ok && lane == 0) attn_fail(p.status, abort_flag, code);
      return ok;
    };
    for (int n = 0; ok && next_piece(p, walk, &pc); ++n) {
      // the piece's queries and tree
      if (!bounded(&sh->q_empty[n & 1], ((n >> 1) & 1) ^ 1, 0x710000u)) break;
      Tree* tree = &sh->tree[n & 1];
      if (w == 0) {
        grow_tree(p, pc.b, tree, lane);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->tree_full[n & 1]));
      }
      uint8_t* q_tile = smem + (n & 1) * TILE;
#pragma unroll 4
      for (int i = 0; i < 32; i += PER) {
        const int r = w * 32 + i + sub, row = pc.rt * kTile + r;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (row < p.rows && chunk_real) {
          const int t = row / p.group, h = pc.hk * p.group + row % p.group;
          x = *reinterpret_cast<const uint4*>(p.q + pc.b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2] + chunk * 8);
        }
        *reinterpret_cast<uint4*>(q_tile + (chunk >> 3) * kBoxBytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = x;
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->q_full[n & 1]));
      if (!bounded(&sh->tree_full[n & 1], (n >> 1) & 1, 0x710002u)) break;

      const int len = p.lengths[pc.b], places = tree_places(p, pc.b);
      const int* table = p.table + pc.b * p.table_stride;
      // page number of this lane's row of a tile, as the table has it; -1: the row does not exist
      auto page_of = [&](int tile) {
        const int j = tile * kTile + w * 32 + lane;
        if (tile >= pc.last || j >= places) return -1;
        if (j >= len && tree->seen[j - len] == 0) return -1;
        return table[j / p.page_size];
      };
      int page = page_of(pc.first);
      for (int tile = pc.first; ok && tile < pc.last; ++tile, ++tile_no) {
        const bool real = page >= 0 && page < p.pages;
        const int here = real ? page : p.pages;     // past the cache: a TMA box of zeros
        page = page_of(tile + 1);                   // on its way while this tile's copies are issued
        const int in_page = (tile * kTile + w * 32 + lane) % p.page_size;
        const uint32_t word = __ballot_sync(~0u, real);
        const bool boxes = p.box_rows && all_cached(tile, len, places);
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
          if (boxes) {
            if (lane == 0) {      // for the 32 arrivals a warp's copies count as
              ptx::mbar_arrive_expect_tx(full, TILE / 4);
              ptx::mbar_arrive_n(full, 31);
            }
            __syncwarp();
            constexpr int WIDE = DP / 64;
            const int r = lane / WIDE * p.box_rows, c = lane % WIDE;
            const int pg = __shfl_sync(~0u, here, r & 31), at_slot = __shfl_sync(~0u, in_page, r & 31);
            if (r < 32) {
              const int32_t at[5] = {c * 64, at_slot, pc.hk, pg, 0};
              ptx::tma_load_nd(4, dst + c * kBoxBytes + r * 128, g ? &maps.v : &maps.k, at, full);
            }
            continue;
          }
          const long long* st = g ? p.v_stride : p.k_stride;
          const long long row_at = real ? here * st[0] + in_page * st[1] + pc.hk * st[2] : 0;
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
    }
    ptx::cp_async_wait_all();      // leave no copy in flight
  } else {
    ptx::regs_more<kTreeMathRegs>();
    // ---------------- weights, epilogue ----------------
    const int t = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + t * kTile, o_tmem = tmem + lanes + 2 * kTile + t * DP;
    const float by = p.scale * kLog2e;
    const float u_by = CAP ? 2.f * kLog2e * p.scale / p.softcap : 0.f, cap_by = p.softcap * kLog2e;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
      if (!ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, abort_flag, kAttnWait)) ok = false;
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) attn_fail(p.status, abort_flag, code);
        ok = false;
      }
      return ok;
    };
    uint32_t scored = 0, tile_no = 0, mine = 0, paired = 0;
    for (int n = 0; ok && next_piece(p, walk, &pc); ++n) {
      const int count = pc.last - pc.first;
      const int row = pc.rt * kTile + quarter * 32 + lane;
      const bool real = row < p.rows, any_row = pc.rt * kTile + quarter * 32 < p.rows;
      const int tok = real ? row / p.group : 0, h = pc.hk * p.group + (real ? row % p.group : 0);
      if (!wait(&sh->q_full[n & 1], (n >> 1) & 1, 0x740000u)) break;
      const Tree* tree = &sh->tree[n & 1];
      const int len = p.lengths[pc.b];
      const unsigned long long seen = real ? tree->seen[tok] : 0;
      const int depth = tree->depth[tok];
      const float slope = BIAS && p.slopes ? p.slopes[h] * kLog2e : 0.f;
      float m = -INFINITY, sum = 0.f;
      for (int i = t; i < count; i += 2) {
        const int j0 = (pc.first + i) * kTile;
        const uint32_t no = tile_no + i;
        if (!wait(&sh->exist_full[no % kMaskRing], (no / kMaskRing) & 1, 0x740001u) ||
            !wait(&sh->s_full[t], scored & 1, 0x740002u))
          break;
        ++scored;
        ptx::tc_fence_after();
        if (!any_row) {       // idle rows: whatever the product makes of what stands there, nobody reads it
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->p_full[t]));
          continue;
        }
        float s[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) ptx::tmem_ld_32x32(s_tmem + c, reinterpret_cast<uint32_t*>(s) + c);
        uint32_t see[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) see[x] = sh->exist[no % kMaskRing][x];
        ptx::tmem_ld_wait();
        if (CAP || BIAS) {
#pragma unroll
          for (int c = 0; c < kTile; ++c) {
            float z = CAP ? cap_by * tanh_of(s[c] * u_by) : s[c] * by;
            if (BIAS) z = fmaf(-slope, (float)(len - j0 - c) + (float)depth, z);     // cached tokens: none is ahead
            s[c] = z;
          }
        }
        if (j0 + kTile > len) {      // drafted tokens among the keys
          const int at = len - j0;   // column of the first; may be negative
          if (BIAS) {                // they stand where their depth says, not their place
#pragma unroll
            for (int c = 0; c < kTile; ++c) {
              const int d = c - at;
              if (d >= 0 && d < p.drafted)
                s[c] = fmaf(-slope, fabsf((float)(depth - tree->depth[d])) - (float)(depth - d), s[c]);
            }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int shift = 32 * x - at;     // draft token of column 32 x
            uint32_t drafted = shift <= -32 || shift >= 64 ? 0u : shift >= 0 ? (uint32_t)(seen >> shift) : (uint32_t)(seen << -shift);
            see[x] &= bits_upto(at - 1, x) | drafted;
          }
        }
        if ((see[0] & see[1] & see[2] & see[3]) != ~0u) {
#pragma unroll
          for (int c = 0; c < kTile; ++c) s[c] = (see[c >> 5] >> (c & 31)) & 1u ? s[c] : -INFINITY;
        }
        weigh_tile<DP, BF16, CAP || BIAS>(s, by, i == t, &m, &sum, s_tmem, o_tmem);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->p_full[t]));
      }
      tile_no += count;
      if (seen == 0) {        // an unused token: no weight, whatever it would have seen
        m = -INFINITY;
        sum = 0.f;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->q_empty[n & 1]));    // done with the tree
      if (!ok) break;
      if (t == 1) {       // leave (m, sum) where the scores were, for the other warpgroup
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
      const float top = fmaxf(m, m1);
      const float mu = top == -INFINITY ? 0.f : top;
      const float f0 = ex2(m - mu), f1 = ex2(m1 - mu);
      const float all = sum * f0 + sum1 * f1;
      const bool whole = pc.first == 0 && pc.last == pc.tiles;
      const bool has = all > 0.f || all != all;
      const float norm = whole ? (has ? 1.f / all : 0.f) : 1.f;
      const float g0 = sum != 0.f ? f0 * norm : 0.f, g1 = sum1 != 0.f ? f1 * norm : 0.f;
      // of an unfinished piece: the run's last when it starts its sequence, else the run's first
      const long long slot = 2 * (long long)blockIdx.x + (pc.first == 0 ? 1 : 0);
      float* part = p.partial + (slot * kTile + quarter * 32 + lane) * DP;
      uint16_t* out = p.o + (((long long)pc.b * p.drafted + tok) * p.q_heads + h) * p.dim;
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32], o1[32];
        ptx::tmem_ld_32x32(o_tmem + c, o);
        if (count >= 2) ptx::tmem_ld_32x32(o_tmem + DP + c, o1);
        ptx::tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          v[x] = g0 != 0.f ? __uint_as_float(o[x]) * g0 : 0.f;
          if (count >= 2 && g1 != 0.f) v[x] = fmaf(__uint_as_float(o1[x]), g1, v[x]);
        }
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
      if (real && !whole) {
        float2* ms = reinterpret_cast<float2*>(p.partial + 2 * (long long)p.runs * kTile * DP);
        ms[slot * kTile + quarter * 32 + lane] = make_float2(top, all);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&sh->o_free));
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
  __shared__ long long words[kJoinThreads / 32];
  __shared__ long long first_unit;
  ptx::grid_dependency_wait();
  const int per_tile = p.k_heads * p.row_tiles;
  const int b = blockIdx.x / per_tile, hr = blockIdx.x % per_tile, hk = hr / p.row_tiles, rt = hr % p.row_tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = tree_tiles(p, b);
  long long total = 0, before;
  for (int base = 0; base < p.batch; base += kJoinThreads) {
    const int i = base + threadIdx.x;
    const long long sum = block_scan<kJoinThreads>(i < p.batch ? (long long)tree_tiles(p, i) * per_tile : 0, &before, words);
    if (i == b) first_unit = total + before + (long long)hr * tiles;
    total += sum;
  }
  __syncthreads();
  int c0 = 0, c1 = -1;
  if (tiles > 0) {
    const int runs = total < p.runs ? (int)total : p.runs;
    auto run_of = [&](long long u) {     // the run that holds unit u
      int c = (int)((double)u * runs / total);
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
    const int tok = row / p.group, h = hk * p.group + row % p.group;
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
