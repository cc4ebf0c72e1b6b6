// Attention of drafted token trees over a paged cache: one warp per query row.
#include "attention.cuh"

namespace lego {
namespace {

constexpr int MAXD = 4;
constexpr int kMaxDraft = LEGO_MAX_DRAFT;

struct TreeProblem {
  int batch, drafted, q_heads, k_heads, dim, group;
  int pages, page_size, max_pages;
  long long table_stride;
  long long q_stride[3], k_stride[3], v_stride[3];
  float scale, softcap;
  const int* table;
  const int* lengths;
  const int* parents;
  const float* slopes;
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

// Ancestors of every drafted token (itself included) as bits, and depths; 0 marks an unused token.
__device__ void ancestors(const TreeProblem& p, int b, unsigned long long* mask, int* depth) {
  for (int t = 0; t < p.drafted; ++t) {
    const int up = p.parents ? p.parents[(long long)b * p.drafted + t] : t - 1;
    const bool root = up == -1, child = up >= 0 && up < t && mask[up] != 0;
    mask[t] = root || child ? (1ull << t) | (child ? mask[up] : 0) : 0;
    depth[t] = child ? depth[up] + 1 : 0;
  }
}

template <typename T>
__global__ void tree_kernel(const __grid_constant__ TreeProblem p, const T* q, const T* kc, const T* vc, T* o) {
  __shared__ unsigned long long mask[kMaxDraft];
  __shared__ int depth[kMaxDraft];
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) ancestors(p, b, mask, depth);
  __syncthreads();
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= p.drafted) return;
  const int ctx = p.lengths[b], hk = h / p.group;
  const T* qr = q + b * p.q_stride[0] + t * p.q_stride[1] + h * p.q_stride[2];
  float qv[MAXD], acc[MAXD] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < MAXD; ++e) qv[e] = lane + 32 * e < p.dim ? to_f32(qr[lane + 32 * e]) : 0.f;
  const long long room = (long long)p.max_pages * p.page_size;
  const long long end = ctx < 0 || !mask[t] ? 0 : ((long long)ctx + p.drafted < room ? (long long)ctx + p.drafted : room);
  for (long long j = 0; j < end; ++j) {
    int at = (int)j;
    if (j >= ctx) {
      const int a = (int)(j - ctx);
      if (!((mask[t] >> a) & 1)) continue;
      at = ctx + depth[a];
    }
    const int page = p.table[b * p.table_stride + j / p.page_size];
    if (page < 0 || page >= p.pages) continue;
    const T* kr = kc + page * p.k_stride[0] + (j % p.page_size) * p.k_stride[1] + hk * p.k_stride[2];
    const T* vr = vc + page * p.v_stride[0] + (j % p.page_size) * p.v_stride[1] + hk * p.v_stride[2];
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < MAXD; ++e) s += lane + 32 * e < p.dim ? qv[e] * to_f32(kr[lane + 32 * e]) : 0.f;
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(~0u, s, w);
    s *= p.scale;
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    if (p.slopes) s -= p.slopes[h] * fabsf((float)(ctx + depth[t] - at));
    const float mn = fmaxf(m, s);
    const float a = mn == -INFINITY ? 1.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < MAXD; ++e) acc[e] = acc[e] * a + (lane + 32 * e < p.dim ? w * to_f32(vr[lane + 32 * e]) : 0.f);
    m = mn;
  }
  T* orow = o + (((long long)b * p.drafted + t) * p.q_heads + h) * p.dim;
  const float by = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < MAXD; ++e)
    if (lane + 32 * e < p.dim) from_f32(acc[e] * by, &orow[lane + 32 * e]);
}

}  // namespace
}  // namespace lego

using namespace lego;

extern "C" {

int64_t lego_tree_attention_workspace_bytes(const lego_tree_attention_t* d) {
  TreeProblem p;
  const int32_t st = tree_problem(d, &p);
  return st != LEGO_OK ? st : 0;
}

int32_t lego_tree_attention(const lego_tree_attention_t* d, const void* q, const void* k_cache, const void* v_cache,
                            const int32_t* page_table, const int32_t* lengths, const int32_t* parents,
                            const float* slopes, void* o, void* workspace, int64_t workspace_bytes, void* stream) {
  TreeProblem p;
  const int32_t st = tree_problem(d, &p);
  if (st != LEGO_OK) return st;
  if (!q || !k_cache || !v_cache || !page_table || !lengths || !o) return LEGO_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)o) & 15) return LEGO_ERR_ALIGN;
  if (workspace_bytes < lego_tree_attention_workspace_bytes(d)) return LEGO_ERR_SIZE;
  (void)workspace;
  p.table = page_table;
  p.lengths = lengths;
  p.parents = parents;
  p.slopes = slopes;
  const dim3 grid((p.drafted + 3) / 4, p.q_heads, p.batch);
  if (d->dtype == LEGO_F16)
    tree_kernel<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(p, (const __half*)q, (const __half*)k_cache,
                                                                (const __half*)v_cache, (__half*)o);
  else
    tree_kernel<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(
        p, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k_cache, (const __nv_bfloat16*)v_cache, (__nv_bfloat16*)o);
  LEGO_CUDA_TRY(cudaGetLastError());
  return LEGO_OK;
}

}  // extern "C"
