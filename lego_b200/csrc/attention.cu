// Attention with a cap on the scores, a bias by distance and causal, prefix and document
// masks, forward and backward: one warp per query (forward, dQ) or per key (dK, dV), a
// value of the head per lane and 32 columns.
#include "attention.cuh"

namespace lego {

int32_t attention_problem(const lego_attention_t* d, AttnProblem* p) {
  if (!d) return LEGO_ERR_NULL;
  if (d->dtype != LEGO_F16 && d->dtype != LEGO_BF16) return LEGO_ERR_UNSUPPORTED;
  if (d->batch < 1 || d->q_len < 1 || d->k_len < 1 || d->q_heads < 1 || d->k_heads < 1 || d->head_dim < 1)
    return LEGO_ERR_DIM;
  if (d->q_heads % d->k_heads || d->head_dim % 8 || d->head_dim > 128) return LEGO_ERR_SIZE;
  if (d->q_len > (1 << 30) || d->k_len > (1 << 30) || d->q_heads > 65535 || d->batch > (1 << 24)) return LEGO_ERR_SIZE;
  if (d->batch * d->q_heads > (1LL << 31) / 64 ) return LEGO_ERR_SIZE;
  if (d->documents && d->q_len > d->k_len) return LEGO_ERR_SIZE;
  if (d->prefix && !d->causal) return LEGO_ERR_SIZE;
  if (!(d->softcap >= 0.f) || d->softcap > 3e38f || !(d->scale >= -3e38f && d->scale <= 3e38f)) return LEGO_ERR_SIZE;
  p->batch = (int)d->batch;
  p->q_len = (int)d->q_len;
  p->k_len = (int)d->k_len;
  p->q_heads = (int)d->q_heads;
  p->k_heads = (int)d->k_heads;
  p->dim = (int)d->head_dim;
  p->group = p->q_heads / p->k_heads;
  p->offset = p->k_len - p->q_len;
  p->causal = d->causal != 0;
  p->scale = d->scale;
  p->softcap = d->softcap;
  for (int i = 0; i < 3; ++i) {
    p->q_stride[i] = d->q_stride[i];
    p->k_stride[i] = d->k_stride[i];
    p->v_stride[i] = d->v_stride[i];
    if (d->q_stride[i] % 8 || d->k_stride[i] % 8 || d->v_stride[i] % 8) return LEGO_ERR_ALIGN;
  }
  p->slopes = d->slopes;
  p->prefix = d->prefix;
  p->documents = d->documents;
  p->key_docs = p->query_docs = nullptr;
  return LEGO_OK;
}

int64_t attention_docs_bytes(const AttnProblem& p) {
  return p.documents ? (int64_t)p.batch * (tiles_of(p.k_len) + tiles_of(p.q_len)) * (int64_t)sizeof(int4) : 0;
}

namespace {

// One block of 128 threads per tile: the range of its documents.
__global__ void __launch_bounds__(kTile) attn_docs_kernel(const int* docs, int4* out, int batch, int q_len, int k_len) {
  __shared__ int lo[4], hi[4], neg[4];
  const int nk = tiles_of(k_len), nq = tiles_of(q_len);
  ptx::grid_dependency_wait();
  const int id = blockIdx.x;
  const bool keys = id < batch * nk;
  const int b = keys ? id / nk : (id - batch * nk) / nq;
  const int tile = keys ? id % nk : (id - batch * nk) % nq;
  const int at = (keys ? 0 : k_len - q_len) + tile * kTile + threadIdx.x;   // queries are the last of the keys
  const int d = at < k_len ? docs[(long long)b * k_len + at] : 0;
  const bool real = at < k_len;
  const int mn = __reduce_min_sync(~0u, real && d >= 0 ? d : 0x7fffffff);
  const int mx = __reduce_max_sync(~0u, real && d >= 0 ? d : -1);
  const int ng = __any_sync(~0u, real && d < 0);
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    lo[w] = mn;
    hi[w] = mx;
    neg[w] = ng;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    out[id] = make_int4(min(min(lo[0], lo[1]), min(lo[2], lo[3])), max(max(hi[0], hi[1]), max(hi[2], hi[3])),
                        neg[0] | neg[1] | neg[2] | neg[3], 0);
}

}  // namespace

int32_t attention_docs(AttnProblem* p, void* where, cudaStream_t s) {
  if (!p->documents) return LEGO_OK;
  const long long nk = (long long)p->batch * tiles_of(p->k_len), nq = (long long)p->batch * tiles_of(p->q_len);
  if (nk + nq > 0x7fffffffLL) return LEGO_ERR_SIZE;
  int4* out = reinterpret_cast<int4*>(where);
  LEGO_CUDA_TRY(launch_overlapped(attn_docs_kernel, dim3((unsigned)(nk + nq)), dim3(kTile), 0, s, p->documents, out,
                                  p->batch, p->q_len, p->k_len));
  p->key_docs = out;
  p->query_docs = out + nk;
  return LEGO_OK;
}

namespace {

constexpr int MAXD = 4;  // values of a head per lane

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

__device__ __forceinline__ bool sees(const AttnProblem& p, int b, int pos, int j) {
  if (p.causal && j > pos && !(p.prefix && j < p.prefix[b])) return false;
  if (p.documents) {
    const int d = p.documents[(long long)b * p.k_len + j];
    return d >= 0 && d == p.documents[(long long)b * p.k_len + pos];
  }
  return true;
}

// score of raw product s, and the cap's derivative
__device__ __forceinline__ float score(const AttnProblem& p, float s, int h, int pos, int j, float* bend) {
  s *= p.scale;
  *bend = 1.f;
  if (p.softcap > 0.f) {
    const float t = tanhf(s / p.softcap);
    *bend = 1.f - t * t;
    s = p.softcap * t;
  }
  if (p.slopes) s -= p.slopes[h] * fabsf((float)(pos - j));
  return s;
}

template <typename T>
__device__ __forceinline__ void load_row(const T* r, int dim, int lane, float* v) {
#pragma unroll
  for (int k = 0; k < MAXD; ++k) v[k] = lane + 32 * k < dim ? to_f32(r[lane + 32 * k]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_row(T* r, int dim, int lane, const float* v, float by) {
#pragma unroll
  for (int k = 0; k < MAXD; ++k)
    if (lane + 32 * k < dim) from_f32(v[k] * by, &r[lane + 32 * k]);
}
__device__ __forceinline__ float dot(const float* a, const float* b) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < MAXD; ++k) s += a[k] * b[k];
  return warp_sum(s);
}

struct Row { int b, h, i; };
__device__ __forceinline__ Row row_of(long long id, int heads, int len) {
  Row r;
  r.i = (int)(id % len);
  r.h = (int)(id / len % heads);
  r.b = (int)(id / len / heads);
  return r;
}
template <typename T>
__device__ __forceinline__ const T* at(const void* x, const long long* st, int b, int i, int h) {
  return reinterpret_cast<const T*>(x) + b * st[0] + i * st[1] + h * st[2];
}

template <typename T>
__global__ void dq_kernel(AttnProblem p, const void* q, const void* k, const void* v, const T* o, const float* lse,
                          const T* d_o, T* dq, float* delta) {
  const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (id >= (long long)p.batch * p.q_heads * p.q_len) return;
  const Row r = row_of(id, p.q_heads, p.q_len);
  const int pos = r.i + p.offset;
  const long long flat = (((long long)r.b * p.q_len + r.i) * p.q_heads + r.h) * p.dim;
  float qv[MAXD], dov[MAXD], acc[MAXD] = {}, kv[MAXD], vv[MAXD], bend;
  load_row(at<T>(q, p.q_stride, r.b, r.i, r.h), p.dim, lane, qv);
  load_row(d_o + flat, p.dim, lane, dov);
  load_row(o + flat, p.dim, lane, kv);
  const float del = dot(dov, kv), ls = lse[id];
  if (lane == 0) delta[id] = del;
  if (ls > -INFINITY)
    for (int j = 0; j < p.k_len; ++j) {
      if (!sees(p, r.b, pos, j)) continue;
      load_row(at<T>(k, p.k_stride, r.b, j, r.h / p.group), p.dim, lane, kv);
      load_row(at<T>(v, p.v_stride, r.b, j, r.h / p.group), p.dim, lane, vv);
      const float w = expf(score(p, dot(qv, kv), r.h, pos, j, &bend) - ls);
      const float ds = w * (dot(dov, vv) - del) * bend;
#pragma unroll
      for (int e = 0; e < MAXD; ++e) acc[e] += ds * kv[e];
    }
  store_row(dq + flat, p.dim, lane, acc, p.scale);
}

template <typename T>
__global__ void dkv_kernel(AttnProblem p, const void* q, const void* k, const void* v, const float* lse,
                           const T* d_o, const float* delta, T* dk, T* dv) {
  const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (id >= (long long)p.batch * p.k_heads * p.k_len) return;
  const Row r = row_of(id, p.k_heads, p.k_len);
  float kv[MAXD], vv[MAXD], ak[MAXD] = {}, av[MAXD] = {}, qv[MAXD], dov[MAXD], bend;
  load_row(at<T>(k, p.k_stride, r.b, r.i, r.h), p.dim, lane, kv);
  load_row(at<T>(v, p.v_stride, r.b, r.i, r.h), p.dim, lane, vv);
  for (int h = r.h * p.group; h < (r.h + 1) * p.group; ++h)
    for (int i = 0; i < p.q_len; ++i) {
      if (!sees(p, r.b, i + p.offset, r.i)) continue;
      const long long row = ((long long)r.b * p.q_heads + h) * p.q_len + i;
      load_row(at<T>(q, p.q_stride, r.b, i, h), p.dim, lane, qv);
      load_row(d_o + (((long long)r.b * p.q_len + i) * p.q_heads + h) * p.dim, p.dim, lane, dov);
      const float w = expf(score(p, dot(qv, kv), h, i + p.offset, r.i, &bend) - lse[row]);
      const float ds = w * (dot(dov, vv) - delta[row]) * bend;
#pragma unroll
      for (int e = 0; e < MAXD; ++e) {
        av[e] += w * dov[e];
        ak[e] += ds * qv[e];
      }
    }
  const long long flat = (((long long)r.b * p.k_len + r.i) * p.k_heads + r.h) * p.dim;
  store_row(dk + flat, p.dim, lane, ak, p.scale);
  store_row(dv + flat, p.dim, lane, av, 1.f);
}

template <typename T>
int32_t backward(const AttnProblem& p, const void* q, const void* k, const void* v, const void* o, const float* lse,
                 const void* d_o, void* dq, void* dk, void* dv, float* delta, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.q_heads * p.q_len, keys = (long long)p.batch * p.k_heads * p.k_len;
  dq_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(p, q, k, v, (const T*)o, lse, (const T*)d_o, (T*)dq, delta);
  LEGO_CUDA_TRY(cudaGetLastError());
  dkv_kernel<T><<<(unsigned)((keys + 7) / 8), 256, 0, s>>>(p, q, k, v, lse, (const T*)d_o, delta, (T*)dk, (T*)dv);
  LEGO_CUDA_TRY(cudaGetLastError());
  return LEGO_OK;
}

}  // namespace
}  // namespace lego

using namespace lego;

extern "C" {

int64_t lego_attention_workspace_bytes(const lego_attention_t* d, int32_t backward) {
  AttnProblem p;
  const int32_t st = attention_problem(d, &p);
  if (st != LEGO_OK) return st;
  return attention_docs_bytes(p) + (backward ? (int64_t)p.batch * p.q_heads * p.q_len * 4 : 0);
}

int32_t lego_attention_bwd(const lego_attention_t* d, const void* q, const void* k, const void* v, const void* o,
                           const float* lse, const void* d_o, void* dq, void* dk, void* dv, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  AttnProblem p;
  const int32_t st = attention_problem(d, &p);
  if (st != LEGO_OK) return st;
  if (!q || !k || !v || !o || !lse || !d_o || !dq || !dk || !dv || !workspace) return LEGO_ERR_NULL;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)d_o | (uintptr_t)dq | (uintptr_t)dk |
       (uintptr_t)dv | (uintptr_t)workspace) & 15)
    return LEGO_ERR_ALIGN;
  if (workspace_bytes < lego_attention_workspace_bytes(d, 1)) return LEGO_ERR_SIZE;
  cudaStream_t s = (cudaStream_t)stream;
  return d->dtype == LEGO_F16
             ? backward<__half>(p, q, k, v, o, lse, d_o, dq, dk, dv, (float*)workspace, s)
             : backward<__nv_bfloat16>(p, q, k, v, o, lse, d_o, dq, dk, dv, (float*)workspace, s);
}

}  // extern "C"
