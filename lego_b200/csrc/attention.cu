// What the forward and the backward pass of attention share on the host: the checks of a
// call, and the summaries of the documents by which tiles nobody sees are left out.
#include "attention.cuh"

namespace lego {

bool scores_ok(float scale, float softcap) {
  const float most = 1e30f;      // what is made of them stays finite
  if (!(softcap >= 0.f && softcap < most) || !(scale > -most && scale < most)) return false;
  return softcap == 0.f || (scale < most * softcap && scale > -most * softcap);
}

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
  if (!scores_ok(d->scale, d->softcap)) return LEGO_ERR_SIZE;
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

}  // namespace lego
