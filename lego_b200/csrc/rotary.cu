// Rotary positions: pairs of a head's values turned by position * frequency.
//
// Every value is read once and written once and nothing else is large, so the kernel is
// bound by memory; what must not cost is the angle.  A block takes a few tokens: its
// threads first put the tokens' cosines and sines (one pair of a token per thread and
// step, shared by all heads of both tensors) into shared memory, then turn the heads with
// 16-byte loads and stores.  The angle is position * frequency in 64 bits, reduced to a
// fraction of a turn there (positions of 10^5 and more leave no digits of a 32-bit angle),
// sine and cosine of the fraction are taken in 32 bits.
//
// 2 x 8192 tokens, 40 heads of 128: 55.5 us in 16 bits (6.05 TB/s), 105 us in 32 (6.4); 64 tokens 3 us.
#include "attention.cuh"
#include "ptx_sm100.cuh"

namespace lego {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxTokens = 8;      // tokens per block at most

struct RotArgs {
  const void* x[2];
  void* y[2];
  long long in_stride[2][3];
  int heads[2];
  const void* positions;
  long long pos_stride[2];
  const double* freqs;
  long long tokens;       // batch * length
  long long length;
  int dim, half;          // head_dim, rotary_dim / 2
  int pos64, inverse;
  float scale;
  int per_block;          // tokens per block
  FastDiv by_units, by_heads;      // units of a head; heads of both tensors
};

// VEC values of T at once: 16 bytes where the tensors' alignment and the borders inside a head allow it, else
// 8 bytes of a 16-bit type (heads of 80 turned by half: 102 -> 48 us for 2 x 8192 tokens x 40 heads), else one value.
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  Pack<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(&r) = __ldcs(reinterpret_cast<const uint2*>(p));
  else r.v[0] = *p;
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& r) {
  if constexpr (VEC * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&r));
  else if constexpr (VEC * sizeof(T) == 8) __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&r));
  else *p = r.v[0];
}

// A unit of work is two packs of VEC values, or one pack of whole pairs where neighbours turn together
// (interleaved, VEC > 1): values of the rotated part and their partners, or of the part that is
// copied (which ends with a pack twice where its packs are odd in number).  A thread has kRotUnits units
// under way: all their loads, then the turns and stores; with a branch for copies before the
// loads, heads turned by half moved 3.2 TB/s where whole ones moved 5.
constexpr int kRotUnits = 4;
constexpr __host__ __device__ bool rot_two_packs(bool half, int vec) { return half || vec == 1; }
__host__ __device__ inline int rot_units(bool half, int vec, int pairs) { return rot_two_packs(half, vec) ? pairs / vec : 2 * pairs / vec; }
__host__ __device__ inline int copy_units(bool half, int vec, int values) {
  return rot_two_packs(half, vec) ? (values / vec + 1) / 2 : values / vec;
}

template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotArgs a) {
  extern __shared__ __align__(16) float2 turn[];   // [token][pair in the order below] (cos, sin), scaled
  __shared__ long long row[2][kRotMaxTokens];      // where a token's heads start in either input
  ptx::launch_dependents();
  ptx::grid_dependency_wait();
  const long long t0 = (long long)blockIdx.x * a.per_block;
  const int nt = (int)(a.tokens - t0 < a.per_block ? a.tokens - t0 : a.per_block);

  // A unit's pairs, two at a time, stand as far apart as there are units: the lanes of a warp then read
  // neighbouring 16 bytes, where a unit's own would be in four lanes' way (2 x 8192 tokens x 40 heads
  // of 128, bf16: 65 -> 55.5 us, 6.05 TB/s).
  constexpr bool TWO = rot_two_packs(HALF, VEC);
  constexpr int PAIRS = TWO ? VEC : VEC / 2;
  const int turned = rot_units(HALF, VEC, a.half);
  __shared__ long long place[kRotMaxTokens];
  if (threadIdx.x < nt) {
    const long long b = (t0 + threadIdx.x) / a.length, s = (t0 + threadIdx.x) - b * a.length;
    row[0][threadIdx.x] = b * a.in_stride[0][0] + s * a.in_stride[0][1];
    row[1][threadIdx.x] = b * a.in_stride[1][0] + s * a.in_stride[1][1];
    place[threadIdx.x] = b * a.pos_stride[0] + s * a.pos_stride[1];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nt * a.half; i += kRotThreads) {
    const int t = i / a.half, p = i - t * a.half;
    const long long at = place[t];
    const double pos = a.pos64 ? (double)reinterpret_cast<const long long*>(a.positions)[at]
                               : (double)reinterpret_cast<const int*>(a.positions)[at];
    double turns = pos * a.freqs[p] * 0.15915494309189533577;   // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.0f * (float)turns, &sn, &cs);
    const int u = p / PAIRS, e = p - u * PAIRS;
    turn[t * a.half + (PAIRS > 1 ? ((e >> 1) * turned + u) * 2 + (e & 1) : p)] =
        make_float2(a.scale * cs, a.scale * (a.inverse ? -sn : sn));
  }
  __syncthreads();

  const int per_head = turned + copy_units(HALF, VEC, a.dim - 2 * a.half);
  const int h0 = a.heads[0], heads = h0 + a.heads[1];
  const int units = nt * heads * per_head;
  for (int i0 = threadIdx.x; i0 < units; i0 += kRotUnits * kRotThreads) {
    Pack<T, VEC> x1[kRotUnits], x2[TWO ? kRotUnits : 1];
    T* y1[kRotUnits];
    int c2[kRotUnits], cs_at[kRotUnits];      // from the first pack to the second; angles, -1: a copy
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      const int i = i0 + k * kRotThreads;
      if (i >= units) break;
      const int head_id = (int)fd_div((uint32_t)i, a.by_units), u = i - head_id * per_head;
      const int t = (int)fd_div((uint32_t)head_id, a.by_heads), hh = head_id - t * heads;
      const bool second = hh >= h0, turn_it = u < turned;
      const int h = second ? hh - h0 : hh;
      int c1;
      if (TWO) {
        const int rest = 2 * a.half + 2 * (u - turned) * VEC;
        c1 = !turn_it ? rest : HALF ? u * VEC : 2 * u;
        c2[k] = !turn_it ? (rest + VEC < a.dim ? VEC : 0) : HALF ? a.half : 1;
      } else {
        c1 = u * VEC;
      }
      cs_at[k] = !turn_it ? -1 : t * a.half + (PAIRS > 1 ? 2 * u : u);
      const T* x = reinterpret_cast<const T*>(second ? a.x[1] : a.x[0]) + row[second ? 1 : 0][t] +
                   h * (second ? a.in_stride[1][2] : a.in_stride[0][2]) + c1;
      y1[k] = reinterpret_cast<T*>(second ? a.y[1] : a.y[0]) + ((t0 + t) * (second ? a.heads[1] : h0) + h) * a.dim + c1;
      x1[k] = load_pack<T, VEC>(x);
      if constexpr (TWO) x2[k] = load_pack<T, VEC>(x + c2[k]);
    }
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      if (i0 + k * kRotThreads >= units) break;
      if (cs_at[k] >= 0) {
        const float2* cs = turn + cs_at[k];
        float2 w[PAIRS];
        if constexpr (PAIRS > 1) {
#pragma unroll
          for (int e = 0; e < PAIRS; e += 2) {
            const float4 z = *reinterpret_cast<const float4*>(cs + e * turned);
            w[e] = make_float2(z.x, z.y);
            w[e + 1] = make_float2(z.z, z.w);
          }
        } else {
          w[0] = cs[0];
        }
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          T* v1 = TWO ? &x1[k].v[e] : &x1[k].v[2 * e];
          T* v2 = TWO ? &x2[TWO ? k : 0].v[e] : &x1[k].v[2 * e + 1];
          const float f1 = to_f32(*v1), f2 = to_f32(*v2);
          from_f32(f1 * w[e].x - f2 * w[e].y, v1);
          from_f32(f2 * w[e].x + f1 * w[e].y, v2);
        }
      }
      store_pack<T, VEC>(y1[k], x1[k]);
      if constexpr (TWO) store_pack<T, VEC>(y1[k] + c2[k], x2[k]);
    }
  }
}

template <typename T, int VEC>
cudaError_t launch_rotary(const RotArgs& a, bool half, long long blocks, size_t smem, cudaStream_t s) {
  return half ? launch_overlapped(rotary_kernel<T, VEC, true>, dim3((unsigned)blocks), dim3(kRotThreads), smem, s, a)
              : launch_overlapped(rotary_kernel<T, VEC, false>, dim3((unsigned)blocks), dim3(kRotThreads), smem, s, a);
}

template <typename T>
cudaError_t launch_rotary_type(const RotArgs& a, bool half, int vec, long long blocks, size_t smem, cudaStream_t s) {
  if (vec == (int)(16 / sizeof(T))) return launch_rotary<T, 16 / sizeof(T)>(a, half, blocks, smem, s);
  if constexpr (sizeof(T) == 2)
    if (vec == 4) return launch_rotary<T, 4>(a, half, blocks, smem, s);
  return launch_rotary<T, 1>(a, half, blocks, smem, s);
}

}  // namespace
}  // namespace lego

using namespace lego;

extern "C" int32_t lego_rotary(const lego_rotary_t* d, const void* x0, const void* x1, void* y0, void* y1,
                               const void* positions, const double* freqs, void* stream) {
  if (!d) return LEGO_ERR_NULL;
  if (d->dtype < LEGO_F16 || d->dtype > LEGO_F32) return LEGO_ERR_UNSUPPORTED;
  if (d->pairs != LEGO_PAIRS_HALF && d->pairs != LEGO_PAIRS_INTERLEAVED) return LEGO_ERR_UNSUPPORTED;
  if (d->position_bytes != 4 && d->position_bytes != 8) return LEGO_ERR_UNSUPPORTED;
  if (d->batch < 0 || d->length < 0 || d->heads[0] < 0 || d->heads[1] < 0) return LEGO_ERR_DIM;
  if (d->head_dim < 1 || d->head_dim > 1024 || d->rotary_dim < 2 || d->rotary_dim > d->head_dim || (d->rotary_dim & 1))
    return LEGO_ERR_SIZE;
  if (d->heads[0] > 65536 || d->heads[1] > 65536) return LEGO_ERR_SIZE;
  if (d->batch == 0 || d->length == 0 || d->heads[0] + d->heads[1] == 0) return LEGO_OK;
  if (!positions || !freqs) return LEGO_ERR_NULL;
  if ((d->heads[0] && (!x0 || !y0)) || (d->heads[1] && (!x1 || !y1))) return LEGO_ERR_NULL;
  if (d->batch > (1LL << 40) / d->length) return LEGO_ERR_OVERFLOW;

  RotArgs a = {};
  const void* xs[2] = {x0, x1};
  void* ys[2] = {y0, y1};
  const int eb = d->dtype == LEGO_F32 ? 4 : 2;
  const bool half = d->pairs == LEGO_PAIRS_HALF;
  // whole packs: every row of a head starts on a pack's boundary and no pack holds the border
  // between the halves, or between the rotated and the copied part
  int64_t borders = d->head_dim | (half ? d->rotary_dim / 2 : d->rotary_dim);      // in values; their common powers of two count
  uint64_t places = 0;                                                             // in bytes
  for (int i = 0; i < 2; ++i) {
    a.x[i] = xs[i];
    a.y[i] = ys[i];
    a.heads[i] = (int)d->heads[i];
    if (!d->heads[i]) continue;
    if (((uintptr_t)xs[i] | (uintptr_t)ys[i]) & (uintptr_t)(eb - 1)) return LEGO_ERR_ALIGN;
    places |= (uintptr_t)xs[i] | (uintptr_t)ys[i];
    for (int k = 0; k < 3; ++k) {
      a.in_stride[i][k] = d->stride[i][k];
      borders |= d->stride[i][k];
    }
  }
  auto fits = [&](int values) { return borders % values == 0 && places % (uint64_t)(values * eb) == 0; };
  const int vec = fits(16 / eb) ? 16 / eb : eb == 2 && fits(4) ? 4 : 1;
  a.positions = positions;
  a.pos_stride[0] = d->position_stride[0];
  a.pos_stride[1] = d->position_stride[1];
  a.freqs = freqs;
  a.tokens = d->batch * d->length;
  a.length = d->length;
  a.dim = (int)d->head_dim;
  a.half = (int)d->rotary_dim / 2;
  a.pos64 = d->position_bytes == 8;
  a.inverse = d->inverse != 0;
  a.scale = d->scale;
  a.per_block = 1;
  while (a.per_block < kRotMaxTokens && a.tokens / (2 * a.per_block) >= 148 * 8) a.per_block *= 2;
  a.by_units = make_fastdiv((uint64_t)(rot_units(half, vec, a.half) + copy_units(half, vec, a.dim - 2 * a.half)));
  a.by_heads = make_fastdiv((uint64_t)(a.heads[0] + a.heads[1]));
  const long long blocks = (a.tokens + a.per_block - 1) / a.per_block;
  if (blocks > 0x7fffffffLL) return LEGO_ERR_SIZE;
  const size_t smem = (size_t)a.per_block * a.half * sizeof(float2);   // at most 8 x 512 x 8 = 32 KiB
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (d->dtype == LEGO_F16) e = launch_rotary_type<__half>(a, half, vec, blocks, smem, s);
  else if (d->dtype == LEGO_BF16) e = launch_rotary_type<__nv_bfloat16>(a, half, vec, blocks, smem, s);
  else e = launch_rotary_type<float>(a, half, vec, blocks, smem, s);
  LEGO_CUDA_TRY(e);
  return LEGO_OK;
}
