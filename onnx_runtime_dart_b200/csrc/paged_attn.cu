// Attention over the paged KV cache, one warp per (token, query head).
#include <cuda_bf16.h>

#include "paged.cuh"

namespace ortc {
namespace {

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

// Lane l owns features l, l + 32, ...; the keys are walked in order with the
// running maximum and sum of the softmax.
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  const PagedView& c = a.c;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0)  // sequences that no token of the call reaches are checked too
    for (int b = threadIdx.x; b < c.batch; b += blockDim.x) paged_seq(c, b, a.max_seq, a.shared);
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= (int64_t)c.num_tokens * a.heads) return;
  const int t = (int)(w / a.heads), h = (int)(w % a.heads), g = h / a.group;
  const int b = paged_find(c, t);
  if (b >= c.batch) return;
  const PagedSeq s = paged_seq(c, b, a.max_seq, a.shared);
  if (t < s.row0 || t >= s.row0 + s.count) return;
  const int pos = s.past + t - s.row0;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < 4; i++)
    q[i] = lane + 32 * i < c.D ? a.q[t * a.q_stride + (int64_t)h * c.D + lane + 32 * i] : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = a.window ? max(0, pos - a.window + 1) : 0; j <= pos; j++) {
    const int64_t off = paged_row(c, j < a.shared ? 0 : b, j);
    if (off < 0) continue;
    const T* kr = static_cast<const T*>(c.key) + off + g * c.D;
    const T* vr = static_cast<const T*>(c.value) + off + g * c.D;
    float d = 0.f;
    for (int i = 0; i < 4; i++)
      if (lane + 32 * i < c.D) d = fmaf(q[i], widen(kr[lane + 32 * i]), d);
    for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(~0u, d, x);
    d *= a.scale;
    if (a.softcap > 0.f) d = a.softcap * tanhf(d / a.softcap);
    const float mn = fmaxf(m, d);
    const float corr = m == mn ? 1.f : expf(m - mn), p = expf(d - mn);
    l = l * corr + p;
    m = mn;
    for (int i = 0; i < 4; i++)
      if (lane + 32 * i < c.D) o[i] = fmaf(p, widen(vr[lane + 32 * i]), o[i] * corr);
  }
  for (int i = 0; i < 4; i++)
    if (lane + 32 * i < c.D)
      a.out[((int64_t)t * a.heads + h) * c.D + lane + 32 * i] = l == 0.f ? 0.f : o[i] / l;
}

}  // namespace

size_t paged_attention_scratch(const PagedAttnArgs&, int) { return 0; }

int launch_paged_attention(const PagedAttnArgs& a, void*, int, cudaStream_t st,
                           int64_t* launches) {
  const unsigned grid = (unsigned)(((int64_t)a.c.num_tokens * a.heads + 3) / 4);
  if (a.c.type == ORT_CUDA_CACHE_F32)
    paged_attn_kernel<float><<<grid, 128, 0, st>>>(a);
  else if (a.c.type == ORT_CUDA_CACHE_F16)
    paged_attn_kernel<__half><<<grid, 128, 0, st>>>(a);
  else
    paged_attn_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
  ORTC_CUDA(cudaGetLastError());
  (*launches)++;
  return ORT_CUDA_OK;
}

}  // namespace ortc
