// Internal declarations of the paged KV cache (csrc/paged.cu: entry points,
// workspaces, append; csrc/paged_attn.cu: attention).
#pragma once

#include "common.cuh"
#include "ptx.cuh"

namespace ortc {

// The cache and the batch of one call, as the kernels see them.
struct PagedView {
  void* key = nullptr;
  void* value = nullptr;
  const int32_t* table = nullptr;
  const int32_t* cu = nullptr;
  const int32_t* past = nullptr;
  int64_t page_elems = 0;  // elements of a page: page_size * kv_heads * D
  int row_elems = 0;       // elements of a token's row: kv_heads * D
  int num_pages = 0, page_size = 0, max_pages = 0, batch = 0;
  int kv_heads = 0, D = 0, type = 0;
  int num_tokens = 0;
  int* err = nullptr;  // host-mapped error word
};

// Sequence b of a call: its first token, its token count and its past; no
// tokens when its lengths do not fit (see fits), a count of -1 when they fall.  Callers
// pass no sequence behind the first whose lengths fall: those before it share no token.
struct PagedSeq {
  int row0, count, past;
};

__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedView& v, int b, int max_seq, int shared) {
  const int c0 = v.cu[b], c1 = v.cu[b + 1], past = v.past[b];
  PagedSeq s = {c0, c1 - c0, past};
  if (c0 >= 0 && c1 == c0) {  // no tokens: nothing to check
    s.count = 0;
    return s;
  }
  // (the shared prefix is worked out for the tokens up to cu[batch])
  const bool fits = c0 >= 0 && c0 < c1 && c1 <= v.num_tokens && c1 <= v.cu[v.batch] &&
                    c1 - c0 <= max_seq && past >= 0 && past >= shared &&
                    (int64_t)past + (c1 - c0) <= (int64_t)v.max_pages * v.page_size;
  if (!fits) {
#ifdef __CUDA_ARCH__
    record_error(v.err, KERR_PAGED_LENGTH);
#endif
    s.count = c1 < c0 ? -1 : 0;
  }
  return s;
}

// The sequence that token t belongs to: the first that ends behind t, `batch`
// when there is none or a sequence before it falls.  Whole warp; the lengths of 32
// sequences a step.
__device__ __forceinline__ int paged_find(const PagedView& v, int t) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < v.batch; b0 += 32) {
    const bool in = b0 + lane < v.batch;
    const int c0 = in ? v.cu[b0 + lane] : 0, c1 = in ? v.cu[b0 + lane + 1] : 0;
    const unsigned m = __ballot_sync(0xffffffffu, in && c1 > t);
    const unsigned f = __ballot_sync(0xffffffffu, c1 < c0);
    if (f && (!m || __ffs(f) < __ffs(m))) break;
    if (m) return b0 + __ffs(m) - 1;
  }
  return v.batch;
}

// floor(x / d) for 0 <= x < 2^31.
struct FastDiv {
  uint32_t mul = 0, shift = 0;  // mul 0: a power of two
  __host__ void set(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    if ((1ull << s) == d) {
      mul = 0, shift = s;
    } else {  // ceil(2^(31 + s) / d) < 2^32: exact for 31-bit x
      mul = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
      shift = s - 1;
    }
  }
  __device__ __forceinline__ int div(int x) const {
    return mul ? (int)(__umulhi((uint32_t)x, mul) >> shift) : x >> shift;
  }
};

// The first bytes of a workspace, zero between calls.
constexpr size_t kTicketBytes = 4096;

struct PagedAttnArgs {
  PagedView c;
  const float* q = nullptr;
  int64_t q_stride = 0;
  float* out = nullptr;
  int heads = 0, group = 1, max_seq = 0, shared = 0;
  int window = 0;  // 0: no window
  float scale = 1.0f, softcap = 0.0f;
};
size_t paged_attention_scratch(const PagedAttnArgs& a, int sm_count);
int launch_paged_attention(const PagedAttnArgs& a, void* scratch, int sm_count, cudaStream_t st,
                           int64_t* launches);

}  // namespace ortc
