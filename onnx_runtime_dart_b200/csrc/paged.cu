// The paged KV cache: C entry points (include/ort_cuda.h), the workspaces of
// its attention, and the append kernel.
#include <algorithm>
#include <climits>
#include <cmath>
#include <map>
#include <memory>
#include <mutex>
#include <type_traits>
#include <utility>
#include <vector>

#include <cuda_bf16.h>

#include "paged.cuh"

namespace ortc {

// ---- workspaces ----------------------------------------------------------------
// A call's workspace belongs to the stream it is launched on, or to the graph
// being captured on that stream: calls on two streams, and two captured graphs
// replayed at once, never share one.  Streams are told apart by their ids: a handle
// may come again when its stream is destroyed, even with work of it still to run.  A
// stream's workspace is kept until the session closes or its handle comes again.  A
// graph's workspace is handed back when the graph and everything instantiated from it
// are gone (a CUDA user object), and is reused by later captures.  The first
// kTicketBytes are zero between calls.
struct PagedScratch {
  struct Buf {
    void* p = nullptr;
    size_t bytes = 0;
  };
  struct Pool {  // outlives the session while a graph still holds a workspace
    std::mutex m;
    std::vector<Buf> idle;
  };
  struct OfStream : Buf {
    cudaStream_t handle = nullptr;
  };
  std::shared_ptr<Pool> pool = std::make_shared<Pool>();
  std::vector<void*> all;
  std::map<unsigned long long, OfStream> streams;  // by the stream's id
  unsigned long long capture = 0;  // the capture `captured` belongs to
  std::map<cudaStream_t, Buf> captured;
};

namespace {

struct GraphHold {
  std::shared_ptr<PagedScratch::Pool> pool;
  PagedScratch::Buf buf;
};

void CUDART_CB release_hold(void* p) {
  auto* h = static_cast<GraphHold*>(p);
  {
    std::lock_guard<std::mutex> lock(h->pool->m);
    h->pool->idle.push_back(h->buf);
  }
  delete h;
}

// Allocating and freeing are allowed in its scope while a stream of this thread, this
// one or another, is being captured.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// A new zeroed workspace.
int new_buf(PagedScratch* w, size_t bytes, PagedScratch::Buf* out) {
  RelaxedCapture relaxed;
  PagedScratch::Buf b;
  cudaStream_t st = nullptr;
  cudaError_t e = cudaMalloc(&b.p, bytes);
  if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
  if (e == cudaSuccess) e = cudaMemsetAsync(b.p, 0, kTicketBytes, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (st) cudaStreamDestroy(st);
  if (e != cudaSuccess && b.p) cudaFree(b.p);
  if (e != cudaSuccess) return cuda_fail(e, "paged attention workspace");
  b.bytes = bytes;
  w->all.push_back(b.p);
  *out = b;
  return ORT_CUDA_OK;
}

// Frees a workspace.  cudaFree waits for what still runs on it.
int free_buf(PagedScratch* w, PagedScratch::Buf* b) {
  if (!b->p) return ORT_CUDA_OK;
  RelaxedCapture relaxed;
  ORTC_CUDA(cudaFree(b->p));
  w->all.erase(std::find(w->all.begin(), w->all.end(), b->p));
  *b = PagedScratch::Buf();
  return ORT_CUDA_OK;
}

int paged_scratch(ort_cuda_session* s, size_t bytes, void** out) {
  *out = nullptr;
  if (bytes == 0) return ORT_CUDA_OK;
  if (!s->paged) s->paged = new PagedScratch();
  PagedScratch* w = s->paged;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  ORTC_CUDA(cudaStreamGetCaptureInfo_v2(s->stream, &status, &id, &graph, nullptr, nullptr));
  if (status == cudaStreamCaptureStatusNone) {
    unsigned long long stream = 0;  // (not to be had while it is captured)
    ORTC_CUDA(cudaStreamGetId(s->stream, &stream));
    auto at = w->streams.find(stream);
    if (at == w->streams.end()) {
      // another stream of this handle is gone, and its workspace goes too (the handle of
      // the per-thread stream is one stream for every host thread)
      for (auto i = w->streams.begin(); i != w->streams.end();)
        if (i->second.handle == s->stream && s->stream != cudaStreamPerThread) {
          const int rc = free_buf(w, &i->second);
          if (rc) return rc;
          i = w->streams.erase(i);
        } else {
          ++i;
        }
      at = w->streams.emplace(stream, PagedScratch::OfStream()).first;
      at->second.handle = s->stream;
    }
    PagedScratch::Buf& b = at->second;
    if (bytes > b.bytes) {
      if (b.p) {
        RelaxedCapture relaxed;
        ORTC_CUDA(cudaStreamSynchronize(s->stream));
      }
      int rc = free_buf(w, &b);
      if (rc) return rc;
      rc = new_buf(w, bytes, &b);
      if (rc) return rc;
    }
    *out = b.p;
    return ORT_CUDA_OK;
  }
  ORTC_CHECK(status == cudaStreamCaptureStatusActive, ORT_CUDA_ERR_CUDA,
             "paged attention: the stream's capture was invalidated");
  if (w->capture != id) {
    w->captured.clear();
    w->capture = id;
  }
  PagedScratch::Buf& b = w->captured[s->stream];
  if (bytes > b.bytes) {
    PagedScratch::Buf got;
    {
      std::lock_guard<std::mutex> lock(w->pool->m);
      auto& idle = w->pool->idle;
      for (size_t i = 0; i < idle.size(); i++)
        if (idle[i].bytes >= bytes) {
          got = idle[i];
          idle.erase(idle.begin() + i);
          break;
        }
    }
    if (!got.p) {
      const int rc = new_buf(w, bytes, &got);
      if (rc) return rc;
    }
    auto* hold = new GraphHold{w->pool, got};
    cudaUserObject_t obj = nullptr;
    cudaError_t e = cudaUserObjectCreate(&obj, hold, release_hold, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
      release_hold(hold);
      return cuda_fail(e, "cudaUserObjectCreate");
    }
    e = cudaGraphRetainUserObject(graph, obj, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) {
      cudaUserObjectRelease(obj, 1);
      return cuda_fail(e, "cudaGraphRetainUserObject");
    }
    b = got;
  }
  *out = b.p;
  return ORT_CUDA_OK;
}

}  // namespace

void paged_free(ort_cuda_session* s) {
  if (!s->paged) return;
  for (void* p : s->paged->all) cudaFree(p);
  delete s->paged;
  s->paged = nullptr;
}

// ---- append ----------------------------------------------------------------------
namespace {

struct AppendArgs {
  PagedView c;
  const float* q = nullptr;
  const float* k = nullptr;
  const float* v = nullptr;
  int64_t q_stride = 0, k_stride = 0, v_stride = 0;
  float* q_out = nullptr;
  int heads = 0;  // query heads, 0 without Q
  const float* cos = nullptr;
  const float* sin = nullptr;
  int half = 0, interleaved = 0;
  int64_t max_pos = 0;
  // filled by the launch
  FastDiv page_div, piece_div;
  int parts = 1;  // CTAs of a token
};

// a b - c d (or + c d), as computed in double and rounded to fp32: the products as
// pairs of floats (exact), their sum with its error.  About 13 fp32 instructions in
// place of 4 conversions to and from double, which run at an eighth of the rate.
// `odd`: rounded to odd instead, so that rounding on to 16 bits rounds once.
template <bool PLUS, bool ODD>
__device__ __forceinline__ float rope_sum(float a, float b, float c, float d) {
  const float p = __fmul_rn(a, b), pe = __fmaf_rn(a, b, -p);
  if (PLUS) c = -c;
  const float q = __fmul_rn(c, d), qe = __fmaf_rn(c, d, -q);
  const float s = __fsub_rn(p, q), z = __fsub_rn(s, p);
  const float e = __fsub_rn(__fsub_rn(p, __fsub_rn(s, z)), __fadd_rn(q, z));
  const float t = __fadd_rn(e, __fsub_rn(pe, qe));
  float r = __fadd_rn(s, t);
  if (!(t == t)) return s;  // infinities and NaN
  if (ODD) {
    const float rest = __fsub_rn(t, __fsub_rn(r, s));
    const int u = __float_as_int(r);
    // an even r that is not exact: its neighbour on the side of the rest
    if (rest != 0.f && !(u & 1) && r != 0.f)
      r = __int_as_float((rest > 0.f) == (r > 0.f) ? u + 1 : u - 1);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ T to_cache(float x);
template <>
__device__ __forceinline__ float to_cache<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half to_cache<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 to_cache<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// The token's sequence, position and row offset, by one warp; b < 0: none, or left out.
struct AppendPlace {
  int b, pos;
  int64_t off;
};
__device__ __forceinline__ AppendPlace append_place(const AppendArgs& a, int t) {
  const PagedView& c = a.c;
  const int b = paged_find(c, t);
  AppendPlace r = {-1, 0, -1};
  const PagedSeq s = b < c.batch ? paged_seq(c, b, INT_MAX, 0) : PagedSeq{0, 0, 0};
  if (t < s.row0 || t >= s.row0 + s.count) return r;
  r.pos = s.past + t - s.row0;
  if (a.half && r.pos >= a.max_pos) {
    record_error(c.err, KERR_PAGED_POSITION);
    return r;
  }
  r.b = b;
  const int pg = a.page_div.div(r.pos), page = __ldg(c.table + (int64_t)b * c.max_pages + pg);
  if (page < 0 || page >= c.num_pages)
    record_error(c.err, KERR_PAGED_PAGE);
  else
    r.off = page * c.page_elems + (int64_t)(r.pos - pg * c.page_size) * c.row_elems;
  return r;
}

// Sequences that no token of the call reaches are checked too (one CTA).
__device__ __forceinline__ void append_check_all(const PagedView& c) {
  for (int b = threadIdx.x; b < c.batch; b += blockDim.x) paged_seq(c, b, INT_MAX, 0);
}

// Any strides, alignments and rotated widths: a CTA per token, a thread per pair.
template <typename T>
__global__ void __launch_bounds__(256) append_any_kernel(const __grid_constant__ AppendArgs a) {
  const PagedView& c = a.c;
  const int t = blockIdx.x;
  if (t == 0) append_check_all(c);
  __shared__ AppendPlace at;
  if (threadIdx.x < 32) {
    const AppendPlace r = append_place(a, t);
    if (threadIdx.x == 0) at = r;
  }
  __syncthreads();
  if (at.b < 0) return;
  const int pos = at.pos, D = c.D, half = a.half;
  const int64_t off = at.off;
  const float* cs = a.cos + (int64_t)pos * half;
  const float* sn = a.sin + (int64_t)pos * half;
  const int per = D - half;  // pairs, then the features behind them
  const int n = (a.heads + 2 * c.kv_heads) * per;
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    int h = e / per;
    const int i = e - h * per;
    const bool pair = i < half;
    const int a0 = pair ? (a.interleaved ? 2 * i : i) : i + half;
    const int a1 = pair ? (a.interleaved ? 2 * i + 1 : i + half) : a0;
    if (h < a.heads) {
      const float* src = a.q + t * a.q_stride + (int64_t)h * D;
      float* dst = a.q_out + ((int64_t)t * a.heads + h) * D;
      const float x0 = src[a0], x1 = src[a1];
      if (pair) {
        dst[a0] = rope_sum<false, false>(x0, cs[i], x1, sn[i]);
        dst[a1] = rope_sum<true, false>(x1, cs[i], x0, sn[i]);
      } else {
        dst[a0] = x0;
      }
      continue;
    }
    if (off < 0) continue;
    h -= a.heads;
    const bool is_v = h >= c.kv_heads;
    if (is_v) h -= c.kv_heads;
    const float* src = (is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) + (int64_t)h * D;
    T* dst = static_cast<T*>(is_v ? c.value : c.key) + off + (int64_t)h * D;
    constexpr bool odd = sizeof(T) == 2;
    const float x0 = src[a0], x1 = src[a1];
    if (pair && !is_v) {
      dst[a0] = to_cache<T>(rope_sum<false, odd>(x0, cs[i], x1, sn[i]));
      dst[a1] = to_cache<T>(rope_sum<true, odd>(x1, cs[i], x0, sn[i]));
    } else {
      dst[a0] = to_cache<T>(x0);
      if (pair) dst[a1] = to_cache<T>(x1);
    }
  }
}

// 16-byte loads: a thread takes pieces of 8 features (4 pairs, or 8 features that are
// not rotated) of a token's heads, IT of them, and has its loads in flight while one
// warp finds the token's place (three dependent loads).  Bound by memory: 8676 tokens
// of 48 heads of
// 128 (393 MB) take 83 us, 4.75 TB/s, 0.73 of the copy (90, 107 us with two pieces, one).
// RoPE as in double, like the dense attention's, rounded once.
template <typename T, int IT>
__global__ void __launch_bounds__(128, 8) append_kernel(const __grid_constant__ AppendArgs a) {
  const PagedView& c = a.c;
  const int t = blockIdx.x / a.parts, part = blockIdx.x - t * a.parts;
  if (blockIdx.x == 0) append_check_all(c);
  const int D = c.D, half = a.half, ppc = D >> 3;  // pieces of a head
  const int n = (a.heads + 2 * c.kv_heads) * ppc;
  float x[IT][8];
  int first[IT], second[IT], head[IT];  // features of x[0..3] and x[4..7]; -1: no piece
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int e = (part * IT + i) * 128 + threadIdx.x;
    head[i] = -1;
    if (e >= n) continue;
    const int h = a.piece_div.div(e), y = e - h * ppc;
    head[i] = h;
    const bool turned = h < a.heads + c.kv_heads && 8 * y < 2 * half;
    if (turned && !a.interleaved) {  // (i, i + half)
      first[i] = 4 * y, second[i] = 4 * y + half;
    } else {
      first[i] = 8 * y, second[i] = 8 * y + 4;
    }
    const float* src = h < a.heads ? a.q + t * a.q_stride + (int64_t)h * D
                       : h < a.heads + c.kv_heads
                           ? a.k + t * a.k_stride + (int64_t)(h - a.heads) * D
                           : a.v + t * a.v_stride + (int64_t)(h - a.heads - c.kv_heads) * D;
    // (not through the read-only path: Q may be rotated in place)
    *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(src + first[i]);
    *reinterpret_cast<float4*>(x[i] + 4) = *reinterpret_cast<const float4*>(src + second[i]);
  }
  __shared__ AppendPlace at;
  if (threadIdx.x < 32) {
    const AppendPlace r = append_place(a, t);
    if (threadIdx.x == 0) at = r;
  }
  __syncthreads();
  if (at.b < 0) return;
  const int64_t off = at.off, cs0 = (int64_t)at.pos * half;
#pragma unroll
  for (int i = 0; i < IT; i++) {
    if (head[i] < 0) continue;
    const int h = head[i];
    const bool is_q = h < a.heads, is_v = h >= a.heads + c.kv_heads;
    if (!is_q && off < 0) continue;
    float(&y)[8] = x[i];
    const int pair0 = a.interleaved ? first[i] >> 1 : first[i];
    if (!is_v && pair0 < half && first[i] < 2 * half) {
      const float4 cv = __ldg(reinterpret_cast<const float4*>(a.cos + cs0 + pair0));
      const float4 sv = __ldg(reinterpret_cast<const float4*>(a.sin + cs0 + pair0));
      const float cd[4] = {cv.x, cv.y, cv.z, cv.w}, sd[4] = {sv.x, sv.y, sv.z, sv.w};
      auto turn = [&](auto odd) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float u = a.interleaved ? y[2 * e] : y[e], v = a.interleaved ? y[2 * e + 1] : y[e + 4];
          const float nu = rope_sum<false, odd>(u, cd[e], v, sd[e]);
          const float nv = rope_sum<true, odd>(v, cd[e], u, sd[e]);
          if (a.interleaved)
            y[2 * e] = nu, y[2 * e + 1] = nv;
          else
            y[e] = nu, y[e + 4] = nv;
        }
      };
      if (is_q || sizeof(T) == 4)
        turn(std::false_type());
      else
        turn(std::true_type());
    }
    if (is_q) {
      float* dst = a.q_out + ((int64_t)t * a.heads + h) * D;
      *reinterpret_cast<float4*>(dst + first[i]) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(dst + second[i]) = make_float4(y[4], y[5], y[6], y[7]);
      continue;
    }
    T* dst = static_cast<T*>(is_v ? c.value : c.key) + off +
             (int64_t)(h - a.heads - (is_v ? c.kv_heads : 0)) * D;
    __align__(16) T w[8];
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = to_cache<T>(y[e]);
    using H = std::conditional_t<sizeof(T) == 4, float4, uint2>;  // four features
    *reinterpret_cast<H*>(dst + first[i]) = *reinterpret_cast<const H*>(w);
    *reinterpret_cast<H*>(dst + second[i]) = *reinterpret_cast<const H*>(w + 4);
  }
}

template <typename T>
int launch_append_type(AppendArgs& a, int sm_count, cudaStream_t st) {
  const PagedView& c = a.c;
  auto ok = [](const void* p, int64_t stride) {
    return ((uintptr_t)p & 15) == 0 && stride % 4 == 0;
  };
  const bool vec = a.half % 4 == 0 && ok(a.k, a.k_stride) && ok(a.v, a.v_stride) &&
                   ok(a.q, a.q_stride) && ok(a.q_out, 0) && ok(a.cos, 0) && ok(a.sin, 0);
  if (!vec) {
    append_any_kernel<T><<<c.num_tokens, 256, 0, st>>>(a);
    ORTC_CUDA(cudaGetLastError());
    return ORT_CUDA_OK;
  }
  const int pieces = (a.heads + 2 * c.kv_heads) * (c.D / 8);
  a.piece_div.set((uint32_t)(c.D / 8));
  // one piece a thread until there are 2048 threads a SM, then three
  const int it = (int64_t)c.num_tokens * pieces > (int64_t)sm_count * 2048 ? 3 : 1;
  a.parts = (pieces + 128 * it - 1) / (128 * it);
  ORTC_CHECK((int64_t)c.num_tokens * a.parts <= INT_MAX, ORT_CUDA_ERR_INVALID_ARG,
             "paged append: sizes too large");
  const unsigned grid = (unsigned)(c.num_tokens * a.parts);
  if (it == 3)
    append_kernel<T, 3><<<grid, 128, 0, st>>>(a);
  else
    append_kernel<T, 1><<<grid, 128, 0, st>>>(a);
  ORTC_CUDA(cudaGetLastError());
  return ORT_CUDA_OK;
}

int launch_append(AppendArgs& a, int sm_count, cudaStream_t st, int64_t* launches) {
  a.page_div.set((uint32_t)a.c.page_size);
  const int rc = a.c.type == ORT_CUDA_CACHE_F32   ? launch_append_type<float>(a, sm_count, st)
                 : a.c.type == ORT_CUDA_CACHE_F16 ? launch_append_type<__half>(a, sm_count, st)
                                                  : launch_append_type<__nv_bfloat16>(a, sm_count, st);
  if (rc == ORT_CUDA_OK) (*launches)++;
  return rc;
}

// Whether two ranges of floats share one.
bool overlap(const float* a, int64_t an, const float* b, int64_t bn) {
  return a && b && a < b + bn && b < a + an;
}

// Whether a range of floats lies in the key or value pages.
bool in_pages(const ort_cuda_paged_cache* c, const float* a, int64_t an) {
  const int64_t bytes = c->num_pages * c->page_size * c->kv_num_heads * c->head_size *
                        (c->type == ORT_CUDA_CACHE_F32 ? 4 : 2);
  const int64_t n = (bytes + 3) / 4;
  return overlap(a, an, static_cast<const float*>(c->key), n) ||
         overlap(a, an, static_cast<const float*>(c->value), n);
}

// Checks what the host can see of a cache and fills the kernels' view.
int paged_view(ort_cuda_session* s, const ort_cuda_paged_cache* c, int64_t num_tokens, int flags,
               PagedView* v) {
  ORTC_CHECK(s && c, ORT_CUDA_ERR_INVALID_ARG, "NULL argument");
  ORTC_CHECK((flags & ORT_CUDA_HOST_IO) == 0, ORT_CUDA_ERR_INVALID_ARG,
             "the paged KV cache takes device tensors");
  ORTC_CHECK(c->type == ORT_CUDA_CACHE_F32 || c->type == ORT_CUDA_CACHE_F16 ||
                 c->type == ORT_CUDA_CACHE_BF16,
             ORT_CUDA_ERR_UNSUPPORTED, "paged KV cache: unknown element type");
  ORTC_CHECK(c->batch >= 0 && c->num_pages >= 0 && c->page_size >= 1 && c->max_pages >= 0 &&
                 c->kv_num_heads >= 1 && c->head_size >= 1 && num_tokens >= 0,
             ORT_CUDA_ERR_INVALID_ARG,
             "paged KV cache: need page_size, kv_num_heads, head_size >= 1 and sizes >= 0");
  ORTC_CHECK(c->head_size % 8 == 0 && c->head_size <= 128, ORT_CUDA_ERR_UNSUPPORTED,
             "paged KV cache: head sizes are multiples of 8 up to 128");
  ORTC_CHECK(c->num_pages <= INT_MAX && c->page_size <= INT_MAX && c->max_pages <= INT_MAX &&
                 c->batch < INT_MAX && num_tokens <= INT_MAX / 2 &&
                 (int64_t)c->kv_num_heads * c->head_size <= INT_MAX / c->page_size &&
                 c->max_pages <= (int64_t)(INT_MAX / 2) / c->page_size,
             ORT_CUDA_ERR_INVALID_ARG, "paged KV cache: sizes too large");
  if (num_tokens == 0 || c->batch == 0) return ORT_CUDA_OK;
  ORTC_CHECK(c->key && c->value && c->block_table && c->cu_seqlens && c->past_lens,
             ORT_CUDA_ERR_INVALID_ARG, "NULL argument");
  ORTC_CHECK(((uintptr_t)c->key & 15) == 0 && ((uintptr_t)c->value & 15) == 0,
             ORT_CUDA_ERR_INVALID_ARG, "paged KV cache: key and value must be 16-byte aligned");
  v->key = c->key, v->value = c->value;
  v->table = c->block_table, v->cu = c->cu_seqlens, v->past = c->past_lens;
  v->kv_heads = c->kv_num_heads, v->D = (int)c->head_size, v->type = c->type;
  v->row_elems = v->kv_heads * v->D;
  v->page_elems = c->page_size * v->row_elems;
  v->num_pages = (int)c->num_pages, v->page_size = (int)c->page_size;
  v->max_pages = (int)c->max_pages, v->batch = (int)c->batch;
  v->num_tokens = (int)num_tokens;
  v->err = s->err_dev;
  return ORT_CUDA_OK;
}

}  // namespace
}  // namespace ortc

using namespace ortc;

extern "C" {

ORT_CUDA_API int ort_cuda_paged_kv_append(ort_cuda_session* s, const ort_cuda_paged_cache* cache,
                                          const float* Q, int64_t q_stride, const float* K,
                                          int64_t k_stride, const float* V, int64_t v_stride,
                                          int64_t num_tokens, int num_heads,
                                          const float* cos_cache, const float* sin_cache,
                                          int64_t rotary_half, int64_t max_pos, float* Q_out,
                                          int flags) try {
  AppendArgs a;
  int rc = paged_view(s, cache, num_tokens, flags, &a.c);
  if (rc) return rc;
  const int64_t D = cache->head_size, row = cache->kv_num_heads * D;
  ORTC_CHECK((Q == nullptr) == (Q_out == nullptr), ORT_CUDA_ERR_INVALID_ARG,
             "paged append: give both Q and Q_out or neither");
  ORTC_CHECK(!Q || (num_heads >= 1 && num_heads % cache->kv_num_heads == 0 &&
                    num_heads <= INT_MAX / D && q_stride >= num_heads * D),
             ORT_CUDA_ERR_INVALID_ARG,
             "paged append: need num_heads a multiple of kv_num_heads and q_stride >= its row");
  ORTC_CHECK((Q ? num_heads : 0) * D + 2 * row <= INT_MAX, ORT_CUDA_ERR_INVALID_ARG,
             "paged append: sizes too large");
  const int64_t rows = std::max<int64_t>(num_tokens - 1, 0), qn = num_heads * D;
  ORTC_CHECK(!Q || num_tokens == 0 ||
                 (Q == Q_out ? q_stride == qn : !overlap(Q_out, (rows + 1) * qn, Q, rows * q_stride + qn)),
             ORT_CUDA_ERR_INVALID_ARG,
             "paged append: Q_out may be Q only when Q is contiguous, and not overlap it else");
  ORTC_CHECK(!Q || num_tokens == 0 ||
                 (!overlap(Q_out, (rows + 1) * qn, K, rows * k_stride + row) &&
                  !overlap(Q_out, (rows + 1) * qn, V, rows * v_stride + row)),
             ORT_CUDA_ERR_INVALID_ARG, "paged append: Q_out overlaps K or V");
  ORTC_CHECK(!Q || num_tokens == 0 || !in_pages(cache, Q_out, (rows + 1) * qn),
             ORT_CUDA_ERR_INVALID_ARG, "paged append: Q_out overlaps the pages");
  ORTC_CHECK(k_stride >= row && v_stride >= row, ORT_CUDA_ERR_INVALID_ARG,
             "paged append: k_stride and v_stride must be at least a row");
  ORTC_CHECK((cos_cache == nullptr) == (sin_cache == nullptr), ORT_CUDA_ERR_INVALID_ARG,
             "paged append: give both cos and sin caches or neither");
  ORTC_CHECK(!cos_cache || (rotary_half >= 1 && 2 * rotary_half <= D && max_pos >= 1),
             ORT_CUDA_ERR_INVALID_ARG,
             "paged append: rotary needs cos/sin caches of rotary_half <= head_size / 2 values");
  if (num_tokens == 0 || cache->batch == 0) return ORT_CUDA_OK;
  ORTC_CHECK(K && V, ORT_CUDA_ERR_INVALID_ARG, "NULL argument");
  ORTC_CHECK(cache->key != cache->value, ORT_CUDA_ERR_INVALID_ARG,
             "paged append: key and value are the same pages");
  a.q = Q, a.q_out = Q_out, a.q_stride = q_stride, a.heads = Q ? num_heads : 0;
  a.k = K, a.k_stride = k_stride, a.v = V, a.v_stride = v_stride;
  if (cos_cache) {
    a.cos = cos_cache, a.sin = sin_cache, a.half = (int)rotary_half, a.max_pos = max_pos;
    a.interleaved = (flags & ORT_CUDA_ROTARY_INTERLEAVED) ? 1 : 0;
  }
  DeviceGuard guard(s->device);
  OpTimer timer(s, "PagedKVAppend");
  return launch_append(a, s->sm_count, s->stream, &s->launches);
} catch (const std::exception& e) {
  return fail(ORT_CUDA_ERR_OOM, std::string("paged append: ") + e.what());
}

ORT_CUDA_API int ort_cuda_paged_attention(ort_cuda_session* s, const ort_cuda_paged_cache* cache,
                                          const float* Q, int64_t q_stride, int64_t num_tokens,
                                          int64_t max_seq, int num_heads, double scale,
                                          double softcap, int64_t window, int64_t shared_len,
                                          float* out, int flags) try {
  PagedAttnArgs a;
  int rc = paged_view(s, cache, num_tokens, flags, &a.c);
  if (rc) return rc;
  const int64_t D = cache->head_size;
  ORTC_CHECK(num_heads >= 1 && num_heads % cache->kv_num_heads == 0 && num_heads <= INT_MAX / D &&
                 q_stride >= num_heads * D,
             ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: need num_heads a multiple of kv_num_heads and q_stride >= its row");
  ORTC_CHECK(max_seq >= 0 && shared_len >= 0, ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: need max_seq, shared_len >= 0");
  ORTC_CHECK(shared_len <= cache->max_pages * cache->page_size, ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: shared_len exceeds max_pages * page_size");
  ORTC_CHECK(std::isfinite(scale) && std::isfinite(softcap), ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: scale and softcap must be finite");
  // Within fp32 with room for their quotient; a cap of 2^20 at most, since weights over
  // fp16 pages have room for tanhf's last bits times the cap (2^15.4 of 2^15.99).
  ORTC_CHECK((scale <= 0 || (scale >= 0x1p-100 && scale <= 0x1p100)) &&
                 (softcap <= 0 || (softcap >= 0x1p-20 && softcap <= 0x1p20)),
             ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: scale lies in [2^-100, 2^100], softcap in [2^-20, 2^20]");
  if (num_tokens == 0 || cache->batch == 0) return ORT_CUDA_OK;
  ORTC_CHECK(Q && out, ORT_CUDA_ERR_INVALID_ARG, "NULL argument");
  ORTC_CHECK(num_tokens * num_heads <= INT_MAX, ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: sizes too large");
  ORTC_CHECK(!overlap(out, num_tokens * num_heads * D, Q, (num_tokens - 1) * q_stride + num_heads * D),
             ORT_CUDA_ERR_INVALID_ARG, "paged attention: out overlaps Q");
  ORTC_CHECK(!in_pages(cache, out, num_tokens * num_heads * D), ORT_CUDA_ERR_INVALID_ARG,
             "paged attention: out overlaps the pages");
  a.q = Q, a.q_stride = q_stride, a.out = out;
  a.heads = num_heads, a.group = num_heads / cache->kv_num_heads;
  a.max_seq = (int)std::min<int64_t>(max_seq, num_tokens);
  a.shared = (int)shared_len;
  a.window = window > 0 && window < INT_MAX ? (int)window : 0;
  a.scale = (float)(scale > 0 ? scale : 1.0 / std::sqrt((double)D));
  a.softcap = softcap > 0 ? (float)softcap : 0.0f;
  DeviceGuard guard(s->device);
  OpTimer timer(s, "PagedAttention");
  void* scratch = nullptr;
  rc = paged_scratch(s, paged_attention_scratch(a, s->sm_count), &scratch);
  if (rc) return rc;
  return launch_paged_attention(a, scratch, s->sm_count, s->stream, &s->launches);
} catch (const std::exception& e) {
  return fail(ORT_CUDA_ERR_OOM, std::string("paged attention: ") + e.what());
}

}  // extern "C"
