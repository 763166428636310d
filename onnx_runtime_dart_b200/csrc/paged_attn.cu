// Launches of the attention over the paged KV cache.
#include <algorithm>
#include <atomic>
#include <climits>

#include "paged_stream.cuh"

namespace ortc {
namespace {

constexpr size_t kTicketBytes = 4096;  // kept zero between calls (csrc/paged.cu)
size_t al256(size_t x) { return (x + 255) & ~(size_t)255; }

// Rows of one MMA tile: 8 when no sequence can have more (a row's parts then
// share an MMA), else 16.
int stream_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }
int padded_head(int D) { return D <= 64 ? 64 : 128; }

template <typename T, int DP, int R>
int launch_one(const StreamArgs& p, int grid, cudaStream_t st) {
  using C = StreamCfg<T, DP, R>;
  static std::atomic<unsigned long long> attr_set{0};  // per device
  int dev = 0;
  ORTC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(attr_set.load() >> dev & 1ull)) {
    ORTC_CUDA(cudaFuncSetAttribute(paged_stream_kernel<T, DP, R>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    if (dev < 64) attr_set.fetch_or(1ull << dev);
  }
  paged_stream_kernel<T, DP, R><<<grid, 256, C::SMEM, st>>>(p);
  ORTC_CUDA(cudaGetLastError());
  return ORT_CUDA_OK;
}

template <typename T>
int launch_type(const StreamArgs& p, int rows, int grid, cudaStream_t st) {
  if (padded_head(p.a.c.D) == 64)
    return rows == 8 ? launch_one<T, 64, 8>(p, grid, st) : launch_one<T, 64, 16>(p, grid, st);
  return rows == 8 ? launch_one<T, 128, 8>(p, grid, st) : launch_one<T, 128, 16>(p, grid, st);
}

int launch_stream(const StreamArgs& p, int rows, int grid, cudaStream_t st, int64_t* launches) {
  int rc;
  if (p.a.c.type == ORT_CUDA_CACHE_F32)
    rc = launch_type<float>(p, rows, grid, st);
  else if (p.a.c.type == ORT_CUDA_CACHE_F16)
    rc = launch_type<__half>(p, rows, grid, st);
  else
    rc = launch_type<__nv_bfloat16>(p, rows, grid, st);
  if (rc == ORT_CUDA_OK) (*launches)++;
  return rc;
}

}  // namespace

size_t paged_attention_scratch(const PagedAttnArgs& a, int sm_count) {
  size_t n = kTicketBytes + al256((size_t)sm_count * 2 * 16 * 2 * 4) +
             al256((size_t)sm_count * 2 * 16 * 128 * 4);
  if (a.shared) {
    const size_t rows = (size_t)a.c.num_tokens * a.heads;
    n += al256(rows * 8) + al256(rows * a.c.D * 4);
  }
  return n;
}

int launch_paged_attention(const PagedAttnArgs& a, void* scratch, int sm_count, cudaStream_t st,
                           int64_t* launches) {
  ORTC_CHECK(sm_count * sizeof(unsigned) <= kTicketBytes, ORT_CUDA_ERR_UNSUPPORTED,
             "paged attention: more SMs than tickets");
  constexpr float kLog2e = 1.4426950408889634f;
  StreamArgs p;
  p.a = a;
  p.page_div.set((uint32_t)a.c.page_size);
  p.q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0;
  p.t_scale = a.softcap > 0.f ? a.scale / a.softcap : a.scale;
  p.t_mul = a.softcap > 0.f ? a.softcap * kLog2e : kLog2e;
  p.max_rows = INT_MAX;
  char* at = static_cast<char*>(scratch);
  p.tickets = reinterpret_cast<unsigned*>(at);
  at += kTicketBytes;
  p.part_ml = reinterpret_cast<float*>(at);
  at += al256((size_t)sm_count * 2 * 16 * 2 * 4);
  p.part_o = reinterpret_cast<float*>(at);
  at += al256((size_t)sm_count * 2 * 16 * 128 * 4);
  if (a.shared) {
    const size_t rows = (size_t)a.c.num_tokens * a.heads;
    p.pre_ml = reinterpret_cast<float*>(at);
    p.pre_o = reinterpret_cast<float*>(at + al256(rows * 8));
    StreamArgs q = p;
    q.prefix = 1;
    const int rc = launch_stream(q, stream_rows((int64_t)a.c.num_tokens * a.group), sm_count, st,
                                 launches);
    if (rc) return rc;
  }
  return launch_stream(p, stream_rows((int64_t)a.max_seq * a.group), sm_count, st, launches);
}

}  // namespace ortc
