// Launches of the attention over the paged KV cache.
#include <algorithm>
#include <atomic>
#include <climits>

#include "paged_rows.cuh"
#include "paged_tile.cuh"

namespace ortc {
namespace {

size_t al256(size_t x) { return (x + 255) & ~(size_t)255; }

// Query rows of a sequence and KV head up to which the stream kernel takes it.  From 33
// to 64 rows over 16-bit pages the tiles win where their segments fill the device, and
// lose where few do.  Tiles and stream, us, 40 and 64 rows over 2000 to 4000 keys of
// heads of 128:
//   segments   fp16, 40        64            bf16, 40        64
//    8         39.3, 22.7      41.2, 22.8    43.2, 24.4      43.4, 25.8
//   16         37.6, 26.6      39.2, 29.5    39.2, 28.9      41.2, 33.0
//   24         40.7, 33.0      41.2, 39.1    44.1, 37.1      45.3, 45.3
//   32         42.6, 39.2      43.3, 47.3    47.3, 45.3      47.9, 55.4
//   48         51.4, 57.5      52.4, 69.9    60.2, 66.8      61.5, 82.3
//   64         59.7, 70.3      61.0, 89.3    71.6, 82.5      72.5, 105
// With 32 rows the stream is ahead at 64 segments too (53, 49); over fp32 pages it wins
// to 64 rows either way (276, 211; one sequence 68, 38; 128 rows: 324, 408).  A shared
// prefix is one sequence.
int stream_limit(const PagedAttnArgs& a, int sequences) {
  const bool many = (int64_t)sequences * a.c.kv_heads > 24;
  return a.c.type != ORT_CUDA_CACHE_F32 && many ? 32 : 64;
}

// Rows of one MMA tile of the stream kernel: 8 when no sequence can have more
// (a row's parts then share an MMA), else 16.
int stream_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }
int padded_head(int D) { return D <= 64 ? 64 : 128; }

// Whether tiles of 128 rows may be used (csrc/paged_tile.cuh for 16-bit pages,
// csrc/paged_rows.cuh for fp32): two tokens' heads at least fit one.  More heads on a KV
// head go to the stream at any length, where every tile of 16 rows reads all keys of its
// sequence: a prompt of 2048 tokens, one KV head of 64, takes 179 us with 64 query heads
// and 1431 with 71 (fp16; bf16 195, 1564; fp32 880, 3068).
bool tile_ok(const PagedAttnArgs& a) { return a.group <= 64; }

template <typename K>
int set_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  ORTC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(done.load() >> dev & 1ull)) {
    ORTC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) done.fetch_or(1ull << dev);
  }
  return ORT_CUDA_OK;
}

template <typename T, int DP, int R>
int launch_stream_one(const StreamArgs& p, int grid, cudaStream_t st) {
  using C = StreamCfg<T, DP, R>;
  static std::atomic<unsigned long long> attr_set{0};  // per device
  const int rc = set_smem(paged_stream_kernel<T, DP, R>, C::SMEM, attr_set);
  if (rc) return rc;
  paged_stream_kernel<T, DP, R><<<grid, 256, C::SMEM, st>>>(p);
  ORTC_CUDA(cudaGetLastError());
  return ORT_CUDA_OK;
}

template <typename T>
int launch_stream_type(const StreamArgs& p, int rows, int grid, cudaStream_t st) {
  if (padded_head(p.a.c.D) == 64)
    return rows == 8 ? launch_stream_one<T, 64, 8>(p, grid, st)
                     : launch_stream_one<T, 64, 16>(p, grid, st);
  return rows == 8 ? launch_stream_one<T, 128, 8>(p, grid, st)
                   : launch_stream_one<T, 128, 16>(p, grid, st);
}

int launch_stream(const StreamArgs& p, int rows, int grid, cudaStream_t st, int64_t* launches) {
  int rc;
  if (p.a.c.type == ORT_CUDA_CACHE_F32)
    rc = launch_stream_type<float>(p, rows, grid, st);
  else if (p.a.c.type == ORT_CUDA_CACHE_F16)
    rc = launch_stream_type<__half>(p, rows, grid, st);
  else
    rc = launch_stream_type<__nv_bfloat16>(p, rows, grid, st);
  if (rc == ORT_CUDA_OK) (*launches)++;
  return rc;
}

template <typename T, int DP, bool CAP>
int launch_tile_cap(const TileArgs& p, int grid, cudaStream_t st) {
  using C = TileCfg<T, DP>;
  static std::atomic<unsigned long long> attr_set{0};
  int dev = 0;
  ORTC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(attr_set.load() >> dev & 1ull)) {
    // the register split draws on what the block is launched with
    cudaFuncAttributes fa;
    ORTC_CUDA(cudaFuncGetAttributes(&fa, paged_tile_kernel<T, DP, CAP>));
    ORTC_CHECK(fa.numRegs >= kTileRegs, ORT_CUDA_ERR_UNSUPPORTED,
               "paged attention: built with too few registers for the warpgroups' split");
  }
  const int rc = set_smem(paged_tile_kernel<T, DP, CAP>, C::SMEM, attr_set);
  if (rc) return rc;
  paged_tile_kernel<T, DP, CAP><<<grid, kTileThreads, C::SMEM, st>>>(p);
  ORTC_CUDA(cudaGetLastError());
  return ORT_CUDA_OK;
}

template <typename T, int DP>
int launch_tile_one(const TileArgs& p, int grid, cudaStream_t st) {
  return p.s.a.softcap > 0.f ? launch_tile_cap<T, DP, true>(p, grid, st)
                           : launch_tile_cap<T, DP, false>(p, grid, st);
}

template <int DP>
int launch_rows(const StreamArgs& p, int grid, cudaStream_t st) {
  static std::atomic<unsigned long long> attr_set{0};
  const int rc = set_smem(paged_rows_kernel<DP>, RowsCfg<DP>::SMEM, attr_set);
  if (rc) return rc;
  paged_rows_kernel<DP><<<grid, 256, RowsCfg<DP>::SMEM, st>>>(p);
  ORTC_CUDA(cudaGetLastError());
  return ORT_CUDA_OK;
}

int launch_tile(const StreamArgs& s, int grid, cudaStream_t st, int64_t* launches) {
  if (s.a.c.type == ORT_CUDA_CACHE_F32) {
    const int rc = padded_head(s.a.c.D) == 64 ? launch_rows<64>(s, grid, st)
                                              : launch_rows<128>(s, grid, st);
    if (rc == ORT_CUDA_OK) (*launches)++;
    return rc;
  }
  TileArgs p;
  p.s = s;
  const PagedView& c = s.a.c;
  const bool f16 = c.type == ORT_CUDA_CACHE_F16;
  const int64_t tokens = (int64_t)c.num_pages * c.page_size;
  if (c.page_size % 8 == 0 && tokens >= 1 && tokens <= INT_MAX) {
    const int most = f16 ? 128 : 64;  // a block's keys
    p.tma_rows = std::min(most, c.page_size & -c.page_size);
    const auto type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int v = 0; v < 2; v++) {
      const int rc = encode_tma_rows(v ? &p.value : &p.key, type, v ? c.value : c.key, c.D,
                                     c.kv_heads, tokens, (uint64_t)c.D * 2,
                                     (uint64_t)c.row_elems * 2, 64, p.tma_rows);
      if (rc) return rc;
    }
  }
  int rc;
  if (f16)
    rc = padded_head(c.D) == 64 ? launch_tile_one<__half, 64>(p, grid, st)
                                : launch_tile_one<__half, 128>(p, grid, st);
  else
    rc = padded_head(c.D) == 64 ? launch_tile_one<__nv_bfloat16, 64>(p, grid, st)
                                : launch_tile_one<__nv_bfloat16, 128>(p, grid, st);
  if (rc == ORT_CUDA_OK) (*launches)++;
  return rc;
}

// Whether the sequences' own keys, and the shared prefix, may need tiles of 128 rows.
bool tile_main(const PagedAttnArgs& a) {
  return tile_ok(a) && (int64_t)a.max_seq * a.group > stream_limit(a, a.c.batch);
}
bool tile_prefix(const PagedAttnArgs& a) {
  return tile_ok(a) && a.shared && (int64_t)a.c.num_tokens * a.group > stream_limit(a, 1);
}
size_t piece_rows(const PagedAttnArgs& a) { return tile_main(a) || tile_prefix(a) ? 128 : 16; }

}  // namespace

size_t paged_attention_scratch(const PagedAttnArgs& a, int sm_count) {
  size_t n = kTicketBytes + al256((size_t)sm_count * 2 * piece_rows(a) * 2 * 4) +
             al256((size_t)sm_count * 2 * piece_rows(a) * 128 * 4);
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
  p.group_div.set((uint32_t)a.group);
  p.q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0;
  p.out_vec = ((uintptr_t)a.out & 15) == 0;
  p.t_scale = a.softcap > 0.f ? a.scale / a.softcap : a.scale;
  p.t_mul = a.softcap > 0.f ? a.softcap * kLog2e : kLog2e;
  char* at = static_cast<char*>(scratch);
  p.tickets = reinterpret_cast<unsigned*>(at);
  at += kTicketBytes;
  p.part_ml = reinterpret_cast<float*>(at);
  at += al256((size_t)sm_count * 2 * piece_rows(a) * 2 * 4);
  p.part_o = reinterpret_cast<float*>(at);
  at += al256((size_t)sm_count * 2 * piece_rows(a) * 128 * 4);
  int rc;
  if (a.shared) {
    const size_t rows = (size_t)a.c.num_tokens * a.heads;
    p.pre_ml = reinterpret_cast<float*>(at);
    p.pre_o = reinterpret_cast<float*>(at + al256(rows * 8));
    StreamArgs q = p;
    q.prefix = 1;
    q.max_rows = INT_MAX;
    rc = tile_prefix(a)
             ? launch_tile(q, sm_count, st, launches)
             : launch_stream(q, stream_rows((int64_t)a.c.num_tokens * a.group), sm_count, st,
                             launches);
    if (rc) return rc;
  }
  p.max_rows = tile_ok(a) ? stream_limit(a, a.c.batch) : INT_MAX;
  if (tile_main(a)) {
    rc = launch_tile(p, sm_count, st, launches);
    if (rc) return rc;
  }
  const int64_t most = (int64_t)a.max_seq * a.group;
  return launch_stream(p, stream_rows(std::min<int64_t>(most, p.max_rows)), sm_count, st, launches);
}

}  // namespace ortc
