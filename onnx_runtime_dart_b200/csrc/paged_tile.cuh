// Attention over the paged KV cache for many query rows per sequence and KV
// head (prompts, a large batch over a shared prefix), 16-bit pages: tiles of
// 128 query rows on tcgen05.
//
// A segment is (sequence, tile of 128 / group tokens with all their query heads
// of one KV head, KV head); its keys are cut into blocks of KB.  The segments
// in order, each as long as its keys are many, are cut into equal runs, one per
// CTA and SM, at block borders; a segment in several runs is joined by the last
// CTA of them (a ticket), in run order.
//
// Roles: two softmax warpgroups, which take the blocks of a segment in turn
// (one works on its block's weights while the tensor cores work for the
// other), an MMA warp, and loaders: TMA boxes of as many tokens as a power of
// two divides the page size, or, where that is below 8, cp.async in pieces of
// 16 bytes by three warps (a 2048-token prompt on pages of 16, 24, 17 tokens:
// 140, 152, 335 us).  A warpgroup's thread owns one query row: it reads the
// row's scores from TMEM, writes the weights back over them as the A operand of p.v, and adds each
// block's product, which comes in TMEM columns of its own, to its fp32 output in
// registers (so sums over many blocks are rounded, where the tensor cores cut
// them off; there is no rescaling in TMEM).  The two warpgroups' states are
// joined at the segment's end.
//
// fp32 results from 16-bit operands: q and the weights are split into parts of
// the pages' type (csrc/paged_stream.cuh), each part an MMA of its own, the
// smallest part first.  fp16: 2 + 2 MMAs a product, bf16: 3 + 3, so the tensor
// bound is 1/2 (1/3) of the dense rate.
//
// Bound by the softmax warpgroups and by what lies between two segments: a
// 4096-token prompt of 32 heads of 128 over fp16 pages takes 340 us, 404 TFLOP/s of
// useful products (tensor pipe 42 %); a mixed bf16 step with capped scores 129.
//
// TMEM columns: scores / weights of the two warpgroups (KB, or KB + KB / 2
// where three parts need more than the scores), then their p.v (DP each).
#pragma once

#include <type_traits>

#include "paged_segments.cuh"
#include "tc.cuh"

namespace ortc {

template <typename T, int DP>
struct TileCfg {
  static constexpr int PARTS = Split<T>::PARTS;
  static constexpr int KB = PARTS == 2 ? 128 : 64;   // keys of a block
  static constexpr int SREG = PARTS == 2 ? KB : KB * 3 / 2;  // TMEM columns of scores / weights
  static constexpr int QPART = 128 * DP * 2;         // bytes of one part of the q tile
  static constexpr int QB = PARTS * QPART;
  static constexpr int STAGE = KB * DP * 2;
  static constexpr int NK = PARTS == 2 && DP == 128 ? 3 : 4;  // ring stages of keys
  static constexpr int NV = PARTS == 2 && DP == 128 ? 2 : 4;  // and of values
  static constexpr int DATA = QB + (NK + NV) * STAGE;
  // What a segment's start and end cost, in keys (its q operands, the first block's
  // latency, the output): a 4096-token fp16 prompt took 383, 345, 340 us at 6, 8, 10
  // blocks, a mixed bf16 step 219, 210, 210, a shared prefix 115, 112, 112.
  static constexpr int EXTRA = (PARTS == 2 ? 10 : 8) * KB;
  // data, (max, sum) of 128 rows by both warpgroups, block validity, barriers
  static constexpr int SMEM = DATA + 2 * 128 * 8 + 8 * 16 + 256;
  static_assert(2 * SREG + 2 * DP <= 512, "TMEM");
  static_assert(DP * 128 * 4 <= QB, "the output is staged in the q tile");
};

struct TileArgs {
  StreamArgs s;
  // pages as [tokens][kv heads][D], boxes of tma_rows tokens x 64 features; 0:
  // page sizes that are no multiple of 8 are loaded by cp.async
  int tma_rows = 0;
  CUtensorMap key, value;
};

__device__ __forceinline__ void bar_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ bool bar_or(int id, int n, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\t"
      "bar.red.or.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(y)
      : "r"(id), "r"(n), "r"((uint32_t)x)
      : "memory");
  return y != 0;
}

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// The parts of a packed pair (Split::pair with the differences in one
// instruction each).
template <typename T>
__device__ __forceinline__ void split2(uint64_t x, uint32_t (&w)[Split<T>::PARTS]) {
  const uint64_t minus1 = pack2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < Split<T>::PARTS; i++) {
    const float2 v = unpack2(x);
    float2 f;
    if constexpr (Split<T>::PARTS == 2) {
      const __half2 h = __floats2half2_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
      f = __half22float2(h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
      f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    if (i + 1 < Split<T>::PARTS) x = fma2(pack2(f.x, f.y), minus1, x);
  }
}

// Registers a thread after the split; they draw on what the block was launched with
// (kTileRegs a thread), which launch_tile_cap checks.  A softmax thread holds its row's
// output (128); 208, 216, 224, 232 for it: a mixed bf16 step 224, 210, 205, 205 us.
constexpr int kTileThreads = 384, kTileSoftRegs = 232, kTileLoadRegs = 40, kTileRegs = 168;
static_assert(256 * kTileSoftRegs + 128 * kTileLoadRegs <= kTileThreads * kTileRegs, "registers");

template <typename T, int DP, bool CAP>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_tile_kernel(const __grid_constant__ TileArgs args) {
  using C = TileCfg<T, DP>;
  constexpr int PARTS = C::PARTS, KB = C::KB, NK = C::NK, NV = C::NV, EX = C::EXTRA;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw;  // 1024-byte aligned: the kernel has no other shared memory
  unsigned char* qs = smem;                 // [part][DP / 64][128 rows][128 B], swizzled
  unsigned char* ks = qs + C::QB;           // [NK][DP / 64][KB rows][128 B]
  unsigned char* vs = ks + NK * C::STAGE;   // [NV] the same
  float* ost = reinterpret_cast<float*>(qs);  // [DP][128] at a segment's end
  float2* stats = reinterpret_cast<float2*>(smem + C::DATA);  // [2][128]
  uint32_t* kvalid = reinterpret_cast<uint32_t*>(stats + 256);  // [8][4]
  uint64_t* bars = reinterpret_cast<uint64_t*>(kvalid + 32);
  uint64_t *kfull = bars, *kempty = kfull + NK, *vfull = kempty + NK, *vempty = vfull + NV,
           *sfull = vempty + NV, *pfull = sfull + 2, *pvfull = pfull + 2, *qfull = pvfull + 2,
           *done = qfull + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);
  int* s_last = reinterpret_cast<int*>(tmem_at + 1);
  static_assert((2 * 4 + 2 * 4 + 8) * 8 + 8 <= 256, "barriers");

  const StreamArgs& p = args.s;
  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = c.D, TT = 128 / a.group;
  const int rows_tma = args.tma_rows, align = max(1, rows_tma);

  // ---- this CTA's run
  TileRun<KB, EX> run;
  if (!run.plan(p, TT, align, stats)) return;
  const long long total = run.total;
  const int runs = run.runs;
  // the segment and its first block here; each role walks the list from here
  TilePos cur = run.cur;
  long long seg = run.seg;  // place of block 0 of the segment
  int k0 = run.k0;
  auto next = [&](TilePos& s, long long& at, int& first) { return run.next(p, s, at, first); };
  auto blocks = [&](const TilePos& s, long long at, int first) { return run.blocks(s, at, first); };

  if (tid == 0) {
    for (int i = 0; i < NK; i++) mbar_init(kfull + i, rows_tma ? 1 : 3), mbar_init(kempty + i, 1);
    for (int i = 0; i < NV; i++) mbar_init(vfull + i, rows_tma ? 1 : 3), mbar_init(vempty + i, 1);
    for (int i = 0; i < 2; i++) mbar_init(sfull + i, 1), mbar_init(pfull + i, 128), mbar_init(pvfull + i, 1);
    mbar_init(qfull, 256);
    mbar_init(done, 1);
    fence_mbarrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_at;
  bool dead = false;  // a wait ran out: no more waits, every barrier is still met

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTileLoadRegs));
    if (warp == 8) {
      // ---- MMA
      constexpr uint32_t id_s = idesc_f16(PARTS == 3, 128, KB);
      constexpr uint32_t id_o = idesc_f16(PARTS == 3, 128, DP) | kIdescBMnMajor;
      const uint32_t k_s = smem_u32(ks), v_s = smem_u32(vs);
      const uint64_t qd = smem_desc_sw128(smem_u32(qs));  // addresses add in its low bits
      int kc = 0, vc = 0, pc[2] = {0, 0}, sc = 0;
      auto wait = [&](uint64_t* bar, int parity) {
        if (!dead && !mbar_wait(bar, parity)) {
          dead = true;
          record_error(c.err, KERR_WAIT_FULL);
        }
        dead = __any_sync(~0u, dead);
        tc_fence_after();
      };
      auto scores = [&](int w) {  // s = q . k of the next block
        const int st = kc % NK;
        wait(kfull + st, (kc / NK) & 1);
        kc++;
        if (dead) return;
        if (elect_one()) {
          const uint64_t kd = smem_desc_sw128(k_s + st * C::STAGE);
#pragma unroll
          for (int pt = PARTS - 1; pt >= 0; pt--)
#pragma unroll
            for (int x = 0; x < DP / 16; x++)
              mma_f16_ss(tmem + w * C::SREG,
                         qd + ((pt * C::QPART + (x >> 2) * 16384 + (x & 3) * 32) >> 4),
                         kd + (((x >> 2) * (KB * 128) + (x & 3) * 32) >> 4), id_s,
                         pt != PARTS - 1 || x);
          mma_commit(kempty + st);
          mma_commit(sfull + w);
        }
        __syncwarp();
      };
      for (;;) {
        const int n = blocks(cur, seg, k0);
        wait(qfull, sc & 1);
        sc++;
        scores(0);
        if (n > 1) scores(1);
        for (int k = 0; k < n; k++) {
          const int w = k & 1, st = vc % NV;
          wait(pfull + w, pc[w] & 1);
          pc[w]++;
          wait(vfull + st, (vc / NV) & 1);
          vc++;
          if (!dead && elect_one()) {
            const uint64_t vd = smem_desc_sw128_mn(v_s + st * C::STAGE, KB * 128);
#pragma unroll
            for (int pt = PARTS - 1; pt >= 0; pt--)
#pragma unroll
              for (int x = 0; x < KB / 16; x++) {
                const int col = pt < 2 ? 16 * x + 8 * pt : KB + 8 * x;
                mma_f16_ts(tmem + 2 * C::SREG + w * DP, tmem + w * C::SREG + col,
                           vd + (x * 2048 >> 4), id_o,
                           pt != PARTS - 1 || x);
              }
            mma_commit(vempty + st);
            mma_commit(pvfull + w);
          }
          __syncwarp();
          if (k + 2 < n) scores(w);
        }
        if (!next(cur, seg, k0)) break;
      }
      // every product has ended before TMEM is given up, also where a wait ran out
      if (elect_one()) mma_commit(done);
      __syncwarp();
      if (!mbar_wait(done, 0)) record_error(c.err, KERR_WAIT_DRAIN);
    } else if (rows_tma) {
      // ---- TMA: warp 9 keys, warp 10 values; lane i the box of tokens i * rows_tma
      if (warp <= 10) {
        const bool is_k = warp == 9;
        const int NS = is_k ? NK : NV, box = lane * rows_tma;
        uint64_t *full = is_k ? kfull : vfull, *empty = is_k ? kempty : vempty;
        const uint32_t ring = smem_u32(is_k ? ks : vs);
        const CUtensorMap* map = is_k ? &args.key : &args.value;
        if (lane == 0) prefetch_tensormap(map);
        int cnt = 0, issued = 0;
        for (;;) {
          const int n = blocks(cur, seg, k0);
#pragma unroll 1
          for (int k = 0; k < n; k++, cnt++) {
            const int st = cnt % NS, j = cur.lo + (k0 + k) * KB + box;
            int page = -2, slot = 0;
            if (box < KB && j < cur.hi) {
              const int pg = p.page_div.div(j);
              slot = j - pg * c.page_size;
              page = __ldg(c.table + (int64_t)(p.prefix ? 0 : cur.b) * c.max_pages + pg);
            }
            const bool ok = page >= 0 && page < c.num_pages;
            if (cnt >= NS && !dead) {
              if (!mbar_wait(empty + st, ((cnt / NS) - 1) & 1)) {
                dead = true;
                record_error(c.err, KERR_WAIT_EMPTY);
              }
              dead = __any_sync(~0u, dead);
            }
            const unsigned there = __ballot_sync(~0u, ok);
            if (is_k) {
              if (!ok && page != -2) record_error(c.err, KERR_PAGED_PAGE);
              if (lane < KB / 32) {  // the word's keys: a bit per box, spread over its rows
                uint32_t m = 0;
                for (int e = 0; e < 32; e++)
                  m |= ((there >> ((32 * lane + e) / rows_tma)) & 1u) << e;
                kvalid[(cnt & 7) * 4 + lane] = m;
              }
              __syncwarp();
            }
            if (!dead) {
              issued = cnt + 1;
              if (lane == 0)
                mbar_arrive_expect_tx(full + st,
                                      (uint32_t)(__popc(there) * rows_tma * 128 * (DP / 64)));
              __syncwarp();
              if (ok) {
#pragma unroll
                for (int hf = 0; hf < DP / 64; hf++)
                  tma_load_3d(ring + st * C::STAGE + hf * (KB * 128) + box * 128, map, full + st,
                              64 * hf, cur.g, page * c.page_size + slot);
              }
            }
          }
          if (!next(cur, seg, k0)) break;
        }
        // the last copies have landed before the block's memory is given up
        for (int i = max(0, issued - NS); i < issued; i++)
          if (!mbar_wait(full + i % NS, (i / NS) & 1)) record_error(c.err, KERR_WAIT_DRAIN);
      }
    } else {
      // ---- loaders: the stages in the order the MMA warp takes them (K0, K1, V0,
      // K2, V1, ...), each by warps 9, 10, 11 together (every warp waits for every
      // stage in turn, so a phase of a barrier is never passed over)
      const uint32_t k_s = smem_u32(ks), v_s = smem_u32(vs);
      constexpr int LK = KB / 32;
      const int chunks = D / 8, ch = lane & 7;
      const int third = warp - 9;
      int kc = 0, vc = 0;
      uint64_t* pending = nullptr;  // a stage whose copies have not been announced
      auto announce = [&] {  // its copies have landed (waited for): hand it to the MMA
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(pending);
        pending = nullptr;
      };
      auto load = [&](bool is_k, int k) {
        const int cnt = is_k ? kc++ : vc++;
        const int NS = is_k ? NK : NV, st = cnt % NS, base = cur.lo + (k0 + k) * KB;
        int page[LK], slot[LK];
#pragma unroll
        for (int i = 0; i < LK; i++) {
          const int j = base + 32 * i + lane, pg = p.page_div.div(j);
          slot[i] = j - pg * c.page_size;
          page[i] = j < cur.hi
                        ? __ldg(c.table + (int64_t)(p.prefix ? 0 : cur.b) * c.max_pages + pg)
                        : -2;
        }
        uint64_t* empty = (is_k ? kempty : vempty) + st;
        if (cnt >= NS && !dead) {
          const int par = ((cnt / NS) - 1) & 1;
          if (!__all_sync(~0u, mbar_try_wait(empty, par))) {
            if (pending) {  // do not hold a landed stage back
              asm volatile("cp.async.wait_group 0;\n" ::: "memory");
              announce();
            }
            if (!mbar_wait(empty, par)) {
              dead = true;
              record_error(c.err, KERR_WAIT_EMPTY);
            }
            dead = __any_sync(~0u, dead);
          }
        }
        const uint32_t at = (is_k ? k_s : v_s) + st * C::STAGE;
        const T* src = static_cast<const T*>(is_k ? c.key : c.value);
#pragma unroll
        for (int i = 0; i < LK; i++) {
          const bool ok = page[i] >= 0 && page[i] < c.num_pages;
          if (is_k && third == 0) {
            if (!ok && page[i] != -2) record_error(c.err, KERR_PAGED_PAGE);
            const unsigned m = __ballot_sync(~0u, ok);
            if (lane == 0) kvalid[(cnt & 7) * 4 + i] = m;
          }
          const T* row = ok ? src + (long long)page[i] * c.page_elems +
                                  (long long)slot[i] * c.row_elems + (long long)cur.g * D
                            : nullptr;
          // 8 lanes a row: its 128-byte halves
#pragma unroll
          for (int y = 0; y < 8; y++) {
            if ((8 * i + y) % 3 != third) continue;
            const int r = 4 * y + (lane >> 3);
            const T* o = reinterpret_cast<const T*>(
                __shfl_sync(~0u, reinterpret_cast<unsigned long long>(row), r));
            const uint32_t dst = at + (32 * i + r) * 128 + ((ch ^ (r & 7)) << 4);
#pragma unroll
            for (int hf = 0; hf < DP / 64; hf++) {
              const int bytes = o && ch + 8 * hf < chunks ? 16 : 0;
              cp16(dst + hf * (KB * 128), bytes ? o + (ch + 8 * hf) * 8 : src, bytes);
            }
          }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        if (pending) {
          asm volatile("cp.async.wait_group 1;\n" ::: "memory");
          announce();
        }
        pending = (is_k ? kfull : vfull) + st;
      };
      for (;;) {
        const int n = blocks(cur, seg, k0);
#pragma unroll 1
        for (int k = -2; k < n; k++) {
          if (k + 2 < n) load(true, k + 2);
          if (k >= 0) load(false, k);
        }
        if (!next(cur, seg, k0)) break;
      }
      asm volatile("cp.async.wait_group 0;\n" ::: "memory");
      if (pending) announce();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTileSoftRegs));
    // ---- softmax warpgroup wg; thread: query row `row` of the tile
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + (((uint32_t)(warp & 3) * 32) << 16);
    const uint32_t ts = tl + wg * C::SREG, to = tl + 2 * C::SREG + wg * DP;
    int sc = 0, gb = 0;  // this warpgroup's blocks so far; all blocks so far
    auto wait = [&](uint64_t* bar, int parity) {
      if (!dead && !mbar_wait(bar, parity)) {
        dead = true;
        record_error(c.err, KERR_WAIT_MMA);
      }
      __syncwarp();
      tc_fence_after();
    };
    // q rows: warp w brings rows 16 w .. 16 w + 15 of a segment's tile, a 16-byte piece
    // a lane, four steps at a time with the next four on their way (the loop is rolled:
    // straight-line code for all rows, run once a segment, waits for its instructions)
    constexpr int LPR = DP / 4, RPI = 32 / LPR, NQ = 16 / RPI, QS = 4;  // lanes a row, rows a step, steps
    auto load_q = [&](const TilePos& s, int i0, float4 (&q4)[QS]) {
      const int t0 = s.rt * TT, rows = min(TT, s.count - t0) * a.group;
      const int f = (lane & (LPR - 1)) * 4;
      const float* base = a.q + (int64_t)(s.row0 + t0) * a.q_stride + (int64_t)(s.g * a.group) * D;
#pragma unroll
      for (int i = 0; i < QS; i++) {
        const int r = warp * 16 + (i0 + i) * RPI + lane / LPR;
        q4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && f < D) {
          const int t = p.group_div.div(r);
          const float* src = base + (int64_t)t * a.q_stride + (int64_t)(r - t * a.group) * D + f;
          if (p.q_vec)
            q4[i] = __ldg(reinterpret_cast<const float4*>(src));
          else
            q4[i] = make_float4(__ldg(src), __ldg(src + 1), __ldg(src + 2), __ldg(src + 3));
        }
      }
    };
    float4 q4[QS];
    load_q(cur, 0, q4);
    for (;;) {
      const int n = blocks(cur, seg, k0);
      const int tok0 = cur.rt * TT, rows_here = min(TT, cur.count - tok0) * a.group;
      const bool has = row < rows_here;
      const int tok = tok0 + (has ? p.group_div.div(row) : 0);
      // the parts of the q tile
#pragma unroll 1
      for (int i0 = 0; i0 < NQ; i0 += QS) {
        float4 nq[QS];
        if (i0 + QS < NQ) load_q(cur, i0 + QS, nq);
#pragma unroll
        for (int i = 0; i < QS; i++) {
          const int r = warp * 16 + (i0 + i) * RPI + lane / LPR, ch = (lane & (LPR - 1)) >> 1;
          float fr = p.t_scale, up = 1.f;
          if constexpr (PARTS == 2) {  // the row's largest value into [2^13, 2^14)
            float mx = fmaxf(fmaxf(fabsf(q4[i].x), fabsf(q4[i].y)),
                             fmaxf(fabsf(q4[i].z), fabsf(q4[i].w)));
            if (LPR == 32) {
              mx = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mx)));
            } else {
#pragma unroll
              for (int x = LPR / 2; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, x));
            }
            int ex = (int)(__float_as_uint(mx) >> 23) - 127;
            ex = max(-100, min(ex, 126));
            up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
            fr *= __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
          }
          uint32_t w0[PARTS], w1[PARTS];
          Split<T>::pair(q4[i].x * up, q4[i].y * up, w0);
          Split<T>::pair(q4[i].z * up, q4[i].w * up, w1);
#pragma unroll
          for (int pt = 0; pt < PARTS; pt++)
            *reinterpret_cast<uint2*>(qs + pt * C::QPART + (ch >> 3) * 16384 + r * 128 +
                                      (((ch & 7) ^ (r & 7)) << 4) + (lane & 1) * 8) =
                make_uint2(w0[pt], w1[pt]);
          if ((lane & (LPR - 1)) == 0) stats[r].x = fr;
          if (NQ > QS) q4[i] = nq[i];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(qfull);
      bar_sync(1, 256);
      const float fac = stats[row].x;
      int pos = -1;  // the row's position (-1: no row), and what all rows see
      int all_hi = cur.past + tok0, all_lo = cur.past + min(tok0 + TT, cur.count) - 1;
      if (p.prefix) {
        pos = all_hi = all_lo = INT_MAX / 2;
        if (a.window) {
          all_hi = -1;  // rows of different sequences: look at each
          if (has) pos = prefix_position(c, tok);
        }
      } else if (has) {
        pos = cur.past + tok;
      }
      const int own = pos;
      pos = min(pos, cur.hi - 1);  // a block's boxes may reach past the last key
      const int first = p.prefix ? 0 : a.shared;
      const int from = max(first, a.window ? own - a.window + 1 : 0);
      const float cmul = fac * p.t_mul;

      float m = -INFINITY, l = 0.f;
      uint64_t o[DP / 2];  // pairs of features
#pragma unroll
      for (int i = 0; i < DP / 2; i++) o[i] = 0;
      for (int k = wg; k < n; k += 2) {
        const int base = cur.lo + (k0 + k) * KB;
        wait(sfull + wg, sc & 1);
        // Whether all rows see the whole block (alike for all threads: a barrier below
        // depends on it), and whether its pages are there too (alike within a warp; where
        // a wait ran out, one warp may read what another does not).
        const bool inner = base + KB - 1 <= all_hi && base + KB <= cur.hi && base >= first &&
                           (!a.window || base > all_lo - a.window);
        const uint32_t* kv = kvalid + ((gb + k) & 7) * 4;
        bool full = inner;
        for (int i = 0; i < KB / 32; i++) full = full && kv[i] == ~0u;
        full = __all_sync(~0u, full);
        auto seen = [&](int i) {  // keys of the block's word i that the row sees
          const int b = base + 32 * i, x0 = max(from - b, 0), x1 = min(pos - b, 31);
          return pos < b || x0 > x1 ? 0u : kv[i] & (~0u >> (31 - x1)) & (~0u << x0);
        };
        // the row's maximum
        float mx = -INFINITY, mx2 = -INFINITY;
        if (full) {
#pragma unroll
          for (int i = 0; i < KB / 64; i++) {
            uint32_t r[64];
            tmem_ld64(ts + 64 * i, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              mx = max3(mx, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
              mx2 = max3(mx2, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
            }
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < KB / 32; i++) {
            uint32_t r[32];
            tmem_ld32(ts + 32 * i, r);
            const uint32_t vw = seen(i);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e++)
              if ((vw >> e) & 1) mx = fmaxf(mx, __uint_as_float(r[e]));
          }
        }
        mx = fmaxf(mx, mx2);
        if (mx != -INFINITY) mx = CAP ? __fmul_rn(tanhf(mx * fac), p.t_mul) : __fmul_rn(mx, cmul);
        const float mn = fmaxf(m, row_base<T>(mx)), sub = mn == -INFINITY ? 0.f : mn;
        const float corr = ex2(m - sub);
        m = mn;

        // values only some rows see: an infinity or NaN among them must not reach
        // the others as 0 * inf (see paged_stream.cuh); rows that hold no key of the
        // segment, whatever a page or an older stage left there, become zeros
        bool odd = false;
        unsigned char* vst = vs + ((gb + k) % NV) * C::STAGE;
        if (!full) {
          wait(vfull + (gb + k) % NV, ((gb + k) / NV) & 1);
          // a thread looks over one row (KB = 64: half a row)
          constexpr int TPR = 128 / KB, CPT = DP / 8 / TPR;
          const int r = row & (KB - 1), j = base + r, ch0 = row / KB * CPT;
          const bool there = j >= first && j < cur.hi && ((kv[r >> 5] >> (r & 31)) & 1);
          constexpr uint32_t up = PARTS == 2 ? 0x04000400u : 0x00800080u;
          uint32_t top = 0;  // exponents of all ones carry into the halves' sign bits
#pragma unroll
          for (int y = 0; y < CPT; y++) {
            const int ch = ch0 + y;
            uint4* at = reinterpret_cast<uint4*>(vst + (ch >> 3) * (KB * 128) + r * 128 +
                                                 (((ch & 7) ^ (r & 7)) << 4));
            if (there) {
              const uint4 v = *at;
              top |= ((v.x & 0x7fff7fffu) + up) | ((v.y & 0x7fff7fffu) + up) |
                     ((v.z & 0x7fff7fffu) + up) | ((v.w & 0x7fff7fffu) + up);
            } else {
              *at = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          odd = (top & 0x80008000u) != 0;
          fence_proxy_async_smem();
          odd = !inner && bar_or(2 + wg, 128, odd);
        }

        // weights, over the scores
        uint64_t sums[2] = {0, 0};
        // The fused product is not rounded as the maximum's was, which below 2^20 is no
        // more than 2^-5 apart.  A warp with a larger base rounds its scores like it.
        const bool big = !CAP && __any_sync(~0u, fabsf(m) >= 1048576.f);
        const uint64_t cmul2 = pack2(cmul, cmul), sub2 = pack2(-sub, -sub);
        // 16 scores: exp2, their sum, the parts
        auto weigh = [&](auto masked, int st, const uint32_t (&r)[16], uint32_t vw) {
          uint64_t x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            float2 t = make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
            if (CAP)
              t = make_float2(fmaf(tanhf(t.x * fac), p.t_mul, -sub),
                              fmaf(tanhf(t.y * fac), p.t_mul, -sub));
            else if (masked && big)
              t = make_float2(__fsub_rn(__fmul_rn(t.x, cmul), sub),
                              __fsub_rn(__fmul_rn(t.y, cmul), sub));
            else
              t = unpack2(fma2(pack2(t.x, t.y), cmul2, sub2));
            t.x = ex2(t.x), t.y = ex2(t.y);
            if (masked) {
              t.x = (vw >> (2 * e)) & 1 ? t.x : 0.f;
              t.y = (vw >> (2 * e + 1)) & 1 ? t.y : 0.f;
            }
            x[e] = pack2(t.x, t.y);
            sums[e & 1] = add2(sums[e & 1], x[e]);
          }
          uint32_t wd[16], w2[8];
          if (masked && odd) {  // kept in fp32 for the sum below
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const float2 t = unpack2(x[e]);
              wd[2 * e] = __float_as_uint(t.x), wd[2 * e + 1] = __float_as_uint(t.y), w2[e] = 0u;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              uint32_t t[PARTS];
              split2<T>(x[e], t);
              wd[e] = t[0], wd[8 + e] = t[1], w2[e] = t[PARTS - 1];
            }
          }
          tmem_st16(ts + 16 * st, wd);
          if (PARTS == 3)
            tmem_st8(ts + KB + 8 * st, make_uint4(w2[0], w2[1], w2[2], w2[3]),
                     make_uint4(w2[4], w2[5], w2[6], w2[7]));
        };
        if (full && !big) {
#pragma unroll 1
          for (int i = 0; i < KB / 32; i++) {
            uint32_t ra[16], rb[16];
            tmem_ld16(ts + 32 * i, ra);
            tmem_ld16(ts + 32 * i + 16, rb);
            tmem_ld_wait();
            weigh(std::false_type(), 2 * i, ra, 0u);
            weigh(std::false_type(), 2 * i + 1, rb, 0u);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < KB / 16; i++) {
            uint32_t r[16];
            tmem_ld16(ts + 16 * i, r);
            const uint32_t vw = seen(i >> 1) >> (16 * (i & 1));
            tmem_ld_wait();
            weigh(std::true_type(), i, r, vw);
          }
        }
        const float2 sa = unpack2(add2(sums[0], sums[1]));
        l = l * corr + (sa.x + sa.y);
        tmem_st_wait();
        const uint64_t corr2 = pack2(corr, corr);
        if (odd) {
#pragma unroll
          for (int i = 0; i < DP / 2; i++) o[i] = fma2(o[i], corr2, 0);
          for (int j = 0; j < KB; j++) {
            uint32_t r;
            tmem_ld1(ts + j, r);
            tmem_ld_wait();
            const float w = __uint_as_float(r);
#pragma unroll
            for (int ch = 0; ch < DP / 8; ch++) {
              const uint4 v = *reinterpret_cast<const uint4*>(
                  vst + (ch >> 3) * (KB * 128) + j * 128 + (((ch & 7) ^ (j & 7)) << 4));
              const T* ve = reinterpret_cast<const T*>(&v);
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (w != 0.f)
                  o[4 * ch + e] = fma2(pack2(w, w), pack2((float)ve[2 * e], (float)ve[2 * e + 1]),
                                       o[4 * ch + e]);
            }
          }
        }
        tc_fence_before();
        mbar_arrive(pfull + wg);
        wait(pvfull + wg, sc & 1);
        sc++;
        if (odd) continue;  // the product of what is not weights
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
          uint32_t r[32];
          tmem_ld32(to + 32 * i, r);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; e++)
            o[16 * i + e] = fma2(o[16 * i + e], corr2, pack2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])));
        }
      }
      gb += n;

      // ---- the segment's end: join the warpgroups, write rows by warps
      auto at = [&](int d, int r) -> float& { return ost[d * 128 + (r ^ (d & 31))]; };
      tc_fence_before();
      bar_sync(1, 256);  // every MMA of the segment is done: the q tile is free
      // each warpgroup hands over half of the features and joins the other half
      auto hand = [&](auto half) {
#pragma unroll
        for (int i = 0; i < DP / 4; i++) {
          const float2 v = unpack2(o[half * (DP / 4) + i]);
          at(half * (DP / 2) + 2 * i, row) = v.x;
          at(half * (DP / 2) + 2 * i + 1, row) = v.y;
        }
      };
      auto join = [&](auto half, float mine, float theirs) {
#pragma unroll
        for (int i0 = 0; i0 < DP / 4; i0 += 8) {
          float2 t[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int d = half * (DP / 2) + 2 * (i0 + i);
            t[i] = make_float2(at(d, row), at(d + 1, row));
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int d = half * (DP / 2) + 2 * (i0 + i);
            const float2 v = unpack2(o[d / 2]);
            at(d, row) = v.x * mine + t[i].x * theirs;
            at(d + 1, row) = v.y * mine + t[i].y * theirs;
          }
        }
      };
      using H0 = std::integral_constant<int, 0>;
      using H1 = std::integral_constant<int, 1>;
      stats[wg * 128 + row] = make_float2(m, l);
      if (wg == 0)
        hand(H1());
      else
        hand(H0());
      bar_sync(1, 256);
      const float2 s2 = stats[(wg ^ 1) * 128 + row];
      const float M = fmaxf(m, s2.x), mb = M == -INFINITY ? 0.f : M;
      const float mine = ex2(m - mb), theirs = ex2(s2.x - mb);
      if (wg == 0)
        join(H0(), mine, theirs);
      else
        join(H1(), mine, theirs);
      bar_sync(1, 256);
      const bool whole = n == cur.nt;
      const int slot = 2 * blockIdx.x + (k0 ? 0 : 1);
      if (wg == 0) {  // the row's place and factors, over the states (read above)
        const float L = l * mine + s2.y * theirs;
        const int64_t to = whole ? tile_place(p, cur, TT, has ? row : 0) : (int64_t)slot * 128 + row;
        float2 f = make_float2(1.f, 0.f);
        if (has && (!whole || p.prefix))
          *reinterpret_cast<float2*>((whole ? p.pre_ml : p.part_ml) + 2 * to) = make_float2(M, L);
        else if (has)
          f = paged_row_scale(p, to, M, L);
        stats[row] = f;
        reinterpret_cast<int64_t*>(stats + 128)[row] = to * (whole ? D : DP);
      }
      // the next segment's first q rows come while this one's are written
      TilePos nx = cur;
      long long nseg = seg;
      int nk0 = k0;
      const bool more = next(nx, nseg, nk0);
      if (more) load_q(nx, 0, q4);
      bar_sync(1, 256);
      auto write = [&](auto add) {
        float* dst = whole ? (p.prefix ? p.pre_o : a.out) : p.part_o;
#pragma unroll 4
        for (int r = warp; r < rows_here; r += 8) {
          const float2 f = stats[r];
          const int64_t to = reinterpret_cast<const int64_t*>(stats + 128)[r];
          float v[DP / 32];
#pragma unroll
          for (int x = 0; x < DP / 32; x++) v[x] = at(lane + 32 * x, r) * f.x;
#pragma unroll
          for (int x = 0; x < DP / 32; x++) {
            const int d = lane + 32 * x;
            if (d >= D) continue;
            if (add) v[x] = fmaf(p.pre_o[to + d], f.y, v[x]);
            dst[to + d] = v[x];
          }
        }
      };
      if (whole && !p.prefix && a.shared)
        write(std::true_type());
      else
        write(std::false_type());
      if (!whole) {
        const int c0 = (int)(((seg + 1) * runs - 1) / total);
        const int c1 = (int)(((seg + (long long)(cur.nt - 1) * KB + 1) * runs - 1) / total);
        const int np = c1 - c0 + 1;
        bar_sync(1, 256);
        if (tid == 0) *s_last = atom_add_acq_rel_gpu(p.tickets + c0, 1u) == (unsigned)(np - 1);
        bar_sync(1, 256);
        if (*s_last) {
          tile_join<DP>(p, cur, TT, c0, np, rows_here, warp, 8);
          if (tid == 0) p.tickets[c0] = 0u;
        }
      }
      bar_sync(1, 256);  // the staged output has been read
      if (!more) break;
      cur = nx, seg = nseg, k0 = nk0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ortc
