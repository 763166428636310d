// Attention over fp32 pages for many query rows per sequence and KV head: tiles of
// 128 query rows, 16 a warp, that read the keys together.
//
// The steps are those of the key stream (csrc/paged_stream.cuh: tf32 products with
// both sides split in two, fp32 softmax and sums); here the eight warps share the
// keys, 32 at a time through a ring of shared memory with one barrier a block, where
// there they share the rows.  Each warp leaves out the steps whose keys none of its rows
// sees (the causal border, the window).  Bound by the latency of eight warps, two a
// scheduler at 230 registers and more (tensor pipe 34 %, issue slots 40 %); each of them
// splits every key and value into its two tf32 parts for itself.  1000 + 300 tokens of 32
// heads of 64: 177 us, 29 TFLOP/s; 2048 tokens of heads of 128: 877 us, 39 TFLOP/s.
#pragma once

#include "paged_segments.cuh"

namespace ortc {

template <int DP>
struct RowsCfg {
  using S = StreamCfg<float, DP, 16>;
  static constexpr int KB = 32;                   // keys of a block
  static constexpr int STAGE = 2 * KB * S::ROWB;  // K rows, V rows
  static constexpr int NS = DP == 128 ? 3 : 4;
  static constexpr int QW = S::QB;                // q operands of a warp
  static constexpr int SMEM = NS * STAGE + 8 * QW;
  // a segment's start and end, in keys (173, 191, 225 us at 4, 8, 16 blocks)
  static constexpr int EXTRA = 4 * KB;
};

template <int DP>
__global__ void __launch_bounds__(256, 1) paged_rows_kernel(const __grid_constant__ StreamArgs p) {
  using C = RowsCfg<DP>;
  using S = StreamCfg<float, DP, 16>;
  constexpr int KB = C::KB, NS = C::NS, ROWB = S::ROWB, CHP = S::CHP, KS = S::KS, E = DP / 32;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ long long s_plan[19];
  __shared__ unsigned char s_ok[NS][KB];
  __shared__ int s_last;
  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, D = c.D, TT = 128 / a.group;
  unsigned char* ring = smem;
  uint4* qs = reinterpret_cast<uint4*>(smem + NS * C::STAGE + w * C::QW);  // this warp's

  TileRun<KB, C::EXTRA> run;
  if (!run.plan(p, TT, 1, s_plan)) return;
  TilePos cur = run.cur;
  long long seg = run.seg;
  int k0 = run.k0;
  const int chunks = D / 4, ch = tid & (CHP - 1);
  for (;;) {
    const int n = run.blocks(cur, seg, k0);
    const int tok0 = cur.rt * TT, rows = min(TT, cur.count - tok0) * a.group;
    auto issue = [&](int i) {  // block i of this run into its stage
      const uint32_t st = smem_u32(ring) + (i % NS) * C::STAGE;
      const int base = cur.lo + (k0 + i) * KB;
#pragma unroll
      for (int y = 0; y < KB * CHP / 256; y++) {
        const int r = (tid + 256 * y) / CHP, j = base + r;
        int64_t off = -1;
        if (j < cur.hi) {
          const int pg = p.page_div.div(j);
          const int page = __ldg(c.table + (int64_t)(p.prefix ? 0 : cur.b) * c.max_pages + pg);
          if (page >= 0 && page < c.num_pages)
            off = (int64_t)page * c.page_elems + (int64_t)(j - pg * c.page_size) * c.row_elems +
                  (int64_t)cur.g * D;
          else
            record_error(c.err, KERR_PAGED_PAGE);
        }
        if (ch == 0) s_ok[i % NS][r] = off >= 0;
        const int bytes = off >= 0 && ch < chunks ? 16 : 0;
        const int64_t e = bytes ? off + ch * 4 : 0;
        cp16(st + r * ROWB + ((ch ^ ((r & 1) << 2)) << 4), static_cast<const float*>(c.key) + e,
             bytes);
        cp16(st + KB * ROWB + r * ROWB + ((ch ^ (((r >> 1) & 3) << 1)) << 4),
             static_cast<const float*>(c.value) + e, bytes);
      }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;\n" ::: "memory"); };
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
      if (i < n) issue(i);
      commit();
    }
    // this warp's rows 16 w .. 16 w + 15, lane's features E lane ..
#pragma unroll 4
    for (int y = 0; y < 16; y++) {
      const int r = 16 * w + y;
      float x[E];
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = 0.f;
      if (r < rows) {
        const int t = p.group_div.div(r);
        const float* src = a.q + (int64_t)(cur.row0 + tok0 + t) * a.q_stride +
                           (int64_t)(cur.g * a.group + r - t * a.group) * D;
#pragma unroll
        for (int e = 0; e < E; e++)
          if (E * lane + e < D) x[e] = __ldg(src + E * lane + e);
      }
      uint32_t* qw = reinterpret_cast<uint32_t*>(qs);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const int d = E * lane + e, cd = d >> 2, s = 2 * (cd >> 2) + ((d >> 1) & 1);
        const int ml = (y & 7) * 4 + (cd & 3);
        uint32_t w0[2], w1[2];
        Split<float>::one(x[e], w0);
        Split<float>::one(x[e + 1], w1);
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
          uint32_t* at = qw + ((pt * KS + s) * 32 + ml) * 4 + (y >> 3);
          at[0] = w0[pt];
          at[2] = w1[pt];
        }
      }
    }
    __syncwarp();
    float fac[2], m[2], l[2], o[DP / 64][8][4];
    int pos[2], pos_lo = INT_MAX, pos_hi = INT_MIN;
#pragma unroll
    for (int rr = 0; rr < 2; rr++) {
      const int r = 16 * w + (lane >> 2) + 8 * rr;
      fac[rr] = p.t_scale, m[rr] = -INFINITY, l[rr] = 0.f;
      pos[rr] = INT_MIN;
      if (r < rows) {
        const int tok = tok0 + p.group_div.div(r);
        pos[rr] = !p.prefix ? cur.past + tok : a.window ? prefix_position(c, tok) : INT_MAX / 2;
        pos_lo = min(pos_lo, pos[rr]);
        pos_hi = max(pos_hi, pos[rr]);
      }
    }
    pos_lo = __reduce_min_sync(~0u, pos_lo);
    pos_hi = __reduce_max_sync(~0u, pos_hi);
#pragma unroll
    for (int x = 0; x < DP / 64; x++)
#pragma unroll
      for (int i = 0; i < 8; i++) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;

    for (int i = 0; i < n; i++) {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(NS - 2) : "memory");
      __syncthreads();  // block i is there for all; block i - 1 has been read by all
      if (i + NS - 1 < n) issue(i + NS - 1);
      commit();
      const unsigned char* kt = ring + (i % NS) * C::STAGE;
      const unsigned there = __ballot_sync(~0u, s_ok[i % NS][lane] != 0);
      const int base = cur.lo + (k0 + i) * KB;
      if (there == 0 || base > pos_hi || (a.window && base + KB - 1 <= pos_lo - a.window)) continue;
      stream_step<float, DP, 16, KB / 8>(qs, kt, kt + KB * ROWB, there, base, fac, pos, pos_lo,
                                         pos_hi, a.window, a.softcap > 0.f, p.t_mul, m, l, o);
    }

    const bool whole = n == cur.nt;
    const int slot = 2 * blockIdx.x + (k0 ? 0 : 1);
    const int cl = lane & 3;
#pragma unroll
    for (int rr = 0; rr < 2; rr++) {
      const int r = 16 * w + (lane >> 2) + 8 * rr;
      l[rr] += __shfl_xor_sync(~0u, l[rr], 1);
      l[rr] += __shfl_xor_sync(~0u, l[rr], 2);
      if (r >= rows) continue;
      const int64_t at = whole ? tile_place(p, cur, TT, r) : (int64_t)slot * 128 + r;
#pragma unroll
      for (int x = 0; x < DP / 64; x++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int i2 = 0; i2 < 8; i2 += 4) {
            const int d = x * 64 + (i2 >> 2) * 32 + (2 * cl + e) * 4;
            const float4 v = make_float4(o[x][i2][2 * rr + e], o[x][i2 + 1][2 * rr + e],
                                         o[x][i2 + 2][2 * rr + e], o[x][i2 + 3][2 * rr + e]);
            if (!whole)
              *reinterpret_cast<float4*>(p.part_o + at * DP + d) = v;
            else if (d < D)
              write4(p, at, d, m[rr], l[rr], v);
          }
      if (!whole && cl == 0)
        *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[rr], l[rr]);
    }
    __syncthreads();  // the ring has been read
    if (!whole) {
      const int c0 = (int)(((seg + 1) * run.runs - 1) / run.total);
      const int c1 = (int)(((seg + (long long)(cur.nt - 1) * KB + 1) * run.runs - 1) / run.total);
      const int np = c1 - c0 + 1;
      if (tid == 0)  // releases this CTA's partials (ordered by the barrier), acquires the others'
        s_last = atom_add_acq_rel_gpu(p.tickets + c0, 1u) == (unsigned)(np - 1);
      __syncthreads();
      if (s_last) {
        tile_join<DP>(p, cur, TT, c0, np, rows, w, 8);
        if (tid == 0) p.tickets[c0] = 0u;
      }
      __syncthreads();
    }
    if (!run.next(p, cur, seg, k0)) break;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

}  // namespace ortc
