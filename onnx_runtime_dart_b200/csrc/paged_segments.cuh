// The list of segments of the kernels that work on tiles of 128 query rows
// (csrc/paged_tile.cuh, csrc/paged_rows.cuh): a segment is (sequence, tile of
// 128 / group tokens with all their query heads of one KV head, KV head), as long as
// its keys are many plus EX for its start and end; the segments in order are cut
// into equal runs, one per CTA, at blocks of KB keys.
//
// A segment in several runs is joined by the last CTA of them, in run order.
#pragma once

#include "paged_stream.cuh"

namespace ortc {

struct TilePos {
  int b, rt, g;
  int row0, count, past;
  int lo, hi, nt, nrt;  // keys and blocks of this segment (lo a multiple of `align`); row tiles
  int len;              // keys it counts as in the list (the causal border unclamped)
  // the sequence: the first key of its row tiles (aligned), tiles that start there
  int base, ramp;
};

// Sets the sequence of `s`; its number of row tiles (0: not this kernel's; count -1: its
// lengths fall).
__device__ __forceinline__ int tile_seq(const StreamArgs& p, TilePos& s, int b, int min_past,
                                        int TT, int align) {
  const PagedAttnArgs& a = p.a;
  s.b = b;
  s.nrt = 0;
  if (p.prefix) {
    s.row0 = 0, s.past = 0;
    s.count = max(0, min(a.c.cu[a.c.batch], a.c.num_tokens));
    s.base = (a.window ? min(a.shared, max(0, min_past + 1 - a.window)) : 0) & -align;
  } else {
    const PagedSeq q = paged_seq(a.c, b, a.max_seq, a.shared);
    s.row0 = q.row0, s.count = q.count, s.past = q.past;
    if ((int64_t)q.count * a.group <= p.max_rows) return 0;
    s.base = a.shared & -align;
  }
  s.nrt = (s.count + TT - 1) / TT;
  s.ramp = s.nrt;
  if (!p.prefix && a.window) {
    const long long x = (long long)s.base + a.window - 1 - s.past;
    s.ramp = x < 0 ? 0 : (int)min((long long)s.nrt, x / TT + 1);
  }
  return s.nrt;
}

// Keys that row tiles 0 .. r - 1 of one KV head count as, with `extra` each.
__device__ __forceinline__ long long tile_sum(const StreamArgs& p, const TilePos& s, int r, int TT,
                                              int align, int extra) {
  if (p.prefix) return (long long)r * (max(1, p.a.shared - s.base) + extra);
  const long long f = min(r, s.ramp), c = r - f;
  return f * (s.past - s.base) + TT * (f * (f + 1) / 2) + c * (TT + p.a.window + align - 2) +
         (long long)r * extra;
}

// Sets the segment (rt, g) of the sequence of `s`.
template <int KB>
__device__ __forceinline__ void tile_segment(const StreamArgs& p, TilePos& s, int rt, int g,
                                             int TT, int align) {
  s.rt = rt, s.g = g;
  if (p.prefix) {
    s.lo = s.base, s.hi = p.a.shared;
    s.len = max(1, s.hi - s.lo);
  } else {
    const int t0 = s.past + rt * TT;
    const bool ramp = rt < s.ramp;
    s.lo = ramp ? s.base : (t0 + 1 - p.a.window) & -align;
    s.hi = min(s.past + s.count, t0 + TT);
    s.len = ramp ? t0 + TT - s.base : TT + p.a.window + align - 2;
  }
  s.nt = max(1, (s.hi - s.lo + KB - 1) / KB);
}

// A CTA's run: the segment and block it starts at, found from a scan over the batch
// (the lengths are on the device), and the walk from there.
template <int KB, int EX>
struct TileRun {
  TilePos cur;
  long long seg;  // place of block 0 of cur in the list
  int k0;         // first block of cur here
  long long total, u0, u1;
  int runs, min_past, TT, align;
  int nb;  // sequences: those before the first whose lengths fall

  // False: nothing to do.  Whole CTA; scratch of 19 * 8 bytes, free again at return.
  __device__ __forceinline__ bool plan(const StreamArgs& p, int TT_, int align_, void* scratch) {
    TT = TT_, align = align_;
    const PagedAttnArgs& a = p.a;
    const PagedView& c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nt = blockDim.x;
    const int G = c.kv_heads;
    nb = p.prefix ? 1 : c.batch;
    // warps, then the start and sequence of u0, the first sequence that falls
    long long* s_scan = static_cast<long long*>(scratch);
    int* s_falls = reinterpret_cast<int*>(s_scan + 18);
    if (tid == 0) *s_falls = INT_MAX;
    min_past = 0;
    if (p.prefix && a.window) {
      int* s_min = static_cast<int*>(scratch);
      min_past = INT_MAX / 2;
      for (int b = tid; b < c.batch; b += nt)
        if (c.cu[b + 1] > c.cu[b]) min_past = min(min_past, max(0, c.past[b]));
      min_past = __reduce_min_sync(~0u, min_past);
      if (lane == 0) s_min[warp] = min_past;
      __syncthreads();
      for (int i = 0; i < nt / 32; i++) min_past = min(min_past, s_min[i]);
      __syncthreads();
    }
    for (int pass = 0; pass < 2; pass++) {  // the total, then the sequence of u0
      long long base = 0;
      for (int b0 = 0; b0 < nb; b0 += nt) {
        TilePos t;
        t.count = 0;
        long long n = 0;
        if (b0 + tid < nb) {
          const int nrt = tile_seq(p, t, b0 + tid, min_past, TT, align);
          if (nrt) n = tile_sum(p, t, nrt, TT, align, EX) * G;
        }
        long long x = n;
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(~0u, x, o);
          if (lane >= o) x += y;
        }
        if (lane == 31) s_scan[warp] = x;
        const bool falls = t.count < 0;
        if (__syncthreads_or(falls)) {  // the list again, without what lies behind
          if (falls) atomicMin(s_falls, b0 + tid);
          __syncthreads();
          nb = *s_falls;
          base = 0, b0 = -nt;
          continue;
        }
        long long all = 0, before = 0;
        for (int i = 0; i < nt / 32; i++) {
          if (i < warp) before += s_scan[i];
          all += s_scan[i];
        }
        if (pass == 1) {
          const long long start = base + before + x - n;
          if (n && start <= u0 && u0 < start + n) {
            s_scan[16] = start;
            s_scan[17] = b0 + tid;
          }
        }
        base += all;
        __syncthreads();
      }
      if (pass == 0) {
        total = base;
        if (total == 0) return false;
        runs = (int)min((long long)gridDim.x, max(1ll, total / KB));  // a run holds a block at least
        if ((int)blockIdx.x >= runs) return false;
        u0 = total * blockIdx.x / runs;
        u1 = total * (blockIdx.x + 1) / runs;
      }
    }
    const long long off = u0 - s_scan[16];
    tile_seq(p, cur, (int)s_scan[17], min_past, TT, align);
    int lo = 0, hi = cur.nrt;  // the last row tile that starts at or before off
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile_sum(p, cur, mid, TT, align, EX) * G <= off)
        lo = mid;
      else
        hi = mid;
    }
    tile_segment<KB>(p, cur, lo, 0, TT, align);
    const long long rem = off - tile_sum(p, cur, lo, TT, align, EX) * G, each = cur.len + EX;
    cur.g = (int)(rem / each);
    const long long in = rem - cur.g * each - EX;
    seg = u0 - in;
    k0 = in <= 0 ? 0 : (int)((in + KB - 1) / KB);
    __syncthreads();  // the scratch has been read
    if (seg + (long long)k0 * KB >= u1 || k0 >= cur.nt) return next(p, cur, seg, k0);
    return true;
  }

  // To the next segment with a block in this run; false: none.
  __device__ __forceinline__ bool next(const StreamArgs& p, TilePos& s, long long& at,
                                       int& first) const {
    at += s.len + EX;
    if (at >= u1) return false;
    first = 0;
    if (s.g + 1 < p.a.c.kv_heads) {
      tile_segment<KB>(p, s, s.rt, s.g + 1, TT, align);
      return true;
    }
    if (s.rt + 1 < s.nrt) {
      tile_segment<KB>(p, s, s.rt + 1, 0, TT, align);
      return true;
    }
    int b = s.b + 1;
    while (b < nb && !tile_seq(p, s, b, min_past, TT, align)) b++;
    if (b >= nb) return false;
    tile_segment<KB>(p, s, 0, 0, TT, align);
    return true;
  }

  // Blocks of the segment at place `at` in this run, from block `first` on.
  __device__ __forceinline__ int blocks(const TilePos& s, long long at, int first) const {
    return (int)min((long long)s.nt, (u1 - at + KB - 1) / KB) - first;
  }
};

// Position of the token `tok` of the prefix pass (rows of different sequences).
__device__ __forceinline__ int prefix_position(const PagedView& c, int tok) {
  int lo = 0, hi = c.batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c.cu[mid + 1] <= tok)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < c.batch ? c.past[lo] + tok - c.cu[lo] : INT_MAX / 2;
}

// Where the row r of a segment's tile is written: (token, head).
__device__ __forceinline__ int64_t tile_place(const StreamArgs& p, const TilePos& s, int TT, int r) {
  const int t = p.group_div.div(r);
  return (int64_t)(s.row0 + s.rt * TT + t) * p.a.heads + s.g * p.a.group + r - t * p.a.group;
}

// Joins the np pieces that CTAs c0 .. c0 + np - 1 left of a segment: warp w of nw
// takes rows w, w + nw, ..., four at a time (their loads are in flight together).
template <int DP>
__device__ __forceinline__ void tile_join(const StreamArgs& p, const TilePos& s, int TT, int c0,
                                          int np, int rows, int w, int nw) {
  const int lane = threadIdx.x & 31, D = p.a.c.D;
  constexpr int L4 = DP / 4;      // lanes of a row: 16 bytes each
  constexpr int RW = 32 / L4;     // rows a warp loads at once
  const int q = lane % L4, sub = lane / L4;
  for (int r0 = w * 4 * RW; r0 < rows; r0 += nw * 4 * RW) {
    float M[4], L[4];
    float4 v[4];
    int r[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
      r[x] = r0 + x * RW + sub;
      M[x] = -INFINITY, L[x] = 0.f, v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = 0; i < np; i++) {
      const int64_t slot = (int64_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * 128;
      float2 ml[4];
      float4 t[4];
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int64_t at = slot + min(r[x], rows - 1);
        ml[x] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
        t[x] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * DP) + q);
      }
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const float mn = fmaxf(M[x], ml[x].x), mb = mn == -INFINITY ? 0.f : mn;
        const float fa = ex2(M[x] - mb), fb = ex2(ml[x].x - mb);
        M[x] = mn;
        L[x] = L[x] * fa + ml[x].y * fb;
        v[x].x = v[x].x * fa + t[x].x * fb, v[x].y = v[x].y * fa + t[x].y * fb;
        v[x].z = v[x].z * fa + t[x].z * fb, v[x].w = v[x].w * fa + t[x].w * fb;
      }
    }
#pragma unroll
    for (int x = 0; x < 4; x++)
      if (r[x] < rows && 4 * q < D) write4(p, tile_place(p, s, TT, r[x]), 4 * q, M[x], L[x], v[x]);
  }
}

}  // namespace ortc
