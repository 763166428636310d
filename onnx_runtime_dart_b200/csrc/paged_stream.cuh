// Attention over the paged KV cache for few query rows per sequence and KV
// head (decode steps, drafted tokens, a batch over a shared prefix): a stream
// over the keys.
//
// One CTA per SM.  A segment is (sequence, tile of R query rows, KV head); its
// keys are cut into tiles of 8 warps x KW keys, and the tiles of all segments,
// in order (and a few places more for each segment), are cut into equal runs,
// one per CTA, whatever the sequences' lengths are (read on the device; every
// CTA finds its run from a scan over the batch).  Each warp owns KW keys of every tile with a ring of
// its own in shared memory, filled by cp.async some tiles ahead, across
// segment borders, and its own running maximum and sum (no CTA barrier inside
// a segment); the warps' states are joined at a segment's end.  A segment that
// lies in several CTAs' runs is joined by the last of them (a ticket), in run
// order, so results do not depend on timing.
//
// The products run on mma.sync (rows as M = 16, so tcgen05's M = 128 would be
// empty for the most part; the bound is the key stream).  They keep fp32
// results from 16-bit operands by splitting the fp32 side, q and the softmax
// weights p, into parts of the cache's type whose products are exact in fp32:
// fp16 hi + lo (22 bits; q scaled by a power of two per row, p by 2^15, so
// that the low part keeps its bits), bf16 hi + mid + lo (24 bits).  fp32 pages
// take tf32 with both sides split in two (hi.hi + lo.hi + hi.lo).  Up to 8
// rows, a row's hi and lo parts are rows r and r + 8 of one MMA, so the split
// costs nothing.
//
// Bound by memory over fp16 pages: 64 sequences of 100 to 8191 keys 84 us, 5.7 TB/s
// (0.87 of the copy); one of 131000 keys 98 us, 5.5 TB/s.  bf16 (100 us) and fp32 pages
// (203 us) take more steps a key with two warps a scheduler, and are bound by their
// latency at 4.8 and 4.7 TB/s, 8 rows with capped scores at 4.1 (tensor pipe 26 %, issue
// slots 38 %).
//
// Operand layouts avoid shuffles and transposes: the feature order of q.k is
// free, so a lane's 16-byte chunk of a key row serves as its B operand of two
// MMAs; the score accumulator is, after exp2, the A operand of p.v; and a
// lane's 16-byte chunks of the value rows 2c, 2c + 1, 2c + 8, 2c + 9 give,
// with byte permutes, its B operand of eight MMAs.
#pragma once

#include <type_traits>

#include <cuda_bf16.h>

#include "paged.cuh"

namespace ortc {

struct StreamArgs {
  PagedAttnArgs a;
  FastDiv page_div, group_div;
  int q_vec = 0, out_vec = 0;  // 16-byte loads of q rows, stores of out
  int prefix = 0;      // 1: rows of all tokens over keys [0, shared) of row 0's pages
  int max_rows = 0;    // sequences with more query rows per KV head are not this kernel's
  float t_scale = 0;   // scale (softcap: scale / softcap)
  float t_mul = 0;     // log2(e) (softcap: softcap * log2(e))
  unsigned* tickets = nullptr;  // one per CTA, zero between calls
  float* part_ml = nullptr;     // [2 * grid][R][2]
  float* part_o = nullptr;      // [2 * grid][R][DP]
  // prefix results per (token, head): maximum and sum, unnormalised output
  float* pre_ml = nullptr;
  float* pre_o = nullptr;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a row's unnormalised values, and those that the prefix pass left, are
// multiplied by, from the row's maximum and sum.
__device__ __forceinline__ float2 paged_row_scale(const StreamArgs& p, int64_t at, float M,
                                                  float L) {
  if (p.prefix) return make_float2(1.f, 0.f);
  float wa = 1.f, wb = 0.f;
  if (p.a.shared) {
    const float2 pm = *reinterpret_cast<const float2*>(p.pre_ml + 2 * at);
    const float mm = fmaxf(M, pm.x), mb = mm == -INFINITY ? 0.f : mm;
    wa = ex2(M - mb), wb = ex2(pm.x - mb);
    L = L * wa + pm.y * wb;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  return make_float2(wa * inv, wb * inv);
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1,
                                          __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1,
                                          __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_1688(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_rna(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return y;
}

// The parts of a pair of fp32 values in the cache's 16-bit type: PARTS words,
// each rounded to nearest from what the ones before it left.
template <typename T>
struct Split;
template <>
struct Split<__half> {
  static constexpr int PARTS = 2;
  static __device__ __forceinline__ void pair(float x, float y, uint32_t (&w)[2]) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    w[0] = *reinterpret_cast<const uint32_t*>(&h);
    w[1] = *reinterpret_cast<const uint32_t*>(&l);
  }
};
template <>
struct Split<__nv_bfloat16> {
  static constexpr int PARTS = 3;
  static __device__ __forceinline__ void pair(float x, float y, uint32_t (&w)[3]) {
#pragma unroll
    for (int i = 0; i < 3; i++) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      const float2 f = __bfloat1622float2(h);
      x -= f.x, y -= f.y;
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <>
struct Split<float> {
  static constexpr int PARTS = 2;
  static __device__ __forceinline__ void one(float x, uint32_t (&w)[2]) {
    w[0] = tf32_rna(x);
    w[1] = tf32_rna(x - __uint_as_float(w[0]));
  }
};

// The base of a row's weights exp2(score - base), from its largest score; what a row
// keeps as its maximum.  fp16: 15 below it, so that the weights' low parts keep their
// bits, rounded up, so that none passes 2^15 however large the scores are (a score of
// 2^24 less 15, rounded to nearest, may be 16 below it, and 2^16 is no fp16 number).
template <typename T>
__device__ __forceinline__ float row_base(float mx) {
  return std::is_same<T, __half>::value ? __fadd_ru(mx, -15.f) : mx;
}

template <typename T, int DP, int R>
struct StreamCfg {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int KW = F32 ? 8 : 16;           // keys of a warp per tile
  static constexpr int TK = 8 * KW;                 // keys of a tile
  static constexpr int CHP = DP * (int)sizeof(T) / 16;  // 16-byte chunks of a padded row
  static constexpr int ROWB = DP * (int)sizeof(T);
  static constexpr int WSTAGE = 2 * KW * ROWB;      // a warp's stage: K rows, V rows
  static constexpr int NS = 3 * 8192 / WSTAGE;      // 24 KB of ring per warp
  static constexpr int KS = F32 ? DP / 8 : DP / 16; // k-steps of q.k
  // q operands: R = 8 packs two parts into the 16 rows of an MMA
  static constexpr int QP = R == 8 ? (Split<T>::PARTS + 1) / 2 : Split<T>::PARTS;
  static constexpr int QB = QP * KS * 512;
  static constexpr int RING = 8 * NS * WSTAGE;
  // A segment's start and end cost about as much as two 64 KB tiles; the list
  // counts them, so that a run of many short sequences is no longer than one of a
  // long sequence.  Measured at 1, 2, 3 tiles: 64 sequences of 100 to 8191 keys 86.2,
  // 82.1, 84.0 us (uncounted 113), one of 131000 keys 95.8, 94.8, 94.8 us.
  static constexpr int EXTRA = 2 * 128 / DP;
  static_assert(R * DP * 4 <= WSTAGE, "a warp's output is handed over in its free stage");
  // the ring, two sets of operands, (max, sum) per warp and row
  static constexpr int SMEM = RING + 2 * QB + 8 * R * 8;
};

// Where a CTA is in the list of tiles: tile `tile` of segment (b, rt, g).
struct StreamPos {
  int b, rt, g, tile;
  int row0, count, past;    // the sequence
  int lo, hi, nt, nrt;      // its keys, key tiles and row tiles
};

// Sets the sequence of `s`; false: nothing for this kernel (count -1: its lengths fall).
template <int R, int TK>
__host__ __device__ __forceinline__ bool stream_seq(const StreamArgs& p, StreamPos& s, int b,
                                                    int min_past) {
  const PagedAttnArgs& a = p.a;
  s.b = b;
  if (p.prefix) {
    s.row0 = 0, s.past = 0;
    s.count = max(0, min(a.c.cu[a.c.batch], a.c.num_tokens));
    s.lo = a.window ? min(a.shared, max(0, min_past + 1 - a.window)) : 0;
    s.hi = a.shared;
  } else {
    const PagedSeq q = paged_seq(a.c, b, a.max_seq, a.shared);
    s.row0 = q.row0, s.count = q.count, s.past = q.past;
    s.lo = max(a.shared, a.window ? q.past + 1 - a.window : 0);
    s.hi = q.past + q.count;
  }
  const int64_t rows = (int64_t)s.count * a.group;
  if (rows <= 0 || (!p.prefix && rows > p.max_rows)) {
    s.nt = s.nrt = 0;
    return false;
  }
  s.nrt = (int)((rows + R - 1) / R);
  s.nt = max(1, (s.hi - s.lo + TK - 1) / TK);
  return true;
}

// The sequence's length in the list per KV head.  It passes 32 bits where a KV head has
// more query heads than a tile takes: 128 heads and 131072 tokens over fp32 pages are
// 1048576 row tiles of 2050 places.
template <int EXTRA>
__host__ __device__ __forceinline__ long long stream_places(const StreamPos& s) {
  return (long long)(s.nt + EXTRA) * s.nrt;
}

// One step of a warp: 8 NT keys at `base` (bit r of `valid`: key r is there) in
// shared memory at kt, vt against its R rows, whose operands are qs, score factors
// fac, positions pos (from pos_lo to pos_hi over the rows); m, l, o: the rows'
// running maximum (row_base), this lane's part of the sum, output.
template <typename T, int DP, int R, int NT = StreamCfg<T, DP, R>::KW / 8>
__device__ __forceinline__ void stream_step(const uint4* qs, const unsigned char* kt,
                                            const unsigned char* vt, unsigned valid, int base,
                                            const float (&fac)[R / 8], const int (&pos)[R / 8],
                                            int pos_lo, int pos_hi, int window, bool softcap,
                                            float t_mul, float (&m)[R / 8], float (&l)[R / 8],
                                            float (&o)[DP / 64][8][R / 4]) {
  using C = StreamCfg<T, DP, R>;
  constexpr bool F32 = C::F32;
  constexpr int KW = 8 * NT, CHP = C::CHP, KS = C::KS, PARTS = Split<T>::PARTS, NPASS = DP / 64;
  constexpr int NR = R / 8;
  constexpr unsigned kAll = ~0u >> (32 - KW);
  const int lane = threadIdx.x & 31;
  // scores
  float s[NT][2][4];  // two chains of products each
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) s[t][0][e] = s[t][1][e] = 0.f;
  const int row = lane >> 2, cl = lane & 3;
#pragma unroll
  for (int ks = 0; ks < KS; ks += 2) {
    const int ch = cl + 4 * (ks >> 1);
    uint4 kv[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
      kv[t] = *reinterpret_cast<const uint4*>(kt + (row + 8 * t) * C::ROWB +
                                              ((ch ^ ((row & 1) << 2)) << 4));
    if constexpr (F32) {
      uint4 qa[2], ql[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        qa[e] = qs[(ks + e) * 32 + lane];
        if (R == 16) ql[e] = qs[(KS + ks + e) * 32 + lane];
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        uint32_t kh[4], kl[4];
        const float kx[4] = {__uint_as_float(kv[t].x), __uint_as_float(kv[t].y),
                             __uint_as_float(kv[t].z), __uint_as_float(kv[t].w)};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t ww[2];
          Split<float>::one(kx[e], ww);
          kh[e] = ww[0], kl[e] = ww[1];
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          mma_1688(s[t][e], qa[e], kl[2 * e], kl[2 * e + 1]);
          if (R == 16) mma_1688(s[t][e], ql[e], kh[2 * e], kh[2 * e + 1]);
          mma_1688(s[t][e], qa[e], kh[2 * e], kh[2 * e + 1]);
        }
      }
    } else {
#pragma unroll
      for (int pt = 0; pt < C::QP; pt++) {
        const uint4 q0 = qs[(pt * KS + ks) * 32 + lane], q1 = qs[(pt * KS + ks + 1) * 32 + lane];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          mma_16816(s[t][0], q0, kv[t].x, kv[t].y, T());
          mma_16816(s[t][1], q1, kv[t].z, kv[t].w, T());
        }
      }
    }
  }

  // softmax weights; rows (lane / 4) + 8 rr, keys base + 8 t + 2 cl + e
  const bool full = valid == kAll && base + KW - 1 <= pos_lo &&
                    (!window || base > pos_hi - window);
  float pr[NR][NT][2];
#pragma unroll
  for (int rr = 0; rr < NR; rr++)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = s[t][0][2 * rr + e] + s[t][1][2 * rr + e];
        if (R == 8) x += s[t][0][e + 2] + s[t][1][e + 2];
        x *= fac[rr];
        if (softcap) x = tanhf(x);
        pr[rr][t][e] = __fmul_rn(x, t_mul);  // not fused with the subtraction of the base below
      }
  if (!full) {
#pragma unroll
    for (int rr = 0; rr < NR; rr++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int k = 8 * t + 2 * cl + e, j = base + k;
          if (!((valid >> k) & 1) || j > pos[rr] || (window && j <= pos[rr] - window))
            pr[rr][t][e] = -INFINITY;
        }
  }
  float corr[NR];
#pragma unroll
  for (int rr = 0; rr < NR; rr++) {
    constexpr bool shifted = std::is_same<T, __half>::value;
    float mx = shifted ? -INFINITY : m[rr];
#pragma unroll
    for (int t = 0; t < NT; t++) mx = fmaxf(mx, fmaxf(pr[rr][t][0], pr[rr][t][1]));
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
    if (shifted) mx = fmaxf(m[rr], row_base<T>(mx));
    const float mb = mx == -INFINITY ? 0.f : mx;
    corr[rr] = ex2(m[rr] - mb);
    m[rr] = mx;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        pr[rr][t][e] = ex2(pr[rr][t][e] - mb);
        sum += pr[rr][t][e];
      }
    l[rr] = l[rr] * corr[rr] + sum;
  }
  // A value that only some rows see must not reach the others as 0 * inf:
  // such tiles (the border of the mask) are looked over, and one that holds
  // an infinity or NaN is summed key by key.
  bool odd = false;
  if (!full) {
#pragma unroll
    for (int x = 0; x < KW * CHP / 32; x++) {
      const uint4 v = reinterpret_cast<const uint4*>(vt)[x * 32 + lane];
      const uint32_t ws[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (F32) {
          odd |= (ws[e] & 0x7f800000u) == 0x7f800000u;
        } else {
          constexpr uint32_t inf = PARTS == 2 ? 0x7c00u : 0x7f80u;
          odd |= (ws[e] & inf) == inf || ((ws[e] >> 16) & inf) == inf;
        }
      }
    }
    odd = __any_sync(~0u, odd);
  }
  if (odd) {
#pragma unroll
    for (int x = 0; x < NPASS; x++)
#pragma unroll
      for (int i2 = 0; i2 < 8; i2++)
#pragma unroll
        for (int e = 0; e < 2 * NR; e++) o[x][i2][e] *= corr[e >> 1];
    for (int k = 0; k < KW; k++) {
      float pk[NR];
#pragma unroll
      for (int rr = 0; rr < NR; rr++) {
        float mine = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (k == 8 * t + 2 * cl + e) mine = pr[rr][t][e];
        pk[rr] = __shfl_sync(~0u, mine, (lane & ~3) | ((k >> 1) & 3));
      }
      const T* vr = reinterpret_cast<const T*>(vt + k * C::ROWB);
#pragma unroll
      for (int x = 0; x < NPASS; x++)
#pragma unroll
        for (int i2 = 0; i2 < 8; i2++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            // feature of accumulator (x, i2, column 2 cl + e)
            const int d = F32 ? x * 64 + (i2 >> 2) * 32 + (2 * cl + e) * 4 + (i2 & 3)
                              : x * 64 + (2 * cl + e) * 8 + i2;
            constexpr int PC = 16 / (int)sizeof(T);
            const int dd = ((d / PC) ^ (((k >> 1) & 3) << 1)) * PC + d % PC;
            const float v = (float)vr[dd];
#pragma unroll
            for (int rr = 0; rr < NR; rr++)
              if (pk[rr] != 0.f) o[x][i2][2 * rr + e] = fmaf(pk[rr], v, o[x][i2][2 * rr + e]);
          }
    }
    return;
  }

  // o = o corr + p . v, the products of a tile in accumulators of their own:
  // the tensor cores' sums are cut off, not rounded, and over a long run of
  // tiles that adds up (1.5e-6 of the result over 131000 keys, against 0.5e-6
  // so)
  auto add = [&](float(&acc)[2 * NR], const float(&d)[4]) {
    if constexpr (R == 8) {
      acc[0] = fmaf(acc[0], corr[0], d[0] + d[2]);
      acc[1] = fmaf(acc[1], corr[0], d[1] + d[3]);
    } else {
      acc[0] = fmaf(acc[0], corr[0], d[0]);
      acc[1] = fmaf(acc[1], corr[0], d[1]);
      acc[2] = fmaf(acc[2], corr[NR - 1], d[2]);
      acc[3] = fmaf(acc[3], corr[NR - 1], d[3]);
    }
  };
  if constexpr (F32) {
    uint4 pa[NT][2];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      uint32_t w0[2], w1[2];
      Split<float>::one(pr[0][t][0], w0);
      Split<float>::one(pr[0][t][1], w1);
      if (R == 8) {
        pa[t][0] = make_uint4(w0[0], w0[1], w1[0], w1[1]);
      } else {
        uint32_t y0[2], y1[2];
        Split<float>::one(pr[NR - 1][t][0], y0);
        Split<float>::one(pr[NR - 1][t][1], y1);
        pa[t][0] = make_uint4(w0[0], y0[0], w1[0], y1[0]);
        pa[t][1] = make_uint4(w0[1], y0[1], w1[1], y1[1]);
      }
    }
#pragma unroll
    for (int x = 0; x < DP / 32; x++) {
      const int ch = row + 8 * x;
      float d[4][4];
#pragma unroll
      for (int e = 0; e < 4; e++) d[e][0] = d[e][1] = d[e][2] = d[e][3] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const unsigned char* vr = vt + (8 * t + 2 * cl) * C::ROWB + ((ch ^ (cl << 1)) << 4);
        const uint4 v0 = *reinterpret_cast<const uint4*>(vr);
        const uint4 v1 = *reinterpret_cast<const uint4*>(vr + C::ROWB);
        const uint32_t a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          uint32_t h0[2], h1[2];
          Split<float>::one(__uint_as_float(a0[e]), h0);
          Split<float>::one(__uint_as_float(a1[e]), h1);
          mma_1688(d[e], pa[t][0], h0[1], h1[1]);
          if (R == 16) mma_1688(d[e], pa[t][1], h0[0], h1[0]);
          mma_1688(d[e], pa[t][0], h0[0], h1[0]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) add(o[x >> 1][(x & 1) * 4 + e], d[e]);
    }
  } else {
    uint4 pa[C::QP];
    {
      uint32_t w0[PARTS], w1[PARTS];
      Split<T>::pair(pr[0][0][0], pr[0][0][1], w0);
      Split<T>::pair(pr[0][NT - 1][0], pr[0][NT - 1][1], w1);
      if (R == 8) {
        pa[0] = make_uint4(w0[0], w0[1], w1[0], w1[1]);
        if (PARTS == 3) pa[C::QP - 1] = make_uint4(w0[PARTS - 1], 0u, w1[PARTS - 1], 0u);
      } else {
        uint32_t y0[PARTS], y1[PARTS];
        Split<T>::pair(pr[NR - 1][0][0], pr[NR - 1][0][1], y0);
        Split<T>::pair(pr[NR - 1][NT - 1][0], pr[NR - 1][NT - 1][1], y1);
#pragma unroll
        for (int pt = 0; pt < PARTS; pt++)
          pa[pt < C::QP ? pt : 0] = make_uint4(w0[pt], y0[pt], w1[pt], y1[pt]);
      }
    }
#pragma unroll
    for (int x = 0; x < NPASS; x++) {
      const int ch = row + 8 * x;
      uint4 v[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = 2 * cl + (e & 1) + 8 * (e >> 1);
        v[e] = *reinterpret_cast<const uint4*>(vt + r * C::ROWB + ((ch ^ (cl << 1)) << 4));
      }
      const uint32_t a0[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
      const uint32_t a1[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
      const uint32_t a8[4] = {v[2].x, v[2].y, v[2].z, v[2].w};
      const uint32_t a9[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
        const uint32_t b0 = __byte_perm(a0[e >> 1], a1[e >> 1], sel);
        const uint32_t b1 = __byte_perm(a8[e >> 1], a9[e >> 1], sel);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int pt = 0; pt < C::QP; pt++) mma_16816(d, pa[pt], b0, b1, T());
        add(o[x][e], d);
      }
    }
  }
}

// Writes features d .. d + 3 of (token, head) `at` (D is a multiple of 8): the output,
// joined with what the prefix pass left, or, in the prefix pass, that.
__device__ __forceinline__ void write4(const StreamArgs& p, int64_t at, int d, float M, float L,
                                       float4 v) {
  const PagedAttnArgs& a = p.a;
  const int D = a.c.D;
  if (p.prefix) {
    *reinterpret_cast<float4*>(p.pre_o + at * D + d) = v;
    if (d == 0) *reinterpret_cast<float2*>(p.pre_ml + 2 * at) = make_float2(M, L);
    return;
  }
  const float2 f = paged_row_scale(p, at, M, L);
  v.x *= f.x, v.y *= f.x, v.z *= f.x, v.w *= f.x;
  if (a.shared) {
    const float4 t = *reinterpret_cast<const float4*>(p.pre_o + at * D + d);
    v.x = fmaf(t.x, f.y, v.x), v.y = fmaf(t.y, f.y, v.y);
    v.z = fmaf(t.z, f.y, v.z), v.w = fmaf(t.w, f.y, v.w);
  }
  float* dst = a.out + at * D + d;
  if (p.out_vec)
    *reinterpret_cast<float4*>(dst) = v;
  else
    dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
}

// The same for query row idx of a segment's sequence and KV head.
__device__ __forceinline__ void stream_finish(const StreamArgs& p, const StreamPos& s, int idx,
                                              int d, float M, float L, float4 v) {
  const int tok = p.group_div.div(idx), h = s.g * p.a.group + idx - tok * p.a.group;
  write4(p, (int64_t)(s.row0 + tok) * p.a.heads + h, d, M, L, v);
}

template <typename T, int DP, int R>
__global__ void __launch_bounds__(256, 1) paged_stream_kernel(const __grid_constant__ StreamArgs p) {
  using C = StreamCfg<T, DP, R>;
  constexpr bool F32 = C::F32;
  constexpr int KW = C::KW, TK = C::TK, EXTRA = C::EXTRA, CHP = C::CHP, NS = C::NS, KS = C::KS, PARTS = Split<T>::PARTS;
  constexpr int NPASS = DP / 64;       // blocks of 64 features of the output
  constexpr int NR = R / 8;            // rows a lane holds
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem;
  uint4* qf = reinterpret_cast<uint4*>(smem + C::RING);  // [2][QP][KS][32]: segments in turn
  float2* wml = reinterpret_cast<float2*>(smem + C::RING + 2 * C::QB);  // [8][R]
  __shared__ long long s_scan[8];
  __shared__ long long s_u0base;
  __shared__ int s_b0, s_min[8], s_last, s_falls;
  __shared__ float s_fac[2][R];   // score factor of a row
  __shared__ int s_pos[2][R];     // position of a row, INT_MIN: no row

  const PagedAttnArgs& a = p.a;
  const PagedView& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int D = c.D, G = c.kv_heads;
  int nb = p.prefix ? 1 : c.batch;  // sequences: those before the first whose lengths fall

  // ---- this CTA's run of tiles
  if (tid == 0) s_falls = INT_MAX;
  int min_past = 0;
  if (p.prefix && a.window) {
    min_past = INT_MAX;
    for (int b = tid; b < c.batch; b += 256)
      if (c.cu[b + 1] > c.cu[b]) min_past = min(min_past, max(0, c.past[b]));
    min_past = __reduce_min_sync(~0u, min_past);
    if (lane == 0) s_min[w] = min_past;
    __syncthreads();
    for (int i = 0; i < 8; i++) min_past = min(min_past, s_min[i]);
    if (min_past > INT_MAX / 2) min_past = INT_MAX / 2;
  }
  StreamPos cur;
  long long total = 0, u0 = 0, u1 = 0;
  int runs = 1;  // CTAs with work: one tile each at least
  for (int pass = 0; pass < 2; pass++) {  // total, then the sequence of u0
    long long base = 0;
    for (int b0 = 0; b0 < nb; b0 += 256) {
      StreamPos t;
      t.count = 0;
      const long long n = b0 + tid < nb && stream_seq<R, TK>(p, t, b0 + tid, min_past)
                              ? stream_places<EXTRA>(t) * G
                              : 0;
      long long x = n;
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[w] = x;
      const bool falls = t.count < 0;
      if (__syncthreads_or(falls)) {  // the list again, without what lies behind
        if (falls) atomicMin(&s_falls, b0 + tid);
        __syncthreads();
        nb = s_falls;
        base = 0, b0 = -256;
        continue;
      }
      long long all = 0, before = 0;
      for (int i = 0; i < 8; i++) {
        if (i < w) before += s_scan[i];
        all += s_scan[i];
      }
      if (pass == 1) {
        const long long start = base + before + x - n;
        if (n && start <= u0 && u0 < start + n) {
          s_b0 = b0 + tid;
          s_u0base = start;
        }
      }
      base += all;
      __syncthreads();
      if (pass == 0 && nb <= 256) {  // one block of sequences: find u0 without a second scan
        total = all;
        runs = (int)min((long long)gridDim.x, max(total, 1ll));
        u0 = total * blockIdx.x / runs;
        const long long start = before + x - n;
        if (n && start <= u0 && u0 < start + n) {
          s_b0 = tid;
          s_u0base = start;
        }
      }
    }
    if (pass == 0) {
      total = base;
      runs = (int)min((long long)gridDim.x, max(total, 1ll));
      u0 = total * blockIdx.x / runs;
      u1 = total * (blockIdx.x + 1) / runs;
      if (nb <= 256) break;
    }
  }
  __syncthreads();
  if ((int)blockIdx.x >= runs || u0 >= u1) return;
  stream_seq<R, TK>(p, cur, s_b0, min_past);
  long long seg_u = s_u0base;  // place of tile 0 of the segment in the list
  {
    const int len = cur.nt + EXTRA;
    const long long off = u0 - s_u0base, sg = off / len;
    cur.tile = max(0, (int)(off - sg * len) - EXTRA);
    cur.g = (int)(sg % G);
    cur.rt = (int)(sg / G);
    seg_u += sg * len + EXTRA;
  }
  if (seg_u + cur.tile >= u1) return;  // a run inside a segment's extra places

  // ---- loads
  unsigned char* wring = ring + w * NS * C::WSTAGE;
  const uint32_t wring_s = smem_u32(wring);
  const int chunks = D * (int)sizeof(T) / 16;
  StreamPos ld = cur;      // the tile to load next
  long long lu = seg_u + cur.tile;  // its place in the list
  int ld_stage = 0;
  unsigned valid_q[NS];    // per stage: bit r set when key r of the warp is there
#pragma unroll
  for (int i = 0; i < NS; i++) valid_q[i] = 0;
  auto advance = [&](StreamPos& s) {
    if (++s.tile < s.nt) return;
    s.tile = 0;
    if (++s.g < G) return;
    s.g = 0;
    if (++s.rt < s.nrt) return;
    s.rt = 0;
    for (int b = s.b + 1; b < nb; b++)
      if (stream_seq<R, TK>(p, s, b, min_past)) return;
  };
  // the page of lane r's key (r < KW) of a tile, and whether it has one
  auto page_of = [&](const StreamPos& s, int& slot) {
    const int j = s.lo + s.tile * TK + w * KW + (lane & (KW - 1));
    slot = 0;
    if (j >= s.hi) return -1;
    const int pg = p.page_div.div(j);
    slot = j - pg * c.page_size;
    return __ldg(c.table + (int64_t)(p.prefix ? 0 : s.b) * c.max_pages + pg);
  };
  int nslot = 0, npage = page_of(ld, nslot);  // of tile lu
  auto issue = [&](unsigned& valid) {  // loads tile lu; fetches the page of the next one
    const int page = npage, slot = nslot, g = ld.g;
    const bool there = ld.lo + ld.tile * TK + w * KW + (lane & (KW - 1)) < ld.hi;
    if (there && (page < 0 || page >= c.num_pages)) record_error(c.err, KERR_PAGED_PAGE);
    const bool ok = there && page >= 0 && page < c.num_pages;
    const long long off =
        ok ? (long long)page * c.page_elems + (long long)slot * c.row_elems + (long long)g * D : -1;
    valid = __ballot_sync(~0u, ok) & ((1u << KW) - 1);
    lu += ld.tile + 1 == ld.nt ? 1 + EXTRA : 1;
    if (lu < u1) {
      advance(ld);
      npage = page_of(ld, nslot);
    }
    const uint32_t st = wring_s + ld_stage * C::WSTAGE;
    constexpr int RPI = CHP >= 32 ? 1 : 32 / CHP;  // rows per instruction
    const int ch = lane & (CHP - 1);
#pragma unroll
    for (int i = 0; i < KW / RPI; i++) {
      const int r = i * RPI + lane / CHP;
      const long long o = __shfl_sync(~0u, off, r);
      const int bytes = o >= 0 && ch < chunks ? 16 : 0;
      const long long e = bytes ? o + ch * (16 / (int)sizeof(T)) : 0;
      cp16(st + r * C::ROWB + ((ch ^ ((r & 1) << 2)) << 4), static_cast<const T*>(c.key) + e, bytes);
      cp16(st + KW * C::ROWB + r * C::ROWB + ((ch ^ (((r >> 1) & 3) << 1)) << 4),
           static_cast<const T*>(c.value) + e, bytes);
    }
    if (++ld_stage == NS) ld_stage = 0;
  };
  auto commit = [] { asm volatile("cp.async.commit_group;\n" ::: "memory"); };
#pragma unroll
  for (int i = 0; i < NS - 1; i++) {
    if (lu < u1) issue(valid_q[i]);
    commit();
  }

  // ---- q rows: warp w brings rows w, w + 8 of a segment's tile into registers and,
  // later, as A operands into one of the two sets
  constexpr int E = DP / 32;  // features of a lane
  float qx[NR][E];
  auto row_of = [&](const StreamPos& s, int r, int& tok, int& h) {
    const int idx = s.rt * R + r;
    const bool row = idx < s.count * a.group;
    tok = row ? p.group_div.div(idx) : 0;
    h = s.g * a.group + (row ? idx - tok * a.group : 0);
    return row;
  };
  auto load_q = [&](const StreamPos& s) {
#pragma unroll
    for (int rr = 0; rr < NR; rr++) {
      int tok, h;
      const bool row = row_of(s, w + 8 * rr, tok, h);
      const float* src = a.q + (int64_t)(s.row0 + tok) * a.q_stride + (int64_t)h * D;
#pragma unroll
      for (int e = 0; e < E; e++) qx[rr][e] = 0.f;
      if (!row) continue;
      if (E == 4 && p.q_vec && 4 * lane + 3 < D) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(src) + lane);
        qx[rr][0] = v.x, qx[rr][1] = v.y, qx[rr][E - 2] = v.z, qx[rr][E - 1] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (E * lane + e < D) qx[rr][e] = __ldg(src + E * lane + e);
      }
    }
  };
  auto build_q = [&](const StreamPos& s, int set) {
    uint32_t* qw = reinterpret_cast<uint32_t*>(qf + set * (C::QB / 16));
    // word `reg` of k-step s of part pt for MMA lane ml
    auto put = [&](int pt, int s, int ml, int reg, uint32_t v) {
      qw[(((pt * KS + s) * 32) + ml) * 4 + reg] = v;
    };
#pragma unroll
    for (int rr = 0; rr < NR; rr++) {
      const int r = w + 8 * rr;
      int tok, h;
      const bool row = row_of(s, r, tok, h);
      int pos = INT_MIN;
      if (row) {
        pos = s.past + tok;
        if (p.prefix) {
          pos = INT_MAX / 2;  // past the prefix
          if (a.window) {
            const int b = paged_find(c, tok);
            pos = b < c.batch ? c.past[b] + tok - c.cu[b] : INT_MAX / 2;
          }
        }
      }
      float(&x)[E] = qx[rr];
      float fac = p.t_scale;
      if constexpr (!F32 && PARTS == 2) {  // fp16: the row's largest value into [2^13, 2^14)
        float mx = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) mx = fmaxf(mx, fabsf(x[e]));
        mx = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mx)));
        int ex = (int)(__float_as_uint(mx) >> 23) - 127;
        ex = max(-100, min(ex, 126));
        const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
#pragma unroll
        for (int e = 0; e < E; e++) x[e] *= up;
        fac *= __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
      }
      if (lane == 0) {
        s_fac[set][r] = fac;
        s_pos[set][r] = pos;
      }
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const int d = E * lane + e;
        if constexpr (F32) {  // chunk of 4: features 0, 1 in k-step 2i, 2, 3 in 2i + 1
          const int ch = d >> 2, s = 2 * (ch >> 2) + ((d >> 1) & 1), ml = (r & 7) * 4 + (ch & 3);
          uint32_t w0[2], w1[2];
          Split<float>::one(x[e], w0);
          Split<float>::one(x[e + 1], w1);
#pragma unroll
          for (int pt = 0; pt < 2; pt++) {
            const int reg = R == 8 ? pt : rr, part = R == 8 ? 0 : pt;
            put(part, s, ml, reg, w0[pt]);
            put(part, s, ml, reg + 2, w1[pt]);
          }
        } else {  // chunk of 8: features 0..3 in k-step 2i, 4..7 in 2i + 1
          const int ch = d >> 3, s = 2 * (ch >> 2) + ((d >> 2) & 1), ml = (r & 7) * 4 + (ch & 3);
          const int hi2 = ((d >> 1) & 1) * 2;
          uint32_t wd[PARTS];
          Split<T>::pair(x[e], x[e + 1], wd);
#pragma unroll
          for (int pt = 0; pt < PARTS; pt++) {
            if (R == 8)
              put(pt >> 1, s, ml, (pt & 1) + hi2, wd[pt]);
            else
              put(pt, s, ml, rr + hi2, wd[pt]);
          }
          if (R == 8 && PARTS == 3) put(1, s, ml, 1 + hi2, 0u);
        }
      }
    }
  };

  // ---- segments
  int stage = 0, set = 0;
  load_q(cur);
  build_q(cur, 0);
  __syncthreads();
  for (;;) {
    const int n = (int)min((long long)cur.nt, u1 - seg_u) - cur.tile;  // tiles of it in this run
    const bool more = seg_u + cur.nt + EXTRA < u1;
    StreamPos nx = cur;  // the next segment: its q rows come while this one's keys do
    if (more) {
      nx.tile = nx.nt - 1;
      advance(nx);
      load_q(nx);
    }
    const uint4* qs = qf + set * (C::QB / 16);
    float fac[NR];
    int pos[NR];
    int pos_lo = INT_MAX, pos_hi = INT_MIN;  // over the tile's rows
#pragma unroll
    for (int rr = 0; rr < NR; rr++) {
      fac[rr] = s_fac[set][(lane >> 2) + 8 * rr];
      pos[rr] = s_pos[set][(lane >> 2) + 8 * rr];
      if (pos[rr] != INT_MIN) {
        pos_lo = min(pos_lo, pos[rr]);
        pos_hi = max(pos_hi, pos[rr]);
      }
    }
    pos_lo = __reduce_min_sync(~0u, pos_lo);
    pos_hi = __reduce_max_sync(~0u, pos_hi);

    float m[NR], l[NR], o[NPASS][8][2 * NR];
#pragma unroll
    for (int rr = 0; rr < NR; rr++) m[rr] = -INFINITY, l[rr] = 0.f;
#pragma unroll
    for (int x = 0; x < NPASS; x++)
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 2 * NR; e++) o[x][i][e] = 0.f;

    for (int i = 0; i < n; i++) {
      // the tile NS - 1 ahead into the stage that was read last
      __syncwarp();
      unsigned next_valid = 0;
      if (lu < u1) issue(next_valid);
      commit();
      asm volatile("cp.async.wait_group %0;\n" ::"n"(NS - 1) : "memory");
      __syncwarp();
      const unsigned valid = valid_q[0];
#pragma unroll
      for (int x = 0; x + 1 < NS - 1; x++) valid_q[x] = valid_q[x + 1];
      valid_q[NS - 2] = next_valid;
      const unsigned char* kt = wring + stage * C::WSTAGE;
      const unsigned char* vt = kt + KW * C::ROWB;
      if (++stage == NS) stage = 0;
      const int base = cur.lo + (cur.tile + i) * TK + w * KW;
      if (valid == 0) continue;

      stream_step<T, DP, R>(qs, kt, vt, valid, base, fac, pos, pos_lo, pos_hi, a.window,
                            a.softcap > 0.f, p.t_mul, m, l, o);
    }

    // ---- the segment's end: each warp hands over its rows' state, the output in the
    // stage of its ring that the next load will fill
    const int row = lane >> 2, cl = lane & 3;
    __syncwarp();  // the stage has been read
    float* mine = reinterpret_cast<float*>(wring + (stage == 0 ? NS - 1 : stage - 1) * C::WSTAGE);
#pragma unroll
    for (int rr = 0; rr < NR; rr++) {
      l[rr] += __shfl_xor_sync(~0u, l[rr], 1);
      l[rr] += __shfl_xor_sync(~0u, l[rr], 2);
      if (cl == 0) wml[w * R + row + 8 * rr] = make_float2(m[rr], l[rr]);
#pragma unroll
      for (int x = 0; x < NPASS; x++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int i2 = 0; i2 < 8; i2 += 4) {
            // features d .. d + 3, pieces of 16 bytes swizzled by the row
            const int d = x * 64 + (F32 ? (i2 >> 2) * 32 + (2 * cl + e) * 4 : (2 * cl + e) * 8 + i2);
            *reinterpret_cast<float4*>(mine + (row + 8 * rr) * DP + (((d >> 2) ^ row) << 2)) =
                make_float4(o[x][i2][2 * rr + e], o[x][i2 + 1][2 * rr + e], o[x][i2 + 2][2 * rr + e],
                            o[x][i2 + 3][2 * rr + e]);
          }
    }
    if (more) build_q(nx, set ^ 1);
    const int free_stage = (stage == 0 ? NS - 1 : stage - 1) * C::WSTAGE;
    __syncthreads();
    const bool whole = n == cur.nt;
    const bool head = cur.tile != 0;  // begun in an earlier CTA
    const int slot = 2 * blockIdx.x + (head ? 0 : 1);
    const int rows_here = min(R, cur.count * a.group - cur.rt * R);
    for (int e = tid; e < rows_here * (DP / 4); e += 256) {
      const int r = e / (DP / 4), q = e % (DP / 4);
      float M = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; i++) M = fmaxf(M, wml[i * R + r].x);
      const float mb = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float2 s2 = wml[i * R + r];
        const float f = ex2(s2.x - mb);
        // every warp is at the same stage of its ring
        const float4 t = *reinterpret_cast<const float4*>(
            ring + i * NS * C::WSTAGE + free_stage + (r * DP + ((q ^ (r & 7)) << 2)) * 4);
        L = fmaf(f, s2.y, L);
        v.x = fmaf(f, t.x, v.x), v.y = fmaf(f, t.y, v.y);
        v.z = fmaf(f, t.z, v.z), v.w = fmaf(f, t.w, v.w);
      }
      if (4 * q >= D) continue;
      if (whole) {
        stream_finish(p, cur, cur.rt * R + r, 4 * q, M, L, v);
      } else {
        const int64_t at = (int64_t)slot * R + r;
        *reinterpret_cast<float4*>(p.part_o + at * DP + 4 * q) = v;
        if (q == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
      }
    }
    if (!whole) {
      // the runs that hold this segment: CTAs c0 .. c1
      const int c0 = (int)(((seg_u + 1) * runs - 1) / total);
      const int c1 = (int)(((seg_u + cur.nt) * runs - 1) / total);
      const int np = c1 - c0 + 1;
      __syncthreads();
      if (tid == 0)  // releases this CTA's partials (ordered by the barrier), acquires the others'
        s_last = atom_add_acq_rel_gpu(p.tickets + c0, 1u) == (unsigned)(np - 1);
      __syncthreads();
      if (s_last) {
        for (int r = w; r < rows_here; r += 8) {
          auto piece = [&](int i) { return (int64_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * R + r; };
          float M = -INFINITY;
          for (int i = lane; i < np; i += 32) M = fmaxf(M, __ldcg(p.part_ml + piece(i) * 2));
          for (int x = 16; x; x >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, x));
          const float mb = M == -INFINITY ? 0.f : M;
          float L = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          const bool in = 4 * lane < D;
          for (int i0 = 0; i0 < np; i0 += 32) {
            float2 q = make_float2(-INFINITY, 0.f);
            if (i0 + lane < np)
              q = __ldcg(reinterpret_cast<const float2*>(p.part_ml + piece(i0 + lane) * 2));
            const float f = ex2(q.x - mb);
            L = fmaf(f, q.y, L);
            const int k = min(32, np - i0);
#pragma unroll 8
            for (int i = 0; i < k; i++) {
              const float f1 = __shfl_sync(~0u, f, i);
              if (!in) continue;
              const float4 t = __ldcg(
                  reinterpret_cast<const float4*>(p.part_o + piece(i0 + i) * DP + 4 * lane));
              v.x = fmaf(f1, t.x, v.x), v.y = fmaf(f1, t.y, v.y);
              v.z = fmaf(f1, t.z, v.z), v.w = fmaf(f1, t.w, v.w);
            }
          }
          for (int x = 16; x; x >>= 1) L += __shfl_xor_sync(~0u, L, x);
          if (in) stream_finish(p, cur, cur.rt * R + r, 4 * lane, M, L, v);
        }
        if (tid == 0) p.tickets[c0] = 0u;
      }
    }
    if (!more) break;
    __syncthreads();  // the handed-over states have been read
    seg_u += cur.nt + EXTRA;
    cur = nx;
    set ^= 1;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

}  // namespace ortc
