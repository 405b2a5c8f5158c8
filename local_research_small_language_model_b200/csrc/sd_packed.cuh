// Packed (ragged) sequences: how a CTA finds its tile, and the arguments that
// the CUDA-core and tensor-core attention kernels share.
#pragma once

#include "sd_common.cuh"

namespace sd {

struct PackedArgs {
  const void *q, *k, *v;                // [total][Hq|Hkv][64], element strides below
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int32_t *cu;                    // [S + 1] sequence bounds in the token rows
  int S, Hq, Hkv;
  int64_t total;
  float scale_log2;                     // softmax scale times log2(e)
  float scale;
  void *out;                            // forward output, row strides o_st, o_sh
  int64_t o_st, o_sh;
  float *lse;                           // [Hq][total] log2 of the row's exponential sum (nullable in the forward)
  void *rest;                           // nullable, contiguous [total][Hq][64]: what rounding took from out (16-bit)
  int zero_rest;                        // write zeros to the rows outside every sequence
  // backward
  const void *dout;
  int64_t g_st, g_sh;
  float *delta;                         // [Hq][total] rowsum(dout * out)
  void *dq, *dk, *dv;                   // contiguous
};

// A tile of kTile rows of one sequence.  start: first row of the sequence,
// len: its rows, row0: the tile's first row within the sequence (row0 < len
// where valid).  rest: the rows belong to no sequence (before cu[0] or from
// cu[S] on).
struct PackedTile {
  int64_t start;
  int len, row0;
  bool valid, rest;
};

// Tile slots need no prefix sums over the sequences: with b_i the bounds
// {0, cu[0], ..., cu[S], total} (S + 2 ranges, the first and the last holding
// the rows outside every sequence), range i owns the slots from
// floor(b_i / tile) + i, and ceil((b_{i+1} - b_i) / tile) of them are never
// more than up to the next range's first.  So total / tile + S + 2 slots hold
// every tile, and a warp finds a slot's range by a 32-way search (two rounds
// of loads for a thousand sequences).  Bounds are clamped to [0, total]: a
// malformed cu gives wrong rows but no access outside the tensors.
__device__ __forceinline__ int64_t packed_bound(const int32_t *cu, int S, int64_t total, int i) {
  if (i <= 0) return 0;
  if (i > S + 1) return total;
  const int64_t b = cu[i - 1];
  return b < 0 ? 0 : (b > total ? total : b);
}

inline int64_t packed_slots(int64_t total, int S, int tile) { return total / tile + S + 2; }

// Called by all 32 lanes of a warp with the same slot.
__device__ __forceinline__ PackedTile packed_find(const int32_t *cu, int S, int64_t total, int64_t slot, int tile) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = S + 2;  // the range is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const bool le = lane * step < n && packed_bound(cu, S, total, i) / tile + i <= slot;
    const unsigned hit = __ballot_sync(0xffffffffu, le);
    const int top = hit ? 31 - __clz(hit) : 0;
    const int end = lo + n;
    lo += top * step;
    n = min(step, end - lo);
  }
  const int64_t b = packed_bound(cu, S, total, lo), e = packed_bound(cu, S, total, lo + 1);
  PackedTile t;
  t.start = b;
  t.len = e > b ? static_cast<int>(e - b) : 0;
  const int64_t nth = slot - (b / tile + lo);
  t.rest = lo == 0 || lo == S + 1;
  t.valid = nth >= 0 && nth * tile < t.len;
  t.row0 = t.valid ? static_cast<int>(nth * tile) : 0;
  return t;
}

// The nth tile in order of falling work, for up to 128 sequences: CTAs start in
// launch order, and a long tile that starts late is what the others wait for
// (11 prompts, 16384 tokens: a fifth of the forward's time).  A tile with i
// tiles before it in its sequence (last_first: query tiles, which see the keys
// before them) or behind it (key tiles, seen by the queries behind them) has
// level i; f(i) = sum_s max(0, T_s - i) tiles have level i or more, so the nth
// tile's level is the largest i with f(i) > n, found by bisection with the
// counts T_s in registers.  Tiles of the rows outside every sequence follow.
// With more sequences than that: the slots above, in their order.
__device__ __forceinline__ PackedTile packed_nth(const int32_t *cu, int S, int64_t total, int64_t n, int64_t slots,
                                                 int tile, bool last_first) {
  constexpr int kEach = 4;  // sequences a lane
  if (S > 32 * kEach) return packed_find(cu, S, total, last_first ? slots - 1 - n : n, tile);
  const int lane = threadIdx.x & 31;
  int start[kEach], len[kEach], tiles[kEach], most = 0, all = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int s = lane + 32 * e;
    start[e] = len[e] = tiles[e] = 0;
    if (s < S) {
      start[e] = static_cast<int>(packed_bound(cu, S, total, s + 1));
      len[e] = max(0, static_cast<int>(packed_bound(cu, S, total, s + 2)) - start[e]);
      tiles[e] = static_cast<int>((static_cast<unsigned>(len[e]) + tile - 1) / tile);
    }
    most = max(most, tiles[e]);
    all += tiles[e];
  }
  PackedTile t = {};
  t.valid = true;
  if (S == 1) {
    all = __shfl_sync(0xffffffffu, tiles[0], 0);
    if (n < all) {
      t.start = __shfl_sync(0xffffffffu, start[0], 0);
      t.len = __shfl_sync(0xffffffffu, len[0], 0);
      t.row0 = (last_first ? all - 1 - static_cast<int>(n) : static_cast<int>(n)) * tile;
      return t;
    }
  } else {
    most = __reduce_max_sync(0xffffffffu, most);
    all = __reduce_add_sync(0xffffffffu, all);
  }
  if (n >= all) {  // the rows before cu[0], then those from cu[S] on
    n -= all;
    const int64_t first = packed_bound(cu, S, total, 1), last = packed_bound(cu, S, total, S + 1);
    const int64_t before = (first + tile - 1) / tile;
    t.rest = true;
    t.start = n < before ? 0 : last;
    t.len = static_cast<int>(n < before ? first : total - last);
    if (n >= before) n -= before;
    t.valid = n * tile < t.len;
    t.row0 = t.valid ? static_cast<int>(n * tile) : 0;
    return t;
  }
  auto from = [&](int i) {
    int c = max(0, tiles[0] - i);
    if (S > 32) {
#pragma unroll
      for (int e = 1; e < kEach; ++e) c += max(0, tiles[e] - i);
    }
    return static_cast<int>(__reduce_add_sync(0xffffffffu, c));
  };
  int lo = 0, hi = most, above = 0;  // f(lo) > n >= f(hi) = above
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, f = from(mid);
    if (f > n)
      lo = mid;
    else
      hi = mid, above = f;
  }
  int rank = static_cast<int>(n) - above;  // among the sequences with more than lo tiles
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const bool mine = tiles[e] > lo;
    const unsigned has = __ballot_sync(0xffffffffu, mine);
    const unsigned hit = __ballot_sync(0xffffffffu, mine && __popc(has & ((1u << lane) - 1u)) == rank);
    if (hit) {
      const int l = __ffs(hit) - 1, held = __shfl_sync(0xffffffffu, tiles[e], l);
      t.start = __shfl_sync(0xffffffffu, start[e], l);
      t.len = __shfl_sync(0xffffffffu, len[e], l);
      t.row0 = (last_first ? lo : held - 1 - lo) * tile;
      break;
    }
    rank -= __popc(has);
  }
  return t;
}

// The columns in which rows from .. to - 1 of v hold a NaN or an infinity, by a
// warp from the last row down until all of `want` are found: bit e of lane n
// stands for column (64 / kLanes) (n % kLanes) + e.
template <typename T>
__device__ __forceinline__ unsigned packed_not_finite(const T *v, int64_t stride, int from, int to, unsigned want) {
  constexpr int kCols = 16 / sizeof(T), kLanes = 64 / kCols, kAtOnce = 32 / kLanes, kUnroll = 8;
  const int lane = threadIdx.x & 31;
  unsigned found = 0;
  for (int r1 = to; r1 > from; r1 -= kAtOnce * kUnroll) {
    uint4 x[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = r1 - 1 - kAtOnce * u - lane / kLanes;
      x[u] = r >= from ? *reinterpret_cast<const uint4 *>(v + r * stride + lane % kLanes * kCols)
                       : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const T *p = reinterpret_cast<const T *>(&x[u]);
#pragma unroll
      for (int e = 0; e < kCols; ++e) found |= static_cast<unsigned>(!(fabsf(to_f(p[e])) < INFINITY)) << e;
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) found |= __shfl_xor_sync(0xffffffffu, found, o);
    if (!__any_sync(0xffffffffu, want & ~found)) break;
  }
  return found;
}

// Rows of the forward again, by a warp and without matrix products, where a masked
// weight of 0 met a NaN or an infinity of a later token's v, which the row does
// not see.  Rows `row` (of the sequence; below 0: none) of head h, with their
// references m and sums l from the fast path, whose blocks held the sequence's
// keys up to `end`.  Only columns are computed that hold such a value behind the
// row and none up to it: with one up to it, or a sum that is not finite, the
// result is not finite whatever is computed.  So a tensor full of NaN costs two
// looks at a few rows of v (32768 tokens: 2.2 ms instead of 1.7, 2.5 with one NaN
// in the first token); it is the rows before a column's first such value, fewer
// than a tile's, that walk over their keys (the worst: it is the last of 8192
// tokens, 17 ms, of 32768, 68 ms).  Two rows at a time: 24 ms with one; four, or a
// function that is not inlined, make the kernels' loops spill.
template <int R> struct PackedRows {
  int row[R];
  float m[R], l[R];
};
template <typename T, int R>
__device__ __forceinline__ void packed_again(const PackedArgs &a, int64_t start, int end, int h, const PackedRows<R> &g) {
  constexpr int kCols = 16 / sizeof(T), kLanes = 64 / kCols, kAtOnce = 32 / kLanes;
  const int lane = threadIdx.x & 31, hk = h / (a.Hq / a.Hkv);
  const T *q = static_cast<const T *>(a.q) + start * a.q_st + h * a.q_sh;
  const T *k = static_cast<const T *>(a.k) + start * a.k_st + hk * a.k_sh;
  const T *v = static_cast<const T *>(a.v) + start * a.v_st + hk * a.v_sh;
  const int c = lane % kLanes * kCols;  // this lane's columns; it reads every kAtOnce-th row of v
  unsigned again[R];                    // those of them to be computed
  int row[R], last = -1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    row[r] = -1, again[r] = 0;
    if (g.row[r] < 0 || !(g.l[r] > 0.f && g.l[r] < INFINITY)) continue;
    again[r] = packed_not_finite(v, a.v_st, g.row[r] + 1, end, (1u << kCols) - 1);
    if (__any_sync(0xffffffffu, again[r])) again[r] &= ~packed_not_finite(v, a.v_st, 0, g.row[r] + 1, again[r]);
    if (__any_sync(0xffffffffu, again[r])) row[r] = g.row[r], last = max(last, row[r]);
  }
  if (last < 0) return;
  float o[R][kCols] = {};
  for (int j0 = 0; j0 <= last; j0 += 32) {
    float p[R] = {};
    const T *kj = k + min(j0 + lane, last) * a.k_st;
#pragma unroll 4
    for (int d = 0; d < 64; d += kCols) {
      const uint4 y = *reinterpret_cast<const uint4 *>(kj + d);
      const T *py = reinterpret_cast<const T *>(&y);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint4 x = *reinterpret_cast<const uint4 *>(q + max(row[r], 0) * a.q_st + d);
        const T *px = reinterpret_cast<const T *>(&x);
#pragma unroll
        for (int e = 0; e < kCols; ++e) p[r] = fmaf(to_f(px[e]), to_f(py[e]), p[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = exp2f(fmaf(p[r], a.scale_log2, g.m[r] == -INFINITY ? 0.f : -g.m[r]));
#pragma unroll 4
    for (int t0 = 0; t0 < 32; t0 += kAtOnce) {
      const int t = t0 + lane / kLanes;
      const uint4 x = *reinterpret_cast<const uint4 *>(v + min(j0 + t, last) * a.v_st + c);
      const T *px = reinterpret_cast<const T *>(&x);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = __shfl_sync(0xffffffffu, p[r], t);
        if (j0 + t > row[r]) continue;
#pragma unroll
        for (int e = 0; e < kCols; ++e) o[r][e] = fmaf(w, to_f(px[e]), o[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int e = 0; e < kCols; ++e)
#pragma unroll
      for (int n = kLanes; n < 32; n <<= 1) o[r][e] += __shfl_xor_sync(0xffffffffu, o[r][e], n);
    if (row[r] < 0 || lane >= kLanes) continue;
    const int64_t at = start + row[r];
    T *out = static_cast<T *>(a.out) + at * a.o_st + h * a.o_sh + c;
#pragma unroll
    for (int e = 0; e < kCols; ++e) {
      if (!(again[r] >> e & 1)) continue;
      const float x = o[r][e] / g.l[r];
      out[e] = from_f<T>(x);
      if (a.rest) static_cast<T *>(a.rest)[(at * a.Hq + h) * 64 + c + e] = from_f<T>(x - round_to<T>(x));
    }
  }
}

// The tensor-core kernels (16-bit types).
int launch_packed_fwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s);
int launch_packed_bwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s);

}  // namespace sd
