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
  float *delta;                         // [Hq][total] rowsum(dout * out), and one word more
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

// One row of the forward again, by a warp and without matrix products, for a
// result that is not finite: there a masked weight of 0 met a NaN or an infinity
// of a later token's v, which the row does not see; or it does see one, and the
// result stays what it is.  Row `row` (of the sequence) of head h, with its
// reference m and sum l from the fast path.
template <typename T>
__device__ __forceinline__ void packed_row(const PackedArgs &a, int64_t start, int row, int h, float m, float l) {
  const int lane = threadIdx.x & 31, hk = h / (a.Hq / a.Hkv);
  const T *q = static_cast<const T *>(a.q) + (start + row) * a.q_st + h * a.q_sh;
  const T *k = static_cast<const T *>(a.k) + start * a.k_st + hk * a.k_sh;
  const T *v = static_cast<const T *>(a.v) + start * a.v_st + hk * a.v_sh;
  float o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 <= row; j0 += 32) {
    float p = 0.f;
    if (j0 + lane <= row) {
      const T *kj = k + (j0 + lane) * a.k_st;
      float s = 0.f;
      for (int d = 0; d < 64; ++d) s = fmaf(to_f(q[d]), to_f(kj[d]), s);
      p = exp2f(fmaf(s, a.scale_log2, m == -INFINITY ? 0.f : -m));
    }
    const int n = min(32, row + 1 - j0);
    for (int t = 0; t < n; ++t) {
      const float w = __shfl_sync(0xffffffffu, p, t);
      const T *vj = v + (j0 + t) * a.v_st + 2 * lane;
      o0 = fmaf(w, to_f(vj[0]), o0);
      o1 = fmaf(w, to_f(vj[1]), o1);
    }
  }
  o0 /= l, o1 /= l;
  T *out = static_cast<T *>(a.out) + (start + row) * a.o_st + h * a.o_sh + 2 * lane;
  out[0] = from_f<T>(o0), out[1] = from_f<T>(o1);
  if (a.rest) {
    T *rest = static_cast<T *>(a.rest) + ((start + row) * a.Hq + h) * 64 + 2 * lane;
    rest[0] = from_f<T>(o0 - round_to<T>(o0)), rest[1] = from_f<T>(o1 - round_to<T>(o1));
  }
}

// The tensor-core kernels (16-bit types).
int launch_packed_fwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s);
int launch_packed_bwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s);

}  // namespace sd
