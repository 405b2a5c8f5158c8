// Paged key-value cache: the append, and the attention of one new token of
// every sequence over its pages.
//
// A pool holds pages of `page` tokens, k_pages and v_pages [P][Hkv][page][64]
// (any strides with an innermost one of 1).  Position t of sequence b lies in
// page table[b][t / page], row t % page.
#include "sd_tma.cuh"

namespace sd {

struct PagedArgs {
  const int32_t *table;  // [B][width]
  int64_t t_sb;
  int width;
  const int32_t *lens;   // [B]
  int B, Hq, Hkv, page;
  int64_t pages, p_sp, p_sh, p_st;  // pool size and element strides
  int32_t *err;
};

namespace pg {

__device__ __forceinline__ void report(int32_t *err, int code) {
  if (err) *err = code;
}

// Tokens that the table can hold, and the sequence's length clamped to them.
__device__ __forceinline__ int seq_len(const PagedArgs &a, int b) {
  const int64_t cap = static_cast<int64_t>(a.width) * a.page;
  const int n = a.lens[b];
  if (n < 0 || n > cap) {
    report(a.err, SD_KERR_BOUNDS);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}

// Element offset of position t of sequence b in the pool, or -1 when its page
// is not a page of the pool.
__device__ __forceinline__ int64_t row_of(const PagedArgs &a, int b, int h, int t) {
  const int nth = t / a.page;
  const int64_t p = a.table[b * a.t_sb + nth];
  if (p < 0 || p >= a.pages) return -1;
  return p * a.p_sp + h * a.p_sh + (t - nth * a.page) * a.p_st;
}

}  // namespace pg

// The append: kTok rows a CTA, whose places the first kTok threads look up; then
// all threads move 16-byte chunks of K and V, several in flight each.  cu
// (nullable): token rows [cu[b], cu[b + 1]) belong to sequence b; without it row
// b is sequence b's one token.  Rows outside every sequence, and those of an
// absent one, are not written anywhere.  HBM-bound: 32768 rows of 4 bf16 heads into pages of 64 tokens in
// 12.4 us (67 MB, 5.4 TB/s with the launch); 64 single tokens 4.2 us, the launch
// and three loads that depend on one another (length, page, value).
template <typename T, int kTok>
__global__ void __launch_bounds__(256)
    paged_append_kernel(PagedArgs a, const int32_t *cu, int64_t N, const T *xk, const T *xv, int64_t k_sn,
                        int64_t k_sh, int64_t v_sn, int64_t v_sh, T *k_pages, T *v_pages) {
  constexpr int kVec = 16 / sizeof(T), kChunks = 64 / kVec, kUnroll = 4;
  __shared__ int64_t place[kTok];  // element offset of the row in the pool, head 0; -1: dropped
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kTok;
  const int rows = static_cast<int>(N - n0 < kTok ? N - n0 : kTok), tid = threadIdx.x;
  if (tid < rows) {
    const int64_t n = n0 + tid;
    int b = static_cast<int>(n);
    int64_t t = 0, off = -1;
    bool held = true;
    if (cu) {
      int lo = 0, hi = a.B;  // the last b with cu[b] <= n, if n < cu[b + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= n) lo = mid; else hi = mid;
      }
      b = lo;
      held = n >= cu[b] && n < cu[b + 1];
      t = n - cu[b];
    }
    const int before = held ? a.lens[b] : SD_LEN_ABSENT;
    if (before != SD_LEN_ABSENT) {
      t += before;
      if (t >= 0 && t < static_cast<int64_t>(a.width) * a.page) off = pg::row_of(a, b, 0, static_cast<int>(t));
      if (off < 0) pg::report(a.err, SD_KERR_BOUNDS);
    }
    place[tid] = off;
  }
  __syncthreads();
  const int chunks = rows * a.Hkv * kChunks;
  for (int e0 = tid; e0 < chunks; e0 += 256 * kUnroll) {
    uint4 k[kUnroll], v[kUnroll];
    int64_t to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int e = e0 + 256 * u;
      to[u] = -1;
      if (e >= chunks) continue;
      const int c = e % kChunks * kVec, hr = e / kChunks, r = hr / a.Hkv, h = hr - r * a.Hkv;
      if (place[r] < 0) continue;
      to[u] = place[r] + h * a.p_sh + c;
      k[u] = *reinterpret_cast<const uint4 *>(xk + (n0 + r) * k_sn + h * k_sh + c);
      v[u] = *reinterpret_cast<const uint4 *>(xv + (n0 + r) * v_sn + h * v_sh + c);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (to[u] >= 0) {
        *reinterpret_cast<uint4 *>(k_pages + to[u]) = k[u];
        *reinterpret_cast<uint4 *>(v_pages + to[u]) = v[u];
      }
  }
}

// ---------------------------------------------------------------- decode
//   out = sum_t exp2(c q.k_t - m) v_t / sum_t exp2(c q.k_t - m),  c = scale log2(e)
//
// HBM-bound: every cached K and V row is read once for all the query heads of
// its kv head.  The work is cut into units (sequence, head group, 64 tokens;
// 32 in fp32), numbered in that order, and each of 3 CTAs an SM takes an equal
// run of them, whatever the lengths are: a CTA may end one sequence's head,
// do several and begin another.  What a CTA holds of a head whole it writes out
// itself; the other parts (running maximum, sum, weighted values) go to the
// workspace, and a second kernel joins them in order.
//
// A warp owns a quarter of every unit's tokens with its own copies (cp.async,
// 16 bytes a lane, kStages units ahead, page ids looked up one unit earlier
// still) and its own softmax state, so the loop has no block barrier; the four
// states meet at the end of a head.  16-bit products are mma.sync m16n8k16 with
// up to 16 query heads as the rows (a kv head has few: a 128-row tcgen05 tile
// would be mostly padding, and the tensor pipe is not what bounds this).
//
// Measured, 12 query and 4 key-value heads: 64 sequences up to 16384 tokens, bf16,
// 738 MB in 121 us (6.1 TB/s); one of 32768 tokens 14.4 us (33.5 MB, 5.1 us of
// reading: start-up of the copies, the join and its launch are the rest); 5 up to
// 1100 tokens in fp32 with pages of 24 tokens 12.5 us (nearly all latency: a
// unit's length, page and rows depend on one another).
namespace pg {

constexpr int kThreads = 128, kWarps = 4, kStages = 4;
constexpr int kMaxHeads = 16;                // query heads of a group
constexpr int kCtas = 148 * 3;
constexpr int kMaxSeqs = 2048;               // sequences of a launch (two ints each in shared memory)
constexpr int kPart = 66;                    // m, l, 64 values
constexpr int kWarpBytes = 4096;             // a warp's K and V rows of one unit
template <typename T> constexpr int kUnit = sizeof(T) == 2 ? 64 : 32;

struct DecodeArgs {
  const void *q;
  int64_t q_sb, q_sh;
  const void *k, *v;
  void *out;
  int64_t o_sb, o_sh;
  float scale_log2;
  int G, Hh;           // query heads of a group, groups of all kv heads (Hkv x groups a kv head)
  uint32_t page_inv;   // floor(2^32 / page), 2^32 - 1 for a page of 1
  int32_t *plan;       // [B + 1] units before each sequence (of one head group), then units a CTA
  float *parts;        // [kCtas][2][G][kPart]
};

struct Cursor {
  int b, hh, tile;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool held) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(held ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// t / page: the estimate is never above and at most one below for t < 2^31.
__device__ __forceinline__ int page_of(int t, int page, uint32_t inv) {
  int p = static_cast<int>(__umulhi(static_cast<uint32_t>(t), inv));
  return t - p * page >= page ? p + 1 : p;
}

// What a part with maximum m weighs under the common maximum.
__device__ __forceinline__ float factor(float m, float top) { return m == -INFINITY ? 0.f : ex2(m - top); }

}  // namespace pg

// kWhole: a warp's tokens of a unit lie in one page (the page size is a multiple
// of them), so a unit takes one look-up and its rows follow each other; kWide:
// more than 8 query heads a group (the fragments' second 8 rows hold heads too).
template <typename T, bool kWhole, bool kWide>
__global__ void __launch_bounds__(pg::kThreads, 3) paged_decode_kernel(const PagedArgs a, const pg::DecodeArgs d) {
  using namespace pg;
  constexpr bool k16 = sizeof(T) == 2;
  constexpr int kTok = kUnit<T>, kMine = kTok / kWarps;  // tokens of a unit, and of a warp
  constexpr int kRow = 64 * sizeof(T), kChunks = kRow / 16, kRowsAt = 32 / kChunks;  // rows of one copy of a warp
  constexpr int kCopies = kMine / kRowsAt;
  extern __shared__ __align__(128) char sm[];
  char *ring = sm;                                                   // [warp][stage][K rows | V rows]
  uint8_t *held = reinterpret_cast<uint8_t *>(sm + kWarps * kStages * kWarpBytes);  // [warp][stage][16]
  float *merge = reinterpret_cast<float *>(held + kWarps * kStages * 16);           // [warp][G][kPart]
  float *sq = merge + kWarps * d.G * kPart;                          // fp32: [G][64]
  int *pre = reinterpret_cast<int *>(k16 ? sq : sq + d.G * 64), *len = pre + a.B + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- lengths, and the units before each sequence
  {
    __shared__ int sums[kWarps];
    int run = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + tid;
      const int n = b < a.B ? seq_len(a, b) : 0;
      int x = (n + kTok - 1) / kTok;
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) sums[warp] = x;
      __syncthreads();
      int before = run, all = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[w];
        all += sums[w];
      }
      if (b < a.B) {
        pre[b] = before + x - own;
        len[b] = n;
      }
      run += all;
      __syncthreads();
    }
    if (tid == 0) pre[a.B] = run;
    __syncthreads();
  }
  const int64_t units = static_cast<int64_t>(pre[a.B]) * d.Hh;
  const int64_t per = units <= 0x7fffffff - kCtas ? (static_cast<uint32_t>(units) + gridDim.x - 1) / gridDim.x
                                                  : (units + gridDim.x - 1) / gridDim.x;
  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.B; b += kThreads) d.plan[b] = pre[b];
    if (tid == 0) d.plan[a.B + 1] = static_cast<int>(per);
  }
  const int64_t u0 = blockIdx.x * per, u1 = u0 + per < units ? u0 + per : units;
  // the joining kernel may be brought in from here on; it waits for this one's end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (u0 >= u1) return;

  // ---- the first unit
  Cursor at;
  {
    int lo = 0, hi = a.B;  // the last b with pre[b] * Hh <= u0 that has units
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<int64_t>(pre[mid]) * d.Hh <= u0) lo = mid; else hi = mid;
    }
    const int tiles = pre[lo + 1] - pre[lo];
    const int64_t in = u0 - static_cast<int64_t>(pre[lo]) * d.Hh;
    if (in <= 0x7fffffff)
      at = {lo, static_cast<int>(in) / tiles, static_cast<int>(in) % tiles};
    else
      at = {lo, static_cast<int>(in / tiles), static_cast<int>(in % tiles)};
  }
  auto advance = [&](Cursor &c) {
    if (++c.tile < pre[c.b + 1] - pre[c.b]) return;
    c.tile = 0;
    if (++c.hh < d.Hh) return;
    c.hh = 0;
    do ++c.b;
    while (c.b < a.B && pre[c.b + 1] == pre[c.b]);
  };
  const int groups = d.Hh / a.Hkv;  // groups of a kv head

  // ---- copies: this lane's rows of a unit
  const int row0 = lane / kChunks, chunk = lane % kChunks;
  Cursor ld = at, ld_at = at;
  int left = static_cast<int>(u1 - u0);  // units not yet looked up
  int page[kWhole ? 1 : kCopies];
  bool more = false;
  const int64_t lane_off = chunk * (16 / static_cast<int>(sizeof(T))) + (kWhole ? row0 * a.p_st : 0);
  auto lookup = [&]() {  // the page ids of unit ld (used when it is copied, a unit later)
    more = left > 0;
    if (!more) return;
    ld_at = ld;
    const int n = len[ld.b], t0 = ld.tile * kTok + warp * kMine;
#pragma unroll
    for (int j = 0; j < (kWhole ? 1 : kCopies); ++j) {
      const int t = kWhole ? t0 : t0 + row0 + kRowsAt * j;
      page[j] = t < n ? a.table[ld.b * a.t_sb + page_of(t, a.page, d.page_inv)] : -1;
    }
    advance(ld);
    --left;
  };
  char *mine = ring + warp * kStages * kWarpBytes;
  uint8_t *mine_held = held + warp * kStages * 16;
  // chunks change places by row so that a warp's reads meet no bank twice
  auto place = [&](int r) { return r * kRow + ((chunk ^ (k16 ? r & 7 : (r & 1) * 4)) << 4); };
  const uint32_t ring_at = smem_u32(mine);
  auto copy = [&](int stage) {
    if (more) {
      const uint32_t dst = ring_at + stage * kWarpBytes;
      const int hk = groups == 1 ? ld_at.hh : ld_at.hh / groups;
      const int t0 = ld_at.tile * kTok + warp * kMine, n = len[ld_at.b];
      if constexpr (kWhole) {
        const bool ok = page[0] >= 0 && page[0] < a.pages;
        const int here = ok ? min(n - t0, kMine) : 0;  // rows held (lane 0 tells the readers)
        if (!ok && t0 < n) report(a.err, SD_KERR_BOUNDS);
        const int64_t off = ok ? page[0] * a.p_sp + hk * a.p_sh +
                                     (t0 - page_of(t0, a.page, d.page_inv) * a.page) * a.p_st + lane_off
                               : lane_off;
        const T *ks = static_cast<const T *>(d.k) + off, *vs = static_cast<const T *>(d.v) + off;
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const bool in = row0 + kRowsAt * j < here;
          const int64_t step = in ? kRowsAt * j * a.p_st : 0;
          cp16(dst + place(row0 + kRowsAt * j), in ? ks + step : static_cast<const T *>(d.k), in);
          cp16(dst + place(row0 + kRowsAt * j) + kWarpBytes / 2, in ? vs + step : static_cast<const T *>(d.v), in);
        }
        if (lane == 0) mine_held[stage * 16] = here > 0 ? here : 0;
      } else {
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const int r = row0 + kRowsAt * j, t = t0 + r;
          const bool ok = page[j] >= 0 && page[j] < a.pages;
          if (!ok && t < n) report(a.err, SD_KERR_BOUNDS);
          const int64_t off = ok ? page[j] * a.p_sp + hk * a.p_sh +
                                       (t - page_of(t, a.page, d.page_inv) * a.page) * a.p_st + lane_off
                                 : 0;
          cp16(dst + place(r), static_cast<const T *>(d.k) + off, ok);
          cp16(dst + place(r) + kWarpBytes / 2, static_cast<const T *>(d.v) + off, ok);
          if (chunk == 0) mine_held[stage * 16 + r] = ok;
        }
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    lookup();
    copy(s);
  }
  lookup();

  // ---- state of the current head group
  // 16-bit: fragments of m16n8k16, rows lane / 4 and lane / 4 + 8 are heads;
  // fp32: every lane keeps all heads, columns 2 lane and 2 lane + 1
  constexpr int kHalves = kWide ? 2 : 1;
  constexpr int kAcc = k16 ? 8 : kMaxHeads, kAccN = k16 ? 4 : 2, kStat = k16 ? kHalves : kMaxHeads;
  float o[kAcc][kAccN], m[kStat], l[kStat];
  uint32_t qa[4][4];
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  auto begin = [&](const Cursor &c) {
    const int h0 = (c.hh / groups) * (a.Hq / a.Hkv) + (c.hh % groups) * kMaxHeads;
    const int n = min(d.G, (a.Hq / a.Hkv) - (c.hh % groups) * kMaxHeads);
    const T *src = static_cast<const T *>(d.q) + c.b * d.q_sb + h0 * d.q_sh;
    if constexpr (k16) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int g = r0 + (e & 1) * 8, col = 16 * k + c0 + (e >> 1) * 8;
          qa[k][e] = (kWide || !(e & 1)) && g < n ? *reinterpret_cast<const uint32_t *>(src + g * d.q_sh + col) : 0u;
        }
    } else {
      __syncthreads();
      for (int e = tid; e < n * 64; e += kThreads) sq[e] = src[(e >> 6) * d.q_sh + (e & 63)];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kAcc; ++i)
#pragma unroll
      for (int e = 0; e < kAccN; ++e) o[i][e] = 0.f;
#pragma unroll
    for (int i = 0; i < kStat; ++i) m[i] = -INFINITY, l[i] = 0.f;
  };
  begin(at);
  int first_tile = at.tile;
  const float c = d.scale_log2;

  const int count = static_cast<int>(u1 - u0);
  for (int it = 0; it < count; ++it) {
    const int stage = it % kStages;
    copy((it + kStages - 1) % kStages);
    lookup();
    cp_wait<kStages - 1>();
    __syncwarp();
    const char *kt = mine + stage * kWarpBytes, *vt = kt + kWarpBytes / 2;
    const uint8_t *ok = mine_held + stage * 16;
    if constexpr (k16) {
      float s[2][4];
      const uint32_t kb = smem_u32(kt), vb = smem_u32(vt);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
        uint32_t b0, b1, b2, b3;
        const int key = 8 * nt + (lane & 7);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ldsm_x4(kb + sw128(key, 4 * half + (lane >> 3)), b0, b1, b2, b3);
          mma16816<T>(s[nt], qa[2 * half], b0, b1);
          mma16816<T>(s[nt], qa[2 * half + 1], b2, b3);
        }
      }
      if constexpr (kWhole) {
        const int here = ok[0];
        if (here < kMine) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (8 * nt + c0 + (e & 1) >= here) s[nt][e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint32_t flags = *reinterpret_cast<const uint16_t *>(ok + 8 * nt + c0);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(e & 1 ? flags >> 8 : flags & 0xff)) s[nt][e] = -INFINITY;
        }
      }
      uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int half = 0; half < kHalves; ++half) {
        float best = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        best *= c;
        if (__any_sync(0xffffffffu, best > m[half])) {  // some head's maximum rises
          const float mn = fmaxf(m[half], best), alpha = m[half] == -INFINITY ? 0.f : ex2(m[half] - mn);
          m[half] = mn;
          l[half] *= alpha;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            o[n][2 * half] *= alpha;
            o[n][2 * half + 1] *= alpha;
          }
        }
        const float neg = m[half] == -INFINITY ? 0.f : -m[half];
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ex2(fmaf(s[e >> 1][2 * half + (e & 1)], c, neg));
        l[half] += (p[0] + p[1]) + (p[2] + p[3]);
        pa[half] = pack2<T>(p[0], p[1]);
        pa[2 + half] = pack2<T>(p[2], p[3]);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(vb + sw128(lane & 15, 2 * n + (lane >> 4)), b0, b1, b2, b3);
        mma16816<T>(o[2 * n], pa, b0, b1);
        mma16816<T>(o[2 * n + 1], pa, b2, b3);
      }
    } else {
      const int key = lane >> 2, quarter = lane & 3, flip = (key & 1) * 4;
      float4 kr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kr[i] = *reinterpret_cast<const float4 *>(kt + key * kRow + (((4 * i + quarter) ^ flip) << 4));
      float2 vr[kMine];
#pragma unroll
      for (int r = 0; r < kMine; ++r)
        vr[r] = *reinterpret_cast<const float2 *>(vt + r * kRow + (((lane >> 1) ^ ((r & 1) * 4)) << 4) + (lane & 1) * 8);
      const bool seen = kWhole ? key < ok[0] : ok[key];
#pragma unroll
      for (int g = 0; g < kMaxHeads; ++g) {
        if (g >= d.G) break;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 x = *reinterpret_cast<const float4 *>(sq + g * 64 + (4 * i + quarter) * 4);
          s = fmaf(x.x, kr[i].x, fmaf(x.y, kr[i].y, fmaf(x.z, kr[i].z, fmaf(x.w, kr[i].w, s))));
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s = seen ? s * c : -INFINITY;
        float best = s;
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, w));
        const float mn = fmaxf(m[g], best), ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = ex2(m[g] - ref), p = ex2(s - ref);
        float sum = p;
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        m[g] = mn;
        l[g] = l[g] * alpha + sum;
        o[g][0] *= alpha, o[g][1] *= alpha;
#pragma unroll
        for (int r = 0; r < kMine; ++r) {
          const float w = __shfl_sync(0xffffffffu, p, 4 * r);
          o[g][0] = fmaf(w, vr[r].x, o[g][0]);
          o[g][1] = fmaf(w, vr[r].y, o[g][1]);
        }
      }
    }
    __syncwarp();
    const int tiles = pre[at.b + 1] - pre[at.b];
    const bool head_ends = at.tile + 1 == tiles;
    if (head_ends || it + 1 == count) {
      // the four warps' states of this head group meet
      float *to = merge + warp * d.G * kPart;
      if constexpr (k16) {
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
          l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
          l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
          const int g = r0 + 8 * half;
          if (g < d.G) {
            if (c0 == 0) to[g * kPart] = m[half], to[g * kPart + 1] = l[half];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              to[g * kPart + 2 + 8 * n + c0] = o[n][2 * half];
              to[g * kPart + 2 + 8 * n + c0 + 1] = o[n][2 * half + 1];
            }
          }
        }
      } else {
#pragma unroll
        for (int g = 0; g < kMaxHeads; ++g) {
          if (g >= d.G) break;
          if (lane == 0) to[g * kPart] = m[g], to[g * kPart + 1] = l[g];
          to[g * kPart + 2 + 2 * lane] = o[g][0];
          to[g * kPart + 2 + 2 * lane + 1] = o[g][1];
        }
      }
      __syncthreads();
      const bool whole = first_tile == 0 && head_ends;
      const int sub = at.hh % groups, h0 = (at.hh / groups) * (a.Hq / a.Hkv) + sub * kMaxHeads;
      const int n = min(d.G, (a.Hq / a.Hkv) - sub * kMaxHeads);
      // a part that begins with the CTA's run is its slot 0, one that begins later slot 1
      float *part = d.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (at.tile - first_tile == it ? 0 : 1)) *
                                  d.G * kPart;
      for (int g = tid >> 6; g < n; g += kThreads / 64) {
        const int e = tid & 63;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge[(w * d.G + g) * kPart]);
        float sum = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float *p = merge + (w * d.G + g) * kPart;
          const float f = factor(p[0], top);
          sum = fmaf(f, p[1], sum);
          val = fmaf(f, p[2 + e], val);
        }
        if (whole) {
          static_cast<T *>(d.out)[at.b * d.o_sb + (h0 + g) * d.o_sh + e] = from_f<T>(sum == 0.f ? 0.f : val / sum);
        } else {
          if (e == 0) part[g * kPart] = top, part[g * kPart + 1] = sum;
          part[g * kPart + 2 + e] = val;
        }
      }
      __syncthreads();
      advance(at);
      if (it + 1 < count) {
        begin(at);
        first_tile = 0;
      }
    } else {
      ++at.tile;
    }
  }
  cp_wait<0>();
}

// Joins the parts of a head that was split over CTAs, in their order, and zeros
// the rows of sequences without tokens.  One CTA per (sequence, query head):
// eight runs of the parts side by side, then the eight.
template <typename T>
__global__ void __launch_bounds__(512) paged_join_kernel(const PagedArgs a, const pg::DecodeArgs d) {
  using namespace pg;
  constexpr int kRuns = 8, kUnroll = 8;
  __shared__ float tops[kRuns], sums[kRuns], vals[kRuns][64];
  pdl_wait();
  const int b = blockIdx.y, group = a.Hq / a.Hkv, groups = d.Hh / a.Hkv, tid = threadIdx.x;
  const int h = blockIdx.x, hh = (h / group) * groups + h % group / kMaxHeads, g = h % group % kMaxHeads;
  T *out = static_cast<T *>(d.out) + b * d.o_sb + h * d.o_sh;
  const int64_t tiles = d.plan[b + 1] - d.plan[b], per = d.plan[a.B + 1];
  if (tiles == 0) {
    if (tid < 64) out[tid] = from_f<T>(0.f);
    return;
  }
  const int64_t u0 = static_cast<int64_t>(d.plan[b]) * d.Hh + hh * tiles, u1 = u0 + tiles;
  int c0, n;  // the parts' CTAs
  if (u1 <= 0x7fffffff) {
    c0 = static_cast<int>(u0) / static_cast<int>(per);
    n = static_cast<int>(u1 - 1) / static_cast<int>(per) - c0 + 1;
  } else {
    c0 = static_cast<int>(u0 / per);
    n = static_cast<int>((u1 - 1) / per) - c0 + 1;
  }
  if (n == 1) return;
  auto part = [&](int i) {
    return d.parts + ((static_cast<int64_t>(c0 + i) * 2 + ((c0 + i) * per < u0 ? 1 : 0)) * d.G + g) * kPart;
  };
  const int run = tid >> 6, e = tid & 63;
  const int i0 = n * run / kRuns, i1 = n * (run + 1) / kRuns;
  float top = -INFINITY, sum = 0.f, val = 0.f;
  for (int i = i0; i < i1; i += kUnroll) {
    float pm[kUnroll], pl[kUnroll], pv[kUnroll], best = top;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const float *p = part(i + u < i1 ? i + u : i);
      pm[u] = i + u < i1 ? p[0] : -INFINITY, pl[u] = p[1], pv[u] = p[2 + e];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) best = fmaxf(best, pm[u]);
    const float f0 = factor(top, best);
    sum *= f0, val *= f0, top = best;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const float f = factor(pm[u], best);
      sum = fmaf(f, pl[u], sum);
      val = fmaf(f, pv[u], val);
    }
  }
  if (e == 0) tops[run] = top;
  if (e == 0) sums[run] = sum;
  vals[run][e] = val;
  __syncthreads();
  if (tid < 64) {
    top = -INFINITY, sum = val = 0.f;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) top = fmaxf(top, tops[i]);
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const float f = factor(tops[i], top);
      sum = fmaf(f, sums[i], sum);
      val = fmaf(f, vals[i][e], val);
    }
    out[e] = from_f<T>(sum == 0.f ? 0.f : val / sum);
  }
}

static int check_pool(const PagedArgs &a, int dtype, int64_t D, const void *k, const void *v) {
  if (!dtype_ok(dtype) || a.B <= 0 || a.Hkv <= 0 || a.page <= 0 || a.pages <= 0 || a.width <= 0 || !a.table ||
      !a.lens || !k || !v)
    return SD_ERR_INVALID;
  if (D != 64 || a.Hkv > 65535 || static_cast<int64_t>(a.width) * a.page > 0x7fffff00ll) return SD_ERR_UNSUPPORTED;
  const int64_t size = dtype_size(dtype);
  if (!aligned16(k) || !aligned16(v) || (a.p_sp * size) % 16 || (a.p_sh * size) % 16 || (a.p_st * size) % 16)
    return SD_ERR_ALIGN;
  return SD_OK;
}

}  // namespace sd

extern "C" {

int sd_paged_append(const void *xk, const void *xv, int dtype, int64_t N, int64_t Hkv, int64_t D, int64_t k_sn,
                    int64_t k_sh, int64_t v_sn, int64_t v_sh, void *k_pages, void *v_pages, int64_t pages, int page,
                    int64_t p_sp, int64_t p_sh, int64_t p_st, const int32_t *table, int64_t t_sb, int width,
                    const int32_t *lens, int B, const int32_t *cu_seqlens, int32_t *err, void *stream) {
  using namespace sd;
  if (!xk || !xv || N <= 0 || Hkv <= 0 || Hkv > 65535 || (!cu_seqlens && N != B)) return SD_ERR_INVALID;
  PagedArgs a = {table, t_sb, width, lens, B, 0, static_cast<int>(Hkv), page, pages, p_sp, p_sh, p_st, err};
  int rc = check_pool(a, dtype, D, k_pages, v_pages);
  if (rc != SD_OK) return rc;
  const int64_t size = dtype_size(dtype);
  if (!aligned16(xk) || !aligned16(xv) || (k_sn * size) % 16 || (k_sh * size) % 16 || (v_sn * size) % 16 ||
      (v_sh * size) % 16)
    return SD_ERR_ALIGN;
  // a decode step's few rows go to more CTAs
  const bool many = N >= 32 * 148;
  const int64_t ctas = many ? (N + 31) / 32 : (N + 3) / 4;
  if (ctas > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  SD_DISPATCH_DTYPE(dtype, T, {
    auto kern = many ? paged_append_kernel<T, 32> : paged_append_kernel<T, 4>;
    kern<<<static_cast<unsigned>(ctas), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        a, cu_seqlens, N, static_cast<const T *>(xk), static_cast<const T *>(xv), k_sn, k_sh, v_sn, v_sh,
        static_cast<T *>(k_pages), static_cast<T *>(v_pages));
  });
  return check_launch();
}

int sd_paged_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t *bytes) {
  using namespace sd;
  if (!bytes || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return SD_ERR_INVALID;
  const int64_t seqs = B < pg::kMaxSeqs ? B : pg::kMaxSeqs, group = Hq / Hkv;
  const int64_t heads = group < pg::kMaxHeads ? group : pg::kMaxHeads;
  *bytes = ((seqs + 2) * 4 + 15) / 16 * 16 + static_cast<int64_t>(pg::kCtas) * 2 * heads * pg::kPart * 4;
  return SD_OK;
}

int sd_paged_decode_attention(const void *q, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t q_sb,
                              int64_t q_sh, const void *k_pages, const void *v_pages, int64_t pages, int page,
                              int64_t p_sp, int64_t p_sh, int64_t p_st, const int32_t *table, int64_t t_sb,
                              int width, const int32_t *lens, float scale, void *out, int64_t o_sb, int64_t o_sh,
                              void *workspace, int64_t workspace_bytes, int32_t *err, void *stream) {
  using namespace sd;
  if (!q || !out || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || !(scale > 0.f) || scale > 3.0e38f || !workspace)
    return SD_ERR_INVALID;
  if (B > 0x7fffffff || Hq > 65535) return SD_ERR_UNSUPPORTED;
  PagedArgs a = {table, t_sb, width, lens, static_cast<int>(B), static_cast<int>(Hq), static_cast<int>(Hkv), page,
                 pages, p_sp, p_sh, p_st, err};
  int rc = check_pool(a, dtype, D, k_pages, v_pages);
  if (rc != SD_OK) return rc;
  int64_t need = 0;
  sd_paged_decode_workspace(B, Hq, Hkv, &need);
  if (workspace_bytes < need) return SD_ERR_INVALID;
  const int64_t size = dtype_size(dtype);
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (q_sb * size) % 16 || (q_sh * size) % 16 ||
      (o_sb * size) % 16 || (o_sh * size) % 16)
    return SD_ERR_ALIGN;
  const int group = a.Hq / a.Hkv;
  pg::DecodeArgs d = {};
  d.q_sb = q_sb, d.q_sh = q_sh, d.k = k_pages, d.v = v_pages, d.o_sb = o_sb, d.o_sh = o_sh;
  d.scale_log2 = scale * 1.4426950408889634f;
  d.G = group < pg::kMaxHeads ? group : pg::kMaxHeads;
  d.Hh = a.Hkv * ((group + pg::kMaxHeads - 1) / pg::kMaxHeads);
  d.page_inv = page == 1 ? 0xffffffffu : static_cast<uint32_t>((1ull << 32) / static_cast<uint64_t>(page));
  const int64_t tokens = static_cast<int64_t>(width) * page;
  // more sequences than one launch plans: the launches follow each other on the stream
  for (int64_t b0 = 0; b0 < B; b0 += pg::kMaxSeqs) {
    a.B = static_cast<int>(B - b0 < pg::kMaxSeqs ? B - b0 : pg::kMaxSeqs);
    a.table = table + b0 * t_sb;
    a.lens = lens + b0;
    d.plan = static_cast<int32_t *>(workspace);
    d.parts = reinterpret_cast<float *>(static_cast<char *>(workspace) + ((a.B + 2) * 4 + 15) / 16 * 16);
    SD_DISPATCH_DTYPE(dtype, T, {
      d.q = static_cast<const T *>(q) + b0 * q_sb;
      d.out = static_cast<T *>(out) + b0 * o_sb;
      // the plan counts units of one head group in 32 bits
      const int64_t most = static_cast<int64_t>(a.B) * ((tokens + pg::kUnit<T> - 1) / pg::kUnit<T>);
      if (most > 0x3fffffffll) return SD_ERR_UNSUPPORTED;
      const unsigned ctas = static_cast<unsigned>(most * d.Hh < pg::kCtas ? most * d.Hh : pg::kCtas);
      const size_t smem = pg::kWarps * pg::kStages * (pg::kWarpBytes + 16) + pg::kWarps * d.G * pg::kPart * 4 +
                          (sizeof(T) == 4 ? d.G * 256 : 0) + (2 * a.B + 1) * 4;
      const bool whole = page % (pg::kUnit<T> / pg::kWarps) == 0, wide = sizeof(T) == 2 && d.G > 8;
      constexpr bool k16 = sizeof(T) == 2;  // fp32 has no wide form
      auto kern = whole ? wide ? paged_decode_kernel<T, true, k16> : paged_decode_kernel<T, true, false>
                  : wide ? paged_decode_kernel<T, false, k16>
                         : paged_decode_kernel<T, false, false>;
      if (ensure_smem(kern, smem) != SD_OK) return SD_ERR_CUDA;
      kern<<<ctas, pg::kThreads, smem, static_cast<cudaStream_t>(stream)>>>(a, d);
      rc = check_launch();
      if (rc != SD_OK) return rc;
      rc = launch(paged_join_kernel<T>, dim3(a.Hq, a.B), dim3(512), 0, static_cast<cudaStream_t>(stream), true, a, d);
      if (rc != SD_OK) return rc;
    });
  }
  return SD_OK;
}

}  // extern "C"
