// Causal grouped-query attention over packed sequences, and its gradients, on
// CUDA cores for fp32 inputs; and the entry points for all types.
//
//   O_i = sum_{j <= i} P_ij v_j,  P_ij = exp(scale q_i.k_j - lse_i)
//   delta_i = dO_i . O_i
//   dS_ij = P_ij (dO_i . v_j - delta_i)
//   dV_j = sum_i P_ij dO_i,  dK_j = scale sum_i dS_ij q_i,  dQ_i = scale sum_j dS_ij k_j
//
// i, j run over the tokens of one sequence; dK and dV also sum over the query
// heads of their key-value head.  Tiles are 64 x 64; a thread of the 128 owns
// 8 rows x 4 columns of every product, with all operands row-major in shared
// memory (row pitch 68 floats: the float4 reads below have no bank conflicts).
// A warp's 16-byte shared loads take 16 cycles of the four schedulers' 32 in each
// of the three forms (row.row, P times rows, P^T times rows); 4 x 4 a thread with
// 256 threads, 12 of 16, was up to 13 % slower where tiles are many.  No atomics:
// every sum has a fixed order.
//
// With few sequences there are few tiles, and the longest decide: so the CTAs of
// a cluster deal out a tile's other axis, and rank 0 joins their parts.
// dK/dV goes before dQ, whose CTAs are shorter and start as the first's last ones
// leave SMs free (8096 tokens: 4.35 ms one after the other, 4.06 ms with dQ first,
// 3.83 ms so).
//
// Measured, 12 query and 4 key-value heads: 1023 tokens in 3 sequences, forward
// 50 us (62 with one CTA a tile), backward 146 us (36 us for all of it at the fp32
// pipe's rate); 8096 tokens, the longest sequence 4096, forward 1.22 ms (34
// TFLOP/s), backward 3.83 ms (38): half of the 69 that the pipe reaches.  What
// bounds them: the latency of shared loads behind each barrier between a tile's
// products, with 8 warps an SM to cover it.
#include "sd_packed.cuh"

namespace sd {

namespace pk {

constexpr int kTile = 64;
constexpr int kThreads = 128;
constexpr int kR = 8;                        // rows of a thread
constexpr int kPitch = 68;
constexpr int kTileFloats = kTile * kPitch;
constexpr float kLog2e = 1.4426950408889634f;

// 64 rows (rows past `rows` zero) of 64 values from global memory into a tile,
// arriving while the caller computes (one copy group of the thread).
__device__ __forceinline__ void start_tile(float *dst, const float *src, int64_t stride, int rows) {
  for (int e = threadIdx.x; e < kTile * 16; e += kThreads) {
    const int r = e >> 4, c = (e & 15) * 4;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * kPitch + c)),
                 "l"(r < rows ? src + r * stride + c : src), "r"(r < rows ? 16 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void start_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest n groups have arrived, for every thread.
template <int n> __device__ __forceinline__ void arrived() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
  __syncthreads();
}

// The rows of a thread: fours, 32 apart, so that the two that a warp reads at a
// time lie in different banks.
__device__ __forceinline__ int row_of(int ty, int i) { return 4 * ty + (i & 3) + 8 * (i & ~3); }

__device__ __forceinline__ float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float dot4(float4 a, float4 b, float c) {
  return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, c))));
}
// Two multiply-adds in one instruction (the same 128 a cycle and SM, in half the
// issue slots, which the shared loads need): {x, y} += {a, b} * {c, d}.
__device__ __forceinline__ void fma2(float &x, float &y, float a, float b, float c, float d) {
  asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(c), "f"(d));
}

// c[i][j] = sum_d A[row i][d] B[tx + 16 j][d], even and odd d apart
__device__ __forceinline__ void mul_rows(const float *A, const float *B, int ty, int tx, float (&c)[kR][4]) {
  float even[kR][4], odd[kR][4];
#pragma unroll
  for (int i = 0; i < kR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) even[i][j] = odd[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < kTile; d += 4) {
    float4 b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = ld4(B + (tx + 16 * j) * kPitch + d);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const float4 a = ld4(A + row_of(ty, i) * kPitch + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fma2(even[i][j], odd[i][j], a.x, a.y, b[j].x, b[j].y);
        fma2(even[i][j], odd[i][j], a.z, a.w, b[j].z, b[j].w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kR; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = even[i][j] + odd[i][j];
}

// c[i][u] += w b[u]
__device__ __forceinline__ void add_row(float (&c)[4], float w, float4 b) {
  fma2(c[0], c[1], w, w, b.x, b.y);
  fma2(c[2], c[3], w, w, b.z, b.w);
}

// c[i][u] += sum_k P[row i][k] B[k][4 tx + u]
__device__ __forceinline__ void mul_p(const float *P, const float *B, int ty, int tx, float (&c)[kR][4]) {
#pragma unroll 4
  for (int k = 0; k < kTile; k += 4) {
    float4 b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = ld4(B + (k + e) * kPitch + 4 * tx);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const float4 p = ld4(P + row_of(ty, i) * kPitch + k);
      add_row(c[i], p.x, b[0]);
      add_row(c[i], p.y, b[1]);
      add_row(c[i], p.z, b[2]);
      add_row(c[i], p.w, b[3]);
    }
  }
}

// c[i][u] += sum_k P[k][row i] B[k][4 tx + u]
__device__ __forceinline__ void mul_pt(const float *P, const float *B, int ty, int tx, float (&c)[kR][4]) {
#pragma unroll 4
  for (int k = 0; k < kTile; ++k) {
    const float4 b = ld4(B + k * kPitch + 4 * tx);
#pragma unroll
    for (int i = 0; i < kR; i += 4) {
      const float4 p = ld4(P + k * kPitch + row_of(ty, i));
      add_row(c[i], p.x, b);
      add_row(c[i + 1], p.y, b);
      add_row(c[i + 2], p.z, b);
      add_row(c[i + 3], p.w, b);
    }
  }
}

__device__ __forceinline__ void store4(float *dst, float a, float b, float c, float d) {
  *reinterpret_cast<float4 *>(dst) = make_float4(a, b, c, d);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four values at p's place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float4 peer4(const float *p, int rank) {
  uint32_t addr;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Sums of a tile that a cluster shares: the other ranks put theirs into their
// own shared memory, rank 0 adds them in their order.
__device__ __forceinline__ void put(float *P, const float (&c)[kR][4], int ty, int tx) {
#pragma unroll
  for (int i = 0; i < kR; ++i) store4(P + row_of(ty, i) * kPitch + 4 * tx, c[i][0], c[i][1], c[i][2], c[i][3]);
}
__device__ __forceinline__ void add_peer(const float *P, int rank, float (&c)[kR][4], int ty, int tx) {
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const float4 x = peer4(P + row_of(ty, i) * kPitch + 4 * tx, rank);
    c[i][0] += x.x, c[i][1] += x.y, c[i][2] += x.z, c[i][3] += x.w;
  }
}

// CTAs that share a tile: as many as make `ctas` in all, so that the longest rows
// of tiles do not outlast the rest, but no more than twice the tiles of an average
// sequence, which would find nothing to do.  Two CTAs fit an SM.  12 query
// and 4 key-value heads, for 2, 3, 4 and 6 times 148: one sequence of 2048 tokens,
// forward 277, 226, 227 us, dQ 408, 363, 350 us, dK/dV (from 3) 474, 440, 439 us;
// 1023 tokens in 3 sequences, forward 58, 57, 64 us, dQ 80, 79, 90 us.
static int cluster_ranks(const PackedArgs &a, int64_t slots, int heads, int ctas) {
  const int64_t most = 2 * ((a.total + kTile * int64_t(a.S) - 1) / (kTile * int64_t(a.S > 0 ? a.S : 1)));
  int ranks = 1;
  while (ranks < 8 && 2 * ranks <= most && slots * heads * ranks < ctas) ranks *= 2;
  return ranks;
}

// The 16 lanes of a row (tx = 0..15).
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace pk

__global__ void __launch_bounds__(pk::kThreads, 2) packed_fwd_kernel(const __grid_constant__ PackedArgs a, int ranks) {
  using namespace pk;
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *K = Q + kTileFloats, *V = K + kTileFloats, *P = V + kTileFloats;
  // the tiles that see the most keys start first
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x, gridDim.x, kTile, true);
  if (!t.valid) return;
  const int h = blockIdx.y / ranks, rank = blockIdx.y % ranks, hk = h / (a.Hq / a.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int rows = min(kTile, t.len - t.row0);
  const int64_t first = t.start + t.row0;
  float *out = static_cast<float *>(a.out) + first * a.o_st + h * a.o_sh;
  if (t.rest) {
    if (a.zero_rest && rank == 0)
      for (int i = 0; i < kR; ++i)
        if (row_of(ty, i) < rows) store4(out + row_of(ty, i) * a.o_st + 4 * tx, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const float *kp = static_cast<const float *>(a.k) + t.start * a.k_st + hk * a.k_sh;
  const float *vp = static_cast<const float *>(a.v) + t.start * a.v_st + hk * a.v_sh;
  start_tile(Q, static_cast<const float *>(a.q) + first * a.q_st + h * a.q_sh, a.q_st, rows);
  auto start = [&](float *dst, const float *src, int64_t st, int k0) {
    if (k0 <= t.row0) start_tile(dst, src + k0 * st, st, min(kTile, t.len - k0));
    start_group();
  };
  start(K, kp, a.k_st, rank * kTile);
  start(V, vp, a.v_st, rank * kTile);
  float o[kR][4] = {}, m[kR], l[kR];
#pragma unroll
  for (int i = 0; i < kR; ++i) m[i] = -INFINITY, l[i] = 0.f;
  for (int k0 = rank * kTile; k0 <= t.row0; k0 += ranks * kTile) {
    // a tile's successor comes in as soon as its last product is done
    const int next = k0 + ranks * kTile;
    float s[kR][4];
    arrived<1>();
    mul_rows(Q, K, ty, tx, s);
    __syncthreads();
    start(K, kp, a.k_st, next);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int row = t.row0 + row_of(ty, i);
      float best = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = k0 + tx + 16 * j <= row ? s[i][j] * a.scale_log2 : -INFINITY;
        best = fmaxf(best, s[i][j]);
      }
      const float mn = fmaxf(m[i], row_max(best));
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m[i] - ref);
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - ref);
        P[row_of(ty, i) * kPitch + tx + 16 * j] = p;
        ps += p;
      }
      l[i] = l[i] * alpha + row_sum(ps);
      m[i] = mn;
#pragma unroll
      for (int u = 0; u < 4; ++u) o[i][u] *= alpha;
    }
    arrived<1>();
    mul_p(P, V, ty, tx, o);
    __syncthreads();
    start(V, vp, a.v_st, next);
  }
  if (ranks > 1) {  // the ranks' parts, in their order; maximum and sum beside the 64 columns
    __syncthreads();
    if (rank > 0) {
      put(P, o, ty, tx);
      if (tx == 0) {
#pragma unroll
        for (int i = 0; i < kR; ++i) P[row_of(ty, i) * kPitch + 64] = m[i], P[row_of(ty, i) * kPitch + 65] = l[i];
      }
    }
    cluster_sync();
    if (rank == 0) {
      for (int c = 1; c < ranks; ++c)
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const float *row = P + row_of(ty, i) * kPitch;
          const float4 ml = peer4(row + 64, c), x = peer4(row + 4 * tx, c);
          const float mn = fmaxf(m[i], ml.x), ref = mn == -INFINITY ? 0.f : mn;
          const float f0 = exp2f(m[i] - ref), f1 = exp2f(ml.x - ref);
          m[i] = mn;
          l[i] = l[i] * f0 + ml.y * f1;
          o[i][0] = o[i][0] * f0 + x.x * f1, o[i][1] = o[i][1] * f0 + x.y * f1;
          o[i][2] = o[i][2] * f0 + x.z * f1, o[i][3] = o[i][3] * f0 + x.w * f1;
        }
    }
    cluster_sync();
    if (rank > 0) return;
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const float inv = 1.0f / l[i];
    bool finite = true;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      o[i][u] *= inv;
      finite = finite && fabsf(o[i][u]) < INFINITY;
    }
    const bool held = row_of(ty, i) < rows;
    if (held) {
      store4(out + row_of(ty, i) * a.o_st + 4 * tx, o[i][0], o[i][1], o[i][2], o[i][3]);
      if (a.lse && tx == 0) a.lse[h * a.total + first + row_of(ty, i)] = m[i] + log2f(l[i]);
    }
    // the warp's two rows, where one is not finite
    const unsigned bad = __ballot_sync(0xffffffffu, held && !finite);
    if (bad) {
      __syncwarp();
      PackedRows<2> g;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = __shfl_sync(0xffffffffu, t.row0 + row_of(ty, i), 16 * half);
        g.row[half] = bad >> (16 * half) & 0xffffu ? row : -1;
        g.m[half] = __shfl_sync(0xffffffffu, m[i], 16 * half), g.l[half] = __shfl_sync(0xffffffffu, l[i], 16 * half);
      }
      packed_again<float>(a, t.start, min(t.len, t.row0 + kTile), h, g);
    }
  }
}

// delta, 16 lanes a row.  A kernel of its own, so that both gradients' kernels can
// read it and the second may start while the first ends.
__global__ void __launch_bounds__(256) packed_delta_kernel(const PackedArgs a) {
  using namespace pk;
  const int64_t n = blockIdx.x * 16ll + (threadIdx.x >> 4);  // row x head
  const int64_t row = n / a.Hq;
  const int h = static_cast<int>(n - row * a.Hq), c = 4 * (threadIdx.x & 15);
  float d = 0.f;
  if (row < a.total)
    d = dot4(ld4(static_cast<const float *>(a.out) + row * a.o_st + h * a.o_sh + c),
             ld4(static_cast<const float *>(a.dout) + row * a.g_st + h * a.g_sh + c), 0.f);
  d = row_sum(d);
  if (row < a.total && c == 0) a.delta[h * a.total + row] = d;
}

// dQ of a query tile, its key tiles dealt out to the CTAs of a cluster.
__global__ void __launch_bounds__(pk::kThreads, 2) packed_bwd_dq_kernel(PackedArgs a, int ranks) {
  using namespace pk;
  // Starts while dK/dV's last CTAs run, of which it reads nothing; what follows on
  // the stream follows both, as one CTA here ends after all of theirs.
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) pdl_wait();
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *G = Q + kTileFloats, *K = G + kTileFloats, *V = K + kTileFloats, *P = V + kTileFloats;
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x, gridDim.x, kTile, true);
  if (!t.valid) return;
  const int h = blockIdx.y / ranks, rank = blockIdx.y % ranks, hk = h / (a.Hq / a.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int rows = min(kTile, t.len - t.row0);
  const int64_t first = t.start + t.row0;
  const int64_t c_st = static_cast<int64_t>(a.Hq) * kTile;  // dq is contiguous
  float *dq = static_cast<float *>(a.dq) + first * c_st + h * kTile;
  if (t.rest) {
    for (int i = 0; i < kR && rank == 0; ++i)
      if (row_of(ty, i) < rows) store4(dq + row_of(ty, i) * c_st + 4 * tx, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  float delta[kR], lse[kR];
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    const int r = row_of(ty, i);
    delta[i] = r < rows ? a.delta[h * a.total + first + r] : 0.f;
    lse[i] = r < rows ? a.lse[h * a.total + first + r] : 0.f;
  }
  const float *kp = static_cast<const float *>(a.k) + t.start * a.k_st + hk * a.k_sh;
  const float *vp = static_cast<const float *>(a.v) + t.start * a.v_st + hk * a.v_sh;
  auto start = [&](float *dst, const float *src, int64_t st, int k0) {
    if (k0 <= t.row0) start_tile(dst, src + k0 * st, st, min(kTile, t.len - k0));
    start_group();
  };
  start_tile(G, static_cast<const float *>(a.dout) + first * a.g_st + h * a.g_sh, a.g_st, rows);
  start_tile(Q, static_cast<const float *>(a.q) + first * a.q_st + h * a.q_sh, a.q_st, rows);
  start(V, vp, a.v_st, rank * kTile);
  start(K, kp, a.k_st, rank * kTile);
  float acc[kR][4] = {};
  for (int k0 = rank * kTile; k0 <= t.row0; k0 += ranks * kTile) {
    float s[kR][4], dp[kR][4];
    arrived<1>();
    mul_rows(G, V, ty, tx, dp);
    __syncthreads();
    start(V, vp, a.v_st, k0 + ranks * kTile);
    arrived<1>();
    mul_rows(Q, K, ty, tx, s);
#pragma unroll
    for (int i = 0; i < kR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool seen = k0 + tx + 16 * j <= t.row0 + row_of(ty, i);
        const float p = exp2f(s[i][j] * a.scale_log2 - lse[i]);
        P[row_of(ty, i) * kPitch + tx + 16 * j] = seen ? p * (dp[i][j] - delta[i]) : 0.f;
      }
    __syncwarp();  // a warp reads only the rows of P that it wrote
    mul_p(P, K, ty, tx, acc);
    __syncthreads();
    start(K, kp, a.k_st, k0 + ranks * kTile);
  }
  if (ranks > 1) {
    __syncthreads();
    if (rank > 0) put(P, acc, ty, tx);
    cluster_sync();
    if (rank == 0)
      for (int c = 1; c < ranks; ++c) add_peer(P, c, acc, ty, tx);
    cluster_sync();
    if (rank > 0) return;
  }
#pragma unroll
  for (int i = 0; i < kR; ++i)
    if (row_of(ty, i) < rows)
      store4(dq + row_of(ty, i) * c_st + 4 * tx, acc[i][0] * a.scale, acc[i][1] * a.scale, acc[i][2] * a.scale,
             acc[i][3] * a.scale);
}

// dK and dV of a key tile: every query tile at or behind it, of every query
// head of the key-value head.  These are dealt out in turn to the CTAs of a
// cluster (blockIdx.y = kv head x ranks + rank): a short batch has few key
// tiles, and the first of a sequence has them all.
__global__ void __launch_bounds__(pk::kThreads, 2) packed_bwd_dkv_kernel(PackedArgs a, int ranks) {
  using namespace pk;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // dQ's CTAs take the SMs that this one's leave
  extern __shared__ __align__(16) float sm[];
  float *K = sm, *V = K + kTileFloats, *Q = V + kTileFloats, *G = Q + kTileFloats, *P = G + kTileFloats,
        *D = P + kTileFloats;
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x, gridDim.x, kTile, false);
  if (!t.valid) return;  // the cluster's CTAs share the tile: all return
  const int hk = blockIdx.y / ranks, rank = blockIdx.y % ranks, group = a.Hq / a.Hkv;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int keys = min(kTile, t.len - t.row0);
  const int64_t first = t.start + t.row0;
  const int64_t c_st = static_cast<int64_t>(a.Hkv) * kTile;
  float *dk = static_cast<float *>(a.dk) + first * c_st + hk * kTile;
  float *dv = static_cast<float *>(a.dv) + first * c_st + hk * kTile;
  float sk[kR][4] = {}, sv[kR][4] = {};
  if (!t.rest) {
    const int per_head = (t.len - t.row0 + kTile - 1) / kTile, items = per_head * group;
    auto start = [&](float *dst, const void *src, int64_t st, int64_t sh, int item) {
      if (item < items) {
        const int q0 = t.row0 + item % per_head * kTile;
        start_tile(dst, static_cast<const float *>(src) + (t.start + q0) * st + (hk * group + item / per_head) * sh, st,
                   min(kTile, t.len - q0));
      }
      start_group();
    };
    start_tile(K, static_cast<const float *>(a.k) + first * a.k_st + hk * a.k_sh, a.k_st, keys);
    start_tile(V, static_cast<const float *>(a.v) + first * a.v_st + hk * a.v_sh, a.v_st, keys);
    start(G, a.dout, a.g_st, a.g_sh, rank);
    start(Q, a.q, a.q_st, a.q_sh, rank);
    for (int item = rank; item < items; item += ranks) {
      const int h = hk * group + item / per_head, q0 = t.row0 + item % per_head * kTile;
      {
        const int rows = min(kTile, t.len - q0);
        const int64_t at = t.start + q0;
        float s[kR][4], dp[kR][4];
        arrived<1>();
        mul_rows(G, V, ty, tx, dp);
        arrived<0>();
        mul_rows(Q, K, ty, tx, s);
#pragma unroll
        for (int i = 0; i < kR; ++i) {
          const int r = row_of(ty, i);
          float lse = 0.f, delta = 0.f;
          if (r < rows) {
            lse = a.lse[h * a.total + at + r];
            delta = a.delta[h * a.total + at + r];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool seen = r < rows && t.row0 + tx + 16 * j <= q0 + r;
            const float p = seen ? exp2f(s[i][j] * a.scale_log2 - lse) : 0.f;
            P[r * kPitch + tx + 16 * j] = p;
            D[r * kPitch + tx + 16 * j] = seen ? p * (dp[i][j] - delta) : 0.f;
          }
        }
        __syncthreads();
        mul_pt(P, G, ty, tx, sv);
        __syncthreads();
        start(G, a.dout, a.g_st, a.g_sh, item + ranks);
        mul_pt(D, Q, ty, tx, sk);
        __syncthreads();
        start(Q, a.q, a.q_st, a.q_sh, item + ranks);
      }
    }
  }
  if (ranks > 1) {
    __syncthreads();  // all have read P and D
    if (rank > 0) put(P, sk, ty, tx), put(D, sv, ty, tx);
    cluster_sync();
    if (rank == 0)
      for (int c = 1; c < ranks; ++c) add_peer(P, c, sk, ty, tx), add_peer(D, c, sv, ty, tx);
    cluster_sync();  // the others' shared memory stays until it is read
    if (rank > 0) return;
  }
#pragma unroll
  for (int i = 0; i < kR; ++i)
    if (row_of(ty, i) < keys) {
      store4(dk + row_of(ty, i) * c_st + 4 * tx, sk[i][0] * a.scale, sk[i][1] * a.scale, sk[i][2] * a.scale,
             sk[i][3] * a.scale);
      store4(dv + row_of(ty, i) * c_st + 4 * tx, sv[i][0], sv[i][1], sv[i][2], sv[i][3]);
    }
}

// Shapes, strides (multiples of 16 bytes) and pointers of one packed tensor.
static int check_rows(const void *p, int dtype, int64_t st, int64_t sh) {
  if (!p) return SD_ERR_INVALID;
  const int64_t size = dtype_size(dtype);
  if (!aligned16(p) || (st * size) % 16 || (sh * size) % 16) return SD_ERR_ALIGN;
  return SD_OK;
}

static int check_packed(const PackedArgs &a, int dtype, int64_t D) {
  if (!dtype_ok(dtype) || a.total <= 0 || a.S < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || !a.cu || !a.out ||
      !(a.scale > 0.f) || a.scale > 3.0e38f)
    return SD_ERR_INVALID;
  if (D != 64 || a.Hq > 8191 || a.total > 0x7fffff00ll || a.S > (1 << 24)) return SD_ERR_UNSUPPORTED;
  int rc = check_rows(a.q, dtype, a.q_st, a.q_sh);
  if (rc == SD_OK) rc = check_rows(a.k, dtype, a.k_st, a.k_sh);
  if (rc == SD_OK) rc = check_rows(a.v, dtype, a.v_st, a.v_sh);
  if (rc == SD_OK) rc = check_rows(a.out, dtype, a.o_st, a.o_sh);
  return rc;
}

}  // namespace sd

extern "C" {

int sd_packed_attention(const void *q, const void *k, const void *v, int dtype, int64_t total, int64_t Hq,
                        int64_t Hkv, int64_t D, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st,
                        int64_t v_sh, const int32_t *cu_seqlens, int nseq, float scale, void *out, int64_t o_st,
                        int64_t o_sh, float *lse, void *rest, int zero_rest, int32_t *err, void *stream) {
  using namespace sd;
  PackedArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  a.cu = cu_seqlens, a.S = nseq, a.total = total;
  if (Hq > 65535 || Hkv > 65535) return SD_ERR_UNSUPPORTED;
  a.Hq = static_cast<int>(Hq), a.Hkv = static_cast<int>(Hkv);
  a.scale = scale, a.scale_log2 = scale * pk::kLog2e;
  a.out = out, a.o_st = o_st, a.o_sh = o_sh;
  a.lse = lse, a.rest = rest, a.zero_rest = zero_rest;
  int rc = check_packed(a, dtype, D);
  if (rc != SD_OK) return rc;
  if (rest && dtype == SD_DTYPE_F32) return SD_ERR_INVALID;
  if (!aligned16(rest)) return SD_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype != SD_DTYPE_F32) return launch_packed_fwd_tc(a, dtype, err, s);
  const size_t smem = 4 * pk::kTileFloats * sizeof(float);
  if (ensure_smem(packed_fwd_kernel, smem) != SD_OK) return SD_ERR_CUDA;
  const unsigned slots = static_cast<unsigned>(packed_slots(total, nseq, pk::kTile));
  const int ranks = pk::cluster_ranks(a, slots, a.Hq, 3 * 148);
  return launch_cluster(packed_fwd_kernel, dim3(slots, a.Hq * ranks), dim3(pk::kThreads), dim3(1, ranks, 1), smem, s,
                        false, a, ranks);
}

int sd_packed_attention_backward(const void *q, const void *k, const void *v, const void *out, const void *dout,
                                 int dtype, int64_t total, int64_t Hq, int64_t Hkv, int64_t D, int64_t q_st,
                                 int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t o_st,
                                 int64_t o_sh, int64_t g_st, int64_t g_sh, const int32_t *cu_seqlens, int nseq,
                                 float scale, const float *lse, const void *rest, float *delta, void *dq, void *dk,
                                 void *dv, int32_t *err, void *stream) {
  using namespace sd;
  PackedArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
  a.cu = cu_seqlens, a.S = nseq, a.total = total;
  if (Hq > 65535 || Hkv > 65535) return SD_ERR_UNSUPPORTED;
  a.Hq = static_cast<int>(Hq), a.Hkv = static_cast<int>(Hkv);
  a.scale = scale, a.scale_log2 = scale * pk::kLog2e;
  a.out = const_cast<void *>(out), a.o_st = o_st, a.o_sh = o_sh;
  a.lse = const_cast<float *>(lse), a.rest = const_cast<void *>(rest), a.delta = delta;
  a.dout = dout, a.g_st = g_st, a.g_sh = g_sh;
  a.dq = dq, a.dk = dk, a.dv = dv;
  int rc = check_packed(a, dtype, D);
  if (rc == SD_OK) rc = check_rows(dout, dtype, g_st, g_sh);
  if (rc != SD_OK) return rc;
  if (!lse || !delta || !dq || !dk || !dv || (rest && dtype == SD_DTYPE_F32)) return SD_ERR_INVALID;
  if (!aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !aligned16(rest)) return SD_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype != SD_DTYPE_F32) return launch_packed_bwd_tc(a, dtype, err, s);
  const unsigned slots = static_cast<unsigned>(packed_slots(total, nseq, pk::kTile));
  const size_t smem_q = 5 * pk::kTileFloats * sizeof(float), smem_kv = 6 * pk::kTileFloats * sizeof(float);
  auto kq = packed_bwd_dq_kernel;
  auto kkv = packed_bwd_dkv_kernel;
  if (ensure_smem(kq, smem_q) != SD_OK || ensure_smem(kkv, smem_kv) != SD_OK) return SD_ERR_CUDA;
  const int64_t delta_ctas = (total * a.Hq + 15) / 16;
  if (delta_ctas > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  packed_delta_kernel<<<static_cast<unsigned>(delta_ctas), 256, 0, s>>>(a);
  rc = check_launch();
  if (rc != SD_OK) return rc;
  int ranks = pk::cluster_ranks(a, slots, a.Hkv, 4 * 148);
  rc = launch_cluster(kkv, dim3(slots, a.Hkv * ranks), dim3(pk::kThreads), dim3(1, ranks, 1), smem_kv, s, false, a,
                      ranks);
  if (rc != SD_OK) return rc;
  ranks = pk::cluster_ranks(a, slots, a.Hq, 3 * 148);
  return launch_cluster(kq, dim3(slots, a.Hq * ranks), dim3(pk::kThreads), dim3(1, ranks, 1), smem_q, s, true, a, ranks);
}

}  // extern "C"
