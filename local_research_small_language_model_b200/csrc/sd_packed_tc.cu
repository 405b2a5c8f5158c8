// Causal attention over packed sequences on the 5th-generation tensor cores,
// 16-bit inputs.
//
//   O_i = sum_{j <= i} exp2(c q_i.k_j - m_i) v_j / l_i,  c = scale log2(e)
//
// Forward.  One CTA per 256 query rows of one sequence and head, two per SM.
// The rows are two 128-row tiles; for every 64 keys up to a tile's own diagonal
//   S_x = Q_x K^T    4 MMAs M=128 N=64 K=16, fp32 in 64 columns
//   P_x = exp2(..)   warpgroup x, one thread a row, 16-bit pairs written over
//                    the first 32 columns of S_x
//   O_x += P_x V     4 MMAs, A from tensor memory
// Warp 8 issues all MMAs, warp 9 all copies (K and V in a ring of 4 stages).
// The four tiles of an SM take turns: while one's products run, the others
// compute exponentials (64 a row and block: at 16 a cycle and SM 512 cycles, 384
// with the quarter of them that is computed elsewhere; the products need 320).
// S_x(i + 1) is issued right behind O_x(i), so its arrival also says that O_x(i)
// is done.
// A row's reference m is its first block's maximum, and stays while a block's
// weights sum to at most 2^14 (16-bit weights and fp32 sums have the same
// relative precision there), so the common path looks for no maximum: the sum,
// needed anyway, tells.  Otherwise m moves to the block's maximum, the weights
// are computed again, and O is rescaled.
//
// Backward, two kernels of one shape: a CTA owns 128 rows, the A operands of its
// products, and walks 128-row blocks of the other side, which serve as B both
// ways.
//   dQ:    rows are queries (A: Q, dO), blocks are keys (B: K, V)
//          S = Q K^T, dP = dO V^T;  dS = P (dP - delta);  dQ += dS K
//   dK/dV: rows are keys (A: K, V), blocks are queries of every head of the
//          group (B: Q, dO)
//          S' = K Q^T, dP' = V dO^T;  dV += P' dO,  dK += dS' Q
// Sixteen warps compute, 32 rows x 32 columns each.  They read a block's S and dP
// into registers at once, which frees the columns for the next block's products,
// and write their 16-bit weights to columns of their own: products, exponentials
// and accumulation of neighbouring blocks run side by side.
// S and dP are computed in both (7 products and 2 exponentials a pair instead
// of 5 and 1): in return every gradient is summed in tensor memory in a fixed
// order, with no atomics and no fp32 buffer to add into and convert.
// P and dS are rounded to 16 bits, as P is in the forward: the products that take
// them have 16-bit operands, and splitting them in two would double four products.
// A small kernel ahead of them computes delta, so that neither needs the other:
// dK/dV, whose CTAs are longer, goes first, and dQ's CTAs take the SMs that its
// last ones leave (one after the other: 457 instead of 416 us at 8192 tokens, 100
// instead of 78 at 2048).
//
// Measured, 12 query and 4 key-value heads, bf16.  One sequence of 32768 tokens:
// forward 1.74 ms as the best of five runs of ten (945 TFLOP/s), 2.0 ms called for
// longer, under the power cap (820); 1.00 ms of products, 1.07 ms of exponentials
// on the special-function units (1.43 if all were there).  Backward 5.9 ms (700
// TFLOP/s of the 5 products a gradient needs, 985 of the 7 it computes).  Training
// on 16000 tokens in 9 sequences: 0.40 to 0.45 ms, forward and backward (f16 0.46).
// Of a sequence's cycles the forward keeps the special-function units, instruction
// issue and the tensor pipe busy for 67, 65 and 44 % at 32768 tokens, 57, 57 and
// 36 % at 8192, 31, 34 and 18 % at 2048: no unit is its bound, but the chain of a
// block's steps, and in short batches the longest tiles.  dQ at 8192: 44, 55 and
// 43 %, dK/dV 38, 62 and 50 %: issue, and its warps' waits for one another between
// the phases of a block.  f16's look at the other side's rows costs a tenth of its
// backward there (435 us; 362 in bf16).  The forward spills 32 bytes a thread.
#include <type_traits>

#include "sd_packed.cuh"
#include "sd_tc.cuh"
#include "sd_tma.cuh"

namespace sd {

namespace pt {

using namespace tc;

constexpr int kRows = 128;                   // MMA M
constexpr int kBlock = 64;                   // rows of a block of the other side
constexpr int kBlockBytes = kBlock * 128;    // of 64 16-bit values
constexpr int kStages = 4;
constexpr int kFwdThreads = 320;             // 2 softmax warpgroups, MMA warp, copy warp
constexpr int kFwdCols = 256, kFwdO = 128;   // tensor-memory columns: S of tile x from 64 x, O_x from 128 + 64 x
constexpr int kTileBytes = kRows * 128;

constexpr float kMostSum = 16384.f;          // of a block's weights against a row's reference

struct FwdBars {
  uint64_t q_full, full[kStages], empty[kStages], s_full[2], p_full[2], o_full[2];
  uint32_t tmem;
};

struct FwdSmem {
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kBlockBytes;
  static constexpr int kBar = kV + kStages * kBlockBytes;
  static constexpr int kBytes = kBar + 256;
};

// 32 consecutive columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ void fma2(float &a, float &b, float c, float d) {  // {a, b} = {a, b} * c + d
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmov.b64 z, {%3, %3};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ void add2(float &a, float &b, float c, float d) {  // {a, b} += {c, d}
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}

__device__ __forceinline__ void fma2v(float &a, float &b, float c, float d, float e) {  // {a, b} = {a, b} * c + {d, e}
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmov.b64 z, {%3, %4};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d), "f"(e));
}
__device__ __forceinline__ void mul2(float &a, float &b, float c, float d) {  // {a, b} *= {c, d}
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}

// 2^a and 2^b on the FMA pipe, to 2^-22, for a, b <= 127; with kUpper 2^127 for
// what is above and for a NaN.  n = round(x) by adding 1.5 2^23, f = x - n in [-1/2, 1/2], 2^f by its
// degree-5 polynomial of least relative error (fitted for this use), n added to
// the exponent.  Below -126: at most 2^-126.
template <bool kUpper> __device__ __forceinline__ void exp2_fma(float &a, float &b) {
  a = fmaxf(kUpper ? fminf(a, 127.f) : a, -126.f);
  b = fmaxf(kUpper ? fminf(b, 127.f) : b, -126.f);
  asm("{\n\t.reg .b64 x, t, n, f, p, c;\n\t.reg .b32 t0, t1, p0, p1;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b32 t0, 0f4B400000;\n\tmov.b64 c, {t0, t0};\n\tadd.rn.f32x2 t, x, c;\n\t"
      "mov.b32 t1, 0fCB400000;\n\tmov.b64 c, {t1, t1};\n\tadd.rn.f32x2 n, t, c;\n\t"
      "mov.b32 t1, 0fBF800000;\n\tmov.b64 c, {t1, t1};\n\tfma.rn.f32x2 f, n, c, x;\n\t"
      "mov.b64 p, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\tfma.rn.f32x2 p, p, f, c;\n\t"
      "mov.b64 c, {%4, %4};\n\tfma.rn.f32x2 p, p, f, c;\n\t"
      "mov.b64 c, {%5, %5};\n\tfma.rn.f32x2 p, p, f, c;\n\t"
      "mov.b64 c, {%6, %6};\n\tfma.rn.f32x2 p, p, f, c;\n\t"
      "mov.b64 c, {%7, %7};\n\tfma.rn.f32x2 p, p, f, c;\n\t"
      "mov.b64 {t0, t1}, t;\n\tmov.b64 {p0, p1}, p;\n\t"
      "shl.b32 t0, t0, 23;\n\tshl.b32 t1, t1, 23;\n\t"
      "add.u32 p0, p0, t0;\n\tadd.u32 p1, p1, t1;\n\tmov.b32 %0, p0;\n\tmov.b32 %1, p1;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(0.001327647129073739f), "f"(0.009675540961325169f), "f"(0.05550713092088699f), "f"(0.24022120237350464f),
        "f"(0.6931469440460205f), "f"(1.0000001192092896f));
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Zeros the rows from `first` on of a tile in shared memory (a warp): the rows
// behind a sequence's end belong to others, and a masked weight of 0 times
// their NaN or infinity would show.
__device__ __forceinline__ void clear_rows(char *tile, int first, int rows) {
  const int lane = threadIdx.x & 31;
  for (int e = first * 8 + lane; e < rows * 8; e += 32)
    *reinterpret_cast<uint4 *>(tile + e * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  __syncwarp();
}

// A warp's 32 accumulator rows of 64 values, scaled, to 16-bit rows `stride`
// apart, the first `rows` of them; with `rest` also what the rounding took from
// them.  Through 4 KB of the warp's own shared memory, so that eight lanes write
// a row's 128 bytes together.  Returns the lanes whose row holds a value that is
// not finite.
template <typename T>
__device__ __forceinline__ unsigned store_rows(T *dst, int64_t stride, int rows, uint32_t taddr, float scale, char *sm,
                                           T *rest = nullptr, int64_t rest_stride = 0) {
  const int lane = threadIdx.x & 31;
  bool finite = true;
#pragma unroll 1
  for (int pass = 0; pass < (rest == nullptr ? 1 : 2); ++pass) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[32];
      tmem_ld32(taddr + 32 * h, v);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 32; c += 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[c + e] *= scale;
          finite = finite && fabsf(v[c + e]) < INFINITY;
          if (pass == 1) v[c + e] -= round_to<T>(v[c + e]);
        }
        *reinterpret_cast<uint4 *>(sm + sw128(lane, 4 * h + (c >> 3))) = make_uint4(
            pack2<T>(v[c], v[c + 1]), pack2<T>(v[c + 2], v[c + 3]), pack2<T>(v[c + 4], v[c + 5]),
            pack2<T>(v[c + 6], v[c + 7]));
      }
    }
    __syncwarp();
    T *to = pass == 0 ? dst : rest;
    const int64_t st = pass == 0 ? stride : rest_stride;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3), c = lane & 7;
      if (r < rows) *reinterpret_cast<uint4 *>(to + r * st + 8 * c) = *reinterpret_cast<const uint4 *>(sm + sw128(r, c));
    }
  }
  return __ballot_sync(0xffffffffu, !finite && lane < rows);
}

// A value that the warp's lanes share, in a form the compiler knows to be shared:
// descriptors and columns derived from it stay in uniform registers, where MMAs
// take them from.
template <typename V> __device__ __forceinline__ V shared_value(V v) { return __shfl_sync(0xffffffffu, v, 0); }

template <typename T> __device__ __forceinline__ void zero_rows(T *dst, int64_t stride, int rows) {
  for (int e = threadIdx.x; e < rows * 8; e += blockDim.x)
    *reinterpret_cast<uint4 *>(dst + (e >> 3) * stride + (e & 7) * 8) = make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace pt

template <typename T>
__global__ void __launch_bounds__(pt::kFwdThreads, 2)
    packed_fwd_tc_kernel(const __grid_constant__ PackedArgs a, const __grid_constant__ CUtensorMap tmq,
                         const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                         int32_t *err) {
  using namespace pt;
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  // heads fastest; the tiles that see the most keys first
  const int h = blockIdx.x % a.Hq;
  const int64_t slots = gridDim.x / a.Hq;
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x / a.Hq, slots, 2 * kRows, true);
  if (!t.valid) return;
  const int rows = min(2 * kRows, t.len - t.row0);
  const int64_t first = t.start + t.row0;
  T *out = static_cast<T *>(a.out) + first * a.o_st + h * a.o_sh;
  if (t.rest) {
    if (a.zero_rest) zero_rows(out, a.o_st, rows);
    return;
  }
  extern __shared__ __align__(1024) char smem_raw[];
  char *sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  FwdBars *bars = reinterpret_cast<FwdBars *>(sm + FwdSmem::kBar);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = h / (a.Hq / a.Hkv);
  // key blocks of each tile: those up to its diagonal
  const int all = (t.len + kBlock - 1) / kBlock;
  const int n0 = min(all, t.row0 / kBlock + 2), n1 = rows > kRows ? min(all, n0 + 2) : 0;
  const int blocks = max(n0, n1);
  if (warp == 8) tmem_alloc(&bars->tmem, kFwdCols);
  if (tid == 288) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bars->s_full[x], 1);
      mbar_init(&bars->p_full[x], 4);
      mbar_init(&bars->o_full[x], 1);
    }
    mbar_init_fence();
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = bars->tmem;
  bool ok = true;
  float l = 0.f, m = -INFINITY;
  const int x = warp >> 2, r = (warp & 3) * 32 + lane;  // of a softmax warp: tile and row
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;

  auto load = [&](int i) {
    const int s = i % kStages, row = static_cast<int>(t.start) + i * kBlock;
    mbar_arrive_expect_tx(&bars->full[s], 2 * kBlockBytes);
    tma_load_4d(sm + FwdSmem::kK + s * kBlockBytes, &tmk, 0, row, hk, 0, &bars->full[s]);
    tma_load_4d(sm + FwdSmem::kV + s * kBlockBytes, &tmv, 0, row, hk, 0, &bars->full[s]);
  };
  if (warp == 9) {
    if (lane == 0) {
      // Q rows behind the sequence are others' (their results go nowhere)
      mbar_arrive_expect_tx(&bars->q_full, (n1 > 0 ? 2 : 1) * kTileBytes);
      for (int i = 0; i < (n1 > 0 ? 4 : 2); ++i)
        tma_load_4d(sm + FwdSmem::kQ + i * kBlockBytes, &tmq, 0, static_cast<int>(first) + i * kBlock, h, 0,
                    &bars->q_full);
      for (int i = 0; i < blocks; ++i) {
        if (i >= kStages) ok = mbar_wait(&bars->empty[i % kStages], (i / kStages - 1) & 1);
        if (!ok) break;
        load(i);
      }
    }
    __syncwarp();
  } else if (warp == 8) {
    constexpr uint32_t id_s = idesc_f16(fmt, false, 64), id_o = idesc_f16(fmt, true, 64);
    const uint64_t dq = umma_desc_sw128(smem_u32(sm + FwdSmem::kQ), 16, 1024);
    const uint64_t dk = umma_desc_sw128(smem_u32(sm + FwdSmem::kK), 16, 1024);
    const uint64_t dv = umma_desc_sw128(smem_u32(sm + FwdSmem::kV), kBlockBytes, 1024);
    const uint32_t tm = shared_value(tmem);
    const int u0 = shared_value(n0), u1 = shared_value(n1), last = max(u0, u1);
    auto issue_s = [&](int y, int i) {
      const int s = i % kStages;
      ok = ok && mbar_wait(&bars->full[s], (i / kStages) & 1);
      fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16(tm + 64 * y, dq + y * (kTileBytes >> 4) + 2 * k, dk + s * (kBlockBytes >> 4) + 2 * k, id_s, k > 0);
        mma_commit(&bars->s_full[y]);
      }
      __syncwarp();
    };
    ok = mbar_wait(&bars->q_full, 0);
    issue_s(0, 0);
    if (u1 > 0) issue_s(1, 0);
    const int tail = shared_value(t.len) / kBlock;  // the block that holds the sequence's end, if it ends inside one
    for (int i = 0; i < last; ++i) {
      const int s = i % kStages;
      if (i == tail) {
        ok = ok && mbar_wait(&bars->full[s], (i / kStages) & 1);
        clear_rows(sm + FwdSmem::kV + s * kBlockBytes, t.len - tail * kBlock, kBlock);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int n = y ? u1 : u0;
        if (i >= n) continue;
        ok = ok && mbar_wait(&bars->p_full[y], i & 1);
        fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16_ts(tm + kFwdO + 64 * y, tm + 64 * y + 8 * k, dv + s * (kBlockBytes >> 4) + 128 * k, id_o,
                       i > 0 || k > 0);
          if (i + 1 == n) mma_commit(&bars->o_full[y]);
        }
        __syncwarp();
        if (i + 1 < n) issue_s(y, i + 1);
      }
      if (i + kStages < last && elect_one()) mma_commit(&bars->empty[s]);
      if (!__all_sync(0xffffffffu, ok)) break;
    }
  } else {
    const int n = x ? n1 : n0, row = t.row0 + x * kRows + r;
    const bool held = x * kRows + r < rows;  // the others' sums move no reference
    const uint32_t t_s = tmem + lane_base + 64 * x, t_o = tmem + lane_base + kFwdO + 64 * x;
    const float c = a.scale_log2;
    for (int i = 0; i < n; ++i) {
      ok = mbar_wait(&bars->s_full[x], i & 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      fence_after_sync();
      const bool edge = i * kBlock + kBlock - 1 > row - r;  // the diagonal's two blocks
      auto scores = [&](int part, float (&s)[16]) {
        tmem_ld16(t_s + 16 * part, s);
        tmem_wait_ld();
        if (edge) {
          const int seen = row + 1 - i * kBlock - 16 * part;
#pragma unroll
          for (int u = 0; u < 16; ++u) s[u] = u < seen ? s[u] : -INFINITY;
        }
      };
      uint32_t w[32];
      auto weights = [&](auto poly, bool raise) {
        constexpr bool kPoly = decltype(poly)::value;
        // without a reference yet: the sum is to say so, unless the block has none to give
        const float neg = m == -INFINITY ? (raise ? 0.f : INFINITY) : -m;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float s[16];
          scores(q, s);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float y0 = s[2 * e], y1 = s[2 * e + 1];
            fma2(y0, y1, c, neg);
            // every fourth pair's exponentials on the FMA pipe: the special-function unit is the busiest (1.90 -> 1.82
            // ms at 32768 tokens)
            if (kPoly && (e & 3) == 3)
              exp2_fma<true>(y0, y1);
            else
              y0 = ex2(y0), y1 = ex2(y1);
            add2(part[2 * (e & 1)], part[2 * (e & 1) + 1], y0, y1);
            w[8 * q + e] = pack2<T>(y0, y1);
          }
        }
        return (part[0] + part[1]) + (part[2] + part[3]);
      };
      float sum;
      for (bool raise = i == 0;;) {
        if (raise) {  // the reference moves to this block's maximum, what is summed so far with it
          float best = -INFINITY;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float s[16];
            scores(q, s);
#pragma unroll
            for (int u = 0; u < 16; ++u) best = fmaxf(best, s[u]);
          }
          best *= c;
          float alpha = 1.f;
          if (best > m) {
            alpha = m == -INFINITY ? 0.f : ex2(m - best);
            m = best;
          }
          l *= alpha;
          if (i > 0) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float o[16];
              tmem_ld16(t_o + 16 * u, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= alpha;
              tmem_st16(t_o + 16 * u, o);
            }
          }
        }
        // masked and first blocks, and what the polynomial's range does not hold (a NaN, an infinity, a weight
        // past 2^127: the sum tells), take the special-function unit for all
        sum = raise || edge ? weights(std::false_type(), raise) : weights(std::true_type(), false);
        if (raise || !__any_sync(0xffffffffu, held && !(sum <= kMostSum))) break;
        raise = true;
      }
      l += sum;
      tmem_st16(t_s, reinterpret_cast<const float(&)[16]>(w[0]));
      tmem_st16(t_s + 16, reinterpret_cast<const float(&)[16]>(w[16]));
      tmem_wait_st();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[x]);
    }
    if (n > 0 && ok) {
      ok = mbar_wait(&bars->o_full[x], 0);
      fence_after_sync();
    }
  }
  const bool failed = __syncthreads_or(!ok);
  if (failed) {  // a bounded wait expired: let copies in flight land, poison the rows
    if (tid == 288) {
      mbar_wait(&bars->q_full, 0, 1000000ull);
      for (int s = 0; s < kStages; ++s) mbar_wait(&bars->full[s], 0, 1000000ull);
    }
    l = __int_as_float(0x7fc00000);
    if (tid == 0 && err) *err = SD_KERR_TIMEOUT;
  }
  if (warp < 8 && (x == 0 || n1 > 0)) {
    fence_after_sync();
    const int row0 = 32 * warp, row = row0 + lane;  // of the CTA's rows
    T *rest = a.rest ? static_cast<T *>(a.rest) + ((first + row0) * a.Hq + h) * 64 : nullptr;
    // the tile's own Q is read no more
    unsigned again = store_rows(out + row0 * a.o_st, a.o_st, rows - row0, tmem + lane_base + kFwdO + 64 * x, 1.0f / l,
                                sm + FwdSmem::kQ + warp * 4096, rest, static_cast<int64_t>(a.Hq) * 64);
    if (again && !failed) {
      __syncwarp();  // a row's first result is written by other lanes than its second
      // the tile is looked up again: nothing is kept for this in the loop's registers
      const PackedTile u = packed_nth(a.cu, a.S, a.total, blockIdx.x / a.Hq, gridDim.x / a.Hq, 2 * kRows, true);
      const int at = u.row0 + 32 * warp, end = min(u.len, (at / kRows + 1) * kRows);  // the tile's keys end with its rows
      while (again) {
        PackedRows<2> g;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = again ? __ffs(again) - 1 : 0;
          g.row[i] = again ? at + n : -1;
          g.m[i] = __shfl_sync(0xffffffffu, m, n), g.l[i] = __shfl_sync(0xffffffffu, l, n);
          again &= again - 1;
        }
        packed_again<T>(a, u.start, end, blockIdx.x % a.Hq, g);
      }
    }
    if (row < rows && a.lse) a.lse[h * a.total + first + row] = m + log2f(l);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    fence_after_sync();
    tmem_dealloc(tmem, kFwdCols);
  }
}

// ---------------------------------------------------------------- backward
namespace pt {

constexpr int kBwdMma = 16, kBwdCopy = 17;    // warps; 0 to 15 compute
constexpr int kBwdThreads = 576;
constexpr int kBwdStages = 4;

struct BwdSmem {
  static constexpr int kRowsA = 0;                              // the CTA's rows: Q or K
  static constexpr int kRowsB = kRowsA + kTileBytes;            // dO or V
  static constexpr int kA = kRowsB + kTileBytes;                // the other side's blocks: K or Q
  static constexpr int kB = kA + kBwdStages * kTileBytes;       // V or dO
  static constexpr int kVec = kB + kBwdStages * kTileBytes;     // dK/dV: 16 warps x (32 lse, 32 delta)
  static constexpr int kTop = kVec + 4096;                      // fp16: the largest |dout|, |v|, |delta| of rows
  static constexpr int kBar = kTop + 2048;
  static constexpr int kBytes = kBar + 256;
};

// Tensor-memory columns: scores, dP, 16-bit weights (dS; for dK/dV P then dS), accumulators.
constexpr int kColS = 0, kColDp = 128, kColW = 256, kColW2 = 320;
constexpr int kDqAcc = 320, kDkvAcc = 384, kDkvAcc2 = 448;

struct BwdBars {
  uint64_t rows, full[kBwdStages], empty[kBwdStages];
  uint64_t sd_full, sd_free;  // S and dP computed; read
  uint64_t w_full, w_free;    // weights written; consumed
  uint32_t tmem;
};

__device__ __forceinline__ void bwd_init(BwdBars *bars) {
  mbar_init(&bars->rows, 1);
  for (int s = 0; s < kBwdStages; ++s) {
    mbar_init(&bars->full[s], 1);
    mbar_init(&bars->empty[s], 1);
  }
  mbar_init(&bars->sd_full, 1);
  mbar_init(&bars->sd_free, 16);
  mbar_init(&bars->w_full, 16);
  mbar_init(&bars->w_free, 1);
  mbar_init_fence();
}

// The copy thread: the CTA's rows, then the blocks; block i lies i % per_head
// blocks behind block_row, in head head0 + i / per_head.
__device__ __forceinline__ bool bwd_copy(BwdBars *bars, char *sm, const CUtensorMap &rows_a, const CUtensorMap &rows_b,
                                         int row, int head, const CUtensorMap &ma, const CUtensorMap &mb, int blocks,
                                         int per_head, int block_row, int head0) {
  mbar_arrive_expect_tx(&bars->rows, 2 * kTileBytes);
  tma_load_4d(sm + BwdSmem::kRowsA, &rows_a, 0, row, head, 0, &bars->rows);
  tma_load_4d(sm + BwdSmem::kRowsB, &rows_b, 0, row, head, 0, &bars->rows);
  int nth = 0;
  for (int i = 0; i < blocks; ++i) {
    const int s = i % kBwdStages;
    if (i >= kBwdStages && !mbar_wait(&bars->empty[s], (i / kBwdStages - 1) & 1)) return false;
    const int at = block_row + nth * kRows;
    mbar_arrive_expect_tx(&bars->full[s], 2 * kTileBytes);
    tma_load_4d(sm + BwdSmem::kA + s * kTileBytes, &ma, 0, at, head0, 0, &bars->full[s]);
    tma_load_4d(sm + BwdSmem::kB + s * kTileBytes, &mb, 0, at, head0, 0, &bars->full[s]);
    if (++nth == per_head) nth = 0, ++head0;
  }
  return true;
}

// A bounded wait expired: copies in flight land before the CTA ends.
__device__ __forceinline__ void bwd_failed(BwdBars *bars, int32_t *err) {
  if (threadIdx.x == 32 * kBwdCopy) {
    mbar_wait(&bars->rows, 0, 1000000ull);
    for (int s = 0; s < kBwdStages; ++s) mbar_wait(&bars->full[s], 0, 1000000ull);
  }
  if (threadIdx.x == 0 && err) *err = SD_KERR_TIMEOUT;
}

// fp16's range is narrow: weights fall as 1 / n, a loss averaged over many tokens
// has small output gradients, a scaled one large ones, and values add up.  So dS is
// held scaled by a power of two per accumulator row, from the pairs of that row
// alone: neither what else is packed beside its sequence nor what the row does not
// see costs it digits.  |dP - delta| is at most 64 max|dout| max|v| + max|delta|,
// which the power takes into [2^14, 2^15): twice that fits.  A look at the other
// side's rows ahead of the loop (the compute warps', while the first products run)
// finds the maxima: 16-bit magnitudes in pairs as integers, whose order is theirs.
__device__ __forceinline__ unsigned top2(uint4 x) {
  constexpr unsigned kAbs = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(x.x & kAbs, x.y & kAbs), __vmaxu2(x.z & kAbs, x.w & kAbs));
}
__device__ __forceinline__ unsigned top1(unsigned pair) { return max(pair & 0xffffu, pair >> 16); }
// What is not finite counts as the largest number: its own rows' gradients are not finite whatever the scale.
__device__ __forceinline__ float top_value(unsigned bits) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(min(bits, 0x7bffu))));
}
__device__ __forceinline__ float range_scale(float bound) {
  const int e = 268 - static_cast<int>(__float_as_uint(bound) >> 23);  // 2^(14 - floor(log2 bound))
  return __uint_as_float(static_cast<uint32_t>(min(max(e, 27), 227)) << 23);
}
constexpr int kComputeThreads = 512;
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// The MMA warp's loop, the same for both kernels: the products of block i + 1
// as soon as block i's are read, then the accumulation of block i once its
// weights are there.  Blocks come in runs of per_head, each over
// rows_left rows.  acc(off, first): issues the accumulating MMAs with the
// block's shared memory `off` (in descriptor units) behind the first stage's.
template <typename T, typename Acc>
__device__ __forceinline__ bool bwd_mma(BwdBars *bars, char *sm, uint32_t tmem, int blocks, int rows_left, int per_head,
                                        bool clear_b, Acc acc) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t id = idesc_f16(fmt, false, 128);
  const uint64_t ra = umma_desc_sw128(smem_u32(sm + BwdSmem::kRowsA), 16, 1024);
  const uint64_t rb = umma_desc_sw128(smem_u32(sm + BwdSmem::kRowsB), 16, 1024);
  const uint64_t da = umma_desc_sw128(smem_u32(sm + BwdSmem::kA), 16, 1024);
  const uint64_t db = umma_desc_sw128(smem_u32(sm + BwdSmem::kB), 16, 1024);
  const int whole = rows_left / kRows;  // a run's blocks that end within the sequence
  int nth = 0;                          // of the next block in its run
  bool ok = mbar_wait(&bars->rows, 0);
  auto products = [&](int i) {
    const int s = i % kBwdStages;
    ok = ok && mbar_wait(&bars->full[s], (i / kBwdStages) & 1);
    if (nth >= whole) {
      const int left = rows_left - nth * kRows;
      clear_rows(sm + BwdSmem::kA + s * kTileBytes, left, kRows);
      if (clear_b) clear_rows(sm + BwdSmem::kB + s * kTileBytes, left, kRows);
    }
    nth = nth + 1 == per_head ? 0 : nth + 1;
    fence_after_sync();
    if (elect_one()) {
      const uint32_t off = s * (kTileBytes >> 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_f16(tmem + kColS, ra + 2 * k, da + off + 2 * k, id, k > 0);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_f16(tmem + kColDp, rb + 2 * k, db + off + 2 * k, id, k > 0);
      mma_commit(&bars->sd_full);
    }
    __syncwarp();
  };
  products(0);
  for (int i = 0; i < blocks; ++i) {
    if (i + 1 < blocks) {
      ok = ok && mbar_wait(&bars->sd_free, i & 1);
      products(i + 1);
    }
    const int s = i % kBwdStages;
    ok = ok && mbar_wait(&bars->w_full, i & 1);
    fence_after_sync();
    if (elect_one()) {
      acc(static_cast<uint32_t>(s * (kTileBytes >> 4)), i == 0);
      mma_commit(&bars->w_free);
      if (i + kBwdStages < blocks) mma_commit(&bars->empty[s]);
    }
    __syncwarp();
    if (!__all_sync(0xffffffffu, ok)) return false;
  }
  return ok;
}

// A compute warp says that it has read its scores, or written its weights.
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
  fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

template <typename T> __device__ __forceinline__ void store_weights(uint32_t taddr, const float (&x)[32]) {
  float w[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) w[u] = __uint_as_float(pack2<T>(x[2 * u], x[2 * u + 1]));
  tmem_st16(taddr, w);
}

}  // namespace pt

// delta = rowsum(dout out), eight lanes a row and head.  A kernel of its own, so
// that both gradients' kernels can read it and the second may start while the first
// ends.
template <typename T> __global__ void __launch_bounds__(256) packed_delta_tc_kernel(const PackedArgs a) {
  const int64_t n = blockIdx.x * 32ll + (threadIdx.x >> 3), row = n / a.Hq;
  const int h = static_cast<int>(n - row * a.Hq), c = 8 * (threadIdx.x & 7);
  float delta = 0.f;
  const bool in = row < a.total;
  if (in) {
    const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.out) + row * a.o_st + h * a.o_sh + c);
    const uint4 y = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.dout) + row * a.g_st + h * a.g_sh + c);
    uint4 z = make_uint4(0u, 0u, 0u, 0u);
    // out in twice its bits: delta's error is the same for a whole row of dS, and would add up
    if (a.rest) z = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.rest) + (row * a.Hq + h) * 64 + c);
    const T *po = reinterpret_cast<const T *>(&x), *pg = reinterpret_cast<const T *>(&y),
            *pz = reinterpret_cast<const T *>(&z);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      delta = fmaf(to_f(po[u]), to_f(pg[u]), delta);
      delta = fmaf(to_f(pz[u]), to_f(pg[u]), delta);
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) delta += __shfl_xor_sync(0xffffffffu, delta, o);
  if (in && c == 0) a.delta[h * a.total + row] = delta;
}


template <typename T>
__global__ void __launch_bounds__(pt::kBwdThreads, 1)
    packed_bwd_dq_tc_kernel(const PackedArgs a, const __grid_constant__ CUtensorMap tmq,
                            const __grid_constant__ CUtensorMap tmg, const __grid_constant__ CUtensorMap tmk,
                            const __grid_constant__ CUtensorMap tmv, int32_t *err) {
  using namespace pt;
  // Starts while dK/dV's last CTAs run, of which it reads nothing; what follows on
  // the stream follows both, as one CTA here ends after all of theirs.
  if (blockIdx.x == gridDim.x - 1) pdl_wait();
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr uint32_t fmt = kHalf ? 0u : 1u;
  const int h = blockIdx.x % a.Hq;
  const int64_t slots = gridDim.x / a.Hq;
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x / a.Hq, slots, kRows, true);
  if (!t.valid) return;
  const int rows = min(kRows, t.len - t.row0);
  const int64_t first = t.start + t.row0, c_st = static_cast<int64_t>(a.Hq) * 64;
  T *dq = static_cast<T *>(a.dq) + first * c_st + h * 64;
  if (t.rest) {
    zero_rows(dq, c_st, rows);
    return;
  }
  extern __shared__ __align__(1024) char smem_raw[];
  char *sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  BwdBars *bars = reinterpret_cast<BwdBars *>(sm + BwdSmem::kBar);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = h / (a.Hq / a.Hkv);
  const int blocks = t.row0 / kRows + 1;  // keys up to the tile's diagonal
  if (warp == kBwdMma) tmem_alloc(&bars->tmem, 512);
  if (tid == 32 * kBwdCopy) bwd_init(bars);
  const int wg = warp >> 2, r = (warp & 3) * 32 + lane;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = bars->tmem;
  float f = 1.f;  // of this thread's query
  bool ok = true;
  if (warp == kBwdCopy) {
    if (lane == 0)
      ok = bwd_copy(bars, sm, tmq, tmg, static_cast<int>(first), h, tmk, tmv, blocks, blocks,
                    static_cast<int>(t.start), hk);
    __syncwarp();
  } else if (warp == kBwdMma) {
    constexpr uint32_t id = idesc_f16(fmt, true, 64);
    const uint64_t dk = umma_desc_sw128(smem_u32(sm + BwdSmem::kA), kTileBytes, 1024);
    const uint32_t tm = shared_value(tmem);
    const int n = shared_value(blocks);
    ok = bwd_mma<T>(bars, sm, tm, n, shared_value(t.len), n + 1, false, [&](uint32_t off, bool start) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        mma_f16_ts(tm + kDqAcc, tm + kColW + 8 * k, dk + off + 128 * k, id, !start || k > 0);
    });
  } else {
    const uint32_t t_s = tmem + lane_base + kColS + 32 * wg;
    const float delta = r < rows ? a.delta[h * a.total + first + r] : 0.f;
    const float lse = r < rows ? a.lse[h * a.total + first + r] : 0.f;
    if (kHalf) {
      // largest |dout| of each query; |v| of each key of the tile's own rows, and of all before them
      unsigned *grads = reinterpret_cast<unsigned *>(sm + BwdSmem::kTop), *vals = grads + kRows, *vals_on = vals + kRows;
      const int part = lane >> 3, c = 8 * (lane & 7);
      const T *v = static_cast<const T *>(a.v) + t.start * a.v_st + hk * a.v_sh + c;
      const T *g = static_cast<const T *>(a.dout) + first * a.g_st + h * a.g_sh + c;
      auto row_top = [&](const T *p) { return top2(*reinterpret_cast<const uint4 *>(p)); };
      for (int row = 4 * warp + part; row < kRows; row += 64) {
        unsigned both = 0;
        if (row < rows) both = top1(row_top(v + (t.row0 + row) * a.v_st)) << 16 | top1(row_top(g + row * a.g_st));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
        if ((lane & 7) == 0) vals[row] = both >> 16, grads[row] = both & 0xffffu;
      }
      unsigned on = 0;
#pragma unroll 8
      for (int row = 4 * warp + part; row < t.row0; row += 64) on = __vmaxu2(on, row_top(v + row * a.v_st));
      on = __reduce_max_sync(0xffffffffu, top1(on));
      if (lane == 0) vals_on[warp] = on;
      compute_sync();
      // over the keys up to this thread's query: the query's 32 rows by a scan, those before them whole
      unsigned top_v = vals_on[lane & 15], own_v = vals[r];
      for (int w = 0; w < (warp & 3); ++w) top_v = max(top_v, vals[32 * w + lane]);
      top_v = __reduce_max_sync(0xffffffffu, top_v);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, own_v, o);
        if (lane >= o) own_v = max(own_v, x);
      }
      f = range_scale(64.f * top_value(grads[r]) * top_value(max(top_v, own_v)) + fminf(fabsf(delta), 3.0e38f));
    }
    for (int i = 0; i < blocks; ++i) {
      ok = mbar_wait(&bars->sd_full, i & 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      fence_after_sync();
      float s[32], d[32];
      tmem_ld32(t_s, s);
      tmem_ld32(t_s + kColDp, d);
      tmem_wait_ld();
      warp_arrive(&bars->sd_free);
      // every fourth pair of exponentials on the FMA pipe where nothing is masked (scores are at most lse; a NaN
      // there is in delta too)
      auto weights = [&](auto poly) {
#pragma unroll
        for (int u = 0; u < 32; u += 2) {
          fma2(s[u], s[u + 1], a.scale_log2, -lse);
          if (decltype(poly)::value && u % 8 == 6)
            exp2_fma<false>(s[u], s[u + 1]);
          else
            s[u] = ex2(s[u]), s[u + 1] = ex2(s[u + 1]);
          if (kHalf)
            fma2(d[u], d[u + 1], f, -delta * f);
          else
            add2(d[u], d[u + 1], -delta, -delta);
          mul2(d[u], d[u + 1], s[u], s[u + 1]);
        }
      };
      if (i + 1 < blocks) {
        weights(std::true_type());
      } else {  // the diagonal block
        weights(std::false_type());
        const int seen = r + 1 - 32 * wg;
#pragma unroll
        for (int u = 0; u < 32; ++u) d[u] = u < seen ? d[u] : 0.f;
      }
      if (i > 0) ok = mbar_wait(&bars->w_free, (i - 1) & 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      fence_after_sync();
      store_weights<T>(tmem + lane_base + kColW + 16 * wg, d);
      tmem_wait_st();
      warp_arrive(&bars->w_full);
    }
    if (ok) {
      ok = mbar_wait(&bars->w_free, (blocks - 1) & 1);
      fence_after_sync();
    }
  }
  const bool failed = __syncthreads_or(!ok);
  if (failed) bwd_failed(bars, err);
  if (warp < 4) {
    fence_after_sync();
    const float back = failed ? __int_as_float(0x7fc00000) : a.scale / f;
    store_rows(dq + 32 * warp * c_st, c_st, rows - 32 * warp, tmem + lane_base + kDqAcc, back,
               sm + BwdSmem::kRowsA + warp * 4096);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == kBwdMma) {
    fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T>
__global__ void __launch_bounds__(pt::kBwdThreads, 1)
    packed_bwd_dkv_tc_kernel(const PackedArgs a, const __grid_constant__ CUtensorMap tmq,
                             const __grid_constant__ CUtensorMap tmg, const __grid_constant__ CUtensorMap tmk,
                             const __grid_constant__ CUtensorMap tmv, int32_t *err) {
  using namespace pt;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // dQ's CTAs take the SMs that this one's leave
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr uint32_t fmt = kHalf ? 0u : 1u;
  const int hk = blockIdx.x % a.Hkv, group = a.Hq / a.Hkv;
  // the keys that are seen by the most queries first
  const PackedTile t = packed_nth(a.cu, a.S, a.total, blockIdx.x / a.Hkv, gridDim.x / a.Hkv, kRows, false);
  if (!t.valid) return;
  const int keys = min(kRows, t.len - t.row0);
  const int64_t first = t.start + t.row0, c_st = static_cast<int64_t>(a.Hkv) * 64;
  T *dk = static_cast<T *>(a.dk) + first * c_st + hk * 64, *dv = static_cast<T *>(a.dv) + first * c_st + hk * 64;
  if (t.rest) {
    zero_rows(dk, c_st, keys);
    zero_rows(dv, c_st, keys);
    return;
  }
  extern __shared__ __align__(1024) char smem_raw[];
  char *sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float *vec = reinterpret_cast<float *>(sm + BwdSmem::kVec);
  BwdBars *bars = reinterpret_cast<BwdBars *>(sm + BwdSmem::kBar);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_head = (t.len - t.row0 + kRows - 1) / kRows, blocks = per_head * group;
  if (warp == kBwdMma) tmem_alloc(&bars->tmem, 512);
  if (tid == 32 * kBwdCopy) bwd_init(bars);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = bars->tmem;
  const int wg = warp >> 2, r = (warp & 3) * 32 + lane;
  const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
  float f = 1.f;  // of this thread's key
  // fp16: P, at most 1, is held as 2^15 P, so that keys with little weight keep the digits of dV
  constexpr float kWeight = kHalf ? 15.f : 0.f, kUnweight = kHalf ? 1.f / 32768.f : 1.f;
  bool ok = true;
  if (warp == kBwdCopy) {
    if (lane == 0)
      ok = bwd_copy(bars, sm, tmk, tmv, static_cast<int>(first), hk, tmq, tmg, blocks, per_head,
                    static_cast<int>(first), hk * group);
    __syncwarp();
  } else if (warp == kBwdMma) {
    constexpr uint32_t id = idesc_f16(fmt, true, 64);
    const uint64_t dq = umma_desc_sw128(smem_u32(sm + BwdSmem::kA), kTileBytes, 1024);
    const uint64_t dg = umma_desc_sw128(smem_u32(sm + BwdSmem::kB), kTileBytes, 1024);
    const uint32_t tm = shared_value(tmem);
    ok = bwd_mma<T>(bars, sm, tm, shared_value(blocks), shared_value(t.len - t.row0), shared_value(per_head), true,
                    [&](uint32_t off, bool start) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        mma_f16_ts(tm + kDkvAcc, tm + kColW + 8 * k, dg + off + 128 * k, id, !start || k > 0);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        mma_f16_ts(tm + kDkvAcc2, tm + kColW2 + 8 * k, dq + off + 128 * k, id, !start || k > 0);
    });
  } else {
    const uint32_t t_s = tmem + lane_base + kColS + 32 * wg;
    // the warp's 32 queries' log sums and deltas, negated: a lane brings one of each, all read them from shared memory
    float *mine = vec + warp * 64;
    const int span = t.len - t.row0 - 32 * wg;  // rows of a head from this warpgroup's first query on
    int64_t at = static_cast<int64_t>(hk) * group * a.total + first + 32 * wg + lane;
    int qn = 0;  // the next block's first query, from the tile's first key
    float next_l, next_d;
    auto fetch = [&](bool more) {
      const bool held = more && qn + lane < span;
      next_l = next_d = 0.f;
      if (held) next_l = a.lse[at + qn], next_d = a.delta[at + qn];  // negated when stored: nothing waits for them here
      qn += kRows;
      if (qn >= span + 32 * wg) qn = 0, at += a.total;
    };
    fetch(true);
    if (kHalf) {
      // largest |v| of each key; |dout| and |delta| of each query of the tile's own rows, and of all behind them
      unsigned *vals = reinterpret_cast<unsigned *>(sm + BwdSmem::kTop), *grads = vals + kRows, *grads_on = grads + kRows;
      float *deltas = reinterpret_cast<float *>(grads_on + 16), *deltas_on = deltas + kRows;
      const int len = t.len - t.row0, part = lane >> 3, c = 8 * (lane & 7);
      const T *v = static_cast<const T *>(a.v) + first * a.v_st + hk * a.v_sh + c;
      const T *g = static_cast<const T *>(a.dout) + first * a.g_st + hk * group * a.g_sh + c;
      auto row_top = [&](const T *p) { return top2(*reinterpret_cast<const uint4 *>(p)); };
      for (int row = 4 * warp + part; row < kRows; row += 64) {
        unsigned big_v = 0, big_g = 0;
        if (row < keys) {
          big_v = row_top(v + row * a.v_st);
          for (int h = 0; h < group; ++h) big_g = __vmaxu2(big_g, row_top(g + row * a.g_st + h * a.g_sh));
        }
        unsigned both = top1(big_v) << 16 | top1(big_g);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
        if ((lane & 7) == 0) vals[row] = both >> 16, grads[row] = both & 0xffffu;
      }
      auto size = [](float x) { return fminf(fabsf(x), 3.0e38f); };  // a NaN as well
      const float *d = a.delta + static_cast<int64_t>(hk) * group * a.total + first;
      if (tid < kRows) {
        float big = 0.f;
        for (int h = 0; h < group; ++h)
          if (tid < keys) big = fmaxf(big, size(d[h * a.total + tid]));
        deltas[tid] = big;
      }
      unsigned on = 0;
      float d_on = 0.f;
      for (int h = 0; h < group; ++h) {
#pragma unroll 8
        for (int row = kRows + 4 * warp + part; row < len; row += 64)
          on = __vmaxu2(on, row_top(g + row * a.g_st + h * a.g_sh));
#pragma unroll 4
        for (int row = kRows + tid; row < len; row += kComputeThreads) d_on = fmaxf(d_on, size(d[h * a.total + row]));
      }
      on = __reduce_max_sync(0xffffffffu, top1(on));
      const unsigned d_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(d_on));
      if (lane == 0) grads_on[warp] = on, deltas_on[warp] = __uint_as_float(d_bits);
      compute_sync();
      // over the queries from this thread's key on: the key's 32 rows by a scan, those behind them whole
      unsigned top_g = grads_on[lane & 15], top_d = __float_as_uint(deltas_on[lane & 15]);
      for (int w = (warp & 3) + 1; w < 4; ++w)
        top_g = max(top_g, grads[32 * w + lane]), top_d = max(top_d, __float_as_uint(deltas[32 * w + lane]));
      top_g = __reduce_max_sync(0xffffffffu, top_g), top_d = __reduce_max_sync(0xffffffffu, top_d);
      unsigned own_g = grads[r], own_d = __float_as_uint(deltas[r]);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_down_sync(0xffffffffu, own_g, o), y = __shfl_down_sync(0xffffffffu, own_d, o);
        if (lane + o < 32) own_g = max(own_g, x), own_d = max(own_d, y);
      }
      f = range_scale(64.f * top_value(max(top_g, own_g)) * top_value(vals[r]) + __uint_as_float(max(top_d, own_d)));
    }
    const float fw = f * kUnweight;  // dP - delta's share: dS = (2^15 P) (fw (dP - delta))
    for (int i = 0; i < blocks; ++i) {
      __syncwarp();
      mine[lane] = kWeight - next_l;
      mine[32 + lane] = -next_d;
      const bool nan = __any_sync(0xffffffffu, next_l != next_l);
      __syncwarp();
      const int q0 = qn == 0 ? (span + 32 * wg - 1) / kRows * kRows : qn - kRows;  // this block's
      fetch(i + 1 < blocks);
      ok = mbar_wait(&bars->sd_full, i & 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      fence_after_sync();
      const int from = r - q0 - 32 * wg, to = span - q0;  // visible columns: from .. to - 1
      const bool plain = q0 > 0 && to >= 32 && !nan;
      // 16 columns at a time: the two weights' 32-bit halves take over the scores' registers
      float wp[16], wd[16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float s[16], d[16];
        tmem_ld16(t_s + 16 * half, s);
        tmem_ld16(t_s + kColDp + 16 * half, d);
        tmem_wait_ld();
        if (half == 1) warp_arrive(&bars->sd_free);
        auto weights = [&](auto poly) {
#pragma unroll
          for (int u = 0; u < 16; u += 4) {
            const float4 l4 = *reinterpret_cast<const float4 *>(mine + 16 * half + u);
            const float4 d4 = *reinterpret_cast<const float4 *>(mine + 32 + 16 * half + u);
            fma2v(s[u], s[u + 1], a.scale_log2, l4.x, l4.y);
            fma2v(s[u + 2], s[u + 3], a.scale_log2, l4.z, l4.w);
            add2(d[u], d[u + 1], d4.x, d4.y);
            add2(d[u + 2], d[u + 3], d4.z, d4.w);
            s[u] = ex2(s[u]), s[u + 1] = ex2(s[u + 1]);
            if (decltype(poly)::value && u % 8 == 4)
              exp2_fma<false>(s[u + 2], s[u + 3]);
            else
              s[u + 2] = ex2(s[u + 2]), s[u + 3] = ex2(s[u + 3]);
            if (kHalf) {
              mul2(d[u], d[u + 1], fw, fw);
              mul2(d[u + 2], d[u + 3], fw, fw);
            }
            mul2(d[u], d[u + 1], s[u], s[u + 1]);
            mul2(d[u + 2], d[u + 3], s[u + 2], s[u + 3]);
          }
        };
        if (plain) {
          weights(std::true_type());
        } else {
          weights(std::false_type());
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const bool seen = 16 * half + u >= from && 16 * half + u < to;
            s[u] = seen ? s[u] : 0.f;
            d[u] = seen ? d[u] : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          wp[8 * half + u] = __uint_as_float(pack2<T>(s[2 * u], s[2 * u + 1]));
          wd[8 * half + u] = __uint_as_float(pack2<T>(d[2 * u], d[2 * u + 1]));
        }
      }
      if (i > 0) ok = mbar_wait(&bars->w_free, (i - 1) & 1);
      if (__any_sync(0xffffffffu, !ok)) break;
      fence_after_sync();
      tmem_st16(tmem + lane_base + kColW + 16 * wg, wp);
      tmem_st16(tmem + lane_base + kColW2 + 16 * wg, wd);
      tmem_wait_st();
      warp_arrive(&bars->w_full);
    }
    if (ok) {
      ok = mbar_wait(&bars->w_free, (blocks - 1) & 1);
      fence_after_sync();
    }
  }
  const bool failed = __syncthreads_or(!ok);
  if (failed) bwd_failed(bars, err);
  if (warp < 8) {
    fence_after_sync();
    const float back = failed ? __int_as_float(0x7fc00000) : wg == 0 ? kUnweight : a.scale / f;
    const int row0 = 32 * (warp & 3);
    store_rows((wg == 0 ? dv : dk) + row0 * c_st, c_st, keys - row0,
               tmem + lane_base + (wg == 0 ? kDkvAcc : kDkvAcc2), back, sm + BwdSmem::kRowsA + warp * 4096);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == kBwdMma) {
    fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Map of a packed tensor [total][H][64]: boxes of `box` rows of one head.
static int packed_map(CUtensorMap *map, const void *p, int dtype, int64_t total, int64_t H, int64_t st, int64_t sh,
                      int box) {
  if (H == 1 && sh <= 0) sh = 64;
  if (total == 1 && st <= 0) st = sh * H;
  return encode_rows_map(map, p, dtype, 64, total, H, 1, st, sh, st, box);
}

int launch_packed_fwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s) {
  CUtensorMap mq, mk, mv;
  int rc = packed_map(&mq, a.q, dtype, a.total, a.Hq, a.q_st, a.q_sh, pt::kBlock);
  if (rc == SD_OK) rc = packed_map(&mk, a.k, dtype, a.total, a.Hkv, a.k_st, a.k_sh, pt::kBlock);
  if (rc == SD_OK) rc = packed_map(&mv, a.v, dtype, a.total, a.Hkv, a.v_st, a.v_sh, pt::kBlock);
  if (rc != SD_OK) return rc;
  const int64_t ctas = packed_slots(a.total, a.S, 2 * pt::kRows) * a.Hq;
  if (ctas > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  const size_t smem = pt::FwdSmem::kBytes + 1024;
  auto run = [&](auto *kern) {
    if (ensure_smem(kern, smem) != SD_OK) return static_cast<int>(SD_ERR_CUDA);
    kern<<<static_cast<unsigned>(ctas), pt::kFwdThreads, smem, s>>>(a, mq, mk, mv, err);
    return check_launch();
  };
  return dtype == SD_DTYPE_BF16 ? run(packed_fwd_tc_kernel<__nv_bfloat16>) : run(packed_fwd_tc_kernel<__half>);
}

int launch_packed_bwd_tc(const PackedArgs &a, int dtype, int32_t *err, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mg;
  int rc = packed_map(&mq, a.q, dtype, a.total, a.Hq, a.q_st, a.q_sh, pt::kRows);
  if (rc == SD_OK) rc = packed_map(&mk, a.k, dtype, a.total, a.Hkv, a.k_st, a.k_sh, pt::kRows);
  if (rc == SD_OK) rc = packed_map(&mv, a.v, dtype, a.total, a.Hkv, a.v_st, a.v_sh, pt::kRows);
  if (rc == SD_OK) rc = packed_map(&mg, a.dout, dtype, a.total, a.Hq, a.g_st, a.g_sh, pt::kRows);
  if (rc != SD_OK) return rc;
  const int64_t slots = packed_slots(a.total, a.S, pt::kRows);
  if (slots * a.Hq > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  const size_t smem = pt::BwdSmem::kBytes + 1024;
  const int64_t delta_ctas = (a.total * a.Hq + 31) / 32;
  if (delta_ctas > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  auto run = [&](auto *delta, auto *dq, auto *dkv) {
    if (ensure_smem(dq, smem) != SD_OK || ensure_smem(dkv, smem) != SD_OK) return static_cast<int>(SD_ERR_CUDA);
    delta<<<static_cast<unsigned>(delta_ctas), 256, 0, s>>>(a);
    int rc = check_launch();
    if (rc != SD_OK) return rc;
    // the kernel with the longer CTAs first: the other's fill the SMs that its last ones leave
    dkv<<<static_cast<unsigned>(slots * a.Hkv), pt::kBwdThreads, smem, s>>>(a, mq, mg, mk, mv, err);
    rc = check_launch();
    if (rc != SD_OK) return rc;
    return launch(dq, dim3(static_cast<unsigned>(slots * a.Hq)), dim3(pt::kBwdThreads), smem, s, true, a, mq, mg, mk,
                  mv, err);
  };
  return dtype == SD_DTYPE_BF16 ? run(packed_delta_tc_kernel<__nv_bfloat16>, packed_bwd_dq_tc_kernel<__nv_bfloat16>,
                                      packed_bwd_dkv_tc_kernel<__nv_bfloat16>)
                                : run(packed_delta_tc_kernel<__half>, packed_bwd_dq_tc_kernel<__half>,
                                      packed_bwd_dkv_tc_kernel<__half>);
}

}  // namespace sd
