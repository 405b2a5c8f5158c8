// Log probabilities of given tokens with the distribution's entropy and its
// likeliest tokens, and the gradient of the logits.
//
//   m = max x,  s = sum exp(x - m),  w = sum exp(x - m) (x - m)
//   log p_j = x_j - m - log s,   H = log s - w / s
//   d/dx_j (g log p_t + h H) = g [j = t] - p_j (g + h (log p_j + H))
//
// m, s and w come from one pass over the row in fp32 (s and w are rescaled when
// m rises).  x - m is formed before it is scaled to base 2: with large common
// offsets a rounded m log2(e) would cost digits.  A logit of -inf has
// probability 0 and adds nothing; a row with a NaN, a +inf or nothing but -inf
// has NaN results, as log_softmax.
//
// HBM-bound where rows are many: 8192 x 32000 bf16 forward 105 us (524 MB, 5.0
// TB/s: the exponentials and the entropy's sum fill the issue slots beside the
// loads), gradient 165 us (1.05 GB read and written, 6.4 TB/s).  64 rows with 8
// alternatives and entropy take 10.4 us, a row's latency: its pass, the joining
// of its threads, and the pass for the alternatives.
#include <type_traits>

#include "sd_common.cuh"

namespace sd {

namespace lp {

// From four rows an SM on, small CTAs win: one's loads cover another's joining
// of its threads (8192 x 32000 bf16: 105 us with 128 threads, 127 with 256, 189
// with 512; the gradient 165 us with 256, 168 with 128, 177 with 512).  With
// fewer rows a row's own latency counts (64 rows: 5.5 us with 512 threads).
constexpr int64_t kManyRows = 4 * 148;
constexpr int kGroups = 128;            // of threads: their maxima bound the top_k-th value (top_k <= 64)
constexpr int kAbove = 4096;            // room for the values above that bound,
constexpr int kTies = 512;              // and for those equal to it
constexpr int kCandidates = kAbove + kTies;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFloor = -1e4f;         // stands for what is below it: its exponential is 0 and 0 * kFloor is 0

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

struct Stat {
  float m, s, w;
};

// m rises to (or stays at) top.
__device__ __forceinline__ void raise(Stat &a, float top) {
  if (!(top > a.m)) return;
  if (a.m == -INFINITY) {
    a.m = top;
    return;  // s and w are 0, or NaN
  }
  // a sum of masked values (the type's lowest, or far below) times their distance would pass the range of fp32
  const float d = fmaxf(a.m - top, kFloor), c = ex2(d * kLog2e);
  a.w = c * fmaf(a.s, d, a.w);
  a.s *= c;
  a.m = top;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 y;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 y;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(y.x), "=f"(y.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return y;
}

// N values (N even) with their largest and smallest (NaNs left out).  Nearly
// always none is -inf or so far below that its distance could overflow, and the
// guard is left out for all.
template <int N> __device__ __forceinline__ void add(Stat &a, const float (&x)[N], float top, float least) {
  raise(a, top);
  const float ref = a.m == -INFINITY ? 0.f : a.m;
  const float2 neg = {-ref, -ref}, log2e = {kLog2e, kLog2e}, zero = {0.f, 0.f};
  float2 s[2] = {}, w[2] = {};
  const bool guard = least - ref < kFloor;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 d = add2({x[i], x[i + 1]}, neg);
    if (guard) d.x = max_nan(d.x, kFloor), d.y = max_nan(d.y, kFloor);
    float2 e = fma2(d, log2e, zero);
    e.x = ex2(e.x), e.y = ex2(e.y);
    s[(i >> 1) & 1] = add2(s[(i >> 1) & 1], e);
    w[(i >> 1) & 1] = fma2(e, d, w[(i >> 1) & 1]);
  }
  a.s += (s[0].x + s[0].y) + (s[1].x + s[1].y);
  a.w += (w[0].x + w[0].y) + (w[1].x + w[1].y);
}
__device__ __forceinline__ void add_one(Stat &a, float x) {
  const float pair[2] = {x, -INFINITY};
  add(a, pair, x, -INFINITY);
}

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float top = fmaxf(a.m, b.m);
  raise(a, top);
  raise(b, top);
  a.s += b.s;
  a.w += b.w;
  return a;
}

// A float's place in the order NaN > +inf > ... > -inf, with -0 = +0.
__device__ __forceinline__ uint32_t place(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Larger for a larger value, for equal ones at the lower index.
__device__ __forceinline__ unsigned long long key_of(float x, int64_t j) {
  return static_cast<unsigned long long>(place(x)) << 32 | (0xfffffffeu - static_cast<uint32_t>(j));
}

template <typename T> struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4 &raw, float *x) {
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y);
      x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
    } else {
      const T *p = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int i = 0; i < kN; ++i) x[i] = to_f(p[i]);
    }
  }
  // Largest and smallest of n pieces: 16-bit types two values an instruction.
  template <int n> static __device__ __forceinline__ void range(const uint4 (&raw)[n], float &top, float &least) {
    if constexpr (sizeof(T) == 4) {
      top = -INFINITY, least = INFINITY;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        float x[4];
        unpack(raw[i], x);
        top = fmaxf(top, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        least = fminf(least, fminf(fminf(x[0], x[1]), fminf(x[2], x[3])));
      }
    } else {
      using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const T2 *p = reinterpret_cast<const T2 *>(&raw[0]);
      T2 hi = p[0], lo = p[0];
#pragma unroll
      for (int i = 1; i < 4 * n; ++i) hi = __hmax2(hi, p[i]), lo = __hmin2(lo, p[i]);
      top = fmaxf(to_f(hi.x), to_f(hi.y));
      least = fminf(to_f(lo.x), to_f(lo.y));
    }
  }
};

// A row in 16-byte pieces: `head` values up to the first aligned address, then
// `vecs` pieces, then the rest.
template <typename T> struct Row {
  const T *p;
  int64_t n;
  int head;
  int64_t vecs, tail;
  __device__ __forceinline__ Row(const T *row, int64_t V) : p(row), n(V) {
    const int64_t off = ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T);
    head = static_cast<int>(off < V ? off : V);
    vecs = (V - head) / Vec<T>::kN;
    tail = head + vecs * Vec<T>::kN;
  }
  __device__ __forceinline__ const uint4 *body() const { return reinterpret_cast<const uint4 *>(p + head); }
};

}  // namespace lp

// One CTA a row.  stats [3][rows]: m, log s, H (kept for the gradient).
//
// top_k: the top_k-th largest of the 128 thread groups' maxima bounds the
// top_k-th largest value from below, so a second pass (the row is in L2, 64 KB
// for 32000 16-bit logits) collects the values above that bound and those equal
// to it (only the first top_k of these, in index order, where they are many); a
// candidate's rank among them is its place in the answer.
template <typename T, bool kTop, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    token_logprobs_kernel(const T *x, int64_t rows, int64_t V, int64_t ld, const int64_t *targets,
                          int64_t ignore_index, float *logprobs, float *entropy, float *stats, int top_k,
                          float *top_logprobs, int64_t *top_ids, int32_t *err) {
  using namespace lp;
  constexpr int kN = Vec<T>::kN, kUnroll = 4, kWarps = kThreads / 32;
  __shared__ Stat part[kWarps];
  const int64_t r = blockIdx.x;
  const Row<T> row(x + r * ld, V);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Stat a = {-INFINITY, 0.f, 0.f};
  float top = -INFINITY;  // largest value of this thread that is a number
  {
    if (tid < row.head) add_one(a, to_f(row.p[tid]));
    if (row.tail + tid < V) add_one(a, to_f(row.p[row.tail + tid]));
    const uint4 *body = row.body();
    int64_t i = tid;
    for (; i + (kUnroll - 1) * kThreads < row.vecs; i += kUnroll * kThreads) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) raw[u] = __ldg(body + i + u * kThreads);
      float y[kUnroll * kN], hi, lo;
      Vec<T>::range(raw, hi, lo);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) Vec<T>::unpack(raw[u], y + kN * u);
      add(a, y, hi, lo);
    }
    for (; i < row.vecs; i += kThreads) {
      uint4 raw[1] = {__ldg(body + i)};
      float y[kN], hi, lo;
      Vec<T>::range(raw, hi, lo);
      Vec<T>::unpack(raw[0], y);
      add(a, y, hi, lo);
    }
    top = a.m;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat b = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                    __shfl_xor_sync(0xffffffffu, a.w, o)};
    // both lanes of a pair join in the same order, so that all end with equal bits
    a = lane & o ? join(b, a) : join(a, b);
  }
  if (lane == 0) part[warp] = a;
  __syncthreads();
  a = part[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) a = join(a, part[i]);
  const float logs = a.s > 0.f ? logf(a.s) : __int_as_float(0x7fc00000);
  if (tid == 0) {
    const float h = logs - a.w / a.s;
    const int64_t t = targets[r];
    float v = 0.f;
    if (t != ignore_index) {
      if (t >= 0 && t < V) {
        v = to_f(row.p[t]) - a.m - logs;
      } else {
        v = __int_as_float(0x7fc00000);
        if (err) *err = SD_KERR_BOUNDS;
      }
    }
    logprobs[r] = v;
    if (entropy) entropy[r] = h;
    if (stats) stats[r] = a.m, stats[rows + r] = logs, stats[2 * rows + r] = h;
  }
  if constexpr (kTop) {
    extern __shared__ unsigned long long cand[];  // [kCandidates]
    __shared__ float group[kGroups];
    __shared__ float bound;
    __shared__ int above, ties;  // values above the bound, and equal to it
    __shared__ int count[kWarps];
    constexpr int kGroup = kThreads / kGroups;  // threads of a group
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (tid % kGroup == 0) group[tid / kGroup] = top;
    if (tid == 0) above = ties = 0;
    __syncthreads();
    if (tid < kGroups) {
      const float mine = group[tid];
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < kGroups; ++i) rank += group[i] > mine || (group[i] == mine && i < tid);
      if (rank == top_k - 1) bound = mine;
    }
    __syncthreads();
    const float low = bound;
    // candidates above the bound fill the buffer from its start, equal ones from
    // its end
    auto take = [&](float v, int64_t j) {
      if (v < low) return;
      if (v == low) {
        const int at = atomicAdd(&ties, 1);
        if (at < kTies) cand[kCandidates - 1 - at] = key_of(v, j);
      } else {
        const int at = atomicAdd(&above, 1);
        if (at < kAbove) cand[at] = key_of(v, j);
      }
    };
    const uint4 *body = row.body();
    auto take_vec = [&](const uint4 &raw, int64_t i) {
      float y[kN];
      Vec<T>::unpack(raw, y);
      bool any = false;
#pragma unroll
      for (int e = 0; e < kN; ++e) any = any || !(y[e] < low);
      if (any) {
#pragma unroll
        for (int e = 0; e < kN; ++e) take(y[e], row.head + i * kN + e);
      }
    };
    if (tid < row.head) take(to_f(row.p[tid]), tid);
    if (row.tail + tid < V) take(to_f(row.p[row.tail + tid]), row.tail + tid);
    for (int64_t i = tid; i < row.vecs; i += kUnroll * kThreads) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i + u * kThreads < row.vecs) raw[u] = __ldg(body + i + u * kThreads);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (i + u * kThreads < row.vecs) take_vec(raw[u], i + u * kThreads);
    }
    __syncthreads();
    if (ties > kTies) {  // (a masked vocabulary, a flat row) keep the first top_k of the equal ones, in index order
      int found = 0;
      __syncthreads();
      // pieces in order: the head, the body's, the tail; a thread's equal values and how many lie before them
      const int64_t steps = (row.vecs + kThreads - 1) / kThreads + 2;
      for (int64_t step = 0; step < steps && found < top_k; ++step) {
        const bool head = step == 0, tail = step == steps - 1;
        const int64_t i = (step - 1) * kThreads + tid;
        int64_t j = head ? tid : tail ? row.tail + tid : row.head + i * kN;
        uint32_t equal = 0;
        if (head || tail) {
          equal = j < (head ? row.head : V) && to_f(row.p[j]) == low;
        } else if (i < row.vecs) {
          float y[kN];
          Vec<T>::unpack(__ldg(body + i), y);
#pragma unroll
          for (int e = 0; e < kN; ++e) equal |= static_cast<uint32_t>(y[e] == low) << e;
        }
        int before = __popc(equal);
        const int own = before;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += y;
        }
        if (lane == 31) count[warp] = before;
        __syncthreads();
        before += found - own;
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) before += count[w];
          all += count[w];
        }
        for (; equal && before < top_k; equal &= equal - 1, ++before)
          cand[kCandidates - 1 - before] = key_of(low, j + __ffs(equal) - 1);
        found += all;
        __syncthreads();
      }
      if (tid == 0) ties = min(found, top_k);
      __syncthreads();
    }
    const int na = above, nt = ties, n = na + nt;
    if (na <= kAbove) {
      auto get = [&](int i) { return cand[i < na ? i : kCandidates - 1 - (i - na)]; };
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long mine = get(i);
        int rank = 0;
        for (int j = 0; j < na; ++j) rank += cand[j] > mine;
        for (int j = 0; j < nt; ++j) rank += cand[kCandidates - 1 - j] > mine;
        if (rank < top_k) {
          const int64_t j = 0xfffffffeu - static_cast<uint32_t>(mine);
          top_ids[r * top_k + rank] = j;
          top_logprobs[r * top_k + rank] = to_f(row.p[j]) - a.m - logs;
        }
      }
    } else {
      // more than fit (many large values in few thread groups): one pass a place
      unsigned long long prev = ~0ull;
      for (int k = 0; k < top_k; ++k) {
        unsigned long long b = 0;
        for (int64_t j = tid; j < V; j += kThreads) {
          const unsigned long long key = key_of(to_f(row.p[j]), j);
          if (key < prev && key > b) b = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        __syncthreads();
        if (lane == 0) cand[warp] = b;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) b = max(b, cand[i]);
        prev = b;
        if (tid == 0) {
          const int64_t j = 0xfffffffeu - static_cast<uint32_t>(b);
          top_ids[r * top_k + k] = j;
          top_logprobs[r * top_k + k] = to_f(row.p[j]) - a.m - logs;
        }
      }
    }
  }
}

// One CTA a row: one read of the logits, one write of their gradient.
template <typename T, bool kEntropy, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    token_logprobs_backward_kernel(const T *x, int64_t rows, int64_t V, int64_t ld, const int64_t *targets,
                                   int64_t ignore_index, const float *stats, const float *g_logprobs,
                                   const float *g_entropy, T *dx, int64_t d_ld) {
  using namespace lp;
  constexpr int kN = Vec<T>::kN, kUnroll = 4;
  const int64_t r = blockIdx.x;
  const Row<T> row(x + r * ld, V);
  T *d = dx + r * d_ld;
  const int tid = threadIdx.x;
  const float m = stats[r], logs = stats[rows + r], h = stats[2 * rows + r];
  const int64_t t = targets[r];
  const float g = g_logprobs && t != ignore_index && t >= 0 && t < V ? g_logprobs[r] : 0.f;
  const float ge = kEntropy ? g_entropy[r] : 0.f;
  auto grad = [&](float v) {
    const float l = max_nan(v - m - logs, kFloor), p = ex2(l * kLog2e);
    return kEntropy ? -p * fmaf(ge, l + h, g) : -p * g;
  };
  auto one = [&](int64_t j) {
    float v = grad(to_f(row.p[j]));
    if (j == t) v += g;
    d[j] = from_f<T>(v);
  };
  if ((reinterpret_cast<uintptr_t>(d + row.head) & 15) != 0) {  // the two rows are aligned differently
    for (int64_t j = tid; j < V; j += kThreads) one(j);
    return;
  }
  if (tid < row.head) one(tid);
  if (row.tail + tid < V) one(row.tail + tid);
  const uint4 *body = row.body();
  uint4 *to = reinterpret_cast<uint4 *>(d + row.head);
  // the piece that holds the target, and the place in it
  const int64_t tv = t >= row.head && t < row.tail ? (t - row.head) / kN : -1;
  for (int64_t i = tid; i < row.vecs; i += kUnroll * kThreads) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < row.vecs) raw[u] = __ldg(body + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t at = i + u * kThreads;
      if (at >= row.vecs) continue;
      float y[kN];
      Vec<T>::unpack(raw[u], y);
#pragma unroll
      for (int e = 0; e < kN; ++e) y[e] = grad(y[e]);
      if (at == tv) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
          if (row.head + at * kN + e == t) y[e] += g;
      }
      uint4 out;
      T *p = reinterpret_cast<T *>(&out);
#pragma unroll
      for (int e = 0; e < kN; ++e) p[e] = from_f<T>(y[e]);
      __stcs(to + at, out);
    }
  }
}

}  // namespace sd

extern "C" {

int sd_token_logprobs(const void *logits, int dtype, int64_t rows, int64_t V, int64_t ld, const int64_t *targets,
                      int64_t ignore_index, float *logprobs, float *entropy, float *stats, int top_k,
                      float *top_logprobs, int64_t *top_ids, int32_t *err, void *stream) {
  using namespace sd;
  if (!logits || !targets || !logprobs || !dtype_ok(dtype) || rows <= 0 || V <= 0 || top_k < 0 || top_k > V ||
      (top_k > 0 && (!top_logprobs || !top_ids)) || ld < 0)
    return SD_ERR_INVALID;
  if (top_k > 64 || rows > 0x7fffffffll || V > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype)) return SD_ERR_ALIGN;
  SD_DISPATCH_DTYPE(dtype, T, {
    auto run = [&](auto *kern, int threads, size_t smem) {
      if (ensure_smem(kern, smem) != SD_OK) return static_cast<int>(SD_ERR_CUDA);
      kern<<<static_cast<unsigned>(rows), threads, smem, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T *>(logits), rows, V, ld, targets, ignore_index, logprobs, entropy, stats, top_k,
          top_logprobs, top_ids, err);
      return check_launch();
    };
    if (top_k > 0) return run(token_logprobs_kernel<T, true, 512>, 512, lp::kCandidates * sizeof(unsigned long long));
    return rows >= lp::kManyRows ? run(token_logprobs_kernel<T, false, 128>, 128, 0)
                                 : run(token_logprobs_kernel<T, false, 512>, 512, 0);
  });
  return SD_OK;
}

int sd_token_logprobs_backward(const void *logits, int dtype, int64_t rows, int64_t V, int64_t ld,
                               const int64_t *targets, int64_t ignore_index, const float *stats,
                               const float *g_logprobs, const float *g_entropy, void *dlogits, int64_t d_ld,
                               void *stream) {
  using namespace sd;
  if (!logits || !targets || !stats || !dlogits || !dtype_ok(dtype) || rows <= 0 || V <= 0 || ld < 0 || d_ld < V)
    return SD_ERR_INVALID;
  if (rows > 0x7fffffffll || V > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(logits) % dtype_size(dtype) ||
      reinterpret_cast<uintptr_t>(dlogits) % dtype_size(dtype))
    return SD_ERR_ALIGN;
  SD_DISPATCH_DTYPE(dtype, T, {
    const bool many = rows >= lp::kManyRows;
    auto kern = g_entropy ? many ? token_logprobs_backward_kernel<T, true, 256> : token_logprobs_backward_kernel<T, true, 512>
                : many    ? token_logprobs_backward_kernel<T, false, 256>
                          : token_logprobs_backward_kernel<T, false, 512>;
    kern<<<static_cast<unsigned>(rows), many ? 256 : 512, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T *>(logits), rows, V, ld, targets, ignore_index, stats, g_logprobs, g_entropy,
        static_cast<T *>(dlogits), d_ld);
  });
  return check_launch();
}

}  // extern "C"
