// Log probabilities of given tokens with the distribution's entropy and its
// likeliest tokens, and the gradient of the logits.
//
//   m = max x,  s = sum exp(x - m),  w = sum exp(x - m) (x - m)
//   log p_j = x_j - m - log s,   H = log s - w / s
//   d/dx_j (g log p_t + h H) = g [j = t] - p_j (g + h (log p_j + H))
//
// m, s and w come from one pass over the row (s and w are rescaled when m
// rises), in fp32.  A logit of -inf has probability 0 and adds nothing; a row
// with a NaN, a +inf or nothing but -inf has NaN results, as log_softmax.
#include "sd_common.cuh"

namespace sd {

namespace lp {

constexpr int kThreads = 256;

struct Stat {
  float m, s, w;
};

__device__ __forceinline__ void add(Stat &a, float x) {
  if (x == -INFINITY) return;
  if (x > a.m) {
    const float c = a.m == -INFINITY ? 0.f : __expf(a.m - x);
    a.w = a.m == -INFINITY ? 0.f : c * (a.w + a.s * (a.m - x));
    a.s *= c;
    a.m = x;
  }
  const float d = x - a.m, e = __expf(d);
  a.s += e;
  a.w = fmaf(e, d, a.w);
}

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  if (b.m > a.m) {
    const Stat t = a;
    a = b;
    b = t;
  }
  if (b.m == -INFINITY) {  // an empty part (s = w = 0), or one that holds NaN only
    a.s += b.s;
    return a;
  }
  const float d = b.m - a.m, c = d == 0.f ? 1.f : __expf(d);
  a.s += c * b.s;
  a.w += c * (b.w + b.s * d);
  return a;
}

// A float's place in the order NaN > +inf > ... > -inf, with -0 = +0.
__device__ __forceinline__ uint32_t place(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

}  // namespace lp

// stats [3][rows]: m, log s, H (kept for the gradient).
template <typename T>
__global__ void __launch_bounds__(lp::kThreads)
    token_logprobs_kernel(const T *x, int64_t rows, int64_t V, int64_t ld, const int64_t *targets,
                          int64_t ignore_index, float *logprobs, float *entropy, float *stats, int top_k,
                          float *top_logprobs, int64_t *top_ids, int32_t *err) {
  using namespace lp;
  __shared__ Stat part[kThreads / 32];
  __shared__ unsigned long long best[kThreads / 32];
  const int64_t r = blockIdx.x;
  const T *row = x + r * ld;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Stat a = {-INFINITY, 0.f, 0.f};
  for (int64_t j = tid; j < V; j += kThreads) add(a, to_f(row[j]));
  for (int o = 16; o > 0; o >>= 1) {
    Stat b = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
              __shfl_xor_sync(0xffffffffu, a.w, o)};
    a = join(a, b);
  }
  if (lane == 0) part[warp] = a;
  __syncthreads();
  a = part[0];
  for (int i = 1; i < kThreads / 32; ++i) a = join(a, part[i]);
  const float logs = logf(a.s);
  if (tid == 0) {
    const float h = logs - a.w / a.s;
    const int64_t t = targets[r];
    float v = 0.f;
    if (t != ignore_index) {
      if (t >= 0 && t < V) {
        v = to_f(row[t]) - a.m - logs;
      } else {
        v = __int_as_float(0x7fc00000);
        if (err) *err = SD_KERR_BOUNDS;
      }
    }
    logprobs[r] = v;
    if (entropy) entropy[r] = h;
    if (stats) stats[r] = a.m, stats[rows + r] = logs, stats[2 * rows + r] = h;
  }
  unsigned long long prev = ~0ull;
  for (int k = 0; k < top_k; ++k) {
    unsigned long long b = 0;
    for (int64_t j = tid; j < V; j += kThreads) {
      const unsigned long long key =
          static_cast<unsigned long long>(place(to_f(row[j]))) << 32 | (0xfffffffeu - static_cast<uint32_t>(j));
      if (key < prev && key > b) b = key;
    }
    for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    for (int i = 0; i < kThreads / 32; ++i) b = max(b, best[i]);
    prev = b;
    if (tid == 0) {
      const int64_t j = 0xfffffffeu - static_cast<uint32_t>(b);
      top_ids[r * top_k + k] = j;
      top_logprobs[r * top_k + k] = to_f(row[j]) - a.m - logs;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(lp::kThreads)
    token_logprobs_backward_kernel(const T *x, int64_t rows, int64_t V, int64_t ld, const int64_t *targets,
                                   int64_t ignore_index, const float *stats, const float *g_logprobs,
                                   const float *g_entropy, T *dx, int64_t d_ld) {
  const int64_t r = blockIdx.x;
  const T *row = x + r * ld;
  T *d = dx + r * d_ld;
  const float m = stats[r], logs = stats[rows + r], h = stats[2 * rows + r];
  const int64_t t = targets[r];
  const float g = g_logprobs && t != ignore_index && t >= 0 && t < V ? g_logprobs[r] : 0.f;
  const float ge = g_entropy ? g_entropy[r] : 0.f;
  for (int64_t j = threadIdx.x; j < V; j += lp::kThreads) {
    const float l = to_f(row[j]) - m - logs, p = __expf(l);
    float v = j == t ? g : 0.f;
    v -= p * g;
    if (ge != 0.f && p > 0.f) v -= p * (ge * (l + h));
    d[j] = from_f<T>(v);
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
  SD_DISPATCH_DTYPE(dtype, T, {
    token_logprobs_kernel<T><<<static_cast<unsigned>(rows), lp::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const T *>(logits), rows, V, ld, targets, ignore_index, logprobs, entropy, stats, top_k,
        top_logprobs, top_ids, err);
  });
  return check_launch();
}

int sd_token_logprobs_backward(const void *logits, int dtype, int64_t rows, int64_t V, int64_t ld,
                               const int64_t *targets, int64_t ignore_index, const float *stats,
                               const float *g_logprobs, const float *g_entropy, void *dlogits, int64_t d_ld,
                               void *stream) {
  using namespace sd;
  if (!logits || !targets || !stats || !dlogits || !dtype_ok(dtype) || rows <= 0 || V <= 0 || ld < 0 || d_ld < V)
    return SD_ERR_INVALID;
  if (rows > 0x7fffffffll || V > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  SD_DISPATCH_DTYPE(dtype, T, {
    token_logprobs_backward_kernel<T>
        <<<static_cast<unsigned>(rows), lp::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T *>(logits), rows, V, ld, targets, ignore_index, stats, g_logprobs, g_entropy,
            static_cast<T *>(dlogits), d_ld);
  });
  return check_launch();
}

}  // extern "C"
