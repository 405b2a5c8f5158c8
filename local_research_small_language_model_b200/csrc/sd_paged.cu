// Paged key-value cache: the append, and the attention of one new token of
// every sequence over its pages.
//
// A pool holds pages of `page` tokens, k_pages and v_pages [P][Hkv][page][64]
// (any strides with an innermost one of 1).  Position t of sequence b lies in
// page table[b][t / page], row t % page.
#include "sd_common.cuh"

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

// One 16-byte chunk of K and of V a thread.  cu (nullable): token rows
// [cu[b], cu[b + 1]) belong to sequence b; without it row b is sequence b's
// one token.  Rows outside every sequence are not written anywhere.
template <typename T>
__global__ void __launch_bounds__(256)
    paged_append_kernel(PagedArgs a, const int32_t *cu, int64_t N, const T *xk, const T *xv, int64_t k_sn,
                        int64_t k_sh, int64_t v_sn, int64_t v_sh, T *k_pages, T *v_pages) {
  constexpr int kVec = 16 / sizeof(T), kChunks = 64 / kVec;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int c = static_cast<int>(e % kChunks) * kVec;
  const int h = static_cast<int>(e / kChunks % a.Hkv);
  const int64_t n = e / (kChunks * a.Hkv);
  if (n >= N) return;
  int b = static_cast<int>(n);
  int64_t t = 0;
  if (cu) {
    int lo = 0, hi = a.B;  // the last b with cu[b] <= n, if n < cu[b + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (cu[mid] <= n) lo = mid; else hi = mid;
    }
    b = lo;
    if (n < cu[b] || n >= cu[b + 1]) return;
    t = n - cu[b];
  }
  t += a.lens[b];
  if (t < 0 || t >= static_cast<int64_t>(a.width) * a.page) {
    pg::report(a.err, SD_KERR_BOUNDS);
    return;
  }
  const int64_t off = pg::row_of(a, b, h, static_cast<int>(t));
  if (off < 0) {
    pg::report(a.err, SD_KERR_BOUNDS);
    return;
  }
  *reinterpret_cast<uint4 *>(k_pages + off + c) = *reinterpret_cast<const uint4 *>(xk + n * k_sn + h * k_sh + c);
  *reinterpret_cast<uint4 *>(v_pages + off + c) = *reinterpret_cast<const uint4 *>(xv + n * v_sn + h * v_sh + c);
}

// One CTA of 128 threads per (sequence, kv head, 16 query heads of it).
template <typename T>
__global__ void __launch_bounds__(128)
    paged_decode_kernel(PagedArgs a, const T *q, int64_t q_sb, int64_t q_sh, const T *k_pages, const T *v_pages,
                        float scale_log2, T *out, int64_t o_sb, int64_t o_sh) {
  constexpr int kG = 16, kPitch = 68;
  __shared__ float sq[kG][64], sp[kG][64], sm_[kG], sl[kG], sa[kG];
  __shared__ float kv[64 * kPitch];
  const int b = blockIdx.z, hk = blockIdx.y, g0 = blockIdx.x * kG;
  const int group = a.Hq / a.Hkv, G = min(kG, group - g0), h0 = hk * group + g0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = pg::seq_len(a, b);
  for (int e = tid; e < G * 64; e += 128) sq[e >> 6][e & 63] = to_f(q[b * q_sb + (h0 + (e >> 6)) * q_sh + (e & 63)]);
  if (tid < kG) sm_[tid] = -INFINITY, sl[tid] = 0.f;
  float acc[kG] = {};
  for (int t0 = 0; t0 < len; t0 += 64) {
    const int n = min(64, len - t0);
    auto load = [&](const T *src) {
      constexpr int kVec = 16 / sizeof(T), kChunks = 64 / kVec;
      for (int e = tid; e < 64 * kChunks; e += 128) {
        const int r = e / kChunks, c = e % kChunks * kVec;
        const int64_t off = r < n ? pg::row_of(a, b, hk, t0 + r) : -1;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (off >= 0) raw = *reinterpret_cast<const uint4 *>(src + off + c);
        const T *p = reinterpret_cast<const T *>(&raw);
        for (int u = 0; u < kVec; ++u) kv[r * kPitch + c + u] = to_f(p[u]);
      }
    };
    __syncthreads();
    load(k_pages);
    __syncthreads();
    const int r = tid >> 1, d0 = (tid & 1) * 32;
    bool held = r < n;
    if (held && pg::row_of(a, b, hk, t0 + r) < 0) {
      pg::report(a.err, SD_KERR_BOUNDS);
      held = false;
    }
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
      for (int d = 0; d < 32; ++d) s = fmaf(sq[g][d0 + d], kv[r * kPitch + d0 + d], s);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      if (d0 == 0) sp[g][r] = held ? s * scale_log2 : -INFINITY;
    }
    __syncthreads();
    load(v_pages);
    for (int g = warp; g < G; g += 4) {
      const float s0 = sp[g][lane], s1 = sp[g][lane + 32];
      float mt = fmaxf(s0, s1);
      for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
      const float mn = fmaxf(sm_[g], mt), ref = mn == -INFINITY ? 0.f : mn;
      const float p0 = exp2f(s0 - ref), p1 = exp2f(s1 - ref);
      float ps = p0 + p1;
      for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      sp[g][lane] = p0, sp[g][lane + 32] = p1;
      __syncwarp();
      if (lane == 0) {
        sa[g] = exp2f(sm_[g] - ref);
        sl[g] = sl[g] * sa[g] + ps;
        sm_[g] = mn;
      }
    }
    __syncthreads();
    const int d = tid & 63, k0 = (tid >> 6) * 32;
    for (int g = 0; g < kG; ++g) {
      if (g >= G) break;
      float s = 0.f;
      for (int k = k0; k < k0 + 32; ++k) s = fmaf(sp[g][k], kv[k * kPitch + d], s);
      acc[g] = acc[g] * sa[g] + s;
    }
  }
  __syncthreads();
  for (int g = 0; g < kG; ++g)
    if (g < G) sp[g][tid & 63] = 0.f;
  __syncthreads();
  if (tid >= 64)
    for (int g = 0; g < kG; ++g)
      if (g < G) sp[g][tid & 63] = acc[g];
  __syncthreads();
  if (tid < 64)
    for (int g = 0; g < kG; ++g)
      if (g < G) {
        const float l = sl[g];
        // a sequence without tokens gives zeros
        out[b * o_sb + (h0 + g) * o_sh + tid] = from_f<T>(l == 0.f ? 0.f : (acc[g] + sp[g][tid]) / l);
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
  const int64_t threads = N * Hkv * (64 * size / 16);
  if ((threads + 255) / 256 > 0x7fffffffll) return SD_ERR_UNSUPPORTED;
  SD_DISPATCH_DTYPE(dtype, T, {
    paged_append_kernel<T><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        a, cu_seqlens, N, static_cast<const T *>(xk), static_cast<const T *>(xv), k_sn, k_sh, v_sn, v_sh,
        static_cast<T *>(k_pages), static_cast<T *>(v_pages));
  });
  return check_launch();
}

int sd_paged_decode_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t *bytes) {
  if (!bytes || B <= 0 || Hq <= 0 || Hkv <= 0) return SD_ERR_INVALID;
  *bytes = 0;
  return SD_OK;
}

int sd_paged_decode_attention(const void *q, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t q_sb,
                              int64_t q_sh, const void *k_pages, const void *v_pages, int64_t pages, int page,
                              int64_t p_sp, int64_t p_sh, int64_t p_st, const int32_t *table, int64_t t_sb,
                              int width, const int32_t *lens, float scale, void *out, int64_t o_sb, int64_t o_sh,
                              void *workspace, int64_t workspace_bytes, int32_t *err, void *stream) {
  using namespace sd;
  (void)workspace, (void)workspace_bytes;
  if (!q || !out || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || !(scale > 0.f) || scale > 3.0e38f)
    return SD_ERR_INVALID;
  if (B > 65535 || Hq > 65535) return SD_ERR_UNSUPPORTED;
  PagedArgs a = {table, t_sb, width, lens, static_cast<int>(B), static_cast<int>(Hq), static_cast<int>(Hkv), page,
                 pages, p_sp, p_sh, p_st, err};
  int rc = check_pool(a, dtype, D, k_pages, v_pages);
  if (rc != SD_OK) return rc;
  const int64_t size = dtype_size(dtype);
  if (!aligned16(q) || !aligned16(out) || (q_sb * size) % 16 || (q_sh * size) % 16 || (o_sb * size) % 16 ||
      (o_sh * size) % 16)
    return SD_ERR_ALIGN;
  const unsigned heads = static_cast<unsigned>((Hq / Hkv + 15) / 16);
  SD_DISPATCH_DTYPE(dtype, T, {
    paged_decode_kernel<T><<<dim3(heads, a.Hkv, a.B), 128, 0, static_cast<cudaStream_t>(stream)>>>(
        a, static_cast<const T *>(q), q_sb, q_sh, static_cast<const T *>(k_pages), static_cast<const T *>(v_pages),
        scale * 1.4426950408889634f, static_cast<T *>(out), o_sb, o_sh);
  });
  return check_launch();
}

}  // extern "C"
