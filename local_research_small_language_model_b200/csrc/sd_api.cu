// Library-wide entry points: error text, version, last CUDA error, length bump.
#include <math.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <type_traits>
#include <utility>

#include "sd_common.cuh"

namespace sd {

static thread_local int g_last_cuda_error = 0;
static std::atomic<int> g_pdl{0};

bool pdl_enabled() { return g_pdl.load(std::memory_order_relaxed) != 0; }

void set_cuda_error(cudaError_t e) { g_last_cuda_error = static_cast<int>(e); }

int check_launch() {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return SD_ERR_CUDA;
  }
  return SD_OK;
}

float inv_sqrt(int64_t d) { return static_cast<float>(1.0 / sqrt(static_cast<double>(d))); }

int set_max_smem_raw(const void *func, size_t bytes) {
  if (bytes <= 48 * 1024) return SD_OK;
  cudaError_t e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return SD_ERR_CUDA;
  }
  return SD_OK;
}

int ensure_smem_raw(const void *func, size_t bytes) {
  if (bytes <= 48 * 1024) return SD_OK;
  struct Limit {
    const void *func;
    int device;
    size_t bytes;
  };
  static std::mutex lock;
  static Limit limits[1024];  // no allocation: nothing may be thrown through a C entry point
  static int known = 0;
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    cudaGetLastError();
    return SD_ERR_CUDA;
  }
  std::lock_guard<std::mutex> hold(lock);
  Limit *at = nullptr;
  for (int i = 0; i < known && !at; ++i)
    if (limits[i].func == func && limits[i].device == device) at = &limits[i];
  if (at && at->bytes >= bytes) return SD_OK;
  const int rc = set_max_smem_raw(func, bytes);
  if (rc != SD_OK) return rc;
  if (at)
    at->bytes = bytes;
  else if (known < static_cast<int>(sizeof(limits) / sizeof(limits[0])))
    limits[known++] = {func, device, bytes};
  return SD_OK;
}

__global__ void advance_len_kernel(int32_t *lens, int n, int delta) {
  pdl_wait();
  int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) lens[i] += delta;
}

// One word of sd_invoke as an argument of type A.
template <typename A> static A from_word(int64_t word) {
  if constexpr (std::is_pointer<A>::value) {
    return reinterpret_cast<A>(static_cast<intptr_t>(word));
  } else if constexpr (std::is_same<A, float>::value) {
    double d;
    memcpy(&d, &word, sizeof(d));
    return static_cast<float>(d);
  } else {
    return static_cast<A>(word);
  }
}

template <typename... A, size_t... I>
static int call_words(int (*f)(A...), const int64_t *words, std::index_sequence<I...>) {
  return f(from_word<A>(words[I])...);
}
template <typename... A> static int invoke(int (*f)(A...), const int64_t *words, int n) {
  if (n != static_cast<int>(sizeof...(A))) return SD_ERR_INVALID;
  return call_words(f, words, std::index_sequence_for<A...>());
}

}  // namespace sd

extern "C" {

int sd_invoke(int call, const int64_t *words, int n) {
  if (!words) return SD_ERR_INVALID;
  switch (call) {
    case SD_CALL_PACKED_ATTENTION: return sd::invoke(sd_packed_attention, words, n);
    case SD_CALL_PACKED_ATTENTION_BACKWARD: return sd::invoke(sd_packed_attention_backward, words, n);
    case SD_CALL_PAGED_APPEND: return sd::invoke(sd_paged_append, words, n);
    case SD_CALL_PAGED_DECODE_ATTENTION: return sd::invoke(sd_paged_decode_attention, words, n);
    case SD_CALL_TOKEN_LOGPROBS: return sd::invoke(sd_token_logprobs, words, n);
    case SD_CALL_TOKEN_LOGPROBS_BACKWARD: return sd::invoke(sd_token_logprobs_backward, words, n);
    default: return SD_ERR_INVALID;
  }
}

const char *sd_strerror(int code) {
  switch (code) {
    case SD_OK: return "ok";
    case SD_ERR_INVALID: return "invalid argument (shape, stride, pointer or value)";
    case SD_ERR_UNSUPPORTED: return "unsupported configuration for the sm_100a kernels";
    case SD_ERR_CUDA: return "CUDA runtime error (see sd_last_cuda_error)";
    case SD_ERR_ALIGN: return "pointer or stride not 16-byte aligned as bulk copies require";
    default: return "unknown error";
  }
}

int sd_version(void) { return 1; }

int sd_last_cuda_error(void) { return sd::g_last_cuda_error; }

int sd_advance_len(int32_t *lens, int n, int delta, void *stream) {
  if (!lens || n <= 0) return SD_ERR_INVALID;
  return sd::launch(sd::advance_len_kernel, dim3((n + 127) / 128), dim3(128), 0, static_cast<cudaStream_t>(stream),
                    sd::pdl_enabled(), lens, n, delta);
}

int sd_set_programmatic_launch(int enable) { return sd::g_pdl.exchange(enable != 0 ? 1 : 0); }

}  // extern "C"
