// Penalties for repeated tokens, biases and a grammar mask on logits.
//
// One CTA takes a slice of one row's vocabulary: it counts in shared memory
// how often each token of the slice occurs in the row's history (integer
// atomics, so the order does not matter), then streams the slice through
// once. The row is read and written once, so HBM bounds it; the history is
// read once per slice, from L2 after the first.
#include <cuda_bf16.h>

#include "runtime.h"

namespace neso {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 8192;  // vocabulary entries per CTA: 32 KB of counts
// A count word: generated occurrences, and two flags.
constexpr uint32_t kSeen = 0x80000000u;    // the token occurs in the history
constexpr uint32_t kBiased = 0x40000000u;  // the token has a bias
constexpr uint32_t kCount = 0x3fffffffu;

struct LogitsParams {
  const void* in;
  void* out;
  const int32_t *history, *history_lens, *prompt_lens, *bias_ids, *mask;
  const float *repetition, *frequency, *presence, *bias;
  int64_t in_stride, out_stride, history_stride, mask_stride;
  int V, T, num_bias, slices;
};

template <typename T>
__device__ __forceinline__ float load_float(T x);
template <>
__device__ __forceinline__ float load_float<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float load_float<__half>(__half x) {
  return __half2float(x);
}
template <>
__device__ __forceinline__ float load_float<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T store_float(float x);
template <>
__device__ __forceinline__ float store_float<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half store_float<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 store_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Pack {
  T e[kVec];
};

template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) process_logits_kernel(const __grid_constant__ LogitsParams p) {
  __shared__ uint32_t counts[kSlice];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(p.in) + b * p.in_stride;
  T* out = static_cast<T*>(p.out) + b * p.out_stride;
  // Slices start on a vector boundary of the row's addresses; the first one
  // also holds the entries before it.
  const int head = kVec == 1 ? 0 : static_cast<int>((kVec - (reinterpret_cast<uintptr_t>(in) / sizeof(T)) % kVec) % kVec);
  const int body = kSlice - kVec;
  const int64_t begin = slice == 0 ? 0 : head + static_cast<int64_t>(slice) * body;
  const int64_t end = head + static_cast<int64_t>(slice + 1) * body;
  if (begin >= p.V) return;
  const int v0 = static_cast<int>(begin), v1 = static_cast<int>(end < p.V ? end : p.V);
  const uint32_t width = static_cast<uint32_t>(v1 - v0);

  for (uint32_t i = tid; i < width; i += kThreads) counts[i] = 0;
  __syncthreads();
  if (p.history != nullptr) {
    int n = p.history_lens[b];
    n = n < 0 ? 0 : (n > p.T ? p.T : n);
    const int prompt = p.prompt_lens != nullptr ? p.prompt_lens[b] : 0;
    const int32_t* ids = p.history + b * p.history_stride;
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t at = static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(v0);
      if (at < width) {
        if (i >= prompt) atomicAdd(&counts[at], 1u);
        atomicOr(&counts[at], kSeen);
      }
    }
  }
  if (p.bias_ids != nullptr) {
    for (int i = tid; i < p.num_bias; i += kThreads) {
      const uint32_t at = static_cast<uint32_t>(p.bias_ids[static_cast<int64_t>(b) * p.num_bias + i]) - static_cast<uint32_t>(v0);
      if (at < width) atomicOr(&counts[at], kBiased);
    }
  }
  __syncthreads();

  const float rep = p.repetition != nullptr ? p.repetition[b] : 1.f;
  const float freq = p.frequency != nullptr ? p.frequency[b] : 0.f;
  const float pres = p.presence != nullptr ? p.presence[b] : 0.f;
  const int32_t* mask = p.mask != nullptr ? p.mask + b * p.mask_stride : nullptr;
  auto one = [&](float x, int v) {
    const uint32_t c = counts[v - v0];
    if (c != 0) {
      if (c & kSeen) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      const uint32_t n = c & kCount;
      if (n != 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(n))), pres);
      if (c & kBiased) {
        for (int i = 0; i < p.num_bias; ++i) {
          const int64_t at = static_cast<int64_t>(b) * p.num_bias + i;
          if (p.bias_ids[at] == v) x = __fadd_rn(x, p.bias[at]);
        }
      }
    }
    if (mask != nullptr && !((static_cast<uint32_t>(mask[v >> 5]) >> (v & 31)) & 1u)) x = -INFINITY;
    return x;
  };
  const int va = slice == 0 ? (head < v1 ? head : v1) : v0;  // first vector
  for (int v = v0 + tid; v < va; v += kThreads) out[v] = store_float<T>(one(load_float<T>(in[v]), v));
  const int nvec = (v1 - va) / kVec;
  for (int i = tid; i < nvec; i += kThreads) {
    const int v = va + i * kVec;
    Pack<T, kVec> x = *reinterpret_cast<const Pack<T, kVec>*>(in + v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) x.e[e] = store_float<T>(one(load_float<T>(x.e[e]), v + e));
    *reinterpret_cast<Pack<T, kVec>*>(out + v) = x;
  }
  for (int v = va + nvec * kVec + tid; v < v1; v += kThreads) out[v] = store_float<T>(one(load_float<T>(in[v]), v));
}

template <typename T>
int launch_logits(LogitsParams p, int B, cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  // Vectors need rows of logits and out that lie the same way to 16 bytes.
  const uintptr_t diff = reinterpret_cast<uintptr_t>(p.in) - reinterpret_cast<uintptr_t>(p.out);
  const bool vec = diff % 16 == 0 && (B == 1 || (p.in_stride - p.out_stride) % kVec == 0);
  const int64_t body = kSlice - (vec ? kVec : 1);
  const int64_t slices = (p.V + body - 1) / body;
  if (slices * B > INT32_MAX) return fail(NESO_ERR_UNSUPPORTED, "batch x vocabulary is too large");
  p.slices = static_cast<int>(slices);
  const dim3 grid(static_cast<unsigned>(slices * B));
  cudaError_t e = vec ? launch_pdl(process_logits_kernel<T, kVec>, grid, dim3(kThreads), 0, stream, p)
                      : launch_pdl(process_logits_kernel<T, 1>, grid, dim3(kThreads), 0, stream, p);
  return e == cudaSuccess ? ok() : cuda_fail(e, "process_logits launch");
}

}  // namespace
}  // namespace neso

using namespace neso;

extern "C" int neso_process_logits(const void* logits, void* out, int32_t dtype, int32_t B, int32_t V,
                                   int64_t logits_stride, int64_t out_stride, const int32_t* history,
                                   const int32_t* history_lens, const int32_t* prompt_lens, int32_t T,
                                   int64_t history_stride, const float* repetition, const float* frequency,
                                   const float* presence, const int32_t* bias_ids, const float* bias, int32_t num_bias,
                                   const int32_t* mask, int64_t mask_stride, neso_stream_t stream) {
  if (dtype != NESO_F16 && dtype != NESO_BF16 && dtype != NESO_F32) {
    return fail(NESO_ERR_INVALID_ARG, "dtype must be f16, bf16 or f32");
  }
  if (B < 0 || V < 0 || T < 0 || num_bias < 0) return fail(NESO_ERR_INVALID_ARG, "negative size");
  if (T >= (1 << 30)) return fail(NESO_ERR_UNSUPPORTED, "history of 2^30 tokens or more");
  if (history != nullptr && history_lens == nullptr) return fail(NESO_ERR_INVALID_ARG, "history needs history_lens");
  if ((bias_ids != nullptr) != (bias != nullptr)) return fail(NESO_ERR_INVALID_ARG, "bias_ids and bias come together");
  if (B == 0 || V == 0) return ok();
  if (logits == nullptr || out == nullptr) return fail(NESO_ERR_INVALID_ARG, "null pointer");
  LogitsParams p{};
  p.in = logits;
  p.out = out;
  p.history = history;
  p.history_lens = history_lens;
  p.prompt_lens = prompt_lens;
  p.bias_ids = bias_ids;
  p.mask = mask;
  p.repetition = repetition;
  p.frequency = frequency;
  p.presence = presence;
  p.bias = bias;
  p.in_stride = logits_stride;
  p.out_stride = out_stride;
  p.history_stride = history_stride;
  p.mask_stride = mask_stride;
  p.V = V;
  p.T = T;
  p.num_bias = num_bias;
  if (dtype == NESO_F32) return launch_logits<float>(p, B, as_stream(stream));
  if (dtype == NESO_BF16) return launch_logits<__nv_bfloat16>(p, B, as_stream(stream));
  return launch_logits<__half>(p, B, as_stream(stream));
}
