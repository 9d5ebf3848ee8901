// Penalties for repeated tokens, biases and a grammar mask on logits.
//
// One CTA takes a slice of one row's vocabulary. Everything that it reads (the
// slice, its mask, the history's first tokens, the biases) is requested before
// the first wait. It counts in shared memory how often each token of the slice
// occurs in the row's history (integer atomics, so the order does not matter)
// and lists the tokens that it meets for the first time. The few listed ones
// are worked out one to a thread, because frequent tokens crowd in a few
// slices; the slice itself passes from registers to memory under the mask, and
// the listed values are written over it. The row is read and written once, so
// HBM bounds it; the history is read once per slice, from L2 after the first.
// 128 rows x 128257 fp32 with up to 4096 tokens of history, 16 biases and a mask
// take 32 us (4.2 TB/s; 24.6 without a history; bf16 27.5 and 18.4), one row of
// 32000 3.3.
#include <cuda_bf16.h>

#include "runtime.h"

namespace neso {
namespace {

// Vocabulary entries per thread and threads per CTA when the slices fill the
// SMs: long slices, because each reads the history once more (128 x 128257: 24 x
// 512 32.1 us, 24 x 256 32.3, 24 x 1024 35.7, 16 x 256 36-46). A few rows would
// leave most SMs idle: one vector a thread then (1 x 32000: 3.2 us, with slices
// of 8192 entries 8.9).
constexpr int kLong = 24, kLongThreads = 512;
constexpr int kShortThreads = 256;
constexpr int kMostThreads = 1024;  // per SM
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

// Entries a CTA covers: kPer per thread, less one vector for the entries before
// the first vector boundary, which the first slice takes as well.
template <int kVec, int kPer, int kThreads>
constexpr int slice_body() {
  return kThreads * kPer - kVec;
}

// Tokens 4 i .. 4 i + 3 of a row of T; -1 behind its end.
__device__ __forceinline__ int4 load_four(const int32_t* ids, int i, int T) {
  if (4 * i + 3 < T && (reinterpret_cast<uintptr_t>(ids) & 15u) == 0) return reinterpret_cast<const int4*>(ids)[i];
  int4 r = make_int4(-1, -1, -1, -1);
  if (4 * i < T) r.x = ids[4 * i];
  if (4 * i + 1 < T) r.y = ids[4 * i + 1];
  if (4 * i + 2 < T) r.z = ids[4 * i + 2];
  if (4 * i + 3 < T) r.w = ids[4 * i + 3];
  return r;
}

template <int kPer, int kThreads>
struct LogitsShared {
  alignas(16) uint32_t counts[kThreads * kPer];  // of entry v0 + i
  uint16_t listed[kThreads * kPer];              // entries with a count
  int num_listed;
  uint32_t allowed[kThreads + 1];  // mask words
  int32_t bias_id[kThreads];       // the row's first biases
  float bias_of[kThreads];
};

template <typename T, int kVec, int kPer, int kThreads>
__global__ void __launch_bounds__(kThreads, kMostThreads / kThreads)
    process_logits_kernel(const __grid_constant__ LogitsParams p) {
  constexpr int kBody = slice_body<kVec, kPer, kThreads>();
  constexpr int kVecs = kPer / kVec;
  static_assert(kPer <= 31, "a slice's mask words fit one per thread");
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sh = *reinterpret_cast<LogitsShared<kPer, kThreads>*>(smem);
  auto& counts = sh.counts;
  auto& listed = sh.listed;
  auto& allowed = sh.allowed;
  auto& bias_id = sh.bias_id;
  auto& bias_of = sh.bias_of;
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(p.in) + b * p.in_stride;
  T* out = static_cast<T*>(p.out) + b * p.out_stride;
  // Slices start on a vector boundary of the row's addresses; the first one
  // also holds the entries before it.
  const int head = kVec == 1 ? 0 : static_cast<int>((kVec - (reinterpret_cast<uintptr_t>(in) / sizeof(T)) % kVec) % kVec);
  const int64_t begin = head + static_cast<int64_t>(slice) * kBody;
  if (slice > 0 && begin >= p.V) return;
  const int va = static_cast<int>(begin < p.V ? begin : p.V);                  // first vector
  const int v0 = slice == 0 ? 0 : va;                                          // first entry
  const int v1 = static_cast<int>(begin + kBody < p.V ? begin + kBody : p.V);  // end
  const uint32_t width = static_cast<uint32_t>(v1 - v0);
  const int nvec = (v1 - va) / kVec;
  const int word0 = v0 >> 5;

  // Requests.
  int n = 0, prompt = 0;
  int4 id;  // four of the history's tokens
  const int32_t* ids = p.history + b * p.history_stride;
  if (p.history != nullptr) {
    n = p.history_lens[b];
    if (p.prompt_lens != nullptr) prompt = p.prompt_lens[b];
    id = load_four(ids, tid, p.T);
  }
  const int32_t* bias_ids = p.bias_ids + static_cast<int64_t>(b) * p.num_bias;
  const float* bias = p.bias + static_cast<int64_t>(b) * p.num_bias;
  int my_bias_id = -1;
  float my_bias = 0.f;
  if (tid < p.num_bias) {
    my_bias_id = bias_ids[tid];
    my_bias = bias[tid];
  }
  uint32_t my_word = 0xffffffffu;
  if (p.mask != nullptr && tid <= ((v1 - 1) >> 5) - word0) {
    my_word = static_cast<uint32_t>(p.mask[b * p.mask_stride + word0 + tid]);
  }
  const float rep = p.repetition != nullptr ? p.repetition[b] : 1.f;
  const float freq = p.frequency != nullptr ? p.frequency[b] : 0.f;
  const float pres = p.presence != nullptr ? p.presence[b] : 0.f;
  Pack<T, kVec> x[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    if (tid + i * kThreads < nvec) x[i] = *reinterpret_cast<const Pack<T, kVec>*>(in + va + (tid + i * kThreads) * kVec);
  }

  for (int i = tid; i < kThreads * kPer / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) sh.num_listed = 0;
  __syncthreads();
  auto list = [&](uint32_t before, uint32_t at) {
    if (before == 0) listed[atomicAdd(&sh.num_listed, 1)] = static_cast<uint16_t>(at);
  };
  if (p.history != nullptr) {
    n = n < 0 ? 0 : (n > p.T ? p.T : n);
    // Most fours hold no token of the slice: one comparison for all of them.
    auto count = [&](int4 four, int i) {
      uint32_t at[4] = {static_cast<uint32_t>(four.x) - static_cast<uint32_t>(v0),
                        static_cast<uint32_t>(four.y) - static_cast<uint32_t>(v0),
                        static_cast<uint32_t>(four.z) - static_cast<uint32_t>(v0),
                        static_cast<uint32_t>(four.w) - static_cast<uint32_t>(v0)};
      if (min(min(at[0], at[1]), min(at[2], at[3])) >= width) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (at[e] < width && 4 * i + e < n) {
          list(4 * i + e >= prompt ? atomicAdd(&counts[at[e]], 1u) : atomicOr(&counts[at[e]], kSeen), at[e]);
        }
      }
    };
    for (int i = tid; 4 * i < n; i += kThreads) {
      if (i != tid) id = load_four(ids, i, p.T);
      count(id, i);
    }
  }
  for (int i = tid; i < p.num_bias; i += kThreads) {
    const uint32_t at = static_cast<uint32_t>(i < kThreads ? my_bias_id : bias_ids[i]) - static_cast<uint32_t>(v0);
    if (at < width) list(atomicOr(&counts[at], kBiased), at);
  }
  bias_id[tid] = my_bias_id;
  bias_of[tid] = my_bias;
  allowed[tid] = my_word;
  __syncthreads();

  // Mask bits of the entries from v on, as many as a vector has.
  auto bits = [&](int v) {
    if (p.mask == nullptr) return 0xffffffffu;
    const int w = (v >> 5) - word0;
    return __funnelshift_r(allowed[w], allowed[w + 1], v & 31);
  };
  const int n_listed = sh.num_listed;
  for (int i = tid; i < n_listed; i += kThreads) {
    const int at = listed[i], v = v0 + at;
    const uint32_t c = counts[at], times = c & kCount;
    float y = load_float<T>(in[v]);
    if (c & (kSeen | kCount)) y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
    if (times != 0) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(times))), pres);
    if (c & kBiased) {
      const int near = p.num_bias < kThreads ? p.num_bias : kThreads;
      for (int j = 0; j < near; ++j) {
        if (bias_id[j] == v) y = __fadd_rn(y, bias_of[j]);
      }
      for (int j = near; j < p.num_bias; ++j) {
        if (bias_ids[j] == v) y = __fadd_rn(y, bias[j]);
      }
    }
    counts[at] = __float_as_uint((bits(v) & 1u) ? y : -INFINITY);  // in the place of its count
  }
  if (p.in == p.out) __syncthreads();  // the listed logits have been read
  // The slice: vectors, and the ragged ends before the first and behind the last.
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int j = tid + i * kThreads;
    if (j < nvec) {
      const int v = va + j * kVec;
      const uint32_t allow = bits(v);
      Pack<T, kVec> y = x[i];
#pragma unroll
      for (int e = 0; e < kVec; ++e) y.e[e] = ((allow >> e) & 1u) ? y.e[e] : store_float<T>(-INFINITY);
      *reinterpret_cast<Pack<T, kVec>*>(out + v) = y;
    }
  }
  const int tail = va + nvec * kVec;
  const int ragged = (va - v0) + (v1 - tail);
  for (int i = tid; i < ragged; i += kThreads) {
    const int v = i < va - v0 ? v0 + i : tail + (i - (va - v0));
    out[v] = (bits(v) & 1u) ? in[v] : store_float<T>(-INFINITY);
  }
  if (n_listed == 0) return;
  __syncthreads();
  for (int i = tid; i < n_listed; i += kThreads) {
    const int at = listed[i];
    out[v0 + at] = store_float<T>(__uint_as_float(counts[at]));
  }
}

template <typename T, int kVec, int kPer, int kThreads>
int launch_slices(LogitsParams p, int B, cudaStream_t stream) {
  constexpr int kBody = slice_body<kVec, kPer, kThreads>();
  constexpr int kSmem = static_cast<int>(sizeof(LogitsShared<kPer, kThreads>));
  const int64_t slices = (static_cast<int64_t>(p.V) + kBody - 1) / kBody;
  if (slices * B > INT32_MAX) return fail(NESO_ERR_UNSUPPORTED, "batch x vocabulary is too large");
  p.slices = static_cast<int>(slices);
  auto* kern = process_logits_kernel<T, kVec, kPer, kThreads>;
  const int rc = kernel_setup(reinterpret_cast<const void*>(kern), kSmem, nullptr);
  if (rc != NESO_OK) return rc;
  cudaError_t e = launch_pdl(kern, dim3(static_cast<unsigned>(slices * B)), dim3(kThreads), kSmem, stream, p);
  return e == cudaSuccess ? ok() : cuda_fail(e, "process_logits launch");
}

template <typename T>
int launch_logits(const LogitsParams& p, int B, cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  // Vectors need rows of logits and out that lie the same way to 16 bytes.
  const uintptr_t diff = reinterpret_cast<uintptr_t>(p.in) - reinterpret_cast<uintptr_t>(p.out);
  const bool vec = diff % 16 == 0 && (B == 1 || (p.in_stride - p.out_stride) % kVec == 0);
  const int64_t entries = static_cast<int64_t>(B) * p.V;
  const bool few = entries < static_cast<int64_t>(sm_count()) * kLong * kLongThreads;
  if (!vec) {
    return few ? launch_slices<T, 1, 4, kShortThreads>(p, B, stream) : launch_slices<T, 1, kLong, kLongThreads>(p, B, stream);
  }
  return few ? launch_slices<T, kVec, kVec, kShortThreads>(p, B, stream)
             : launch_slices<T, kVec, kLong, kLongThreads>(p, B, stream);
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
  p.num_bias = bias != nullptr ? num_bias : 0;
  if (dtype == NESO_F32) return launch_logits<float>(p, B, as_stream(stream));
  if (dtype == NESO_BF16) return launch_logits<__nv_bfloat16>(p, B, as_stream(stream));
  return launch_logits<__half>(p, B, as_stream(stream));
}
