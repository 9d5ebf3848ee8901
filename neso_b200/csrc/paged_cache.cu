// Writing to and trimming the paged key-value cache.
//
// rope_paged_append: new tokens' queries and keys are rotated in fp32 (products
// and sums rounded separately, then once to 16 bits) and keys and values go to
// their slots. One pass: every input byte is read once and every output byte
// written once, so HBM bounds it (launch latency for a few tokens): 8192 tokens
// of 32 + 8 + 8 heads x 128 in 37.0 us, 5.6 TB/s read and written.
//
// kv_evict, first kernel: for each (sequence, kv head) the kept set is found by
// a radix selection on the weights' bits. Up to kShortLen tokens one CTA does
// it in registers and shared memory (a cluster's common count costs two cluster
// barriers a digit: 66 us for the case below when every length took it, 43.6
// without); longer sequences are counted by a cluster through its shared memory.
// Second kernel: the kept rows move together, in order. Under a table of their
// own they move independently of each other. In place, a cluster moves the rows
// of one (sequence, kv head) a step at a time: row j comes from row src_j >= j,
// so when all rows of a step are in shared memory (a cluster barrier), the rows
// that it overwrites are not the source of any later step, and later steps may
// already be on their way in. 8 sequences x 8 heads of up to 4096 tokens to
// 2048, D = 128: 34.3 us under a table of their own, of which the rows take 22.3
// (6 TB/s read and written, as a plain copy) and the selection the rest; 44.1 in
// place, a cluster barrier per step.
#include <cooperative_groups.h>

#include "paged.h"

namespace neso {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxAxes = 4;

struct RopeParams {
  const uint16_t *q, *k, *v;
  const float *cos, *sin;
  const int32_t* positions;  // [axes, N]
  const int64_t* slots;      // [N]
  uint16_t* q_out;           // [N, hq, D]
  PagedCache kc, vc;
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, slot_count;
  int N, hq, hkv, D, half, table_rows, axes;
  int section_end[kMaxAxes];
  int group;  // tokens per CTA
  PageDivisor page, per_head, heads;  // heads: of q, k and v
};

template <bool kBf16>
__device__ __forceinline__ float to_float(uint16_t x) {
  if (kBf16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  return __half2float(__ushort_as_half(x));
}
template <bool kBf16>
__device__ __forceinline__ uint16_t from_float(float x) {
  if (kBf16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

template <int N>
struct alignas(N == 8 ? 16 : 2) Vec {
  uint16_t e[N];
};

// Where the angle of pair d lies among `half` of them. Vectors of eight keep the
// first fours of all columns, then the second ones, so that neighbouring lanes
// read neighbouring float4.
template <int kVec>
__device__ __forceinline__ int angle_place(int d, int half) {
  return kVec == 8 ? (d & 4) * (half >> 3) + (d >> 3) * 4 + (d & 3) : d;
}
template <int N>
__device__ __forceinline__ Vec<N> load_vec(const uint16_t* p) {
  Vec<N> r;
  if (N == 8) {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  } else {
    r.e[0] = *p;
  }
  return r;
}
template <int N>
__device__ __forceinline__ void store_vec(uint16_t* p, const Vec<N>& r) {
  if (N == 8) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  } else {
    *p = r.e[0];
  }
}

constexpr int kRopeTokens = 2;   // tokens per CTA when there are many
constexpr int kMaxRopeDim = 1024;

// kThreads per CTA, kBatch items requested at a time by each. Many tokens run
// fastest in small CTAs with few registers (8192 tokens of 48 heads x 128: 128
// threads, 2 items, 2 tokens 37.2 us; 256, 3, 4 41.7; 128, 3, 2 38.7; 64, 3, 1
// 38.7), few tokens with a CTA for each that requests all its items at once (187 tokens: 256
// threads, 3 items 4.4 us; 128, 2 5.0).
// A CTA takes p.group tokens. Every head of q, k and v is D / (2 kVec) items
// of two vectors: a rotated pair, or two that are copied (the rest of a
// rotated head, and values). The first items are requested before the chain
// position -> angles, which is walked once per CTA into shared memory.
template <bool kBf16, int kVec, int kThreads, int kBatch>
__global__ void __launch_bounds__(kThreads) rope_paged_append_kernel(const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float angles[];  // [group][2][half]
  __shared__ int64_t places[kRopeTokens][2];        // element offsets in k_cache and v_cache, or -1
  const int tid = threadIdx.x;
  const int n0 = blockIdx.x * p.group;
  const int tokens = min(p.group, p.N - n0);
  const int rotated = p.hq + p.hkv, heads = rotated + p.hkv;
  const int per_head = p.D / (2 * kVec);
  const int items = tokens * heads * per_head;
  pdl_launch_dependents();
  pdl_wait();

  struct Item {
    int n, h, d, second;  // token, head, first element, distance of the second
    bool turned;
  };
  auto item_at = [&](int i) {
    Item it;
    const int hn = static_cast<int>(page_of(p.per_head, i));
    const int c = i - hn * per_head;
    it.n = static_cast<int>(page_of(p.heads, hn));
    it.h = hn - it.n * heads;
    const int turn = it.h < rotated ? p.half : 0;  // pairs that turn
    it.turned = c * kVec < turn;
    it.d = it.turned ? c * kVec : c * kVec + turn;
    it.second = it.turned ? p.half : p.D / 2 - turn;
    return it;
  };
  auto source = [&](const Item& it) {
    const int64_t n = n0 + it.n;
    if (it.h < p.hq) return p.q + n * p.q_sn + it.h * p.q_sh + it.d;
    if (it.h < rotated) return p.k + n * p.k_sn + (it.h - p.hq) * p.k_sh + it.d;
    return p.v + n * p.v_sn + (it.h - rotated) * p.v_sh + it.d;
  };
  Vec<kVec> x[kBatch], y[kBatch];
  auto request = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kThreads;
      if (i < items) {
        const Item it = item_at(i);
        const uint16_t* src = source(it);
        x[j] = load_vec<kVec>(src);
        y[j] = load_vec<kVec>(src + it.second);
      }
    }
  };
  request(tid);

  if (tid < tokens) {
    const int64_t slot = p.slots[n0 + tid];
    int64_t ko = -1, vo = -1;
    if (slot >= 0 && slot < p.slot_count) {
      const int64_t page = p.slot_count <= INT32_MAX ? static_cast<int64_t>(page_of(p.page, static_cast<uint32_t>(slot)))
                                                     : slot / p.page.size;
      const int64_t row = slot - page * p.page.size;
      ko = page * p.kc.page_stride + row * p.kc.token_stride;
      vo = page * p.vc.page_stride + row * p.vc.token_stride;
    }
    places[tid][0] = ko;
    places[tid][1] = vo;
  }
  for (int i = tid; i < tokens * p.half; i += kThreads) {
    const int n = i / p.half, d = i - n * p.half;
    int axis = 0;
    while (axis < p.axes - 1 && d >= p.section_end[axis]) ++axis;
    const int pos = p.positions[static_cast<int64_t>(axis) * p.N + n0 + n];
    const bool in = pos >= 0 && pos < p.table_rows;
    const int64_t row = static_cast<int64_t>(pos) * p.half + d;
    const int place = 2 * n * p.half + angle_place<kVec>(d, p.half);
    angles[place] = in ? p.cos[row] : __int_as_float(0x7fc00000);
    angles[place + p.half] = in ? p.sin[row] : __int_as_float(0x7fc00000);
  }
  __syncthreads();

  for (int i0 = tid; i0 < items; i0 += kBatch * kThreads) {
    if (i0 != tid) request(i0);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kThreads;
      if (i >= items) break;
      const Item it = item_at(i);  // again: kept, it costs registers and 39.8 us
      const int64_t ko = places[it.n][0], vo = places[it.n][1];
      uint16_t* dst;
      if (it.h < p.hq) {
        dst = p.q_out + (static_cast<int64_t>(n0 + it.n) * p.hq + it.h) * p.D + it.d;
        if (ko < 0) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[j].e[e] = y[j].e[e] = 0;
        }
      } else {
        if (ko < 0) continue;
        dst = it.h < rotated ? static_cast<uint16_t*>(p.kc.base) + ko + (it.h - p.hq) * p.kc.head_stride + it.d
                             : static_cast<uint16_t*>(p.vc.base) + vo + (it.h - rotated) * p.vc.head_stride + it.d;
      }
      if (it.turned && ko >= 0) {
        const float* cs = angles + 2 * it.n * p.half + angle_place<kVec>(it.d, p.half);
        if (kVec == 8) {
          uint32_t* xw = reinterpret_cast<uint32_t*>(&x[j]);
          uint32_t* yw = reinterpret_cast<uint32_t*>(&y[j]);
#pragma unroll
          for (int q4 = 0; q4 < 2; ++q4) {
            const float4 c4 = *reinterpret_cast<const float4*>(cs + q4 * (p.half / 2));
            const float4 s4 = *reinterpret_cast<const float4*>(cs + p.half + q4 * (p.half / 2));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 u = unpack16<kBf16>(xw[2 * q4 + e]), w = unpack16<kBf16>(yw[2 * q4 + e]);
              const float c0 = e ? c4.z : c4.x, c1 = e ? c4.w : c4.y, s0 = e ? s4.z : s4.x, s1 = e ? s4.w : s4.y;
              xw[2 * q4 + e] = pack16<kBf16>(__fsub_rn(__fmul_rn(u.x, c0), __fmul_rn(w.x, s0)),
                                             __fsub_rn(__fmul_rn(u.y, c1), __fmul_rn(w.y, s1)));
              yw[2 * q4 + e] = pack16<kBf16>(__fadd_rn(__fmul_rn(u.x, s0), __fmul_rn(w.x, c0)),
                                             __fadd_rn(__fmul_rn(u.y, s1), __fmul_rn(w.y, c1)));
            }
          }
        } else {
          const float u = to_float<kBf16>(x[j].e[0]), w = to_float<kBf16>(y[j].e[0]);
          x[j].e[0] = from_float<kBf16>(__fsub_rn(__fmul_rn(u, cs[0]), __fmul_rn(w, cs[p.half])));
          y[j].e[0] = from_float<kBf16>(__fadd_rn(__fmul_rn(u, cs[p.half]), __fmul_rn(w, cs[0])));
        }
      }
      store_vec<kVec>(dst, x[j]);
      store_vec<kVec>(dst + it.second, y[j]);
    }
  }
}

template <bool kBf16, int kVec>
int launch_rope(RopeParams p, cudaStream_t stream) {
  const bool many = p.N >= 8 * sm_count();
  p.group = many ? kRopeTokens : 1;
  p.per_head = page_divisor(static_cast<uint32_t>(p.D / (2 * kVec)));
  const unsigned grid = static_cast<unsigned>((p.N + p.group - 1) / p.group);
  const size_t smem = static_cast<size_t>(p.group) * 2 * p.half * sizeof(float);
  cudaError_t e = many ? launch_pdl(rope_paged_append_kernel<kBf16, kVec, 128, 2>, dim3(grid), dim3(128), smem, stream, p)
                       : launch_pdl(rope_paged_append_kernel<kBf16, kVec, 256, 3>, dim3(grid), dim3(256), smem, stream, p);
  return e == cudaSuccess ? ok() : cuda_fail(e, "rope_paged_append launch");
}

// ------------------------------------------------------------------- evict --
struct EvictParams {
  PagedCache k, v;
  const int32_t *tables, *out_tables, *lens;
  const float* win;
  float* wout;
  int32_t *kept, *new_lens;
  int64_t table_stride, out_stride, win_sb, win_sh, wout_sb, wout_sh;
  int hkv, D, budget, recent, sink, num_pages, capacity, out_capacity;
  int row_shift;  // log2 of the pieces of a K row and a V row, or -1
  PageDivisor page;
};

// Threads of a CTA that selects: 1024 where the tables hold more than
// kSmallTable tokens, 512 otherwise (64 sequences of up to 4096 tokens: 34.6
// against 37.2 us for the whole eviction; 8 of 1023: 11.8 against 10.3).
constexpr int kSmallTable = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMostTokens = 1 << 30;
constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kCopiesOfHist = 8;   // counters of a digit, so that equal digits of a warp collide less
constexpr int kHistPitch = kDigits + 1;
constexpr int kShortLen = 8192;    // tokens of a short sequence
constexpr int kMoveThreads = 512;
constexpr int kMoveStages = 4;     // steps of rows in flight, one 16-byte piece per thread and cache each
constexpr int kMoveBytes = kMoveStages * 2 * kMoveThreads * 16;

// Larger weights get larger keys; NaN the largest; -0 and +0 the same key.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Execution barrier of the cluster that does not wait for stores on their way
// to memory (the ordinary one does, microseconds at a time): for steps whose
// loads have completed and whose stores nobody reads.
__device__ __forceinline__ void cluster_barrier_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

struct EvictShared {
  int hist[2][kCopiesOfHist * kHistPitch];
  alignas(16) int total[kDigits];
  int warp_sum[2][32];
  int slice[2];  // long sequences: kept for sure and ties of this CTA's slice
};
// Short sequences, dynamic shared memory: the weights (padded), then the kept
// tokens and their weights.
constexpr int kPadded = kShortLen + kShortLen / 16;
constexpr int kSelectBytes = (kPadded + kShortLen) * 4;

// Count this thread's digit, in its copy of the histogram.
__device__ __forceinline__ void count_digit(int* hist, uint32_t key, uint32_t prefix, int shift) {
  if (shift == 32 - kDigitBits || ((key ^ prefix) >> (shift + kDigitBits)) == 0) {
    atomicAdd(&hist[(threadIdx.x % kCopiesOfHist) * kHistPitch + ((key >> shift) & (kDigits - 1))], 1);
  }
}

// The digit that holds the need-th largest key, how many of its keys are wanted
// and how many it has. Every warp works it out for itself.
struct Pick {
  int digit, wanted, has;
};
__device__ __forceinline__ Pick pick_digit(const int* total, int need) {
  constexpr int kPer = kDigits / 32;
  const int lane = threadIdx.x & 31;
  int of[kPer];  // digits from the largest down, kPer to a lane
  int mine = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    of[j] = total[kDigits - 1 - (lane * kPer + j)];
    mine += of[j];
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  const uint32_t reached = __ballot_sync(0xffffffffu, need <= incl);
  int before = incl - mine;
  Pick pick{0, 0, 0};
  bool found = false;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (!found && before + of[j] >= need) {
      pick = Pick{kDigits - 1 - (lane * kPer + j), need - before, of[j]};
      found = true;
    }
    before += of[j];
  }
  const int src = __ffs(reached) - 1;
  return Pick{__shfl_sync(0xffffffffu, pick.digit, src), __shfl_sync(0xffffffffu, pick.wanted, src),
              __shfl_sync(0xffffffffu, pick.has, src)};
}

// What a selection found: keys above `bound` are kept, and the first `ties`
// tokens whose key equals it.
struct Selected {
  uint32_t bound;
  int ties;
};

template <int kEvictThreads>
__global__ void __launch_bounds__(kEvictThreads, 1024 / kEvictThreads)
    kv_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int kEvictWarps = kEvictThreads / 32;
  constexpr int kItems = kShortLen / kEvictThreads;  // tokens per thread of a short sequence
  __shared__ EvictShared sh;
  extern __shared__ __align__(16) int lists[];
  int* list = lists;
  int* kept_bits = lists + kPadded;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int seg = blockIdx.x / ctas;
  const int b = seg / p.hkv, h = seg % p.hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  auto sync_cluster = [&] {
    if (ctas > 1) {
      cluster.sync();
    } else {
      __syncthreads();
    }
  };

  const float* win = p.win + b * p.win_sb + h * p.win_sh;
  // A short sequence's weights are requested along with its length.
  float early[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int t = i * kEvictThreads + tid;
    early[i] = rank == 0 && t < p.capacity ? win[t] : 0.f;
  }
  int len = p.lens[b];
  len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
  const int keep = len < p.budget ? len : p.budget;
  float* wout = p.wout + b * p.wout_sb + h * p.wout_sh;
  int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  // Candidates [lo, hi) are ranked; tokens outside are kept.
  const bool all = len <= p.budget;
  const int lo = all ? 0 : p.sink, hi = all ? 0 : len - p.recent;
  const int wanted = all ? 0 : keep - p.sink - p.recent;  // candidates to keep
  const bool is_short = len <= kShortLen;

  if (is_short) {
    if (rank > 0) return;
    // Thread i takes tokens [i * items, (i + 1) * items), through shared
    // memory (one word of padding after 16) so that the loads are coalesced.
    const int items = (len + kEvictThreads - 1) / kEvictThreads;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = i * kEvictThreads + tid;
      if (i >= items) break;
      if (t < len) list[t + (t >> 4)] = __float_as_int(early[i]);
    }
    for (int i = tid; i < 2 * kCopiesOfHist * kHistPitch; i += kEvictThreads) sh.hist[0][i] = 0;
    __syncthreads();
    int bits[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = tid * items + i;
      if (i >= items) break;
      bits[i] = t < len ? list[t + (t >> 4)] : 0;
    }
    auto key_of = [&](int i) { return weight_key(__int_as_float(bits[i])); };
    Selected sel{0xffffffffu, 0};
    if (wanted > 0) {
      uint32_t prefix = 0;
      int need = wanted;
      for (int shift = 32 - kDigitBits, pass = 0; shift >= 0; shift -= kDigitBits, ++pass) {
        int* hist = sh.hist[pass & 1];
        int* next = sh.hist[~pass & 1];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int t = tid * items + i;
          if (i >= items) break;
          if (t >= lo && t < hi) count_digit(hist, key_of(i), prefix, shift);
        }
        __syncthreads();
        if (tid < kDigits) {
          int sum = 0;
#pragma unroll
          for (int c = 0; c < kCopiesOfHist; ++c) sum += hist[c * kHistPitch + tid];
          sh.total[tid] = sum;
        } else if (pass > 0) {
          for (int i = tid - kDigits; i < kCopiesOfHist * kHistPitch; i += kEvictThreads - kDigits) next[i] = 0;
        }
        __syncthreads();
        const Pick pick = pick_digit(sh.total, need);
        prefix |= static_cast<uint32_t>(pick.digit) << shift;
        need = pick.wanted;
        if (need == pick.has) {
          // Every key of this digit is wanted: the ones from prefix up. (prefix
          // is not 0: then all candidates would be kept.)
          prefix -= 1;
          need = 0;
          break;
        }
      }
      sel = Selected{prefix, need};
    }
    // Ranks: kept-for-sure tokens in the low half, ties in the high half.
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = tid * items + i;
      if (i >= items) break;
      if (t < len) {
        const bool in = t >= lo && t < hi;
        mine += (!in || (wanted > 0 && key_of(i) > sel.bound)) ? 1u : 0u;
        mine += (in && sel.ties > 0 && key_of(i) == sel.bound) ? 0x10000u : 0u;
      }
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) sh.warp_sum[0][warp] = static_cast<int>(incl);
    __syncthreads();  // also: every weight is in registers, list may be overwritten
    uint32_t at = incl - mine;
#pragma unroll
    for (int i = 0; i < kEvictWarps; ++i) at += i < warp ? static_cast<uint32_t>(sh.warp_sum[0][i]) : 0u;
    int sure = static_cast<int>(at & 0xffffu), tied = static_cast<int>(at >> 16);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = tid * items + i;
      if (i >= items) break;
      if (t < len) {
        const bool in = t >= lo && t < hi;
        const bool yes = !in || (wanted > 0 && key_of(i) > sel.bound);
        const bool tie = in && sel.ties > 0 && key_of(i) == sel.bound;
        // Kept before this token: the sure ones and the ties among the first `ties`.
        if (yes || (tie && tied < sel.ties)) {
          const int j = sure + (tied < sel.ties ? tied : sel.ties);
          list[j] = t;
          kept_bits[j] = bits[i];
        }
        sure += yes;
        tied += tie;
      }
    }
    __syncthreads();
    for (int j = tid; j < p.budget; j += kEvictThreads) kept[j] = j < keep ? list[j] : -1;
    for (int j = tid; j < len; j += kEvictThreads) wout[j] = j < keep ? __int_as_float(kept_bits[j]) : 0.f;
  } else {
    // Counted together: every CTA takes a slice.
    const int per = (len + ctas - 1) / ctas;
    const int t0 = min(len, rank * per), t1 = min(len, t0 + per);
    uint32_t prefix = 0xffffffffu;
    int need = wanted;
    if (need > 0) {
      prefix = 0;
      int* hist = sh.hist[0];
      for (int shift = 32 - kDigitBits; shift >= 0; shift -= kDigitBits) {
        for (int i = tid; i < kCopiesOfHist * kHistPitch; i += kEvictThreads) hist[i] = 0;
        __syncthreads();
        for (int t = max(t0, lo) + tid; t < min(t1, hi); t += kEvictThreads) count_digit(hist, weight_key(win[t]), prefix, shift);
        __syncthreads();
        if (tid < kDigits) {
          int sum = 0;
#pragma unroll
          for (int c = 0; c < kCopiesOfHist; ++c) sum += hist[c * kHistPitch + tid];
          hist[tid] = sum;  // the first copy: only this thread reads and writes column tid
        }
        sync_cluster();
        if (tid < kDigits) {
          int sum = 0;
          for (int r = 0; r < ctas; ++r) sum += ctas > 1 ? cluster.map_shared_rank(hist, r)[tid] : hist[tid];
          sh.total[tid] = sum;
        }
        sync_cluster();  // the totals are there, and every CTA has read the counts
        const Pick pick = pick_digit(sh.total, need);
        prefix |= static_cast<uint32_t>(pick.digit) << shift;
        need = pick.wanted;
        if (need == pick.has) {
          prefix -= 1;
          need = 0;
          break;
        }
      }
    }
    const bool some = wanted > 0;
    int n_sure = 0, n_tie = 0;
    for (int t = t0 + tid; t < t1; t += kEvictThreads) {
      const bool in = t >= lo && t < hi;
      const uint32_t key = in ? weight_key(win[t]) : 0u;
      n_sure += !in || (some && key > prefix);
      n_tie += in && need > 0 && key == prefix;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      n_sure += __shfl_xor_sync(0xffffffffu, n_sure, o);
      n_tie += __shfl_xor_sync(0xffffffffu, n_tie, o);
    }
    if (lane == 0) {
      sh.warp_sum[0][warp] = n_sure;
      sh.warp_sum[1][warp] = n_tie;
    }
    __syncthreads();
    if (tid == 0) {
      int a = 0, c = 0;
      for (int i = 0; i < kEvictWarps; ++i) {
        a += sh.warp_sum[0][i];
        c += sh.warp_sum[1][i];
      }
      sh.slice[0] = a;
      sh.slice[1] = c;
    }
    sync_cluster();
    int base_sure = 0, base_tie = 0;
    for (int r = 0; r < rank; ++r) {
      base_sure += cluster.map_shared_rank(sh.slice, r)[0];
      base_tie += cluster.map_shared_rank(sh.slice, r)[1];
    }
    for (int c0 = t0; c0 < t1; c0 += kEvictThreads) {
      const int t = c0 + tid;
      const bool in = t >= lo && t < hi;
      const uint32_t key = (t < t1 && in) ? weight_key(win[t]) : 0u;
      const bool sure = t < t1 && (!in || (some && key > prefix));
      const bool tie = t < t1 && in && need > 0 && key == prefix;
      const uint32_t bs = __ballot_sync(0xffffffffu, sure), bt = __ballot_sync(0xffffffffu, tie);
      __syncthreads();
      if (lane == 0) {
        sh.warp_sum[0][warp] = __popc(bs);
        sh.warp_sum[1][warp] = __popc(bt);
      }
      __syncthreads();
      int a = base_sure, c = base_tie;
#pragma unroll
      for (int i = 0; i < kEvictWarps; ++i) {
        if (i < warp) {
          a += sh.warp_sum[0][i];
          c += sh.warp_sum[1][i];
        }
        base_sure += sh.warp_sum[0][i];
        base_tie += sh.warp_sum[1][i];
      }
      const uint32_t below = (1u << lane) - 1u;
      a += __popc(bs & below);
      c += __popc(bt & below);
      if (sure || (tie && c < need)) kept[a + (c < need ? c : need)] = t;
    }
    for (int j = keep + rank * kEvictThreads + tid; j < p.budget; j += ctas * kEvictThreads) kept[j] = -1;
    __threadfence();
    sync_cluster();  // the list is there for all
    // The weights move a step at a time, as the rows below.
    for (int j0 = 0; j0 < len; j0 += ctas * kEvictThreads) {
      const int j = j0 + rank * kEvictThreads + tid;
      const float x = j < keep ? win[kept[j]] : 0.f;
      sync_cluster();
      if (j < len) wout[j] = x;
    }
  }
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = keep;

}

// The length of a sequence as the select kernel sees it, and what it keeps.
__device__ __forceinline__ int kept_tokens(const EvictParams& p, int b) {
  int len = p.lens[b];
  len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
  return len < p.budget ? len : p.budget;
}

// Where token `t` of sequence b lies: page (negative: nowhere) and row.
__device__ __forceinline__ int2 place_of(const EvictParams& p, const int32_t* table, int t) {
  const int block = static_cast<int>(page_of(p.page, t));
  const int page = table[block];
  return make_int2(page < p.num_pages ? page : -1, t - block * static_cast<int>(p.page.size));
}

// Apart: a warp takes kApartRows kept tokens; each half of it looks up one end
// of the moves, a token to a lane, so that the chain index -> table -> row is
// walked once for all of them, and the rows then pass through registers with
// kApartLoads vectors per lane in flight.
constexpr int kApartWarps = 8;
constexpr int kApartRows = 16;
constexpr int kApartLoads = 4;

// A sequence whose out table names one of its pages at the page's old place (a copy
// of the block table, or a table that keeps some pages) has rows that are a source
// for one move and the end of another. One CTA moves all of them then, in order: the
// rows of a step are all loaded before the first is stored, and later steps read
// behind the rows that it stores. The case above takes 180 us so, 44 where the
// caller says that it is in place.
__device__ __forceinline__ void move_ordered(const EvictParams& p, int b, int h, int keep, const int32_t* kept) {
  constexpr int kThreads = kApartWarps * 32;
  const int pieces = p.D / 8, row_items = 2 * pieces;
  const int rows = kThreads * kApartLoads / row_items;
  for (int j0 = 0; j0 < keep; j0 += rows) {
    uint4 x[kApartLoads];
    uint16_t* dst[kApartLoads];
#pragma unroll
    for (int i = 0; i < kApartLoads; ++i) {
      const int item = i * kThreads + threadIdx.x;
      const int r = item / row_items, j = j0 + r;
      dst[i] = nullptr;
      if (r < rows && j < keep) {
        const int2 from = place_of(p, p.tables + b * p.table_stride, kept[j]);
        const int2 to = place_of(p, p.out_tables + b * p.out_stride, j);
        if (from.x >= 0 && to.x >= 0) {
          const int at = item - r * row_items;
          const PagedCache& cache = at < pieces ? p.k : p.v;
          uint16_t* head = static_cast<uint16_t*>(cache.base) + h * cache.head_stride + (at < pieces ? at : at - pieces) * 8;
          x[i] = *reinterpret_cast<const uint4*>(head + from.x * cache.page_stride + from.y * cache.token_stride);
          dst[i] = head + to.x * cache.page_stride + to.y * cache.token_stride;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kApartLoads; ++i) {
      if (dst[i] != nullptr) *reinterpret_cast<uint4*>(dst[i]) = x[i];
    }
  }
}

__global__ void __launch_bounds__(kApartWarps * 32) kv_move_apart_kernel(const __grid_constant__ EvictParams p) {
  const int seg = blockIdx.x;
  const int b = seg / p.hkv, h = seg % p.hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int keep = min(kept_tokens(p, b), p.out_capacity);
  const int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  const int pieces = p.D / 8, row_items = 2 * pieces;
  bool shared = false;  // a page of this sequence stays where it was
  if (keep > 0) {
    const int blocks = static_cast<int>(page_of(p.page, keep - 1)) + 1;
    for (int i = threadIdx.x; i < blocks; i += kApartWarps * 32) {
      shared = shared || p.tables[b * p.table_stride + i] == p.out_tables[b * p.out_stride + i];
    }
  }
  shared = __syncthreads_or(shared);  // while the selection runs
  pdl_wait();
  pdl_launch_dependents();
  if (shared) {
    if (blockIdx.y == 0) move_ordered(p, b, h, keep, kept);
    return;
  }
  for (int j0 = (blockIdx.y * kApartWarps + warp) * kApartRows; j0 < keep; j0 += gridDim.y * kApartWarps * kApartRows) {
    const int mine = j0 + (lane & (kApartRows - 1));
    int2 place = make_int2(-1, 0);
    if (mine < keep) {
      place = lane < kApartRows ? place_of(p, p.tables + b * p.table_stride, kept[mine])
                                : place_of(p, p.out_tables + b * p.out_stride, mine);
    }
    const int items = min(kApartRows, keep - j0) * row_items;
    for (int i0 = 0; i0 < items; i0 += 32 * kApartLoads) {
      uint4 x[kApartLoads];
      uint16_t* dst[kApartLoads];
#pragma unroll
      for (int i = 0; i < kApartLoads; ++i) {
        const int item = i0 + i * 32 + lane;
        const int r = min(p.row_shift >= 0 ? item >> p.row_shift : item / row_items, kApartRows - 1);
        const int sp = __shfl_sync(0xffffffffu, place.x, r), sr = __shfl_sync(0xffffffffu, place.y, r);
        const int dp = __shfl_sync(0xffffffffu, place.x, kApartRows + r);
        const int dr = __shfl_sync(0xffffffffu, place.y, kApartRows + r);
        dst[i] = nullptr;
        if (item < items && sp >= 0 && dp >= 0) {
          const int at = item - r * row_items;
          const PagedCache& cache = at < pieces ? p.k : p.v;
          uint16_t* head = static_cast<uint16_t*>(cache.base) + h * cache.head_stride + (at < pieces ? at : at - pieces) * 8;
          x[i] = *reinterpret_cast<const uint4*>(head + sp * cache.page_stride + sr * cache.token_stride);
          dst[i] = head + dp * cache.page_stride + dr * cache.token_stride;
        }
      }
#pragma unroll
      for (int i = 0; i < kApartLoads; ++i) {
        if (dst[i] != nullptr) *reinterpret_cast<uint4*>(dst[i]) = x[i];
      }
    }
  }
}

// In place: a cluster per (sequence, kv head).
__global__ void __launch_bounds__(kMoveThreads) kv_move_in_place_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) unsigned char move_ring[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int seg = blockIdx.x / ctas;
  const int b = seg / p.hkv, h = seg % p.hkv;
  const int tid = threadIdx.x;
  const int keep = kept_tokens(p, b);
  const int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;
  pdl_wait();
  pdl_launch_dependents();
  // The rows move through a ring in shared memory that cp.async fills; a thread
  // moves one piece of one row per step and cache, and reads only what it
  // copied itself.
  const int pieces = p.D / 8;                 // 16-byte pieces per row
  const int rows_cta = kMoveThreads / pieces;  // kept tokens per CTA and step
  const int step = rows_cta * ctas;
  const int row = tid / pieces, piece = tid - row * pieces;
  const int steps = (keep + step - 1) / step;
  const uint32_t ring = smem_u32(move_ring) + tid * 16;
  uint32_t live = 0;  // bit k: the newest step but k moves this thread's piece
  auto fetch = [&](int k) {
    const int j = k * step + rank * rows_cta + row;
    bool moves = k < steps && row < rows_cta && j < keep && j < p.out_capacity;
    if (moves) {
      const int src = kept[j];
      const int sb = static_cast<int>(page_of(p.page, src)), db = static_cast<int>(page_of(p.page, j));
      const int sp = p.tables[b * p.table_stride + sb], dp = p.out_tables[b * p.out_stride + db];
      const int srow = src - sb * static_cast<int>(p.page.size), drow = j - db * static_cast<int>(p.page.size);
      moves = sp >= 0 && sp < p.num_pages && dp >= 0 && dp < p.num_pages && !(sp == dp && srow == drow);
      if (moves) {
        const uint32_t dst = ring + (k % kMoveStages) * (2 * kMoveThreads * 16);
        cp_async16(dst, static_cast<const uint16_t*>(p.k.base) + sp * p.k.page_stride + h * p.k.head_stride +
                            srow * p.k.token_stride + piece * 8);
        cp_async16(dst + kMoveThreads * 16, static_cast<const uint16_t*>(p.v.base) + sp * p.v.page_stride +
                                                 h * p.v.head_stride + srow * p.v.token_stride + piece * 8);
      }
    }
    cp_async_commit();
    live = (live << 1) | (moves ? 1u : 0u);
  };
#pragma unroll
  for (int k = 0; k < kMoveStages - 1; ++k) fetch(k);
  for (int k = 0; k < steps; ++k) {
    // This thread's piece of step k has landed, then everybody's: from here on
    // the rows that step k overwrites are read by nobody.
    cp_async_wait<kMoveStages - 2>();
    if (ctas > 1) {
      cluster_barrier_relaxed();
    } else {
      __syncthreads();
    }
    if ((live >> (kMoveStages - 2)) & 1) {
      const int j = k * step + rank * rows_cta + row;
      const int db = static_cast<int>(page_of(p.page, j));
      const int dp = p.out_tables[b * p.out_stride + db];
      const int drow = j - db * static_cast<int>(p.page.size);
      const unsigned char* at = move_ring + tid * 16 + (k % kMoveStages) * (2 * kMoveThreads * 16);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k.base) + dp * p.k.page_stride + h * p.k.head_stride +
                                drow * p.k.token_stride + piece * 8) = *reinterpret_cast<const uint4*>(at);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v.base) + dp * p.v.page_stride + h * p.v.head_stride +
                                drow * p.v.token_stride + piece * 8) =
          *reinterpret_cast<const uint4*>(at + kMoveThreads * 16);
    }
    fetch(k + kMoveStages - 1);
  }
}

}  // namespace
}  // namespace neso

using namespace neso;

extern "C" {

int neso_rope_paged_append(const void* q, const void* k, const void* v, const float* cos, const float* sin,
                           const int32_t* positions, const int64_t* slots, void* q_out, void* k_cache, void* v_cache,
                           int32_t dtype, int32_t N, int32_t Hq, int32_t Hkv, int32_t D, int32_t half,
                           int32_t table_rows, int32_t axes, const int32_t* sections, int64_t q_stride_n,
                           int64_t q_stride_h, int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n,
                           int64_t v_stride_h, int32_t num_pages, int32_t page_size, int64_t kc_stride_page,
                           int64_t kc_stride_head, int64_t kc_stride_token, int64_t vc_stride_page,
                           int64_t vc_stride_head, int64_t vc_stride_token, neso_stream_t stream) {
  if (dtype != NESO_F16 && dtype != NESO_BF16) return fail(NESO_ERR_INVALID_ARG, "dtype must be f16 or bf16");
  if (N < 0 || Hq < 0 || Hkv < 0 || D < 1 || half < 0 || table_rows < 0 || num_pages < 0) {
    return fail(NESO_ERR_INVALID_ARG, "negative size");
  }
  if (D % 8 != 0) return fail(NESO_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 (got %d)", D);
  if (half > D / 2) return fail(NESO_ERR_INVALID_ARG, "half = %d rotates more than head_dim = %d", half, D);
  if (page_size < 1) return fail(NESO_ERR_INVALID_ARG, "page_size must be at least 1 (got %d)", page_size);
  if (axes < 1 || axes > kMaxAxes) return fail(NESO_ERR_INVALID_ARG, "axes must be in [1, %d] (got %d)", kMaxAxes, axes);
  if (axes > 1 && sections == nullptr) return fail(NESO_ERR_INVALID_ARG, "several axes need their sections");
  if (D > kMaxRopeDim) return fail(NESO_ERR_UNSUPPORTED, "head_dim is limited to %d (got %d)", kMaxRopeDim, D);
  if (static_cast<int64_t>(Hq) + 2 * static_cast<int64_t>(Hkv) > 65536) {
    return fail(NESO_ERR_UNSUPPORTED, "a token has more than 65536 heads");
  }
  RopeParams p{};
  int at = 0;
  for (int a = 0; a < axes; ++a) {
    const int width = sections != nullptr ? sections[a] : half;
    if (width < 0 || width > half - at) return fail(NESO_ERR_INVALID_ARG, "sections do not add up to half = %d", half);
    at += width;
    p.section_end[a] = at;
  }
  if (at != half) return fail(NESO_ERR_INVALID_ARG, "sections do not add up to half = %d", half);
  if (N == 0) return ok();
  if (slots == nullptr || (Hq > 0 && (q == nullptr || q_out == nullptr)) || (Hkv > 0 && (k == nullptr || v == nullptr)) ||
      (half > 0 && (positions == nullptr || (table_rows > 0 && (cos == nullptr || sin == nullptr))))) {
    return fail(NESO_ERR_INVALID_ARG, "null pointer");
  }
  p.kc = PagedCache{k_cache, kc_stride_page, kc_stride_head, kc_stride_token};
  p.vc = PagedCache{v_cache, vc_stride_page, vc_stride_head, vc_stride_token};
  if (num_pages > 0) {
    int rc = check_cache(p.kc, "k_cache");
    if (rc == NESO_OK) rc = check_cache(p.vc, "v_cache");
    if (rc != NESO_OK) return rc;
  }
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.cos = cos;
  p.sin = sin;
  p.positions = positions;
  p.slots = slots;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.q_sn = q_stride_n;
  p.q_sh = q_stride_h;
  p.k_sn = k_stride_n;
  p.k_sh = k_stride_h;
  p.v_sn = v_stride_n;
  p.v_sh = v_stride_h;
  p.slot_count = static_cast<int64_t>(num_pages) * page_size;
  p.N = N;
  p.hq = Hq;
  p.hkv = Hkv;
  p.D = D;
  p.half = half;
  p.table_rows = table_rows;
  p.axes = axes;
  p.page = page_divisor(static_cast<uint32_t>(page_size));
  p.heads = page_divisor(static_cast<uint32_t>(Hq + 2 * Hkv > 0 ? Hq + 2 * Hkv : 1));
  // 16-byte vectors where the rows of q, k, v and q_out start on them and the
  // rotated part and the rest are pairs of them.
  const bool vec = D % 16 == 0 && half % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                   (q_stride_n | q_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h) % 8 == 0;
  if (dtype == NESO_BF16) return vec ? launch_rope<true, 8>(p, as_stream(stream)) : launch_rope<true, 1>(p, as_stream(stream));
  return vec ? launch_rope<false, 8>(p, as_stream(stream)) : launch_rope<false, 1>(p, as_stream(stream));
}

int neso_kv_evict(void* k_cache, void* v_cache, const int32_t* block_tables, const int32_t* out_tables,
                  const int32_t* seq_lens, const float* weights_in, float* weights_out, int32_t* kept,
                  int32_t* new_lens, int32_t B, int32_t Hkv, int32_t D, int32_t budget, int32_t recent, int32_t sink,
                  int32_t num_pages, int32_t page_size, int64_t k_stride_page, int64_t k_stride_head,
                  int64_t k_stride_token, int64_t v_stride_page, int64_t v_stride_head, int64_t v_stride_token,
                  int32_t table_width, int64_t table_stride, int32_t out_width, int64_t out_stride,
                  int64_t win_stride_b, int64_t win_stride_h, int64_t wout_stride_b, int64_t wout_stride_h,
                  neso_stream_t stream) {
  if (B < 0 || Hkv < 1 || num_pages < 0 || table_width < 0 || out_width < 0) {
    return fail(NESO_ERR_INVALID_ARG, "bad batch, head count, page count or table width");
  }
  if (D < 8 || D % 8 != 0 || D > 256) {
    return fail(NESO_ERR_UNSUPPORTED, "head_dim must be a multiple of 8, at most 256 (got %d)", D);
  }
  if (page_size < 1) return fail(NESO_ERR_INVALID_ARG, "page_size must be at least 1 (got %d)", page_size);
  if (budget < 1 || recent < 0 || sink < 0 || static_cast<int64_t>(recent) + sink > budget) {
    return fail(NESO_ERR_INVALID_ARG, "need budget >= 1 and 0 <= recent + sink <= budget");
  }
  // The selection requests the weights of a whole table before it knows the length.
  // Rows of a buffer that ends with the longest sequence are closer together.
  const int64_t tokens = static_cast<int64_t>(table_width) * page_size;
  if ((Hkv > 1 && win_stride_h > 0 && win_stride_h < tokens) || (B > 1 && win_stride_b > 0 && win_stride_b < tokens)) {
    return fail(NESO_ERR_INVALID_ARG, "rows of weights_in must hold table_width * page_size = %lld tokens",
                static_cast<long long>(tokens));
  }
  // As for lengths: steps past the end of a row of `kept` stay in 32 bits.
  if (budget > kMostTokens) return fail(NESO_ERR_UNSUPPORTED, "budget is limited to 2^30 tokens (got %d)", budget);
  if (static_cast<int64_t>(B) * Hkv * kMaxCluster > INT32_MAX) {
    return fail(NESO_ERR_UNSUPPORTED, "batch x heads is too large");
  }
  if (B == 0) return ok();
  if (seq_lens == nullptr || kept == nullptr || new_lens == nullptr ||
      (table_width > 0 && (block_tables == nullptr || weights_in == nullptr || weights_out == nullptr)) || (out_width > 0 && out_tables == nullptr)) {
    return fail(NESO_ERR_INVALID_ARG, "null pointer");
  }
  EvictParams p{};
  p.k = PagedCache{k_cache, k_stride_page, k_stride_head, k_stride_token};
  p.v = PagedCache{v_cache, v_stride_page, v_stride_head, v_stride_token};
  if (num_pages > 0) {
    int rc = check_cache(p.k, "k_cache");
    if (rc == NESO_OK) rc = check_cache(p.v, "v_cache");
    if (rc != NESO_OK) return rc;
  }
  const int64_t cap = static_cast<int64_t>(table_width) * page_size, ocap = static_cast<int64_t>(out_width) * page_size;
  p.tables = block_tables;
  p.out_tables = out_tables;
  p.lens = seq_lens;
  p.win = weights_in;
  p.wout = weights_out;
  p.kept = kept;
  p.new_lens = new_lens;
  p.table_stride = table_stride;
  p.out_stride = out_stride;
  p.win_sb = win_stride_b;
  p.win_sh = win_stride_h;
  p.wout_sb = wout_stride_b;
  p.wout_sh = wout_stride_h;
  p.hkv = Hkv;
  p.D = D;
  p.budget = budget;
  p.recent = recent;
  p.sink = sink;
  p.num_pages = num_pages;
  // At most 2^30, so that the kernel's steps past the end stay in 32 bits.
  p.capacity = static_cast<int>(cap < kMostTokens ? cap : kMostTokens);
  p.out_capacity = static_cast<int>(ocap < kMostTokens ? ocap : kMostTokens);
  p.page = page_divisor(static_cast<uint32_t>(page_size));
  const int64_t segments = static_cast<int64_t>(B) * Hkv;
  const int pieces = D / 8;
  p.row_shift = -1;
  for (int i = 0; i < 7; ++i) {
    if ((1 << i) == 2 * pieces) p.row_shift = i;
  }
  auto launch = [&](void (*kern)(EvictParams), int ctas, int threads, int smem) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(segments * ctas));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, p);
  };
  // CTAs that count one long sequence: as many as the SMs hold two deep.
  int ctas = 1;
  while (cap > kShortLen && ctas < kMaxCluster && segments * ctas * 2 <= 2 * sm_count()) ctas *= 2;
  auto* select = cap > kSmallTable ? kv_select_kernel<1024> : kv_select_kernel<512>;
  int rc = kernel_setup(reinterpret_cast<const void*>(select), kSelectBytes, nullptr);
  if (rc != NESO_OK) return rc;
  cudaError_t e = launch(select, ctas, cap > kSmallTable ? 1024 : 512, kSelectBytes);
  if (e != cudaSuccess) return cuda_fail(e, "kv_evict select launch");
  const int64_t most = budget < cap ? budget : cap;
  if (out_tables != block_tables || (B > 1 && out_stride != table_stride)) {
    const int64_t blocks = (most + kApartWarps * kApartRows - 1) / (kApartWarps * kApartRows);
    if (blocks == 0) return ok();
    e = launch_pdl(kv_move_apart_kernel, dim3(static_cast<unsigned>(segments), static_cast<unsigned>(blocks < 65535 ? blocks : 65535)),
                   dim3(kApartWarps * 32), 0, as_stream(stream), p);
  } else {
    rc = kernel_setup(reinterpret_cast<const void*>(kv_move_in_place_kernel), kMoveBytes, nullptr);
    if (rc != NESO_OK) return rc;
    // As many as fill the SMs two deep, no more than have a step's rows to move.
    const int rows = kMoveThreads / pieces;
    for (ctas = 1; ctas < kMaxCluster && segments * ctas * 2 <= 2 * sm_count() && static_cast<int64_t>(rows) * ctas < most;) ctas *= 2;
    e = launch(kv_move_in_place_kernel, ctas, kMoveThreads, kMoveBytes);
  }
  return e == cudaSuccess ? ok() : cuda_fail(e, "kv_evict move launch");
}

}  // extern "C"
