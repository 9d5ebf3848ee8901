// Writing to and trimming the paged key-value cache.
//
// rope_paged_append: new tokens' queries and keys are rotated in fp32 (products
// and sums rounded separately, then once to 16 bits) and keys and values go to
// their slots. One pass: every input byte is read once and every output byte
// written once, so HBM bounds it (launch latency for a few tokens).
//
// kv_evict: for each (sequence, kv head) the kept set is found by a radix
// selection on the weights' bits and the kept rows are moved together, in order.
// A cluster of CTAs owns one (sequence, kv head): it counts digits in its
// CTAs' shared memory, ranks the kept tokens by a scan, and moves the rows in
// steps, all CTAs side by side. Moving in place is safe because row j comes
// from row src_j >= j: when a step's rows are all in registers (a cluster
// barrier), the rows that it overwrites are not the source of any later step.
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
  PageDivisor page;
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
struct Vec {
  uint16_t e[N];
};
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

constexpr int kRopeThreads = 256;

// One CTA per token (grid-stride). A work item is kVec rotated pairs of one
// head, or kVec elements that are copied.
template <bool kBf16, int kVec>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_append_kernel(const __grid_constant__ RopeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int hv = p.half / kVec, rest = p.D / kVec - 2 * hv, dv = p.D / kVec;
  const int per_head = hv + rest;
  const int items = (p.hq + p.hkv) * per_head + p.hkv * dv;
  for (int n = blockIdx.x; n < p.N; n += gridDim.x) {
    const int64_t slot = p.slots[n];
    const bool pad = slot < 0 || slot >= p.slot_count;
    uint16_t* q_row = p.q_out + static_cast<int64_t>(n) * p.hq * p.D;
    if (pad) {
      Vec<kVec> zero;
#pragma unroll
      for (int i = 0; i < kVec; ++i) zero.e[i] = 0;
      for (int i = threadIdx.x; i < p.hq * dv; i += kRopeThreads) store_vec<kVec>(q_row + i * kVec, zero);
      continue;
    }
    const int64_t page = slot / p.page.size;
    const int64_t row = slot - page * p.page.size;
    uint16_t* kc = static_cast<uint16_t*>(p.kc.base) + page * p.kc.page_stride + row * p.kc.token_stride;
    uint16_t* vc = static_cast<uint16_t*>(p.vc.base) + page * p.vc.page_stride + row * p.vc.token_stride;
    for (int i = threadIdx.x; i < items; i += kRopeThreads) {
      if (i >= (p.hq + p.hkv) * per_head) {
        const int j = i - (p.hq + p.hkv) * per_head;
        const int h = j / dv, d = (j % dv) * kVec;
        store_vec<kVec>(vc + h * p.vc.head_stride + d, load_vec<kVec>(p.v + n * p.v_sn + h * p.v_sh + d));
        continue;
      }
      const int h = i / per_head, c = i % per_head;
      const uint16_t* src = h < p.hq ? p.q + n * p.q_sn + h * p.q_sh : p.k + n * p.k_sn + (h - p.hq) * p.k_sh;
      uint16_t* dst = h < p.hq ? q_row + static_cast<int64_t>(h) * p.D : kc + (h - p.hq) * p.kc.head_stride;
      if (c >= hv) {
        const int d = 2 * p.half + (c - hv) * kVec;
        store_vec<kVec>(dst + d, load_vec<kVec>(src + d));
        continue;
      }
      const int d = c * kVec;
      const Vec<kVec> a = load_vec<kVec>(src + d), b = load_vec<kVec>(src + d + p.half);
      Vec<kVec> x, y;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        int axis = 0;
        while (axis < p.axes - 1 && d + e >= p.section_end[axis]) ++axis;
        const int pos = p.positions[static_cast<int64_t>(axis) * p.N + n];
        float cs = __int_as_float(0x7fc00000), sn = cs;
        if (pos >= 0 && pos < p.table_rows) {
          cs = p.cos[static_cast<int64_t>(pos) * p.half + d + e];
          sn = p.sin[static_cast<int64_t>(pos) * p.half + d + e];
        }
        const float u = to_float<kBf16>(a.e[e]), w = to_float<kBf16>(b.e[e]);
        x.e[e] = from_float<kBf16>(__fsub_rn(__fmul_rn(u, cs), __fmul_rn(w, sn)));
        y.e[e] = from_float<kBf16>(__fadd_rn(__fmul_rn(u, sn), __fmul_rn(w, cs)));
      }
      store_vec<kVec>(dst + d, x);
      store_vec<kVec>(dst + d + p.half, y);
    }
  }
}

template <bool kBf16, int kVec>
int launch_rope(const RopeParams& p, cudaStream_t stream) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * 64;
  const unsigned grid = static_cast<unsigned>(p.N < cap ? p.N : cap);
  cudaError_t e = launch_pdl(rope_paged_append_kernel<kBf16, kVec>, dim3(grid), dim3(kRopeThreads), 0, stream, p);
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
  PageDivisor page;
};

constexpr int kEvictThreads = 512;
constexpr int kEvictCluster = 8;
constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kMoveRows = 2;  // 16-byte pieces per thread, cache and step

// Larger weights get larger keys; NaN the largest; -0 and +0 the same key.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __cluster_dims__(kEvictCluster, 1, 1) __launch_bounds__(kEvictThreads)
    kv_evict_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int hist[kDigits];
  __shared__ int total[kDigits];
  __shared__ int above_of[2];   // this CTA's slice: tokens above the threshold, tokens at it
  __shared__ int warp_sum[2][kEvictThreads / 32];
  __shared__ int pick[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int seg = blockIdx.x / kEvictCluster;
  const int b = seg / p.hkv, h = seg % p.hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();

  int len = p.lens[b];
  len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
  const int keep = len < p.budget ? len : p.budget;
  const float* win = p.win + b * p.win_sb + h * p.win_sh;
  float* wout = p.wout + b * p.wout_sb + h * p.wout_sh;
  int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.hkv + h) * p.budget;

  // Candidates [lo, hi) are ranked; tokens outside are kept.
  const bool all = len <= p.budget;
  const int lo = all ? 0 : p.sink, hi = all ? 0 : len - p.recent;
  int need = all ? 0 : keep - p.sink - p.recent;  // candidates to keep
  // This CTA's slice of the whole sequence.
  const int per = (len + kEvictCluster - 1) / kEvictCluster;
  const int t0 = min(len, rank * per), t1 = min(len, t0 + per);

  // The need-th largest key, digit by digit from the top: `prefix` holds the
  // digits found so far, `need` how many of the keys that share it are kept.
  uint32_t prefix = 0;
  if (need > 0) {
    for (int shift = 32 - kDigitBits; shift >= 0; shift -= kDigitBits) {
      for (int i = tid; i < kDigits; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int t = max(t0, lo) + tid; t < min(t1, hi); t += kEvictThreads) {
        const uint32_t key = weight_key(win[t]);
        if (shift == 32 - kDigitBits || (key >> (shift + kDigitBits)) == (prefix >> (shift + kDigitBits))) {
          atomicAdd(&hist[(key >> shift) & (kDigits - 1)], 1);
        }
      }
      cluster.sync();
      for (int i = tid; i < kDigits; i += kEvictThreads) {
        int sum = 0;
        for (int r = 0; r < kEvictCluster; ++r) sum += cluster.map_shared_rank(hist, r)[i];
        total[i] = sum;
      }
      __syncthreads();
      if (warp == 0) {
        // Digits from the largest down, eight to a lane.
        constexpr int kPer = kDigits / 32;
        int mine = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) mine += total[kDigits - 1 - (lane * kPer + j)];
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        int before = incl - mine;
        if (before < need && need <= incl) {
          for (int j = 0; j < kPer; ++j) {
            const int digit = kDigits - 1 - (lane * kPer + j);
            if (before + total[digit] >= need) {
              pick[0] = digit;
              pick[1] = need - before;
              break;
            }
            before += total[digit];
          }
        }
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(pick[0]) << shift;
      need = pick[1];
      cluster.sync();  // every CTA has read the counts before they are cleared
    }
  }
  // Now keys above `prefix` are kept, and the first `need` that equal it.

  int n_above = 0, n_at = 0;
  for (int t = t0 + tid; t < t1; t += kEvictThreads) {
    const bool in = t >= lo && t < hi;
    const uint32_t key = in ? weight_key(win[t]) : 0u;
    n_above += !in || (need > 0 && key > prefix);
    n_at += in && need > 0 && key == prefix;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    n_above += __shfl_xor_sync(0xffffffffu, n_above, o);
    n_at += __shfl_xor_sync(0xffffffffu, n_at, o);
  }
  if (lane == 0) {
    warp_sum[0][warp] = n_above;
    warp_sum[1][warp] = n_at;
  }
  __syncthreads();
  if (tid == 0) {
    int a = 0, c = 0;
    for (int i = 0; i < kEvictThreads / 32; ++i) {
      a += warp_sum[0][i];
      c += warp_sum[1][i];
    }
    above_of[0] = a;
    above_of[1] = c;
  }
  cluster.sync();
  int base_above = 0, base_at = 0;
  for (int r = 0; r < rank; ++r) {
    base_above += cluster.map_shared_rank(above_of, r)[0];
    base_at += cluster.map_shared_rank(above_of, r)[1];
  }
  // Ranks within the slice: running counts of kept-for-sure and of ties.
  for (int c0 = t0; c0 < t1; c0 += kEvictThreads) {
    const int t = c0 + tid;
    const bool in = t >= lo && t < hi;
    const uint32_t key = (t < t1 && in) ? weight_key(win[t]) : 0u;
    const bool sure = t < t1 && (!in || (need > 0 && key > prefix));
    const bool tie = t < t1 && in && need > 0 && key == prefix;
    const uint32_t bs = __ballot_sync(0xffffffffu, sure), bt = __ballot_sync(0xffffffffu, tie);
    __syncthreads();
    if (lane == 0) {
      warp_sum[0][warp] = __popc(bs);
      warp_sum[1][warp] = __popc(bt);
    }
    __syncthreads();
    int a = base_above, c = base_at;
    for (int i = 0; i < kEvictThreads / 32; ++i) {
      if (i < warp) {
        a += warp_sum[0][i];
        c += warp_sum[1][i];
      }
      base_above += warp_sum[0][i];
      base_at += warp_sum[1][i];
    }
    const uint32_t below = (1u << lane) - 1u;
    a += __popc(bs & below);
    c += __popc(bt & below);
    // Kept before this token: the sure ones and the ties among the first `need`.
    if (sure || (tie && c < need)) kept[a + (c < need ? c : need)] = t;
  }
  for (int j = keep + rank * kEvictThreads + tid; j < p.budget; j += kEvictCluster * kEvictThreads) kept[j] = -1;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = keep;
  __threadfence();
  cluster.sync();

  // Move rows and weights, a step of kStep kept tokens at a time.
  const int pieces = p.D / 8;                              // 16-byte pieces per row
  const int rows_cta = kEvictThreads * kMoveRows / pieces;  // kept tokens per CTA and step
  const int step = rows_cta * kEvictCluster;
  for (int j0 = 0; j0 < keep; j0 += step) {
    uint4 kx[kMoveRows], vx[kMoveRows];
    int64_t kd[kMoveRows], vd[kMoveRows];
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      const int r = (tid + i * kEvictThreads) / pieces, piece = (tid + i * kEvictThreads) % pieces;
      const int j = j0 + rank * rows_cta + r;
      kd[i] = -1;
      if (r < rows_cta && j < keep && j < p.out_capacity) {
        const int src = kept[j];
        const int sb = static_cast<int>(page_of(p.page, src)), db = static_cast<int>(page_of(p.page, j));
        const int sp = p.tables[b * p.table_stride + sb], dp = p.out_tables[b * p.out_stride + db];
        if (sp >= 0 && sp < p.num_pages && dp >= 0 && dp < p.num_pages) {
          const int64_t srow = src - static_cast<int64_t>(sb) * p.page.size, drow = j - static_cast<int64_t>(db) * p.page.size;
          const uint16_t* ks = static_cast<const uint16_t*>(p.k.base) + sp * p.k.page_stride + h * p.k.head_stride +
                               srow * p.k.token_stride + piece * 8;
          const uint16_t* vs = static_cast<const uint16_t*>(p.v.base) + sp * p.v.page_stride + h * p.v.head_stride +
                               srow * p.v.token_stride + piece * 8;
          if (!(sp == dp && srow == drow)) {
            kx[i] = *reinterpret_cast<const uint4*>(ks);
            vx[i] = *reinterpret_cast<const uint4*>(vs);
            kd[i] = dp * p.k.page_stride + h * p.k.head_stride + drow * p.k.token_stride + piece * 8;
            vd[i] = dp * p.v.page_stride + h * p.v.head_stride + drow * p.v.token_stride + piece * 8;
          }
        }
      }
    }
    cluster.sync();  // the step's rows are in registers everywhere
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      if (kd[i] >= 0) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k.base) + kd[i]) = kx[i];
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v.base) + vd[i]) = vx[i];
      }
    }
  }
  // The weights move the same way, one token per thread.
  for (int j0 = 0; j0 < len; j0 += kEvictCluster * kEvictThreads) {
    const int j = j0 + rank * kEvictThreads + tid;
    const float x = j < keep ? win[kept[j]] : 0.f;
    cluster.sync();
    if (j < len) wout[j] = x;
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
  if (static_cast<int64_t>(Hq + static_cast<int64_t>(Hkv) * 2) * D > INT32_MAX) {
    return fail(NESO_ERR_UNSUPPORTED, "a token has more than 2^31 - 1 elements");
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
  // 16-byte vectors where the rows of q, k, v and q_out start on them and the
  // rotated part ends on one.
  const bool vec = half % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
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
  if (static_cast<int64_t>(B) * Hkv * kEvictCluster > INT32_MAX) {
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
  // Below 2^30, so that the kernel's steps past the end stay in 32 bits.
  p.capacity = static_cast<int>(cap < (1 << 30) ? cap : (1 << 30));
  p.out_capacity = static_cast<int>(ocap < (1 << 30) ? ocap : (1 << 30));
  p.page = page_divisor(static_cast<uint32_t>(page_size));
  cudaError_t e = launch_pdl(kv_evict_kernel, dim3(static_cast<unsigned>(B) * Hkv * kEvictCluster), dim3(kEvictThreads), 0,
                             as_stream(stream), p);
  return e == cudaSuccess ? ok() : cuda_fail(e, "kv_evict launch");
}

}  // extern "C"
