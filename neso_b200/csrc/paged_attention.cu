// Attention of one new token per sequence over a paged key-value cache.
//
//   s[h, t] = scale * q[h] . k[t]                      (fp32)
//   s       = cap * tanh(s / cap)                      if cap > 0
//   s      += slope[h] * (t - (len - 1))               if slopes are given
//   o[h]    = sum_t p[h, t] v[t],  p = softmax over the visible t < len,
//             t > len - 1 - window if window > 0
//   weights_out[b, kv, t] = weights_in[b, kv, t] + sum over the kv head's
//             query heads of p[h, t]                   if weights are given
//
// Every visible key and value is read once for up to 16 query heads of its kv
// head (larger groups in several passes): 4 D bytes per token and kv head against
// 4 D FLOP per token and query head, far below the tensor cores' ridge, so HBM
// bounds it.
//
// Work: the cache is cut into units of 16 tokens of one (sequence, kv head).
// All units of the batch, in order, are dealt out in equal contiguous runs to
// the warps of the grid, whatever the sequences' lengths are; nothing about
// the lengths is needed on the host, so a captured graph follows them. A warp
// works alone: its own ring of three units in shared memory filled by
// cp.async (no block barrier), its own running maximum and sum. A run that
// holds a whole (sequence, kv head) writes the output itself; a run's first
// and last pieces leave their maximum, sum and unnormalised output in the
// workspace, and a second kernel joins them. Where the tables are short and
// the (sequence, kv head) pairs few, a cluster of CTAs takes each pair and joins
// its warps' parts itself: one launch, and no search for the runs.
//
// Products: the tokens are the M rows of mma.m16n8k16 and the query heads its
// N columns (S^T = K Q^T, O^T = V^T P^T), so a group of up to 8 heads costs one
// instruction per 16 x 16 block of the cache and ldmatrix reads each byte of
// it once; groups up to 16 take two column tiles, larger ones several passes.
// P goes into the second product as a sum of 16-bit values, the next one the
// remainder of those before (three in bf16: 2^-25 of the weight is left; two in
// fp16: 2^-22, see kParts and kRaise), so the output's own rounding is what
// remains; the tensor cores are idle enough to do it several times.
//
// Measured (B200, D = 128): one sequence of 131071 tokens, 32 / 8 heads, 92.5 us =
// 5.8 TB/s of keys and values, 88 % of the rate of a large copy; 64 ragged
// sequences of 5 to 8192 tokens, 64 / 8 heads, 75 us = 5.5 TB/s. What is
// missing: 5 us until the first keys arrive, the join (4 us), and equal runs
// that end at different times, because SMs reach memory at different rates (the
// last 16 us after the first in a run slowed by time stamps).
#include <cooperative_groups.h>

#include <map>
#include <mutex>

#include "paged.h"

namespace neso {
namespace {

namespace cg = cooperative_groups;

constexpr int kUnit = 16;      // tokens per unit
constexpr int kStages = 3;     // units in flight per warp
constexpr int kWarps = 4;      // warps per CTA
constexpr int kThreads = kWarps * 32;
// Cost of starting a segment, in units. With 0 / 1 / 2 / 4 / 8: 64 ragged sequences
// 85.6 / 76.5 / 76.8 / 76.8 / 76.7 us, 48 sequences under a window 25.8 / 25.1 / 25.1 /
// 25.5 / 26.3, 256 sequences of 500 tokens 98.3 / 95.3 / 97.0 / 99.1 / 97.2.
constexpr int kStart = 1;
// Least points of a run: shorter ones leave more pieces to join, longer ones
// fewer warps (8192 tokens of 16 / 1 heads as runs: 15.4 us with 2, 13.6 with 4, 15.8
// with 6; 2048 of 32 / 8: 11.2, 11.2, 14.4).
constexpr int kMinRun = 4;
constexpr float kLog2e = 1.4426950408889634f;

// A segment that several runs share: its index (sequence, kv head, tile), its
// first run, the number of runs, and the slot of the first run's piece; the
// other runs' pieces lie in their first slots.
struct Split {
  int seg, w0, count, first_slot;
  __device__ __forceinline__ int64_t slot(int i) const { return i == 0 ? first_slot : (w0 + i) * 2; }
};

struct AttnParams {
  const uint16_t* q;
  PagedCache k, v;
  const int32_t* tables;
  const int32_t* lens;
  const float* slopes;      // [Hq] or null
  uint16_t* out;            // [B, Hq, D]
  float4* partials;         // [2 warps][NT][D/16][32]
  float4* stats;            // [2 warps][NT][4]: m, l of heads 2c, 2c+1 (log2 units)
  Split* splits;            // [warps][2]
  float* scores;            // [B, Hq, score_stride], log2 units, when weights are wanted
  float2* head_stats;       // [B, Hq]: m, l of heads that were not split, when weights are wanted
  const float* win;
  float* wout;
  int64_t q_sb, q_sh, table_stride, win_sb, win_sh, wout_sb, wout_sh, score_stride;
  int B, hq, hkv, group, tiles, rows;  // tiles of `rows` query heads per kv head
  int num_pages, capacity, window, warps;
  bool whole_units;  // the page size is a multiple of kUnit
  int join_ctas;
  PageDivisor page;
  float score_scale;          // scale * log2(e), or scale / softcap when scores are capped
  float softcap;
};

// Visible token range [lo, len) of sequence b and its unit range.
struct Span {
  int len, lo, u0, u1;
};
__device__ __forceinline__ Span span_of(const AttnParams& p, int b) {
  Span s;
  int n = p.lens[b];
  n = n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
  s.len = n;
  s.lo = (p.window > 0 && n > p.window) ? n - p.window : 0;
  s.u0 = s.lo / kUnit;
  s.u1 = n / kUnit + (n % kUnit != 0);
  return s;
}

// The batch's work as a line: each segment, one (sequence, kv head, tile) with
// visible tokens, is kStart points for starting it (its queries, its output)
// followed by one point per unit. Runs are equal pieces of this line, whose
// length the host has checked to fit 31 bits.
__device__ __forceinline__ int cost_of(const Span& s) { return s.u1 > s.u0 ? s.u1 - s.u0 + kStart : 0; }

// Points per (kv head, tile) of the sequences before `b`, and of all of them;
// a whole warp calls it.
__device__ __forceinline__ void line_sums(const AttnParams& p, int b, int* before, int* all) {
  int lo = 0, sum = 0;
  for (int i = threadIdx.x & 31; i < p.B; i += 32) {
    const int cost = cost_of(span_of(p, i));
    sum += cost;
    if (i < b) lo += cost;
  }
  *all = __reduce_add_sync(0xffffffffu, sum);
  *before = __reduce_add_sync(0xffffffffu, lo);
}

// The line of `total` points is cut into `count` runs; the first `longer` of
// them have len + 1 points, the others len.
struct Runs {
  int count, len, longer;
  Runs() = default;
  __device__ __forceinline__ Runs(const AttnParams& p, int total) {
    const int most = total / kMinRun;
    count = most < 1 ? 1 : (most < p.warps ? most : p.warps);
    len = total / count;
    longer = total - len * count;
  }
  __device__ __forceinline__ int begin(int w) const { return w * len + (w < longer ? w : longer); }
  __device__ __forceinline__ int holding(int x) const {
    const int bound = longer * (len + 1);
    return x < bound ? x / (len + 1) : longer + (x - bound) / len;
  }
};

// Which runs share the segment of `per` units that starts at point s0: only
// the first of them can hold units of an earlier segment, and then its piece
// is its last one.
__device__ __forceinline__ Split split_of(const Runs& runs, int seg, int s0, int per) {
  const int w0 = runs.holding(s0 + kStart), w1 = runs.holding(s0 + kStart + per - 1);
  return Split{seg, w0, w1 - w0 + 1, w0 * 2 + (runs.begin(w0) >= s0 ? 0 : 1)};
}

// A position in the batch's order of units: sequence, (kv head, tile), unit.
struct Cursor {
  int b, hx, u;
  Span s;
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++u < s.u1) return;
    if (++hx < p.hkv * p.tiles) {
      u = s.u0;
      return;
    }
    hx = 0;
    do {
      if (++b >= p.B) return;
      s = span_of(p, b);
    } while (s.u0 == s.u1);
    u = s.u0;
  }
};

// Run w: its first unit, where that unit's segment starts on the line, and how
// many units the run has; a whole warp calls it.
__device__ __forceinline__ int find_run(const AttnParams& p, int w, Cursor* first, int* line, Runs* cut) {
  const int lane = threadIdx.x & 31;
  const int heads = p.hkv * p.tiles;
  const int cost0 = lane < p.B ? cost_of(span_of(p, lane)) : 0;
  int sum = cost0;
  for (int i = lane + 32; i < p.B; i += 32) sum += cost_of(span_of(p, i));
  const int total = __reduce_add_sync(0xffffffffu, sum) * heads;
  const Runs runs(p, total);
  *cut = runs;
  if (total == 0 || w >= runs.count) return 0;
  const int from = runs.begin(w), to = runs.begin(w + 1);
  int units_from = 0, units_to = 0;
  int past = 0, segments = 0;  // of the sequences before the 32 in hand
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int cost = b0 == 0 ? cost0 : (b0 + lane < p.B ? cost_of(span_of(p, b0 + lane)) : 0);
    int end = cost * heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += t;
    }
    end += past;
    const uint32_t filled = __ballot_sync(0xffffffffu, cost > 0);
    const int all = __shfl_sync(0xffffffffu, end, 31);
    // The first unit at or after point `at`, and the units before it.
    auto locate = [&](int at, Cursor* c) {
      const int src = __ffs(__ballot_sync(0xffffffffu, at < end)) - 1;
      const int b_cost = __shfl_sync(0xffffffffu, cost, src);
      const int start = __shfl_sync(0xffffffffu, end, src) - b_cost * heads;
      const int hx = (at - start) / b_cost;
      const int in = at - start - hx * b_cost;
      const int unit = in > kStart ? in - kStart : 0;
      const int seg = segments + __popc(filled & ((1u << src) - 1u)) * heads + hx;
      if (c != nullptr) {
        c->b = b0 + src;
        c->s = span_of(p, c->b);
        c->hx = hx;
        c->u = c->s.u0 + unit;
        *line = at - in;
      }
      return at - in + unit - seg * kStart;
    };
    if (from >= past && from < all) units_from = locate(from, first);
    if (to >= past && to < all) {
      units_to = locate(to, nullptr);
      return units_to - units_from;
    }
    segments += __popc(filled) * heads;
    past = all;
  }
  return total - segments * kStart - units_from;  // the last run ends with the line
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transpose of an 8 x 8 matrix of 16-bit values held one pair per lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kBf16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Write a 16 x 8 tile of O^T (rows d, columns heads) as 16-bit output: two
// 8 x 8 transposes give each lane one head and two neighbouring d.
template <bool kBf16>
__device__ __forceinline__ void store_out_tile(const AttnParams& p, const float (&o)[4], uint16_t* head0, int D, int nt,
                                               int dt, int nrows) {
  const int lane = threadIdx.x & 31;
  const uint32_t t0 = transpose8x8(pack16<kBf16>(o[0], o[1]));
  const uint32_t t1 = transpose8x8(pack16<kBf16>(o[2], o[3]));
  const int row = nt * 8 + (lane >> 2);
  if (row < nrows) {
    uint16_t* dst = head0 + static_cast<int64_t>(row) * D + dt * 16 + (lane & 3) * 2;
    *reinterpret_cast<uint32_t*>(dst) = t0;
    *reinterpret_cast<uint32_t*>(dst + 8) = t1;
  }
}

// The reference point of a row that has seen nothing yet is 0, so that its
// exponentials come out as 0 rather than exp(-inf + inf).
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.f : m; }
// 1 / l, and 0 for a row that saw no token (l == 0); NaN stays NaN.
__device__ __forceinline__ float inv_sum(float l) { return l == 0.f ? 0.f : __fdiv_rn(1.f, l); }

// One warp's work: a ring of units, and the state of the segment in hand.
// kBias: scores are capped or get a distance bias. kScores: they are kept for
// the weights.
template <bool kBf16, int D, int NT, bool kBias, bool kScores>
struct Warp {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kHalf = kUnit * kRowBytes;  // K or V of one unit
  static constexpr int kRing = kStages * 2 * kHalf;
  static constexpr int kChunks = kRowBytes / 16;   // 16-byte chunks per row
  static constexpr int kRowsPerCopy = 32 / kChunks;
  static constexpr int kCopies = kUnit / kRowsPerCopy;
  // fp16 ends at 2^-24: of weights up to 1, the value and the remainder would both
  // lose what lies below 2^-25, which the sum counts. Weights up to kRaise keep
  // 22 bits down to 2^-17 of the largest, and are off by 2^-40 of it below.
  static constexpr float kRaise = kBf16 ? 1.f : 32768.f;
  // Parts of a weight: 8 bits each in bf16, 11 in fp16. Two in bf16 leave 2^-17
  // of the weight, more than the rest of the arithmetic (48 sequences of up to 1025
  // visible tokens: results off by 1.0e-6 before their rounding, 4.0e-7 with three;
  // 22.9 against 23.4 us).
  static constexpr int kParts = kBf16 ? 3 : 2;

  const AttnParams& p;
  const int lane;
  const uint32_t ring;
  uint64_t masks;  // 16 validity bits per unit in flight, newest in the low bits
  uint32_t qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2], slope[NT][2];
  int h0, nrows;

  __device__ __forceinline__ Warp(const AttnParams& params, uint32_t ring_addr)
      : p(params), lane(threadIdx.x & 31), ring(ring_addr), masks(0) {}

  // Request unit c.u into a stage; with any = false only the group is counted.
  __device__ __forceinline__ void request(const Cursor& c, int stage, bool any) {
    uint32_t valid_bits = 0;
    if (any) {
      const int chunk = lane % kChunks;
      const uint32_t base = ring + stage * (2 * kHalf);
      const int64_t head = c.hx / p.tiles;
      const int t0 = c.u * kUnit;
      if (p.whole_units) {
        // A unit lies in one page: one table entry, rows a constant stride apart.
        const uint32_t block = page_of(p.page, t0);
        const int page = p.tables[c.b * p.table_stride + block];
        if (page >= 0 && page < p.num_pages) {
          const int a = c.s.lo - t0, z = c.s.len - t0;  // rows [a, z) are visible
          valid_bits = (z >= 16 ? 0xffffu : (1u << z) - 1u) & (a > 0 ? ~0u << a : ~0u);
        }
        const int64_t at = t0 - static_cast<int64_t>(block) * p.page.size + lane / kChunks;
        const bool in = valid_bits != 0;
        const char* ks = static_cast<const char*>(p.k.base) + chunk * 16 +
                         (in ? 2 * (page * p.k.page_stride + head * p.k.head_stride + at * p.k.token_stride) : 0);
        const char* vs = static_cast<const char*>(p.v.base) + chunk * 16 +
                         (in ? 2 * (page * p.v.page_stride + head * p.v.head_stride + at * p.v.token_stride) : 0);
        const int64_t kstep = in ? 2 * kRowsPerCopy * p.k.token_stride : 0;
        const int64_t vstep = in ? 2 * kRowsPerCopy * p.v.token_stride : 0;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int row = i * kRowsPerCopy + lane / kChunks;
          const uint32_t dst = base + row * kRowBytes + ((chunk ^ (row & 7)) << 4);
          cp_async16(dst, ks + i * kstep, (valid_bits >> row) & 1);
          cp_async16(dst + kHalf, vs + i * vstep, (valid_bits >> row) & 1);
        }
      } else {
        // Lane r < 16 finds the address of key row r of the unit, lane 16 + r
        // that of value row r; the copies fetch them by shuffle.
        const int t = t0 + (lane & 15);
        bool valid = t >= c.s.lo && t < c.s.len;
        const PagedCache& cache = lane < 16 ? p.k : p.v;
        int64_t off = 0;
        if (valid) {
          const uint32_t block = page_of(p.page, t);
          const int page = p.tables[c.b * p.table_stride + block];
          valid = page >= 0 && page < p.num_pages;
          if (valid) {
            off = page * cache.page_stride + head * cache.head_stride +
                  static_cast<int64_t>(t - block * p.page.size) * cache.token_stride;
          }
        }
        const uint16_t* src = static_cast<const uint16_t*>(cache.base) + off;
        valid_bits = __ballot_sync(0xffffffffu, valid) & 0xffffu;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int i = 0; i < kCopies; ++i) {
            const int row = i * kRowsPerCopy + lane / kChunks;
            const uint16_t* rsrc = reinterpret_cast<const uint16_t*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), half * 16 + row));
            cp_async16(base + half * kHalf + row * kRowBytes + ((chunk ^ (row & 7)) << 4), rsrc + chunk * 8,
                       (valid_bits >> row) & 1);
          }
        }
      }
    }
    masks = (masks << 16) | valid_bits;
    cp_async_commit();
  }

  // A new segment: its queries as the B operand (a head per lane quad), empty
  // statistics.
  __device__ __forceinline__ void start(const Cursor& c) {
    const int tile = c.hx % p.tiles;
    h0 = (c.hx / p.tiles) * p.group + tile * p.rows;
    nrows = p.group - tile * p.rows < p.rows ? p.group - tile * p.rows : p.rows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + (lane >> 2);
      const uint16_t* qrow = p.q + c.b * p.q_sb + static_cast<int64_t>(h0 + row) * p.q_sh + (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[nt][ks][0] = row < nrows ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16) : 0u;
        qf[nt][ks][1] = row < nrows ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8) : 0u;
        o[nt][ks][0] = o[nt][ks][1] = o[nt][ks][2] = o[nt][ks][3] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = -INFINITY;
        l[nt][j] = 0.f;
        const int col = nt * 8 + (lane & 3) * 2 + j;
        slope[nt][j] = (kBias && p.slopes != nullptr && col < nrows) ? p.slopes[h0 + col] * kLog2e : 0.f;
      }
    }
  }

  // Add the unit that lies in a stage, the oldest requested.
  __device__ __forceinline__ void add(const Cursor& c, int stage) {
    const uint32_t valid_bits = static_cast<uint32_t>(masks >> (16 * (kStages - 1))) & 0xffffu;
    const uint32_t base = ring + stage * (2 * kHalf);
    // S^T = K Q^T: rows are tokens lane/4 and lane/4 + 8, columns heads.
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    {
      const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
      const uint32_t rbase = base + row * kRowBytes;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[4];
        ldmatrix4(rbase + (((ks * 2 + (lane >> 4)) ^ (row & 7)) << 4), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<kBf16>(s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
    }
    const bool v0 = (valid_bits >> (lane >> 2)) & 1, v1 = (valid_bits >> ((lane >> 2) + 8)) & 1;
    uint32_t part[kParts][NT][2];
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = s[nt][j] * p.score_scale;
        if (kBias) {
          if (p.softcap > 0.f) x = p.softcap * kLog2e * tanhf(x);
          const int t = c.u * kUnit + (lane >> 2) + (j >> 1) * 8;
          x = fmaf(slope[nt][j & 1], static_cast<float>(t - (c.s.len - 1)), x);
        }
        s[nt][j] = ((j >> 1) ? v1 : v0) ? x : -INFINITY;
      }
      if (kScores) {
        const int t = c.u * kUnit + (lane >> 2);
        const int col = nt * 8 + (lane & 3) * 2;
        float* dst = p.scores + (static_cast<int64_t>(c.b) * p.hq + h0 + col) * p.score_stride + t;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (col + j < nrows) {
            dst[j * p.score_stride] = s[nt][j];
            dst[j * p.score_stride + 8] = s[nt][2 + j];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = fmaxf(s[nt][j], s[nt][2 + j]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx = fmaxf(mx, m[nt][j]);
        const float ref = safe_max(mx);
        alpha[nt][j] = ex2_approx(m[nt][j] - ref);
        m[nt][j] = mx;
        s[nt][j] = ex2_approx(s[nt][j] - ref) * kRaise;  // an exact product
        s[nt][2 + j] = ex2_approx(s[nt][2 + j] - ref) * kRaise;
        l[nt][j] = fmaf(l[nt][j], alpha[nt][j], s[nt][j] + s[nt][2 + j]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float2 rest = make_float2(s[nt][2 * j], s[nt][2 * j + 1]);
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
          const uint32_t h = pack16<kBf16>(rest.x, rest.y);
          const float2 f = unpack16<kBf16>(h);
          part[k][nt][j] = transpose8x8(h);
          rest = make_float2(rest.x - f.x, rest.y - f.y);
        }
      }
    }
    // O^T = alpha O^T + V^T P^T: rows are d, read through transposing ldmatrix. The
    // tensor cores cut each product off at the last bit of the sum they add to. A
    // sum over all tokens would lose that much per token (32768 tokens of one sign in
    // one run: 3e-4 of the result), so each unit's starts from zero, with the small
    // parts, and an FMA adds it to the scaled output.
    {
      const int row = (lane & 7) + (lane >> 4) * 8;
      const uint32_t rbase = base + kHalf + row * kRowBytes;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        uint32_t a[4];
        ldmatrix4_trans(rbase + (((dt * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = kParts - 1; k >= 0; --k) mma16816<kBf16>(sum, a, part[k][nt][0], part[k][nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][dt][e] = fmaf(o[nt][dt][e], alpha[nt][e & 1], sum[e]);
        }
      }
    }
  }

  // The sums of the segment's weights, over the lanes; weights count from 1 again.
  __device__ __forceinline__ void close() {
    constexpr float kLower = 1.f / kRaise;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
        l[nt][j] *= kLower;
      }
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][dt][e] *= kLower;
      }
    }
  }
  __device__ __forceinline__ float4 fragment(int nt, int dt) const {
    return make_float4(o[nt][dt][0], o[nt][dt][1], o[nt][dt][2], o[nt][dt][3]);
  }
  __device__ __forceinline__ float4 stats(int nt) const { return make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]); }
};

template <bool kBf16, int D, int NT, bool kBias, bool kScores>
__global__ void __launch_bounds__(kThreads, D == 128 ? 2 : 4)
    paged_attention_kernel(const __grid_constant__ AttnParams p) {
  using W = Warp<kBf16, D, NT, kBias, kScores>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Released only here: the join kernel reads the lengths before its own wait,
  // so everything launched before this grid has to be complete by then.
  pdl_wait();
  pdl_launch_dependents();

  // Neighbouring runs go to different CTAs, so a small batch spreads over the SMs.
  const int w = warp * gridDim.x + blockIdx.x;
  for (int b = w; b < p.B; b += p.warps) {
    if (cost_of(span_of(p, b)) == 0) {  // no token is visible
      uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + static_cast<int64_t>(b) * p.hq * D);
      for (int i = lane; i < p.hq * (D / 2); i += 32) dst[i] = 0u;
    }
  }
  Cursor ld;
  Runs runs;
  int line = 0;
  const int n = find_run(p, w, &ld, &line, &runs);
  Split first_split{0, 0, 0, 0}, started{0, 0, 0, 0};
  if (n == 0) {
    if (lane == 0) p.splits[w * 2] = p.splits[w * 2 + 1] = started;
    return;
  }
  Cursor c = ld;
  W my(p, smem_u32(smem) + warp * W::kRing);
  auto request = [&](int stage, bool any) {
    my.request(ld, stage, any);
    if (any) ld.next(p);
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request(s, s < n);

  bool fresh = true, whole = false, first_piece = true;
  for (int i = 0, stage = 0; i < n; ++i) {
    if (fresh) {
      fresh = false;
      whole = c.u == c.s.u0;
      my.start(c);
    }
    cp_async_wait<kStages - 2>();
    __syncwarp();
    {
      const int next = stage + kStages - 1;
      request(next >= kStages ? next - kStages : next, i + kStages - 1 < n);
    }
    my.add(c, stage);

    const bool seg_end = c.u + 1 == c.s.u1;
    if (seg_end || i + 1 == n) {
      my.close();
      const int64_t head = static_cast<int64_t>(c.b) * p.hq + my.h0;
      const int64_t slot = w * 2 + (first_piece ? 0 : 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (whole && seg_end) {
          const float r0 = inv_sum(my.l[nt][0]), r1 = inv_sum(my.l[nt][1]);
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const float4 f = my.fragment(nt, dt);
            const float t[4] = {f.x * r0, f.y * r1, f.z * r0, f.w * r1};
            store_out_tile<kBf16>(p, t, p.out + head * D, D, nt, dt, my.nrows);
          }
          if (kScores && lane < 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int col = nt * 8 + lane * 2 + j;
              if (col < my.nrows) p.head_stats[head + col] = make_float2(my.m[nt][j], my.l[nt][j]);
            }
          }
        } else {
          if (nt == 0) {
            const Split sp = split_of(runs, c.b * p.hkv * p.tiles + c.hx, line, c.s.u1 - c.s.u0);
            if (first_piece) first_split = sp;
            if (sp.w0 == w) started = sp;
          }
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) p.partials[((slot * NT + nt) * (D / 16) + dt) * 32 + lane] = my.fragment(nt, dt);
          if (lane < 4) p.stats[(slot * NT + nt) * 4 + lane] = my.stats(nt);
        }
      }
      fresh = true;
      first_piece = false;
      line += c.s.u1 - c.s.u0 + kStart;
    }
    c.next(p);
    if (++stage == kStages) stage = 0;
  }
  if (lane == 0) {
    p.splits[w * 2] = first_split;
    p.splits[w * 2 + 1] = started;
  }
}

// A cluster of CTAs per (sequence, kv head) of one tile, its units dealt to the
// warps of all of them in turn. Each CTA joins its warps' parts in its shared
// memory, then the CTAs take the fragments in turn and join them across the
// cluster, all in a fixed order.
constexpr int kSegWarps = 8;
constexpr int kSegThreads = kSegWarps * 32;
constexpr int kMaxCluster = 8;
// Very few pairs: clusters of this size, which a GPC of the B200 still holds (a
// CTA to an SM at D = 128, so that only half the SMs are counted on). One
// sequence of 8192 tokens: 16 / 1 heads x 128 17.8 -> 12.5 us, 32 / 8 x 64
// 11.9 -> 9.8; 32 / 8 x 128 would take 20.1 instead of 14.7, as the eight
// clusters are not on the SMs together.
constexpr int kBigCluster = 16;

// Statistics and fragment of some pieces, added up one after the other.
struct Joined {
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(const float4& st, const float4& x) {
    const float n0 = fmaxf(m0, st.x), n1 = fmaxf(m1, st.z);
    const float a0 = ex2_approx(m0 - safe_max(n0)), a1 = ex2_approx(m1 - safe_max(n1));
    const float b0 = ex2_approx(st.x - safe_max(n0)), b1 = ex2_approx(st.z - safe_max(n1));
    l0 = fmaf(st.y, b0, l0 * a0);
    l1 = fmaf(st.w, b1, l1 * a1);
    o.x = fmaf(x.x, b0, o.x * a0);
    o.y = fmaf(x.y, b1, o.y * a1);
    o.z = fmaf(x.z, b0, o.z * a0);
    o.w = fmaf(x.w, b1, o.w * a1);
    m0 = n0;
    m1 = n1;
  }
  __device__ __forceinline__ float4 stats() const { return make_float4(m0, l0, m1, l1); }
};

// As many CTAs an SM as the rings let in: left to itself the compiler keeps to 128
// registers, and the products wait for one another (one sequence of 8192 tokens,
// 32 / 8 heads x 128: 15.9 us, with 200 registers 14.8).
template <bool kBf16, int D, int NT, bool kBias, bool kScores>
__global__ void __launch_bounds__(kSegThreads, D == 128 ? 1 : 2) paged_attention_segment_kernel(const __grid_constant__ AttnParams p) {
  using W = Warp<kBf16, D, NT, kBias, kScores>;
  constexpr int kFrags = NT * (D / 16);
  static_assert(kFrags * 32 * sizeof(float4) <= W::kRing, "a warp's part fits its ring");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float4 stats[kSegWarps][NT][4];
  __shared__ float4 cta_stats[NT][4];
  __shared__ float4 cta_part[kFrags][32];
  __shared__ float2 final_stats[NT * 8];  // reference point, 1 / l
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int segment = blockIdx.x / ctas, step = ctas * kSegWarps;
  Cursor c;
  c.b = segment / p.hkv;
  c.hx = segment % p.hkv;
  c.s = span_of(p, c.b);
  c.u = c.s.u0 + warp * ctas + rank;
  const int n = c.u < c.s.u1 ? (c.s.u1 - c.u + step - 1) / step : 0;
  Cursor ld = c;
  W my(p, smem_u32(smem) + warp * W::kRing);
  auto request = [&](int stage, bool any) {
    my.request(ld, stage, any);
    ld.u += step;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request(s, s < n);
  my.start(c);
  for (int i = 0, stage = 0; i < n; ++i) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const int next = stage + kStages - 1;
    request(next >= kStages ? next - kStages : next, i + kStages - 1 < n);
    my.add(c, stage);
    c.u += step;
    if (++stage == kStages) stage = 0;
  }
  my.close();
  // The ring is empty: every requested unit has been added.
  float4* part = reinterpret_cast<float4*>(smem + warp * W::kRing);
  __syncwarp();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) part[(nt * (D / 16) + dt) * 32 + lane] = my.fragment(nt, dt);
    if (lane < 4) stats[warp][nt][lane] = my.stats(nt);
  }
  __syncthreads();
  uint16_t* head0 = p.out + (static_cast<int64_t>(c.b) * p.hq + my.h0) * D;
  auto write = [&](const Joined& j, int frag) {
    const float i0 = inv_sum(j.l0), i1 = inv_sum(j.l1);
    const float t[4] = {j.o.x * i0, j.o.y * i1, j.o.z * i0, j.o.w * i1};
    store_out_tile<kBf16>(p, t, head0, D, frag / (D / 16), frag % (D / 16), my.nrows);
  };
  for (int frag = warp; frag < kFrags; frag += kSegWarps) {
    const int nt = frag / (D / 16);
    Joined j;
#pragma unroll
    for (int k = 0; k < kSegWarps; ++k) {
      j.add(stats[k][nt][lane & 3], reinterpret_cast<const float4*>(smem + k * W::kRing)[frag * 32 + lane]);
    }
    if (ctas == 1) {
      write(j, frag);
    } else {
      cta_part[frag][lane] = j.o;
    }
    if (frag % (D / 16) == 0 && lane < 4) cta_stats[nt][lane] = j.stats();
  }
  if (ctas > 1) {
    cluster.sync();  // also: the scores of every CTA are written
    for (int frag = rank + warp * ctas; frag < kFrags; frag += step) {
      const int nt = frag / (D / 16);
      Joined j;
#pragma unroll 4
      for (int k = 0; k < ctas; ++k) {
        j.add(cluster.map_shared_rank(&cta_stats[nt][lane & 3], k)[0], cluster.map_shared_rank(&cta_part[frag][lane], k)[0]);
      }
      write(j, frag);
    }
  } else if (kScores) {
    __syncthreads();
  }
  if constexpr (kScores) {
    if (warp < NT && lane < 4) {
      const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
      Joined j;
      for (int k = 0; k < ctas; ++k) j.add(ctas == 1 ? cta_stats[warp][lane] : cluster.map_shared_rank(&cta_stats[warp][lane], k)[0], none);
      final_stats[warp * 8 + lane * 2] = make_float2(safe_max(j.m0), inv_sum(j.l0));
      final_stats[warp * 8 + lane * 2 + 1] = make_float2(safe_max(j.m1), inv_sum(j.l1));
    }
    __syncthreads();
    const float* in = p.win + c.b * p.win_sb + c.hx * p.win_sh;
    float* out = p.wout + c.b * p.wout_sb + c.hx * p.wout_sh;
    const float* scores = p.scores + (static_cast<int64_t>(c.b) * p.hq + my.h0) * p.score_stride;
    for (int t = rank * kSegThreads + threadIdx.x; t < c.s.len; t += ctas * kSegThreads) {
      float w = in[t];
      if (t >= c.s.lo) {
#pragma unroll 4
        for (int h = 0; h < my.nrows; ++h) {
          w = fmaf(ex2_approx(scores[h * p.score_stride + t] - final_stats[h].x), final_stats[h].y, w);
        }
      }
      out[t] = w;
    }
  }
  if (ctas > 1) cluster.sync();  // nobody reads this CTA's shared memory any more
}

// The second kernel. CTAs below p.join_ctas join the pieces of split segments.
// Each takes consecutive runs, as many as make some 300 CTAs, and the segments
// that start in them. A warp joins kPairFrags fragments (of 16 d x 8 heads) at
// a time of a segment in two or three pieces, one fragment of a segment in more;
// what matters is that all it reads is requested at once. The runs of a segment
// of more than kFewPieces pieces fill several CTAs: those take its fragments in
// turn, each warp an equal part of the pieces. Everything adds up in a fixed
// order. The other CTAs, when the weights are wanted, take kWeightTokens tokens
// of one (sequence, kv head):
//   weights_out[t] = weights_in[t] + sum_h exp2(s[h, t] - m[h]) / l[h].
constexpr int kJoinWarps = 8;
constexpr int kJoinThreads = kJoinWarps * 32;
constexpr int kPairFrags = 2;
constexpr int kFewPieces = 16;
constexpr int kJoinBatch = 4;  // pieces that a warp has requested
constexpr int kWeightTokens = 1024;
constexpr int kWeightSteps = kWeightTokens / kJoinThreads;
constexpr int kWeightHeads = 4;  // heads whose scores a thread has requested

struct JoinShared {
  float4 acc[kJoinWarps][32];
  float4 sums[kJoinWarps][4];
};

template <int D, int NT>
__device__ __forceinline__ void add_pieces(const AttnParams& p, const Split& sp, int frag, int first, int step, Joined& j) {
  const int lane = threadIdx.x & 31;
  const int nt = frag / (D / 16), dt = frag % (D / 16);
  for (int i0 = first; i0 < sp.count; i0 += kJoinBatch * step) {
    float4 st[kJoinBatch], x[kJoinBatch];
#pragma unroll
    for (int k = 0; k < kJoinBatch; ++k) {
      const int i = i0 + k * step;
      if (i < sp.count) {
        const int64_t slot = sp.slot(i) * NT + nt;
        st[k] = p.stats[slot * 4 + (lane & 3)];
        x[k] = p.partials[(slot * (D / 16) + dt) * 32 + lane];
      }
    }
#pragma unroll
    for (int k = 0; k < kJoinBatch; ++k) {
      if (i0 + k * step < sp.count) j.add(st[k], x[k]);
    }
  }
}

template <int D>
constexpr int join_runs() {
  return D == 64 ? 8 : 4;
}

template <bool kBf16, int D, int NT>
__device__ __forceinline__ void join_segments(const AttnParams& p, JoinShared& sh) {
  constexpr int kJoinRuns = join_runs<D>();
  constexpr int kFrags = NT * (D / 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.hkv * p.tiles;
  auto write = [&](const Split& sp, int frag, const Joined& j) {
    const int b = sp.seg / heads, hx = sp.seg - b * heads;
    const int kv = hx / p.tiles, tile = hx - kv * p.tiles;
    const int nrows = p.group - tile * p.rows < p.rows ? p.group - tile * p.rows : p.rows;
    const float i0 = inv_sum(j.l0), i1 = inv_sum(j.l1);
    const float t[4] = {j.o.x * i0, j.o.y * i1, j.o.z * i0, j.o.w * i1};
    store_out_tile<kBf16>(p, t, p.out + (static_cast<int64_t>(b) * p.hq + kv * p.group + tile * p.rows) * D, D,
                          frag / (D / 16), frag % (D / 16), nrows);
  };
  // Lane i has run i / 2's first piece (even) or the segment that starts in it (odd).
  const int run0 = blockIdx.x * kJoinRuns;
  Split mine{0, 0, 0, 0};
  if (lane < 2 * kJoinRuns && run0 + lane / 2 < p.warps) mine = p.splits[run0 * 2 + lane];
  auto split = [&](int i) {
    return Split{__shfl_sync(0xffffffffu, mine.seg, i), __shfl_sync(0xffffffffu, mine.w0, i),
                 __shfl_sync(0xffffffffu, mine.count, i), __shfl_sync(0xffffffffu, mine.first_slot, i)};
  };
  const uint32_t few = __ballot_sync(0xffffffffu, (lane & 1) && mine.count > 1 && mine.count <= kFewPieces);
  int task = 0;
  for (uint32_t left = few; left != 0; left &= left - 1) {
    const Split sp = split(__ffs(left) - 1);
    if (sp.count <= 3) {
      for (int frag0 = 0; frag0 < kFrags; frag0 += kPairFrags, ++task) {
        if (task % kJoinWarps != warp) continue;
        const int nt = frag0 / (D / 16);  // kPairFrags divides D / 16
        float4 st[3], x[3][kPairFrags];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (i < sp.count) {
            const int64_t slot = sp.slot(i) * NT;
            st[i] = p.stats[(slot + nt) * 4 + (lane & 3)];
#pragma unroll
            for (int f = 0; f < kPairFrags; ++f) x[i][f] = p.partials[(slot * (D / 16) + frag0 + f) * 32 + lane];
          }
        }
#pragma unroll
        for (int f = 0; f < kPairFrags; ++f) {
          Joined j;
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            if (i < sp.count) j.add(st[i], x[i][f]);
          }
          write(sp, frag0 + f, j);
        }
      }
      continue;
    }
    for (int frag = 0; frag < kFrags; ++frag, ++task) {
      if (task % kJoinWarps != warp) continue;
      Joined j;
      add_pieces<D, NT>(p, sp, frag, 0, 1, j);
      write(sp, frag, j);
    }
  }
  uint32_t many = __ballot_sync(0xffffffffu, !(lane & 1) && mine.count > kFewPieces && run0 + lane / 2 != mine.w0);
  int before = -1;
  for (; many != 0; many &= many - 1) {
    const Split sp = split(__ffs(many) - 1);
    if (sp.seg == before) continue;
    before = sp.seg;
    const int cta0 = (sp.w0 + 1) / kJoinRuns, ctas = (sp.w0 + sp.count - 1) / kJoinRuns - cta0 + 1;
    for (int frag = blockIdx.x - cta0; frag < kFrags; frag += ctas) {
      Joined j;
      add_pieces<D, NT>(p, sp, frag, warp, kJoinWarps, j);
      __syncthreads();  // the last fragment's sums have been read
      sh.acc[warp][lane] = j.o;
      if (lane < 4) sh.sums[warp][lane] = make_float4(j.m0, j.l0, j.m1, j.l1);
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int k = 1; k < kJoinWarps; ++k) j.add(sh.sums[k][lane & 3], sh.acc[k][lane]);
        write(sp, frag, j);
      }
    }
  }
}

// Reference point and 1 / l of the NT * 8 heads of one tile, into shared memory.
template <int NT>
__device__ __forceinline__ void tile_stats(const AttnParams& p, const Split& sp, int64_t head, int nrows, float2* stat) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= NT) return;
  // Lane quads take two heads each of every eighth piece.
  const int col = warp * 8 + (lane & 3) * 2;
  Joined j;
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
  if (sp.count == 1) {
    float2 st[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
    for (int k = 0; k < 2; ++k) {
      if (col + k < nrows) st[k] = p.head_stats[head + col + k];
    }
    j.m0 = st[0].x;
    j.l0 = st[0].y;
    j.m1 = st[1].x;
    j.l1 = st[1].y;
  } else {
#pragma unroll 4
    for (int i = lane >> 2; i < sp.count; i += 8) j.add(p.stats[(sp.slot(i) * NT + warp) * 4 + (lane & 3)], none);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
      const float4 other = make_float4(__shfl_xor_sync(0xffffffffu, j.m0, d), __shfl_xor_sync(0xffffffffu, j.l0, d),
                                       __shfl_xor_sync(0xffffffffu, j.m1, d), __shfl_xor_sync(0xffffffffu, j.l1, d));
      j.add(other, none);
    }
  }
  if (lane < 4) {
    stat[col] = make_float2(safe_max(j.m0), inv_sum(j.l0));
    stat[col + 1] = make_float2(safe_max(j.m1), inv_sum(j.l1));
  }
}

template <bool kBf16, int D, int NT, bool kScores>
__global__ void __launch_bounds__(kJoinThreads, kScores ? 4 : 2) paged_attention_join_kernel(const __grid_constant__ AttnParams p) {
  __shared__ JoinShared sh;
  if (!kScores || blockIdx.x < p.join_ctas) {
    pdl_wait();
    pdl_launch_dependents();
    join_segments<kBf16, D, NT>(p, sh);
    return;
  }
  if constexpr (kScores) {
    const int pair = (blockIdx.x - p.join_ctas) % (p.B * p.hkv), chunk = (blockIdx.x - p.join_ctas) / (p.B * p.hkv);
    const int b = pair / p.hkv, kv = pair % p.hkv;
    const Span s = span_of(p, b);
    const int per = s.u1 - s.u0, heads = p.hkv * p.tiles;
    int before, all;
    line_sums(p, b, &before, &all);
    const Runs runs(p, all * heads);
    pdl_wait();
    pdl_launch_dependents();
    if (chunk * kWeightTokens >= s.len) return;
    float2* stat = reinterpret_cast<float2*>(&sh.sums[0][0]);
    const float* in = p.win + b * p.win_sb + kv * p.win_sh;
    float* out = p.wout + b * p.wout_sb + kv * p.wout_sh;
    const int begin = chunk * kWeightTokens + threadIdx.x;
    float w[kWeightSteps];
#pragma unroll
    for (int i = 0; i < kWeightSteps; ++i) {
      const int t = begin + i * kJoinThreads;
      w[i] = t < s.len ? in[t] : 0.f;
    }
    for (int tile = 0; tile < p.tiles; ++tile) {
      const int h0 = kv * p.group + tile * p.rows;
      const int nrows = p.group - tile * p.rows < p.rows ? p.group - tile * p.rows : p.rows;
      const int64_t head = static_cast<int64_t>(b) * p.hq + h0;
      const float* scores = p.scores + head * p.score_stride;
      const Split sp = split_of(runs, 0, before * heads + (kv * p.tiles + tile) * (per + kStart), per);
      for (int g = 0; g < nrows; g += kWeightHeads) {
        float x[kWeightHeads][kWeightSteps];
#pragma unroll
        for (int h = 0; h < kWeightHeads; ++h) {
#pragma unroll
          for (int i = 0; i < kWeightSteps; ++i) {
            const int t = begin + i * kJoinThreads;
            x[h][i] = g + h < nrows && t >= s.lo && t < s.len ? scores[(g + h) * p.score_stride + t] : -INFINITY;
          }
        }
        if (g == 0) {  // while the scores are on their way
          __syncthreads();
          tile_stats<NT>(p, sp, head, nrows, stat);
          __syncthreads();
        }
#pragma unroll
        for (int h = 0; h < kWeightHeads; ++h) {
          if (g + h >= nrows) break;
          const float2 st = stat[g + h];
#pragma unroll
          for (int i = 0; i < kWeightSteps; ++i) w[i] = fmaf(ex2_approx(x[h][i] - st.x), st.y, w[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kWeightSteps; ++i) {
      const int t = begin + i * kJoinThreads;
      if (t < s.len) out[t] = w[i];
    }
  }
}

// A cluster per (sequence, kv head) where the clusters fit the SMs (two CTAs each
// at D = 64: 256 pairs of up to 300 tokens 7.3 us, as runs 12.2; at D = 128 one:
// 160 pairs of up to 900 tokens 17.2 us so, 16.6 as runs) and the tables hold at most
// kSegTokens tokens per CTA. One sequence, 32 / 8 heads,
// D = 128, 512 / 1024 / 2048 / 8192 tokens: 6.1 / 6.7 / 8.2 / 14.7 us so,
// 10.9 / 13.3 / 11.2 / 16.4 us as runs; beyond, the few CTAs' share of the
// bandwidth falls behind (8 pairs of up to 9000 tokens: 19.2 against 16.8 us; at
// D = 128 and 16 CTAs beyond half of that, 16384 tokens: 18.0 against 17.2).
constexpr int kSegTokens = 1024;
// A CTA is worth having for this many tokens.
constexpr int kSegLeast = 128;

void cluster_launch(cudaLaunchConfig_t* cfg, cudaLaunchAttribute (&attr)[2], int clusters, int size, int smem,
                    cudaStream_t stream) {
  *cfg = cudaLaunchConfig_t{};
  cfg->gridDim = dim3(static_cast<unsigned>(clusters * size));
  cfg->blockDim = dim3(kSegThreads);
  cfg->dynamicSmemBytes = smem;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(size);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 2;
}

// Whether the current device can hold a cluster of sixteen, which is more than
// every device has to (asked once, of the variant that needs most; without a
// device, the B200's answer).
template <int D>
bool holds_big_cluster() {
  static std::mutex mu;
  static std::map<int, bool> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return true;
  }
  std::lock_guard<std::mutex> lock(mu);
  const auto it = known.find(dev);
  if (it != known.end()) return it->second;
  constexpr int smem = kSegWarps * Warp<true, D, 2, true, true>::kRing;
  auto* kern = paged_attention_segment_kernel<true, D, 2, true, true>;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  cluster_launch(&cfg, attr, 1, kBigCluster, smem, nullptr);
  cfg.numAttrs = 1;  // the cluster's size
  int most = 0;
  if (kernel_setup(reinterpret_cast<const void*>(kern), smem, nullptr) != NESO_OK ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    most = 0;
  }
  return known[dev] = most > 0;
}

struct Plan {
  int group, tiles, rows, nt, ctas, warps;
  int64_t capacity;
  bool by_segment;
  int cluster;  // CTAs per segment then
  size_t partials, stats, splits, scores, head_stats, score_stride, bytes;
};

size_t round_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

int make_plan(int B, int hq, int hkv, int D, int width, int page_size, bool weights, Plan* out) {
  if (B < 0 || hq < 1 || hkv < 1 || width < 0) return fail(NESO_ERR_INVALID_ARG, "bad batch, head count or table width");
  if (hq % hkv != 0) return fail(NESO_ERR_INVALID_ARG, "%d query heads are not a multiple of %d kv heads", hq, hkv);
  if (D != 64 && D != 128) return fail(NESO_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", D);
  if (page_size < 1) return fail(NESO_ERR_INVALID_ARG, "page_size must be at least 1 (got %d)", page_size);
  Plan pl{};
  pl.group = hq / hkv;
  pl.tiles = (pl.group + 15) / 16;
  pl.rows = (pl.group + pl.tiles - 1) / pl.tiles;
  pl.nt = pl.rows > 8 ? 2 : 1;
  pl.capacity = static_cast<int64_t>(width) * page_size;
  if (pl.capacity > INT32_MAX - kUnit) pl.capacity = INT32_MAX - kUnit;
  // 192 KB of rings per SM: two CTAs of four warps at D = 128, four at 64.
  const int64_t units = (pl.capacity + kUnit - 1) / kUnit * B * hkv * pl.tiles;
  const int64_t segments = static_cast<int64_t>(B) * hkv * pl.tiles;
  if (segments > INT32_MAX || units + segments * kStart > INT32_MAX) {
    return fail(NESO_ERR_UNSUPPORTED, "batch x heads x table width exceeds 2^31 units of %d tokens", kUnit);
  }
  pl.cluster = 1;
  while (pl.cluster < kMaxCluster && segments * pl.cluster * 2 <= sm_count() && pl.cluster * kSegLeast < pl.capacity) pl.cluster *= 2;
  if (pl.cluster == kMaxCluster && pl.cluster * kSegLeast < pl.capacity &&
      segments * kBigCluster * (D == 64 ? 1 : 2) <= sm_count() && (D == 64 ? holds_big_cluster<64>() : holds_big_cluster<128>())) {
    pl.cluster = kBigCluster;
  }
  pl.by_segment = segments <= sm_count() * (D == 64 ? 2 : 1) && pl.tiles == 1 &&
                  pl.capacity <= static_cast<int64_t>(pl.cluster) * (D == 128 && pl.cluster > kMaxCluster ? kSegTokens / 2 : kSegTokens);
  const int64_t full = static_cast<int64_t>(sm_count()) * (D == 128 ? 2 : 4);
  pl.ctas = static_cast<int>(units < full ? (units > 1 ? units : 1) : full);
  pl.warps = pl.ctas * kWarps;
  pl.partials = 0;
  size_t at = 0;
  if (!pl.by_segment) {
    at = round_up(static_cast<size_t>(pl.warps) * 2 * pl.nt * (D / 16) * 32 * sizeof(float4));
    pl.stats = at;
    at += round_up(static_cast<size_t>(pl.warps) * 2 * pl.nt * 4 * sizeof(float4));
    pl.splits = at;
    at += round_up(static_cast<size_t>(pl.warps) * 2 * sizeof(Split));
  }
  if (weights) {
    pl.score_stride = static_cast<size_t>((pl.capacity + kUnit - 1) / kUnit * kUnit);
    pl.scores = at;
    at += round_up(pl.score_stride * static_cast<size_t>(B) * hq * sizeof(float));
    pl.head_stats = at;
    at += round_up(static_cast<size_t>(B) * hq * sizeof(float2));
  }
  pl.bytes = at;
  *out = pl;
  return NESO_OK;
}

template <bool kBf16, int D, int NT, bool kBias, bool kScores>
int launch_attention(const AttnParams& p, const Plan& pl, cudaStream_t stream) {
  using W = Warp<kBf16, D, NT, kBias, kScores>;
  if (pl.by_segment) {
    constexpr int smem = kSegWarps * W::kRing;
    auto* kern = paged_attention_segment_kernel<kBf16, D, NT, kBias, kScores>;
    const int rc = kernel_setup(reinterpret_cast<const void*>(kern), smem, nullptr);
    if (rc != NESO_OK) return rc;
    if (pl.cluster > kMaxCluster) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    }
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    cluster_launch(&cfg, attr, p.B * p.hkv, pl.cluster, smem, stream);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    return e == cudaSuccess ? ok() : cuda_fail(e, "paged_attention launch");
  }
  constexpr int smem = kWarps * W::kRing;
  auto* kern = paged_attention_kernel<kBf16, D, NT, kBias, kScores>;
  int rc = kernel_setup(reinterpret_cast<const void*>(kern), smem, nullptr);
  if (rc != NESO_OK) return rc;
  cudaError_t e = launch_pdl(kern, dim3(pl.ctas), dim3(kThreads), smem, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention launch");
  const int64_t pairs = static_cast<int64_t>(p.B) * p.hkv;
  const int64_t weight_ctas = kScores ? (pl.capacity + kWeightTokens - 1) / kWeightTokens * pairs : 0;
  e = launch_pdl(paged_attention_join_kernel<kBf16, D, NT, kScores>, dim3(static_cast<unsigned>(p.join_ctas + weight_ctas)),
                 dim3(kJoinThreads), 0, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention join launch");
  return ok();
}

template <bool kBf16, int D, int NT>
int launch_modes(const AttnParams& p, const Plan& pl, bool bias, cudaStream_t stream) {
  if (p.wout != nullptr) {
    return bias ? launch_attention<kBf16, D, NT, true, true>(p, pl, stream)
                : launch_attention<kBf16, D, NT, false, true>(p, pl, stream);
  }
  return bias ? launch_attention<kBf16, D, NT, true, false>(p, pl, stream)
              : launch_attention<kBf16, D, NT, false, false>(p, pl, stream);
}

template <bool kBf16>
int launch_shapes(const AttnParams& p, const Plan& pl, int D, bool bias, cudaStream_t stream) {
  if (D == 128) {
    return pl.nt == 2 ? launch_modes<kBf16, 128, 2>(p, pl, bias, stream) : launch_modes<kBf16, 128, 1>(p, pl, bias, stream);
  }
  return pl.nt == 2 ? launch_modes<kBf16, 64, 2>(p, pl, bias, stream) : launch_modes<kBf16, 64, 1>(p, pl, bias, stream);
}

}  // namespace
}  // namespace neso

using namespace neso;

extern "C" {

int64_t neso_paged_attention_workspace(int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t table_width,
                                       int32_t page_size, int32_t with_weights) {
  Plan pl;
  const int rc = make_plan(B, Hq, Hkv, D, table_width, page_size, with_weights != 0, &pl);
  if (rc != NESO_OK) return rc;
  ok();
  return static_cast<int64_t>(pl.bytes);
}

int neso_paged_attention(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                         const int32_t* seq_lens, const float* slopes, const float* weights_in, float* weights_out,
                         void* out, void* workspace, int64_t workspace_bytes, int32_t dtype, int32_t B, int32_t Hq,
                         int32_t Hkv, int32_t D, float scale, float softcap, int32_t window, int64_t q_stride_b,
                         int64_t q_stride_h, int32_t num_pages, int32_t page_size, int64_t k_stride_page,
                         int64_t k_stride_head, int64_t k_stride_token, int64_t v_stride_page, int64_t v_stride_head,
                         int64_t v_stride_token, int32_t table_width, int64_t table_stride, int64_t win_stride_b,
                         int64_t win_stride_h, int64_t wout_stride_b, int64_t wout_stride_h, neso_stream_t stream) {
  if (dtype != NESO_F16 && dtype != NESO_BF16) return fail(NESO_ERR_INVALID_ARG, "dtype must be f16 or bf16");
  Plan pl;
  int rc = make_plan(B, Hq, Hkv, D, table_width, page_size, weights_out != nullptr, &pl);
  if (rc != NESO_OK) return rc;
  if (num_pages < 0) return fail(NESO_ERR_INVALID_ARG, "num_pages must be >= 0");
  if (window < 0) return fail(NESO_ERR_INVALID_ARG, "window must be >= 0 (0 = no window)");
  if (!(softcap >= 0.f) || softcap > 1e30f || (softcap > 0.f && !(fabsf(scale / softcap) <= 1e30f))) {
    return fail(NESO_ERR_INVALID_ARG, "softcap must be >= 0 and finite, and scale / softcap finite");
  }
  if ((weights_in != nullptr) != (weights_out != nullptr)) {
    return fail(NESO_ERR_INVALID_ARG, "weights_in and weights_out come together");
  }
  if (B == 0) return ok();
  if (q == nullptr || seq_lens == nullptr || out == nullptr || (table_width > 0 && block_tables == nullptr)) {
    return fail(NESO_ERR_INVALID_ARG, "null pointer");
  }
  AttnParams p{};
  p.k = PagedCache{const_cast<void*>(k_cache), k_stride_page, k_stride_head, k_stride_token};
  p.v = PagedCache{const_cast<void*>(v_cache), v_stride_page, v_stride_head, v_stride_token};
  if (num_pages == 0) {
    // No page is valid and nothing is read, but copies of no bytes name an address all
    // the same, and it has to lie on 16 bytes as any other (q need not).
    p.k.base = p.v.base = reinterpret_cast<void*>(reinterpret_cast<uintptr_t>(q) & ~static_cast<uintptr_t>(15));
  } else {
    if ((rc = check_cache(p.k, "k_cache")) != NESO_OK) return rc;
    if ((rc = check_cache(p.v, "v_cache")) != NESO_OK) return rc;
  }
  if ((reinterpret_cast<uintptr_t>(q) & 3u) != 0 || (reinterpret_cast<uintptr_t>(out) & 3u) != 0 || q_stride_b % 2 != 0 ||
      q_stride_h % 2 != 0) {
    return fail(NESO_ERR_MISALIGNED, "q, out and q's strides must be multiples of 4 bytes");
  }
  if (pl.bytes > 0 && (workspace == nullptr || workspace_bytes < static_cast<int64_t>(pl.bytes))) {
    return fail(NESO_ERR_INVALID_ARG, "workspace holds %lld bytes, %lld are needed",
                static_cast<long long>(workspace == nullptr ? 0 : workspace_bytes), static_cast<long long>(pl.bytes));
  }
  if (!aligned16(workspace)) return fail(NESO_ERR_MISALIGNED, "workspace is not 16-byte aligned");
  if (weights_out != nullptr &&
      (pl.capacity + kWeightTokens - 1) / kWeightTokens * (static_cast<int64_t>(B) * Hkv) > INT32_MAX - pl.warps) {
    return fail(NESO_ERR_UNSUPPORTED, "batch x kv heads x table width is too large for weights");
  }
  p.q = static_cast<const uint16_t*>(q);
  p.tables = block_tables;
  p.lens = seq_lens;
  p.slopes = slopes;
  p.out = static_cast<uint16_t*>(out);
  char* ws = static_cast<char*>(workspace);
  p.partials = reinterpret_cast<float4*>(ws + pl.partials);
  p.stats = reinterpret_cast<float4*>(ws + pl.stats);
  p.splits = reinterpret_cast<Split*>(ws + pl.splits);
  p.scores = reinterpret_cast<float*>(ws + pl.scores);
  p.head_stats = reinterpret_cast<float2*>(ws + pl.head_stats);
  p.win = weights_in;
  p.wout = weights_out;
  p.q_sb = q_stride_b;
  p.q_sh = q_stride_h;
  p.table_stride = table_stride;
  p.win_sb = win_stride_b;
  p.win_sh = win_stride_h;
  p.wout_sb = wout_stride_b;
  p.wout_sh = wout_stride_h;
  p.score_stride = static_cast<int64_t>(pl.score_stride);
  p.B = B;
  p.hq = Hq;
  p.hkv = Hkv;
  p.group = pl.group;
  p.tiles = pl.tiles;
  p.rows = pl.rows;
  p.num_pages = num_pages;
  p.capacity = static_cast<int>(pl.capacity);
  p.window = window;
  p.warps = pl.warps;
  p.whole_units = page_size % kUnit == 0;
  const int join = D == 64 ? join_runs<64>() : join_runs<128>();
  p.join_ctas = (pl.warps + join - 1) / join;
  p.page = page_divisor(static_cast<uint32_t>(page_size));
  p.score_scale = softcap > 0.f ? scale / softcap : scale * kLog2e;
  p.softcap = softcap;
  const bool bias = softcap > 0.f || slopes != nullptr;
  return dtype == NESO_BF16 ? launch_shapes<true>(p, pl, D, bias, as_stream(stream))
                            : launch_shapes<false>(p, pl, D, bias, as_stream(stream));
}

}  // extern "C"
