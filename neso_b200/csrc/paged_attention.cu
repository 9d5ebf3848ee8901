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
// Every visible key and value is read once for all the query heads of its kv
// head: 4 D bytes per token and kv head against 4 D FLOP per token and query
// head, far below the tensor cores' ridge, so HBM bounds it.
//
// Work: the cache is cut into units of 16 tokens of one (sequence, kv head).
// All units of the batch, in order, are dealt out in equal contiguous runs to
// the warps of the grid, whatever the sequences' lengths are; nothing about
// the lengths is needed on the host, so a captured graph follows them. A warp
// works alone: its own ring of three units in shared memory filled by
// cp.async (no block barrier), its own running maximum and sum. A run that
// holds a whole (sequence, kv head) writes the output itself; a run's first
// and last pieces leave their maximum, sum and unnormalised output in the
// workspace, and a second kernel joins them.
//
// Products: the tokens are the M rows of mma.m16n8k16 and the query heads its
// N columns (S^T = K Q^T, O^T = V^T P^T), so a group of up to 8 heads costs one
// instruction per 16 x 16 block of the cache and ldmatrix reads each byte of
// it once; groups up to 16 take two column tiles, larger ones several passes.
// P goes into the second product as a 16-bit value plus the 16-bit remainder
// (relative error 2^-16 for bf16, 2^-22 for fp16), so the output's own
// rounding is what remains; the tensor cores are idle enough to do it twice.
#include "paged.h"

namespace neso {
namespace {

constexpr int kUnit = 16;      // tokens per unit
constexpr int kStages = 3;     // units in flight per warp
constexpr int kWarps = 4;      // warps per CTA
constexpr int kThreads = kWarps * 32;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const uint16_t* q;
  PagedCache k, v;
  const int32_t* tables;
  const int32_t* lens;
  const float* slopes;      // [Hq] or null
  uint16_t* out;            // [B, Hq, D]
  float4* partials;         // [2 warps][NT][D/16][32]
  float4* stats;            // [2 warps][NT][4]: m, l of heads 2c, 2c+1 (log2 units)
  float* scores;            // [B, Hq, score_stride], log2 units, when weights are wanted
  float2* head_stats;       // [B, Hq]: final m, l, when weights are wanted
  const float* win;
  float* wout;
  int64_t q_sb, q_sh, table_stride, win_sb, win_sh, wout_sb, wout_sh, score_stride;
  int B, hq, hkv, group, tiles, rows;  // tiles of `rows` query heads per kv head
  int num_pages, capacity, window, warps;
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

// The units of all sequences before `b`, and of the whole batch, per (kv
// head, tile); a whole warp calls it.
__device__ __forceinline__ void unit_sums(const AttnParams& p, int b, int64_t* before, int64_t* all) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, sum = 0;
  for (int i = lane; i < p.B; i += 32) {
    const Span s = span_of(p, i);
    sum += s.u1 - s.u0;
    if (i < b) lo += s.u1 - s.u0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    lo += __shfl_xor_sync(0xffffffffu, lo, o);
  }
  *before = lo;
  *all = sum;
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

__device__ __forceinline__ Cursor find_unit(const AttnParams& p, int64_t at) {
  const int lane = threadIdx.x & 31;
  const int heads = p.hkv * p.tiles;
  Cursor c{0, 0, 0, {0, 0, 0, 0}};
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + lane;
    int64_t mine = 0;
    if (b < p.B) {
      const Span s = span_of(p, b);
      mine = static_cast<int64_t>(s.u1 - s.u0) * heads;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, at < incl);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      const int64_t rest = at - __shfl_sync(0xffffffffu, incl - mine, src);
      c.b = b0 + src;
      c.s = span_of(p, c.b);
      const int per = c.s.u1 - c.s.u0;
      c.hx = static_cast<int>(rest / per);
      c.u = c.s.u0 + static_cast<int>(rest % per);
      return c;
    }
    at -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return c;
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

// The two 16-bit types: pack with one rounding, unpack exactly, multiply.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
  if (kBf16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
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

// kBias: scores are capped or get a distance bias. kScores: they are kept for
// the weights kernel.
template <bool kBf16, int D, int NT, bool kBias, bool kScores>
__global__ void __launch_bounds__(kThreads, D == 128 ? 2 : 4)
    paged_attention_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kRowBytes = D * 2;
  constexpr int kHalf = kUnit * kRowBytes;  // K or V of one unit
  constexpr int kChunks = kRowBytes / 16;   // 16-byte chunks per row
  constexpr int kRowsPerCopy = 32 / kChunks;
  constexpr int kCopies = kUnit / kRowsPerCopy;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * kHalf);

  pdl_launch_dependents();
  pdl_wait();

  int64_t unused, per_head;
  unit_sums(p, 0, &unused, &per_head);
  const int64_t total = per_head * p.hkv * p.tiles;
  const int64_t nw = total < p.warps ? total : p.warps;
  // Neighbouring runs go to different CTAs, so a small batch spreads over the SMs.
  const int64_t w = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x;
  if (w >= nw) return;
  const int64_t first = w * total / nw, last = (w + 1) * total / nw;
  const int n = static_cast<int>(last - first);

  Cursor ld = find_unit(p, first);
  Cursor c = ld;
  uint64_t masks = 0;  // 16 validity bits per unit in flight, newest in the low bits

  // Lane r < 16 finds the address of key row r of the unit, lane 16 + r that
  // of value row r; the copies fetch them by shuffle.
  auto issue = [&](int stage, bool any) {
    uint32_t valid_bits = 0;
    if (any) {
      const int r = lane & 15;
      const int t = ld.u * kUnit + r;
      bool valid = t >= ld.s.lo && t < ld.s.len;
      const PagedCache& cache = lane < 16 ? p.k : p.v;
      int64_t off = 0;
      if (valid) {
        const uint32_t block = page_of(p.page, t);
        const int page = p.tables[ld.b * p.table_stride + block];
        valid = page >= 0 && page < p.num_pages;
        if (valid) {
          off = page * cache.page_stride + (ld.hx / p.tiles) * cache.head_stride +
                static_cast<int64_t>(t - block * p.page.size) * cache.token_stride;
        }
      }
      const uint16_t* src = static_cast<const uint16_t*>(cache.base) + off;
      valid_bits = __ballot_sync(0xffffffffu, valid) & 0xffffu;
      const int chunk = lane % kChunks;
      const uint32_t base = ring + stage * (2 * kHalf);
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
      ld.next(p);
    }
    masks = (masks << 16) | valid_bits;
    cp_async_commit();
  };

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s, s < n);

  uint32_t qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2], slope[NT][2];
  bool fresh = true, whole = false, first_piece = true;
  int nrows = 0;

  for (int i = 0, stage = 0; i < n; ++i) {
    if (fresh) {
      // A new (sequence, kv head, tile): its queries as the B operand (one
      // head per lane quad row), empty statistics.
      fresh = false;
      whole = c.u == c.s.u0;
      const int tile = c.hx % p.tiles;
      const int h0 = (c.hx / p.tiles) * p.group + tile * p.rows;
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

    cp_async_wait<kStages - 2>();
    __syncwarp();
    {
      const int next = stage + kStages - 1;
      issue(next >= kStages ? next - kStages : next, i + kStages - 1 < n);
    }
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
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x;
        if (kBias) {
          x = s[nt][j] * p.score_scale;
          if (p.softcap > 0.f) x = p.softcap * kLog2e * tanhf(x);
          const int t = c.u * kUnit + (lane >> 2) + (j >> 1) * 8;
          x = fmaf(slope[nt][j & 1], static_cast<float>(t - (c.s.len - 1)), x);
        } else {
          x = s[nt][j] * p.score_scale;
        }
        s[nt][j] = ((j >> 1) ? v1 : v0) ? x : -INFINITY;
      }
      if (kScores) {
        const int t = c.u * kUnit + (lane >> 2);
        const int col = nt * 8 + (lane & 3) * 2;
        const int h0 = (c.hx / p.tiles) * p.group + (c.hx % p.tiles) * p.rows;
        float* dst = p.scores + (static_cast<int64_t>(c.b) * p.hq + h0 + col) * p.score_stride + t;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (col + j < nrows) {
            dst[j * p.score_stride] = s[nt][j];
            dst[j * p.score_stride + 8] = s[nt][2 + j];
          }
        }
      }
      float alpha[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = fmaxf(s[nt][j], s[nt][2 + j]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        mx = fmaxf(mx, m[nt][j]);
        const float ref = safe_max(mx);
        alpha[j] = ex2_approx(m[nt][j] - ref);
        m[nt][j] = mx;
        s[nt][j] = ex2_approx(s[nt][j] - ref);
        s[nt][2 + j] = ex2_approx(s[nt][2 + j] - ref);
        l[nt][j] = fmaf(l[nt][j], alpha[j], s[nt][j] + s[nt][2 + j]);
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          o[nt][dt][0] *= alpha[0];
          o[nt][dt][1] *= alpha[1];
          o[nt][dt][2] *= alpha[0];
          o[nt][dt][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t h = pack16<kBf16>(s[nt][2 * j], s[nt][2 * j + 1]);
        const float2 f = unpack16<kBf16>(h);
        hi[nt][j] = transpose8x8(h);
        lo[nt][j] = transpose8x8(pack16<kBf16>(s[nt][2 * j] - f.x, s[nt][2 * j + 1] - f.y));
      }
    }
    // O^T += V^T P^T: rows are d, read through transposing ldmatrix.
    {
      const int row = (lane & 7) + (lane >> 4) * 8;
      const uint32_t rbase = base + kHalf + row * kRowBytes;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        uint32_t a[4];
        ldmatrix4_trans(rbase + (((dt * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4), a);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816<kBf16>(o[nt][dt], a, hi[nt][0], hi[nt][1]);
          mma16816<kBf16>(o[nt][dt], a, lo[nt][0], lo[nt][1]);
        }
      }
    }

    const bool seg_end = c.u + 1 == c.s.u1;
    if (seg_end || i + 1 == n) {
      const int h0 = (c.hx / p.tiles) * p.group + (c.hx % p.tiles) * p.rows;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
        }
        if (whole && seg_end) {
          const float r0 = inv_sum(l[nt][0]), r1 = inv_sum(l[nt][1]);
          uint16_t* head0 = p.out + (static_cast<int64_t>(c.b) * p.hq + h0) * D;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const float t[4] = {o[nt][dt][0] * r0, o[nt][dt][1] * r1, o[nt][dt][2] * r0, o[nt][dt][3] * r1};
            store_out_tile<kBf16>(p, t, head0, D, nt, dt, nrows);
          }
          if (kScores && lane < 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int col = nt * 8 + lane * 2 + j;
              if (col < nrows) p.head_stats[static_cast<int64_t>(c.b) * p.hq + h0 + col] = make_float2(m[nt][j], l[nt][j]);
            }
          }
        } else {
          const int64_t slot = w * 2 + (first_piece ? 0 : 1);
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            p.partials[((slot * NT + nt) * (D / 16) + dt) * 32 + lane] =
                make_float4(o[nt][dt][0], o[nt][dt][1], o[nt][dt][2], o[nt][dt][3]);
          }
          if (lane < 4) p.stats[(slot * NT + nt) * 4 + lane] = make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]);
        }
      }
      fresh = true;
      first_piece = false;
    }
    c.next(p);
    if (++stage == kStages) stage = 0;
  }
}

// One CTA per (sequence, kv head, tile): joins the pieces that the runs left
// when the segment was split, and writes zeros where no token is visible.
// Warps take fragments of 16 d x 8 heads; spare warps share the pieces of one
// fragment and add up in shared memory in a fixed order.
constexpr int kJoinWarps = 16;

template <bool kBf16, int D, int NT, bool kScores>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attention_join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kFrags = NT * (D / 16);
  constexpr int kParts = kJoinWarps / kFrags;
  __shared__ float4 acc[kJoinWarps][32];
  __shared__ float4 sums[kJoinWarps][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int heads = p.hkv * p.tiles;
  const int b = blockIdx.x / heads, hx = blockIdx.x % heads;
  const int tile = hx % p.tiles;
  const int h0 = (hx / p.tiles) * p.group + tile * p.rows;
  const int nrows = p.group - tile * p.rows < p.rows ? p.group - tile * p.rows : p.rows;
  uint16_t* head0 = p.out + (static_cast<int64_t>(b) * p.hq + h0) * D;
  const Span s = span_of(p, b);
  const int per = s.u1 - s.u0;
  if (per == 0) {
    uint32_t* dst = reinterpret_cast<uint32_t*>(head0);
    for (int i = threadIdx.x; i < nrows * D / 2; i += blockDim.x) dst[i] = 0u;
    return;
  }
  int64_t before, all;
  unit_sums(p, b, &before, &all);
  const int64_t total = all * heads;
  const int64_t nw = total < p.warps ? total : p.warps;
  const int64_t s0 = before * heads + static_cast<int64_t>(hx) * per;
  // The run that holds unit x is the largest w with w * total / nw <= x.
  const int64_t w0 = ((s0 + 1) * nw - 1) / total, w1 = ((s0 + per) * nw - 1) / total;
  if (w0 == w1) return;
  const int pieces = static_cast<int>(w1 - w0 + 1);
  // Piece i's slot: only the first run can have begun before the segment.
  const int64_t head_slot = w0 * 2 + (w0 * total / nw == s0 ? 0 : 1);
  auto slot_of = [&](int i) { return i == 0 ? head_slot : (w0 + i) * 2; };

  const int part = warp / kFrags, frag = warp % kFrags, nt = frag / (D / 16);
  float m0 = -INFINITY, m1 = -INFINITY;
  for (int i = lane >> 2; i < pieces; i += 8) {
    const float4 st = p.stats[(slot_of(i) * NT + nt) * 4 + (lane & 3)];
    m0 = fmaxf(m0, st.x);
    m1 = fmaxf(m1, st.z);
  }
#pragma unroll
  for (int d = 4; d < 32; d <<= 1) {
    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, d));
    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, d));
  }
  const float r0 = safe_max(m0), r1 = safe_max(m1);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l0 = 0.f, l1 = 0.f;
#pragma unroll 4
  for (int i = part; i < pieces; i += kParts) {
    const int64_t slot = slot_of(i) * NT + nt;
    const float4 st = p.stats[slot * 4 + (lane & 3)];
    const float4 x = p.partials[(slot * (D / 16) + frag % (D / 16)) * 32 + lane];
    const float a0 = ex2_approx(st.x - r0), a1 = ex2_approx(st.z - r1);
    l0 = fmaf(st.y, a0, l0);
    l1 = fmaf(st.w, a1, l1);
    o.x = fmaf(x.x, a0, o.x);
    o.y = fmaf(x.y, a1, o.y);
    o.z = fmaf(x.z, a0, o.z);
    o.w = fmaf(x.w, a1, o.w);
  }
  if (kParts > 1) {
    acc[warp][lane] = o;
    if (lane < 4) sums[warp][lane] = make_float4(l0, l1, 0.f, 0.f);
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) {
      const float4 x = acc[k * kFrags + frag][lane], y = sums[k * kFrags + frag][lane & 3];
      o.x += x.x;
      o.y += x.y;
      o.z += x.z;
      o.w += x.w;
      l0 += y.x;
      l1 += y.y;
    }
  }
  const float i0 = inv_sum(l0), i1 = inv_sum(l1);
  const float t[4] = {o.x * i0, o.y * i1, o.z * i0, o.w * i1};
  store_out_tile<kBf16>(p, t, head0, D, nt, frag % (D / 16), nrows);
  if (kScores && frag % (D / 16) == 0 && lane < 4) {
    float2* hs = p.head_stats + static_cast<int64_t>(b) * p.hq + h0;
    const int col = nt * 8 + lane * 2;
    if (col < nrows) hs[col] = make_float2(m0, l0);
    if (col + 1 < nrows) hs[col + 1] = make_float2(m1, l1);
  }
}

// weights_out[b, kv, t] = weights_in[b, kv, t] + sum_h exp2(s[h, t] - m[h]) / l[h].
constexpr int kWeightThreads = 256;
constexpr int kWeightTokens = 1024;

__global__ void __launch_bounds__(kWeightThreads) paged_attention_weights_kernel(const __grid_constant__ AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / p.hkv, kv = blockIdx.x % p.hkv;
  const Span s = span_of(p, b);
  const int64_t head = static_cast<int64_t>(b) * p.hq + static_cast<int64_t>(kv) * p.group;
  const float* in = p.win + b * p.win_sb + kv * p.win_sh;
  float* out = p.wout + b * p.wout_sb + kv * p.wout_sh;
  const int begin = blockIdx.y * kWeightTokens;
  const int end = s.len - begin > kWeightTokens ? begin + kWeightTokens : s.len;
  for (int t = begin + threadIdx.x; t < end; t += kWeightThreads) {
    float sum = 0.f;
    if (t >= s.lo) {
      for (int h = 0; h < p.group; ++h) {
        const float2 st = p.head_stats[head + h];
        sum = fmaf(ex2_approx(p.scores[(head + h) * p.score_stride + t] - safe_max(st.x)), inv_sum(st.y), sum);
      }
    }
    out[t] = in[t] + sum;
  }
}

struct Plan {
  int group, tiles, rows, nt, ctas, warps;
  int64_t capacity;
  size_t partials, stats, scores, head_stats, score_stride, bytes;
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
  if (static_cast<int64_t>(B) * hkv * pl.tiles > INT32_MAX) {
    return fail(NESO_ERR_UNSUPPORTED, "batch x heads exceeds 2^31 - 1");
  }
  // 192 KB of rings per SM: two CTAs of four warps at D = 128, four at 64.
  const int64_t units = (pl.capacity + kUnit - 1) / kUnit * B * hkv * pl.tiles;
  const int64_t full = static_cast<int64_t>(sm_count()) * (D == 128 ? 2 : 4);
  pl.ctas = static_cast<int>(units < full ? (units > 1 ? units : 1) : full);
  pl.warps = pl.ctas * kWarps;
  pl.partials = 0;
  size_t at = round_up(static_cast<size_t>(pl.warps) * 2 * pl.nt * (D / 16) * 32 * sizeof(float4));
  pl.stats = at;
  at += round_up(static_cast<size_t>(pl.warps) * 2 * pl.nt * 4 * sizeof(float4));
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
  constexpr int smem = kWarps * kStages * 2 * kUnit * D * 2;
  auto* kern = paged_attention_kernel<kBf16, D, NT, kBias, kScores>;
  int rc = kernel_setup(reinterpret_cast<const void*>(kern), smem, nullptr);
  if (rc != NESO_OK) return rc;
  cudaError_t e = launch_pdl(kern, dim3(pl.ctas), dim3(kThreads), smem, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention launch");
  e = launch_pdl(paged_attention_join_kernel<kBf16, D, NT, kScores>, dim3(p.B * p.hkv * p.tiles),
                 dim3(kJoinWarps * 32), 0, stream, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention join launch");
  if (kScores) {
    const int64_t chunks = (pl.capacity + kWeightTokens - 1) / kWeightTokens;
    e = launch_pdl(paged_attention_weights_kernel, dim3(p.B * p.hkv, static_cast<unsigned>(chunks)),
                   dim3(kWeightThreads), 0, stream, p);
    if (e != cudaSuccess) return cuda_fail(e, "paged_attention weights launch");
  }
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
  if (!(softcap >= 0.f) || softcap > 1e30f) return fail(NESO_ERR_INVALID_ARG, "softcap must be >= 0 and finite");
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
    p.k.base = p.v.base = const_cast<void*>(q);  // nothing is read from it: no page is valid
  } else {
    if ((rc = check_cache(p.k, "k_cache")) != NESO_OK) return rc;
    if ((rc = check_cache(p.v, "v_cache")) != NESO_OK) return rc;
  }
  if ((reinterpret_cast<uintptr_t>(q) & 3u) != 0 || (reinterpret_cast<uintptr_t>(out) & 3u) != 0 || q_stride_b % 2 != 0 ||
      q_stride_h % 2 != 0) {
    return fail(NESO_ERR_MISALIGNED, "q, out and q's strides must be multiples of 4 bytes");
  }
  if (workspace == nullptr || workspace_bytes < static_cast<int64_t>(pl.bytes)) {
    return fail(NESO_ERR_INVALID_ARG, "workspace holds %lld bytes, %lld are needed",
                static_cast<long long>(workspace == nullptr ? 0 : workspace_bytes), static_cast<long long>(pl.bytes));
  }
  if (!aligned16(workspace)) return fail(NESO_ERR_MISALIGNED, "workspace is not 16-byte aligned");
  if (weights_out != nullptr && (pl.capacity + kWeightTokens - 1) / kWeightTokens > 65535) {
    return fail(NESO_ERR_UNSUPPORTED, "weights are limited to tables of 65535 x %d tokens", kWeightTokens);
  }
  p.q = static_cast<const uint16_t*>(q);
  p.tables = block_tables;
  p.lens = seq_lens;
  p.slopes = slopes;
  p.out = static_cast<uint16_t*>(out);
  char* ws = static_cast<char*>(workspace);
  p.partials = reinterpret_cast<float4*>(ws + pl.partials);
  p.stats = reinterpret_cast<float4*>(ws + pl.stats);
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
  p.page = page_divisor(static_cast<uint32_t>(page_size));
  p.score_scale = softcap > 0.f ? scale / softcap : scale * kLog2e;
  p.softcap = softcap;
  const bool bias = softcap > 0.f || slopes != nullptr;
  return dtype == NESO_BF16 ? launch_shapes<true>(p, pl, D, bias, as_stream(stream))
                            : launch_shapes<false>(p, pl, D, bias, as_stream(stream));
}

}  // extern "C"
