// Attention of new tokens over the paged cache, split over its length and
// joined.
//
// Row (t, g) of kv head h is query token t of T under query head h G + g, with
// G = Hq / Hkv. For its scores x_s = scale (q . k_s) over the visible slots,
//
//   asinh    w_s = rho(x_s)^n          softmax   w_s = exp(x_s)   (2^x_s, log2(e) in scale)
//   l = sum_s w_s + w(sink)            o = sum_s w_s v_s / l
//
// with every weight taken relative to a running reference score, so that no sum
// overflows (algebraic.py:186-204; the shifted form of kernels/flash.py:240-284).
// A row that sees no slot, or whose weights are all zero, gives zeros.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"
#include "sm100.cuh"
#include "tmap.h"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace algx {
namespace {

constexpr int kD = 64;
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kSms = 148;
// Slots a warp takes at least: fewer make more parts to join, more leave a short
// cache to few warps. bf16: one user over 2048 slots 10.2 us a pass with 64, 11.4
// with 128. float32, whose parts are joined with exact roots: 4 users over 4096
// slots 22.0 us with 64, 19.9 with 128, 26.3 with 256.
constexpr int kMinSlotsBf16 = 64, kMinSlotsF32 = 128;

struct PagedAttnArgs {
  const void *q, *k, *v;
  const float *sink, *scores;
  float* scores_out;
  void* o;
  float2* part_ml;  // (warps + items, tile_rows): reference score, sum of weights
  float* part_o;    // (warps + items, tile_rows, 64)
  float* xs;        // (B, Hkv, rows, S) scores, when weights are accumulated
  int* err;
  int64_t slots;    // S: slots of one sequence's table
  int B, T, G, rows, tile_rows, tiles, warps, log2n;
  int shift, least;  // log2 of the slots of a group; groups a warp takes at least
  int cluster;       // CTAs of an item where clusters join, 0 where a second launch does
  float scale, inv_unit;
  Sight sight;
};

// ------------------------------------------------------------- division of work
// An item is one tile of up to tile_rows rows of one kv head of one sequence; its
// work is the groups of 16 or 32 slots that its rows look at. All items' groups stand in
// one line, (sequence, head, tile, group), which is cut into equal shares, one a
// warp, whatever the sequences' lengths: a share can end one item and begin the
// next ones. Every warp writes one partial result for every item it touches, at
// index warp + item, which is different for every pair that occurs because along
// the line either the warp or the item moves on.

// Rows of an item, and the span of slots they look at.
struct Rows {
  int r0, nr, lo, hi;
  __device__ __forceinline__ Rows(const PagedAttnArgs& a, int len, int tile) {
    r0 = tile * a.tile_rows;
    nr = min(a.tile_rows, a.rows - r0);
    lo = len - a.T + r0 / a.G;
    hi = len - a.T + (r0 + nr - 1) / a.G;
  }
};
__device__ __forceinline__ Span item_span(const PagedAttnArgs& a, int len, int tile) {
  const Rows r(a, len, tile);
  return Span(a.sight, a.shift, r.lo, r.hi);
}
// Groups of one kv head of a sequence: all tiles', or those before `tiles`.
__device__ __forceinline__ int head_groups(const PagedAttnArgs& a, int len, int tiles) {
  int n = 0;
  for (int i = 0; i < tiles; ++i) n += item_span(a, len, i).total;
  return n;
}

// The line as one warp counts it, 32 sequences at a time: its length, and the
// groups before sequence `upto`. (The host refuses calls whose line could pass
// 2^31 groups.)
struct Line {
  int before, total, share;
  __device__ __forceinline__ Line(const PagedAttnArgs& a, const PagedView& pv, int upto) {
    before = total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int b = b0 + (threadIdx.x & 31);
      const int n = b < a.B ? head_groups(a, paged_len(pv, b, a.err), a.tiles) * pv.heads : 0;
      total += __reduce_add_sync(0xffffffffu, n);
      before += __reduce_add_sync(0xffffffffu, b < upto ? n : 0);
    }
    share = max(a.least, (int)(((unsigned)total + a.warps - 1) / (unsigned)a.warps));
  }
};

// A place on the line.
struct Cursor {
  int b, h, tile, item, grp, len;
  Span span;

  // The `at`-th group, found by the whole warp.
  __device__ __forceinline__ Cursor(const PagedAttnArgs& a, const PagedView& pv, int at) : span(a.sight, a.shift, -1, -1) {
    const int lane = threadIdx.x & 31;
    int per = 0;
    for (int b0 = 0;; b0 += 32) {
      const int mine = b0 + lane < a.B ? paged_len(pv, b0 + lane, a.err) : 0;
      const int each = b0 + lane < a.B ? head_groups(a, mine, a.tiles) : 0, n = each * pv.heads;
      int upto = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto > at);
      if (past == 0) {
        at -= __shfl_sync(0xffffffffu, upto, 31);
        continue;
      }
      const int src = __ffs(past) - 1;
      at -= __shfl_sync(0xffffffffu, upto - n, src);
      per = __shfl_sync(0xffffffffu, each, src);
      len = __shfl_sync(0xffffffffu, mine, src);
      b = b0 + src;
      break;
    }
    h = at / per;
    at -= h * per;
    tile = 0;
    for (;;) {
      span = item_span(a, len, tile);
      if (at < span.total) break;
      at -= span.total;
      ++tile;
    }
    grp = at;
    item = (b * pv.heads + h) * a.tiles + tile;
  }
  // The grp_-th group of one item.
  __device__ __forceinline__ Cursor(const PagedAttnArgs& a, const PagedView& pv, int item_, const Span& span_, int len_,
                                    int grp_) : item(item_), grp(grp_), len(len_), span(span_) {
    tile = item % a.tiles;
    h = item / a.tiles % pv.heads;
    b = item / a.tiles / pv.heads;
  }
  __device__ __forceinline__ int slot(const PagedAttnArgs& a) const { return span.group(grp) << a.shift; }
  // On to the next group, if there is one.
  __device__ __forceinline__ void next(const PagedAttnArgs& a, const PagedView& pv) {
    if (++grp < span.total) return;
    grp = 0;
    do {
      ++item;
      if (++tile == a.tiles) {
        tile = 0;
        if (++h == pv.heads) {
          h = 0;
          if (++b == a.B) return;
          len = paged_len(pv, b, a.err);
        }
      }
      span = item_span(a, len, tile);
    } while (span.total == 0);
  }
};

// Final factor of a row: 1 / l with the sink's weight in l, 0 for an empty row.
__device__ __forceinline__ float row_scale(float l) { return l == 0.f ? 0.f : 1.f / l; }

__device__ __forceinline__ float sink_score(const PagedAttnArgs& a, int h, int row) {
  return a.sink ? a.sink[h * a.G + row % a.G] * a.inv_unit : kNegInf;
}

// What a warp needs to know of the item it works on.
struct Item {
  int b, h, len, r0, nr, lo, hi;
  __device__ __forceinline__ Item(const PagedAttnArgs& a, const PagedView& pv, int item) {
    const int tile = item % a.tiles, bh = item / a.tiles;
    b = bh / pv.heads;
    h = bh - b * pv.heads;
    len = paged_len(pv, b, a.err);
    const Rows r(a, len, tile);
    r0 = r.r0; nr = r.nr; lo = r.lo; hi = r.hi;
  }
  // Row of q or o (in units of 64 elements), and of xs (in units of S).
  __device__ __forceinline__ int64_t q_row(const PagedAttnArgs& a, const PagedView& pv, int r) const {
    const int t = (r0 + r) / a.G;
    return (((int64_t)b * a.T + t) * pv.heads + h) * a.G + (r0 + r - t * a.G);
  }
  __device__ __forceinline__ float* x_row(const PagedAttnArgs& a, const PagedView& pv, int r) const {
    return a.xs + (((int64_t)b * pv.heads + h) * a.rows + r0 + r) * a.slots;
  }
  __device__ __forceinline__ int last_of(const PagedAttnArgs& a, int r) const { return len - a.T + (r0 + r) / a.G; }
};

// Weights are relative to a per-row reference that moves only when a weight (or the
// sum of a few) passes 2^8, so most groups need no reduction over lanes at all.
constexpr float kMove = 256.f;

// ------------------------------------------------------- float32, FMA units
// A row of 64 elements lies across 16 lanes, two slots a step. The 8 partial
// products of a lane are summed over the 16 lanes by exchanging halves (8
// shuffles for 16 slots), which leaves every slot's score in a pair of lanes, so
// each weight is evaluated once, and handed back by one shuffle a step.
template <int KIND_, int R>
struct FmaEngine {
  using T = float;
  static constexpr int kSlots = 16, kStages = 2, kCtas = 3, kRowBytes = kD * 4, kKind = KIND_;
  static constexpr bool kSwizzle = false;
  float4 q[R], acc[R];
  float m[R], turn[R], l[R];
  int last[R];

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const PagedView& pv, const Item& w) {
    const int sub = threadIdx.x & 15;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float* row = static_cast<const float*>(a.q) + w.q_row(a, pv, min(r, w.nr - 1)) * kD;
      q[r] = reinterpret_cast<const float4*>(row)[sub];
      acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      m[r] = kNegInf;
      turn[r] = weight_turn<KIND_, true>(kNegInf);
      l[r] = 0.f;
      last[r] = r < w.nr ? w.last_of(a, r) : -1;
    }
  }
  __device__ __forceinline__ void compute(const PagedAttnArgs& a, const PagedView& pv, const Item& w,
                                          const unsigned char* group, int base, int live) {
    const int lane = threadIdx.x & 31, sub = lane & 15, rl = lane >> 4;
    const float4* k = reinterpret_cast<const float4*>(group) + lane;
    const float4* v = k + kSlots * kRowBytes / 16;
    const int slot = base + (sub & ~1) + rl;  // whose score this lane ends up with
    float p[R];
    float high = 0.f;
    float x[R][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 kv = k[i * 32];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][i] = fmaf(q[r].w, kv.w, fmaf(q[r].z, kv.z, fmaf(q[r].y, kv.y, q[r].x * kv.x)));
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int half = 4; half > 0; half >>= 1) {
        const bool upper = sub & (2 * half);
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float give = upper ? x[r][i] : x[r][i + half], hold = upper ? x[r][i + half] : x[r][i];
          x[r][i] = hold + __shfl_xor_sync(0xffffffffu, give, 2 * half);
        }
      }
      float s = (x[r][0] + __shfl_xor_sync(0xffffffffu, x[r][0], 1)) * a.scale;
      if (slot >= live || !a.sight.sees(slot, last[r])) s = kNegInf;
      if (a.xs != nullptr && r < w.nr && !(sub & 1)) w.x_row(a, pv, r)[slot] = s;
      x[r][0] = s;
      p[r] = weight_of<KIND_, true>(s, turn[r], a.log2n);
      high = fmaxf(high, p[r]);
    }
    if (__any_sync(0xffffffffu, high > kMove)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = x[r][0];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (top > m[r]) {
          turn[r] = weight_turn<KIND_, true>(top);
          const float f = m[r] == kNegInf ? 0.f : weight_of<KIND_, true>(m[r], turn[r], a.log2n);
          m[r] = top;
          l[r] *= f;
          acc[r].x *= f; acc[r].y *= f; acc[r].z *= f; acc[r].w *= f;
          p[r] = weight_of<KIND_, true>(x[r][0], turn[r], a.log2n);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) l[r] += p[r];
    const bool whole = base + kSlots <= live && a.sight.sees_all(base, kSlots, w.lo, w.hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 vv = v[i * 32];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float f = __shfl_sync(0xffffffffu, p[r], (lane & 16) + 2 * i);
        if (whole || f != 0.f) {  // a weight of zero does not hide an infinity or NaN in a value
          acc[r].x = fmaf(f, vv.x, acc[r].x); acc[r].y = fmaf(f, vv.y, acc[r].y);
          acc[r].z = fmaf(f, vv.z, acc[r].z); acc[r].w = fmaf(f, vv.w, acc[r].w);
        }
      }
    }
  }
  __device__ __forceinline__ void flush(const Item& w, float2* ml, float* o) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float sum = 0.5f * row_sum<32>(l[r]);  // every slot's weight stands in two lanes
      float4 y = acc[r];
      y.x += __shfl_xor_sync(0xffffffffu, y.x, 16); y.y += __shfl_xor_sync(0xffffffffu, y.y, 16);
      y.z += __shfl_xor_sync(0xffffffffu, y.z, 16); y.w += __shfl_xor_sync(0xffffffffu, y.w, 16);
      if (r < w.nr) {
        if (lane == 0) ml[r] = make_float2(m[r], sum);
        if (lane < 16) reinterpret_cast<float4*>(o + r * kD)[lane] = y;
      }
    }
  }
};

// ----------------------------------------------------- bfloat16, matrix units
// Scores: the keys are the 16-row operand, up to 8 query rows the other one
// (S^T = K Q^T). Output: O^T = V^T P^T, the values transposed on the way from
// shared memory. The scores come out as (slot, row) and go in as (row, slot),
// one 8 x 8 transposition in registers. mma.sync rather than tcgen05: at 8 to 32
// rows the matrix work is a few percent of either unit's rate, and tcgen05 would
// put the weights through shared memory and the scores through TMEM and give up
// the independence of the warps, which hides the latency of one group's chain
// (products, weights, products) behind those of the others.
//
// Weights go into the second product as two bf16 parts each. One part, as the
// training kernels round them (kernels/flash.py:262), adds 1.6e-3 to the output's
// relative error of 1.7e-3; the second product's time does not show.
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// A pair of floats as the sum of two bf16 pairs (16 bits of each).
__device__ __forceinline__ void split_pair(float2 x, uint32_t& high, uint32_t& low) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
  const float2 r = sub2(x, __bfloat1622float2(h));
  const __nv_bfloat162 l = __floats2bfloat162_rn(r.x, r.y);
  high = *reinterpret_cast<const uint32_t*>(&h);
  low = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void load_matrices_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}


template <int KIND_, int LOG2N, int NT, bool ONE>
struct MmaEngine {
  using T = __nv_bfloat16;
  // Groups of 32 slots: copies of 4 KB. Read in 2 KB pieces memory gives a tenth
  // less (6.0 TB/s instead of 6.6 in a bare ring of this form).
  static constexpr int kSlots = 32, kStages = NT <= 2 ? 2 : 3, kCtas = NT <= 2 ? 3 : 2, kRowBytes = kD * 2,
                       kKind = KIND_;
  static constexpr int kSub = NT == 1 ? 2 : 1;  // 16-slot steps worked on together
  static constexpr bool kSwizzle = true;
  // Scores are worked on in pairs: of both columns of a lane, or, with a single
  // row (only the first column counts), of its two slots.
  static constexpr int NP = ONE ? 1 : 2;
  uint32_t q[NT][8];
  // the lane's two columns of every tile are rows 8 nt + 2 t and + 1
  float m[NT][2], o[NT][4][4];
  float2 turn[NT], l[NT];  // turn: of weight_scaled
  int last[NT][2];  // last slot the column's row sees

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const PagedView& pv, const Item& w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // row 8 nt + g, elements 16 s + 2 t and 16 s + 8 + 2 t of every step s
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const uint32_t* row =
          reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + w.q_row(a, pv, min(r, w.nr - 1)) * kD) + t;
#pragma unroll
      for (int i = 0; i < 8; ++i) q[nt][i] = r < w.nr ? row[i * 4] : 0u;
      m[nt][0] = m[nt][1] = kNegInf;
      turn[nt].x = turn[nt].y = signed_turn(weight_turn<KIND_, false>(kNegInf));
      l[nt] = make_float2(0.f, 0.f);
      last[nt][0] = w.last_of(a, nt * 8 + 2 * t);
      last[nt][1] = w.last_of(a, nt * 8 + 2 * t + 1);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][j][i] = 0.f;
    }
  }
  // O^T += V^T P^T for 16 slots. PART: values outside keep0, keep1 (bits of slots
  // 2 t, 2 t + 1 and 2 t + 8, 2 t + 9) are taken as zero. ONLY: of the rows, those
  // whose last visible slot is `only` receive the sum.
  enum { WHOLE, PART, ONLY };
  template <int MODE>
  __device__ __forceinline__ void add_values(uint32_t v_at, const uint32_t (&p)[NT][4], uint32_t keep0, uint32_t keep1,
                                             int only) {
    uint32_t b[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) b[nt][i] = transpose_8x8(p[nt][i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t v[4];
      load_matrices_trans(v, v_at ^ (j << 5));
      if constexpr (MODE != WHOLE) {
        v[0] &= keep0; v[1] &= keep0; v[2] &= keep1; v[3] &= keep1;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (MODE == ONLY) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(sum, v[0], v[1], v[2], v[3], b[nt][0], b[nt][1]);
          mma_16816(sum, v[0], v[1], v[2], v[3], b[nt][2], b[nt][3]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (last[nt][i & 1] == only) o[nt][j][i] += sum[i];
        } else {
          mma_16816(o[nt][j], v[0], v[1], v[2], v[3], b[nt][0], b[nt][1]);
          mma_16816(o[nt][j], v[0], v[1], v[2], v[3], b[nt][2], b[nt][3]);
        }
      }
    }
  }
  // Whether a kept value of the 16 slots is an infinity or NaN.
  __device__ __forceinline__ bool odd_values(uint32_t v_at, uint32_t keep0, uint32_t keep1) const {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t v[4];
      load_matrices_trans(v, v_at ^ (j << 5));
      v[0] &= keep0; v[1] &= keep0; v[2] &= keep1; v[3] &= keep1;
#pragma unroll
      for (int i = 0; i < 4; ++i) odd = odd || (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
    }
    return __any_sync(0xffffffffu, odd);
  }
  __device__ __forceinline__ float2 pair(const float (&s)[4], int i) const {
    return ONE ? make_float2(s[0], s[2]) : make_float2(s[2 * i], s[2 * i + 1]);
  }
  static __device__ __forceinline__ float signed_turn(float t) { return KIND_ == kSoftmax ? -t : t; }
  __device__ __forceinline__ float2 turns(int nt) const { return ONE ? make_float2(turn[nt].x, turn[nt].x) : turn[nt]; }

  __device__ __forceinline__ void compute(const PagedAttnArgs& a, const PagedView& pv, const Item& w,
                                          const unsigned char* group, int base, int live) {
    const bool whole = base + kSlots <= live && a.sight.sees_all(base, kSlots, w.lo, w.hi);
#pragma unroll 1
    for (int i = 0; i < kSlots / 16; i += kSub) step(a, pv, w, sm100::smem_u32(group) + i * 16 * kRowBytes, base + i * 16, live, whole);
  }
  __device__ __forceinline__ void step(const PagedAttnArgs& a, const PagedView& pv, const Item& w, uint32_t at, int base,
                                       int live, bool whole) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // what this lane points ldmatrix at: keys by (row, chunk), values by (chunk, row)
    const int r8 = lane & 7, mi = lane >> 3;
    const uint32_t k_at = at + (r8 + (mi & 1) * 8) * 128 + (((mi >> 1) ^ r8) << 4);
    const uint32_t v_at = at + kSlots * kRowBytes + (r8 + (mi >> 1) * 8) * 128 + (((mi & 1) ^ r8) << 4);
    float s[kSub][NT][4];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][nt][i] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        uint32_t k[4];
        load_matrices(k, (k_at + u * 16 * kRowBytes) ^ (c << 5));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816(s[u][nt], k[0], k[1], k[2], k[3], q[nt][2 * c], q[nt][2 * c + 1]);
      }
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = base + u * 16 + g + (i >> 1) * 8;
          if (!whole && (slot >= live || !a.sight.sees(slot, last[nt][i & 1])))
            s[u][nt][i] = kNegInf;
        }
    if (a.xs != nullptr) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = nt * 8 + 2 * t + (i & 1), slot = base + u * 16 + g + (i >> 1) * 8;
            if (r < w.nr && slot < a.slots) w.x_row(a, pv, r)[slot] = s[u][nt][i] * a.scale;
          }
    }
    float2 p[kSub][NT][NP], inc[NT];
    const float2 scale = make_float2(a.scale, a.scale);
    auto weigh = [&](int nt) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          p[u][nt][i] = weight_scaled<KIND_, LOG2N>(pair(s[u][nt], i), scale, turns(nt), a.log2n);
          inc[nt] = u + i ? add2(inc[nt], p[u][nt][i]) : p[u][nt][i];
        }
    };
    float high = 0.f;  // a weight above kMove shows in its sum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      weigh(nt);
      high = fmaxf(high, fmaxf(inc[nt].x, inc[nt].y));
    }
    if (__any_sync(0xffffffffu, high > kMove)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          float top = kNegInf;
#pragma unroll
          for (int u = 0; u < kSub; ++u) top = fmaxf(top, fmaxf(s[u][nt][c], s[u][nt][c + 2]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          top *= a.scale;
          if (top > m[nt][c]) {
            const float to = weight_turn<KIND_, false>(top);
            const float f = m[nt][c] == kNegInf ? 0.f : weight_of<KIND_, false>(m[nt][c], to, a.log2n);
            m[nt][c] = top;
            (c ? turn[nt].y : turn[nt].x) = signed_turn(to);
            (c ? l[nt].y : l[nt].x) *= f;
            if (ONE) l[nt].y *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[nt][j][c] *= f;
              o[nt][j][c + 2] *= f;
            }
          }
        }
        weigh(nt);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt] = add2(l[nt], inc[nt]);
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t pk[NT][4];  // slots g and g + 8: high parts, low parts
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 x = p[u][nt][0], y = p[u][nt][NP - 1];
        split_pair(ONE ? make_float2(x.x, 0.f) : x, pk[nt][0], pk[nt][2]);
        split_pair(ONE ? make_float2(x.y, 0.f) : y, pk[nt][1], pk[nt][3]);
      }
      const uint32_t vu = v_at + u * 16 * kRowBytes;
      if (whole) {
        add_values<WHOLE>(vu, pk, 0u, 0u, 0);
        continue;
      }
      // Slots that a row does not see hold anything, and a weight of zero does not
      // hide an infinity or NaN in a value: values that no row sees are cleared,
      // and where one of the others is not finite and the rows' tokens differ in
      // what they see, the 16 slots are added token by token.
      const int slot = base + u * 16 + 2 * t;
      auto keep = [&](int slot, int lo, int hi) {  // seen by some query with lo <= last <= hi
        auto seen = [&](int s) {
          return s < live && s <= hi && (a.sight.window == 0 || s > max(lo, 0) - a.sight.window || s < a.sight.first);
        };
        return (seen(slot) ? 0xffffu : 0u) | (seen(slot + 1) ? 0xffff0000u : 0u);
      };
      const uint32_t keep0 = keep(slot, w.lo, w.hi), keep1 = keep(slot + 8, w.lo, w.hi);
      if (w.lo == w.hi || !odd_values(vu, keep0, keep1)) {
        add_values<PART>(vu, pk, keep0, keep1, 0);
        continue;
      }
      for (int l = w.lo; l <= w.hi; ++l) add_values<ONLY>(vu, pk, keep(slot, l, l), keep(slot + 8, l, l), l);
    }
  }
  __device__ __forceinline__ void flush(const Item& w, float2* ml, float* dst) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        float sum = ONE ? l[nt].x + l[nt].y : c ? l[nt].y : l[nt].x;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int r = nt * 8 + 2 * t + c;
        if (r >= w.nr) continue;
        if (g == 0) ml[r] = make_float2(m[nt][c], sum);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dst[r * kD + 16 * j + g] = o[nt][j][c];
          dst[r * kD + 16 * j + 8 + g] = o[nt][j][c + 2];
        }
      }
  }
};

// ------------------------------------------------------------------ the kernel
// Decoding reads every key and value once and does little with it, so the kernel
// is built around the loads. Every warp works for itself: one lane asks TMA for
// the groups of the warp's share, rows of keys and of values contiguous in a page,
// kStages - 1 groups ahead into the warp's ring, across the ends of items;
// the warp takes them from there. (bf16 boxes are swizzled by 128 bytes, so that
// ldmatrix meets no bank twice.) Three CTAs of four warps with one 8 KB group on its
// way and one at work keep 96 KB an SM in flight.
// Measured: 638 MB of 8 ragged sequences up to 32768 slots, 16 heads, 105 us (6.1
// TB/s; a plain copy reads and writes 6.55); 134 MB of 512 windows of 1024 slots 31
// us; 20 rows a head over 150 MB 51 us, there bound by latency: 253 registers leave
// two warps a scheduler (0.28 instructions a cycle).
template <typename E>
constexpr int group_bytes() { return 2 * E::kSlots * E::kRowBytes; }
template <typename E>
constexpr int ring_smem() { return 1024 + kWarps * E::kStages * group_bytes<E>(); }

// Joins the CTA's warps' partial results (s_ml, s_o: by warp and row) in one, then
// the cluster's CTAs', a share of the outputs each.
template <typename E>
__device__ __forceinline__ void join_cluster(const PagedAttnArgs& a, const PagedView& pv, const Item& w, float2* s_ml,
                                             float* s_o) {
  using T = typename E::T;
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int kKind = E::kKind, kMost = 8;
  cg::cluster_group cluster = cg::this_cluster();
  const int R = a.tile_rows, C = a.cluster;
  float2* const c_ml = s_ml + kWarps * R;
  float* const c_o = s_o + kWarps * R * kD;
  for (int i = threadIdx.x; i < w.nr * kD; i += kThreads) {
    const int r = i / kD, d = i % kD;
    float M = kNegInf, L = 0.f, O = 0.f;
#pragma unroll
    for (int p = 0; p < kWarps; ++p) M = fmaxf(M, s_ml[p * R + r].x);
    const float turn = weight_turn<kKind, EXACT>(M);
#pragma unroll
    for (int p = 0; p < kWarps; ++p) {
      const float2 ml = s_ml[p * R + r];
      const float f = ml.x == kNegInf ? 0.f : weight_of<kKind, EXACT>(ml.x, turn, a.log2n);
      L = fmaf(ml.y, f, L);
      O = fmaf(s_o[(p * R + r) * kD + d], f, O);
    }
    c_o[i] = O;
    if (d == 0) c_ml[r] = make_float2(M, L);
  }
  cluster.sync();
  for (int i = (int)cluster.block_rank() * kThreads + threadIdx.x; i < w.nr * kD; i += C * kThreads) {
    const int r = i / kD, d = i % kD;
    const float sink = sink_score(a, w.h, w.r0 + r);
    float2 ml[kMost];
    float x[kMost];
    float M = sink;
#pragma unroll
    for (int c = 0; c < kMost; ++c)
      if (c < C) {
        ml[c] = *cluster.map_shared_rank(c_ml + r, c);
        x[c] = *cluster.map_shared_rank(c_o + i, c);
        M = fmaxf(M, ml[c].x);
      }
    const float turn = weight_turn<kKind, EXACT>(M);
    float L = sink == kNegInf ? 0.f : weight_of<kKind, EXACT>(sink, turn, a.log2n), O = 0.f;
#pragma unroll
    for (int c = 0; c < kMost; ++c)
      if (c < C) {
        const float f = ml[c].x == kNegInf ? 0.f : weight_of<kKind, EXACT>(ml[c].x, turn, a.log2n);
        L = fmaf(ml[c].y, f, L);
        O = fmaf(x[c], f, O);
      }
    static_cast<T*>(a.o)[w.q_row(a, pv, r) * kD + d] = from_f32<T>(O * row_scale(L));
  }
  cluster.sync();  // nobody leaves while others read its shared memory
}

// CLUSTER: a cluster of a.cluster CTAs takes one item, its groups cut evenly over
// the cluster's warps, and joins the result itself. For short caches: no line has
// to be counted and no second launch waits, which are half of their time.
template <typename E, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, E::kCtas)
    paged_attn_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                      const PagedAttnArgs a, const PagedView pv) {
  constexpr int kStages = E::kStages, kBytes = group_bytes<E>();
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t s_full[kWarps][kStages];
  __shared__ int4 s_meta[kWarps][kStages];  // item, first slot, live slots
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned char* const rings = smem_raw + (1024 - (sm100::smem_u32(smem_raw) & 1023));
  unsigned char* const ring = rings + warp * kStages * kBytes;
  uint64_t* const full = s_full[warp];
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_mbar_init();
    if (warp == 0) {
      abort_flag = 0;
      sm100::prefetch_tmap(&k_map);
      sm100::prefetch_tmap(&v_map);
    }
  }
  __syncthreads();
  pdl_wait();
  int wid = 0, left = 0, start = 0;
  if constexpr (!CLUSTER) {
    const Line line(a, pv, 0);
    wid = warp * gridDim.x + blockIdx.x;  // neighbours in the line sit on different SMs
    const int64_t from = (int64_t)wid * line.share;
    if (from >= line.total) return;  // also where no sequence has a group, which Cursor would look for
    start = (int)from;
    left = min(line.share, line.total - start);
  }
  Cursor at = [&] {
    if constexpr (CLUSTER) {
      const int item = blockIdx.x / (unsigned)a.cluster, rank = blockIdx.x - item * a.cluster;
      const int len = paged_len(pv, item / a.tiles / pv.heads, a.err);
      const Span span = item_span(a, len, item % a.tiles);
      const int n = a.cluster * kWarps, r = rank * kWarps + warp;
      start = (int)((int64_t)span.total * r / n);
      left = (int)((int64_t)span.total * (r + 1) / n) - start;
      return Cursor(a, pv, item, span, len, start);
    } else {
      return Cursor(a, pv, start);
    }
  }();
  int to_issue = left;

  // A group lies in one page, or, with pages of 16 slots and groups of 32, in two.
  const int boxes = (1 << pv.page_shift) < E::kSlots ? 2 : 1;
  int2 pid = make_int2(0, 0);
  auto read_pages = [&]() {
    if (to_issue <= 0) return;
    const int slot = at.slot(a), page = slot >> pv.page_shift;
    const int32_t* table = pv.table + (int64_t)at.b * pv.max_pages;
    pid.x = table[page];
    pid.y = boxes == 2 && slot + 16 < at.len ? table[page + 1] : pid.x;
  };
  // One lane fetches. A page that does not exist is replaced by page 0 and the
  // group's slots are masked; a box beyond the sequence is left out.
  auto issue = [&](int stage) {
    if (to_issue <= 0) return;
    const bool known = (unsigned)pid.x < (unsigned)pv.num_pages && (unsigned)pid.y < (unsigned)pv.num_pages;
    const int slot = at.slot(a);
    if (lane == 0) {
      if (!known) atomicOr(a.err, DEV_ERR_BAD_PAGE);
      s_meta[warp][stage] = make_int4(at.item, slot, known ? at.len : 0, 0);
      const bool second = boxes == 2 && slot + 16 < at.len;
      sm100::mbar_expect_tx(&full[stage], boxes == 1 || second ? kBytes : kBytes / 2);
      unsigned char* k = ring + stage * kBytes;
      const int row = (int)(paged_row(pv, known ? pid.x : 0, at.h, slot) / kD);
      sm100::tma_load_2d(k, &k_map, &full[stage], 0, row);
      sm100::tma_load_2d(k + kBytes / 2, &v_map, &full[stage], 0, row);
      if (second) {
        const int next = (int)(paged_row(pv, known ? pid.y : 0, at.h, slot + 16) / kD);
        sm100::tma_load_2d(k + kBytes / 4, &k_map, &full[stage], 0, next);
        sm100::tma_load_2d(k + 3 * kBytes / 4, &v_map, &full[stage], 0, next);
      }
    }
    if (--to_issue > 0) at.next(a, pv);
    read_pages();  // one group further ahead than the copy that needs them
  };
  read_pages();
  int item = at.item;
  Item w(a, pv, item);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);
  E e;
  e.begin(a, pv, w);

  volatile int* const abort_v = &abort_flag;
  uint32_t parity = 0;
  int stage = 0, in = kStages - 1;
  while (left > 0) {
    __syncwarp();  // every lane has taken the group whose place this copy gets
    issue(in);
    if (!sm100::mbar_wait_warp(&full[stage], parity, abort_v, a.err)) break;
    const int4 meta = s_meta[warp][stage];
    if (meta.x != item) {
      e.flush(w, a.part_ml + (int64_t)(wid + item) * a.tile_rows, a.part_o + (int64_t)(wid + item) * a.tile_rows * kD);
      item = meta.x;
      w = Item(a, pv, item);
      e.begin(a, pv, w);
    }
    e.compute(a, pv, w, ring + stage * kBytes, meta.y, meta.z);
    --left;
    in = stage;
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  pdl_trigger();  // not earlier: the join's CTAs would only wait beside this kernel's (34.0 us a pass instead of 33.0)
  if constexpr (!CLUSTER)
    e.flush(w, a.part_ml + (int64_t)(wid + item) * a.tile_rows, a.part_o + (int64_t)(wid + item) * a.tile_rows * kD);
  if (left > 0) {  // a copy did not arrive in time: let those on their way land, within limits, before the CTA ends
    volatile int quiet = 0;
    for (int i = 0; i < kStages && i < left - to_issue; ++i)
      sm100::mbar_wait(&full[(stage + i) % kStages], parity ^ (stage + i >= kStages), &quiet, nullptr);
  }
  if constexpr (CLUSTER) {
    __syncthreads();  // the rings are free
    float* const s_o = reinterpret_cast<float*>(rings);
    float2* const s_ml = reinterpret_cast<float2*>(s_o + (kWarps + 1) * a.tile_rows * kD);
    e.flush(w, s_ml + warp * a.tile_rows, s_o + warp * a.tile_rows * kD);
    __syncthreads();
    join_cluster<E>(a, pv, w, s_ml, s_o);
  }
}

// ------------------------------------------------------------------------ join
// The first blocks of a kv head join its rows' partial results, the others add the
// weights of kScoreSlots slots each over the rows. A row takes a CTA, or, where the
// rows alone fill the device, a warp: 512 rows of 14 parts
// 33.4 us a pass with CTAs and 33.7 with warps, 48 rows of 37 parts 21 and 30, 2560
// rows of 10 parts 57 and 52.
constexpr int kScoreSlots = 1024;
constexpr int kRowChunk = 64;
// Threads of a row: a warp of a CTA of four (kNarrow), a CTA of 128, each of whose
// warps finds the row's reference and sum for itself (kUsual), or, for few rows, one
// of 512 that finds them together (kWide), as the way through hundreds of parts is
// then all latency. 35 rows of 250 parts 32.2 us a pass with kUsual, 17.1 with kWide,
// 27 rows of 400 parts 21.2 and 16.3, 3 heads of 8 scored rows 19.8 and 15.5; 48 rows
// of 37 parts 19.5 and 19.9, 512 rows of 14 parts 34.4 and 41.5.
enum JoinForm { kNarrow, kUsual, kWide };
constexpr int join_threads(int form) { return form == kWide ? 512 : 128; }

// The partial results of one item: indices first .. first + count - 1, and the row
// in its tile.
struct Parts {
  int64_t first;
  int count, row;
  __device__ __forceinline__ Parts(const PagedAttnArgs& a, const PagedView& pv, const Line& line, int b, int h, int len,
                                   int r) {
    const int tile = r / a.tile_rows;
    row = r - tile * a.tile_rows;
    const int begin = line.before + h * head_groups(a, len, a.tiles) + head_groups(a, len, tile);
    const int groups = item_span(a, len, tile).total;
    const int lo = begin / line.share, hi = (begin + groups - 1) / line.share;
    first = lo + ((int64_t)b * pv.heads + h) * a.tiles + tile;
    count = groups ? hi - lo + 1 : 0;
  }
};

// Reference and sum of one row over its parts and the sink, by one warp or by all
// WARPS of the CTA, over shared memory (2 WARPS floats).
template <int KIND, bool EXACT, int WARPS>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, const Parts& p, float sink, float* s_x, float& turn,
                                         float& L) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = WARPS == 1 ? lane : threadIdx.x;
  const float2* ml = a.part_ml + p.first * a.tile_rows + p.row;
  float M = sink;  // -inf without a sink
  for (int s = at; s < p.count; s += WARPS * 32) M = fmaxf(M, ml[(int64_t)s * a.tile_rows].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  if constexpr (WARPS > 1) {
    if (lane == 0) s_x[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) M = fmaxf(M, s_x[i]);
  }
  turn = weight_turn<KIND, EXACT>(M);
  L = at == 0 && sink != kNegInf ? weight_of<KIND, EXACT>(sink, turn, a.log2n) : 0.f;
  for (int s = at; s < p.count; s += WARPS * 32) {
    const float2 x = ml[(int64_t)s * a.tile_rows];
    if (x.x != kNegInf || x.y != 0.f) L = fmaf(x.y, weight_of<KIND, EXACT>(x.x, turn, a.log2n), L);
  }
  L = row_sum<32>(L);
  if constexpr (WARPS > 1) {
    if (lane == 0) s_x[WARPS + warp] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) L += s_x[WARPS + i];
  }
}

__device__ __forceinline__ void store_row(float* o, int quad, const float4& y) { reinterpret_cast<float4*>(o)[quad] = y; }
__device__ __forceinline__ void store_row(__nv_bfloat16* o, int quad, const float4& y) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
  reinterpret_cast<uint2*>(o)[quad] =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <typename T, int KIND, int FORM>
__global__ void __launch_bounds__(join_threads(FORM)) paged_join_kernel(const PagedAttnArgs a, const PagedView pv,
                                                                        int blocks, int row_blocks) {
  constexpr bool NARROW = FORM == kNarrow;
  constexpr int kThreads = join_threads(FORM), kWarps = kThreads / 32;
  constexpr bool EXACT = sizeof(T) == 4;
  // 16 lanes hold a part's 64 values; kSets such sets work on a row, each with
  // kAhead parts loaded before the row's reference is known
  constexpr int kSets = NARROW ? 2 : kThreads / 16, kAhead = NARROW ? 8 : 4;
  const int64_t bh = blockIdx.x / (unsigned)blocks;
  const int which = (int)(blockIdx.x - bh * blocks);
  const int h = (int)(bh % pv.heads), b = (int)(bh / pv.heads);
  // lengths and sinks were there before the kernel that this one waits for
  const int len = paged_len(pv, b, a.err);
  const Line line(a, pv, b);
  if (which < row_blocks) {
    const int row = NARROW ? which * kWarps + (threadIdx.x >> 5) : which;
    if (row >= a.rows) return;  // a warp of a NARROW block
    const Parts p(a, pv, line, b, h, len, row);
    const float sink = sink_score(a, h, row);
    const int quad = threadIdx.x & 15, set = (NARROW ? threadIdx.x & 31 : threadIdx.x) >> 4;
    auto place = [&](int s) { return (p.first + s) * a.tile_rows + p.row; };
    pdl_wait();
    float ref[kAhead];
    float4 x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = set + i * kSets;
      ref[i] = s < p.count ? a.part_ml[place(s)].x : kNegInf;
      x[i] = s < p.count ? reinterpret_cast<const float4*>(a.part_o)[place(s) * 16 + quad] : make_float4(0, 0, 0, 0);
    }
    __shared__ float s_x[2 * kWarps];
    float turn, L;
    join_row<KIND, EXACT, FORM == kWide ? kWarps : 1>(a, p, sink, s_x, turn, L);
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    // a part that saw nothing has the reference -inf and zeros; one that saw only
    // NaN has -inf too, and its sums are NaN, which a factor of zero keeps
    auto add = [&](float r, const float4& y) {
      const float f = r == kNegInf ? 0.f : weight_of<KIND, EXACT>(r, turn, a.log2n);
      O.x = fmaf(y.x, f, O.x); O.y = fmaf(y.y, f, O.y); O.z = fmaf(y.z, f, O.z); O.w = fmaf(y.w, f, O.w);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(ref[i], x[i]);
#pragma unroll 4
    for (int s = set + kAhead * kSets; s < p.count; s += kSets)
      add(a.part_ml[place(s)].x, reinterpret_cast<const float4*>(a.part_o)[place(s) * 16 + quad]);
    O.x += __shfl_xor_sync(0xffffffffu, O.x, 16); O.y += __shfl_xor_sync(0xffffffffu, O.y, 16);
    O.z += __shfl_xor_sync(0xffffffffu, O.z, 16); O.w += __shfl_xor_sync(0xffffffffu, O.w, 16);
    if constexpr (!NARROW) {
      __shared__ float4 s_part[kWarps][16];
      if ((threadIdx.x & 31) < 16) s_part[threadIdx.x >> 5][quad] = O;
      __syncthreads();
      O = s_part[0][quad];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) {
        const float4 y = s_part[i][quad];
        O.x += y.x; O.y += y.y; O.z += y.z; O.w += y.w;
      }
    }
    const float inv = row_scale(L);
    const int t = row / a.G, g = row - t * a.G;
    const int64_t at = (((int64_t)b * a.T + t) * pv.heads + h) * a.G + g;
    if (set == 0)
      store_row(static_cast<T*>(a.o) + at * kD, quad, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
    return;
  }
  constexpr int kEach = kScoreSlots / kThreads;
  __shared__ float s_turn[kRowChunk], s_inv[kRowChunk];
  const int64_t s0 = (int64_t)(which - row_blocks) * kScoreSlots + threadIdx.x;
  float old[kEach], sum[kEach], next[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t s = s0 + i * kThreads;
    old[i] = s < len - a.T ? a.scores[bh * a.slots + s] : 0.f;
    sum[i] = 0.f;
  }
  auto read = [&](int r) {  // the scores of row r, one row ahead of their use
    const float* x = a.xs + (bh * a.rows + r) * a.slots;
    const int last = len - a.T + r / a.G;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t s = s0 + i * kThreads;
      next[i] = r < a.rows && s < len && a.sight.sees((int)s, last) ? x[s] : kNegInf;
    }
  };
  pdl_wait();
  read(0);
  for (int r0 = 0; r0 < a.rows; r0 += kRowChunk) {
    const int nr = min(kRowChunk, a.rows - r0);
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < nr; r += kWarps) {
      float turn, L;
      join_row<KIND, EXACT, 1>(a, Parts(a, pv, line, b, h, len, r0 + r), sink_score(a, h, r0 + r), nullptr, turn, L);
      s_turn[r] = turn;
      s_inv[r] = row_scale(L);
    }
    __syncthreads();
    for (int r = 0; r < nr; ++r) {
      float x[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) x[i] = next[i];
      read(r0 + r + 1);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (x[i] != kNegInf) sum[i] += weight_of<KIND, EXACT>(x[i], s_turn[r], a.log2n) * s_inv[r];
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t s = s0 + i * kThreads;
    if (s < a.slots) a.scores_out[bh * a.slots + s] = old[i] + sum[i];
  }
}

// Scores of a call without tokens: those of the cached slots stay, the others are zero.
__global__ void __launch_bounds__(256) paged_scores_kernel(const PagedAttnArgs a, const PagedView pv) {
  pdl_wait();
  const int64_t all = (int64_t)a.B * pv.heads * a.slots;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t bh = i / a.slots, s = i - bh * a.slots;
    const int len = pv.lens[bh / pv.heads];
    if (s == 0 && len > a.slots) atomicOr(a.err, DEV_ERR_BAD_PAGE);
    a.scores_out[i] = s < len ? a.scores[i] : 0.f;
  }
}

// ------------------------------------------------------------------------ host
struct Plan {
  int64_t rows, tile_rows, tiles, items, warps;
  size_t o, xs, bytes;
};

Plan make_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t S, bool scored, bool wide) {
  Plan p = {};
  p.rows = T * (Hq / Hkv);
  int ctas = 3;
  if (wide) {  // bf16: tiles of up to 32 rows, as even as they come
    const int64_t tiles = (p.rows + 31) / 32;
    p.tile_rows = ((p.rows + tiles - 1) / tiles + 7) / 8 * 8;
    ctas = p.tile_rows <= 16 ? 3 : 2;
  } else {
    p.tile_rows = p.rows <= 1 ? 1 : p.rows <= 2 ? 2 : p.rows <= 4 ? 4 : 8;
  }
  p.tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  p.items = B * Hkv * p.tiles;
  // one wave of CTAs, fewer where even the full tables hold less than the least a warp takes
  const int64_t least = wide ? kMinSlotsBf16 : kMinSlotsF32;
  const int64_t most = (p.items * ((S + 31) / 32 * 32) + least - 1) / least;
  p.warps = std::min<int64_t>(kSms * ctas, (most + kWarps - 1) / kWarps) * kWarps;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t parts = (size_t)((p.warps + p.items) * p.tile_rows);
  p.o = up(parts * sizeof(float2));
  p.xs = p.o + up(parts * kD * sizeof(float));
  p.bytes = p.xs + (scored ? up((size_t)(B * Hkv * p.rows * S) * sizeof(float)) : 0);
  return p;
}

// Clusters join where the caller's table bounds a warp's work to kFewGroups groups:
// CTAs an item (at most 8, one wave of them), or 0. One user over 2048 slots: 8.6 us
// a pass, 9.8 along the line; 512 windows of 1024 slots, 9 groups a warp: 39.9 us by
// clusters, 33.4 along the line, which balances them.
constexpr int kFewGroups = 4;

template <typename E>
int cluster_of(const PagedAttnArgs& a, int64_t items) {
  if (a.xs != nullptr) return 0;
  int64_t slots = a.slots;
  if (a.sight.window) slots = std::min<int64_t>(slots, (int64_t)a.sight.window + a.T + a.sight.first + 2 * E::kSlots);
  int c = 8;
  while (c > 1 && items * c > kSms * E::kCtas) c /= 2;
  const int64_t groups = (slots + E::kSlots - 1) / E::kSlots;
  return groups <= (int64_t)c * kWarps * kFewGroups && items * c <= INT32_MAX ? c : 0;
}

template <typename E, bool CLUSTER>
int attn_kernel(const PagedAttnArgs& a, const PagedView& pv, const CUtensorMap& k, const CUtensorMap& v, int64_t grid,
                cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};  // one bit per device: its shared memory limit is raised
  auto* kern = paged_attn_kernel<E, CLUSTER>;
  int dev = 0;
  ALGX_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    ALGX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_smem<E>()));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = ring_smem<E>();
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CLUSTER ? a.cluster : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  ALGX_CUDA(cudaLaunchKernelEx(&cfg, kern, k, v, a, pv));
  ALGX_LAUNCHED("paged_attn_kernel");
  return ALGX_OK;
}

template <typename E>
int attn_launch(PagedAttnArgs& a, const PagedView& pv, cudaStream_t st) {
  constexpr int dtype = sizeof(typename E::T) == 2 ? ALGX_BF16 : ALGX_F32;
  const int64_t rows = ((int64_t)pv.num_pages * pv.heads) << pv.page_shift;
  ALGX_REQUIRE(rows <= INT32_MAX, "paged cache too large");
  CUtensorMap k, v;
  const uint32_t box = std::min(E::kSlots, 1 << pv.page_shift);
  if (int e = make_tmap_2d(&k, a.k, dtype, kD, (uint64_t)rows, E::kRowBytes, kD, box, E::kSwizzle)) return e;
  if (int e = make_tmap_2d(&v, a.v, dtype, kD, (uint64_t)rows, E::kRowBytes, kD, box, E::kSwizzle)) return e;
  const int64_t items = (int64_t)a.B * pv.heads * a.tiles;
  a.cluster = cluster_of<E>(a, items);
  return a.cluster ? attn_kernel<E, true>(a, pv, k, v, items * a.cluster, st)
                   : attn_kernel<E, false>(a, pv, k, v, a.warps / kWarps, st);
}

template <int KIND, int LOG2N>
int mma_launch(PagedAttnArgs& a, const PagedView& pv, cudaStream_t st) {
  return a.rows == 1         ? attn_launch<MmaEngine<KIND, LOG2N, 1, true>>(a, pv, st)
         : a.tile_rows == 8  ? attn_launch<MmaEngine<KIND, LOG2N, 1, false>>(a, pv, st)
         : a.tile_rows == 16 ? attn_launch<MmaEngine<KIND, LOG2N, 2, false>>(a, pv, st)
         : a.tile_rows == 24 ? attn_launch<MmaEngine<KIND, LOG2N, 3, false>>(a, pv, st)
                             : attn_launch<MmaEngine<KIND, LOG2N, 4, false>>(a, pv, st);
}

template <typename T, int KIND>
int paged_launch(PagedAttnArgs& a, const PagedView& pv, cudaStream_t st) {
  int e;
  if constexpr (sizeof(T) == 2)
    e = KIND == kAsinh && a.log2n == 4 ? mma_launch<KIND, 4>(a, pv, st) : mma_launch<KIND, 0>(a, pv, st);
  else
    e = a.tile_rows == 1   ? attn_launch<FmaEngine<KIND, 1>>(a, pv, st)
        : a.tile_rows == 2 ? attn_launch<FmaEngine<KIND, 2>>(a, pv, st)
        : a.tile_rows == 4 ? attn_launch<FmaEngine<KIND, 4>>(a, pv, st)
                           : attn_launch<FmaEngine<KIND, 8>>(a, pv, st);
  if (e) return e;
  if (a.cluster) return ALGX_OK;
  const int64_t heads = (int64_t)a.B * pv.heads;
  const int64_t score_blocks = a.xs ? (a.slots + kScoreSlots - 1) / kScoreSlots : 0;
  const bool few = heads * (a.rows + score_blocks) <= kSms && (a.xs || a.warps > 64 * heads * a.tiles);
  const int form = heads * a.rows > kSms * 8 ? kNarrow : few ? kWide : kUsual;
  const int64_t row_blocks = form == kNarrow ? (a.rows + kWarps - 1) / kWarps : a.rows;
  const int64_t blocks = row_blocks + score_blocks;
  const int64_t grid = blocks * heads;
  ALGX_REQUIRE(grid <= INT32_MAX, "too many rows");
  auto* join = form == kNarrow ? paged_join_kernel<T, KIND, kNarrow>
               : form == kWide ? paged_join_kernel<T, KIND, kWide>
                               : paged_join_kernel<T, KIND, kUsual>;
  ALGX_CUDA(launch_dependent(join, dim3((unsigned)grid), dim3(join_threads(form)), 0, st, a, pv, (int)blocks,
                             (int)row_blocks));
  ALGX_LAUNCHED("paged_join_kernel");
  return ALGX_OK;
}

}  // namespace
}  // namespace algx

extern "C" {

size_t algx_paged_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t page_size,
                                      int64_t max_pages, int32_t scored, int32_t dtype) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || page_size <= 0 || max_pages <= 0) return 0;
  return algx::make_plan(B, T, Hq, Hkv, page_size * max_pages, scored != 0, dtype == ALGX_BF16).bytes;
}

int algx_paged_attn(const algx_paged_config* cfg, const void* q, const void* k_pages, const void* v_pages,
                    const int32_t* table, const int32_t* lens, const float* sink, const float* scores,
                    float* scores_out, void* o, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t num_pages,
                    int64_t page_size, int64_t max_pages, int64_t D, int32_t dtype, void* workspace,
                    size_t workspace_bytes, void* stream) {
  using namespace algx;
  PagedView pv;
  if (int s = paged_view(&pv, table, lens, B, Hkv, num_pages, page_size, max_pages, D)) return s;
  ALGX_REQUIRE(cfg != nullptr, "cfg is NULL");
  ALGX_REQUIRE(dtype == ALGX_F32 || dtype == ALGX_BF16, "dtype must be f32 or bf16");
  ALGX_REQUIRE(cfg->kind == ALGX_ATTN_ASINH || cfg->kind == ALGX_ATTN_SOFTMAX, "unknown attention kind");
  ALGX_REQUIRE(cfg->kind == ALGX_ATTN_SOFTMAX || (cfg->n >= 2 && (cfg->n & (cfg->n - 1)) == 0),
               "n must be a power of two");
  ALGX_REQUIRE(T >= 0 && Hq >= 1 && Hq % Hkv == 0, "query heads must be a multiple of the cache's heads");
  ALGX_REQUIRE(cfg->scale > 0.f && std::isfinite(cfg->scale) && cfg->inv_unit > 0.f && std::isfinite(cfg->inv_unit),
               "scale and inv_unit must be positive and finite");
  ALGX_REQUIRE(cfg->window >= 0 && cfg->first >= 0, "window and first must not be negative");
  ALGX_REQUIRE((scores == nullptr) == (scores_out == nullptr), "give scores and scores_out or neither");
  if (B == 0 || (T == 0 && scores == nullptr)) return ALGX_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    PagedAttnArgs a = {};
    a.scores = scores; a.scores_out = scores_out; a.B = (int)B; a.slots = page_size * max_pages;
    a.err = device_error_word();
    ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
    const int64_t blocks = (B * Hkv * a.slots + 1023) / 1024;
    ALGX_CUDA(launch_dependent(paged_scores_kernel, dim3((unsigned)std::min<int64_t>(blocks, kSms * 8)), dim3(256), 0, st,
                               a, pv));
    ALGX_LAUNCHED("paged_scores_kernel");
    return ALGX_OK;
  }
  ALGX_REQUIRE(q && k_pages && v_pages && o, "NULL tensor");
  ALGX_REQUIRE((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)workspace) & 15) == 0,
               "tensors must be 16-byte aligned");
  ALGX_REQUIRE(T <= INT32_MAX && T * (Hq / Hkv) <= INT32_MAX / 64, "too many rows");
  const int64_t S = page_size * max_pages;
  const Plan p = make_plan(B, T, Hq, Hkv, S, scores != nullptr, dtype == ALGX_BF16);
  ALGX_REQUIRE(p.items + p.warps <= INT32_MAX && p.items * ((S + 15) / 16) <= INT32_MAX - p.warps, "too many rows");
  ALGX_REQUIRE(workspace && workspace_bytes >= p.bytes, "workspace too small");
  PagedAttnArgs a = {};
  a.q = q; a.k = k_pages; a.v = v_pages; a.sink = sink; a.scores = scores; a.scores_out = scores_out; a.o = o;
  char* ws = static_cast<char*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(ws);
  a.part_o = reinterpret_cast<float*>(ws + p.o);
  a.xs = scores ? reinterpret_cast<float*>(ws + p.xs) : nullptr;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  a.slots = S; a.B = (int)B; a.T = (int)T; a.G = (int)(Hq / Hkv); a.rows = (int)p.rows;
  a.tile_rows = (int)p.tile_rows; a.tiles = (int)p.tiles; a.warps = (int)p.warps;
  const bool soft = cfg->kind == ALGX_ATTN_SOFTMAX;
  if (!soft)
    while ((1 << a.log2n) < cfg->n) ++a.log2n;
  a.scale = soft ? cfg->scale * kLog2e : cfg->scale;
  a.inv_unit = soft ? cfg->inv_unit * kLog2e : cfg->inv_unit;
  a.sight = {cfg->window, cfg->first};
  a.shift = dtype == ALGX_BF16 ? 5 : 4;
  a.least = (dtype == ALGX_BF16 ? kMinSlotsBf16 : kMinSlotsF32) >> a.shift;
  if (dtype == ALGX_BF16)
    return soft ? paged_launch<__nv_bfloat16, kSoftmax>(a, pv, st) : paged_launch<__nv_bfloat16, kAsinh>(a, pv, st);
  return soft ? paged_launch<float, kSoftmax>(a, pv, st) : paged_launch<float, kAsinh>(a, pv, st);
}

}  // extern "C"
