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
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged_common.cuh"
#include "sm100.cuh"
#include "tmap.h"
#include "vec_io.cuh"

namespace algx {
namespace {

constexpr int kD = 64;
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMinGroups = 8;  // groups of 16 slots a split takes at least

struct PagedAttnArgs {
  const void *q, *k, *v;
  const float *sink, *scores;
  float* scores_out;
  void* o;
  float2* part_ml;  // (B, Hkv, rows, splits): reference score, sum of weights
  float* part_o;    // (B, Hkv, rows, splits, 64)
  float* xs;        // (B, Hkv, rows, S) scores, when weights are accumulated
  int* err;
  int64_t slots;    // S: slots of one sequence's table
  int T, G, rows, tile_rows, tiles, splits, log2n;
  bool direct;      // one split and no scores: outputs are written without a join
  float scale, inv_unit;
  Sight sight;
};

// Final factor of a row: 1 / l with the sink's weight in l, 0 for an empty row.
__device__ __forceinline__ float row_scale(float l) { return l == 0.f ? 0.f : 1.f / l; }

// What one CTA works on.
struct Work {
  int b, h, split, r0, nr, len, lo, hi;
  __device__ __forceinline__ Work(const PagedAttnArgs& a, const PagedView& pv) {
    unsigned idx = blockIdx.x;
    const unsigned tile = idx % (unsigned)a.tiles;
    idx /= (unsigned)a.tiles;
    split = (int)(idx % (unsigned)a.splits);
    idx /= (unsigned)a.splits;
    b = (int)(idx / (unsigned)pv.heads);
    h = (int)(idx - (unsigned)b * (unsigned)pv.heads);
    len = paged_len(pv, b, a.err);
    r0 = (int)tile * a.tile_rows;
    nr = min(a.tile_rows, a.rows - r0);
    lo = len - a.T + r0 / a.G;
    hi = len - a.T + (r0 + nr - 1) / a.G;
  }
  __device__ __forceinline__ int64_t kv(const PagedView& pv) const { return (int64_t)b * pv.heads + h; }
  // Element offset / 64 of a row of q or o.
  __device__ __forceinline__ int64_t q_row(const PagedAttnArgs& a, const PagedView& pv, int row) const {
    const int t = row / a.G;
    return (((int64_t)b * a.T + t) * pv.heads + h) * a.G + (row - t * a.G);
  }
};

__device__ __forceinline__ float sink_score(const PagedAttnArgs& a, int h, int row) {
  return a.sink ? a.sink[h * a.G + row % a.G] * a.inv_unit : kNegInf;
}

// Joins the CTA's PARTS partial results of each row: into the workspace, or, when
// no other split has a share, into the output.
template <typename T, int KIND, int PARTS>
__device__ __forceinline__ void merge_parts(const PagedAttnArgs& a, const PagedView& pv, const Work& w,
                                            const float* s_o, const float2* s_ml) {
  constexpr bool EXACT = sizeof(T) == 4;
  for (int i = threadIdx.x; i < w.nr * kD; i += kThreads) {
    const int r = i / kD, d = i % kD;
    const float sink = a.direct ? sink_score(a, w.h, w.r0 + r) : kNegInf;
    float M = sink;
    for (int p = 0; p < PARTS; ++p) M = fmaxf(M, s_ml[r * PARTS + p].x);
    const float t = weight_turn<KIND, EXACT>(M);
    float L = sink == kNegInf ? 0.f : weight_of<KIND, EXACT>(sink, t, a.log2n), O = 0.f;
    for (int p = 0; p < PARTS; ++p) {
      const float2 ml = s_ml[r * PARTS + p];
      if (ml.x == kNegInf && ml.y == 0.f) continue;
      const float f = weight_of<KIND, EXACT>(ml.x, t, a.log2n);
      L = fmaf(ml.y, f, L);
      O = fmaf(s_o[(r * PARTS + p) * kD + d], f, O);
    }
    if (a.direct) {
      static_cast<T*>(a.o)[w.q_row(a, pv, w.r0 + r) * kD + d] = from_f32<T>(O * row_scale(L));
    } else {
      const int64_t at = (w.kv(pv) * a.rows + w.r0 + r) * a.splits + w.split;
      if (d == 0) a.part_ml[at] = make_float2(M, L);
      a.part_o[at * kD + d] = O;
    }
  }
}

// ------------------------------------------------------- any I/O type, FMA units
// One CTA per (split, row tile, kv head, sequence); a warp takes every fourth
// group of the split. A row of 64 elements lies across TPR lanes, so a warp
// reads 32 / TPR slots at once, and each such lane group keeps its own running
// reference, sum and output, merged over the CTA at the end.
template <typename T, int KIND, int R>
__global__ void __launch_bounds__(kThreads) paged_attn_kernel(const PagedAttnArgs a, const PagedView pv) {
  using V = Vec<T>;
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int kParts = kWarps * V::RPW;
  __shared__ float s_o[R][kParts][kD];
  __shared__ float2 s_ml[R][kParts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % V::TPR, rl = lane / V::TPR;
  const Work w(a, pv);
  const Span span(a.sight, w.lo, w.hi);
  const int per = max(kMinGroups, (span.total + a.splits - 1) / a.splits);
  const int g_end = (int)min((int64_t)span.total, (int64_t)(w.split + 1) * per);

  float q[R][V::N];
  int last[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(w.r0 + r, a.rows - 1);
    last[r] = r < w.nr ? w.len - a.T + row / a.G : -1;
    unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + w.q_row(a, pv, row) * kD + sub * V::N), q[r]);
  }
  float m[R], turn[R], l[R], acc[R][V::N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = kNegInf;
    turn[r] = weight_turn<KIND, EXACT>(kNegInf);
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < V::N; ++i) acc[r][i] = 0.f;
  }
  for (int64_t g = (int64_t)w.split * per + warp; g < g_end; g += kWarps) {
    const int base = span.slot((int)g);
    const int pid = pv.table[(int64_t)w.b * pv.max_pages + (base >> pv.page_shift)];
    if (pid < 0 || pid >= pv.num_pages) {
      if (lane == 0) atomicOr(a.err, DEV_ERR_BAD_PAGE);
      if (a.xs != nullptr && lane < 16)
        for (int r = 0; r < w.nr; ++r) a.xs[(w.kv(pv) * a.rows + w.r0 + r) * a.slots + base + lane] = kNegInf;
      continue;
    }
    const int64_t at = paged_row(pv, pid, w.h, base) + sub * V::N;
#pragma unroll 2
    for (int j = 0; j < 16; j += V::RPW) {
      const int s = base + j + rl;
      float kf[V::N], vf[V::N];
      const bool live = s < w.len;
      unpack<T>(live ? ld_stream(static_cast<const T*>(a.k) + at + (j + rl) * kD) : make_uint4(0, 0, 0, 0), kf);
      unpack<T>(live ? ld_stream(static_cast<const T*>(a.v) + at + (j + rl) * kD) : make_uint4(0, 0, 0, 0), vf);
      float xr[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < V::N; ++i) x = fmaf(q[r][i], kf[i], x);
        xr[r] = row_sum<V::TPR>(x) * a.scale;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float x = xr[r];
        if (!a.sight.sees(s, last[r])) continue;
        if (a.xs != nullptr && sub == 0)
          a.xs[(w.kv(pv) * a.rows + w.r0 + r) * a.slots + s] = x;
        if (x == kNegInf) continue;  // weight 0
        if (x > m[r]) {
          const float nt = weight_turn<KIND, EXACT>(x);
          const float f = m[r] == kNegInf ? 0.f : weight_of<KIND, EXACT>(m[r], nt, a.log2n);
          m[r] = x;
          turn[r] = nt;
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < V::N; ++i) acc[r][i] *= f;
        }
        const float p = weight_of<KIND, EXACT>(x, turn[r], a.log2n);
        l[r] += p;
#pragma unroll
        for (int i = 0; i < V::N; ++i) acc[r][i] = fmaf(p, vf[i], acc[r][i]);
      }
    }
  }
  const int part = warp * V::RPW + rl;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (sub == 0) s_ml[r][part] = make_float2(m[r], l[r]);
#pragma unroll
    for (int i = 0; i < V::N; ++i) s_o[r][part][sub * V::N + i] = acc[r][i];
  }
  __syncthreads();
  merge_parts<T, KIND, kParts>(a, pv, w, &s_o[0][0][0], &s_ml[0][0]);
}

// ----------------------------------------------------- bfloat16, matrix units
// Decoding reads every key and value once and does little with it, so this
// kernel is built around the loads. Every warp works for itself: one lane asks
// TMA for groups of 16 slots (2 KB of keys, 2 KB of values, contiguous in a
// page) into the warp's ring, kStages - 1 groups ahead, and the warp takes them
// from there in the registers of the matrix instructions. The boxes are swizzled
// by 128 bytes, so reading eight rows at once meets no bank twice.
//
// Scores: the keys are the 16-row operand, up to 8 query rows the other one
// (S^T = K Q^T). Output: O^T = V^T P^T, the values transposed on the way from
// shared memory. The scores come out as (slot, row) and go in as (row, slot),
// one 8 x 8 transposition in registers. mma.sync rather than tcgen05: at 8 to 32
// rows the matrix work is a few percent of either unit's rate, and tcgen05 would
// put the weights through shared memory and the scores through TMEM and give up
// the independence of the warps, which hides the latency of one group's chain
// (products, weights, products) behind those of the others.
//
// Weights are relative to a per-row reference that moves only when a weight
// passes 2^8, so most groups need no reduction over lanes at all. Weights are
// rounded to bf16 for the second product, as the forward kernels round them
// (kernels/flash.py:262), while their sum keeps the unrounded ones.
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
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
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

constexpr int kGroupBytes = 2 * 16 * kD * 2;  // keys and values of 16 slots
__host__ __device__ constexpr int mma_ctas(int nt) { return nt == 1 ? 4 : nt == 2 ? 3 : 2; }
__host__ __device__ constexpr int mma_stages(int nt) { return nt == 1 ? 3 : nt == 2 ? 4 : 6; }
__host__ __device__ constexpr int mma_smem(int nt) {
  return 1024 + kWarps * mma_stages(nt) * (kGroupBytes + (int)sizeof(uint64_t));
}
constexpr float kMove = 256.f;  // a weight above it moves the row's reference

template <int KIND, int LOG2N, int NT, bool ONE>
__global__ void __launch_bounds__(kThreads, mma_ctas(NT))
    paged_attn_mma_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                          const PagedAttnArgs a, const PagedView pv) {
  using T = __nv_bfloat16;
  // Scores are worked on in pairs: of both columns of a lane, or, with a single
  // row (only the first column counts), of its two slots.
  constexpr int NP = ONE ? 1 : 2, kStages = mma_stages(NT);
  extern __shared__ unsigned char smem_raw[];
  __shared__ int abort_flag;
  unsigned char* const smem = smem_raw + (1024 - (sm100::smem_u32(smem_raw) & 1023));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* const ring = smem + warp * kStages * kGroupBytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + kWarps * kStages * kGroupBytes) + warp * kStages;
  float* const s_o = reinterpret_cast<float*>(smem);  // takes the rings' place once the groups are done
  float2* const s_ml = reinterpret_cast<float2*>(s_o + NT * 8 * kWarps * kD);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&full[i], 1);
    sm100::fence_mbar_init();
  }
  if (threadIdx.x == 0) abort_flag = 0;
  const Work w(a, pv);
  const Span span(a.sight, w.lo, w.hi);
  const int per = max(kMinGroups, (span.total + a.splits - 1) / a.splits);
  const int g_end = (int)min((int64_t)span.total, (int64_t)(w.split + 1) * per);
  const int32_t* table = pv.table + (int64_t)w.b * pv.max_pages;

  // One lane fetches; a page that does not exist is replaced by page 0 and its
  // slots are masked.
  auto page_of = [&](int grp) { return grp < g_end ? table[span.slot(grp) >> pv.page_shift] : 0; };
  uint32_t missing = 0;  // stages whose page does not exist
  auto issue = [&](int stage, int grp, int pid) {
    if (grp >= g_end) return;
    missing &= ~(1u << stage);
    if ((unsigned)pid >= (unsigned)pv.num_pages) {
      missing |= 1u << stage;
      if (lane == 0) atomicOr(a.err, DEV_ERR_BAD_PAGE);
      pid = 0;
    }
    if (lane != 0) return;
    const int row = (int)(paged_row(pv, pid, w.h, span.slot(grp)) / kD);
    sm100::mbar_expect_tx(&full[stage], kGroupBytes);
    sm100::tma_load_2d(ring + stage * kGroupBytes, &k_map, &full[stage], 0, row);
    sm100::tma_load_2d(ring + stage * kGroupBytes + kGroupBytes / 2, &v_map, &full[stage], 0, row);
  };
  int grp = (int)min((int64_t)g_end, (int64_t)w.split * per + warp);
  int ahead = page_of(grp);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    const int pid = ahead;
    ahead = page_of(grp + (i + 1) * kWarps);
    issue(i, grp + i * kWarps, pid);
  }

  // queries: row 8 nt + g, elements 16 s + 2 t and 16 s + 8 + 2 t of every step
  uint32_t q[NT][8];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g;
    const uint32_t* row = reinterpret_cast<const uint32_t*>(
        static_cast<const T*>(a.q) + w.q_row(a, pv, w.r0 + min(r, w.nr - 1)) * kD) + t;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[nt][i] = r < w.nr ? row[i * 4] : 0u;
  }
  // what this lane points ldmatrix at: keys by (row, chunk), values by (chunk, row)
  const uint32_t ring_at = sm100::smem_u32(ring);
  const int r8 = lane & 7, mi = lane >> 3;
  const uint32_t k_at = ring_at + (r8 + (mi & 1) * 8) * 128 + (((mi >> 1) ^ r8) << 4);
  const uint32_t v_at = ring_at + kGroupBytes / 2 + (r8 + (mi >> 1) * 8) * 128 + (((mi & 1) ^ r8) << 4);
  // the lane's two columns of every tile are rows 8 nt + 2 t and + 1
  float m[NT][2], o[NT][4][4];
  float2 turn[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kNegInf;
    turn[nt].x = turn[nt].y = weight_turn<KIND, false>(kNegInf);
    l[nt] = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][j][i] = 0.f;
  }

  auto last_of = [&](int r) { return w.len - a.T + (w.r0 + r) / a.G; };
  // O^T += V^T P^T for the weights p (two packed pairs a tile) and the group's
  // values. keep(i): bits of the values of slots 2 t, 2 t + 1 (i = 0) or 2 t + 8,
  // 2 t + 9 that exist. With one_token, only for the rows whose last visible slot
  // is `only`.
  auto add_values = [&](int stage, const uint32_t (&p)[NT][2], auto masked, uint32_t keep0, uint32_t keep1,
                        auto one_token, int only) {
    uint32_t b[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      b[nt][0] = transpose_8x8(p[nt][0]);
      b[nt][1] = transpose_8x8(p[nt][1]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t v[4];
      load_matrices_trans(v, (v_at + stage * kGroupBytes) ^ (j << 5));
      if constexpr (decltype(masked)::value) {
        v[0] &= keep0; v[1] &= keep0; v[2] &= keep1; v[3] &= keep1;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (decltype(one_token)::value) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(sum, v[0], v[1], v[2], v[3], b[nt][0], b[nt][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (last_of(nt * 8 + 2 * t + (i & 1)) == only) o[nt][j][i] += sum[i];
        } else {
          mma_16816(o[nt][j], v[0], v[1], v[2], v[3], b[nt][0], b[nt][1]);
        }
      }
    }
  };
  // pair i of a tile's four scores, and its reference
  auto pair = [&](const float (&s)[4], int i) { return ONE ? make_float2(s[0], s[2]) : make_float2(s[2 * i], s[2 * i + 1]); };
  auto turns = [&](int nt) { return ONE ? make_float2(turn[nt].x, turn[nt].x) : turn[nt]; };

  auto compute = [&](int stage, int base, int live) {
    float s[NT][4], s2[NT][4];  // two chains of products, for shorter ones
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.f;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      uint32_t k[4];
      load_matrices(k, (k_at + stage * kGroupBytes) ^ (step << 5));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma_16816(step & 1 ? s2[nt] : s[nt], k[0], k[1], k[2], k[3], q[nt][2 * step], q[nt][2 * step + 1]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = (s[nt][i] + s2[nt][i]) * a.scale;
    const bool whole = base + 16 <= live && a.sight.sees_group(base, w.lo, w.hi);
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = base + g + (i >> 1) * 8;
          if (slot >= live || !a.sight.sees(slot, last_of(nt * 8 + 2 * t + (i & 1)))) s[nt][i] = kNegInf;
        }
    }
    if (a.xs != nullptr) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = nt * 8 + 2 * t + (i & 1), slot = base + g + (i >> 1) * 8;
          if (r < w.nr) a.xs[(w.kv(pv) * a.rows + w.r0 + r) * a.slots + slot] = s[nt][i];
        }
    }
    float2 p[NT][NP];
    float high = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        p[nt][i] = weight_pair<KIND, LOG2N>(pair(s[nt], i), turns(nt), a.log2n);
        high = fmaxf(high, fmaxf(p[nt][i].x, p[nt][i].y));
      }
    if (__any_sync(0xffffffffu, high > kMove)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          float top = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          if (top > m[nt][c]) {
            const float to = weight_turn<KIND, false>(top);
            const float f = m[nt][c] == kNegInf ? 0.f : weight_of<KIND, false>(m[nt][c], to, a.log2n);
            m[nt][c] = top;
            (c ? turn[nt].y : turn[nt].x) = to;
            (c ? l[nt].y : l[nt].x) *= f;
            if (ONE) l[nt].y *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[nt][j][c] *= f;
              o[nt][j][c + 2] *= f;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) p[nt][i] = weight_pair<KIND, LOG2N>(pair(s[nt], i), turns(nt), a.log2n);
      }
    }
    uint32_t pk[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < NP; ++i) l[nt] = add2(l[nt], p[nt][i]);
      pk[nt][0] = ONE ? pack_pair(p[nt][0].x, 0.f) : pack_pair(p[nt][0].x, p[nt][0].y);
      pk[nt][1] = ONE ? pack_pair(p[nt][0].y, 0.f) : pack_pair(p[nt][NP - 1].x, p[nt][NP - 1].y);
    }
    if (whole) {
      add_values(stage, pk, std::false_type{}, 0u, 0u, std::false_type{}, 0);
      return;
    }
    // Slots beyond the sequence hold anything: a weight of zero does not hide an
    // infinity or NaN in a value, so their values are cleared. Where the rows of
    // different tokens see different slots, the group is added token by token.
    auto keep = [&](int i, int last) {
      const int slot = base + 2 * t + i * 8;
      return (slot < live && a.sight.sees(slot, last) ? 0xffffu : 0u) |
             (slot + 1 < live && a.sight.sees(slot + 1, last) ? 0xffff0000u : 0u);
    };
    if (w.lo == w.hi) {
      add_values(stage, pk, std::true_type{}, keep(0, w.hi), keep(1, w.hi), std::false_type{}, 0);
    } else {
      for (int last = w.lo; last <= w.hi; ++last)
        add_values(stage, pk, std::true_type{}, keep(0, last), keep(1, last), std::true_type{}, last);
    }
  };

  // Page numbers are read one group further ahead than the copies that need them.
  volatile int* const abort_v = &abort_flag;
  uint32_t parity = 0;
  int stage = 0, in = kStages - 1;
  bool ok = true;
  __syncthreads();
  while (grp < g_end) {
    __syncwarp();  // every lane has taken the group whose place this copy gets
    issue(in, grp + (kStages - 1) * kWarps, ahead);
    ahead = page_of(grp + kStages * kWarps);
    ok = sm100::mbar_wait_warp(&full[stage], parity, abort_v, a.err);
    if (!ok) break;
    compute(stage, span.slot(grp), missing >> stage & 1 ? 0 : w.len);
    grp += kWarps;
    in = stage;
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (!ok) {  // a copy did not arrive in time: let those on their way land, within limits, before the CTA ends
    volatile int quiet = 0;
    for (int i = 0; i < kStages && grp + i * kWarps < g_end; ++i)
      sm100::mbar_wait(&full[(stage + i) % kStages], parity ^ (stage + i >= kStages), &quiet, nullptr);
  }
  pdl_trigger();
  __syncthreads();  // the rings are free

#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float sum = c ? (ONE ? 0.f : l[nt].y) : (ONE ? l[nt].x + l[nt].y : l[nt].x);
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      const int r = nt * 8 + 2 * t + c;
      if (g == 0) s_ml[r * kWarps + warp] = make_float2(m[nt][c], sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s_o[(r * kWarps + warp) * kD + 16 * j + g] = o[nt][j][c];
        s_o[(r * kWarps + warp) * kD + 16 * j + 8 + g] = o[nt][j][c + 2];
      }
    }
  }
  __syncthreads();
  merge_parts<T, KIND, kWarps>(a, pv, w, s_o, s_ml);
}

// ------------------------------------------------------------------------ join
// Blocks below `rows` join one row's splits; the others add the weights of their
// slots over the rows of one kv head.
constexpr int kScoreSlots = 1024;
constexpr int kRowChunk = 64;

// Reference and sum of one row over its splits and the sink, by one warp.
template <int KIND, bool EXACT>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, int64_t row, float sink, float& turn, float& L) {
  const int lane = threadIdx.x & 31;
  const float2* ml = a.part_ml + row * a.splits;
  float M = sink;  // -inf without a sink
  for (int s = lane; s < a.splits; s += 32) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  turn = weight_turn<KIND, EXACT>(M);
  L = lane == 0 && sink != kNegInf ? weight_of<KIND, EXACT>(sink, turn, a.log2n) : 0.f;
  for (int s = lane; s < a.splits; s += 32) {
    const float2 x = ml[s];
    if (x.x != kNegInf || x.y != 0.f) L = fmaf(x.y, weight_of<KIND, EXACT>(x.x, turn, a.log2n), L);
  }
  L = row_sum<32>(L);
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const PagedAttnArgs a, const PagedView pv, int blocks) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int kQuads = kD / 4, kGroups = kThreads / kQuads;
  pdl_wait();
  const int64_t bh = blockIdx.x / (unsigned)blocks;
  const int which = (int)(blockIdx.x - bh * blocks);
  const int h = (int)(bh % pv.heads), b = (int)(bh / pv.heads);
  if (which < a.rows) {
    __shared__ float4 s_part[kGroups][kQuads];
    const int64_t row = bh * a.rows + which;
    float turn, L;
    join_row<KIND, EXACT>(a, row, sink_score(a, h, which), turn, L);
    const int quad = threadIdx.x % kQuads, grp = threadIdx.x / kQuads;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = grp; s < a.splits; s += kGroups) {
      const float2 ml = a.part_ml[row * a.splits + s];
      const float4 x = reinterpret_cast<const float4*>(a.part_o)[(row * a.splits + s) * kQuads + quad];
      const float f = ml.x == kNegInf && ml.y == 0.f ? 0.f : weight_of<KIND, EXACT>(ml.x, turn, a.log2n);
      O.x = fmaf(x.x, f, O.x); O.y = fmaf(x.y, f, O.y); O.z = fmaf(x.z, f, O.z); O.w = fmaf(x.w, f, O.w);
    }
    s_part[grp][quad] = O;
    __syncthreads();
    if (threadIdx.x < kD) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) sum += reinterpret_cast<const float*>(s_part[i])[threadIdx.x];
      const int t = which / a.G, g = which - t * a.G;
      const int64_t at = (((int64_t)b * a.T + t) * pv.heads + h) * a.G + g;
      static_cast<T*>(a.o)[at * kD + threadIdx.x] = from_f32<T>(sum * row_scale(L));
    }
    return;
  }
  __shared__ float s_turn[kRowChunk], s_inv[kRowChunk];
  const int len = paged_len(pv, b, a.err);
  const int64_t s0 = (int64_t)(which - a.rows) * kScoreSlots;
  float sum[kScoreSlots / kThreads];
#pragma unroll
  for (int i = 0; i < kScoreSlots / kThreads; ++i) sum[i] = 0.f;
  for (int r0 = 0; r0 < a.rows; r0 += kRowChunk) {
    const int nr = min(kRowChunk, a.rows - r0);
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < nr; r += kWarps) {
      float turn, L;
      join_row<KIND, EXACT>(a, bh * a.rows + r0 + r, sink_score(a, h, r0 + r), turn, L);
      s_turn[r] = turn;
      s_inv[r] = row_scale(L);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kScoreSlots / kThreads; ++i) {
      const int64_t s = s0 + threadIdx.x + (int64_t)i * kThreads;
      if (s >= len) continue;
      for (int r = 0; r < nr; ++r) {
        if (!a.sight.sees((int)s, len - a.T + (r0 + r) / a.G)) continue;
        const float x = a.xs[(bh * a.rows + r0 + r) * a.slots + s];
        sum[i] += weight_of<KIND, EXACT>(x, s_turn[r], a.log2n) * s_inv[r];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kScoreSlots / kThreads; ++i) {
    const int64_t s = s0 + threadIdx.x + (int64_t)i * kThreads;
    if (s >= a.slots) continue;
    const float old = s < len - a.T ? a.scores[bh * a.slots + s] : 0.f;
    a.scores_out[bh * a.slots + s] = old + sum[i];
  }
}

// ------------------------------------------------------------------------ host
struct Plan {
  int64_t rows, tile_rows, tiles, splits;
  size_t ml, o, xs, bytes;
};

// Slots a query can see at most, in groups of 16.
int64_t visible_groups(int64_t S, int64_t T, int64_t window, int64_t first) {
  const int64_t all = (S + 15) / 16;
  if (window == 0) return all;
  return std::min(all, (window + T + 15) / 16 + 1 + (std::min(first, S) + 15) / 16);
}

Plan make_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t S, int64_t window, int64_t first, bool scored,
               bool wide) {
  Plan p = {};
  p.rows = T * (Hq / Hkv);
  if (wide)  // bf16: tiles of up to 32 rows, as even as they come
    p.tile_rows = (((p.rows + 31) / 32 - 1 + p.rows) / ((p.rows + 31) / 32) + 7) / 8 * 8;
  else
    p.tile_rows = p.rows <= 1 ? 1 : p.rows <= 2 ? 2 : p.rows <= 4 ? 4 : 8;
  p.tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  const int64_t groups = visible_groups(S, T, window, first);
  const int64_t base = std::max<int64_t>(1, B * Hkv * p.tiles);
  const int64_t want = (148 * 8 + base - 1) / base;
  p.splits = std::max<int64_t>(1, std::min(want, (groups + kMinGroups - 1) / kMinGroups));
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.ml = 0;
  p.o = up((size_t)(B * Hkv * p.rows * p.splits) * sizeof(float2));
  p.xs = p.o + up((size_t)(B * Hkv * p.rows * p.splits) * kD * sizeof(float));
  p.bytes = p.xs + (scored ? up((size_t)(B * Hkv * p.rows * S) * sizeof(float)) : 0);
  return p;
}

template <int KIND, int LOG2N, int NT, bool ONE>
int mma_launch(const PagedAttnArgs& a, const PagedView& pv, const CUtensorMap& k, const CUtensorMap& v, unsigned grid,
               cudaStream_t st) {
  auto* kern = paged_attn_mma_kernel<KIND, LOG2N, NT, ONE>;
  static std::atomic<uint64_t> ready{0};  // one bit per device: its shared memory limit is raised
  int dev = 0;
  ALGX_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    ALGX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, mma_smem(NT)));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  kern<<<grid, kThreads, mma_smem(NT), st>>>(k, v, a, pv);
  return ALGX_OK;
}

template <int KIND, int LOG2N>
int mma_launch_rows(const PagedAttnArgs& a, const PagedView& pv, unsigned grid, cudaStream_t st) {
  const int64_t rows = ((int64_t)pv.num_pages * pv.heads) << pv.page_shift;
  ALGX_REQUIRE(rows <= INT32_MAX, "paged cache too large");
  CUtensorMap k, v;
  if (int e = make_tmap_2d(&k, a.k, ALGX_BF16, kD, (uint64_t)rows, kD * 2, kD, 16, true)) return e;
  if (int e = make_tmap_2d(&v, a.v, ALGX_BF16, kD, (uint64_t)rows, kD * 2, kD, 16, true)) return e;
  return a.rows == 1         ? mma_launch<KIND, LOG2N, 1, true>(a, pv, k, v, grid, st)
         : a.tile_rows == 8  ? mma_launch<KIND, LOG2N, 1, false>(a, pv, k, v, grid, st)
         : a.tile_rows == 16 ? mma_launch<KIND, LOG2N, 2, false>(a, pv, k, v, grid, st)
         : a.tile_rows == 24 ? mma_launch<KIND, LOG2N, 3, false>(a, pv, k, v, grid, st)
                             : mma_launch<KIND, LOG2N, 4, false>(a, pv, k, v, grid, st);
}

template <typename T, int KIND>
int paged_launch(const PagedAttnArgs& a, const PagedView& pv, const Plan& p, int64_t B, cudaStream_t st) {
  const int64_t grid = B * pv.heads * p.splits * p.tiles;
  ALGX_REQUIRE(grid <= INT32_MAX, "too many rows");
  if constexpr (sizeof(T) == 2) {
    const int e = KIND == kAsinh && a.log2n == 4 ? mma_launch_rows<KIND, 4>(a, pv, (unsigned)grid, st)
                                                 : mma_launch_rows<KIND, 0>(a, pv, (unsigned)grid, st);
    if (e) return e;
  } else {
    auto* kern = p.tile_rows == 1   ? paged_attn_kernel<T, KIND, 1>
                 : p.tile_rows == 2 ? paged_attn_kernel<T, KIND, 2>
                 : p.tile_rows == 4 ? paged_attn_kernel<T, KIND, 4>
                                    : paged_attn_kernel<T, KIND, 8>;
    kern<<<(unsigned)grid, kThreads, 0, st>>>(a, pv);
  }
  ALGX_LAUNCHED("paged_attn_kernel");
  if (a.direct) return ALGX_OK;
  const int64_t blocks = a.rows + (a.xs ? (a.slots + kScoreSlots - 1) / kScoreSlots : 0);
  ALGX_REQUIRE(blocks * B * pv.heads <= INT32_MAX, "too many rows");
  ALGX_CUDA(launch_dependent(paged_join_kernel<T, KIND>, dim3((unsigned)(blocks * B * pv.heads)), dim3(kThreads), 0, st,
                             a, pv, (int)blocks));
  ALGX_LAUNCHED("paged_join_kernel");
  return ALGX_OK;
}

}  // namespace
}  // namespace algx

extern "C" {

size_t algx_paged_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t page_size,
                                      int64_t max_pages, int64_t window, int64_t first, int32_t scored,
                                      int32_t dtype) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || page_size <= 0 || max_pages <= 0) return 0;
  return algx::make_plan(B, T, Hq, Hkv, page_size * max_pages, window, first, scored != 0,
                         dtype == ALGX_BF16).bytes;
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
  ALGX_REQUIRE(cfg->window >= 0 && cfg->first >= 0, "window and first must not be negative");
  if (B == 0 || T == 0) return ALGX_OK;
  ALGX_REQUIRE(q && k_pages && v_pages && o, "NULL tensor");
  ALGX_REQUIRE((scores == nullptr) == (scores_out == nullptr), "give scores and scores_out or neither");
  ALGX_REQUIRE((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o | (uintptr_t)workspace) & 15) == 0,
               "tensors must be 16-byte aligned");
  ALGX_REQUIRE(T * (Hq / Hkv) <= INT32_MAX / 64, "too many rows");
  const int64_t S = page_size * max_pages;
  const Plan p = make_plan(B, T, Hq, Hkv, S, cfg->window, cfg->first, scores != nullptr, dtype == ALGX_BF16);
  ALGX_REQUIRE(workspace && workspace_bytes >= p.bytes, "workspace too small");
  PagedAttnArgs a = {};
  a.q = q; a.k = k_pages; a.v = v_pages; a.sink = sink; a.scores = scores; a.scores_out = scores_out; a.o = o;
  char* ws = static_cast<char*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ml);
  a.part_o = reinterpret_cast<float*>(ws + p.o);
  a.xs = scores ? reinterpret_cast<float*>(ws + p.xs) : nullptr;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  a.slots = S; a.T = (int)T; a.G = (int)(Hq / Hkv); a.rows = (int)p.rows; a.tiles = (int)p.tiles;
  a.splits = (int)p.splits;
  while ((1 << a.log2n) < cfg->n) ++a.log2n;
  const bool soft = cfg->kind == ALGX_ATTN_SOFTMAX;
  a.scale = soft ? cfg->scale * kLog2e : cfg->scale;
  a.inv_unit = soft ? cfg->inv_unit * kLog2e : cfg->inv_unit;
  a.tile_rows = (int)p.tile_rows;
  a.direct = p.splits == 1 && scores == nullptr;
  a.sight = {cfg->window, cfg->first};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == ALGX_BF16)
    return soft ? paged_launch<__nv_bfloat16, kSoftmax>(a, pv, p, B, st)
                : paged_launch<__nv_bfloat16, kAsinh>(a, pv, p, B, st);
  return soft ? paged_launch<float, kSoftmax>(a, pv, p, B, st) : paged_launch<float, kAsinh>(a, pv, p, B, st);
}

}  // extern "C"
