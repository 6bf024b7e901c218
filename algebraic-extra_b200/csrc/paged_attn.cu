// Attention of new tokens over the paged cache, split over its length and
// joined.
//
// Row (t, g) of kv head h is query token t of T under query head h G + g, with
// G = Hq / Hkv. For its scores x_s = scale (q . k_s) over the visible slots,
//
//   asinh    w_s = rho(x_s)^n          softmax   w_s = exp(x_s)
//   l = sum_s w_s + w(sink)            o = sum_s w_s v_s / l
//
// with every weight taken relative to a running reference score, so that no sum
// overflows (algebraic.py:186-204; the shifted form of kernels/flash.py:240-284).
// A row that sees no slot, or whose weights are all zero, gives zeros.
#include <algorithm>

#include "paged_common.cuh"
#include "vec_io.cuh"

namespace algx {
namespace {

constexpr int kD = 64;
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMinGroups = 8;  // groups of 16 slots a split takes at least
constexpr float kNegInf = -INFINITY;

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
  int T, G, rows, tiles, splits, log2n;
  float scale, inv_unit;
  Sight sight;
};

// Final factor of a row: 1 / l with the sink's weight in l, 0 for an empty row.
__device__ __forceinline__ float row_scale(float l) { return l == 0.f ? 0.f : 1.f / l; }

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
  int64_t idx = blockIdx.x;
  const int tile = (int)(idx % a.tiles);
  idx /= a.tiles;
  const int split = (int)(idx % a.splits);
  idx /= a.splits;
  const int h = (int)(idx % pv.heads), b = (int)(idx / pv.heads);
  const int len = paged_len(pv, b, a.err);
  const int r0 = tile * R, nr = min(R, a.rows - r0);
  const int lo = len - a.T + r0 / a.G, hi = len - a.T + (r0 + nr - 1) / a.G;
  const Span span(a.sight, lo, hi);
  const int per = max(kMinGroups, (span.total + a.splits - 1) / a.splits);
  const int g_end = (int)min((int64_t)span.total, (int64_t)(split + 1) * per);

  float q[R][V::N];
  int last[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(r0 + r, a.rows - 1), t = row / a.G, g = row - t * a.G;
    last[r] = r < nr ? len - a.T + t : -1;
    const int64_t at = (((int64_t)b * a.T + t) * pv.heads + h) * a.G + g;
    unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at * kD + sub * V::N), q[r]);
  }
  float m[R], turn[R], l[R], acc[R][V::N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = kNegInf;
    turn[r] = 0.f;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < V::N; ++i) acc[r][i] = 0.f;
  }
  for (int64_t g = (int64_t)split * per + warp; g < g_end; g += kWarps) {
    const int base = span.slot((int)g);
    const int pid = pv.table[(int64_t)b * pv.max_pages + (base >> pv.page_shift)];
    if (pid < 0 || pid >= pv.num_pages) {
      if (lane == 0) atomicOr(a.err, DEV_ERR_BAD_PAGE);
      continue;
    }
    const int64_t at = paged_row(pv, pid, h, base) + sub * V::N;
#pragma unroll 2
    for (int j = 0; j < 16; j += V::RPW) {
      const int s = base + j + rl;
      float kf[V::N], vf[V::N];
      const bool live = s < len;
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
          a.xs[(((int64_t)b * pv.heads + h) * a.rows + r0 + r) * a.slots + s] = x;
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
        const float w = weight_of<KIND, EXACT>(x, turn[r], a.log2n);
        l[r] += w;
#pragma unroll
        for (int i = 0; i < V::N; ++i) acc[r][i] = fmaf(w, vf[i], acc[r][i]);
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
  for (int i = threadIdx.x; i < nr * kD; i += kThreads) {
    const int r = i / kD, d = i % kD;
    float M = kNegInf;
    for (int p = 0; p < kParts; ++p) M = fmaxf(M, s_ml[r][p].x);
    const float t = weight_turn<KIND, EXACT>(M);
    float L = 0.f, O = 0.f;
    for (int p = 0; p < kParts; ++p) {
      const float2 ml = s_ml[r][p];
      if (ml.x == kNegInf && ml.y == 0.f) continue;
      const float f = weight_of<KIND, EXACT>(ml.x, t, a.log2n);
      L = fmaf(ml.y, f, L);
      O = fmaf(s_o[r][p][d], f, O);
    }
    const int64_t row = ((int64_t)b * pv.heads + h) * a.rows + r0 + r;
    if (d == 0) a.part_ml[row * a.splits + split] = make_float2(M, L);
    a.part_o[(row * a.splits + split) * kD + d] = O;
  }
}

// ------------------------------------------------------------------------ join
// Blocks below `rows` join one row's splits; the others add the weights of their
// slots over the rows of one kv head.
constexpr int kScoreSlots = 1024;
constexpr int kRowChunk = 64;

template <int KIND, bool EXACT>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, int64_t row, float sink, float& M, float& L) {
  M = sink;  // -inf without a sink
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.part_ml[row * a.splits + s].x);
  const float t = weight_turn<KIND, EXACT>(M);
  L = sink == kNegInf ? 0.f : weight_of<KIND, EXACT>(sink, t, a.log2n);
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = a.part_ml[row * a.splits + s];
    if (ml.x == kNegInf && ml.y == 0.f) continue;
    L = fmaf(ml.y, weight_of<KIND, EXACT>(ml.x, t, a.log2n), L);
  }
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const PagedAttnArgs a, const PagedView pv, int blocks) {
  constexpr bool EXACT = sizeof(T) == 4;
  const int64_t bh = blockIdx.x / blocks;
  const int which = (int)(blockIdx.x - bh * blocks);
  const int h = (int)(bh % pv.heads), b = (int)(bh / pv.heads);
  if (which < a.rows) {
    __shared__ float s_half[kD];
    const int64_t row = bh * a.rows + which;
    const int t = which / a.G, g = which - t * a.G;
    const float sink = a.sink ? a.sink[h * a.G + g] * a.inv_unit : kNegInf;
    float M, L, O = 0.f;
    join_row<KIND, EXACT>(a, row, sink, M, L);
    const float turn = weight_turn<KIND, EXACT>(M);
    const int d = threadIdx.x % kD, half = threadIdx.x / kD;
    for (int s = half; s < a.splits; s += kThreads / kD) {
      const float2 ml = a.part_ml[row * a.splits + s];
      if (ml.x == kNegInf && ml.y == 0.f) continue;
      O = fmaf(a.part_o[(row * a.splits + s) * kD + d], weight_of<KIND, EXACT>(ml.x, turn, a.log2n), O);
    }
    if (half == 1) s_half[d] = O;
    __syncthreads();
    if (half == 0) {
      O = (O + s_half[d]) * row_scale(L);
      const int64_t at = (((int64_t)b * a.T + t) * pv.heads + h) * a.G + g;
      static_cast<T*>(a.o)[at * kD + d] = from_f32<T>(O);
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
    for (int r = threadIdx.x; r < nr; r += kThreads) {
      const int g = (r0 + r) % a.G;
      const float sink = a.sink ? a.sink[h * a.G + g] * a.inv_unit : kNegInf;
      float M, L;
      join_row<KIND, EXACT>(a, bh * a.rows + r0 + r, sink, M, L);
      s_turn[r] = weight_turn<KIND, EXACT>(M);
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

Plan make_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t S, int64_t window, int64_t first, bool scored) {
  Plan p = {};
  p.rows = T * (Hq / Hkv);
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

template <typename T, int KIND>
int paged_launch(const PagedAttnArgs& a, const PagedView& pv, const Plan& p, int64_t B, cudaStream_t st) {
  const int64_t grid = B * pv.heads * p.splits * p.tiles;
  ALGX_REQUIRE(grid <= INT32_MAX, "too many rows");
  auto* kern = p.tile_rows == 1   ? paged_attn_kernel<T, KIND, 1>
               : p.tile_rows == 2 ? paged_attn_kernel<T, KIND, 2>
               : p.tile_rows == 4 ? paged_attn_kernel<T, KIND, 4>
                                  : paged_attn_kernel<T, KIND, 8>;
  kern<<<(unsigned)grid, kThreads, 0, st>>>(a, pv);
  ALGX_LAUNCHED("paged_attn_kernel");
  const int64_t blocks = a.rows + (a.xs ? (a.slots + kScoreSlots - 1) / kScoreSlots : 0);
  ALGX_REQUIRE(blocks * B * pv.heads <= INT32_MAX, "too many rows");
  paged_join_kernel<T, KIND><<<(unsigned)(blocks * B * pv.heads), kThreads, 0, st>>>(a, pv, (int)blocks);
  ALGX_LAUNCHED("paged_join_kernel");
  return ALGX_OK;
}

}  // namespace
}  // namespace algx

extern "C" {

size_t algx_paged_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t page_size,
                                      int64_t max_pages, int64_t window, int64_t first, int32_t scored) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || page_size <= 0 || max_pages <= 0) return 0;
  return algx::make_plan(B, T, Hq, Hkv, page_size * max_pages, window, first, scored != 0).bytes;
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
  const Plan p = make_plan(B, T, Hq, Hkv, S, cfg->window, cfg->first, scores != nullptr);
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
  a.scale = cfg->scale; a.inv_unit = cfg->inv_unit;
  a.sight = {cfg->window, cfg->first};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool soft = cfg->kind == ALGX_ATTN_SOFTMAX;
  if (dtype == ALGX_BF16)
    return soft ? paged_launch<__nv_bfloat16, kSoftmax>(a, pv, p, B, st)
                : paged_launch<__nv_bfloat16, kAsinh>(a, pv, p, B, st);
  return soft ? paged_launch<float, kSoftmax>(a, pv, p, B, st) : paged_launch<float, kAsinh>(a, pv, p, B, st);
}

}  // extern "C"
