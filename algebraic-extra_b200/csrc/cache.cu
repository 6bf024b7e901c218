// The paged key/value cache's own kernels: appending the keys and values of new
// tokens (QK norm and rotation on the way in) and evicting slots by accumulated
// attention weight.
#include <algorithm>

#include "paged_common.cuh"
#include "vec_io.cuh"

namespace algx {
namespace {

constexpr int kD = 64;

// ------------------------------------------------------------------- append
constexpr int kAppThreads = 256;
constexpr int kAppPasses = 4;  // row groups of one warp, loaded together

struct AppendArgs {
  const void* qkv;
  const float *gain_q, *gain_k, *rot_cos, *rot_sin;
  const int32_t *positions, *counts;
  void *q, *k_pages, *v_pages;
  int32_t* slot_positions;
  int* err;
  int64_t tokens;  // B * T
  int T, Hq, rot_rows, passes, segs;
  float eps;
};

// One warp takes `passes` groups of RPW head rows of one token, so the token's
// slot, page and rotation angles are found once for all of them. y = rms(x) g,
// then (y1 c - y2 s, y1 s + y2 c), all in fp32 with one rounding at the store:
// the cache holds the nearest bf16 of the exact key. Bound by memory: each row
// is read once and written once.
template <typename T, bool NORM, bool ROT>
__global__ void __launch_bounds__(kAppThreads) cache_append_kernel(const AppendArgs a, const PagedView pv) {
  using V = Vec<T>;
  constexpr int kHalfT = V::TPR / 2;
  const int lane = threadIdx.x & 31, sub = lane % V::TPR, rl = lane / V::TPR;
  const int64_t w = (int64_t)blockIdx.x * (kAppThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = w / a.segs;
  if (tok >= a.tokens) return;
  const int seg = (int)(w - tok * a.segs);
  const int heads = a.Hq + 2 * pv.heads;
  const int h0 = seg * a.passes * V::RPW + rl;

  uint4 raw[kAppPasses];
#pragma unroll
  for (int p = 0; p < kAppPasses; ++p) {
    const int h = h0 + p * V::RPW;
    raw[p] = p < a.passes && h < heads
                 ? ld_stream(static_cast<const T*>(a.qkv) + (tok * heads + h) * kD + sub * V::N)
                 : make_uint4(0, 0, 0, 0);
  }
  const int b = (int)(tok / a.T), t = (int)(tok - (int64_t)b * a.T);
  const int len = pv.lens[b];
  const bool live = a.counts == nullptr || t < a.counts[b];
  const int64_t slot = (int64_t)len + t;
  int pos = (a.positions ? a.positions[b] : len) + t;
  int pid = -1;
  const bool fits = len >= 0 && slot < ((int64_t)pv.max_pages << pv.page_shift);
  if (live && fits) pid = pv.table[(int64_t)b * pv.max_pages + (slot >> pv.page_shift)];
  const bool stored = live && fits && pid >= 0 && pid < pv.num_pages;
  bool bad = live && !stored;
  float c[V::N], s[V::N];
  if constexpr (ROT) {
    if (pos < 0 || pos >= a.rot_rows) {
      bad = bad || live;
      pos = pos < 0 ? 0 : a.rot_rows - 1;
    }
    const int j0 = (sub % kHalfT) * V::N;
#pragma unroll
    for (int i = 0; i < V::N; i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(a.rot_cos + (int64_t)pos * (kD / 2) + j0 + i);
      const float4 sv = *reinterpret_cast<const float4*>(a.rot_sin + (int64_t)pos * (kD / 2) + j0 + i);
      c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
      s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
    }
  }
  if (bad && lane == 0) atomicOr(a.err, DEV_ERR_BAD_PAGE);

#pragma unroll
  for (int p = 0; p < kAppPasses; ++p) {
    if (p >= a.passes) break;
    const int h = h0 + p * V::RPW;
    const bool is_v = h >= a.Hq + pv.heads;
    float x[V::N];
    unpack<T>(raw[p], x);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < V::N; ++i) ss = fmaf(x[i], x[i], ss);
      ss = row_sum<V::TPR>(ss);
      const float tau = rsqrtf(ss * (1.0f / kD) + a.eps);
      const float* g = (h < a.Hq ? a.gain_q : a.gain_k) + sub * V::N;
#pragma unroll
      for (int i = 0; i < V::N; ++i) x[i] = (x[i] * tau) * __ldg(g + i);
    }
    if constexpr (ROT) {
#pragma unroll
      for (int i = 0; i < V::N; ++i) {
        const float other = __shfl_xor_sync(0xffffffffu, x[i], kHalfT);
        x[i] = sub < kHalfT ? x[i] * c[i] - other * s[i] : x[i] * c[i] + other * s[i];
      }
    }
    if (h >= heads) continue;
    const uint4 y = is_v ? raw[p] : pack<T>(x);
    if (h < a.Hq) {
      *reinterpret_cast<uint4*>(static_cast<T*>(a.q) + (tok * a.Hq + h) * kD + sub * V::N) =
          live ? y : make_uint4(0, 0, 0, 0);
    } else if (stored) {
      const int g = h - a.Hq - (is_v ? pv.heads : 0);
      T* dst = static_cast<T*>(is_v ? a.v_pages : a.k_pages) + paged_row(pv, pid, g, (int)slot) + sub * V::N;
      *reinterpret_cast<uint4*>(dst) = y;
      if (!is_v && sub == 0 && a.slot_positions != nullptr)
        a.slot_positions[((int64_t)b * pv.heads + g) * ((int64_t)pv.max_pages << pv.page_shift) + slot] =
            (a.positions ? a.positions[b] : len) + t;
    }
  }
}

template <typename T>
int append_launch(const AppendArgs& a, const PagedView& pv, int64_t blocks, cudaStream_t st) {
  const bool norm = a.gain_q != nullptr, rot = a.rot_cos != nullptr;
  auto* kern = norm ? (rot ? cache_append_kernel<T, true, true> : cache_append_kernel<T, true, false>)
                    : (rot ? cache_append_kernel<T, false, true> : cache_append_kernel<T, false, false>);
  kern<<<(unsigned)blocks, kAppThreads, 0, st>>>(a, pv);
  ALGX_LAUNCHED("cache_append_kernel");
  return ALGX_OK;
}

// ------------------------------------------------------------------ eviction
constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;

struct EvictArgs {
  void *k_pages, *v_pages;
  const float* scores;
  const int32_t* positions;
  float* new_scores;
  int32_t *new_positions, *new_lens, *kept;
  int32_t* holes;  // workspace (B, Hkv, budget)
  int* err;
  int budget, first, recent;
  int row_bytes;
};

// Order-preserving map of a float to an unsigned key (NaN below everything).
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  x += 0.f;  // -0 and +0 are equal scores
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of two counts over the block; totals in tot.
__device__ __forceinline__ int2 block_scan2(int2 v, int2* warp_sums, int2& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 s = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s.x, off), y = __shfl_up_sync(0xffffffffu, s.y, off);
    if (lane >= off) { s.x += x; s.y += y; }
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int2 t = lane < kEvWarps ? warp_sums[lane] : make_int2(0, 0);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, t.x, off), y = __shfl_up_sync(0xffffffffu, t.y, off);
      if (lane >= off) { t.x += x; t.y += y; }
    }
    warp_sums[lane] = t;
  }
  __syncthreads();
  const int2 before = warp > 0 ? warp_sums[warp - 1] : make_int2(0, 0);
  tot = warp_sums[kEvWarps - 1];
  return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// One CTA per (sequence, kv head). The budget-th largest key is found by four
// rounds of 8-bit counting; slots above it stay, and of those equal to it the
// lowest slots. The kept slots at or above the budget then move, in order, into
// the holes below it, so a row that is already below the budget never moves.
__global__ void __launch_bounds__(kEvThreads) cache_evict_kernel(const EvictArgs a, const PagedView pv) {
  __shared__ int hist[256];
  __shared__ int2 warp_sums[32];
  __shared__ int s_newest, s_digit, s_left;
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / pv.heads), h = (int)(bh - (int64_t)b * pv.heads);
  const int len = paged_len(pv, b, a.err);
  const int64_t S = (int64_t)pv.max_pages << pv.page_shift;
  const float* scores = a.scores + bh * S;
  const int32_t* positions = a.positions + bh * S;
  float* new_scores = a.new_scores + bh * S;
  int32_t* new_positions = a.new_positions + bh * S;
  int32_t* kept = a.kept + bh * a.budget;
  int32_t* holes = a.holes + bh * a.budget;
  const int out_len = len < a.budget ? len : a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = out_len;

  if (len > a.budget) {
    if (tid == 0) s_newest = -1;
    __syncthreads();
    int newest = -1;
    for (int s = tid; s < len; s += kEvThreads) newest = max(newest, positions[s]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if ((tid & 31) == 0) atomicMax(&s_newest, newest);
    __syncthreads();
    newest = s_newest;
    const int64_t from = (int64_t)newest - a.recent;  // positions above it are recent
    auto key_at = [&](int s) -> uint32_t {
      const int p = positions[s];
      return p < a.first || p > from ? score_key(__int_as_float(0x7f800000)) : score_key(scores[s]);
    };
    // the budget-th largest key, and how many of its equals stay
    uint32_t prefix = 0;
    int left = a.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kEvThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t high = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int s = tid; s < len; s += kEvThreads) {
        const uint32_t k = key_at(s);
        if ((k & high) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int above = 0, d = 255;
        while (d > 0 && above + hist[d] < left) above += hist[d--];
        s_digit = d;
        s_left = left - above;
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      left = s_left;
      __syncthreads();
    }
    // holes below the budget, then movers above it, both in slot order
    int equal_before = 0, holes_before = 0;
    for (int s0 = 0; s0 < len; s0 += kEvThreads) {
      const int s = s0 + tid;
      const uint32_t k = s < len ? key_at(s) : 0u;
      const bool equal = s < len && k == prefix;
      int2 tot;
      const int2 r = block_scan2(make_int2(equal, 0), warp_sums, tot);
      const bool keep = s < len && (k > prefix || (equal && equal_before + r.x < left));
      equal_before += tot.x;
      const bool hole = s < a.budget && !keep;
      const bool mover = s >= a.budget && keep;
      const int2 q = block_scan2(make_int2(hole, mover), warp_sums, tot);
      // equal counts of holes and movers: the running index serves both lists
      if (hole) holes[holes_before + q.x] = s;
      if (s < a.budget && keep) kept[s] = s;
      holes_before += tot.x;
      (void)q;
    }
    __syncthreads();
    equal_before = 0;
    int movers_before = 0;
    for (int s0 = 0; s0 < len; s0 += kEvThreads) {
      const int s = s0 + tid;
      const uint32_t k = s < len ? key_at(s) : 0u;
      const bool equal = s < len && k == prefix;
      int2 tot;
      const int2 r = block_scan2(make_int2(equal, 0), warp_sums, tot);
      const bool keep = s < len && (k > prefix || (equal && equal_before + r.x < left));
      equal_before += tot.x;
      const bool mover = s >= a.budget && keep;
      const int2 q = block_scan2(make_int2(mover, 0), warp_sums, tot);
      if (mover) kept[holes[movers_before + q.x]] = s;
      movers_before += tot.x;
    }
    __syncthreads();
    // the rows themselves: 16 bytes a thread
    const int lanes = a.row_bytes / 16;
    const int64_t chunks = (int64_t)movers_before * lanes;
    for (int64_t i = tid; i < chunks; i += kEvThreads) {
      const int dst = holes[i / lanes], part = (int)(i % lanes);
      const int src = kept[dst];
      const int pd = pv.table[(int64_t)b * pv.max_pages + (dst >> pv.page_shift)];
      const int ps = pv.table[(int64_t)b * pv.max_pages + (src >> pv.page_shift)];
      if (pd < 0 || pd >= pv.num_pages || ps < 0 || ps >= pv.num_pages) {
        atomicOr(a.err, DEV_ERR_BAD_PAGE);
        continue;
      }
      const int64_t to = paged_row(pv, pd, h, dst) / kD * a.row_bytes + part * 16;
      const int64_t of = paged_row(pv, ps, h, src) / kD * a.row_bytes + part * 16;
      const uint4 kv = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.k_pages) + of);
      const uint4 vv = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.v_pages) + of);
      *reinterpret_cast<uint4*>(static_cast<char*>(a.k_pages) + to) = kv;
      *reinterpret_cast<uint4*>(static_cast<char*>(a.v_pages) + to) = vv;
    }
  } else {
    for (int s = tid; s < len; s += kEvThreads) kept[s] = s;
    __syncthreads();
  }
  for (int s = out_len + tid; s < a.budget; s += kEvThreads) kept[s] = -1;
  for (int64_t s = tid; s < S; s += kEvThreads) {
    const int src = s < out_len ? kept[s] : -1;
    new_scores[s] = src >= 0 ? scores[src] : 0.f;
    new_positions[s] = src >= 0 ? positions[src] : -1;
  }
}

}  // namespace

int paged_view(PagedView* pv, const void* table, const void* lens, int64_t B, int64_t Hkv, int64_t num_pages,
               int64_t page_size, int64_t max_pages, int64_t D) {
  ALGX_REQUIRE(B == 0 || (table && lens), "table or lens is NULL");
  ALGX_REQUIRE(D == 64, "head_dim must be 64");
  ALGX_REQUIRE(B >= 0 && Hkv >= 1 && num_pages >= 1 && max_pages >= 1, "paged cache sizes must be positive");
  ALGX_REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
               "page_size must be a power of two from 16 to 256");
  ALGX_REQUIRE(num_pages <= INT32_MAX && max_pages * page_size <= INT32_MAX, "paged cache too large");
  ALGX_REQUIRE(B * Hkv <= INT32_MAX, "too many sequences");
  pv->table = static_cast<const int32_t*>(table);
  pv->lens = static_cast<const int32_t*>(lens);
  pv->num_pages = (int32_t)num_pages;
  pv->max_pages = (int32_t)max_pages;
  pv->heads = (int32_t)Hkv;
  pv->page_shift = 0;
  while ((1 << pv->page_shift) < page_size) ++pv->page_shift;
  return ALGX_OK;
}

}  // namespace algx

extern "C" {

int algx_cache_append(const void* qkv, const float* gain_q, const float* gain_k, const float* rope_cos,
                      const float* rope_sin, int64_t rope_rows, const int32_t* table, const int32_t* lens,
                      const int32_t* positions, const int32_t* counts, void* q, void* k_pages, void* v_pages,
                      int32_t* slot_positions, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t num_pages,
                      int64_t page_size, int64_t max_pages, int64_t D, int32_t dtype, float eps, void* stream) {
  using namespace algx;
  PagedView pv;
  if (int s = paged_view(&pv, table, lens, B, Hkv, num_pages, page_size, max_pages, D)) return s;
  ALGX_REQUIRE(dtype == ALGX_F32 || dtype == ALGX_BF16, "dtype must be f32 or bf16");
  ALGX_REQUIRE(T >= 0 && Hq >= 0, "negative size");
  if (B == 0 || T == 0) return ALGX_OK;
  ALGX_REQUIRE(qkv && (q || Hq == 0) && k_pages && v_pages, "NULL tensor");
  ALGX_REQUIRE((gain_q == nullptr) == (gain_k == nullptr), "give both gains or neither");
  ALGX_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "give both rotary tables or neither");
  ALGX_REQUIRE(rope_cos == nullptr || (rope_rows >= 1 && rope_rows <= INT32_MAX), "rotary tables have no rows");
  ALGX_REQUIRE(eps > 0.f, "eps must be positive");
  ALGX_REQUIRE(((((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)rope_cos |
                  (uintptr_t)rope_sin)) & 15) == 0,
               "tensors must be 16-byte aligned");
  const int64_t heads = Hq + 2 * Hkv;
  ALGX_REQUIRE(heads <= 65536 && T <= INT32_MAX && B * T <= INT32_MAX, "too many rows");
  AppendArgs a = {};
  a.qkv = qkv; a.gain_q = gain_q; a.gain_k = gain_k; a.rot_cos = rope_cos; a.rot_sin = rope_sin;
  a.positions = positions; a.counts = counts; a.q = q; a.k_pages = k_pages; a.v_pages = v_pages;
  a.slot_positions = slot_positions;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  a.tokens = B * T; a.T = (int)T; a.Hq = (int)Hq; a.rot_rows = (int)rope_rows; a.eps = eps;
  const int rpw = dtype == ALGX_BF16 ? 4 : 2;
  // Few rows: one group a warp, so the rows spread over the SMs; from 48 warps
  // an SM on, more groups a warp share the token's lookups.
  const int64_t groups = (heads + rpw - 1) / rpw * a.tokens;
  a.passes = (int)std::min<int64_t>(kAppPasses, std::max<int64_t>(1, groups / (148 * 48)));
  a.segs = (int)((heads + rpw * a.passes - 1) / (rpw * a.passes));
  const int64_t blocks = (a.tokens * a.segs + kAppThreads / 32 - 1) / (kAppThreads / 32);
  ALGX_REQUIRE(blocks <= INT32_MAX, "too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == ALGX_BF16 ? append_launch<__nv_bfloat16>(a, pv, blocks, st) : append_launch<float>(a, pv, blocks, st);
}

size_t algx_cache_evict_workspace_size(int64_t B, int64_t Hkv, int64_t budget) {
  return B > 0 && Hkv > 0 && budget > 0 ? (size_t)(B * Hkv * budget) * sizeof(int32_t) : 0;
}

int algx_cache_evict(void* k_pages, void* v_pages, const int32_t* table, const int32_t* lens, const float* scores,
                     const int32_t* positions, int64_t budget, int64_t first, int64_t recent, int32_t* new_lens,
                     float* new_scores, int32_t* new_positions, int32_t* kept, int64_t B, int64_t Hkv,
                     int64_t num_pages, int64_t page_size, int64_t max_pages, int64_t D, int32_t dtype,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace algx;
  PagedView pv;
  if (int s = paged_view(&pv, table, lens, B, Hkv, num_pages, page_size, max_pages, D)) return s;
  ALGX_REQUIRE(dtype == ALGX_F32 || dtype == ALGX_BF16, "dtype must be f32 or bf16");
  ALGX_REQUIRE(budget >= 1 && budget <= INT32_MAX, "budget must be positive");
  ALGX_REQUIRE(first >= 0 && recent >= 0 && first <= budget && recent <= budget - first,
               "first + recent must fit the budget");
  if (B == 0) return ALGX_OK;
  ALGX_REQUIRE(k_pages && v_pages && scores && positions && new_lens && new_scores && new_positions && kept,
               "NULL tensor");
  ALGX_REQUIRE(scores != new_scores && positions != new_positions && lens != new_lens,
               "the new scores, positions and lengths need their own buffers");
  ALGX_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "tensors must be 16-byte aligned");
  ALGX_REQUIRE(workspace && workspace_bytes >= algx_cache_evict_workspace_size(B, Hkv, budget),
               "workspace too small");
  EvictArgs a = {};
  a.k_pages = k_pages; a.v_pages = v_pages; a.scores = scores; a.positions = positions;
  a.new_scores = new_scores; a.new_positions = new_positions; a.new_lens = new_lens; a.kept = kept;
  a.holes = static_cast<int32_t*>(workspace);
  a.budget = (int)budget; a.first = (int)first; a.recent = (int)recent;
  a.row_bytes = dtype == ALGX_BF16 ? 128 : 256;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  cache_evict_kernel<<<(unsigned)(B * Hkv), kEvThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, pv);
  ALGX_LAUNCHED("cache_evict_kernel");
  return ALGX_OK;
}

}  // extern "C"
