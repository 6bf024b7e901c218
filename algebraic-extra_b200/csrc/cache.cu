// The paged key/value cache's own kernels: appending the keys and values of new
// tokens (QK norm and rotation on the way in) and evicting slots by accumulated
// attention weight.
#include <algorithm>
#include <atomic>

#include "paged_common.cuh"
#include "vec_io.cuh"

namespace algx {
namespace {

constexpr int kD = 64;

// ------------------------------------------------------------------- append
constexpr int kAppThreads = 128;
constexpr int kAppPasses = 5;  // row groups of one warp, loaded together

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

// One warp takes `passes` groups of head rows of one token, so the token's slot,
// page and rotation angles are found once for all of them. A lane holds a 16-byte
// chunk of a row's first half and the chunk 32 elements on, which the rotation
// pairs: it needs no exchange, and the norm two shuffles (bf16: 4 lanes a row, 8
// rows a group). y = rms(x) g, then (y1 c - y2 s, y1 s + y2 c), all in fp32 with
// one rounding at the store: the cache holds the nearest bf16 of the exact key.
// Bound by memory: each row is read once and written once. Measured: 16384 tokens of
// 36 rows (155 MB) 32 us a pass, 4.8 TB/s, of 6.55 a plain copy reaches, at 14 warps an
// SM; with a row across 8 lanes, halves exchanged by
// shuffles, 47 us; three row groups a warp instead of five 34 us.
template <typename T, bool NORM, bool ROT>
__global__ void __launch_bounds__(kAppThreads, 4) cache_append_kernel(const AppendArgs a, const PagedView pv) {
  using V = Vec<T>;
  constexpr int N = V::N, kLanes = V::TPR / 2, kRows = 32 / kLanes;
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % kLanes, rl = lane / kLanes;
  const int64_t w = (int64_t)blockIdx.x * (kAppThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = w / a.segs;
  if (tok >= a.tokens) return;
  const int seg = (int)(w - tok * a.segs);
  const int heads = a.Hq + 2 * pv.heads;
  const int h0 = seg * a.passes * kRows + rl;
  const T* src = static_cast<const T*>(a.qkv) + tok * heads * kD + sub * N;

  uint4 raw[kAppPasses][2];
#pragma unroll
  for (int p = 0; p < kAppPasses; ++p) {
    const int h = h0 + p * kRows;
    const bool in = p < a.passes && h < heads;
#pragma unroll
    for (int i = 0; i < 2; ++i) raw[p][i] = in ? ld_stream(src + h * kD + i * (kD / 2)) : make_uint4(0, 0, 0, 0);
  }
  const int b = (int)(tok / a.T), t = (int)(tok - (int64_t)b * a.T);
  const int len = pv.lens[b], start = a.positions ? a.positions[b] : len;
  const bool live = a.counts == nullptr || t < a.counts[b];
  const int64_t slot = (int64_t)len + t;
  int pid = -1;
  const bool fits = len >= 0 && slot < ((int64_t)pv.max_pages << pv.page_shift);
  if (live && fits) pid = pv.table[(int64_t)b * pv.max_pages + (slot >> pv.page_shift)];
  const bool stored = live && fits && pid >= 0 && pid < pv.num_pages;
  bool bad = live && !stored;
  float2 c[N / 2], s[N / 2];
  if constexpr (ROT) {
    int64_t pos = (int64_t)start + t;
    if (pos < 0 || pos >= a.rot_rows) {
      bad = bad || live;
      pos = pos < 0 ? 0 : a.rot_rows - 1;
    }
#pragma unroll
    for (int i = 0; i < N / 2; i += 2) {
      const float4 cv = __ldg(reinterpret_cast<const float4*>(a.rot_cos + pos * (kD / 2) + sub * N) + i / 2);
      const float4 sv = __ldg(reinterpret_cast<const float4*>(a.rot_sin + pos * (kD / 2) + sub * N) + i / 2);
      c[i] = make_float2(cv.x, cv.y); c[i + 1] = make_float2(cv.z, cv.w);
      s[i] = make_float2(sv.x, sv.y); s[i + 1] = make_float2(sv.z, sv.w);
    }
  }
  if (bad && lane == 0) atomicOr(a.err, DEV_ERR_BAD_PAGE);

#pragma unroll
  for (int p = 0; p < kAppPasses; ++p) {
    if (p >= a.passes) break;
    const int h = h0 + p * kRows;
    const bool is_v = h >= a.Hq + pv.heads;
    float x0[N], x1[N];
    unpack<T>(raw[p][0], x0);
    unpack<T>(raw[p][1], x1);
    float2 y[2][N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      y[0][i] = make_float2(x0[2 * i], x0[2 * i + 1]);
      y[1][i] = make_float2(x1[2 * i], x1[2 * i + 1]);
    }
    if constexpr (NORM) {
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) ss = fma2(y[1][i], y[1][i], fma2(y[0][i], y[0][i], ss));
      const float sum = row_sum<kLanes>(ss.x + ss.y);
      const float tau = rsqrtf(sum * (1.0f / kD) + a.eps);
      const float* g = (h < a.Hq ? a.gain_q : a.gain_k) + sub * N;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < N / 2; i += 2) {
          const float4 gv = __ldg(reinterpret_cast<const float4*>(g + half * (kD / 2)) + i / 2);
          const float2 tt = make_float2(tau, tau);
          y[half][i] = mul2(mul2(y[half][i], tt), make_float2(gv.x, gv.y));
          y[half][i + 1] = mul2(mul2(y[half][i + 1], tt), make_float2(gv.z, gv.w));
        }
    }
    if constexpr (ROT) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 u = y[0][i], v = y[1][i], minus = make_float2(-v.x, -v.y);
        y[0][i] = fma2(u, c[i], mul2(minus, s[i]));
        y[1][i] = fma2(u, s[i], mul2(v, c[i]));
      }
    }
    if (h >= heads) continue;
    uint4 out[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float z[N];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        z[2 * i] = y[half][i].x;
        z[2 * i + 1] = y[half][i].y;
      }
      out[half] = is_v ? raw[p][half] : pack<T>(z);
    }
    T* dst = nullptr;
    if (h < a.Hq) {
      dst = static_cast<T*>(a.q) + (tok * a.Hq + h) * kD;
      if (!live) out[0] = out[1] = make_uint4(0, 0, 0, 0);
    } else if (stored) {
      const int g = h - a.Hq - (is_v ? pv.heads : 0);
      dst = static_cast<T*>(is_v ? a.v_pages : a.k_pages) + paged_row(pv, pid, g, (int)slot);
      if (!is_v && sub == 0 && a.slot_positions != nullptr)
        a.slot_positions[((int64_t)b * pv.heads + g) * ((int64_t)pv.max_pages << pv.page_shift) + slot] = start + t;
    }
    if (dst != nullptr) {
      *reinterpret_cast<uint4*>(dst + sub * N) = out[0];
      *reinterpret_cast<uint4*>(dst + kD / 2 + sub * N) = out[1];
    }
  }
}

template <typename T>
int append_launch(const AppendArgs& a, const PagedView& pv, int64_t blocks, cudaStream_t st) {
  const bool norm = a.gain_q != nullptr, rot = a.rot_cos != nullptr;
  auto* kern = norm ? (rot ? cache_append_kernel<T, true, true> : cache_append_kernel<T, true, false>)
                    : (rot ? cache_append_kernel<T, false, true> : cache_append_kernel<T, false, false>);
  ALGX_CUDA(launch_dependent(kern, dim3((unsigned)blocks), dim3(kAppThreads), 0, st, a, pv));
  ALGX_LAUNCHED("cache_append_kernel");
  return ALGX_OK;
}

// ------------------------------------------------------------------ eviction
constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvChunk = 4 * kEvThreads;     // slots of one sweep of the block, four a thread
constexpr int kEvCached = 48 * 1024;         // keys kept in shared memory
constexpr int kBins = 4 * kEvThreads;        // 11 bits a round, 10 in the last
constexpr int kInplace = 1024;

struct EvictArgs {
  void *k_pages, *v_pages;
  const float* scores;
  const int32_t* positions;
  float* new_scores;
  int32_t *new_positions, *new_lens, *kept;
  int2* moves;  // workspace (B, Hkv, budget): (to, from) slots
  int* counts;  // workspace (B, Hkv): moves of each item
  int* err;
  int budget, first, recent;
  int lanes;    // 16-byte pieces of a row
  int cached;   // whether the keys fit shared memory
  int inplace;  // whether the CTA that chose the rows moves them too
};

// Order-preserving map of a float to an unsigned key (NaN below everything).
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  x += 0.f;  // -0 and +0 are equal scores
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Inclusive sum over the block of one int a thread; the total goes to `total`.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += x;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kEvWarps; ++i) {
    const int x = warp_sums[i];
    if (i < warp) before += x;
    total += x;
  }
  __syncthreads();
  return before + v;
}

// Rows i0, i0 + step, ... of an item's moves, counted in 16-byte pieces: keys and
// values, kFly pieces of each in flight.
template <int kFly>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const PagedView& pv, int64_t bh, int i0, int end, int step) {
  const int b = (int)(bh / pv.heads), h = (int)(bh - (int64_t)b * pv.heads);
  const int32_t* table = pv.table + (int64_t)b * pv.max_pages;
  const int2* moves = a.moves + bh * a.budget;
  const int row_bytes = a.lanes * 16, row_shift = a.lanes == 8 ? 3 : 4;
  for (; i0 < end; i0 += step * kFly) {
    uint4 kv[kFly], vv[kFly];
    int64_t to[kFly], of[kFly];
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      const int i = i0 + j * step;
      to[j] = -1;
      if (i >= end) continue;
      const int2 move = moves[i >> row_shift];
      const int pd = table[move.x >> pv.page_shift], ps = table[move.y >> pv.page_shift];
      if ((unsigned)pd >= (unsigned)pv.num_pages || (unsigned)ps >= (unsigned)pv.num_pages) {
        atomicOr(a.err, DEV_ERR_BAD_PAGE);
        continue;
      }
      const int part = (i & (a.lanes - 1)) * 16;
      to[j] = paged_row(pv, pd, h, move.x) / kD * row_bytes + part;
      of[j] = paged_row(pv, ps, h, move.y) / kD * row_bytes + part;
    }
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      if (to[j] < 0) continue;
      kv[j] = ld_stream(static_cast<const char*>(a.k_pages) + of[j]);
      vv[j] = ld_stream(static_cast<const char*>(a.v_pages) + of[j]);
    }
#pragma unroll
    for (int j = 0; j < kFly; ++j) {
      if (to[j] < 0) continue;
      *reinterpret_cast<uint4*>(static_cast<char*>(a.k_pages) + to[j]) = kv[j];
      *reinterpret_cast<uint4*>(static_cast<char*>(a.v_pages) + to[j]) = vv[j];
    }
  }
}

// One CTA per (sequence, kv head). The budget-th largest key is found by three
// rounds of counting 11 bits; slots above it stay, and of those equal to it the
// lowest slots. One sweep over the slots then numbers the holes below the budget
// and the kept slots at or above it: the i-th such slot moves to the i-th hole, so
// a row that is below the budget never moves. This is a chain of block-wide steps: some
// twenty, and two barriers (four where scores are equal at the limit) for every 2048
// slots of the last sweep. Measured: 12 items of 2560 slots, with the moves, 10.9 us a
// pass (19 as one cold launch under the profiler), 192 items of 8192 slots 27 us. (Counting with one addition for all lanes
// that meet in a bin took 40 us: their matching costs more than the conflicts.)
__global__ void __launch_bounds__(kEvThreads, 2) cache_evict_kernel(const EvictArgs a, const PagedView pv) {
  extern __shared__ uint4 s_keys[];
  __shared__ int4 hist[kBins / 4];
  __shared__ int warp_sums[kEvWarps];
  __shared__ int s_newest, s_digit, s_left, s_equal;
  int* const bins = reinterpret_cast<int*>(hist);
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / pv.heads), h = (int)(bh - (int64_t)b * pv.heads);
  const int len = paged_len(pv, b, a.err);
  const int S = pv.max_pages << pv.page_shift;  // a multiple of 16
  const float* scores = a.scores + bh * S;
  const int32_t* positions = a.positions + bh * S;
  float* new_scores = a.new_scores + bh * S;
  int32_t* new_positions = a.new_positions + bh * S;
  int32_t* kept = a.kept + bh * a.budget;
  int2* moves = a.moves + bh * a.budget;
  const int out_len = min(len, a.budget);
  if (h == 0 && tid == 0) a.new_lens[b] = out_len;
  // Everything below the new length first as if nothing moved; the moves write
  // over their holes later.
  auto copy_row = [&](int s, const float4& x, const int4& p) {
    if (s + 4 <= out_len) {
      *reinterpret_cast<float4*>(new_scores + s) = x;
      *reinterpret_cast<int4*>(new_positions + s) = p;
    } else {
      const float xs[4] = {x.x, x.y, x.z, x.w};
      const int ps[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        new_scores[s + i] = s + i < out_len ? xs[i] : 0.f;
        new_positions[s + i] = s + i < out_len ? ps[i] : -1;
      }
    }
  };
  for (int s = tid; s < a.budget; s += kEvThreads) kept[s] = s < out_len ? s : -1;
  for (int i = tid; i < kBins / 4; i += kEvThreads) hist[i] = make_int4(0, 0, 0, 0);
  if (tid == 0) s_newest = -1;
  __syncthreads();
  int newest = -1;
#pragma unroll 4
  for (int s = 4 * tid; s < S; s += kEvChunk) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    int4 p = make_int4(-1, -1, -1, -1);
    if (s < len) {
      x = *reinterpret_cast<const float4*>(scores + s);
      p = *reinterpret_cast<const int4*>(positions + s);
      newest = max(newest, p.x);
      if (s + 1 < len) newest = max(newest, p.y);
      if (s + 2 < len) newest = max(newest, p.z);
      if (s + 3 < len) newest = max(newest, p.w);
    }
    copy_row(s, x, p);
  }
  int movers = 0;
  if (len > a.budget) {
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&s_newest, newest);
    __syncthreads();
    const int64_t from = (int64_t)s_newest - a.recent;  // positions above it are recent
    // protected slots stand above every score, an infinite one too (0xff800000)
    auto key = [&](float x, int p) { return p < a.first || p > from ? 0xffffffffu : score_key(x); };
    auto make_keys = [&](int s) {
      const float4 x = *reinterpret_cast<const float4*>(scores + s);
      const int4 p = *reinterpret_cast<const int4*>(positions + s);
      return make_uint4(key(x.x, p.x), key(x.y, p.y), key(x.z, p.z), key(x.w, p.w));
    };

    // the budget-th largest key, and how many of its equals stay
    uint32_t limit = 0;
    int left = a.budget;
#pragma unroll
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, mask = round == 2 ? 1023 : kBins - 1;
#pragma unroll 4
      for (int s = 4 * tid; s < len; s += kEvChunk) {
        const uint4 k4 = round > 0 && a.cached ? s_keys[s >> 2] : make_keys(s);
        if (round == 0 && a.cached) s_keys[s >> 2] = k4;  // read by the same thread only
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = s + i < len && (round == 0 || (k[i] >> (round == 1 ? 21 : 10)) == limit);
          const int bin = (int)((k[i] >> shift) & mask);
          if (in) atomicAdd(&bins[bin], 1);
        }
      }
      __syncthreads();
      // the bin where the count from above reaches `left`: four bins a thread
      const int quad = kEvThreads - 1 - tid;
      const int4 q = hist[quad];
      const int c[4] = {q.w, q.z, q.y, q.x};
      int total;
      const int mine = c[0] + c[1] + c[2] + c[3], upto = block_scan(mine, warp_sums, total);
      if (upto >= left && upto - mine < left) {
        int above = upto - mine, d = 0;
        while (above + c[d] < left) above += c[d++];
        s_digit = 4 * quad + 3 - d;
        s_left = left - above;
        s_equal = c[d];
      }
      hist[quad] = make_int4(0, 0, 0, 0);
      __syncthreads();
      limit = round == 0 ? (uint32_t)s_digit : (limit << (round == 1 ? 11 : 10)) | (uint32_t)s_digit;
      left = s_left;
    }
    const bool all_equals = s_equal == left;  // the usual case: no ties at the limit

    int equals = 0, holes = 0;
    for (int s0 = 0; s0 < len; s0 += kEvChunk) {
      const int s = s0 + 4 * tid;
      const uint4 k4 = s < len ? (a.cached ? s_keys[s >> 2] : make_keys(s)) : make_uint4(0, 0, 0, 0);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
      bool keep[4];
      if (all_equals) {
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = s + i < len && k[i] >= limit;
      } else {
        int n = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += s + i < len && k[i] == limit;
        int rank = equals + block_scan(n, warp_sums, total) - n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool equal = s + i < len && k[i] == limit;
          keep[i] = s + i < len && (k[i] > limit || (equal && rank < left));
          rank += equal;
        }
        equals += total;
      }
      int n = 0, total;  // holes in the low half, movers in the high one
#pragma unroll
      for (int i = 0; i < 4; ++i) n += s + i < a.budget ? (s + i < len && !keep[i]) : keep[i] << 16;
      const int upto = block_scan(n, warp_sums, total) - n;
      int hole = holes + (upto & 0xffff), mover = movers + (upto >> 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (s + i < a.budget && s + i < len && !keep[i]) moves[hole++].x = s + i;
        if (s + i >= a.budget && keep[i]) moves[mover++].y = s + i;
      }
      holes += total & 0xffff;
      movers += total >> 16;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < movers; i += kEvThreads) {
      const int2 move = moves[i];
      kept[move.x] = move.y;
      new_scores[move.x] = scores[move.y];
      new_positions[move.x] = positions[move.y];
    }
    if (a.inplace) move_rows<4>(a, pv, bh, tid, movers * a.lanes, kEvThreads);
  }
  if (tid == 0) a.counts[bh] = movers;
}

// The moves of all items, spread over the device: kMovePieces 16-byte pieces of
// keys and of values a CTA at a time. Bound by memory at single 128-byte rows;
// measured: 201 MB 41 us, 4.9 TB/s.
constexpr int kMoveThreads = 256;
constexpr int kMoveFly = 4;
constexpr int kMovePieces = kMoveThreads * kMoveFly;

__global__ void __launch_bounds__(kMoveThreads, 4) cache_move_kernel(const EvictArgs a, const PagedView pv, int items,
                                                                  int chunks) {
  pdl_wait();
  for (int64_t i = blockIdx.x; i < (int64_t)items * chunks; i += gridDim.x) {
    const int chunk = (int)(i / items), item = (int)(i - (int64_t)chunk * items);
    const int begin = chunk * kMovePieces, end = min(begin + kMovePieces, a.counts[item] * a.lanes);
    if (begin < end) move_rows<kMoveFly>(a, pv, item, begin + threadIdx.x, end, kMoveThreads);
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
  // slots are counted in 32 bits, up to the end of the group of 32 that holds the last one
  ALGX_REQUIRE(num_pages <= INT32_MAX && max_pages <= (INT32_MAX - 64) / page_size, "paged cache too large");
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
                  (uintptr_t)rope_sin | (uintptr_t)gain_q | (uintptr_t)gain_k)) & 15) == 0,
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
  const int rows = dtype == ALGX_BF16 ? 8 : 4;  // of one group
  // Few rows: one group a warp, so the rows spread over the SMs; from 48 warps
  // an SM on, more groups a warp share the token's lookups.
  const int64_t groups = (heads + rows - 1) / rows;
  const int64_t most = std::min<int64_t>(kAppPasses, std::max<int64_t>(1, groups * a.tokens / (148 * 48)));
  a.segs = (int)((groups + most - 1) / most);
  a.passes = (int)((groups + a.segs - 1) / a.segs);
  const int64_t blocks = (a.tokens * a.segs + kAppThreads / 32 - 1) / (kAppThreads / 32);
  ALGX_REQUIRE(blocks <= INT32_MAX, "too many rows");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == ALGX_BF16 ? append_launch<__nv_bfloat16>(a, pv, blocks, st) : append_launch<float>(a, pv, blocks, st);
}

size_t algx_cache_evict_workspace_size(int64_t B, int64_t Hkv, int64_t budget) {
  return B > 0 && Hkv > 0 && budget > 0 ? (size_t)(B * Hkv * budget) * sizeof(int2) + (size_t)(B * Hkv) * sizeof(int) : 0;
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
  const int64_t S = page_size * max_pages;
  // Rows an item can move at most.
  const int64_t most = std::min<int64_t>(budget, std::max<int64_t>(0, S - budget));
  // The kernels count slots and 16-byte pieces of moved rows in 32 bits, up to a step past the end.
  const int64_t lanes = dtype == ALGX_BF16 ? 8 : 16;
  ALGX_REQUIRE(S <= INT32_MAX - kEvChunk && budget <= INT32_MAX - kEvThreads && most * lanes <= INT32_MAX - 2 * kMovePieces,
               "paged cache too large");
  if (B == 0) return ALGX_OK;
  ALGX_REQUIRE(k_pages && v_pages && scores && positions && new_lens && new_scores && new_positions && kept,
               "NULL tensor");
  ALGX_REQUIRE(scores != new_scores && positions != new_positions && lens != new_lens,
               "the new scores, positions and lengths need their own buffers");
  ALGX_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)scores | (uintptr_t)positions |
                  (uintptr_t)new_scores | (uintptr_t)new_positions) & 15) == 0 &&
                   ((uintptr_t)workspace & 7) == 0,
               "tensors must be 16-byte aligned");
  ALGX_REQUIRE(workspace && workspace_bytes >= algx_cache_evict_workspace_size(B, Hkv, budget),
               "workspace too small");
  EvictArgs a = {};
  a.k_pages = k_pages; a.v_pages = v_pages; a.scores = scores; a.positions = positions;
  a.new_scores = new_scores; a.new_positions = new_positions; a.new_lens = new_lens; a.kept = kept;
  a.moves = static_cast<int2*>(workspace);
  a.counts = reinterpret_cast<int*>(a.moves + B * Hkv * budget);
  a.budget = (int)budget; a.first = (int)first; a.recent = (int)recent;
  a.lanes = (int)lanes;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  // Up to kInplace rows an item's own CTA moves them, which saves a launch (12
  // items of at most 512 rows: 11 us a pass in one launch); more are spread over the
  // device (192 items of 2050 rows: 69 us a pass in two launches, 138 in one).
  a.inplace = most <= kInplace;
  a.cached = S <= kEvCached;
  const size_t smem = a.cached ? (size_t)S * sizeof(uint32_t) : 0;
  static std::atomic<uint64_t> ready{0};  // one bit per device: its shared memory limit is raised
  int dev = 0;
  ALGX_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    ALGX_CUDA(cudaFuncSetAttribute(cache_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   kEvCached * (int)sizeof(uint32_t)));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  ALGX_CUDA(launch_dependent(cache_evict_kernel, dim3((unsigned)(B * Hkv)), dim3(kEvThreads), smem,
                             static_cast<cudaStream_t>(stream), a, pv));
  ALGX_LAUNCHED("cache_evict_kernel");
  if (a.inplace) return ALGX_OK;
  const int64_t items = B * Hkv, chunks = (most * a.lanes + kMovePieces - 1) / kMovePieces;
  ALGX_CUDA(launch_dependent(cache_move_kernel, dim3((unsigned)std::min<int64_t>(items * chunks, 148 * 8)),
                             dim3(kMoveThreads), 0, static_cast<cudaStream_t>(stream), a, pv, (int)items, (int)chunks));
  ALGX_LAUNCHED("cache_move_kernel");
  return ALGX_OK;
}

}  // extern "C"
