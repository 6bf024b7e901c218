// Verification of drafted tokens against the target model's probabilities, and
// the draw of the token that follows the accepted ones.
//
// Row probabilities are p_v = w(z_v) / sum w, with w(z) = exp(z) (ce) or
// rho(z / c)^n (alg_ce, algebraic.py:266-301), taken relative to the row's
// maximum. Draft token x_i is accepted while u_i q_i(x_i) < p_i(x_i). After the
// first refusal at i the next token has the distribution max(p_i - q_i, 0)
// normalised, after K acceptances p_K; with exponential variates e_v it is
// argmax_v weight_v / e_v, so no sum over the residual is needed, ties going to
// the lowest index.
//
// One cluster of CTAs per sequence, one launch: each CTA reads its slice of the
// vocabulary of every row, the CTAs exchange the rows' partial sums through
// distributed shared memory, each decides the (same) accepted count, races over
// its slice of the one row that counts, and the winners meet in CTA 0.
//
// One cluster barrier a round and two a race: three to six a call, whose chain is the
// time where there are few sequences (one of 4 drafts, bf16, 10.8 us a pass). Where
// there are many, memory is far from busy: 64 sequences of 7 drafts over 50304 float32
// logits take 55 us a pass and read 119 of 193 MB, 2.2 TB/s, a third of a copy's rate,
// at 0.48 instructions a scheduler and cycle; some 30 us are sums, 8 the race.
//
// The sums use the MUFU forms of the weights (measured at most 7.5 n 2^-24 off an
// element for alg_ce, mostly averaged out by the sum); everything a decision
// compares - the drafted tokens' weights and the race's candidates - is evaluated
// with correctly rounded roots and divisions or expf. A draft whose u q(x) lies within
// the sums' error of p(x) can fall the other way than in 64 bits.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace algx {
namespace {

constexpr int kMaxRows = 64;  // of one round: 32 target rows, 31 draft rows

struct VerifyArgs {
  const void *target, *draft;
  const int32_t *tokens, *counts;
  const float *u, *race;
  int32_t *out, *accepted;
  int* err;
  int64_t V, slice;  // slice: vocabulary columns of one CTA
  int K, log2n;
  int round;  // draft positions looked at in the first round
  float scale;  // 1 / temperature (ce) or 1 / c (alg_ce)
  float margin;  // of the race's fast weights, relative (race_margin)
};

// How far the race's fast weights may be from the exact ones that decide, relative to
// themselves, with u = 2^-24. alg_ce: root and reciprocal of 2 u each, a sum and a
// product of u make 6 u for the fast form of rho(x) turn, 4 u for the exact one, 10 u
// together, n times that in the power, whose squarings add less than n u a side;
// 12 n u + 12 u for the factors after it is below 2^-19 n from n = 2 on (measured:
// 7.5 n u at most). ce: the argument, at most 126 in units of log2(e), is rounded to
// 2^-18, its factor to 2 u, the exact form's to 2^-18: 2^-16 of a weight, 2^-14 with
// the factors after it to spare. Below 2^-126 the fast forms flush to zero: kFlushed
// bounds that.
constexpr float kFlushed = 0x1p-125f;
inline float race_margin(int32_t kind, int32_t n) {
  return kind == ALGX_HEAD_CE ? 0x1p-14f : std::min(1.f, (float)n * 0x1p-19f);
}

// The score of a logit: the logit itself for ce, so that differences from the
// maximum are exact, z / c for alg_ce. NaN counts as -inf.
template <int KIND>
__device__ __forceinline__ float score_of(const VerifyArgs& a, float z) {
  z = fmaxf(z, kNegInf);
  return KIND == kSoftmax ? z : z * a.scale;
}
template <int KIND>
__device__ __forceinline__ float exact_weight(const VerifyArgs& a, float x, float turn) {
  if constexpr (KIND == kSoftmax) return expf((x - turn) * a.scale);
  else return weight_of<kAsinh, true>(x, turn, a.log2n);
}
template <int KIND>
__device__ __forceinline__ float fast_weight(const VerifyArgs& a, float x, float turn) {
  if constexpr (KIND == kSoftmax) return weight_of<kSoftmax, false>((x - turn) * (a.scale * kLog2e), 0.f, 0);
  else return weight_of<kAsinh, false>(x, turn, a.log2n);
}
template <int KIND, int LOG2N>
__device__ __forceinline__ float2 fast_weights(const VerifyArgs& a, float2 x, float2 turn) {
  if constexpr (KIND == kSoftmax) {
    const float k = a.scale * kLog2e;
    return weight_pair<kSoftmax, 0>(mul2(sub2(x, turn), make_float2(k, k)), make_float2(0.f, 0.f), 0);
  } else {
    return weight_pair<kAsinh, LOG2N>(x, turn, a.log2n);
  }
}

// Running reference (a score) and sum of weights of one lane. The reference is
// the first vector's maximum until a weight passes 2^60 of it; smaller moves
// would cost a warp a rescaling at nearly every vector, for some lane of it.
constexpr float kFar = 0x1p60f;

template <int KIND, int LOG2N>
struct RowSum {
  float m, turn;
  float2 l;
  __device__ __forceinline__ void clear() {
    m = kNegInf;
    turn = KIND == kSoftmax ? -FLT_MAX : weight_turn<KIND, true>(kNegInf);
    l = make_float2(0.f, 0.f);
  }
  // The score that l is relative to. Before the reference has moved, ce weights are
  // relative to the lowest finite logit, so a row of nothing else counts too.
  __device__ __forceinline__ float reference() const {
    return KIND == kSoftmax && m == kNegInf && l.x + l.y > 0.f ? -FLT_MAX : m;
  }
  // CLEAN: NaN logits count as -inf. Without it one spoils the sum, which then is
  // taken again with it.
  template <bool CLEAN, int N>
  __device__ __forceinline__ void add(const VerifyArgs& a, const float (&z)[N]) {
    constexpr int P = (N + 1) / 2;
    float2 x[P], w[P];
    auto weigh = [&]() {
      float2 sum;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        w[i] = fast_weights<KIND, LOG2N>(a, x[i], make_float2(turn, turn));
        sum = i ? add2(sum, w[i]) : w[i];
      }
      return sum;
    };
#pragma unroll
    for (int i = 0; i < P; ++i) {
      x[i] = make_float2(z[2 * i], 2 * i + 1 < N ? z[2 * i + 1] : kNegInf);
      if (CLEAN) x[i] = make_float2(fmaxf(x[i].x, kNegInf), fmaxf(x[i].y, kNegInf));
      if (KIND == kAsinh) x[i] = mul2(x[i], make_float2(a.scale, a.scale));
    }
    float2 inc = weigh();
    if (fmaxf(inc.x, inc.y) > kFar) {  // the reference moves
      float top = m;
#pragma unroll
      for (int i = 0; i < P; ++i) top = fmaxf(top, fmaxf(x[i].x, x[i].y));
      const float to = weight_turn<KIND, true>(top);
      const float f = m == kNegInf ? 0.f : exact_weight<KIND>(a, m, to);
      l = mul2(l, make_float2(f, f));
      m = top;
      turn = to;
      inc = weigh();
    }
    l = add2(l, inc);
  }
};

__device__ __forceinline__ uint64_t pack_best(float value, int64_t v) {
  return ((uint64_t)__float_as_uint(value) << 32) | (uint32_t)~(uint32_t)v;
}

// Columns [begin, end) of a row: 16-byte vectors in the aligned middle, counted in
// blocks of kBlock, and up to 2 (N - 1) single columns at the ends, which go with
// the first block.
constexpr int kBlock = 64;
template <typename T>
struct Columns {
  static constexpr int N = Vec<T>::N;
  const T* row;
  int64_t begin, end, mid;
  int vecs;
  __device__ __forceinline__ Columns(const T* r, int64_t b, int64_t e) : row(r), begin(b), end(e) {
    const uintptr_t addr = reinterpret_cast<uintptr_t>(r + b);
    mid = min(e, b + (int64_t)(((16 - (addr & 15)) & 15) / sizeof(T)));
    vecs = (int)((e - mid) / N);
  }
  __device__ __forceinline__ int ends() const { return (int)((mid - begin) + (end - mid - (int64_t)vecs * N)); }
  __device__ __forceinline__ int64_t end_column(int i) const {
    return i < mid - begin ? begin + i : mid + (int64_t)vecs * N + (i - (mid - begin));
  }
};

template <typename T, int KIND, int LOG2N, int kCluster, int kThreads>
__global__ void __launch_bounds__(kThreads, kCluster == 16 ? 1 : 1024 / kThreads) verify_kernel(const VerifyArgs a) {
  using V = Vec<T>;
  constexpr int kWarps = kThreads / 32;
  // 16-byte loads of a lane on their way while as many are worked on
  constexpr int kFly = kCluster == 16 ? 4 : 2;
  using Cols = Columns<T>;
  __shared__ float2 s_part[kWarps + kMaxRows];  // (reference, sum) of every (warp, row) that meets, at warp + row
  __shared__ float2 s_row[2][kMaxRows];         // this CTA's (reference, sum) of every row, for two rounds
  __shared__ float s_turn[kMaxRows], s_l[kMaxRows];
  __shared__ uint64_t s_best[kWarps];
  __shared__ uint64_t s_cta_best;
  __shared__ int s_accepted;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / kCluster;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  const int K = a.counts ? min(max(a.counts[b], 0), a.K) : a.K;
  const bool has_draft = a.draft != nullptr;
  const int64_t begin = min(a.V, rank * a.slice), end = min(a.V, begin + a.slice);
  const T* target = static_cast<const T*>(a.target) + b * (a.K + 1) * a.V;
  const T* draft = static_cast<const T*>(a.draft) + b * a.K * a.V;
  const float* race = a.race + b * a.V;
  // what the decision will need, asked for early: the drafted tokens, their
  // logits, and (into L2) the race's variates
  float u = 0.f, zp = 0.f, zq = 0.f;
  bool valid = false;
  if (warp == 0 && lane < K) {
    const int32_t x = a.tokens[b * a.K + lane];
    valid = x >= 0 && x < a.V;
    if (!valid && rank == 0) atomicOr(a.err, DEV_ERR_BAD_LABEL);
    u = a.u[b * a.K + lane];
    if (valid) {
      zp = to_f32(target[(int64_t)lane * a.V + x]);
      if (has_draft) zq = to_f32(draft[(int64_t)lane * a.V + x]);
    }
  }
  for (int64_t v = begin + threadIdx.x * 32; v < end; v += kThreads * 32)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(race + v));

  // joins parts one by one; each has a reference and a sum
  auto join = [&](int count, auto part) {
    float M = kNegInf, L = 0.f;
    for (int i = 0; i < count; ++i) M = fmaxf(M, part(i).x);
    const float turn = weight_turn<KIND, true>(M);
    for (int i = 0; i < count; ++i) {
      const float2 p = part(i);
      if (p.x != kNegInf) L = fmaf(p.y, fast_weight<KIND>(a, p.x, turn), L);
    }
    return make_float2(M, L);
  };
  auto prob = [&](int r, float z) {
    const float x = score_of<KIND>(a, z);
    return x > kNegInf ? exact_weight<KIND>(a, x, s_turn[r]) / s_l[r] : 0.f;
  };
  const int blocks = (int)max((int64_t)1, (end - begin + V::N * kBlock - 1) / (V::N * kBlock));

  // Two rounds at most, the first of a.round positions: rows after a refusal are not
  // needed. Row r of a round is target row i0 + r, then draft row i0 + (r - nt).
  int acc = -1, i0 = 0, nt = 0;
  for (int turn_no = 0; acc < 0; ++turn_no) {
    i0 += nt;
    nt = turn_no == 0 ? min(K + 1, a.round) : K + 1 - i0;
    const int nd = min(K - i0, nt), rows = nt + (has_draft ? nd : 0);
    float2* const s_mine = s_row[turn_no & 1];
    // the blocks of the round's rows stand in one line, cut into equal shares of the warps
    const int share = (rows * blocks + kWarps - 1) / kWarps;
    int at = warp * share;
    const int stop = min(rows * blocks, at + share);
    while (at < stop) {
      const int r = at / blocks;
      const Cols c(r < nt ? target + (int64_t)(i0 + r) * a.V : draft + (int64_t)(i0 + r - nt) * a.V, begin, end);
      const uint4* mid = reinterpret_cast<const uint4*>(c.row + c.mid);
      const int to = min(stop, (r + 1) * blocks);
      const int v_begin = (at - r * blocks) * kBlock + lane, v_end = min(c.vecs, (to - r * blocks) * kBlock);
      const bool has_ends = at == r * blocks && lane < c.ends();
      at = to;
      RowSum<KIND, LOG2N> sum;
      auto add_up = [&](auto clean) {
        constexpr bool CLEAN = decltype(clean)::value;
        sum.clear();
        int v = v_begin;
        uint4 next[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i)
          if (v + i * 32 < v_end) next[i] = __ldg(mid + v + i * 32);
        if (has_ends) {
          const float z[1] = {to_f32(c.row[c.end_column(lane)])};
          sum.template add<CLEAN>(a, z);
        }
        for (; v < v_end; v += 32 * kFly) {
          uint4 raw[kFly];
#pragma unroll
          for (int i = 0; i < kFly; ++i) {
            raw[i] = next[i];
            if (v + (i + kFly) * 32 < v_end) next[i] = __ldg(mid + v + (i + kFly) * 32);
          }
#pragma unroll
          for (int i = 0; i < kFly; ++i)
            if (v + i * 32 < v_end) {
              float z[V::N];
              unpack<T>(raw[i], z);
              sum.template add<CLEAN>(a, z);
            }
        }
      };
      add_up(std::false_type{});
      if (__any_sync(0xffffffffu, !(sum.l.x + sum.l.y < INFINITY))) add_up(std::true_type{});
      const float mine = sum.reference();
      float M = mine;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
      float L = mine == kNegInf ? 0.f : (sum.l.x + sum.l.y) * fast_weight<KIND>(a, mine, weight_turn<KIND, true>(M));
      L = row_sum<32>(L);
      if (lane == 0) s_part[warp + r] = make_float2(M, L);
    }
    __syncthreads();
    if (threadIdx.x < rows) {
      const int r = threadIdx.x, lo = r * blocks / share, hi = ((r + 1) * blocks - 1) / share;
      s_mine[r] = join(hi - lo + 1, [&](int i) { return s_part[lo + i + r]; });
    }
    cluster.sync();
    if (threadIdx.x < rows) {
      const int r = threadIdx.x;
      float2 part[kCluster];
#pragma unroll
      for (int c = 0; c < kCluster; ++c) part[c] = *cluster.map_shared_rank(&s_mine[r], c);
      float M = kNegInf, L = 0.f;
#pragma unroll
      for (int c = 0; c < kCluster; ++c) M = fmaxf(M, part[c].x);
      const float turn = weight_turn<KIND, true>(M);
#pragma unroll
      for (int c = 0; c < kCluster; ++c)
        if (part[c].x != kNegInf) L = fmaf(part[c].y, fast_weight<KIND>(a, part[c].x, turn), L);
      s_turn[r] = turn;
      s_l[r] = L > 0.f ? L : 1.f;
    }
    __syncthreads();
    if (warp == 0) {
      bool refused = false;
      const int i = lane - i0;  // this lane's draft in the round
      if (i >= 0 && i < nd) refused = !valid || !(u * (has_draft ? prob(nt + i, zq) : 1.f) < prob(i, zp));
      const unsigned mask = __ballot_sync(0xffffffffu, refused);
      if (lane == 0) s_accepted = mask ? __ffs(mask) - 1 : i0 + nt > K ? K : -1;
    }
    __syncthreads();
    acc = s_accepted;
  }
  const T* row_p = target + (int64_t)acc * a.V;
  const T* row_q = has_draft && acc < K ? draft + (int64_t)acc * a.V : nullptr;
  const int64_t drafted = !has_draft && acc < K ? a.tokens[b * a.K + acc] : -1;
  const int rp = acc - i0, rq = nt + acc - i0;  // their rows in the last round
  const float turn_p = s_turn[rp], l_p = s_l[rp];
  const float turn_q = row_q ? s_turn[rq] : 0.f, l_q = row_q ? s_l[rq] : 1.f;
  const float inv_p = 1.f / l_p, inv_q = 1.f / l_q;
  // weight / variate of one column, as the result is compared
  auto exact_ratio = [&](bool rest, int64_t v, float xp, float xq, float e) {
    float w = xp > kNegInf ? exact_weight<KIND>(a, xp, turn_p) / l_p : 0.f;
    if (rest) w -= row_q ? (xq > kNegInf ? exact_weight<KIND>(a, xq, turn_q) / l_q : 0.f) : v == drafted ? 1.f : 0.f;
    const float ratio = w > 0.f ? w / e : 0.f;
    return ratio > 0.f ? ratio : 0.f;
  };
  // pass 0 races over the residual; where nothing of it is left, pass 1 over p
  for (int pass = acc < K ? 0 : 1; pass < 2; ++pass) {
    // The fast weights' error (race_margin) bounds every ratio from both sides. A
    // lane keeps the column that no other can be above; only where two overlap are
    // they evaluated exactly, and at the end the lanes that could hold the winner.
    float low = 0.f, up = 0.f, xp_b = kNegInf, xq_b = kNegInf, e_b = 1.f;
    int64_t v_b = min(begin + threadIdx.x, a.V - 1);
    auto enter = [&](int64_t v, float z, float zd, float e) {
      const float xp = score_of<KIND>(a, z), xq = score_of<KIND>(a, zd);
      const float2 f = fast_weights<KIND, LOG2N>(a, make_float2(xp, xq), make_float2(turn_p, turn_q));
      const float p = f.x * inv_p, q = pass == 1 ? 0.f : row_q ? f.y * inv_q : v == drafted ? 1.f : 0.f;
      const float r = rcp_fast(e), mid = (p - q) * r, off = fmaf(p + q, a.margin, kFlushed) * r;
      if (!(mid + off > low) || !(xp > kNegInf)) return;  // the latter: no probability
      bool take = mid - off > up;
      float lo = mid - off, hi = mid + off;
      if (!take) {
        const float mine = exact_ratio(pass == 0, v, xp, xq, e);
        const float held = up > 0.f ? exact_ratio(pass == 0, v_b, xp_b, xq_b, e_b) : 0.f;
        take = mine > held || (mine == held && v < v_b);
        lo = hi = mine;
        if (!take) low = up = held;
      }
      if (take) {
        low = lo; up = hi; xp_b = xp; xq_b = xq; e_b = e; v_b = v;
      }
    };
    const bool rest = pass == 0 && row_q;
    const Cols c(row_p, begin, end);
    if (threadIdx.x < c.ends()) {
      const int64_t v = c.end_column(threadIdx.x);
      enter(v, to_f32(row_p[v]), rest ? to_f32(row_q[v]) : kNegInf, race[v]);
    }
    // the three rows need not be aligned alike: vectors where they are
    const bool vec = ((reinterpret_cast<uintptr_t>(race + c.mid) & 15) == 0) &&
                     (!rest || (reinterpret_cast<uintptr_t>(row_q + c.mid) & 15) == 0);
    if (vec) {
      struct Three {
        uint4 p, q;
        float4 e[V::N / 4];
      };
      auto load = [&](Three& x, int i) {
        if (i >= c.vecs) return;
        const int64_t v = c.mid + (int64_t)i * V::N;
        x.p = __ldg(reinterpret_cast<const uint4*>(row_p + v));
        if (rest) x.q = __ldg(reinterpret_cast<const uint4*>(row_q + v));
#pragma unroll
        for (int j = 0; j < V::N / 4; ++j) x.e[j] = __ldg(reinterpret_cast<const float4*>(race + v) + j);
      };
      Three next;
      load(next, threadIdx.x);
      for (int i = threadIdx.x; i < c.vecs; i += kThreads) {
        const Three x = next;
        load(next, i + kThreads);
        float z[V::N], zd[V::N];
        unpack<T>(x.p, z);
        if (rest) unpack<T>(x.q, zd);
        const float* e = reinterpret_cast<const float*>(x.e);
#pragma unroll
        for (int j = 0; j < V::N; ++j) enter(c.mid + (int64_t)i * V::N + j, z[j], rest ? zd[j] : kNegInf, e[j]);
      }
    } else {
      for (int64_t v = c.mid + threadIdx.x; v < c.mid + (int64_t)c.vecs * V::N; v += kThreads)
        enter(v, to_f32(row_p[v]), rest ? to_f32(row_q[v]) : kNegInf, race[v]);
    }
    float sure = low;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sure = fmaxf(sure, __shfl_xor_sync(0xffffffffu, sure, off));
    uint64_t best_at = pack_best(0.f, v_b);
    if (up > 0.f && up >= sure) best_at = pack_best(exact_ratio(pass == 0, v_b, xp_b, xq_b, e_b), v_b);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, best_at, off);
      best_at = best_at > o ? best_at : o;
    }
    if (lane == 0) s_best[warp] = best_at;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 1; i < kWarps; ++i) best_at = best_at > s_best[i] ? best_at : s_best[i];
      s_cta_best = best_at;
    }
    cluster.sync();
    uint64_t all = 0;
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      const uint64_t o = *cluster.map_shared_rank(&s_cta_best, c);
      all = all > o ? all : o;
    }
    const bool empty = (all >> 32) == 0;
    if (rank == 0 && (int)threadIdx.x <= a.K && (pass == 1 || !empty)) {
      const int i = threadIdx.x;
      a.out[b * (a.K + 1) + i] = i < acc ? a.tokens[b * a.K + i] : i == acc ? (int32_t)~(uint32_t)all : -1;
      if (i == 0) a.accepted[b] = acc;
    }
    cluster.sync();  // nobody leaves, or writes its best again, while others read it
    if (!empty) break;
  }
}

template <int CL, int TH, typename T>
auto pick(int32_t kind, int log2n) -> void (*)(VerifyArgs) {
  if (kind == ALGX_HEAD_CE) return verify_kernel<T, kSoftmax, 0, CL, TH>;
  return log2n == 3 ? verify_kernel<T, kAsinh, 3, CL, TH> : verify_kernel<T, kAsinh, 0, CL, TH>;
}

template <int CL, int TH>
int verify_launch(const VerifyArgs& a, int32_t kind, int32_t dtype, int64_t B, cudaStream_t st) {
  auto* kern = dtype == ALGX_BF16 ? pick<CL, TH, __nv_bfloat16>(kind, a.log2n) : pick<CL, TH, float>(kind, a.log2n);
  if (CL > 8)  // clusters above 8 CTAs are this device's, not every one's
    ALGX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * CL));
  cfg.blockDim = dim3(TH);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CL;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  ALGX_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  ALGX_LAUNCHED("verify_kernel");
  return ALGX_OK;
}

}  // namespace
}  // namespace algx

extern "C" int algx_verify_draft(int32_t kind, int32_t n, float scale, const void* target, const void* draft,
                                 const int32_t* tokens, const int32_t* counts, const float* u, const float* race,
                                 int32_t* out, int32_t* accepted, int64_t B, int64_t K, int64_t V, int32_t dtype,
                                 void* stream) {
  using namespace algx;
  ALGX_REQUIRE(dtype == ALGX_F32 || dtype == ALGX_BF16, "dtype must be f32 or bf16");
  ALGX_REQUIRE(kind == ALGX_HEAD_CE || kind == ALGX_HEAD_ALG_CE, "unknown head kind");
  ALGX_REQUIRE(kind == ALGX_HEAD_CE || (n >= 2 && (n & (n - 1)) == 0), "n must be a power of two");
  ALGX_REQUIRE(B >= 0 && K >= 0 && K < 32, "at most 31 drafted tokens");
  ALGX_REQUIRE(V >= 1 && V <= INT32_MAX, "the vocabulary must not be empty");
  ALGX_REQUIRE(scale > 0.f && std::isfinite(scale), "scale must be positive and finite");
  if (B == 0) return ALGX_OK;
  ALGX_REQUIRE(B <= INT32_MAX / 16, "too many sequences");
  ALGX_REQUIRE(target && race && out && accepted && (K == 0 || (tokens && u)), "NULL tensor");
  VerifyArgs a = {};
  a.target = target; a.draft = K > 0 ? draft : nullptr; a.tokens = tokens; a.counts = counts; a.u = u; a.race = race;
  a.out = out; a.accepted = accepted; a.V = V; a.K = (int)K;
  a.scale = scale;
  a.margin = race_margin(kind, n);
  while ((1 << a.log2n) < n) ++a.log2n;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Few sequences: all rows in one round, whose time is latency, over as many SMs
  // as a cluster spans. Where the clusters fill the device, four positions
  // first, as rows behind a refusal are mostly not read, and smaller CTAs, four
  // an SM, which leave less of a last wave. (64 sequences of 7 drafts: 60.8, 55.8,
  // 56.5, 54.6, 57.3 us with one to five positions first, 60 with all; two CTAs of 512
  // threads an SM took 100 instead of 74 at an earlier step.)
  //
  // Clusters of 16 only where a thread of 8 CTAs would read 96 logits or more. (16
  // CTAs and 8: one user's 4 drafts over 50304 10.9 us and 13.9, 7 drafts over 32000
  // 10.4 and 12.4; 4 drafts over 32000 with alg_ce 17.8 and 16.6, 9 sequences of one
  // draft over 3968 24.2 and 10.4.)
  const bool wide = B * 8 <= 2 * 148, few = B * 16 <= 148 && (2 * K + 1) * V >= 96 * 8 * 512;
  const int64_t cluster = few ? 16 : 8;
  a.round = wide ? (int)K + 1 : 4;
  a.slice = ((V + cluster - 1) / cluster + 7) / 8 * 8;
  return few    ? verify_launch<16, 512>(a, kind, dtype, B, st)
         : wide ? verify_launch<8, 512>(a, kind, dtype, B, st)
                : verify_launch<8, 256>(a, kind, dtype, B, st);
}
