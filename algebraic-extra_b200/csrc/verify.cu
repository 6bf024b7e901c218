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
#include <cooperative_groups.h>

#include <algorithm>

#include "paged_common.cuh"
#include "vec_io.cuh"

namespace cg = cooperative_groups;

namespace algx {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kMaxDraft = 32;

struct VerifyArgs {
  const void *target, *draft;
  const int32_t *tokens, *counts;
  const float *u, *race;
  int32_t *out, *accepted;
  int* err;
  int64_t V, slice;  // slice: vocabulary columns of one CTA, a multiple of 8
  int K, log2n;
  float scale;  // log2(e) / temperature (ce) or 1 / c (alg_ce)
};

// Running reference and sum of one lane over one row's elements.
template <int KIND>
struct RowSum {
  float m = kNegInf, turn = 0.f, l = 0.f;
  __device__ __forceinline__ void add(float x, int log2n) {
    if (!(x > kNegInf)) return;  // -inf and NaN logits have no probability
    if (x > m) {
      const float t = weight_turn<KIND, true>(x);
      l = m == kNegInf ? 0.f : l * weight_of<KIND, true>(m, t, log2n);
      m = x;
      turn = t;
    }
    l += weight_of<KIND, true>(x, turn, log2n);
  }
};

// f(column, value) over the columns [begin, end) of a row, 16-byte loads on the
// aligned middle, spread over `lanes` threads.
template <typename T, typename F>
__device__ __forceinline__ void for_columns(const T* row, int64_t begin, int64_t end, int me, int lanes, F f) {
  using V = Vec<T>;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(row + begin);
  int64_t head = (int64_t)(((16 - (addr & 15)) & 15) / sizeof(T));
  if (head > end - begin) head = end - begin;
  for (int64_t v = begin + me; v < begin + head; v += lanes) f(v, to_f32(row[v]));
  const int64_t mid = begin + head, vecs = (end - mid) / V::N;
#pragma unroll 4
  for (int64_t i = me; i < vecs; i += lanes) {
    float x[V::N];
    unpack<T>(*reinterpret_cast<const uint4*>(row + mid + i * V::N), x);
#pragma unroll
    for (int j = 0; j < V::N; ++j) f(mid + i * V::N + j, x[j]);
  }
  for (int64_t v = mid + vecs * V::N + me; v < end; v += lanes) f(v, to_f32(row[v]));
}

__device__ __forceinline__ uint64_t pack_best(float value, int64_t v) {
  return ((uint64_t)__float_as_uint(value) << 32) | (uint32_t)~(uint32_t)v;
}

template <typename T, int KIND>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) verify_kernel(const VerifyArgs a) {
  __shared__ float2 s_part[2 * kMaxDraft + 1];  // this CTA's (reference, sum) of every row
  __shared__ float s_m[2 * kMaxDraft + 1], s_l[2 * kMaxDraft + 1];
  __shared__ uint64_t s_best[kWarps];
  __shared__ uint64_t s_cta_best;
  __shared__ int s_accepted;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / kCluster;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int K = a.counts ? min(max(a.counts[b], 0), a.K) : a.K;
  const bool has_draft = a.draft != nullptr;
  const int rows = K + 1 + (has_draft ? K : 0);
  const int64_t begin = min(a.V, rank * a.slice), end = min(a.V, begin + a.slice);
  const T* target = static_cast<const T*>(a.target) + b * (a.K + 1) * a.V;
  const T* draft = static_cast<const T*>(a.draft) + b * a.K * a.V;
  auto row_of = [&](int r) { return r <= K ? target + (int64_t)r * a.V : draft + (int64_t)(r - K - 1) * a.V; };

  for (int r = warp; r < rows; r += kWarps) {
    RowSum<KIND> sum;
    for_columns(row_of(r), begin, end, lane, 32, [&](int64_t, float z) { sum.add(z * a.scale, a.log2n); });
    float M = sum.m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float L = sum.m == kNegInf ? 0.f : sum.l * weight_of<KIND, true>(sum.m, weight_turn<KIND, true>(M), a.log2n);
    L = row_sum<32>(L);
    if (lane == 0) s_part[r] = make_float2(M, L);
  }
  cluster.sync();
  for (int r = threadIdx.x; r < rows; r += kThreads) {
    float2 part[kCluster];
    float M = kNegInf, L = 0.f;
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      part[c] = *cluster.map_shared_rank(&s_part[r], c);
      M = fmaxf(M, part[c].x);
    }
    const float turn = weight_turn<KIND, true>(M);
#pragma unroll
    for (int c = 0; c < kCluster; ++c)
      if (part[c].x != kNegInf) L = fmaf(part[c].y, weight_of<KIND, true>(part[c].x, turn, a.log2n), L);
    s_m[r] = turn;
    s_l[r] = L > 0.f ? L : 1.f;
  }
  __syncthreads();
  auto prob = [&](int r, float z) {
    const float x = z * a.scale;
    return x > kNegInf ? weight_of<KIND, true>(x, s_m[r], a.log2n) / s_l[r] : 0.f;
  };
  if (warp == 0) {
    bool refused = false;
    if (lane < K) {
      const int32_t x = a.tokens[b * a.K + lane];
      if (x < 0 || x >= a.V) {
        refused = true;
        if (rank == 0) atomicOr(a.err, DEV_ERR_BAD_LABEL);
      } else {
        const float p = prob(lane, to_f32(target[(int64_t)lane * a.V + x]));
        const float q = has_draft ? prob(K + 1 + lane, to_f32(draft[(int64_t)lane * a.V + x])) : 1.f;
        refused = !(a.u[b * a.K + lane] * q < p);
      }
    }
    const unsigned mask = __ballot_sync(0xffffffffu, refused);
    if (lane == 0) s_accepted = mask ? __ffs(mask) - 1 : K;
  }
  __syncthreads();
  const int acc = s_accepted;
  const float* race = a.race + b * a.V;
  const T* zp = target + (int64_t)acc * a.V;
  const T* zq = has_draft && acc < K ? draft + (int64_t)acc * a.V : nullptr;
  const int64_t drafted = !has_draft && acc < K ? a.tokens[b * a.K + acc] : -1;
  // pass 0 races over the residual; where nothing of it is left, pass 1 over p
  for (int pass = acc < K ? 0 : 1; pass < 2; ++pass) {
    uint64_t best = 0;
    for_columns(zp, begin, end, threadIdx.x, kThreads, [&](int64_t v, float z) {
      float w = prob(acc, z);
      if (pass == 0) {
        const float q = zq ? prob(K + 1 + acc, to_f32(zq[v])) : v == drafted ? 1.f : 0.f;
        w = fmaxf(w - q, 0.f);
      }
      const float ratio = w > 0.f ? w / race[v] : 0.f;
      const uint64_t at = pack_best(ratio > 0.f ? ratio : 0.f, v);
      best = best > at ? best : at;
    });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, best, off);
      best = best > o ? best : o;
    }
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kWarps; ++i) best = best > s_best[i] ? best : s_best[i];
      s_cta_best = best;
    }
    cluster.sync();
    uint64_t all = 0;
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      const uint64_t o = *cluster.map_shared_rank(&s_cta_best, c);
      all = all > o ? all : o;
    }
    const bool empty = (all >> 32) == 0;
    if (rank == 0 && threadIdx.x == 0 && (pass == 1 || !empty)) {
      for (int i = 0; i <= a.K; ++i)
        a.out[b * (a.K + 1) + i] =
            i < acc ? a.tokens[b * a.K + i] : i == acc ? (int32_t)~(uint32_t)all : -1;
      a.accepted[b] = acc;
    }
    cluster.sync();  // nobody leaves, or writes its best again, while others read it
    if (!empty) break;
  }
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
  ALGX_REQUIRE(scale > 0.f, "scale must be positive");
  if (B == 0) return ALGX_OK;
  ALGX_REQUIRE(B <= INT32_MAX / kCluster, "too many sequences");
  ALGX_REQUIRE(target && race && out && accepted && (K == 0 || (tokens && u)), "NULL tensor");
  ALGX_REQUIRE((((uintptr_t)target | (uintptr_t)draft) & 3) == 0, "logits must be 4-byte aligned");
  VerifyArgs a = {};
  a.target = target; a.draft = K > 0 ? draft : nullptr; a.tokens = tokens; a.counts = counts; a.u = u; a.race = race;
  a.out = out; a.accepted = accepted; a.V = V; a.K = (int)K;
  a.scale = kind == ALGX_HEAD_CE ? scale * kLog2e : scale;
  a.slice = ((V + kCluster - 1) / kCluster + 7) / 8 * 8;
  while ((1 << a.log2n) < n) ++a.log2n;
  a.err = device_error_word();
  ALGX_REQUIRE(a.err != nullptr, "device error word unavailable");
  auto* kern = dtype == ALGX_BF16 ? (kind == ALGX_HEAD_CE ? verify_kernel<__nv_bfloat16, kSoftmax>
                                                          : verify_kernel<__nv_bfloat16, kAsinh>)
                                  : (kind == ALGX_HEAD_CE ? verify_kernel<float, kSoftmax>
                                                          : verify_kernel<float, kAsinh>);
  kern<<<(unsigned)(B * kCluster), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  ALGX_LAUNCHED("verify_kernel");
  return ALGX_OK;
}
