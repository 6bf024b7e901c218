// What the paged-cache kernels share: the cache's layout and the two score
// weights, asinh-power (algebraic.py:186-204) and softmax.
#pragma once

#include "algx_common.cuh"

namespace algx {

// Keys and values live in pages: k_pages, v_pages (num_pages, Hkv, page_size,
// 64). Slot s of sequence b lies in page table[b * max_pages + s / page_size] at
// row s % page_size. page_size is a power of two of at least 16, so an aligned
// group of 16 slots never straddles two pages.
struct PagedView {
  const int32_t* table;
  const int32_t* lens;
  int32_t num_pages;
  int32_t max_pages;
  int32_t page_shift;  // log2(page_size)
  int32_t heads;       // Hkv
};

// The view of a call's arguments, or an error status (cache.cu).
int paged_view(PagedView* pv, const void* table, const void* lens, int64_t B, int64_t Hkv, int64_t num_pages,
               int64_t page_size, int64_t max_pages, int64_t D);
int* device_error_word();

// First element of the row that holds slot `s` for head h in page `pid`.
__device__ __forceinline__ int64_t paged_row(const PagedView& pv, int pid, int h, int s) {
  const int64_t in_page = s & ((1 << pv.page_shift) - 1);
  return ((((int64_t)pid * pv.heads + h) << pv.page_shift) + in_page) * 64;
}

// Slots of sequence b that the table can address, 0 for a negative length.
__device__ __forceinline__ int paged_len(const PagedView& pv, int b, int* err) {
  const int len = pv.lens[b];
  const int64_t cap = (int64_t)pv.max_pages << pv.page_shift;
  if (len > cap) {
    if (threadIdx.x == 0) atomicOr(err, DEV_ERR_BAD_PAGE);
    return (int)cap;
  }
  return len < 0 ? 0 : len;
}

// rho(x) for either sign (kernels/flash.py:76-80): |x| + sqrt(1 + x^2), or its
// reciprocal for x < 0. EXACT uses correctly rounded square root and division
// (float32 I/O); otherwise the MUFU forms with about 2^-22 relative error,
// 16 times that in a 16th power, far below bf16's 2^-9.
template <bool EXACT>
__device__ __forceinline__ float rho_any(float x) {
  const float rad = fmaf(x, x, 1.f);
  if constexpr (EXACT) {
    const float t = fabsf(x) + sqrtf(rad);
    return x >= 0.f ? t : 1.f / t;
  } else {
    float s;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(rad));
    const float t = fabsf(x) + s;
    return x >= 0.f ? t : rcp_fast(t);
  }
}

__device__ __forceinline__ float pow_log2(float x, int log2n) {
  for (int i = 0; i < log2n; ++i) x *= x;
  return x;
}

// Weight of a score x against a reference score m: (rho(x) rho(-m))^n for the
// asinh kind, 2^(x - m) for softmax, whose scores carry a factor log2(e). `turn`
// is the reference's part, computed once per reference; before any score is seen
// (m = -inf) it is so large that every finite score has a huge weight, and a
// masked one (x = -inf) none.
constexpr int kAsinh = ALGX_ATTN_ASINH, kSoftmax = ALGX_ATTN_SOFTMAX;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -INFINITY;

template <int KIND, bool EXACT>
__device__ __forceinline__ float weight_turn(float m) {
  if constexpr (KIND == kAsinh) return m == kNegInf ? 3e38f : rho_any<EXACT>(-m);
  else return m == kNegInf ? -3e38f : m;
}
template <int KIND, bool EXACT>
__device__ __forceinline__ float weight_of(float x, float turn, int log2n) {
  if constexpr (KIND == kSoftmax) {
    if constexpr (EXACT) return exp2f(x - turn);
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x - turn));
    return y;
  } else {
    return pow_log2(rho_any<EXACT>(x) * turn, log2n);
  }
}

// The same weights for two scores at once on packed fp32 pairs, MUFU forms.
// LOG2N > 0: the power is known when compiling.
template <int KIND, int LOG2N>
__device__ __forceinline__ float2 weight_pair(float2 x, float2 turn, int log2n) {
  float2 y;
  if constexpr (KIND == kSoftmax) {
    y = sub2(x, turn);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(y.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(y.y));
    return y;
  } else {
    y = fma2(x, x, make_float2(1.f, 1.f));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(y.x));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(y.y));
    y.x += fabsf(x.x);
    y.y += fabsf(x.y);
    const float rx = rcp_fast(y.x), ry = rcp_fast(y.y);
    y.x = x.x >= 0.f ? y.x : rx;
    y.y = x.y >= 0.f ? y.y : ry;
    y = mul2(y, turn);
    if constexpr (LOG2N > 0) {
#pragma unroll
      for (int i = 0; i < LOG2N; ++i) y = mul2(y, y);
    } else {
      for (int i = 0; i < log2n; ++i) y = mul2(y, y);
    }
    return y;
  }
}

// weight_pair of the scores scale x; softmax takes the negative reference, -m.
template <int KIND, int LOG2N>
__device__ __forceinline__ float2 weight_scaled(float2 x, float2 scale, float2 turn, int log2n) {
  if constexpr (KIND == kSoftmax) {
    float2 y = fma2(x, scale, turn);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(y.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(y.y));
    return y;
  } else {
    return weight_pair<KIND, LOG2N>(mul2(x, scale), turn, log2n);
  }
}

// Which slots a query sees. Query token t of T new ones stands at slot
// last = len - T + t and sees slots s <= last with s > last - window or
// s < first (window 0: no window).
struct Sight {
  int window;
  int first;
  __device__ __forceinline__ bool sees(int s, int last) const {
    return s <= last && (window == 0 || s > last - window || s < first);
  }
  // Whether every query with lo <= last <= hi sees every slot of s .. s + n - 1.
  __device__ __forceinline__ bool sees_all(int s, int n, int lo, int hi) const {
    return s + n - 1 <= lo && (window == 0 || s > hi - window || s + n - 1 < first);
  }
};

// The aligned groups of 2^shift slots that queries with lo <= last <= hi look at:
// the groups of the first visible slots, then those from the window's left end on.
struct Span {
  int head_groups;  // groups before the gap
  int skip;         // groups in the gap
  int total;        // groups to visit
  __device__ __forceinline__ Span(const Sight& w, int shift, int lo, int hi) {
    const int end = max(0, hi + 1), more = (1 << shift) - 1;
    const int groups = (end + more) >> shift;
    head_groups = 0;
    skip = 0;
    if (w.window != 0) {
      const int left = max(0, max(lo, 0) - w.window + 1) >> shift;  // queries before slot 0 see nothing
      const int head = (min(w.first, end) + more) >> shift;
      if (head < left) {
        head_groups = head;
        skip = min(left, groups) - head;
      }
    }
    total = groups - skip;
  }
  // Number of the i-th group to visit.
  __device__ __forceinline__ int group(int i) const { return i < head_groups ? i : i + skip; }
};

}  // namespace algx
