// Shared by the operators on rows of logits (ag_logprobs.cu, ag_distill.cu): argument checks, the exponential, softmax
// statistics that can be merged.
#pragma once

#include <math.h>

#include "ag_common.cuh"

constexpr float AG_LN2 = 0.69314718055994531f, AG_LOG2E = 1.44269504088896341f;

// Launches go to the context's device, whichever is current in the calling thread.
struct AgOnDevice {
  int before = -1;
  explicit AgOnDevice(const ag_ctx* ctx) {
    int now = -1;
    if (cudaGetDevice(&now) == cudaSuccess && now != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess) before = now;
  }
  ~AgOnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

struct AgVocabShape {
  int64_t N, ld, ld_grad;
  int V, top, dtype;
  float temperature;
  size_t size() const { return dtype == AG_F32 ? 4 : 2; }
};

static inline int ag_vocab_check(ag_ctx* ctx, const char* who, const AgVocabShape& s, int max_v, int max_top, const void* logits,
                                 const void* dres, const void* dlogits) {
  AG_REQUIRE(ctx, s.N >= 0 && s.N < (1ll << 31) && s.V > 0 && s.V <= max_v, "%s: bad shape N=%lld V=%d (V up to %d)", who,
             (long long)s.N, s.V, max_v);
  AG_REQUIRE(ctx, s.dtype == AG_F32 || s.dtype == AG_BF16, "%s: unknown dtype %d", who, s.dtype);
  AG_REQUIRE(ctx, s.temperature >= 1e-4f && s.temperature <= 1e4f, "%s: temperature %g outside 1e-4 to 1e4", who, s.temperature);
  AG_REQUIRE(ctx, s.top >= 0 && s.top <= max_top && s.top <= s.V, "%s: %d tokens per row, up to %d and V", who, s.top, max_top);
  // beyond 2^40 elements the products below would overflow before they could be compared with anything
  AG_REQUIRE(ctx, s.ld >= s.V && s.ld < (1ll << 31), "%s: row stride %lld smaller than V=%d, or too large", who, (long long)s.ld, s.V);
  AG_REQUIRE(ctx, logits || s.N == 0, "%s: null logits", who);
  const uintptr_t mask = s.size() - 1;
  AG_REQUIRE(ctx, ((uintptr_t)logits & mask) == 0, "%s: logits not aligned to their type", who);
  if (s.ld_grad < 0) return AG_OK;  // no gradient in this call
  AG_REQUIRE(ctx, s.ld_grad >= s.V && s.ld_grad < (1ll << 31), "%s: gradient row stride %lld smaller than V=%d, or too large", who,
             (long long)s.ld_grad, s.V);
  AG_REQUIRE(ctx, dlogits || s.N == 0, "%s: null gradient", who);
  AG_REQUIRE(ctx, (((uintptr_t)dlogits | (uintptr_t)dres) & mask) == 0, "%s: gradient not aligned to its type", who);
  if (s.N == 0) return AG_OK;
  // A block writes its row's gradient while others still read theirs: apart, or row for row in the same place.
  auto apart = [&](const void* a, int64_t lda, const void* b, int64_t ldb) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b, a1 = a0 + ((size_t)(s.N - 1) * lda + s.V) * s.size(),
                    b1 = b0 + ((size_t)(s.N - 1) * ldb + s.V) * s.size();
    return a1 <= b0 || b1 <= a0 || (a0 == b0 && (lda == ldb || s.N == 1));
  };
  AG_REQUIRE(ctx, apart(logits, s.ld, dlogits, s.ld_grad), "%s: gradient overlaps the logits otherwise than in place", who);
  AG_REQUIRE(ctx, !dres || apart(dres, s.ld_grad, dlogits, s.ld_grad), "%s: gradient overlaps dres otherwise than in place", who);
  return AG_OK;
}

#ifdef __CUDACC__

// 2^x to 2^-22 of the result (what a sum of thousands of terms in 32 bits loses anyway); -inf gives 0.
__device__ __forceinline__ float ag_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Statistics of a part of a row in units of log 2: m the largest logit, s = sum 2^d, t = sum 2^d d with d = (x - m) * c,
// c = log2(e) / temperature.  Terms whose 2^d is 0 add nothing to t, however small d is.  m = -inf: nothing above -inf yet,
// s = t = 0.  A NaN or +inf among the logits makes s NaN.
struct AgStat {
  float m, s, t;
};
__device__ __forceinline__ AgStat ag_stat_none() { return {-INFINITY, 0.0f, 0.0f}; }
__device__ __forceinline__ AgStat ag_stat_merge(const AgStat& a, const AgStat& b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.t + b.t};
  const float da = (a.m - m) * c, db = (b.m - m) * c;  // one of them 0, the other possibly -inf: of an empty part
  const float ea = ag_ex2(da), eb = ag_ex2(db);
  // s 2^d, and t 2^d + s 2^d d; NaN stays in s
  return {m, a.s * ea + b.s * eb, (ea > 0.0f ? ea * (a.t + a.s * da) : 0.0f) + (eb > 0.0f ? eb * (b.t + b.s * db) : 0.0f)};
}

__device__ __forceinline__ AgStat ag_stat_warp(AgStat v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const AgStat w = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o), __shfl_xor_sync(0xffffffffu, v.t, o)};
    v = ag_stat_merge(v, w, c);
  }
  return v;
}

// The order of the alternatives: larger logits first (NaN before all, -0 beside +0), equal ones by the lower index.
__device__ __forceinline__ uint32_t ag_order(float x) {
  if (x != x) return 0xfffffffeu;  // above every other, below the start of a search
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 + 0 = +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ag_of_order(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);  // 0xfffffffe becomes a NaN again
}

#endif  // __CUDACC__
