// Log-probabilities of given tokens, entropies and likeliest tokens of rows of logits, and their gradient.
//
//   z = x / temperature,  m = max x,  L = ln sum exp((x - m) / temperature),  log p_j = (x_j - m) / temperature - L
//   entropy H = L - sum_j p_j (x_j - m) / temperature
//   d logits_j = (a (delta_j,id - p_j) - b p_j (log p_j + H)) / temperature,  a = dlogprob (0 without a token), b = dentropy
//
// A block takes a row and reads it once for the statistics, once more from L2 for each alternative.
#include "ag_vocab.cuh"

namespace {

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;

template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
logprobs_kernel(const T* __restrict__ logits, int64_t ld, const int32_t* __restrict__ ids, float* logprob, float* entropy,
                float4* stats, int32_t* top_ids, float* top_logprobs, int V, int top, float inv_tau) {
  __shared__ AgStat s_stat[LP_WARPS];
  __shared__ unsigned long long s_key[LP_WARPS];
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const float c = inv_tau * AG_LOG2E;
  AgStat v = ag_stat_none();
  for (int j = threadIdx.x; j < V; j += LP_THREADS) {
    const float xj = Pack<T>::load1(x + j);
    v = ag_stat_merge(v, {xj, xj == -INFINITY ? 0.0f : xj - xj + 1.0f, 0.0f}, c);  // inf - inf and NaN: a NaN for the sum
  }
  v = ag_stat_warp(v, c);
  if ((threadIdx.x & 31) == 0) s_stat[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_stat[0];
  for (int w = 1; w < LP_WARPS; ++w) v = ag_stat_merge(v, s_stat[w], c);
  const float L = logf(v.s), H = v.m == -INFINITY && v.s == 0.0f ? 0.0f : L - AG_LN2 * (v.t / v.s);
  auto log_p = [&](float xj) { return xj == -INFINITY && !(v.s != v.s) ? -INFINITY : (xj - v.m) * inv_tau - L; };
  if (threadIdx.x == 0) {
    if (logprob) {
      const int id = ids[row];
      logprob[row] = id >= 0 && id < V ? log_p(Pack<T>::load1(x + id)) : 0.0f;
    }
    if (entropy) entropy[row] = H;
    if (stats) stats[row] = make_float4(v.m, L, H, 0.0f);
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < V; j += LP_THREADS) {
      const unsigned long long key = (unsigned long long)ag_order(Pack<T>::load1(x + j)) << 32 | (uint32_t)(~j);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long w = __shfl_xor_sync(0xffffffffu, best, o);
      best = w > best ? w : best;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_key[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < LP_WARPS; ++w) best = s_key[w] > best ? s_key[w] : best;
    if (threadIdx.x == 0) {
      top_ids[row * top + k] = (int32_t)~(uint32_t)best;
      top_logprobs[row * top + k] = log_p(ag_of_order((uint32_t)(best >> 32)));
    }
    last = best;
  }
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
logprobs_backward_kernel(const T* logits, int64_t ld, const int32_t* __restrict__ ids, const float4* __restrict__ stats,
                         const float* __restrict__ dlogprob, const float* __restrict__ dentropy, const T* dres, T* dlogits,
                         int64_t ld_grad, int V, float inv_tau) {
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t row = blockIdx.x;
  const float4 st = stats[row];
  const int id = ids ? ids[row] : -1;
  const float a = dlogprob && id >= 0 && id < V ? dlogprob[row] * inv_tau : 0.0f, b = dentropy ? dentropy[row] * inv_tau : 0.0f;
  const bool none = (a == 0.0f && b == 0.0f) || (st.x == -INFINITY && st.y == -INFINITY);
  for (int j = threadIdx.x; j < V; j += LP_THREADS) {
    const float xj = Pack<T>::load1(logits + row * ld + j);
    const float lp = fmaxf((xj - st.x) * inv_tau, -1e4f) - st.y;  // -inf: p = 0, and 0 times something finite
    const float p = ag_ex2(lp * AG_LOG2E);
    float g = none ? 0.0f : (j == id ? a : 0.0f) - p * (a + b * (lp + st.z));
    if (dres) g += Pack<T>::load1(dres + row * ld_grad + j);
    Pack<T>::store1(dlogits + row * ld_grad + j, g);
  }
}

}  // namespace

extern "C" int ag_token_logprobs_forward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* ids, float* logprob,
                                         float* entropy, float* stats, int32_t* top_ids, float* top_logprobs, int64_t N, int V,
                                         int top, float temperature, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  const char* who = "ag_token_logprobs_forward";
  if (int rc = ag_vocab_check(ctx, who, {N, ld, -1, V, top, dtype, temperature}, AG_VOCAB_MAX, AG_TOP_MAX, logits, nullptr, nullptr))
    return rc;
  AG_REQUIRE(ctx, !logprob || ids, "%s: log-probabilities of no tokens", who);
  AG_REQUIRE(ctx, top == 0 || (top_ids && top_logprobs) || N == 0, "%s: null pointer", who);
  AG_REQUIRE(ctx, ag_aligned16(stats), "%s: stats not 16-byte aligned", who);
  if (N == 0) return AG_OK;
  AgOnDevice on(ctx);
  const float inv = 1.0f / temperature;
  if (dtype == AG_F32)
    AG_LAUNCH_PDL(ctx, "logprobs_kernel", logprobs_kernel<float>, (unsigned)N, LP_THREADS, 0, (const float*)logits, ld, ids, logprob,
                  entropy, (float4*)stats, top_ids, top_logprobs, V, top, inv);
  else
    AG_LAUNCH_PDL(ctx, "logprobs_kernel", logprobs_kernel<__nv_bfloat16>, (unsigned)N, LP_THREADS, 0, (const __nv_bfloat16*)logits, ld,
                  ids, logprob, entropy, (float4*)stats, top_ids, top_logprobs, V, top, inv);
  return AG_OK;
}

extern "C" int ag_token_logprobs_backward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* ids, const float* stats,
                                          const float* dlogprob, const float* dentropy, const void* dres, void* dlogits,
                                          int64_t ld_grad, int64_t N, int V, float temperature, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  const char* who = "ag_token_logprobs_backward";
  AG_REQUIRE(ctx, ld_grad >= 0, "%s: negative gradient row stride", who);
  if (int rc = ag_vocab_check(ctx, who, {N, ld, ld_grad, V, 0, dtype, temperature}, INT32_MAX, 0, logits, dres, dlogits)) return rc;
  AG_REQUIRE(ctx, !dlogprob || ids, "%s: a gradient of log-probabilities of no tokens", who);
  AG_REQUIRE(ctx, stats || N == 0, "%s: null stats", who);
  AG_REQUIRE(ctx, ag_aligned16(stats), "%s: stats not 16-byte aligned", who);
  if (N == 0) return AG_OK;
  AgOnDevice on(ctx);
  const float inv = 1.0f / temperature;
  if (dtype == AG_F32)
    AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", logprobs_backward_kernel<float>, (unsigned)N, LP_THREADS, 0, (const float*)logits,
                  ld, ids, (const float4*)stats, dlogprob, dentropy, (const float*)dres, (float*)dlogits, ld_grad, V, inv);
  else
    AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", logprobs_backward_kernel<__nv_bfloat16>, (unsigned)N, LP_THREADS, 0,
                  (const __nv_bfloat16*)logits, ld, ids, (const float4*)stats, dlogprob, dentropy, (const __nv_bfloat16*)dres,
                  (__nv_bfloat16*)dlogits, ld_grad, V, inv);
  return AG_OK;
}
