// Distillation from a teacher's top logits: a row's loss against the teacher's distribution over a list of tokens, and its
// gradient.  With p = softmax(x / temperature) over the V tokens, slots k of the row's list with token id_k and value t_k:
//
//   RENORM  q = softmax(t / temperature) over the slots, r = 0
//   REST    q_k = exp(t_k), r = max(0, 1 - sum q): t are log-probabilities, r what they leave to all other tokens together
//   row_loss = sum_k q_k (ln q_k - ln p_id_k) + r (ln r - ln p_rest),  p_rest = sum of p over the tokens not listed
//   d logits_j = s / temperature (p_j (Q + r) - sum_{k: id_k = j} q_k - r [j not listed] p_j / p_rest),  Q = sum q
//
// p_rest is summed over the unlisted logits themselves: 1 - sum_k p_id_k would keep nothing of a small rest.  A slot with a
// negative id is not in use.  A block takes a row; a bitmap of the row's listed tokens in shared memory tells them apart.
#include "ag_vocab.cuh"

namespace {

constexpr int DI_THREADS = 512;
constexpr int DI_WARPS = DI_THREADS / 32;

struct DistillArgs {
  const int32_t* ids;
  const float* teacher;
  const float* row_scale;  // null: 1 / N
  const float* dloss;      // null: no gradient
  float* row_loss;         // null: no loss
  float4* stats;           // (m, L, ln p_rest, 0)
  int64_t N, ld, ld_grad;
  int V, top, rest;
  float inv_tau;
  int* status;
};

// The row's list in shared memory: token (-1: not in use), teacher's probability, its logarithm.
struct DistillList {
  int id[AG_DISTILL_MAX];
  float q[AG_DISTILL_MAX], log_q[AG_DISTILL_MAX], x[AG_DISTILL_MAX];
  float mass, left;  // Q and r
  int used;
};

// By all threads of the block; ends with a barrier.
__device__ void distill_list(DistillList& l, const DistillArgs& a, int64_t row) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    float m = -INFINITY;
    bool nan = false;
    for (int k = lane; k < a.top; k += 32) {
      int id = a.ids[row * a.top + k];
      if (id >= a.V) {
        atomicOr(a.status, AG_STATUS_BAD_INDEX);
        id = -1;
      }
      const float t = id < 0 ? -INFINITY : a.teacher[row * a.top + k];
      l.id[k] = id;
      l.log_q[k] = t;
      m = fmaxf(m, t);
      nan |= t != t;
    }
    m = ag_warp_max(m);
    nan = __any_sync(0xffffffffu, nan);
    const bool used = m > -INFINITY || nan;
    double mass = 0.0;
    float sum = 0.0f;
    for (int k = lane; k < a.top; k += 32) {
      float t = l.log_q[k];
      if (!a.rest) t = t == -INFINITY ? t : (t - m) * a.inv_tau;
      const float q = expf(t);
      l.log_q[k] = t;
      l.q[k] = q;
      sum += q;
      mass += q;
    }
    sum = ag_warp_sum(sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    if (!a.rest && used) {
      const float log_sum = logf(sum), inv = 1.0f / sum;
      for (int k = lane; k < a.top; k += 32) {
        l.log_q[k] -= log_sum;
        l.q[k] *= inv;
      }
    }
    if (lane == 0) {
      l.used = used;
      l.mass = !used ? 0.0f : a.rest ? (float)mass : sum != sum ? sum : 1.0f;
      l.left = a.rest && used ? (float)(1.0 - mass > 0.0 ? 1.0 - mass : mass != mass ? mass : 0.0) : 0.0f;
    }
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(DI_THREADS)
distill_kernel(const T* logits, const T* dres, T* dlogits, DistillArgs a, int have_stats) {
  extern __shared__ uint32_t s_listed[];  // a bit per token
  __shared__ DistillList l;
  __shared__ AgStat s_stat[DI_WARPS];
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t row = blockIdx.x;
  const T* x = logits + row * a.ld;
  const float c = a.inv_tau * AG_LOG2E;
  for (int j = threadIdx.x; j < (a.V + 31) / 32; j += DI_THREADS) s_listed[j] = 0;
  distill_list(l, a, row);
  for (int k = threadIdx.x; k < a.top; k += DI_THREADS)
    if (l.id[k] >= 0) {
      atomicOr(&s_listed[l.id[k] >> 5], 1u << (l.id[k] & 31));
      l.x[k] = Pack<T>::load1(x + l.id[k]);
    }
  __syncthreads();
  float m, L, log_rest;
  if (have_stats) {
    const float4 st = a.stats[row];
    m = st.x, L = st.y, log_rest = st.z;
  } else {
    AgStat in = ag_stat_none(), out = ag_stat_none();
    for (int j = threadIdx.x; j < a.V; j += DI_THREADS) {
      const float xj = Pack<T>::load1(x + j);
      const AgStat one = {xj, xj == -INFINITY ? 0.0f : xj - xj + 1.0f, 0.0f};
      if (s_listed[j >> 5] >> (j & 31) & 1) in = ag_stat_merge(in, one, c);
      else out = ag_stat_merge(out, one, c);
    }
    out = ag_stat_warp(out, c);
    in = ag_stat_warp(in, c);
    if ((threadIdx.x & 31) == 0) s_stat[threadIdx.x >> 5] = out;
    __syncthreads();
    out = s_stat[0];
    for (int w = 1; w < DI_WARPS; ++w) out = ag_stat_merge(out, s_stat[w], c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_stat[threadIdx.x >> 5] = in;
    __syncthreads();
    in = s_stat[0];
    for (int w = 1; w < DI_WARPS; ++w) in = ag_stat_merge(in, s_stat[w], c);
    const AgStat all = ag_stat_merge(in, out, c);
    m = all.m;
    L = logf(all.s);
    log_rest = out.m == -INFINITY && out.s == 0.0f ? -INFINITY : (out.m - m) * a.inv_tau + logf(out.s) - L;
    if (threadIdx.x == 0 && a.stats) a.stats[row] = make_float4(m, L, a.rest ? log_rest : 0.0f, 0.0f);
  }
  auto log_p = [&](float xj) { return xj == -INFINITY && !(L != L) ? -INFINITY : (xj - m) * a.inv_tau - L; };
  if (a.row_loss && threadIdx.x < 32) {
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.top; k += 32)
      if (l.id[k] >= 0 && l.q[k] != 0.0f) sum += l.q[k] * (l.log_q[k] - log_p(l.x[k]));
    sum = ag_warp_sum(sum);
    if (l.left != 0.0f) sum += l.left * (logf(l.left) - log_rest);
    if (threadIdx.x == 0) a.row_loss[row] = l.used ? sum : 0.0f;
  }
  if (!a.dloss) return;
  const float w = a.row_scale ? a.row_scale[row] : 1.0f / (float)a.N;
  const float s = w == 0.0f ? 0.0f : a.dloss[0] * w * a.inv_tau;
  const bool none = s == 0.0f || !l.used || (m == -INFINITY && L == -INFINITY);
  const float r = l.left;
  const float outside = l.mass + r - (r != 0.0f && log_rest > -INFINITY ? r * expf(-log_rest) : 0.0f), inside = l.mass + r;
  for (int j = threadIdx.x; j < a.V; j += DI_THREADS) {
    const bool listed = s_listed[j >> 5] >> (j & 31) & 1;
    float g = 0.0f;
    if (!none) {
      const float p = ag_ex2(((Pack<T>::load1(x + j) - m) * a.inv_tau - L) * AG_LOG2E);
      g = p * (listed ? inside : outside);
      if (listed)
        for (int k = 0; k < a.top; ++k)
          if (l.id[k] == j) g -= l.q[k];
      g *= s;
    }
    if (dres) g += Pack<T>::load1(dres + row * a.ld_grad + j);
    Pack<T>::store1(dlogits + row * a.ld_grad + j, g);
  }
}

// loss = sum of the weighted rows, in an order that N fixes; a row of weight 0 takes no part, whatever its loss.
__global__ void __launch_bounds__(1024)
distill_loss_kernel(const float* __restrict__ row_loss, const float* __restrict__ row_scale, int64_t N, float* loss) {
  __shared__ double s_sum[32];
  ag_pdl_wait();
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < N; i += 1024) {
    const float w = row_scale ? row_scale[i] : 1.0f;
    if (w != 0.0f) sum += (double)w * row_loss[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x < 32) {
    sum = s_sum[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) loss[0] = (float)(row_scale || N == 0 ? sum : sum / (double)N);
  }
}

template <typename T>
int distill_t(ag_ctx* ctx, const void* logits, const void* dres, void* dlogits, const DistillArgs& a, int have_stats) {
  const size_t smem = (size_t)(a.V + 31) / 32 * 4;
  static bool ready[AG_MAX_DEVICES];
  if (!ready[ag_dev_slot(ctx)]) {
    AG_CUDA(ctx, cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (AG_VOCAB_MAX + 31) / 32 * 4));
    ready[ag_dev_slot(ctx)] = true;
  }
  AG_LAUNCH_PDL(ctx, "distill_kernel", distill_kernel<T>, (unsigned)a.N, DI_THREADS, smem, (const T*)logits, (const T*)dres, (T*)dlogits,
                a, have_stats);
  return AG_OK;
}

int distill(ag_ctx* ctx, const char* who, const void* logits, int64_t ld, const int32_t* ids, const float* teacher,
            const float* row_scale, const float* dloss, float* loss, float* row_loss, float* stats, const void* dres, void* dlogits,
            int64_t ld_grad, int64_t N, int V, int top, float temperature, int mode, int dtype, bool backward) {
  if (int rc = ag_vocab_check(ctx, who, {N, ld, ld_grad, V, top, dtype, temperature}, AG_VOCAB_MAX, AG_DISTILL_MAX, logits, dres, dlogits))
    return rc;
  AG_REQUIRE(ctx, mode == AG_DISTILL_RENORM || mode == AG_DISTILL_REST, "%s: unknown mode %d", who, mode);
  AG_REQUIRE(ctx, top > 0, "%s: a list of no tokens", who);
  AG_REQUIRE(ctx, (ids && teacher && (backward ? stats : row_loss) && (dloss || ld_grad < 0)) || N == 0, "%s: null pointer", who);
  AG_REQUIRE(ctx, ag_aligned16(stats), "%s: stats not 16-byte aligned", who);
  if (N == 0 && !loss) return AG_OK;
  AgOnDevice on(ctx);
  const DistillArgs a = {ids, teacher, row_scale, dloss, row_loss, (float4*)stats, N, ld, ld_grad, V, top, mode == AG_DISTILL_REST,
                         1.0f / temperature, ctx->d_status};
  if (int rc = N == 0 ? AG_OK
               : dtype == AG_F32 ? distill_t<float>(ctx, logits, dres, dlogits, a, backward)
                                 : distill_t<__nv_bfloat16>(ctx, logits, dres, dlogits, a, backward))
    return rc;
  if (loss)
    AG_LAUNCH_PDL(ctx, "distill_loss_kernel", distill_loss_kernel, 1, 1024, 0, (const float*)row_loss, row_scale, N, loss);
  return AG_OK;
}

}  // namespace

extern "C" int ag_distill_forward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* teacher_ids, const float* teacher_logits,
                                  const float* row_scale, float* loss, float* row_loss, float* stats, int64_t N, int V, int top,
                                  float temperature, int mode, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  return distill(ctx, "ag_distill_forward", logits, ld, teacher_ids, teacher_logits, row_scale, nullptr, loss, row_loss, stats, nullptr,
                 nullptr, -1, N, V, top, temperature, mode, dtype, false);
}

extern "C" int ag_distill_backward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* teacher_ids, const float* teacher_logits,
                                   const float* row_scale, const float* stats, const float* dloss, const void* dres, void* dlogits,
                                   int64_t ld_grad, int64_t N, int V, int top, float temperature, int mode, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  AG_REQUIRE(ctx, ld_grad >= 0, "ag_distill_backward: negative gradient row stride");
  return distill(ctx, "ag_distill_backward", logits, ld, teacher_ids, teacher_logits, row_scale, dloss, nullptr, nullptr,
                 const_cast<float*>(stats), dres, dlogits, ld_grad, N, V, top, temperature, mode, dtype, true);
}

extern "C" int ag_distill_forward_backward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* teacher_ids,
                                           const float* teacher_logits, const float* row_scale, const float* dloss, float* loss,
                                           float* row_loss, float* stats, void* dlogits, int64_t ld_grad, int64_t N, int V, int top,
                                           float temperature, int mode, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  AG_REQUIRE(ctx, ld_grad >= 0, "ag_distill_forward_backward: negative gradient row stride");
  return distill(ctx, "ag_distill_forward_backward", logits, ld, teacher_ids, teacher_logits, row_scale, dloss, loss, row_loss, stats,
                 nullptr, dlogits, ld_grad, N, V, top, temperature, mode, dtype, false);
}
