// Shared by the operators on rows of logits (ag_logprobs.cu, ag_distill.cu): argument checks, softmax statistics that can be
// merged, rows in 16-byte packets, what the blocks of a row tell one another.
#pragma once

#include <math.h>

#include <atomic>

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

// Pointers to 32-bit numbers, or null
template <typename... P>
static inline bool ag_aligned4(const P*... p) {
  return ((((uintptr_t)p & 3) == 0) && ...);
}

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
  AG_REQUIRE(ctx, s.top >= 0 && s.top <= max_top, "%s: %d tokens per row, up to %d", who, s.top, max_top);
  // strides below 2^31: the products below stay below 2^64
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
__device__ __forceinline__ float ag_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float ag_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// Statistics of a part of a row: m its largest logit, s = sum 2^(c y), t = sum 2^(c y) y with y = x - m, c = log2(e) / temperature.
// The difference is formed before the product: x c - m c in one fma would be off by the rounding of m c, which differs between the
// parts of a row, and overflows for rows of the lowest numbers.  Terms whose power is 0 add nothing to t, however far y is.
// m = -inf: nothing above -inf, s = t = 0.  A NaN or +inf among the logits makes s NaN.
struct AgStat {
  float m, s, t;
};
__device__ __forceinline__ AgStat ag_stat_none() { return {-INFINITY, 0.0f, 0.0f}; }
// v as part of something with the largest logit m >= v.m
__device__ __forceinline__ void ag_stat_scale(AgStat& v, float m, float c) {
  const float y = m == -INFINITY ? 0.0f : v.m - m, e = ag_ex2(y * c);
  v.t = e > 0.0f ? e * (v.t + v.s * y) : 0.0f;
  v.s *= e;  // a NaN stays
  v.m = m;
}
__device__ __forceinline__ AgStat ag_stat_merge(AgStat a, AgStat b, float c) {
  const float m = fmaxf(a.m, b.m);
  ag_stat_scale(a, m, c);
  ag_stat_scale(b, m, c);
  return {m, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ AgStat ag_stat_warp(AgStat v, float c) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v.m));
  ag_stat_scale(v, m, c);
  uint64_t st = ag_pair(v.s, v.t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) st = ag_add2(st, __shfl_xor_sync(0xffffffffu, st, o));
  ag_unpair(st, v.s, v.t);
  return v;
}

// What 16 bytes of a row hold: 4 fp32 or 8 bf16.
template <typename T>
constexpr int AG_PACKET = 16 / (int)sizeof(T);
__device__ __forceinline__ void ag_widen(const uint4& w, float (&x)[4]) { Pack<float>::unpack_raw(*reinterpret_cast<const float4*>(&w), x); }
__device__ __forceinline__ void ag_widen(const uint4& w, float (&x)[8]) { Pack<__nv_bfloat16>::unpack(w, x); }

// The largest logit of packets as they lie in memory (NaN ignored).
template <int U>
__device__ __forceinline__ float ag_largest(const uint4 (&w)[U], float) {
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m = ag_max3(m, __uint_as_float(w[u].x), __uint_as_float(w[u].y));
    m = ag_max3(m, __uint_as_float(w[u].z), __uint_as_float(w[u].w));
  }
  return m;
}
__device__ __forceinline__ uint32_t ag_max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
template <int U>
__device__ __forceinline__ float ag_largest(const uint4 (&w)[U], __nv_bfloat16) {
  uint32_t m = 0xff80ff80u;
#pragma unroll
  for (int u = 0; u < U; ++u) m = ag_max_bf16x2(m, ag_max_bf16x2(ag_max_bf16x2(w[u].x, w[u].y), ag_max_bf16x2(w[u].z, w[u].w)));
  return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}

// U packets, the largest of which is `most`, onto v; t only if it is wanted.  A batch costs one more exponential, for what is there
// already.
template <bool WITH_T, typename T, int U>
__device__ __forceinline__ void ag_stat_add(AgStat& v, const uint4 (&w)[U], float most, float c) {
  constexpr int NV = AG_PACKET<T>;
  const float m = fmaxf(v.m, most);
  ag_stat_scale(v, m, c);
  const float ref = m == -INFINITY ? 0.0f : -m;
  const uint64_t ref2 = ag_pair(ref, ref), c2 = ag_pair(c, c);
  uint64_t s2 = ag_pair(v.s, 0.0f), t2 = ag_pair(v.t, 0.0f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float x[NV];
    ag_widen(w[u], x);
#pragma unroll
    for (int i = 0; i < NV; i += 2) {
      const uint64_t y2 = ag_add2(ag_pair(x[i], x[i + 1]), ref2);
      float d0, d1, y0, y1;
      ag_unpair(ag_mul2(y2, c2), d0, d1);
      const uint64_t e2 = ag_pair(ag_ex2(d0), ag_ex2(d1));
      s2 = ag_add2(s2, e2);
      if (!WITH_T) continue;
      ag_unpair(y2, y0, y1);
      t2 = ag_fma2(e2, ag_pair(fmaxf(y0, -1e30f), fmaxf(y1, -1e30f)), t2);  // 0 times -inf
    }
  }
  float a, b;
  ag_unpair(s2, a, b);
  v.s = a + b;
  if (!WITH_T) return;
  ag_unpair(t2, a, b);
  v.t = a + b;
}

// A packet of a gradient, whose rows may lie otherwise than the logits' with respect to 16 bytes
template <typename T>
__device__ __forceinline__ void ag_store_packet(T* to, const float (&g)[AG_PACKET<T>], bool whole) {
  if (whole) {
    Pack<T>::store_stream(to, g);
  } else {
#pragma unroll
    for (int e = 0; e < AG_PACKET<T>; ++e) Pack<T>::store1(to + e, g[e]);
  }
}

template <typename T>
__device__ __forceinline__ void ag_load_packet(const T* from, float (&d)[AG_PACKET<T>], bool whole) {
  if (whole) {
    Pack<T>::load_stream(from, d);
  } else {
#pragma unroll
    for (int e = 0; e < AG_PACKET<T>; ++e) d[e] = Pack<T>::load1(from + e);
  }
}

// A row as its cluster sees it: `head` elements before the first 16-byte boundary, `body` packets, `tail` elements behind them.
// Block `rank` has the packets from rank * per; head and tail are the first block's, an element per thread (0.., 16..).
template <typename T>
struct AgRow {
  const T* x;
  int head, body, tail;
  __device__ __forceinline__ AgRow(const T* row, int V) : x(row) {
    constexpr int NV = AG_PACKET<T>;
    const int past = (int)((uintptr_t)row & 15) / (int)sizeof(T);
    head = past ? min(NV - past, V) : 0;
    body = (V - head) / NV;
    tail = V - head - body * NV;
  }
  __device__ __forceinline__ int mine(int rank, int per) const { return max(0, min(body - rank * per, per)); }
  // index of this thread's own element of the edges, -1 without one
  __device__ __forceinline__ int edge(int rank) const {
    const int t = threadIdx.x;
    return rank ? -1 : t < head ? t : t >= 16 && t < 16 + tail ? head + body * AG_PACKET<T> + t - 16 : -1;
  }
  __device__ __forceinline__ int owner(int id, int per) const {
    const int q = id - head;
    return q < 0 || q >= body * AG_PACKET<T> ? 0 : q / AG_PACKET<T> / per;
  }
};

// Statistics of this thread's part of n packets, U at a time, and of its element of the edges (-inf without one).  `most` (null: not
// wanted): the largest logit of each batch, and of each packet that is left behind the last whole batch, this thread's
// TH (the threads of the block) apart, the first one that far behind `most`.
template <bool WITH_T, typename T, int U, int TH, bool AHEAD = true>
__device__ __forceinline__ AgStat ag_part_stat(const uint4* at, int n, float edge, float c, float* most = nullptr) {
  AgStat v = {edge == edge ? edge : -INFINITY, edge == -INFINITY ? 0.0f : edge - edge + 1.0f, 0.0f};  // NaN and inf - inf: a NaN for the sum
  const uint4* p = at + threadIdx.x;
  int left = n - (int)threadIdx.x;
  for (; left > (U - 1) * TH; left -= U * TH, p += U * TH) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = p[u * TH];
    const float m = ag_largest(w, T());
    if (most) *(most += TH) = m;
    ag_stat_add<WITH_T, T>(v, w, m, c);
  }
  // what is left of a batch: all loads under way before the first is used, where there are registers for it (AHEAD)
  constexpr int R = AHEAD ? 4 : 1;
  for (; left > 0; left -= R * TH, p += R * TH) {
    uint4 w[R][1];
#pragma unroll
    for (int u = 0; u < R; ++u)
      if (left > u * TH) w[u][0] = p[u * TH];
#pragma unroll
    for (int u = 0; u < R; ++u)
      if (left > u * TH) {
        const float m = ag_largest(w[u], T());
        if (most) *(most += TH) = m;
        ag_stat_add<WITH_T, T>(v, w[u], m, c);
      }
  }
  return v;
}

// ---- clusters --------------------------------------------------------------------------
__device__ __forceinline__ int ag_cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Every thread of every block of the cluster.
__device__ __forceinline__ void ag_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// What the lanes of this warp have read and written comes before what any of them sends afterwards.
__device__ __forceinline__ void ag_cluster_fence() {
  __syncwarp();
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// address in block `rank` of what lies at p in this one
__device__ __forceinline__ uint32_t ag_peer(const void* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ag_smem_u32(p)), "r"(rank));
  return a;
}
// Stores to a block of the cluster that count themselves at a barrier of that block when they are there: no thread waits for them,
// and there is no fence, which a barrier of the whole cluster would have (a sixth of the stalls of 4 blocks per row of 32768 fp32).
__device__ __forceinline__ void ag_send(uint32_t to, float4 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool ag_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(ag_smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void ag_wait_cluster(uint64_t* bar, uint32_t parity, int* status) {
  for (uint32_t i = 0; i < 1u << 20; ++i) {
    if (ag_try_wait_cluster(bar, parity)) return;
    if (i > 64) __nanosleep(32);
  }
  atomicOr(status, AG_STATUS_WAIT_EXPIRED);
}

// What each warp of a cluster tells the others about its part of a row, once: one float4 per warp.  S = 1: a block by itself.
template <int TH>
struct AgExchange {
  float4* box;    // [S * warps of a block]
  uint64_t* bar;
  int S, rank;
  int* status;
  __device__ __forceinline__ void start() const {
    if (S == 1) return;
    if (threadIdx.x == 0) {
      ag_mbar_init(bar, 1);
      ag_fence_mbar_init();
    }
    ag_cluster_sync();  // all of them run, with barriers set up, before one sends
  }
  // To block 0 only, or to all; by whole warps, every lane with the same v.  The box is returned, in which all entries are then; null
  // where nothing was sent to, which has no more to do here.
  template <bool ALL>
  __device__ __forceinline__ const float4* tell(float4 v) const {
    const int lane = threadIdx.x & 31;
    float4* to = box + rank * (TH / 32) + (threadIdx.x >> 5);
    if (S == 1) {
      if (lane == 0) *to = v;
      __syncthreads();
      return box;
    }
    if (lane < (ALL ? S : 1)) ag_send(ag_peer(to, lane), v, ag_peer(bar, lane));
    if (!ALL && rank) return nullptr;
    if (threadIdx.x == 0) ag_mbar_expect_tx(bar, S * (TH / 32) * 16);
    ag_wait_cluster(bar, 0, status);
    return box;
  }
};
// Where the launch counts what a block's pointers into shared memory span: aligned as the real ones are.
static inline float4* ag_counted_shared() { return reinterpret_cast<float4*>((uintptr_t)1 << 20); }
template <typename T>
static inline size_t ag_counted_bytes(const T* end) { return (size_t)((uintptr_t)end - ((uintptr_t)1 << 20)); }

__device__ __forceinline__ void ag_peer_store(uint32_t to, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
}
__device__ __forceinline__ void ag_peer_store(uint32_t to, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(v) : "memory");
}
// one arrival at a barrier of another block, after everything that this thread has seen done
__device__ __forceinline__ void ag_peer_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
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

// ---- launches ---------------------------------------------------------------------------
// Blocks per row of a kernel whose blocks need nothing of one another: one, unless that leaves SMs without work.
static inline int ag_row_parts(const ag_ctx* ctx, int64_t N, int packets) {
  int S = 1;
  while (N * S < 4 * ctx->sm_count && packets / S >= 1024) S *= 2;
  return S;
}

// Blocks of a cluster that share a row, where they have something to tell one another: more while the SMs have about one block each,
// and the blocks at least two packets per thread.  Us, by 1.0 / 1.4 / 2.8 blocks per SM up to which they are doubled: 200 rows of
// 32768 bf16, 20 alternatives 10.4 / 9.3 / 9.3; 64 rows 7.1 / 7.1 / 10.4; distillation loss of 200 rows fp32 9.6 / 9.0 / 9.0.
static inline int ag_cluster_parts(const ag_ctx* ctx, int64_t N, int packets) {
  int S = 1;
  while (S < 8 && N * S * 5 <= 7 * ctx->sm_count && packets / S >= 512) S *= 2;
  return S;
}

// Threads of a block with a row to itself: up to p64 packets 64, up to p128 128; not 64 for a few rows, which wait for their own loads.
static inline int ag_row_threads(const ag_ctx* ctx, int64_t N, int packets, int p64, int p128) {
  return packets > p128 ? 256 : packets > p64 || N < 4 * ctx->sm_count ? 128 : 64;
}

// Launch of n clusters of S blocks.
template <typename... P, typename... A>
static inline int ag_launch_clusters(ag_ctx* ctx, const char* name, void (*kern)(P...), int S, int threads, size_t smem, int64_t n,
                                     A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(n * S);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = ctx->pdl;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = S;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) AG_FAIL(ctx, AG_ERR_CUDA, "launch of %s failed: %s", name, cudaGetErrorString(e));
  ctx->launches++;
  ag_enqueued(ctx);
  return AG_OK;
}

