// Log-probabilities of given tokens, entropies and likeliest tokens of rows of logits, and their gradient.
//
//   z = x / temperature,  m = max x,  L = ln sum exp((x - m) / temperature),  log p_j = (x_j - m) / temperature - L
//   entropy H = L - sum_j p_j (x_j - m) / temperature
//   d logits_j = (a (delta_j,id - p_j) - b p_j (log p_j + H)) / temperature,  a = dlogprob (0 without a token), b = dentropy
//
// Forward: a block, or for few rows a cluster of 2 to 8, streams a row through registers.  The alternatives come from a second look
// at the row, which L2 still holds:
//   each warp tells, along with its statistics, its J-th largest lane maximum; the (top / J)-th largest of these is a bound that at
//   least `top` logits reach, and up to twice as many do, since the lanes' logits lie spread over the row;
//   the logits that reach it are collected, (order, index) as one key each, by the threads whose maximum does;
//   one block of the cluster counts for each how many are larger, which is its place.
// A block that collects more than `cap` (many equal logits, or the largest ones all in a few lanes) searches a bound of its own,
// bit by bit, and takes logits that equal it in the order of their index.
#include "ag_vocab.cuh"

namespace {

constexpr int LP_THREADS = AG_ROW_THREADS, LP_WARPS = LP_THREADS / 32;
static_assert(3 * AG_TOP_MAX + 64 + 1 <= 2 * LP_THREADS, "two keys per thread are moved");

struct LpArgs {
  const int32_t* ids;
  float *logprob, *entropy;
  float4* stats;
  int32_t* top_ids;
  float* top_logprobs;
  int64_t N, ld;
  int V, top;
  float inv_tau;
  int S, per;  // blocks per row, packets per block
  int J, need, cap;  // which lane maximum of a warp, how many of these the bound has to meet, keys per block
  int* status;
};

constexpr int LP_BATCH = 4;  // packets
// whole batches of a thread before which (and at which) `left` packets of the block lie, and packets behind them
__host__ __device__ constexpr int lp_whole(int left) {
  return left > (LP_BATCH - 1) * LP_THREADS ? (left - (LP_BATCH - 1) * LP_THREADS - 1) / (LP_BATCH * LP_THREADS) + 1 : 0;
}
__host__ __device__ constexpr int lp_rest(int left) {
  return left > lp_whole(left) * LP_BATCH * LP_THREADS ? (left - lp_whole(left) * LP_BATCH * LP_THREADS - 1) / LP_THREADS + 1 : 0;
}

// the exchange, a barrier, a block's keys, those of all blocks at block 0, batches with a logit that passes, counters, the batches'
// largest logits
size_t lp_smem(int S, int cap, int per) {
  return AgExchange::bytes(S) + 16 + (size_t)cap * (8 * (S == 1 ? 1 : 1 + S) + 8) + 48 +
         (cap ? (size_t)(lp_whole(per) + LP_BATCH - 1) * LP_THREADS * 4 : 0);
}

__device__ __forceinline__ unsigned long long lp_key(float x, int index) { return (unsigned long long)ag_order(x) << 32 | (uint32_t)~index; }

// The need-th largest of the n <= 64 numbers box[].w, or one that an eighth more of them reach; by one warp.
__device__ __forceinline__ float lp_bound(const float4* box, int n, int need) {
  const int lane = threadIdx.x & 31;
  if (n <= 16) {  // a lane each, which counts the larger ones: the bisection takes some 20 steps
    const float mine = lane < n ? box[lane].w : -INFINITY;
    int place = 0;
    for (int g = 0; g < n; ++g) {
      const float w = box[g].w;
      place += w > mine || (w == mine && g < lane);
    }
    return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, lane < n && place == need - 1)) - 1);
  }
  const bool one = lane < n, two = lane + 32 < n;
  const uint32_t a = one ? ag_order(box[lane].w) : 0u, b = two ? ag_order(box[lane + 32].w) : 0u;
  uint32_t lo = __reduce_min_sync(0xffffffffu, min(one ? a : 0xffffffffu, two ? b : 0xffffffffu));
  uint32_t hi = __reduce_max_sync(0xffffffffu, max(a, b));
  const int enough = need + max(1, need >> 3);
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const int count = __popc(__ballot_sync(0xffffffffu, a >= mid)) + __popc(__ballot_sync(0xffffffffu, b >= mid));
    if (count >= need) {
      lo = mid;
      if (count <= enough) break;
    } else {
      hi = mid - 1;
    }
  }
  return ag_of_order(lo);
}

template <typename T>
struct LpPart {
  const uint4* at;
  int n, first;  // packets, index of the first one's first logit
  float edge;
  int edge_index;  // -1: none
  // f(logit, its index) for this thread's logits
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int NV = AG_PACKET<T>;
    if (edge_index >= 0) f(edge, edge_index);
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
      float x[NV];
      ag_widen(at[i], x);
#pragma unroll
      for (int e = 0; e < NV; ++e) f(x[e], first + i * NV + e);
    }
  }
};

// The block's logits whose order is `bound` or more are more than `cap`: leaves the keys of its `top` largest at least, `cap` at
// most, in `keys` and returns how many.  By all threads of the block.  A block that has this many has more than `top` logits.
template <typename T>
__device__ __noinline__ int lp_search(const LpPart<T>& sl, uint32_t lo, int top, int cap, unsigned long long* keys, int* s_count) {
  uint32_t hi = 0xffffffffu;
  auto count_from = [&](uint32_t k) {
    int c = 0;
    sl.each([&](float x, int) { c += ag_order(x) >= k; });
    c = __reduce_add_sync(0xffffffffu, c);
    if (threadIdx.x == 0) *s_count = 0;
    __syncthreads();
    if ((threadIdx.x & 31) == 0 && c) atomicAdd(s_count, c);
    __syncthreads();
    c = *s_count;
    __syncthreads();
    return c;
  };
  bool fits = false;
  while (lo < hi && !fits) {
    const uint32_t mid = lo + (hi - lo) / 2 + 1;
    const int c = count_from(mid);
    if (c >= top) lo = mid, fits = c <= cap;
    else hi = mid - 1;
  }
  // fits: all that reach lo.  Otherwise lo is the top-th largest itself: all above it (fewer than top), and then equal ones.
  if (threadIdx.x == 0) *s_count = 0;
  __syncthreads();
  sl.each([&](float x, int j) {
    const uint32_t k = ag_order(x);
    if (k > lo || (fits && k == lo)) keys[atomicAdd(s_count, 1)] = lp_key(x, j);
  });
  __syncthreads();
  int have = *s_count;
  if (fits) return have;
  // in the order of the index: the elements before the first packet, then packets by rounds of the block, then those behind
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ int s_warp[LP_WARPS];
  constexpr int NV = AG_PACKET<T>;
  const int rounds = (sl.n + LP_THREADS - 1) / LP_THREADS;
  for (int r = -1; r <= rounds && have < top; ++r) {
    float x[NV];
    int mine = 0, first = 0;
    const int i = r * LP_THREADS + threadIdx.x;
    if (r < 0 || r == rounds) {
      const bool head = sl.edge_index >= 0 && threadIdx.x < 16;
      mine = sl.edge_index >= 0 && head == (r < 0) && ag_order(sl.edge) == lo;
    } else if (i < sl.n) {
      ag_widen(sl.at[i], x);
      first = sl.first + i * NV;
#pragma unroll
      for (int e = 0; e < NV; ++e) mine += ag_order(x[e]) == lo;
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) s_warp[warp] = before;
    __syncthreads();
    int at = have + before - mine, all = 0;
    for (int w = 0; w < LP_WARPS; ++w) {
      if (w < warp) at += s_warp[w];
      all += s_warp[w];
    }
    if (mine && at < top) {
      if (r < 0 || r == rounds) {
        keys[at] = lp_key(sl.edge, sl.edge_index);
      } else {
#pragma unroll
        for (int e = 0; e < NV; ++e)
          if (ag_order(x[e]) == lo && at < top) keys[at++] = lp_key(x[e], first + e);
      }
    }
    have = min(have + all, top);
    __syncthreads();
  }
  return have;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, 6)
logprobs_kernel(const T* __restrict__ logits, const LpArgs a) {
  extern __shared__ float4 s_box[];
  const int S = a.S, tid = threadIdx.x, lane = tid & 31, rank = S > 1 ? ag_cluster_rank() : 0;
  const int groups = S * LP_WARPS;
  uint64_t* s_bars = reinterpret_cast<uint64_t*>(s_box + 2 * groups);
  const AgExchange exchange = {s_box, s_bars, S, rank, a.status};
  uint64_t* s_keys_bar = s_bars + 2;                                                   // every block's keys are at block 0
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(s_keys_bar + 2);    // [cap], cap even
  unsigned long long* all = S == 1 ? keys : keys + a.cap;                              // [S * cap], of block 0
  int* batches = reinterpret_cast<int*>(keys + (S == 1 ? 1 : 1 + S) * a.cap);          // [cap]
  float* list_most = reinterpret_cast<float*>(batches + a.cap);                        // [cap]
  int* counts = reinterpret_cast<int*>(list_most + a.cap);                             // [8]
  int* n_keys = counts + 8;                                                            // keys, batches, a counter, a bound
  uint32_t* s_bound = reinterpret_cast<uint32_t*>(n_keys + 3);
  float* most = reinterpret_cast<float*>(n_keys + 4);                                  // [batches and packets of a thread][threads]
  const float c = a.inv_tau * AG_LOG2E;
  if (TOP && tid == 0) {
    n_keys[0] = n_keys[1] = n_keys[3] = 0;
    ag_mbar_init(s_keys_bar, S);
    ag_fence_mbar_init();
  }
  exchange.start();
  ag_pdl_wait();
  ag_pdl_trigger();

  const int64_t row = blockIdx.x / S;
  const AgRow<T> r(logits + row * a.ld, a.V);
  const int edge_index = r.edge(rank);
  const float edge = edge_index >= 0 ? Pack<T>::load1(r.x + edge_index) : -INFINITY;
  const int n = r.mine(rank, a.per), first = r.head + rank * a.per * AG_PACKET<T>;
  const uint4* at = reinterpret_cast<const uint4*>(r.x + first);
  const int id = tid == 0 && rank == 0 && a.logprob ? a.ids[row] : -1;
  const AgStat own = ag_part_stat<true, T, LP_BATCH>(at, n, edge, c, TOP ? most + tid - LP_THREADS : nullptr);
  const bool has = id >= 0 && id < a.V;
  const float x_id = has ? Pack<T>::load1(r.x + id) : 0.0f;  // not before: the warp's packets would wait for the id
  AgStat v = ag_stat_warp(own, c);
  float reached = v.m;
  if (TOP) {
    float left = own.m;
    for (int j = 1; j < a.J; ++j) {
      const uint32_t who = __ballot_sync(0xffffffffu, left == reached);
      if (lane == __ffs(who) - 1) left = -INFINITY;
      asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(reached) : "f"(left));
    }
  }
  const float4 word = make_float4(v.m, v.s, v.t, reached);
  const float4* told = TOP ? exchange.tell(0, word) : exchange.tell_first(word);
  if (!TOP && (rank || tid >= 32)) return;
  v = lane < groups ? AgStat{told[lane].x, told[lane].y, told[lane].z} : ag_stat_none();
  if (lane + 32 < groups) v = ag_stat_merge(v, {told[lane + 32].x, told[lane + 32].y, told[lane + 32].z}, c);
  v = ag_stat_warp(v, c);
  const float L = logf(v.s);
  auto log_p = [&](float x) { return x == -INFINITY && !(L != L) ? -INFINITY : (x - v.m) * a.inv_tau - L; };
  if (rank == 0 && tid == 0) {
    const float H = v.m == -INFINITY && v.s == 0.0f ? 0.0f : L - v.t / v.s * a.inv_tau;
    if (a.logprob) a.logprob[row] = has ? log_p(x_id) : 0.0f;
    if (a.entropy) a.entropy[row] = H;
    if (a.stats) a.stats[row] = make_float4(v.m, L, H, 0.0f);
  }
  if (!TOP) return;
  float bound = lp_bound(told, groups, a.need);
  const bool nan = L != L;  // NaN may lie in any batch, whatever its largest number is
  const LpPart<T> part = {at, n, first, edge, edge_index};
  // Batches with something in them go on a list, whose packets all threads then fetch from L2 and take apart.
  if (own.m >= bound || own.s != own.s) {
    const int entries = lp_whole(n - tid) + lp_rest(n - tid);
    for (int b = 0; b < entries; ++b) {
      const float m = most[b * LP_THREADS + tid];
      if (m < bound && own.s == own.s) continue;
      const int k = atomicAdd(n_keys + 1, 1);
      if (k < a.cap) batches[k] = b * LP_THREADS + tid, list_most[k] = m;
    }
  }
  __syncthreads();
  const int listed = min(n_keys[1], a.cap);
  // With `top` batches and more, the top-th largest of their maxima is a bound that hardly more than `top` logits reach; what it
  // leaves out need not be fetched, or counted against all others.
  if (listed > a.top && !nan) {
    for (int k = tid; k < listed; k += LP_THREADS) {
      const float m = list_most[k];
      int place = 0;
#pragma unroll 4
      for (int g = 0; g < listed; ++g) place += list_most[g] > m;
      if (place < a.top) atomicMax(s_bound, ag_order(m) ^ 0xffffffffu);
    }
    __syncthreads();
    bound = fmaxf(bound, ag_of_order(*s_bound ^ 0xffffffffu));
  }
  if (edge_index >= 0 && !(edge < bound)) keys[atomicAdd(n_keys, 1)] = lp_key(edge, edge_index);
  for (int k = tid; k < listed * LP_BATCH; k += LP_THREADS) {
    if (list_most[k / LP_BATCH] < bound && !nan) continue;
    const int b = batches[k / LP_BATCH] / LP_THREADS, of = batches[k / LP_BATCH] % LP_THREADS, whole = lp_whole(n - of);
    if (b >= whole && k % LP_BATCH) continue;  // a packet by itself
    const int i = (b < whole ? b * LP_BATCH + k % LP_BATCH : whole * LP_BATCH + b - whole) * LP_THREADS + of;
    float x[AG_PACKET<T>];
    ag_widen(at[i], x);
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < AG_PACKET<T>; ++e) hits |= x[e] < bound ? 0u : 1u << e;
    for (; hits; hits &= hits - 1) {
      const int index = first + i * AG_PACKET<T> + __ffs(hits) - 1, to = atomicAdd(n_keys, 1);
      if (to < a.cap) keys[to] = lp_key(Pack<T>::load1(r.x + index), index);
    }
  }
  __syncthreads();
  int total = n_keys[0];
  if (total > a.cap || n_keys[1] > a.cap) total = lp_search<T>(part, ag_order(bound), a.top, a.cap, keys, n_keys + 2);
  if (S > 1) {
    // to block 0, each to its own place there
    const uint32_t to = ag_peer(all + (size_t)rank * a.cap, 0);
    for (int k = tid; k < total; k += LP_THREADS) ag_peer_store(to + k * 8, keys[k]);
    if (tid == 0) ag_peer_store(ag_peer(counts + rank, 0), total);
    __syncthreads();
    if (tid == 0) ag_peer_arrive(ag_peer(s_keys_bar, 0));
    if (rank) return;
    ag_wait_cluster(s_keys_bar, 0, a.status);
    // side by side
    total = counts[0];
    for (int p = 1; p < S; ++p) {
      const int more = counts[p];
      unsigned long long mine[2];  // cap <= 2 * LP_THREADS, and what is moved down may lie over what is not yet
      for (int k = 0; k < 2; ++k)
        if (tid + k * LP_THREADS < more) mine[k] = all[(size_t)p * a.cap + tid + k * LP_THREADS];
      __syncthreads();
      for (int k = 0; k < 2; ++k)
        if (tid + k * LP_THREADS < more) all[total + tid + k * LP_THREADS] = mine[k];
      total += more;
    }
    __syncthreads();
  }
  // a key's place is the number of larger ones; where there are threads for it, several count for each key
  auto put = [&](unsigned long long key, int place) {
    if (place >= a.top) return;
    const int64_t to = row * a.top + place;
    a.top_ids[to] = (int32_t)~(uint32_t)key;
    a.top_logprobs[to] = log_p(ag_of_order((uint32_t)(key >> 32)));
  };
  auto larger = [&](unsigned long long key, int from, int step) {  // pairs of keys from, from + step, ...; the last one may stand alone
    int place = 0;
#pragma unroll 4
    for (int k = 2 * from; k < total - 1; k += 2 * step) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(all + k);
      place += two.x > key;
      place += two.y > key;
    }
    return place + ((total & 1) && from == 0 && all[total - 1] > key);
  };
  __shared__ int s_place[LP_THREADS / 2];
  if (total <= LP_THREADS / 2) {
    const int lanes = (total + 31) & ~31, parts = LP_THREADS / lanes, i = tid % lanes;
    if (tid < lanes) s_place[i] = 0;
    __syncthreads();
    if (i < total && tid < parts * lanes) {
      const int place = larger(all[i], tid / lanes, parts);
      if (place) atomicAdd(&s_place[i], place);
    }
    __syncthreads();
    if (tid < total) put(all[tid], s_place[tid]);
  } else {
    for (int i = tid; i < total; i += LP_THREADS) put(all[i], larger(all[i], 0, 1));
  }
}

// Gradient: a block takes `per` packets of a row.
struct LbArgs {
  const int32_t* ids;
  const float4* stats;
  const float *dlogprob, *dentropy;
  int64_t ld, ld_grad;
  int V, S, per;
  float inv_tau;
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4)
logprobs_backward_kernel(const T* logits, const T* dres, T* dlogits, const LbArgs p) {
  constexpr int NV = AG_PACKET<T>, U = 4;
  const int tid = threadIdx.x;
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t row = blockIdx.x / p.S;
  const int rank = (int)(blockIdx.x - row * p.S);
  const AgRow<T> r(logits + row * p.ld, p.V);
  const int n = r.mine(rank, p.per), first = r.head + rank * p.per * NV;
  const uint4* at = reinterpret_cast<const uint4*>(r.x + first);
  const int edge_index = r.edge(rank);
  const float x_edge = edge_index >= 0 ? Pack<T>::load1(r.x + edge_index) : 0.0f;
  const float4 st = p.stats[row];
  const int id = p.ids ? p.ids[row] : -1;
  const float a = p.dlogprob && id >= 0 && id < p.V ? p.dlogprob[row] * p.inv_tau : 0.0f;
  const float b = p.dentropy ? p.dentropy[row] * p.inv_tau : 0.0f;
  const bool none = (a == 0.0f && b == 0.0f) || (st.x == -INFINITY && st.y == -INFINITY);
  T* g_row = dlogits + row * p.ld_grad;
  const T* d_row = dres ? dres + row * p.ld_grad : nullptr;
  const bool packets = (((uintptr_t)(g_row + first)) & 15) == 0, d_packets = (((uintptr_t)(d_row + first)) & 15) == 0;
  // p (a + b (ln p + H)) = p (a + b H + b ln p); a logit of -inf: p = 0, and 0 times something finite
  const float k = a + b * st.z;
  auto local = [&](float x) {
    const float lp = fmaxf((x - st.x) * p.inv_tau, -1e4f) - st.y;
    return -ag_ex2(lp * AG_LOG2E) * (k + b * lp);
  };
  auto put = [&](const uint4& w, int i) {
    float x[NV], g[NV];
    ag_widen(w, x);
#pragma unroll
    for (int e = 0; e < NV; ++e) g[e] = none ? 0.0f : local(x[e]);
    const int to = first + i * NV, hit = id - to;
    if (hit >= 0 && hit < NV && !none) {
#pragma unroll
      for (int e = 0; e < NV; ++e) g[e] += e == hit ? a : 0.0f;
    }
    if (d_row) {
      float d[NV];
      ag_load_packet<T>(d_row + to, d, d_packets);
#pragma unroll
      for (int e = 0; e < NV; ++e) g[e] += d[e];
    }
    ag_store_packet<T>(g_row + to, g, packets);
  };
  int i = tid;
  for (; i + (U - 1) * LP_THREADS < n; i += U * LP_THREADS) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldcs(at + i + u * LP_THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) put(w[u], i + u * LP_THREADS);
  }
  for (; i < n; i += LP_THREADS) put(__ldcs(at + i), i);
  if (edge_index >= 0) {
    const float g = none ? 0.0f : local(x_edge) + (edge_index == id ? a : 0.0f);
    Pack<T>::store1(g_row + edge_index, g + (d_row ? Pack<T>::load1(d_row + edge_index) : 0.0f));
  }
}

template <typename T>
int logprobs_backward(ag_ctx* ctx, const void* logits, const void* dres, void* dlogits, LbArgs p, int64_t N) {
  p.S = ag_row_parts(ctx, N, p.V / AG_PACKET<T>);
  p.per = (p.V / AG_PACKET<T> + p.S - 1) / p.S;
  AG_REQUIRE(ctx, N * p.S < (1ll << 31), "ag_token_logprobs_backward: too many rows for V=%d", p.V);
  AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", logprobs_backward_kernel<T>, (unsigned)(N * p.S), LP_THREADS, 0, (const T*)logits,
                (const T*)dres, (T*)dlogits, p);
  return AG_OK;
}

template <typename T, bool TOP>
int logprobs(ag_ctx* ctx, const void* logits, LpArgs a) {
  const int packets = (a.V + AG_PACKET<T> - 1) / AG_PACKET<T>;
  a.S = 1;
  while (a.S < 8 && a.N * a.S * 2 <= 2 * ctx->sm_count && packets / a.S >= 512) a.S *= 2;
  a.per = (packets + a.S - 1) / a.S;
  a.cap = TOP ? 3 * a.top + 64 + (a.top & 1) : 0;
  // Lane maxima: where nearly all warps have to meet the bound, the one with the smallest logits decides, and many more than
  // `top` pass.  33 of 32 warps: the smallest of the second ones is passed by 200, the 17th of them by 55.
  const int groups = a.S * LP_WARPS;
  a.J = (a.top + groups - 1) / groups;
  while (TOP && a.J < 32 && (a.top + a.J - 1) / a.J * 20 > groups * 17) ++a.J;
  a.need = TOP ? (a.top + a.J - 1) / a.J : 0;
  a.status = ctx->d_status;
  AG_REQUIRE(ctx, a.N * a.S < (1ll << 31), "ag_token_logprobs_forward: too many rows");
  const size_t smem = lp_smem(a.S, a.cap, a.per);
  if (smem > 47 * 1024) {
    static std::atomic<bool> ready[AG_MAX_DEVICES];
    if (!ready[ag_dev_slot(ctx)].load(std::memory_order_acquire)) {
      AG_CUDA(ctx, cudaFuncSetAttribute(logprobs_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
      ready[ag_dev_slot(ctx)].store(true, std::memory_order_release);
    }
  }
  return ag_launch_clusters(ctx, "logprobs_kernel", logprobs_kernel<T, TOP>, a.S, smem, a.N, (const T*)logits, a);
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
  const LpArgs a = {ids, logprob, entropy, (float4*)stats, top_ids, top_logprobs, N, ld, V, top, 1.0f / temperature, 0, 0, 0, 0, 0, nullptr};
  if (dtype == AG_F32)
    return top ? logprobs<float, true>(ctx, logits, a) : logprobs<float, false>(ctx, logits, a);
  return top ? logprobs<__nv_bfloat16, true>(ctx, logits, a) : logprobs<__nv_bfloat16, false>(ctx, logits, a);
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
  const LbArgs p = {ids, (const float4*)stats, dlogprob, dentropy, ld, ld_grad, V, 0, 0, 1.0f / temperature};
  return dtype == AG_F32 ? logprobs_backward<float>(ctx, logits, dres, dlogits, p, N)
                         : logprobs_backward<__nv_bfloat16>(ctx, logits, dres, dlogits, p, N);
}
