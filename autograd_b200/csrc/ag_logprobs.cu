// Log-probabilities of given tokens, entropies and likeliest tokens of rows of logits, and their gradient.
//
//   z = x / temperature,  m = max x,  L = ln sum exp((x - m) / temperature),  log p_j = (x_j - m) / temperature - L
//   entropy H = L - sum_j p_j (x_j - m) / temperature
//   d logits_j = (a (delta_j,id - p_j) - b p_j (log p_j + H)) / temperature,  a = dlogprob (0 without a token), b = dentropy
//
// Forward: a block, or for few rows a cluster of 2 to 8, streams a row through registers.  For the alternatives it notes the largest
// logit of every batch of packets that a thread reads at a time:
//   a block with a row to itself takes the top-th largest of these (or a little less: lp_threshold) as a bound, which `top` logits
//   at least reach, and hardly more do;
//   the blocks of a cluster, which would find a bound each, tell one another their warps' J-th largest lane maxima instead, and take
//   the (top / J)-th largest of these, which up to twice as many reach (8 rows of 151936 bf16, 20 alternatives: 10.4 / 7.7 us);
//   the batches that reach it, still in L2, are fetched again and their logits that do collected, (order, index) as one key each;
//   the first block of the cluster counts for each how many are larger, which is its place.
// A block that collects more than `cap` (many equal logits, many in one batch) searches a bound among the logits themselves, bit by
// bit, and takes those that equal it in the order of their index.
#include "ag_vocab.cuh"

namespace {

// Packets of a row up to which a block has 64 or 128 threads: without alternatives, with them, for the gradient.  16384 rows (of
// 32768: 8192), 64 / 128 / 256 threads, us: none 640 bf16 18 / 19 / 30, 5003 fp32 55 / 57 / 68, 32768 bf16 93 / 89 / 87; 20 alternatives
// 5003 bf16 69 / 86 / 156, 10007 fp32 144 / 148 / 203; 64 of 32768 bf16 - / 125 / 141, fp32 - / 206 / 197; gradient 640 fp32
// 24 / 27 / 40, 5003 bf16 67 / 68 / 108, 5003 fp32 116 / 111 / 121, 32768 bf16 193 / 182 / 178.
constexpr int LP_PACKETS_64 = 1300, LP_PACKETS_128 = 2560, LP_TOP_64 = 2500, LP_TOP_128 = 8191, LB_PACKETS_64 = 800, LB_PACKETS_128 = 2560;

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
template <int TH>
__host__ __device__ constexpr int lp_whole(int left) {
  return left > (LP_BATCH - 1) * TH ? (left - (LP_BATCH - 1) * TH - 1) / (LP_BATCH * TH) + 1 : 0;
}
template <int TH>
__host__ __device__ constexpr int lp_rest(int left) {
  return left > lp_whole<TH>(left) * LP_BATCH * TH ? (left - lp_whole<TH>(left) * LP_BATCH * TH - 1) / TH + 1 : 0;
}

// Keys that a block has room for.  A multiple of four: keys are read in pairs, the histogram behind them 16 bytes at a time.
constexpr int lp_cap(int top) { return top ? (3 * top + 64 + 3) & ~3 : 0; }

// Shared memory from the exchange's box on, for the kernel and for the launch that counts it.  All lengths before `most` are
// multiples of 16 bytes.
template <int TH>
struct LpShared {
  uint64_t* bars;            // [2] one of the exchange
  uint64_t* keys_bar;        // [2] every block's keys are at block 0
  unsigned long long* keys;  // [cap]
  unsigned long long* all;   // [S * cap], of block 0; a block with a row to itself has only those
  int* batches;              // [cap] with a logit that passes
  int* counts;               // [8]
  int* n_keys;               // [4] keys, batches, a counter
  uint32_t* hist;            // [256]
  float* most;               // [batches and packets of a thread][threads] their largest logits
  __host__ __device__ __forceinline__ LpShared(float4* box, int S, int cap) {
    bars = reinterpret_cast<uint64_t*>(box + S * (TH / 32));
    keys_bar = bars + 2;
    keys = reinterpret_cast<unsigned long long*>(keys_bar + 2);
    all = S == 1 ? keys : keys + cap;
    batches = reinterpret_cast<int*>(keys + (S == 1 ? 1 : 1 + S) * cap);
    counts = batches + cap;
    n_keys = counts + 8;
    hist = reinterpret_cast<uint32_t*>(n_keys + 4);
    most = reinterpret_cast<float*>(hist + 256);
  }
  static size_t bytes(int S, int cap, int per) {
    const LpShared at(ag_counted_shared(), S, cap);
    return ag_counted_bytes(cap ? reinterpret_cast<char*>(at.most + (lp_whole<TH>(per) + LP_BATCH - 1) * TH)
                                : reinterpret_cast<char*>(at.keys_bar));
  }
};
constexpr bool lp_lengths() {
  for (int top = 1; top <= AG_TOP_MAX; ++top)
    if (lp_cap(top) % 4 || lp_cap(top) < 3 * top + 64) return false;
  return true;
}
static_assert(lp_lengths(), "keys, batches and what lies behind them start at multiples of 16 bytes");

__device__ __forceinline__ unsigned long long lp_key(float x, int index) { return (unsigned long long)ag_order(x) << 32 | (uint32_t)~index; }

// An order that at least `need` of the block's values reach and, unless many are equal, `enough` at most; 0 if there are fewer than
// `need` from lo on.  each(f) calls f(order) for this thread's values; lo <= the need-th largest if it exists, hi >= all.  hist: 256
// zeros, which it does not leave.  A histogram of the range finds the 256th of it where the need-th lies, until that is narrow
// enough; from the smallest of the lanes' largest logits on the first one usually is.  By all threads of the block.
template <int TH, typename F>
__device__ __forceinline__ uint32_t lp_threshold(F each, uint32_t lo, uint32_t hi, int need, int enough, uint32_t* hist) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (;;) {
    const int shift = max(0, 24 - __clz(hi - lo));
    each([&](uint32_t k) {
      if (k >= lo && k <= hi) atomicAdd(hist + ((k - lo) >> shift), 1u);
    });
    __syncthreads();
    // every warp: bins 8 * lane .. 8 * lane + 7, and how many values lie in those of the lanes above
    uint32_t bin[8];
    *reinterpret_cast<uint4*>(bin) = *reinterpret_cast<const uint4*>(hist + 8 * lane);
    *reinterpret_cast<uint4*>(bin + 4) = *reinterpret_cast<const uint4*>(hist + 8 * lane + 4);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine += bin[i];
    int upto = mine;  // of this lane and those above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_down_sync(0xffffffffu, upto, o);
      if (lane + o < 32) upto += w;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, upto >= need);
    if (!who) return 0;  // too few values
    int above = upto - mine, at = 0, reach = 0;
    bool found = false;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      if (!found && above + (int)bin[i] >= need) found = true, at = 8 * lane + i, reach = above + bin[i];
      if (!found) above += bin[i];
    }
    const int from = 31 - __clz(who);  // the highest lane that gets there
    at = __shfl_sync(0xffffffffu, at, from);
    above = __shfl_sync(0xffffffffu, above, from);
    reach = __shfl_sync(0xffffffffu, reach, from);
    lo += (uint32_t)at << shift;
    if (reach <= enough || shift == 0) return lo;
    need -= above;
    enough -= above;
    hi = min(hi, lo + (1u << shift) - 1);
    __syncthreads();
    for (int b = tid; b < 256; b += TH) hist[b] = 0;
    __syncthreads();
  }
}

// The order of the need-th largest of the n <= 64 numbers box[].w, or of one that an eighth more of them reach; by one warp.
__device__ __forceinline__ uint32_t lp_bound(const float4* box, int n, int need) {
  const int lane = threadIdx.x & 31;
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
  return lo;
}

template <typename T, int TH>
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
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += TH) {
      float x[NV];
      ag_widen(at[i], x);
#pragma unroll
      for (int e = 0; e < NV; ++e) f(x[e], first + i * NV + e);
    }
  }
};

// The block's logits whose order is `bound` or more are more than `cap`: leaves the keys of its `top` largest at least, `cap` at
// most, in `keys` and returns how many.  By all threads of the block.  A block that has this many has more than `top` logits.
template <typename T, int TH>
__device__ __noinline__ int lp_search(const LpPart<T, TH>& sl, uint32_t lo, int top, int cap, unsigned long long* keys, int* s_count) {
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
  lo = max(lo, ag_order(-INFINITY));
  // first whether the logits that equal lo make up the number: rows where fewer than `top` tokens are allowed, and all others are
  // masked with one value
  for (bool first = true; lo < hi && !fits; first = false) {
    const uint32_t mid = first ? lo + 1 : lo + (hi - lo) / 2 + 1;
    const int c = count_from(mid);
    if (c >= top) lo = mid, fits = c <= cap;
    else hi = mid - 1;  // the first time lo itself
  }
  // fits: all that reach lo.  Otherwise lo is the top-th largest itself: all above it (fewer than top), and then equal ones.
  if (threadIdx.x == 0) *s_count = 0;
  __syncthreads();
  sl.each([&](float x, int j) {
    const uint32_t k = ag_order(x);
    if (k > lo || (fits && k == lo)) {
      const int to = atomicAdd(s_count, 1);
      if (to < cap) keys[to] = lp_key(x, j);  // always, unless the logits change under way
    }
  });
  __syncthreads();
  int have = min(*s_count, cap);
  if (fits) return have;
  // in the order of the index: the elements before the first packet, then packets by rounds of the block, then those behind
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ int s_warp[(TH / 32)];
  constexpr int NV = AG_PACKET<T>;
  const int rounds = (sl.n + TH - 1) / TH;
  for (int r = -1; r <= rounds && have < top; ++r) {
    float x[NV];
    int mine = 0, first = 0;
    const int i = r * TH + threadIdx.x;
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
    for (int w = 0; w < (TH / 32); ++w) {
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

// MANY: the blocks of a cluster may share a row.  Six blocks of 256 threads per SM (40 registers), with alternatives of fp32 five:
// 64 of 8192 x 32768, at 6 / 5 of 256 threads: bf16 170 / 176 us, fp32 237 / 223.
template <typename T, bool TOP, int TH, bool MANY>
__global__ void __launch_bounds__(TH, (TOP && sizeof(T) == 4 ? 5 : 6) * 256 / TH)
logprobs_kernel(const T* __restrict__ logits, const LpArgs a) {
  extern __shared__ float4 s_box[];
  const int S = MANY || !TOP ? a.S : 1, tid = threadIdx.x, lane = tid & 31, rank = S > 1 ? ag_cluster_rank() : 0;
  const int groups = S * (TH / 32);
  const LpShared<TH> s(s_box, S, a.cap);
  const AgExchange<TH> exchange = {s_box, s.bars, S, rank, a.status};
  uint64_t* s_keys_bar = s.keys_bar;
  unsigned long long *keys = s.keys, *all = s.all;
  int *batches = s.batches, *counts = s.counts, *n_keys = s.n_keys;
  uint32_t* hist = s.hist;
  float* most = s.most;
  const float c = a.inv_tau * AG_LOG2E;
  for (int b = tid; TOP && !MANY && b < 256; b += TH) hist[b] = 0;
  if (TOP && tid == 0) {
    n_keys[0] = n_keys[1] = 0;
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
  const AgStat own = ag_part_stat<true, T, LP_BATCH, TH>(at, n, edge, c, TOP ? most + tid - TH : nullptr);
  const bool has = id >= 0 && id < a.V;
  const float x_id = has ? Pack<T>::load1(r.x + id) : 0.0f;  // not before: the warp's packets would wait for the id
  AgStat v = ag_stat_warp(own, c);
  float reached = v.m;
  if (TOP && MANY) {  // the J-th largest of the lanes' maxima
    float left = own.m;
    for (int j = 1; j < a.J; ++j) {
      const uint32_t who = __ballot_sync(0xffffffffu, left == reached);
      if (lane == __ffs(who) - 1) left = -INFINITY;
      asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(reached) : "f"(left));
    }
  } else if (TOP) {  // the smallest
    asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(reached) : "f"(own.m));
  }
  const float4 word = make_float4(v.m, v.s, v.t, reached);
  const float4* told = exchange.template tell<TOP>(word);
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
  const int entries = lp_whole<TH>(n - tid) + lp_rest<TH>(n - tid);
  uint32_t least = 0;  // the order of a NaN, which nothing is below
  if (MANY) {
    if (L == L) least = lp_bound(told, groups, a.need);
  } else if (L == L) {  // with NaN or +inf in the row the batches' largest logits say little
    reached = lane < groups ? told[lane].w : INFINITY;
    asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(reached) : "f"(reached));
    auto each = [&](auto f) {
      for (int b = 0; b < entries; ++b) f(ag_order(most[b * TH + tid]));
    };
    least = lp_threshold<TH>(each, ag_order(reached), ag_order(v.m), a.top, a.top + (a.top >> 1) + 16, hist);
  }
  const float bound = ag_of_order(least);
  // Counted even where there is no room: warps are at different places here, so that any of them may come behind `cap` others.
  auto take = [&](float x, int index) {
    const int to = atomicAdd(n_keys, 1);
    if (to < a.cap) keys[to] = lp_key(x, index);
  };
  for (int b = 0; b < entries; ++b) {
    if (most[b * TH + tid] < bound) continue;
    const int k = atomicAdd(n_keys + 1, 1);
    if (k < a.cap) batches[k] = b * TH + tid;
  }
  __syncthreads();
  const int listed = min(n_keys[1], a.cap);
  if (edge_index >= 0 && !(edge < bound)) take(edge, edge_index);
  for (int k = tid; k < listed * LP_BATCH; k += TH) {
    const int b = batches[k / LP_BATCH] / TH, of = batches[k / LP_BATCH] % TH, whole = lp_whole<TH>(n - of);
    if (b >= whole && k % LP_BATCH) continue;  // a packet by itself
    const int i = (b < whole ? b * LP_BATCH + k % LP_BATCH : whole * LP_BATCH + b - whole) * TH + of;
    float x[AG_PACKET<T>];
    ag_widen(at[i], x);
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < AG_PACKET<T>; ++e) hits |= x[e] < bound ? 0u : 1u << e;
    for (; hits; hits &= hits - 1) {
      const int index = first + i * AG_PACKET<T> + __ffs(hits) - 1;
      take(Pack<T>::load1(r.x + index), index);
    }
  }
  __syncthreads();
  int total = n_keys[0];
  if (total > a.cap || n_keys[1] > a.cap) {
    const LpPart<T, TH> part = {at, n, first, edge, edge_index};
    total = lp_search<T, TH>(part, least, a.top, a.cap, keys, n_keys + 2);
  }
  if (MANY) {
    // to block 0, each to its own place there
    const uint32_t to = ag_peer(all + (size_t)rank * a.cap, 0);
    for (int k = tid; k < total; k += TH) ag_peer_store(to + k * 8, keys[k]);
    if (tid == 0) ag_peer_store(ag_peer(counts + rank, 0), total);
    __syncthreads();
    if (tid == 0) ag_peer_arrive(ag_peer(s_keys_bar, 0));
    if (rank) return;
    ag_wait_cluster(s_keys_bar, 0, a.status);
    // side by side
    constexpr int MOVE = (lp_cap(AG_TOP_MAX) + TH - 1) / TH;  // keys of a block per thread, at most
    // (a count may be anything if the wait has expired)
    total = max(0, min(counts[0], a.cap));
    for (int p = 1; p < S; ++p) {
      const int more = max(0, min(counts[p], a.cap));
      unsigned long long mine[MOVE];  // what is moved down may lie over what is not yet
      for (int k = 0; k < MOVE; ++k)
        if (tid + k * TH < more) mine[k] = all[(size_t)p * a.cap + tid + k * TH];
      __syncthreads();
      for (int k = 0; k < MOVE; ++k)
        if (tid + k * TH < more) all[total + tid + k * TH] = mine[k];
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
  __shared__ int s_place[TH / 2];
  if (total <= TH / 2) {
    const int lanes = max(32, (total + 31) & ~31), parts = TH / lanes, i = tid % lanes;
    if (tid < lanes) s_place[i] = 0;
    __syncthreads();
    if (i < total && tid < parts * lanes) {
      const int place = larger(all[i], tid / lanes, parts);
      if (place) atomicAdd(&s_place[i], place);
    }
    __syncthreads();
    if (tid < total) put(all[tid], s_place[tid]);
  } else {
    for (int i = tid; i < total; i += TH) put(all[i], larger(all[i], 0, 1));
  }
}

// Gradient: a block takes `per` packets of a row.  fp32 gains by twice as many under way (8192 x 32768 334 / 328 us), bf16 by more
// blocks (179 / 171, which is nearer to what its exponentials take).
struct LbArgs {
  const int32_t* ids;
  const float4* stats;
  const float *dlogprob, *dentropy;
  int64_t ld, ld_grad;
  int V, S, per;
  float inv_tau;
};

template <typename T, int TH>
__global__ void __launch_bounds__(TH, (sizeof(T) == 4 ? 4 : 5) * 256 / TH)
logprobs_backward_kernel(const T* logits, const T* dres, T* dlogits, const LbArgs p) {
  constexpr int NV = AG_PACKET<T>, U = sizeof(T) == 4 ? 8 : 4;
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
  // p (a + b (ln p + H)) = p (k + b ln p) with ln p = d ln 2, p = 2^d.  A logit of -inf: p = 0, and 0 times something finite; a NaN
  // has to stay one.
  const float c = p.inv_tau * AG_LOG2E, shift = -st.y * AG_LOG2E, k = -(a + b * st.z), bd = -b * AG_LN2;
  const uint64_t ref2 = ag_pair(-st.x, -st.x), c2 = ag_pair(c, c), shift2 = ag_pair(shift, shift), k2 = ag_pair(k, k),
                 bd2 = ag_pair(bd, bd);
  auto local = [&](float x0, float x1, float& g0, float& g1) {
    float d0, d1;
    ag_unpair(ag_fma2(ag_add2(ag_pair(x0, x1), ref2), c2, shift2), d0, d1);
    d0 = ag_max_nan(d0, -1e4f);
    d1 = ag_max_nan(d1, -1e4f);
    ag_unpair(ag_mul2(ag_pair(ag_ex2(d0), ag_ex2(d1)), ag_fma2(bd2, ag_pair(d0, d1), k2)), g0, g1);
  };
  auto add = [&](float (&g)[NV], int i) {
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
  auto put = [&](const uint4& w, int i) {
    float x[NV], g[NV];
    ag_widen(w, x);
#pragma unroll
    for (int e = 0; e < NV; e += 2) local(x[e], x[e + 1], g[e], g[e + 1]);
    add(g, i);
  };
  int i = tid;
  if (none)  // 0, whatever the logits are
    for (; i < n; i += TH) {
      float g[NV] = {};
      add(g, i);
    }
  for (; i + (U - 1) * TH < n; i += U * TH) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldcs(at + i + u * TH);
#pragma unroll
    for (int u = 0; u < U; ++u) put(w[u], i + u * TH);
  }
  for (; i < n; i += 4 * TH) {  // what is left of a batch
    uint4 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * TH < n) w[u] = __ldcs(at + i + u * TH);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * TH < n) put(w[u], i + u * TH);
  }
  if (edge_index >= 0) {
    float g = 0.0f, other;
    if (!none) local(x_edge, x_edge, g, other);
    if (!none && edge_index == id) g += a;
    Pack<T>::store1(g_row + edge_index, g + (d_row ? Pack<T>::load1(d_row + edge_index) : 0.0f));
  }
}

template <typename T>
int logprobs_backward(ag_ctx* ctx, const void* logits, const void* dres, void* dlogits, LbArgs p, int64_t N) {
  const int packets = p.V / AG_PACKET<T>;
  p.S = ag_row_parts(ctx, N, packets);
  p.per = (packets + p.S - 1) / p.S;
  AG_REQUIRE(ctx, N * p.S < (1ll << 31), "ag_token_logprobs_backward: too many rows for V=%d", p.V);
  const T *x = static_cast<const T*>(logits), *d = static_cast<const T*>(dres);
  T* g = static_cast<T*>(dlogits);
  const unsigned grid = (unsigned)(N * p.S);
  const int th = p.S > 1 ? 256 : ag_row_threads(ctx, N, packets, LB_PACKETS_64, LB_PACKETS_128);
  if (th == 64) AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", (logprobs_backward_kernel<T, 64>), grid, 64, 0, x, d, g, p);
  else if (th == 128) AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", (logprobs_backward_kernel<T, 128>), grid, 128, 0, x, d, g, p);
  else AG_LAUNCH_PDL(ctx, "logprobs_backward_kernel", (logprobs_backward_kernel<T, 256>), grid, 256, 0, x, d, g, p);
  return AG_OK;
}

template <typename T, bool TOP, int TH, bool MANY>
int logprobs_launch(ag_ctx* ctx, const T* logits, const LpArgs& a) {
  const size_t smem = LpShared<TH>::bytes(a.S, a.cap, a.per);
  static std::atomic<bool> ready[AG_MAX_DEVICES];
  if (smem > 47 * 1024 && !ready[ag_dev_slot(ctx)].load(std::memory_order_acquire)) {
    AG_CUDA(ctx, cudaFuncSetAttribute(logprobs_kernel<T, TOP, TH, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    ready[ag_dev_slot(ctx)].store(true, std::memory_order_release);
  }
  return ag_launch_clusters(ctx, "logprobs_kernel", logprobs_kernel<T, TOP, TH, MANY>, a.S, TH, smem, a.N, logits, a);
}

template <typename T>
int logprobs(ag_ctx* ctx, const void* x, LpArgs a) {
  const T* logits = static_cast<const T*>(x);
  const int packets = (a.V + AG_PACKET<T> - 1) / AG_PACKET<T>;
  a.S = ag_cluster_parts(ctx, a.N, packets);
  a.per = (packets + a.S - 1) / a.S;
  a.status = ctx->d_status;
  AG_REQUIRE(ctx, a.N * a.S < (1ll << 31), "ag_token_logprobs_forward: too many rows");
  if (a.top == 0) {
    const int th = a.S > 1 ? 256 : ag_row_threads(ctx, a.N, packets, LP_PACKETS_64, LP_PACKETS_128);
    return th == 64    ? logprobs_launch<T, false, 64, true>(ctx, logits, a)
           : th == 128 ? logprobs_launch<T, false, 128, true>(ctx, logits, a)
                       : logprobs_launch<T, false, 256, true>(ctx, logits, a);
  }
  a.cap = lp_cap(a.top);
  if (a.S > 1) {
    // Lane maxima: where nearly all warps have to meet the bound, the one with the smallest logits decides, and many more than
    // `top` pass.  33 of 32 warps: the smallest of the second ones is passed by 200, the 17th of them by 55.
    const int groups = a.S * 8;
    a.J = (a.top + groups - 1) / groups;
    while (a.J < 32 && (a.top + a.J - 1) / a.J * 20 > groups * 17) ++a.J;
    a.need = (a.top + a.J - 1) / a.J;
    return logprobs_launch<T, true, 256, true>(ctx, logits, a);
  }
  // Short rows: what each warp does once per row weighs more than what more threads read at a time.
  const int th = ag_row_threads(ctx, a.N, packets, LP_TOP_64, LP_TOP_128);
  return th == 64    ? logprobs_launch<T, true, 64, false>(ctx, logits, a)
         : th == 128 ? logprobs_launch<T, true, 128, false>(ctx, logits, a)
                     : logprobs_launch<T, true, 256, false>(ctx, logits, a);
}

}  // namespace

extern "C" int ag_token_logprobs_forward(ag_ctx* ctx, const void* logits, int64_t ld, const int32_t* ids, float* logprob,
                                         float* entropy, float* stats, int32_t* top_ids, float* top_logprobs, int64_t N, int V,
                                         int top, float temperature, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  const char* who = "ag_token_logprobs_forward";
  if (int rc = ag_vocab_check(ctx, who, {N, ld, -1, V, top, dtype, temperature}, AG_VOCAB_MAX, AG_TOP_MAX, logits, nullptr, nullptr))
    return rc;
  AG_REQUIRE(ctx, top <= V, "%s: %d of %d tokens", who, top, V);
  AG_REQUIRE(ctx, !logprob || ids, "%s: log-probabilities of no tokens", who);
  AG_REQUIRE(ctx, top == 0 || (top_ids && top_logprobs) || N == 0, "%s: null pointer", who);
  AG_REQUIRE(ctx, ag_aligned16(stats), "%s: stats not 16-byte aligned", who);
  AG_REQUIRE(ctx, ag_aligned4(ids, logprob, entropy, top_ids, top_logprobs), "%s: pointer not aligned to its type", who);
  if (N == 0) return AG_OK;
  AgOnDevice on(ctx);
  const LpArgs a = {ids, logprob, entropy, (float4*)stats, top_ids, top_logprobs, N, ld, V, top, 1.0f / temperature, 0, 0, 0, 0, 0, nullptr};
  return dtype == AG_F32 ? logprobs<float>(ctx, logits, a) : logprobs<__nv_bfloat16>(ctx, logits, a);
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
  AG_REQUIRE(ctx, ag_aligned4(ids, dlogprob, dentropy), "%s: pointer not aligned to its type", who);
  if (N == 0) return AG_OK;
  AgOnDevice on(ctx);
  const LbArgs p = {ids, (const float4*)stats, dlogprob, dentropy, ld, ld_grad, V, 0, 0, 1.0f / temperature};
  return dtype == AG_F32 ? logprobs_backward<float>(ctx, logits, dres, dlogits, p, N)
                         : logprobs_backward<__nv_bfloat16>(ctx, logits, dres, dlogits, p, N);
}
