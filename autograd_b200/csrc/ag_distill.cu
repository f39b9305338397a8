// Distillation from a teacher's top logits: a row's loss against the teacher's distribution over a list of tokens, and its
// gradient.  With p = softmax(x / temperature) over the V tokens, slots k of the row's list with token id_k and value t_k:
//
//   RENORM  q = softmax(t / temperature) over the slots, r = 0
//   REST    q_k = exp(t_k), r = 1 - sum q, none up to DI_LEAST: t are log-probabilities, r what they leave to all other tokens together
//   row_loss = sum_k q_k (ln q_k - ln p_id_k) + r (ln r - ln p_rest),  p_rest = sum of p over the tokens not listed
//   d logits_j = s / temperature (p_j (Q + r) - sum_{k: id_k = j} q_k - r [j not listed] p_j / p_rest),  Q = sum q
//
// p_rest is summed over the unlisted logits themselves: 1 - sum_k p_id_k would keep nothing of a small rest.  A slot with a
// negative id is not in use.
// p_j / p_rest of an unlisted token is at most 1, but neither p_j nor 1 / p_rest need be a number of 32 bits: where ln p_rest is
// below DI_FAR it is one power, 2^((x_j - m') c - log2 sum') with the largest logit m' and the sum of the unlisted tokens alone,
// and p_j (Q + r) lies below its rounding (2^-46 against r / 2^24).
//
// Loss, and loss with gradient: a block, or a cluster of 2 to 8, streams a row through registers, thread k has slot k.  A bit per
// token tells what is listed: in the sum over the others those logits count as -inf, and the listed ones are added from the threads
// that have them, each token once.  The gradient comes from a second look at the row, which L2 still holds: rows under way take
// up to DI_IN_FLIGHT bytes, more blocks per row where they would take more.  The listed tokens' entries are written after it.
// Gradient alone: the same, without the first look, but twice as many packets under way (8192 x 32768 bf16, lists of 64: 204 / 195
// us, fp32 365 / 353).
#include "ag_vocab.cuh"

namespace {

// Blocks of 256 threads per SM, packets per thread under way in the first look.  Without a gradient and with the map more packets
// gain what more blocks do otherwise: us, 4 packets and 5 blocks (REST 4) / 8 packets and 4 blocks: loss of 512 x 32768 fp32 RENORM
// 17.0 / 15.2, REST 17.5 / 16.5, gradient REST of 8192 x 50257 bf16 341 / 322, 16384 x 32768 fp32 800 / 758, RENORM 734 / 827.
constexpr int distill_blocks(bool train, bool rest) { return train && !rest ? 5 : 4; }
constexpr int distill_batch(bool train, bool rest) { return train && !rest ? 4 : 8; }
// Packets of a row up to which a block has 64 or 128 threads.  16384 rows (of 32768: 8192), lists of 20 to 64, 64 / 128 / 256 threads,
// us: loss REST 640 fp32 34 / 53 / 98, 5003 66 / 85 / 143; with gradient RENORM 640 fp32 36 / 50 / 86, 5003 130 / 129 / 155, REST 10007
// bf16 156 / 179 / 256; gradient alone 5003 bf16 51 / 54 / 91, 10007 85 / 84 / 106, 32768 224 / 205 / 209.
constexpr int DI_PACKETS_64 = 2048, DI_PACKETS_128 = 4096;
// Bytes of the rows that are under way at a time, above which more blocks share a row: what is written then pushes out of L2 what is
// to be read again.  Us, 1 / 2 / 4 blocks per row: 16384 x 32768 fp32 RENORM (97, 48, 24 MB) 942 / 713 / 833; REST 8192 x 50257 bf16 (60,
// 30, 15 MB) 337 / 420 / 652; 4096 x 151936 bf16 (180, 90, 45 MB) 576 / 585 / 520.
constexpr int64_t DI_IN_FLIGHT = 64 << 20;
constexpr float DI_FAR = -32.0f;  // ln p_rest
// What 1 - sum q may be of a list that leaves nothing: of log-probabilities t in 32 bits, each within 7 u |t| and together with exp
// 25 u (u = 2^-24: differences from the largest logit, their product, the logarithm of the sum, its roundings, t's own, exp), of a
// distribution over 256 tokens at most, sum q |t| <= ln 256: 7 * 5.6 + 25 = 64 u.  Against a p_rest of 0, or of forbidden tokens,
// such an r would count without limit.
constexpr double DI_LEAST = 64.0 / (1 << 24);

struct DistillArgs {
  const int32_t* ids;
  const float* teacher;
  const float* row_scale;  // null: 1 / N
  const float* dloss;      // null: no gradient
  float* row_loss;
  float4* stats;           // (m, L, ln p_rest, 0), of a far rest (m, L, 1 + ln sum', m')
  int64_t N, ld, ld_grad;
  int V, top, rest;
  float inv_tau, inv_n;
  int* status;
  int S, per;  // blocks per row, packets per block
};

// Part of a list, and the whole of it merged from parts: m the largest t, sum = sum exp((t - m) / temperature) (RENORM) or the
// mass in 64 bits (REST).
struct DistillPart {
  float m;
  int nan;
  double sum;
};
struct DistillList {
  float m, log_sum, inv_sum;  // RENORM
  float mass, left;           // sum q and r
  bool used;
};
__device__ __forceinline__ DistillPart distill_part(float t, bool rest, float inv_tau) {
  DistillPart p;
  p.m = ag_warp_max(t);  // ignores NaN
  p.nan = __any_sync(0xffffffffu, t != t);
  if (rest) {
    p.sum = expf(t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) p.sum += __shfl_xor_sync(0xffffffffu, p.sum, o);
  } else {
    p.sum = ag_warp_sum(t == -INFINITY ? 0.0f : expf((t - p.m) * inv_tau));
  }
  return p;
}
// by whole warps; n <= 8 parts
__device__ __forceinline__ DistillList distill_list(const DistillPart* part, int n, bool rest, float inv_tau) {
  const int lane = threadIdx.x & 31;
  const DistillPart p = lane < n ? part[lane] : DistillPart{-INFINITY, 0, 0.0};
  DistillList l;
  l.m = ag_warp_max(p.m);
  const bool nan = __any_sync(0xffffffffu, p.nan);
  l.used = l.m > -INFINITY || nan;
  l.log_sum = 0.0f, l.inv_sum = 1.0f, l.left = 0.0f;
  if (rest) {
    double mass = p.sum;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    mass = __shfl_sync(0xffffffffu, mass, 0);
    l.mass = (float)mass;
    l.left = (float)(1.0 - mass > DI_LEAST ? 1.0 - mass : mass != mass ? mass : 0.0);
  } else {
    float sum = ag_warp_sum(p.m == -INFINITY ? 0.0f : (float)p.sum * expf((p.m - l.m) * inv_tau));
    if (nan) sum = NAN;
    l.log_sum = logf(sum);
    l.inv_sum = 1.0f / sum;
    l.mass = sum != sum ? sum : 1.0f;
  }
  if (!l.used) l.mass = l.left = 0.0f;
  return l;
}
// ln q and q of a slot with value t
__device__ __forceinline__ void distill_slot(const DistillList& l, float t, bool rest, float inv_tau, float& log_q, float& q) {
  const float d = rest || t == -INFINITY ? t : (t - l.m) * inv_tau;
  log_q = d - l.log_sum;
  q = l.used ? expf(d) * l.inv_sum : 0.0f;
}
// The gradient of the unlisted tokens as scale * 2^((x + ref) c + shift).  The listed ones, whose place it takes for a while, may
// be anything.  log_rest = ln p_rest; far: p / p_rest = 2^((x - m_out) c - log_out * log2(e)).  Nothing is left of p_rest = 0.
struct DistillDense {
  float scale, ref, shift;
};
__device__ __forceinline__ bool distill_far(float log_rest) { return log_rest < DI_FAR && log_rest > -INFINITY; }
__device__ __forceinline__ DistillDense distill_unlisted(const DistillList& l, float s, float m, float L, bool far, float log_rest,
                                                         float m_out, float log_out) {
  if (far && l.left != 0.0f) return {-s * l.left, -m_out, -log_out * AG_LOG2E};
  const float rest = l.left != 0.0f && log_rest > -INFINITY ? l.left * expf(-log_rest) : 0.0f;
  return {s * (l.mass + l.left - rest), -m, -L * AG_LOG2E};
}
__device__ __forceinline__ float distill_scale(const DistillArgs& a, int64_t row) {
  const float w = a.row_scale ? a.row_scale[row] : a.inv_n;
  return w == 0.0f ? 0.0f : a.dloss[0] * w * a.inv_tau;
}

// -inf in the places of a packet whose bits are set
__device__ __forceinline__ void distill_mask(uint4& w, uint32_t bits, float) {
  if (bits & 1) w.x = 0xff800000u;
  if (bits & 2) w.y = 0xff800000u;
  if (bits & 4) w.z = 0xff800000u;
  if (bits & 8) w.w = 0xff800000u;
}
__device__ __forceinline__ void distill_mask(uint4& w, uint32_t bits, __nv_bfloat16) {
  uint32_t* v = &w.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bits >> (2 * i) & 1) v[i] = (v[i] & 0xffff0000u) | 0xff80u;
    if (bits >> (2 * i) & 2) v[i] = (v[i] & 0xffffu) | 0xff800000u;
  }
}

// Statistics of the unlisted logits of this thread's part; as ag_part_stat.  map: a byte per packet.
template <typename T, int U, int TH>
__device__ __forceinline__ AgStat distill_part_stat(const uint4* at, const uint8_t* map, int n, float edge, float c) {
  AgStat v = {edge == edge ? edge : -INFINITY, edge == -INFINITY ? 0.0f : edge - edge + 1.0f, 0.0f};
  const uint4* p = at + threadIdx.x;
  const uint8_t* b = map + threadIdx.x;
  int left = n - (int)threadIdx.x;
  for (; left > (U - 1) * TH; left -= U * TH, p += U * TH, b += U * TH) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = p[u * TH];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (const uint32_t bits = b[u * TH]) distill_mask(w[u], bits, T());
    ag_stat_add<false, T>(v, w, ag_largest(w, T()), c);
  }
  for (; left > 0; left -= 4 * TH, p += 4 * TH, b += 4 * TH) {
    uint4 w[4][1];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (left > u * TH) w[u][0] = p[u * TH];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (left > u * TH) {
        distill_mask(w[u][0], b[u * TH], T());
        ag_stat_add<false, T>(v, w[u], ag_largest(w[u], T()), c);
      }
  }
  return v;
}

// scale * 2^((x + ref) c + shift) of a packet's logits
template <typename T>
__device__ __forceinline__ void distill_dense(const uint4& w, uint64_t ref2, uint64_t c2, uint64_t shift2, float scale,
                                              float (&g)[AG_PACKET<T>]) {
  float x[AG_PACKET<T>];
  ag_widen(w, x);
#pragma unroll
  for (int e = 0; e < AG_PACKET<T>; e += 2) {
    float d0, d1;
    ag_unpair(ag_fma2(ag_add2(ag_pair(x[e], x[e + 1]), ref2), c2, shift2), d0, d1);
    g[e] = scale * ag_ex2(d0);  // not as a pair: 16384 x 32768 fp32 749 us that way, 700 this way
    g[e + 1] = scale * ag_ex2(d1);
  }
}

// Shared memory from the exchange's box on, for the kernel and for the launch that counts it.  All lengths are multiples of 16 bytes.
static_assert(sizeof(DistillPart) == 16 && AG_DISTILL_MAX % 4 == 0, "marks are cleared 16 bytes at a time");
template <int TH>
struct DistillShared {
  uint64_t* bars;      // [2] one of the exchange
  DistillPart* parts;  // [warps of a block] of the list
  int* ids;            // [AG_DISTILL_MAX] slots' tokens
  float* q;            // [AG_DISTILL_MAX] and masses
  float* sum;          // [8] loss per warp
  uint32_t* marks;     // [4] bits of the edges, whether a token is listed twice
  uint8_t* map;        // a byte per packet
  __host__ __device__ __forceinline__ DistillShared(float4* box, int S) {
    bars = reinterpret_cast<uint64_t*>(box + S * (TH / 32));
    parts = reinterpret_cast<DistillPart*>(bars + 2);
    ids = reinterpret_cast<int*>(parts + (TH / 32));
    q = reinterpret_cast<float*>(ids + AG_DISTILL_MAX);
    sum = q + AG_DISTILL_MAX;
    marks = reinterpret_cast<uint32_t*>(sum + 8);
    map = reinterpret_cast<uint8_t*>(marks + 4);
  }
  static size_t bytes(int S, int per, bool map) {
    return ag_counted_bytes(DistillShared(ag_counted_shared(), S).map + (map ? (per + 15) / 16 * 16 : 0));
  }
};

template <typename T, bool TRAIN, bool REST, int TH>
__global__ void __launch_bounds__(TH, distill_blocks(TRAIN, REST) * 256 / TH)
distill_kernel(const T* logits, T* dlogits, const DistillArgs a) {
  constexpr int NV = AG_PACKET<T>, BATCH = distill_batch(TRAIN, REST);
  extern __shared__ float4 s_box[];
  const int S = a.S, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = S > 1 ? ag_cluster_rank() : 0;
  const int groups = S * (TH / 32), parts = (a.top + 31) / 32;
  const DistillShared<TH> shared(s_box, S);
  const AgExchange<TH> exchange = {s_box, shared.bars, S, rank, a.status};
  DistillPart* s_parts = shared.parts;
  int* s_ids = shared.ids;
  float *s_q = shared.q, *s_sum = shared.sum;
  uint32_t* s_marks = shared.marks;  // [0] edges, [1] a token is listed twice, [4..] packets
  uint8_t* s_map = shared.map;
  const float c = a.inv_tau * AG_LOG2E;
  exchange.start();
  ag_pdl_wait();
  ag_pdl_trigger();

  const int64_t row = blockIdx.x / S;
  const AgRow<T> r(logits + row * a.ld, a.V);
  const int n = r.mine(rank, a.per), first = r.head + rank * a.per * NV;
  const uint4* at = reinterpret_cast<const uint4*>(r.x + first);
  int id = tid < a.top ? a.ids[row * a.top + tid] : -1;
  float t = tid < a.top ? a.teacher[row * a.top + tid] : -INFINITY;
  const float s = TRAIN ? distill_scale(a, row) : 0.0f;
  const int edge_index = r.edge(rank);
  float edge = edge_index >= 0 ? Pack<T>::load1(r.x + edge_index) : -INFINITY;
  if (TRAIN || REST) {
    for (int i = tid; i < (a.per + 15) / 16 + 1; i += TH) reinterpret_cast<uint4*>(s_marks)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  if (id >= a.V) {
    if (rank == 0) atomicOr(a.status, AG_STATUS_BAD_INDEX);
    id = -1;
  }
  if (id < 0) t = -INFINITY;
  const bool own = id >= 0 && r.owner(id, a.per) == rank;
  float x_id = -INFINITY;
  if (id >= 0 && (rank == 0 || own)) x_id = Pack<T>::load1(r.x + id);
  if ((TRAIN || REST) && own) {
    const int q = id - first;  // among this block's packets, or in the edges: 0.. before them, 16.. behind them
    const bool body = id >= r.head && id < r.head + r.body * NV;
    const int edge_bit = id < r.head ? id : 16 + id - r.head - r.body * NV;
    const uint32_t bit = body ? 1u << ((q / NV & 3) * 8 + q % NV) : 1u << edge_bit;
    if (atomicOr(body ? s_marks + 4 + q / NV / 4 : s_marks, bit) & bit) s_marks[1] = 1;
  }
  if (tid < a.top) s_ids[tid] = id;
  if (warp < parts) {
    const DistillPart p = distill_part(t, REST, a.inv_tau);
    if (lane == 0) s_parts[warp] = p;
  }
  __syncthreads();
  bool once = own;
  if ((TRAIN || REST) && s_marks[1] && own)
    for (int k = 0; k < tid; ++k) once &= s_ids[k] != id;
  const float x_edge = edge;
  if (REST && edge_index >= 0 && s_marks[0] >> tid & 1) edge = -INFINITY;

  const AgStat mine = ag_stat_warp(REST ? distill_part_stat<T, BATCH, TH>(at, s_map, n, edge, c)
                                          : ag_part_stat<false, T, BATCH, TH, !TRAIN>(at, n, edge, c), c);
  AgStat in = ag_stat_none();
  if (REST && warp < parts) {
    if (once) in = {x_id == x_id ? x_id : -INFINITY, x_id == -INFINITY ? 0.0f : x_id - x_id + 1.0f, 0.0f};
    in = ag_stat_warp(in, c);
  }
  // If the gradient takes the logits' place: the first block has read those of other blocks' parts before its word goes out, on which
  // they are overwritten.  (Otherwise they are apart altogether, and go without: 16384 x 32768 fp32 REST 775 / 761 us.)
  if (TRAIN && S > 1 && rank == 0 && warp < parts && logits == dlogits) ag_cluster_fence();
  const float4 word = make_float4(mine.m, mine.s, in.m, in.s);
  const float4* told = exchange.template tell<TRAIN>(word);
  if (!TRAIN && rank) return;
  AgStat out = ag_stat_none();
  in = ag_stat_none();
  if (lane < groups) {
    const float4 w = told[lane];
    out = {w.x, w.y, 0.0f};
    if (REST) in = {w.z, w.w, 0.0f};
  }
  if (lane + 32 < groups) {
    const float4 w = told[lane + 32];
    out = ag_stat_merge(out, {w.x, w.y, 0.0f}, c);
    if (REST) in = ag_stat_merge(in, {w.z, w.w, 0.0f}, c);
  }
  out = ag_stat_warp(out, c);
  AgStat all = out;
  float log_rest = 0.0f;
  if (REST) {
    all = ag_stat_merge(ag_stat_warp(in, c), out, c);
    log_rest = out.m == -INFINITY && out.s == 0.0f ? -INFINITY : (out.m - all.m) * a.inv_tau + logf(out.s) - logf(all.s);
  }
  const float m = all.m, L = logf(all.s);
  const DistillList list = distill_list(s_parts, parts, REST, a.inv_tau);
  auto log_p = [&](float x) { return x == -INFINITY && !(L != L) ? -INFINITY : (x - m) * a.inv_tau - L; };
  float q = 0.0f;
  if (warp < parts) {
    float log_q = 0.0f;
    if (id >= 0) distill_slot(list, t, REST, a.inv_tau, log_q, q);
    if (TRAIN && tid < a.top) s_q[tid] = q;
    if (rank == 0) {
      const float sum = ag_warp_sum(id >= 0 && q != 0.0f ? q * (log_q - log_p(x_id)) : 0.0f);
      if (lane == 0) s_sum[warp] = sum;
    }
  }
  const bool none = s == 0.0f || !list.used || (m == -INFINITY && L == -INFINITY);
  const bool far = REST && distill_far(log_rest);
  T* g_row = dlogits + row * a.ld_grad;
  if (TRAIN) {
    const DistillDense u = distill_unlisted(list, s, m, L, far, log_rest, out.m, logf(out.s));
    const uint64_t ref2 = ag_pair(u.ref, u.ref), c2 = ag_pair(c, c), shift2 = ag_pair(u.shift, u.shift);
    const bool packets = (((uintptr_t)(g_row + first)) & 15) == 0;
    auto put = [&](const uint4& w, int i) {
      float g[NV];
      distill_dense<T>(w, ref2, c2, shift2, u.scale, g);
      ag_store_packet<T>(g_row + first + (int64_t)i * NV, g, packets);
    };
    constexpr int U = 4;
    int i = tid;
    if (none) {  // 0, whatever the logits are
      const float g[NV] = {};
      for (; i < n; i += TH) ag_store_packet<T>(g_row + first + (int64_t)i * NV, g, packets);
    }
    for (; i + (U - 1) * TH < n; i += U * TH) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = at[i + u * TH];
#pragma unroll
      for (int u = 0; u < U; ++u) put(w[u], i + u * TH);
    }
    for (; i < n; i += TH) put(at[i], i);
    if (edge_index >= 0) Pack<T>::store1(g_row + edge_index, none ? 0.0f : u.scale * ag_ex2((x_edge + u.ref) * c + u.shift));
  }
  __syncthreads();  // the loss of each warp is there; the entries of listed tokens are written once more
  if (rank == 0 && tid == 0) {
    float sum = list.left != 0.0f ? list.left * (logf(list.left) - log_rest) : 0.0f;
    for (int w = 0; w < parts; ++w) sum += s_sum[w];
    a.row_loss[row] = list.used ? sum : 0.0f;
    if (a.stats) a.stats[row] = far ? make_float4(m, L, 1.0f + logf(out.s), out.m) : make_float4(m, L, log_rest, 0.0f);
  }
  if (TRAIN && once) {
    if (s_marks[1])
      for (int k = tid + 1; k < a.top; ++k)
        if (s_ids[k] == id) q += s_q[k];
    const float p = ag_ex2((x_id - m) * c - L * AG_LOG2E);
    Pack<T>::store1(g_row + id, none ? 0.0f : s * (p * (list.mass + list.left) - q));
  }
}

// The gradient alone, from the statistics that the loss left: a block takes `per` packets of a row.
template <typename T, bool REST, int TH>
__global__ void __launch_bounds__(TH, 3 * 256 / TH)
distill_backward_kernel(const T* logits, const T* dres, T* dlogits, const DistillArgs a) {
  constexpr int NV = AG_PACKET<T>, U = 8;
  __shared__ DistillPart s_parts[(TH / 32)];
  __shared__ int s_ids[AG_DISTILL_MAX];
  __shared__ float s_q[AG_DISTILL_MAX];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, parts = (a.top + 31) / 32;
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t row = blockIdx.x / a.S;
  const int rank = (int)(blockIdx.x - row * a.S);
  const AgRow<T> r(logits + row * a.ld, a.V);
  const int n = r.mine(rank, a.per), first = r.head + rank * a.per * NV;
  const uint4* at = reinterpret_cast<const uint4*>(r.x + first);
  T* g_row = dlogits + row * a.ld_grad;
  const T* d_row = dres ? dres + row * a.ld_grad : nullptr;
  const float4 st = a.stats[row];
  const float m = st.x, L = st.y, c = a.inv_tau * AG_LOG2E;
  int id = -1;
  float t = -INFINITY, x_id = 0.0f, d_id = 0.0f;
  if (tid < a.top) {
    id = a.ids[row * a.top + tid];
    t = a.teacher[row * a.top + tid];
    if (id >= a.V) {
      if (rank == 0) atomicOr(a.status, AG_STATUS_BAD_INDEX);
      id = -1;
    }
    if (id < 0) t = -INFINITY;
    s_ids[tid] = id;
  }
  const float s = distill_scale(a, row);
  const int edge_index = r.edge(rank);
  const float x_edge = edge_index >= 0 ? Pack<T>::load1(r.x + edge_index) : 0.0f;
  const bool own = id >= 0 && r.owner(id, a.per) == rank;
  if (own) {
    x_id = Pack<T>::load1(r.x + id);
    if (d_row) d_id = Pack<T>::load1(d_row + id);
  }
  if (warp < parts) {
    const DistillPart p = distill_part(t, REST, a.inv_tau);
    if (lane == 0) s_parts[warp] = p;
  }
  __syncthreads();
  const DistillList list = distill_list(s_parts, parts, REST, a.inv_tau);
  if (tid < a.top) {
    float log_q, q = 0.0f;
    if (id >= 0) distill_slot(list, t, REST, a.inv_tau, log_q, q);
    s_q[tid] = q;
  }
  const bool none = s == 0.0f || !list.used || (m == -INFINITY && L == -INFINITY);
  // A far rest as the loss leaves it; ln p_rest that comes from elsewhere serves as well, to 2^-22 |ln p_rest| of the result.
  const bool left = REST && st.z >= 0.5f, far = REST && (left || distill_far(st.z));
  const DistillDense v = distill_unlisted(list, s, m, L, far, st.z, left ? st.w : m, left ? st.z - 1.0f : L + st.z);
  const uint64_t ref2 = ag_pair(v.ref, v.ref), c2 = ag_pair(c, c), shift2 = ag_pair(v.shift, v.shift);
  const bool packets = (((uintptr_t)(g_row + first)) & 15) == 0, d_packets = (((uintptr_t)(d_row + first)) & 15) == 0;
  auto add = [&](float (&g)[NV], int i) {
    const int to = first + i * NV;
    if (d_row) {
      float d[NV];
      ag_load_packet<T>(d_row + to, d, d_packets);
#pragma unroll
      for (int e = 0; e < NV; ++e) g[e] += d[e];
    }
    ag_store_packet<T>(g_row + to, g, packets);
  };
  auto put = [&](const uint4& w, int i) {
    float g[NV];
    distill_dense<T>(w, ref2, c2, shift2, v.scale, g);
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
  for (; i < n; i += TH) put(__ldcs(at + i), i);
  if (edge_index >= 0) {
    const float d = d_row ? Pack<T>::load1(d_row + edge_index) : 0.0f;
    Pack<T>::store1(g_row + edge_index, (none ? 0.0f : v.scale * ag_ex2((x_edge + v.ref) * c + v.shift)) + d);
  }
  __syncthreads();  // the entries of listed tokens are written once more
  if (own) {
    bool once = true;
    float q = 0.0f;
    for (int k = 0; k < a.top; ++k)
      if (s_ids[k] == id) {
        once &= k >= tid;
        q += s_q[k];
      }
    const float p = ag_ex2((x_id - m) * c - L * AG_LOG2E);
    if (once) Pack<T>::store1(g_row + id, (none ? 0.0f : s * (p * (list.mass + list.left) - q)) + d_id);
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

// Threads of a block: short rows leave most of 256 idle, but a slot of the list needs one.
static_assert(AG_DISTILL_MAX <= 256, "a slot per thread, and eight warps' parts of the list and of the loss");
int distill_threads(const ag_ctx* ctx, int64_t N, int packets, int top) {
  const int th = ag_row_threads(ctx, N, packets, DI_PACKETS_64, DI_PACKETS_128);
  return th >= top ? th : top <= 128 ? 128 : 256;
}

template <typename T, bool TRAIN, bool REST, int TH>
int distill_launch(ag_ctx* ctx, const T* logits, T* dlogits, const DistillArgs& a) {
  static std::atomic<bool> ready[AG_MAX_DEVICES];
  const size_t smem = DistillShared<TH>::bytes(a.S, a.per, TRAIN || REST);
  if (smem > 48 * 1024 && !ready[ag_dev_slot(ctx)].load(std::memory_order_acquire)) {
    AG_CUDA(ctx, cudaFuncSetAttribute(distill_kernel<T, TRAIN, REST, TH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)DistillShared<TH>::bytes(8, AG_VOCAB_MAX / AG_PACKET<T> + 1, true)));
    ready[ag_dev_slot(ctx)].store(true, std::memory_order_release);
  }
  return ag_launch_clusters(ctx, "distill_kernel", distill_kernel<T, TRAIN, REST, TH>, a.S, TH, smem, a.N, logits, dlogits, a);
}

template <typename T, bool TRAIN, bool REST>
int distill_forward(ag_ctx* ctx, const void* logits, void* dlogits, DistillArgs a) {
  const int packets = (a.V + AG_PACKET<T> - 1) / AG_PACKET<T>, blocks = distill_blocks(TRAIN, REST);
  a.S = ag_cluster_parts(ctx, a.N, packets);
  if (TRAIN)
    while (a.S < 8 && (int64_t)packets * 16 * ctx->sm_count * blocks > DI_IN_FLIGHT * a.S && packets / a.S >= 512) a.S *= 2;
  a.per = (packets + a.S - 1) / a.S;
  AG_REQUIRE(ctx, a.N * a.S < (1ll << 31), "distillation: too many rows");
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(dlogits);
  const int th = a.S > 1 || (TRAIN && packets > DI_PACKETS_64) ? 256 : distill_threads(ctx, a.N, packets, a.top);
  return th == 64 ? distill_launch<T, TRAIN, REST, 64>(ctx, x, g, a) : th == 128 ? distill_launch<T, TRAIN, REST, 128>(ctx, x, g, a)
                                                                               : distill_launch<T, TRAIN, REST, 256>(ctx, x, g, a);
}

template <typename T, bool REST>
int distill_backward(ag_ctx* ctx, const void* logits, const void* dres, void* dlogits, DistillArgs a) {
  const int packets = a.V / AG_PACKET<T>;
  a.S = ag_row_parts(ctx, a.N, packets);
  a.per = (packets + a.S - 1) / a.S;
  AG_REQUIRE(ctx, a.N * a.S < (1ll << 31), "ag_distill_backward: too many rows for V=%d", a.V);
  const T *x = static_cast<const T*>(logits), *d = static_cast<const T*>(dres);
  T* g = static_cast<T*>(dlogits);
  const unsigned grid = (unsigned)(a.N * a.S);
  const int th = a.S > 1 ? 256 : distill_threads(ctx, a.N, packets, a.top);
  if (th == 64) AG_LAUNCH_PDL(ctx, "distill_backward_kernel", (distill_backward_kernel<T, REST, 64>), grid, 64, 0, x, d, g, a);
  else if (th == 128) AG_LAUNCH_PDL(ctx, "distill_backward_kernel", (distill_backward_kernel<T, REST, 128>), grid, 128, 0, x, d, g, a);
  else AG_LAUNCH_PDL(ctx, "distill_backward_kernel", (distill_backward_kernel<T, REST, 256>), grid, 256, 0, x, d, g, a);
  return AG_OK;
}

template <typename T>
int distill_t(ag_ctx* ctx, const void* x, const void* d, void* g, const DistillArgs& a, bool backward) {
  if (backward) return a.rest ? distill_backward<T, true>(ctx, x, d, g, a) : distill_backward<T, false>(ctx, x, d, g, a);
  if (a.dloss) return a.rest ? distill_forward<T, true, true>(ctx, x, g, a) : distill_forward<T, true, false>(ctx, x, g, a);
  return a.rest ? distill_forward<T, false, true>(ctx, x, g, a) : distill_forward<T, false, false>(ctx, x, g, a);
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
  AG_REQUIRE(ctx, ag_aligned4(ids, teacher, row_scale, dloss, loss, row_loss), "%s: pointer not aligned to its type", who);
  if (N == 0 && !loss) return AG_OK;
  AgOnDevice on(ctx);
  const DistillArgs a = {ids, teacher, row_scale, dloss, row_loss, (float4*)stats, N, ld, ld_grad, V, top, mode == AG_DISTILL_REST,
                         1.0f / temperature, N ? (float)(1.0 / (double)N) : 0.0f, ctx->d_status, 0, 0};
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
