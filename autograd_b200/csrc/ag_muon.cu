// The orthogonal factor of matrices by Newton-Schulz products, and the optimizer step that moves a matrix along the factor
// of its momentum.
//
//   m <- m + (1 - beta) (g - m),  u = g + beta (m - g) or m,  X = u / max(|u|_F, eps), transposed where it has more rows
//   than columns (all of this is about singular values, which the transpose shares);
//   steps times:  A = X X^T,  Q = a I + b A + c A A,  X <- Q X,  which takes every singular value s of X to a s + b s^3 + c s^5;
//   p <- (1 - lr decay) p - lr scale X.
//
// Matrices of one size go through every kernel together, as many at a time as the workspace holds.
#include <stdlib.h>

#include <algorithm>

#include "ag_tma.cuh"

namespace {

constexpr int NS_BATCH = 32;          // matrices of one launch
constexpr int NS_NORM_BLOCKS = 128;   // blocks per matrix of the momentum kernel, at most
constexpr int NS_THREADS = 256;
constexpr int NS_PAD_M = 128, NS_PAD_N = 64;
constexpr int NS_MAX_SHORT = 16384, NS_MAX_LONG = 1 << 20, NS_MAX_STEPS = 32;
constexpr size_t NS_WORKSPACE = (size_t)512 << 20;

struct NsMatrices {
  float* p[NS_BATCH];
  const void* g[NS_BATCH];
  float* m[NS_BATCH];  // null: the factor of g itself
};

struct NsUpdate {
  float beta, grad_scale;
  int nesterov;
};

// Buffers of a batch.  Matrices are stored [m][n], m <= n, in rows of np, mp rows each
struct NsPlan {
  int rows, cols, m, n, mp, np, batch;
  size_t x_bytes, a_bytes, norm_bytes, total;
};

NsPlan ns_plan(int count, int rows, int cols) {
  NsPlan s = {};
  s.rows = rows; s.cols = cols;
  s.m = rows < cols ? rows : cols;
  s.n = rows < cols ? cols : rows;
  s.mp = (s.m + NS_PAD_M - 1) / NS_PAD_M * NS_PAD_M;
  s.np = (s.n + NS_PAD_N - 1) / NS_PAD_N * NS_PAD_N;
  const size_t x = (size_t)s.mp * s.np * 4, a = (size_t)s.mp * s.mp * 4, norm = NS_NORM_BLOCKS * sizeof(double);
  const size_t one = 2 * x + 2 * a + norm;
  size_t batch = NS_WORKSPACE / one;
  if (batch < 1) batch = 1;
  if (batch > (size_t)NS_BATCH) batch = NS_BATCH;
  if (batch > (size_t)count) batch = count;
  // as many in every batch
  const int rounds = (count + (int)batch - 1) / (int)batch;
  s.batch = (count + rounds - 1) / rounds;
  s.x_bytes = x * s.batch; s.a_bytes = a * s.batch; s.norm_bytes = norm * s.batch;
  s.total = 2 * s.x_bytes + 2 * s.a_bytes + s.norm_bytes;
  return s;
}

__device__ __forceinline__ float ns_load(const void* g, int bf16, int64_t i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]) : static_cast<const float*>(g)[i];
}
__device__ __forceinline__ float ns_direction(float g, float m, const NsUpdate& s) {
  return s.nesterov ? fmaf(s.beta, m - g, g) : m;
}

// m <- m + (1 - beta) (g - m); the squares of the update's elements, in 64 bits, summed by every block.  VEC: four elements to a
// thread, all addresses being aligned to that.
template <bool VEC>
__global__ void __launch_bounds__(NS_THREADS) ns_momentum_kernel(const NsMatrices mats, int64_t elements, int bf16, NsUpdate s,
                                                                 double* norms) {
  __shared__ double part[NS_THREADS / 32];
  ag_pdl_wait();
  ag_pdl_trigger();
  const void* g = mats.g[blockIdx.y];
  float* m = mats.m[blockIdx.y];
  double sum = 0.0;
  auto element = [&](float gi, float& mi) {
    float u = gi * s.grad_scale;
    if (m) {
      mi = fmaf(1.0f - s.beta, u - mi, mi);
      u = ns_direction(u, mi, s);
    }
    sum = fma((double)u, (double)u, sum);
  };
  constexpr int EACH = VEC ? 4 : 1, AHEAD = 4;
  const int64_t stride = (int64_t)gridDim.x * NS_THREADS, packets = elements / EACH;
  for (int64_t i = (int64_t)blockIdx.x * NS_THREADS + threadIdx.x; i < packets; i += stride * AHEAD) {
    float gv[AHEAD][EACH], mv[AHEAD][EACH];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t at = (i + k * stride) * EACH;
      if (i + k * stride >= packets) continue;
      if constexpr (VEC) {
        if (bf16) {
          const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(g) + at);
          gv[k][0] = __uint_as_float(w.x << 16); gv[k][1] = __uint_as_float(w.x & 0xffff0000u);
          gv[k][2] = __uint_as_float(w.y << 16); gv[k][3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
          Pack<float>::load(static_cast<const float*>(g) + at, gv[k]);
        }
        if (m) Pack<float>::load(m + at, mv[k]);
      } else {
        gv[k][0] = ns_load(g, bf16, at);
        if (m) mv[k][0] = m[at];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t at = (i + k * stride) * EACH;
      if (i + k * stride >= packets) continue;
#pragma unroll
      for (int e = 0; e < EACH; ++e) element(gv[k][e], mv[k][e]);
      if (m) {
        if constexpr (VEC) Pack<float>::store(m + at, mv[k]);
        else m[at] = mv[k][0];
      }
    }
  }
  if (VEC && blockIdx.x == 0 && threadIdx.x < elements % EACH) {
    const int64_t at = elements - 1 - threadIdx.x;
    float mi = m ? m[at] : 0.0f;
    element(ns_load(g, bf16, at), mi);
    if (m) m[at] = mi;
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NS_THREADS / 32; ++w) sum += part[w];
    norms[blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = sum;
  }
}

// What is kept between products: x * 2^12 as one or two 16-bit floats (`hi`, and what hi leaves), in planes of padded rows.
// Singular values stay near 1 or below, so that no element of X, A or Q is beyond a few units, and the smallest that
// keep all bits are 2^-26 (one word) or next to nothing (two): elements err by at most 2^-37 or 2^-38 beside that.
constexpr float NS_SCALE = 4096.0f;

struct NsPlane {
  __half *hi, *lo;  // lo null: one word
};

__device__ __forceinline__ float ns_get(const NsPlane& s, int64_t i) {
  return (__half2float(s.hi[i]) + (s.lo ? __half2float(s.lo[i]) : 0.0f)) * (1.0f / NS_SCALE);
}

// X = u / max(|u|, eps) in padded rows, transposed where the matrix is tall: tiles of 64 x 64
__global__ void __launch_bounds__(NS_THREADS) ns_start_kernel(const NsMatrices mats, NsPlan t, int bf16, NsUpdate s, float eps,
                                                              const double* norms, int norm_blocks, NsPlane X) {
  __shared__ float tile[64][65];
  __shared__ double factor;
  ag_pdl_wait();
  ag_pdl_trigger();
  const void* g = mats.g[blockIdx.z];
  const float* m = mats.m[blockIdx.z];
  const bool tall = t.rows > t.cols;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of X
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  float u[16], mv[16];
  const int row = tall ? c0 + ty : r0 + ty, col = tall ? r0 + tx : c0 + tx;  // of the matrix: rows 4 apart
  const int64_t at = (int64_t)row * t.cols + col;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const bool in = row + 4 * k < t.rows && col < t.cols;
    u[k] = in ? ns_load(g, bf16, at + (int64_t)(4 * k) * t.cols) : 0.0f;
    mv[k] = in && m ? m[at + (int64_t)(4 * k) * t.cols] : 0.0f;
  }
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < norm_blocks; i += 32) sum += norms[blockIdx.z * NS_NORM_BLOCKS + i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double norm = sqrt(sum);
    if (threadIdx.x == 0) factor = (double)NS_SCALE / (norm > eps || norm != norm ? norm : (double)eps);
  }
  __syncthreads();
  const double by = factor;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float v = u[k] * s.grad_scale;
    if (m) v = ns_direction(v, mv[k], s);
    tile[ty + 4 * k][tx] = (float)(v * by);
  }
  __syncthreads();
  const int64_t x = (int64_t)blockIdx.z * t.mp * t.np;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // eight neighbours of a row of X to a thread
    const int i = threadIdx.x + h * NS_THREADS, r = i >> 3, c = (i & 7) * 8;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = tall ? tile[c + 2 * k][r] : tile[r][c + 2 * k], b = tall ? tile[c + 2 * k + 1][r] : tile[r][c + 2 * k + 1];
      split_f16x2(a, b, hi[k], lo[k]);
    }
    const int64_t to = x + (int64_t)(r0 + r) * t.np + c0 + c;
    *reinterpret_cast<uint4*>(X.hi + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (X.lo) *reinterpret_cast<uint4*>(X.lo + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// ---------------------------------------------------------------------------- products
// One persistent kernel, D = f(L R) for every matrix of the batch: TMA producer, MMA issuer and epilogue warps as in
// ag_flce_tc.cu, on single CTAs (128 x BN) or on pairs of them (256 x BN).  Operands are planes, three MMAs per 16 elements of
// the contraction (hi lo, lo hi, hi hi) where there are two.
//   GRAM:  A = X X^T             both K-major
//   POLY:  Q = a I + b A + c AA  both symmetric
//   NEXT:  X' = Q X              symmetric, X MN-major
//   LAST:  the same, straight into p or out
// A and Q are symmetric (polynomials of one matrix commute): only the tiles on and above the diagonal are computed and
// stored.  A tile of an operand that lies below is read as the transpose of the one above, as an MN-major tile: which of the
// two is a matter of the map, the descriptor and a bit of the instruction, chosen for every 64 columns.
enum { NS_GRAM, NS_POLY, NS_NEXT, NS_LAST };
constexpr bool ns_symmetric(int kind) { return kind <= NS_POLY; }

constexpr int NS_EPI_WARPS = 8;
constexpr int NS_TC_THREADS = 128 + 32 * NS_EPI_WARPS;
constexpr int NS_MAX_STAGES = 6;
constexpr int NS_SMEM_LIMIT = 227 * 1024;
constexpr int NS_STAGING = NS_EPI_WARPS * 2048;  // 32 rows of 64 bytes on their way to p or out
constexpr int NS_SMEM_FIXED = 1024 + NS_STAGING + 256;
// The tensor core's sums truncate: chains of at most this many steps of 64 elements, added in registers
#ifndef CH
#define CH 1
#endif
constexpr int NS_CHAIN_PAIRS = CH, NS_CHAIN_SINGLE = 128;

// Tensor maps of a plane: tiles with the contraction along its rows (k), and along its columns (mn)
struct NsMaps {
  CUtensorMap k_hi, k_lo, mn_hi, mn_lo;
};

struct NsGemm {
  NsMaps l, r;
  int batch, tiles_m, tiles_n, tiles;  // tiles of a matrix; symmetric: those on and above the diagonal
  int k_iters, chain, stages;
  int M, N;            // rows and columns of a matrix that are stored (padded)
  int64_t ldd;
  NsPlane D, A;        // POLY reads A where D is written
  float diag, add, mul;
  // LAST
  NsMatrices mats;
  int rows, cols, tall, out_kind;
  float keep, by;
  int* status;
};

struct NsTile {
  int mat, tm, tn;
};

template <int KIND>
__device__ __forceinline__ bool ns_tile(const NsGemm& p, int unit, int units, int step, NsTile& t) {
  int i = unit + step * units;
  if (i >= p.batch * p.tiles) return false;
  t.mat = i / p.tiles;
  i -= t.mat * p.tiles;
  if (ns_symmetric(KIND)) {  // columns of tiles, the diagonal last in each
    int n = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while (n * (n + 1) / 2 > i) --n;
    while ((n + 1) * (n + 2) / 2 <= i) ++n;
    t.tn = n;
    t.tm = i - n * (n + 1) / 2;
  } else {
    t.tn = i / p.tiles_m;
    t.tm = i - t.tn * p.tiles_m;
  }
  return true;
}

// 32 columns of a lane's row as words
template <bool SPLIT>
__device__ __forceinline__ void ns_store_row(const NsPlane& d, int64_t at, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) split_f16x2(v[16 * j + 2 * k], v[16 * j + 2 * k + 1], hi[k], lo[k]);
    tc_st_global_v8(d.hi + at + 16 * j, hi);
    if (SPLIT) tc_st_global_v8(d.lo + at + 16 * j, lo);
  }
}
// p <- keep p - by v (kind 0), or v in fp32 (1) or bf16 (2)
__device__ __forceinline__ void ns_apply(void* p, int64_t i, float v, float old, float keep, float by, int kind) {
  if (kind == 2) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = kind == 0 ? fmaf(-by, v, keep * old) : v;
}

// 32 values of the lane in a column of the matrix, `n` of them inside
__device__ __forceinline__ void ns_apply_column(const NsGemm& p, int mat, int64_t at, const float (&v)[32], int n) {
  float* d = p.mats.p[mat];
#pragma unroll
  for (int h = 0; h < 32; h += 16) {
    float old[16];
    if (p.out_kind == 0) {
#pragma unroll
      for (int j = 0; j < 16; ++j) old[j] = h + j < n ? d[at + (int64_t)(h + j) * p.cols] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (h + j < n) ns_apply(d, at + (int64_t)(h + j) * p.cols, v[h + j], old[j], p.keep, p.by, p.out_kind);
  }
}

// 32 rows x 16 columns from (row0, col), v = the lane's row: four lanes per row, or two rows at a time where rows are not aligned
__device__ __forceinline__ void ns_apply_block(const NsGemm& p, int mat, unsigned char* stg, int lane, const float* v, int row0, int col) {
  float* d = p.mats.p[mat];
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) *tc_stage_at(stg, lane, j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  if (p.out_kind < 2 && (p.cols & 3) == 0 && (reinterpret_cast<uintptr_t>(d) & 15) == 0 && col + 16 <= p.cols) {
    const int r4 = lane >> 2, piece = lane & 3;
    float4* q = reinterpret_cast<float4*>(d + (int64_t)(row0 + r4) * p.cols + col) + piece;
    const int64_t next = (int64_t)p.cols * 2;  // eight rows, in float4
    float4 old[4];
    if (p.out_kind == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row0 + r4 + 8 * i < p.rows) old[i] = q[i * next];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (row0 + r4 + 8 * i >= p.rows) continue;
      float4 x = *tc_stage_at(stg, r4 + 8 * i, piece);
      if (p.out_kind == 0)
        x = make_float4(fmaf(-p.by, x.x, p.keep * old[i].x), fmaf(-p.by, x.y, p.keep * old[i].y), fmaf(-p.by, x.z, p.keep * old[i].z),
                        fmaf(-p.by, x.w, p.keep * old[i].w));
      q[i * next] = x;
    }
    return;
  }
  const int c = lane & 15, first = lane >> 4;
  if (col + c >= p.cols) return;
  const int64_t at = (int64_t)(row0 + first) * p.cols + col + c;
  float old[16];
  if (p.out_kind == 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) old[i] = row0 + first + 2 * i < p.rows ? d[at + (int64_t)(2 * i) * p.cols] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (row0 + first + 2 * i < p.rows)
      ns_apply(d, at + (int64_t)(2 * i) * p.cols, reinterpret_cast<const float*>(tc_stage_at(stg, first + 2 * i, c >> 2))[c & 3], old[i],
               p.keep, p.by, p.out_kind);
}

// All MMAs of a stage.  The products with a low part come first: what the tensor core cuts off a sum grows with it, and theirs is
// 2^-11 of the whole.
template <bool SPLIT, bool PAIR>
__device__ __forceinline__ void ns_stage_mmas(uint32_t acc, uint32_t lh, uint32_t ll, uint32_t l_step, uint32_t rh, uint32_t rl,
                                              uint32_t r_step, uint32_t idesc, uint32_t not_first) {
  constexpr uint32_t hi = TcDesc::hi;
  if (SPLIT) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k == 0) tc_mma<2, PAIR>(acc, lh, hi, rl, hi, idesc, not_first);
      else tc_mma<1, PAIR>(acc, lh + k * l_step, hi, rl + k * r_step, hi, idesc, 1u);
      tc_mma<1, PAIR>(acc, ll + k * l_step, hi, rh + k * r_step, hi, idesc, 1u);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!SPLIT && k == 0) tc_mma<2, PAIR>(acc, lh, hi, rh, hi, idesc, not_first);
    else tc_mma<1, PAIR>(acc, lh + k * l_step, hi, rh + k * r_step, hi, idesc, 1u);
  }
}

// four 16-byte loads at once of 32 words of 16 bits
struct NsWords {
  uint4 v[4];
  __device__ __forceinline__ void load(const __half* p) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(p + 8 * j);
  }
  __device__ __forceinline__ float2 pair(int k) const {  // words 2 k and 2 k + 1
    const uint4& q = v[k >> 2];
    const uint32_t w = (k & 3) == 0 ? q.x : (k & 3) == 1 ? q.y : (k & 3) == 2 ? q.z : q.w;
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
};

template <int KIND, bool SPLIT, bool PAIR, int BN>
__global__ void __launch_bounds__(NS_TC_THREADS, 1) ns_gemm_kernel(const __grid_constant__ NsGemm p) {
  extern __shared__ unsigned char ns_smem_raw[];
  constexpr bool R_MN = !ns_symmetric(KIND);          // the right operand is stored with its columns contiguous
  constexpr uint32_t A_BYTES = TC_BM * 128, BN_CTA = PAIR ? BN / 2 : BN, B_BYTES = BN_CTA * 128;
  constexpr uint32_t STAGE = (A_BYTES + B_BYTES) * (SPLIT ? 2 : 1);
  constexpr int BM = PAIR ? 2 * TC_BM : TC_BM;
  constexpr uint32_t COLUMNS = 2 * BN;                // of tensor memory: two accumulators
  constexpr int CHUNKS = BN / 64;                     // 32-column chunks of an epilogue warp
  constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  static_assert(!ns_symmetric(KIND) || BM == BN, "tiles on the diagonal are square");
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ns_smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* staging = tiles + (size_t)p.stages * STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + NS_STAGING);
  uint64_t* empty = full + NS_MAX_STAGES;
  uint64_t* acc_full = empty + NS_MAX_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? tc_cluster_rank() : 0u;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int row_off = PAIR ? (int)rank * TC_BM : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ag_mbar_init(&full[s], 1);
      ag_mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      ag_mbar_init(&acc_full[b], 1);
      ag_mbar_init(&acc_empty[b], PAIR ? 2 * NS_EPI_WARPS : NS_EPI_WARPS);
    }
    *abort_flag = 0;
    ag_fence_mbar_init();
  }
  if (PAIR) tc_cluster_sync(); else __syncthreads();
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ag_smem_u32(tmem_slot)), "r"(COLUMNS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ag_smem_u32(tmem_slot)), "r"(COLUMNS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool expired = false;
  ag_pdl_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      uint32_t stage = 0, phase = 0;
      NsTile t;
      for (int step = 0; !expired && ns_tile<KIND>(p, unit, units, step, t); ++step) {
        const int l_at = t.tm * BM + row_off;
        const int r_at = t.tn * BN + (int)rank * (PAIR ? (int)BN_CTA : 0);
        for (int k = 0; k < p.k_iters; ++k) {
          if (!tc_wait(&empty[stage], phase ^ 1u, abort_flag)) {
            expired = true;
            break;
          }
          unsigned char* s = tiles + (size_t)stage * STAGE;
          uint32_t full_addr = ag_smem_u32(&full[stage]);
          if (PAIR) {
            if (rank == 0) ag_mbar_expect_tx(&full[stage], 2u * STAGE);
            full_addr = tc_map_to_cta(full_addr, 0u);
          } else {
            ag_mbar_expect_tx(&full[stage], STAGE);
          }
          const int kx = k * TC_BK;
          const int blk = kx / BM;  // tile of the contraction
          auto load = [&](const CUtensorMap& k_map, const CUtensorMap& mn_map, unsigned char* dst, int at, bool mn) {
            if (!mn) {
              if (PAIR) tc_tma_load_2d_pair(&k_map, dst, full_addr, kx, t.mat * p.M + at);
              else tc_tma_load_2d(&k_map, dst, &full[stage], kx, t.mat * p.M + at);
            } else {
              if (PAIR) tc_tma_load_3d_pair(&mn_map, dst, full_addr, 0, t.mat * p.M + kx, at / TC_MN_GROUP);
              else tc_tma_load_3d(&mn_map, dst, &full[stage], 0, t.mat * p.M + kx, at / TC_MN_GROUP);
            }
          };
          const bool l_mn = KIND != NS_GRAM && t.tm > blk, r_mn = R_MN || (KIND == NS_POLY && t.tn > blk);
          load(p.l.k_hi, p.l.mn_hi, s, l_at, l_mn);
          if (SPLIT) {
            load(p.l.k_lo, p.l.mn_lo, s + A_BYTES, l_at, l_mn);
            load(p.r.k_hi, p.r.mn_hi, s + 2 * A_BYTES, r_at, r_mn);
            load(p.r.k_lo, p.r.mn_lo, s + 2 * A_BYTES + B_BYTES, r_at, r_mn);
          } else {
            load(p.r.k_hi, p.r.mn_hi, s + A_BYTES, r_at, r_mn);
          }
          if (++stage == (uint32_t)p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------------------------------------------------------- MMA issuer (pair: the leader only)
      uint32_t stage = 0, phase = 0, acc_par = 0;
      int buf = 0;
      const uint32_t tiles_u = ag_smem_u32(tiles) >> 4;
      TcDesc dk, dmn;
      dk.init(0);
      dmn.init(1);
      NsTile t;
      for (int step = 0; !expired && ns_tile<KIND>(p, unit, units, step, t); ++step) {
        uint32_t tacc = 0;
        int left = 0;
        for (int k = 0; k < p.k_iters; ++k) {
          uint32_t not_first = 1u;
          if (left == 0) {
            if (!tc_wait(&acc_empty[buf], ((acc_par >> buf) & 1u) ^ 1u, abort_flag)) {
              expired = true;
              break;
            }
            acc_par ^= 1u << buf;
            tacc = tmem_base + (uint32_t)buf * BN;
            left = p.k_iters - k < p.chain ? p.k_iters - k : p.chain;
            not_first = 0u;
          }
          if (!tc_wait(&full[stage], phase, abort_flag)) {
            expired = true;
            break;
          }
          tc_fence_after();
          const uint32_t su = tiles_u + stage * (STAGE >> 4);
          const int blk = k * TC_BK / BM;
          const bool l_mn = KIND != NS_GRAM && t.tm > blk, r_mn = R_MN || (KIND == NS_POLY && t.tn > blk);
          const uint32_t ah = su + (l_mn ? dmn.lo_const : dk.lo_const), al = ah + (A_BYTES >> 4);
          const uint32_t bh = su + ((SPLIT ? 2u * A_BYTES : A_BYTES) >> 4) + (r_mn ? dmn.lo_const : dk.lo_const), bl = bh + (B_BYTES >> 4);
          ns_stage_mmas<SPLIT, PAIR>(tacc, ah, al, l_mn ? dmn.step : dk.step, bh, bl, r_mn ? dmn.step : dk.step,
                                     IDESC | (l_mn ? 1u << 15 : 0u) | (r_mn ? 1u << 16 : 0u), not_first);
          if (PAIR) {
            const uint32_t e = ag_smem_u32(&empty[stage]);
            tc_commit_pair(tc_map_to_cta(e, 0u));
            tc_commit_pair(tc_map_to_cta(e, 1u));
          } else {
            tc_commit(&empty[stage]);
          }
          if (++stage == (uint32_t)p.stages) {
            stage = 0;
            phase ^= 1u;
          }
          if (--left == 0) {
            if (PAIR) {
              const uint32_t f = ag_smem_u32(&acc_full[buf]);
              tc_commit_pair(tc_map_to_cta(f, 0u));
              tc_commit_pair(tc_map_to_cta(f, 1u));
            } else {
              tc_commit(&acc_full[buf]);
            }
            buf ^= 1;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 4..11)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3, slice = (warp - 4) >> 2;
    unsigned char* stg = staging + (warp - 4) * 2048;
    uint32_t full_par = 0;
    int buf = 0;
    NsTile t;
    for (int step = 0; !expired && ns_tile<KIND>(p, unit, units, step, t); ++step) {
      const int row0 = t.tm * BM + row_off + quarter * 32, row = row0 + lane, col0 = t.tn * BN + slice * (BN / 2);
      const uint32_t toff = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slice * (BN / 2));
      const bool rows_in = row0 < p.M;  // padded sizes are multiples of 32
      const int64_t at = (int64_t)t.mat * p.M * p.ldd + (int64_t)row * p.ldd + col0;
      NsWords ah[2], al[2];             // POLY: A where the tile goes, a chunk ahead
      auto fetch = [&](const int c) {
        if (KIND == NS_POLY && rows_in && col0 + c * 32 < p.N) {
          ah[c & 1].load(p.A.hi + at + c * 32);
          if (SPLIT) al[c & 1].load(p.A.lo + at + c * 32);
        }
      };
      auto chunk = [&](const int c, float (&v)[32]) {
        const int col = col0 + c * 32;
        if (c + 1 < CHUNKS) fetch(c + 1);
        if (!rows_in || col >= p.N) return;
        if constexpr (KIND != NS_LAST) {
          if constexpr (KIND == NS_POLY) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float2 x = ah[c & 1].pair(k);
              if (SPLIT) {
                const float2 y = al[c & 1].pair(k);
                x.x += y.x; x.y += y.y;
              }
              v[2 * k] = fmaf(p.mul, v[2 * k], p.add * x.x);
              v[2 * k + 1] = fmaf(p.mul, v[2 * k + 1], p.add * x.y);
            }
            const int hit = row - col;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == hit) v[j] += p.diag;
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= p.mul;
          }
          ns_store_row<SPLIT>(p.D, at + c * 32, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= p.mul;
          if (p.tall) {  // row of X = column of the matrix: lanes are neighbours in memory
            if (row < p.cols) ns_apply_column(p, t.mat, (int64_t)col * p.cols + row, v, p.rows - col);
          } else {       // through shared memory, 32 rows x 16 columns at a time
#pragma unroll
            for (int h = 0; h < 2; ++h) ns_apply_block(p, t.mat, stg, lane, v + 16 * h, row0, col + 16 * h);
          }
        }
      };
      auto wait_full = [&]() {
        if (!tc_wait(&acc_full[buf], (full_par >> buf) & 1u, abort_flag)) {
          expired = true;
          return false;
        }
        full_par ^= 1u << buf;
        tc_fence_after();
        return true;
      };
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) tc_mbar_arrive_cluster(tc_map_to_cta(ag_smem_u32(&acc_empty[buf]), 0u));
          else ag_mbar_arrive(&acc_empty[buf]);
        }
        buf ^= 1;
      };
      float acc[CHUNKS][32];
      bool gone = false;
      for (int k = 0; k < p.k_iters; k += p.chain) {
        if (k + p.chain >= p.k_iters) fetch(0);
        if (!wait_full()) {
          gone = true;
          break;
        }
        const uint32_t from = toff + (uint32_t)buf * BN;
        if (k == 0) {
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) tc_tmem_ld32(from + c * 32, reinterpret_cast<uint32_t(&)[32]>(acc[c]));
          tc_tmem_ld_wait();
          release();
        } else {  // two chunks at a time: a load's latency is about what their additions take
#pragma unroll
          for (int c = 0; c < CHUNKS; c += 2) {
            uint32_t r[2][32];
            tc_tmem_ld32(from + c * 32, r[0]);
            if (CHUNKS > 1) tc_tmem_ld32(from + (c + 1) * 32, r[1]);
            tc_tmem_ld_wait();
            if (c + 2 >= CHUNKS) release();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c][j] += __uint_as_float(r[0][j]);
            if (CHUNKS > 1) {
#pragma unroll
              for (int j = 0; j < 32; ++j) acc[(c + 1) % CHUNKS][j] += __uint_as_float(r[1][j]);
            }
          }
        }
      }
      if (gone) break;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) chunk(c, acc[c]);
    }
  }
  if (expired && lane == 0) atomicOr(p.status, AG_STATUS_WAIT_EXPIRED);
  tc_fence_before();
  if (PAIR) tc_cluster_sync(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLUMNS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLUMNS) : "memory");
  }
}

// No steps: X itself
__global__ void __launch_bounds__(NS_THREADS) ns_finish_kernel(const NsMatrices mats, NsPlan t, NsPlane X, float keep, float by,
                                                               int out_kind) {
  ag_pdl_wait();
  ag_pdl_trigger();
  const int64_t x = (int64_t)blockIdx.y * t.mp * t.np, elements = (int64_t)t.rows * t.cols;
  for (int64_t i = (int64_t)blockIdx.x * NS_THREADS + threadIdx.x; i < elements; i += (int64_t)gridDim.x * NS_THREADS) {
    const int64_t row = i / t.cols, col = i - row * t.cols;
    float* p = mats.p[blockIdx.y];
    ns_apply(p, i, ns_get(X, x + (t.rows > t.cols ? col * t.np + row : row * t.np + col)), out_kind == 0 ? p[i] : 0.0f, keep, by, out_kind);
  }
}

// ---------------------------------------------------------------------------- host side
// Tensor map of a plane of `rows` rows (of all matrices) of `cols` columns: tiles of TC_BK columns and box_rows rows, or seen as
// {64, rows, cols / 64}, for the columns of a product, boxes of TC_BK rows and `box_rows` columns.
int ns_map(ag_ctx* ctx, CUtensorMap* tm, const void* plane, int64_t rows, int64_t cols, int box, bool mn_major) {
  EncodeTiledFn encode = tc_encode_fn(ctx);
  if (!encode) return AG_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1}, strides[2] = {(cuuint64_t)cols * 2, TC_MN_GROUP * 2};
  cuuint32_t boxes[3] = {TC_BK, (cuuint32_t)box, 1}, estr[3] = {1, 1, 1};
  if (mn_major) {
    dims[0] = TC_MN_GROUP; dims[2] = (cuuint64_t)(cols / TC_MN_GROUP);
    boxes[0] = TC_MN_GROUP; boxes[1] = TC_BK; boxes[2] = (cuuint32_t)(box / TC_MN_GROUP);
  }
  const CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, mn_major ? 3 : 2, const_cast<void*>(plane), dims, strides, boxes, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    AG_FAIL(ctx, AG_ERR_CUDA, "cuTensorMapEncodeTiled failed: CUresult %d (ptr %p, %lld x %lld, box %d)", (int)r, plane, (long long)rows,
            (long long)cols, box);
  return AG_OK;
}

int ns_maps(ag_ctx* ctx, NsMaps& m, const NsPlane& plane, int64_t rows, int64_t cols, int box) {
  int rc;
  if ((rc = ns_map(ctx, &m.k_hi, plane.hi, rows, cols, box, false)) || (rc = ns_map(ctx, &m.mn_hi, plane.hi, rows, cols, box, true))) return rc;
  m.k_lo = m.k_hi;
  m.mn_lo = m.mn_hi;
  if (plane.lo && ((rc = ns_map(ctx, &m.k_lo, plane.lo, rows, cols, box, false)) || (rc = ns_map(ctx, &m.mn_lo, plane.lo, rows, cols, box, true))))
    return rc;
  return AG_OK;
}

template <int KIND, bool SPLIT, bool PAIR, int BN>
int ns_launch(ag_ctx* ctx, NsGemm& p) {
  constexpr int BM = PAIR ? 256 : 128, BN_CTA = PAIR ? BN / 2 : BN;
  constexpr size_t STAGE = (size_t)(TC_BM + BN_CTA) * 128 * (SPLIT ? 2 : 1);
  static std::atomic<int> known[AG_MAX_DEVICES];  // 1 + units that are resident at once
  auto kern = ns_gemm_kernel<KIND, SPLIT, PAIR, BN>;
  std::atomic<int>& slot = known[ag_dev_slot(ctx)];
  int units = slot.load(std::memory_order_relaxed) - 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.blockDim = dim3(NS_TC_THREADS);
  cfg.dynamicSmemBytes = NS_SMEM_LIMIT;
  cfg.attrs = at;
  if (PAIR) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (units < 0) {
    AG_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM_LIMIT));
    units = ctx->sm_count;
    if (PAIR) {
      cfg.gridDim = dim3(2 * ctx->sm_count);
      AG_CUDA(ctx, cudaOccupancyMaxActiveClusters(&units, kern, &cfg));
      AG_REQUIRE(ctx, units > 0, "ns_gemm_kernel: no pair of CTAs fits the device");
    }
    slot.store(1 + units, std::memory_order_relaxed);
  }
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  p.tiles = ns_symmetric(KIND) ? p.tiles_n * (p.tiles_n + 1) / 2 : p.tiles_m * p.tiles_n;
  const int chain = SPLIT ? NS_CHAIN_PAIRS : NS_CHAIN_SINGLE, parts = (p.k_iters + chain - 1) / chain;
  p.chain = (p.k_iters + parts - 1) / parts;
  p.stages = std::min<int>(NS_MAX_STAGES, (int)((NS_SMEM_LIMIT - NS_SMEM_FIXED) / STAGE));
  units = std::min<int64_t>(units, (int64_t)p.batch * p.tiles);
  cfg.gridDim = dim3(PAIR ? 2 * units : units);
  cfg.dynamicSmemBytes = NS_SMEM_FIXED + p.stages * STAGE;
  cfg.stream = ctx->stream;
  if (ctx->pdl) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  AG_CUDA(ctx, cudaLaunchKernelEx(&cfg, kern, p));
  ctx->launches++;
  ag_enqueued(ctx);
  return AG_OK;
}

template <int KIND, bool SPLIT>
int ns_product(ag_ctx* ctx, NsGemm& p) {
  return p.M > 256 ? ns_launch<KIND, SPLIT, true, 256>(ctx, p) : ns_launch<KIND, SPLIT, false, 128>(ctx, p);
}

struct NsBuffer {
  NsPlane plane;
  NsMaps maps;
};

template <bool SPLIT>
int ns_iterate(ag_ctx* ctx, const NsPlan& t, NsGemm& p, NsPlane Xp, NsPlane Yp, NsPlane Ap, NsPlane Qp, const float* coefficients,
               int steps) {
  NsBuffer X[2], A, Q;
  X[0].plane = Xp; X[1].plane = Yp; A.plane = Ap; Q.plane = Qp;
  const int64_t rows = (int64_t)p.batch * t.mp;
  int rc;
  for (NsBuffer* b : {&X[0], &X[1], &A, &Q})
    if ((rc = ns_maps(ctx, b->maps, b->plane, rows, b == &A || b == &Q ? t.mp : t.np, TC_BM))) return rc;
  for (int i = 0; i < steps; ++i) {
    const float *co = coefficients + 3 * i, unit = 1.0f / NS_SCALE;
    NsBuffer &x = X[i & 1], &y = X[~i & 1];
    p.M = p.N = t.mp; p.ldd = t.mp;
    p.k_iters = t.np / TC_BK;
    p.l = p.r = x.maps;
    p.D = A.plane; p.mul = unit;
    if ((rc = ns_product<NS_GRAM, SPLIT>(ctx, p))) return rc;
    p.k_iters = t.mp / TC_BK;
    p.l = p.r = A.maps;
    p.D = Q.plane; p.A = A.plane;
    p.diag = co[0] * NS_SCALE; p.add = co[1]; p.mul = co[2] * unit;
    if ((rc = ns_product<NS_POLY, SPLIT>(ctx, p))) return rc;
    p.N = t.np; p.ldd = t.np;
    p.l = Q.maps; p.r = x.maps;
    p.D = y.plane;
    if (i + 1 < steps) {
      p.mul = unit;
      rc = ns_product<NS_NEXT, SPLIT>(ctx, p);
    } else {
      p.mul = unit * unit;
      rc = ns_product<NS_LAST, SPLIT>(ctx, p);
    }
    if (rc) return rc;
  }
  return AG_OK;
}

int ns_run(ag_ctx* ctx, const NsPlan& t, const NsMatrices& mats, int count, int bf16, const NsUpdate& s, float eps,
           const float* coefficients, int steps, float keep, float by, int out_kind, char* scratch, bool split) {
  auto plane = [&](size_t at, size_t bytes) {
    NsPlane r = {reinterpret_cast<__half*>(scratch + at), nullptr};
    if (split || steps == 0) r.lo = reinterpret_cast<__half*>(scratch + at + bytes / 2);
    return r;
  };
  const NsPlane X = plane(0, t.x_bytes), Y = plane(t.x_bytes, t.x_bytes), A = plane(2 * t.x_bytes, t.a_bytes),
                Q = plane(2 * t.x_bytes + t.a_bytes, t.a_bytes);
  double* norms = reinterpret_cast<double*>(scratch + 2 * t.x_bytes + 2 * t.a_bytes);
  const int64_t elements = (int64_t)t.rows * t.cols;
  bool vec = true;
  for (int i = 0; i < count; ++i)
    vec = vec && ag_aligned16(mats.m[i]) && ((uintptr_t)mats.g[i] & (bf16 ? 7 : 15)) == 0;
  const int each = vec ? 4 : 1;
  int blocks = ag_ceil_div(elements, (int64_t)NS_THREADS * 4 * each);
  if (blocks > NS_NORM_BLOCKS) blocks = NS_NORM_BLOCKS;
  if (vec)
    AG_LAUNCH_PDL(ctx, "ns_momentum_kernel", ns_momentum_kernel<true>, dim3(blocks, count), NS_THREADS, 0, mats, elements, bf16, s, norms);
  else
    AG_LAUNCH_PDL(ctx, "ns_momentum_kernel", ns_momentum_kernel<false>, dim3(blocks, count), NS_THREADS, 0, mats, elements, bf16, s, norms);
  AG_LAUNCH_PDL(ctx, "ns_start_kernel", ns_start_kernel, dim3(t.np / 64, t.mp / 64, count), NS_THREADS, 0, mats, t, bf16, s, eps,
                (const double*)norms, blocks, X);
  if (steps == 0) {
    int many = ag_ceil_div(elements, NS_THREADS * 4);
    if (many > 1024) many = 1024;
    AG_LAUNCH_PDL(ctx, "ns_finish_kernel", ns_finish_kernel, dim3(many, count), NS_THREADS, 0, mats, t, X, keep, by, out_kind);
    return AG_OK;
  }
  NsGemm p = {};
  p.batch = count;
  p.mats = mats;
  p.rows = t.rows; p.cols = t.cols; p.tall = t.rows > t.cols; p.out_kind = out_kind;
  p.keep = keep; p.by = by;
  p.status = ctx->d_status;
  return split ? ns_iterate<true>(ctx, t, p, X, Y, A, Q, coefficients, steps) : ns_iterate<false>(ctx, t, p, X, Y, A, Q, coefficients, steps);
}

bool ns_fits(int rows, int cols) {
  const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m > 0 && m <= NS_MAX_SHORT && n <= NS_MAX_LONG && (int64_t)rows * cols < (1ll << 31);
}

bool ns_finite(double x) { return x - x == 0.0; }

int ns_check(ag_ctx* ctx, const char* name, int count, int rows, int cols, const float* coefficients, int steps, float eps,
             int precision, const void* scratch) {
  AG_REQUIRE(ctx, count >= 0 && rows > 0 && cols > 0, "%s: bad shape count=%d rows=%d cols=%d", name, count, rows, cols);
  AG_REQUIRE(ctx, ns_fits(rows, cols), "%s: %d x %d is too large", name, rows, cols);
  AG_REQUIRE(ctx, steps >= 0 && steps <= NS_MAX_STEPS && (steps == 0 || coefficients), "%s: %d steps", name, steps);
  for (int i = 0; i < 3 * steps; ++i) AG_REQUIRE(ctx, ns_finite(coefficients[i]), "%s: coefficient %g", name, (double)coefficients[i]);
  AG_REQUIRE(ctx, eps > 0.0f && ns_finite(eps), "%s: eps %g", name, (double)eps);
  AG_REQUIRE(ctx, precision == AG_CE_3XTF32 || precision == AG_CE_BF16, "%s: precision %d", name, precision);
  AG_REQUIRE(ctx, count == 0 || (scratch && ((uintptr_t)scratch & 255) == 0), "%s: the workspace has to be 256-byte aligned", name);
  return AG_OK;
}

struct NsRange {
  uintptr_t from, to;
  bool written;
};

// Whether no range that is written meets another one; sorts them
bool ns_apart(NsRange* r, size_t n) {
  std::sort(r, r + n, [](const NsRange& x, const NsRange& y) { return x.from < y.from; });
  uintptr_t any = 0, written = 0;  // where those before end
  for (size_t i = 0; i < n; ++i) {
    if (r[i].from < (r[i].written ? any : written)) return false;
    any = std::max(any, r[i].to);
    if (r[i].written) written = std::max(written, r[i].to);
  }
  return true;
}

// All matrices of a call and its workspace: what one of them reads, another must not write, and no two write the same
int ns_check_ranges(ag_ctx* ctx, const char* name, const void* const* p, size_t p_size, const void* const* g, size_t g_size,
                    const void* const* m, int count, size_t elements, const void* scratch, size_t scratch_bytes) {
  NsRange few[96 + 1];
  const size_t most = 3 * (size_t)count + 1;
  NsRange* r = most <= 97 ? few : static_cast<NsRange*>(malloc(most * sizeof(NsRange)));
  if (!r) AG_FAIL(ctx, AG_ERR_INVALID, "%s: no memory to look %d matrices over", name, count);
  size_t n = 0;
  auto add = [&](const void* at, size_t bytes, bool written) {
    r[n++] = {(uintptr_t)at, (uintptr_t)at + bytes, written};
  };
  for (int i = 0; i < count; ++i) {
    add(p[i], elements * p_size, true);
    if (m) add(m[i], elements * 4, true);
    if (m || g[i] != p[i] || g_size < p_size) add(g[i], elements * g_size, false);  // the factor may take its matrix's place
  }
  add(scratch, scratch_bytes, true);
  const bool apart = ns_apart(r, n);
  if (r != few) free(r);
  AG_REQUIRE(ctx, apart, "%s: matrices overlap one another or the workspace", name);
  return AG_OK;
}

}  // namespace

extern "C" size_t ag_orthogonalise_scratch_bytes(int count, int rows, int cols, int precision) {
  if (count <= 0 || !ns_fits(rows, cols) || (precision != AG_CE_3XTF32 && precision != AG_CE_BF16)) return 0;
  return ns_plan(count, rows, cols).total;
}

extern "C" int ag_orthogonalise(ag_ctx* ctx, const void* const* g, void* const* out, int count, int rows, int cols,
                                const float* coefficients, int steps, float eps, int precision, int dtype, int out_dtype,
                                void* scratch, size_t scratch_bytes) {
  if (!ctx) return AG_ERR_INVALID;
  if (int rc = ns_check(ctx, "ag_orthogonalise", count, rows, cols, coefficients, steps, eps, precision, scratch)) return rc;
  if (count == 0) return AG_OK;
  AG_REQUIRE(ctx, g && out, "ag_orthogonalise: null pointer");
  AG_REQUIRE(ctx, (dtype == AG_F32 || dtype == AG_BF16) && (out_dtype == AG_F32 || out_dtype == AG_BF16),
             "ag_orthogonalise: unknown dtype %d or %d", dtype, out_dtype);
  for (int i = 0; i < count; ++i)
    AG_REQUIRE(ctx, g[i] && out[i] && ((uintptr_t)g[i] & (dtype == AG_F32 ? 3 : 1)) == 0 && ((uintptr_t)out[i] & (out_dtype == AG_F32 ? 3 : 1)) == 0,
               "ag_orthogonalise: null or misaligned matrix %d", i);
  const NsPlan t = ns_plan(count, rows, cols);
  if (scratch_bytes < t.total)
    AG_FAIL(ctx, AG_ERR_SCRATCH, "ag_orthogonalise: %zu bytes of workspace, %zu needed", scratch_bytes, t.total);
  if (int rc = ns_check_ranges(ctx, "ag_orthogonalise", out, out_dtype == AG_F32 ? 4 : 2, g, dtype == AG_F32 ? 4 : 2, nullptr, count,
                               (size_t)rows * cols, scratch, t.total))
    return rc;
  const NsUpdate s = {0.0f, 1.0f, 0};
  for (int first = 0; first < count; first += t.batch) {
    NsMatrices mats = {};
    const int here = count - first < t.batch ? count - first : t.batch;
    for (int i = 0; i < here; ++i) {
      mats.g[i] = g[first + i];
      mats.p[i] = static_cast<float*>(out[first + i]);
    }
    if (int rc = ns_run(ctx, t, mats, here, dtype == AG_BF16, s, eps, coefficients, steps, 0.0f, 0.0f, out_dtype == AG_F32 ? 1 : 2,
                        static_cast<char*>(scratch), precision == AG_CE_3XTF32))
      return rc;
  }
  return AG_OK;
}

extern "C" int ag_muon_step(ag_ctx* ctx, float* const* p, const void* const* g, float* const* m, int count, int rows, int cols,
                            double lr, double momentum, int nesterov, double weight_decay, double scale, double grad_scale,
                            const float* coefficients, int steps, float eps, int precision, int grad_dtype, void* scratch,
                            size_t scratch_bytes) {
  if (!ctx) return AG_ERR_INVALID;
  if (int rc = ns_check(ctx, "ag_muon_step", count, rows, cols, coefficients, steps, eps, precision, scratch)) return rc;
  if (count == 0) return AG_OK;
  AG_REQUIRE(ctx, p && g && m, "ag_muon_step: null pointer");
  AG_REQUIRE(ctx, grad_dtype == AG_F32 || grad_dtype == AG_BF16, "ag_muon_step: unknown dtype %d", grad_dtype);
  AG_REQUIRE(ctx, ns_finite(lr) && ns_finite(weight_decay) && ns_finite(scale) && ns_finite(grad_scale) && momentum >= 0.0 && momentum <= 1.0,
             "ag_muon_step: lr %g momentum %g weight_decay %g scale %g grad_scale %g", lr, momentum, weight_decay, scale, grad_scale);
  for (int i = 0; i < count; ++i)
    AG_REQUIRE(ctx, p[i] && g[i] && m[i] && (((uintptr_t)p[i] | (uintptr_t)m[i]) & 3) == 0 &&
                        ((uintptr_t)g[i] & (grad_dtype == AG_F32 ? 3 : 1)) == 0, "ag_muon_step: null or misaligned matrix %d", i);
  const NsPlan t = ns_plan(count, rows, cols);
  if (scratch_bytes < t.total)
    AG_FAIL(ctx, AG_ERR_SCRATCH, "ag_muon_step: %zu bytes of workspace, %zu needed", scratch_bytes, t.total);
  if (int rc = ns_check_ranges(ctx, "ag_muon_step", reinterpret_cast<const void* const*>(p), 4, g, grad_dtype == AG_F32 ? 4 : 2,
                               reinterpret_cast<const void* const*>(m), count, (size_t)rows * cols, scratch, t.total))
    return rc;
  const NsUpdate s = {(float)momentum, (float)grad_scale, nesterov != 0};
  for (int first = 0; first < count; first += t.batch) {
    NsMatrices mats = {};
    const int here = count - first < t.batch ? count - first : t.batch;
    for (int i = 0; i < here; ++i) {
      mats.p[i] = p[first + i];
      mats.g[i] = g[first + i];
      mats.m[i] = m[first + i];
    }
    if (int rc = ns_run(ctx, t, mats, here, grad_dtype == AG_BF16, s, eps, coefficients, steps, (float)(1.0 - lr * weight_decay),
                        (float)(lr * scale), 0, static_cast<char*>(scratch), precision == AG_CE_3XTF32))
      return rc;
  }
  return AG_OK;
}
