// The orthogonal factor of matrices by Newton-Schulz products, and the optimizer step that moves a matrix along the factor
// of its momentum.
//
//   m <- m + (1 - beta) (g - m),  u = g + beta (m - g) or m,  X = u / max(|u|_F, eps), transposed where it has more rows
//   than columns (all of this is about singular values, which the transpose shares);
//   steps times:  A = X X^T,  Q = a I + b A + c A A,  X <- Q X,  which takes every singular value s of X to a s + b s^3 + c s^5;
//   p <- (1 - lr decay) p - lr scale X.
//
// Matrices of one size go through every kernel together, as many at a time as the workspace holds.
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "ag_tma.cuh"

namespace {

constexpr int NS_BATCH = 96;          // matrices of one launch
constexpr int NS_NORM_BLOCKS = 256;   // blocks per matrix of the momentum kernel, at most
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

__device__ __forceinline__ float ns_direction(float g, float m, const NsUpdate& s) {
  return s.nesterov ? fmaf(s.beta, m - g, g) : m;
}

// EACH consecutive elements of a gradient; EACH 1: any address
template <typename T, int EACH>
__device__ __forceinline__ void ns_load(const void* g, int64_t at, float (&v)[EACH]) {
  const T* p = static_cast<const T*>(g) + at;
  if constexpr (EACH == 1) {
    v[0] = Pack<T>::load1(p);
  } else if constexpr (sizeof(T) == 2) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
    v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    Pack<float>::load(p, v);
  }
}
template <int EACH>
__device__ __forceinline__ void ns_load_f32(const float* p, float (&v)[EACH]) {
  if constexpr (EACH == 1) v[0] = *p;
  else Pack<float>::load(p, v);
}

// Sum of squares of numbers of any size: those whose square is well inside 32 bits are added in 32 bits, a few dozen at a time, the
// others, and NaN, in 64 (which alone would take twice the time of reading bf16 gradients: 124 us for 55 million).
struct NsSquares {
  double sum = 0.0;
  float some = 0.0f;
  __device__ __forceinline__ void add(float u) {
    const float t = u * u;
    if (t > 0x1p-100f && t < 0x1p100f) some += t;
    else if (u != 0.0f) sum = fma((double)u, (double)u, sum);
  }
  __device__ __forceinline__ void flush() {
    sum += (double)some;
    some = 0.0f;
  }
};

// m <- m + (1 - beta) (g - m); the squares of the update's elements, summed by every block.  EACH elements to an access:
// 4 where all addresses are aligned to that, else 1; four or eight accesses of each array under way in a thread.
// HAS: there is a momentum.
template <typename T, int EACH, bool HAS>
__global__ void __launch_bounds__(NS_THREADS, 4) ns_momentum_kernel(const NsMatrices mats, int64_t elements, NsUpdate s, double* norms) {
  __shared__ double part[NS_THREADS / 32];
  ag_pdl_wait();
  ag_pdl_trigger();
  const void* g = mats.g[blockIdx.y];
  float* m = HAS ? mats.m[blockIdx.y] : nullptr;
  NsSquares squares;
  auto element = [&](float gi, float& mi) {
    float u = gi * s.grad_scale;
    if (HAS) {
      mi = fmaf(1.0f - s.beta, u - mi, mi);
      u = ns_direction(u, mi, s);
    }
    squares.add(u);
  };
  constexpr int AHEAD = EACH == 1 || !HAS ? 8 : 4;
  const int64_t stride = (int64_t)gridDim.x * NS_THREADS, packets = elements / EACH;
  int64_t i = (int64_t)blockIdx.x * NS_THREADS + threadIdx.x;
  auto run = [&](auto count) {
    constexpr int N = decltype(count)::value;
    float gv[N][EACH], mv[N][EACH];
#pragma unroll
    for (int k = 0; k < N; ++k) ns_load<T, EACH>(g, (i + k * stride) * EACH, gv[k]);
    if (HAS) {
#pragma unroll
      for (int k = 0; k < N; ++k) ns_load_f32<EACH>(m + (i + k * stride) * EACH, mv[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) element(gv[k][e], mv[k][e]);
      if (HAS) {
        if constexpr (EACH == 4) Pack<float>::store(m + (i + k * stride) * EACH, mv[k]);
        else m[i + k * stride] = mv[k][0];
      }
    }
    squares.flush();
  };
  for (; i + (AHEAD - 1) * stride < packets; i += AHEAD * stride) run(std::integral_constant<int, AHEAD>());
  for (; i < packets; i += stride) run(std::integral_constant<int, 1>());
  if (EACH > 1 && blockIdx.x == 0 && threadIdx.x < elements % EACH) {
    const int64_t at = elements - 1 - threadIdx.x;
    float gi[1], mi = m ? m[at] : 0.0f;
    ns_load<T, 1>(g, at, gi);
    element(gi[0], mi);
    if (m) m[at] = mi;
    squares.flush();
  }
  double sum = squares.sum;
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NS_THREADS / 32; ++w) sum += part[w];
    norms[blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = sum;
  }
}

// What is kept between products: x * 2^12 as one or two 16-bit floats (`hi`, and what hi leaves), in planes of padded rows.
// Singular values stay near 1 or below, so that no element of X, A or Q is beyond a few units (15.99 is the largest: a limit on what
// coefficients of the caller's may do, A = X X^T + h I being the first to reach it), and the smallest that
// keep all bits are 2^-26 (one word) or next to nothing (two): elements err by at most 2^-37 or 2^-38 beside that.
constexpr float NS_SCALE = 4096.0f;

struct NsPlane {
  __half *hi, *lo;  // lo null: one word
};

// What an element of the update is multiplied by: NS_SCALE over its norm, whose square is `sum`; NaN, and so a matrix of NaN after any
// number of steps, where the norm is infinite or none (32-bit numbers have squares that 64 bits can add up)
__device__ __forceinline__ double ns_factor(double sum, float eps) {
  const double norm = sqrt(sum), none = norm - norm;
  return none != 0.0 ? none : (double)NS_SCALE / (norm > eps ? norm : (double)eps);
}

// X = u / max(|u|, eps) in padded rows, transposed where the matrix is tall: tiles of 64 x 64, EACH elements to an access of the matrix
template <typename T, int EACH>
__global__ void __launch_bounds__(NS_THREADS) ns_start_kernel(const NsMatrices mats, NsPlan t, NsUpdate s, float eps, const double* norms,
                                                              int norm_blocks, NsPlane X) {
  __shared__ float tile[64][65];
  __shared__ double factor;
  ag_pdl_wait();
  ag_pdl_trigger();
  const void* g = mats.g[blockIdx.z];
  const float* m = mats.m[blockIdx.z];
  const bool tall = t.rows > t.cols;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of X
  constexpr int ACROSS = 64 / EACH, DOWN = NS_THREADS / ACROSS, TIMES = 64 / DOWN;
  const int tx = threadIdx.x % ACROSS * EACH, ty = threadIdx.x / ACROSS;
  float u[TIMES][EACH], mv[TIMES][EACH];
  const int row = (tall ? c0 : r0) + ty, col = (tall ? r0 : c0) + tx;  // of the matrix: rows DOWN apart
  const int64_t at = (int64_t)row * t.cols + col;
#pragma unroll
  for (int k = 0; k < TIMES; ++k) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) u[k][e] = mv[k][e] = 0.0f;
    if (row + DOWN * k < t.rows && col < t.cols) {
      ns_load<T, EACH>(g, at + (int64_t)(DOWN * k) * t.cols, u[k]);
      if (m) ns_load_f32<EACH>(m + at + (int64_t)(DOWN * k) * t.cols, mv[k]);
    }
  }
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < norm_blocks; i += 32) sum += norms[blockIdx.z * NS_NORM_BLOCKS + i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) factor = ns_factor(sum, eps);
  }
  __syncthreads();
  const double by = factor;
#pragma unroll
  for (int k = 0; k < TIMES; ++k)
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      float v = u[k][e] * s.grad_scale;
      if (m) v = ns_direction(v, mv[k][e], s);
      tile[ty + DOWN * k][tx + e] = (float)(v * by);
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
// the contraction (hi lo, lo hi, hi hi) where there are two.  What one thread issues between MMAs takes their time where they do not
// queue up, a tcgen05.commit above all (ten of them to 24 MMAs: 171 cycles for each of 128): slots hold 128 elements, a commit
// arrives in both CTAs of a pair, and where a chain is a slot, the commit that hands its sum over frees it too.
// A step X <- (a I + b G + c G G) X, G = X X^T, is a square once it is completed: with h = b / 2 c
//   GRAM:  A = G + h I                    both operands K-major
//   POLY:  Q = (a - h h c) I + c A A      both symmetric
//   NEXT:  X' = Q X                       symmetric, X MN-major
// so that no product needs anything beside its operands, and every epilogue is a factor and a number on the diagonal.  Where c is 0,
// GRAM writes Q = a I + b G itself.
// A and Q are symmetric (polynomials of one matrix commute): only the 256 x 256 blocks on and above the diagonal are computed and
// stored, by tiles of either size.  A tile of an operand that lies below is read as the transpose of the one above, as an MN-major
// tile: which of the two is a matter of the map, the descriptor and a bit of the instruction.
// Few tiles with a long contraction (X X^T of a wide matrix) are shared by a cluster of up to 8 CTAs, each with a part of the contraction (ZSPLIT):
// they send their sums to the CTA that owns the rows, which adds them in the order of the ranks.
enum { NS_GRAM, NS_POLY, NS_NEXT };
constexpr bool ns_symmetric(int kind) { return kind <= NS_POLY; }

constexpr int NS_EPI_WARPS = 8;
constexpr int NS_TC_THREADS = 128 + 32 * NS_EPI_WARPS;
constexpr int NS_MAX_SLOTS = 4;
constexpr int NS_SMEM_LIMIT = 227 * 1024;
constexpr int NS_STAGING = NS_EPI_WARPS * 4096;  // per epilogue warp: 32 rows of 64 bytes, twice, on their way to memory
constexpr int NS_SMEM_FIXED = 1024 + NS_STAGING + 512;
// The tensor core truncates a sum at every addition, by an amount that grows with it.  So chains are short, 128 elements
// (single words: 8192, their operands are off by more), the epilogue adds them in registers, and the products with a low part come
// first, whose sum is 2^-11 of the whole.  What truncation takes of a sum on average, NS_LOSS of it at each of the later additions of
// 16 elements, is put back by the factor of the epilogue.  Error of the factor of 333 x 1001 with 0, 4e-8, 7e-8 and 1e-7: 3.8e-6, 1.9e-6, 2.9e-6, 4.7e-6
// (plain fp32 products: 2.6e-6); without it, low parts first in every step, chains of 1, 2 and 4 steps: 2.6e-6, 5.7e-6, 8.7e-6.
constexpr int NS_CHAIN_PAIRS = 1, NS_CHAIN_SINGLE = 64;  // in double steps of 128 elements
constexpr double NS_LOSS = 4.6e-8;

// Tensor maps of a plane: tiles with the contraction along its rows (k), and along its columns (mn)
struct NsMaps {
  CUtensorMap k_hi, k_lo, mn_hi, mn_lo;
};

struct NsGemm {
  NsMaps l, r;
  CUtensorMap d_hi, d_lo;  // of the result: boxes of 32 rows x 32 columns
  int batch, tiles_m, tiles_n, tiles;  // tiles of a matrix; symmetric: those on and above the diagonal
  int k_iters, chain, k_real;  // steps of 64 elements of the contraction; double steps to a chain; elements that are not padding
  int slots;                   // of operand tiles of a double step
  int M, N;                // rows and columns of a matrix that are stored (padded)
  int two;                 // the result has a low part
  int cluster, k_each;     // ZSPLIT: CTAs to a tile, steps of each (even)
  NsPlane D;               // and where the result goes
  float diag, mul;
  int expire;              // the issuer gives up at once
  int* status;
};

struct NsTile {
  int mat, tm, tn;
};

template <int KIND, bool PAIR>
__device__ __forceinline__ bool ns_tile(const NsGemm& p, int unit, int units, int step, NsTile& t) {
  int i = unit + step * units;
  if (i >= p.batch * p.tiles) return false;
  t.mat = i / p.tiles;
  i -= t.mat * p.tiles;
  if (ns_symmetric(KIND) && PAIR) {  // columns of tiles, the diagonal last in each
    int n = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while (n * (n + 1) / 2 > i) --n;
    while ((n + 1) * (n + 2) / 2 <= i) ++n;
    t.tn = n;
    t.tm = i - n * (n + 1) / 2;
  } else if (ns_symmetric(KIND)) {   // two columns of 128-row tiles to a block: 2 j + 2 tiles in each
    int j = (int)((sqrtf(2.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while (2 * j * (j + 1) > i) --j;
    while (2 * (j + 1) * (j + 2) <= i) ++j;
    i -= 2 * j * (j + 1);
    const int rows = min(2 * j + 2, p.tiles_m);
    t.tn = 2 * j + i / rows;
    t.tm = i - i / rows * rows;
  } else {
    t.tn = i / p.tiles_m;
    t.tm = i - t.tn * p.tiles_m;
  }
  return true;
}

// 32 x 32 words of 16 bits from a warp's buffer (64 bytes a row, swizzled as tc_stage_at has it) to memory, as a bulk store
__device__ __forceinline__ void ns_tma_store(const CUtensorMap* tm, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tm), "r"(ag_smem_u32(src)), "r"(x), "r"(y)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// all but the last `N` stores of this thread have read their buffers
template <int N>
__device__ __forceinline__ void ns_stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

// an arrival at the barrier of both CTAs of a pair once the MMAs so far are done
__device__ __forceinline__ void ns_commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(ag_smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}

// The MMAs of a step of 64 elements: products with a low part, or those of the high parts
template <bool LOW, bool PAIR>
__device__ __forceinline__ void ns_step_mmas(uint32_t acc, uint32_t lh, uint32_t ll, uint32_t l_step, uint32_t rh, uint32_t rl,
                                             uint32_t r_step, uint32_t idesc, uint32_t not_first) {
  constexpr uint32_t hi = TcDesc::hi;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t lo = k * l_step, ro = k * r_step, r0 = LOW ? rl : rh;
    if (k == 0) tc_mma<2, PAIR>(acc, lh, hi, r0, hi, idesc, not_first);
    else tc_mma<1, PAIR>(acc, lh + lo, hi, r0 + ro, hi, idesc, 1u);
    if (LOW) tc_mma<1, PAIR>(acc, ll + lo, hi, rh + ro, hi, idesc, 1u);
  }
}

// into the shared memory of a CTA of the cluster
__device__ __forceinline__ void ns_st_cluster(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void ns_st_cluster(uint32_t addr, uint32_t x, uint32_t y) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void ns_st_cluster(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

template <int KIND, bool SPLIT, bool PAIR, int BN, bool ZSPLIT = false>
__global__ void __launch_bounds__(NS_TC_THREADS, 1) ns_gemm_kernel(const __grid_constant__ NsGemm p) {
  static_assert(!ZSPLIT || (KIND == NS_GRAM && !PAIR), "sums of a cluster: X X^T on single CTAs");
  extern __shared__ unsigned char ns_smem_raw[];
  constexpr bool R_MN = !ns_symmetric(KIND);          // the right operand is stored with its columns contiguous
  constexpr uint32_t A_BYTES = TC_BM * 128, BN_CTA = PAIR ? BN / 2 : BN, B_BYTES = BN_CTA * 128;
  constexpr uint32_t STEP = A_BYTES + B_BYTES;        // both operands' tiles of 64 elements of the contraction
  constexpr uint32_t SLOT = 2 * STEP;
  constexpr int BM = PAIR ? 2 * TC_BM : TC_BM;
  constexpr uint32_t COLUMNS = 2 * BN;                // of tensor memory: two accumulators
  constexpr int CHUNKS = BN / 64;                     // 32-column chunks of an epilogue warp
  constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  static_assert(!ns_symmetric(KIND) || BM == BN, "tiles on the diagonal are square");
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ns_smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* lows = tiles + (size_t)p.slots * SLOT;  // SPLIT: two slots of a step's low parts
  unsigned char* staging = lows + (SPLIT ? SLOT : 0);
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + NS_STAGING);
  uint64_t* empty = full + NS_MAX_SLOTS;              // not SPLIT: a chain's slot is free when its sum is complete
  uint64_t* low_full = empty + NS_MAX_SLOTS;
  uint64_t* low_empty = low_full + 2;
  uint64_t* acc_full = low_empty + 2;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? tc_cluster_rank() : 0u;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : ZSPLIT ? (int)blockIdx.x / p.cluster : (int)blockIdx.x;
  const int units = PAIR ? (int)(gridDim.x >> 1) : ZSPLIT ? (int)gridDim.x / p.cluster : (int)gridDim.x;  // ZSPLIT: one tile each
  const int zrank = ZSPLIT ? (int)blockIdx.x - unit * p.cluster : 0;
  const int k_first = ZSPLIT ? zrank * p.k_each : 0, k_last = ZSPLIT ? min(p.k_iters, k_first + p.k_each) : p.k_iters;
  const int row_off = PAIR ? (int)rank * TC_BM : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.slots; ++s) {
      ag_mbar_init(&full[s], 1);
      ag_mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      ag_mbar_init(&low_full[b], 1);
      ag_mbar_init(&low_empty[b], 1);
      ag_mbar_init(&acc_full[b], 1);
      ag_mbar_init(&acc_empty[b], PAIR ? 2 * NS_EPI_WARPS : NS_EPI_WARPS);
    }
    *abort_flag = 0;
    ag_fence_mbar_init();
  }
  if (PAIR || ZSPLIT) tc_cluster_sync(); else __syncthreads();
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
  // a wait ran out: all roles give up, those of the pair's other CTA too
  auto give_up = [&]() {
    expired = true;
    *abort_flag = 1;
    if (PAIR) tc_st_cluster(tc_map_to_cta(ag_smem_u32(tmem_slot + 1), rank ^ 1u), 1);
  };
  ag_pdl_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      uint32_t slot = 0, phase = 0, low = 0, low_phase = 0;
      NsTile t;
      for (int step = 0; !expired && ns_tile<KIND, PAIR>(p, unit, units, step, t); ++step) {
        const int l_at = t.tm * BM + row_off, r_at = t.tn * BN + (int)rank * (PAIR ? (int)BN_CTA : 0);
        for (int k = k_first; k < k_last && !expired; k += 2) {
          const int n = k_last - k < 2 ? 1 : 2, blk = k * TC_BK / 256;  // blk: block of the contraction
          const bool l_mn = KIND != NS_GRAM && t.tm * BM / 256 > blk, r_mn = R_MN || (KIND == NS_POLY && t.tn * BN / 256 > blk);
          auto load = [&](const CUtensorMap& k_map, const CUtensorMap& mn_map, uint64_t* bar, unsigned char* dst, int kx, int row, bool mn) {
            const uint32_t at = PAIR ? tc_map_to_cta(ag_smem_u32(bar), 0u) : 0u;  // the leader counts the bytes of both
            if (!mn) {
              if (PAIR) tc_tma_load_2d_pair(&k_map, dst, at, kx, t.mat * p.M + row);
              else tc_tma_load_2d(&k_map, dst, bar, kx, t.mat * p.M + row);
            } else {
              if (PAIR) tc_tma_load_3d_pair(&mn_map, dst, at, 0, t.mat * p.M + kx, row / TC_MN_GROUP);
              else tc_tma_load_3d(&mn_map, dst, bar, 0, t.mat * p.M + kx, row / TC_MN_GROUP);
            }
          };
          if (!tc_wait(SPLIT ? &acc_full[slot] : &empty[slot], phase ^ 1u, abort_flag)) {
            give_up();
            break;
          }
          unsigned char* s = tiles + (size_t)slot * SLOT;
          if (rank == 0) ag_mbar_expect_tx(&full[slot], (PAIR ? 2u : 1u) * n * STEP);
          for (int j = 0; j < n; ++j, s += STEP) {
            const int kx = (k + j) * TC_BK;
            load(p.l.k_hi, p.l.mn_hi, &full[slot], s, kx, l_at, l_mn);
            load(p.r.k_hi, p.r.mn_hi, &full[slot], s + A_BYTES, kx, r_at, r_mn);
            if (SPLIT) {
              if (!tc_wait(&low_empty[low], low_phase ^ 1u, abort_flag)) {
                give_up();
                break;
              }
              unsigned char* d = lows + (size_t)low * STEP;
              if (rank == 0) ag_mbar_expect_tx(&low_full[low], (PAIR ? 2u : 1u) * STEP);
              load(p.l.k_lo, p.l.mn_lo, &low_full[low], d, kx, l_at, l_mn);
              load(p.r.k_lo, p.r.mn_lo, &low_full[low], d + A_BYTES, kx, r_at, r_mn);
              low ^= 1u;
              low_phase ^= low ^ 1u;
            }
          }
          if (++slot == (uint32_t)p.slots) slot = 0, phase ^= 1u;
        }
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------------------------------------------------------- MMA issuer (pair: the leader only)
      uint32_t slot = 0, phase = 0, low = 0, low_phase = 0, acc_par = 0;
      int buf = 0;
      // descriptors take the address within the CTA: higher bits may name the CTA of the cluster
      const uint32_t tiles_u = (ag_smem_u32(tiles) & 0x3FFFFu) >> 4, lows_u = (ag_smem_u32(lows) & 0x3FFFFu) >> 4;
      TcDesc dk, dmn;
      dk.init(0);
      dmn.init(1);
      auto arrive = [&](uint64_t* bar) {  // when the MMAs so far are done (pair: in both CTAs)
        if (PAIR) ns_commit_both(bar);
        else tc_commit(bar);
      };
      if (p.expire) give_up();
      NsTile t;
      for (int step = 0; !expired && ns_tile<KIND, PAIR>(p, unit, units, step, t); ++step) {
        uint32_t tacc = 0, more = 0;
        int left = 0;  // double steps of the chain
        for (int k = k_first; k < k_last; k += 2) {
          const int n = k_last - k < 2 ? 1 : 2, blk = k * TC_BK / 256;
          const bool l_mn = KIND != NS_GRAM && t.tm * BM / 256 > blk, r_mn = R_MN || (KIND == NS_POLY && t.tn * BN / 256 > blk);
          const uint32_t idesc = IDESC | (l_mn ? 1u << 15 : 0u) | (r_mn ? 1u << 16 : 0u);
          const uint32_t l_step = l_mn ? dmn.step : dk.step, r_step = r_mn ? dmn.step : dk.step;
          const uint32_t l_const = l_mn ? dmn.lo_const : dk.lo_const, r_const = (A_BYTES >> 4) + (r_mn ? dmn.lo_const : dk.lo_const);
          // the accumulator last: it is what is late
          if (!tc_wait(&full[slot], phase, abort_flag) || (SPLIT && !tc_wait(&low_full[low], low_phase, abort_flag)) ||
              (left == 0 && !tc_wait(&acc_empty[buf], ((acc_par >> buf) & 1u) ^ 1u, abort_flag))) {
            give_up();
            break;
          }
          tc_fence_after();
          if (left == 0) {
            acc_par ^= 1u << buf;
            tacc = tmem_base + (uint32_t)buf * BN;
            left = p.chain;
            more = 0u;
          }
          const uint32_t hs = tiles_u + slot * (SLOT >> 4);
          if (SPLIT) {
            for (int j = 0; j < n; ++j) {
              if (j > 0) {
                if (!tc_wait(&low_full[low], low_phase, abort_flag)) {
                  give_up();
                  break;
                }
                tc_fence_after();
              }
              const uint32_t h = hs + j * (STEP >> 4), l = lows_u + low * (STEP >> 4);
              ns_step_mmas<true, PAIR>(tacc, h + l_const, l + l_const, l_step, h + r_const, l + r_const, r_step, idesc, more);
              more = 1u;
              arrive(&low_empty[low]);
              low ^= 1u;
              low_phase ^= low ^ 1u;
            }
            if (expired) break;
          }
          for (int j = 0; j < n; ++j) {
            const uint32_t h = hs + j * (STEP >> 4);
            ns_step_mmas<false, PAIR>(tacc, h + l_const, 0, l_step, h + r_const, 0, r_step, idesc, more);
            more = 1u;
          }
          if (!SPLIT) arrive(&empty[slot]);
          if (++slot == (uint32_t)p.slots) slot = 0, phase ^= 1u;
          if (--left == 0 || k + 2 >= k_last) {
            arrive(&acc_full[buf]);
            buf ^= 1;
            left = 0;
          }
        }
      }
    }
    if constexpr (ZSPLIT) {
      __syncwarp();
      tc_cluster_sync();
      tc_cluster_sync();
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 4..11)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3, slice = (warp - 4) >> 2;
    unsigned char* stg = staging + (warp - 4) * 4096;
    uint32_t full_par = 0;
    int buf = 0, half = 0;
    NsTile t;
    for (int step = 0; !expired && ns_tile<KIND, PAIR>(p, unit, units, step, t); ++step) {
      const int row0 = t.tm * BM + row_off + quarter * 32, col0 = t.tn * BN + slice * (BN / 2);
      const uint32_t toff = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slice * (BN / 2));
      const bool rows_in = row0 < p.M;  // padded sizes are multiples of 32
      // one word of each of the lane's 32 columns: through the half of the buffer that was stored from before the last
      auto put = [&](const CUtensorMap& map, const uint32_t (&w)[16], int col) {
        if (lane == 0) ns_stores_read<1>();
        __syncwarp();
        unsigned char* s = stg + half * 2048;
        half ^= 1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(tc_stage_at(s, lane, j)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        ag_fence_proxy_async();
        __syncwarp();
        if (lane == 0) ns_tma_store(&map, s, col, t.mat * p.M + row0);
      };
      auto chunk = [&](const int c, float (&v)[32]) {
        const int col = col0 + c * 32;
        if (!rows_in || col >= p.N) return;
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= p.mul;
        if (ns_symmetric(KIND) && row0 == col) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (j == lane) v[j] += p.diag;
        }
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) split_f16x2(v[2 * k], v[2 * k + 1], hi[k], lo[k]);
        put(p.d_hi, hi, col);
        if (SPLIT || p.two) put(p.d_lo, lo, col);
      };
      auto wait_full = [&]() {
        // one answer for the warp: what follows is for all lanes together
        if (!__all_sync(0xffffffffu, tc_wait(&acc_full[buf], (full_par >> buf) & 1u, abort_flag))) {
          give_up();
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
      if (ZSPLIT) {  // a part may be empty
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] = 0.0f;
      }
      bool gone = false;
      for (int k = k_first; k < k_last; k += 2 * p.chain) {
        if (!wait_full()) {
          gone = true;
          break;
        }
        const uint32_t from = toff + (uint32_t)buf * BN;
        if (k == k_first) {
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
      if constexpr (ZSPLIT) {
        // The sums go to the CTAs that own the rows, where the operands were (all CTAs meet twice, whatever became of them)
        const int own = TC_BM / p.cluster, r = quarter * 32 + lane;
        tc_cluster_sync();
        const uint32_t to = tc_map_to_cta(ag_smem_u32(tiles), r / own) + (uint32_t)(zrank * own + r % own) * 512u;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            ns_st_cluster(to + ((((uint32_t)(slice * (BN / 8) + c * 8 + j)) ^ ((uint32_t)r & 7u)) << 4),
                          make_float4(acc[c][4 * j], acc[c][4 * j + 1], acc[c][4 * j + 2], acc[c][4 * j + 3]));
        tc_cluster_sync();
        for (int i = threadIdx.x - 128; i < own * 32; i += 32 * NS_EPI_WARPS) {
          const int q = i & 31, at = zrank * own + (i >> 5), row = t.tm * BM + at, col = t.tn * BN + q * 4;
          if (row >= p.M || col >= p.N) continue;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int s = 0; s < p.cluster; ++s) {
            const float4 x = *reinterpret_cast<const float4*>(tiles + (uint32_t)(s * own + (i >> 5)) * 512u + ((uint32_t)(q ^ (at & 7)) << 4));
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
          }
          const int d = row - col;  // the diagonal's place among the four
          uint32_t hi[2], lo[2];
          split_f16x2(v.x * p.mul + (d == 0 ? p.diag : 0.f), v.y * p.mul + (d == 1 ? p.diag : 0.f), hi[0], lo[0]);
          split_f16x2(v.z * p.mul + (d == 2 ? p.diag : 0.f), v.w * p.mul + (d == 3 ? p.diag : 0.f), hi[1], lo[1]);
          const int64_t out = ((int64_t)t.mat * p.M + row) * p.M + col;
          *reinterpret_cast<uint2*>(p.D.hi + out) = make_uint2(hi[0], hi[1]);
          if (SPLIT || p.two) *reinterpret_cast<uint2*>(p.D.lo + out) = make_uint2(lo[0], lo[1]);
        }
        break;
      }
      if (gone) break;
      // one copy of the code for all chunks, which move up to acc[0] one after the other: what every tile runs through once is
      // fetched anew each time
#pragma unroll 1
      for (int c = 0; c < CHUNKS; ++c) {
        chunk(c, acc[0]);
#pragma unroll
        for (int k = 1; k < CHUNKS; ++k)
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[k - 1][j] = acc[k][j];
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  if (expired && lane == 0) atomicOr(p.status, AG_STATUS_WAIT_EXPIRED);
  tc_fence_before();
  tc_meet<PAIR || ZSPLIT>();
  if (warp == 1) {
    tc_drain(abort_flag);
    tc_fence_after();
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLUMNS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(COLUMNS) : "memory");
  }
}

// p <- keep p - by X (NS_STEP), or X in fp32 (NS_F32) or bf16 (NS_BF16)
enum { NS_STEP, NS_F32, NS_BF16 };
template <int EACH>
__device__ __forceinline__ void ns_put(float* p, int64_t at, float (&v)[EACH], const float (&old)[EACH], float keep, float by, int kind) {
  if (kind == NS_BF16) {
    __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(p) + at;
    if constexpr (EACH == 4) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(q) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      *q = __float2bfloat16_rn(v[0]);
    }
    return;
  }
  if (kind == NS_STEP) {
#pragma unroll
    for (int e = 0; e < EACH; ++e) v[e] = fmaf(-by, v[e], keep * old[e]);
  }
  if constexpr (EACH == 4) Pack<float>::store(p + at, v);
  else p[at] = v[0];
}

// The factor goes where it belongs: tiles of 64 x 64 of X, as in ns_start_kernel
template <int EACH>
__global__ void __launch_bounds__(NS_THREADS) ns_finish_kernel(const NsMatrices mats, NsPlan t, NsPlane X, float keep, float by, int kind) {
  __shared__ float tile[64][65];
  ag_pdl_wait();
  ag_pdl_trigger();
  const bool tall = t.rows > t.cols;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of X
  constexpr int ACROSS = 64 / EACH, DOWN = NS_THREADS / ACROSS, TIMES = 64 / DOWN;
  const int tx = threadIdx.x % ACROSS * EACH, ty = threadIdx.x / ACROSS;
  const int row = (tall ? c0 : r0) + ty, col = (tall ? r0 : c0) + tx;  // of the matrix: rows DOWN apart
  const int64_t at = (int64_t)row * t.cols + col, x = (int64_t)blockIdx.z * t.mp * t.np;
  float* p = mats.p[blockIdx.z];
  float old[TIMES][EACH];
#pragma unroll
  for (int k = 0; k < TIMES; ++k) {
    if (kind == NS_STEP && row + DOWN * k < t.rows && col < t.cols) ns_load_f32<EACH>(p + at + (int64_t)(DOWN * k) * t.cols, old[k]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * NS_THREADS, r = i >> 3, c = (i & 7) * 8;
    const int64_t from = x + (int64_t)(r0 + r) * t.np + c0 + c;
    const uint4 hi = *reinterpret_cast<const uint4*>(X.hi + from);
    uint4 lo = make_uint4(0u, 0u, 0u, 0u);
    if (X.lo) lo = *reinterpret_cast<const uint4*>(X.lo + from);
    const uint32_t hw[4] = {hi.x, hi.y, hi.z, hi.w}, lw[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&hw[k])), v = __half22float2(*reinterpret_cast<const __half2*>(&lw[k]));
      const float a = (u.x + v.x) * (1.0f / NS_SCALE), b = (u.y + v.y) * (1.0f / NS_SCALE);
      tile[tall ? c + 2 * k : r][tall ? r : c + 2 * k] = a;
      tile[tall ? c + 2 * k + 1 : r][tall ? r : c + 2 * k + 1] = b;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < TIMES; ++k) {
    if (row + DOWN * k >= t.rows || col >= t.cols) continue;
    float v[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) v[e] = tile[ty + DOWN * k][tx + e];
    ns_put<EACH>(p, at + (int64_t)(DOWN * k) * t.cols, v, old[k], keep, by, kind);
  }
}

// ---------------------------------------------------------------------------- small matrices
// Matrices of up to 128 rows (their shorter side) in one launch, from gradient to parameter: a cluster of CTAs per matrix, each with a
// slice of 64 to 320 columns of X in shared memory, as pairs in the layout that serves as a K-major operand (X X^T) and as an MN-major
// one (Q X) alike.  A step is three products of 128 rows:
//   G = X X^T of the slice into tensor memory; each CTA of the cluster owns 128 / S rows of the sum: it gets the others' parts of them
//   through distributed shared memory, adds them in the order of the ranks, and sends A = G + h I to all;
//   Q = (a - h h c) I + c A A and X <- Q X by every CTA for itself.
// What bounds it is latency: 15 dependent products of a few thousand cycles, where the launches of the general path cost 7 us each.
constexpr int NS_SMALL_THREADS = 512, NS_SMALL_M = 128, NS_SMALL_GROUPS = 5, NS_SMALL_APART = 3, NS_SMALL_CLUSTER = 16;
constexpr uint32_t NS_GROUP_BYTES = NS_SMALL_M * 128;       // 64 columns of one plane
constexpr uint32_t NS_SQUARE_BYTES = 4 * NS_GROUP_BYTES;    // 128 x 128: two planes, or 32-bit sums

struct NsSmall {
  NsMatrices mats;
  NsUpdate s;
  int rows, cols, m, n, groups, cluster, steps, out_kind;
  float eps, keep, by, loss_gram, loss_square;
  float co[3 * NS_MAX_STEPS];
  uint32_t wait_limit;  // polls of a wait for products
  int* status;
};

// generic writes before it, of this CTA's memory or another's, and products after it
__device__ __forceinline__ void ns_fence_proxy() { asm volatile("fence.proxy.async;" ::: "memory"); }

// Byte of (row, byte of the row) in a group of rows of 128 bytes, swizzled as the products read it
__device__ __forceinline__ uint32_t ns_swizzled(int row, uint32_t byte) { return (uint32_t)row * 128u + (byte ^ (((uint32_t)row & 7u) << 4)); }

template <typename T, bool SPLIT>
__global__ void __launch_bounds__(NS_SMALL_THREADS, 1) ns_small_kernel(const __grid_constant__ NsSmall p) {
  extern __shared__ unsigned char ns_smem_raw[];
  unsigned char* X = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ns_smem_raw) + 1023) & ~(uintptr_t)1023);
  const int G = p.groups, S = p.cluster, W = G * 64;
  const uint32_t plane = (uint32_t)G * NS_GROUP_BYTES;                 // X: high words, low words; at the end its 32-bit values
  unsigned char* AQ = X + 2 * plane;                                   // A or Q: high words, low words
  const bool apart = S > 1 && G <= NS_SMALL_APART;                     // there is room for partial sums beside it
  unsigned char* parts = apart ? AQ + NS_SQUARE_BYTES : AQ;
  double* norms = reinterpret_cast<double*>(parts + NS_SQUARE_BYTES);  // of every rank
  uint64_t* bar = reinterpret_cast<uint64_t*>(norms + NS_SMALL_CLUSTER);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  double* part = reinterpret_cast<double*>(tmem_slot + 2);             // of every warp
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int mat = blockIdx.x / S, rank = blockIdx.x - mat * S;
  auto cluster_sync = [&]() {
    if (S > 1) tc_cluster_sync(); else __syncthreads();
  };
  if (tid == 0) {
    ag_mbar_init(bar, 1);
    *abort_flag = 0;
    ag_fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ag_smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync();  // all CTAs are there, too, before anything goes to their memory
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ag_pdl_wait();
  ag_pdl_trigger();

  // ---- the momentum and the norm; then X.  Elements in the order of memory: a slice is whole rows of a tall matrix, pieces of the
  // rows of another
  const bool tall = p.rows > p.cols;
  const int first = rank * W, width = max(0, min(W, p.n - first)), inner = tall ? p.m : width, count = p.m * width;
  auto place = [&](int i, int& r, int& c) {  // row and column of the slice of X
    const int q = i / inner, k = i - q * inner;
    r = tall ? k : q;
    c = tall ? q : k;
    return tall ? (int64_t)(first + q) * p.cols + k : (int64_t)q * p.cols + first + k;
  };
  const void* g = p.mats.g[mat];
  float* mom = p.mats.m[mat];
  constexpr int AHEAD = 8;
  NsSquares squares;
  for (int i = tid; i < count; i += NS_SMALL_THREADS * AHEAD) {
    float gv[AHEAD][1], mv[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      gv[k][0] = mv[k] = 0.0f;
      if (j < count) {
        int r, c;
        const int64_t at = place(j, r, c);
        ns_load<T, 1>(g, at, gv[k]);
        if (mom) mv[k] = mom[at];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      if (j >= count) continue;
      float u = gv[k][0] * p.s.grad_scale;
      if (mom) {
        int r, c;
        const float v = fmaf(1.0f - p.s.beta, u - mv[k], mv[k]);
        mom[place(j, r, c)] = v;
        u = ns_direction(u, v, p.s);
      }
      squares.add(u);
    }
    squares.flush();
  }
  double sum = squares.sum;
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) part[warp] = sum;
  // padding of X is zero, and rows and columns of the square that are not written
  for (uint32_t i = tid; i < (2 * plane + NS_SQUARE_BYTES) / 16; i += NS_SMALL_THREADS) reinterpret_cast<uint4*>(X)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  if (tid < S) {
    sum = 0.0;
    for (int w = 0; w < NS_SMALL_THREADS / 32; ++w) sum += part[w];
    if (S > 1) ns_st_cluster(tc_map_to_cta(ag_smem_u32(norms + rank), tid), sum);
    else norms[0] = sum;
  }
  cluster_sync();
  sum = 0.0;
  for (int r = 0; r < S; ++r) sum += norms[r];
  const double by = ns_factor(sum, p.eps);
  for (int i = tid; i < count; i += NS_SMALL_THREADS * AHEAD) {
    float gv[AHEAD][1], mv[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      gv[k][0] = mv[k] = 0.0f;
      if (j < count) {
        int r, c;
        const int64_t at = place(j, r, c);
        ns_load<T, 1>(g, at, gv[k]);
        if (mom) mv[k] = mom[at];
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      if (j >= count) continue;
      int r, c;
      place(j, r, c);
      float u = gv[k][0] * p.s.grad_scale;
      if (mom) u = ns_direction(u, mv[k], p.s);
      u = (float)(u * by);
      const __half h = __float2half_rn(u);
      const uint32_t at = (uint32_t)(c >> 6) * NS_GROUP_BYTES + ns_swizzled(r, (uint32_t)(c & 63) * 2u);
      *reinterpret_cast<__half*>(X + at) = h;
      if (SPLIT || p.steps == 0) *reinterpret_cast<__half*>(X + plane + at) = __float2half_rn(u - __half2float(h));
    }
  }
  ns_fence_proxy();
  // without steps nothing else stands between what a CTA reads and what another may write in its place (narrower words)
  if (p.steps == 0) cluster_sync();
  __syncthreads();

  // ---- the steps
  uint32_t phase = 0;
  bool expired = false;
  auto products_done = [&]() {
    if (!tc_wait(bar, phase, abort_flag, p.wait_limit)) expired = true;  // the steps go on without products, all CTAs meet at the same barriers
    __syncwarp();
    phase ^= 1u;
    tc_fence_after();
  };
  constexpr uint32_t HI = TcDesc::hi, K_CONST = 1u << 16, MN_CONST = (NS_GROUP_BYTES >> 4) << 16;
  auto idesc = [](uint32_t n, bool mn) { return (1u << 4) | (mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((NS_SMALL_M >> 4) << 24); };
  // D (at column `d` of tensor memory) = B B^T over `steps16` steps of a K-major buffer: the products with a low part first
  auto gram = [&](uint32_t d, uint32_t hi, uint32_t lo, int steps16, uint32_t n) {
    const uint32_t form = idesc(n, false);
    uint32_t more = 0;
    if (SPLIT)
      for (int k = 0; k < steps16; ++k) {
        const uint32_t at = (uint32_t)(k >> 2) * (NS_GROUP_BYTES >> 4) + (uint32_t)(k & 3) * 2u + K_CONST;
        tc_mma<2, false>(d, hi + at, HI, lo + at, HI, form, more);
        tc_mma<1, false>(d, lo + at, HI, hi + at, HI, form, 1u);
        more = 1u;
      }
    for (int k = 0; k < steps16; ++k) {
      const uint32_t at = (uint32_t)(k >> 2) * (NS_GROUP_BYTES >> 4) + (uint32_t)(k & 3) * 2u + K_CONST;
      tc_mma<2, false>(d, hi + at, HI, hi + at, HI, form, more);
      more = 1u;
    }
  };
  // descriptors take the address within the CTA: higher bits, which may name the CTA of the cluster, would run into the next field
  const uint32_t xu = (ag_smem_u32(X) & 0x3FFFFu) >> 4, xl = xu + (plane >> 4), au = (ag_smem_u32(AQ) & 0x3FFFFu) >> 4, al = au + ((2 * NS_GROUP_BYTES) >> 4);
  constexpr int SLICES = NS_SMALL_THREADS / 128;
  const int quarter = warp & 3, slice = warp >> 2, row = quarter * 32 + lane;
  // what is not padding: steps of 16 elements, chunks of 32 columns of a square
  const int m16 = (p.m + 15) / 16, m32 = (p.m + 31) / 32;
  const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
  const int w16 = max(1, (width + 15) / 16), chain16 = SPLIT ? 8 : 4 * NS_SMALL_GROUPS, chains = (w16 + chain16 - 1) / chain16;
  // 32 columns of the lane's row into the words of a buffer; rows of padding are zero
  auto put = [&](unsigned char* dst, uint32_t low, int col, const float (&v)[32]) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      split_f16x2(v[2 * k], v[2 * k + 1], hi[k], lo[k]);
      if (row >= p.m) hi[k] = lo[k] = 0u;
    }
    unsigned char* d = dst + (uint32_t)(col >> 6) * NS_GROUP_BYTES;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = ns_swizzled(row, (uint32_t)(col & 63) * 2u + 16u * j);
      *reinterpret_cast<uint4*>(d + at) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
      if (SPLIT) *reinterpret_cast<uint4*>(d + low + at) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
    }
  };
  auto finish_value = [&](int col, const float (&v)[32]) {  // 32-bit values in X's place, in the order in which they leave
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      if (tall) {
        reinterpret_cast<float*>(X)[(col + j) * NS_SMALL_M + row] = v[j];
      } else if ((j & 3) == 0) {
        *reinterpret_cast<float4*>(X + (uint32_t)row * W * 4u + ((((uint32_t)(col + j) >> 2) ^ ((uint32_t)row & 7u)) << 4)) =
            make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
  };
  const float unit = 1.0f / NS_SCALE;
  for (int step = 0; step < p.steps; ++step) {
    const float a = p.co[3 * step], b = p.co[3 * step + 1], c = p.co[3 * step + 2];
    const bool square = c != 0.0f;
    const float h = square ? b / (2.0f * c) : 0.0f;
    const float gram_mul = (square ? 1.0f : b) * unit * p.loss_gram, gram_diag = (square ? h : a) * NS_SCALE;
    if (tid == 0 && !expired) {
      for (int i = 0; i < chains; ++i)
        gram(tmem + i * 128, xu + 2 * i * (NS_GROUP_BYTES >> 4), xl + 2 * i * (NS_GROUP_BYTES >> 4), min(chain16, w16 - i * chain16), m16 * 16);
      tc_commit(bar);
    }
    products_done();
    const int own = NS_SMALL_M / S;          // rows of the sum that a CTA owns
    if (S > 1 && !apart) tc_cluster_sync();  // nobody multiplies with its Q any more
    for (int ch = slice; ch < m32; ch += SLICES) {
      const int col = ch * 32;
      float v[32];
      tc_tmem_ld32(trow + col, reinterpret_cast<uint32_t(&)[32]>(v));
      tc_tmem_ld_wait();
      for (int i = 1; i < chains; ++i) {
        uint32_t r[32];
        tc_tmem_ld32(trow + i * 128 + col, r);
        tc_tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(r[j]);
      }
      if (S == 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = v[j] * gram_mul + (row == col + j ? gram_diag : 0.0f);
        put(AQ, 2 * NS_GROUP_BYTES, col, v);
      } else {
        const uint32_t to = tc_map_to_cta(ag_smem_u32(parts), row / own) + (uint32_t)(rank * own + row % own) * 512u;
        if (row < p.m) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            ns_st_cluster(to + (((((uint32_t)col >> 2) + j) ^ ((uint32_t)row & 7u)) << 4), make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        }
        __syncwarp();
      }
    }
    if (S > 1) {
      tc_cluster_sync();
      // own rows: four columns to a thread and turn, 32 x own of them
      constexpr int TURNS = NS_SMALL_M / 2 * 32 / NS_SMALL_THREADS;
      float4 sums[TURNS];
#pragma unroll
      for (int k = 0; k < TURNS; ++k) {
        const int i = tid + k * NS_SMALL_THREADS, r = i >> 5, q = i & 31, global = rank * own + r;
        if (r >= own || global >= m16 * 16 || q >= m32 * 8) continue;
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < (global < p.m ? S : 0); ++s) {
          const float4 x = *reinterpret_cast<const float4*>(parts + (uint32_t)(s * own + r) * 512u + ((uint32_t)(q ^ (global & 7)) << 4));
          t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
        }
        const int d = global < p.m ? global - q * 4 : -1;  // the diagonal's place among the four; rows of padding are zero
        t.x = t.x * gram_mul + (d == 0 ? gram_diag : 0.f);
        t.y = t.y * gram_mul + (d == 1 ? gram_diag : 0.f);
        t.z = t.z * gram_mul + (d == 2 ? gram_diag : 0.f);
        t.w = t.w * gram_mul + (d == 3 ? gram_diag : 0.f);
        sums[k] = t;
      }
      if (!apart) tc_cluster_sync();  // all have read the parts: A takes their place
#pragma unroll
      for (int k = 0; k < TURNS; ++k) {
        const int i = tid + k * NS_SMALL_THREADS, r = i >> 5, q = i & 31, global = rank * own + r;
        if (r >= own || global >= m16 * 16 || q >= m32 * 8) continue;
        uint32_t hi[2], lo[2];
        split_f16x2(sums[k].x, sums[k].y, hi[0], lo[0]);
        split_f16x2(sums[k].z, sums[k].w, hi[1], lo[1]);
        const uint32_t at = ag_smem_u32(AQ) + (uint32_t)(q >> 4) * NS_GROUP_BYTES + ns_swizzled(global, (uint32_t)(q & 15) * 8u);
        for (int s = 0; s < S; ++s) {
          const uint32_t to = tc_map_to_cta(at, s);
          ns_st_cluster(to, hi[0], hi[1]);
          if (SPLIT) ns_st_cluster(to + 2 * NS_GROUP_BYTES, lo[0], lo[1]);
        }
      }
    }
    ns_fence_proxy();
    tc_fence_before();
    cluster_sync();
    if (square) {
      if (tid == 0 && !expired) {
        tc_fence_after();
        ns_fence_proxy();
        gram(tmem, au, al, m16, m16 * 16);
        tc_commit(bar);
      }
      products_done();
      const float mul = c * unit * p.loss_square, diag = (a - h * h * c) * NS_SCALE;
      for (int ch = slice; ch < m32; ch += SLICES) {
        const int col = ch * 32;
        float v[32];
        tc_tmem_ld32(trow + col, reinterpret_cast<uint32_t(&)[32]>(v));
        tc_tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = v[j] * mul + (row == col + j ? diag : 0.0f);
        put(AQ, 2 * NS_GROUP_BYTES, col, v);
      }
      ns_fence_proxy();
      tc_fence_before();
      __syncthreads();
    }
    if (tid == 0 && !expired) {
      tc_fence_after();
      ns_fence_proxy();
      for (int c0 = 0; c0 < G; c0 += 4) {  // up to 256 columns at a time
        const uint32_t n = (uint32_t)min(4, G - c0) * 64u, d = tmem + c0 * 64, x0 = c0 * (NS_GROUP_BYTES >> 4) + MN_CONST;
        uint32_t more = 0;
        if (SPLIT)
          for (int k = 0; k < m16; ++k) {
            const uint32_t l = (uint32_t)(k >> 2) * (NS_GROUP_BYTES >> 4) + (uint32_t)(k & 3) * 2u + K_CONST, r = x0 + k * 128;
            tc_mma<2, false>(d, au + l, HI, xl + r, HI, idesc(n, true), more);
            tc_mma<1, false>(d, al + l, HI, xu + r, HI, idesc(n, true), 1u);
            more = 1u;
          }
        for (int k = 0; k < m16; ++k) {
          const uint32_t l = (uint32_t)(k >> 2) * (NS_GROUP_BYTES >> 4) + (uint32_t)(k & 3) * 2u + K_CONST, r = x0 + k * 128;
          tc_mma<2, false>(d, au + l, HI, xu + r, HI, idesc(n, true), more);
          more = 1u;
        }
      }
      tc_commit(bar);
    }
    products_done();
    const bool last = step + 1 == p.steps;
    const float mul = (last ? unit * unit : unit) * p.loss_square;
    for (int ch = slice; ch < 2 * G; ch += SLICES) {
      float v[32];
      tc_tmem_ld32(trow + ch * 32, reinterpret_cast<uint32_t(&)[32]>(v));
      tc_tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= mul;
      if (last) finish_value(ch * 32, v);
      else put(X, plane, ch * 32, v);
    }
    ns_fence_proxy();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  // ---- out
  float* out = p.mats.p[mat];
  for (int i = tid; i < count; i += NS_SMALL_THREADS * AHEAD) {
    float old[AHEAD][1];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      int r, c;
      if (j < count && p.out_kind == NS_STEP) old[k][0] = out[place(j, r, c)];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int j = i + k * NS_SMALL_THREADS;
      if (j >= count) continue;
      int r, c;
      const int64_t at = place(j, r, c);
      float v[1];
      if (p.steps == 0) {
        const uint32_t x = (uint32_t)(c >> 6) * NS_GROUP_BYTES + ns_swizzled(r, (uint32_t)(c & 63) * 2u);
        v[0] = (__half2float(*reinterpret_cast<const __half*>(X + x)) + __half2float(*reinterpret_cast<const __half*>(X + plane + x))) * unit;
      } else if (tall) {
        v[0] = reinterpret_cast<const float*>(X)[c * NS_SMALL_M + r];
      } else {
        v[0] = *reinterpret_cast<const float*>(X + (uint32_t)r * W * 4u + ((((uint32_t)c >> 2) ^ ((uint32_t)r & 7u)) << 4) + ((uint32_t)c & 3u) * 4u);
      }
      ns_put<1>(out, at, v, old[k], p.keep, p.by, p.out_kind);
    }
  }
  if (expired) atomicOr(p.status, AG_STATUS_WAIT_EXPIRED);
  tc_fence_before();
  if (S > 1) tc_meet<true>(); else tc_meet<false>();
  if (warp == 0) {
    tc_drain(abort_flag);
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------------------- host side
// Tensor maps of a plane of `rows` rows (of all matrices) of `cols` columns.  NS_K: tiles of TC_BK columns and `box` rows; NS_MN: seen
// as {64, rows, cols / 64}, boxes of TC_BK rows and `box` columns; NS_OUT: 32 x 32.
enum { NS_K, NS_MN, NS_OUT };
int ns_map(ag_ctx* ctx, CUtensorMap* tm, const void* plane, int64_t rows, int64_t cols, int box, int form) {
  EncodeTiledFn encode = tc_encode_fn(ctx);
  if (!encode) return AG_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1}, strides[2] = {(cuuint64_t)cols * 2, TC_MN_GROUP * 2};
  cuuint32_t boxes[3] = {TC_BK, (cuuint32_t)box, 1}, estr[3] = {1, 1, 1};
  if (form == NS_MN) {
    dims[0] = TC_MN_GROUP; dims[2] = (cuuint64_t)(cols / TC_MN_GROUP);
    boxes[0] = TC_MN_GROUP; boxes[1] = TC_BK; boxes[2] = (cuuint32_t)(box / TC_MN_GROUP);
  } else if (form == NS_OUT) {
    boxes[0] = boxes[1] = 32;
  }
  const CUresult r = encode(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, form == NS_MN ? 3 : 2, const_cast<void*>(plane), dims, strides, boxes, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, form == NS_OUT ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    AG_FAIL(ctx, AG_ERR_CUDA, "cuTensorMapEncodeTiled failed: CUresult %d (ptr %p, %lld x %lld, box %d)", (int)r, plane, (long long)rows,
            (long long)cols, box);
  return AG_OK;
}

// Planes and their maps: as operands, and as a result
struct NsBuffer {
  NsPlane plane;
  NsMaps maps;
  CUtensorMap out_hi, out_lo;
};

int ns_maps(ag_ctx* ctx, NsBuffer& b, int64_t rows, int64_t cols) {
  int rc = AG_OK;
  auto make = [&](CUtensorMap& hi, CUtensorMap& lo, int form) {
    if (!rc) rc = ns_map(ctx, &hi, b.plane.hi, rows, cols, TC_BM, form);
    lo = hi;
    if (!rc && b.plane.lo) rc = ns_map(ctx, &lo, b.plane.lo, rows, cols, TC_BM, form);
  };
  make(b.maps.k_hi, b.maps.k_lo, NS_K);
  make(b.maps.mn_hi, b.maps.mn_lo, NS_MN);
  make(b.out_hi, b.out_lo, NS_OUT);
  return rc;
}

int ns_tiles(int kind, int M, int N, int BM, int BN) {
  const int m = (M + BM - 1) / BM, n = (N + BN - 1) / BN;
  if (!ns_symmetric(kind)) return m * n;
  if (BM == 256) return n * (n + 1) / 2;
  return 2 * (n / 2) * (n / 2 + 1) + (n & 1 ? n : 0);  // two columns of 2 j + 2 each, and what an odd number leaves
}

template <int KIND, bool SPLIT, bool PAIR, int BN, bool ZSPLIT>
int ns_launch(ag_ctx* ctx, NsGemm& p) {
  constexpr int BM = PAIR ? 256 : 128, BN_CTA = PAIR ? BN / 2 : BN;
  constexpr size_t SLOT = (size_t)(TC_BM + BN_CTA) * 256;
  static std::atomic<int> known[AG_MAX_DEVICES];  // 1 + units that are resident at once
  auto kern = ns_gemm_kernel<KIND, SPLIT, PAIR, BN, ZSPLIT>;
  std::atomic<int>& slot = known[ag_dev_slot(ctx)];
  int units = slot.load(std::memory_order_relaxed) - 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.blockDim = dim3(NS_TC_THREADS);
  cfg.dynamicSmemBytes = NS_SMEM_LIMIT;
  cfg.attrs = at;
  if (PAIR || ZSPLIT) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PAIR ? 2 : p.cluster;
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
  p.tiles = ns_tiles(KIND, p.M, p.N, BM, BN);
  p.chain = SPLIT ? NS_CHAIN_PAIRS : NS_CHAIN_SINGLE;
  const int chains = (p.k_iters + 2 * p.chain - 1) / (2 * p.chain);  // parts of a cluster are whole chains
  if (SPLIT) p.mul *= (float)(1.0 + NS_LOSS * std::max(0.0, ((p.k_real + 15) / 16 - chains) / (double)chains));
  // a slot per accumulator, and two steps' low parts: more slots would be free no earlier
  constexpr int SLOTS = SPLIT ? 2 : std::min<int>(NS_MAX_SLOTS, (int)((NS_SMEM_LIMIT - NS_SMEM_FIXED) / SLOT));
  static_assert(NS_SMEM_FIXED + (SLOTS + (SPLIT ? 1 : 0)) * SLOT <= NS_SMEM_LIMIT && SLOTS >= 2, "operand tiles");
  p.slots = SLOTS;
  p.expire = tc_expires(ctx);
  const int64_t work = (int64_t)p.batch * p.tiles;
  cfg.gridDim = dim3(ZSPLIT ? work * p.cluster : (PAIR ? 2 : 1) * std::min<int64_t>(units, work));
  cfg.dynamicSmemBytes = NS_SMEM_FIXED + (SLOTS + (SPLIT ? 1 : 0)) * SLOT;
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

// Tiles of 256 x 256 on pairs of CTAs or of 128 x 128 on single ones: a round of them takes 7 + 1.15 k or 6 + 0.78 k us for k steps of 64
// elements with pairs of words (1280 x 1280 alone: 402 us on pairs, 327 on single CTAs; four of them 630 and 737).  Where X X^T
// leaves most SMs without a tile, clusters share the contraction, four steps or more to each CTA.
int ns_form(ag_ctx* ctx, int kind, int batch, int M, int N, int k_iters, int* cluster) {
  const int64_t pairs = (int64_t)batch * ns_tiles(kind, M, N, 256, 256), singles = (int64_t)batch * ns_tiles(kind, M, N, 128, 128);
  const double on_pairs = ag_ceil_div(pairs, ctx->sm_count / 2) * (7.0 + 1.15 * k_iters);
  const double on_singles = ag_ceil_div(singles, ctx->sm_count) * (6.0 + 0.78 * k_iters);
  if (M > 256 && on_pairs <= on_singles) return AG_NS_PAIRS;
  if (kind != NS_GRAM) return AG_NS_SINGLE;
  int z = 8;
  while (z > 1 && (singles * z > ctx->sm_count || k_iters < 4 * z)) z /= 2;
  *cluster = z;
  return z > 1 ? AG_NS_CLUSTERS : AG_NS_SINGLE;
}

template <int KIND, bool SPLIT>
int ns_product(ag_ctx* ctx, NsGemm& p) {
  const int form = ns_form(ctx, KIND, p.batch, p.M, p.N, p.k_iters, &p.cluster);
  if (form == AG_NS_PAIRS) return ns_launch<KIND, SPLIT, true, 256, false>(ctx, p);
  if constexpr (KIND == NS_GRAM) {
    if (form == AG_NS_CLUSTERS) {
      p.k_each = ((p.k_iters + p.cluster - 1) / p.cluster + 1) & ~1;
      return ns_launch<KIND, SPLIT, false, 128, true>(ctx, p);
    }
  }
  return ns_launch<KIND, SPLIT, false, 128, false>(ctx, p);
}

// X[0] -> the factor in X[steps & 1]
template <bool SPLIT>
int ns_iterate(ag_ctx* ctx, const NsPlan& t, NsGemm& p, NsBuffer* X, NsBuffer& A, NsBuffer& Q, const float* coefficients, int steps) {
  const float unit = 1.0f / NS_SCALE;  // operands carry NS_SCALE each, a result one of them
  for (int i = 0; i < steps; ++i) {
    const double a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2], h = c != 0.0 ? b / (2.0 * c) : 0.0;
    NsBuffer &x = X[i & 1], &y = X[~i & 1];
    auto product = [&](auto kind, const NsMaps& l, const NsMaps& r, NsBuffer& d, int n, int k, double mul, double diag) {
      p.l = l; p.r = r;
      p.d_hi = d.out_hi; p.d_lo = d.out_lo; p.D = d.plane;
      p.two = d.plane.lo && (SPLIT || (&d == &y && i + 1 == steps));
      p.N = n; p.k_iters = (k + TC_BK - 1) / TC_BK; p.k_real = k;
      p.mul = (float)mul * unit; p.diag = (float)(diag * NS_SCALE);
      return ns_product<decltype(kind)::value, SPLIT>(ctx, p);
    };
    int rc = product(std::integral_constant<int, NS_GRAM>(), x.maps, x.maps, c != 0.0 ? A : Q, t.mp, t.n, c != 0.0 ? 1.0 : b, c != 0.0 ? h : a);
    if (!rc && c != 0.0) rc = product(std::integral_constant<int, NS_POLY>(), A.maps, A.maps, Q, t.mp, t.m, c, a - h * h * c);
    if (!rc) rc = product(std::integral_constant<int, NS_NEXT>(), Q.maps, x.maps, y, t.np, t.m, 1.0, 0.0);
    if (rc) return rc;
  }
  return AG_OK;
}

void ns_cluster_launch(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* at, int cluster, int blocks) {
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(NS_SMALL_THREADS);
  cfg.dynamicSmemBytes = NS_SMEM_LIMIT;  // whatever the slice needs: a CTA has its SM, and all of tensor memory, for itself
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
}

template <typename T, bool SPLIT>
int ns_small_setup(ag_ctx* ctx) {
  static std::atomic<bool> done[AG_MAX_DEVICES];
  auto kern = ns_small_kernel<T, SPLIT>;
  if (!done[ag_dev_slot(ctx)].load(std::memory_order_relaxed)) {
    AG_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, NS_SMEM_LIMIT));
    AG_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    done[ag_dev_slot(ctx)].store(true, std::memory_order_relaxed);
  }
  return AG_OK;
}

// Clusters of 2^log2 CTAs of the small kernel that are resident at once; 0: none, or not known
int ns_small_resident(ag_ctx* ctx, int log2) {
  static std::atomic<int> known[AG_MAX_DEVICES][5];  // 1 + the answer
  std::atomic<int>& slot = known[ag_dev_slot(ctx)][log2];
  if (const int k = slot.load(std::memory_order_relaxed)) return k - 1;
  int n = 0;
  if (ns_small_setup<float, true>(ctx) == AG_OK) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    ns_cluster_launch(cfg, at, 1 << log2, ctx->sm_count << log2);
    if (cudaOccupancyMaxActiveClusters(&n, ns_small_kernel<float, true>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
  }
  slot.store(1 + n, std::memory_order_relaxed);
  return n;
}

// How the columns of X, in groups of 64, go to the CTAs of a cluster; false where the general path serves the matrices better.  Times in
// us, fitted to measurements of 16 to 128 rows and 16 to 5000 columns: a round of clusters takes 13 + 0.17 m, 3 + 0.15 m a group and, with
// S > 1 CTAs, 12 + m m S / 10^4 (64 x 256: 51 on four CTAs, 64 on two, 73 on one; 128 x 256: 78, 93, 116; 64 x 64: 36 on one, 49 on four;
// 128 x 1024, 2048, 4096 on sixteen: 93, 114, 160), and there are as many rounds as it takes to hold all matrices; the general path
// 85 + 0.065 n + 0.0013 n for each matrix (64 x 64: 90, 2 of 64 x 1024: 154, 2 of 128 x 4096: 355, 16 of them: 433 against 501, 32 of 100 x
// 5000: 656 against 836).
bool ns_small_shape(ag_ctx* ctx, const NsPlan& t, int count, int* cluster, int* groups) {
  if (t.m > NS_SMALL_M) return false;
  const int all = (t.n + 63) / 64;
  double best = 85.0 + 0.065 * t.n + 0.0013 * t.n * count;
  bool found = false;
  for (int log2 = 0; (1 << log2) <= NS_SMALL_CLUSTER && (log2 == 0 || (1 << log2) < 2 * all); ++log2) {
    const int g = (all + (1 << log2) - 1) >> log2;
    if (g > NS_SMALL_GROUPS) continue;
    const int resident = ns_small_resident(ctx, log2);
    if (resident < 1) continue;
    const double cost = ((count + resident - 1) / resident) *
                        (13.0 + 0.17 * t.m + (3.0 + 0.15 * t.m) * g + (log2 ? 12.0 + 1e-4 * t.m * t.m * (1 << log2) : 0.0));
    if (cost < best) {
      best = cost;
      found = true;
      *cluster = 1 << log2;
      *groups = g;
    }
  }
  return found;
}

template <typename T, bool SPLIT>
int ns_small_launch(ag_ctx* ctx, NsSmall& p, int count) {
  static_assert(1024 + 2 * NS_SMALL_GROUPS * NS_GROUP_BYTES + NS_SQUARE_BYTES + 512 <= NS_SMEM_LIMIT &&
                1024 + 2 * NS_SMALL_APART * NS_GROUP_BYTES + 2 * NS_SQUARE_BYTES + 512 <= NS_SMEM_LIMIT, "slice and square");
  if (int rc = ns_small_setup<T, SPLIT>(ctx)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  ns_cluster_launch(cfg, at, p.cluster, count * p.cluster);
  cfg.stream = ctx->stream;
  if (ctx->pdl) {
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  AG_CUDA(ctx, cudaLaunchKernelEx(&cfg, ns_small_kernel<T, SPLIT>, p));
  ctx->launches++;
  ag_enqueued(ctx);
  return AG_OK;
}

int ns_run(ag_ctx* ctx, const NsPlan& t, const NsMatrices& mats, int count, int bf16, const NsUpdate& s, float eps,
           const float* coefficients, int steps, float keep, float by, int out_kind, char* scratch, bool split) {
  int cluster, groups;
  if (ns_small_shape(ctx, t, count, &cluster, &groups)) {
    NsSmall p = {};
    p.mats = mats; p.s = s;
    p.rows = t.rows; p.cols = t.cols; p.m = t.m; p.n = t.n; p.groups = groups; p.cluster = cluster; p.steps = steps; p.out_kind = out_kind;
    p.eps = eps; p.keep = keep; p.by = by; p.wait_limit = tc_expires(ctx) ? 0u : TC_WAIT_LIMIT; p.status = ctx->d_status;
    const double chains = cluster * ((groups + 1) / 2);
    p.loss_gram = split ? (float)(1.0 + NS_LOSS * std::max(0.0, ((t.n + 15) / 16 - chains) / chains)) : 1.0f;
    p.loss_square = split ? (float)(1.0 + NS_LOSS * ((t.m + 15) / 16 - 1)) : 1.0f;
    for (int i = 0; i < 3 * steps; ++i) p.co[i] = coefficients[i];
    if (bf16) return split ? ns_small_launch<__nv_bfloat16, true>(ctx, p, count) : ns_small_launch<__nv_bfloat16, false>(ctx, p, count);
    return split ? ns_small_launch<float, true>(ctx, p, count) : ns_small_launch<float, false>(ctx, p, count);
  }
  // 16-bit operands have one word, but for the last result, which nothing multiplies
  auto plane = [&](size_t at, size_t bytes, bool two) {
    return NsPlane{reinterpret_cast<__half*>(scratch + at), two ? reinterpret_cast<__half*>(scratch + at + bytes / 2) : nullptr};
  };
  NsBuffer X[2], A, Q;
  for (int i = 0; i < 2; ++i) X[i].plane = plane(i * t.x_bytes, t.x_bytes, split || i == (steps & 1));
  A.plane = plane(2 * t.x_bytes, t.a_bytes, split);
  Q.plane = plane(2 * t.x_bytes + t.a_bytes, t.a_bytes, split);
  double* norms = reinterpret_cast<double*>(scratch + 2 * t.x_bytes + 2 * t.a_bytes);
  const int64_t elements = (int64_t)t.rows * t.cols;
  // accesses of four elements where all addresses are multiples of their size, in every row for the tiles
  bool vec = true, vec_out = true;
  for (int i = 0; i < count; ++i) {
    vec = vec && ag_aligned16(mats.m[i]) && ((uintptr_t)mats.g[i] & (bf16 ? 7 : 15)) == 0;
    vec_out = vec_out && ((uintptr_t)mats.p[i] & (out_kind == NS_BF16 ? 7 : 15)) == 0;
  }
  const bool vec_rows = vec && (t.cols & 3) == 0;
  vec_out = vec_out && (t.cols & 3) == 0;
  int blocks = ag_ceil_div(elements, (int64_t)NS_THREADS * 4 * (vec ? 4 : 1));
  if (blocks > NS_NORM_BLOCKS) blocks = NS_NORM_BLOCKS;
  const dim3 tiles(t.np / 64, t.mp / 64, count);
#define NS_FORMS(T, EACH_M, EACH_S)                                                                                              \
  do {                                                                                                                           \
    if (mats.m[0])                                                                                                                \
      AG_LAUNCH_PDL(ctx, "ns_momentum_kernel", (ns_momentum_kernel<T, EACH_M, true>), dim3(blocks, count), NS_THREADS, 0, mats, elements, s, norms); \
    else                                                                                                                         \
      AG_LAUNCH_PDL(ctx, "ns_momentum_kernel", (ns_momentum_kernel<T, EACH_M, false>), dim3(blocks, count), NS_THREADS, 0, mats, elements, s, norms); \
    AG_LAUNCH_PDL(ctx, "ns_start_kernel", (ns_start_kernel<T, EACH_S>), tiles, NS_THREADS, 0, mats, t, s, eps, (const double*)norms, blocks, \
                  X[0].plane);                                                                                                    \
  } while (0)
  if (bf16) {
    if (vec_rows) NS_FORMS(__nv_bfloat16, 4, 4);
    else if (vec) NS_FORMS(__nv_bfloat16, 4, 1);
    else NS_FORMS(__nv_bfloat16, 1, 1);
  } else {
    if (vec_rows) NS_FORMS(float, 4, 4);
    else if (vec) NS_FORMS(float, 4, 1);
    else NS_FORMS(float, 1, 1);
  }
#undef NS_FORMS
  if (steps > 0) {
    const int64_t rows = (int64_t)count * t.mp;
    int rc;
    if ((rc = ns_maps(ctx, X[0], rows, t.np)) || (rc = ns_maps(ctx, X[1], rows, t.np)) || (rc = ns_maps(ctx, A, rows, t.mp)) ||
        (rc = ns_maps(ctx, Q, rows, t.mp)))
      return rc;
    NsGemm p = {};
    p.batch = count;
    p.M = t.mp;
    p.status = ctx->d_status;
    if ((rc = split ? ns_iterate<true>(ctx, t, p, X, A, Q, coefficients, steps) : ns_iterate<false>(ctx, t, p, X, A, Q, coefficients, steps)))
      return rc;
  }
  if (vec_out)
    AG_LAUNCH_PDL(ctx, "ns_finish_kernel", ns_finish_kernel<4>, tiles, NS_THREADS, 0, mats, t, X[steps & 1].plane, keep, by, out_kind);
  else
    AG_LAUNCH_PDL(ctx, "ns_finish_kernel", ns_finish_kernel<1>, tiles, NS_THREADS, 0, mats, t, X[steps & 1].plane, keep, by, out_kind);
  return AG_OK;
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
  for (int i = 0; i < steps; ++i) {
    const double b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    AG_REQUIRE(ctx, c == 0.0 || (fabs(b) <= 16.0 * fabs(c) && b * b <= 256.0 * fabs(c)), "%s: coefficients b %g and c %g are too far apart",
               name, b, c);
  }
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
    const bool in_place = !m && g[i] == p[i] && g_size >= p_size;  // the factor may take its matrix's place
    add(p[i], elements * (in_place ? g_size : p_size), true);
    if (m) add(m[i], elements * 4, true);
    if (!in_place) add(g[i], elements * g_size, false);
  }
  add(scratch, scratch_bytes, true);
  const bool apart = ns_apart(r, n);
  if (r != few) free(r);
  AG_REQUIRE(ctx, apart, "%s: matrices overlap one another or the workspace", name);
  return AG_OK;
}

}  // namespace

extern "C" int ag_orthogonalise_form(ag_ctx* ctx, int count, int rows, int cols, int product, int* form, int* batch) {
  if (!ctx) return AG_ERR_INVALID;
  AG_REQUIRE(ctx, count > 0 && rows > 0 && cols > 0 && ns_fits(rows, cols), "ag_orthogonalise_form: bad shape count=%d rows=%d cols=%d", count, rows,
             cols);
  AG_REQUIRE(ctx, product >= NS_GRAM && product <= NS_NEXT && form && batch, "ag_orthogonalise_form: product %d", product);
  const NsPlan t = ns_plan(count, rows, cols);
  int cluster = 1, groups;
  *batch = t.batch;
  *form = ns_small_shape(ctx, t, t.batch, &cluster, &groups)
              ? AG_NS_ONE_LAUNCH
              : ns_form(ctx, product, t.batch, t.mp, product == NS_NEXT ? t.np : t.mp, ((product == NS_GRAM ? t.n : t.m) + TC_BK - 1) / TC_BK, &cluster);
  return AG_OK;
}

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
    if (int rc = ns_run(ctx, t, mats, here, dtype == AG_BF16, s, eps, coefficients, steps, 0.0f, 0.0f, out_dtype == AG_F32 ? NS_F32 : NS_BF16,
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
                        (float)(lr * scale), NS_STEP, static_cast<char*>(scratch), precision == AG_CE_3XTF32))
      return rc;
  }
  return AG_OK;
}
