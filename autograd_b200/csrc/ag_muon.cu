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

#include "ag_common.cuh"

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

// m <- m + (1 - beta) (g - m); the squares of the update's elements, in 64 bits, summed by every block
__global__ void __launch_bounds__(NS_THREADS) ns_momentum_kernel(const NsMatrices mats, int64_t elements, int bf16, NsUpdate s,
                                                                 double* norms) {
  __shared__ double part[NS_THREADS / 32];
  ag_pdl_wait();
  ag_pdl_trigger();
  const void* g = mats.g[blockIdx.y];
  float* m = mats.m[blockIdx.y];
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * NS_THREADS + threadIdx.x; i < elements; i += (int64_t)gridDim.x * NS_THREADS) {
    float u = ns_load(g, bf16, i) * s.grad_scale;
    if (m) {
      const float t = fmaf(1.0f - s.beta, u - m[i], m[i]);
      m[i] = t;
      u = ns_direction(u, t, s);
    }
    sum = fma((double)u, (double)u, sum);
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NS_THREADS / 32; ++w) sum += part[w];
    norms[blockIdx.y * NS_NORM_BLOCKS + blockIdx.x] = sum;
  }
}

// X = u / max(|u|, eps) in padded rows, transposed where the matrix is tall
__global__ void __launch_bounds__(NS_THREADS) ns_start_kernel(const NsMatrices mats, NsPlan t, int bf16, NsUpdate s, float eps,
                                                              const double* norms, int norm_blocks, float* X) {
  __shared__ float tile[32][33];
  ag_pdl_wait();
  ag_pdl_trigger();
  double sum = 0.0;
  for (int i = 0; i < norm_blocks; ++i) sum += norms[blockIdx.z * NS_NORM_BLOCKS + i];
  const double norm = sqrt(sum), by = 1.0 / (norm > eps || norm != norm ? norm : (double)eps);
  const void* g = mats.g[blockIdx.z];
  const float* m = mats.m[blockIdx.z];
  const bool tall = t.rows > t.cols;
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;  // of X
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int k = ty; k < 32; k += NS_THREADS / 32) {
    const int row = tall ? c0 + k : r0 + k, col = tall ? r0 + tx : c0 + tx;  // of the matrix
    float u = 0.0f;
    if (row < t.rows && col < t.cols) {
      const int64_t i = (int64_t)row * t.cols + col;
      u = ns_load(g, bf16, i) * s.grad_scale;
      if (m) u = ns_direction(u, m[i], s);
      u = (float)(u * by);
    }
    tile[k][tx] = u;
  }
  __syncthreads();
  float* x = X + (int64_t)blockIdx.z * t.mp * t.np;
  for (int k = ty; k < 32; k += NS_THREADS / 32) {
    const int row = r0 + k, col = c0 + tx;
    if (row < t.mp && col < t.np) x[(int64_t)row * t.np + col] = tall ? tile[tx][k] : tile[k][tx];
  }
}

// D = diag I + add A + mul L R of every matrix, R as stored or transposed
template <bool TRANSPOSED>
__global__ void __launch_bounds__(NS_THREADS) ns_product_kernel(const float* L, int64_t ldl, const float* R, int64_t ldr, float* D,
                                                                int64_t ldd, const float* A, int M, int N, int K, int64_t l_next,
                                                                int64_t r_next, int64_t d_next, float diag, float add, float mul) {
  __shared__ float ls[16][65], rs[16][65];
  ag_pdl_wait();
  ag_pdl_trigger();
  L += blockIdx.z * l_next; R += blockIdx.z * r_next; D += blockIdx.z * d_next;
  if (A) A += blockIdx.z * d_next;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += NS_THREADS) {
      const int k = i & 15, r = i >> 4;
      ls[k][r] = m0 + r < M && k0 + k < K ? L[(m0 + r) * ldl + k0 + k] : 0.0f;
      if (TRANSPOSED) {
        rs[k][r] = n0 + r < N && k0 + k < K ? R[(n0 + r) * ldr + k0 + k] : 0.0f;
      } else {
        const int c = i & 63, kk = i >> 6;
        rs[kk][c] = n0 + c < N && k0 + kk < K ? R[(k0 + kk) * ldr + n0 + c] : 0.0f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ls[k][ty * 4 + i], rs[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
      if (r >= M || c >= N) continue;
      float v = mul * acc[i][j] + (r == c ? diag : 0.0f);
      if (A) v = fmaf(add, A[r * ldd + c], v);
      D[r * ldd + c] = v;
    }
}

// p <- keep p - by X, or out = X in its type
__global__ void __launch_bounds__(NS_THREADS) ns_finish_kernel(const NsMatrices mats, NsPlan t, const float* X, float keep, float by,
                                                               int out_kind) {
  ag_pdl_wait();
  ag_pdl_trigger();
  const float* x = X + (int64_t)blockIdx.y * t.mp * t.np;
  float* p = mats.p[blockIdx.y];
  const bool tall = t.rows > t.cols;
  const int64_t elements = (int64_t)t.rows * t.cols;
  for (int64_t i = (int64_t)blockIdx.x * NS_THREADS + threadIdx.x; i < elements; i += (int64_t)gridDim.x * NS_THREADS) {
    const int64_t row = i / t.cols, col = i - row * t.cols;
    const float v = tall ? x[col * t.np + row] : x[row * t.np + col];
    if (out_kind == 0) p[i] = fmaf(-by, v, keep * p[i]);
    else if (out_kind == 1) p[i] = v;
    else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  }
}

int ns_run(ag_ctx* ctx, const NsPlan& t, const NsMatrices& mats, int count, int bf16, const NsUpdate& s, float eps,
           const float* coefficients, int steps, float keep, float by, int out_kind, char* scratch) {
  float* X[2] = {reinterpret_cast<float*>(scratch), reinterpret_cast<float*>(scratch + t.x_bytes)};
  float* A = reinterpret_cast<float*>(scratch + 2 * t.x_bytes);
  float* Q = reinterpret_cast<float*>(scratch + 2 * t.x_bytes + t.a_bytes);
  double* norms = reinterpret_cast<double*>(scratch + 2 * t.x_bytes + 2 * t.a_bytes);
  const int64_t elements = (int64_t)t.rows * t.cols;
  int blocks = ag_ceil_div(elements, NS_THREADS * 4);
  if (blocks > NS_NORM_BLOCKS) blocks = NS_NORM_BLOCKS;
  AG_LAUNCH_PDL(ctx, "ns_momentum_kernel", ns_momentum_kernel, dim3(blocks, count), NS_THREADS, 0, mats, elements, bf16, s, norms);
  AG_LAUNCH_PDL(ctx, "ns_start_kernel", ns_start_kernel, dim3(t.np / 32, t.mp / 32, count), NS_THREADS, 0, mats, t, bf16, s, eps,
                (const double*)norms, blocks, X[0]);
  const int64_t xn = (int64_t)t.mp * t.np, an = (int64_t)t.mp * t.mp;
  const dim3 ga((t.m + 63) / 64, (t.m + 63) / 64, count), gx((t.n + 63) / 64, (t.m + 63) / 64, count);
  for (int i = 0; i < steps; ++i) {
    const float a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
    AG_LAUNCH_PDL(ctx, "ns_product_kernel", ns_product_kernel<true>, ga, NS_THREADS, 0, (const float*)X[0], (int64_t)t.np,
                  (const float*)X[0], (int64_t)t.np, A, (int64_t)t.mp, (const float*)nullptr, t.m, t.m, t.n, xn, xn, an, 0.0f, 0.0f, 1.0f);
    AG_LAUNCH_PDL(ctx, "ns_product_kernel", ns_product_kernel<true>, ga, NS_THREADS, 0, (const float*)A, (int64_t)t.mp,
                  (const float*)A, (int64_t)t.mp, Q, (int64_t)t.mp, (const float*)A, t.m, t.m, t.m, an, an, an, a, b, c);
    AG_LAUNCH_PDL(ctx, "ns_product_kernel", ns_product_kernel<false>, gx, NS_THREADS, 0, (const float*)Q, (int64_t)t.mp,
                  (const float*)X[0], (int64_t)t.np, X[1], (int64_t)t.np, (const float*)nullptr, t.m, t.n, t.m, an, xn, xn, 0.0f, 0.0f, 1.0f);
    float* swap = X[0];
    X[0] = X[1];
    X[1] = swap;
  }
  int many = ag_ceil_div(elements, NS_THREADS * 4);
  if (many > 1024) many = 1024;
  AG_LAUNCH_PDL(ctx, "ns_finish_kernel", ns_finish_kernel, dim3(many, count), NS_THREADS, 0, mats, t, (const float*)X[0], keep, by,
                out_kind);
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
                        static_cast<char*>(scratch)))
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
                        (float)(lr * scale), 0, static_cast<char*>(scratch)))
      return rc;
  }
  return AG_OK;
}
