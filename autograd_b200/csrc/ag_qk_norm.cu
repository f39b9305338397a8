// Queries and keys normalised per head, scaled by a weight per column and rotated by their position, in one pass, and the
// gradient of that.
//
//   y = R(pos) (gamma * x * inv),  inv = 1 / sqrt(mean(x^2) + eps) over the D columns of a head
//   w = R(pos)^T dy;  dgamma = sum over tokens and heads of w x inv;  v = gamma w;
//   dx = inv (v - x inv^2 mean(v x))
// R turns columns (c, c + rot / 2), c < rot / 2, by the angle of (position, c); columns from rot on stay as they are.
//
// A group of 1 to 32 lanes owns a head: a lane has S slots, a slot two packets that the rotation mixes (columns rot and
// more are split into two halves in the same way, with nothing to mix), so that statistics and rotation need one read, a
// few shuffles and no shared memory.  A thread has one or two heads of a token under way, loads the angles once for them, and goes on to the next
// token of its turn with the weights in registers.  Packets are as wide as addresses, strides and halves allow, one to four
// elements: every shape takes the same code.  All sums are fp32.
// Bound: HBM with fp32 rows (16 x 2048 tokens of 2 x 10 heads of 128: 108 us, 0.95 of the copy rate; the gradient 167 us, 0.92); with bf16 ones (73 us, 0.70;
// the gradient 117 us, 0.66) waits for loads at 31 to 41 % of the warps beside two thirds of the issue slots; instructions with packets of one
// element (heads of 74 columns: 93 us fp32, 0.64; the gradient 143).
#include <type_traits>

#include "ag_common.cuh"

namespace {

constexpr int QK_THREADS = 256;
constexpr int QK_BLOCKS_PER_SM = 8;  // at most: 256 threads each

// One fp32 number, or two that arithmetic takes at once: bf16 rows, where instructions count (gradient of 8192 tokens of 12 + 2
// heads 34 -> 27 us; fp32 rows are bound by memory and lost 3 % with pairs, 114 -> 119 us for 16 x 2048 tokens of 2 x 10 heads).
struct QkOne {
  float v;
  __device__ __forceinline__ static QkOne make(float a, float = 0.0f) { return {a}; }
  __device__ __forceinline__ void get(float& a, float&) const { a = v; }
  __device__ __forceinline__ float sum() const { return v; }
};
struct QkTwo {
  uint64_t v;
  __device__ __forceinline__ static QkTwo make(float a, float b) { return {ag_pair(a, b)}; }
  __device__ __forceinline__ void get(float& a, float& b) const { ag_unpair(v, a, b); }
  __device__ __forceinline__ float sum() const {
    float a, b;
    get(a, b);
    return a + b;
  }
};
__device__ __forceinline__ QkOne qk_mul(QkOne a, QkOne b) { return {a.v * b.v}; }
__device__ __forceinline__ QkOne qk_add(QkOne a, QkOne b) { return {a.v + b.v}; }
__device__ __forceinline__ QkOne qk_fma(QkOne a, QkOne b, QkOne c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ QkTwo qk_mul(QkTwo a, QkTwo b) { return {ag_mul2(a.v, b.v)}; }
__device__ __forceinline__ QkTwo qk_add(QkTwo a, QkTwo b) { return {ag_add2(a.v, b.v)}; }
__device__ __forceinline__ QkTwo qk_fma(QkTwo a, QkTwo b, QkTwo c) { return {ag_fma2(a.v, b.v, c.v)}; }

// NV values of type T as they lie in memory
template <int BYTES> struct QkWord;
template <> struct QkWord<2> { using Raw = uint16_t; };
template <> struct QkWord<4> { using Raw = uint32_t; };
template <> struct QkWord<8> { using Raw = uint2; };
template <> struct QkWord<16> { using Raw = uint4; };

// and as numbers: N of E, TWO in each or one
template <typename T, int NV>
struct QkVec {
  static constexpr bool TWO = NV > 1 && sizeof(T) == 2;
  using E = std::conditional_t<TWO, QkTwo, QkOne>;
  static constexpr int N = TWO ? NV / 2 : NV;
  E e[N];
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = E::make(x, x);
  }
};

template <typename T, int NV>
struct QkPack {
  using Raw = typename QkWord<sizeof(T) * NV>::Raw;
  using V = QkVec<T, NV>;
  union Bits {
    Raw raw;
    uint16_t half[sizeof(T) * NV / 2];
    uint32_t word[sizeof(T) * NV >= 4 ? sizeof(T) * NV / 4 : 1];
    __device__ Bits() {}
  };
  __device__ __forceinline__ static Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  // What is read or written once leaves the cache first (114 -> 108 us forward for the tokens above, fp32), but for narrow packets, whose
  // neighbours read the same sectors again (93 us against 99 with heads of 74 columns)
  __device__ __forceinline__ static Raw load_once(const T* p) {
    if constexpr (NV >= 4) return __ldcs(reinterpret_cast<const Raw*>(p));
    else return load(p);
  }
  __device__ __forceinline__ static void unpack(const Raw& r, V& f) {
    Bits b;
    b.raw = r;
#pragma unroll
    for (int i = 0; i < V::N; ++i) {
      if constexpr (sizeof(T) == 4) f.e[i] = V::E::make(__uint_as_float(b.word[i]));
      else if constexpr (NV == 1) f.e[i] = V::E::make(__uint_as_float((uint32_t)b.half[0] << 16));
      else f.e[i] = V::E::make(__uint_as_float(b.word[i] << 16), __uint_as_float(b.word[i] & 0xffff0000u));
    }
  }
  template <bool ONCE>
  __device__ __forceinline__ static void store(T* p, const V& f) {
    Bits b;
#pragma unroll
    for (int i = 0; i < V::N; ++i) {
      float x, y = 0.0f;
      f.e[i].get(x, y);
      if constexpr (sizeof(T) == 4) {
        b.word[i] = __float_as_uint(x);
      } else if constexpr (NV == 1) {
        b.half[0] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        b.word[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (NV >= 4 && ONCE) __stcs(reinterpret_cast<Raw*>(p), b.raw);
    else *reinterpret_cast<Raw*>(p) = b.raw;
  }
};

template <typename T, int NV>
__device__ __forceinline__ void qk_load_f32(const float* p, QkVec<T, NV>& f) {
  using V = QkVec<T, NV>;
  float v[NV];
  if constexpr (NV >= 4) {
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = __ldg(p + i);
  }
#pragma unroll
  for (int i = 0; i < V::N; ++i) f.e[i] = V::TWO ? V::E::make(v[2 * i % NV], v[(2 * i + 1) % NV]) : V::E::make(v[i], 0.0f);
}

// Queries or keys.  Rows of a token are `*_stride` elements apart, its heads follow one another.
struct QkSide {
  const void* x;
  const void* dy;      // backward
  void* y;             // forward: output; backward: dx
  const float* gamma;  // may be null
  float* dgamma;       // backward, may be null
  int64_t x_stride, dy_stride, y_stride;
  int heads;
  int blocks;          // of U heads each
};

struct QkArgs {
  QkSide side[2];
  const float* cos_tab;
  const float* sin_tab;
  const int32_t* positions;  // null: token % seq
  int64_t tokens;
  int seq, rows;             // rows of the tables
  int D, half, slots;        // half = rot / 2, slots = D / 2 / NV
  int lanes_log2;
  float eps, sgn;
  int accumulate;            // backward: dx += ...
  float* partials;           // backward: [grid.y][grid.x][D]
  int* status;
};

struct QkPlace {  // where a lane stands
  int64_t tok;
  int side, head;  // first head of the block
  bool in;         // the token exists
};

// Columns of a slot: its first packet's and how far the second one is
__device__ __forceinline__ void qk_columns(const QkArgs& a, int first, bool& turns, int& col, int& apart) {
  turns = first < a.half;
  col = turns ? first : a.half + first;
  apart = turns ? a.half : (a.D >> 1) - a.half;
}

// The row of the tables of the token that a group has, which goes `stride` tokens on: no division on the way
struct QkTurn {
  uint32_t pos, step;
  __device__ __forceinline__ QkTurn(const QkArgs& a, int64_t first, int64_t stride) {
    pos = step = 0;
    if (a.half && !a.positions) {
      pos = (uint32_t)first % (uint32_t)a.seq;  // both are below 2^32: there are fewer than 2^31 tokens
      step = (uint32_t)stride % (uint32_t)a.seq;
    }
  }
  __device__ __forceinline__ void next(const QkArgs& a) {
    pos += step;  // both below seq, which is below 2^31
    if (pos >= (uint32_t)a.seq) pos -= (uint32_t)a.seq;
  }
};

// Cosines, and sines with the direction's sign, of a token; 1 and 0 for columns that do not turn.  False: a bad position
template <typename T, int S, int NV>
__device__ __forceinline__ bool qk_angles(const QkArgs& a, int64_t tok, uint32_t pos, bool in, int lane, QkVec<T, NV> (&c)[S], QkVec<T, NV> (&s)[S]) {
  bool ok = true;
  if (in && a.half && a.positions) {
    pos = (uint32_t)a.positions[tok];
    ok = pos < (uint32_t)a.rows;
    if (!ok && lane == 0) atomicOr(a.status, AG_STATUS_BAD_INDEX);
    if (!ok) pos = 0;
  }
#pragma unroll
  for (int k = 0; k < S; ++k) {
    const int first = (lane + (k << a.lanes_log2)) * NV;
    if (in && first < a.half) {
      qk_load_f32<T, NV>(a.cos_tab + (int64_t)pos * a.half + first, c[k]);
      qk_load_f32<T, NV>(a.sin_tab + (int64_t)pos * a.half + first, s[k]);
    } else {
      c[k].fill(1.0f);
      s[k].fill(0.0f);
    }
  }
  return ok;
}

template <typename T, int S, int NV>
__device__ __forceinline__ void qk_gamma(const QkArgs& a, const float* gamma, int lane, QkVec<T, NV> (&lo)[S], QkVec<T, NV> (&hi)[S]) {
#pragma unroll
  for (int k = 0; k < S; ++k) {
    const int slot = lane + (k << a.lanes_log2);
    bool turns;
    int col, apart;
    qk_columns(a, slot * NV, turns, col, apart);
    if (gamma && slot < a.slots) {
      qk_load_f32<T, NV>(gamma + col, lo[k]);
      qk_load_f32<T, NV>(gamma + col + apart, hi[k]);
    } else {
      lo[k].fill(1.0f);
      hi[k].fill(1.0f);
    }
  }
}

// A group goes from token to token with its weights in registers
template <typename T, int NV, int S, int U>
__global__ void __launch_bounds__(QK_THREADS) qk_forward_kernel(const QkArgs a) {
  using P = QkPack<T, NV>;
  ag_pdl_wait();
  ag_pdl_trigger();
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const int per_block = QK_THREADS >> a.lanes_log2;
  const int which = (int)blockIdx.y >= a.side[0].blocks;
  const QkSide& q = a.side[which];
  const int head = ((int)blockIdx.y - (which ? a.side[0].blocks : 0)) * U, heads = min(U, q.heads - head);
  using V = QkVec<T, NV>;
  using E = typename V::E;
  V glo[S], ghi[S];
  qk_gamma<T, S, NV>(a, q.gamma, lane, glo, ghi);
  int col[S], apart[S];
  bool turns[S];
#pragma unroll
  for (int k = 0; k < S; ++k) qk_columns(a, (lane + (k << a.lanes_log2)) * NV, turns[k], col[k], apart[k]);
  const float over = 1.0f / (float)a.D;
  const int64_t first = (int64_t)blockIdx.x * per_block + (threadIdx.x >> a.lanes_log2), stride = (int64_t)gridDim.x * per_block;
  const T* x = static_cast<const T*>(q.x) + first * q.x_stride + (int64_t)head * a.D;
  T* out = static_cast<T*>(q.y) + first * q.y_stride + (int64_t)head * a.D;
  QkTurn turn(a, first, stride);
  const E sign = E::make(a.sgn, a.sgn), minus = E::make(-a.sgn, -a.sgn);
  // all threads of a block make as many turns: the sums are over groups of lanes
  for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.tokens; base += stride) {
    const int64_t tok = base + (threadIdx.x >> a.lanes_log2);
    const bool in = tok < a.tokens;
    typename P::Raw xl[U][S], xh[U][S];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < S; ++k) {
        xl[u][k] = xh[u][k] = typename P::Raw{};
        if (in && u < heads && lane + (k << a.lanes_log2) < a.slots) {
          xl[u][k] = P::load_once(x + u * a.D + col[k]);
          xh[u][k] = P::load_once(x + u * a.D + col[k] + apart[k]);
        }
      }
    V c[S], s[S];
    const bool good = qk_angles<T, S, NV>(a, tok, turn.pos, in, lane, c, s);
    turn.next(a);
    float sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      E all = E::make(0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < S; ++k) {
        V vx, vy;
        P::unpack(xl[u][k], vx);
        P::unpack(xh[u][k], vy);
#pragma unroll
        for (int i = 0; i < V::N; ++i) all = qk_fma(vx.e[i], vx.e[i], qk_fma(vy.e[i], vy.e[i], all));
      }
      sum[u] = all.sum();
    }
    for (int o = (1 << a.lanes_log2) >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in || u >= heads) continue;
      const float inv = rsqrtf(sum[u] * over + a.eps);
      const E by = E::make(inv, inv);
#pragma unroll
      for (int k = 0; k < S; ++k) {
        if (lane + (k << a.lanes_log2) >= a.slots) continue;
        V vx, vy;
        P::unpack(xl[u][k], vx);
        P::unpack(xh[u][k], vy);
#pragma unroll
        for (int i = 0; i < V::N; ++i) {
          vx.e[i] = qk_mul(qk_mul(vx.e[i], by), glo[k].e[i]);
          vy.e[i] = qk_mul(qk_mul(vy.e[i], by), ghi[k].e[i]);
        }
        if (turns[k]) {
#pragma unroll
          for (int i = 0; i < V::N; ++i) {
            const E xn = vx.e[i], yn = vy.e[i];
            vx.e[i] = qk_fma(xn, c[k].e[i], qk_mul(yn, qk_mul(s[k].e[i], minus)));
            vy.e[i] = qk_fma(yn, c[k].e[i], qk_mul(xn, qk_mul(s[k].e[i], sign)));
          }
        }
        if (!good) {
          vx.fill(0.0f);
          vy.fill(0.0f);
        }
        T* d = out + u * a.D + col[k];
        P::template store<true>(d, vx);
        P::template store<true>(d + apart[k], vy);
      }
    }
    x += stride * q.x_stride;
    out += stride * q.y_stride;
  }
}

// W: the gradients of the weights are wanted (of either side).  A group goes from token to token, with the sums of its columns in
// registers.  What keeps memory busy is blocks, not packets a token ahead: with those, registers leave half of the blocks (187 us
// instead of 165 for 16 x 2048 tokens of 2 x 10 heads fp32).  bf16 rows get three or two blocks to an SM by the bound on registers (heads of 80 columns, 40 of
// which rotate, S = 3: 188 -> 92 us); fp32 ones that many by themselves, and three are too many (177 us), as is a hint that they leave the cache.
template <typename T, int NV, int S, int U, bool W>
__global__ void __launch_bounds__(QK_THREADS, sizeof(T) == 4 || S * NV > 12 ? 1 : S == 1 ? 3 : 2) qk_backward_kernel(const QkArgs a) {
  using P = QkPack<T, NV>;
  extern __shared__ float qk_smem[];  // W: [warps][D]
  ag_pdl_wait();
  ag_pdl_trigger();
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const int per_block = QK_THREADS >> a.lanes_log2;
  const int which = (int)blockIdx.y >= a.side[0].blocks;
  const QkSide& q = a.side[which];
  const int head = ((int)blockIdx.y - (which ? a.side[0].blocks : 0)) * U, heads = min(U, q.heads - head);
  using V = QkVec<T, NV>;
  using E = typename V::E;
  V glo[S], ghi[S];
  qk_gamma<T, S, NV>(a, q.gamma, lane, glo, ghi);
  int col[S], apart[S];
  bool turns[S];
#pragma unroll
  for (int k = 0; k < S; ++k) qk_columns(a, (lane + (k << a.lanes_log2)) * NV, turns[k], col[k], apart[k]);
  V dlo[W ? S : 1], dhi[W ? S : 1];
#pragma unroll
  for (int k = 0; k < (W ? S : 1); ++k) {
    dlo[k].fill(0.0f);
    dhi[k].fill(0.0f);
  }
  const float over = 1.0f / (float)a.D;
  const int64_t first = (int64_t)blockIdx.x * per_block + (threadIdx.x >> a.lanes_log2), stride = (int64_t)gridDim.x * per_block;
  const T* x = static_cast<const T*>(q.x) + first * q.x_stride + (int64_t)head * a.D;
  const T* dy = static_cast<const T*>(q.dy) + first * q.dy_stride + (int64_t)head * a.D;
  T* out = static_cast<T*>(q.y) + first * q.y_stride + (int64_t)head * a.D;
  QkTurn turn(a, first, stride);
  const E sign = E::make(a.sgn, a.sgn), minus = E::make(-a.sgn, -a.sgn);
  constexpr bool ONCE = sizeof(T) == 2;  // see above
  // What turns, and what has a place, is selected in fp32 rows where a lane has four pairs of columns or fewer, and branched on elsewhere
  // (16 x 2048 tokens of 2 x 10 heads fp32: 166.6 us with selects, 168.9 with branches; heads of 74 columns 143 and 149, heads of 80, 40 of which
  // rotate, twelve pairs of columns to a lane, 150.6 and 149.0)
  constexpr bool SELECT = sizeof(T) == 4 && S * NV <= 4;
  auto fetch = [](const T* p) {
    if constexpr (ONCE) return P::load_once(p);
    else return P::load(p);
  };
  // all threads of a block make as many turns: the sums are over groups of lanes
  for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.tokens; base += stride) {
    const int64_t tok = base + (threadIdx.x >> a.lanes_log2);
    const bool in = tok < a.tokens;
    typename P::Raw xl[U][S], xh[U][S], gl[U][S], gh[U][S];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < S; ++k) {
        xl[u][k] = xh[u][k] = gl[u][k] = gh[u][k] = typename P::Raw{};
        if (in && u < heads && lane + (k << a.lanes_log2) < a.slots) {
          const int at = u * a.D + col[k];
          xl[u][k] = fetch(x + at);
          xh[u][k] = fetch(x + at + apart[k]);
          gl[u][k] = fetch(dy + at);
          gh[u][k] = fetch(dy + at + apart[k]);
        }
      }
    V c[S], s[S];
    const bool good = qk_angles<T, S, NV>(a, tok, turn.pos, in, lane, c, s);
    turn.next(a);
    x += stride * q.x_stride;
    dy += stride * q.dy_stride;
    V vx[U][S], vy[U][S], wl[U][S], wh[U][S];
    float sum[U], dot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      E squares = E::make(0.0f, 0.0f), products = squares;
#pragma unroll
      for (int k = 0; k < S; ++k) {
        P::unpack(xl[u][k], vx[u][k]);
        P::unpack(xh[u][k], vy[u][k]);
        P::unpack(gl[u][k], wl[u][k]);
        P::unpack(gh[u][k], wh[u][k]);
        if (SELECT || turns[k]) {
#pragma unroll
          for (int i = 0; i < V::N; ++i) {
            const E p = wl[u][k].e[i], r = wh[u][k].e[i];
            const E tl = qk_fma(p, c[k].e[i], qk_mul(r, qk_mul(s[k].e[i], sign)));
            const E th = qk_fma(r, c[k].e[i], qk_mul(p, qk_mul(s[k].e[i], minus)));
            wl[u][k].e[i] = !SELECT || turns[k] ? tl : p;
            wh[u][k].e[i] = !SELECT || turns[k] ? th : r;
          }
        }
#pragma unroll
        for (int i = 0; i < V::N; ++i) {
          squares = qk_fma(vx[u][k].e[i], vx[u][k].e[i], qk_fma(vy[u][k].e[i], vy[u][k].e[i], squares));
          products = qk_fma(vx[u][k].e[i], qk_mul(wl[u][k].e[i], glo[k].e[i]), products);
          products = qk_fma(vy[u][k].e[i], qk_mul(wh[u][k].e[i], ghi[k].e[i]), products);
        }
      }
      sum[u] = squares.sum();
      dot[u] = products.sum();
    }
    for (int o = (1 << a.lanes_log2) >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
        dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!in || u >= heads) continue;
      const float inv = rsqrtf(sum[u] * over + a.eps);
      const float back = -(inv * inv * (dot[u] * over));
      const E by = E::make(inv, inv), less = E::make(back, back);
#pragma unroll
      for (int k = 0; k < S; ++k) {
        if (lane + (k << a.lanes_log2) >= a.slots) continue;
        T* d = out + u * a.D + col[k];
        V ol, oh;
        if (SELECT || good) {
#pragma unroll
          for (int i = 0; i < V::N; ++i) {
            const E xi = vx[u][k].e[i], yi = vy[u][k].e[i], wi = wl[u][k].e[i], ui = wh[u][k].e[i];
            if (W && (!SELECT || good)) {
              dlo[k].e[i] = qk_fma(wi, qk_mul(xi, by), dlo[k].e[i]);
              dhi[k].e[i] = qk_fma(ui, qk_mul(yi, by), dhi[k].e[i]);
            }
            ol.e[i] = qk_mul(by, qk_fma(wi, glo[k].e[i], qk_mul(xi, less)));
            oh.e[i] = qk_mul(by, qk_fma(ui, ghi[k].e[i], qk_mul(yi, less)));
          }
        }
        if (!good) {
          ol.fill(0.0f);
          oh.fill(0.0f);
        }
        if (a.accumulate) {
          V pl, ph;
          P::unpack(P::load(d), pl);
          P::unpack(P::load(d + apart[k]), ph);
#pragma unroll
          for (int i = 0; i < V::N; ++i) ol.e[i] = qk_add(ol.e[i], pl.e[i]), oh.e[i] = qk_add(oh.e[i], ph.e[i]);
        }
        P::template store<ONCE>(d, ol);
        P::template store<ONCE>(d + apart[k], oh);
      }
    }
    out += stride * q.y_stride;
  }
  if constexpr (W) {
    // the groups of a warp, then the warps, in a fixed order
    const int warp = threadIdx.x >> 5, wl = threadIdx.x & 31;
    float* mine = qk_smem + warp * a.D;
#pragma unroll
    for (int k = 0; k < S; ++k) {
      const int slot = lane + (k << a.lanes_log2);
      bool turns;
      int col, apart;
      qk_columns(a, slot * NV, turns, col, apart);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        constexpr int EACH = V::TWO ? 2 : 1;
        float of_lo[2] = {}, of_hi[2] = {};
        dlo[k].e[i / EACH].get(of_lo[0], of_lo[1]);
        dhi[k].e[i / EACH].get(of_hi[0], of_hi[1]);
        float u = of_lo[i % EACH], v = of_hi[i % EACH];
        for (int o = 16; o >= (1 << a.lanes_log2); o >>= 1) {
          u += __shfl_xor_sync(0xffffffffu, u, o);
          v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        if (wl < (1 << a.lanes_log2) && slot < a.slots) {
          mine[col + i] = u;
          mine[col + apart + i] = v;
        }
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += QK_THREADS) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < QK_THREADS / 32; ++w) t += qk_smem[w * a.D + d];
      a.partials[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.D + d] = t;
    }
  }
}

// dgamma += the partial rows of its side: those of queries are the first (one weight for both sides: all rows are its).  A block has 32 columns of one side, its warps take rows in
// turn, eight under way each (one at a time, of eight warps, took 72 us for 1183 rows of 128).
constexpr int QK_FOLD_WARPS = 32;
__global__ void __launch_bounds__(32 * QK_FOLD_WARPS) qk_fold_kernel(const float* __restrict__ partials, int q_rows, int k_rows, int D,
                                                                     float* dq_gamma, float* dk_gamma) {
  __shared__ float part[QK_FOLD_WARPS][33];
  ag_pdl_wait();
  ag_pdl_trigger();
  float* out = blockIdx.y ? dk_gamma : dq_gamma;
  if (!out) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = blockIdx.x * 32 + lane;
  const int rows = blockIdx.y ? k_rows : q_rows;
  const float* p = partials + (blockIdx.y ? (int64_t)q_rows * D : 0) + d;
  float t = 0.0f;
  for (int r = warp; r < rows; r += 8 * QK_FOLD_WARPS) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = d < D && r + k * QK_FOLD_WARPS < rows ? p[(int64_t)(r + k * QK_FOLD_WARPS) * D] : 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += v[k];
  }
  part[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && d < D) {
    t = 0.0f;
#pragma unroll
    for (int w = 0; w < QK_FOLD_WARPS; ++w) t += part[w][lane];
    out[d] += t;
  }
}

// ---------------------------------------------------------------------------- host side
struct QkShape {
  int nv, lanes_log2, S;
};

// The widest packets that everything allows, then lanes and slots with as few idle ones as possible
template <typename T>
QkShape qk_shape(const QkArgs& a) {
  int nv = 4;
  auto fits = [&](int n) {
    if (a.half % n || ((a.D >> 1) - a.half) % n) return false;
    const uintptr_t bytes = n * sizeof(T), wide = n >= 4 ? 15u : 3u;
    uintptr_t f = (uintptr_t)a.cos_tab | (uintptr_t)a.sin_tab;
    for (const QkSide& q : a.side) {
      if (!q.x) continue;
      if ((((uintptr_t)q.x | (uintptr_t)q.dy | (uintptr_t)q.y) & (bytes - 1)) || q.x_stride % n || q.dy_stride % n || q.y_stride % n)
        return false;
      f |= (uintptr_t)q.gamma;
    }
    return (f & wide) == 0;
  };
  while (nv > 1 && !fits(nv)) nv >>= 1;
  const int slots = a.D / 2 / nv;
  QkShape best = {nv, 0, 0};
  int best_cost = 1 << 30;
  for (int s = 1; s <= 16; s = s < 4 ? s + 1 : s * 2)
    for (int g = 0; g <= 5; ++g)
      if ((s << g) >= slots) {
        const int cost = (s << g) * 8 + s;
        if (cost < best_cost) best_cost = cost, best = {nv, g, s};
        break;
      }
  return best;
}

template <typename T, int NV, int S, int U, bool BACK, bool W>
int qk_launch(ag_ctx* ctx, QkArgs& a, const QkShape& sh) {
  for (QkSide& q : a.side) q.blocks = q.x ? (q.heads + U - 1) / U : 0;
  const int gy = a.side[0].blocks + a.side[1].blocks, per_block = QK_THREADS >> sh.lanes_log2;
  AG_REQUIRE(ctx, gy <= 65535, "too many heads");
  int64_t gx = (a.tokens + per_block - 1) / per_block;
  const size_t smem = BACK && W ? QK_THREADS / 32 * a.D * sizeof(float) : 0;
  // blocks that are resident at once, with as many turns each
  static AgOccupancy known[AG_MAX_DEVICES];
  const auto resident = [&] {
    int n = 0;
    cudaError_t e;
    if constexpr (BACK) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, qk_backward_kernel<T, NV, S, U, W>, QK_THREADS, smem);
    else e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, qk_forward_kernel<T, NV, S, U>, QK_THREADS, smem);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    return n;
  };
  int occ = known[ag_dev_slot(ctx)].get(QK_THREADS, smem, resident);
  occ = occ < 1 ? 1 : occ > QK_BLOCKS_PER_SM ? QK_BLOCKS_PER_SM : occ;
  const int64_t most = ctx->sm_count * occ / gy > 0 ? ctx->sm_count * occ / gy : 1, turns = (gx + most - 1) / most;
  gx = (gx + turns - 1) / turns;
  if constexpr (!BACK) {
    AG_LAUNCH_PDL(ctx, "qk_forward_kernel", (qk_forward_kernel<T, NV, S, U>), dim3((unsigned)gx, gy), QK_THREADS, 0, a);
  } else {
    AG_LAUNCH_PDL(ctx, "qk_backward_kernel", (qk_backward_kernel<T, NV, S, U, W>), dim3((unsigned)gx, gy), QK_THREADS, smem, a);
    if (W) {
      const int q_rows = (int)gx * a.side[0].blocks, k_rows = (int)gx * a.side[1].blocks;
      const bool one = a.side[0].dgamma == a.side[1].dgamma;
      AG_LAUNCH_PDL(ctx, "qk_fold_kernel", qk_fold_kernel, dim3((a.D + 31) / 32, one ? 1 : 2), 32 * QK_FOLD_WARPS, 0, a.partials,
                    one ? q_rows + k_rows : q_rows, k_rows, a.D, a.side[0].dgamma, a.side[1].dgamma);
    }
  }
  return AG_OK;
}

// Heads that a thread has under way.  Forward, two where a lane has 16 bytes of a half or fewer, else one (16 x 2048 tokens of 2 x 10 heads of 128
// with two, one and four: fp32 108, 114 and 116 us, bf16 71, 84 and 77; heads of 256 columns fp32 214, 214 and 230).  Backward, two where a
// lane has four pairs of columns or fewer, else one (with two and one: the same tokens fp32 164 and 174 us, bf16 112 and 136; 8192 of 12 + 2
// heads bf16 26 and 30).
template <typename T, int NV, int S>
int qk_kind(ag_ctx* ctx, QkArgs& a, const QkShape& sh, bool back, bool w) {
  constexpr int BYTES = S * NV * (int)sizeof(T), U = BYTES < 32 ? 2 : 1, B = S * NV <= 4 ? 2 : 1;
  if (!back) return qk_launch<T, NV, S, U, false, false>(ctx, a, sh);
  return w ? qk_launch<T, NV, S, B, true, true>(ctx, a, sh) : qk_launch<T, NV, S, B, true, false>(ctx, a, sh);
}

template <typename T, int NV>
int qk_slots(ag_ctx* ctx, QkArgs& a, const QkShape& sh, bool back, bool w) {
  a.lanes_log2 = sh.lanes_log2;
  a.slots = a.D / 2 / NV;
  switch (sh.S) {
    case 1: return qk_kind<T, NV, 1>(ctx, a, sh, back, w);
    case 2: return qk_kind<T, NV, 2>(ctx, a, sh, back, w);
    case 3: return qk_kind<T, NV, 3>(ctx, a, sh, back, w);
    case 4: return qk_kind<T, NV, 4>(ctx, a, sh, back, w);
  }
  if constexpr (NV < 4) {  // packets of four: 32 lanes of 4 slots hold 1024 columns
    if (sh.S == 8) return qk_kind<T, NV, 8>(ctx, a, sh, back, w);
    if constexpr (NV == 1)
      if (sh.S == 16) return qk_kind<T, NV, 16>(ctx, a, sh, back, w);
  }
  AG_FAIL(ctx, AG_ERR_INVALID, "no kernel for heads of %d columns", a.D);
}

template <typename T>
int qk_run(ag_ctx* ctx, QkArgs& a, bool back, bool w) {
  const QkShape sh = qk_shape<T>(a);
  switch (sh.nv) {
    case 1: return qk_slots<T, 1>(ctx, a, sh, back, w);
    case 2: return qk_slots<T, 2>(ctx, a, sh, back, w);
    default: return qk_slots<T, 4>(ctx, a, sh, back, w);
  }
}

// Rows of `width` elements, `stride` apart
struct QkRows {
  const void* p;
  int64_t stride, width;
};

// Whether two sets of rows share an element: not if their ranges are apart, nor if rows of the same stride lie beside each
// other (slices of one packed row)
bool qk_overlap(const QkRows& x, const QkRows& y, int64_t rows, int64_t size) {
  if (!x.p || !y.p) return false;
  const int64_t a = (int64_t)(uintptr_t)x.p, b = (int64_t)(uintptr_t)y.p;
  const int64_t a_end = a + ((rows - 1) * x.stride + x.width) * size, b_end = b + ((rows - 1) * y.stride + y.width) * size;
  if (a_end <= b || b_end <= a) return false;
  if (x.stride != y.stride) return true;
  const int64_t pitch = x.stride * size, off = (((b - a) % pitch) + pitch) % pitch;  // of y's rows behind x's
  return off < x.width * size || off + y.width * size > pitch;
}

int qk_check(ag_ctx* ctx, const char* name, const QkArgs& a, int seq, int rot, float eps, int dtype, bool back) {
  AG_REQUIRE(ctx, a.tokens > 0 && a.tokens < (1ll << 31), "%s: bad number of tokens %lld", name, (long long)a.tokens);
  AG_REQUIRE(ctx, a.D > 0 && a.D <= AG_QK_MAX_D && a.D % 2 == 0, "%s: heads of %d columns (even, at most %d)", name, a.D, AG_QK_MAX_D);
  AG_REQUIRE(ctx, rot >= 0 && rot <= a.D && rot % 2 == 0, "%s: %d of %d columns rotate", name, rot, a.D);
  AG_REQUIRE(ctx, dtype == AG_F32 || dtype == AG_BF16, "%s: unknown dtype %d", name, dtype);
  AG_REQUIRE(ctx, eps >= 0.0f && eps <= 1e30f, "%s: eps %g", name, (double)eps);
  AG_REQUIRE(ctx, rot == 0 || (a.cos_tab && a.sin_tab), "%s: null table", name);
  AG_REQUIRE(ctx, rot == 0 || (a.rows > 0 && (a.positions || (seq > 0 && seq <= a.rows))),
             "%s: sequences of %d positions, tables of %d", name, seq, a.rows);
  AG_REQUIRE(ctx, a.side[0].x || a.side[1].x, "%s: neither queries nor keys", name);
  const int64_t size = dtype == AG_F32 ? 4 : 2;
  for (const QkSide& q : a.side) {
    if (!q.x) continue;
    AG_REQUIRE(ctx, q.y && (!back || q.dy), "%s: null pointer", name);
    AG_REQUIRE(ctx, q.heads > 0 && q.heads <= 65535, "%s: %d heads", name, q.heads);
    const int64_t w = (int64_t)q.heads * a.D;
    AG_REQUIRE(ctx, q.x_stride >= w && q.y_stride >= w && (!back || q.dy_stride >= w), "%s: token stride smaller than heads * D", name);
    AG_REQUIRE(ctx, q.x_stride < (1ll << 31) && q.y_stride < (1ll << 31) && q.dy_stride < (1ll << 31), "%s: token stride too large", name);
    AG_REQUIRE(ctx, (((uintptr_t)q.x | (uintptr_t)q.y | (uintptr_t)q.dy) & (size - 1)) == 0 &&
                        (((uintptr_t)q.gamma | (uintptr_t)q.dgamma) & 3) == 0, "%s: misaligned pointer", name);
  }
  AG_REQUIRE(ctx, (((uintptr_t)a.cos_tab | (uintptr_t)a.sin_tab | (uintptr_t)a.positions) & 3) == 0, "%s: misaligned table", name);
  const uintptr_t dg[2] = {(uintptr_t)a.side[0].dgamma, (uintptr_t)a.side[1].dgamma}, wide = (uintptr_t)a.D * 4;
  AG_REQUIRE(ctx, !dg[0] || !dg[1] || dg[0] == dg[1] || dg[0] + wide <= dg[1] || dg[1] + wide <= dg[0],
             "%s: the weights' gradients overlap", name);
  // an output may be one of its own side's inputs, row by row; otherwise it shares nothing with any operand
  for (int i = 0; i < 2; ++i) {
    const QkSide& q = a.side[i];
    if (!q.x) continue;
    const QkRows out = {q.y, q.y_stride, (int64_t)q.heads * a.D};
    for (int j = 0; j < 2; ++j) {
      const QkSide& o = a.side[j];
      if (!o.x) continue;
      const QkRows rows[3] = {{o.x, o.x_stride, (int64_t)o.heads * a.D},
                              {back ? o.dy : nullptr, o.dy_stride, (int64_t)o.heads * a.D},
                              {i != j ? o.y : nullptr, o.y_stride, (int64_t)o.heads * a.D}};
      for (const QkRows& r : rows) {
        const bool same = i == j && r.p == q.y && r.stride == q.y_stride;
        AG_REQUIRE(ctx, same || !qk_overlap(out, r, a.tokens, size), "%s: an output overlaps another operand", name);
      }
    }
  }
  return AG_OK;
}

}  // namespace

extern "C" int ag_qk_norm_rope_forward(ag_ctx* ctx, const void* q, const void* k, const float* q_gamma, const float* k_gamma,
                                       const float* cos_tab, const float* sin_tab, const int32_t* positions, void* q_out,
                                       void* k_out, int64_t tokens, int seq, int table_rows, int H, int HKV, int D, int rot,
                                       int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                                       float eps, int sin_sign, int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  if (tokens == 0) return AG_OK;
  QkArgs a = {};
  a.side[0] = {q, nullptr, q_out, q_gamma, nullptr, q_stride, 0, q_out_stride, H, 0};
  a.side[1] = {k, nullptr, k_out, k_gamma, nullptr, k_stride, 0, k_out_stride, HKV, 0};
  a.cos_tab = cos_tab; a.sin_tab = sin_tab; a.positions = positions;
  a.tokens = tokens; a.seq = seq; a.rows = table_rows; a.D = D; a.half = rot / 2;
  a.eps = eps; a.sgn = sin_sign >= 0 ? 1.0f : -1.0f; a.status = ctx->d_status;
  if (int rc = qk_check(ctx, "ag_qk_norm_rope_forward", a, seq, rot, eps, dtype, false)) return rc;
  if (rot == 0) a.cos_tab = a.sin_tab = nullptr;
  return dtype == AG_F32 ? qk_run<float>(ctx, a, false, false) : qk_run<__nv_bfloat16>(ctx, a, false, false);
}

extern "C" size_t ag_qk_norm_partials_bytes(ag_ctx* ctx, int H, int HKV, int D) {
  if (!ctx || D <= 0 || H < 0 || HKV < 0) return 0;
  // a row of D per block: QK_BLOCKS_PER_SM of them per SM, or one per head where there are more heads
  const int64_t blocks = (int64_t)ctx->sm_count * QK_BLOCKS_PER_SM, heads = (int64_t)H + HKV;
  return (size_t)((blocks > heads ? blocks : heads) * D) * sizeof(float);
}

extern "C" int ag_qk_norm_rope_backward(ag_ctx* ctx, const void* dq_out, const void* dk_out, const void* q, const void* k,
                                        const float* q_gamma, const float* k_gamma, const float* cos_tab,
                                        const float* sin_tab, const int32_t* positions, void* dq, void* dk,
                                        float* dq_gamma, float* dk_gamma, void* partials, size_t partials_bytes,
                                        int64_t tokens, int seq, int table_rows, int H, int HKV, int D, int rot,
                                        int64_t dq_out_stride, int64_t dk_out_stride, int64_t q_stride, int64_t k_stride,
                                        int64_t dq_stride, int64_t dk_stride, float eps, int sin_sign, int accumulate,
                                        int dtype) {
  if (!ctx) return AG_ERR_INVALID;
  if (tokens == 0) return AG_OK;
  QkArgs a = {};
  a.side[0] = {q, dq_out, dq, q_gamma, q ? dq_gamma : nullptr, q_stride, dq_out_stride, dq_stride, H, 0};
  a.side[1] = {k, dk_out, dk, k_gamma, k ? dk_gamma : nullptr, k_stride, dk_out_stride, dk_stride, HKV, 0};
  a.cos_tab = cos_tab; a.sin_tab = sin_tab; a.positions = positions;
  a.tokens = tokens; a.seq = seq; a.rows = table_rows; a.D = D; a.half = rot / 2;
  a.eps = eps; a.sgn = sin_sign >= 0 ? 1.0f : -1.0f; a.status = ctx->d_status; a.accumulate = accumulate != 0;
  if (int rc = qk_check(ctx, "ag_qk_norm_rope_backward", a, seq, rot, eps, dtype, true)) return rc;
  if (rot == 0) a.cos_tab = a.sin_tab = nullptr;
  const bool w = a.side[0].dgamma || a.side[1].dgamma;
  if (w) {
    const size_t need = ag_qk_norm_partials_bytes(ctx, q ? H : 0, k ? HKV : 0, D);
    AG_REQUIRE(ctx, partials && ((uintptr_t)partials & 3) == 0, "ag_qk_norm_rope_backward: weight gradients need partials");
    if (partials_bytes < need)
      AG_FAIL(ctx, AG_ERR_SCRATCH, "ag_qk_norm_rope_backward: %zu bytes of partials, %zu needed", partials_bytes, need);
    a.partials = static_cast<float*>(partials);
  }
  return dtype == AG_F32 ? qk_run<float>(ctx, a, true, w) : qk_run<__nv_bfloat16>(ctx, a, true, w);
}
