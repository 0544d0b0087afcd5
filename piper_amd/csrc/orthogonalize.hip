// Newton-Schulz orthogonalization of matrices, and the optimizer step built on it.
//
//   X = U / max(|U|_F, eps);   `steps` times:  A = X X^T,  B = a + b A + c A A,  X <- B X
//
// An odd polynomial of X's singular values, applied again and again, which drives them towards 1 without computing them.  U [r, c]
// is worked on with the shorter side as rows: X [m, n], m = min(r, c).  The step: m <- m + (1 - mu)(g - m), U = g + mu (m - g)
// (nesterov; otherwise m), w <- w (1 - lr decay) - lr s X.
//
// Numbers.  X lives between the products as two planes of fp16 (hi + lo: 22 bits), scaled by a power of two so that its typical
// value is near 1, A times 2^8, B as it is: their values are at most a few units and their absolute error is what counts beside
// a X.  All sums are fp32.  Results take three products, hi hi + lo hi + hi lo, of all operands: 1e-6 to 2e-6 off, what products in fp32
// give or less, in a third of the time of fp32 instructions; a bf16 result is then the rounding of one in fp32 (1.7e-3 off 64 bits).
//
// Where the caller asks for it, single products, of the upper planes alone, with a X from both: a third of the matrix operations.  An
// error of a product is bounded by the strong directions and turns them a little, while an error of X itself, a full matrix of noise, grows
// with the weak ones, up to 3.4 times a step.  (256 x 683, relative to 64 bits: gradients with 8 strong directions 4e-4 as here, 0.04
// with X in one plane, 0.3 with everything in bf16; random ones 1.7e-3.)  Errors of a few directions do not average out: matrices with
// few rows that are not zero 2e-3 to 7e-3, scaled identities up to 0.012, any one direction below 0.04.  Those with a side of
// at most 128 take three products in any case, as they cost next to nothing.
//
// Work is laid out for many matrices: a launch runs one product of all matrices of a group, as many as the workspace holds.  Padded
// to multiples of 128 with zeros there (zeros stay zeros under the products), so that only the first and the last kernel see
// where a matrix ends.
#include "pk_common.h"
#include "lds_tiles.h"
#include "launch_rules.h"
#include <algorithm>
#include <cmath>
#include <limits>

namespace {

using namespace pk_lds;

typedef _Float16 f16_t;
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

constexpr int kPad = 128;
// Stacks of matrices in a launch of the kernels at both ends, these launches in a group, and sizes in one of a product: keeps the kernels'
// arguments below 4 KiB.
constexpr int kMaxEntries = 40, kMaxEnds = 8, kMaxShapes = 100;
constexpr int kChunk = 8192;                 // elements a workgroup of begin_kernel takes
constexpr int kThreads = 256;
// Workspace that is asked for.  Groups that stay in the 256 MiB memory-side cache leave too few workgroups a launch, whose last round is
// rarely full: 128 matrices of 768 x 2048, single / three products, ms with 192 MiB 8.1 / 12.8, 384 6.2 / 11.4, 768 5.4 / 11.0, 1,536 5.0 / 9.9, 2,560 4.5 / 9.6.
constexpr int64_t kGroupBytes = 2560ll << 20;

// Matrices of one shape that lie one behind the other, as the kernels at both ends see them.
struct Entry {
  const void* src;       // what is orthogonalized, or the gradients (may be null: zeros)
  float* flat;           // step: fp32 gradients to add to them (may be null)
  float* momentum;       // step only
  float* master;         // step only
  void* out;             // the result, or the step's bf16 weights (may be null)
  int64_t ws;            // bytes from the workspace to the first matrix's buffers
  int32_t rows, cols, count;
  int32_t mp, np;        // padded sides, mp the shorter
  int32_t first_chunk, first_tile;
  float rate;            // step: lr * s
};
struct Ends {
  Entry e[kMaxEntries];
  char* ws;
  int32_t n;
  float mu, keep, eps;   // keep: 1 - lr decay
  int32_t nesterov, zero_flat, precise;
};
static_assert(sizeof(Ends) <= 4096, "kernel arguments");
struct Gemm {
  // (first_unit: the number of matrices, until they are numbered; first_k: with shares, the pairs of k-tiles before the shape's first unit)
  struct Shape { int64_t ws, stride; int32_t mp, np, first_unit, first_k; } e[kMaxShapes];
  char* ws;
  int32_t n, units, blocks, chunk, wide;      // blocks: of units in the order they are dealt
  int32_t shares, pairs, slots;               // X X^T in shares of all units' pairs of k-tiles; a unit's sums lie in `slots` places
  int32_t from;          // which of the two X the products read
  int32_t lower;         // whether UPDATE's result needs its lower plane
  float a, b, c;
};
static_assert(sizeof(Gemm) <= 4096, "kernel arguments");

// X is held times 2^12 and A times 2^8: elements of large normalised matrices are small, as A's off the diagonal are, and
// the lower plane of a small one would be below fp16's range.  Singular values up to 15 stay in it (2^12 * 15 and 2^8 * 15^2 are below
// 65504), and calls whose coefficients may lead past that are refused (settings_ok); those of the usual ones stay below 1.3.
constexpr int kXLog2 = 12, kALog2 = 8;
constexpr float kX = 1 << kXLog2, kA = 1 << kALog2;

// Buffers of one matrix: X twice, each as hi and lo; A, B (with precise sums hi and lo); for each wave of the 128 x 128 tiles on and below A's
// diagonal, how many sums of shares of k there are; partial sums of squares.
__host__ __device__ inline int64_t plane_x(int mp, int np) { return (int64_t)mp * np * 2; }
__host__ __device__ inline int64_t plane_a(int mp) { return (int64_t)mp * mp * 2; }
__host__ __device__ inline int64_t at_a(int mp, int np) { return 4 * plane_x(mp, np); }
__host__ __device__ inline int64_t at_b(int mp, int np, bool precise) { return at_a(mp, np) + (precise ? 2 : 1) * plane_a(mp); }
__host__ __device__ inline int64_t at_counts(int mp, int np, bool precise) { return at_a(mp, np) + (precise ? 4 : 2) * plane_a(mp); }
__host__ __device__ inline int64_t counts_of(int mp) { return (int64_t)(mp / 128) * (mp / 128 + 1) / 2 * 8; }
__host__ __device__ inline int64_t at_sums(int mp, int np, bool precise) { return at_counts(mp, np, precise) + counts_of(mp) * 4; }
__host__ __device__ inline int64_t matrix_bytes(int rows, int cols, int mp, int np, bool precise) {
  const int64_t chunks = ((int64_t)rows * cols + kChunk - 1) / kChunk;
  return (at_sums(mp, np, precise) + chunks * 8 + 255) / 256 * 256;
}
// Where element (row, col) of a matrix of ld columns is, in fp16 values from its first one, and its lower part from there.  Single products
// read the upper plane alone: one plane behind the other.  Three products read both: 32 columns of one, then of the other, so that a k-tile
// of both is 128 consecutive bytes of a row.
__host__ __device__ inline int64_t place(bool precise, int row, int col, int ld) {
  return precise ? (int64_t)row * 2 * ld + (col >> 5) * 64 + (col & 31) : (int64_t)row * ld + col;
}
__host__ __device__ inline int64_t to_lower(bool precise, int rows, int ld) { return precise ? 32 : (int64_t)rows * ld; }

template <typename F>
__device__ __forceinline__ int entry_of(int n, int block, F&& first) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first(mid) <= block) lo = mid; else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------- the ends
// Memory bounds them: 128 matrices of 768 x 2048 in bf16 90 + 256 + 232 us (4.5, 4.7, 5.2 TB/s), a step of 170 million bf16 values 336 + 359 + 487.
// N neighbouring values at p as fp32; VEC: p is on a boundary of their size.
template <int N, bool VEC, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
  typedef T vec_t __attribute__((ext_vector_type(VEC ? (sizeof(T) == 2 ? N : 4) : 1)));
  constexpr int PER = VEC ? (sizeof(T) == 2 ? N : 4) : 1;
#pragma unroll
  for (int v = 0; v < N / PER; ++v) {
    const vec_t t = reinterpret_cast<const vec_t*>(p)[v];
#pragma unroll
    for (int k = 0; k < PER; ++k) x[v * PER + k] = (float)t[k];
  }
}
template <int N, bool VEC, typename T>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
  typedef T vec_t __attribute__((ext_vector_type(VEC ? (sizeof(T) == 2 ? N : 4) : 1)));
  constexpr int PER = VEC ? (sizeof(T) == 2 ? N : 4) : 1;
#pragma unroll
  for (int v = 0; v < N / PER; ++v) {
    vec_t t;
#pragma unroll
    for (int k = 0; k < PER; ++k) t[k] = (T)x[v * PER + k];
    reinterpret_cast<vec_t*>(p)[v] = t;
  }
}
// Whether every buffer of an entry has 16-byte boundaries where a multiple of `piece` elements begins in a matrix.
__device__ __forceinline__ bool aligned(const Entry& e, int piece) {
  return ((reinterpret_cast<uintptr_t>(e.src) | reinterpret_cast<uintptr_t>(e.flat) | reinterpret_cast<uintptr_t>(e.momentum) |
           reinterpret_cast<uintptr_t>(e.master) | reinterpret_cast<uintptr_t>(e.out)) & 15u) == 0 && piece;
}
// The gradients of elements i .. i + N - 1 of an entry; the momentum after this step and U, from the momentum before.
template <int N, bool VEC, typename TG>
__device__ __forceinline__ void gradient(const Entry& e, int64_t i, float (&g)[N]) {
  float f[N] = {};
#pragma unroll
  for (int k = 0; k < N; ++k) g[k] = 0.f;
  if (e.flat) load_n<N, VEC>(e.flat + i, f);
  if (e.src) load_n<N, VEC>(reinterpret_cast<const TG*>(e.src) + i, g);
  if (e.flat) {
#pragma unroll
    for (int k = 0; k < N; ++k) g[k] = f[k] + g[k];
  }
}
__device__ __forceinline__ float next_momentum(float m, float g, float mu) { return m + (1.f - mu) * (g - m); }
__device__ __forceinline__ float update_of(float m, float g, float mu, bool nesterov) { return nesterov ? g + mu * (m - g) : m; }

template <int N, bool VEC, typename TG, bool STEP>
__device__ __forceinline__ void begin_piece(const Ends& p, const Entry& e, int64_t i, double& sum) {
  float u[N];
  gradient<N, VEC, TG>(e, i, u);
  if (STEP) {
    float m[N];
    load_n<N, VEC>(e.momentum + i, m);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      m[k] = next_momentum(m[k], u[k], p.mu);
      u[k] = update_of(m[k], u[k], p.mu, p.nesterov);
    }
    store_n<N, VEC>(e.momentum + i, m);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sum += (double)u[k] * u[k];
}

// Momentum, and the sum of squares of every chunk of a matrix of U, in 64 bits (squares of fp32 values reach past fp32's range); counts of
// zero.
template <typename TG, bool STEP>
__global__ __launch_bounds__(kThreads) void begin_kernel(const Ends p) {
  __shared__ double part[kThreads / 64];
  const int en = entry_of(p.n, blockIdx.x, [&](int i) { return p.e[i].first_chunk; });
  const Entry& e = p.e[en];
  const int64_t size = (int64_t)e.rows * e.cols;
  const int chunks = (int)((size + kChunk - 1) / kChunk);
  const int local = blockIdx.x - e.first_chunk, mat = local / chunks, chunk = local % chunks;
  const int64_t base = (int64_t)mat * size + (int64_t)chunk * kChunk;
  const int n = (int)min((int64_t)kChunk, size - (int64_t)chunk * kChunk);
  char* const mem = p.ws + e.ws + mat * matrix_bytes(e.rows, e.cols, e.mp, e.np, p.precise);
  double sum = 0.0;
  if (n == kChunk && aligned(e, size % 8 == 0)) {
#pragma unroll
    for (int i = 0; i < kChunk / (kThreads * 8); ++i) begin_piece<8, true, TG, STEP>(p, e, base + (i * kThreads + threadIdx.x) * 8, sum);
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads) begin_piece<1, false, TG, STEP>(p, e, base + i, sum);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < kThreads / 64; ++w) s += part[w];
    reinterpret_cast<double*>(mem + at_sums(e.mp, e.np, p.precise))[chunk] = s;
  }
  if (chunk == 0) {
    uint32_t* const counts = reinterpret_cast<uint32_t*>(mem + at_counts(e.mp, e.np, p.precise));
    for (int i = threadIdx.x; i < (int)counts_of(e.mp); i += kThreads) counts[i] = 0;
  }
}

struct Tile {            // 64 x 64 of a matrix's padded X
  const Entry& e;
  int mat, i0, j0;
  bool tall;
  char* mem;
  int row0, col0;        // the same in the matrix itself, turned where that is taller than wide
  int64_t base;          // elements to the matrix
  bool whole;            // four neighbours at a time: no end of a row inside, 16-byte boundaries
};
__device__ __forceinline__ Tile tile_of(const Ends& p, int block) {
  const Entry& e = p.e[entry_of(p.n, block, [&](int i) { return p.e[i].first_tile; })];
  const int tm = e.mp / 64, tn = e.np / 64, local = block - e.first_tile;
  const int mat = local / (tm * tn), t = local % (tm * tn);
  const bool tall = e.rows > e.cols;
  const int i0 = t / tn * 64, j0 = t % tn * 64;
  return Tile{e, mat, i0, j0, tall, p.ws + e.ws + mat * matrix_bytes(e.rows, e.cols, e.mp, e.np, p.precise), tall ? j0 : i0, tall ? i0 : j0,
              (int64_t)mat * e.rows * e.cols, aligned(e, e.cols % 4 == 0)};
}
// f(row in the tile, first of four columns in it, its element, whether all four are there as a vector) for this thread's share of a tile in the
// matrix's own order
template <typename F>
__device__ __forceinline__ void for_pieces(const Tile& t, F&& f) {
#pragma unroll
  for (int it = 0; it < 64 * 16 / kThreads; ++it) {
    const int q = it * kThreads + threadIdx.x, r = q >> 4, c = (q & 15) * 4;
    f(r, c, t.base + (int64_t)(t.row0 + r) * t.e.cols + t.col0 + c, t.row0 + r < t.e.rows ? min(4, t.e.cols - t.col0 - c) : 0);
  }
}

// X = U / max(|U|, eps) in two planes, its longer side along the rows in memory, zeros around it.
template <typename TG, bool STEP>
__global__ __launch_bounds__(kThreads) void convert_kernel(const Ends p) {
  __shared__ double part[kThreads / 64];
  __shared__ float turned[64][65];
  const Tile t = tile_of(p, blockIdx.x);
  const Entry& e = t.e;
  const int tid = threadIdx.x;
  const int64_t size = (int64_t)e.rows * e.cols;
  const int chunks = (int)((size + kChunk - 1) / kChunk);
  const double* sums = reinterpret_cast<const double*>(t.mem + at_sums(e.mp, e.np, p.precise));
  double sum = 0.0;
  for (int i = tid; i < chunks; i += kThreads) sum += sums[i];
  float u[4][4];
  int it = 0;
  const auto piece = [&](int64_t i, int n, float (&x)[4]) {
    if (t.whole && n == 4) {
      gradient<4, true, TG>(e, i, x);
      if (STEP) {
        float m[4];
        load_n<4, true>(e.momentum + i, m);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = update_of(m[k], x[k], p.mu, p.nesterov);
        const float zero[4] = {};
        if (p.zero_flat && e.flat) store_n<4, true>(e.flat + i, zero);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = 0.f;
        if (k < n) {
          float g[1];
          gradient<1, false, TG>(e, i + k, g);
          x[k] = STEP ? update_of(e.momentum[i + k], g[0], p.mu, p.nesterov) : g[0];
          if (STEP && p.zero_flat && e.flat) e.flat[i + k] = 0.f;
        }
      }
    }
  };
  for_pieces(t, [&](int, int, int64_t i, int n) { piece(i, n, u[it++]); });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((tid & 63) == 0) part[tid >> 6] = sum;
  __syncthreads();
  const double norm = sqrt(part[0] + part[1] + part[2] + part[3]);
  const double factor = (double)kX / (norm < (double)p.eps ? (double)p.eps : norm);   // (NaN stays)
  // in two steps of fp32, the first one a power of two: the quotient may be far outside its range, and so may U
  const int half = factor > 0.0 ? ilogb(factor) / 2 : 0;
  const float f1 = ldexpf(1.f, half), f2 = (float)ldexp(factor, -half);
  f16_t* const hi = reinterpret_cast<f16_t*>(t.mem);
  f16_t* const lo = hi + to_lower(p.precise, e.mp, e.np);
  const auto put = [&](int i, int j, const float (&x)[4]) {
    f16x4_t h, l;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      h[v] = (f16_t)x[v];
      l[v] = (f16_t)(x[v] - (float)h[v]);
    }
    const int64_t at = place(p.precise, t.i0 + i, t.j0 + j, e.np);
    *reinterpret_cast<f16x4_t*>(hi + at) = h;
    *reinterpret_cast<f16x4_t*>(lo + at) = l;
  };
  it = 0;
  for_pieces(t, [&](int r, int c, int64_t, int) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = u[it][k] * f1 * f2;
    ++it;
    if (!t.tall) return put(r, c, x);
#pragma unroll
    for (int k = 0; k < 4; ++k) turned[r][c + k] = x[k];
  });
  if (!t.tall) return;
  __syncthreads();
  for (int q = tid; q < 64 * 16; q += kThreads) {
    const int i = q >> 4, j = (q & 15) * 4;
    const float x[4] = {turned[j][i], turned[j + 1][i], turned[j + 2][i], turned[j + 3][i]};
    put(i, j, x);
  }
}

// The result (TG), or with STEP the weights and their bf16 copy.  lower: whether X has its lower plane.
template <typename TG, bool STEP>
__global__ __launch_bounds__(kThreads) void finish_kernel(const Ends p, int from, int lower) {
  __shared__ float turned[64][65];
  const Tile t = tile_of(p, blockIdx.x);
  const Entry& e = t.e;
  const int tid = threadIdx.x;
  const f16_t* const hi = reinterpret_cast<const f16_t*>(t.mem + 2 * from * plane_x(e.mp, e.np));
  const f16_t* const lo = hi + to_lower(p.precise, e.mp, e.np);
  const auto get = [&](int i, int j, float (&x)[4]) {
    const int64_t at = place(p.precise, t.i0 + i, t.j0 + j, e.np);
    const f16x4_t h = *reinterpret_cast<const f16x4_t*>(hi + at), l = lower ? *reinterpret_cast<const f16x4_t*>(lo + at) : f16x4_t{};
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] = ((float)h[v] + (float)l[v]) * (1.f / kX);
  };
  if (t.tall) {
    for (int q = tid; q < 64 * 16; q += kThreads) {
      const int i = q >> 4, j = (q & 15) * 4;
      float x[4];
      get(i, j, x);
#pragma unroll
      for (int v = 0; v < 4; ++v) turned[j + v][i] = x[v];
    }
    __syncthreads();
  }
  for_pieces(t, [&](int r, int c, int64_t i, int n) {
    if (n <= 0) return;
    float o[4];
    if (t.tall) {
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = turned[r][c + k];
    } else {
      get(r, c, o);
    }
    if (t.whole && n == 4) {
      if (STEP) {
        float w[4];
        load_n<4, true>(e.master + i, w);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = w[k] * p.keep - e.rate * o[k];
        store_n<4, true>(e.master + i, w);
        if (e.out) store_n<4, true>(reinterpret_cast<bf16_t*>(e.out) + i, w);
      } else {
        store_n<4, true>(reinterpret_cast<TG*>(e.out) + i, o);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= n) continue;
      if (STEP) {
        const float w = e.master[i + k] * p.keep - e.rate * o[k];
        e.master[i + k] = w;
        if (e.out) reinterpret_cast<bf16_t*>(e.out)[i + k] = (bf16_t)w;
      } else {
        reinterpret_cast<TG*>(e.out)[i + k] = pk_from_float<TG>(o[k]);
      }
    }
  });
}

// ---------------------------------------------------------------- the products
enum Product { GRAM, POLY, UPDATE };

// Row tiles (of BM) of the BN x BN blocks on and below the diagonal of a symmetric mp x mp result, block row by block row: a full
// block row r has r + 1 blocks of BN / BM tiles, the last one may be half a block high.
template <int BM, int BN>
__host__ __device__ inline int units_of_symmetric(int mp) {
  constexpr int R = BN / BM;
  const int tm = (mp + BM - 1) / BM, whole = tm / R;
  return whole * (whole + 1) / 2 * R + (tm % R) * (whole + 1);
}

// BM x BN outputs of one product of one matrix (more rows and columns than there are: read from the last ones, not stored).
//   GRAM    A = X X^T              rows of X against rows of X
//   POLY    B = a + b A + c A A    A is symmetric: its rows against its rows
//   UPDATE  X' = B X               X comes as [k][columns] and through the transposing LDS read
// Single products of B and X's upper plane leave out B times its lower one; a times it is added, all of it that matters where A is small.
// GRAM and POLY are symmetric: the BN x BN blocks on and below the diagonal are computed, those below it stored twice.
// PRECISE: three products, lo hi + hi lo + hi hi, of both planes of a k-tile.  The matrix instructions cut what they add to a sum
// off at its last bit instead of rounding it, which makes long sums of one sign too small (diagonals of 1,100 products by 8e-7, and
// the result by ten times that): every 64 values of k the accumulators go into a second set by ordinary additions.
//
// Eight waves, 64 columns of outputs each, in two groups half a k-tile apart, one wave of each on a SIMD: while one multiplies a k-tile
// out of registers, the other reads its next k-tile's fragments from LDS and requests a later k-tile from memory; a barrier,
// and they swap (the k-loop of the grouped products).  k-tiles go straight to LDS, NS - 1 of them ahead.  A k-tile has KT values of k; W
// fp16 values of a row (both planes with PRECISE).
//
// us a launch, 128 matrices of 768 x 2048, three products: X X^T 564, A A 282, B X 918 (1.05 PFLOP/s of the products that it needs), single ones:
// 216, 126, 473 (of which its products are 295 and its 1.6 GB 310: the stores of a unit's end are not under the next one's products);
// one of 2048 x 4096, three products: 81, 54, 102 (1.0 PFLOP/s).
//
// SHARED (GRAM and POLY with few units, 128 x 128): the pairs of k-tiles of all units, one unit's behind the other's, are cut into
// p.shares equal shares, one to a workgroup.  A wave leaves its sums of a part of a unit as they are in Xn, which nobody needs then, and
// counts them; the one that finds the others' there adds them up in their order and goes on to the epilogue.
template <int KIND, bool PRECISE, int BM, int BN, int KT, int NS, bool SHARED = false>
__global__ __launch_bounds__(512) void product_kernel(const Gemm p) {
  constexpr int NW = 8, WNW = BN / 64, WM = BM / (NW / WNW), TM = WM / 32, TN = 2, KS = KT / 16;
  constexpr int P = PRECISE ? 2 : 1, W = KT * P;
  constexpr int A_BYTES = BM * W * 2, STAGE = (BM + BN) * W * 2, LA = A_BYTES / (NW * 1024), LB = BN * W * 2 / (NW * 1024), L = LA + LB;
  constexpr int STAGING = 32 * 128;                     // of a wave: 32 rows of one plane of its outputs
  static_assert(NS * STAGE <= 160 * 1024 && NW * STAGING <= STAGE, "LDS budget");
  static_assert(W == 32 || W == 64, "rows of the LDS tiles");
  static_assert(!PRECISE || KT == 32, "blocks of 32 of either plane");
  __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WNW, wn = wave % WNW;
  const int grp = wave >> 2;

  struct Unit {
    int mp, np, N;                                      // N: columns of the result
    int row0, col0, in_matrix, part, parts, nkt;        // parts: shares that the unit is in, part: which of them this is
    bool mirrored;                                      // off the diagonal of a symmetric result
    char *X, *Xn, *A, *B;
    uint32_t* counts;
  };
  Unit u;
  // ---- the loader: a lane's byte offsets from two wave-uniform pointers that advance by a constant per k-tile
  uint32_t va[LA], vb[LB];
  const char *ld_a, *ld_b;
  int64_t step_b;
  // this workgroup's units: neighbours share operands in an XCD's L2; with SHARED, its pairs of k-tiles
  int at = SHARED ? (int)(blockIdx.x * p.pairs / p.shares) : (int)blockIdx.x;
  const int end = SHARED ? (int)((blockIdx.x + 1) * p.pairs / p.shares) : p.blocks;
  auto share_of = [&](int pair) { return ((pair + 1) * p.shares - 1) / p.pairs; };      // the last that starts at or before it
  auto enter = [&](int dealt) {
    const int en = entry_of(p.n, dealt, [&](int i) { return SHARED ? p.e[i].first_k : p.e[i].first_unit; });
    const int mp = u.mp = p.e[en].mp, np = u.np = p.e[en].np;
    const int N = u.N = KIND == UPDATE ? np : mp;
    const int tm = (mp + BM - 1) / BM, tn = (N + BN - 1) / BN;
    const int pairs = (KIND == GRAM ? np : mp) / (2 * KT);       // of k-tiles: k is a multiple of 128
    const int local = SHARED ? (dealt - p.e[en].first_k) / pairs : dealt - p.e[en].first_unit;
    const int first_pair = p.e[en].first_k + local * pairs, pair0 = SHARED ? dealt - first_pair : 0;
    if (SHARED) {
      u.part = blockIdx.x - share_of(first_pair);
      u.parts = share_of(first_pair + pairs - 1) - share_of(first_pair) + 1;
    }
    int mat, mt, nt;
    if (KIND == UPDATE) {
      mat = local / (tm * tn);
      u.in_matrix = local % (tm * tn);
      mt = u.in_matrix / tn;
      nt = u.in_matrix % tn;
    } else {
      constexpr int R = BN / BM;                        // row tiles of a block
      const int per = units_of_symmetric<BM, BN>(mp);
      mat = local / per;
      const int t = u.in_matrix = local % per;
      nt = (int)((sqrtf(8.f * (t / R) + 1.f) - 1.f) * 0.5f);     // row of blocks, corrected, and the column in it
      while ((nt + 1) * (nt + 2) / 2 * R <= t) ++nt;
      while (nt * (nt + 1) / 2 * R > t) --nt;
      const int in_row = t - nt * (nt + 1) / 2 * R, rows = min(R, tm - nt * R);
      mt = nt * R + in_row % rows;
      nt = in_row / rows;
    }
    u.mirrored = KIND != UPDATE && mt / (BN / BM) != nt;
    const int row0 = u.row0 = __builtin_amdgcn_readfirstlane(mt * BM), col0 = u.col0 = __builtin_amdgcn_readfirstlane(nt * BN);
    char* const mem = const_cast<char*>(uniform_ptr(p.ws + p.e[en].ws + (int64_t)mat * p.e[en].stride));
    const int64_t px = plane_x(mp, np);
    u.X = mem + 2 * p.from * px;
    u.Xn = mem + 2 * (1 - p.from) * px;
    u.A = mem + at_a(mp, np);
    u.B = mem + at_b(mp, np, PRECISE);
    u.counts = reinterpret_cast<uint32_t*>(mem + at_counts(mp, np, PRECISE)) + u.in_matrix * 8;
    const char* const left = KIND == GRAM ? u.X : KIND == POLY ? u.A : u.B;
    const char* const right = KIND == POLY ? u.A : u.X;
    const int lda = (KIND == GRAM ? np : mp) * P, ldb = (KIND == POLY ? mp : np) * P;    // of a row in memory
    const int kt0 = 2 * pair0;
    u.nkt = __builtin_amdgcn_readfirstlane(2 * (SHARED ? min(pairs - pair0, end - dealt) : pairs));
    if (SHARED) at = dealt + u.nkt / 2;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      int r, k;
      kc_slot<W>(wave * LA + i, lane, r, k);
      va[i] = (uint32_t)(min(r, mp - 1 - row0) * lda + k) * 2u;
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      int r, k;
      if (KIND == UPDATE) {
        mn_slot<BN * P>(wave * LB + i, lane, r, k);
        vb[i] = (uint32_t)(r * ldb + min(k, (N - col0) * P - 8)) * 2u;
      } else {
        kc_slot<W>(wave * LB + i, lane, r, k);
        vb[i] = (uint32_t)(min(r, N - 1 - col0) * ldb + k) * 2u;
      }
    }
    ld_a = uniform_ptr(left + (int64_t)row0 * lda * 2 + (int64_t)kt0 * W * 2);
    ld_b = uniform_ptr(right + (KIND == UPDATE ? (int64_t)col0 * P * 2 : (int64_t)col0 * ldb * 2 + (int64_t)kt0 * W * 2));
    step_b = KIND == UPDATE ? (int64_t)KT * ldb * 2 : W * 2;
  };
  auto request = [&](int stage) {
    const uint32_t to = lds_addr(smem) + stage * STAGE;
    static_for<LA>([&](auto i) { dma16_s<decltype(i)::value * 1024>(va[i], ld_a, to + wave * (LA * 1024)); });
    static_for<LB>([&](auto i) { dma16_s<A_BYTES + decltype(i)::value * 1024>(vb[i], ld_b, to + wave * (LB * 1024)); });
    ld_a += W * 2;
    ld_b += step_b;
  };
  int cur = 0;                                          // stage of the unit's first k-tile
  auto request_first = [&]() {
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
      if (s < u.nkt) request(cur + s >= NS ? cur + s - NS : cur + s);
  };

  auto next = [&]() {                                   // -1: none
    if (SHARED) return at < end ? at : -1;
    for (; at < end; at += gridDim.x) {
      const int d = pk_rules::dealt_unit(at, p.chunk);
      if (d < p.units) {
        at += gridDim.x;
        return d;
      }
    }
    return -1;
  };
  int dealt = next();
  if (dealt < 0) return;
  enter(dealt);
  request_first();
  int stored = 0;                                       // store instructions since those requests

  for (;;) {
    const Unit w = u;
    const bool live = w.row0 + wm * WM < w.mp && w.col0 + wn * 64 < w.N;
    floatx16_t acc[TM][TN] = {}, sum[PRECISE ? TM : 1][TN] = {};
    {
      // k-tile 0 has landed once only the younger ones and the stores behind them are on their way
      wait_vm_le((min(w.nkt, NS - 1) - 1) * L + stored);
      block_barrier();
      if (grp == 1) block_barrier();
      f16x8_t fa[P][KS][TM], fb[P][KS][TN];             // upper and lower plane
      // FIRST: the accumulators go into the second set and start again
      auto k_tile = [&](int kt, auto first) __attribute__((always_inline)) {
        constexpr bool FIRST = decltype(first)::value;
        // ---- memory phase
        const char* const st = smem + cur * STAGE;
        if (live) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int pl = 0; pl < P; ++pl) {
#pragma unroll
              for (int i = 0; i < TM; ++i) fa[pl][ks][i] = frag_kc<W, f16x8_t>(st, wm * WM + 32 * i, ks + pl * KS, lane);
#pragma unroll
              for (int j = 0; j < TN; ++j)
                fb[pl][ks][j] = KIND == UPDATE ? frag_mn<BN * P, f16x8_t>(st + A_BYTES, (wn * 64 + 32 * j) * P + 32 * pl, ks, lane)
                                               : frag_kc<W, f16x8_t>(st + A_BYTES, wn * 64 + 32 * j, ks + pl * KS, lane);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (kt + NS - 1 < w.nkt) request(cur == 0 ? NS - 1 : cur - 1);      // the stage of k-tile kt - 1
        cur = cur + 1 == NS ? 0 : cur + 1;
        if (FIRST && live) {      // (while the other group multiplies)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) sum[PRECISE ? i : 0][j] += acc[i][j];
        }
        // a wave's own part of k-tile kt + 1 has landed when the phase before its first read ends; younger than it are the k-tiles after
        // it and, while it is one of those requested before the epilogue, that one's stores
        const int tiles = min(NS - 2, w.nkt - 2 - kt);
        auto wait_next = [&]() {
          if (kt <= NS - 3) wait_vm_le(max(tiles, 0) * L + stored);
          else wait_tiles<L, NS - 2>(tiles);
        };
        if (grp == 1) wait_next();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        block_barrier();
        // ---- compute phase
        if (live) {
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int pr = PRECISE ? 0 : 2; pr < 3; ++pr)        // lo hi, hi lo, hi hi
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                  acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[pr == 1 ? P - 1 : 0][ks][j], fa[pr == 0 ? P - 1 : 0][ks][i],
                                                                     FIRST && pr == 0 && ks == 0 ? floatx16_t{} : acc[i][j], 0, 0, 0);
          __builtin_amdgcn_s_setprio(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (grp == 0) wait_next();
        block_barrier();
      };
      if constexpr (PRECISE) {
        for (int kt = 0; kt < w.nkt; kt += 2) {
          k_tile(kt, std::true_type{});
          k_tile(kt + 1, std::false_type{});
        }
      } else {
        for (int kt = 0; kt < w.nkt; ++kt) k_tile(kt, std::false_type{});
      }
      if constexpr (PRECISE) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] += sum[i][j];
      }
      if (grp == 0) block_barrier();        // the whole ring is free
    }
    // the next unit's first k-tiles come while this one's results go
    dealt = next();
    if (dealt >= 0) {
      enter(dealt);
      request_first();
    }
    stored = 0;

    bool last = true;
    if (SHARED && live && w.parts > 1) {
      // [unit of the matrix][slot][8 bytes of every lane in turn].  Other XCDs read them: these stores go through the L2 to memory and the loads
      // past it, which costs less than fences, each of which walks a whole L2 (2048 x 4096 in fp32: X X^T 162 us with fences).
      typedef uint32_t uintx2_t __attribute__((ext_vector_type(2)));
      constexpr int VECS = TM * TN * 8;
      uint64_t* const sums = reinterpret_cast<uint64_t*>(w.Xn) + (int64_t)w.in_matrix * p.slots * (VECS * 512) + wave * (VECS * 64) + lane;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uintx2_t v = {__float_as_uint(acc[i][j][2 * q]), __float_as_uint(acc[i][j][2 * q + 1])};
            __hip_atomic_store(sums + (int64_t)w.part * (VECS * 512) + ((i * TN + j) * 8 + q) * 64, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
          }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // they are there
      uint32_t before = 0;
      if (lane == 0) before = __hip_atomic_fetch_add(w.counts + wave, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __builtin_amdgcn_readfirstlane(before) == (uint32_t)w.parts - 1;
      asm volatile("" ::: "memory");
      if (last) {
        if (lane == 0) __hip_atomic_store(w.counts + wave, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // (for the next launch)
        for (int z = 0; z < w.parts; ++z)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const uintx2_t v = __builtin_bit_cast(uintx2_t, __hip_atomic_load(sums + (int64_t)z * (VECS * 512) + ((i * TN + j) * 8 + q) * 64,
                                                                                  __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
                for (int k = 0; k < 2; ++k) acc[i][j][2 * q + k] = z == 0 ? __uint_as_float(v[k]) : acc[i][j][2 * q + k] + __uint_as_float(v[k]);
              }
      }
    }
    // ---- epilogue, 32 rows of a wave at a time.  acc[i][j][v] is row 32 i + lane % 32, column 32 j + 8 (v / 4) + 4 (lane / 32) + v % 4.  Memory
    // is read and written 16 bytes a lane, 64 columns a row; LDS turns one into the other: fp16 rows of 128 bytes, their 16-byte
    // pieces swizzled by the row, in the stage that the coming k-tiles leave free.
    if (last && live) {
      const int ldc = w.N;
      const int64_t lower = to_lower(PRECISE, w.mp, ldc) * 2;     // bytes
      char* const out = KIND == GRAM ? w.A : KIND == POLY ? w.B : w.Xn;
      const char* const old = KIND == POLY ? w.A : w.X;           // what b or a multiplies
      constexpr float unscale = KIND == GRAM ? kA / (kX * kX) : KIND == POLY ? 1.f / (kA * kA) : 1.f;
      constexpr bool OLD_HI = KIND == POLY, OLD_LO = PRECISE ? KIND == POLY : KIND == UPDATE, OUT_LO = KIND == UPDATE || PRECISE;
      char* const buf = smem + (cur == 0 ? NS - 1 : cur - 1) * STAGE + wave * STAGING;
      int lane_e = lane;                                // (so that its addresses are formed here, not kept in registers through the k-loop)
      asm volatile("" : "+v"(lane_e));
      const int lr = lane_e >> 3, lc = lane_e & 7;      // a lane's row (of 8 in a pass) and piece of it in memory
      const int row = lane_e & 31, col = 4 * (lane_e >> 5);       // and in acc: column 32 j + 8 q + col
      const auto piece_at = [&](int r, int c) { return buf + r * 128 + ((c ^ (r & 7)) << 4); };
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r0 = w.row0 + wm * WM + 32 * i, c0 = w.col0 + wn * 64;
        f16x8_t from_memory[2][4];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
          if (pl ? OLD_LO : OLD_HI) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              from_memory[pl][q] = *reinterpret_cast<const f16x8_t*>(old + place(PRECISE, r0 + 8 * q + lr, c0 + 8 * lc, ldc) * 2 + pl * lower);
          }
        f16x4_t o[2][TN][4];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl)
          if (pl ? OLD_LO : OLD_HI) {
            wave_lds_fence();
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<f16x8_t*>(piece_at(8 * q + lr, lc)) = from_memory[pl][q];
            wave_lds_fence();
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) o[pl][j][q] = *reinterpret_cast<const f16x4_t*>(piece_at(row, 4 * j + q) + col * 2);
          }
        f16x4_t res[2][TN][4];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float x = acc[i][j][4 * q + k] * unscale;
              if (KIND == POLY) {
                const float before = OLD_LO ? (float)o[0][j][q][k] + (float)o[1][j][q][k] : (float)o[0][j][q][k];
                x = p.b * (before * (1.f / kA)) + p.c * x;
                if (r0 + row == c0 + 32 * j + 8 * q + col + k) x += p.a;
              } else if (OLD_LO) {
                x += p.a * (float)o[1][j][q][k];
              }
              res[0][j][q][k] = (f16_t)x;
              res[1][j][q][k] = (f16_t)(x - (float)res[0][j][q][k]);
            }
#pragma unroll
        for (int pl = 0; pl < (OUT_LO ? 2 : 1); ++pl) {
          if (KIND == UPDATE && !PRECISE && pl == 1 && !p.lower) break;
          wave_lds_fence();
#pragma unroll
          for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<f16x4_t*>(piece_at(row, 4 * j + q) + col * 2) = res[pl][j][q];
          wave_lds_fence();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f16x8_t*>(out + place(PRECISE, r0 + 8 * q + lr, c0 + 8 * lc, ldc) * 2 + pl * lower) =
                *reinterpret_cast<const f16x8_t*>(piece_at(8 * q + lr, lc));
          stored += 4;
          if (KIND != UPDATE && w.mirrored) {
            // turned: within 16 lanes of the transposing read, lane t points at row t / 4, columns 4 (t % 4) .. and receives rows 0 .. 3 of
            // column t
            const int t = lane_e & 15, ra = 8 * (lane_e >> 4) + (t >> 2), rb = ra + 4;
#pragma unroll
            for (int q = 0; q < 4; ++q) {               // columns 16 q ..
              const int c = 16 * q + 4 * (t & 3);
              const shortx4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4_t*)(piece_at(ra, c >> 3) + (c & 7) * 2));
              const shortx4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4_t*)(piece_at(rb, c >> 3) + (c & 7) * 2));
              typedef short shortx8_t __attribute__((ext_vector_type(8)));
              *reinterpret_cast<shortx8_t*>(out + pl * lower + place(PRECISE, c0 + 16 * q + t, r0 + 8 * (lane_e >> 4), ldc) * 2) =
                  __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            stored += 4;
          }
        }
      }
    }
    if (dealt < 0) return;
  }
}

// ---------------------------------------------------------------- host
struct Item {
  const void* src;
  float *flat, *momentum, *master;
  void* out;
  int64_t count, rows, cols;
  float rate;
  bool precise;
};
struct Settings {
  bool step, bf16_src;
  float mu, keep, eps;
  bool nesterov, zero_flat;
  int steps;
  float a, b, c;
};
int padded(int64_t n) { return (int)(pk_ceil_div(n, kPad) * kPad); }
int64_t bytes_of(int64_t rows, int64_t cols, bool precise) {
  return matrix_bytes((int)rows, (int)cols, padded(std::min(rows, cols)), padded(std::max(rows, cols)), precise);
}
bool sides_ok(int64_t rows, int64_t cols) { return rows <= PK_MAX_MATRIX_SIDE && cols <= PK_MAX_MATRIX_SIDE; }

// The tiles: wide ones, 256 x 256 (single products) or 128 x 256, or 128 x 128, by the rounds that their units take on the CUs; a round of wide
// ones takes 2.5 to 3 (1.5 to 1.75 with three products) of the others.  us of the five steps, wide / narrow, X X^T and A A together, the
// update, and in brackets their wide units; fp32: three products, bf16: single ones: 24 x 256 x 512, fp32, 225 / 174, 97 / 80 (48, 96); 24 x 363 x 1000, bf16, 244 / 147, 127 / 154 (72, 192),
// fp32 351 / 260, 223 / 220 (96, 288); 2048 x 4096, fp32, 1,020 / 644, 483 / 636 (72, 256), bf16 695 / 389, 285 / 270 (36, 128); 16 x 768 x 2048, fp32,
// 726 / 797, 657 / 753 (192, 768); 64 x 512 x 512, fp32, 612 / 599, 318 / 368 (384, 512); 128 x 768 x 2048, bf16, 1,713 / 1,923, 2,342 / 3,256
// (3 and 12 rounds), fp32 4,261 / 4,456, 4,541 / 5,661 (6 and 24).  (Half of a wide tile on the diagonal is of no use.)
bool pays_wide(bool precise, int64_t wide, int64_t narrow) {
  return pk_ceil_div(wide, 256) * (precise ? 5 / 3.0 : 11 / 4.0) < (double)pk_ceil_div(narrow, 256);
}
constexpr int kWideRows[2] = {256, 128};               // [precise]
constexpr unsigned kGrid = 256;                         // workgroups at most, one to a CU; each takes every kGrid-th unit
template <int KIND>
void launch_product(const Gemm& g, bool precise, int id, hipStream_t s) {
  const dim3 grid(std::min<unsigned>(g.blocks, kGrid)), block(512);
#define PK_LAUNCH(...) PK_LAUNCH_NOCHECK(id, s, (product_kernel<KIND, __VA_ARGS__>), grid, block, 0, s, g)
  if constexpr (KIND != UPDATE)
    if (g.shares > 0) {
      const dim3 grid(g.shares);
      if (precise) PK_LAUNCH(true, 128, 128, 32, 4, true); else PK_LAUNCH(false, 128, 128, 64, 4, true);
      return;
    }
  if (g.wide) { if (precise) PK_LAUNCH(true, 128, 256, 32, 3); else PK_LAUNCH(false, 256, 256, 32, 4); }
  else if (precise) PK_LAUNCH(true, 128, 128, 32, 4);
  else PK_LAUNCH(false, 128, 128, 64, 4);
#undef PK_LAUNCH
}
void deal(Gemm& g, int64_t units) {
  g.chunk = (int32_t)pk_rules::deal_chunk(units, 32);
  g.blocks = (int32_t)pk_rules::dealt_blocks(units, g.chunk);
}
int64_t wide_symmetric(bool precise, int mp) { return precise ? units_of_symmetric<128, 256>(mp) : units_of_symmetric<256, 256>(mp); }
int64_t wide_update(bool precise, int mp, int np) { return pk_ceil_div(mp, kWideRows[precise]) * pk_ceil_div(np, 256); }
template <typename F>
int64_t count_units(const Gemm& g, F&& per) {
  int64_t units = 0;
  for (int i = 0; i < g.n; ++i) units += g.e[i].first_unit * (int64_t)per(g.e[i].mp, g.e[i].np);
  return units;
}
// Whether X X^T (A A with poly) of `units` (at most one to a CU) is cut into shares, of at least 256 values of k: where a unit's sums fit Xn
// and the longest unit is kLeastSaved k-tiles of 32 longer than a share, about what leaving and adding the sums takes.  2048 x 4096 in fp32,
// 136 units: X X^T (60 k-tiles saved of 128) 101 -> 81 us, A A (30 of 64) 57 -> 53; 128 x 2048, one unit: the orthogonalization 188 -> 180
// against shares whose sums a second launch adds up, which 2048 x 4096 runs in 1,147 us and this in 1,058.
constexpr int kLeastSaved = 16;
void cut(Gemm& g, bool precise, bool poly, int64_t units) {
  if (units == 0 || units > kGrid) return;
  const int64_t per_pair = precise ? 64 : 128;          // values of k
  int64_t pairs = 0, longest = 0;
  for (int i = 0, at = 0; i < g.n; ++i) {
    const int64_t matrices = g.e[i].first_unit, of_unit = (poly ? g.e[i].mp : g.e[i].np) / per_pair;
    g.e[i].first_k = at;
    pairs += matrices * units_of_symmetric<128, 128>(g.e[i].mp) * of_unit;
    at = (int)pairs;
    longest = std::max(longest, of_unit);
  }
  const auto slots = [&](int64_t shares) {              // a unit's ends may lie inside shares, unless shares and units end together
    const bool whole = g.n == 1 && shares % units == 0;
    return pk_ceil_div(longest * shares, pairs) + (whole ? 0 : 1);
  };
  int64_t room = kGrid + 1, shares = std::min<int64_t>(kGrid, pairs * per_pair / 256);
  for (int i = 0; i < g.n; ++i)
    room = std::min(room, 2 * plane_x(g.e[i].mp, g.e[i].np) / (units_of_symmetric<128, 128>(g.e[i].mp) * (int64_t)(128 * 128 * 4)));
  while (shares > units && slots(shares) > room) --shares;
  if (shares <= units || (longest - pk_ceil_div(pairs, shares)) * per_pair < kLeastSaved * 32) return;
  g.shares = (int)shares; g.pairs = (int)pairs; g.slots = (int)slots(shares);
}
// Units of a launch: per(mp, np) of them for each matrix.
template <typename F>
int64_t number_units(Gemm& g, F&& per) {
  int64_t at = 0;
  for (int i = 0; i < g.n; ++i) {
    const int64_t units = g.e[i].first_unit * (int64_t)per(g.e[i].mp, g.e[i].np);
    g.e[i].first_unit = (int32_t)at;
    at += units;
  }
  g.units = (int32_t)at;
  deal(g, at);
  return at;
}
// A group of matrices.
struct Group {
  Ends ends[kMaxEnds];
  int64_t chunks[kMaxEnds], tiles[kMaxEnds];            // workgroups of the launches
  int n;
  Gemm sym, poly, upd;
};
template <typename TG, bool STEP>
int run_group(Group& g, const Settings& o, hipStream_t s) {
  const bool precise = g.ends[0].precise != 0;
  for (int i = 0; i < g.n; ++i)
    PK_LAUNCH_NOCHECK(pk_timing::K_MUON_BEGIN, s, (begin_kernel<TG, STEP>), dim3((unsigned)g.chunks[i]), dim3(kThreads), 0, s, g.ends[i]);
  for (int i = 0; i < g.n; ++i)
    PK_LAUNCH_NOCHECK(pk_timing::K_MUON_CONVERT, s, (convert_kernel<TG, STEP>), dim3((unsigned)g.tiles[i]), dim3(kThreads), 0, s, g.ends[i]);
  // Single products end with the upper plane alone, off by 2^-12 where they are by 2e-3: 16 bits a value less to write and to read
  const auto lower = [&](int step) { return precise || step == 0 || step < o.steps; };
  int from = 0;
  for (int i = 0; i < o.steps; ++i) {
    g.sym.from = g.poly.from = g.upd.from = from;
    g.upd.lower = lower(i + 1);
    launch_product<GRAM>(g.sym, precise, pk_timing::K_NS_GRAM, s);
    launch_product<POLY>(g.poly, precise, pk_timing::K_NS_POLY, s);
    launch_product<UPDATE>(g.upd, precise, pk_timing::K_NS_UPDATE, s);
    from = 1 - from;
  }
  for (int i = 0; i < g.n; ++i)
    PK_LAUNCH_NOCHECK(pk_timing::K_MUON_FINISH, s, (finish_kernel<TG, STEP>), dim3((unsigned)g.tiles[i]), dim3(kThreads), 0, s, g.ends[i], from, (int)lower(o.steps));
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

// Whether all operands take part with both planes.
bool precise_result(bool asked, int64_t rows, int64_t cols) { return asked || std::min(rows, cols) <= kPad; }

// All matrices of the items 0 .. n - 1 (item(i); one without matrices has count 0), in groups of what the workspace holds.
template <typename F>
int run(int64_t n, F&& item, const Settings& o, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  bool some = false;
  int64_t all = 0;
  for (int64_t i = 0; i < n; ++i) {
    const Item it = item(i);
    if (it.count == 0) continue;
    some = true;
    all += it.count * bytes_of(it.rows, it.cols, it.precise);
    if (!workspace || !pk_aligned16(workspace) || bytes_of(it.rows, it.cols, it.precise) > workspace_bytes) return PK_ERR_WORKSPACE;
  }
  if (!some) return PK_OK;
  const int64_t share = pk_ceil_div(all, pk_ceil_div(all, workspace_bytes));      // groups of about the same size
  const int64_t es = o.bf16_src ? 2 : 4;
  int64_t i = 0, done = 0;        // done: matrices of item i
  while (i < n) {
    Group g;
    g.n = 0;
    Gemm sym = {};
    sym.ws = static_cast<char*>(workspace);
    sym.a = o.a; sym.b = o.b; sym.c = o.c;
    int64_t used = 0;
    bool precise = false;
    while (i < n) {
      const Item it = item(i);
      if (it.count == 0) { ++i; continue; }
      if (used > 0 && it.precise != precise) break;                // the kernels of a group are of one kind
      precise = it.precise;
      const int64_t each = bytes_of(it.rows, it.cols, precise), left = std::min(workspace_bytes - used, std::max<int64_t>(share - used, 0) + each - 1);
      const int64_t fit = std::min(left / each, it.count - done);
      const int mp = padded(std::min(it.rows, it.cols)), np = padded(std::max(it.rows, it.cols));
      const bool like_last = sym.n > 0 && sym.e[sym.n - 1].mp == mp && sym.e[sym.n - 1].np == np && sym.e[sym.n - 1].stride == each;
      if (fit <= 0 || (!like_last && sym.n == kMaxShapes)) break;
      if (g.n == 0 || g.ends[g.n - 1].n == kMaxEntries) {
        if (g.n == kMaxEnds) break;
        Ends& e = g.ends[g.n];
        e.ws = static_cast<char*>(workspace);
        e.n = 0;
        e.mu = o.mu; e.keep = o.keep; e.eps = o.eps; e.nesterov = o.nesterov; e.zero_flat = o.zero_flat; e.precise = precise;
        g.chunks[g.n] = g.tiles[g.n] = 0;
        ++g.n;
      }
      Ends& e = g.ends[g.n - 1];
      int64_t &chunks = g.chunks[g.n - 1], &tiles = g.tiles[g.n - 1];
      const int64_t at = done * it.rows * it.cols;
      Entry& x = e.e[e.n++];
      x.src = it.src ? static_cast<const char*>(it.src) + at * es : nullptr;
      x.flat = it.flat ? it.flat + at : nullptr;
      x.momentum = it.momentum ? it.momentum + at : nullptr;
      x.master = it.master ? it.master + at : nullptr;
      x.out = it.out ? static_cast<char*>(it.out) + at * (o.step ? 2 : es) : nullptr;
      x.ws = used;
      x.rows = (int)it.rows; x.cols = (int)it.cols; x.count = (int)fit; x.mp = mp; x.np = np;
      x.first_chunk = (int)chunks; x.first_tile = (int)tiles;
      x.rate = it.rate;
      if (like_last) sym.e[sym.n - 1].first_unit += (int32_t)fit;
      else sym.e[sym.n++] = {used, each, mp, np, (int32_t)fit};
      chunks += fit * pk_ceil_div(it.rows * it.cols, kChunk);
      tiles += fit * (mp / 64) * (np / 64);
      if (std::max(chunks, tiles) > 0x3fffffffll) return PK_ERR_SHAPE;
      used += fit * each;
      done += fit;
      if (done == it.count) { ++i; done = 0; }
    }
    if (g.n == 0) break;
    // long products first: what is left for the end is short
    std::sort(sym.e, sym.e + sym.n, [](const auto& x, const auto& y) { return (int64_t)x.mp * x.np > (int64_t)y.mp * y.np; });
    g.sym = g.upd = sym;
    const int64_t narrow_sym = count_units(sym, [](int mp, int) { return units_of_symmetric<128, 128>(mp); });
    g.sym.wide = pays_wide(precise, count_units(sym, [&](int mp, int) { return wide_symmetric(precise, mp); }), narrow_sym);
    g.upd.wide = pays_wide(precise, count_units(sym, [&](int mp, int np) { return wide_update(precise, mp, np); }),
                           count_units(sym, [](int mp, int np) { return (int64_t)(mp / 128) * (np / 128); }));
    g.poly = g.sym;
    if (!g.sym.wide) {
      cut(g.sym, precise, false, narrow_sym);
      cut(g.poly, precise, true, narrow_sym);
    }
    const auto of_symmetric = [&](int mp, int) { return g.sym.wide ? wide_symmetric(precise, mp) : units_of_symmetric<128, 128>(mp); };
    const int64_t sym_units = number_units(g.sym, of_symmetric);
    number_units(g.poly, of_symmetric);
    const int64_t upd_units =
        number_units(g.upd, [&](int mp, int np) { return g.upd.wide ? wide_update(precise, mp, np) : (int64_t)(mp / 128) * (np / 128); });
    if (std::max(sym_units, upd_units) > 0x3fffffffll) return PK_ERR_SHAPE;
    const int rc = o.step ? (o.bf16_src ? run_group<bf16_t, true>(g, o, s) : run_group<float, true>(g, o, s))
                          : (o.bf16_src ? run_group<bf16_t, false>(g, o, s) : run_group<float, false>(g, o, s));
    if (rc != PK_OK) return rc;
  }
  return PK_OK;
}

bool settings_ok(int steps, float a, float b, float c, float eps) {
  return steps >= 0 && steps <= 100 && eps > 0.f && pk_newton_schulz_range(steps, a, b, c) <= PK_NEWTON_SCHULZ_RANGE;
}

}  // namespace

extern "C" {

// A step takes singular values x in [0, m] onto p(x) = a x + b x^3 + c x^5, an interval around 0, whose ends are p at m or where p' = a + 3 b
// x^2 + 5 c x^4 is 0.  2^-6 at the start and at every step is room for the roundings (single products: below 2^-8 of a value, the
// head of this file), which coefficients that hold 1 in place without holding its neighbours would carry on.  B = p(x) / x is fp16 too: it
// counts with a factor of 15 / 60000.
double pk_newton_schulz_range(int steps, float a, float b, float c) {
  const double room = 1.0 + 1.0 / 64, none = std::numeric_limits<double>::infinity();
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return none;
  double m = room, most = m;
  for (int i = 0; i < steps; ++i) {
    const auto poly = [&](double t) { return a + t * (b + t * (double)c); };      // of t = x^2
    const double end = m * m;
    double at[5] = {0.0, end, end, end, end};
    const double disc = 9.0 * b * b - 20.0 * a * (double)c;
    if (c != 0 && disc >= 0)
      for (int k = 0; k < 2; ++k) at[2 + k] = (-3.0 * b + (k ? 1 : -1) * std::sqrt(disc)) / (10.0 * c);
    else if (c == 0 && b != 0)
      at[2] = -(double)a / (3.0 * b);
    if (c != 0) at[4] = -(double)b / (2.0 * c);                                   // where B turns
    double next = 0.0;
    for (const double t : at) {
      if (!(t >= 0.0 && t <= end)) continue;
      next = std::max(next, std::abs(std::sqrt(t) * poly(t)));
      most = std::max(most, std::abs(poly(t)) * (PK_NEWTON_SCHULZ_RANGE / 60000.0));
    }
    m = next * room;
    most = std::max(most, m);
    if (!(most <= PK_NEWTON_SCHULZ_RANGE)) return std::isfinite(most) ? most : none;
  }
  return most;
}

int64_t pk_orthogonalize_workspace_bytes(const int64_t* counts, const int64_t* rows, const int64_t* cols, int64_t n, int precise) {
  if (n < 0 || (n > 0 && (!counts || !rows || !cols))) return PK_ERR_ARG;
  int64_t all = 0, most = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] < 0 || rows[i] < 0 || cols[i] < 0) return PK_ERR_ARG;
    if (!sides_ok(rows[i], cols[i])) return PK_ERR_SHAPE;
    if (counts[i] == 0 || rows[i] == 0 || cols[i] == 0) continue;
    const int64_t each = bytes_of(rows[i], cols[i], precise_result(precise != 0, rows[i], cols[i]));
    most = std::max(most, each);
    all = std::min(all, kGroupBytes) + std::min(counts[i], kGroupBytes / each + 1) * each;
  }
  return std::max(most, std::min(all, kGroupBytes));
}

static int orthogonalize(bool precise, const void* x, int dtype, void* out, int64_t count, int64_t rows, int64_t cols, int steps, float a,
                         float b, float c, float eps, void* workspace, int64_t workspace_bytes, pk_stream_t stream) {
  if (count < 0 || rows < 0 || cols < 0 || !pk_dtype_ok(dtype) || !settings_ok(steps, a, b, c, eps)) return PK_ERR_ARG;
  if (!sides_ok(rows, cols)) return PK_ERR_SHAPE;
  if (count == 0 || rows == 0 || cols == 0) return PK_OK;
  if (!x || !out) return PK_ERR_ARG;
  Settings o = {};
  o.bf16_src = dtype == PK_BF16;
  o.eps = eps; o.steps = steps; o.a = a; o.b = b; o.c = c;
  const Item only{x, nullptr, nullptr, nullptr, out, count, rows, cols, 0.f, precise_result(precise, rows, cols)};
  return run(1, [&](int64_t) { return only; }, o, workspace, workspace_bytes, (hipStream_t)stream);
}
int pk_orthogonalize(const void* x, int dtype, void* out, int64_t count, int64_t rows, int64_t cols, int steps, float a, float b, float c,
                     float eps, void* workspace, int64_t workspace_bytes, pk_stream_t stream) {
  return orthogonalize(true, x, dtype, out, count, rows, cols, steps, a, b, c, eps, workspace, workspace_bytes, stream);
}
int pk_orthogonalize_half(const void* x, int dtype, void* out, int64_t count, int64_t rows, int64_t cols, int steps, float a, float b, float c,
                          float eps, void* workspace, int64_t workspace_bytes, pk_stream_t stream) {
  return orthogonalize(false, x, dtype, out, count, rows, cols, steps, a, b, c, eps, workspace, workspace_bytes, stream);
}

int pk_muon_fused(float* const* masters, float* const* momenta, const void* const* grads, float* const* flat_grads, void* const* shadows,
                  const int64_t* counts, const int64_t* rows, const int64_t* cols, int64_t n, int grad_dtype, double lr, double momentum,
                  double weight_decay, int nesterov, int adjust, int zero_flat, int precise, int steps, float a, float b, float c, float eps,
                  void* workspace, int64_t workspace_bytes, pk_stream_t stream) {
  if (n < 0 || !pk_dtype_ok(grad_dtype) || !settings_ok(steps, a, b, c, eps) || (adjust != PK_MUON_ASPECT && adjust != PK_MUON_RMS)) return PK_ERR_ARG;
  if (n == 0) return PK_OK;
  if (!masters || !momenta || !counts || !rows || !cols) return PK_ERR_ARG;
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] < 0 || rows[i] < 0 || cols[i] < 0) return PK_ERR_ARG;
    if (!sides_ok(rows[i], cols[i])) return PK_ERR_SHAPE;
    if (counts[i] > 0 && rows[i] > 0 && cols[i] > 0 && (!masters[i] || !momenta[i])) return PK_ERR_ARG;
  }
  const auto item = [&](int64_t i) {
    const double r = (double)rows[i], k = (double)cols[i];
    const double scale = adjust == PK_MUON_RMS ? 0.2 * std::sqrt(std::max(r, k)) : std::sqrt(std::max(1.0, r / k));
    return Item{grads ? grads[i] : nullptr, flat_grads ? flat_grads[i] : nullptr, momenta[i], masters[i], shadows ? shadows[i] : nullptr,
                rows[i] > 0 && cols[i] > 0 ? counts[i] : 0, rows[i], cols[i], (float)(lr * scale), precise_result(precise != 0, rows[i], cols[i])};
  };
  Settings o = {};
  o.step = true; o.bf16_src = grad_dtype == PK_BF16;
  o.mu = (float)momentum; o.keep = (float)(1.0 - lr * weight_decay); o.eps = eps;
  o.nesterov = nesterov != 0; o.zero_flat = zero_flat != 0;
  o.steps = steps; o.a = a; o.b = b; o.c = c;
  return run(n, item, o, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
