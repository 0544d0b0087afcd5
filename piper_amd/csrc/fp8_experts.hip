// The experts' products in 8-bit floating point: e4m3 values with a power of two for each block of 128 (fp8_blocks.h).
//   rows:     [R][K'] codes, K' = K rounded up to 128 (the rest zeros), and K'/128 scale bytes a row, rows of whole words
//   weights:  [E][N][K'] codes and [E][N/128][K'/128] bytes, blocks of 128 x 128; the transposed codes [E][K][N'] share the bytes
// Values are decoded into bf16, their power of two included, and multiplied there: products are exact, and added in fp32.
// v_mfma_scale_f32_32x32x64_f8f6f4 takes codes and scale bytes as they are, at twice the rate (measured 4.5 PFLOP/s against 2.2), but of 8
// neighbouring products' sum it keeps 13 bits below the largest product's leading one (measured; the other instructions for 8-bit values
// do the same, those for bf16 keep all).  An error of 2^-13 is small next to the codes' own 2^-4, but g, u and d_h are rounded to
// bf16 next, and h, d_g and d_u to codes again: a value that falls to the other side there is a step off, 2^-8 or 2^-3.  Against
// exact sums y of one token was off by 0.007 of its size, four times bf16's own rounding, y of many rows by 0.0013 and d_w by 0.001.
// So these short sums are for callers who ask for them (the entry points ending in _short), where they are faster.
#include "fp8_blocks.h"
#include "launch_rules.h"
#include "unit_index.h"

#include <type_traits>

namespace {

constexpr int BLOCK = PK_FP8_BLOCK;
constexpr int THREADS = 256;
using pk_units::FastDiv;

inline int64_t blocks_of(int64_t n) { return pk_ceil_div(n, BLOCK); }
// bytes of a row of scales: whole words
__host__ __device__ inline int scale_row(int blocks) { return (blocks + 3) & ~3; }

// 8 neighbouring values, zeros behind the first `have`.  Rows of odd widths start anywhere: 16-byte loads need no alignment (24 experts'
// weights of 363 x 1000 in fp32 41 -> 34 us against value by value, 10,975 rows of 1145 bf16 values 19 -> 10).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int have, float (&f)[8]) {
  if (have >= 8) {
    T v[8];
    __builtin_memcpy(v, p, sizeof v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < have ? pk_to_float<T>(p[i]) : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------ rows
// 16 lanes to a block, one pass: 2 (bf16) or 4 bytes read and 1 written per value, bound by the memory (32,768 x 2048 bf16: 35 us,
// 5.7 TB/s, where a copy of 2 GiB reaches 4.9; with one or four blocks on their way in a lane 38).
// N blocks of rows, by 16 lanes; block i is number `unit` + i * step of all, and there if below `units`.  source(r): the row of x that
// is row r, negative where there is none: such rows are NaN.
template <typename T, int N, typename Source>
__device__ __forceinline__ void quantize_blocks(const T* x, Source&& source, uint8_t* q, uint8_t* s, int64_t unit, int step, int64_t units, int K,
                                                int kb, FastDiv by_kb) {
  const int lane = threadIdx.x & 15;
  int r[N], b[N];
  float f[N][8];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t u = min(unit + i * step, units - 1);
    r[i] = pk_units::fastdiv((int)u, by_kb);
    b[i] = (int)(u - (int64_t)r[i] * kb);
    const int k = b[i] * BLOCK + lane * 8;
    const int64_t from = source(r[i]);
    load8<T>(x + (from < 0 ? 0 : from) * K + k, from < 0 ? 0 : K - k, f[i]);
    if (from < 0) f[i][0] = __builtin_nanf("");
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (unit + i * step >= units) return;    // whole groups of 16 lanes
    uint32_t codes[2], byte;
    pk_fp8::quantize8(f[i], codes, byte);
    *reinterpret_cast<u32x2_t*>(q + (unit + i * step) * BLOCK + lane * 8) = u32x2_t{codes[0], codes[1]};
    if (lane == 0) s[(int64_t)r[i] * scale_row(kb) + b[i]] = (uint8_t)byte;
  }
}
constexpr int ROW_BLOCKS = 2;
template <typename T>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ row_map, int64_t entries,
                                                                FastDiv map_div, uint8_t* __restrict__ q, uint8_t* __restrict__ s, int64_t units,
                                                                int K, int kb, FastDiv by_kb) {
  const auto source = [&](int r) -> int64_t {
    if (!row_map) return (int64_t)(uint32_t)r;
    const int entry = row_map[r];
    return entry < 0 || entry >= entries ? -1 : (int64_t)(uint32_t)pk_units::fastdiv(entry, map_div);
  };
  quantize_blocks<T, ROW_BLOCKS>(x, source, q, s, (int64_t)blockIdx.x * (THREADS / 16 * ROW_BLOCKS) + (threadIdx.x >> 4), THREADS / 16, units, K, kb, by_kb);
}

// ------------------------------------------------------------------------------------------------ weights
// A workgroup has one block of 128 x 128: 16 lanes to a row of it, the codes once row-major and once, through the LDS, transposed.  Bound
// by the memory: 128 experts' three weights of 2048 x 768 in bf16 take 457 us, 5.3 TB/s.  All weights of a call share a launch (24 experts'
// three of 363 x 1000 in fp32, 576 workgroups each: three launches took 57 us where one took 41; those 469).
struct Weights {
  const void* w[PK_FP8_MAX_WEIGHTS];
  uint8_t *q[PK_FP8_MAX_WEIGHTS], *t[PK_FP8_MAX_WEIGHTS], *s[PK_FP8_MAX_WEIGHTS];
  int32_t first[PK_FP8_MAX_WEIGHTS], N[PK_FP8_MAX_WEIGHTS], K[PK_FP8_MAX_WEIGHTS];      // first: its first workgroup
  FastDiv by_nb[PK_FP8_MAX_WEIGHTS], by_kb[PK_FP8_MAX_WEIGHTS];
  int32_t count;
};
template <typename T>
__global__ __launch_bounds__(THREADS) void quantize_weights_kernel(const Weights p) {
  constexpr int LD = BLOCK + 4;              // of the LDS rows: columns of bytes spread over the banks
  __shared__ uint32_t amax_of[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[BLOCK * LD];
  int which = 0;
  while (which + 1 < p.count && (int)blockIdx.x >= p.first[which + 1]) ++which;
  const int N = p.N[which], K = p.K[which], kb = (K + BLOCK - 1) / BLOCK, nb = (N + BLOCK - 1) / BLOCK;
  uint8_t *const __restrict__ q = p.q[which], *const __restrict__ t = p.t[which], *const __restrict__ s = p.s[which];
  const int local = (int)blockIdx.x - p.first[which], row_block = pk_units::fastdiv(local, p.by_kb[which]), kblock = local - row_block * kb;
  const int64_t e = pk_units::fastdiv(row_block, p.by_nb[which]);
  const int nblock = row_block - (int)e * nb;
  const int n0 = nblock * BLOCK, k0 = kblock * BLOCK, Kp = kb * BLOCK, Np = nb * BLOCK;
  const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, k = k0 + lane * 8;
  const T* const __restrict__ src = reinterpret_cast<const T*>(p.w[which]) + e * N * K;
  float f[8][8];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + row + 16 * i;
    load8<T>(src + (int64_t)(n < N ? n : n0) * K + k, n < N ? K - k : 0, f[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(f[i][j]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
  }
  m = pk_fp8::row_max(m);
  {
    const uint32_t a = __shfl_xor(m, 16), b = a > m ? a : m, c = __shfl_xor(b, 32);
    m = c > b ? c : b;
  }
  if ((threadIdx.x & 63) == 0) amax_of[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = amax_of[i] > m ? amax_of[i] : m;
  const bool finite = m < pk_fp8::INF_BITS;
  const uint32_t byte = finite ? pk_fp8::scale_byte(m, pk_fp8::TOP_E4M3) : 127u;
  const float inv = pk_fp8::inverse_scale_of(byte);
  if (threadIdx.x == 0) s[(e * nb + nblock) * kb + kblock] = (uint8_t)byte;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    u32x2_t c;
    c[0] = pk_fp8::e4m3x4(f[i][0] * inv, f[i][1] * inv, f[i][2] * inv, f[i][3] * inv);
    c[1] = pk_fp8::e4m3x4(f[i][4] * inv, f[i][5] * inv, f[i][6] * inv, f[i][7] * inv);
    if (!finite) c[0] = c[1] = pk_fp8::NAN_CODE * 0x01010101u;
    const int n = n0 + row + 16 * i;
    if (n < N) *reinterpret_cast<u32x2_t*>(q + (e * N + n) * Kp + k) = c;
    if (t) {
      *reinterpret_cast<uint32_t*>(tile + (row + 16 * i) * LD + lane * 8) = c[0];
      *reinterpret_cast<uint32_t*>(tile + (row + 16 * i) * LD + lane * 8 + 4) = c[1];
    }
  }
  if (!t) return;
  __syncthreads();
  // a NaN block's padding is NaN as well: it never leaves the block's own rows and columns
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = threadIdx.x + THREADS * i, kr = p >> 3, c = (p & 7) * 16;
    if (k0 + kr >= K) continue;
    u32x4_t v;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      uint32_t d = 0u;
#pragma unroll
      for (int b = 0; b < 4; ++b) d |= (uint32_t)tile[(c + 4 * a + b) * LD + kr] << (8 * b);
      v[a] = d;
    }
    *reinterpret_cast<u32x4_t*>(t + (e * K + k0 + kr) * Np + n0 + c) = v;
  }
}

// ------------------------------------------------------------------------------------------------ plan
// Where every expert's rows are and which expert a tile of TILE_ROWS rows belongs to, once for all products of a pass: a workgroup of a product
// then finds its next unit with one read of the table, requested while it multiplies the one before, where a search through starts[] takes
// three dependent ones, 2 us each while the chip is busy.
//   [E + 1] starts (cut off at A), tiles, padding to 8; then for every tile 8 words: expert, its first tile, its tiles, its first
//   row and the row behind its last, padding.  Counts that do not fit into A rows, or are negative, cannot lead a kernel out of bounds.
constexpr int TILE_ROWS = pk_rules::FP8_TILE_ROWS, PLAN_THREADS = 1024, ENTRY = 8;
__host__ __device__ inline int64_t plan_head(int64_t E) { return (E + 2 + ENTRY - 1) / ENTRY * ENTRY; }
inline int64_t plan_tiles(int64_t A, int64_t E) { return pk_rules::fp8_tiles(A, E, TILE_ROWS); }

// sum over the threads before this one (exclusive), all of PLAN_THREADS; *total: over all of them
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* waves /* 16 */, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = __shfl_up(incl, off, PK_WAVE);
    if (lane >= off) incl += o;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int i = 0; i < PLAN_THREADS / 64; ++i) {
    before += i < wave ? waves[i] : 0;
    all += waves[i];
  }
  *total = all;
  return before + incl - v;
}
__device__ __forceinline__ void make_plan(const void* counts, int is_i64, int E, int64_t A, int32_t* plan) {
  __shared__ int64_t waves[16];
  __shared__ int32_t first[PK_MAX_EXPERTS + 1], begin[PK_MAX_EXPERTS + 1];
  const int e = threadIdx.x;
  int64_t n = 0, total;
  if (e < E) n = is_i64 ? reinterpret_cast<const int64_t*>(counts)[e] : reinterpret_cast<const int32_t*>(counts)[e];
  n = n < 0 ? 0 : n > A ? A : n;
  int64_t start = block_scan(n, waves, &total);
  start = start > A ? A : start;
  const int64_t end = start + n > A ? A : start + n;
  const int64_t tiles = (end - start + TILE_ROWS - 1) / TILE_ROWS;
  const int64_t f = block_scan(tiles, waves, &total);
  if (e < E) {
    plan[e] = begin[e] = (int32_t)start;
    first[e] = (int32_t)f;
    if (e == E - 1) {
      plan[E] = begin[E] = (int32_t)end;
      plan[E + 1] = first[E] = (int32_t)total;
    }
  }
  __syncthreads();
  int32_t* const table = plan + plan_head(E);
  for (int t = threadIdx.x; t < (int)total; t += PLAN_THREADS) {
    int lo = 0, hi = E;                      // first[lo] <= t < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= t) lo = mid; else hi = mid;
    }
    // (of experts without tiles, which share their first one with the next, the last one is found)
    *reinterpret_cast<u32x4_t*>(table + t * ENTRY) = u32x4_t{(uint32_t)lo, (uint32_t)first[lo], (uint32_t)(first[lo + 1] - first[lo]), (uint32_t)begin[lo]};
    table[t * ENTRY + 4] = begin[lo + 1];
  }
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_kernel(const void* counts, int is_i64, int E, int64_t A, int32_t* plan) {
  make_plan(counts, is_i64, E, A, plan);
}

// What a pass begins with, in one launch: its rows in blocks, and in front of the forward its plan (by the first workgroup), in front of
// the backward a row map.  (1,777 tokens of 2048 in 8 places each: 17 us, and 5 for either of the others by itself.)
// The map: every row its own number, those of no expert the last one that has one, for pk_grouped_swiglu_wgrad_scaled_t, whose loader
// may stand behind the last expert's rows.  What is in rows of no expert (it may be anything) is thereby not read.
struct Begin {
  const bf16_t* x;
  uint8_t *q, *s;
  int64_t units, A;
  int32_t K, kb, E, is_i64;
  FastDiv by_kb;
  const void* counts;       // forward
  int32_t* plan;
  const int32_t* owned;     // backward: rows that have an expert
  int32_t* map;
};
template <bool FORWARD>
__global__ __launch_bounds__(PLAN_THREADS) void begin_kernel(const Begin p) {
  if (FORWARD && blockIdx.x == 0) {
    make_plan(p.counts, p.is_i64, p.E, p.A, p.plan);
    return;
  }
  const int group = threadIdx.x >> 4;
  const int64_t unit = (int64_t)(blockIdx.x - (FORWARD ? 1 : 0)) * (PLAN_THREADS / 16 * ROW_BLOCKS) + group;
  quantize_blocks<bf16_t, ROW_BLOCKS>(p.x, [](int r) { return (int64_t)(uint32_t)r; }, p.q, p.s, unit, PLAN_THREADS / 16, p.units, p.K, p.kb, p.by_kb);
  if (!FORWARD && p.map) {
    const int64_t r = (int64_t)blockIdx.x * PLAN_THREADS + threadIdx.x;
    if (r < p.A) p.map[r] = (int32_t)(r < *p.owned ? r : *p.owned > 0 ? *p.owned - 1 : 0);
  }
}

// ------------------------------------------------------------------------------------------------ products
// C[rows_e, N] = sum_seg A_seg[rows_e, K] . B_seg[e][N, K]^T in tiles (units) of 128 rows and 256 columns (gate and up: 128 of each).
enum Epilogue { PLAIN = 0, GATE_UP = 1, BWD = 2 };

typedef int intx8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// 8 codes and their power of two
__device__ __forceinline__ bf16x8_t decode8(uint32_t lo, uint32_t hi, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8_t{(bf16_t)a[0], (bf16_t)a[1], (bf16_t)b[0], (bf16_t)b[1], (bf16_t)c[0], (bf16_t)c[1], (bf16_t)d[0], (bf16_t)d[1]};
}

struct Product {
  const uint8_t* A[2];      // codes of the rows, by segment [., lda]
  const uint8_t* As[2];     // and their scales [., scale_row(kt)]
  const uint8_t* B[2];      // weights of a segment (GATE_UP: gate, up), rows of ld codes
  const uint8_t* Bs[2];     // scale of block (n, k) of expert e: Bs[e * bs_e + n * bs_n + k * bs_k]
  int64_t ld, strideB, bs_e;
  int32_t bs_n, bs_k;
  const int32_t* plan;
  FastDiv by_n_tiles;
  int32_t E, kt, nseg, N, n_tiles;
  bool vec;                 // rows of the bf16 tensors are whole 16-byte pieces
  bf16_t* O0;               // C;  GATE_UP: g (optional);  BWD: d_g
  bf16_t* O1;               //     GATE_UP: u (optional);  BWD: d_u
  bf16_t* O2;               //                             BWD: h;  with TRANSPOSED the transposed copies
  uint8_t* Q[2];            //     GATE_UP: h;             BWD: d_g, d_u   in blocks
  uint8_t* Qs[2];
  const bf16_t* G;          // BWD: g and u of the forward
  const bf16_t* U;
  int64_t A_rows;
  int32_t head;             // words in front of the plan's table
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }
// 16 bytes per lane straight into LDS, lane l's at lds_base + 16 l, from a wave-uniform base and an offset per lane.  The
// compiler does not see the transfer: dma_wait and a barrier stand before what reads it.
__device__ __forceinline__ void dma4(uint32_t voff, const void* sbase, uint32_t lds_base) {      // lane l's 4 bytes at lds_base + 4 l
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_base), "v"(voff), "s"(sbase) : "memory");
}
__device__ __forceinline__ void dma16(uint32_t voff, const void* sbase, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(voff), "s"(sbase) : "memory");
}
template <int N>
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // what the wave has read of the LDS or written to it is done
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// A k-tile is a block: 128 bytes of every row, a whole line of the caches (64 bytes at a time come at 39 bytes a cycle and CU out of
// the L2, 128 at 65).  16-byte pieces of a row are XOR-ed with bits of the row, so that 16 neighbouring rows' pieces of one number
// cover the banks.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

// 32 of the 64 reduction bytes of step `half` of a k-tile, for row row0 + lane % 32.  Both operands are dealt alike, and a
// k-tile has one scale, so it does not matter which lane holds which of them.
__device__ __forceinline__ intx8_t fragment(const char* tile, int row0, int half, int lane) {
  const int r = row0 + (lane & 31), c = 4 * half + 2 * (lane >> 5);
  const char* const p = tile + r * BLOCK;
  const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(p + ((c ^ swz(r)) << 4));
  const u32x4_t hi = *reinterpret_cast<const u32x4_t*>(p + (((c + 1) ^ swz(r)) << 4));
  return intx8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// the value of the lane 32 further or back
__device__ __forceinline__ uint32_t other_half(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (threadIdx.x & 32) ? r[0] : r[1];
}
// From fours of 32 columns, dealt to the lower and upper lanes in turn, 16 neighbouring ones to each.
__device__ __forceinline__ void exchange_halves(const floatx16_t& x, float (&f)[16]) {
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[v]), __float_as_uint(x[v + 8]), false, false);
    const int to = (v & 3) + (v & 4) * 2;
    f[to] = __uint_as_float(r[0]);
    f[to + 4] = __uint_as_float(r[1]);
  }
}
__device__ __forceinline__ bf16x8_t pack8(const float (&f)[8]) {
  bf16x8_t v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (bf16_t)f[i];
  return v;
}
// In this form: the compiler would keep the eight floats of a value that is unpacked again, twice the registers.
__device__ __forceinline__ bf16x8_t kept(bf16x8_t v) {
  u32x4_t w = __builtin_bit_cast(u32x4_t, v);
  asm volatile("" : "+v"(w));
  return __builtin_bit_cast(bf16x8_t, w);
}
// Eight neighbouring bf16 of a row in whole 16-byte pieces, of which the first `have` are there (any number)
__device__ __forceinline__ void store8(bf16_t* p, int have, bf16x8_t v) {      // whole pieces
  if (have > 0) *reinterpret_cast<bf16x8_t*>(p) = v;
}
// 16 values as two pieces
__device__ __forceinline__ void pack16(const float (&f)[16], bf16x8_t (&v)[2]) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { a[i] = f[i]; b[i] = f[8 + i]; }
  v[0] = pack8(a);
  v[1] = pack8(b);
}
__device__ __forceinline__ void load16(const bf16_t* p, int have, bf16x8_t (&v)[2]) {      // whole pieces
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[h] = bf16x8_t{};
    if (have > 8 * h) v[h] = *reinterpret_cast<const bf16x8_t*>(p + 8 * h);
  }
}
__device__ __forceinline__ float held(float v) { return (float)(bf16_t)v; }
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// A wave's way of 32 rows x 64 columns of bf16 to 64 columns of 32 rows.  16-byte pieces of a row are XOR-ed with a mix of the row's bits
// that spreads 8 neighbouring rows' writes, and the four rows of a group of a transposing read, over the banks.
constexpr int TR_BYTES = 32 * 64 * 2;
typedef short shortx4_t __attribute__((ext_vector_type(4)));
typedef short shortx8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ int tr_swz(int r) { return ((r & 3) << 1 | (r >> 2 & 1)) ^ (r >> 3 & 1); }
__device__ __forceinline__ void put_row(char* t, int row, int piece, bf16x8_t v) {
  *reinterpret_cast<bf16x8_t*>(t + row * 128 + ((piece ^ tr_swz(row)) << 4)) = v;
}
__device__ __forceinline__ bf16x8_t get_row(const char* t, int row, int piece) {
  return *reinterpret_cast<const bf16x8_t*>(t + row * 128 + ((piece ^ tr_swz(row)) << 4));
}
__device__ __forceinline__ int tr_value(int row, int col) { return row * 128 + (((col >> 3) ^ tr_swz(row)) << 4) + (col & 7) * 2; }
// Rows whose pieces are not 16-byte aligned: a row's 64 columns at a time, a lane to a column, `to` its place in row 0.  (Values by themselves
// from where the products leave them touch 64 lines with an instruction: 4 experts of 2,700 rows 1145 x 1536, down 91 -> 45 us,
// d_x 116 -> 71; 24 of 200 rows 1001 x 361, gate and up 44 -> 25, d_h 62 -> 31.)
__device__ __forceinline__ void store_rows(const char* t, int lane, bf16_t* to, int64_t ld, int rows, bool in) {
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {
    bf16_t v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = *reinterpret_cast<const bf16_t*>(t + tr_value(r0 + r, lane));
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (in && r0 + r < rows) to[(r0 + r) * ld] = v[r];
  }
}
__device__ __forceinline__ void load_rows(char* t, int lane, const bf16_t* from, int64_t ld, int rows, bool in) {
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 8) {
    bf16_t v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = in && r0 + r < rows ? from[(r0 + r) * ld] : (bf16_t)0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) *reinterpret_cast<bf16_t*>(t + tr_value(r0 + r, lane)) = v[r];
  }
}
__device__ __forceinline__ void store_columns(const char* t, int lane, bf16_t* to) {
  // within 16 lanes, lane i points at 4 neighbouring columns of row i / 4 and receives 4 neighbouring rows of column i
  const int g = lane >> 4, i = lane & 15;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    shortx4_t half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 8 * g + 4 * h + (i >> 2), col = 16 * c + 4 * (i & 3);
      half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) shortx4_t*)(t + row * 128 + (((col >> 3) ^ tr_swz(row)) << 4) + (col & 7) * 2));
    }
    *reinterpret_cast<shortx8_t*>(to + (16 * c + i) * 32 + 8 * g) = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

constexpr int unit_chunk = 16;
__device__ __forceinline__ int unit_of_block(int b) {      // neighbouring units on one XCD
  const int x = b % pk_rules::NXCD, q = b / pk_rules::NXCD;
  return ((q / unit_chunk) * pk_rules::NXCD + x) * unit_chunk + (q % unit_chunk);
}

// One persistent workgroup to a CU, eight waves (2 x 4) of 64 x 64 outputs, a ring of three k-tiles.  A workgroup goes through its
// units one after the other: behind a unit's last k-tile it requests the first two of the next one, and the epilogue, which
// needs the LDS for the blocks' maxima alone, runs while they are on their way.
// What bounds it: multiplying and decoding.  With 128 experts of 2048 x 768 and 256 rows each gate and up take 295 us, in which the matrix
// units are busy for 40 % of the cycles and the vector units, which mostly decode (a wave 128 pairs a lane and k-tile for its 32
// products of 32 x 32 x 16), for another 40 %; with 111 rows 156.
// With short sums: a CU has no more than some 128 cache lines (16 KB) on their way from the L2, in order; with 512 rows each a line of
// gate and up takes 664 cycles on average (7 of 10 are in the L2), which is the 24 bytes a cycle that the transfers reach by themselves
// (a unit's first wait, for a scale byte and the first k-tile, takes the stores of the one before along; what that costs is not known).
// Two halves of the waves that took turns at reading the LDS and at multiplying changed nothing, nor did dealing neighbouring units
// by 8, 16 or 32 to an XCD, or experts that start at different k-tiles.  512 rows each, us, against two workgroups of four waves to a CU with
// half-block k-tiles: gate and up 363 : 376, down 225 : 261, d_h (row-major copies) 326 : 354; with 111 rows each 105 : 110 and 64 : 68,
// which is 4.2 TB/s.
// TRANSPOSED (BWD, N a multiple of 256): O0 to O2 are the transposed copies that pk_grouped_swiglu_wgrad_scaled_t reads,
// [padded rows / 32][N][32], expert e's rows from (begin & ~63) + 64 e on, zeros behind its last row up to the end of its last block.
// NARROW (not GATE_UP, whose unit has to have whole blocks of h): units of 128 columns, waves (4 x 2) of 32 x 64, for launches that
// leave CUs without a unit.
constexpr int NT = 512, BM = TILE_ROWS, WIDE = pk_rules::FP8_WIDE, STAGES = 3, A_BYTES = BM * BLOCK, STAGE = A_BYTES + WIDE * BLOCK;
inline int product_lds(int nblk4) { return STAGES * STAGE + nblk4 * BM + 2 * nblk4; }

template <int EPI, bool VEC, bool TRANSPOSED, bool EXACT, bool NARROW>
__global__ __launch_bounds__(NT, 2) void product_kernel(const Product p) {
  constexpr int BN = NARROW ? BLOCK : WIDE, TM = NARROW ? 1 : 2, TN = 2, LA = BM * 8 / NT, LB = BN * 8 / NT, L = LA + LB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = NARROW ? wave >> 1 : wave >> 2, wn = NARROW ? wave & 1 : wave & 3;
  const int wave_row = wm * 32 * TM;         // the wave's first row in the unit
  const int kt4 = scale_row(p.kt), nblk = p.kt * p.nseg, n_blocks = (p.N + BLOCK - 1) / BLOCK, out4 = scale_row(n_blocks);
  const int total = pk_units::as_const(p.plan)[p.E + 1] * p.n_tiles;
  if constexpr (EPI == PLAIN) {              // rows of no expert: zeros
    const int64_t end = p.A_rows * p.N, at = (int64_t)blockIdx.x * NT + tid, threads = (int64_t)gridDim.x * NT;
    const int64_t first = (int64_t)pk_units::as_const(p.plan)[p.E] * p.N;
    if constexpr (VEC) {
      for (int64_t i = first + at * 8; i < end; i += threads * 8) *reinterpret_cast<u32x4_t*>(p.O0 + i) = u32x4_t{};
    } else {
      for (int64_t i = first + at; i < end; i += threads) p.O0[i] = (bf16_t)0.f;
    }
  }
  int step = blockIdx.x;
  if (unit_of_block(step) >= total) return;
  char* const sa = smem + STAGES * STAGE;    // scales of the unit's rows, [words of a row][128]
  char* const sb = sa + kt4 * p.nseg * BM;   // and of its two blocks of columns (GATE_UP: gate, up), [2][nblk]

  // units of an expert are laid out [column tile][row tile]: neighbours share the weights
  int e = 0, nt = 0, mt = 0, begin = 0, rows = 0, row0 = 0, n0 = 0;
  const auto take = [&](int unit, u32x4_t entry, int end) {
    e = __builtin_amdgcn_readfirstlane((int)entry[0]);
    const int first = __builtin_amdgcn_readfirstlane((int)entry[1]), tiles = __builtin_amdgcn_readfirstlane((int)entry[2]);
    begin = __builtin_amdgcn_readfirstlane((int)entry[3]);
    const int local = unit - first * p.n_tiles;
    nt = __builtin_amdgcn_readfirstlane(local / tiles);
    mt = local - nt * tiles;
    row0 = begin + mt * BM;
    rows = min(BM, __builtin_amdgcn_readfirstlane(end) - row0);
    n0 = nt * (EPI == GATE_UP ? BLOCK : BN);
  };
  const auto entry_of = [&](int unit) { return p.plan + p.head + (int64_t)pk_units::fastdiv(unit, p.by_n_tiles) * ENTRY; };

  // Byte offsets of the 16-byte pieces that the thread brings; rows past the expert's end and columns past N read the tile's first
  // ones instead, and what comes of them is stored nowhere.
  uint32_t a_off[LA], b_off[LB];
  uint32_t scale_b = 0;                      // of the unit that comes next, on its way into sb
  const uint32_t ring = lds_addr(smem) + wave * 1024, ring_sa = lds_addr(sa);
  const auto source = [&](int r) { return (int64_t)row0 + (r < rows ? r : 0); };
  const auto fetch = [&](int kt, int stage) {
    const int seg = kt >= p.kt, k = (seg ? kt - p.kt : kt) * BLOCK;
    const uint8_t* const a = uniform(p.A[seg] + k);
    // GATE_UP: a wave's 64 columns are 32 of gate and 32 of up, and so are the tile's rows of B
    const uint8_t* const b = uniform(p.B[EPI == GATE_UP ? wave >> 2 & 1 : seg] + e * p.strideB + k);
    const uint32_t at = ring + stage * STAGE;
#pragma unroll
    for (int i = 0; i < LA; ++i) dma16(a_off[i], a, at + i * NT * 16);
#pragma unroll
    for (int i = 0; i < LB; ++i) dma16(b_off[i], b, at + A_BYTES + i * NT * 16);
  };
  // everything that the k-loop of the unit taken needs, up to two k-tiles, the first one into `stage`
  const auto start = [&](int stage) {
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int s = tid + i * NT, r = s >> 3;
      a_off[i] = (uint32_t)(source(r) * p.ld + ((s & 7) ^ swz(r)) * 16);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int s = tid + i * NT, r = s >> 3;
      const int n = n0 + (EPI == GATE_UP ? (r >> 6) * 32 + (r & 31) : r);
      b_off[i] = (uint32_t)((int64_t)(n < p.N ? n : n0) * p.ld + ((s & 7) ^ swz(r)) * 16);
    }
    const uint32_t s_off = (uint32_t)(source((wave & 1) * 64 + lane) * kt4);
    for (int w = wave; w < kt4 / 2 * p.nseg; w += 8) {      // words of scales, 64 rows at a time
      const int seg = w >= kt4 / 2, d = (seg ? w - kt4 / 2 : w) >> 1;
      dma4(s_off, uniform(p.As[seg] + d * 4), ring_sa + w * 256);
    }
    if (tid < 2 * nblk) {
      const int b = tid >= nblk, k = b ? tid - nblk : tid, seg = k >= p.kt;
      const int nb = EPI == GATE_UP ? nt : min(nt * (BN / BLOCK) + b, n_blocks - 1);
      scale_b = p.Bs[EPI == GATE_UP ? b : seg][e * p.bs_e + (int64_t)nb * p.bs_n + (int64_t)(seg ? k - p.kt : k) * p.bs_k];
    }
    fetch(0, stage);
    if (nblk > 1) fetch(1, stage == STAGES - 1 ? 0 : stage + 1);
  };

  {
    const int unit = unit_of_block(step);
    const int32_t* const entry = entry_of(unit);
    take(unit, *reinterpret_cast<const u32x4_t*>(entry), entry[4]);
  }
  int stage = 0;
  start(stage);
  for (;;) {
    if (tid < 2 * nblk) sb[tid] = (char)scale_b;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    floatx16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    const bool wave_has_rows = wave_row < rows;
    step += gridDim.x;
    const int next_unit = unit_of_block(step);
    const bool more = next_unit < total;
    u32x4_t next_entry = {};
    int next_end = 0;
    for (int kt = 0; kt < nblk; ++kt) {
      // all but the youngest k-tile have landed, everywhere; the stage that the next one goes to has been read
      if (kt + 1 < nblk) dma_wait<L>();
      else dma_wait<0>();
      block_barrier();
      if (kt == 0 && more) {                 // (behind the wait for what it is not to hold up)
        const int32_t* const entry = entry_of(next_unit);
        next_entry = *reinterpret_cast<const u32x4_t*>(entry);
        next_end = entry[4];
      }
      if (kt + 2 < nblk) fetch(kt + 2, stage == 0 ? STAGES - 1 : stage - 1);
      if (wave_has_rows) {
        const char* const at = smem + stage * STAGE;
        const int seg = kt >= p.kt, k = seg ? kt - p.kt : kt;
        const char* const sa_at = sa + (seg * kt4 + (k & ~3)) * BM + (k & 3) + (wave_row + (lane & 31)) * 4;
        const int sc0 = (unsigned char)sb[(EPI == GATE_UP ? 0 : wn >> 1) * nblk + kt];
        const int sc1 = EPI == GATE_UP ? (unsigned char)sb[nblk + kt] : sc0;
        int scale_a[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) scale_a[i] = (unsigned char)sa_at[i * 128];
        intx8_t a[2][TM], b[2][TN];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
          for (int i = 0; i < TM; ++i) a[half][i] = fragment(at, wave_row + i * 32, half, lane);
#pragma unroll
          for (int j = 0; j < TN; ++j) b[half][j] = fragment(at + A_BYTES, wn * 64 + j * 32, half, lane);
        }
        // operands swapped: a lane then holds 4 neighbouring columns of one row,
        //   acc[v] = C[row = lane % 32][col = 8 * (v / 4) + 4 * (lane / 32) + v % 4]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if constexpr (EXACT) {
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
              bf16x8_t av[TM], bv[TN];
#pragma unroll
              for (int i = 0; i < TM; ++i) av[i] = decode8(a[half][i][c], a[half][i][c + 1], pk_fp8::scale_of(scale_a[i]));
#pragma unroll
              for (int j = 0; j < TN; ++j) bv[j] = decode8(b[half][j][c], b[half][j][c + 1], pk_fp8::scale_of(j ? sc1 : sc0));
#pragma unroll
              for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bv[j], av[i], acc[i][j], 0, 0, 0);
            }
          } else {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[half][j], a[half][i], acc[i][j], 0, 0, 0, j ? sc1 : sc0, 0, scale_a[i]);
          }
        }
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    block_barrier();                         // the scales and the last k-tile have been read
    char* const spare = smem + (stage == 0 ? STAGES - 1 : stage - 1) * STAGE;      // its place, free until the next unit's third one

    // The unit that is stored from here on, while the next one is taken.
    const int u_e = e, u_rows = rows, u_row0 = row0, u_n0 = n0, u_nt = nt, u_begin = begin, u_mt = mt;
    const int half16 = (lane >> 5) * 16;
    // BWD: the wave's part of g and u, requested before the next unit's k-tiles, which would be waited for as well
    bf16x8_t gs[TM][TN][2], us[TM][TN][2];
    [[maybe_unused]] char* const tr = spare + 8 * BM * 4 + wave * TR_BYTES;
    [[maybe_unused]] const int col = u_n0 + wn * 64 + lane;      // of a lane that has a column
    if constexpr (EPI == BWD) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (VEC) {
          const int r = wave_row + 32 * i + (lane & 31);
          const int64_t row = u_row0 + (r < u_rows ? r : 0);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int n = u_n0 + wn * 64 + 32 * j + half16;
            load16(p.G + row * p.N + n, p.N - n, gs[i][j]);
            load16(p.U + row * p.N + n, p.N - n, us[i][j]);
          }
        } else {
          const int64_t at = (int64_t)(u_row0 + wave_row + 32 * i) * p.N + col;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            load_rows(tr, lane, (w ? p.U : p.G) + at, p.N, u_rows - wave_row - 32 * i, col < p.N);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int k = 0; k < 2; ++k) (w ? us : gs)[i][j][k] = get_row(tr, lane & 31, 4 * j + 2 * (lane >> 5) + k);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more) {
      take(next_unit, next_entry, next_end);
      start(stage);
    }

    // A lane and the one 32 further have the 32 columns of a row of acc[i][j], in fours; after exchanging halves of them each has 16
    // neighbouring ones, so that loads and stores are 16 bytes wide without a way through the LDS.
    if constexpr (EPI == PLAIN) {
      if (wave_has_rows) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = wave_row + 32 * i + (lane & 31);
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            float f[16];
            bf16x8_t v[2];
            exchange_halves(acc[i][j], f);
            pack16(f, v);
            const int n = u_n0 + wn * 64 + 32 * j + half16;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if constexpr (!VEC) put_row(tr, lane & 31, 4 * j + 2 * (lane >> 5) + k, v[k]);
              else if (r < u_rows) store8(p.O0 + (int64_t)(u_row0 + r) * p.N + n + 8 * k, p.N - n - 8 * k, v[k]);
            }
          }
          if constexpr (!VEC) {
            const int first = wave_row + 32 * i;
            store_rows(tr, lane, p.O0 + (int64_t)(u_row0 + first) * p.N + col, p.N, u_rows - first, col < p.N);
          }
        }
      }
    } else if constexpr (EPI == GATE_UP) {
      // 32 columns of h in a wave, four waves to a block
      const int n = u_n0 + wn * 32 + half16;
      uint32_t* const amax = reinterpret_cast<uint32_t*>(spare);      // [4 waves][128 rows]
      float h[TM][16];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r = wave_row + 32 * i + (lane & 31);
        const bool live = r < u_rows;        // the same in both lanes of a row
        float g[16], u[16];
        exchange_halves(acc[i][0], g);
        exchange_halves(acc[i][1], u);
        uint32_t m = 0u;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          g[v] = held(g[v]);                 // g and u are bf16 tensors, written or not
          u[v] = held(u[v]);
          h[i][v] = (VEC ? p.N - n > v / 8 * 8 : p.N - n > v) ? g[v] * sigmoid(g[v]) * u[v] : 0.f;
          m = umax(m, __float_as_uint(h[i][v]) & 0x7fffffffu);
        }
        amax[wn * BM + r] = umax(m, other_half(m));
        if (p.O0) {
          const int64_t o = (int64_t)(u_row0 + r) * p.N + n;
          bf16x8_t gv[2], uv[2];
          pack16(g, gv);
          pack16(u, uv);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if constexpr (!VEC) {              // 32 columns of g, then those of u
              put_row(tr, lane & 31, 2 * (lane >> 5) + k, gv[k]);
              put_row(tr, lane & 31, 4 + 2 * (lane >> 5) + k, uv[k]);
            } else if (live) {
              store8(p.O0 + o + 8 * k, p.N - n - 8 * k, gv[k]);
              store8(p.O1 + o + 8 * k, p.N - n - 8 * k, uv[k]);
            }
          }
          if constexpr (!VEC) {
            const int first = wave_row + 32 * i, c = u_n0 + wn * 32 + (lane & 31);
            store_rows(tr, lane, (lane < 32 ? p.O0 : p.O1) + (int64_t)(u_row0 + first) * p.N + c, p.N, u_rows - first, c < p.N);
          }
        }
      }
      block_barrier();
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int r = wave_row + 32 * i + (lane & 31);
        const pk_fp8::BlockScale sc = pk_fp8::block_scale(umax(umax(amax[r], amax[BM + r]), umax(amax[2 * BM + r], amax[3 * BM + r])));
        if (r < u_rows) {
          const int64_t row = u_row0 + r;
          *reinterpret_cast<u32x4_t*>(p.Q[0] + (row * n_blocks + u_nt) * BLOCK + wn * 32 + half16) = pk_fp8::codes16(h[i], sc);
          if (wn == 0 && lane < 32) p.Qs[0][row * out4 + u_nt] = (uint8_t)sc.byte;
        }
      }
    } else {
      const int nb = u_nt * (BN / BLOCK) + (wn >> 1);      // the wave's block of columns, shared with its neighbour
      uint32_t* const amax = reinterpret_cast<uint32_t*>(spare);      // [2: d_g, d_u][4 waves][128 rows]
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        asm volatile("" ::: "memory");       // the second half's work not before the first half has left its registers
        __builtin_amdgcn_sched_barrier(0);
        const int r = wave_row + 32 * i + (lane & 31);
        const bool live = r < u_rows;        // the same in both lanes of a row
        const int64_t row = u_row0 + (live ? r : 0);
        const bool chunk = wave_row + 32 * i < u_rows;      // (the same for the whole wave)
        uint32_t mg = 0u, mu = 0u;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          float f[16];
          exchange_halves(acc[i][j], f);
#pragma unroll
          for (int k = 0; k < 2; ++k) {      // eight columns at a time
            const int n = u_n0 + wn * 64 + 32 * j + half16 + 8 * k;
            int have = p.N - n;
            asm volatile("" : "+v"(have));   // compared here and not kept: 32 such masks are more than there are scalar registers
            float g[8], u[8], h[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const float gv = (float)gs[i][j][k][v], uv = (float)us[i][j][k][v], d = f[8 * k + v];
              const float sg = sigmoid(gv), silu = gv * sg;
              const bool in = TRANSPOSED ? live : VEC ? have > 0 : have > v;
              h[v] = !TRANSPOSED || in ? silu * uv : 0.f;
              const float dg = d * uv * (sg * (1.f + gv * (1.f - sg))), du = d * silu;
              g[v] = in ? held(dg) : 0.f;    // bf16 tensors, whose blocks are of what they hold
              u[v] = in ? held(du) : 0.f;
              mg = umax(mg, __float_as_uint(g[v]) & 0x7fffffffu);
              mu = umax(mu, __float_as_uint(u[v]) & 0x7fffffffu);
            }
            asm volatile("" : "+v"(mg), "+v"(mu));      // step by step: as one reduction it would keep all values
            gs[i][j][k] = kept(pack8(g));    // d_g and d_u take the place of g and u
            us[i][j][k] = kept(pack8(u));
            if constexpr (TRANSPOSED || !VEC) {
              put_row(tr, lane & 31, 4 * j + 2 * (lane >> 5) + k, pack8(h));
            } else if (live) {
              store8(p.O0 + row * p.N + n, have, gs[i][j][k]);
              store8(p.O1 + row * p.N + n, have, us[i][j][k]);
              store8(p.O2 + row * p.N + n, have, pack8(h));
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if constexpr (TRANSPOSED || !VEC) {
          if (chunk) {
            const int first = wave_row + 32 * i;
            const auto store = [&](bf16_t* out) {
              if constexpr (TRANSPOSED) {
                const int64_t padded = (u_begin & ~63) + 64 * (int64_t)u_e + u_mt * BM + first;
                store_columns(tr, lane, out + (padded / 32 * p.N + u_n0 + wn * 64) * 32);
              } else {
                store_rows(tr, lane, out + (int64_t)(u_row0 + first) * p.N + col, p.N, u_rows - first, col < p.N);
              }
            };
            store(p.O2);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int k = 0; k < 2; ++k) put_row(tr, lane & 31, 4 * j + 2 * (lane >> 5) + k, gs[i][j][k]);
            store(p.O0);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int k = 0; k < 2; ++k) put_row(tr, lane & 31, 4 * j + 2 * (lane >> 5) + k, us[i][j][k]);
            store(p.O1);
          }
        }
        amax[wn * BM + r] = umax(mg, other_half(mg));
        amax[(4 + wn) * BM + r] = umax(mu, other_half(mu));
      }
      block_barrier();
      if (nb < n_blocks) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = wave_row + 32 * i + (lane & 31);
          const pk_fp8::BlockScale scg = pk_fp8::block_scale(umax(amax[wn * BM + r], amax[(wn ^ 1) * BM + r]));
          const pk_fp8::BlockScale scu = pk_fp8::block_scale(umax(amax[(4 + wn) * BM + r], amax[(4 + (wn ^ 1)) * BM + r]));
          if (r < u_rows) {
            const int64_t row = u_row0 + r, at = (row * n_blocks + nb) * BLOCK + (wn & 1) * 64 + half16;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              float g[16], u[16];
#pragma unroll
              for (int v = 0; v < 16; ++v) { g[v] = (float)gs[i][j][v >> 3][v & 7]; u[v] = (float)us[i][j][v >> 3][v & 7]; }
              *reinterpret_cast<u32x4_t*>(p.Q[0] + at + 32 * j) = pk_fp8::codes16(g, scg);
              *reinterpret_cast<u32x4_t*>(p.Q[1] + at + 32 * j) = pk_fp8::codes16(u, scu);
            }
            if ((wn & 1) == 0 && lane < 32) {
              p.Qs[0][row * out4 + nb] = (uint8_t)scg.byte;
              p.Qs[1][row * out4 + nb] = (uint8_t)scu.byte;
            }
          }
        }
      }
    }
    if (!more) return;
  }
}

template <int EPI>
int launch_product(Product p, int64_t A, int kernel_id, hipStream_t s, bool short_sums, bool transposed = false) {
  const bool narrow = EPI != GATE_UP && !transposed && pk_rules::fp8_narrow(A, p.E, p.N);
  p.n_tiles = (int32_t)pk_ceil_div(p.N, EPI == GATE_UP || narrow ? BLOCK : WIDE);
  p.by_n_tiles = pk_units::make_fastdiv(p.n_tiles);
  p.head = (int32_t)plan_head(p.E);
  p.A_rows = A;
  const int64_t units = plan_tiles(A, p.E) * p.n_tiles;
  if (units > 0x7fff0000ll) return PK_ERR_SHAPE;      // (steps past the last unit are formed as well)
  const int64_t per = unit_chunk * pk_rules::NXCD, all = pk_ceil_div(units, per) * per;
  const dim3 grid((unsigned)(all < 256 ? all : 256)), block(NT);      // one for every CU
  const int lds = product_lds(scale_row(p.kt) * p.nseg);
  const auto launch = [&](auto kernel, bool (&ready)[PK_MAX_DEVICES]) -> int {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= PK_MAX_DEVICES) return PK_ERR_UNSUPPORTED;
    if (!ready[dev]) {                       // (more than one thread may do it)
      const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
      if (err != hipSuccess) return (int)err;
      ready[dev] = true;
    }
    PK_LAUNCH_NOCHECK(kernel_id, s, kernel, grid, block, lds, s, p);
    PK_RETURN_IF_LAUNCH_FAILED();
    return PK_OK;
  };
  static bool ready[10][PK_MAX_DEVICES] = {};
  const bool exact = pk_rules::fp8_exact(short_sums, A, p.E);
  if constexpr (EPI == BWD)
    if (transposed)
      return exact ? launch(product_kernel<EPI, true, true, true, false>, ready[9]) : launch(product_kernel<EPI, true, true, false, false>, ready[8]);
  const auto pick = [&](auto wide_or_narrow, bool (*done)[PK_MAX_DEVICES]) {
    constexpr bool N = decltype(wide_or_narrow)::value;
    if (exact)
      return p.vec ? launch(product_kernel<EPI, true, false, true, N>, done[3]) : launch(product_kernel<EPI, false, false, true, N>, done[2]);
    return p.vec ? launch(product_kernel<EPI, true, false, false, N>, done[1]) : launch(product_kernel<EPI, false, false, false, N>, done[0]);
  };
  if constexpr (EPI != GATE_UP)
    if (narrow) return pick(std::true_type(), ready + 4);
  return pick(std::false_type(), ready);
}

// ------------------------------------------------------------------------------------------------ few rows
// A handful of rows an expert: the weights are the traffic (one token, 8 of 128 experts, 2048 x 768: 38 MB), so every wave requests
// all it needs of them at once, straight into registers, and nothing runs before that needs a launch of its own.  The rows are
// quantized on their way in, and a workgroup finds its expert in the row counts by itself.  Four v_mfma_f32_16x16x32_bf16: 16
// rows of x, 16 of a weight, one block of both.
//   gate_up_few: 16 columns of gate and up to a workgroup, its eight waves take every eighth block of the reduction; h stays fp32,
//                since a block of it belongs to eight workgroups
//   down_few:    h in blocks into the LDS, then 16 columns to each of four waves
// One token of 8 experts of 2048 x 768 takes 11.9 + 7.1 us, of which the weights are 7.7 at the rate of a copy: the rest is the chain of
// counts, weights, sums, twice.  24 tokens (some 100 of 128 experts) 73 + 44 us for 470 MB, 4.0 TB/s.  Where H is no multiple of 8
// gate_up_few loads its rows value by value (8 rows of 8 experts, 2048 x 768 16 us, 2047 x 767 21; 128 of 64, 1000 x 360 37, 1001 x 361 55).
constexpr int FEW_ROWS = pk_rules::FP8_FEW_ROWS;

struct Few {
  const void* counts;
  int32_t is_i64, E, H, I;
  int64_t A;
  const bf16_t* x;
  const uint8_t *q1, *s1, *q3, *s3, *q2, *s2;
  bf16_t *g, *u;            // optional
  float* h;                 // [A, I]
  bf16_t* y;
  int32_t n_cols;           // column tiles
  bool whole;               // H is a multiple of 8
  FastDiv by_cols;
};

// Sums over the lanes up to this one, cut off at `cap` (of numbers up to 2^31 that are not negative cutting off can be done at every
// step): shifts within rows of 16 lanes, then the rows' last lanes to the rows behind them.
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t cap) {
#define PK_STEP(CTRL, ROWS)                                                                                    \
  {                                                                                                            \
    const uint32_t sum = v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); \
    v = sum < cap ? sum : cap;                                                                                 \
  }
  PK_STEP(0x111, 0xf) PK_STEP(0x112, 0xf) PK_STEP(0x114, 0xf) PK_STEP(0x118, 0xf) PK_STEP(0x142, 0xa) PK_STEP(0x143, 0xc)
#undef PK_STEP
  return v;
}

// The row tile of that number: its expert and rows.  Every wave looks for itself.  total_rows: rows that belong to an expert.
__device__ __forceinline__ bool find_rows(const Few& p, int tile, int& e_out, int& row0, int& rows, int& total_rows) {
  const int lane = threadIdx.x & 63, epl = (p.E + 63) >> 6, lo = lane * epl, hi = min(p.E, lo + epl);
  const uint32_t A = (uint32_t)p.A;
  const auto count = [&](int e) -> uint32_t {
    const int64_t n = p.is_i64 ? reinterpret_cast<const int64_t*>(p.counts)[e] : reinterpret_cast<const int32_t*>(p.counts)[e];
    return n < 0 ? 0u : n > p.A ? A : (uint32_t)n;
  };
  uint32_t mine = 0u;
  for (int e = lo; e < hi; ++e) mine = min(mine + count(e), A);
  const uint32_t incl = scan(mine, A);
  const uint32_t begin = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)incl, 0x138, 0xf, 0xf, false);      // of the lane before
  total_rows = (int)__builtin_amdgcn_readlane((int)incl, 63);
  uint32_t tiles = 0u;
  for (uint32_t e = lo, at = begin; (int)e < hi; ++e) {
    const uint32_t end = min(at + count((int)e), A);
    tiles += (end - at + FEW_ROWS - 1) / FEW_ROWS;
    at = end;
  }
  const uint32_t sum = scan(tiles, 0x7fffffffu);
  const unsigned long long owner = __ballot(tile >= (int)(sum - tiles) && tile < (int)sum);
  if (owner == 0ull) return false;
  const int src = __ffsll((long long)owner) - 1;
  uint32_t left = (uint32_t)(tile - __builtin_amdgcn_readlane((int)(sum - tiles), src));
  uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)begin, src);
  int e = src * epl;
  for (;; ++e) {                             // ends: the tile is one of this lane's experts'
    const uint32_t end = min(at + count(e), A), n = (end - at + FEW_ROWS - 1) / FEW_ROWS;
    if (left < n) {
      e_out = __builtin_amdgcn_readfirstlane(e);
      row0 = __builtin_amdgcn_readfirstlane((int)(at + left * FEW_ROWS));
      rows = __builtin_amdgcn_readfirstlane((int)min((uint32_t)FEW_ROWS, end - at - left * FEW_ROWS));
      return true;
    }
    left -= n;
    at = end;
  }
}

__device__ __forceinline__ uint32_t max_of_row(uint32_t m) {      // over the four lanes that share a row of 16
  m = umax(m, __shfl_xor(m, 16));
  return umax(m, __shfl_xor(m, 32));
}
// a block: 32 codes of each to a lane
__device__ __forceinline__ floatx4_t multiply_block(intx8_t w, int sw, intx8_t x, int sx, floatx4_t acc) {
  const float fw = pk_fp8::scale_of((uint32_t)sw), fx = pk_fp8::scale_of((uint32_t)sx);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decode8(w[2 * c], w[2 * c + 1], fw), decode8(x[2 * c], x[2 * c + 1], fx), acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ intx8_t as_fragment(u32x4_t a, u32x4_t b) {
  return intx8_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

__global__ __launch_bounds__(512, 2) void gate_up_few_kernel(const Few p) {
  constexpr int WAVES = 8, AHEAD = 2;        // blocks of a wave that are requested at once
  __shared__ float part[WAVES][2][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = pk_units::fastdiv((int)blockIdx.x, p.by_cols), ct = (int)blockIdx.x - tile * p.n_cols;
  int e, row0, rows, total_rows;
  if (!find_rows(p, tile, e, row0, rows, total_rows)) return;
  const int hb = (p.H + BLOCK - 1) / BLOCK, ib = (p.I + BLOCK - 1) / BLOCK, Hp = hb * BLOCK;
  const int r = lane & 15, quarter = lane >> 4, n0 = ct * 16;
  const int64_t wrow = (int64_t)e * p.I + (n0 + r < p.I ? n0 + r : n0);
  const uint8_t* const w1 = p.q1 + wrow * Hp + quarter * 32;
  const uint8_t* const w3 = p.q3 + wrow * Hp + quarter * 32;
  const int64_t srow = ((int64_t)e * ib + n0 / BLOCK) * hb;
  const bf16_t* const x = p.x + (int64_t)(row0 + (r < rows ? r : 0)) * p.H + quarter * 32;
  floatx4_t ag = {0.f, 0.f, 0.f, 0.f}, au = ag;
  for (int b0 = wave; b0 < hb; b0 += WAVES * AHEAD) {
    u32x4_t wg[AHEAD][2], wu[AHEAD][2];
    int sg[AHEAD], su[AHEAD];
    bf16x8_t xs[AHEAD][4];
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
      const int b = b0 + t * WAVES < hb ? b0 + t * WAVES : b0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        wg[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w1 + b * BLOCK + 16 * i));
        wu[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w3 + b * BLOCK + 16 * i));
      }
      sg[t] = p.s1[srow + b];
      su[t] = p.s3[srow + b];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = b * BLOCK + quarter * 32 + 8 * i, have = r < rows ? p.H - k : 0;
        if (p.whole) {
          xs[t][i] = bf16x8_t{};
          if (have > 0) __builtin_memcpy(&xs[t][i], x + b * BLOCK + 8 * i, 16);
        } else {
#pragma unroll
          for (int v = 0; v < 8; ++v) xs[t][i][v] = v < have ? x[b * BLOCK + 8 * i + v] : (bf16_t)0.f;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
      if (b0 + t * WAVES >= hb) break;
      float f[2][16];
      uint32_t m = 0u;
#pragma unroll
      for (int v = 0; v < 32; ++v) {
        f[v >> 4][v & 15] = (float)xs[t][v >> 3][v & 7];
        m = umax(m, __float_as_uint(f[v >> 4][v & 15]) & 0x7fffffffu);
      }
      const pk_fp8::BlockScale sc = pk_fp8::block_scale(max_of_row(m));
      const intx8_t xf = as_fragment(pk_fp8::codes16(f[0], sc), pk_fp8::codes16(f[1], sc));
      ag = multiply_block(as_fragment(wg[t][0], wg[t][1]), sg[t], xf, (int)sc.byte, ag);
      au = multiply_block(as_fragment(wu[t][0], wu[t][1]), su[t], xf, (int)sc.byte, au);
    }
  }
  // acc[v] = C[row = lane % 16][col = 4 * (lane / 16) + v]
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    part[wave][0][v][lane] = ag[v];
    part[wave][1][v][lane] = au[v];
  }
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int v = threadIdx.x >> 6, n = n0 + 4 * quarter + v;
  float g = 0.f, u = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    g += part[w][0][v][lane];
    u += part[w][1][v][lane];
  }
  if (r >= rows || n >= p.I) return;
  const int64_t o = (int64_t)(row0 + r) * p.I + n;
  g = held(g);
  u = held(u);
  if (p.g) {
    p.g[o] = (bf16_t)g;
    p.u[o] = (bf16_t)u;
  }
  p.h[o] = g * sigmoid(g) * u;
}

// A row tile's rows of K values in blocks into the LDS, 16 lanes to a block; rows that are not there stay as they are, since no other
// row sees them.
template <typename T>
__device__ __forceinline__ void rows_into_lds(const T* from, int64_t ld_from, int rows, int K, uint8_t* q, int ld, uint8_t* qs) {
  const int nb = (K + BLOCK - 1) / BLOCK;
  for (int i = threadIdx.x >> 4; i < rows * nb; i += (int)blockDim.x >> 4) {
    const int r = i / nb, b = i - r * nb, k = b * BLOCK + (threadIdx.x & 15) * 8;
    float f[8];
    load8<T>(from + r * ld_from + k, K - k, f);
    uint32_t codes[2], byte;
    pk_fp8::quantize8(f, codes, byte);
    *reinterpret_cast<u32x2_t*>(q + r * ld + k) = u32x2_t{codes[0], codes[1]};
    if ((threadIdx.x & 15) == 0) qs[r * nb + b] = (uint8_t)byte;
  }
}
__host__ __device__ inline int few_lds(int64_t K) {
  const int nb = (int)((K + BLOCK - 1) / BLOCK);
  return FEW_ROWS * (nb * BLOCK + 16) + FEW_ROWS * nb;
}

// The products of a row tile in the LDS with `tiles` times 16 columns of MATS weights, block after block, each requested D steps ahead (but
// a step waits for its scale byte, requested last, and memory answers in order: what was requested before is waited for as well);
// done(c, acc) for every 16 columns.  w: the lane's part of column tile 0, `next` bytes further for the next one.
template <int MATS, int D, typename Done>
__device__ __forceinline__ void stream_columns(const uint8_t* const (&w)[MATS], int64_t next, const uint8_t* const (&sw)[MATS], int64_t next_scale,
                                               int nb, int tiles, const uint8_t* q, int ld, const uint8_t* qs, bool ready, Done&& done) {
  const int r = threadIdx.x & 15, quarter = (threadIdx.x >> 4) & 3, steps = tiles * nb;
  u32x4_t ring[D][MATS][2];
  int fc = 0, fb = 0;                        // what is requested next; the last one again where nothing is left
  const auto request = [&](auto& slot) {
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) slot[m][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w[m] + fc * next + fb * BLOCK + 16 * i));
    if (fc * nb + fb + 1 < steps) {
      ++fb;
      if (fb == nb) { fb = 0; ++fc; }
    }
  };
#pragma unroll
  for (int t = 0; t < D; ++t) {
    request(ring[t]);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (!ready) __syncthreads();               // the rows are in the LDS
  floatx4_t acc[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) acc[m] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  int c = 0, b = 0;
  const auto step = [&](auto& slot) {
    const u32x4_t* const f = reinterpret_cast<const u32x4_t*>(q + r * ld + b * BLOCK + quarter * 32);
    const intx8_t x = as_fragment(f[0], f[1]);
    const int sx = qs[r * nb + b];
#pragma unroll
    for (int m = 0; m < MATS; ++m) acc[m] = multiply_block(as_fragment(slot[m][0], slot[m][1]), sw[m][c * next_scale + b], x, sx, acc[m]);
    if (++b == nb) {
      done(c, acc);
#pragma unroll
      for (int m = 0; m < MATS; ++m) acc[m] = floatx4_t{0.f, 0.f, 0.f, 0.f};
      b = 0;
      ++c;
    }
  };
  int s = 0;
  for (; s + D < steps; s += D) {
#pragma unroll
    for (int t = 0; t < D; ++t) {
      step(ring[t]);
      request(ring[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int t = 0; t < D; ++t)
    if (s + t < steps) step(ring[t]);
}

// gate and up with more workgroups than it takes to fill the chip: 16 columns and the whole reduction to a wave, nothing to add up.
__global__ __launch_bounds__(512, 4) void gate_up_stream_kernel(const Few p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tile = pk_units::fastdiv((int)blockIdx.x, p.by_cols), ct = (int)blockIdx.x - tile * p.n_cols;
  int e, row0, rows, total_rows;
  if (!find_rows(p, tile, e, row0, rows, total_rows)) return;
  const int hb = (p.H + BLOCK - 1) / BLOCK, ib = (p.I + BLOCK - 1) / BLOCK, Hp = hb * BLOCK, ld = Hp + 16;
  const int r = lane & 15, quarter = lane >> 4, n0 = (ct * 8 + wave) * 16;
  uint8_t* const q = reinterpret_cast<uint8_t*>(smem);
  uint8_t* const qs = q + FEW_ROWS * ld;
  // (a wave behind the last column reads the first ones' weights and stores nothing)
  const int64_t at = ((int64_t)e * p.I + (n0 + r < p.I ? n0 + r : 0)) * Hp + quarter * 32, sat = ((int64_t)e * ib + ct) * hb;
  const uint8_t* const w[2] = {p.q1 + at, p.q3 + at};
  const uint8_t* const sw[2] = {p.s1 + sat, p.s3 + sat};
  rows_into_lds<bf16_t>(p.x + (int64_t)row0 * p.H, p.H, rows, p.H, q, ld, qs);
  stream_columns<2, 4>(w, 0, sw, 0, hb, 1, q, ld, qs, false, [&](int, const floatx4_t (&acc)[2]) {
    if (r >= rows) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int n = n0 + 4 * quarter + v;
      if (n >= p.I) continue;
      const int64_t o = (int64_t)(row0 + r) * p.I + n;
      const float g = held(acc[0][v]), u = held(acc[1][v]);
      if (p.g) {
        p.g[o] = (bf16_t)g;
        p.u[o] = (bf16_t)u;
      }
      p.h[o] = g * sigmoid(g) * u;
    }
  });
}

// `tiles` times 64 columns to a workgroup of four waves.
__global__ __launch_bounds__(256, 4) void down_few_kernel(const Few p, int units, int tiles) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int hb = (p.H + BLOCK - 1) / BLOCK, ib = (p.I + BLOCK - 1) / BLOCK, Ip = ib * BLOCK, ld = Ip + 16;
  int e, row0, rows, total_rows;
  if ((int)blockIdx.x >= units) {            // rows of no expert: zeros
    find_rows(p, -1, e, row0, rows, total_rows);
    const int64_t first = (int64_t)total_rows * p.H, step = (int64_t)(gridDim.x - units) * blockDim.x;
    for (int64_t i = first + (int64_t)(blockIdx.x - units) * blockDim.x + threadIdx.x; i < p.A * p.H; i += step) p.y[i] = (bf16_t)0.f;
    return;
  }
  const int tile = pk_units::fastdiv((int)blockIdx.x, p.by_cols), ct = (int)blockIdx.x - tile * p.n_cols;
  if (!find_rows(p, tile, e, row0, rows, total_rows)) return;
  // the wave's columns: 16 * tiles of them from n0 on
  const int r = lane & 15, quarter = lane >> 4, n0 = (ct * 4 + wave) * 16 * tiles;
  uint8_t* const q = reinterpret_cast<uint8_t*>(smem);
  uint8_t* const qs = q + FEW_ROWS * ld;
  const int mine = min(tiles, (p.H - n0 + 15) / 16);
  rows_into_lds<float>(p.h + (int64_t)row0 * p.I, p.I, rows, p.I, q, ld, qs);
  __syncthreads();
  if (mine <= 0) return;
  for (int c0 = 0; c0 < mine;) {             // columns that share a row of scales, and whole tiles or a last one that is not
    const int n = n0 + 16 * c0;
    int take = min(mine - c0, (BLOCK - n % BLOCK) / 16);
    if (n + 16 * take > p.H && take > 1) --take;
    const uint8_t* const w[1] = {p.q2 + ((int64_t)e * p.H + (n + r < p.H ? n + r : n)) * Ip + quarter * 32};
    const uint8_t* const sw[1] = {p.s2 + ((int64_t)e * hb + n / BLOCK) * ib};
    stream_columns<1, 6>(w, (int64_t)16 * Ip, sw, 0, ib, take, q, ld, qs, true, [&](int c, const floatx4_t (&acc)[1]) {
      if (r >= rows) return;
      const int at = n + 16 * c + 4 * quarter;
      bf16_t* const to = p.y + (int64_t)(row0 + r) * p.H + at;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (at + v < p.H) to[v] = (bf16_t)acc[0][v];
    });
    c0 += take;
  }
}

// Common checks of the products.  Offsets from an operand's first row are 32 bits wide.
int check(int64_t A, int64_t H, int64_t I, int64_t E) {
  if (A < 0 || H <= 0 || I <= 0 || E <= 0) return PK_ERR_ARG;
  if (A > 0x7fffffffll || E > PK_MAX_EXPERTS || H > PK_FP8_MAX_HIDDEN || I > PK_FP8_MAX_INTER) return PK_ERR_SHAPE;
  if (A * blocks_of(H) * BLOCK > 0xffffffffll || A * blocks_of(I) * BLOCK > 0xffffffffll) return PK_ERR_SHAPE;
  return PK_OK;
}
bool all_aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!pk_aligned16(q)) return false;
  return true;
}
bool word_aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if ((uintptr_t)q & 3) return false;
  return true;
}
bool all_set(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!q) return false;
  return true;
}
bool bf16_pieces(int64_t width, std::initializer_list<const void*> ps) { return width % 8 == 0 && all_aligned(ps); }

}  // namespace

extern "C" {

int pk_fp8_quantize_rows_of(const void* x, int dtype, int64_t x_rows, const int32_t* row_map, int64_t row_map_div, uint8_t* q, uint8_t* scales,
                            int64_t rows, int64_t K, pk_stream_t stream) {
  if (rows < 0 || x_rows < 0 || K <= 0 || row_map_div < 1 || !pk_dtype_ok(dtype) || (!row_map && rows > x_rows)) return PK_ERR_ARG;
  if (rows == 0) return PK_OK;
  if (!all_set({x, q, scales})) return PK_ERR_ARG;
  if (!pk_aligned16(q)) return PK_ERR_ALIGN;
  const int64_t kb = blocks_of(K), units = rows * kb;
  if (K > 0x7fffff00ll || rows > 0x7fffffffll || units > 0x7fffffffll || row_map_div > 0x7fffffffll) return PK_ERR_SHAPE;
  const FastDiv div = pk_units::make_fastdiv(row_map_div), by_kb = pk_units::make_fastdiv(kb);
  // of the row map, those that name a row of x
  const int64_t entries = x_rows > 0x7fffffffll / row_map_div ? 0x80000000ll : x_rows * row_map_div;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)pk_ceil_div(units, THREADS / 16 * ROW_BLOCKS)), block(THREADS);
  if (dtype == PK_BF16)
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_rows_kernel<bf16_t>), grid, block, 0, s, (const bf16_t*)x, row_map, entries, div, q,
                      scales, units, (int)K, (int)kb, by_kb);
  else
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_rows_kernel<float>), grid, block, 0, s, (const float*)x, row_map, entries, div, q,
                      scales, units, (int)K, (int)kb, by_kb);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int pk_fp8_quantize_rows(const void* x, int dtype, const int32_t* row_map, int64_t row_map_div, uint8_t* q, uint8_t* scales, int64_t rows,
                         int64_t K, pk_stream_t stream) {
  return pk_fp8_quantize_rows_of(x, dtype, 0x7fffffffffffffffll, row_map, row_map_div, q, scales, rows, K, stream);
}

int pk_fp8_quantize_weights(int count, const void* const* w, int dtype, uint8_t* const* q, uint8_t* const* q_t, uint8_t* const* scales, int64_t E,
                            const int64_t* N, const int64_t* K, pk_stream_t stream) {
  if (count < 0 || count > PK_FP8_MAX_WEIGHTS || E < 0 || !pk_dtype_ok(dtype)) return PK_ERR_ARG;
  if (count == 0 || E == 0) return PK_OK;
  if (!all_set({w, q, scales, N, K})) return PK_ERR_ARG;
  Weights p = {};
  p.count = count;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (N[i] <= 0 || K[i] <= 0 || !all_set({w[i], q[i], scales[i]})) return PK_ERR_ARG;
    if (!all_aligned({q[i], q_t ? q_t[i] : nullptr})) return PK_ERR_ALIGN;
    if (N[i] > 0x7fffff00ll || K[i] > 0x7fffff00ll) return PK_ERR_SHAPE;
    const int64_t nb = blocks_of(N[i]), kb = blocks_of(K[i]);
    if (E > 0x7fffffffll / nb || E * nb > (0x7fffffffll - blocks) / kb) return PK_ERR_SHAPE;
    p.w[i] = w[i]; p.q[i] = q[i]; p.t[i] = q_t ? q_t[i] : nullptr; p.s[i] = scales[i];
    p.first[i] = (int32_t)blocks; p.N[i] = (int32_t)N[i]; p.K[i] = (int32_t)K[i];
    p.by_nb[i] = pk_units::make_fastdiv(nb); p.by_kb[i] = pk_units::make_fastdiv(kb);
    blocks += E * nb * kb;
  }
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks), block(THREADS);
  if (dtype == PK_BF16) PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_weights_kernel<bf16_t>), grid, block, 0, s, p);
  else PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_weights_kernel<float>), grid, block, 0, s, p);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int64_t pk_fp8_plan_bytes(int64_t A, int64_t E) {
  if (A < 0 || E <= 0 || E > PK_MAX_EXPERTS || A > 0x7fffffffll) return PK_ERR_ARG;
  return (plan_head(E) + plan_tiles(A, E) * ENTRY) * 4;
}

int pk_fp8_plan(const void* counts, int counts_is_i64, int64_t E, int64_t A, int32_t* plan, pk_stream_t stream) {
  if (A < 0 || E <= 0) return PK_ERR_ARG;
  if (E > PK_MAX_EXPERTS || A > 0x7fffffffll) return PK_ERR_SHAPE;
  if (!counts || !plan) return PK_ERR_ARG;
  if (!pk_aligned16(plan)) return PK_ERR_ALIGN;
  PK_LAUNCH_NOCHECK(pk_timing::K_COUNTS_TO_STARTS, (hipStream_t)stream, plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, (hipStream_t)stream, counts,
                    counts_is_i64, (int)E, A, plan);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

static int begin(Begin p, const void* x, uint8_t* q, uint8_t* scales, int64_t A, int64_t K, int64_t E, bool forward, pk_stream_t stream) {
  if (!all_set({x, q, scales, p.plan})) return PK_ERR_ARG;
  if (!all_aligned({q, p.plan})) return PK_ERR_ALIGN;
  p.x = (const bf16_t*)x; p.q = q; p.s = scales; p.A = A; p.K = (int32_t)K; p.E = (int32_t)E; p.kb = (int32_t)blocks_of(K);
  p.by_kb = pk_units::make_fastdiv(p.kb);
  p.units = A * p.kb;
  if (p.units > 0x7fffffffll) return PK_ERR_SHAPE;
  const dim3 grid((unsigned)(pk_ceil_div(p.units, PLAN_THREADS / 16 * ROW_BLOCKS) + (forward ? 1 : 0))), block(PLAN_THREADS);
  const hipStream_t s = (hipStream_t)stream;
  if (forward) PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (begin_kernel<true>), grid, block, 0, s, p);
  else PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (begin_kernel<false>), grid, block, 0, s, p);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int pk_fp8_begin(const void* x, const void* counts, int counts_is_i64, uint8_t* q, uint8_t* scales, int32_t* plan, int64_t A, int64_t H, int64_t E,
                 pk_stream_t stream) {
  if (const int rc = check(A, H, 1, E)) return rc;
  if (A == 0) return pk_fp8_plan(counts, counts_is_i64, E, A, plan, stream);
  if (!counts) return PK_ERR_ARG;
  Begin p = {};
  p.counts = counts; p.is_i64 = counts_is_i64; p.plan = plan;
  return begin(p, x, q, scales, A, H, E, true, stream);
}

int pk_fp8_begin_backward(const void* d_y, const int32_t* plan, uint8_t* q, uint8_t* scales, int32_t* row_map, int64_t A, int64_t H, int64_t E,
                          pk_stream_t stream) {
  if (const int rc = check(A, H, 1, E)) return rc;
  if (A == 0) return PK_OK;
  if (!plan) return PK_ERR_ARG;
  Begin p = {};
  p.plan = const_cast<int32_t*>(plan); p.owned = plan + E; p.map = row_map;
  return begin(p, d_y, q, scales, A, H, E, false, stream);
}

static int gate_up(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w1, const uint8_t* s1, const uint8_t* w3, const uint8_t* s3,
                   const int32_t* plan, void* g, void* u, uint8_t* h, uint8_t* h_scales, int64_t A, int64_t H, int64_t I, int64_t E,
                   pk_stream_t stream, bool short_sums) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({x, x_scales, w1, s1, w3, s3, plan, h, h_scales}) || !g != !u) return PK_ERR_ARG;
  if (!all_aligned({x, w1, w3, h, plan}) || !word_aligned({x_scales})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = p.A[1] = x; p.As[0] = p.As[1] = x_scales;
  p.B[0] = w1; p.B[1] = w3; p.Bs[0] = s1; p.Bs[1] = s3;
  p.kt = (int32_t)blocks_of(H); p.nseg = 1; p.N = (int32_t)I; p.E = (int32_t)E; p.plan = plan;
  p.ld = blocks_of(H) * BLOCK; p.strideB = I * p.ld;
  p.bs_n = p.kt; p.bs_k = 1; p.bs_e = blocks_of(I) * p.kt;
  p.vec = bf16_pieces(I, {g, u});
  p.O0 = (bf16_t*)g; p.O1 = (bf16_t*)u; p.Q[0] = h; p.Qs[0] = h_scales;
  return launch_product<GATE_UP>(p, A, pk_timing::K_FP8_GATE_UP, (hipStream_t)stream, short_sums);
}

int pk_fp8_gate_up(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w1, const uint8_t* s1, const uint8_t* w3, const uint8_t* s3,
                   const int32_t* plan, void* g, void* u, uint8_t* h, uint8_t* h_scales, int64_t A, int64_t H, int64_t I, int64_t E,
                   pk_stream_t stream) {
  return gate_up(x, x_scales, w1, s1, w3, s3, plan, g, u, h, h_scales, A, H, I, E, stream, false);
}

int pk_fp8_gate_up_short(const uint8_t* x, const uint8_t* x_scales, const uint8_t* w1, const uint8_t* s1, const uint8_t* w3, const uint8_t* s3,
                         const int32_t* plan, void* g, void* u, uint8_t* h, uint8_t* h_scales, int64_t A, int64_t H, int64_t I, int64_t E,
                         pk_stream_t stream) {
  return gate_up(x, x_scales, w1, s1, w3, s3, plan, g, u, h, h_scales, A, H, I, E, stream, true);
}

static int down(const uint8_t* h, const uint8_t* h_scales, const uint8_t* w2, const uint8_t* s2, const int32_t* plan, void* y, int64_t A,
                int64_t H, int64_t I, int64_t E, pk_stream_t stream, bool short_sums) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({h, h_scales, w2, s2, plan, y})) return PK_ERR_ARG;
  if (!all_aligned({h, w2, plan}) || !word_aligned({h_scales})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = p.A[1] = h; p.As[0] = p.As[1] = h_scales;
  p.B[0] = p.B[1] = w2; p.Bs[0] = p.Bs[1] = s2;
  p.kt = (int32_t)blocks_of(I); p.nseg = 1; p.N = (int32_t)H; p.E = (int32_t)E; p.plan = plan;
  p.ld = blocks_of(I) * BLOCK; p.strideB = H * p.ld;
  p.bs_n = p.kt; p.bs_k = 1; p.bs_e = blocks_of(H) * p.kt;
  p.vec = bf16_pieces(H, {y});
  p.O0 = (bf16_t*)y;
  return launch_product<PLAIN>(p, A, pk_timing::K_FP8_DOWN, (hipStream_t)stream, short_sums);
}

int pk_fp8_down(const uint8_t* h, const uint8_t* h_scales, const uint8_t* w2, const uint8_t* s2, const int32_t* plan, void* y, int64_t A,
                int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  return down(h, h_scales, w2, s2, plan, y, A, H, I, E, stream, false);
}

int pk_fp8_down_short(const uint8_t* h, const uint8_t* h_scales, const uint8_t* w2, const uint8_t* s2, const int32_t* plan, void* y, int64_t A,
                      int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  return down(h, h_scales, w2, s2, plan, y, A, H, I, E, stream, true);
}

static int dgrad_dh(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                    const int32_t* plan, void* d_g, void* d_u, void* h, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8, uint8_t* d_u_scales,
                    int64_t A, int64_t H, int64_t I, int64_t E, bool transposed, pk_stream_t stream, bool short_sums) {
  if (A == 0) return PK_OK;
  if (!all_set({d_y, d_y_scales, w2_t, s2, g, u, plan, d_g, d_u, h, d_g8, d_g_scales, d_u8, d_u_scales})) return PK_ERR_ARG;
  if (!all_aligned({d_y, w2_t, d_g8, d_u8, plan}) || !word_aligned({d_y_scales})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = p.A[1] = d_y; p.As[0] = p.As[1] = d_y_scales;
  p.B[0] = p.B[1] = w2_t; p.Bs[0] = p.Bs[1] = s2;
  p.kt = (int32_t)blocks_of(H); p.nseg = 1; p.N = (int32_t)I; p.E = (int32_t)E; p.plan = plan;
  p.ld = blocks_of(H) * BLOCK; p.strideB = I * p.ld;
  p.bs_n = 1; p.bs_k = (int32_t)blocks_of(I); p.bs_e = blocks_of(H) * blocks_of(I);
  p.vec = bf16_pieces(I, {g, u, d_g, d_u, h});
  if (transposed && !p.vec) return PK_ERR_ALIGN;
  p.O0 = (bf16_t*)d_g; p.O1 = (bf16_t*)d_u; p.O2 = (bf16_t*)h;
  p.Q[0] = d_g8; p.Qs[0] = d_g_scales; p.Q[1] = d_u8; p.Qs[1] = d_u_scales;
  p.G = (const bf16_t*)g; p.U = (const bf16_t*)u;
  return launch_product<BWD>(p, A, pk_timing::K_FP8_DGRAD_DH, (hipStream_t)stream, short_sums, transposed);
}

int pk_fp8_dgrad_dh(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                    const int32_t* plan, void* d_g, void* d_u, void* h, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8, uint8_t* d_u_scales,
                    int64_t A, int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  return dgrad_dh(d_y, d_y_scales, w2_t, s2, g, u, plan, d_g, d_u, h, d_g8, d_g_scales, d_u8, d_u_scales, A, H, I, E, false, stream, false);
}

int pk_fp8_dgrad_dh_short(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                          const int32_t* plan, void* d_g, void* d_u, void* h, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8, uint8_t* d_u_scales,
                          int64_t A, int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  return dgrad_dh(d_y, d_y_scales, w2_t, s2, g, u, plan, d_g, d_u, h, d_g8, d_g_scales, d_u8, d_u_scales, A, H, I, E, false, stream, true);
}

static int dgrad_dh_t(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                      const int32_t* plan, void* d_gT, void* d_uT, void* hT, int64_t ldt, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8,
                      uint8_t* d_u_scales, int64_t A, int64_t H, int64_t I, int64_t E, pk_stream_t stream, bool short_sums) {
  if (const int rc = check(A, H, I, E)) return rc;
  const int64_t need = pk_grouped_swiglu_transposed_ld(A, H, I, E, PK_BF16);
  if (need <= 0) return PK_ERR_SHAPE;
  if (A > 0 && (ldt < need || ldt % 64 != 0)) return PK_ERR_ARG;
  return dgrad_dh(d_y, d_y_scales, w2_t, s2, g, u, plan, d_gT, d_uT, hT, d_g8, d_g_scales, d_u8, d_u_scales, A, H, I, E, true, stream, short_sums);
}

int pk_fp8_dgrad_dh_t(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                      const int32_t* plan, void* d_gT, void* d_uT, void* hT, int64_t ldt, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8,
                      uint8_t* d_u_scales, int64_t A, int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  return dgrad_dh_t(d_y, d_y_scales, w2_t, s2, g, u, plan, d_gT, d_uT, hT, ldt, d_g8, d_g_scales, d_u8, d_u_scales, A, H, I, E, stream, false);
}

int pk_fp8_dgrad_dh_t_short(const uint8_t* d_y, const uint8_t* d_y_scales, const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u,
                            const int32_t* plan, void* d_gT, void* d_uT, void* hT, int64_t ldt, uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8,
                            uint8_t* d_u_scales, int64_t A, int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  return dgrad_dh_t(d_y, d_y_scales, w2_t, s2, g, u, plan, d_gT, d_uT, hT, ldt, d_g8, d_g_scales, d_u8, d_u_scales, A, H, I, E, stream, true);
}

static int dgrad_dx(const uint8_t* d_g8, const uint8_t* d_g_scales, const uint8_t* d_u8, const uint8_t* d_u_scales, const uint8_t* w1_t,
                    const uint8_t* s1, const uint8_t* w3_t, const uint8_t* s3, const int32_t* plan, void* d_x, int64_t A, int64_t H, int64_t I,
                    int64_t E, pk_stream_t stream, bool short_sums) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({d_g8, d_g_scales, d_u8, d_u_scales, w1_t, s1, w3_t, s3, plan, d_x})) return PK_ERR_ARG;
  if (!all_aligned({d_g8, d_u8, w1_t, w3_t, plan}) || !word_aligned({d_g_scales, d_u_scales})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = d_g8; p.As[0] = d_g_scales; p.A[1] = d_u8; p.As[1] = d_u_scales;
  p.B[0] = w1_t; p.Bs[0] = s1; p.B[1] = w3_t; p.Bs[1] = s3;
  p.kt = (int32_t)blocks_of(I); p.nseg = 2; p.N = (int32_t)H; p.E = (int32_t)E; p.plan = plan;
  p.ld = blocks_of(I) * BLOCK; p.strideB = H * p.ld;
  p.bs_n = 1; p.bs_k = (int32_t)blocks_of(H); p.bs_e = blocks_of(H) * blocks_of(I);
  p.vec = bf16_pieces(H, {d_x});
  p.O0 = (bf16_t*)d_x;
  return launch_product<PLAIN>(p, A, pk_timing::K_FP8_DGRAD_DX, (hipStream_t)stream, short_sums);
}

int pk_fp8_dgrad_dx(const uint8_t* d_g8, const uint8_t* d_g_scales, const uint8_t* d_u8, const uint8_t* d_u_scales, const uint8_t* w1_t,
                    const uint8_t* s1, const uint8_t* w3_t, const uint8_t* s3, const int32_t* plan, void* d_x, int64_t A, int64_t H, int64_t I,
                    int64_t E, pk_stream_t stream) {
  return dgrad_dx(d_g8, d_g_scales, d_u8, d_u_scales, w1_t, s1, w3_t, s3, plan, d_x, A, H, I, E, stream, false);
}

int pk_fp8_dgrad_dx_short(const uint8_t* d_g8, const uint8_t* d_g_scales, const uint8_t* d_u8, const uint8_t* d_u_scales, const uint8_t* w1_t,
                          const uint8_t* s1, const uint8_t* w3_t, const uint8_t* s3, const int32_t* plan, void* d_x, int64_t A, int64_t H, int64_t I,
                          int64_t E, pk_stream_t stream) {
  return dgrad_dx(d_g8, d_g_scales, d_u8, d_u_scales, w1_t, s1, w3_t, s3, plan, d_x, A, H, I, E, stream, true);
}

int pk_fp8_few_rows_pays(int64_t A, int64_t H, int64_t I, int64_t E) {
  if (check(A, H, I, E) != PK_OK || A == 0) return 0;
  return pk_rules::fp8_few_rows(A, E);
}

int pk_fp8_experts_few_rows(const void* x, const void* counts, int counts_is_i64, const uint8_t* w1, const uint8_t* s1, const uint8_t* w2,
                            const uint8_t* s2, const uint8_t* w3, const uint8_t* s3, void* g, void* u, float* h, void* y, int64_t A, int64_t H,
                            int64_t I, int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({x, counts, w1, s1, w2, s2, w3, s3, h, y}) || !g != !u) return PK_ERR_ARG;
  if (!all_aligned({w1, w2, w3})) return PK_ERR_ALIGN;
  Few p = {};
  p.counts = counts; p.is_i64 = counts_is_i64; p.E = (int32_t)E; p.H = (int32_t)H; p.I = (int32_t)I; p.A = A;
  p.x = (const bf16_t*)x; p.q1 = w1; p.s1 = s1; p.q2 = w2; p.s2 = s2; p.q3 = w3; p.s3 = s3;
  p.g = (bf16_t*)g; p.u = (bf16_t*)u; p.h = h; p.y = (bf16_t*)y;
  p.whole = H % 8 == 0;
  const int64_t tiles = pk_rules::fp8_tiles(A, E, FEW_ROWS);
  const bool stream_up = pk_rules::fp8_stream_up(A, E, I);
  const int64_t up = stream_up ? blocks_of(I) : pk_ceil_div(I, 16), per = pk_rules::fp8_down_tiles(A, E, H), down = pk_ceil_div(H, 64 * per);
  if (tiles * up > 0x7fffff00ll || tiles * down > 0x7fffff00ll) return PK_ERR_SHAPE;
  static bool ready[PK_MAX_DEVICES] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= PK_MAX_DEVICES) return PK_ERR_UNSUPPORTED;
  if (!ready[dev]) {
    for (const void* k : {reinterpret_cast<const void*>(down_few_kernel), reinterpret_cast<const void*>(gate_up_stream_kernel)}) {
      const hipError_t err = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, few_lds(PK_FP8_MAX_HIDDEN));
      if (err != hipSuccess) return (int)err;
    }
    ready[dev] = true;
  }
  hipStream_t s = (hipStream_t)stream;
  p.n_cols = (int32_t)up; p.by_cols = pk_units::make_fastdiv(up);
  if (stream_up)
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_GATE_UP, s, gate_up_stream_kernel, dim3((unsigned)(tiles * up)), dim3(512), few_lds(H), s, p);
  else
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_GATE_UP, s, gate_up_few_kernel, dim3((unsigned)(tiles * up)), dim3(512), 0, s, p);
  PK_RETURN_IF_LAUNCH_FAILED();
  p.n_cols = (int32_t)down; p.by_cols = pk_units::make_fastdiv(down);
  const int units = (int)(tiles * down), zeros = (int)(A < 32 ? A : 32);
  PK_LAUNCH_NOCHECK(pk_timing::K_FP8_DOWN, s, down_few_kernel, dim3((unsigned)(units + zeros)), dim3(256), few_lds(I), s, p, units, (int)per);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

}  // extern "C"
