// The experts' products in 8-bit floating point: e4m3 values with a power of two for each block of 128 (fp8_blocks.h).
//   rows:     [R][K'] codes, K' = K rounded up to 128 (the rest zeros), and [R][K'/128] scale bytes
//   weights:  [E][N][K'] codes and [E][N/128][K'/128] bytes, blocks of 128 x 128; the transposed codes [E][K][N'] share the bytes
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies the codes at twice the rate of bf16, applies both scale bytes to the products and
// adds in fp32.
#include "fp8_blocks.h"
#include "launch_rules.h"
#include "unit_index.h"

namespace {

constexpr int BLOCK = PK_FP8_BLOCK;
constexpr int THREADS = 256;
using pk_units::FastDiv;

inline int64_t blocks_of(int64_t n) { return pk_ceil_div(n, BLOCK); }

template <typename T>
__device__ __forceinline__ void load8(const T* p, int have, bool vec, float (&f)[8]) {
  if (vec && have >= 8) {
    if constexpr (sizeof(T) == 2) {
      const bf16x8_t v = *reinterpret_cast<const bf16x8_t*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
    } else {
      const floatx4_t a = *reinterpret_cast<const floatx4_t*>(p), b = *reinterpret_cast<const floatx4_t*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < have ? pk_to_float<T>(p[i]) : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------ rows
// 16 lanes to a block, one pass: 2 (bf16) or 4 bytes read and 1 written per value, bound by the memory.
template <typename T>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ row_map, FastDiv map_div,
                                                                uint8_t* __restrict__ q, uint8_t* __restrict__ s, int64_t units, int K, int kb,
                                                                FastDiv by_kb, bool vec) {
  const int64_t unit = (int64_t)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4);
  if (unit >= units) return;                 // whole groups of 16 lanes
  const int lane = threadIdx.x & 15;
  const int r = pk_units::fastdiv((int)unit, by_kb), b = (int)unit - r * kb;
  const int64_t src = row_map ? pk_units::fastdiv(row_map[r], map_div) : r;
  const int k = b * BLOCK + lane * 8;
  float f[8];
  load8<T>(x + src * K + k, K - k, vec, f);
  uint32_t codes[2], byte;
  pk_fp8::quantize8(f, codes, byte);
  *reinterpret_cast<u32x2_t*>(q + unit * BLOCK + lane * 8) = u32x2_t{codes[0], codes[1]};
  if (lane == 0) s[unit] = (uint8_t)byte;
}

// ------------------------------------------------------------------------------------------------ weights
// A workgroup has one block of 128 x 128: 16 lanes to a row of it, the codes once row-major and once, through the LDS, transposed.
template <typename T>
__global__ __launch_bounds__(THREADS) void quantize_weights_kernel(const T* __restrict__ w, uint8_t* __restrict__ q, uint8_t* __restrict__ t,
                                                                   uint8_t* __restrict__ s, int N, int K, bool vec) {
  constexpr int LD = BLOCK + 4;              // of the LDS rows: columns of bytes spread over the banks
  __shared__ uint32_t amax_of[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[BLOCK * LD];
  const int kb = gridDim.x, nb = gridDim.y;
  const int64_t e = blockIdx.z;
  const int n0 = blockIdx.y * BLOCK, k0 = blockIdx.x * BLOCK, Kp = kb * BLOCK, Np = nb * BLOCK;
  const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, k = k0 + lane * 8;
  const T* const src = w + e * N * K;
  float f[8][8];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int n = n0 + row + 16 * i;
    load8<T>(src + (int64_t)(n < N ? n : n0) * K + k, n < N ? K - k : 0, vec, f[i]);
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
  if (threadIdx.x == 0) s[(e * nb + blockIdx.y) * kb + blockIdx.x] = (uint8_t)byte;
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

// ------------------------------------------------------------------------------------------------ products
// C[rows_e, N] = sum_seg A_seg[rows_e, K] . B_seg[e][N, K]^T, one workgroup to a tile of BM rows and 256 columns (gate and up: 128
// of each).
enum Epilogue { PLAIN = 0, GATE_UP = 1, BWD = 2, BWD_SCALED = 3 };

typedef int intx8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

struct Product {
  const uint8_t* A[2];      // codes of the rows, by segment [., lda]
  const uint8_t* As[2];     // and their scales [., kt]
  const int32_t* row_map;   // optional gather: A row = row_map[sorted row] / map_div
  FastDiv map_div;
  const uint8_t* B[2];      // weights of a segment (GATE_UP: gate, up), rows of ld codes
  const uint8_t* Bs[2];     // scale of block (n, k) of expert e: Bs[e * bs_e + n * bs_n + k * bs_k]
  int64_t ld, strideB, bs_e;
  int32_t bs_n, bs_k;
  const int32_t* starts;
  int32_t E, kt, nseg, N, n_tiles;
  bool vec;                 // rows of the bf16 tensors are whole 16-byte pieces
  bf16_t* O0;               // C;  GATE_UP: g (optional);  BWD: d_g
  bf16_t* O1;               //     GATE_UP: u (optional);  BWD: d_u
  bf16_t* O2;               //                             BWD: h (BWD_SCALED: score * h)
  uint8_t* Q[2];            //     GATE_UP: h;             BWD: d_g, d_u   in blocks
  uint8_t* Qs[2];
  const bf16_t* G;          // BWD: g and u of the forward
  const bf16_t* U;
  const float* scores;      // BWD_SCALED: of every routed slot
  float* ds_part;           //             [N / 128][total_rows]: the score gradient in parts
  int64_t total_rows;
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_ptr_t)p; }
// 16 bytes per lane straight into LDS, lane l's at lds_base + 16 l, from a wave-uniform base and an offset per lane.  The
// compiler does not see the transfer: dma_wait and a barrier stand before what reads it.
__device__ __forceinline__ void dma16(uint32_t voff, const void* sbase, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(voff), "s"(sbase) : "memory");
}
template <int N>
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

constexpr int KT_BYTES = 128;                // a k-tile is one block: 128 bytes of every row
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

// 32 of the 64 reduction bytes of step `half` of a k-tile, for row row0 + lane % 32.  Both operands are dealt alike, and a
// k-tile has one scale, so it does not matter which lane holds which of them.
__device__ __forceinline__ intx8_t fragment(const char* tile, int row0, int half, int lane) {
  const int r = row0 + (lane & 31), c = 4 * half + 2 * (lane >> 5);
  const char* const p = tile + r * KT_BYTES;
  const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(p + ((c ^ swz(r)) << 4));
  const u32x4_t hi = *reinterpret_cast<const u32x4_t*>(p + (((c + 1) ^ swz(r)) << 4));
  return intx8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// fp32 staging of a tile's rows in LDS, 16-byte units of a row XOR-ed with the row against bank conflicts
template <int X>
__device__ __forceinline__ void stage4(float* lds, int row, int col, const float* four) {
  *reinterpret_cast<floatx4_t*>(lds + row * X + (((col >> 2) ^ (row & (X / 4 - 1))) << 2)) = floatx4_t{four[0], four[1], four[2], four[3]};
}
template <int X>
__device__ __forceinline__ void staged8(const float* lds, int row, int col, float (&f)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const floatx4_t v = *reinterpret_cast<const floatx4_t*>(lds + row * X + ((((col >> 2) + h) ^ (row & (X / 4 - 1))) << 2));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 * h + i] = v[i];
  }
}
__device__ __forceinline__ void store8(bf16_t* p, int have, bool vec, const float (&f)[8]) {
  if (vec && have >= 8) {
    bf16x8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16_t)f[i];
    *reinterpret_cast<bf16x8_t*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) p[i] = (bf16_t)f[i];
  }
}
__device__ __forceinline__ float held(float v) { return (float)(bf16_t)v; }
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

constexpr int unit_chunk = 16;
__device__ __forceinline__ int unit_of_block(int b) {      // neighbouring units on one XCD
  const int x = b % pk_rules::NXCD, q = b / pk_rules::NXCD;
  return ((q / unit_chunk) * pk_rules::NXCD + x) * unit_chunk + (q % unit_chunk);
}

// WM x 2 waves of 64 x 128 outputs.
template <int WM, int NS, int EPI>
__global__ __launch_bounds__(128 * WM) void product_kernel(const Product p) {
  constexpr int NT = 128 * WM, BM = 64 * WM, BN = 256, TM = 2, TN = 4;
  constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT, L = LA + LB;
  constexpr int A_BYTES = BM * KT_BYTES, STAGE = A_BYTES + BN * KT_BYTES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
  const pk_units::UnitIndex ui = pk_units::build_unit_index<BM>(p.starts, p.E, p.n_tiles);
  const int unit = unit_of_block(blockIdx.x);
  if (unit >= ui.total) return;
  int e, mt, nt;
  pk_units::locate_unit<BM>(ui, pk_units::as_const(p.starts), p.E, p.n_tiles, unit, e, mt, nt);
  const int row0 = p.starts[e] + mt * BM, rows = min(BM, p.starts[e + 1] - row0);
  const int nkt = p.kt * p.nseg;
  const int n0 = nt * (EPI == GATE_UP ? BLOCK : BN);

  // scales of the tile's rows and columns, behind the ring: a row of them is nkt bytes
  char* const sa = smem + NS * STAGE;
  const int sld = (nkt + 7) / 8 * 8 + 4;
  char* const sb = sa + BM * sld;
  for (int i = tid; i < BM * nkt; i += NT) {
    const int r = i / nkt, k = i - r * nkt, seg = k >= p.kt;
    int64_t src = row0 + (r < rows ? r : 0);
    if (p.row_map) src = pk_units::fastdiv(p.row_map[src], p.map_div);
    sa[r * sld + k] = (char)p.As[seg][src * p.kt + (seg ? k - p.kt : k)];
  }
  const int n_blocks = (p.N + BLOCK - 1) / BLOCK;
  for (int i = tid; i < 2 * nkt; i += NT) {
    const int b = i >= nkt, k = b ? i - nkt : i, seg = k >= p.kt;
    const int nb = EPI == GATE_UP ? nt : min(2 * nt + b, n_blocks - 1);
    sb[i] = (char)p.Bs[EPI == GATE_UP ? b : seg][e * p.bs_e + (int64_t)nb * p.bs_n + (int64_t)(seg ? k - p.kt : k) * p.bs_k];
  }

  // Byte offsets of the 16-byte pieces that the thread brings; rows past the expert's end and columns past N read the tile's first
  // ones instead, and what comes of them is stored nowhere.
  uint32_t a_off[LA], b_off[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int s = tid + i * NT, r = s >> 3, c = (s & 7) ^ swz(r);
    int64_t src = row0 + (r < rows ? r : 0);
    if (p.row_map) src = pk_units::fastdiv(p.row_map[src], p.map_div);
    a_off[i] = (uint32_t)(src * p.ld + c * 16);
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int s = tid + i * NT, r = s >> 3, c = (s & 7) ^ swz(r);
    const int n = n0 + (EPI == GATE_UP ? r & (BLOCK - 1) : r);
    b_off[i] = (uint32_t)((int64_t)(n < p.N ? n : n0) * p.ld + c * 16);
  }
  const uint32_t ring = lds_addr(smem) + wave * 1024;
  const auto fetch = [&](int kt, int stage) {
    const int seg = kt >= p.kt, k = (seg ? kt - p.kt : kt) * KT_BYTES;
    const uint8_t* const a = uniform(p.A[seg] + k);
    const uint32_t at = ring + stage * STAGE;
#pragma unroll
    for (int i = 0; i < LA; ++i) dma16(a_off[i], a, at + i * NT * 16);
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      // GATE_UP: the first half of the tile's rows are gate weights, the second half up weights
      const int which = EPI == GATE_UP ? (i >= LB / 2) : seg;
      dma16(b_off[i], uniform(p.B[which] + e * p.strideB + k), at + A_BYTES + i * NT * 16);
    }
  };

  floatx16_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  __syncthreads();                           // the scales are there; every ordinary load has been waited for
#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < nkt) fetch(s, s);
  int stage = 0;
  for (int kt = 0; kt < nkt; ++kt) {
    // all but the youngest NS - 2 k-tiles have landed, everywhere; the stage that the next one goes to has been read
    if (NS > 2 && kt + 1 < nkt) dma_wait<(NS - 2) * L>();
    else dma_wait<0>();
    block_barrier();
    const int next = stage == 0 ? NS - 1 : stage - 1;
    if (kt + NS - 1 < nkt) fetch(kt + NS - 1, next);
    const char* const at = smem + stage * STAGE;
    const int scale_b = (unsigned char)sb[wn * nkt + kt];
    int scale_a[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) scale_a[i] = (unsigned char)sa[(wm * 64 + i * 32 + (lane & 31)) * sld + kt];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      intx8_t a[TM], b[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = fragment(at, wm * 64 + i * 32, half, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = fragment(at + A_BYTES, wn * 128 + j * 32, half, lane);
      // operands swapped: a lane then holds 4 neighbouring columns of one row,
      //   acc[v] = C[row = lane % 32][col = 8 * (v / 4) + 4 * (lane / 32) + v % 4]
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[i][j], 0, 0, 0, scale_b, 0, scale_a[i]);
    }
    stage = stage == NS - 1 ? 0 : stage + 1;
  }

  // 32 rows of every wave at a time through the LDS; then 16 lanes have 128 columns, a block, of a row
  constexpr int CHUNK = 32 * WM;
  static_assert(CHUNK * BN * 4 <= NS * STAGE, "the staged rows reuse the ring");
  float* const lds = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    __syncthreads();                         // the LDS has been read for the last time
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        stage4<BN>(lds, 32 * wm + (lane & 31), wn * 128 + 32 * j + 8 * q + 4 * (lane >> 5), reinterpret_cast<const float*>(&acc[i][j]) + 4 * q);
    __syncthreads();
    constexpr int PIECES = (EPI == GATE_UP ? BLOCK : BN) / 8;
    for (int s = tid; s < CHUNK * PIECES; s += NT) {
      const int lr = s / PIECES, c = (s % PIECES) * 8, n = n0 + c;
      const int r = (lr >> 5) * 64 + 32 * i + (lr & 31);
      const bool live = r < rows;            // the same for the 16 lanes of a block
      const int have = live ? p.N - n : 0;
      const int64_t o = (int64_t)(row0 + r) * p.N + n;
      const int64_t unit_out = (int64_t)(row0 + r) * n_blocks + n / BLOCK;
      float a[8];
      staged8<BN>(lds, lr, c, a);
      if constexpr (EPI == PLAIN) {
        store8(p.O0 + o, have, p.vec, a);
      } else if constexpr (EPI == GATE_UP) {
        float u[8], h[8];
        staged8<BN>(lds, lr, c + BLOCK, u);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          a[t] = held(a[t]);                 // g and u are bf16 tensors, written or not
          u[t] = held(u[t]);
          h[t] = t < have ? a[t] * sigmoid(a[t]) * u[t] : 0.f;
        }
        uint32_t codes[2], byte;
        pk_fp8::quantize8(h, codes, byte);
        if (live) {
          if (p.O0) store8(p.O0 + o, have, p.vec, a);
          if (p.O1) store8(p.O1 + o, have, p.vec, u);
          *reinterpret_cast<u32x2_t*>(p.Q[0] + unit_out * BLOCK + (n & (BLOCK - 1))) = u32x2_t{codes[0], codes[1]};
          if ((tid & 15) == 0) p.Qs[0][unit_out] = (uint8_t)byte;
        }
      } else {
        float g[8], u[8], h[8], ds = 0.f;
        load8<bf16_t>(p.G + o, have, p.vec, g);
        load8<bf16_t>(p.U + o, have, p.vec, u);
        const float sc = EPI == BWD_SCALED && live ? p.scores[p.row_map[row0 + r]] : 1.f;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float sg = sigmoid(g[t]), silu = g[t] * sg, hv = silu * u[t];
          if (EPI == BWD_SCALED) ds += t < have ? a[t] * hv : 0.f;
          const float d = sc * a[t];
          h[t] = sc * hv;
          const float dg = d * u[t] * (sg * (1.f + g[t] * (1.f - sg))), du = d * silu;
          g[t] = t < have ? held(dg) : 0.f;  // bf16 tensors, whose blocks are of what they hold
          u[t] = t < have ? held(du) : 0.f;
        }
        uint32_t cg[2], cu[2], bg, bu;
        pk_fp8::quantize8(g, cg, bg);
        pk_fp8::quantize8(u, cu, bu);
        if (EPI == BWD_SCALED) ds = pk_fp8::row_sum(ds);
        if (live) {
          store8(p.O0 + o, have, p.vec, g);
          store8(p.O1 + o, have, p.vec, u);
          store8(p.O2 + o, have, p.vec, h);
          if (n / BLOCK < n_blocks) {
            const int64_t at = unit_out * BLOCK + (n & (BLOCK - 1));
            *reinterpret_cast<u32x2_t*>(p.Q[0] + at) = u32x2_t{cg[0], cg[1]};
            *reinterpret_cast<u32x2_t*>(p.Q[1] + at) = u32x2_t{cu[0], cu[1]};
            if ((tid & 15) == 0) {
              p.Qs[0][unit_out] = (uint8_t)bg;
              p.Qs[1][unit_out] = (uint8_t)bu;
              if (EPI == BWD_SCALED) p.ds_part[(int64_t)(n / BLOCK) * p.total_rows + row0 + r] = ds;
            }
          }
        }
      }
    }
  }
}

template <int WM, int NS, int EPI>
int launch_tiles(Product p, int64_t A, int kernel_id, hipStream_t s) {
  constexpr int BM = 64 * WM, STAGE = (BM + 256) * KT_BYTES;
  p.n_tiles = (int32_t)pk_ceil_div(p.N, EPI == GATE_UP ? BLOCK : 256);
  const int64_t units = (A / BM + (A < p.E ? A : p.E)) * p.n_tiles;
  if (units > 0x7fffff00ll) return PK_ERR_SHAPE;
  if (units == 0) return PK_OK;
  const int nkt = p.kt * p.nseg, sld = (nkt + 7) / 8 * 8 + 4;
  const int lds = NS * STAGE + BM * sld + 2 * nkt;
  static bool ready[PK_MAX_DEVICES] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= PK_MAX_DEVICES) return PK_ERR_UNSUPPORTED;
  if (!ready[dev]) {
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void*>(product_kernel<WM, NS, EPI>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               160 * 1024);
    if (err != hipSuccess) return (int)err;
    ready[dev] = true;
  }
  const int64_t per = unit_chunk * pk_rules::NXCD;
  PK_LAUNCH_NOCHECK(kernel_id, s, (product_kernel<WM, NS, EPI>), dim3((unsigned)(pk_ceil_div(units, per) * per)), dim3(128 * WM), lds, s, p);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

template <int EPI>
int launch_product(const Product& p, int64_t A, int kernel_id, hipStream_t s) {
  return launch_tiles<4, 2, EPI>(p, A, kernel_id, s);
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
bool all_set(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!q) return false;
  return true;
}
bool bf16_pieces(int64_t width, std::initializer_list<const void*> ps) { return width % 8 == 0 && all_aligned(ps); }

}  // namespace

extern "C" {

int pk_fp8_quantize_rows(const void* x, int dtype, const int32_t* row_map, int64_t row_map_div, uint8_t* q, uint8_t* scales, int64_t rows,
                         int64_t K, pk_stream_t stream) {
  if (rows < 0 || K <= 0 || row_map_div < 1 || !pk_dtype_ok(dtype)) return PK_ERR_ARG;
  if (rows == 0) return PK_OK;
  if (!all_set({x, q, scales})) return PK_ERR_ARG;
  if (!pk_aligned16(q)) return PK_ERR_ALIGN;
  const int64_t kb = blocks_of(K), units = rows * kb;
  if (K > 0x7fffff00ll || rows > 0x7fffffffll || units > 0x7fffffffll || row_map_div > 0x7fffffffll) return PK_ERR_SHAPE;
  const bool vec = K * (int64_t)pk_dtype_size(dtype) % 16 == 0 && pk_aligned16(x);
  const FastDiv div = pk_units::make_fastdiv(row_map_div), by_kb = pk_units::make_fastdiv(kb);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)pk_ceil_div(units, THREADS / 16)), block(THREADS);
  if (dtype == PK_BF16)
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_rows_kernel<bf16_t>), grid, block, 0, s, (const bf16_t*)x, row_map, div, q, scales,
                      units, (int)K, (int)kb, by_kb, vec);
  else
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_rows_kernel<float>), grid, block, 0, s, (const float*)x, row_map, div, q, scales,
                      units, (int)K, (int)kb, by_kb, vec);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int pk_fp8_quantize_weights(const void* w, int dtype, uint8_t* q, uint8_t* q_t, uint8_t* scales, int64_t E, int64_t N, int64_t K,
                            pk_stream_t stream) {
  if (E < 0 || N <= 0 || K <= 0 || !pk_dtype_ok(dtype)) return PK_ERR_ARG;
  if (E == 0) return PK_OK;
  if (!all_set({w, q, scales})) return PK_ERR_ARG;
  if (!all_aligned({q, q_t})) return PK_ERR_ALIGN;
  const int64_t nb = blocks_of(N), kb = blocks_of(K);
  if (E > 65535 || nb > 65535 || kb > 0x7fffffll) return PK_ERR_SHAPE;
  const bool vec = K * (int64_t)pk_dtype_size(dtype) % 16 == 0 && pk_aligned16(w);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)kb, (unsigned)nb, (unsigned)E), block(THREADS);
  if (dtype == PK_BF16)
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_weights_kernel<bf16_t>), grid, block, 0, s, (const bf16_t*)w, q, q_t, scales, (int)N,
                      (int)K, vec);
  else
    PK_LAUNCH_NOCHECK(pk_timing::K_FP8_QUANTIZE, s, (quantize_weights_kernel<float>), grid, block, 0, s, (const float*)w, q, q_t, scales, (int)N,
                      (int)K, vec);
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int pk_fp8_gate_up(const uint8_t* x, const uint8_t* x_scales, const int32_t* row_map, int64_t row_map_div, const uint8_t* w1, const uint8_t* s1,
                   const uint8_t* w3, const uint8_t* s3, const int32_t* starts, void* g, void* u, uint8_t* h, uint8_t* h_scales, int64_t A,
                   int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (row_map_div < 1 || row_map_div > 0x7fffffffll) return PK_ERR_ARG;
  if (A == 0) return PK_OK;
  if (!all_set({x, x_scales, w1, s1, w3, s3, starts, h, h_scales}) || !g != !u) return PK_ERR_ARG;
  if (!all_aligned({x, w1, w3, h})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = x; p.As[0] = x_scales; p.row_map = row_map; p.map_div = pk_units::make_fastdiv(row_map_div);
  p.A[1] = x; p.As[1] = x_scales;
  p.B[0] = w1; p.B[1] = w3; p.Bs[0] = s1; p.Bs[1] = s3;
  p.kt = (int32_t)blocks_of(H); p.nseg = 1; p.N = (int32_t)I; p.E = (int32_t)E; p.starts = starts;
  p.ld = blocks_of(H) * BLOCK; p.strideB = I * p.ld;
  p.bs_n = p.kt; p.bs_k = 1; p.bs_e = blocks_of(I) * p.kt;
  p.vec = bf16_pieces(I, {g, u});
  p.O0 = (bf16_t*)g; p.O1 = (bf16_t*)u; p.Q[0] = h; p.Qs[0] = h_scales;
  return launch_product<GATE_UP>(p, A, pk_timing::K_FP8_GATE_UP, (hipStream_t)stream);
}

int pk_fp8_down(const uint8_t* h, const uint8_t* h_scales, const uint8_t* w2, const uint8_t* s2, const int32_t* starts, void* y, int64_t A,
                int64_t H, int64_t I, int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({h, h_scales, w2, s2, starts, y})) return PK_ERR_ARG;
  if (!all_aligned({h, w2})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = p.A[1] = h; p.As[0] = p.As[1] = h_scales;
  p.B[0] = p.B[1] = w2; p.Bs[0] = p.Bs[1] = s2;
  p.kt = (int32_t)blocks_of(I); p.nseg = 1; p.N = (int32_t)H; p.E = (int32_t)E; p.starts = starts;
  p.ld = blocks_of(I) * BLOCK; p.strideB = H * p.ld;
  p.bs_n = p.kt; p.bs_k = 1; p.bs_e = blocks_of(H) * p.kt;
  p.vec = bf16_pieces(H, {y});
  p.O0 = (bf16_t*)y;
  return launch_product<PLAIN>(p, A, pk_timing::K_FP8_DOWN, (hipStream_t)stream);
}

int pk_fp8_dgrad_dh(const uint8_t* d_y, const uint8_t* d_y_scales, const int32_t* row_map, int64_t row_map_div, const float* scores,
                    const uint8_t* w2_t, const uint8_t* s2, const void* g, const void* u, const int32_t* starts, void* d_g, void* d_u, void* h,
                    uint8_t* d_g8, uint8_t* d_g_scales, uint8_t* d_u8, uint8_t* d_u_scales, float* ds_part, int64_t A, int64_t H, int64_t I,
                    int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (row_map_div < 1 || row_map_div > 0x7fffffffll) return PK_ERR_ARG;
  if (A == 0) return PK_OK;
  if (!all_set({d_y, d_y_scales, w2_t, s2, g, u, starts, d_g, d_u, h, d_g8, d_g_scales, d_u8, d_u_scales})) return PK_ERR_ARG;
  if (!scores != !ds_part || (scores && !row_map)) return PK_ERR_ARG;
  if (!all_aligned({d_y, w2_t, d_g8, d_u8})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = p.A[1] = d_y; p.As[0] = p.As[1] = d_y_scales; p.row_map = row_map; p.map_div = pk_units::make_fastdiv(row_map_div);
  p.B[0] = p.B[1] = w2_t; p.Bs[0] = p.Bs[1] = s2;
  p.kt = (int32_t)blocks_of(H); p.nseg = 1; p.N = (int32_t)I; p.E = (int32_t)E; p.starts = starts;
  p.ld = blocks_of(H) * BLOCK; p.strideB = I * p.ld;
  p.bs_n = 1; p.bs_k = (int32_t)blocks_of(I); p.bs_e = blocks_of(H) * blocks_of(I);
  p.vec = bf16_pieces(I, {g, u, d_g, d_u, h});
  p.O0 = (bf16_t*)d_g; p.O1 = (bf16_t*)d_u; p.O2 = (bf16_t*)h;
  p.Q[0] = d_g8; p.Qs[0] = d_g_scales; p.Q[1] = d_u8; p.Qs[1] = d_u_scales;
  p.G = (const bf16_t*)g; p.U = (const bf16_t*)u;
  p.scores = scores; p.ds_part = ds_part; p.total_rows = A;
  return scores ? launch_product<BWD_SCALED>(p, A, pk_timing::K_FP8_DGRAD_DH, (hipStream_t)stream)
                : launch_product<BWD>(p, A, pk_timing::K_FP8_DGRAD_DH, (hipStream_t)stream);
}

int pk_fp8_dgrad_dx(const uint8_t* d_g8, const uint8_t* d_g_scales, const uint8_t* d_u8, const uint8_t* d_u_scales, const uint8_t* w1_t,
                    const uint8_t* s1, const uint8_t* w3_t, const uint8_t* s3, const int32_t* starts, void* d_x, int64_t A, int64_t H, int64_t I,
                    int64_t E, pk_stream_t stream) {
  if (const int rc = check(A, H, I, E)) return rc;
  if (A == 0) return PK_OK;
  if (!all_set({d_g8, d_g_scales, d_u8, d_u_scales, w1_t, s1, w3_t, s3, starts, d_x})) return PK_ERR_ARG;
  if (!all_aligned({d_g8, d_u8, w1_t, w3_t})) return PK_ERR_ALIGN;
  Product p = {};
  p.A[0] = d_g8; p.As[0] = d_g_scales; p.A[1] = d_u8; p.As[1] = d_u_scales;
  p.B[0] = w1_t; p.Bs[0] = s1; p.B[1] = w3_t; p.Bs[1] = s3;
  p.kt = (int32_t)blocks_of(I); p.nseg = 2; p.N = (int32_t)H; p.E = (int32_t)E; p.starts = starts;
  p.ld = blocks_of(I) * BLOCK; p.strideB = H * p.ld;
  p.bs_n = 1; p.bs_k = (int32_t)blocks_of(H); p.bs_e = blocks_of(H) * blocks_of(I);
  p.vec = bf16_pieces(H, {d_x});
  p.O0 = (bf16_t*)d_x;
  return launch_product<PLAIN>(p, A, pk_timing::K_FP8_DGRAD_DX, (hipStream_t)stream);
}

}  // extern "C"
