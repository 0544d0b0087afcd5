// The router's balance loss over packed sequences, with every sequence's tokens per expert, and the gradient of its logits
// (formulas in balance.h).
//
// Memory is what bounds long inputs, 4 bytes a logit forward and 8 backward, launches and their dependent loads short ones.  Forward: a
// workgroup sums the softmax of up to `chunk` tokens of one sequence, a second launch adds the chunks of every sequence up in a fixed
// order and 64 bits, and its last workgroup the sequences.  No chunk belongs to two sequences: that of a sequence which starts at
// token b has the units b / chunk + s and on, which cannot meet (as padded_start in the weight gradients), so that the host needs
// no look at the lengths.  Backward: one pass, the softmax formed again.  131,072 tokens of 128 experts in 512 sequences: 21 + 9 + 23 us (the
// logits once in 67 MB, twice in the backward), 256 of 8 experts 4.6 + 4.8 + 3.0.
#include "balance.h"
#include <algorithm>

namespace {

using namespace pk_balance;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kChunk = 64, kMostChunks = 512;       // tokens of a chunk: a multiple of kChunk that leaves about kMostChunks of them

// A token's logits lie on LPT lanes, EPL to a lane, 64 / LPT tokens to a wave: lane g of a token has the pieces of four neighbouring
// experts g, g + LPT, ..
template <int LPT>
__device__ __forceinline__ float group_sum(float v) {
#define PK_STEP(CTRL) v += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true))
  if (LPT > 1) PK_STEP(0xb1);          // quad_perm 1 0 3 2
  if (LPT > 2) PK_STEP(0x4e);          // quad_perm 2 3 0 1
  if (LPT > 4) PK_STEP(0x141);         // row_half_mirror: the other quad of 8 lanes
  if (LPT > 8) PK_STEP(0x140);         // row_mirror: the other 8 of a row of 16
#undef PK_STEP
  const auto add = [](auto r) { return __uint_as_float(r[0]) + __uint_as_float(r[1]); };
  if (LPT > 16) v = add(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  if (LPT > 32) v = add(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return v;
}
template <int LPT>
__device__ __forceinline__ float group_max(float v) {
#define PK_STEP(CTRL) v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true)))
  if (LPT > 1) PK_STEP(0xb1);
  if (LPT > 2) PK_STEP(0x4e);
  if (LPT > 4) PK_STEP(0x141);
  if (LPT > 8) PK_STEP(0x140);
#undef PK_STEP
  const auto most = [](auto r) { return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])); };
  if (LPT > 16) v = most(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  if (LPT > 32) v = most(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return v;
}
template <int LPT>
__device__ __forceinline__ int expert_of(int j, int g) { return ((j >> 2) * LPT + g) * 4 + (j & 3); }

// VEC: rows are whole 16-byte pieces on their boundaries
template <int LPT, int EPL, bool VEC>
__device__ __forceinline__ void load_row(const float* __restrict__ row, int E, int g, float absent, float (&x)[EPL]) {
  if (VEC && E == LPT * EPL) {
#pragma unroll
    for (int j = 0; j < EPL; j += 4) {
      const floatx4_t v = *reinterpret_cast<const floatx4_t*>(row + expert_of<LPT>(j, g));
#pragma unroll
      for (int k = 0; k < 4; ++k) x[j + k] = v[k];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < EPL; j += 4) {
    const int e = expert_of<LPT>(j, g);
    if (VEC) {
      const floatx4_t v = e < E ? *reinterpret_cast<const floatx4_t*>(row + e) : floatx4_t{absent, absent, absent, absent};
#pragma unroll
      for (int k = 0; k < 4; ++k) x[j + k] = v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[j + k] = e + k < E ? row[e + k] : absent;
    }
  }
}
// x becomes the softmax (0 where there is no expert: -inf there); returns log(sum exp).  2^t is the hardware's, 1 ulp.  Rounding
// t = (x - max) log2 e makes 2^t off by 2^-24 ln 2 |t| of itself, which is least for the largest probabilities; with this and
// rows of E = LPT * EPL read without a test, 131,072 tokens' sums take 21 us against 25.
template <int LPT, int EPL>
__device__ __forceinline__ float softmax(float (&x)[EPL]) {
  float mx = x[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) mx = fmaxf(mx, x[j]);
  mx = group_max<LPT>(mx);
  float total = 0.f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    x[j] = __builtin_amdgcn_exp2f((x[j] - mx) * 1.44269504088896340736f);
    total += x[j];
  }
  total = group_sum<LPT>(total);
  const float inv = 1.f / total;
#pragma unroll
  for (int j = 0; j < EPL; ++j) x[j] *= inv;
  return mx + logf(total);
}

struct Forward {
  const float* logits;
  const int32_t* top_idx;
  const int32_t* sequences;
  int32_t T, E, K, S, chunk, units;
  float balance_coeff, z_coeff;
  float* part_p;          // [units][E] sums of the softmax
  int32_t* part_c;        // [units][E] counts
  float* part_z;          // [units]
  double* seq;            // [workgroups of the second launch][4], see there
  uint32_t* done;         // workgroups of the second launch that have finished
  float* loss;
  int32_t* counts;
  float* table;
};

// How many of n things hold, over the workgroup
template <typename F>
__device__ __forceinline__ int count_of(int n, int* box, F&& holds) {
  int c = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) c += holds(i) ? 1 : 0;
  for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = c;
  __syncthreads();
  c = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) c += box[w];
  return c;
}

// As wave_leading, for a workgroup of kThreads: up to 1,024 things take four loads of a thread at once.
template <typename F>
__device__ __forceinline__ int block_leading(int n, int* box, F&& holds) {
  return leading<kThreads>(n, 4 * kThreads, [&](int m, auto&& f) { return __builtin_amdgcn_readfirstlane(count_of(m, box, f)); }, holds);
}

template <int LPT, int EPL, bool VEC>
__global__ __launch_bounds__(kThreads) void balance_partial_kernel(const Forward p) {
  constexpr int EM = LPT * EPL, TPW = 64 / LPT;
  __shared__ float sum_p[kWaves][EM];
  __shared__ float sum_z[kWaves];
  __shared__ int hist[EM];
  __shared__ int box[kWaves];
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;
  const int unit = blockIdx.x;
  const int s = p.sequences ? block_leading(p.S, box, [&](int i) { return begin_of(p.sequences, i, p.T) / p.chunk + i <= unit; }) - 1 : 0;
  if (s < 0) return;
  const int b = begin_of(p.sequences, s, p.T), e = end_of(p.sequences, s, p.T);
  const int64_t from = b + (int64_t)(unit - (b / p.chunk + s)) * p.chunk;
  if (from < b || from >= e) return;                    // (the former only where the offsets do not ascend)
  const int first = (int)from, n = min(p.chunk, e - first);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane % LPT, slot = lane / LPT;
  // two steps' logits are on their way while those of the two before are worked on
  constexpr int AT_ONCE = 2, STEP = kWaves * TPW;
  const float* const logits = p.logits + (int64_t)first * p.E;
  float next[AT_ONCE][EPL];
  const auto request = [&](int i) {
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) {
      const int t = i + q * STEP + slot;
      load_row<LPT, EPL, VEC>(logits + (int64_t)min(t, n - 1) * p.E, p.E, g, -INFINITY, next[q]);
    }
  };
  request(wave * TPW);
  for (int i = tid; i < EM; i += kThreads) hist[i] = 0;
  __syncthreads();
  constexpr int IDS = 8;                                // of a thread on their way at once
  const int32_t* const ids = p.top_idx + (int64_t)first * p.K;
  for (int i = tid; i < n * p.K; i += IDS * kThreads) {
    uint32_t id[IDS];
#pragma unroll
    for (int q = 0; q < IDS; ++q) id[q] = i + q * kThreads < n * p.K ? (uint32_t)ids[i + q * kThreads] : 0xffffffffu;
#pragma unroll
    for (int q = 0; q < IDS; ++q)
      if (id[q] < (uint32_t)p.E) atomicAdd(&hist[id[q]], 1);
  }
  float sum[EPL] = {}, z = 0.f;
  for (int i = wave * TPW; i < n; i += AT_ONCE * STEP) {
    float x[AT_ONCE][EPL], lse[AT_ONCE];
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q)
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[q][j] = next[q][j];
    if (i + AT_ONCE * STEP < n) request(i + AT_ONCE * STEP);
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) lse[q] = softmax<LPT, EPL>(x[q]);
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q)
      if (i + q * STEP + slot < n) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) sum[j] += x[q][j];
        z += lse[q] * lse[q];
      }
  }
#pragma unroll
  for (int off = LPT; off < 64; off <<= 1) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) sum[j] += __shfl_xor(sum[j], off, 64);
    z += __shfl_xor(z, off, 64);
  }
  if (lane < LPT) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) sum_p[wave][expert_of<LPT>(j, g)] = sum[j];
  }
  if (lane == 0) sum_z[wave] = z;
  __syncthreads();
  for (int i = tid; i < p.E; i += kThreads) {
    float v = 0.f;
    for (int w = 0; w < kWaves; ++w) v += sum_p[w][i];
    p.part_p[(int64_t)unit * p.E + i] = v;
    p.part_c[(int64_t)unit * p.E + i] = hist[i];
  }
  if (tid == 0) p.part_z[unit] = sum_z[0] + sum_z[1] + sum_z[2] + sum_z[3];
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// v[q] becomes its sum over the workgroup, in the lanes of wave 0
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double (*box)[N]) {
#pragma unroll
  for (int q = 0; q < N; ++q) v[q] = wave_sum(v[q]);
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int q = 0; q < N; ++q) box[threadIdx.x >> 6][q] = v[q];
  }
  __syncthreads();
  if (threadIdx.x < 64) {
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = wave_sum(threadIdx.x < blockDim.x / 64 ? box[threadIdx.x][q] : 0.0);
  }
}

// Chunks added up in their order: a sequence's row of the table and of the counts, and what the last workgroup adds up to the loss.
// A workgroup's slices of `width` threads, one for each expert, share the chunks of a sequence, or (TOGETHER) take a sequence each.
// What a workgroup costs beside its loads (a barrier, a fence, one addition to `done`) is then paid once for all its sequences:
// 512 sequences, 1,025 chunks and 128 experts take 9.1 us with TOGETHER and 15.2 without, 61 sequences, 318 chunks and 60 experts
// 15.3 with and 6.8 without.  The host does not know the lengths and decides by the mean.
constexpr int kSumThreads = 1024;                       // at most, and with TOGETHER
__host__ __device__ inline int sum_width(int E) { return (E + 63) / 64 * 64; }
template <bool TOGETHER>
__global__ __launch_bounds__(kSumThreads) void balance_sum_kernel(const Forward p) {
  __shared__ double sum_p[TOGETHER ? 1 : kSumThreads];
  __shared__ int sum_c[TOGETHER ? 1 : kSumThreads];
  __shared__ double box[kSumThreads / 64][4];
  const int tid = threadIdx.x, width = sum_width(p.E), slices = (int)blockDim.x / width, slice = tid / width, ex = tid % width;
  const int s = TOGETHER ? blockIdx.x * slices + slice : blockIdx.x;
  const int from = TOGETHER ? 0 : slice, step = TOGETHER ? 1 : slices;
  double all[4] = {0.0, 0.0, 0.0, 0.0};      // sum_e f_e P_e, sum of lse^2, tokens, sequences that have some
  const bool mine = slice < slices && s < p.S;
  const int b = mine ? begin_of(p.sequences, s, p.T) : 0, L = mine ? end_of(p.sequences, s, p.T) - b : 0;
  const int unit0 = b / p.chunk + s, chunks = mine ? min((L + p.chunk - 1) / p.chunk, p.units - unit0) : 0;
  const double inv = L > 0 ? (double)p.E / ((double)p.K * L * L) : 0.0;
  if (mine)
    for (int q = TOGETHER ? ex : tid; q < chunks; q += TOGETHER ? width : slices * width) all[1] += (double)p.part_z[unit0 + q];
  double v = 0.0;
  int c = 0;
  if (mine && ex < p.E) {
    constexpr int AHEAD = 8;                 // chunks on their way at once
    for (int q0 = from; q0 < chunks; q0 += AHEAD * step) {
      float pv[AHEAD];
      int cv[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const bool there = q0 + q * step < chunks;
        const int64_t at = (int64_t)(unit0 + (there ? q0 + q * step : q0)) * p.E + ex;
        pv[q] = there ? p.part_p[at] : 0.f;
        cv[q] = there ? p.part_c[at] : 0;
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        v += (double)pv[q];
        c += cv[q];
      }
    }
  }
  if (!TOGETHER) {
    sum_p[tid] = v;
    sum_c[tid] = c;
    __syncthreads();
  }
  if (mine && (TOGETHER || slice == 0) && ex < p.E) {
    if (!TOGETHER)
      for (int q = 1; q < slices; ++q) {
        v += sum_p[q * width + ex];
        c += sum_c[q * width + ex];
      }
    p.counts[(int64_t)s * p.E + ex] = c;
    p.table[(int64_t)s * p.E + ex] = (float)((double)p.balance_coeff * inv * (c - (double)p.K * L / p.E));
    all[0] = inv * c * v;
    if (ex == 0) {
      all[2] = L;
      all[3] = L > 0;
    }
  }
  block_sums(all, box);
  const auto finish = [&]() {
    const double per = all[3] > 0 ? 1.0 / all[3] : 0.0, each = all[2] > 0 ? (double)p.z_coeff / all[2] : 0.0;
    *p.loss = (float)((double)p.balance_coeff * all[0] * per + each * all[1]);
    p.table[(int64_t)p.S * p.E] = (float)all[3];        // (below 2^20: as it is)
    p.table[(int64_t)p.S * p.E + 1] = (float)(2.0 * each);
  };
  if (gridDim.x == 1) {
    if (tid == 0) finish();
    return;
  }
  if (tid >= 64) return;
  if (tid == 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) __hip_atomic_store(&p.seq[4 * blockIdx.x + q], all[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  int last = 0;
  if (tid == 0) last = __hip_atomic_fetch_add(p.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  if (!__builtin_amdgcn_readfirstlane(last)) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) all[q] = 0.0;
  for (int i = tid; i < (int)gridDim.x; i += 64)
#pragma unroll
    for (int q = 0; q < 4; ++q) all[q] += __hip_atomic_load(&p.seq[4 * i + q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int q = 0; q < 4; ++q) all[q] = wave_sum(all[q]);
  if (tid == 0) finish();
}

// A wave takes `steps` times 64 / LPT neighbouring tokens.
template <int LPT, int EPL, bool VEC>
__global__ __launch_bounds__(kThreads) void balance_bwd_kernel(const float* __restrict__ logits, const Grad gr, int T, int E, int steps,
                                                               float* __restrict__ d_logits) {
  constexpr int TPW = 64 / LPT;
  __shared__ int box[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane % LPT;
  const int block0 = blockIdx.x * kWaves * steps * TPW;
  const int t0 = block0 + wave * steps * TPW + lane / LPT;
  float next[EPL];
  const auto request = [&](int t) { load_row<LPT, EPL, VEC>(logits + (int64_t)min(t, T - 1) * E, E, g, -INFINITY, next); };
  request(t0);
  const float slope_z = gr.table[(int64_t)gr.S * E + 1], d_loss = *gr.d_loss;
  const Factor of_h = factor_of(d_loss, gr.table[(int64_t)gr.S * E]);
  // (the workgroup's first token's sequence: the offsets up to it, less one)
  int s = gr.sequences ? max(block_leading(gr.S + 1, box, [&](int i) { return gr.sequences[i] <= block0; }) - 1, 0) : 0;
  int row_of = -2;                    // whose table row h is
  float h[EPL];
  for (int i = 0; i < steps; ++i) {
    const int t = t0 + i * TPW;
    if (t >= T) break;                // (a token's lanes together)
    float x[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) x[j] = next[j];
    if (i + 1 < steps) request(t + TPW);
    s = sequence_of(gr, max(s, 0), t);
    const bool owned = s >= 0 && s < gr.S;
    if (s != row_of) {
      load_row<LPT, EPL, VEC>(gr.table + (int64_t)(owned ? s : 0) * E, E, g, 0.f, h);
      row_of = s;
    }
    const float lse = softmax<LPT, EPL>(x);
    float mean = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) mean += h[j] * x[j];
    mean = group_sum<LPT>(mean);
    const float of_lse = d_loss * slope_z * lse;
    float* const to = d_logits + (int64_t)t * E;
#pragma unroll
    for (int j = 0; j < EPL; j += 4) {
      floatx4_t d;
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = owned ? x[j + k] * (of_h.times(h[j + k] - mean) + of_lse) : 0.f;
      const int e = expert_of<LPT>(j, g);
      if (VEC) {
        if (e < E) *reinterpret_cast<floatx4_t*>(to + e) = d;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (e + k < E) to[e + k] = d[k];
      }
    }
  }
}

#define PK_BALANCE_DISPATCH(E, vec, LAUNCH)                                                  \
  do {                                                                                       \
    if ((E) <= 8) { if (vec) LAUNCH(2, 4, true); else LAUNCH(2, 4, false); }                 \
    else if ((E) <= 16) { if (vec) LAUNCH(4, 4, true); else LAUNCH(4, 4, false); }           \
    else if ((E) <= 32) { if (vec) LAUNCH(8, 4, true); else LAUNCH(8, 4, false); }           \
    else if ((E) <= 64) { if (vec) LAUNCH(16, 4, true); else LAUNCH(16, 4, false); }         \
    else if ((E) <= 128) { if (vec) LAUNCH(16, 8, true); else LAUNCH(16, 8, false); }        \
    else if ((E) <= 256) { if (vec) LAUNCH(32, 8, true); else LAUNCH(32, 8, false); }        \
    else if ((E) <= 512) { if (vec) LAUNCH(64, 8, true); else LAUNCH(64, 8, false); }        \
    else { if (vec) LAUNCH(64, 16, true); else LAUNCH(64, 16, false); }                      \
  } while (0)
// tokens that a wave of the above takes at a time
int tokens_at_once(int64_t E) { return E <= 8 ? 32 : E <= 16 ? 16 : E <= 32 ? 8 : E <= 128 ? 4 : E <= 256 ? 2 : 1; }

int64_t chunk_of(int64_t T) { return kChunk * std::max<int64_t>(1, pk_ceil_div(T, (int64_t)kChunk * kMostChunks)); }
int64_t units_of(int64_t T, int64_t S) { return T / chunk_of(T) + S + 1; }
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

extern "C" {

int64_t pk_balance_workspace_bytes(int64_t T, int64_t E, int64_t S) {
  if (T < 0 || E <= 0 || S <= 0) return PK_ERR_ARG;
  const int64_t units = units_of(T, S);
  return 2 * align256(units * E * 4) + align256(units * 4) + align256(S * 32) + 256;
}

int pk_balance_loss(const float* logits, const int32_t* top_idx, const int32_t* sequences, int64_t T, int64_t E, int64_t K, int64_t S,
                    float balance_coeff, float z_coeff, float* loss, int32_t* counts, float* table, void* workspace,
                    int64_t workspace_bytes, pk_stream_t stream) {
  if (T < 0 || E <= 0 || K <= 0 || S <= 0 || (!sequences && S != 1)) return PK_ERR_ARG;
  if (E > PK_MAX_EXPERTS || K > PK_MAX_TOPK || T > 0x7fffffffll / K || S > kMostSequences) return PK_ERR_SHAPE;
  if ((T > 0 && (!logits || !top_idx)) || !loss || !counts || !table) return PK_ERR_ARG;
  if (!workspace || workspace_bytes < pk_balance_workspace_bytes(T, E, S) || !pk_aligned16(workspace)) return PK_ERR_WORKSPACE;
  const int64_t units = units_of(T, S);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](int64_t bytes) { char* const r = at; at += align256(bytes); return r; };
  Forward p = {};
  p.logits = logits; p.top_idx = top_idx; p.sequences = sequences;
  p.T = (int32_t)T; p.E = (int32_t)E; p.K = (int32_t)K; p.S = (int32_t)S; p.chunk = (int32_t)chunk_of(T); p.units = (int32_t)units;
  p.balance_coeff = balance_coeff; p.z_coeff = z_coeff;
  p.part_p = reinterpret_cast<float*>(take(units * E * 4));
  p.part_c = reinterpret_cast<int32_t*>(take(units * E * 4));
  p.part_z = reinterpret_cast<float*>(take(units * 4));
  p.seq = reinterpret_cast<double*>(take(S * 32));
  p.done = reinterpret_cast<uint32_t*>(at);
  p.loss = loss; p.counts = counts; p.table = table;
  hipStream_t s = (hipStream_t)stream;
  const bool vec = E % 4 == 0 && pk_aligned16(logits);
#define PK_LAUNCH(...) \
  PK_LAUNCH_NOCHECK(pk_timing::K_BALANCE, s, (balance_partial_kernel<__VA_ARGS__>), dim3((unsigned)units), dim3(kThreads), 0, s, p)
  PK_BALANCE_DISPATCH(E, vec, PK_LAUNCH);
#undef PK_LAUNCH
  // (few chunks leave most of 1,024 threads nothing to add: 61 sequences of 5 on average take 6.8 to 7.2 us with 256, 7.0 with 1,024)
  const int width = sum_width((int)E), slices = kSumThreads / width;
  if (units / S >= 4 || slices == 1) {
    const int threads = std::max(width, units / S >= 32 ? kSumThreads : 256);
    PK_LAUNCH_NOCHECK(pk_timing::K_BALANCE, s, (balance_sum_kernel<false>), dim3((unsigned)S), dim3(threads), 0, s, p);
  } else {
    PK_LAUNCH_NOCHECK(pk_timing::K_BALANCE, s, (balance_sum_kernel<true>), dim3((unsigned)pk_ceil_div(S, slices)), dim3(kSumThreads), 0, s, p);
  }
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

int pk_balance_loss_bwd(const float* logits, const int32_t* sequences, const float* table, const float* d_loss, float* d_logits,
                        int64_t T, int64_t E, int64_t S, pk_stream_t stream) {
  if (T < 0 || E <= 0 || S <= 0 || (!sequences && S != 1)) return PK_ERR_ARG;
  if (E > PK_MAX_EXPERTS || T > 0x7fffffffll || S > kMostSequences) return PK_ERR_SHAPE;
  if (T == 0) return PK_OK;
  if (!logits || !table || !d_loss || !d_logits) return PK_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const Grad g{table, sequences, d_loss, (int32_t)S};
  // four steps a wave where that leaves every CU eight waves
  const int64_t at_once = (int64_t)kWaves * tokens_at_once(E), steps = T >= at_once * 4 * 512 ? 4 : 1;
  const bool vec = E % 4 == 0 && pk_aligned16(logits) && pk_aligned16(table) && pk_aligned16(d_logits);
#define PK_LAUNCH(...)                                                                                                                        \
  PK_LAUNCH_NOCHECK(pk_timing::K_BALANCE_BWD, s, (balance_bwd_kernel<__VA_ARGS__>), dim3((unsigned)pk_ceil_div(T, at_once * steps)), dim3(kThreads), 0, s, \
                    logits, g, (int)T, (int)E, (int)steps, d_logits)
  PK_BALANCE_DISPATCH(E, vec, PK_LAUNCH);
#undef PK_LAUNCH
  PK_RETURN_IF_LAUNCH_FAILED();
  return PK_OK;
}

}  // extern "C"
