// The router's balance loss: what its own kernels and the region's router backward share.
//
//   for a sequence of L tokens:  f_e = counts_e E / (K L),  P_e = mean of softmax(logits)_e over its tokens
//   loss = balance_coeff mean over the sequences that have tokens of sum_e f_e P_e + z_coeff mean over the tokens of lse^2
//
// The counts have no gradient.  A token's softmax p sees dloss/dp_e = h_e with h_e = balance_coeff E counts_e / (K L^2 S'), and
//   d_logit_e = d_loss p_e (h_e - sum_j h_j p_j + 2 z_coeff lse / N).
// Since the p_j add up to 1, the same constant may be taken from all h: the table holds h - mean(h), from the whole numbers
// counts_e - K L / E, so that nothing cancels where the experts are nearly balanced.
#pragma once
#include "pk_common.h"

namespace pk_balance {

// of a call: the first launch has a workgroup for each and more
constexpr int64_t kMostSequences = 0xfffff;

// What a backward needs beside the logits.  table: [S][E] of h - mean(h) without the 1 / S', then S' and 2 z_coeff / N.
struct Grad {
  const float* table;
  const int32_t* sequences;   // [S + 1], or nullptr: one sequence of all T tokens
  const float* d_loss;
  int32_t S;
};

// d_loss / S', a factor of every element: its rounding would make all of them too large or too small together, so it comes in two parts.
struct Factor {
  float hi, lo;
  __device__ __forceinline__ float times(float v) const { return fmaf(hi, v, lo * v); }
};
__device__ __forceinline__ Factor factor_of(float d_loss, float some) {
  const double f = (double)d_loss / some;
  const float hi = (float)f;
  return {hi, __builtin_isfinite(hi) ? (float)(f - hi) : 0.f};
}

// Bounds of sequence s.  Offsets ascend within 0 .. T; whatever else they hold, the range stays inside.
__device__ __forceinline__ int begin_of(const int32_t* sequences, int s, int T) { return sequences ? min(max(sequences[s], 0), T) : 0; }
__device__ __forceinline__ int end_of(const int32_t* sequences, int s, int T) {
  return sequences ? min(max(sequences[s + 1], begin_of(sequences, s, T)), T) : T;
}

// How many of the first n things hold, where whatever follows one that does not hold does not either: WIDTH things are looked at together,
// evenly spaced in what is left while that is more than `scan`.  count(m, f): how many of f(0) .. f(m - 1) hold, the same for all of those
// who ask.  (Things in another order: some number from 0 to n.)
template <int WIDTH, typename C, typename F>
__device__ __forceinline__ int leading(int n, int scan, C&& count, F&& holds) {
  int lo = 0, left = n;
  while (left > scan) {
    const int stride = (left + WIDTH - 1) / WIDTH;
    const int c = count(WIDTH, [&](int k) { return (k + 1) * stride <= left && holds(lo + (k + 1) * stride - 1); });
    lo += c * stride;
    left = min(stride - 1, left - c * stride);
  }
  return lo + count(left, [&](int i) { return holds(lo + i); });
}
// For a wave: up to 128 things take two loads of a lane at once, 2^20 three rounds of one and the same.
template <typename F>
__device__ __forceinline__ int wave_leading(int n, F&& holds) {
  const int lane = threadIdx.x & 63;
  return leading<64>(n, 128, [&](int m, auto&& f) {
    int c = 0;
    for (int i = 0; i < m; i += 64) c += __popcll(__ballot(i + lane < m && f(i + lane)));
    return c;
  }, holds);
}

// The sequence that token t is in, searched from s on; S: behind the last one, -1: in front of the first one.
__device__ __forceinline__ int sequence_of(const Grad& g, int s, int t) {
  if (!g.sequences) return 0;
  for (int n = 0; s < g.S && g.sequences[s + 1] <= t; ++s)
    if (++n == 4) {                  // (many without tokens)
      int end = g.S;                 // the first of s .. S that ends behind t, or S
      while (s < end) {
        const int mid = s + (end - s) / 2;
        if (g.sequences[mid + 1] <= t) s = mid + 1; else end = mid;
      }
      break;
    }
  return s == 0 && t < g.sequences[0] ? -1 : s;
}

}  // namespace pk_balance
