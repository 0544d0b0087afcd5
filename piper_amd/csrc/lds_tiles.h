// Tiles of 16-bit operands in LDS for the matrix instructions: loads that go there directly, the layouts, the fragments.
#pragma once
#include "pk_common.h"
#include <type_traits>

namespace pk_lds {

typedef short shortx4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Direct global->LDS load of 16 bytes per lane: lane l's bytes land at lds_base + 16*l.
// Issued from inline asm so that the compiler does not serialise later LDS reads behind it;
// completion is tracked by hand with vmcnt (wait_dma) followed by a workgroup barrier.
// The statement sets M0 and uses it at once.  M0 cannot be named as clobbered (the compiler
// treats it as reserved and rejects the promise to preserve it), and nothing else in these
// kernels keeps a value in it: on gfx9 ordinary LDS accesses do not read M0, and the kernels
// use no indirect register indexing, readlane with a register index excepted, which takes an
// SGPR operand and not M0.
__device__ __forceinline__ void dma16(const void* gptr, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(gptr)
               : "memory");
}
// The same load with the address split into a wave-uniform 64-bit base (scalar registers) and a
// 32-bit byte offset per lane: a k-loop then advances one scalar pointer per operand and k-tile
// instead of forming a 64-bit address per lane and load.  The LDS destination is lds_base + IMM.
template <int IMM>
__device__ __forceinline__ void dma16_s(uint32_t voff, const void* sbase, uint32_t lds_base) {
  asm volatile("s_add_i32 m0, %0, %3\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(lds_base), "v"(voff), "s"(sbase), "n"(IMM)
               : "memory", "scc");
}
// Four bytes per lane straight into LDS (lane l's dword lands at lds_base + 4*l), same address form.
__device__ __forceinline__ void dma4_s(uint32_t voff, const void* sbase, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2"
               :: "s"(lds_base), "v"(voff), "s"(sbase)
               : "memory");
}
// f(std::integral_constant<int, 0>{}), ..., f(std::integral_constant<int, N-1>{}) in order
template <int I0, int N, typename F>
__device__ __forceinline__ void static_for_impl(F&& f) {
  if constexpr (I0 < N) {
    f(std::integral_constant<int, I0>{});
    static_for_impl<I0 + 1, N>(f);
  }
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) { static_for_impl<0, N>(f); }
template <int N>
__device__ __forceinline__ void wait_dma() {
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// A wave-uniform 64-bit value that the compiler could not prove uniform: into scalar registers.
__device__ __forceinline__ int64_t uniform_i64(int64_t x) {
  const uint64_t v = (uint64_t)x;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ const char* uniform_ptr(const char* p) {
  return (const char*)(uintptr_t)uniform_i64((int64_t)(uintptr_t)p);
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(lds_ptr_t)p;
}

// ---------------------------------------------------------------------------------------------
// LDS tile layouts (BK = 64 or 32 deep).  16-byte chunks are XOR-swizzled so that the fragment
// reads below touch every bank once.
//
// KC tile: [ROWS rows of the M or N index][BK k], k contiguous (2*BK bytes per row, BK/8 chunks).
//          chunk c of row r sits at position c ^ swz(r): (r >> 1) & 7 for BK 64, (r >> 2) & 3 for BK 32.
// MN tile: [BK k][COLS of the M or N index], the M/N index contiguous (COLS/8 chunks per row).
//          chunk c of row k sits at position c ^ ((k & 3) << 2).
//
// A wave-level dma16 fills 64 consecutive 16-byte slots; which global chunk a lane fetches is
// chosen so that the swizzled layout comes out.

// Global element offset (within the operand) of the chunk that lane `lane` of load `G`
// (G-th group of 64 slots of the tile) must fetch, for a KC tile: returns row and k offset.
template <int BK>
__device__ __forceinline__ int kc_swz(int row) { return BK == 64 ? ((row >> 1) & 7) : ((row >> 2) & 3); }
template <int BK>
__device__ __forceinline__ void kc_slot(int G, int lane, int& row, int& kofs) {
  constexpr int CPR = BK / 8;
  const int slot = G * 64 + lane;
  row = slot / CPR;
  kofs = ((slot % CPR) ^ kc_swz<BK>(row)) * 8;
}
template <int COLS>
__device__ __forceinline__ void mn_slot(int G, int lane, int& krow, int& cofs) {
  constexpr int CPR = COLS / 8;
  const int slot = G * 64 + lane;
  krow = slot / CPR;
  cofs = ((slot % CPR) ^ ((krow & 3) << 2)) * 8;
}

// MFMA operand fragment (8 values of 16 bits per lane: row lane%32, k = 16*ks + 8*(lane/32) + 0..7).
template <int BK, typename V = bf16x8_t>
__device__ __forceinline__ V frag_kc(const char* tile, int row0, int ks, int lane) {
  const int r = row0 + (lane & 31);
  const int c = 2 * ks + (lane >> 5);
  return *reinterpret_cast<const V*>(tile + r * (2 * BK) + ((c ^ kc_swz<BK>(r)) << 4));
}
// Same fragment out of an MN tile through the transposing LDS read: within 16 lanes, lane i
// points at 4 consecutive columns of k-row i/4 and receives 4 consecutive k of column i.
template <int COLS, typename V = bf16x8_t>
__device__ __forceinline__ V frag_mn(const char* tile, int col0, int ks, int lane) {
  const int i = lane & 15;
  const int krow = ks * 16 + 8 * (lane >> 5) + (i >> 2);
  const int col = col0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
  const int pos = (col >> 3) ^ ((i >> 2) << 2);
  const char* p = tile + krow * (COLS * 2) + pos * 16 + (col & 7) * 2;
  const shortx4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4_t*)(p));
  const shortx4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4_t*)(p + 4 * COLS * 2));
  typedef short shortx8_t __attribute__((ext_vector_type(8)));
  shortx8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(V, v);
}

// LDS traffic of one wave is ordered by the hardware; this only stops the compiler from
// moving the staged reads above the writes.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Wait until at most `t` (0..MAXT) whole tiles of L loads each are still in flight.
template <int L, int MAXT>
__device__ __forceinline__ void wait_tiles(int t) {
  if (MAXT <= 0 || t <= 0) { wait_dma<0>(); return; }
  if (t >= MAXT) { wait_dma<(MAXT > 0 ? MAXT : 0) * L>(); return; }
  wait_tiles<L, (MAXT > 0 ? MAXT - 1 : 0)>(t);
}

// Wait until at most n (wave-uniform, rounded down to a multiple of 4, capped at 60) vector-memory
// operations are outstanding.  Loads, stores and atomics retire from the counter in issue
// order, so with n = a lower bound of the operations issued AFTER the ones of interest this
// waits for those without waiting for the younger ones (for example an epilogue's stores).
__device__ __forceinline__ void wait_vm_le(int n) {
  switch ((n < 60 ? n : 60) >> 2) {
    case 0: wait_dma<0>(); break;    case 1: wait_dma<4>(); break;    case 2: wait_dma<8>(); break;
    case 3: wait_dma<12>(); break;   case 4: wait_dma<16>(); break;   case 5: wait_dma<20>(); break;
    case 6: wait_dma<24>(); break;   case 7: wait_dma<28>(); break;   case 8: wait_dma<32>(); break;
    case 9: wait_dma<36>(); break;   case 10: wait_dma<40>(); break;  case 11: wait_dma<44>(); break;
    case 12: wait_dma<48>(); break;  case 13: wait_dma<52>(); break;  case 14: wait_dma<56>(); break;
    default: wait_dma<60>(); break;
  }
}

}  // namespace pk_lds
