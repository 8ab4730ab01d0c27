// What the 32-queries-per-wave attention kernels (attn32_fwd.hpp, attn_paged_tile.hpp) share: ring geometry, the LDS image of an operand
// tile, lane swaps, the end of a cluster.
#pragma once
#include <utility>
#include "vm_tile.hpp"

namespace a32 {

constexpr int TILE = 64 * ROWB;                 // one 64-row operand tile (16 KiB)
constexpr int SLAB_PITCH = 272;                 // epilogue slab: [32 q][head_dim] bf16 rows, 16-byte aligned, 2-way on the 8-byte writes
constexpr int SLAB = 32 * SLAB_PITCH;
constexpr int NW = 8;                           // waves per workgroup (measured: 4-wave workgroups, two per CU, tie on 8 x 785 and lose 6 % on 4 x 4609)
constexpr int NS = 3;                           // ring slots per operand: tile t+2 is staged while the late half of the workgroup still reads tile t
constexpr int RING_LDS = (2 * NS * TILE > NW * SLAB) ? 2 * NS * TILE : NW * SLAB;      // K ring | V ring; the epilogue slabs overlay them

// lanes 32..63 of `a` <-> lanes 0..31 of `b`. Inline assembly on purpose: given the same VALUE for both operands, hipcc 7.2 folds the
// builtin's two results into ONE register (max(r[0], r[1]) became r[0]: every half kept only the OTHER half's maximum — 5 % errors).
// The s_nop covers the VALU-write -> permlane-read wait states nobody inserts for inline code.
__device__ __forceinline__ void swap_halves(float& a, float& b) {
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}

__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// LDS image of a 64-row x 256-byte operand tile (guide T10, image (a)): 8-row x 64-byte subtiles of 512 B,
//   off(row, ch) = 2048 (row >> 3) + 512 (ch >> 2) + 64 (row & 7) + 16 ((ch & 3) ^ ((row >> 2) & 3))        ch = 16-byte chunk of the row
// Both kinds of read are conflict-free on it AND need only two lane-constant base addresses each — everything that varies inside the
// tile loop (32-key half, k-step, d-tile) is an instruction immediate. (On the plain 256-byte-row image of vm_tile.hpp the XOR term
// depends on the k-step / d-tile: 15 address registers, which at 250 live registers were spilled INTO the tile loop.)
//  * row fragment of the 32x32x16 A operand, lane (r = lane & 31, h = lane >> 5), rows 32 kt + r, chunk 2 ks + h:
//      base[ks & 1] + 8192 kt + 512 (ks >> 1),   base[e] = 2048 (r >> 3) + 64 (r & 7) + 16 ((2 e + h) ^ ((r >> 2) & 3))
//  * transposed fragment (ds_read_b64_tr_b16 x 2), lane (i = lane & 15, g = (lane >> 4) & 1, h), rows 16 m + 4 h + (i >> 2) (+ 8), d-tile b:
//      baseA + 4096 m + 512 b,  baseB + 4096 m + 512 b   (baseB = the +8 rows: + 2048 and the XOR term of (h + 2) & 3)
__device__ __forceinline__ int row_base(int lane, int e) {
  const int r = lane & 31, h = lane >> 5;
  return 2048 * (r >> 3) + 64 * (r & 7) + 16 * ((2 * e + h) ^ ((r >> 2) & 3));
}
__device__ __forceinline__ int tr_base(int lane, int second) {
  const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
  const int q4 = i >> 2, pp = i & 3;
  return 2048 * second + 64 * (4 * h + q4) + 16 * ((2 * g + (pp >> 1)) ^ ((h + 2 * second) & 3)) + 8 * (pp & 1);
}
__device__ __forceinline__ bf16x8_t ld_row(const char* base, int imm) {
  return *reinterpret_cast<const bf16x8_t*>(base + imm);
}
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) { static_for_impl(f, std::make_integer_sequence<int, N>{}); }
// end of a cluster: at most VM VMEM operations stay in flight (the younger DMA groups), the LDS reads of this cluster are done (their
// slot may be restaged once every wave has passed), then the workgroup barrier — fenced for the compiler on both sides: s_barrier
// itself is no memory fence (IntrNoMem) and register-only MFMAs are not ordered by a "memory" clobber (guide rule 18).
template <int VM>
__device__ __forceinline__ void cluster_end() {
  if constexpr (VM == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  else if constexpr (VM == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
  else if constexpr (VM == 6) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
  else if constexpr (VM == -2) asm volatile("" ::: "memory");     // the caller has waited already
  else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // VM == -1: no DMA group to retire here
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace a32
