// Weights of 4 bits with group scales: their layout, and what the kernels that read them share.
//
//   W[f, k] = scale[f, k / group] * (code[f, k] - zero[f, k / group]),   code 0 .. 15, zero 0 .. 15 (8 where there is none), group 32, 64 or 128
//
// A matrix is cut into strips of 16 rows, tiles of eight strips and steps of 128 along K (skein_b200/ops/int4.py packs it; rows and K are padded with
// zero scales). For a pair of matrices (gate and up of a SwiGLU) a strip holds 8 gate rows and the 8 up rows of the same features, so that whoever
// holds accumulator row r of a strip has its partner at r + 8.
// A step of a tile is one run of memory, a multiple of 128 bytes: the codes of its strips, then their scales, then their zeros where there are any. One
// bulk copy fetches it. (Strips with scales of their own, 1056 bytes each, made the copies start off 128-byte boundaries, which the copy engine
// takes 16 bytes at a time: 140 cycles per KB, three quarters of the tensor-memory kernel's time.)
//   codes  [2][t 4][g 8][16 bytes]: lane (g = lane / 4, t = lane % 4) of half j owns rows g and g + 8 at k = 64 j + 8 t .. + 7 and
//          64 j + 32 + 8 t .. + 7: words {row g, first; row g, second; row g + 8, first; row g + 8, second}. One 16-byte load of a warp is 16 rows x
//          64 k in the order in which mma.sync's A operand wants them (any order of k is right as long as B has the same). The row's eight
//          codes of a word are neighbours in k, so that the tensor-memory kernel takes its rows from the same bytes, eight bytes at a time and
//          without bank conflicts (that is why g runs fastest).
//          Inside a word the codes of even k are the low half's nibbles, those of odd k the high half's: (word >> 4 i) & 0x000f000f is the
//          pair (k = 2 i, 2 i + 1).
//   scales [g 8][128 / group][2] 16-bit: rows g and g + 8 side by side; zeros the same in bytes.
#pragma once
#include "gemm_sched.cuh"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace skein {

constexpr int I4_STEP = 128;                       // elements of K
constexpr int I4_CODES = 16 * I4_STEP / 2;         // bytes of a strip's codes in a step
// bytes of a tile's step; gp: groups of a step
__host__ __device__ constexpr int i4_record(int gp, bool zero) { return 8 * (I4_CODES + 32 * gp + (zero ? 16 * gp : 0)); }
constexpr int I4_SCALES = 8 * I4_CODES;            // where its scales begin
__host__ __device__ constexpr int i4_zeros(int gp) { return I4_SCALES + 8 * 32 * gp; }

// Codes as bf16 pairs (code - zero) / 64. A 16-bit pattern P below 256 is the bf16 number P 2^-133 (subnormals, and the first exponent whose steps are
// as wide), so a masked code needs no exponent of its own: one multiply-add by 2^127 (2^123 for a code four bits up) and -zero / 64 gives the
// difference, a whole number below 16 over 64, exactly. Nine instructions per word of eight codes: a shift, four masks, four multiply-adds.
// Spelled out so that no fast-math flag flushes the subnormal operands.
__device__ __forceinline__ uint32_t i4_fma(uint32_t v, uint32_t m, uint32_t a) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(m), "r"(a));
  return r;
}
constexpr uint32_t I4_EIGHT = 0xbe00be00u;      // -8 / 64
__device__ __forceinline__ uint32_t i4_zero(uint32_t zero) { return i4_fma(zero | (zero << 16), 0xff00ff00u, 0x80008000u); }   // -zero / 64
__device__ __forceinline__ void i4_expand(uint32_t word, uint32_t zero, uint32_t* r) {
  const uint32_t up = word >> 8;
  r[0] = i4_fma(word & 0x000f000fu, 0x7f007f00u, zero);
  r[1] = i4_fma(word & 0x00f000f0u, 0x7d007d00u, zero);
  r[2] = i4_fma(up & 0x000f000fu, 0x7f007f00u, zero);
  r[3] = i4_fma(up & 0x00f000f0u, 0x7d007d00u, zero);
}
// a scale times the 64 of its codes
__device__ __forceinline__ float i4_scale(uint32_t raw, bool half) {
  return 64.f * (half ? __half2float(__ushort_as_half((unsigned short)raw)) : __uint_as_float(raw << 16));
}

}  // namespace skein
