// Microscaled 4-bit matrices (OCP MX, MXFP4): what their kernels share.
//
// A row of K values is NB = ceil(K / 32) blocks of 32. Block b holds 32 e2m1 codes, 16 bytes with the first of a pair in
// the low nibble, and one e8m0 byte s: its values are e2m1(code) * 2^(s - 127), NaN for s = 255. Codes past K are zero. Codes
// (rows x 16 NB bytes) and scales (rows x NB bytes) are separate arrays, row-major and without padding, so that a
// block's codes are one aligned 16-byte piece: what a lane of the 16x16x128 MFMA takes (32 values of one row).
//
// K order. The kernels walk a row in slabs of 16 blocks (512 values, 256 bytes of codes, 16 scales). MFMA step j = 0 .. 3
// of a slab gives lane group g = lane / 16 block 4 j + g, so a step reads 64 consecutive bytes of each of 16 rows. The
// instruction takes a lane's scale from one byte of a register, the same byte for every lane: byte j here, so a lane packs
// byte g of each of its row's four scale words of the slab into one word, once a slab.
#pragma once
#include "gemm_parts.h"

namespace krn {

constexpr int MX_BLOCK = 32;
constexpr int SLAB = 16;          // blocks of a slab

__host__ __device__ inline int64_t mx_blocks(int64_t k) { return (k + MX_BLOCK - 1) / MX_BLOCK; }

// A row whose end cuts its last slab has that slab taken from its last 16 blocks: those of them that the slab before holds
// already count as zeros there (the callers give their codes so), and the scales are 16 bytes of the row as they lie. (A
// scale of 255 among the blocks taken twice makes both products NaN, as one does.) A row of fewer than 16 blocks is
// one slab; its scales go word by word, 2^0 past its end. No byte outside the row is read.
__device__ __forceinline__ int slab_block(int slab, int nb) { return nb < SLAB ? 0 : min(slab * SLAB, nb - SLAB); }

// Whether block `block` counts in slab `slab` of a row of `nb` blocks
__device__ __forceinline__ bool in_slab(int block, int slab, int nb) { return block >= slab * SLAB && block < nb; }

__device__ __forceinline__ u32x4 long_scales(const uint8_t* row, int slab, int nb) {  // nb >= 16
  return *reinterpret_cast<const u32x4_any*>(row + min(slab * SLAB, nb - SLAB));
}

__device__ __forceinline__ u32x4 short_scales(const uint8_t* row, int nb) {  // nb < 16
  typedef uint32_t u32_any __attribute__((aligned(1)));
  constexpr uint32_t UNIT = 0x7f7f7f7f;
  u32x4 w = {UNIT, UNIT, UNIT, UNIT};
  if (nb < 4) {
    const uint32_t b0 = row[0], b1 = nb > 1 ? row[1] : 0x7f, b2 = nb > 2 ? row[2] : 0x7f;
    w[0] = b0 | b1 << 8 | b2 << 16 | 0x7fu << 24;
    return w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // the word that the row's end cuts is its last four bytes, shifted
    const int at = min(4 * i, nb - 4), cut = 4 * i - at;
    const uint32_t v = *reinterpret_cast<const u32_any*>(row + at);
    w[i] = cut < 4 ? __builtin_amdgcn_alignbyte(UNIT, v, cut) : UNIT;
  }
  return w;
}

__device__ __forceinline__ u32x4 slab_scales(const uint8_t* row, int slab, int nb) {
  return nb < SLAB ? short_scales(row, nb) : long_scales(row, slab, nb);
}

// Byte g of each of four words, in one word
__device__ __forceinline__ uint32_t scale_bytes(const u32x4& w, int g) {
  const uint32_t pick = (uint32_t)g | (uint32_t)(g + 4) << 8;
  const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], pick), hi = __builtin_amdgcn_perm(w[3], w[2], pick);
  return (lo & 0xffffu) | hi << 16;
}

// C += A B^T of one step: 16 rows of A by 16 of B, 128 values of K, step J of the slab (byte J of the packed scales)
template <int J>
__device__ __forceinline__ f32x4 mx_mfma(const u32x4& a, const u32x4& b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x4 x = __builtin_bit_cast(i32x4, a), y = __builtin_bit_cast(i32x4, b);
  const i32x8 xa = {x[0], x[1], x[2], x[3], 0, 0, 0, 0}, yb = {y[0], y[1], y[2], y[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xa, yb, c, 4, 4, J, (int)sa, J, (int)sb);  // format 4: e2m1
}

}  // namespace krn
