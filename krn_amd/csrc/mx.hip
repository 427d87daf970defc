// Values to microscaled 4-bit blocks and back, for gfx950 (the format: mx_parts.h).
//
// Quantisation of a block of 32 (OCP MX): with E the biased float32 exponent of the largest magnitude, the scale byte is
// max(E - 2, 0), so that this magnitude lies in [4, 8) and the largest e2m1 value, 6, has its exponent; a code is x times the scale's
// inverse rounded to the nearest e2m1 value, halves to the even code, 6 beyond 6, sign kept (zeros too). A block with a NaN
// or an infinity gets scale 255, which reads back as NaN throughout, and zero codes. Everything is exact but that one
// rounding, which v_cvt_scalef32_pk_fp4_f32 does (checked against the formula for every scale byte below 255, at the halves
// between neighbours, beyond 6 and at -0; a scale of 2^-127, exponent field 0, included).
//
// Both are bound by memory: values are read or written once, with 17 bytes for each 32 of them. Four lanes share a
// block, eight values each, so that a wave's access to values is 16 bytes a lane and contiguous; the block's
// maximum goes through two DPP exchanges.
#include "mx_parts.h"

namespace krn {

template <int KIND>
struct Eight {  // eight consecutive values of a row, from value `col` of `k`; zeros past the end
  float v[8];
  __device__ static Eight load(const uint8_t* row, int64_t col, int64_t k) {
    Eight x;
    if (col + 8 <= k) {
      if constexpr (KIND == F32) {
        const u32x4_any* p = reinterpret_cast<const u32x4_any*>(row + col * 4);
        const u32x4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = __uint_as_float(a[i]), x.v[4 + i] = __uint_as_float(b[i]);
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4_any*>(row + col * 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t h = (uint16_t)(w[i >> 1] >> ((i & 1) * 16));
          x.v[i] = KIND == F16 ? h2f(h) : bf2f(h);
        }
      }
      return x;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x.v[i] = 0.0f;
      if (col + i < k) {
        if constexpr (KIND == F32) x.v[i] = reinterpret_cast<const float*>(row)[col + i];
        else if constexpr (KIND == F16) x.v[i] = h2f(reinterpret_cast<const uint16_t*>(row)[col + i]);
        else x.v[i] = bf2f(reinterpret_cast<const uint16_t*>(row)[col + i]);
      }
    }
    return x;
  }
};

// The largest of the four lanes of a block, and the block's scale byte
__device__ __forceinline__ uint32_t block_scale(const float (&v)[8]) {
  uint32_t top = 0;  // magnitudes order as their bits do, NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xF, 0xF, true));  // lane ^ 1
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xF, 0xF, true));  // lane ^ 2
  const uint32_t e = top >> 23;
  return e == 255 ? 255 : max(e, 2u) - 2;
}

__device__ __forceinline__ uint32_t eight_codes(const float (&v)[8], uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
  return scale == 255 ? 0 : w;
}

// `blocks` blocks of rows of `nb`; workgroup w takes blocks 64 U w .. + 64 U - 1, quad q of it block q of each run of 64.
// ROWS: rows end inside a block (K is no multiple of 32), so a block has to know its row.
template <int KIND, int U, bool ROWS>
__global__ __launch_bounds__(256) void mx_quantize(const uint8_t* __restrict__ X, uint8_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales, int64_t blocks, int64_t k, uint32_t nb) {
  constexpr int SIZE = KIND == F32 ? 4 : 2;
  const int64_t first = (int64_t)blockIdx.x * (64 * U);
  const int quad = threadIdx.x >> 2, part = threadIdx.x & 3;
  const int64_t row0 = ROWS ? first / nb : 0;
  const uint32_t in_row = ROWS ? (uint32_t)(first - row0 * nb) : 0;
  Eight<KIND> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b = first + u * 64 + quad;
    if (b < blocks) {
      if constexpr (ROWS) {
        const uint32_t at = in_row + u * 64 + quad, row = at / nb;
        x[u] = Eight<KIND>::load(X + (row0 + row) * k * SIZE, (int64_t)(at - row * nb) * 32 + part * 8, k);
      } else {
        x[u] = Eight<KIND>::load(X, b * 32 + part * 8, blocks * 32);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b = first + u * 64 + quad;
    if (b < blocks) {  // the four lanes of a quad alike
      const uint32_t s = block_scale(x[u].v);
      reinterpret_cast<uint32_t*>(codes)[b * 4 + part] = eight_codes(x[u].v, s);
      if (part == 0) scales[b] = (uint8_t)s;
    }
  }
}

template <int KIND, int U, bool ROWS>
__global__ __launch_bounds__(256) void mx_dequantize(const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, uint8_t* __restrict__ Y,
                                                     int64_t blocks, int64_t k, uint32_t nb) {
  constexpr int SIZE = KIND == F32 ? 4 : 2;
  const int64_t first = (int64_t)blockIdx.x * (64 * U);
  const int quad = threadIdx.x >> 2, part = threadIdx.x & 3;
  const int64_t row0 = ROWS ? first / nb : 0;
  const uint32_t in_row = ROWS ? (uint32_t)(first - row0 * nb) : 0;
  uint32_t w[U], s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b = first + u * 64 + quad;
    if (b < blocks) w[u] = reinterpret_cast<const uint32_t*>(codes)[b * 4 + part], s[u] = scales[b];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b = first + u * 64 + quad;
    if (b >= blocks) continue;
    const float scale = __uint_as_float(s[u] << 23);
    float v[8];
#define KRN_TWO(i)                                                                       \
  {                                                                                      \
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, i);             \
    v[2 * (i)] = p[0], v[2 * (i) + 1] = p[1];                                            \
  }
    KRN_TWO(0) KRN_TWO(1) KRN_TWO(2) KRN_TWO(3)
#undef KRN_TWO
    int64_t col = b * 32 + part * 8, end = blocks * 32;
    uint8_t* row = Y;
    if constexpr (ROWS) {
      const uint32_t at = in_row + u * 64 + quad, r = at / nb;
      row = Y + (row0 + r) * k * SIZE;
      col = (int64_t)(at - r * nb) * 32 + part * 8, end = k;
    }
    if constexpr (KIND == F32) {
      float* out = reinterpret_cast<float*>(row) + col;
      if (col + 8 <= end) {
        u32x4_any* p = reinterpret_cast<u32x4_any*>(out);
        p[0] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
        p[1] = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < end) out[i] = v[i];
      }
    } else {
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] = KIND == BF16 ? f2bf2(v[2 * i], v[2 * i + 1]) : (uint32_t)f2h(v[2 * i]) | (uint32_t)f2h(v[2 * i + 1]) << 16;
      uint16_t* out = reinterpret_cast<uint16_t*>(row) + col;
      if (col + 8 <= end) {
        *reinterpret_cast<u32x4_any*>(out) = u32x4{h[0], h[1], h[2], h[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < end) out[i] = (uint16_t)(h[i >> 1] >> ((i & 1) * 16));
      }
    }
  }
}

}  // namespace krn

using namespace krn;

// The arguments both entry points share, checked; -1 with a message, or 0
static int mx_arguments(const char* who, int kind, const void* values, const void* codes, const void* scales, int64_t rows,
                        int64_t k) {
  if (kind != F32 && kind != F16 && kind != BF16) {
    krn_set_error("%s: element kind %d; float32, f16 or bf16 values are taken", who, kind);
    return -1;
  }
  // 2^31 blocks are 2^23 workgroups: a launch's threads along an axis stay below 2^32
  if (rows < 0 || k < 1 || k > 0x7fffffff || rows > ((int64_t)1 << 31) / mx_blocks(k)) {
    krn_set_error("%s: %lld rows of %lld values; rows of 1 to 2^31 - 1 values, at most 2^31 blocks of 32 in all", who,
                  (long long)rows, (long long)k);
    return -1;
  }
  if ((uintptr_t)codes % 16 != 0) {
    krn_set_error("%s: codes start at a 16-byte aligned address", who);
    return -1;
  }
  const int64_t nb = mx_blocks(k), bytes = rows * k * (kind == F32 ? 4 : 2);
  if (share_memory(values, bytes, codes, rows * nb * 16) || share_memory(values, bytes, scales, rows * nb) ||
      share_memory(codes, rows * nb * 16, scales, rows * nb)) {
    krn_set_error("%s: values, codes and scales share memory", who);
    return -1;
  }
  return 0;
}

static int launched(const char* who) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("%s launch: %s", who, hipGetErrorString(err));
  return (int)err;
}

extern "C" {

// See include/krn_amd.h for the contract of each entry point.
int krn_mx_quantize(int kind, const void* x, void* codes, void* scales, int64_t rows, int64_t k, void* stream) {
  if (mx_arguments("mx_quantize", kind, x, codes, scales, rows, k)) return -1;
  const int64_t nb = mx_blocks(k), blocks = rows * nb;
  if (blocks == 0) return 0;
  const bool many = blocks >= 64 * 1024;
  const int64_t groups = many ? (blocks + 255) / 256 : (blocks + 63) / 64;
#define KRN_GO(KIND, U, ROWS)                                                                                      \
  hipLaunchKernelGGL((mx_quantize<KIND, U, ROWS>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream,      \
                     (const uint8_t*)x, (uint8_t*)codes, (uint8_t*)scales, blocks, k, (uint32_t)nb)
#define KRN_KIND(KIND)                                 \
  do {                                                 \
    if (k % 32 == 0) {                                 \
      if (many) KRN_GO(KIND, 4, false);                \
      else KRN_GO(KIND, 1, false);                     \
    } else {                                           \
      if (many) KRN_GO(KIND, 4, true);                 \
      else KRN_GO(KIND, 1, true);                      \
    }                                                  \
  } while (0)
  if (kind == F32) KRN_KIND(F32);
  else if (kind == F16) KRN_KIND(F16);
  else KRN_KIND(BF16);
#undef KRN_GO
  return launched("mx_quantize");
}

int krn_mx_dequantize(const void* codes, const void* scales, int kind, void* y, int64_t rows, int64_t k, void* stream) {
  if (mx_arguments("mx_dequantize", kind, y, codes, scales, rows, k)) return -1;
  const int64_t nb = mx_blocks(k), blocks = rows * nb;
  if (blocks == 0) return 0;
  const bool many = blocks >= 64 * 1024;
  const int64_t groups = many ? (blocks + 255) / 256 : (blocks + 63) / 64;
#define KRN_GO(KIND, U, ROWS)                                                                                      \
  hipLaunchKernelGGL((mx_dequantize<KIND, U, ROWS>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream,    \
                     (const uint8_t*)codes, (const uint8_t*)scales, (uint8_t*)y, blocks, k, (uint32_t)nb)
  if (kind == F32) KRN_KIND(F32);
  else if (kind == F16) KRN_KIND(F16);
  else KRN_KIND(BF16);
#undef KRN_KIND
#undef KRN_GO
  return launched("mx_dequantize");
}

}  // extern "C"
