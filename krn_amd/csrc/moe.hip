// A mixture-of-experts layer for a few tokens on gfx950, experts in microscaled 4 bits (mx_parts.h):
//   y_t = sum over the top_k experts e of token t of  w_te * down_e (silu(gate_e x_t) * up_e x_t),
// w_t the softmax of the chosen experts' router logits x_t . router_e. Ties go to the expert of the lower index; a NaN logit
// counts as the largest.
//
// Bound by reading the chosen experts' weights, each once whatever the number of its tokens (up to 16). Four launches:
//   logits  x router^T in 16-bit MFMAs (products exact, float32 sums), K split over workgroups, partial sums to memory
//   route   one workgroup: a wave chooses a token's experts; every expert's tokens as a 64-bit mask, so that its count and a
//           token's place in it are population counts and no order of atomics shows; the chosen experts in a row
//   up      a workgroup per 16 inner values of a chosen expert: gate and up rows, silu(gate) * up * w to memory in bf16
//   down    a workgroup per 16 outputs: all chosen experts' rows, added per token
// Weights go to bf16 exactly (v_cvt_scalef32_pk_bf16_fp4: two bits of mantissa and a power of two) and are multiplied in
// 16x16x32 bf16 MFMAs, 16 weight rows by up to 16 tokens. bfloat16 tokens are taken as they are and the inner values
// rounded to bfloat16, as a bf16 layer stores them; float16 tokens and their inner values are split into a bf16 and
// the bf16 of the remainder, which holds all of a float16, so that nothing is lost and nothing overflows.
#include "mx_parts.h"

namespace krn {

constexpr int MOE_TOKENS = 64, MOE_EXPERTS = 1024, MOE_TOP_K = 16;

// What the launches hand on, in the workspace
struct Routing {
  int* active;         // number of chosen experts, then the experts
  int* offset;         // of the i-th chosen expert's tokens among `token`, and the end of the last
  int* token;          // by expert, in the order of the tokens
  float* weight;
};

// Eight values of a row from value `at` of `k` as raw 16-bit words; zeros past the end
__device__ __forceinline__ u32x4 eight16(const uint16_t* row, int64_t at, int64_t k) {
  if (at + 8 <= k) return *reinterpret_cast<const u32x4_any*>(row + at);
  u32x4 w = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (at + i < k) w[i >> 1] |= (uint32_t)row[at + i] << ((i & 1) * 16);
  return w;
}

template <int KIND>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (KIND == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Partial logits of 16 experts and 16 tokens over the K steps of part blockIdx.z: partial[part][token][expert]
template <int KIND>
__global__ __launch_bounds__(256) void moe_logits(const uint16_t* __restrict__ X, const uint16_t* __restrict__ router,
                                                  float* __restrict__ partial, int T, int64_t H, int E, int steps) {
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const uint16_t* w = router + (int64_t)min(e0 + r, E - 1) * H;
  const uint16_t* x = X + (int64_t)min(t0 + r, T - 1) * H;
  f32x4 acc = {};
  const int64_t first = ((int64_t)blockIdx.z * 4 + wave) * steps * 32;
  for (int s = 0; s < steps; ++s) {
    const int64_t at = first + s * 32 + g * 8;
    acc = mfma16<KIND>(eight16(w, at, H), eight16(x, at, H), acc);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && t0 + r < T) {
    const f32x4 v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (e0 + 4 * g + q < E) partial[((int64_t)blockIdx.z * T + t0 + r) * E + e0 + 4 * g + q] = v[q];
  }
}

// A float32 as an unsigned number in the same order, never 0; NaN above everything
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(1024) void moe_route(const float* __restrict__ partial, int parts, int T, int E, int top_k,
                                                  Routing out) {
  __shared__ uint32_t key[16][MOE_EXPERTS];  // a wave's token's logits in order, 0 once chosen
  __shared__ unsigned long long mask[MOE_EXPERTS];
  __shared__ uint32_t base[MOE_EXPERTS], wave_sum[16];
  __shared__ int chosen[MOE_TOKENS * MOE_TOP_K];
  __shared__ float weight[MOE_TOKENS * MOE_TOP_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  mask[threadIdx.x] = 0;
  __syncthreads();
  for (int t = wave; t < T; t += 16) {
    for (int e = lane; e < E; e += 64) {
      float v = 0.0f;
      for (int p = 0; p < parts; ++p) v += partial[((int64_t)p * T + t) * E + e];
      key[wave][e] = ordered(v);
    }
    float mine = -INFINITY;  // lane j: the logit of choice j
    int pick = 0;
    for (int j = 0; j < top_k; ++j) {
      unsigned long long best = 0;
      for (int e = lane; e < E; e += 64) {
        const unsigned long long v = (unsigned long long)key[wave][e] << 32 | (uint32_t)~e;
        best = v > best ? v : best;
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const unsigned long long v = __shfl_xor(best, d);
        best = v > best ? v : best;
      }
      const int e = (int)~(uint32_t)best;
      const uint32_t u = (uint32_t)(best >> 32);
      if (lane == j) mine = __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u), pick = e;
      if (lane == (e & 63)) key[wave][e] = 0;
    }
    const float top = __shfl(mine, 0);
    const float p = lane < top_k ? expf(mine - top) : 0.0f;
    float sum = p;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) sum += __shfl_xor(sum, d);
    if (lane < top_k) {
      chosen[t * top_k + lane] = pick;
      weight[t * top_k + lane] = p / sum;
      atomicOr(&mask[pick], 1ull << t);
    }
  }
  __syncthreads();
  // places: tokens in the low half, chosen experts in the high half of one sum over the experts before
  const int e = threadIdx.x;
  const uint32_t count = e < E ? (uint32_t)__popcll(mask[e]) : 0, own = count | (count > 0 ? 1u << 16 : 0);
  uint32_t scan = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t v = __shfl_up(scan, d);
    if (lane >= d) scan += v;
  }
  if (lane == 63) wave_sum[wave] = scan;
  __syncthreads();
  uint32_t before = scan - own, total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += wave_sum[w];
    total += wave_sum[w];
  }
  base[e] = before & 0xffff;
  if (count > 0) out.active[1 + (before >> 16)] = e, out.offset[before >> 16] = (int)(before & 0xffff);
  if (e == 0) out.active[0] = (int)(total >> 16), out.offset[total >> 16] = (int)(total & 0xffff);
  __syncthreads();
  for (int i = threadIdx.x; i < T * top_k; i += 1024) {
    const int t = i / top_k, expert = chosen[i];
    const int at = (int)base[expert] + __popcll(mask[expert] & ((1ull << t) - 1));
    out.token[at] = t, out.weight[at] = weight[i];
  }
}

// Eight codes of a block as bf16 values
__device__ __forceinline__ u32x4 bf16_codes(uint32_t w, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
               __builtin_bit_cast(uint32_t, d)};
}

// Eight float16 values as the bf16 nearest to each and the bf16 of what is left (exact: 11 bits in two times 8)
__device__ __forceinline__ void split_f16(const u32x4& x, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = h2f((uint16_t)x[i]), b = h2f((uint16_t)(x[i] >> 16));
    hi[i] = f2bf2(a, b);
    lo[i] = f2bf2(a - bf2f((uint16_t)hi[i]), b - bf2f((uint16_t)(hi[i] >> 16)));
  }
}

// One lane's part of a slab of a weight row: blocks 4 j + g of it (j = 0 .. 3), and the row's scales
struct WeightSlab {
  u32x4 code[4], scale;
  __device__ void load(const uint8_t* codes, const uint8_t* scales, int slab, int nb, int g) {
    const int block = slab_block(slab, nb) + g;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      code[j] = in_slab(block + 4 * j, slab, nb) ? *reinterpret_cast<const u32x4*>(codes + (int64_t)(block + 4 * j) * 16) : u32x4{};
    scale = slab_scales(scales, slab, nb);
  }
  __device__ float factor(int j, int g) const { return __uint_as_float((scale[j] >> (8 * g) & 255u) << 23); }
};

__device__ __forceinline__ float silu_times(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

// Inner values i0 .. i0 + 15 of the chosen expert blockIdx.y, for its tokens, 16 at a time: lane (r, q) row r of the 16 gate
// and up rows. Four waves split the slabs. Past the inner size, up to whole blocks, zeros.
template <int KIND>
__global__ __launch_bounds__(256) void moe_up(const uint16_t* __restrict__ X, const uint8_t* __restrict__ W,
                                              const uint8_t* __restrict__ S, uint16_t* __restrict__ inner, Routing route,
                                              int64_t H, int I, int pairs) {
  __shared__ f32x4 sums[4][2][64];
  const int a = blockIdx.y;
  if (a >= route.active[0]) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int e = route.active[1 + a], begin = route.offset[a], count = route.offset[a + 1] - begin;
  const int i0 = blockIdx.x * 16, nb = (int)mx_blocks(H), slabs = (nb + SLAB - 1) / SLAB;
  const int64_t pitch = mx_blocks(I) * MX_BLOCK, row = (int64_t)e * 2 * I + min(i0 + r, I - 1);
  const uint8_t *gw = W + row * nb * 16, *uw = W + (row + I) * nb * 16, *gs = S + row * nb, *us = S + (row + I) * nb;
  const int from = slabs * wave / 4, to = slabs * (wave + 1) / 4;
  for (int f = 0; f < count; f += 16) {
    const int at = begin + min(f + r, count - 1), t = route.token[at];
    const float weight = route.weight[at];
    const uint16_t* x = X + (int64_t)t * H;
    f32x4 gate = {}, up = {};
    if (i0 < I) {
      for (int s = from; s < to; ++s) {
        WeightSlab gc, uc;
        gc.load(gw, gs, s, nb, g);
        uc.load(uw, us, s, nb, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float gf = gc.factor(j, g), uf = uc.factor(j, g);
          const int block = slab_block(s, nb) + 4 * j + g;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u32x4 v = in_slab(block, s, nb) ? eight16(x, (int64_t)block * 32 + 8 * q, H) : u32x4{};
            const u32x4 gv = bf16_codes(gc.code[j][q], gf), uv = bf16_codes(uc.code[j][q], uf);
            if constexpr (KIND == BF16) {
              gate = mfma16<BF16>(gv, v, gate), up = mfma16<BF16>(uv, v, up);
            } else {
              u32x4 hi, lo;
              split_f16(v, hi, lo);
              gate = mfma16<BF16>(gv, hi, gate), up = mfma16<BF16>(uv, hi, up);
              gate = mfma16<BF16>(gv, lo, gate), up = mfma16<BF16>(uv, lo, up);
            }
          }
        }
      }
    }
    sums[wave][0][lane] = gate, sums[wave][1][lane] = up;
    __syncthreads();
    if (wave == 0 && f + r < count) {
      gate = (sums[0][0][lane] + sums[1][0][lane]) + (sums[2][0][lane] + sums[3][0][lane]);
      up = (sums[0][1][lane] + sums[1][1][lane]) + (sums[2][1][lane] + sums[3][1][lane]);
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = i0 + 4 * g + q < I ? silu_times(gate[q], up[q]) * weight : 0.0f;
      uint16_t* out = inner + (int64_t)(begin + f + r) * pitch + i0 + 4 * g;
      const uint32_t h0 = f2bf2(v[0], v[1]), h1 = f2bf2(v[2], v[3]);
      *reinterpret_cast<u32x2*>(out) = u32x2{h0, h1};
      if constexpr (KIND == F16) {
        const uint32_t l0 = f2bf2(v[0] - bf2f((uint16_t)h0), v[1] - bf2f((uint16_t)(h0 >> 16)));
        const uint32_t l1 = f2bf2(v[2] - bf2f((uint16_t)h1), v[3] - bf2f((uint16_t)(h1 >> 16)));
        *reinterpret_cast<u32x2*>(out + pairs * pitch) = u32x2{l0, l1};
      }
    }
    __syncthreads();
  }
}

// Outputs n0 .. n0 + 15 of every token: the eight waves split the chosen experts' slabs, each adding an expert's part for
// its tokens into sums of its own, which meet at the end in the order of the waves.
template <int KIND>
__global__ __launch_bounds__(512) void moe_down(const uint16_t* __restrict__ inner, const uint8_t* __restrict__ W,
                                                const uint8_t* __restrict__ S, uint16_t* __restrict__ Y, Routing route,
                                                int T, int64_t H, int I, int pairs) {
  constexpr int WAVES = 8;
  __shared__ f32x4 sums[WAVES][MOE_TOKENS][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  for (int i = lane; i < T * 4; i += 64) sums[wave][i >> 2][i & 3] = f32x4{};
  const int nb = (int)mx_blocks(I), slabs = (nb + SLAB - 1) / SLAB, items = route.active[0] * slabs;
  const int64_t pitch = (int64_t)nb * MX_BLOCK;
  int item = items * wave / WAVES;
  const int end = items * (wave + 1) / WAVES;
  while (item < end) {
    const int a = item / slabs, from = item - a * slabs, to = min(slabs, from + end - item);
    item += to - from;
    const int begin = route.offset[a], count = route.offset[a + 1] - begin;
    const int64_t row = (int64_t)route.active[1 + a] * H + min(n0 + r, H - 1);
    const uint8_t *w = W + row * nb * 16, *sc = S + row * nb;
    for (int f = 0; f < count; f += 16) {
      const int at = begin + min(f + r, count - 1);
      const uint16_t* x = inner + at * pitch;
      f32x4 acc = {};
      for (int s = from; s < to; ++s) {
        WeightSlab c;
        c.load(w, sc, s, nb, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float factor = c.factor(j, g);
          const int block = slab_block(s, nb) + 4 * j + g;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u32x4 v = bf16_codes(c.code[j][q], factor);
            const int64_t from_x = (int64_t)block * 32 + 8 * q;
            acc = mfma16<BF16>(v, in_slab(block, s, nb) ? *reinterpret_cast<const u32x4*>(x + from_x) : u32x4{}, acc);
            if constexpr (KIND == F16)
              acc = mfma16<BF16>(v, in_slab(block, s, nb) ? *reinterpret_cast<const u32x4*>(x + pairs * pitch + from_x) : u32x4{}, acc);
          }
        }
      }
      if (f + r < count) sums[wave][route.token[at]][g] += acc;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < T * 16; i += WAVES * 64) {
    const int t = i >> 4, n = i & 15;
    float v = 0.0f;
#pragma unroll
    for (int s = 0; s < WAVES; ++s) v += reinterpret_cast<const float*>(&sums[s][t][0])[n];
    if (n0 + n < H) Y[(int64_t)t * H + n0 + n] = KIND == BF16 ? f2bf(v) : f2h(v);
  }
}

}  // namespace krn

using namespace krn;

namespace {

struct Layout {  // of the workspace, in bytes
  int parts, steps;
  int64_t partial, active, offset, token, weight, inner, bytes;
};

Layout layout_of(int kind, int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k) {
  Layout w{};
  const int64_t steps = (h + 31) / 32, pairs = t * top_k;
  w.steps = steps <= 256 ? 4 : (int)((steps + 63) / 64);  // of each of a workgroup's four waves
  w.parts = (int)((steps + 4 * w.steps - 1) / (4 * w.steps));
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  w.partial = take(w.parts * t * experts * 4);
  w.active = take((experts + 1) * 4);
  w.offset = take((experts + 1) * 4);
  w.token = take(pairs * 4);
  w.weight = take(pairs * 4);
  w.inner = take(pairs * mx_blocks(i) * MX_BLOCK * 2 * (kind == F16 ? 2 : 1));
  return w;
}

bool moe_sizes(int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k) {
  return t >= 0 && t <= MOE_TOKENS && h >= 1 && h < (int64_t)1 << 24 && i >= 1 && i < (int64_t)1 << 24 && experts >= 1 &&
         experts <= MOE_EXPERTS && top_k >= 1 && top_k <= MOE_TOP_K && top_k <= experts;
}

}  // namespace

template <int KIND>
static int launch_moe(const uint16_t* x, const uint16_t* router, const uint8_t* gate_up, const uint8_t* gate_up_scales,
                      const uint8_t* down, const uint8_t* down_scales, uint16_t* y, int t, int64_t h, int i, int experts,
                      int top_k, uint8_t* ws, hipStream_t stream) {
  const Layout w = layout_of(KIND, t, h, i, experts, top_k);
  const Routing route{(int*)(ws + w.active), (int*)(ws + w.offset), (int*)(ws + w.token), (float*)(ws + w.weight)};
  float* partial = (float*)(ws + w.partial);
  uint16_t* inner = (uint16_t*)(ws + w.inner);
  const int pairs = t * top_k, most = pairs < experts ? pairs : experts;
  hipLaunchKernelGGL((moe_logits<KIND>), dim3((unsigned)((experts + 15) / 16), (unsigned)((t + 15) / 16), (unsigned)w.parts),
                     dim3(256), 0, stream, x, router, partial, t, h, experts, w.steps);
  hipLaunchKernelGGL(moe_route, dim3(1), dim3(1024), 0, stream, partial, w.parts, t, experts, top_k, route);
  hipLaunchKernelGGL((moe_up<KIND>), dim3((unsigned)(mx_blocks(i) * 2), (unsigned)most), dim3(256), 0, stream, x, gate_up,
                     gate_up_scales, inner, route, h, i, pairs);
  hipLaunchKernelGGL((moe_down<KIND>), dim3((unsigned)((h + 15) / 16)), dim3(512), 0, stream, inner, down, down_scales, y, route,
                     t, h, i, pairs);
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("moe launch: %s", hipGetErrorString(err));
  return (int)err;
}

extern "C" {

// See include/krn_amd.h for the contract of each entry point.
int64_t krn_moe_workspace(int kind, int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k) {
  return moe_sizes(t, h, i, experts, top_k) && t > 0 ? layout_of(kind, t, h, i, experts, top_k).bytes : 0;
}

int krn_moe(int kind, const void* x, const void* router, const void* gate_up, const void* gate_up_scales, const void* down,
            const void* down_scales, void* y, int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k, void* workspace,
            int64_t workspace_bytes, void* stream) {
  if (kind != F16 && kind != BF16) {
    krn_set_error("moe: element kind %d; f16 or bf16 tokens are taken", kind);
    return -1;
  }
  if (!moe_sizes(t, h, i, experts, top_k)) {
    krn_set_error("moe: %lld tokens of %lld, %lld inner values, %lld of %lld experts; at most %d tokens, %d experts and %d of "
                  "them for a token, sizes of 1 to 2^24 - 1", (long long)t, (long long)h, (long long)i, (long long)top_k,
                  (long long)experts, MOE_TOKENS, MOE_EXPERTS, MOE_TOP_K);
    return -1;
  }
  if (t == 0) return 0;
  if ((uintptr_t)gate_up % 16 != 0 || (uintptr_t)down % 16 != 0 || (uintptr_t)workspace % 16 != 0) {
    krn_set_error("moe: codes and workspace start at 16-byte aligned addresses");
    return -1;
  }
  const Layout w = layout_of(kind, t, h, i, experts, top_k);
  if (workspace == nullptr || workspace_bytes < w.bytes) {
    krn_set_error("moe: a workspace of %lld bytes is needed", (long long)w.bytes);
    return -1;
  }
  const int64_t nb_h = mx_blocks(h), nb_i = mx_blocks(i), up_rows = experts * 2 * i, down_rows = experts * h;
  const struct { const void* p; int64_t bytes; } inputs[] = {
      {x, t * h * 2}, {router, experts * h * 2}, {gate_up, up_rows * nb_h * 16}, {gate_up_scales, up_rows * nb_h},
      {down, down_rows * nb_i * 16}, {down_scales, down_rows * nb_i}};
  for (const auto& in : inputs)
    if (share_memory(y, t * h * 2, in.p, in.bytes)) {
      krn_set_error("moe: the result shares memory with an input");
      return -1;
    }
  auto go = kind == BF16 ? launch_moe<BF16> : launch_moe<F16>;
  return go((const uint16_t*)x, (const uint16_t*)router, (const uint8_t*)gate_up, (const uint8_t*)gate_up_scales,
            (const uint8_t*)down, (const uint8_t*)down_scales, (uint16_t*)y, (int)t, h, (int)i, (int)experts, (int)top_k,
            (uint8_t*)workspace, (hipStream_t)stream);
}

}  // extern "C"
