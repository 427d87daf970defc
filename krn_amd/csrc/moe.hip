// A mixture-of-experts layer for a few tokens on gfx950, experts in microscaled 4 bits (mx_parts.h):
//   y_t = sum over the top_k experts e of token t of  w_te * down_e (silu(gate_e x_t) * up_e x_t),
// w_t the softmax of the chosen experts' router logits x_t . router_e. Ties go to the expert of the lower index; a NaN logit
// counts as the largest.
//
// Bound by reading the chosen experts' weights, each once whatever the number of its tokens (up to 16). The launches:
//   logits  x router^T in 16-bit MFMAs (products exact, float32 sums), in parts of K
//   route   one workgroup: a wave chooses a token's experts; every expert's tokens as a 64-bit mask, so that its count and a
//           token's place in it are population counts and no order of atomics shows; the chosen experts in a row
//   up      16 inner values of a chosen expert a wave: gate and up rows, w silu(gate) up to memory
//   down    256 outputs a workgroup: all chosen experts' rows, added per token, in parts
//   sum     the parts, in their order
// One or two tokens, which wait for launches more than for memory, have no second one: every workgroup of `up` routes for
// itself (of 64 experts 4096 x 2048, us: 1 token 28.6 -> 26.0, 2 tokens 45.0 -> 42.6; but 4 tokens 68.8 -> 73.1, where
// more workgroups do it one after the other). The sum stays a launch of its own (2.6 us): with the last workgroup at its
// outputs adding the parts up, the fence between them took `down` from 8 us to 18.
// Weights go to bf16 exactly (v_cvt_scalef32_pk_bf16_fp4: two bits of mantissa and a power of two) and are multiplied in
// 16x16x32 bf16 MFMAs, 16 weight rows by up to 16 tokens. bfloat16 tokens are taken as they are; float16 tokens are split
// into the nearest bf16 and the bf16 of what is left, which holds all of a float16. The inner values are handed on as two
// such parts for both types, 2^-16 relative: one bf16 would add as much error as the result's own rounding (1 token of
// 4096: 2.4e-3 against 1.7e-3), and the second MFMA hides behind the weights' way from memory.
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

// Logits of 16 experts and 16 tokens over one of PARTS runs of K (blockIdx.z), which its four waves split again
constexpr int PARTS = 8;
template <int KIND>
__global__ __launch_bounds__(256) void moe_logits(const uint16_t* __restrict__ X, const uint16_t* __restrict__ router,
                                                  float* __restrict__ partial, int T, int64_t H, int E) {
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16, run = blockIdx.z * 4 + wave;
  const uint16_t* w = router + (int64_t)min(e0 + r, E - 1) * H + 8 * g;
  const uint16_t* x = X + (int64_t)min(t0 + r, T - 1) * H + 8 * g;
  f32x4 acc = {};
  const int steps = (int)((H + 31) / 32), whole = (int)(H / 32);
  const int to = (int)((int64_t)steps * (run + 1) / (4 * PARTS));
  int s = (int)((int64_t)steps * run / (4 * PARTS));
  for (; s + 4 <= min(to, whole); s += 4) {
    u32x4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = *reinterpret_cast<const u32x4_any*>(w + (s + i) * 32);
      b[i] = *reinterpret_cast<const u32x4_any*>(x + (s + i) * 32);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = mfma16<KIND>(a[i], b[i], acc);
  }
  for (; s < to; ++s) acc = mfma16<KIND>(eight16(w, s * 32, H - 8 * g), eight16(x, s * 32, H - 8 * g), acc);
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && t0 + r < T) {
    const f32x4 v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (e0 + 4 * g + q < E) partial[((int64_t)blockIdx.z * T + t0 + r) * E + e0 + 4 * g + q] = v[q];
  }
}

// The largest (smallest) of a wave's values, in every lane: four DPP steps within 16 lanes, then the four rows' results
template <bool MAX>
__device__ __forceinline__ uint32_t wave_extreme(uint32_t v) {
  auto pick = [](uint32_t a, uint32_t b) { return MAX ? max(a, b) : min(a, b); };
  v = pick(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  v = pick(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));   // lane ^ 2
  v = pick(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));  // half row mirrored
  v = pick(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));  // row mirrored
  return pick(pick((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
              pick((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

// A float32 as an unsigned number in the same order, never 0; NaN above everything
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The experts of token t, by one wave: lane j < top_k gets choice j and its weight. EPL: experts a lane. WAVES16: one of sixteen
// waves, whose 128 registers do not hold all loads of sixteen experts (67 spilled: 64 tokens, 8 of 1024 experts 170 -> 84 us
// for the layer); one of eight has room for them (2 tokens, 16 of 1024 29.1, 32 loads at a time 29.8)
template <int EPL, bool WAVES16>
__device__ __forceinline__ void choose(const float* __restrict__ partial, int t, int T, int E, int top_k, int lane, int& pick,
                                       float& weight) {
  uint32_t key[EPL];  // expert lane + 64 i, 0 once chosen and past the last
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 64 * i;
    float v[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) v[p] = partial[((int64_t)p * T + t) * E + min(e, E - 1)];
    float sum = v[0];
#pragma unroll
    for (int p = 1; p < PARTS; ++p) sum += v[p];
    key[i] = e < E ? ordered(sum) : 0;
    if (WAVES16 && EPL > 4 && i % 4 == 3)  // 32 loads at a time, the address of the next after their sums
      asm volatile("" : "+s"(partial) : "v"(key[i]), "v"(key[i - 1]), "v"(key[i - 2]), "v"(key[i - 3]));
  }
  float mine = -INFINITY;  // lane j: the logit of choice j
  pick = 0;
  for (int j = 0; j < top_k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) best = max(best, key[i]);
    best = wave_extreme<true>(best);
    uint32_t e = MOE_EXPERTS;  // the lowest expert with that logit
#pragma unroll
    for (int i = EPL - 1; i >= 0; --i) e = key[i] == best ? lane + 64 * i : e;
    e = wave_extreme<false>(e);
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = lane + 64 * i == (int)e ? 0 : key[i];
    if (lane == j) mine = __uint_as_float(best & 0x80000000u ? best ^ 0x80000000u : ~best), pick = (int)e;
  }
  const float top = __shfl(mine, 0);
  const float p = lane < top_k ? expf(mine - top) : 0.0f;
  float sum = p;
#pragma unroll
  for (int d = 1; d < 16; d *= 2) sum += __shfl_xor(sum, d);
  weight = p / sum;
}

template <int EPL>
__global__ __launch_bounds__(1024) void moe_route(const float* __restrict__ partial, int T, int E, int top_k, Routing out) {
  __shared__ unsigned long long mask[MOE_EXPERTS];
  __shared__ uint32_t base[MOE_EXPERTS], wave_sum[16];
  __shared__ int chosen[MOE_TOKENS * MOE_TOP_K];
  __shared__ float weight[MOE_TOKENS * MOE_TOP_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  mask[threadIdx.x] = 0;
  __syncthreads();
  for (int t = wave; t < T; t += 16) {
    int pick;
    float w;
    choose<EPL, true>(partial, t, T, E, top_k, lane, pick, w);
    if (lane < top_k) {
      chosen[t * top_k + lane] = pick, weight[t * top_k + lane] = w;
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

// The routing of up to FEW tokens by one workgroup, in its LDS: a pair (token, choice) finds its place by counting the pairs of
// lower experts and the earlier ones of its own
constexpr int FEW = 2, FEW_PAIRS = FEW * MOE_TOP_K;
struct FewRouting {
  int active[FEW_PAIRS + 1], offset[FEW_PAIRS + 1], token[FEW_PAIRS], chosen[FEW_PAIRS];
  float weight[FEW_PAIRS], given[FEW_PAIRS];
  bool first[FEW_PAIRS];
};

template <int EPL>
__device__ __forceinline__ void route_few(FewRouting& out, const float* __restrict__ partial, int T, int E, int top_k) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = threadIdx.x, pairs = T * top_k;
  if (wave < T) {
    int pick;
    float w;
    choose<EPL, false>(partial, wave, T, E, top_k, lane, pick, w);
    if (lane < top_k) out.chosen[wave * top_k + lane] = pick, out.given[wave * top_k + lane] = w;
  }
  __syncthreads();
  int below = 0, before = 0;
  const int e = i < pairs ? out.chosen[i] : 0;
  if (i < pairs) {
    for (int j = 0; j < pairs; ++j) below += out.chosen[j] < e, before += j < i && out.chosen[j] == e;
    out.first[i] = before == 0;
    out.token[below + before] = i / top_k, out.weight[below + before] = out.given[i];
  }
  __syncthreads();
  if (i < pairs && before == 0) {
    int rank = 0;
    for (int j = 0; j < pairs; ++j) rank += out.first[j] && out.chosen[j] < e;
    out.active[1 + rank] = e, out.offset[rank] = below;
  }
  if (i == 0) {
    int active = 0;
    for (int j = 0; j < pairs; ++j) active += out.first[j];
    out.active[0] = active, out.offset[active] = pairs;
  }
  __syncthreads();
}

// Eight codes of a block as bf16 values
__device__ __forceinline__ u32x4 bf16_codes(uint32_t w, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
               __builtin_bit_cast(uint32_t, d)};
}

// What is left of a value when its bf16 is taken away; nothing of one that is, or becomes, infinite
__device__ __forceinline__ float rest(float v, uint16_t bf) {
  const float h = bf2f(bf);
  return __builtin_isinf(h) ? 0.0f : v - h;
}

// Eight float16 values as the bf16 nearest to each and the bf16 of what is left (exact: 11 bits in two times 8)
__device__ __forceinline__ void split_f16(const u32x4& x, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = h2f((uint16_t)x[i]), b = h2f((uint16_t)(x[i] >> 16));
    hi[i] = f2bf2(a, b);
    lo[i] = f2bf2(rest(a, (uint16_t)hi[i]), rest(b, (uint16_t)(hi[i] >> 16)));
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

// Tokens' values for one slab in LDS, where the waves take their MFMA operands from: a row of 512 values is 1024 bytes, and
// rows lie 1040 apart, so that the 16 rows a read touches are on different banks. A token's slab is one access of
// a wave to memory; as operands straight from memory it would be 16, whatever the number of tokens, and the address
// path would bound the kernel (down, 16 tokens of 4: 127 us).
constexpr int STAGED_ROW = 1040;

// Operand (j, q) of lane (r, g): values 8 q .. + 7 of block 4 j + g of the slab, of row min(r, rows - 1)
__device__ __forceinline__ u32x4 staged(const uint8_t* slab, int row, int j, int q, int g) {
  return *reinterpret_cast<const u32x4*>(slab + row * STAGED_ROW + (4 * j + g) * 64 + q * 16);
}

// Inner values of the chosen expert blockIdx.y for its tokens, `rows` (at most 16) at a time. Eight waves: `kparts` of them
// split the slabs of 16 gate and 16 up rows, so that a workgroup has 8 / kparts times 16 inner values. Past the
// inner size, up to whole blocks, zeros. Dynamic LDS: kparts slabs of `rows` tokens (float16: of both parts).
// EPL > 0: of up to FEW tokens, whose routing the workgroup does itself, the first one for `down` as well.
template <int KIND, int EPL>
__global__ __launch_bounds__(512) void moe_up(const uint16_t* __restrict__ X, const uint8_t* __restrict__ W,
                                              const uint8_t* __restrict__ S, uint16_t* __restrict__ inner, Routing given,
                                              int64_t H, int I, int pairs, int kparts, int rows,
                                              const float* __restrict__ partial, int T, int E, int top_k) {
  constexpr int PLANES = KIND == F16 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t tokens[];
  __shared__ f32x4 sums[8][2][64];
  __shared__ FewRouting few;
  Routing route = given;
  if constexpr (EPL > 0) {
    route_few<EPL>(few, partial, T, E, top_k);
    route = Routing{few.active, few.offset, few.token, few.weight};
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x <= pairs) {
      const int i = threadIdx.x, active = few.active[0];
      if (i <= active) given.active[i] = few.active[i], given.offset[i] = few.offset[i];
      if (i < pairs) given.token[i] = few.token[i], given.weight[i] = few.weight[i];
    }
  }
  const int a = blockIdx.y;
  if (a >= route.active[0]) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int e = route.active[1 + a], begin = route.offset[a], count = route.offset[a + 1] - begin;
  const int part = wave % kparts, i0 = (blockIdx.x * (8 / kparts) + wave / kparts) * 16;
  const int nb = (int)mx_blocks(H), slabs = (nb + SLAB - 1) / SLAB;
  const int64_t pitch = mx_blocks(I) * MX_BLOCK, row = (int64_t)e * 2 * I + min(i0 + r, I - 1);
  const uint8_t *gw = W + row * nb * 16, *uw = W + (row + I) * nb * 16, *gs = S + row * nb, *us = S + (row + I) * nb;
  const int plane = kparts * rows * STAGED_ROW;
  const uint8_t* mine = tokens + part * rows * STAGED_ROW;
  for (int f = 0; f < count; f += rows) {
    const int here = min(count - f, rows), own = min(r, here - 1);
    f32x4 gate = {}, up = {};
    for (int from = 0; from < slabs; from += kparts) {
      const int slab = from + part;
      const bool work = slab < slabs && i0 < I;
      WeightSlab gc, uc;
      if (work) gc.load(gw, gs, slab, nb, g), uc.load(uw, us, slab, nb, g);
      if (from > 0 || f > 0) __syncthreads();  // the tokens before have been read
      for (int i = wave; i < here * kparts; i += 8) {
        const int s = from + i % kparts, t = i / kparts, block = slab_block(s, nb) + (lane >> 2);
        if (s >= slabs) continue;
        const u32x4 v = in_slab(block, s, nb) ? eight16(X + (int64_t)route.token[begin + f + t] * H,
                                                        (int64_t)block * 32 + 8 * (lane & 3), H)
                                              : u32x4{};
        uint8_t* to = tokens + ((i % kparts) * rows + t) * STAGED_ROW + lane * 16;
        if constexpr (KIND == F16) {
          u32x4 hi, lo;
          split_f16(v, hi, lo);
          *reinterpret_cast<u32x4*>(to) = hi, *reinterpret_cast<u32x4*>(to + plane) = lo;
        } else {
          *reinterpret_cast<u32x4*>(to) = v;
        }
      }
      __syncthreads();
      if (!work) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float gf = gc.factor(j, g), uf = uc.factor(j, g);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x4 gv = bf16_codes(gc.code[j][q], gf), uv = bf16_codes(uc.code[j][q], uf);
#pragma unroll
          for (int p = 0; p < PLANES; ++p) {
            const u32x4 v = staged(mine + p * plane, own, j, q, g);
            gate = mfma16<BF16>(gv, v, gate), up = mfma16<BF16>(uv, v, up);
          }
        }
        __builtin_amdgcn_sched_barrier(0);  // operands of one step at a time in registers, not of all four
      }
    }
    sums[wave][0][lane] = gate, sums[wave][1][lane] = up;
    __syncthreads();
    if (part == 0 && r < here && i0 < pitch) {
      for (int p = 1; p < kparts; ++p) gate += sums[wave + p][0][lane], up += sums[wave + p][1][lane];
      const float weight = route.weight[begin + f + r];
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = i0 + 4 * g + q < I ? silu_times(gate[q], up[q]) * weight : 0.0f;
      uint16_t* out = inner + (int64_t)(begin + f + r) * pitch + i0 + 4 * g;
      const uint32_t h0 = f2bf2(v[0], v[1]), h1 = f2bf2(v[2], v[3]);
      const uint32_t l0 = f2bf2(rest(v[0], (uint16_t)h0), rest(v[1], (uint16_t)(h0 >> 16)));
      const uint32_t l1 = f2bf2(rest(v[2], (uint16_t)h1), rest(v[3], (uint16_t)(h1 >> 16)));
      *reinterpret_cast<u32x2*>(out) = u32x2{h0, h1};
      *reinterpret_cast<u32x2*>(out + pairs * pitch) = u32x2{l0, l1};
    }
  }
}

// Outputs n0 .. n0 + 255 of every token over part blockIdx.y of the chosen experts' slabs: each of the eight waves has 32
// weight rows and goes through all of the part. The waves share the tokens' inner values in LDS, `rows` tokens (at
// most 16) a step, in two places in turn; a step's inner values and a slab's weights are on their way while the step
// before is multiplied. An expert's part goes to its tokens' sums, which only the wave with those rows touches.
// Dynamic LDS: two places of `rows` tokens in two parts, then the sums of T tokens.
__global__ __launch_bounds__(512) void moe_down(const uint16_t* __restrict__ inner, const uint8_t* __restrict__ W,
                                                const uint8_t* __restrict__ S, float* __restrict__ partial, Routing route,
                                                int T, int64_t H, int I, int pairs, int rows) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tokens[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int plane = rows * STAGED_ROW;
  f32x4* sums = reinterpret_cast<f32x4*>(tokens + 4 * plane) + wave * 8;  // [token][64], this wave's eight
  const int64_t n0 = (int64_t)blockIdx.x * 256 + wave * 32;
  for (int i = lane; i < T * 8; i += 64) sums[(i >> 3) * 64 + (i & 7)] = f32x4{};
  const int nb = (int)mx_blocks(I), slabs = (nb + SLAB - 1) / SLAB, items = route.active[0] * slabs;
  const int64_t pitch = (int64_t)nb * MX_BLOCK;
  const int first = (int)((int64_t)items * blockIdx.y / gridDim.y), end = (int)((int64_t)items * (blockIdx.y + 1) / gridDim.y);
  struct Step {  // tokens f .. of the expert of item `item`, `begin` .. `begin + count` among the pairs
    int item, slab, f, begin, count, expert;
  };
  auto at_item = [&](int item) {
    const int a = item / slabs, begin = route.offset[a];
    return Step{item, item - a * slabs, 0, begin, route.offset[a + 1] - begin, route.active[1 + a]};
  };
  auto load = [&](WeightSlab (&w)[2], const Step& s) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = ((int64_t)s.expert * H + min(n0 + 16 * i + r, H - 1)) * nb;
      w[i].load(W + at * 16, S + at, s.slab, nb, g);
    }
  };
  // row i of a step: token i / 2, part i % 2; this wave's rows are wave, wave + 8, ...
  auto fetch = [&](u32x4 (&v)[4], const Step& s) {
    const int block = slab_block(s.slab, nb) + (lane >> 2), here = min(s.count - s.f, rows);
    const bool in = in_slab(block, s.slab, nb);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = wave + 8 * k;
      v[k] = u32x4{};
      if (i < 2 * here && in)
        v[k] = *reinterpret_cast<const u32x4*>(inner + ((i & 1) * pairs + s.begin + s.f + (i >> 1)) * pitch +
                                               (int64_t)block * 32 + 8 * (lane & 3));
    }
  };
  auto put = [&](const u32x4 (&v)[4], uint8_t* place, const Step& s) {
    const int here = min(s.count - s.f, rows);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = wave + 8 * k;
      if (i < 2 * here) *reinterpret_cast<u32x4*>(place + (i & 1) * plane + (i >> 1) * STAGED_ROW + lane * 16) = v[k];
    }
  };
  if (first < end) {
    Step step = at_item(first);
    WeightSlab now[2];
    u32x4 v[4];
    load(now, step);
    fetch(v, step);
    put(v, tokens, step);
    for (int place = 0;; place ^= 1) {
      __syncthreads();  // the step's values are there, and every wave is done with the other place
      Step next = step;
      next.f += rows;
      const bool new_item = next.f >= step.count, more = !new_item || step.item + 1 < end;
      if (new_item) next = at_item(min(step.item + 1, end - 1));
      WeightSlab after[2];
      load(after, next);  // the same again within an item: from the cache, and no branch around loads in flight
      if (more) fetch(v, next);
      const uint8_t* at = tokens + place * 2 * plane;
      const int here = min(step.count - step.f, rows), own = min(r, here - 1);
      f32x4 acc[2] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f0 = now[0].factor(j, g), f1 = now[1].factor(j, g);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x4 v0 = bf16_codes(now[0].code[j][q], f0), v1 = bf16_codes(now[1].code[j][q], f1);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const u32x4 x = staged(at + p * plane, own, j, q, g);
            acc[0] = mfma16<BF16>(v0, x, acc[0]), acc[1] = mfma16<BF16>(v1, x, acc[1]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (r < here) {
        f32x4* sum = sums + route.token[step.begin + step.f + r] * 64 + g;
        sum[0] += acc[0], sum[4] += acc[1];
      }
      if (!more) break;
      put(v, tokens + (place ^ 1) * 2 * plane, next);
      now[0] = after[0], now[1] = after[1];
      step = next;
    }
  }
  for (int i = lane; i < T * 8; i += 64) {
    const int t = i >> 3;
    const f32x4 v = sums[t * 64 + (i & 7)];
    float* out = partial + ((int64_t)blockIdx.y * T + t) * H + n0 + 4 * (i & 7);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n0 + 4 * (i & 7) + q < H) out[q] = v[q];
  }
}

// y = the sum of the parts, in their order
template <int KIND>
__global__ __launch_bounds__(256) void moe_sum(const float* __restrict__ partial, uint16_t* __restrict__ Y, int64_t values,
                                               int parts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= values) return;
  float v = 0.0f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) v += partial[p * values + i];
  Y[i] = KIND == BF16 ? f2bf(v) : f2h(v);
}

}  // namespace krn

using namespace krn;

namespace {

struct Layout {  // of the workspace, in bytes
  int parts;  // of the down products, so that their workgroups fill the chip
  int64_t logits, active, offset, token, weight, inner, partial, bytes;
};

Layout layout_of(int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k) {
  Layout w{};
  const int64_t pairs = t * top_k, most = pairs < experts ? pairs : experts, blocks = (h + 255) / 256;
  const int64_t items = most * ((mx_blocks(i) + SLAB - 1) / SLAB), fill = (256 + blocks - 1) / blocks;
  w.parts = (int)(items < fill ? items : fill);
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  w.logits = take(PARTS * t * experts * 4);
  w.active = take((experts + 1) * 4);
  w.offset = take((experts + 1) * 4);
  w.token = take(pairs * 4);
  w.weight = take(pairs * 4);
  w.inner = take(pairs * mx_blocks(i) * MX_BLOCK * 4);
  w.partial = take(w.parts * t * h * 4);
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
  const Layout w = layout_of(t, h, i, experts, top_k);
  const Routing route{(int*)(ws + w.active), (int*)(ws + w.offset), (int*)(ws + w.token), (float*)(ws + w.weight)};
  float* logits = (float*)(ws + w.logits);
  uint16_t* inner = (uint16_t*)(ws + w.inner);
  const int pairs = t * top_k, most = pairs < experts ? pairs : experts;
  const int64_t slabs = (mx_blocks(h) + SLAB - 1) / SLAB;
  float* partial = (float*)(ws + w.partial);
  const bool few = t <= FEW;
  // tokens gone through at a time: room for twice an expert's average, so that few experts are read twice for the rest
  int rows = 4;
  while (rows < 16 && rows < t && rows * experts < 2 * pairs) rows *= 2;
  rows = rows < t ? rows : t;
  // as many waves to a row's slabs as these leave LDS for two workgroups on a CU, and no more than there are slabs
  int kparts = 8;
  while (kparts > 1 && (kparts > slabs || kparts * rows * STAGED_ROW * (KIND == F16 ? 2 : 1) > 56 * 1024)) kparts /= 2;
  hipLaunchKernelGGL((moe_logits<KIND>), dim3((unsigned)((experts + 15) / 16), (unsigned)((t + 15) / 16), PARTS), dim3(256), 0,
                     stream, x, router, logits, t, h, experts);
  if (!few) {
    auto choose = experts <= 64 ? moe_route<1> : experts <= 256 ? moe_route<4> : moe_route<16>;
    hipLaunchKernelGGL(choose, dim3(1), dim3(1024), 0, stream, logits, t, experts, top_k, route);
  }
  auto up = !few ? moe_up<KIND, 0> : experts <= 64 ? moe_up<KIND, 1> : experts <= 256 ? moe_up<KIND, 4> : moe_up<KIND, 16>;
  hipLaunchKernelGGL(up, dim3((unsigned)((mx_blocks(i) * 2 * kparts + 7) / 8), (unsigned)most), dim3(512),
                     (unsigned)(kparts * rows * STAGED_ROW * (KIND == F16 ? 2 : 1)), stream, x, gate_up, gate_up_scales, inner,
                     route, h, i, pairs, kparts, rows, logits, t, experts, top_k);
  hipLaunchKernelGGL(moe_down, dim3((unsigned)((h + 255) / 256), (unsigned)w.parts), dim3(512),
                     (unsigned)(4 * rows * STAGED_ROW + t * 1024), stream, inner, down, down_scales, partial, route, t, h, i, pairs,
                     rows);
  hipLaunchKernelGGL((moe_sum<KIND>), dim3((unsigned)((t * h + 255) / 256)), dim3(256), 0, stream, partial, y, t * h, w.parts);
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("moe launch: %s", hipGetErrorString(err));
  return (int)err;
}

extern "C" {

// See include/krn_amd.h for the contract of each entry point.
int64_t krn_moe_workspace(int kind, int64_t t, int64_t h, int64_t i, int64_t experts, int64_t top_k) {
  return moe_sizes(t, h, i, experts, top_k) && t > 0 ? layout_of(t, h, i, experts, top_k).bytes : 0;
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
  const Layout w = layout_of(t, h, i, experts, top_k);
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
