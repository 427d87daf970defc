// Products of microscaled 4-bit matrices for gfx950: C[m, n] = epilogue(sum_k A[m, k] * B[n, k]), both operands K-contiguous
// (the format and the order in which K is taken: mx_parts.h). v_mfma_scale_f32_16x16x128_f8f6f4 multiplies the codes and
// applies both blocks' scales, so the operands stay in 4 bits until the matrix core; sums are float32 and every result is
// rounded once. Every kernel computes blocks transposed (B A^T), so that a lane holds four neighbouring columns of one row.
#include "gemm_split.h"
#include "mx_parts.h"

namespace krn {

struct MxCall {
  const uint8_t *a, *as, *b, *bs;
  void* c;
  int64_t m, n;
  int nb;
  int64_t ldc;
  Epilogue e;
  hipStream_t stream;
};

typedef u32x2 u32x2_any __attribute__((aligned(1)));  // an 8-byte access at any address

// Columns n .. n + 3 of row m through the epilogue, each operation rounded to float32, and to C
__device__ __forceinline__ void store4(const Epilogue& e, f32x4 x, void* C, int64_t ldc, int64_t m, int64_t n, int64_t M,
                                       int64_t N) {
  if (m >= M || n >= N) return;
  float v[4] = {x[0], x[1], x[2], x[3]};
  for (int i = 0; i < e.nops; ++i) {
    const int op = e.op[i] & ((1 << VEC_KIND_SHIFT) - 1), kind = e.op[i] >> VEC_KIND_SHIFT;
    if (op >= RELU) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = activation(op, v[c]);
      continue;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float s = op % 3 == 0 ? e.scalar[i] : bits_value(kind, vec_bits(e.vec[i], kind, op % 3 == 1 ? m : min(n + c, N - 1)));
      v[c] = op < 3 ? __fmul_rn(v[c], s) : __fadd_rn(v[c], s);
    }
  }
  if (e.out_kind == F32) {
    float* out = static_cast<float*>(C) + m * ldc + n;
    if (n + 4 <= N) {
      *reinterpret_cast<u32x4_any*>(out) = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (n + c < N) out[c] = v[c];
    }
    return;
  }
  const uint32_t lo = e.out_kind == BF16 ? f2bf2(v[0], v[1]) : (uint32_t)f2h(v[0]) | (uint32_t)f2h(v[1]) << 16;
  const uint32_t hi = e.out_kind == BF16 ? f2bf2(v[2], v[3]) : (uint32_t)f2h(v[2]) | (uint32_t)f2h(v[3]) << 16;
  uint16_t* out = static_cast<uint16_t*>(C) + m * ldc + n;
  if (n + 4 <= N) {
    *reinterpret_cast<u32x2_any*>(out) = u32x2{lo, hi};
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < N) out[c] = (uint16_t)((c < 2 ? lo : hi) >> ((c & 1) * 16));
  }
}

// Few rows (M <= 16 MT), bound by reading B once. A workgroup owns 16 NT columns and all rows; its waves split K into
// runs of slabs. Operands go from memory straight to registers: step j of a slab reads 64 consecutive bytes of each of 16
// rows, lane (r, g) the 16 that the MFMA takes from it. Rows past the end of A or B read the last row: their results are
// not stored. The waves' sums meet in LDS, in the order of the waves.
template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mx_few(const uint8_t* __restrict__ A, const uint8_t* __restrict__ AS,
                                                     const uint8_t* __restrict__ B, const uint8_t* __restrict__ BS,
                                                     void* __restrict__ C, int64_t M, int64_t N, int nb, int64_t ldc,
                                                     Epilogue e) {
  __shared__ f32x4 sums[WAVES][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  const uint8_t *a[MT], *as[MT], *b[NT], *bs[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t row = min((int64_t)(16 * t + r), M - 1);
    a[t] = A + row * nb * 16 + g * 16, as[t] = AS + row * nb;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = min(n0 + 16 * t + r, N - 1);
    b[t] = B + row * nb * 16 + g * 16, bs[t] = BS + row * nb;
  }
  const int slabs = (nb + SLAB - 1) / SLAB;
  const int from = (int)((int64_t)slabs * wave / WAVES), to = (int)((int64_t)slabs * (wave + 1) / WAVES);
  f32x4 acc[MT][NT] = {};
  for (int s = from; s < to; ++s) {
    const int block = s * SLAB;
    const int64_t at = (int64_t)block * 16;
    u32x4 x[MT][4], y[NT][4];
    uint32_t sx[MT], sy[NT];
    if (block + SLAB <= nb) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int t = 0; t < NT; ++t) y[t][j] = *reinterpret_cast<const u32x4*>(b[t] + at + 64 * j);
#pragma unroll
        for (int t = 0; t < MT; ++t) x[t][j] = *reinterpret_cast<const u32x4*>(a[t] + at + 64 * j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = block + 4 * j + g < nb;
#pragma unroll
        for (int t = 0; t < NT; ++t) y[t][j] = in ? *reinterpret_cast<const u32x4*>(b[t] + at + 64 * j) : u32x4{};
#pragma unroll
        for (int t = 0; t < MT; ++t) x[t][j] = in ? *reinterpret_cast<const u32x4*>(a[t] + at + 64 * j) : u32x4{};
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) sy[t] = scale_bytes(slab_scales(bs[t], block, nb), g);
#pragma unroll
    for (int t = 0; t < MT; ++t) sx[t] = scale_bytes(slab_scales(as[t], block, nb), g);
#define KRN_STEP(J)                                                                                                  \
  _Pragma("unroll") for (int t = 0; t < MT; ++t) _Pragma("unroll") for (int u = 0; u < NT; ++u) acc[t][u] =          \
      mx_mfma<J>(y[u][J], x[t][J], acc[t][u], sy[u], sx[t]);
    KRN_STEP(0) KRN_STEP(1) KRN_STEP(2) KRN_STEP(3)
#undef KRN_STEP
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) sums[wave][t * NT + u][lane] = acc[t][u];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += WAVES) {
    f32x4 v = sums[0][f][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += sums[w][f][lane];
    store4(e, v, C, ldc, 16 * (f / NT) + r, n0 + 16 * (f % NT) + 4 * g, M, N);
  }
}

// The scale words of four 16-row blocks for one slab: lane 16 f + r brings row r of block f's 16 scales (slab_scales), and
// lane (r, g) gets, for each block, byte g of its row's four words packed into one. First the bytes within a lane, then
// the words between the four lane groups (two permlane swaps a word).
__device__ __forceinline__ void spread_scales(const u32x4& d, uint32_t (&out)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400), t1 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602);
  const uint32_t t2 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400), t3 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602);
  const uint32_t o0 = __builtin_amdgcn_perm(t2, t0, 0x05040100), o1 = __builtin_amdgcn_perm(t2, t0, 0x07060302);
  const uint32_t o2 = __builtin_amdgcn_perm(t3, t1, 0x05040100), o3 = __builtin_amdgcn_perm(t3, t1, 0x07060302);
  const auto p01 = __builtin_amdgcn_permlane16_swap(o0, o1, false, false);
  const auto p23 = __builtin_amdgcn_permlane16_swap(o2, o3, false, false);
  const auto q02 = __builtin_amdgcn_permlane32_swap(p01[0], p23[0], false, false);
  const auto q13 = __builtin_amdgcn_permlane32_swap(p01[1], p23[1], false, false);
  out[0] = q02[0], out[2] = q02[1], out[1] = q13[0], out[3] = q13[1];
}

// Tiles of 32 TM x 32 TN, four waves of 16 TM x 16 TN each. Slices of 128 bytes a row (half a slab) go from memory
// straight into a ring of LDS stages, chunk c of row r at slot c ^ ((r >> 1) & 7), STAGES - 1 slices ahead; one barrier
// a slice publishes the landed one and frees the oldest. Past the end of a row, and of the matrix, the buffer loads give
// zeros. Scales go to registers, a slab ahead.
template <int TM, int TN, int STAGES>
__global__ __launch_bounds__(256) void mx_tile(const uint8_t* __restrict__ A, const uint8_t* __restrict__ AS,
                                               const uint8_t* __restrict__ B, const uint8_t* __restrict__ BS,
                                               void* __restrict__ C, int64_t M, int64_t N, int nb, int64_t ldc, Epilogue e) {
  static_assert(TM <= 4 && TN <= 4, "a wave's scales are one row a lane");
  constexpr int BM = 32 * TM, BN = 32 * TN, STAGE = (BM + BN) * 128;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES][STAGE];
  int tm, tn;
  tile_of((int)((M + BM - 1) / BM), (int)((N + BN - 1) / BN), tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  const int64_t ld = (int64_t)nb * 16;
  auto uniform = [](const void* p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const void*)(((uint64_t)hi << 32) | (uint64_t)lo);
  };
  const __amdgpu_buffer_rsrc_t a_rsrc = panel_rsrc(uniform(A + m0 * ld), (M - m0) * ld),
                               b_rsrc = panel_rsrc(uniform(B + n0 * ld), (N - n0) * ld);
  // load item j: rows 8 TM wave + 8 j .. + 7 of A (TN: of B), lane i row i / 8 and the chunk that belongs at slot i % 8
  uint32_t ga[TM], gb[TN];
  int ca[TM], cb[TN];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int row = wave * (8 * TM) + 8 * j + (lane >> 3);
    ca[j] = (lane & 7) ^ swz8(row), ga[j] = (uint32_t)(row * ld + ca[j] * 16);
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int row = wave * (8 * TN) + 8 * j + (lane >> 3);
    cb[j] = (lane & 7) ^ swz8(row), gb[j] = (uint32_t)(row * ld + cb[j] * 16);
  }
  const int slabs = (nb + SLAB - 1) / SLAB, slices = 2 * slabs;
  auto issue = [&](int slice, int stage) {
    uint8_t* la = ring[stage] + wave * (8 * TM * 128);
    uint8_t* lb = ring[stage] + BM * 128 + wave * (8 * TN * 128);
    const int left = nb - slice * 8;  // blocks of the row from this slice on
#pragma unroll
    for (int j = 0; j < TM; ++j) buffer_to_lds16(a_rsrc, la + j * 1024, ca[j] < left ? ga[j] : 0x80000000u, slice * 128);
#pragma unroll
    for (int j = 0; j < TN; ++j) buffer_to_lds16(b_rsrc, lb + j * 1024, cb[j] < left ? gb[j] : 0x80000000u, slice * 128);
  };
  // the row whose scales this lane brings: of the wave's 16 TM (TN) rows, row lane % (16 TM)
  const uint8_t* as = AS + min(m0 + wm * (16 * TM) + lane % (16 * TM), M - 1) * nb;
  const uint8_t* bs = BS + min(n0 + wn * (16 * TN) + lane % (16 * TN), N - 1) * nb;
  int read[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) read[s] = r * 128 + (((4 * s + g) ^ swz8(r)) * 16);
  f32x4 acc[TM][TN] = {};
#pragma unroll
  for (int p = 0; p < STAGES - 1; ++p) issue(min(p, slices - 1), p);
  u32x4 next_a = slab_scales(as, 0, nb), next_b = slab_scales(bs, 0, nb);
  int stage = 0;
  for (int slab = 0; slab < slabs; ++slab) {
    uint32_t sa[4], sb[4];
    spread_scales(next_a, sa);
    spread_scales(next_b, sb);
    if (slab + 1 < slabs) next_a = slab_scales(as, (slab + 1) * SLAB, nb), next_b = slab_scales(bs, (slab + 1) * SLAB, nb);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // all but the newest STAGES - 2 slices' loads have landed (scale loads among them only make this wait longer)
      constexpr int AHEAD = (STAGES - 2) * (TM + TN);
      __builtin_amdgcn_s_waitcnt(0x0070 | (AHEAD & 15) | ((AHEAD >> 4) << 14));  // vmcnt(AHEAD) lgkmcnt(0)
      asm volatile("" ::: "memory");  // no LDS read crosses the barrier, which is none to the compiler
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      issue(min(2 * slab + u + STAGES - 1, slices - 1), (stage + STAGES - 1) % STAGES);
      const uint8_t* la = ring[stage] + wm * (16 * TM * 128);
      const uint8_t* lb = ring[stage] + BM * 128 + wn * (16 * TN * 128);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 x[TM], y[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) x[i] = *reinterpret_cast<const u32x4*>(la + i * 2048 + read[s]);
#pragma unroll
        for (int i = 0; i < TN; ++i) y[i] = *reinterpret_cast<const u32x4*>(lb + i * 2048 + read[s]);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int k = 0; k < TN; ++k) {
            if (u == 0 && s == 0) acc[i][k] = mx_mfma<0>(y[k], x[i], acc[i][k], sb[k], sa[i]);
            else if (u == 0) acc[i][k] = mx_mfma<1>(y[k], x[i], acc[i][k], sb[k], sa[i]);
            else if (s == 0) acc[i][k] = mx_mfma<2>(y[k], x[i], acc[i][k], sb[k], sa[i]);
            else acc[i][k] = mx_mfma<3>(y[k], x[i], acc[i][k], sb[k], sa[i]);
          }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070 | 0x0f00);  // no load still writes the ring when the workgroup's LDS is given away
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int k = 0; k < TN; ++k)
      store4(e, acc[i][k], C, ldc, m0 + wm * (16 * TM) + 16 * i + r, n0 + wn * (16 * TN) + 16 * k + 4 * g, M, N);
}

}  // namespace krn

using namespace krn;

static int launched(const char* who) {
  const hipError_t err = hipGetLastError();
  if (err == hipSuccess) return 0;
  krn_set_error("%s launch: %s", who, hipGetErrorString(err));
  return (int)err;
}

template <int MT, int NT, int WAVES>
static void launch_few(const MxCall& g) {
  hipLaunchKernelGGL((mx_few<MT, NT, WAVES>), dim3((unsigned)((g.n + 16 * NT - 1) / (16 * NT))), dim3(WAVES * 64), 0, g.stream,
                     g.a, g.as, g.b, g.bs, g.c, g.m, g.n, g.nb, g.ldc, g.e);
}

template <int TM, int TN, int STAGES>
static void launch_tile(const MxCall& g) {
  const int64_t tiles = ((g.m + 32 * TM - 1) / (32 * TM)) * ((g.n + 32 * TN - 1) / (32 * TN));
  hipLaunchKernelGGL((mx_tile<TM, TN, STAGES>), dim3((unsigned)tiles), dim3(256), 0, g.stream, g.a, g.as, g.b, g.bs, g.c, g.m,
                     g.n, g.nb, g.ldc, g.e);
}

// The epilogue chain of a launch, checked as krn_gemm's is
static bool mx_epilogue(Epilogue& e, int out_kind, int nops, const int* ops, const float* scalars,
                        const void* const* vectors) {
  if (out_kind != F32 && out_kind != F16 && out_kind != BF16) {
    krn_set_error("mx_gemm: output kind %d; float32, f16 or bf16 results are stored", out_kind);
    return false;
  }
  return epilogue_of(e, out_kind, nops, ops, scalars, vectors, "mx_gemm");
}

extern "C" {

int krn_mx_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, void* c, int out_kind, int64_t m,
                int64_t n, int64_t k, int nops, const int* ops, const float* scalars, const void* const* vectors,
                void* workspace, int64_t workspace_bytes, void* stream) {
  MxCall g{};
  if (!mx_epilogue(g.e, out_kind, nops, ops, scalars, vectors)) return -1;
  // rows of 2^19 blocks: 256 rows of codes are addressed by 31-bit offsets; tiles as a launch's threads allow
  if (m < 0 || n < 0 || k < 1 || k >= (int64_t)1 << 24 || m >= (int64_t)1 << 31 || n >= (int64_t)1 << 31 ||
      ((m + 127) / 128) * ((n + 127) / 128) >= (int64_t)1 << 24) {
    krn_set_error("mx_gemm: %lld x %lld x %lld; rows of 1 to 2^24 - 1 values, m and n below 2^31, fewer than 2^24 tiles of "
                  "128 x 128", (long long)m, (long long)n, (long long)k);
    return -1;
  }
  if ((uintptr_t)a % 16 != 0 || (uintptr_t)b % 16 != 0) {
    krn_set_error("mx_gemm: codes start at a 16-byte aligned address");
    return -1;
  }
  if (m == 0 || n == 0) return 0;
  const int64_t nb = mx_blocks(k), c_bytes = m * n * (out_kind == F32 ? 4 : 2);
  if (share_memory(c, c_bytes, a, m * nb * 16) || share_memory(c, c_bytes, b, n * nb * 16) ||
      share_memory(c, c_bytes, a_scales, m * nb) || share_memory(c, c_bytes, b_scales, n * nb)) {
    krn_set_error("mx_gemm: the result shares memory with an operand");
    return -1;
  }
  g.a = (const uint8_t*)a, g.as = (const uint8_t*)a_scales, g.b = (const uint8_t*)b, g.bs = (const uint8_t*)b_scales;
  g.c = c, g.m = m, g.n = n, g.nb = (int)nb, g.ldc = n, g.stream = (hipStream_t)stream;
  if (m <= 16) launch_few<1, 1, 4>(g);
  else if (m <= 32) launch_few<2, 1, 4>(g);
  else if (m <= 64) launch_few<4, 1, 4>(g);
  else launch_tile<4, 4, 4>(g);
  return launched("mx_gemm");
}

int64_t krn_mx_gemm_workspace(int64_t m, int64_t n, int64_t k) { return 0; }

}  // extern "C"
