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
  Epilogue e;
  void* workspace;  // the planes of K parts (gemm_split.h)
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
  auto slab = [&](int s, auto whole) {  // CUT: the row ends inside the slab
    constexpr bool CUT = !decltype(whole)::value;
    const int block = CUT ? slab_block(s, nb) : s * SLAB;
    const int64_t at = (int64_t)block * 16;
    u32x4 x[MT][4], y[NT][4];
    uint32_t sx[MT], sy[NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = !CUT || in_slab(block + 4 * j + g, s, nb);
#pragma unroll
      for (int t = 0; t < NT; ++t) y[t][j] = in ? *reinterpret_cast<const u32x4*>(b[t] + at + 64 * j) : u32x4{};
#pragma unroll
      for (int t = 0; t < MT; ++t) x[t][j] = in ? *reinterpret_cast<const u32x4*>(a[t] + at + 64 * j) : u32x4{};
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) sy[t] = scale_bytes(CUT ? slab_scales(bs[t], s, nb) : long_scales(bs[t], s, nb), g);
#pragma unroll
    for (int t = 0; t < MT; ++t) sx[t] = scale_bytes(CUT ? slab_scales(as[t], s, nb) : long_scales(as[t], s, nb), g);
#define KRN_STEP(J)                                                                                                  \
  _Pragma("unroll") for (int t = 0; t < MT; ++t) _Pragma("unroll") for (int u = 0; u < NT; ++u) acc[t][u] =          \
      mx_mfma<J>(y[u][J], x[t][J], acc[t][u], sy[u], sx[t]);
    KRN_STEP(0) KRN_STEP(1) KRN_STEP(2) KRN_STEP(3)
#undef KRN_STEP
  };
  const int whole = nb / SLAB;
  for (int s = from; s < min(to, whole); ++s) slab(s, std::true_type{});
  if (to > whole) slab(whole, std::false_type{});
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

// Scales are read for four slabs at a time, 64 bytes of a row together (a slab at a time, a line is fetched from L2 for 16
// bytes of it, as much traffic as the codes): lane (r, q) brings the 16 scales of row r of a 16-row block in slab q of
// the four. Lane (r, g) then gets, for each slab, byte g of its row's four words, packed into one: first the bytes
// within a lane, then the words between the four lane groups (two permlane swaps a word).
struct Spread {  // in six steps of two instructions, to go between MFMAs
  uint32_t t[4], o[4];
  __device__ __forceinline__ void step(int n, const u32x4& d, uint32_t (&out)[4]) {
    if (n == 0) t[0] = __builtin_amdgcn_perm(d[1], d[0], 0x05010400), t[1] = __builtin_amdgcn_perm(d[1], d[0], 0x07030602);
    if (n == 1) t[2] = __builtin_amdgcn_perm(d[3], d[2], 0x05010400), t[3] = __builtin_amdgcn_perm(d[3], d[2], 0x07030602);
    if (n == 2) o[0] = __builtin_amdgcn_perm(t[2], t[0], 0x05040100), o[1] = __builtin_amdgcn_perm(t[2], t[0], 0x07060302);
    if (n == 3) o[2] = __builtin_amdgcn_perm(t[3], t[1], 0x05040100), o[3] = __builtin_amdgcn_perm(t[3], t[1], 0x07060302);
    if (n == 4) {
      const auto p = __builtin_amdgcn_permlane16_swap(o[0], o[1], false, false);
      const auto q = __builtin_amdgcn_permlane16_swap(o[2], o[3], false, false);
      o[0] = p[0], o[1] = p[1], o[2] = q[0], o[3] = q[1];
    }
    if (n == 5) {
      const auto p = __builtin_amdgcn_permlane32_swap(o[0], o[2], false, false);
      const auto q = __builtin_amdgcn_permlane32_swap(o[1], o[3], false, false);
      out[0] = p[0], out[2] = p[1], out[1] = q[0], out[3] = q[1];
    }
  }
};

__device__ __forceinline__ void spread_scales(const u32x4& d, uint32_t (&out)[4]) {
  Spread s;
#pragma unroll
  for (int n = 0; n < 6; ++n) s.step(n, d, out);
}

// An activation of four values. Out of line, so that its registers are not the store's as well: three workgroups of 64 x 64
// tiles share a CU instead of two (1000 x 3001 x 777 with bias and gelu 22.7 -> 18.9 us)
__device__ __noinline__ f32x4 activate4(f32x4 x, int op) {
#define KRN_ALL(OP) f32x4{activation(OP, x[0]), activation(OP, x[1]), activation(OP, x[2]), activation(OP, x[3])}
  if (op == RELU) return KRN_ALL(RELU);
  return op == GELU ? KRN_ALL(GELU) : KRN_ALL(SILU);
#undef KRN_ALL
}

// One 32 x 32 block from its patch through the epilogue to C, rows at any alignment: lane l has columns 16 (l & 1) .. + 15 of
// row l / 2. Out of line, each wave storing several blocks. What an operation does is decided once for four or more
// values. WIDE: the four-wave loop's, which has a CU to itself: activations of sixteen values in line, whose chains overlap
// (4096 x 14336 x 4096 with silu: 297 us in calls of four, 253; bias and gelu 515, 450).
template <bool WIDE>
__device__ __noinline__ void store_patch(uint32_t* patch, void* C, int64_t ldc, int64_t row0, int64_t col0, int64_t M,
                                         int64_t N, const Epilogue& e, int lane) {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the patch is written before any lane reads it
  __builtin_amdgcn_wave_barrier();
  const int rr = lane >> 1, c0 = (lane & 1) * 16;
  float v[16];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(patch + rr * PATCH_STRIDE + c0 + 4 * q);
    v[4 * q] = w[0], v[4 * q + 1] = w[1], v[4 * q + 2] = w[2], v[4 * q + 3] = w[3];
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();  // the next block may overwrite the patch
  const int64_t m = row0 + rr, n = col0 + c0;
  if (m >= M || n >= N) return;
  const int cols = (int)min(N - n, (int64_t)16);
  for (int i = 0; i < e.nops; ++i) {
    const int op = e.op[i] & ((1 << VEC_KIND_SHIFT) - 1), kind = e.op[i] >> VEC_KIND_SHIFT;
#define KRN_ALL(x) _Pragma("unroll") for (int c = 0; c < 16; ++c) v[c] = x
    if (WIDE && op >= RELU) {
      if (op == RELU) { KRN_ALL(activation(RELU, v[c])); }
      else if (op == GELU) { KRN_ALL(activation(GELU, v[c])); }
      else { KRN_ALL(activation(SILU, v[c])); }
    } else if (op >= RELU) {
#pragma unroll
      for (int c = 0; c < 16; c += 4) {
        const f32x4 x = activate4(f32x4{v[c], v[c + 1], v[c + 2], v[c + 3]}, op);
        v[c] = x[0], v[c + 1] = x[1], v[c + 2] = x[2], v[c + 3] = x[3];
      }
    } else if (op % 3 == 2) {
#pragma unroll
      for (int h = 0; h < 16; h += 4) {
        float s[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) s[c] = bits_value(kind, vec_bits(e.vec[i], kind, n + min(h + c, cols - 1)));
#pragma unroll
        for (int c = 0; c < 4; ++c) v[h + c] = op == MUL_COL ? __fmul_rn(v[h + c], s[c]) : __fadd_rn(v[h + c], s[c]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      const float s = op % 3 == 0 ? e.scalar[i] : bits_value(kind, vec_bits(e.vec[i], kind, m));
      if (op < 3) { KRN_ALL(__fmul_rn(v[c], s)); }
      else { KRN_ALL(__fadd_rn(v[c], s)); }
    }
#undef KRN_ALL
  }
  if (e.out_kind == F32) {
    float* out = static_cast<float*>(C) + m * ldc + n;
    if (cols == 16) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        reinterpret_cast<u32x4_any*>(out)[q] = __builtin_bit_cast(u32x4, f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
    } else {
#pragma unroll
      for (int c = 0; c < 16; ++c)
        if (c < cols) out[c] = v[c];
    }
    return;
  }
  uint32_t h[8];
#pragma unroll
  for (int c = 0; c < 8; ++c)
    h[c] = e.out_kind == BF16 ? f2bf2(v[2 * c], v[2 * c + 1]) : (uint32_t)f2h(v[2 * c]) | (uint32_t)f2h(v[2 * c + 1]) << 16;
  uint16_t* out = static_cast<uint16_t*>(C) + m * ldc + n;
  if (cols == 16) {
    reinterpret_cast<u32x4_any*>(out)[0] = u32x4{h[0], h[1], h[2], h[3]};
    reinterpret_cast<u32x4_any*>(out)[1] = u32x4{h[4], h[5], h[6], h[7]};
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (c < cols) out[c] = (uint16_t)(h[c >> 1] >> ((c & 1) * 16));
  }
}

// Tiles of 32 TM x 32 TN, four waves of 16 TM x 16 TN each, K in `parts` runs of slabs (blockIdx.y). Slices of 128 bytes a
// row (half a slab, two MFMA steps) go from memory straight into a ring of LDS stages, chunk c of row r at slot
// c ^ ((r >> 1) & 7), STAGES - 1 slices ahead. Past the end of a row, and of the matrix, the buffer loads give zeros.
// Fragments are read a step ahead of the MFMAs that use them; the one barrier a slice, after its second step's reads,
// publishes the next slice and frees this one's stage. Scales go to registers, four slabs ahead.
// CUT: rows end inside a slab.
template <int TM, int TN, int STAGES, bool CUT>
__global__ __launch_bounds__(256) void mx_tile(const uint8_t* __restrict__ A, const uint8_t* __restrict__ AS,
                                               const uint8_t* __restrict__ B, const uint8_t* __restrict__ BS,
                                               void* __restrict__ C, int64_t M, int64_t N, int nb, int64_t ldc, Epilogue e,
                                               int parts) {
  static_assert(TM <= 4 && TN <= 4 && TM % 2 == 0 && TN % 2 == 0, "a wave's scales are one row a lane, its blocks stored 32 x 32");
  constexpr int BM = 32 * TM, BN = 32 * TN, STAGE = (BM + BN) * 128, LOADS = TM + TN;
  static_assert(STAGES * STAGE >= 4 * PATCH_WORDS * 4, "the store patches fit the ring");
  __shared__ __attribute__((aligned(1024))) uint8_t ring[STAGES * STAGE];
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
  const int all = (nb + SLAB - 1) / SLAB, part = blockIdx.y;
  const int first = (int)((int64_t)all * part / parts), end = (int)((int64_t)all * (part + 1) / parts), last = 2 * end - 1;
  if (parts > 1) C = static_cast<uint8_t*>(C) + part * (M * ldc * 4);
  // slice `slice` (clamped to the last), whose first block in memory is `block`
#define KRN_ISSUE(NAME, TX, rsrc, off, chunk, base)                                                                 \
  auto NAME = [&](int slice) {                                                                                      \
    const int sl = min(slice, last), block = CUT ? slab_block(sl >> 1, nb) + 8 * (sl & 1) : sl * 8;                 \
    uint8_t* to = ring + (slice & (STAGES - 1)) * STAGE + base + wave * (8 * TX * 128);                             \
    _Pragma("unroll") for (int j = 0; j < TX; ++j)                                                                  \
        buffer_to_lds16(rsrc, to + j * 1024, !CUT || in_slab(block + chunk[j], sl >> 1, nb) ? off[j] : 0x80000000u, block * 16); \
  };
  KRN_ISSUE(issue_a, TM, a_rsrc, ga, ca, 0)
  KRN_ISSUE(issue_b, TN, b_rsrc, gb, cb, BM * 128)
#undef KRN_ISSUE
  // the rows whose scales this lane brings: row r of each of the wave's blocks
  const uint8_t *as[TM], *bs[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) as[i] = AS + min(m0 + wm * (16 * TM) + 16 * i + r, M - 1) * nb;
#pragma unroll
  for (int i = 0; i < TN; ++i) bs[i] = BS + min(n0 + wn * (16 * TN) + 16 * i + r, N - 1) * nb;
  int ra[2], rb[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int chunk = r * 128 + (((4 * s + g) ^ swz8(r)) * 16);
    ra[s] = wm * (16 * TM * 128) + chunk, rb[s] = BM * 128 + wn * (16 * TN * 128) + chunk;
  }
  // all but the newest AHEAD loads have landed (scale loads among them only make this wait longer), this wave's LDS reads
  // are done, and then every wave's; no access crosses it
#define KRN_PUBLISH(AHEAD)                                                                               \
  do {                                                                                                   \
    __builtin_amdgcn_sched_barrier(0);                                                                   \
    asm volatile("" ::: "memory");                                                                       \
    __builtin_amdgcn_s_waitcnt(0x0070 | ((AHEAD) & 15) | (((AHEAD) >> 4) << 14)); /* vmcnt(AHEAD) lgkmcnt(0) */ \
    __builtin_amdgcn_s_barrier();                                                                        \
    asm volatile("" ::: "memory");                                                                       \
    __builtin_amdgcn_sched_barrier(0);                                                                   \
  } while (0)
#define KRN_READ(set, slice, s)                                                                                         \
  do {                                                                                                                  \
    const uint8_t* at = ring + ((slice) & (STAGES - 1)) * STAGE;                                                        \
    _Pragma("unroll") for (int i = 0; i < TM; ++i) x##set[i] = *reinterpret_cast<const u32x4*>(at + ra[s] + i * 2048);  \
    _Pragma("unroll") for (int i = 0; i < TN; ++i) y##set[i] = *reinterpret_cast<const u32x4*>(at + rb[s] + i * 2048);  \
  } while (0)
#define KRN_MMA(set, J, q)                                                                                                 \
  _Pragma("unroll") for (int i = 0; i < TM; ++i) _Pragma("unroll") for (int k = 0; k < TN; ++k)                         \
      acc[i][k] = mx_mfma<J>(y##set[k], x##set[i], acc[i][k], sb[k][q], sa[i][q]);
  // One slice: its second step's reads and A's loads of the slice STAGES - 1 ahead go between the MFMAs of the first
  // step, the next slice's first reads (past the end: a slice that is not used) and B's loads between those of the
  // second. A wave issues in order, so a burst of either would hold the MFMAs behind it back.
#define KRN_SPREAD(LOADS_)                                                                                              \
  _Pragma("unroll") for (int i = 0; i < TM * TN; ++i) {                                                                 \
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                                                  \
    if (i < TM + TN) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                 \
    if (i >= TM * TN - (LOADS_)) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                                       \
  }
#define KRN_SLICE(kt, J0, J1, q)                                                                                        \
  do {                                                                                                                  \
    KRN_READ(1, kt, 1);                                                                                                 \
    issue_a((kt) + STAGES - 1);                                                                                         \
    if (STAGES == 2) issue_b((kt) + 1); /* two stages: the next slice whole, to land by the barrier */                  \
    KRN_MMA(0, J0, q);                                                                                                  \
    KRN_SPREAD(STAGES == 2 ? TM + TN : TM);                                                                             \
    KRN_PUBLISH(STAGES == 2 ? 0 : (STAGES - 3) * LOADS + TM);                                                           \
    KRN_READ(0, (kt) + 1, 0);                                                                                           \
    if (STAGES > 2) issue_b((kt) + STAGES - 1);                                                                         \
    KRN_MMA(1, J1, q);                                                                                                  \
    KRN_SPREAD(TN);                                                                                                     \
    __builtin_amdgcn_sched_barrier(0);                                                                                  \
  } while (0)
  f32x4 acc[TM][TN] = {};
  u32x4 x0[TM], y0[TN], x1[TM], y1[TN];
#pragma unroll
  for (int p = 0; p < STAGES - 1; ++p) issue_a(2 * first + p), issue_b(2 * first + p);
  u32x4 next_a[TM], next_b[TN];
  auto fetch = [&](int slab) {
#pragma unroll
    for (int i = 0; i < TM; ++i) next_a[i] = long_scales(as[i], slab + g, nb);
#pragma unroll
    for (int i = 0; i < TN; ++i) next_b[i] = long_scales(bs[i], slab + g, nb);
  };
  if (nb < SLAB) {
#pragma unroll
    for (int i = 0; i < TM; ++i) next_a[i] = short_scales(as[i], nb);
#pragma unroll
    for (int i = 0; i < TN; ++i) next_b[i] = short_scales(bs[i], nb);
  } else {
    fetch(first);
  }
  KRN_PUBLISH((STAGES - 2) * LOADS);
  KRN_READ(0, 2 * first, 0);
  for (int group = first; group < end; group += 4) {
    uint32_t sa[TM][4], sb[TN][4];
#pragma unroll
    for (int i = 0; i < TM; ++i) spread_scales(next_a[i], sa[i]);
#pragma unroll
    for (int i = 0; i < TN; ++i) spread_scales(next_b[i], sb[i]);
    if (group + 4 < end) fetch(group + 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int slab = group + q;
      if (slab < end) {
        KRN_SLICE(2 * slab, 0, 1, q);
        KRN_SLICE(2 * slab + 1, 2, 3, q);
      }
    }
  }
#undef KRN_PUBLISH
#undef KRN_READ
#undef KRN_MMA
#undef KRN_SPREAD
#undef KRN_SLICE
  __builtin_amdgcn_s_waitcnt(0x0070);  // no load still writes the ring
  __syncthreads();
  // 32 x 32 blocks through a patch of the wave's own: lane (r, g) holds row r and columns 4 g .. + 3 of each 16 x 16 block
  uint32_t* patch = reinterpret_cast<uint32_t*>(ring) + wave * PATCH_WORDS;
  const Epilogue local = e;  // taken by address by the out-of-line store
#pragma unroll
  for (int i = 0; i < TM; i += 2)
#pragma unroll
    for (int k = 0; k < TN; k += 2) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<f32x4*>(patch + (16 * p + r) * PATCH_STRIDE + 16 * q + 4 * g) = acc[i + p][k + q];
      store_patch<false>(patch, C, ldc, m0 + wm * (16 * TM) + 16 * i, n0 + wn * (16 * TN) + 16 * k, M, N, local, lane);
    }
}

// The four-wave loop for many 256 x 256 tiles, as gemm_quad16 (gemm.hip) runs the other formats. Each wave owns a
// 128 x 128 quarter (wave w: rows 128 (w >> 1), columns 128 (w & 1)) as 8 x 8 blocks of 16 x 16 in AGPRs. Slices of 128 bytes
// a row (half a slab) go straight into LDS stages, two for A and three for B (160 KiB), each stage an array of its own
// so that the compiler can tell fragment reads from the loads in flight; wave w loads rows 64 w .. 64 w + 63 of both, 8 rows a
// load, chunk c of row r at slot c ^ ((r >> 1) & 7).
//
// One set of fragments (four 32-row blocks of A and of B, two 16-row halves each, both steps of a slice) is refilled in
// place: slices alternate between running their 16 blocks of 32 x 32 row by row (block (I, J) is group 4 I + J of eight
// MFMAs) and column by column, so a block's fragments are dead after its last group and take the next slice's behind
// the MFMAs of the group after it. The one barrier a slice sits after group 3: this wave has read all of slice kt, and
// its loads of slice kt + 1 have landed (the two issued last are B's of slice kt + 2). B's slice kt + 2 is loaded
// through the slice, A's after the barrier.
//
// Scales are brought for two slabs at a time, 32 bytes of a row together: lane (r, q) the 16 of slab q % 2 and of row r
// of half q / 2 of a 32-row block. The next two slabs' are loaded at the ends of the second and third slice, and spread
// between the MFMAs of the fourth.
//
// CUT: rows end inside a slab. Rows hold a slab at least. DIRECT: the epilogue and N are the direct
// store's (quad16_direct), whose stores past the last row do nothing; otherwise all blocks go through patches. (Both
// stores in one kernel leave the loop too few registers.)
template <bool CUT, bool DIRECT>
__global__ __launch_bounds__(256, 1) void mx_quad(const uint8_t* __restrict__ A, const uint8_t* __restrict__ AS,
                                                  const uint8_t* __restrict__ B, const uint8_t* __restrict__ BS,
                                                  void* __restrict__ C, int64_t M, int64_t N, int nb, int64_t ldc, Epilogue e) {
  constexpr int NA = 2, NB = 3, BM = 256, BN = 256, HALF = BM * 128;
  __shared__ __attribute__((aligned(1024))) uint8_t la0[HALF];
  __shared__ __attribute__((aligned(1024))) uint8_t la1[HALF];
  __shared__ __attribute__((aligned(1024))) uint8_t lb0[HALF];
  __shared__ __attribute__((aligned(1024))) uint8_t lb1[HALF];
  __shared__ __attribute__((aligned(1024))) uint8_t lb2[HALF];
  int tm, tn;
  tile_of((int)((M + BM - 1) / BM), (int)((N + BN - 1) / BN), tm, tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN, ld = (int64_t)nb * 16;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave >> 1, wn = wave & 1, r16 = lane & 15, g4 = lane >> 4;
  auto uniform = [](const void* p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const void*)(((uint64_t)hi << 32) | (uint64_t)lo);
  };
  const __amdgpu_buffer_rsrc_t a_rsrc = panel_rsrc(uniform(A + m0 * ld), __builtin_amdgcn_readfirstlane((int)min((M - m0) * ld, (int64_t)0x7fffffff))),
                               b_rsrc = panel_rsrc(uniform(B + n0 * ld), __builtin_amdgcn_readfirstlane((int)min((N - n0) * ld, (int64_t)0x7fffffff)));
  // load item j of an operand: rows 64 wave + 8 j .. + 7, lane i row i / 8 and the chunk that belongs at slot i % 8; the
  // swizzle depends on j through j & 1
  uint32_t go[2];
  int chunk[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = wave * 64 + p * 8 + (lane >> 3);
    chunk[p] = (lane & 7) ^ swz8(row), go[p] = (uint32_t)(row * ld + chunk[p] * 16);
  }
  const int wbase = wave * 8192;
  int ra[2], rb[2];  // fragment reads: row r16 of a half, chunk 4 step + g4
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int part = r16 * 128 + (((4 * x + g4) ^ swz8(r16)) * 16);
    ra[x] = part + wm * 128 * 128, rb[x] = part + wn * 128 * 128;
  }
  const int slabs = (nb + SLAB - 1) / SLAB, nk = 2 * slabs;
  // the scales this lane brings: of row 32 k + 16 (g4 / 2) + r16 of the wave's 128, the matrix's last row past its
  // end, by 32-bit offsets from the tile's first row
  const uint8_t *as = AS + m0 * nb, *bs = BS + n0 * nb;
  const int srow = 16 * (g4 >> 1) + r16, slab_of = g4 & 1;
  const int a_last = (int)min(M - 1 - m0, (int64_t)(BM - 1)), b_last = (int)min(N - 1 - n0, (int64_t)(BN - 1));

  u32x4 F[16][2];  // A block I half R at 2 I + R, B block J half Q at 8 + 2 J + Q; both steps
  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{};
  u32x4 raw[8];          // the next two slabs' scales as loaded: A's four, B's four
  uint32_t sc[8][4];     // spread: [load][slab + 2 half]
  uint32_t cur[2];       // load offsets of the slice being loaded, outside the matrix for blocks that count in the slab before
  int at;                // and its first block

#define MQ_A(p) ((p) == 0 ? la0 : la1)
#define MQ_B(p) ((p) == 0 ? lb0 : (p) == 1 ? lb1 : lb2)
#define MQ_AT(sl)                                                                                              \
  do {                                                                                                         \
    at = CUT ? slab_block((sl) >> 1, nb) + 8 * ((sl) & 1) : (sl) * 8;                                          \
    _Pragma("unroll") for (int p = 0; p < 2; ++p)                                                              \
      cur[p] = !CUT || at + chunk[p] >= ((sl) >> 1) * SLAB ? go[p] : 0x80000000u;                              \
  } while (0)
#define MQ_LOADA(j, pa) buffer_to_lds16(a_rsrc, MQ_A(pa) + wbase + (j) * 1024, cur[(j) & 1], (int)(at * 16 + ((j) & 6) * 8 * ld))
#define MQ_LOADB(j, pb) buffer_to_lds16(b_rsrc, MQ_B(pb) + wbase + (j) * 1024, cur[(j) & 1], (int)(at * 16 + ((j) & 6) * 8 * ld))
#define MQ_READ(r, c, x, pa, pb)                                                                               \
  F[(r) * 2 + (c)][x] = *reinterpret_cast<const u32x4*>(                                                       \
      ((r) < 4 ? MQ_A(pa) + ra[x] : MQ_B(pb) + rb[x]) + (((r) & 3) * 32 + (c) * 16) * 128)
#define MQ_FENCE() __builtin_amdgcn_sched_barrier(0)
// scale load k (0-3 A's, 4-7 B's) of the slabs from `slab`
// (the row is opaque to the compiler, which would otherwise keep eight products of it in registers)
#define MQ_SCALES(k, slab)                                                                                     \
  do {                                                                                                         \
    int row = srow;                                                                                            \
    asm volatile("" : "+v"(row));                                                                                       \
    row = (k) < 4 ? min(wm * 128 + 32 * ((k) & 3) + row, a_last) : min(wn * 128 + 32 * ((k) & 3) + row, b_last); \
    const uint32_t off = __umul24((uint32_t)row, (uint32_t)nb) + (uint32_t)min(((slab) + slab_of) * SLAB, nb - SLAB); \
    raw[k] = *reinterpret_cast<const u32x4_any*>(((k) < 4 ? as : bs) + off);                                   \
  } while (0)
#define MQ_ONE(X, SEL)                                                                                         \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL " cbsz:4 blgp:4"                \
               : "+a"(acc[mi][mj])                                                                             \
               : "v"(F[8 + mj][X]), "v"(F[mi][X]), "v"(sb), "v"(sa))
// MFMA n of block (I, J) of slice U of a run: step n / 4 of its 16 x 16 block (R, Q) = (n / 2 % 2, n % 2), with scale byte
// 2 (U & 1) + step of slab (U >> 1) & 1
#define MQ_MMA(I, J, U, n)                                                                                     \
  do {                                                                                                         \
    const int X = (n) >> 2, R = ((n) >> 1) & 1, Q = (n) & 1, mi = 2 * (I) + R, mj = 2 * (J) + Q;               \
    const uint32_t sa = sc[I][(((U) >> 1) & 1) + 2 * R], sb = sc[4 + (J)][(((U) >> 1) & 1) + 2 * Q];           \
    if (((U) & 1) == 0 && X == 0) MQ_ONE(0, "op_sel:[0,0,0] op_sel_hi:[0,0,0]");                               \
    else if (((U) & 1) == 0) MQ_ONE(1, "op_sel:[1,1,0] op_sel_hi:[0,0,0]");                                    \
    else if (X == 0) MQ_ONE(0, "op_sel:[0,0,0] op_sel_hi:[1,1,0]");                                            \
    else MQ_ONE(1, "op_sel:[1,1,0] op_sel_hi:[1,1,0]");                                                        \
  } while (0)
// Which spread (scale load) runs beside group g of slice U of a run, none: -1. Beside the last slice of two slabs go those
// whose scales no later group of it takes (column order: B's J after group 4 J + 3, A's I after 12 + I), beside the next
// slice, before the groups that need them, the other two.
#define MQ_WHICH(U, g)                                                                                         \
  ((U) % 4 == 3 ? ((g) == 5 ? 4 : (g) == 9 ? 5 : (g) == 12 ? 6 : (g) >= 13 ? (g) - 13 : -1)                    \
                : (U) % 4 == 0 ? ((g) == 0 ? 7 : (g) == 1 ? 3 : -1) : -1)
// Slice kt, u-th of an unrolled run: stages PA, PB, order u & 1. Behind every MFMA at most one memory instruction or
// step of a spread; the fragments that a group leaves dead are read behind the MFMAs of the next.
#define MQ_SLICE(u, kt)                                                                                        \
  do {                                                                                                         \
    const int PA = (u) % NA, PB = (u) % NB, NA_ = (PA + 1) % NA, NB_ = (PB + 1) % NB, ord = (u) & 1;           \
    const int ahead = min((kt) + 2, nk - 1);                                                                   \
    MQ_AT(ahead);                                                                                              \
    _Pragma("unroll") for (int g = 0; g < 16; ++g) {                                                           \
      const int I = ord ? (g & 3) : (g >> 2), J = ord ? (g >> 2) : (g & 3), k = MQ_WHICH(u, g);                \
      /* the block the group before left dead, at g = 0 both that the slice before left last */                \
      const int f = g - 1, fi = ord ? (f & 3) : (f >> 2), fj = ord ? (f >> 2) : (f & 3);                       \
      const int dead = g == 0 ? 3 : fj == 3 && (ord == 0 || fi != 3) && (ord == 0 || f >= 12) ? fi             \
                               : fi == 3 && (ord == 1 || f >= 12) ? 4 + fj : -1;                               \
      Spread spread;                                                                                           \
      _Pragma("unroll") for (int n = 0; n < 8; ++n) {                                                          \
        MQ_MMA(I, J, u, n);                                                                                    \
        MQ_FENCE();                                                                                            \
        if (g == 0) { if (n < 4) MQ_READ(3, n >> 1, n & 1, PA, PB); else MQ_READ(7, (n >> 1) & 1, n & 1, PA, PB); } \
        else if (dead >= 0 && n < 4) MQ_READ(dead, n >> 1, n & 1, NA_, NB_);                                   \
        if (n == 4 && (g & 1) == 0) MQ_LOADB(g >> 1, (PB + 2) % NB);                                           \
        if (n == 5 && g >= 4 && g < 12) MQ_LOADA(g - 4, PA);                                                   \
        if (n == 6 && ((u) % 4 == 1 || (u) % 4 == 2) && g >= 12)                                               \
          MQ_SCALES(((u) % 4 - 1) * 4 + g - 12, (kt) / 2 - ((u) % 4) / 2 + 2);                                 \
        if (k >= 0 && n < 6) spread.step(n, raw[k < 0 ? 0 : k], sc[k < 0 ? 0 : k]);                            \
        MQ_FENCE();                                                                                            \
      }                                                                                                        \
      if (g == 3) {                                                                                            \
        __builtin_amdgcn_s_waitcnt(0x0070 | 2); /* vmcnt(2) lgkmcnt(0) */                                      \
        __builtin_amdgcn_s_barrier();                                                                          \
        MQ_FENCE();                                                                                            \
      }                                                                                                        \
    }                                                                                                          \
  } while (0)

  // the prologue: the first scales, slices 0 and 1 of A and B (B's slice 2 loads during slice 0, as in the loop); once
  // slice 0 has landed everywhere, its fragments
#pragma unroll
  for (int k = 0; k < 8; ++k) MQ_SCALES(k, 0);
#pragma unroll
  for (int sl = 0; sl < 2; ++sl) {
    MQ_AT(sl);
#pragma unroll
    for (int j = 0; j < 8; ++j) MQ_LOADA(j, sl);
#pragma unroll
    for (int j = 0; j < 8; ++j) MQ_LOADB(j, sl);
  }
  __builtin_amdgcn_s_waitcnt(0x0070 | 0x4000);  // vmcnt(16): slice 0's 16 loads came before slice 1's
  __builtin_amdgcn_s_barrier();
  MQ_FENCE();
#pragma unroll
  for (int k = 0; k < 8; ++k) spread_scales(raw[k], sc[k]);
#pragma unroll
  for (int x = 0; x < 6; ++x) {  // in the order a slice reads them (blocks 3 and 7 behind its first group)
    const int r = x < 3 ? 4 + x : x - 3;
#pragma unroll
    for (int n = 0; n < 4; ++n) MQ_READ(r, n >> 1, n & 1, 0, 0);
    MQ_FENCE();
  }
  // twelve slices a turn: every stage index, scale byte and order is a constant (slices come in pairs)
#define MQ_PAIR(u)                                                                                             \
  MQ_SLICE(u, kt + (u));                                                                                       \
  MQ_SLICE((u) + 1, kt + (u) + 1);
  int kt = 0;
  for (; kt + 12 <= nk; kt += 12) {
    MQ_PAIR(0) MQ_PAIR(2) MQ_PAIR(4) MQ_PAIR(6) MQ_PAIR(8) MQ_PAIR(10)
  }
  if (kt + 0 < nk) { MQ_PAIR(0) }
  if (kt + 2 < nk) { MQ_PAIR(2) }
  if (kt + 4 < nk) { MQ_PAIR(4) }
  if (kt + 6 < nk) { MQ_PAIR(6) }
  if (kt + 8 < nk) { MQ_PAIR(8) }
#undef MQ_PAIR
#undef MQ_A
#undef MQ_B
#undef MQ_AT
#undef MQ_LOADA
#undef MQ_LOADB
#undef MQ_READ
#undef MQ_FENCE
#undef MQ_SCALES
#undef MQ_WHICH
#undef MQ_ONE
#undef MQ_MMA
#undef MQ_SLICE
  __builtin_amdgcn_s_waitcnt(0x0070);  // no load still writes the stages
  // the MFMAs are assembly, so the compiler inserts no wait states before the first read of their results
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  __syncthreads();
  const int64_t row0 = m0 + wm * 128, col0 = n0 + wn * 128;
  if constexpr (DIRECT) {
    if (row0 >= M || col0 >= N) return;  // N is a multiple of 128
    const int64_t rows = min(M - row0, (int64_t)128);
    Quad16Generic ops;
    quad16_generic(ops, e, row0, col0, lane);
    if (e.out_kind == BF16) store16t_direct<false, true>(acc, ops, C, ldc, row0, col0, lane, rows);
    else store16t_direct<false, false>(acc, ops, C, ldc, row0, col0, lane, rows);
    return;
  }
  uint32_t* patch = reinterpret_cast<uint32_t*>(la0) + wave * PATCH_WORDS;
  const Epilogue local = e;  // taken by address by the out-of-line store
#pragma unroll
  for (int i = 0; i < 8; i += 2)
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<f32x4*>(patch + (16 * p + r16) * PATCH_STRIDE + 16 * q + 4 * g4) = agpr_block(acc[i + p][k + q]);
      store_patch<true>(patch, C, ldc, row0 + 16 * i, col0 + 16 * k, M, N, local, lane);
    }
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
static int launch_few(const MxCall& g) {
  hipLaunchKernelGGL((mx_few<MT, NT, WAVES>), dim3((unsigned)((g.n + 16 * NT - 1) / (16 * NT))), dim3(WAVES * 64), 0, g.stream,
                     g.a, g.as, g.b, g.bs, g.c, g.m, g.n, g.nb, g.n, g.e);
  return launched("mx_gemm");
}

template <int TM, int TN, int STAGES>
static int launch_tile(const MxCall& g, int parts) {
  const int64_t tiles = ((g.m + 32 * TM - 1) / (32 * TM)) * ((g.n + 32 * TN - 1) / (32 * TN));
  const bool split = parts > 1;
  auto kernel = g.nb % SLAB == 0 ? mx_tile<TM, TN, STAGES, false> : mx_tile<TM, TN, STAGES, true>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)parts), dim3(256), 0, g.stream, g.a, g.as, g.b, g.bs,
                     split ? g.workspace : g.c, g.m, g.n, g.nb, split ? split_ld(g.n) : g.n,
                     split ? plane_epilogue(FMT_FP8) : g.e, parts);
  const int rc = launched("mx_gemm");
  if (rc != 0 || !split) return rc;
  return launch_reduce(FMT_FP8, parts, SplitCall{nullptr, nullptr, g.c, g.m, g.n, 0, 0, 0, g.e, g.workspace, g.stream});
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

// Few rows: 16 x (16 NT) columns a workgroup; then tiles, by their stages; then the four-wave loop on 256 x 256 tiles
enum MxShape : int { FEW_16x16, FEW_16x32, FEW_16x64, FEW_32x16, FEW_32x32, TILE_64_SHORT, TILE_64, TILE_64_DEEP, TILE_64x128, TILE_128, QUAD };
static const char* const SHAPE_NAMES[] = {"few_16x16", "few_16x32", "few_16x64", "few_32x16", "few_32x32", "tile_64x64_short",
                                          "tile_64x64", "tile_64x64_deep", "tile_64x128", "tile_128x128", "quad_256x256"};
struct MxPlan {
  int shape, parts;
  int64_t workspace;
};

static MxPlan mx_plan(int64_t m, int64_t n, int64_t nb, bool activation, int64_t workspace) {
  const int64_t slabs = (nb + SLAB - 1) / SLAB;
  // A launch has fewer than 2^32 threads: 512 for 32 columns reach that at the last n below 2^28, which others take
  constexpr int64_t MOST_32 = ((int64_t)1 << 28) - 32;
  // Up to 32 rows: wider workgroups read A less often, narrower ones fill the chip. Up to 16 rows (us, on 16 / 32 / 64 columns,
  // three sets of operands in turn): 1 x 8192 x 8192 9.1 / 8.4 / 14.7, 1 x 14336 x 4096 8.5 / 8.0 / 9.2, 16 x 8192 x 4096 7.2 /
  // 6.4 / 9.3, 16 x 14336 x 4096 11.4 / 9.5 / 9.8; one row at 9216 to 12288 columns is 10 % faster on 16, sixteen rows are equal.
  // 64 columns pay from nine rows, where the launch fills its rounds: a CU holds three such workgroups, and takes twice as
  // many of 32 columns (16 rows, K = 4096, on 32 / 64: n = 20480 12.8 / 14.3, 28672 16.1 / 14.7, 32768 16.2 / 15.4, 40960 21.5 /
  // 22.3, 49152 28.0 / 26.1, 65536 38.5 / 44.1, 81920 47.1 / 49.0, 98304 55.7 / 52.1, 131072 72.9 / 73.4; 8 rows: 28672 14.5 / 14.2,
  // with K = 8192 33.0 / 33.1; 1 row: 13.0 / 13.8).
  if (m <= 16) {
    const int64_t wide = (n + 64 * 256 - 1) / (64 * 256), half = (n + 32 * 256 - 1) / (32 * 256);  // workgroups a CU
    if (n > MOST_32 || (m > 8 && (wide == 2 || wide % 3 == 0) && 2 * wide <= half)) return {FEW_16x64, 1, 0};
    return {n >= 32 * 256 ? FEW_16x32 : FEW_16x16, 1, 0};
  }
  // (us, on 16 / 32 columns: 24 x 4096 x 4096 5.5 / 6.9, 32 x 8192 x 8192 15.9 / 11.7, tiles of 64 x 64 7.7 and 11.9)
  if (m <= 32 && n <= MOST_32) return {n >= 32 * 256 ? FEW_32x32 : FEW_32x16, 1, 0};
  // Estimated microseconds beyond a launch: what a slab takes the CU that holds most workgroups, measured at K = 8192
  // (64 x 64 tiles, 256 workgroups 14.1 us, 512 21.8, 1024 39.1; eight stages 13.5, 24.5; 64 x 128 17.2, 35.3; 128 x 128 22.4,
  // 52.3; 256 x 256 tiles, 128 of them 52.6, 256 66.3), and what parts add: their planes' way to the second launch and back
  auto rounds = [&](int bm, int bn, int parts) {
    return (double)((((m + bm - 1) / bm) * ((n + bn - 1) / bn) * parts + 255) / 256);
  };
  MxPlan best{TILE_64, 1, 0};
  double least = 1e30;
  for (int shape = TILE_64_SHORT; shape <= QUAD; ++shape)
    for (int parts = 1; parts <= (shape == QUAD || shape == TILE_64_SHORT ? 1 : 8) && (parts == 1 || slabs / parts >= 2); ++parts) {
      if (shape == QUAD && nb < SLAB) break;  // its scale loads take 16 bytes of a row
      const int bm = shape <= TILE_64x128 ? 64 : shape == TILE_128 ? 128 : 256, bn = shape <= TILE_64_DEEP ? 64 : shape <= TILE_128 ? 128 : 256;
      const double r = rounds(bm, bn, parts);
      double slab = shape == TILE_64_SHORT ? 0.57 * r + 0.2 : shape == TILE_64 ? (r > 1 ? 0.53 * r : 0.57)
                  : shape == TILE_64_DEEP ? (r > 1 ? 0.62 * r : 0.52) : shape == TILE_64x128 ? 0.93 * r : shape == TILE_128 ? 1.45 * r
                                          : 3.0 * r + (rounds(256, 128, 1) > r ? 0.8 * r : 0);
      // two stages let three workgroups share a CU and hide each other's first loads and stores, which is what a short K
      // is made of (1000 x 3001 x 777, bias and gelu: 22.2 us with four, 17.4)
      double us = (double)((slabs + parts - 1) / parts) * slab + (shape == TILE_64_SHORT ? 1.5 : 3.0) * r;
      const int64_t need = parts > 1 ? parts * split_plane(m, n) : 0;
      // an activation takes a CU's waves a time of its own for each 32 x 32 block they store, less where workgroups share it
      if (activation && parts == 1)
        us += r * (shape <= TILE_64 ? 1.6 : 2.2 * (bm / 64) * (bn / 64));
      if (parts > 1) us += 4.0 + (double)need / 5e6;
      if (need <= workspace && us < least) best = {shape, parts, need}, least = us;
    }
  return best;
}

static int launch_planned(const MxPlan& p, const MxCall& g) {
  switch (p.shape) {
    case FEW_16x16: return launch_few<1, 1, 8>(g);
    case FEW_16x32: return launch_few<1, 2, 8>(g);
    case FEW_16x64: return launch_few<1, 4, 4>(g);
    case FEW_32x16: return launch_few<2, 1, 4>(g);
    case FEW_32x32: return launch_few<2, 2, 8>(g);
    case TILE_64_SHORT: return launch_tile<2, 2, 2>(g, p.parts);
    case TILE_64: return launch_tile<2, 2, 4>(g, p.parts);
    case TILE_64_DEEP: return launch_tile<2, 2, 8>(g, p.parts);
    case TILE_64x128: return launch_tile<2, 4, 4>(g, p.parts);
    case TILE_128: return launch_tile<4, 4, 4>(g, p.parts);
  }
  const dim3 tiles((unsigned)(((g.m + 255) / 256) * ((g.n + 255) / 256)));
  bool direct = (g.e.out_kind == BF16 || g.e.out_kind == F16) && g.e.nops <= DIRECT_OPS && g.n % 128 == 0 &&
                (uintptr_t)g.c % 8 == 0 && 256 * g.n <= 0x7fffffff;
  for (int i = 0; i < g.e.nops; ++i) {
    const int op = g.e.op[i] & ((1 << VEC_KIND_SHIFT) - 1);
    direct &= op < RELU && (op % 3 != 1 || g.m % 128 == 0);  // it reads a row vector for whole quarters
  }
  auto kernel = g.nb % SLAB == 0 ? (direct ? mx_quad<false, true> : mx_quad<false, false>)
                                 : (direct ? mx_quad<true, true> : mx_quad<true, false>);
  hipLaunchKernelGGL(kernel, tiles, dim3(256), 0, g.stream, g.a, g.as, g.b, g.bs, g.c, g.m, g.n, g.nb, g.n, g.e);
  return launched("mx_gemm");
}

// Whether a product of these sizes is taken
static bool mx_sizes(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 1 && k < (int64_t)1 << 23 && m < (int64_t)1 << 28 && n < (int64_t)1 << 28 &&
         ((m + 63) / 64) * ((n + 63) / 64) < (int64_t)1 << 24;
}

extern "C" {

int krn_mx_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, void* c, int out_kind, int64_t m,
                int64_t n, int64_t k, int nops, const int* ops, const float* scalars, const void* const* vectors,
                void* workspace, int64_t workspace_bytes, void* stream) {
  MxCall g{};
  if (!mx_epilogue(g.e, out_kind, nops, ops, scalars, vectors)) return -1;
  // 256 rows of codes are addressed by 31-bit offsets; a launch has fewer than 2^32 threads, 256 for a tile of 64 x 64 (few rows:
  // mx_plan)
  if (!mx_sizes(m, n, k)) {
    krn_set_error("mx_gemm: %lld x %lld x %lld; rows of 1 to 2^23 - 1 values, m and n below 2^28, fewer than 2^24 tiles of "
                  "64 x 64", (long long)m, (long long)n, (long long)k);
    return -1;
  }
  if ((uintptr_t)a % 16 != 0 || (uintptr_t)b % 16 != 0 || (uintptr_t)workspace % 16 != 0) {
    krn_set_error("mx_gemm: codes and workspace start at 16-byte aligned addresses");
    return -1;
  }
  if (m == 0 || n == 0) return 0;
  const int64_t nb = mx_blocks(k), c_bytes = m * n * (out_kind == F32 ? 4 : 2);
  if (share_memory(c, c_bytes, a, m * nb * 16) || share_memory(c, c_bytes, b, n * nb * 16) ||
      share_memory(c, c_bytes, a_scales, m * nb) || share_memory(c, c_bytes, b_scales, n * nb)) {
    krn_set_error("mx_gemm: the result shares memory with an operand");
    return -1;
  }
  for (int i = 0; i < nops; ++i) {
    const int op = ops[i] & ((1 << VEC_KIND_SHIFT) - 1), size = ops[i] >> VEC_KIND_SHIFT ? 2 : 4;
    if (op < RELU && op % 3 != 0 && share_memory(c, c_bytes, vectors[i], (op % 3 == 1 ? m : n) * size)) {
      krn_set_error("mx_gemm: the result shares memory with a vector of the epilogue");
      return -1;
    }
  }
  g.a = (const uint8_t*)a, g.as = (const uint8_t*)a_scales, g.b = (const uint8_t*)b, g.bs = (const uint8_t*)b_scales;
  g.c = c, g.m = m, g.n = n, g.nb = (int)nb, g.workspace = workspace, g.stream = (hipStream_t)stream;
  bool activation = false;
  for (int i = 0; i < nops; ++i) activation |= (ops[i] & ((1 << VEC_KIND_SHIFT) - 1)) >= RELU;
  return launch_planned(mx_plan(m, n, nb, activation, workspace ? workspace_bytes : 0), g);
}

int64_t krn_mx_gemm_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const int64_t plain = mx_plan(m, n, mx_blocks(k), false, INT64_MAX).workspace, with = mx_plan(m, n, mx_blocks(k), true, INT64_MAX).workspace;
  return plain > with ? plain : with;
}

const char* krn_mx_gemm_kernel(int64_t m, int64_t n, int64_t k, int activation, int64_t workspace_bytes) {
  if (!mx_sizes(m, n, k) || m == 0 || n == 0) return "";
  const MxPlan p = mx_plan(m, n, mx_blocks(k), activation != 0, workspace_bytes);
  if (p.parts == 1) return SHAPE_NAMES[p.shape];
  thread_local char name[48];
  snprintf(name, sizeof name, "%s in %d parts", SHAPE_NAMES[p.shape], p.parts);
  return name;
}

}  // extern "C"
