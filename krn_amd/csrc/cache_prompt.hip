// Causal attention of packed prompts over a paged cache, for rows enough to fill the matrix cores.
//
// A workgroup has 256 rows of one key head: row r of a sequence is its token r / group, query head r % group of the key head's
// `group`. So shared heads lie side by side, short prompts fill tiles, and a causal tile is 256 / group tokens wide. Each of
// its eight waves owns 32 rows and computes S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs: a lane holds one row
// (lane & 31) and half of the keys (its partner is lane ^ 32), P stays in its lane.
//
// The matrix cores bound it, and a SIMD has two waves, one of the workgroup's lower four and one of its upper four. They
// take turns: a tile of 64 keys is four phases, S(t + 1) | half of the weights of t, V's fragments | O += P V | the maximum of t + 1
// and half of its weights, K's fragments; a barrier ends each, and the upper waves are one phase behind. While one wave's
// MFMAs run, the other's vector instructions and LDS reads do.
//
// K and V come into rings of four tiles by direct loads, K four tiles ahead of its use and V three, so that a wait finds them
// there; tiles past the end are asked for with no bytes, which keeps the count of loads on their way the same. Sixteen
// keys lie in one page, whose rows up to the sequence's end are a buffer resource: rows past it, and pages that are not
// there, read as zeros.
#include "attention_parts.h"
#include "cache_parts.h"

namespace krn {

constexpr int PROMPT_TILE = 64;                         // keys
constexpr int PROMPT_RING = 4;                          // tiles of K, and of V

// The tokens of slot `slot`: 256 rows of a sequence. Sequence i has the slots from first_slot(i) on, enough for its rows since
// starts are sums of what came before; a wave looks at 64 sequences at a time.
struct PromptTile {
  int seq, row0;
  TokenRange range;
};
__device__ __forceinline__ int64_t first_slot(const PromptCall& c, int i) {
  const int start = min(max(c.s.starts[i], 0), c.s.tokens);
  return (int64_t)start * c.group / PROMPT_ROWS + i;
}
__device__ __forceinline__ bool find_tile(const PromptCall& c, int slot, PromptTile& tile) {
  int seq, at;
  if (c.s.starts) {
    const int lane = threadIdx.x & 63;
    int low = 0, count = c.s.n;  // the last sequence of low to low + count - 1 whose first slot is this one or before
    while (count > 1) {
      const int step = (count + 63) / 64, i = lane * step;
      const uint64_t before = __builtin_amdgcn_ballot_w64(i < count && first_slot(c, low + min(i, count - 1)) <= slot);
      const int k = before ? 63 - __builtin_clzll(before) : 0;
      low += k * step;
      count = min(step, count - k * step);
    }
    seq = __builtin_amdgcn_readfirstlane(low);
    const int64_t from = slot - first_slot(c, seq);
    at = from < 0 || from > 0xffffff ? -1 : (int)from;
  } else {
    const int per = (c.s.step * c.group + PROMPT_ROWS - 1) / PROMPT_ROWS;
    seq = slot / per, at = slot % per;
  }
  tile.seq = __builtin_amdgcn_readfirstlane(seq);
  tile.range = token_range(c.s, tile.seq);
  tile.range.first = __builtin_amdgcn_readfirstlane(tile.range.first);
  tile.range.count = __builtin_amdgcn_readfirstlane(tile.range.count);
  at = __builtin_amdgcn_readfirstlane(at);
  tile.row0 = at * PROMPT_ROWS;
  return at >= 0 && (int64_t)at * PROMPT_ROWS < (int64_t)tile.range.count * c.group;
}

// V^T fragments of a tile: [step][block of 32 columns], a lane the keys of its P and one column. One assembly block with
// its wait: as builtins the compiler waits for the tiles on their way before the first of them.
template <int D>
__device__ __forceinline__ void value_tile(uint32_t at, u32x4 (&v)[4][D / 32]) {
  u32x2 w[4 * (D / 32) * 2];
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %32\n\t"
        "ds_read_b64_tr_b16 %1, %32 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %33\n\t"
        "ds_read_b64_tr_b16 %3, %33 offset:2048\n\t"
        "ds_read_b64_tr_b16 %4, %34\n\t"
        "ds_read_b64_tr_b16 %5, %34 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %35\n\t"
        "ds_read_b64_tr_b16 %7, %35 offset:2048\n\t"
        "ds_read_b64_tr_b16 %8, %32 offset:4096\n\t"
        "ds_read_b64_tr_b16 %9, %32 offset:6144\n\t"
        "ds_read_b64_tr_b16 %10, %33 offset:4096\n\t"
        "ds_read_b64_tr_b16 %11, %33 offset:6144\n\t"
        "ds_read_b64_tr_b16 %12, %34 offset:4096\n\t"
        "ds_read_b64_tr_b16 %13, %34 offset:6144\n\t"
        "ds_read_b64_tr_b16 %14, %35 offset:4096\n\t"
        "ds_read_b64_tr_b16 %15, %35 offset:6144\n\t"
        "ds_read_b64_tr_b16 %16, %32 offset:8192\n\t"
        "ds_read_b64_tr_b16 %17, %32 offset:10240\n\t"
        "ds_read_b64_tr_b16 %18, %33 offset:8192\n\t"
        "ds_read_b64_tr_b16 %19, %33 offset:10240\n\t"
        "ds_read_b64_tr_b16 %20, %34 offset:8192\n\t"
        "ds_read_b64_tr_b16 %21, %34 offset:10240\n\t"
        "ds_read_b64_tr_b16 %22, %35 offset:8192\n\t"
        "ds_read_b64_tr_b16 %23, %35 offset:10240\n\t"
        "ds_read_b64_tr_b16 %24, %32 offset:12288\n\t"
        "ds_read_b64_tr_b16 %25, %32 offset:14336\n\t"
        "ds_read_b64_tr_b16 %26, %33 offset:12288\n\t"
        "ds_read_b64_tr_b16 %27, %33 offset:14336\n\t"
        "ds_read_b64_tr_b16 %28, %34 offset:12288\n\t"
        "ds_read_b64_tr_b16 %29, %34 offset:14336\n\t"
        "ds_read_b64_tr_b16 %30, %35 offset:12288\n\t"
        "ds_read_b64_tr_b16 %31, %35 offset:14336\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]),
          "=&v"(w[8]), "=&v"(w[9]), "=&v"(w[10]), "=&v"(w[11]), "=&v"(w[12]), "=&v"(w[13]), "=&v"(w[14]), "=&v"(w[15]),
          "=&v"(w[16]), "=&v"(w[17]), "=&v"(w[18]), "=&v"(w[19]), "=&v"(w[20]), "=&v"(w[21]), "=&v"(w[22]), "=&v"(w[23]),
          "=&v"(w[24]), "=&v"(w[25]), "=&v"(w[26]), "=&v"(w[27]), "=&v"(w[28]), "=&v"(w[29]), "=&v"(w[30]), "=&v"(w[31])
        : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16\n\t"
        "ds_read_b64_tr_b16 %1, %16 offset:1024\n\t"
        "ds_read_b64_tr_b16 %2, %17\n\t"
        "ds_read_b64_tr_b16 %3, %17 offset:1024\n\t"
        "ds_read_b64_tr_b16 %4, %16 offset:2048\n\t"
        "ds_read_b64_tr_b16 %5, %16 offset:3072\n\t"
        "ds_read_b64_tr_b16 %6, %17 offset:2048\n\t"
        "ds_read_b64_tr_b16 %7, %17 offset:3072\n\t"
        "ds_read_b64_tr_b16 %8, %16 offset:4096\n\t"
        "ds_read_b64_tr_b16 %9, %16 offset:5120\n\t"
        "ds_read_b64_tr_b16 %10, %17 offset:4096\n\t"
        "ds_read_b64_tr_b16 %11, %17 offset:5120\n\t"
        "ds_read_b64_tr_b16 %12, %16 offset:6144\n\t"
        "ds_read_b64_tr_b16 %13, %16 offset:7168\n\t"
        "ds_read_b64_tr_b16 %14, %17 offset:6144\n\t"
        "ds_read_b64_tr_b16 %15, %17 offset:7168\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]),
          "=&v"(w[8]), "=&v"(w[9]), "=&v"(w[10]), "=&v"(w[11]), "=&v"(w[12]), "=&v"(w[13]), "=&v"(w[14]), "=&v"(w[15])
        : "v"(at), "v"(at ^ 64)
        : "memory");
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const u32x2 a = w[(s * (D / 32) + i) * 2], b = w[(s * (D / 32) + i) * 2 + 1];
      v[s][i] = u32x4{a[0], a[1], b[0], b[1]};
    }
}

#define KRN_PHASE()                         \
  do {                                      \
    __builtin_amdgcn_sched_barrier(0);      \
    asm volatile("" ::: "memory");          \
    __builtin_amdgcn_s_barrier();           \
    asm volatile("" ::: "memory");          \
    __builtin_amdgcn_sched_barrier(0);      \
  } while (0)

template <bool BF, int D>
__global__ __launch_bounds__(512, 2) void cache_prompt(PromptCall c) {
  constexpr int RB = D * 2, DCH = D / 8, TILE = PROMPT_TILE * RB, LOADS = TILE / 8 / 1024, STEPS = D / 16, BLOCKS = D / 32;
  static_assert(LOADS >= 1, "whole loads a wave");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * PROMPT_RING * TILE];
  const int column = (int)(blockIdx.x % c.kv_heads), slot = c.slots - 1 - (int)(blockIdx.x / c.kv_heads);
  PromptTile tile;
  if (!find_tile(c, slot, tile)) return;
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5, r32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int length = __builtin_amdgcn_readfirstlane(sequence_length(c.s, tile.seq));
  const int end = __builtin_amdgcn_readfirstlane(held_keys(c.s, length, c.cache.page_shift));
  const int before = length - tile.range.count;  // the position of the sequence's first token here

  // this lane's row, the keys that it sees, and those that all or some rows of the wave and the workgroup see
  const int row = tile.row0 + wave * 32 + r32, j = row / c.group;
  const bool real = j < tile.range.count;
  const int limit = min(before + min(j, tile.range.count - 1) + 1, end), low = first_key(before + min(j, tile.range.count - 1), c.window);
  const int all_limit = __builtin_amdgcn_readfirstlane(limit), all_low = __builtin_amdgcn_readlane(low, 31);
  const int last_token = __builtin_amdgcn_readfirstlane(min((tile.row0 + PROMPT_ROWS - 1) / c.group, tile.range.count - 1));
  const int key_end = min(before + last_token + 1, end);
  const int first = __builtin_amdgcn_readfirstlane(first_key(before + tile.row0 / c.group, c.window) / PROMPT_TILE);
  const int n = __builtin_amdgcn_readfirstlane((key_end + PROMPT_TILE - 1) / PROMPT_TILE) - first;
  const int64_t place = ((int64_t)(tile.range.first + j) * c.heads + column * c.group + (row - j * c.group)) * D;
  if (n <= 0 || key_end <= 0) {  // no row sees a key
    if (real)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) *reinterpret_cast<u32x4*>(c.o + place + s * 16 + half * 8) = u32x4{};
    return;
  }

  u32x4 qf[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) qf[s] = real ? *reinterpret_cast<const u32x4*>(c.q + place + s * 16 + half * 8) : u32x4{};

  // this wave's eight keys of a tile, half of a group of sixteen
  const int group = wave >> 1;
  uint32_t koff[LOADS], voff[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int key = (wave & 1) * 8 + i * (1024 / RB) + lane / DCH, s = lane % DCH;  // in the group
    const int in_tile = group * 16 + key;
    koff[i] = (uint32_t)(key * RB + k_slot<D>(in_tile, s) * 16);
    voff[i] = (uint32_t)(key * RB + v_slot<D>(in_tile, s) * 16);
  }
  const __attribute__((address_space(4))) int* table =
      (const __attribute__((address_space(4))) int*)(uintptr_t)(c.s.table + (int64_t)tile.seq * c.s.width);
  const int shift = c.cache.page_shift;
  // the page of this wave's group in tile u, or -1
  const auto page_of = [&](int u) {
    const int at = ((first + u) * PROMPT_TILE + group * 16) >> shift;
    return u < n && at < c.s.width ? table[at] : -1;
  };
  const auto load = [&](const void* data, int number, int u, int ring, const uint32_t(&off)[LOADS]) {
    const int key0 = (first + u) * PROMPT_TILE + group * 16;
    const bool there = (uint32_t)number < (uint32_t)c.cache.pages;
    const int64_t at = ((((int64_t)(there ? number : 0) * c.kv_heads + column) << shift) + (key0 & ((1 << shift) - 1))) * RB;
    const int bytes = __builtin_amdgcn_readfirstlane(there ? max(0, min(16, end - key0)) * RB : 0);
    const __amdgpu_buffer_rsrc_t r = panel_rsrc((const uint8_t*)data + at, bytes);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) buffer_to_lds16(r, lds + ring + wave * (TILE / 8) + i * 1024, off[i], 0);
  };
  constexpr int V_RING = PROMPT_RING * TILE;
  const auto ring_of = [](int u) { return (u & (PROMPT_RING - 1)) * TILE; };

  // fragments: K's as A operands (lane = key, 8 columns of step s), V^T's (lane = column, keys as the lane's P has them)
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const uint32_t kat = lds_at + r32 * RB + k_slot<D>(r32, half) * 16;
  const int a16 = lane & 15, tr_key = (lane >> 5) * 4 + (a16 >> 2), tr_col = ((lane >> 4) & 1) * 16 + 4 * (a16 & 3);
  const uint32_t vat = lds_at + V_RING + tr_key * RB + v_slot<D>(tr_key, tr_col >> 3) * 16 + (tr_col & 7) * 2;
  u32x4 kf[2][STEPS];
  const auto read_keys = [&](int ring) {
    const uint32_t at = kat + ring;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        kf[h][s] = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)((at ^ (s << 5)) + h * 32 * RB);
  };
  u32x4 vf[4][BLOCKS];

  f32x16 acc[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) acc[i] = f32x16{};
  float m = -INFINITY, base = 0.0f, total = 0.0f;  // base: m, or 0 while no key has been seen
  f32x16 s0, s1;  // scores of both halves
  u32x4 pf[4];
  const auto scores = [&]() {
    s0 = f32x16{}, s1 = f32x16{};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      Half<BF>::mma(s0, kf[0][s], qf[s]);
      Half<BF>::mma(s1, kf[1][s], qf[s]);
    }
  };
  // weights of one half: p = 2^(s scale - base), packed as two steps of P^T
  const auto weights = [&](const f32x16& s, int h) {
    float sum = 0.0f;
#pragma unroll
    for (int step = 0; step < 2; ++step)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step * 8 + 2 * e], c.scale, -base));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step * 8 + 2 * e + 1], c.scale, -base));
        sum += p0 + p1;
        pf[h * 2 + step][e] = Half<BF>::pack(p0, p1);
      }
    total += sum;
  };
  // the maximum and the weights of tile u
  const auto begin = [&](int u) {
    const int key0 = (first + u) * PROMPT_TILE;
    if (key0 < all_low || key0 + PROMPT_TILE > all_limit) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = key0 + half * 4 + (r >> 2) * 8 + (r & 3);
        s0[r] = key >= limit || key < low ? -INFINITY : s0[r];
        s1[r] = key + 32 >= limit || key + 32 < low ? -INFINITY : s1[r];
      }
    }
    float top = s0[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s0[r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s1[r]);
    top *= c.scale;
    // the base moves only when a weight would exceed 2^8: then acc and total are rescaled
    if (__builtin_amdgcn_ballot_w64(top > m + 8.0f) != 0) {
      const float next = fmaxf(m, pair_max(top)), to_base = next == -INFINITY ? 0.0f : next;
      const float corr = __builtin_amdgcn_exp2f(m - to_base);
      total *= corr;
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= corr;
      m = next, base = to_base;
    }
    weights(s0, 0);
    weights(s1, 1);
  };

  // page numbers one load ahead
  int k_page[PROMPT_RING], next_k, next_v;
#pragma unroll
  for (int u = 0; u < PROMPT_RING; ++u) k_page[u] = page_of(u);
  next_k = page_of(PROMPT_RING), next_v = k_page[3];
  load(c.cache.keys, k_page[0], 0, ring_of(0), koff);
  load(c.cache.keys, k_page[1], 1, ring_of(1), koff);
  load(c.cache.values, k_page[0], 0, V_RING + ring_of(0), voff);
  load(c.cache.keys, k_page[2], 2, ring_of(2), koff);
  load(c.cache.values, k_page[1], 1, V_RING + ring_of(1), voff);
  load(c.cache.keys, k_page[3], 3, ring_of(3), koff);
  load(c.cache.values, k_page[2], 2, V_RING + ring_of(2), voff);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * LOADS) : "memory");  // the first two K tiles and the first V tile
#pragma unroll
  for (int s = 0; s < STEPS; ++s) asm volatile("" : "+v"(qf[s]));  // older loads: no wait for them in the loop
  KRN_PHASE();
  read_keys(ring_of(0));
  scores();
  begin(0);
  read_keys(ring_of(1));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  KRN_PHASE();  // everyone has read the first tile: its place may be loaded
  if (wave >= 4) KRN_PHASE();
  for (int u = 0; u < n; ++u) {
    load(c.cache.keys, next_k, u + 4, ring_of(u), koff);
    load(c.cache.values, next_v, u + 3, V_RING + ring_of(u + 3), voff);
    __builtin_amdgcn_s_setprio(1);
    scores();
    asm volatile("" : "+v"(s0), "+v"(s1));  // here, not where they are used
    __builtin_amdgcn_s_setprio(0);
    KRN_PHASE();
    value_tile<D>(vat + ring_of(u), vf);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * LOADS) : "memory");  // K of u + 2 and V of u + 1
    KRN_PHASE();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) Half<BF>::mma(acc[i], vf[s][i], pf[s]);
    __builtin_amdgcn_s_setprio(0);
    KRN_PHASE();
    next_v = next_k, next_k = page_of(u + 5);
    read_keys(ring_of(u + 2));
    if (u + 1 < n) begin(u + 1);
    KRN_PHASE();
  }
  if (wave < 4) KRN_PHASE();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup

  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(total), __float_as_uint(total), false, false);
    total = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // no key: zeros
  // lane (r32, half) has columns i * 32 + gq * 8 + half * 4 to + 3; its partner's four complete 16 bytes
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
    for (int gp = 0; gp < 2; ++gp) {
      uint32_t w[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = (2 * gp + e) * 4;
        w[e][0] = Half<BF>::pack(acc[i][at] * inv, acc[i][at + 1] * inv);
        w[e][1] = Half<BF>::pack(acc[i][at + 2] * inv, acc[i][at + 3] * inv);
      }
      uint32_t got[2];
#pragma unroll
      for (int word = 0; word < 2; ++word) {
        const auto sw = __builtin_amdgcn_permlane32_swap(w[0][word], w[1][word], false, false);
        got[word] = half ? sw[0] : sw[1];
      }
      const u32x4 piece = half ? u32x4{got[0], got[1], w[1][0], w[1][1]} : u32x4{w[0][0], w[0][1], got[0], got[1]};
      if (real) *reinterpret_cast<u32x4*>(c.o + place + i * 32 + (2 * gp + half) * 8) = piece;
    }
}
#undef KRN_PHASE

}  // namespace krn

using namespace krn;

int64_t krn::prompt_slots(int64_t tokens, int64_t step, int64_t group, int64_t sequences) {
  if (step > 0) return sequences * ((step * group + PROMPT_ROWS - 1) / PROMPT_ROWS);
  return tokens * group / PROMPT_ROWS + sequences;
}

void krn::launch_cache_prompt(bool bf, int d, const PromptCall& c, hipStream_t stream) {
  const dim3 grid((unsigned)(c.slots * c.kv_heads)), block(512);
  if (bf && d == 128) hipLaunchKernelGGL((cache_prompt<true, 128>), grid, block, 0, stream, c);
  else if (bf) hipLaunchKernelGGL((cache_prompt<true, 64>), grid, block, 0, stream, c);
  else if (d == 128) hipLaunchKernelGGL((cache_prompt<false, 128>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((cache_prompt<false, 64>), grid, block, 0, stream, c);
}
