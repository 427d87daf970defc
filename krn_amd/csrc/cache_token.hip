// Attention of a few new tokens a sequence over a paged cache: the rows of one key head (its query heads times the new tokens)
// are multiplied with the head's keys and values, which are read once. What bounds it is that stream, so the keys of a
// sequence are shared out over workgroups and joined by a second kernel.
//
// Shares. A tile is 32 keys. With T tiles in all sequences and C key heads, a part has at most chunk = max(TOKEN_CHUNK, T C
// / TOKEN_PARTS) tiles, and sequence i is ceil(tiles_i / chunk) parts of equal size: long and short sequences together keep
// every CU busy to the end. Only the device knows the lengths, so each wave counts the parts before its own or, with more
// than 128 sequences, a workgroup does for all (2000 sequences, one of 60000 keys and the others of 100: 259 us, by each
// wave 866).
//
// A wave computes S^T = K Q^T and O^T += V^T P^T with 16x16x32 MFMAs on its own tiles. A lane then holds one query row
// (lane & 15) and eight keys of a tile: keys 4 g + r and 16 + 4 g + r, g = lane / 16, which are also the eight that it gives
// the second product, so P goes from registers to registers. The maximum is exchanged between lanes only when a row exceeds the
// running one by more than 2^8 in weight. P is kept in two 16-bit parts (what is left: 2^-17 of a weight in bf16; 2^-23 in f16,
// or 2^-32 of the largest weight if that is more): the matrix cores are idle nine tenths of the time.
//
// K and V tiles come into LDS by direct loads, one buffer each a wave and no barrier: K's next tile leaves when this one's
// fragments are in registers, V's likewise, so 8 to 16 KiB a wave are always on their way. The loads are non-temporal: a step
// reads its whole cache before it reads a line again (196 us with plain ones, 176 with these; caches that stay in the last-level
// cache between steps lose nothing: one sequence of 4096 keys 11.8 and 11.3). Sixteen keys lie in one page,
// whose rows up to the sequence's end are a buffer resource: rows past it, and pages that are not there, read as zeros.
#include "cache_parts.h"

namespace krn {

// the B operand's 16-bit parts and the products, by format
template <bool BF>
struct Narrow {
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return f2bf2(lo, hi); }
  static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <>
struct Narrow<false> {
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return (uint32_t)f2h(lo) | ((uint32_t)f2h(hi) << 16); }
  static __device__ __forceinline__ float low(uint32_t w) { return h2f((uint16_t)(w & 0xffff)); }
  static __device__ __forceinline__ float high(uint32_t w) { return h2f((uint16_t)(w >> 16)); }
};

// The 16-byte chunk of a row that lies in slot `slot` of its row in LDS, so that reads of sixteen rows spread over the banks:
// K's take one chunk of each row, V's transposed reads 32 bytes of each.
template <int D>
__device__ __forceinline__ int key_chunk(int row, int slot) {
  return D == 128 ? slot ^ (row & 15) : slot ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int value_chunk(int row, int slot) {
  return D == 128 ? slot ^ ((row & 7) << 1) : slot ^ (((row >> 1) & 3) << 1);
}

// fragments of both 16-key halves of a K tile: A operands, lane = key, 8 columns of step s
template <int D>
__device__ __forceinline__ void key_fragments(uint32_t at, u32x4 (&k)[2][D / 32]) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
        "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\t"
        "ds_read_b128 %7, %11 offset:4096\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(k[1][2]),
          "=&v"(k[1][3])
        : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %5 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[1][0]), "=&v"(k[1][1])
        : "v"(at), "v"(at ^ 64)
        : "memory");
  }
}

// V^T fragments of four blocks of 16 columns, each four keys of both halves
template <int D>
__device__ __forceinline__ void value_fragments(uint32_t at, u32x4 (&v)[4]) {
  u32x2 w[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\tds_read_b64_tr_b16 %2, %9\n\t"
      "ds_read_b64_tr_b16 %3, %9 offset:%12\n\tds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7])
      : "v"(at), "v"(at ^ 32), "v"(at ^ 64), "v"(at ^ 96), "n"(16 * D * 2)
      : "memory");
#pragma unroll
  for (int b = 0; b < 4; ++b) v[b] = u32x4{w[2 * b][0], w[2 * b][1], w[2 * b + 1][0], w[2 * b + 1][1]};
}

// the largest value of the four lanes that hold one row
__device__ __forceinline__ float row_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The tiles of a sequence that its new tokens see: keys from the first one's window to the end
struct TileRange {
  int first, count;
};
__device__ __forceinline__ TileRange tiles_of(const TokenCall& c, int length) {
  const int end = held_keys(c.s, length, c.cache.page_shift);
  const int low = first_key(length - c.s.step, c.window);
  const int first = low / 32;
  return {first, low < end ? (end + 31) / 32 - first : 0};
}

// What workgroup w of a column does: part `part` of `parts` of sequence `seq`, the `order`-th of those in several parts
struct Share {
  int seq, part, parts, order;
};

__device__ __forceinline__ uint32_t weight_of(const TokenCall& c, int i) {
  return (uint32_t)min(tiles_of(c, sequence_length(c.s, i)).count, TOKEN_TILES);
}
__device__ __forceinline__ uint32_t chunk_of(const TokenCall& c, uint32_t tiles) {
  return max((uint32_t)TOKEN_CHUNK, (tiles + c.shares - 1) / c.shares);
}
__device__ __forceinline__ uint32_t parts_of(uint32_t weight, uint32_t chunk) { return max(1u, (weight + chunk - 1) / chunk); }
// parts in the low half, sequences of several in the high one
__device__ __forceinline__ uint32_t packed(uint32_t parts) { return parts + (parts > 1 ? 0x10000u : 0u); }

// Every wave counts for itself, a lane for up to TOKEN_HELD sequences in a row, so that no barrier is needed. More
// sequences are counted by a launch before this one.
__device__ __forceinline__ bool find_share(const TokenCall& c, int w, bool writes, Share& share) {
  if (!c.split) {
    share = {w, 0, 1, 0};
    return true;
  }
  if (c.map) {
    const int4 at = c.map[w];
    share = {__builtin_amdgcn_readfirstlane(at.x), __builtin_amdgcn_readfirstlane(at.y), __builtin_amdgcn_readfirstlane(at.z),
             __builtin_amdgcn_readfirstlane(at.w)};
    return share.seq >= 0;
  }
  const int lane = threadIdx.x & 63, per = (c.s.n + 63) / 64, first = lane * per, mine = max(0, min(per, c.s.n - first));
  uint32_t held[TOKEN_HELD], tiles = 0;
#pragma unroll
  for (int k = 0; k < TOKEN_HELD; ++k) {
    held[k] = k < mine ? weight_of(c, first + k) : 0;
    tiles += held[k];
  }
  tiles = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(tiles), 63);
  const uint32_t chunk = chunk_of(c, tiles);
  uint32_t count = 0;
#pragma unroll
  for (int k = 0; k < TOKEN_HELD; ++k) {
    held[k] = k < mine ? parts_of(held[k], chunk) : 0;
    count += packed(held[k]);
  }
  const uint32_t upto = wave_scan(count), all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  if (writes && w == 0 && threadIdx.x == 0) c.header[0] = {(int)(all >> 16), 0, 0, 0};
  uint32_t before = upto - count;
  const uint64_t owner = __builtin_amdgcn_ballot_w64((int)(before & 0xffff) <= w && w < (int)(upto & 0xffff));
  if (owner == 0) return false;
  int seq = first, parts = 1;
  bool found = false;
#pragma unroll
  for (int k = 0; k < TOKEN_HELD; ++k) {  // in the owner's lane: its sequence
    if (found || k >= mine) continue;
    seq = first + k, parts = (int)held[k];
    found = w < (int)(before & 0xffff) + parts;
    if (!found) before += packed(held[k]);
  }
  const int from = __builtin_ctzll(owner);
  share.seq = __builtin_amdgcn_readlane(seq, from), share.parts = __builtin_amdgcn_readlane(parts, from);
  before = (uint32_t)__builtin_amdgcn_readlane((int)before, from);
  share.part = w - (int)(before & 0xffff), share.order = (int)(before >> 16);
  return true;
}

// The same for many sequences, once: the share of every workgroup of a column, a thread for `per` sequences in a row
constexpr int MAP_THREADS = 1024;
__global__ __launch_bounds__(MAP_THREADS) void cache_shares(TokenCall c, int workgroups) {
  __shared__ uint32_t sums[2][MAP_THREADS / 64];
  const int t = threadIdx.x, lane = t & 63, per = (c.s.n + MAP_THREADS - 1) / MAP_THREADS, first = t * per;
  const int mine = max(0, min(per, c.s.n - first));
  // the sum up to this thread, and of all
  const auto scan = [&](uint32_t x, uint32_t* wave, uint32_t& all) {
    const uint32_t upto = wave_scan(x);
    if (lane == 63) wave[t / 64] = upto;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
    for (int i = 0; i < MAP_THREADS / 64; ++i) {
      before += i < t / 64 ? wave[i] : 0;
      all += wave[i];
    }
    return before + upto;
  };
  uint32_t tiles = 0, all;
  for (int k = 0; k < mine; ++k) tiles += weight_of(c, first + k);
  scan(tiles, sums[0], all);
  const uint32_t chunk = chunk_of(c, all);
  uint32_t count = 0;
  for (int k = 0; k < mine; ++k) count += packed(parts_of(weight_of(c, first + k), chunk));
  uint32_t before = scan(count, sums[1], all) - count;
  for (int k = 0; k < mine; ++k) {
    const int parts = (int)parts_of(weight_of(c, first + k), chunk), from = (int)(before & 0xffff), order = (int)(before >> 16);
    for (int p = 0; p < parts && from + p < workgroups; ++p) c.map[from + p] = {first + k, p, parts, order};
    before += packed((uint32_t)parts);
  }
  for (int w = (int)(all & 0xffff) + t; w < workgroups; w += MAP_THREADS) c.map[w] = {-1, 0, 0, 0};
  if (t == 0) c.header[0] = {(int)(all >> 16), 0, 0, 0};
}

template <bool BF, int D, int NB>
__global__ __launch_bounds__(64 * TOKEN_WAVES, 2) void cache_tokens(TokenCall c) {
  constexpr int RB = D * 2, DCH = D / 8, HALF = 16 * RB, TILE = 2 * HALF, LOADS = HALF / 1024;
  constexpr int OLD = D + 4;  // floats per row of a wave's O in LDS
  static_assert(16 * OLD * 4 <= 2 * TILE, "a wave's rows fit its buffers");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[TOKEN_WAVES * 2 * TILE];
  __shared__ float stat[2][TOKEN_WAVES][16];
  const int w = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / c.cache.kv_heads)), kv = (int)blockIdx.x - w * c.cache.kv_heads;
  Share share;
  if (!find_share(c, w, kv == 0, share)) return;
  const int seq = share.seq, part = share.part, parts = share.parts;
  const int t = threadIdx.x, lane = t & 63, g = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // parts of the sequences in several before this one: all parts, less the sequences in one
  const int place = w - (seq - share.order);
  if (parts > 1 && part == 0 && kv == 0 && t == 0) c.header[1 + share.order] = {seq, place, parts, 0};

  const int length = __builtin_amdgcn_readfirstlane(sequence_length(c.s, seq)), end = held_keys(c.s, length, c.cache.page_shift);
  const TileRange range = tiles_of(c, length);
  // the part's tiles and this wave's (below 2^26), in scalar registers, where a division leaves none
  const int even = __builtin_amdgcn_readfirstlane(range.count / parts), over = range.count - even * parts;
  const int begin = range.first + even * part + min(part, over), count = even + (part < over ? 1 : 0);
  const int first = begin + count * wave / TOKEN_WAVES, last = begin + count * (wave + 1) / TOKEN_WAVES;

  // queries as B operands (lane = row, 8 columns of step s) and the keys that each row sees, [low, limit)
  u32x4 qf[NB][D / 32];
  int limit[NB], low[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int r = b * 16 + col, j = r / c.group;
    const bool real = r < c.rows;
    const uint16_t* q = c.q + (((int64_t)seq * c.s.step + j) * c.heads + kv * c.group + (r - j * c.group)) * D;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) qf[b][s] = real ? *reinterpret_cast<const u32x4*>(q + s * 32 + g * 8) : u32x4{};
    const int position = length - c.s.step + j;
    limit[b] = real ? min(position + 1, end) : end;
    low[b] = real ? first_key(position, c.window) : 0;
  }
  // tiles in these bounds have no masked key
  const int all_low = first_key(length - 1, c.window), all_limit = min(length - c.s.step + 1, end);

  uint8_t *kbuf = lds + wave * 2 * TILE, *vbuf = kbuf + TILE;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)kbuf;
  const uint32_t kat = lds_at + col * RB + key_chunk<D>(col, g) * 16;
  const int vrow = g * 4 + (col >> 2);
  const uint32_t vat = lds_at + TILE + vrow * RB + value_chunk<D>(vrow, 0) * 16 + (col & 3) * 8;
  uint32_t koff[LOADS], voff[LOADS];  // byte offsets within sixteen keys
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int row = j * (1024 / RB) + lane / DCH, s = lane % DCH;
    koff[j] = (uint32_t)(row * RB + key_chunk<D>(row, s) * 16);
    voff[j] = (uint32_t)(row * RB + value_chunk<D>(row, s) * 16);
  }

  // page numbers of 64 groups of sixteen keys, a lane each
  const int* table = c.s.table + (int64_t)seq * c.s.width;
  const int shift = c.cache.page_shift;
  int ids = -1, ids_from = 0;
  const auto fetch_ids = [&](int tile) {
    ids_from = tile * 2;
    const int64_t at = ((int64_t)(ids_from + lane) * 16) >> shift;
    ids = at < c.s.width ? table[at] : -1;
    asm volatile("" : "+v"(ids));  // waited for here: a use in the loop would wait for the tiles on their way each time
  };
  // the rows of sixteen keys from key0 on: where they start and how many bytes the sequence has there
  struct Group {
    int64_t at;
    int bytes;
  };
  const auto group_of = [&](int tile, int h) {
    const int number = __builtin_amdgcn_readlane(ids, tile * 2 + h - ids_from), key0 = tile * 32 + h * 16;
    const bool there = (uint32_t)number < (uint32_t)c.cache.pages;
    const int64_t row = ((((int64_t)(there ? number : 0) * c.cache.kv_heads + kv) << shift) + (key0 & ((1 << shift) - 1)));
    return Group{row * RB, __builtin_amdgcn_readfirstlane(there ? max(0, min(16, end - key0)) * RB : 0)};
  };
  Group now[2];  // of the tile whose V is next
  const auto load_keys = [&](int tile) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      now[h] = group_of(tile, h);
      const __amdgpu_buffer_rsrc_t r = panel_rsrc((const uint8_t*)c.cache.keys + now[h].at, now[h].bytes);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) buffer_to_lds16<true>(r, kbuf + h * HALF + j * 1024, koff[j], 0);
    }
  };
  const auto load_values = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __amdgpu_buffer_rsrc_t r = panel_rsrc((const uint8_t*)c.cache.values + now[h].at, now[h].bytes);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) buffer_to_lds16<true>(r, vbuf + h * HALF + j * 1024, voff[j], 0);
    }
  };

  f32x4 acc[NB][D / 16];
  // weights are 2^(x - base); exponents above `margin` move the base, to LIFT below them: the first one, then those 8 above that
  constexpr float BEGUN = LIFT<BF> + 8.0f;
  float base[NB], margin[NB], total[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    base[b] = 0.0f, margin[b] = -INFINITY, total[b] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[b][i] = f32x4{};
  }
  if (first < last) fetch_ids(first);
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int s = 0; s < D / 32; ++s) asm volatile("" : "+v"(qf[b][s]));  // here too, for the same reason
  if (first < last) load_keys(first), load_values();
  for (int tile = first; tile < last; ++tile) {
    const bool more = tile + 1 < last;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");  // K is here, V may be on its way
    u32x4 kf[2][D / 32];
    key_fragments<D>(kat, kf);
    if (more) {
      if ((tile + 1) * 2 - ids_from >= 64) fetch_ids(tile + 1);
      load_keys(tile + 1);
    }
    u32x4 ph[NB], pl[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x4 s[2] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) s[h] = Narrow<BF>::mma(kf[h][i], qf[b][i], s[h]);
      float x[8], top = -INFINITY;
      const int key = tile * 32 + g * 4;
      const bool masked = tile * 32 < all_low || tile * 32 + 32 > all_limit;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * c.scale;
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = key + (e >> 2) * 16 + (e & 3);
          if (k >= limit[b] || k < low[b]) x[e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
      // the base moves only when a weight would exceed its first by 2^8: then maxima meet, and acc and total are rescaled. What
      // is compared is the rounded exponent, so that no weight exceeds 2^15, f16's range, however large the scores are
      if (__builtin_amdgcn_ballot_w64(top - base[b] > margin[b]) != 0) {
        const float most = row_max(top);
        const bool moves = most - base[b] > margin[b], began = margin[b] == BEGUN;
        const float next = moves ? most - LIFT<BF> : base[b], corr = began ? __builtin_amdgcn_exp2f(base[b] - next) : 1.0f;
        total[b] *= corr;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[b][i] *= corr;
        base[b] = next, margin[b] = moves ? BEGUN : margin[b];
      }
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(x[2 * e] - base[b]), p1 = __builtin_amdgcn_exp2f(x[2 * e + 1] - base[b]);
        sum += p0 + p1;
        ph[b][e] = Narrow<BF>::pack(p0, p1);
        pl[b][e] = Narrow<BF>::pack(p0 - Narrow<BF>::low(ph[b][e]), p1 - Narrow<BF>::high(ph[b][e]));
      }
      total[b] += sum;
    }
    if (more)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");  // V is here, the next K may be on its way
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (tile * 32 < all_low || min(tile * 32 + 32, end) > all_limit) {  // keys that some rows see and some do not
      u32x4* here = reinterpret_cast<u32x4*>(vbuf) + lane;
      u32x4 held[TILE / 1024];
#pragma unroll
      for (int i = 0; i < TILE / 1024; ++i) held[i] = here[i * 64];
      if (__builtin_amdgcn_ballot_w64(any_endless<BF>(held)) != 0) {
#pragma unroll 1
        for (int k = 0; k < 32; ++k)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const f32x4 v = only_endless<BF>(
                *reinterpret_cast<const u32x2*>(vbuf + k * RB + value_chunk<D>(k % 16, i * 2 + g / 2) * 16 + g % 2 * 8));
#pragma unroll
            for (int b = 0; b < NB; ++b)
              if (tile * 32 + k < limit[b] && tile * 32 + k >= low[b]) acc[b][i] += v;
          }
#pragma unroll
        for (int i = 0; i < TILE / 1024; ++i) here[i * 64] = without_endless<BF>(held[i]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
#pragma unroll
    for (int q = 0; q < D / 64; ++q) {
      u32x4 vf[4];
      value_fragments<D>(vat ^ (q * 128), vf);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          acc[b][q * 4 + i] = Narrow<BF>::mma(vf[i], ph[b], acc[b][q * 4 + i]);
          acc[b][q * 4 + i] = Narrow<BF>::mma(vf[i], pl[b], acc[b][q * 4 + i]);
        }
    }
    if (more) load_values();
  }

  // the waves' rows meet in LDS, sixteen at a time: a lane has columns i * 16 + 4 g to + 3 of its row
  float* mine = reinterpret_cast<float*>(kbuf);
  float* plane = c.planes + ((int64_t)place * c.cache.kv_heads + kv) * c.rows * (D + 4);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (b * 16 >= c.rows) break;
    const float sum = row_sum(total[b]);
    __syncthreads();  // every wave is done with its tiles, or with the rows before
    if (g == 0) stat[0][wave][col] = margin[b] == BEGUN ? base[b] : -INFINITY, stat[1][wave][col] = sum;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(mine + col * OLD + i * 16 + g * 4) = acc[b][i];
    __syncthreads();
    for (int at = t; at < min(16, c.rows - b * 16) * (D / 4); at += 64 * TOKEN_WAVES) {
      const int row = at / (D / 4), d = at % (D / 4) * 4;
      float top = stat[0][0][row];
#pragma unroll
      for (int x = 1; x < TOKEN_WAVES; ++x) top = fmaxf(top, stat[0][x][row]);
      const float to_base = top == -INFINITY ? 0.0f : top;
      float all = 0.0f;
      f32x4 o = f32x4{};
#pragma unroll
      for (int x = 0; x < TOKEN_WAVES; ++x) {
        const float f = __builtin_amdgcn_exp2f(stat[0][x][row] - to_base);
        all += f * stat[1][x][row];
        o += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * 2 * TILE) + row * OLD + d);
      }
      if (parts > 1) {  // unnormalised rows, then their bases and sums
        const int r = b * 16 + row;
        *reinterpret_cast<f32x4*>(plane + r * D + d) = o;
        if (d == 0) plane[c.rows * D + r * 2] = top, plane[c.rows * D + r * 2 + 1] = all;
      } else {
        const int r = b * 16 + row, j = r / c.group;
        const float inv = all == 0.0f ? 0.0f : 1.0f / all;  // no key: zeros
        const u32x2 y = {Narrow<BF>::pack(o[0] * inv, o[1] * inv), Narrow<BF>::pack(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2*>(c.o + (((int64_t)seq * c.s.step + j) * c.heads + kv * c.group + (r - j * c.group)) * D + d) = y;
      }
    }
  }
}

// One row of a split sequence from its parts: JOIN_THREADS / (D / 4) parts side by side, four columns a thread
constexpr int JOIN_THREADS = 512;
template <bool BF, int D>
__global__ __launch_bounds__(JOIN_THREADS) void cache_join(TokenCall c) {
  constexpr int LANES = JOIN_THREADS / (D / 4);
  __shared__ f32x4 sums[LANES][D / 4];
  __shared__ float stat[2][LANES];
  const int rest = (int)(blockIdx.x / c.cache.kv_heads), kv = (int)(blockIdx.x % c.cache.kv_heads), order = rest / c.rows, r = rest % c.rows;
  if (order >= c.header[0].x) return;
  const int4 head = c.header[1 + order];
  const int t = threadIdx.x, side = t / (D / 4), d = t % (D / 4) * 4;
  const int64_t stride = (int64_t)c.cache.kv_heads * c.rows * (D + 4);
  const float* plane = c.planes + head.y * stride + (int64_t)kv * c.rows * (D + 4);
  float m = -INFINITY, total = 0.0f;
  f32x4 o = f32x4{};
#pragma unroll 4
  for (int p = side; p < head.z; p += LANES) {
    const float* at = plane + p * stride;
    const float top = at[c.rows * D + r * 2], sum = at[c.rows * D + r * 2 + 1], next = fmaxf(m, top);
    const float to_base = next == -INFINITY ? 0.0f : next;
    const float f = __builtin_amdgcn_exp2f(m - to_base), h = __builtin_amdgcn_exp2f(top - to_base);
    total = total * f + sum * h;
    o = o * f + h * *reinterpret_cast<const f32x4*>(at + r * D + d);
    m = next;
  }
  sums[side][d / 4] = o;
  if (d == 0) stat[0][side] = m, stat[1][side] = total;
  __syncthreads();
  if (side != 0) return;
  float top = stat[0][0];
#pragma unroll
  for (int x = 1; x < LANES; ++x) top = fmaxf(top, stat[0][x]);
  const float to_base = top == -INFINITY ? 0.0f : top;
  float all = 0.0f;
  o = f32x4{};
#pragma unroll
  for (int x = 0; x < LANES; ++x) {
    const float f = __builtin_amdgcn_exp2f(stat[0][x] - to_base);
    all += f * stat[1][x];
    o += f * sums[x][d / 4];
  }
  const float inv = all == 0.0f ? 0.0f : 1.0f / all;
  const int j = r / c.group;
  const u32x2 y = {Narrow<BF>::pack(o[0] * inv, o[1] * inv), Narrow<BF>::pack(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u32x2*>(c.o + (((int64_t)head.x * c.s.step + j) * c.heads + kv * c.group + (r - j * c.group)) * D + d) = y;
}

}  // namespace krn

using namespace krn;

TokenPlan krn::token_plan(int64_t step, int64_t group, int64_t kv_heads, int64_t d, int64_t page, int64_t sequences, int64_t width) {
  TokenPlan p{};
  p.rows = step * group;
  const int64_t tiles = (width * page < 0x7fffffff ? width * page : 0x7fffffff) / 32 + 1;  // of a sequence, at most
  // parts beyond the first of all sequences, for each key head: no more than shares, nor than parts have tiles
  p.shares = TOKEN_PARTS / kv_heads;
  int64_t extra = p.shares;
  if (sequences * ((tiles - 1) / TOKEN_CHUNK) < extra) extra = sequences * ((tiles - 1) / TOKEN_CHUNK);
  if (sequences > TOKEN_SPLIT || tiles - 1 <= TOKEN_WHOLE) extra = 0;
  p.workgroups = sequences + extra;
  p.split = extra > 0, p.mapped = p.split && sequences > 64 * TOKEN_HELD;
  p.joins = sequences < extra ? sequences : extra;
  p.header_bytes = p.split ? (p.joins + 1) * 16 : 0;
  p.map_bytes = p.mapped ? p.workgroups * 16 : 0;
  // planes of the parts beyond the first, and of the first ones of the sequences that have those
  p.bytes = p.split ? p.header_bytes + p.map_bytes + (extra + p.joins) * kv_heads * p.rows * (d + 4) * 4 : 0;
  return p;
}

template <bool BF, int D>
static void launch(const TokenCall& c, const TokenPlan& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.workgroups * c.cache.kv_heads)), block(64 * TOKEN_WAVES);
  if (c.map) hipLaunchKernelGGL(cache_shares, dim3(1), dim3(MAP_THREADS), 0, stream, c, (int)p.workgroups);
  if (p.rows <= 16) hipLaunchKernelGGL((cache_tokens<BF, D, 1>), grid, block, 0, stream, c);
  else hipLaunchKernelGGL((cache_tokens<BF, D, 2>), grid, block, 0, stream, c);
  if (c.split)
    hipLaunchKernelGGL((cache_join<BF, D>), dim3((unsigned)(p.joins * p.rows * c.cache.kv_heads)), dim3(JOIN_THREADS), 0, stream, c);
}

void krn::launch_cache_tokens(bool bf, int d, TokenCall c, const TokenPlan& p, void* workspace, hipStream_t stream) {
  c.rows = (int)p.rows, c.split = p.split, c.shares = (uint32_t)p.shares;
  c.header = (int4*)workspace, c.map = p.mapped ? (int4*)((char*)workspace + p.header_bytes) : nullptr;
  c.planes = (float*)((char*)workspace + p.header_bytes + p.map_bytes);
  if (bf) d == 128 ? launch<true, 128>(c, p, stream) : launch<true, 64>(c, p, stream);
  else d == 128 ? launch<false, 128>(c, p, stream) : launch<false, 64>(c, p, stream);
}
