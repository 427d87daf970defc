// Causal attention of packed prompts over a paged cache, for rows enough to fill the matrix cores.
//
// A workgroup has 128 rows of one key head: row r of a sequence is its token r / group, query head r % group of the key head's
// `group`. So shared heads lie side by side, short prompts fill tiles, and a causal tile is 128 / group tokens wide. Each of
// its four waves owns 32 rows and computes S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs: a lane holds one row
// (lane & 31) and half of the keys (its partner is lane ^ 32), P stays in its lane.
//
// The matrix cores and the power that they draw bound it (16384 tokens, 32 heads of 128 on 8: 1.85 to 1.99 ms by the card,
// 1105 to 1185 TFLOP/s; a large library product reaches 1380). Two workgroups share a CU, two waves a SIMD. Each wave
// interleaves its own work: scores of the next tile beside the weights of this one, then O += P V beside the exponents of
// the next, one MFMA and a few other instructions at a time in the order written (left to the compiler, 2 % slower). The
// other workgroup covers what comes before and after the loop: one workgroup of eight waves a CU reads keys half as often
// and has 0 to 2 % on that one prompt, 5 on 512 tokens after 15900, but 12 prompts of 8192 tokens take 153 us in place of
// 144, 16 of 500 10.0 and 8.5, 1024 tokens 29.0 and 22.5. (Eight waves in two groups that take turns by barriers: 2.06 ms.
// Four of 64 rows halve the LDS reads, but need more than 256 registers: 2.27 ms with the compiler's copies, 2.04 with
// accumulators that products alone touch.)
//
// K and V come into rings of three and two tiles by direct loads, more than a tile ahead of their use; tiles past the end are
// asked for with no bytes, which keeps the count of loads on their way the same. Sixteen keys, a wave's part of a tile, lie in
// one page, whose rows up to the sequence's end are a buffer resource: rows past it, and pages that are not there, read as zeros.
//
// Weights are rounded to 16 bits before O += P V, half a step (2^-8 in bf16) of each, as in attention.hip: two parts of them, which
// cache_token.hip can afford, would be half as many products again.
#include "attention_parts.h"
#include "cache_parts.h"

namespace krn {

constexpr int PROMPT_TILE = 64;  // keys
constexpr int PROMPT_WAVES = PROMPT_ROWS / 32;
constexpr int PROMPT_KEYS = 3, PROMPT_VALUES = 2;  // tiles of each in their rings

// The tokens of slot `slot`: 128 rows of a sequence. Sequence i has the slots from slot_of(its start, i) on, enough for its
// rows since starts are sums of what came before; a wave looks at 64 sequences at a time.
struct PromptTile {
  int seq, row0;
  TokenRange range;
  int length;
};
__device__ __forceinline__ int64_t slot_of(const PromptCall& c, int start, int i) {
  return (int64_t)min(max(start, 0), c.s.tokens) * c.group / PROMPT_ROWS + i;
}
__device__ __forceinline__ bool find_tile(const PromptCall& c, int slot, PromptTile& tile) {
  int at;
  if (c.s.starts) {
    const int lane = threadIdx.x & 63;
    int low = 0, count = c.s.n;  // the last sequence of low to low + count - 1 whose first slot is this one or before
    while (count > 64) {
      const int step = (count + 63) / 64, i = low + min(lane * step, count - 1);
      const uint64_t before = __builtin_amdgcn_ballot_w64(lane * step < count && slot_of(c, c.s.starts[i], i) <= slot);
      const int k = before ? 63 - __builtin_clzll(before) : 0;
      low += k * step;
      count = min(step, count - k * step);
    }
    // one more look, with what is needed of the sequence
    const int i = low + min(lane, count - 1), start = c.s.starts[i], next = c.s.starts[i + 1], length = sequence_length(c.s, i);
    const uint64_t before = __builtin_amdgcn_ballot_w64(lane < count && slot_of(c, start, i) <= slot);
    const int k = __builtin_amdgcn_readfirstlane(before ? 63 - __builtin_clzll(before) : 0);
    const int first = min(max(start, 0), c.s.tokens);
    tile.seq = __builtin_amdgcn_readfirstlane(low) + k;
    tile.range.first = __builtin_amdgcn_readlane(first, k);
    tile.range.count = __builtin_amdgcn_readlane(min(max(next, first), c.s.tokens) - first, k);
    tile.length = __builtin_amdgcn_readlane(length, k);
    const int64_t from = slot - slot_of(c, tile.range.first, tile.seq);
    at = from < 0 || from > 0xffffff ? -1 : (int)from;
  } else {
    const int per = (c.s.step * c.group + PROMPT_ROWS - 1) / PROMPT_ROWS;
    tile.seq = __builtin_amdgcn_readfirstlane(slot / per), at = slot - tile.seq * per;
    tile.range = token_range(c.s, tile.seq);
    tile.length = __builtin_amdgcn_readfirstlane(sequence_length(c.s, tile.seq));
  }
  at = __builtin_amdgcn_readfirstlane(at);
  tile.row0 = at * PROMPT_ROWS;
  return at >= 0 && (int64_t)at * PROMPT_ROWS < (int64_t)tile.range.count * c.group;
}

// The key tiles that 128 rows from row0 on see: from the first row's window to the last row's position
struct KeyTiles {
  int first, count;
};
__device__ __forceinline__ KeyTiles tiles_seen(const PromptCall& c, const TokenRange& range, int length, int row0) {
  const int before = length - range.count, last = min((row0 + PROMPT_ROWS - 1) / c.group, range.count - 1);
  const int end = min(before + last + 1, held_keys(c.s, length, c.cache.page_shift));
  const int first = first_key(before + row0 / c.group, c.window) / PROMPT_TILE;
  return {first, max(0, (max(end, 0) + PROMPT_TILE - 1) / PROMPT_TILE - first)};
}

// Rows before many keys are shared out: workgroup w of a column does part `part` of `parts` of a tile of rows. All tiles of
// rows of a sequence have as many parts, so that nothing loops over them: with R of them of up to T key tiles each, ceil(T
// / chunk), and chunk is the sum of all R T over `spare`, the workgroups that are there beyond one for each tile of rows. That
// sum has the rows that stay whole in it too, so a few long rows beside many short ones are in fewer parts than there are
// workgroups for (1 token after 65000 keys 62 us, 2000 tokens 47, packed together 123).
// Every wave counts for itself, a lane for ceil(n / 64) sequences in a row. Sequences of R T above 2^22 (16 ms of the whole
// chip a key head at d = 128, half of that for a prompt) stay whole and are not counted, which keeps the sum over up to
// 512 sequences in 32 bits.
struct PromptPart {
  int part, parts, plane, order;  // plane: of the first part, among all planes; order: of the rows, among those in several parts
};
__device__ __forceinline__ bool find_part(const PromptCall& c, int w, bool writes, PromptTile& tile, PromptPart& share) {
  constexpr uint32_t MOST = 1 << 22;
  const int lane = threadIdx.x & 63, per = (c.s.n + 63) / 64, from = lane * per, to = min(from + per, c.s.n);
  struct Rows {
    uint32_t rows, tiles;  // tiles of rows, and the key tiles of the last one
  };
  const auto rows_of = [&](const TokenRange& range, int length) {
    const uint32_t rows = (range.count * c.group + PROMPT_ROWS - 1) / PROMPT_ROWS;
    int first = 0;
    if (c.window) first = first_key(length - range.count + (int)(rows - 1) * PROMPT_ROWS / c.group, c.window) / PROMPT_TILE;
    const int end = held_keys(c.s, length, c.cache.page_shift);
    return Rows{rows, rows ? (uint32_t)max((end + PROMPT_TILE - 1) / PROMPT_TILE - first, 1) : 0};
  };
  const auto work_of = [&](const Rows& r) { return (uint64_t)r.tiles * r.rows > MOST ? 0 : r.tiles * r.rows; };
  // a lane's first sequence stays in registers
  const int own = min(from, c.s.n - 1);
  const TokenRange range = token_range(c.s, own);
  const int length = sequence_length(c.s, own);
  const Rows held = from < to ? rows_of(range, length) : Rows{0, 0};
  uint32_t work = work_of(held), items = held.rows;
  for (int i = from + 1; i < to; ++i) {
    const Rows r = rows_of(token_range(c.s, i), sequence_length(c.s, i));
    work += work_of(r), items += r.rows;
  }
  uint32_t upto = wave_scan(items), before = upto - items;
  work = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(work), 63);
  const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  const uint32_t spare = all < c.shares ? min(c.shares - all, c.spare) : 0;
  const uint32_t chunk = spare ? max((uint32_t)PROMPT_CHUNK, (work + spare - 1) / spare) : 0x7fffffff;
  const auto parts_of = [&](const Rows& r) {
    return r.tiles <= chunk || (uint64_t)r.tiles * r.rows > MOST ? 1u : (r.tiles + chunk - 1) / chunk;
  };
  // parts, and of rows in several of them the parts in the low half, the rows in the high one
  const uint32_t parts = parts_of(held);
  uint32_t count = held.rows * parts, joined = parts > 1 ? held.rows << 16 | count : 0;
  for (int i = from + 1; i < to; ++i) {
    const Rows r = rows_of(token_range(c.s, i), sequence_length(c.s, i));
    const uint32_t p = parts_of(r);
    count += r.rows * p, joined += p > 1 ? r.rows << 16 | r.rows * p : 0;
  }
  uint32_t joined_upto = 0;
  if (__builtin_amdgcn_ballot_w64(joined != 0) != 0) {
    upto = wave_scan(count), before = upto - count;
    joined_upto = wave_scan(joined);
  }
  if (writes && w == 0 && threadIdx.x == 63) c.header[0] = {(int)(joined_upto >> 16), 0, 0, 0};
  const uint64_t owner = __builtin_amdgcn_ballot_w64(before <= (uint32_t)w && (uint32_t)w < upto);
  if (owner == 0) return false;
  // in the owner's lane: the sequence
  uint32_t joined_before = joined_upto - joined, at = (uint32_t)w - before;
  Rows r = held;
  uint32_t p = parts;
  int seq = from;
  while (at >= r.rows * p && seq + 1 < to) {
    at -= r.rows * p, joined_before += p > 1 ? r.rows << 16 | r.rows * p : 0;
    ++seq;
    r = rows_of(token_range(c.s, seq), sequence_length(c.s, seq)), p = parts_of(r);
  }
  const uint32_t row = p > 1 ? at / p : at;  // late rows, the long ones, first
  joined_before += p > 1 ? row << 16 | row * p : 0;
  const int of = __builtin_ctzll(owner);
  const auto get = [&](auto x) { return __builtin_amdgcn_readlane((int)x, of); };
  share.part = get(at - row * p), share.parts = get(p), share.plane = get(joined_before & 0xffff), share.order = get(joined_before >> 16);
  tile.seq = get(seq), tile.row0 = get(r.rows - 1 - row) * PROMPT_ROWS;
  if (tile.seq == of * per) {
    tile.range = {get(range.first), get(range.count)}, tile.length = get(length);
  } else {
    const TokenRange other = token_range(c.s, tile.seq);
    tile.range = {get(other.first), get(other.count)}, tile.length = get(sequence_length(c.s, tile.seq));
  }
  return tile.row0 >= 0;
}

#define KRN_BARRIER()                       \
  do {                                      \
    asm volatile("" ::: "memory");          \
    __builtin_amdgcn_s_barrier();           \
    asm volatile("" ::: "memory");          \
  } while (0)

// `table` is restrict for what that says about the other memory: without any such word on a transposed LDS read the
// compiler waits for all loads to LDS before it.
template <bool BF, int D>
__device__ __forceinline__ void prompt_tile(const PromptCall& c, const PromptTile& tile, int column, int part, int parts,
                                            float* plane, const int* __restrict__ table, uint8_t* lds) {
  constexpr int RB = D * 2, DCH = D / 8, TILE = PROMPT_TILE * RB, LOADS = TILE / PROMPT_WAVES / 1024;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  static_assert(PROMPT_TILE == PROMPT_WAVES * 16, "sixteen keys a wave");
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5, r32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int length = tile.length;
  const int end = __builtin_amdgcn_readfirstlane(held_keys(c.s, length, c.cache.page_shift));
  const int before = length - tile.range.count;  // the position of the sequence's first token here

  // this lane's row, the keys that it sees, and those that all or some rows of the wave and the workgroup see
  const int row = tile.row0 + wave * 32 + r32, j = row / c.group;
  const bool real = j < tile.range.count;
  const int position = before + min(j, tile.range.count - 1), limit = min(position + 1, end), low = first_key(position, c.window);
  const int all_limit = __builtin_amdgcn_readfirstlane(limit), all_low = __builtin_amdgcn_readlane(low, 31);
  // tiles within these bounds have keys that all rows of the workgroup see, or that lie past the end and are zeros
  const int last_token = min((tile.row0 + PROMPT_ROWS - 1) / c.group, tile.range.count - 1);
  const int whole_low = __builtin_amdgcn_readfirstlane(first_key(before + last_token, c.window));
  const int whole_limit = __builtin_amdgcn_readfirstlane(min(before + tile.row0 / c.group + 1, end));
  const KeyTiles seen = tiles_seen(c, tile.range, length, tile.row0);
  const int even = __builtin_amdgcn_readfirstlane(seen.count / parts), over = seen.count - even * parts;
  const int first = __builtin_amdgcn_readfirstlane(seen.first + even * part + min(part, over));
  const int n = __builtin_amdgcn_readfirstlane(even + (part < over ? 1 : 0));
  const int64_t place = ((int64_t)(tile.range.first + j) * c.heads + column * c.group + (row - j * c.group)) * D;
  if (n <= 0) {  // no row sees a key
    if (real)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) *reinterpret_cast<u32x4*>(c.o + place + s * 16 + half * 8) = u32x4{};
    return;
  }

  u32x4 qf[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) qf[s] = real ? *reinterpret_cast<const u32x4*>(c.q + place + s * 16 + half * 8) : u32x4{};

  // this wave's sixteen keys of a tile
  uint32_t koff[LOADS], voff[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int key = i * (1024 / RB) + lane / DCH, s = lane % DCH;  // in the group
    const int in_tile = wave * 16 + key;
    koff[i] = (uint32_t)(key * RB + k_slot<D>(in_tile, s) * 16);
    voff[i] = (uint32_t)(key * RB + v_slot<D>(in_tile, s) * 16);
  }
  const int shift = c.cache.page_shift;
  // page numbers of this wave's keys in 64 tiles, a lane each
  int ids = -1, ids_from = 0;
  const auto fetch_ids = [&](int u) {
    ids_from = u;
    const int64_t at = ((int64_t)(first + u + lane) * PROMPT_TILE + wave * 16) >> shift;
    ids = u + lane < n && at < c.s.width ? table[at] : -1;
    asm volatile("" : "+v"(ids));  // waited for here: a use in the loop would wait for the tiles on their way each time
  };
  // where they lie in tile u, and how many bytes the sequence has there
  struct Group {
    int64_t at;
    int bytes;
  };
  const auto group_of = [&](int u) {
    const int number = __builtin_amdgcn_readlane(ids, u - ids_from), key0 = (first + u) * PROMPT_TILE + wave * 16;
    const bool there = (uint32_t)number < (uint32_t)c.cache.pages;
    const int64_t page = (int64_t)(there ? number : 0) * c.kv_heads + column;
    return Group{((page << shift) + (key0 & ((1 << shift) - 1))) * RB,
                 __builtin_amdgcn_readfirstlane(there ? max(0, min(16, end - key0)) * RB : 0)};
  };
  const auto load = [&](const void* data, const Group& g, int ring, const uint32_t(&off)[LOADS], int i) {
    buffer_to_lds16(panel_rsrc((const uint8_t*)data + g.at, g.bytes), lds + ring + wave * (TILE / PROMPT_WAVES) + i * 1024, off[i], 0);
  };
  constexpr int V_RING = PROMPT_KEYS * TILE;
  const auto key_ring = [](int u) { return u % PROMPT_KEYS * TILE; };
  const auto value_ring = [](int u) { return V_RING + u % PROMPT_VALUES * TILE; };

  // fragments: K's as A operands (lane = key, 8 columns of step s), V^T's (lane = column, keys as the lane's P has them)
  const uint32_t kat = r32 * RB + k_slot<D>(r32, half) * 16;
  const int a16 = lane & 15, tr_key = (lane >> 5) * 4 + (a16 >> 2), tr_col = ((lane >> 4) & 1) * 16 + 4 * (a16 & 3);
  const uint32_t vat = tr_key * RB + v_slot<D>(tr_key, tr_col >> 3) * 16 + (tr_col & 7) * 2;
  constexpr int K_AHEAD = 3, V_AHEAD = 2;  // steps whose fragments are held
  u32x4 kf[K_AHEAD][2], vf[V_AHEAD][BLOCKS];
  const auto read_keys = [&](uint32_t at, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) kf[s % K_AHEAD][h] = *reinterpret_cast<const u32x4*>(lds + ((at ^ (s << 5)) + h * 32 * RB));
  };
  const auto read_values = [&](uint32_t at, int s, int i) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) v4s*)(lds + ((at ^ (i << 6)) + (s * 16 + part * 8) * RB))));
      vf[s % V_AHEAD][i][part * 2] = w[0], vf[s % V_AHEAD][i][part * 2 + 1] = w[1];
    }
  };

  f32x16 acc[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) acc[i] = f32x16{};
  // a score's exponent is s scale - base; exponents above `margin` move the base, to LIFT below them: the first one, then
  // those 8 above that
  constexpr float BEGUN = LIFT<BF> + 8.0f;
  float base = 0.0f, margin = -INFINITY, total = 0.0f;
  u32x4 pf[4];

  // The weights of a tile from its exponents, 2^x packed as P^T, in 34 pieces of work, each on two of a lane's 32: piece 2 x
  // raises 2 to pair x, 2 x + 1 adds up and packs pair x - 1
  constexpr int PIECES = 34;
  const auto piece = [&](f32x16(&s)[2], int at) {
    const int pair = at / 2 - at % 2;
    if (pair < 0 || pair > 15) return;
    f32x16& v = s[pair / 8];
    const int e = pair % 8 * 2;
    if (at % 2 == 0) {
      v[e] = __builtin_amdgcn_exp2f(v[e]), v[e + 1] = __builtin_amdgcn_exp2f(v[e + 1]);
    } else {
      total += v[e] + v[e + 1];
      pf[pair / 4][pair % 4] = Half<BF>::pack(v[e], v[e + 1]);
    }
  };
  // exponents of a pair of scores, and their largest (scaled ones: the compiler quiets a product's scores first)
  const auto scaled = [&](f32x16& v, int e, float& top) {
    v[e] = __builtin_fmaf(v[e], c.scale, -base), v[e + 1] = __builtin_fmaf(v[e + 1], c.scale, -base);
    top = fmaxf(fmaxf(top, v[e]), v[e + 1]);
  };
  // Masks the exponents of tile u, whose largest is `top` before that, and settles the base: it moves only when a weight would
  // exceed its first by 2^8, and then exponents, acc and total with it.
  const auto settle = [&](f32x16(&s)[2], float top, int u) {
    const int key0 = (first + u) * PROMPT_TILE;
    if (key0 < all_low || key0 + PROMPT_TILE > all_limit) {
      top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = key0 + half * 4 + (r >> 2) * 8 + (r & 3);
        s[0][r] = key >= limit || key < low ? -INFINITY : s[0][r];
        s[1][r] = key + 32 >= limit || key + 32 < low ? -INFINITY : s[1][r];
        top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
      }
    }
    if (__builtin_amdgcn_ballot_w64(top > margin) != 0) {
      top = pair_max(top);
      const bool moves = top > margin, began = margin == BEGUN;
      const float by = moves ? top - LIFT<BF> : 0.0f, corr = moves && began ? __builtin_amdgcn_exp2f(-by) : 1.0f;
      total *= corr;
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= corr;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] -= by, s[1][r] -= by;
      base += by;
      margin = moves ? BEGUN : margin;
    }
  };
  // Tile u has keys that some rows see and some do not: if values of it are not finite, which every wave looks for in what it
  // loaded, all of them add what their rows see of those and clear them away. (The look costs 1 % of prompts of some hundred
  // tokens. It comes before the step's products: beside them the compiler would move weights behind its branch, and behind
  // them copy the sums.)
  const auto separate = [&](int u) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");  // this wave's part of V of u
    KRN_BARRIER();
    u32x4* mine = reinterpret_cast<u32x4*>(lds + value_ring(u) + wave * (TILE / PROMPT_WAVES)) + lane;
    uint32_t* flags = reinterpret_cast<uint32_t*>(lds + value_ring(u + 1));  // a wave each: that tile comes in this step
    u32x4 held[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) held[i] = mine[i * 64];
    flags[wave] = __builtin_amdgcn_ballot_w64(any_endless<BF>(held)) != 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    KRN_BARRIER();
    if (__builtin_amdgcn_ballot_w64(flags[lane & (PROMPT_WAVES - 1)] != 0) != 0) {
#pragma unroll 1
      for (int k = 0; k < PROMPT_TILE; ++k) {
        const int key = (first + u) * PROMPT_TILE + k;
        const bool sees = key >= low && key < limit;
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
          for (int gq = 0; gq < 4; ++gq) {
            const f32x4 v = only_endless<BF>(*reinterpret_cast<const u32x2*>(
                lds + value_ring(u) + k * RB + v_slot<D>(k, i * 4 + gq) * 16 + half * 8));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][gq * 4 + e] += sees ? v[e] : 0.0f;
          }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      KRN_BARRIER();
#pragma unroll
      for (int i = 0; i < LOADS; ++i) mine[i * 64] = without_endless<BF>(mine[i * 64]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      KRN_BARRIER();
    }
  };
  // Tile u, whose exponents `s` are settled: the scores `next` of tile u + 1 beside most weights of u, then O += P V beside the
  // others and the exponents of u + 1. One MFMA and a little of the other work at a time, in this order.
  // Once every wave has K's fragments of u + 1, and V of u is there, V's tile u + 1 and K's u + 4 leave; `at` says where the
  // tiles u + 1, u + 2 and u + 3 lie.
  const auto step = [&](f32x16(&s)[2], f32x16(&next)[2], int u, Group(&at)[3]) {
    const uint32_t k_at = kat + key_ring(u + 1), k_then = kat + key_ring(u + 2), v_at = vat + value_ring(u);
    constexpr int FIRST = 24, SCORES = 2 * STEPS, PRODUCTS = 4 * BLOCKS;
    if ((first + u) * PROMPT_TILE < whole_low || min((first + u + 1) * PROMPT_TILE, end) > whole_limit) separate(u);
    next[0] = f32x16{}, next[1] = f32x16{};
#pragma unroll
    for (int i = 0; i < SCORES; ++i) {
      if (i % 2 == 0 && i / 2 + 2 < STEPS) read_keys(k_at, i / 2 + 2);
      if (i == SCORES - BLOCKS) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");  // this wave's part of K of u + 2 and V of u
        KRN_BARRIER();
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i >= SCORES - BLOCKS) read_values(v_at, 0, i - (SCORES - BLOCKS));
      Half<BF>::mma(next[i % 2], kf[i / 2 % K_AHEAD][i % 2], qf[i / 2]);
#pragma unroll
      for (int x = i * FIRST / SCORES; x < (i + 1) * FIRST / SCORES; ++x) piece(s, x);
      __builtin_amdgcn_sched_barrier(0);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      if (i / BLOCKS < 3) read_values(v_at, i / BLOCKS + 1, i % BLOCKS);
      if (i >= PRODUCTS - 4 && i % 2 == 0) read_keys(k_then, (i - (PRODUCTS - 4)) / 2);
      Half<BF>::mma(acc[i % BLOCKS], vf[i / BLOCKS % V_AHEAD][i % BLOCKS], pf[i / BLOCKS]);
      constexpr int LAST = 3 * BLOCKS;  // products before those of the last weights
      if (i < LAST)
#pragma unroll
        for (int x = FIRST + i * (PIECES - FIRST) / LAST; x < FIRST + (i + 1) * (PIECES - FIRST) / LAST; ++x) piece(s, x);
#pragma unroll
      for (int x = i * 16 / PRODUCTS; x < (i + 1) * 16 / PRODUCTS; ++x) scaled(next[x / 8], x % 8 * 2, top[x / 8]);
      // a lane's addresses and loads here and there between the products: all at once they would hold them up
      if (i < LOADS) load(c.cache.values, at[0], value_ring(u + 1), voff, i);
      if (i == PRODUCTS / 4) at[0] = at[1], at[1] = at[2], at[2] = group_of(u + 4);
      if (i >= PRODUCTS / 2 && i < PRODUCTS / 2 + LOADS) load(c.cache.keys, at[2], key_ring(u + 1), koff, i - PRODUCTS / 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" : "+v"(top[0]), "+v"(top[1]), "+v"(total));  // here, not in the branches that follow
    if (u + 5 - ids_from >= 64) fetch_ids(u + 5);
    if (u + 1 < n) settle(next, fmaxf(top[0], top[1]), u + 1);  // no tile: its scores must not move the base
  };

  // tiles on their way in the order that the loop keeps: V of u + 1, then K of u + 4
  fetch_ids(0);
  Group at[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) at[u] = group_of(u);
  const auto load_keys = [&](int u) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(c.cache.keys, at[u], key_ring(u), koff, i);
  };
  load_keys(0), load_keys(1), load_keys(2);
#pragma unroll
  for (int i = 0; i < LOADS; ++i) load(c.cache.values, at[0], value_ring(0), voff, i);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * LOADS) : "memory");  // the first K tile
#pragma unroll
  for (int s = 0; s < STEPS; ++s) asm volatile("" : "+v"(qf[s]));  // older loads: no wait for them in the loop
  KRN_BARRIER();
  f32x16 sa[2], sb[2];
  sa[0] = f32x16{}, sa[1] = f32x16{};
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    read_keys(kat, s);
    Half<BF>::mma(sa[0], kf[s % K_AHEAD][0], qf[s]);
    Half<BF>::mma(sa[1], kf[s % K_AHEAD][1], qf[s]);
  }
  {
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x) scaled(sa[x / 8], x % 8 * 2, top);
    settle(sa, top, 0);
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");  // the second
  KRN_BARRIER();  // everyone has read the first tile: its place may be loaded
  read_keys(kat + key_ring(1), 0);
  read_keys(kat + key_ring(1), 1);
  load_keys(3);
  Group coming[3] = {at[1], at[2], at[3]};
  for (int u = 0;;) {
    step(sa, sb, u, coming);
    if (++u >= n) break;
    step(sb, sa, u, coming);
    if (++u >= n) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup

  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(total), __float_as_uint(total), false, false);
    total = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if (parts > 1) {  // unnormalised rows, then their bases and sums
    float* at = plane + (wave * 32 + r32) * D + half * 4;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<f32x4*>(at + i * 32 + gq * 8) =
            f32x4{acc[i][gq * 4], acc[i][gq * 4 + 1], acc[i][gq * 4 + 2], acc[i][gq * 4 + 3]};
    if (half == 0) {
      plane[PROMPT_ROWS * D + (wave * 32 + r32) * 2] = margin == BEGUN ? base : -INFINITY;
      plane[PROMPT_ROWS * D + (wave * 32 + r32) * 2 + 1] = total;
    }
    return;
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
#undef KRN_BARRIER

template <bool BF, int D>
__global__ __launch_bounds__(64 * PROMPT_WAVES, 2) void cache_prompt(PromptCall c) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[(PROMPT_KEYS + PROMPT_VALUES) * PROMPT_TILE * D * 2];
  const int w = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / c.kv_heads)), column = (int)blockIdx.x - w * c.kv_heads;
  PromptTile tile;
  PromptPart share{0, 1, 0, 0};
  if (c.shares) {
    if (!find_part(c, w, column == 0, tile, share)) return;
    if (share.parts > 1) {
      const int parts = min(share.parts, max(tiles_seen(c, tile.range, tile.length, tile.row0).count, 1));  // of these rows
      if (share.part == 0 && column == 0 && threadIdx.x == 0)
        c.header[1 + share.order] = {tile.seq, tile.row0, share.plane, parts > 1 ? parts : 0};
      if (share.part >= parts) return;
      share.parts = parts;
    }
  } else if (!find_tile(c, c.slots - 1 - w, tile)) {  // late rows, the long ones, first
    return;
  }
  float* plane = c.planes + ((int64_t)(share.plane + share.part) * c.kv_heads + column) * (PROMPT_ROWS * (D + 2));
  prompt_tile<BF, D>(c, tile, column, share.part, share.parts, plane, c.s.table + (int64_t)tile.seq * c.s.width, lds);
}

// Rows in several parts: four columns of a row a thread, the parts one after the other. No more workgroups than run at once: most
// calls have far fewer rows to join than they may have.
constexpr int JOIN_GROUPS = 2048;
template <bool BF, int D>
__global__ __launch_bounds__(256) void cache_prompt_join(PromptCall c) {
  constexpr int ROWS = 256 / (D / 4), BLOCKS = PROMPT_ROWS / ROWS;  // of a workgroup, of a tile of rows
  const int items = c.header[0].x * BLOCKS * c.kv_heads;
  for (int item = (int)blockIdx.x; item < items; item += (int)gridDim.x) {
    const int column = item % c.kv_heads, rest = item / c.kv_heads;
    const int4 head = c.header[1 + rest / BLOCKS];
    const TokenRange range = token_range(c.s, head.x);
    const int r = rest % BLOCKS * ROWS + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    const int row = head.y + r, j = row / c.group;
    if (head.w == 0 || j >= range.count) continue;  // too few keys after all, or no row
    const int64_t stride = (int64_t)c.kv_heads * (PROMPT_ROWS * (D + 2));
    const float* plane = c.planes + head.z * stride + (int64_t)column * (PROMPT_ROWS * (D + 2));
    float m = -INFINITY, all = 0.0f;
    f32x4 o = f32x4{};
#pragma unroll 4
    for (int p = 0; p < head.w; ++p) {
      const float* at = plane + p * stride;
      const float top = at[PROMPT_ROWS * D + r * 2], next = fmaxf(m, top), to_base = next == -INFINITY ? 0.0f : next;
      const float f = __builtin_amdgcn_exp2f(m - to_base), h = __builtin_amdgcn_exp2f(top - to_base);
      all = all * f + at[PROMPT_ROWS * D + r * 2 + 1] * h;
      o = o * f + h * *reinterpret_cast<const f32x4*>(at + r * D + d);
      m = next;
    }
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;  // no key: zeros
    const u32x2 y = {Half<BF>::pack(o[0] * inv, o[1] * inv), Half<BF>::pack(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2*>(c.o + ((int64_t)(range.first + j) * c.heads + column * c.group + (row - j * c.group)) * D + d) = y;
  }
}

}  // namespace krn

using namespace krn;

PromptPlan krn::prompt_plan(int64_t tokens, int64_t step, int64_t group, int64_t kv_heads, int64_t d, int64_t page,
                            int64_t sequences, int64_t width, int64_t bytes) {
  PromptPlan p{};
  p.slots = p.workgroups = step > 0 ? sequences * ((step * group + PROMPT_ROWS - 1) / PROMPT_ROWS)
                                    : tokens * group / PROMPT_ROWS + sequences;
  // parts beyond the first of all tiles of rows, in each column: as many as run at once without them, or half of that
  const int64_t at_once = PROMPT_PLACES / kv_heads, tiles = width * page / PROMPT_TILE;
  if (at_once == 0 || tiles <= PROMPT_CHUNK || (p.slots >= at_once && (tiles <= PROMPT_LONG || sequences > 256))) return p;
  const int64_t header = (at_once + 1) * 16, need = header + 2 * at_once * kv_heads * PROMPT_ROWS * (d + 2) * 4;
  if (need > bytes) return p;
  p.shares = p.workgroups = at_once > p.slots + at_once / 2 ? at_once : p.slots + at_once / 2;
  p.spare = p.joins = at_once, p.header_bytes = header, p.bytes = need;
  return p;
}

template <bool BF, int D>
static void launch(const PromptCall& c, const PromptPlan& p, hipStream_t stream) {
  hipLaunchKernelGGL((cache_prompt<BF, D>), dim3((unsigned)(p.workgroups * c.kv_heads)), dim3(64 * PROMPT_WAVES), 0, stream, c);
  const int64_t items = p.joins * (PROMPT_ROWS * (D / 4) / 256) * c.kv_heads;
  if (p.shares)
    hipLaunchKernelGGL((cache_prompt_join<BF, D>), dim3((unsigned)(items < JOIN_GROUPS ? items : JOIN_GROUPS)), dim3(256), 0, stream, c);
}

void krn::launch_cache_prompt(bool bf, int d, PromptCall c, const PromptPlan& p, void* workspace, hipStream_t stream) {
  c.slots = (int)p.slots, c.shares = (uint32_t)p.shares, c.spare = (uint32_t)p.spare;
  c.header = (int4*)workspace, c.planes = (float*)((char*)workspace + p.header_bytes);
  if (bf) d == 128 ? launch<true, 128>(c, p, stream) : launch<true, 64>(c, p, stream);
  else d == 128 ? launch<false, 128>(c, p, stream) : launch<false, 64>(c, p, stream);
}
