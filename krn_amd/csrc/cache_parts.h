// A paged key-value cache and the sequences of a step, as the kernels on them see both (include/krn_amd.h describes the
// layout). What lies on the device is checked on the device: token ranges are cut to the tokens there are, a length to the
// pages that the table has room for, and a page number outside of the cache reads as zeros and is never written.
#pragma once
#include "common.h"

namespace krn {

struct CacheView {
  const void *keys, *values;  // (pages, kv_heads, page, d) of 16-bit elements
  int pages, kv_heads, page_shift;  // a page holds 2^page_shift keys, 16 or more
};

struct SequencesView {
  const int *starts, *lengths, *table;  // (n + 1) or none, (n), (n, width)
  int n, width, step, tokens;           // without starts every sequence has `step` tokens
};

// The tokens of sequence i
struct TokenRange {
  int first, count;
};
__device__ __forceinline__ TokenRange token_range(const SequencesView& s, int i) {
  if (!s.starts) return {i * s.step, s.step};
  const int first = min(max(s.starts[i], 0), s.tokens), end = min(max(s.starts[i + 1], first), s.tokens);
  return {first, end - first};
}

// The length of sequence i, which positions count from, and how many of its keys the table can hold
__device__ __forceinline__ int sequence_length(const SequencesView& s, int i) { return max(s.lengths[i], 0); }
__device__ __forceinline__ int held_keys(const SequencesView& s, int length, int page_shift) {
  return (int)min((int64_t)length, (int64_t)s.width << page_shift);
}

// The first key that a token at `position` sees through a window of that many keys (0: all)
__device__ __forceinline__ int first_key(int position, int window) {
  return window ? (int)max((int64_t)0, (int64_t)position + 1 - window) : 0;
}

// Softmax weights are rounded to 16 bits before their products. In f16, whose last step is 2^-24, they are 2^7 times as large,
// up to 2^15 with the margin of 2^8 by which a weight may exceed the first: what is below 2^-32 of the largest is lost (2^-25
// without the factor, 0.4 % of a result of 131000 keys behind one large weight). The sums of weights have it too.
template <bool BF>
constexpr float LIFT = BF ? 0.0f : 7.0f;

// Values that are not finite: a weight of zero does not make them zero. Where a tile has keys that some rows see and some do
// not, the products take its values without those, and each row adds the ones that it sees: its sum is not finite either way.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <bool BF>
constexpr uint32_t ENDLESS = BF ? 0x7f80 : 0x7c00;  // infinity; NaN are above
template <bool BF, int N>
__device__ __forceinline__ bool any_endless(const u32x4 (&w)[N]) {
  u16x2 top = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i][e] & 0x7fff7fffu));
  return top[0] >= ENDLESS<BF> || top[1] >= ENDLESS<BF>;
}
template <bool BF>
__device__ __forceinline__ u32x4 without_endless(u32x4 w) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((w[e] & 0x7fff) >= ENDLESS<BF>) w[e] &= 0xffff0000u;
    if ((w[e] >> 16 & 0x7fff) >= ENDLESS<BF>) w[e] &= 0xffffu;
  }
  return w;
}
template <bool BF>
__device__ __forceinline__ f32x4 only_endless(u32x2 w) {
  f32x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint16_t v = (uint16_t)(w[e / 2] >> (e % 2 * 16));
    x[e] = (v & 0x7fff) >= ENDLESS<BF> ? (BF ? bf2f(v) : h2f(v)) : 0.0f;
  }
  return x;
}

// The sum over lanes up to this one: rows of sixteen by shifts, then the rows' ends
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += from_lane<0x111, 0xf>(x);
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);  // lane 15 to the second row, lane 47 to the fourth
  x += from_lane<0x143, 0xc>(x);  // lane 31 to the upper half
  return x;
}

// Attention of new tokens, a few of every sequence (cache_token.hip)
constexpr int TOKEN_WAVES = 4;
// Rows of a key head, at most; more are a prompt's. What is faster hangs on the batch, which this rule does not look at: it is
// set for large ones and costs small ones of 33 to 64 rows up to half of their time. (d = 128, 8 key heads, here and there:
// 64 sequences of 4000 keys, 32 rows 207 and 189 us, 64 rows, in two more blocks of sixteen, 270 and 193; one sequence of
// 4000, 32 rows 12 and 24, 48 rows 20 and 37, 64 rows 20 and 24, of 500 and 48 rows 16 and 25. One key head, 8 sequences of
// 2000, 40 and 64 rows: 16 and 25, 18 and 26.)
constexpr int TOKEN_ROWS = 32;
// Parts that the keys of all sequences and columns are shared out to: two for each workgroup that runs at once. (64 sequences of
// 4096 keys on average, d = 128: 512 parts 179 us, 1024 173, 2048 176; of 4096 each 164, 170, 175; 2 of 131000 103, 99, 102.)
constexpr int TOKEN_PARTS = 1024;
// Tiles of a part, at least, one a wave (one sequence of 4096 keys 10.6 us, with 8 11.0, with 16 12.7)
constexpr int TOKEN_CHUNK = 4;
// Tables of no more tiles a sequence keep each in one workgroup, which saves the joining launch (8 key heads, d = 128, one launch
// and two: 300 keys 5.8 and 8.5 us, 256 sequences of 100 26.3 and 37.4, 16 of 200 8.7 and 10.5; 1000 keys 9.4 and 8.7)
constexpr int TOKEN_WHOLE = 24;
constexpr int TOKEN_SPLIT = 8192;  // sequences; more keep the keys of each in one workgroup
// Sequences that a lane counts; beyond 64 times as many a launch counts them first (128 sequences of 100 keys 19.2 us, 19.8
// with it, 256 36.2 and 31)
constexpr int TOKEN_HELD = 2;
constexpr int TOKEN_TILES = 1 << 18;  // of a sequence, as far as shares go by them: the sum of all stays below 2^32
static_assert(TOKEN_PARTS + TOKEN_SPLIT < 1 << 16, "parts are counted in 16 bits");

struct TokenCall {
  const uint16_t* q;
  uint16_t* o;
  CacheView cache;
  SequencesView s;
  int heads, group, window;  // group: query heads of a key head
  float scale;               // of the scores, times log2(e)
  int rows, split;  // of TokenPlan
  uint32_t shares;  // the parts of a key head, with all sequences in one row
  int4* header;     // the number of sequences in several parts, then of each (sequence, first plane, parts, -)
  int4* map;        // of a workgroup (sequence or -1, part, parts, order of a sequence in several), if counted before
  float* planes;    // of a part of a sequence in several, and key head: `rows` rows of sums, then their bases and sums of weights
};

// rows: of a key head
struct TokenPlan {
  int64_t rows, shares, workgroups, joins, header_bytes, map_bytes, bytes;
  bool split, mapped;
};
TokenPlan token_plan(int64_t step, int64_t group, int64_t kv_heads, int64_t d, int64_t page, int64_t sequences, int64_t width);
void launch_cache_tokens(bool bf, int d, TokenCall c, const TokenPlan& p, void* workspace, hipStream_t stream);

// Attention of packed prompts (cache_prompt.hip)
constexpr int PROMPT_ROWS = 128;  // of a workgroup: tokens times query heads of a key head

// Tiles of 64 keys of a part, at least: a part costs 67 KB of sums written and read (128 tokens after 8000, 32 heads on 8:
// 32.5 us, with 8 36.6, with 32 41.9)
constexpr int PROMPT_CHUNK = 16;
// Tiles of a table, beyond which rows are shared out where they fill the chip as well: a single token before 65000 keys, packed
// with a prompt of 2000 tokens, would run on alone (891 us, shared out 131). Counting parts and the joining launch cost 60
// prompts of 150 tokens with such a table 53.0 and 56.7.
constexpr int PROMPT_LONG = 128;
constexpr int PROMPT_PLACES = 512;  // workgroups that run at once, two a CU

struct PromptCall {
  const uint16_t* q;
  uint16_t* o;
  CacheView cache;
  SequencesView s;
  int heads, kv_heads, group, window;  // group: query heads of a key head
  float scale;                         // of the scores, times log2(e)
  int slots;        // workgroups of a key head without parts
  uint32_t shares;  // workgroups of a key head with parts, or 0
  uint32_t spare;   // those of them that parts beyond the first may take
  int4* header;     // the number of tiles of rows in several parts, then of each (sequence, first row, first plane, parts)
  float* planes;    // of a part: PROMPT_ROWS rows of sums, then their bases and sums of weights
};
// slots: tiles of rows of a key head, without starts those of `step` tokens a sequence, else enough for any lengths (step 0)
struct PromptPlan {
  int64_t slots, shares, spare, workgroups, joins, header_bytes, bytes;
};
PromptPlan prompt_plan(int64_t tokens, int64_t step, int64_t group, int64_t kv_heads, int64_t d, int64_t page, int64_t sequences,
                       int64_t width, int64_t bytes);
void launch_cache_prompt(bool bf, int d, PromptCall c, const PromptPlan& p, void* workspace, hipStream_t stream);

}  // namespace krn

// Host side: what every entry point on a cache checks; false leaves a message.
struct CacheArguments {
  const char* name;
  int kind;
  const void *keys, *values, *starts, *lengths, *table;
  int64_t tokens, heads, kv_heads, d, pages, page, step, sequences, width;
};
bool krn_cache_arguments(const CacheArguments& a, krn::CacheView& cache, krn::SequencesView& sequences);
